// Token embedding: lookup with scaling, and the table's gradient by sorted tokens.
//
//   out[i]  = s * W[id_i]                          (id < 0: a zero row; id >= V: a NaN row + the error word)
//   dW[v]   = s * sum_{i : id_i = v, v != pad} dout[i]
//
// Used by the word lookup of SpeakerDecoder (model.py:1061) and the word-embedding gradient of BertEmbeddings
// (vilmodel.py:161-176 under autograd).
//
// Lookup: bound by HBM (ids + one row read and one written a token); no arithmetic to speak of. 131072 rows of 1024
// bf16 from a table of 50021: 75.6 us, 268 MB written and 102 MB of table read at least: 4.9 TB/s, a large copy's 5.2.
//
// The gradient is deterministic: the rows of one token are summed in fp32 in the order of their positions, so there
// is no float atomic, and every table row is written once, in its type. What it has to move is dout once and the table
// once; the sort that gives the order comes on top, so the sort keeps to few launches and small lists:
//   T <= 8192      one launch: each workgroup sorts its share of the ids into LDS and sums its rows.
//                  (1600 x 768 fp32 into 30522 rows: 20.8 us; the table's 94 MB alone take a fill kernel 13.6.)
//   more           token_sort_kernel, rows, join. A workgroup of the sort owns a share of the ids, reads every token
//                  (T x 8 B, an L2-resident list), counts its own per wave segment and those of the shares before it
//                  (its base), and writes its tokens' positions at their stable rank. No workgroup waits for another.
//   T >= 49152     (more for large tables: split_sort) token_count_kernel, token_place_kernel, rows, join: reading every
//                  id in every workgroup is what bounds the one-launch sort there.
//                  (131072 x 1024 bf16, a third of them padding, into 50021 rows: 7.0 + 16.1 us sort, 72.5 rows
//                  (174 MB read, 102 MB written: 3.8 TB/s; a large sum reads at 4.0), 7.9 join.)
#include "common.h"
#include "../../include/dasa_hip.h"

#include <algorithm>
#include <type_traits>

namespace {

constexpr int kMostSize = 1 << 30;    // of a table: index arithmetic adds tiles to it in 32 bits
constexpr int kMostSlices = 65535;    // of a row, in the grid's second dimension
constexpr unsigned kErrTokenId = 8;   // bit of the error word (ops._ERR_BITS)

// 16 bytes of a row. Rows of odd width or stride start anywhere, so the vector types are element-aligned (global loads
// and stores take any alignment). The last unit of a row that is no multiple of them ends at the row's end and repeats
// columns of the unit before it: no lane takes a partial load of its own, whose branch holds the wave's other loads up
// (gradient of 4099 x 257 fp32 into 1001 rows: 12.2 us against 15.8; lookup of 131072 x 1001 bf16: 98 against
// 111). NARROW: rows of less than one unit.
template <class T> struct Vec;
template <> struct Vec<float> {
  static constexpr int N = 4;
  typedef float type __attribute__((ext_vector_type(4), aligned(4)));
};
template <> struct Vec<__bf16> {
  static constexpr int N = 8;
  typedef __bf16 type __attribute__((ext_vector_type(8), aligned(2)));
};

template <bool NARROW, class T>
__device__ __forceinline__ typename Vec<T>::type load_unit(const T* p, int E) {
  typedef typename Vec<T>::type V;
  if constexpr (!NARROW) return *reinterpret_cast<const V*>(p);
  V v;
#pragma unroll
  for (int e = 0; e < Vec<T>::N; ++e) v[e] = e < E ? p[e] : (T)0.f;
  return v;
}

// columns from `skip` on
template <bool NARROW, class T>
__device__ __forceinline__ void store_unit(T* p, int E, int skip, typename Vec<T>::type v) {
  typedef typename Vec<T>::type V;
  if (!NARROW && skip == 0) {
    *reinterpret_cast<V*>(p) = v;
  } else {
#pragma unroll
    for (int e = 0; e < Vec<T>::N; ++e)
      if (e >= skip && (!NARROW || e < E)) p[e] = v[e];
  }
}

// ------------------------------------------------------------------ lookup
struct LookupArgs {
  const void* table; long ldt;
  const void* ids;
  void* out; long ldo;
  unsigned units;        // 16-B units per row
  unsigned total;        // rows * units (< 2^31)
  int V, E;
  float scale;
  unsigned* err;
};

// Thread = ILP units, the ILP table loads in flight together; consecutive threads take consecutive units, so narrow
// rows still fill a wave's loads.
template <class T, class I, int ILP, bool NARROW>
__global__ __launch_bounds__(256) void embedding_fwd_kernel(LookupArgs a) {
  constexpr int N = Vec<T>::N;
  typedef typename Vec<T>::type V;
  const unsigned u0 = blockIdx.x * (256u * ILP) + threadIdx.x;
  const I* ids = reinterpret_cast<const I*>(a.ids);
  unsigned row[ILP], c[ILP];
  long id[ILP];
#pragma unroll
  for (int k = 0; k < ILP; ++k) {
    const unsigned u = min(u0 + 256u * k, a.total - 1);
    row[k] = u / a.units;
    c[k] = NARROW ? 0 : min((u - row[k] * a.units) * N, (unsigned)(a.E - N));
    id[k] = (long)ids[row[k]];
  }
  V v[ILP];
#pragma unroll
  for (int k = 0; k < ILP; ++k) {
    const long r = (id[k] >= 0 && id[k] < a.V) ? id[k] : 0;
    v[k] = load_unit<NARROW>(reinterpret_cast<const T*>(a.table) + r * a.ldt + c[k], a.E);
  }
  __builtin_amdgcn_sched_barrier(0);     // all loads before the first value is needed (131072 x 1024: 91.5 us without)
#pragma unroll
  for (int k = 0; k < ILP; ++k) {
    if (u0 + 256u * k >= a.total) continue;
    V o;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      float x = (float)v[k][e] * a.scale;
      if (id[k] < 0) x = 0.f;
      if (id[k] >= a.V) x = __builtin_nanf("");
      o[e] = (T)x;
    }
    if (id[k] >= a.V && c[k] == 0 && a.err) atomicOr(a.err, kErrTokenId);
    store_unit<NARROW>(reinterpret_cast<T*>(a.out) + (long)row[k] * a.ldo + c[k], a.E, 0, o);
  }
}

template <class T, class I>
int launch_fwd(LookupArgs a, long rows, hipStream_t st) {
  a.units = (unsigned)((a.E + Vec<T>::N - 1) / Vec<T>::N);
  const long per = ((1L << 31) - 4096) / a.units;    // rows of one launch: 32-bit unit indexes
  const char* ids = reinterpret_cast<const char*>(a.ids);
  char* out = reinterpret_cast<char*>(a.out);
  for (long r = 0; r < rows; r += per) {
    const long n = rows - r < per ? rows - r : per;
    a.ids = ids + r * (long)sizeof(I);
    a.out = out + r * a.ldo * (long)sizeof(T);
    a.total = (unsigned)(n * a.units);
    // four units a thread once that still gives every CU eight waves
    if (a.E < Vec<T>::N)
      hipLaunchKernelGGL((embedding_fwd_kernel<T, I, 1, true>), dim3((a.total + 255) / 256), dim3(256), 0, st, a);
    else if (a.total >= 4u * 256u * 512u)
      hipLaunchKernelGGL((embedding_fwd_kernel<T, I, 4, false>), dim3((a.total + 1023) / 1024), dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL((embedding_fwd_kernel<T, I, 1, false>), dim3((a.total + 255) / 256), dim3(256), 0, st, a);
    DASA_CHECK_LAUNCH();
  }
  return 0;
}

// ------------------------------------------------------------------ tokens in sorted order
constexpr int kSortWaves = 16;
constexpr int kMaxBins = 896;        // vocabulary rows of one sort workgroup (its counters: 56 KB of LDS)
constexpr int kList = 1024;           // tokens of its share that a wave notes on the first pass (96 KB of LDS)

// Which workgroup sorts an id: G = 2^lg owners take the ids in turn (id u: owner u % G, its R bins u / G), since
// vocabularies are often in the order of their words' frequencies: owners of ranges would leave most tokens to the
// first (8192 such tokens x 1024 bf16, 50021 ids: 186 us with ranges, 32 in turn). The sorted order is by owner, then bin.
struct Owners {
  int lg, R;
  __device__ __forceinline__ unsigned place(unsigned u) const { return (u & ((1u << lg) - 1)) * R + (u >> lg); }
};

struct SortArgs {
  const void* ids;
  int T, V;
  Owners own;
  unsigned pad;   // the id without a gradient, or 2^32 - 1
  int* start;     // [G R + 1] first sorted index of every bin; the last: all tokens
  int* order;     // [T] positions in sorted order
};

// at least `least` owners (if V has as many), `bins` bins at most
inline Owners owners(int V, int least, int bins) {
  Owners o{0, 0};
  while ((1 << o.lg) < least && (1 << o.lg) < V) ++o.lg;
  while (((long)V + (1L << o.lg) - 1) >> o.lg > bins) ++o.lg;
  o.R = (int)(((long)V + (1L << o.lg) - 1) >> o.lg);
  return o;
}
inline int64_t bins_of(const Owners& o) { return ((int64_t)1 << o.lg) * o.R; }

// An owner's tokens among the ids
struct Mine {
  unsigned low, V, g, pad;
  int lg;
  __device__ __forceinline__ Mine(const SortArgs& a, unsigned owner)
      : low((1u << a.own.lg) - 1), V(a.V), g(owner), pad(a.pad), lg(a.own.lg) {}
  __device__ __forceinline__ bool counts(unsigned u) const { return u < V && u != pad; }
  __device__ __forceinline__ bool owns(unsigned u) const { return (u & low) == g && counts(u); }
  __device__ __forceinline__ bool below(unsigned u) const { return (u & low) < g && counts(u); }
  __device__ __forceinline__ int bin(unsigned u) const { return (int)(u >> lg); }
};

// An id as a 32-bit token: 2^32 - 1, which no vocabulary holds, for an id outside 32 bits.
__device__ __forceinline__ unsigned token(uint2 v) { return v.y == 0 ? v.x : ~0u; }
__device__ __forceinline__ unsigned token(unsigned v) { return v; }

// f(position, token) for the ids [t0, t1) of a wave, 64 at a time, U loads in flight (and U more of the next group);
// f is called by whole waves
template <class W, int U, class F>
__device__ __forceinline__ void each_token(const W* ids, int t0, int t1, int lane, F f) {
  int t = t0;
  const int last = t1 - 64 * U;
  if (t <= last) {
    W v[U], next[U];
#pragma unroll
    for (int k = 0; k < U; ++k) v[k] = ids[t + lane + 64 * k];
    for (; t <= last; t += 64 * U) {
      const W* p = ids + min(t + 64 * U, last) + lane;      // the next group, or the last again
#pragma unroll
      for (int k = 0; k < U; ++k) next[k] = p[64 * k];
#pragma unroll
      for (int k = 0; k < U; ++k) f(t + 64 * k + lane, token(v[k]));
#pragma unroll
      for (int k = 0; k < U; ++k) v[k] = next[k];
    }
  }
#pragma unroll 1
  for (; t < t1; t += 64) {
    const unsigned u = token(ids[min(t + lane, t1 - 1)]);
    f(t + lane, t + lane < t1 ? u : ~0u);
  }
}

// Write the positions of up to 64 tokens of the share (lanes with `in`, in lane order) at their ranks, one distinct
// id at a time: a frequent id is one turn.
template <class O>
__device__ __forceinline__ void place(int* cursor, O* order, int lane, bool in, int bin, int pos) {
  unsigned long long m = __builtin_amdgcn_ballot_w64(in);
  while (m) {
    const int b = __builtin_amdgcn_readlane(bin, __builtin_ctzll(m));
    const unsigned long long same = __builtin_amdgcn_ballot_w64(in && bin == b);
    const int c = cursor[b];
    if ((same >> lane) & 1) order[c + __popcll(same & ((1ull << lane) - 1))] = (O)pos;
    cursor[b] = c + __popcll(same);                  // every lane stores the same value
    m &= ~same;
  }
}

// f(position, bin, in, lanes with `in`) for the steps of a wave that hold a token of the owner
template <class W, class F>
__device__ __forceinline__ void each_of_mine(const W* ids, int t0, int t1, int lane, const Mine& own, F f) {
  each_token<W, 8>(ids, t0, t1, lane, [&](int pos, unsigned u) {
    const bool in = own.owns(u);
    const unsigned long long m = __builtin_amdgcn_ballot_w64(in);
    if (m) f(pos, own.bin(u), in, m);
  });
}

// hist[bin] += 1 for the lanes of m; PACK: two bins of 16 bits a word. Dense steps add their first id's lanes at once: a
// frequent id would be one address for most lanes.
template <bool PACK>
__device__ __forceinline__ void add_bins(int* hist, int bin, bool in, unsigned long long m) {
  auto add = [&](int b, int c) { atomicAdd(&hist[PACK ? b >> 1 : b], PACK ? c << (16 * (b & 1)) : c); };
  if (__popcll(m) > 8) {
    const int lane = threadIdx.x & 63, lead = __builtin_ctzll(m), b = __builtin_amdgcn_readlane(bin, lead);
    const unsigned long long same = __builtin_amdgcn_ballot_w64(in && bin == b);
    if (lane == lead) add(b, (int)__popcll(same));
    in = in && bin != b;
  }
  if (in) add(bin, 1);
}

// inclusive sum over the workgroup's threads; wsum holds one int a wave
__device__ __forceinline__ int block_scan(int v, int* wsum) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(v, o, 64);
    if (lane >= o) v += y;
  }
  if (lane == 63) wsum[w] = v;
  __syncthreads();
  for (int k = 0; k < w; ++k) v += wsum[k];
  return v;
}

// the wave's part of [t0, t1): multiples of 64 tokens
__device__ __forceinline__ void wave_part(int& t0, int& t1, int w) {
  const int part = (((t1 - t0 + kSortWaves - 1) / kSortWaves) + 63) & ~63;
  const int b = min(t0 + w * part, t1);
  t1 = min(b + part, t1);
  t0 = b;
}

// One launch: an owner's base is the number of tokens of the owners before it, which it counts on the way.
template <class W>
__global__ __launch_bounds__(64 * kSortWaves) void token_sort_kernel(SortArgs a) {
  const int R = a.own.R;
  extern __shared__ int lpos[];                    // [waves][kList] positions, [waves][R] counts (then write
  int* const hist = lpos + kSortWaves * kList;     // cursors), [waves][kList] bins
  unsigned short* const lbin = reinterpret_cast<unsigned short*>(hist + kSortWaves * R);
  __shared__ int below[kSortWaves], wsum[kSortWaves];
  const W* ids = reinterpret_cast<const W*>(a.ids);
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Mine own(a, blockIdx.x);
  for (int i = tid; i < kSortWaves * R; i += 64 * kSortWaves) hist[i] = 0;
  __syncthreads();
  int t0 = 0, t1 = a.T;
  wave_part(t0, t1, w);
  int* mine = hist + w * R;
  int nb = 0, found = 0;
  each_token<W, 8>(ids, t0, t1, lane, [&](int pos, unsigned u) {
    nb += __popcll(__builtin_amdgcn_ballot_w64(own.below(u)));
    const int bin = own.bin(u);
    const bool in = own.owns(u);
    const unsigned long long m = __builtin_amdgcn_ballot_w64(in);
    if (!m) return;
    const int at = found + __popcll(m & ((1ull << lane) - 1));
    if (in && at < kList) {
      lpos[w * kList + at] = pos;
      lbin[w * kList + at] = (unsigned short)bin;
    }
    found += __popcll(m);
    add_bins<false>(mine, bin, in, m);
  });
  if (lane == 0) below[w] = nb;
  __syncthreads();
  // exclusive scan over the bins (thread = bin), then over the waves of one bin
  int tot = 0;
  if (tid < R)
    for (int k = 0; k < kSortWaves; ++k) tot += hist[k * R + tid];
  int at = block_scan(tot, wsum) - tot;
  for (int k = 0; k < kSortWaves; ++k) at += below[k];
  if (tid < R) {
    const long p = (long)blockIdx.x * R + tid;
    a.start[p] = at;
    for (int k = 0; k < kSortWaves; ++k) {
      const int c = hist[k * R + tid];
      hist[k * R + tid] = at;
      at += c;
    }
    if (tid == R - 1 && blockIdx.x == gridDim.x - 1) a.start[p + 1] = at;
  }
  __syncthreads();
  if (found <= kList) {
    for (int i = 0; i < found; i += 64) {
      const int j = min(i + lane, found - 1);
      place(mine, a.order, lane, i + lane < found, lbin[w * kList + j], lpos[w * kList + j]);
    }
    return;
  }
  each_of_mine<W>(ids, t0, t1, lane, own, [&](int pos, int bin, bool in, unsigned long long) {
    place(mine, a.order, lane, in, bin, pos);      // many tokens: the ids again
  });
}

// Two launches for many tokens: workgroup = (owner of more bins, segment of the tokens). The first counts its bins;
// the second adds up what lies before each (owners and bins before it, and the same bin in earlier segments) and places
// its tokens.
constexpr int kWideBins = 1600;
constexpr int kSegmentTokens = 65024;              // of a segment at most: counts and offsets within it fit 16 bits

struct SplitArgs {
  int segments;
  int* counts;     // [segments][G R]
  int* totals;     // [G][segments]
};

__device__ __forceinline__ void segment_of(int T, int segments, int& t0, int& t1) {
  const int seg = (((T + segments - 1) / segments) + 63) & ~63;
  t0 = (int)min((long)blockIdx.y * seg, (long)T);
  t1 = (int)min((long)t0 + seg, (long)T);
}

template <class W>
__global__ __launch_bounds__(64 * kSortWaves) void token_count_kernel(SortArgs a, SplitArgs p) {
  __shared__ int hist[kWideBins];
  __shared__ int found[kSortWaves];
  const W* ids = reinterpret_cast<const W*>(a.ids);
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int R = a.own.R;
  for (int i = tid; i < R; i += 64 * kSortWaves) hist[i] = 0;
  __syncthreads();
  int t0, t1, total = 0;
  segment_of(a.T, p.segments, t0, t1);
  wave_part(t0, t1, w);
  each_of_mine<W>(ids, t0, t1, lane, Mine(a, blockIdx.x), [&](int, int bin, bool in, unsigned long long m) {
    total += __popcll(m);
    add_bins<false>(hist, bin, in, m);
  });
  if (lane == 0) found[w] = total;
  __syncthreads();
  int* counts = p.counts + ((long)blockIdx.y * gridDim.x + blockIdx.x) * R;
  for (int i = tid; i < R; i += 64 * kSortWaves) counts[i] = hist[i];
  if (tid == 0) {
    for (int k = 1; k < kSortWaves; ++k) total += found[k];
    p.totals[blockIdx.x * p.segments + blockIdx.y] = total;
  }
}

template <class W>
__global__ __launch_bounds__(64 * kSortWaves) void token_place_kernel(SortArgs a, SplitArgs p) {
  // a wave's counts, later its offset into a bin's run: two bins of 16 bits a word
  __shared__ int count[kSortWaves][kWideBins / 2];
  __shared__ int first[kWideBins];                // where a bin's tokens of this segment begin
  extern __shared__ int lpos[];                    // [waves][kList] positions, [waves][kList] bins
  unsigned short* const lbin = reinterpret_cast<unsigned short*>(lpos + kSortWaves * kList);
  __shared__ int wsum[kSortWaves], wbase[kSortWaves];
  const W* ids = reinterpret_cast<const W*>(a.ids);
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int R = a.own.R;
  const long all_bins = (long)gridDim.x * R;
  for (int i = tid; i < kSortWaves * kWideBins / 2; i += 64 * kSortWaves) count[0][i] = 0;
  // thread = two bins: all their tokens, those of the earlier segments, and the tokens of the owners before (asked for
  // before the scan, which hides them)
  constexpr int PER = (kWideBins + 64 * kSortWaves - 1) / (64 * kSortWaves);
  static_assert(PER == 2, "two bins share a counter word");
  int all[PER] = {0, 0}, before[PER] = {0, 0}, base = 0;
  for (int k = 0; k < p.segments; ++k) {
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      const int b = tid * PER + q;
      const int c = b < R ? p.counts[k * all_bins + (long)blockIdx.x * R + b] : 0;
      all[q] += c;
      before[q] += k < (int)blockIdx.y ? c : 0;
    }
  }
  for (int i = tid; i < (int)blockIdx.x * p.segments; i += 64 * kSortWaves) base += p.totals[i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) base += __shfl_xor(base, o, 64);
  if (lane == 0) wbase[w] = base;
  __syncthreads();
  int t0, t1, found = 0;
  segment_of(a.T, p.segments, t0, t1);
  wave_part(t0, t1, w);
  each_of_mine<W>(ids, t0, t1, lane, Mine(a, blockIdx.x), [&](int pos, int bin, bool in, unsigned long long m) {
    const int at = found + __popcll(m & ((1ull << lane) - 1));
    if (in && at < kList) {
      lpos[w * kList + at] = pos;
      lbin[w * kList + at] = (unsigned short)bin;
    }
    found += __popcll(m);
    add_bins<true>(count[w], bin, in, m);
  });
  int at = block_scan(all[0] + all[1], wsum) - all[0] - all[1];      // (its barrier also ends the counting)
  for (int k = 0; k < kSortWaves; ++k) at += wbase[k];
  if (tid * PER < R) {
    const int second = at + all[0];
    first[tid * PER] = at + before[0];
    first[tid * PER + 1] = second + before[1];
    if (blockIdx.y == 0) {
      int* start = a.start + (long)blockIdx.x * R + tid * PER;
      const bool two = tid * PER + 1 < R;
      start[0] = at;
      if (two) start[1] = second;
      if (tid * PER + PER >= R && blockIdx.x == gridDim.x - 1) start[two ? 2 : 1] = second + all[1];
    }
    int c[kSortWaves], run = 0;
#pragma unroll
    for (int k = 0; k < kSortWaves; ++k) c[k] = count[k][tid];
#pragma unroll
    for (int k = 0; k < kSortWaves; ++k) {
      count[k][tid] = run;
      run += c[k];
    }
  }
  __syncthreads();
  auto put = [&](bool in, int bin, int pos) {        // place(), with the packed cursors
    unsigned long long m = __builtin_amdgcn_ballot_w64(in);
    while (m) {
      const int b = __builtin_amdgcn_readlane(bin, __builtin_ctzll(m)), sh = 16 * (b & 1);
      const unsigned long long same = __builtin_amdgcn_ballot_w64(in && bin == b);
      const int word = count[w][b >> 1];
      if ((same >> lane) & 1) a.order[first[b] + ((word >> sh) & 0xffff) + __popcll(same & ((1ull << lane) - 1))] = pos;
      count[w][b >> 1] = word + (__popcll(same) << sh);                  // every lane stores the same value
      m &= ~same;
    }
  };
  if (found <= kList) {
    for (int i = 0; i < found; i += 64) {
      const int j = min(i + lane, found - 1);
      put(i + lane < found, lbin[w * kList + j], lpos[w * kList + j]);
    }
    return;
  }
  each_of_mine<W>(ids, t0, t1, lane, Mine(a, blockIdx.x), [&](int pos, int bin, bool in, unsigned long long) {
    put(in, bin, pos);
  });
}

// One launch against two (whole gradient of 8-wide bf16 rows, us; Zipf / uniform / one id). Two launches read every id
// twice in each of their G owners, one launch once in at least 256, and places a frequent id's tokens by one workgroup:
// two are taken from 1536 tokens an owner on, 49152 at least.
//     50021 ids, G 32:  49152 tokens 32 / 32 / 35, one launch 34 / 30 / 55;  131072: 43 / 45 / 56, 60 / 49 / 116
//    100000 ids, G 64:  49152 tokens 46 / 46 / 51, one launch 41 / 37 / 62;  131072: 61 / 63 / 80, 67 / 57 / 122
//    200000 ids, G 128: 131072 tokens 99 / 100 / 112, one launch 81 / 71 / 136;  524288: 202 / 217 / 268, 333 / 174 / 432
// Placing reads the counts of all segments in every segment, bins segments^2 in all: two launches up to 256 a token.
//     50021 ids: 16.8 M tokens (200 a token) 4.9 / 5.3 / 7.2 ms, one launch 9.9 / 6.0 / 13.3
//                33.6 M (399) 14.7 / 15.4 / 18.9, one launch 20.5 / 12.2 / 27.7
//    200000 ids: 4.2 M (202) 1.8 / 1.9 / 2.2, one launch 2.4 / 1.5 / 3.2;  16.8 M (800) 15.2 / 15.6 / 17.2, 10.0 / 6.0 / 13.3
constexpr long kOwnerTokens = 1536, kCountsToken = 256;

inline int sort_segments(int64_t T) { return (int)std::max<int64_t>(8, (T + kSegmentTokens - 1) / kSegmentTokens); }
inline bool split_sort(int64_t T, int V) {
  const Owners o = owners(V, 32, kWideBins);
  const int64_t s = sort_segments(T);
  return T >= kOwnerTokens * std::max(32L, 1L << o.lg) && bins_of(o) * s * s <= kCountsToken * T;
}

inline int64_t round16(int64_t n) { return (n + 15) & ~(int64_t)15; }

inline Owners sort_owners(int64_t T, int V) { return split_sort(T, V) ? owners(V, 32, kWideBins) : owners(V, 256, kMaxBins); }

template <class W>
int launch_sort(SortArgs a, void* split, hipStream_t st) {
  const dim3 block(64 * kSortWaves);
  const unsigned G = 1u << a.own.lg;
  if (split_sort(a.T, a.V)) {
    SplitArgs p;
    p.segments = sort_segments(a.T);
    p.counts = reinterpret_cast<int*>(split);
    p.totals = p.counts + p.segments * bins_of(a.own);
    const dim3 grid(G, p.segments);
    hipLaunchKernelGGL(token_count_kernel<W>, grid, block, 0, st, a, p);
    DASA_CHECK_LAUNCH();
    hipLaunchKernelGGL(token_place_kernel<W>, grid, block, (size_t)kSortWaves * kList * 6, st, a, p);
    DASA_CHECK_LAUNCH();
    return 0;
  }
  hipLaunchKernelGGL(token_sort_kernel<W>, dim3(G), block, (size_t)kSortWaves * (a.own.R * 4 + kList * 6), st, a);
  DASA_CHECK_LAUNCH();
  return 0;
}

// ------------------------------------------------------------------ gradient rows
// A lane's unit of a slice. Lanes past the row's end take its first unit and store nothing, so that whole waves reach
// every lane exchange.
struct Unit {
  int col, skip;   // its first column; the columns that the unit before it writes
  bool live;
};
template <class T>
__device__ __forceinline__ Unit unit_of(int unit, int E) {
  constexpr int N = Vec<T>::N;
  const int col = unit * N;
  if (col >= E) return Unit{0, 0, false};
  const int over = E < N ? 0 : max(col + N - E, 0);
  return Unit{col - over, over, true};
}

// A table row of up to kChunk tokens is summed by one wave per slice of 64 units. Longer (hot) rows are cut at the
// multiples of kChunk in the sorted order, so that a padding or stop word with a tenth of the tokens does not run on
// one wave: each chunk leaves the sum of its part of at most two hot rows (one that reaches into it, one that reaches
// out of it: a hot row is longer than a chunk), and a third launch adds a row's parts in chunk order. Where one row owns
// all chunks of a workgroup, the workgroup leaves one sum, in its first chunk's place (131072 x 1024 bf16 of one id: the
// join 145 -> 37 us; of Zipf ids 14.7 -> 9.1).
constexpr int kChunk = 32;
constexpr int kRowWaves = 4;
constexpr int kJoinWaves = 16;

struct BwdArgs {
  const void* dout; long ldd;
  const void* ids; int ids64;
  const int* start;
  const int* order;
  Owners own;
  float* parts;            // [chunks][2][ldp] sums of hot rows' parts
  long ldp;
  void* dtable; long ldt;
  int V, E;
  long bins;               // of the sort: start[bins] is the number of tokens
  unsigned chunk_blocks;   // blocks of the rows kernel that take chunks (first: they are the longer ones)
  long row0;               // the first table row of the others
  float scale;
  int accumulate;
};

// acc += the dout rows of n <= 64 tokens whose positions the lanes hold, tokens lane0 .. lane0 + n in order; K rows in
// flight at a time.
template <class T, bool NARROW, int K>
__device__ __forceinline__ int add_rows_by(float (&acc)[Vec<T>::N], const T* d, long ldd, int E, int pos, int lane0,
                                           int j, int n) {
  for (; j + K <= n; j += K) {
    typename Vec<T>::type x[K];
#pragma unroll
    for (int k = 0; k < K; ++k)
      x[k] = load_unit<NARROW>(d + (long)__builtin_amdgcn_readlane(pos, lane0 + j + k) * ldd, E);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < Vec<T>::N; ++e) acc[e] += (float)x[k][e];
  }
  return j;
}
template <class T, bool NARROW>
__device__ __forceinline__ void add_rows(float (&acc)[Vec<T>::N], const T* d, long ldd, int E, int pos, int lane0,
                                         int n) {
  int j = add_rows_by<T, NARROW, 8>(acc, d, ldd, E, pos, lane0, 0, n);
  j = add_rows_by<T, NARROW, 2>(acc, d, ldd, E, pos, lane0, j, n);
  add_rows_by<T, NARROW, 1>(acc, d, ldd, E, pos, lane0, j, n);
}

template <class T, bool NARROW>
__device__ __forceinline__ void write_row(const BwdArgs& a, long v, int col, int skip, const float (&acc)[Vec<T>::N]) {
  constexpr int N = Vec<T>::N;
  T* o = reinterpret_cast<T*>(a.dtable) + v * a.ldt + col;
  typename Vec<T>::type y;
  if (a.accumulate) y = load_unit<NARROW>(o, a.E);
#pragma unroll
  for (int e = 0; e < N; ++e) y[e] = (T)(a.accumulate ? (float)y[e] + acc[e] * a.scale : acc[e] * a.scale);
  store_unit<NARROW>(o, a.E, skip, y);
}

__device__ __forceinline__ long id_at(const BwdArgs& a, int pos) {
  return a.ids64 ? (long)reinterpret_cast<const int64_t*>(a.ids)[pos] : (long)reinterpret_cast<const int32_t*>(a.ids)[pos];
}

// One wave = (table row, slice) or (chunk, slice).
template <class T, bool NARROW>
__global__ __launch_bounds__(64 * kRowWaves) void embedding_bwd_rows_kernel(BwdArgs a) {
  constexpr int N = Vec<T>::N;
  __shared__ float sum[kRowWaves][64][N];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const auto [col, skip, live] = unit_of<T>(blockIdx.y * 64 + lane, a.E);
  const T* d = reinterpret_cast<const T*>(a.dout) + col;
  float acc[N];
#pragma unroll
  for (int e = 0; e < N; ++e) acc[e] = 0.f;
  if (blockIdx.x >= a.chunk_blocks) {
    const long v = a.row0 + (long)(blockIdx.x - a.chunk_blocks) * kRowWaves + w;
    if (v >= a.V) return;
    const int* at = a.start + a.own.place((unsigned)v);
    const int s = at[0], n = at[1] - s;
    if (n > kChunk || (a.accumulate && n == 0)) return;
    const int pos = lane < n ? a.order[s + lane] : 0;
    add_rows<T, NARROW>(acc, d, a.ldd, a.E, pos, 0, n);
    if (live) write_row<T, NARROW>(a, v, col, skip, acc);
    return;
  }
  const long c = (long)blockIdx.x * kRowWaves + w;
  const int j0 = (int)(c * kChunk), total = a.start[a.bins];
  if (j0 >= total) return;
  const int m = min(kChunk, total - j0);
  const int pos = a.order[j0 + min(lane, m - 1)];
  const int* at = a.start + a.own.place((unsigned)id_at(a, pos));
  const int rs = at[0], re = at[1];
  const bool hot = re - rs > kChunk;
  float* part = a.parts + c * 2 * a.ldp + col;
  const long b0 = (long)blockIdx.x * kRowWaves * kChunk;
  const bool whole = rs <= b0 && re >= b0 + kRowWaves * kChunk;
  if (__builtin_amdgcn_readlane((int)whole, 0)) {          // of the first token, then of every token of the workgroup
    add_rows<T, NARROW>(acc, d, a.ldd, a.E, pos, 0, m);
#pragma unroll
    for (int e = 0; e < N; ++e) sum[w][lane][e] = acc[e];
    __syncthreads();
    if (w != 0 || !live) return;
    for (int k = 1; k < kRowWaves; ++k)
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] += sum[k][lane][e];
#pragma unroll
    for (int e = 0; e < N; ++e) part[e] = acc[e];
    return;
  }
  // the row that owns the chunk's first token, then the row that owns its last
  const int ea = __builtin_amdgcn_readlane(hot ? min(re - j0, m) : 0, 0);
  if (ea > 0) {
    add_rows<T, NARROW>(acc, d, a.ldd, a.E, pos, 0, ea);
    if (live)
#pragma unroll
      for (int e = 0; e < N; ++e) part[e] = acc[e];
  }
  const int sb = __builtin_amdgcn_readlane(hot ? max(rs - j0, 0) : m, m - 1);
  if (sb > 0 && sb < m) {
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = 0.f;
    add_rows<T, NARROW>(acc, d, a.ldd, a.E, pos, sb, m - sb);
    if (live)
#pragma unroll
      for (int e = 0; e < N; ++e) part[a.ldp + e] = acc[e];
  }
}

// Where the sums of a hot row's sorted places [rs, re) are: chunks, whole workgroups of them, chunks.
struct Parts {
  int c0, first, head, b0, whole, n;
  __device__ __forceinline__ Parts(int rs, int re) {
    constexpr int B = kRowWaves * kChunk;
    c0 = rs / kChunk;
    first = rs > c0 * kChunk;                     // the slot of the first chunk: another row owns its first token
    const int last = (re - 1) / kChunk, lo = (int)(((long)rs + B - 1) / B), hi = re / B;
    b0 = lo;
    whole = max(hi - lo, 0);
    head = whole ? lo * kRowWaves - c0 : last + 1 - c0;
    n = whole ? head + whole + last + 1 - hi * kRowWaves : head;
  }
  __device__ __forceinline__ long place(int i) const {
    if (i < head) return (long)(c0 + i) * 2 + (i == 0 ? first : 0);
    if (i < head + whole) return (long)(b0 + i - head) * kRowWaves * 2;
    return (long)((b0 + whole) * kRowWaves + i - head - whole) * 2;
  }
};

// parts [k0, k1) of a hot row, added in order, eight in flight
template <class T>
__device__ __forceinline__ void add_parts(float (&acc)[Vec<T>::N], const BwdArgs& a, const Parts& p, int k0, int k1,
                                          int col) {
  constexpr int N = Vec<T>::N, K = 8;
  typedef float V __attribute__((ext_vector_type(N), aligned(4)));
  auto part = [&](int k) { return *reinterpret_cast<const V*>(a.parts + p.place(k) * a.ldp + col); };
  int k = k0;
  for (; k + K <= k1; k += K) {
    V x[K];
#pragma unroll
    for (int i = 0; i < K; ++i) x[i] = part(k + i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < K; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] += x[i][e];
  }
#pragma unroll 2
  for (; k < k1; ++k) {
    const V x = part(k);
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] += x[e];
  }
}

// One workgroup = (kJoinWaves chunks, slice). A hot row that starts in a chunk reaches past its end, so the chunk's
// last token names it. Rows of up to kJoinWaves parts: one wave each. The one longer row that may start in the group
// (it reaches past the group's end) takes the whole workgroup: the waves add runs of parts, joined in order.
template <class T, bool NARROW>
__global__ __launch_bounds__(64 * kJoinWaves) void embedding_bwd_join_kernel(BwdArgs a) {
  constexpr int N = Vec<T>::N;
  __shared__ float sum[kJoinWaves][64][N];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const auto [col, skip, live] = unit_of<T>(blockIdx.y * 64 + lane, a.E);
  const int total = a.start[a.bins];
  float acc[N];
#pragma unroll
  for (int e = 0; e < N; ++e) acc[e] = 0.f;
  const long c = (long)blockIdx.x * kJoinWaves + w;
  const long j0 = c * kChunk;
  if (j0 < total) {
    const long v = id_at(a, a.order[min(j0 + kChunk, (long)total) - 1]);
    const int* at = a.start + a.own.place((unsigned)v);
    const int rs = at[0], re = at[1];
    const Parts p(rs, re);
    if (re - rs > kChunk && rs >= j0 && p.n <= kJoinWaves) {
      add_parts<T>(acc, a, p, 0, p.n, col);
      if (live) write_row<T, NARROW>(a, v, col, skip, acc);
    }
  }
  const long g0 = (long)blockIdx.x * kJoinWaves * kChunk;
  if (g0 >= total) return;
  const long v = id_at(a, a.order[min(g0 + kJoinWaves * kChunk, (long)total) - 1]);
  const int* at = a.start + a.own.place((unsigned)v);
  const int rs = at[0], re = at[1];
  const Parts p(rs, re);
  const int n = p.n;
  if (rs < g0 || n <= kJoinWaves) return;
  const int per = (n + kJoinWaves - 1) / kJoinWaves, k0 = min(w * per, n), k1 = min(k0 + per, n);
#pragma unroll
  for (int e = 0; e < N; ++e) acc[e] = 0.f;
  add_parts<T>(acc, a, p, k0, k1, col);
#pragma unroll
  for (int e = 0; e < N; ++e) sum[w][lane][e] = acc[e];
  __syncthreads();
  if (w != 0 || !live) return;
  for (int k = 1; k < kJoinWaves; ++k)
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] += sum[k][lane][e];
  write_row<T, NARROW>(a, v, col, skip, acc);
}

// ------------------------------------------------------------------ few tokens: one launch
// Up to kFewTokens tokens: three launches become one, and no workspace is needed. Every workgroup reads all ids and
// sorts its own tokens into LDS as above (every token of a wave's segment fits its list); then it sums their rows
// itself, groups of lanes a row each.
//   Cold workgroups = (share of the ids, slice of LANES units): ids of up to kChunk tokens, a group each, and the rows
//   without tokens; then ids of up to kHot tokens, all groups together: each a run of them, joined in order.
//   Hot workgroups (first in the grid) = (larger share, slice of 16 units): the ids of more tokens (padding that no
//   padding_idx names), which they find with a count of their share first, all groups together. The narrow slices put
//   an id on several CUs: one CU reads a 1 KB row in 22 cycles, whatever is in flight (4096 x 768 fp32 of one id 139 us
//   without the hot workgroups, 30 with them; 4099 x 257, two fifths of them one id, 36 and 16; they cost about 1 us
//   where there is no such id).
constexpr int kFewTokens = 8192;
constexpr int kFewWaves = 8;
constexpr int kFewBins = 256;         // ids of a cold workgroup
constexpr int kHot = 256;             // 1024 x 768 fp32, two fifths one id: 18.7 us, 28.0 with 512 (4099 x 256: 10.8, 8.8)
constexpr int kHotBins = 4096;        // ids of a hot workgroup's share
constexpr int kHotLanes = 16;
static_assert(kFewTokens / (kHot + 1) <= kFewBins && kFewBins < 64 * kFewWaves, "a thread a bin");

inline int few_segment(int T) { return (((T + kFewWaves - 1) / kFewWaves) + 63) & ~63; }

struct FewArgs {
  Owners cold, hot;
  unsigned hot_blocks, hot_slices;
  int seg;
};

// acc = the sum of the c tokens from sorted place s on; the groups of a wave go on together to the longest of them
template <class T, bool NARROW, int LANES>
__device__ __forceinline__ void add_places(float (&acc)[Vec<T>::N], const T* d, const BwdArgs& a,
                                           const unsigned short* order, int s, int c) {
  constexpr int N = Vec<T>::N;
#pragma unroll
  for (int e = 0; e < N; ++e) acc[e] = 0.f;
  if constexpr (LANES == 64) {
    const int lane = threadIdx.x & 63;
    for (int k = 0; k < c; k += 64) {
      const int pos = order[s + min(k + lane, c - 1)];
      add_rows<T, NARROW>(acc, d, a.ldd, a.E, pos, 0, min(64, c - k));
    }
    return;
  }
  int m = c;
#pragma unroll
  for (int o = LANES; o < 64; o <<= 1) m = max(m, __shfl_xor(m, o, 64));
  m = __builtin_amdgcn_readfirstlane(m);
  auto turn = [&](int j, auto rows) {
    constexpr int K = decltype(rows)::value;
    typename Vec<T>::type x[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {            // a place past the group's last: some token of the workgroup, not added
      const int pos = order[j + k < c ? s + j + k : 0];
      x[k] = load_unit<NARROW>(d + (long)pos * a.ldd, a.E);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] += j + k < c ? (float)x[k][e] : 0.f;
  };
  int j = 0;
  for (; j + 4 <= m; j += 4) turn(j, std::integral_constant<int, 4>{});
  if (j + 2 <= m) { turn(j, std::integral_constant<int, 2>{}); j += 2; }
  if (j < m) turn(j, std::integral_constant<int, 1>{});
}

// The row of c tokens from sorted place s on, summed by the whole workgroup; sum: [groups][LANES][N] of LDS
template <class T, bool NARROW, int LANES>
__device__ __forceinline__ void long_row(const BwdArgs& a, const unsigned short* order, float* sum, int s, int c, long row,
                                         int slice) {
  constexpr int N = Vec<T>::N, GROUPS = 64 / LANES * kFewWaves;
  const int tid = threadIdx.x, group = tid / LANES;
  const auto [col, skip, live] = unit_of<T>(slice * LANES + (tid & (LANES - 1)), a.E);
  const T* d = reinterpret_cast<const T*>(a.dout) + col;
  const int per = (c + GROUPS - 1) / GROUPS, k0 = min(group * per, c), k1 = min(k0 + per, c);
  float acc[N];
  add_places<T, NARROW, LANES>(acc, d, a, order, s + k0, k1 - k0);
  float* mine = sum + (tid & (LANES - 1)) * N;
#pragma unroll
  for (int e = 0; e < N; ++e) mine[group * LANES * N + e] = acc[e];
  __syncthreads();
  if (tid < LANES && live) {
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = 0.f;
#pragma unroll 8
    for (int k = 0; k < GROUPS; ++k)
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] += mine[k * LANES * N + e];
    write_row<T, NARROW>(a, row, col, skip, acc);
  }
  __syncthreads();
}

template <class T, class W, bool NARROW, int LANES>
__global__ __launch_bounds__(64 * kFewWaves, 4) void embedding_bwd_few_kernel(BwdArgs a, SortArgs g, FewArgs f) {
  constexpr int N = Vec<T>::N;
  __shared__ int hist[kFewWaves][kFewBins], first[kFewBins + 1], wsum[kFewWaves], longs[kFewBins], nlong;
  __shared__ int share[kHotBins / 2];              // two bins of 16 bits a word: a count, then a hot id's number + 1
  // the sorted positions [waves seg]; the waves' tokens [waves][seg] as positions and bins, later the hot rows' sums
  extern __shared__ __attribute__((aligned(16))) unsigned short order[];
  const int seg = f.seg;
  unsigned short* const lpos = order + kFewWaves * seg;
  unsigned short* const lbin = lpos + kFewWaves * seg;
  float* const sum = reinterpret_cast<float*>(lpos);       // [groups][lanes][N]
  const W* ids = reinterpret_cast<const W*>(a.ids);
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int t0 = min(w * seg, g.T), t1 = min(t0 + seg, g.T);
  const bool is_hot = blockIdx.x < f.hot_blocks;
  const unsigned b = is_hot ? blockIdx.x : blockIdx.x - f.hot_blocks;
  g.own = is_hot ? f.hot : f.cold;
  const unsigned owner = is_hot ? b / f.hot_slices : b & ((1u << g.own.lg) - 1);
  const int slice = is_hot ? b % f.hot_slices : b >> g.own.lg;
  const Mine own(g, owner);
  int n = (int)((a.V + own.low - owner) >> own.lg);        // its ids: owner + bin G
  for (int i = tid; i < kFewWaves * kFewBins; i += 64 * kFewWaves) hist[0][i] = 0;
  if (tid == 0) nlong = 0;
  if (is_hot) {
    for (int i = tid; i < kHotBins / 2; i += 64 * kFewWaves) share[i] = 0;
    __syncthreads();
    each_token<W, 4>(ids, t0, t1, lane, [&](int, unsigned u) {
      const bool in = own.owns(u);
      const unsigned long long m = __builtin_amdgcn_ballot_w64(in);
      if (m) add_bins<true>(share, own.bin(u), in, m);
    });
    __syncthreads();
    for (int i = tid; i < kHotBins / 2; i += 64 * kFewWaves) {
      unsigned word = (unsigned)share[i], number = 0;
      if (word == 0) continue;
      for (int h = 0; h < 2; ++h)
        if (((word >> (16 * h)) & 0xffff) > (unsigned)kHot) {
          const int r = atomicAdd(&nlong, 1);
          longs[r] = 2 * i + h;
          number |= (unsigned)(r + 1) << (16 * h);
        }
      share[i] = (int)number;
    }
    __syncthreads();
    n = nlong;
    if (n == 0) return;
  }
  __syncthreads();
  int found = 0;
  auto note = [&](int pos, int bin, bool in, auto dense) {
    const unsigned long long m = __builtin_amdgcn_ballot_w64(in);
    if (!m) return;
    if (in) {
      const int at = found + __popcll(m & ((1ull << lane) - 1));
      lpos[w * seg + at] = (unsigned short)pos;
      lbin[w * seg + at] = (unsigned short)bin;
    }
    found += __popcll(m);
    if constexpr (decltype(dense)::value) add_bins<false>(hist[w], bin, in, m);
    else if (in) atomicAdd(&hist[w][bin], 1);
  };
  if (is_hot)
    each_token<W, 4>(ids, t0, t1, lane, [&](int pos, unsigned u) {
      const int bin = own.bin(u), number = own.owns(u) ? (share[bin >> 1] >> (16 * (bin & 1))) & 0xffff : 0;
      note(pos, number - 1, number > 0, std::true_type{});
    });
  else
    each_token<W, 4>(ids, t0, t1, lane,
                     [&](int pos, unsigned u) { note(pos, own.bin(u), own.owns(u), std::false_type{}); });
  __syncthreads();
  int tot = 0;
  if (tid < n)
    for (int k = 0; k < kFewWaves; ++k) tot += hist[k][tid];
  int at = block_scan(tot, wsum) - tot;
  if (tid <= n) first[tid] = at;              // thread n: the total
  if (tid < n) {
    for (int k = 0; k < kFewWaves; ++k) {
      const int c = hist[k][tid];
      hist[k][tid] = at;
      at += c;
    }
    if (!is_hot && tot > kChunk && tot <= kHot) longs[atomicAdd(&nlong, 1)] = tid;
  }
  __syncthreads();
  for (int i = 0; i < found; i += 64) {
    const int j = min(i + lane, found - 1);
    place(hist[w], order, lane, i + lane < found, lbin[w * seg + j], lpos[w * seg + j]);
  }
  __syncthreads();
  if (is_hot) {
    for (int r = 0; r < n; ++r)
      long_row<T, NARROW, kHotLanes>(a, order, sum, first[r], first[r + 1] - first[r], owner + ((long)longs[r] << own.lg),
                                     slice);
    return;
  }
  constexpr int PER = 64 / LANES;             // groups of a wave
  const auto [col, skip, live] = unit_of<T>(slice * LANES + (lane & (LANES - 1)), a.E);
  const T* d = reinterpret_cast<const T*>(a.dout) + col;
  float acc[N];
  for (int r0 = w * PER; r0 < n; r0 += kFewWaves * PER) {      // (a wave's groups end together)
    const int r = PER == 1 ? r0 : r0 + lane / LANES;
    const int s = first[PER == 1 ? r : min(r, n)], c = first[PER == 1 ? r + 1 : min(r + 1, n)] - s;
    add_places<T, NARROW, LANES>(acc, d, a, order, s, c > kChunk ? 0 : c);
    if (r < n && c <= kChunk && live && !(a.accumulate && c == 0))
      write_row<T, NARROW>(a, owner + ((long)r << own.lg), col, skip, acc);
  }
  const int h = nlong;
  for (int i = 0; i < h; ++i) {
    const int r = longs[i];
    long_row<T, NARROW, LANES>(a, order, sum, first[r], first[r + 1] - first[r], owner + ((long)r << own.lg), slice);
  }
}

template <class T, bool NARROW, int LANES>
int launch_few_as(const BwdArgs& a, const SortArgs& g, hipStream_t st) {
  const int units = (a.E + Vec<T>::N - 1) / Vec<T>::N, slices = (units + LANES - 1) / LANES;
  FewArgs f;
  f.cold = owners(a.V, 256, kFewBins);
  f.hot = owners(a.V, 4, kHotBins);
  f.hot_slices = (units + kHotLanes - 1) / kHotLanes;
  f.hot_blocks = g.T > kHot ? f.hot_slices << f.hot.lg : 0;
  f.seg = few_segment(g.T);
  const long blocks = f.hot_blocks + ((long)slices << f.cold.lg);
  if (!threads_fit(blocks, 64 * kFewWaves)) return (int)hipErrorInvalidValue;
  const size_t lists = (size_t)kFewWaves * f.seg * 4, sums = (size_t)kFewWaves * 64 * Vec<T>::N * 4;
  const size_t lds = (size_t)kFewWaves * f.seg * 2 + (lists > sums ? lists : sums);
  const dim3 grid((unsigned)blocks), block(64 * kFewWaves);
  if (a.ids64) hipLaunchKernelGGL((embedding_bwd_few_kernel<T, uint2, NARROW, LANES>), grid, block, lds, st, a, g, f);
  else hipLaunchKernelGGL((embedding_bwd_few_kernel<T, unsigned, NARROW, LANES>), grid, block, lds, st, a, g, f);
  DASA_CHECK_LAUNCH();
  return 0;
}

// Narrow rows share a wave's loads and stores: 1600 x 64 bf16 into 50021 rows 8.2 us with 16 lanes, 14.3 with 64; rows
// of 64 units keep whole waves (4096 x 256 fp32 into 1001 rows 5.2 us, 6.7 with 16 lanes and four slices).
template <class T>
int launch_few(const BwdArgs& a, const SortArgs& g, hipStream_t st) {
  constexpr int N = Vec<T>::N;
  if (a.E < N) return launch_few_as<T, true, 16>(a, g, st);
  if (a.E <= 16 * N) return launch_few_as<T, false, 16>(a, g, st);
  return launch_few_as<T, false, 64>(a, g, st);
}

inline long part_stride(int E, int bf16) {      // whole units, so a partial unit's sums stay inside
  const int n = bf16 ? 8 : 4;
  return (long)(E + n - 1) / n * n;
}

template <class T, bool NARROW>
int launch_rows_as(BwdArgs a, long tokens, hipStream_t st) {
  const int slices = (a.E + 64 * Vec<T>::N - 1) / (64 * Vec<T>::N);
  const long chunks = (tokens + kChunk - 1) / kChunk;
  a.chunk_blocks = (unsigned)((chunks + kRowWaves - 1) / kRowWaves);
  const long blocks = ((long)a.V + kRowWaves - 1) / kRowWaves, most = kMostThreads / (64 * kRowWaves);
  for (long b = 0; b < blocks;) {            // tables of more than 2^26 rows: several launches
    const long n = std::min(blocks - b, most - a.chunk_blocks);
    a.row0 = b * kRowWaves;
    const dim3 grid(a.chunk_blocks + (unsigned)n, slices);
    hipLaunchKernelGGL((embedding_bwd_rows_kernel<T, NARROW>), grid, dim3(64 * kRowWaves), 0, st, a);
    DASA_CHECK_LAUNCH();
    a.chunk_blocks = 0;
    b += n;
  }
  hipLaunchKernelGGL((embedding_bwd_join_kernel<T, NARROW>), dim3((unsigned)((chunks + kJoinWaves - 1) / kJoinWaves), slices),
                     dim3(64 * kJoinWaves), 0, st, a);
  DASA_CHECK_LAUNCH();
  return 0;
}
template <class T>
int launch_rows(const BwdArgs& a, long tokens, hipStream_t st) {
  return a.E < Vec<T>::N ? launch_rows_as<T, true>(a, tokens, st) : launch_rows_as<T, false>(a, tokens, st);
}

}  // namespace

extern "C" int dasa_embedding_fwd(const void* table, int64_t ldt, const void* ids, int32_t ids_bytes, int64_t T,
                                  int32_t V, int32_t E, float scale, int32_t bf16, void* out, int64_t ldo,
                                  uint32_t* err, void* stream) {
  if (T < 0 || V < 0 || E < 0 || V > kMostSize || E > kMostSize || (ids_bytes != 4 && ids_bytes != 8))
    return (int)hipErrorInvalidValue;
  if (T == 0 || E == 0) return 0;
  if (V == 0 || !table || !ids || !out || ldt < E || ldo < E) return (int)hipErrorInvalidValue;
  LookupArgs a{table, (long)ldt, ids, out, (long)ldo, 0, 0, V, E, scale, err};
  hipStream_t st = (hipStream_t)stream;
  if (bf16) return ids_bytes == 8 ? launch_fwd<__bf16, int64_t>(a, T, st) : launch_fwd<__bf16, int32_t>(a, T, st);
  return ids_bytes == 8 ? launch_fwd<float, int64_t>(a, T, st) : launch_fwd<float, int32_t>(a, T, st);
}

extern "C" int64_t dasa_embedding_bwd_workspace(int64_t T, int32_t V, int32_t E) {
  if (T <= kFewTokens || T >= (1LL << 31) || V < 0 || E < 0 || V > kMostSize || E > kMostSize) return 0;
  const int64_t chunks = (T + kChunk - 1) / kChunk;
  const Owners own = sort_owners(T, V);
  const int64_t split = split_sort(T, V) ? (bins_of(own) + (1 << own.lg)) * sort_segments(T) * 4 : 0;
  return round16((bins_of(own) + 1) * 4) + round16(T * 4) + chunks * 2 * part_stride(E, 1) * 4 + split;
}

extern "C" int dasa_embedding_bwd(const void* dout, int64_t ldd, const void* ids, int32_t ids_bytes, int64_t T,
                                  int32_t V, int32_t E, float scale, int32_t padding_idx, int32_t bf16, void* dtable,
                                  int64_t ldt, int32_t accumulate, void* ws, int64_t ws_bytes, void* stream) {
  if (T < 0 || T >= (1LL << 31) - 65536 || V < 0 || E < 0 || V > kMostSize || E > kMostSize ||
      (ids_bytes != 4 && ids_bytes != 8))
    return (int)hipErrorInvalidValue;
  if (V == 0 || E == 0) return 0;
  if (!dtable || ldt < E || ws_bytes < dasa_embedding_bwd_workspace(T, V, E) ||
      (T > kFewTokens && (!ws || !aligned16(ws))))
    return (int)hipErrorInvalidValue;
  if (T > 0 && (!ids || !dout || ldd < E)) return (int)hipErrorInvalidValue;
  if (T > kFewTokens && E > kMostSlices * 64 * Vec<float>::N) return (int)hipErrorInvalidValue;
  hipStream_t st = (hipStream_t)stream;
  BwdArgs ba{};
  ba.dout = dout; ba.ldd = (long)ldd; ba.ids = ids; ba.ids64 = ids_bytes == 8;
  ba.dtable = dtable; ba.ldt = (long)ldt; ba.V = V; ba.E = E; ba.scale = scale; ba.accumulate = accumulate;
  SortArgs sa{ids, (int)T, V, Owners{0, 0}, padding_idx < 0 ? ~0u : (unsigned)padding_idx, nullptr, nullptr};
  if (T <= kFewTokens) return bf16 ? launch_few<__bf16>(ba, sa, st) : launch_few<float>(ba, sa, st);
  ba.own = sa.own = sort_owners(T, V);
  ba.bins = (long)bins_of(ba.own);
  int* start = reinterpret_cast<int*>(ws);
  int* order = reinterpret_cast<int*>(reinterpret_cast<char*>(ws) + round16((bins_of(ba.own) + 1) * 4));
  ba.start = sa.start = start;
  ba.order = sa.order = order;
  ba.parts = reinterpret_cast<float*>(reinterpret_cast<char*>(order) + round16(T * 4));
  ba.ldp = part_stride(E, bf16);
  void* split = ba.parts + (T + kChunk - 1) / kChunk * 2 * part_stride(E, 1);
  const int rc = ids_bytes == 8 ? launch_sort<uint2>(sa, split, st) : launch_sort<unsigned>(sa, split, st);
  if (rc) return rc;
  return bf16 ? launch_rows<__bf16>(ba, T, st) : launch_rows<float>(ba, T, st);
}
