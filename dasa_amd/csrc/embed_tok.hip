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
//   T <= 8192      one launch: each workgroup sorts its vocabulary range into LDS and sums its rows.
//                  (1600 x 768 fp32 into 30522 rows: 20.2 us; the table's 94 MB alone take a fill kernel 13.6.)
//   T <  49152     token_sort_kernel, rows, join. Workgroup g of the sort owns the range [g R, (g + 1) R), reads every
//                  id (T x 8 B, an L2-resident list), counts its own tokens per wave segment and the tokens below the
//                  range (its base), and writes its tokens' positions at their stable rank. No workgroup waits for
//                  another.
//   above          token_count_kernel, token_place_kernel, rows, join: reading every id in every workgroup is what
//                  bounds the one-launch sort there.
//                  (131072 x 1024 bf16, a third of them padding, into 50021 rows: 7.1 + 16.2 us sort, 73.5 rows
//                  (174 MB read, 102 MB written: 3.8 TB/s; a large sum reads at 4.0), 8.6 join.)
#include "common.h"
#include "../../include/dasa_hip.h"

#include <algorithm>

namespace {

constexpr unsigned kErrTokenId = 8;   // bit of the error word (ops._ERR_BITS)

// 16 bytes of a row. Rows of odd width or stride start anywhere, so the vector types are element-aligned (global loads
// and stores take any alignment); the last unit of a row may be partial.
template <class T> struct Vec;
template <> struct Vec<float> {
  static constexpr int N = 4;
  typedef float type __attribute__((ext_vector_type(4), aligned(4)));
};
template <> struct Vec<__bf16> {
  static constexpr int N = 8;
  typedef __bf16 type __attribute__((ext_vector_type(8), aligned(2)));
};

template <class T>
__device__ __forceinline__ typename Vec<T>::type load_unit(const T* p, int left) {
  typedef typename Vec<T>::type V;
  if (left >= Vec<T>::N) return *reinterpret_cast<const V*>(p);
  V v;
#pragma unroll
  for (int e = 0; e < Vec<T>::N; ++e) v[e] = e < left ? p[e] : (T)0.f;
  return v;
}

template <class T>
__device__ __forceinline__ void store_unit(T* p, int left, typename Vec<T>::type v) {
  typedef typename Vec<T>::type V;
  if (left >= Vec<T>::N) {
    *reinterpret_cast<V*>(p) = v;
  } else {
#pragma unroll
    for (int e = 0; e < Vec<T>::N; ++e)
      if (e < left) p[e] = v[e];
  }
}

// ------------------------------------------------------------------ lookup
struct LookupArgs {
  const void* table; long ldt;
  const void* ids;
  void* out; long ldo;
  unsigned units;        // 16-B units per row, the last one partial if the width is odd
  unsigned total;        // rows * units (< 2^31)
  int V, E;
  float scale;
  unsigned* err;
};

// Thread = ILP units, the ILP table loads in flight together; consecutive threads take consecutive units, so narrow
// rows still fill a wave's loads.
template <class T, class I, int ILP>
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
    c[k] = (u - row[k] * a.units) * N;
    id[k] = (long)ids[row[k]];
  }
  V v[ILP];
#pragma unroll
  for (int k = 0; k < ILP; ++k) {
    const long r = (id[k] >= 0 && id[k] < a.V) ? id[k] : 0;
    v[k] = load_unit(reinterpret_cast<const T*>(a.table) + r * a.ldt + c[k], a.E - (int)c[k]);
  }
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
    store_unit(reinterpret_cast<T*>(a.out) + (long)row[k] * a.ldo + c[k], a.E - (int)c[k], o);
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
    if (a.total >= 4u * 256u * 512u)
      hipLaunchKernelGGL((embedding_fwd_kernel<T, I, 4>), dim3((a.total + 1023) / 1024), dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL((embedding_fwd_kernel<T, I, 1>), dim3((a.total + 255) / 256), dim3(256), 0, st, a);
    DASA_CHECK_LAUNCH();
  }
  return 0;
}

// ------------------------------------------------------------------ tokens in sorted order
constexpr int kSortWaves = 16;
constexpr int kMaxRange = 896;        // vocabulary rows of one sort workgroup (its counters: 56 KB of LDS)
constexpr int kList = 1024;           // tokens of its range that a wave notes on the first pass (96 KB of LDS)

struct SortArgs {
  const void* ids;
  int T, V, R;
  unsigned pad;   // the id without a gradient, or 2^32 - 1
  int* start;     // [V + 1] first sorted index of every token id
  int* order;     // [T] positions in sorted order
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

// Write the positions of up to 64 tokens of the range (lanes with `in`, in lane order) at their ranks, one distinct
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

// f(position, bin, in, lanes with `in`) for the steps of a wave that hold a token of the range [lo, lo + n)
template <class W, class F>
__device__ __forceinline__ void each_in_range(const W* ids, int t0, int t1, int lane, unsigned lo, unsigned n,
                                              unsigned pad, F f) {
  each_token<W, 8>(ids, t0, t1, lane, [&](int pos, unsigned u) {
    const unsigned bin = u - lo;
    const bool in = bin < n && u != pad;
    const unsigned long long m = __builtin_amdgcn_ballot_w64(in);
    if (m) f(pos, (int)bin, in, m);
  });
}

// hist[bin] += 1 for the lanes of m; PACK: two bins of 16 bits a word
template <bool PACK>
__device__ __forceinline__ void add_bins(int* hist, int bin, bool in, unsigned long long m) {
  auto add = [&](int b, int c) { atomicAdd(&hist[PACK ? b >> 1 : b], PACK ? c << (16 * (b & 1)) : c); };
  if (__popcll(m) <= 8) {
    if (in) add(bin, 1);
    return;
  }
  const int lane = threadIdx.x & 63;               // dense: a frequent id would be one address for most lanes
  while (m) {
    const int lead = __builtin_ctzll(m), b = __builtin_amdgcn_readlane(bin, lead);
    const unsigned long long same = __builtin_amdgcn_ballot_w64(in && bin == b);
    if (lane == lead) add(b, (int)__popcll(same));
    m &= ~same;
  }
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

// One launch: a workgroup's base is the number of tokens below its range, which it counts on the way.
template <class W>
__global__ __launch_bounds__(64 * kSortWaves) void token_sort_kernel(SortArgs a) {
  extern __shared__ int lpos[];                    // [waves][kList] positions, [waves][R] counts (then write
  int* const hist = lpos + kSortWaves * kList;     // cursors), [waves][kList] bins
  unsigned short* const lbin = reinterpret_cast<unsigned short*>(hist + kSortWaves * a.R);
  __shared__ int below[kSortWaves], wsum[kSortWaves];
  const W* ids = reinterpret_cast<const W*>(a.ids);
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const unsigned lo = blockIdx.x * (unsigned)a.R, n = min((unsigned)a.R, a.V - lo);
  for (int i = tid; i < kSortWaves * a.R; i += 64 * kSortWaves) hist[i] = 0;
  __syncthreads();
  int t0 = 0, t1 = a.T;
  wave_part(t0, t1, w);
  int* mine = hist + w * a.R;
  int nb = 0, found = 0;
  each_token<W, 8>(ids, t0, t1, lane, [&](int pos, unsigned u) {
    nb += __popcll(__builtin_amdgcn_ballot_w64(u < lo && u != a.pad));
    const unsigned bin = u - lo;
    const bool in = bin < n && u != a.pad;
    const unsigned long long m = __builtin_amdgcn_ballot_w64(in);
    if (!m) return;
    const int at = found + __popcll(m & ((1ull << lane) - 1));
    if (in && at < kList) {
      lpos[w * kList + at] = pos;
      lbin[w * kList + at] = (unsigned short)bin;
    }
    found += __popcll(m);
    add_bins<false>(mine, (int)bin, in, m);
  });
  if (lane == 0) below[w] = nb;
  __syncthreads();
  // exclusive scan over the range's ids (thread = id), then over the waves of one id
  int tot = 0;
  if (tid < (int)n)
    for (int k = 0; k < kSortWaves; ++k) tot += hist[k * a.R + tid];
  int at = block_scan(tot, wsum) - tot;
  for (int k = 0; k < kSortWaves; ++k) at += below[k];
  if (tid < (int)n) {
    a.start[lo + tid] = at;
    for (int k = 0; k < kSortWaves; ++k) {
      const int c = hist[k * a.R + tid];
      hist[k * a.R + tid] = at;
      at += c;
    }
    if ((int)lo + tid == a.V - 1) a.start[a.V] = at;
  }
  __syncthreads();
  if (found <= kList) {
    for (int i = 0; i < found; i += 64) {
      const int j = min(i + lane, found - 1);
      place(mine, a.order, lane, i + lane < found, lbin[w * kList + j], lpos[w * kList + j]);
    }
    return;
  }
  each_in_range<W>(ids, t0, t1, lane, lo, n, a.pad, [&](int pos, int bin, bool in, unsigned long long) {
    place(mine, a.order, lane, in, bin, pos);      // a hot range: its ids again
  });
}

// Two launches for many tokens: workgroup = (wider range, segment of the tokens). The first counts its ids; the second
// adds up what lies before each of its ids (smaller ids, and the same id in earlier segments) and places its tokens.
constexpr int kWideRange = 1600;
constexpr int kSegmentTokens = 65024;              // of a segment at most: counts and offsets within it fit 16 bits

struct SplitArgs {
  int ranges, segments;
  int* counts;     // [segments][V]
  int* totals;     // [ranges][segments]
};

__device__ __forceinline__ void segment_of(int T, int segments, int& t0, int& t1) {
  const int seg = (((T + segments - 1) / segments) + 63) & ~63;
  t0 = (int)min((long)blockIdx.y * seg, (long)T);
  t1 = (int)min((long)t0 + seg, (long)T);
}

template <class W>
__global__ __launch_bounds__(64 * kSortWaves) void token_count_kernel(SortArgs a, SplitArgs p) {
  __shared__ int hist[kWideRange];
  __shared__ int found[kSortWaves];
  const W* ids = reinterpret_cast<const W*>(a.ids);
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const unsigned lo = blockIdx.x * (unsigned)a.R, n = min((unsigned)a.R, a.V - lo);
  for (int i = tid; i < (int)n; i += 64 * kSortWaves) hist[i] = 0;
  __syncthreads();
  int t0, t1, total = 0;
  segment_of(a.T, p.segments, t0, t1);
  wave_part(t0, t1, w);
  each_in_range<W>(ids, t0, t1, lane, lo, n, a.pad, [&](int, int bin, bool in, unsigned long long m) {
    total += __popcll(m);
    add_bins<false>(hist, bin, in, m);
  });
  if (lane == 0) found[w] = total;
  __syncthreads();
  for (int i = tid; i < (int)n; i += 64 * kSortWaves) p.counts[(long)blockIdx.y * a.V + lo + i] = hist[i];
  if (tid == 0) {
    for (int k = 1; k < kSortWaves; ++k) total += found[k];
    p.totals[blockIdx.x * p.segments + blockIdx.y] = total;
  }
}

template <class W>
__global__ __launch_bounds__(64 * kSortWaves) void token_place_kernel(SortArgs a, SplitArgs p) {
  // a wave's counts, later its offset into an id's run: two ids of 16 bits a word
  __shared__ int count[kSortWaves][kWideRange / 2];
  __shared__ int first[kWideRange];                // where an id's tokens of this segment begin
  extern __shared__ int lpos[];                    // [waves][kList] positions, [waves][kList] bins
  unsigned short* const lbin = reinterpret_cast<unsigned short*>(lpos + kSortWaves * kList);
  __shared__ int wsum[kSortWaves], wbase[kSortWaves];
  const W* ids = reinterpret_cast<const W*>(a.ids);
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const unsigned lo = blockIdx.x * (unsigned)a.R, n = min((unsigned)a.R, a.V - lo);
  for (int i = tid; i < kSortWaves * kWideRange / 2; i += 64 * kSortWaves) count[0][i] = 0;
  // thread = two ids: all their tokens, those of the earlier segments, and the tokens of smaller ranges (asked for
  // before the scan, which hides them)
  constexpr int PER = (kWideRange + 64 * kSortWaves - 1) / (64 * kSortWaves);
  static_assert(PER == 2, "two ids share a counter word");
  int all[PER] = {0, 0}, before[PER] = {0, 0}, base = 0;
  for (int k = 0; k < p.segments; ++k) {
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      const int b = tid * PER + q;
      const int c = b < (int)n ? p.counts[(long)k * a.V + lo + b] : 0;
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
  each_in_range<W>(ids, t0, t1, lane, lo, n, a.pad, [&](int pos, int bin, bool in, unsigned long long m) {
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
  if (tid * PER < (int)n) {
    const int second = at + all[0];
    first[tid * PER] = at + before[0];
    first[tid * PER + 1] = second + before[1];
    if (blockIdx.y == 0) {
      const int v = (int)lo + tid * PER;
      a.start[v] = at;
      if (v == a.V - 1) a.start[a.V] = second;
      if (tid * PER + 1 < (int)n) {
        a.start[v + 1] = second;
        if (v + 1 == a.V - 1) a.start[a.V] = second + all[1];
      }
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
  each_in_range<W>(ids, t0, t1, lane, lo, n, a.pad, [&](int pos, int bin, bool in, unsigned long long) {
    put(in, bin, pos);
  });
}

inline int sort_ranges(int V) {
  const int need = (V + kWideRange - 1) / kWideRange, most = V < 32 ? V : 32;
  return need > most ? need : most;
}
// One launch against two, 50021 ids, Zipf / uniform / one id: 49152 tokens x 64 bf16, the whole gradient, 34.4 / 28.9 /
// 64.7 us against 33.6 / 30.8 / 45.3; 131072 tokens, the sort alone, 39 / 30 / 72 against 27.5 / 27.9 / 25.5. Above
// 4 M tokens the counts of the segments would outgrow the tokens.
constexpr long kManyTokens = 49152, kMostTokens = 4 << 20;

inline bool split_sort(int64_t T) { return T >= kManyTokens && T <= kMostTokens; }
inline int sort_segments(int64_t T) { return (int)std::max<int64_t>(8, (T + kSegmentTokens - 1) / kSegmentTokens); }

inline int64_t round16(int64_t n) { return (n + 15) & ~(int64_t)15; }

template <class W>
int launch_sort(SortArgs a, void* split, hipStream_t st) {
  const dim3 block(64 * kSortWaves);
  if (split_sort(a.T)) {
    SplitArgs p;
    p.segments = sort_segments(a.T);
    p.ranges = sort_ranges(a.V);
    a.R = (a.V + p.ranges - 1) / p.ranges;
    p.ranges = (a.V + a.R - 1) / a.R;
    p.counts = reinterpret_cast<int*>(split);
    p.totals = p.counts + (long)p.segments * a.V;
    const dim3 grid(p.ranges, p.segments);
    hipLaunchKernelGGL(token_count_kernel<W>, grid, block, 0, st, a, p);
    DASA_CHECK_LAUNCH();
    hipLaunchKernelGGL(token_place_kernel<W>, grid, block, (size_t)kSortWaves * kList * 6, st, a, p);
    DASA_CHECK_LAUNCH();
    return 0;
  }
  int G = (a.V + kMaxRange - 1) / kMaxRange;
  if (G < 256) G = a.V < 256 ? a.V : 256;
  a.R = (a.V + G - 1) / G;
  G = (a.V + a.R - 1) / a.R;
  hipLaunchKernelGGL(token_sort_kernel<W>, dim3(G), block, (size_t)kSortWaves * (a.R * 4 + kList * 6), st, a);
  DASA_CHECK_LAUNCH();
  return 0;
}

// ------------------------------------------------------------------ gradient rows
// A lane's unit of a slice. Lanes past the row's end take its first unit and store nothing, so that whole waves reach
// every lane exchange.
struct Unit {
  int col, left;
  bool live;
};
template <class T>
__device__ __forceinline__ Unit unit_of(int slice, int lane, int E) {
  const int col = (slice * 64 + lane) * Vec<T>::N;
  const bool live = col < E;
  return Unit{live ? col : 0, live ? E - col : E, live};
}

// A table row of up to kChunk tokens is summed by one wave per slice of 64 units. Longer (hot) rows are cut at the
// multiples of kChunk in the sorted order, so that a padding or stop word with a tenth of the tokens does not run on
// one wave: each chunk leaves the sum of its part of at most two hot rows (one that reaches into it, one that reaches
// out of it: a hot row is longer than a chunk), and a third launch adds a row's parts in chunk order.
constexpr int kChunk = 32;
constexpr int kJoinWaves = 16;

struct BwdArgs {
  const void* dout; long ldd;
  const void* ids; int ids64;
  const int* start;
  const int* order;
  float* parts;            // [chunks][2][ldp] sums of hot rows' parts
  long ldp;
  void* dtable; long ldt;
  int V, E;
  unsigned chunk_blocks;   // blocks of the rows kernel that take chunks (first: they are the longer ones)
  float scale;
  int accumulate;
};

// acc += the dout rows of n <= 64 tokens whose positions the lanes hold, tokens lane0 .. lane0 + n in order; K rows in
// flight at a time.
template <class T, int K>
__device__ __forceinline__ int add_rows_by(float (&acc)[Vec<T>::N], const T* d, long ldd, int left, int pos, int lane0,
                                           int j, int n) {
  for (; j + K <= n; j += K) {
    typename Vec<T>::type x[K];
#pragma unroll
    for (int k = 0; k < K; ++k)
      x[k] = load_unit(d + (long)__builtin_amdgcn_readlane(pos, lane0 + j + k) * ldd, left);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < Vec<T>::N; ++e) acc[e] += (float)x[k][e];
  }
  return j;
}
template <class T>
__device__ __forceinline__ void add_rows(float (&acc)[Vec<T>::N], const T* d, long ldd, int left, int pos, int lane0,
                                         int n) {
  int j = add_rows_by<T, 8>(acc, d, ldd, left, pos, lane0, 0, n);
  j = add_rows_by<T, 2>(acc, d, ldd, left, pos, lane0, j, n);
  add_rows_by<T, 1>(acc, d, ldd, left, pos, lane0, j, n);
}

template <class T>
__device__ __forceinline__ void write_row(const BwdArgs& a, long v, int col, int left, const float (&acc)[Vec<T>::N]) {
  constexpr int N = Vec<T>::N;
  T* o = reinterpret_cast<T*>(a.dtable) + v * a.ldt + col;
  typename Vec<T>::type y;
  if (a.accumulate) y = load_unit(o, left);
#pragma unroll
  for (int e = 0; e < N; ++e) y[e] = (T)(a.accumulate ? (float)y[e] + acc[e] * a.scale : acc[e] * a.scale);
  store_unit(o, left, y);
}

__device__ __forceinline__ long id_at(const BwdArgs& a, int pos) {
  return a.ids64 ? (long)reinterpret_cast<const int64_t*>(a.ids)[pos] : (long)reinterpret_cast<const int32_t*>(a.ids)[pos];
}

// One wave = (table row, slice) or (chunk, slice).
template <class T>
__global__ __launch_bounds__(256) void embedding_bwd_rows_kernel(BwdArgs a) {
  constexpr int N = Vec<T>::N;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const auto [col, left, live] = unit_of<T>(blockIdx.y, lane, a.E);
  const T* d = reinterpret_cast<const T*>(a.dout) + col;
  float acc[N];
#pragma unroll
  for (int e = 0; e < N; ++e) acc[e] = 0.f;
  if (blockIdx.x >= a.chunk_blocks) {
    const long v = (long)(blockIdx.x - a.chunk_blocks) * 4 + w;
    if (v >= a.V) return;
    const int s = a.start[v], n = a.start[v + 1] - s;
    if (n > kChunk || (a.accumulate && n == 0)) return;
    const int pos = lane < n ? a.order[s + lane] : 0;
    add_rows<T>(acc, d, a.ldd, left, pos, 0, n);
    if (live) write_row<T>(a, v, col, left, acc);
    return;
  }
  const long c = (long)blockIdx.x * 4 + w;
  const int j0 = (int)(c * kChunk), total = a.start[a.V];
  if (j0 >= total) return;
  const int m = min(kChunk, total - j0);
  const int pos = a.order[j0 + min(lane, m - 1)];
  const long id = id_at(a, pos);
  const int rs = a.start[id], re = a.start[id + 1];
  const bool hot = re - rs > kChunk;
  float* part = a.parts + c * 2 * a.ldp + col;
  // the row that owns the chunk's first token, then the row that owns its last
  const int ea = __builtin_amdgcn_readlane(hot ? min(re - j0, m) : 0, 0);
  if (ea > 0) {
    add_rows<T>(acc, d, a.ldd, left, pos, 0, ea);
    if (live)
#pragma unroll
      for (int e = 0; e < N; ++e) part[e] = acc[e];
  }
  const int sb = __builtin_amdgcn_readlane(hot ? max(rs - j0, 0) : m, m - 1);
  if (sb > 0 && sb < m) {
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = 0.f;
    add_rows<T>(acc, d, a.ldd, left, pos, sb, m - sb);
    if (live)
#pragma unroll
      for (int e = 0; e < N; ++e) part[a.ldp + e] = acc[e];
  }
}

// parts [k0, k1) of the hot row whose first part is slot `first` of chunk c, added in order
template <class T>
__device__ __forceinline__ void add_parts(float (&acc)[Vec<T>::N], const BwdArgs& a, long c, int first, int k0, int k1,
                                          int col) {
#pragma unroll 2
  for (int k = k0; k < k1; ++k) {
    const float* p = a.parts + ((c + k) * 2 + (k == 0 ? first : 0)) * a.ldp + col;
#pragma unroll
    for (int e = 0; e < Vec<T>::N; ++e) acc[e] += p[e];
  }
}

// One workgroup = (kJoinWaves chunks, slice). A hot row that starts in a chunk reaches past its end, so the chunk's
// last token names it. Rows of up to kJoinWaves parts: one wave each. The one longer row that may start in the group
// (it reaches past the group's end) takes the whole workgroup: the waves add runs of parts, joined in order.
template <class T>
__global__ __launch_bounds__(64 * kJoinWaves) void embedding_bwd_join_kernel(BwdArgs a) {
  constexpr int N = Vec<T>::N;
  __shared__ float sum[kJoinWaves][64][N];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const auto [col, left, live] = unit_of<T>(blockIdx.y, lane, a.E);
  const int total = a.start[a.V];
  float acc[N];
#pragma unroll
  for (int e = 0; e < N; ++e) acc[e] = 0.f;
  const long c = (long)blockIdx.x * kJoinWaves + w;
  const long j0 = c * kChunk;
  if (j0 < total) {
    const long v = id_at(a, a.order[min(j0 + kChunk, (long)total) - 1]);
    const int rs = a.start[v], re = a.start[v + 1], n = (re - 1) / kChunk - (int)c + 1;
    if (re - rs > kChunk && rs >= j0 && n <= kJoinWaves) {
      add_parts<T>(acc, a, c, rs > j0, 0, n, col);
      if (live) write_row<T>(a, v, col, left, acc);
    }
  }
  const long g0 = (long)blockIdx.x * kJoinWaves * kChunk;
  if (g0 >= total) return;
  const long v = id_at(a, a.order[min(g0 + kJoinWaves * kChunk, (long)total) - 1]);
  const int rs = a.start[v], re = a.start[v + 1];
  const int c0 = rs / kChunk, n = (re - 1) / kChunk - c0 + 1;
  if (rs < g0 || n <= kJoinWaves) return;
  const int per = (n + kJoinWaves - 1) / kJoinWaves, k0 = min(w * per, n), k1 = min(k0 + per, n);
#pragma unroll
  for (int e = 0; e < N; ++e) acc[e] = 0.f;
  add_parts<T>(acc, a, c0, rs > c0 * kChunk, k0, k1, col);
#pragma unroll
  for (int e = 0; e < N; ++e) sum[w][lane][e] = acc[e];
  __syncthreads();
  if (w != 0 || !live) return;
  for (int k = 1; k < kJoinWaves; ++k)
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] += sum[k][lane][e];
  write_row<T>(a, v, col, left, acc);
}

// ------------------------------------------------------------------ few tokens: one launch
// Up to kFewTokens tokens: workgroup = (vocabulary range, slice). It sorts its range's tokens into LDS as above (every
// token of a wave's segment fits its list) and sums its rows itself: ids of up to kChunk tokens a wave each, the others
// by all waves, whose parts are joined in order. Three launches become one, and no workspace is needed.
constexpr int kFewTokens = 8192;
constexpr int kFewWaves = 8;
constexpr int kFewRange = 256;

inline int few_segment(int T) { return (((T + kFewWaves - 1) / kFewWaves) + 63) & ~63; }

template <class T, class W>
__global__ __launch_bounds__(64 * kFewWaves, 4) void embedding_bwd_few_kernel(BwdArgs a, SortArgs g, int seg) {
  constexpr int N = Vec<T>::N;
  __shared__ int hist[kFewWaves][kFewRange], first[kFewRange + 1], wsum[kFewWaves], hot[kFewRange], nhot;
  // the sorted positions [waves seg]; the waves' tokens [waves][seg] as positions and ids, later the hot rows' sums
  extern __shared__ __attribute__((aligned(16))) unsigned short order[];
  unsigned short* const lpos = order + kFewWaves * seg;
  unsigned short* const lbin = lpos + kFewWaves * seg;
  float* const sum = reinterpret_cast<float*>(lpos);       // [waves][64][N]
  const W* ids = reinterpret_cast<const W*>(a.ids);
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const unsigned lo = blockIdx.x * (unsigned)g.R, n = min((unsigned)g.R, a.V - lo);
  const auto [col, left, live] = unit_of<T>(blockIdx.y, lane, a.E);
  for (int i = tid; i < kFewWaves * kFewRange; i += 64 * kFewWaves) hist[0][i] = 0;
  if (tid == 0) nhot = 0;
  __syncthreads();
  const int t0 = min(w * seg, g.T), t1 = min(t0 + seg, g.T);
  int found = 0;
  each_token<W, 4>(ids, t0, t1, lane, [&](int pos, unsigned u) {
    const unsigned bin = u - lo;
    const bool in = bin < n && u != g.pad;
    const unsigned long long m = __builtin_amdgcn_ballot_w64(in);
    if (!m) return;
    if (in) {
      const int at = found + __popcll(m & ((1ull << lane) - 1));
      lpos[w * seg + at] = (unsigned short)pos;
      lbin[w * seg + at] = (unsigned short)bin;
      atomicAdd(&hist[w][bin], 1);
    }
    found += __popcll(m);
  });
  __syncthreads();
  int tot = 0;
  if (tid < (int)n)
    for (int k = 0; k < kFewWaves; ++k) tot += hist[k][tid];
  int incl = tot;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(incl, o, 64);
    if (lane >= o) incl += y;
  }
  if (lane == 63) wsum[w] = incl;
  __syncthreads();
  int at = incl - tot;
  for (int k = 0; k < w; ++k) at += wsum[k];
  if (tid <= (int)n) first[tid] = at;              // thread n: the total
  if (tid < (int)n) {
    for (int k = 0; k < kFewWaves; ++k) {
      const int c = hist[k][tid];
      hist[k][tid] = at;
      at += c;
    }
    if (tot > kChunk) hot[atomicAdd(&nhot, 1)] = tid;
  }
  __syncthreads();
  for (int i = 0; i < found; i += 64) {
    const int j = min(i + lane, found - 1);
    place(hist[w], order, lane, i + lane < found, lbin[w * seg + j], lpos[w * seg + j]);
  }
  __syncthreads();
  const T* d = reinterpret_cast<const T*>(a.dout) + col;
  float acc[N];
  for (int r = w; r < (int)n; r += kFewWaves) {
    const int s = first[r], c = first[r + 1] - s;
    if (c > kChunk || (a.accumulate && c == 0)) continue;
    const int pos = lane < c ? order[s + lane] : 0;
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = 0.f;
    add_rows<T>(acc, d, a.ldd, left, pos, 0, c);
    if (live) write_row<T>(a, lo + r, col, left, acc);
  }
  const int h = nhot;
  if (h == 0) return;
  for (int i = 0; i < h; ++i) {
    const int r = hot[i], s = first[r], c = first[r + 1] - s;
    const int per = (c + kFewWaves - 1) / kFewWaves, k0 = min(w * per, c), k1 = min(k0 + per, c);
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = 0.f;
    for (int k = k0; k < k1; k += 64) {
      const int pos = order[s + min(k + lane, k1 - 1)];
      add_rows<T>(acc, d, a.ldd, left, pos, 0, min(64, k1 - k));
    }
#pragma unroll
    for (int e = 0; e < N; ++e) sum[(w * 64 + lane) * N + e] = acc[e];
    __syncthreads();
    if (w == 0 && live) {
      for (int k = 1; k < kFewWaves; ++k)
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] += sum[(k * 64 + lane) * N + e];
      write_row<T>(a, lo + r, col, left, acc);
    }
    __syncthreads();
  }
}

template <class T>
int launch_few(const BwdArgs& a, SortArgs g, hipStream_t st) {
  const int slices = (a.E + 64 * Vec<T>::N - 1) / (64 * Vec<T>::N);
  int G = (a.V + kFewRange - 1) / kFewRange;
  if (G < 256) G = a.V < 256 ? a.V : 256;
  g.R = (a.V + G - 1) / G;
  const int seg = few_segment(g.T);
  const size_t lists = (size_t)kFewWaves * seg * 4, sums = (size_t)kFewWaves * 64 * Vec<T>::N * 4;
  const size_t lds = (size_t)kFewWaves * seg * 2 + (lists > sums ? lists : sums);
  const dim3 grid((a.V + g.R - 1) / g.R, slices), block(64 * kFewWaves);
  if (a.ids64) hipLaunchKernelGGL((embedding_bwd_few_kernel<T, uint2>), grid, block, lds, st, a, g, seg);
  else hipLaunchKernelGGL((embedding_bwd_few_kernel<T, unsigned>), grid, block, lds, st, a, g, seg);
  DASA_CHECK_LAUNCH();
  return 0;
}

inline long part_stride(int E, int bf16) {      // whole units, so a partial unit's sums stay inside
  const int n = bf16 ? 8 : 4;
  return (long)(E + n - 1) / n * n;
}

template <class T>
int launch_rows(BwdArgs a, long tokens, hipStream_t st) {
  const int slices = (a.E + 64 * Vec<T>::N - 1) / (64 * Vec<T>::N);
  const long chunks = (tokens + kChunk - 1) / kChunk;
  a.chunk_blocks = (unsigned)((chunks + 3) / 4);
  const dim3 grid(a.chunk_blocks + (unsigned)((a.V + 3) / 4), slices);
  hipLaunchKernelGGL(embedding_bwd_rows_kernel<T>, grid, dim3(256), 0, st, a);
  DASA_CHECK_LAUNCH();
  hipLaunchKernelGGL(embedding_bwd_join_kernel<T>, dim3((unsigned)((chunks + kJoinWaves - 1) / kJoinWaves), slices),
                     dim3(64 * kJoinWaves), 0, st, a);
  DASA_CHECK_LAUNCH();
  return 0;
}


}  // namespace

extern "C" int dasa_embedding_fwd(const void* table, int64_t ldt, const void* ids, int32_t ids_bytes, int64_t T,
                                  int32_t V, int32_t E, float scale, int32_t bf16, void* out, int64_t ldo,
                                  uint32_t* err, void* stream) {
  if (T < 0 || V < 0 || E < 0 || (ids_bytes != 4 && ids_bytes != 8)) return (int)hipErrorInvalidValue;
  if (T == 0 || E == 0) return 0;
  if (V == 0 || !table || !ids || !out || ldt < E || ldo < E) return (int)hipErrorInvalidValue;
  LookupArgs a{table, (long)ldt, ids, out, (long)ldo, 0, 0, V, E, scale, err};
  hipStream_t st = (hipStream_t)stream;
  if (bf16) return ids_bytes == 8 ? launch_fwd<__bf16, int64_t>(a, T, st) : launch_fwd<__bf16, int32_t>(a, T, st);
  return ids_bytes == 8 ? launch_fwd<float, int64_t>(a, T, st) : launch_fwd<float, int32_t>(a, T, st);
}

extern "C" int64_t dasa_embedding_bwd_workspace(int64_t T, int32_t V, int32_t E) {
  if (T <= kFewTokens || T >= (1LL << 31) || V < 0 || E < 0) return 0;
  const int64_t chunks = (T + kChunk - 1) / kChunk;
  const int64_t split = split_sort(T) ? ((int64_t)V + sort_ranges(V)) * sort_segments(T) * 4 : 0;
  return round16(((int64_t)V + 1) * 4) + round16(T * 4) + chunks * 2 * part_stride(E, 1) * 4 + split;
}

extern "C" int dasa_embedding_bwd(const void* dout, int64_t ldd, const void* ids, int32_t ids_bytes, int64_t T,
                                  int32_t V, int32_t E, float scale, int32_t padding_idx, int32_t bf16, void* dtable,
                                  int64_t ldt, int32_t accumulate, void* ws, int64_t ws_bytes, void* stream) {
  if (T < 0 || T >= (1LL << 31) - 65536 || V < 0 || E < 0 || (ids_bytes != 4 && ids_bytes != 8))
    return (int)hipErrorInvalidValue;
  if (V == 0 || E == 0) return 0;
  if (!dtable || ldt < E || ws_bytes < dasa_embedding_bwd_workspace(T, V, E) || (T > kFewTokens && !ws))
    return (int)hipErrorInvalidValue;
  if (T > 0 && (!ids || !dout || ldd < E)) return (int)hipErrorInvalidValue;
  hipStream_t st = (hipStream_t)stream;
  BwdArgs ba{};
  ba.dout = dout; ba.ldd = (long)ldd; ba.ids = ids; ba.ids64 = ids_bytes == 8;
  ba.dtable = dtable; ba.ldt = (long)ldt; ba.V = V; ba.E = E; ba.scale = scale; ba.accumulate = accumulate;
  SortArgs sa{ids, (int)T, V, 0, padding_idx < 0 ? ~0u : (unsigned)padding_idx, nullptr, nullptr};
  if (T <= kFewTokens) return bf16 ? launch_few<__bf16>(ba, sa, st) : launch_few<float>(ba, sa, st);
  int* start = reinterpret_cast<int*>(ws);
  int* order = reinterpret_cast<int*>(reinterpret_cast<char*>(ws) + round16(((int64_t)V + 1) * 4));
  ba.start = sa.start = start;
  ba.order = sa.order = order;
  ba.parts = reinterpret_cast<float*>(reinterpret_cast<char*>(order) + round16(T * 4));
  ba.ldp = part_stride(E, bf16);
  void* split = ba.parts + (T + kChunk - 1) / kChunk * 2 * part_stride(E, 1);
  const int rc = ids_bytes == 8 ? launch_sort<uint2>(sa, split, st) : launch_sort<unsigned>(sa, split, st);
  if (rc) return rc;
  return bf16 ? launch_rows<__bf16>(ba, T, st) : launch_rows<float>(ba, T, st);
}
