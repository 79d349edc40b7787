// Token embedding: lookup with scaling, and the table's gradient by sorted tokens.
//
//   out[i]  = s * W[id_i]                          (id < 0: a zero row; id >= V: a NaN row + the error word)
//   dW[v]   = s * sum_{i : id_i = v, v != pad} dout[i]
//
// Used by the word lookup of SpeakerDecoder (model.py:1061) and the word-embedding gradient of BertEmbeddings
// (vilmodel.py:161-176 under autograd).
//
// The gradient is deterministic: the rows of one token are summed in fp32 in the order of their positions, so there
// is no float atomic. The order comes from a one-launch sort: workgroup g owns the vocabulary range
// [g R, (g + 1) R), reads every id (T x 8 B, an L2-resident list), counts its own range's tokens per wave
// segment and the tokens below the range (its base), and writes its tokens' positions at their stable rank. No
// workgroup waits for another.
#include "common.h"
#include "../../include/dasa_hip.h"

namespace {

constexpr unsigned kErrTokenId = 8;   // bit of the error word (ops._ERR_BITS)

template <class T> struct Vec;   // 16 bytes of a row
template <> struct Vec<float> {
  static constexpr int N = 4;
  typedef float type __attribute__((ext_vector_type(4)));
};
template <> struct Vec<__bf16> {
  static constexpr int N = 8;
  typedef __bf16 type __attribute__((ext_vector_type(8)));
};

// ------------------------------------------------------------------ lookup
struct LookupArgs {
  const void* table; long ldt;
  const void* ids;
  void* out; long ldo;
  unsigned units;        // VEC-element units per row
  unsigned total;        // rows * units (< 2^31)
  int V;
  float scale;
  unsigned* err;
};

// Thread = ILP units of VEC elements, the ILP table loads in flight together; consecutive threads take consecutive
// units, so narrow rows still fill a wave's loads.
template <class T, class I, int VEC, int ILP>
__global__ __launch_bounds__(256) void embedding_fwd_kernel(LookupArgs a) {
  typedef T V __attribute__((ext_vector_type(VEC)));
  const unsigned u0 = blockIdx.x * (256u * ILP) + threadIdx.x;
  const I* ids = reinterpret_cast<const I*>(a.ids);
  unsigned row[ILP], c[ILP];
  long id[ILP];
#pragma unroll
  for (int k = 0; k < ILP; ++k) {
    const unsigned u = min(u0 + 256u * k, a.total - 1);
    row[k] = u / a.units;
    c[k] = u - row[k] * a.units;
    id[k] = (long)ids[row[k]];
  }
  V v[ILP];
#pragma unroll
  for (int k = 0; k < ILP; ++k) {
    const long r = (id[k] >= 0 && id[k] < a.V) ? id[k] : 0;
    v[k] = *reinterpret_cast<const V*>(reinterpret_cast<const T*>(a.table) + r * a.ldt + (long)c[k] * VEC);
  }
#pragma unroll
  for (int k = 0; k < ILP; ++k) {
    if (u0 + 256u * k >= a.total) continue;
    V o;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float x = (float)v[k][e] * a.scale;
      if (id[k] < 0) x = 0.f;
      if (id[k] >= a.V) x = __builtin_nanf("");
      o[e] = (T)x;
    }
    if (id[k] >= a.V && c[k] == 0 && a.err) atomicOr(a.err, kErrTokenId);
    *reinterpret_cast<V*>(reinterpret_cast<T*>(a.out) + (long)row[k] * a.ldo + (long)c[k] * VEC) = o;
  }
}

template <class T, class I, int VEC>
int launch_fwd(LookupArgs a, long rows, int E, hipStream_t st) {
  a.units = (unsigned)(E / VEC);
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
      hipLaunchKernelGGL((embedding_fwd_kernel<T, I, VEC, 4>), dim3((a.total + 1023) / 1024), dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL((embedding_fwd_kernel<T, I, VEC, 1>), dim3((a.total + 255) / 256), dim3(256), 0, st, a);
    DASA_CHECK_LAUNCH();
  }
  return 0;
}

// ------------------------------------------------------------------ tokens in sorted order
constexpr int kSortWaves = 16;
constexpr int kMaxRange = 960;        // vocabulary rows of one sort workgroup (its counters: 60 KB of LDS)

struct SortArgs {
  const void* ids;
  int T, V, R, pad;
  int* start;     // [V + 1] first sorted index of every token id
  int* order;     // [T] positions in sorted order
};

// Every token of one 64-token step that lies in this workgroup's range, one distinct id at a time: f(bin, same-id
// lanes). Few tokens of a step lie in one range (64 / gridDim on average), and a frequent id is one turn.
template <class F>
__device__ __forceinline__ void each_bin(int bin, bool in, F f) {
  unsigned long long m = __ballot(in);
  while (m) {
    const int lead = __builtin_ctzll(m);
    const int b = __builtin_amdgcn_readlane(bin, lead);
    const unsigned long long same = __ballot(in && bin == b);
    f(b, same);
    m &= ~same;
  }
}

template <class I>
__global__ __launch_bounds__(64 * kSortWaves) void token_sort_kernel(SortArgs a) {
  extern __shared__ int hist[];                    // [waves][R] counts, then write cursors
  __shared__ int below[kSortWaves], wsum[kSortWaves];
  const I* ids = reinterpret_cast<const I*>(a.ids);
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int lo = blockIdx.x * a.R, n = min(a.R, a.V - lo);
  for (int i = tid; i < kSortWaves * a.R; i += 64 * kSortWaves) hist[i] = 0;
  __syncthreads();
  const int seg = (((a.T + kSortWaves - 1) / kSortWaves) + 63) & ~63;
  const int t0 = min(w * seg, a.T), t1 = min(t0 + seg, a.T);
  int* mine = hist + w * a.R;
  int nb = 0;
  constexpr int U = 8;                             // id loads in flight
  for (int t = t0; t < t1; t += 64 * U) {
    long v[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int i = t + 64 * k + lane;
      v[k] = i < t1 ? (long)ids[i] : -1;
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const bool ok = v[k] >= 0 && v[k] < a.V && v[k] != a.pad;
      nb += __popcll(__ballot(ok && v[k] < lo));
      const int bin = (int)v[k] - lo;
      each_bin(bin, ok && v[k] >= lo && v[k] < lo + n, [&](int b, unsigned long long same) {
        mine[b] += __popcll(same);                 // every lane stores the same value
      });
    }
  }
  if (lane == 0) below[w] = nb;
  __syncthreads();
  // exclusive scan over the range's ids (thread = id), then over the waves of one id
  int tot = 0;
  if (tid < n)
    for (int k = 0; k < kSortWaves; ++k) tot += hist[k * a.R + tid];
  int incl = tot;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(incl, o, 64);
    if (lane >= o) incl += y;
  }
  if (lane == 63) wsum[w] = incl;
  __syncthreads();
  int base = 0;
  for (int k = 0; k < kSortWaves; ++k) base += below[k] + (k < w ? wsum[k] : 0);
  int at = base + incl - tot;
  if (tid < n) {
    a.start[lo + tid] = at;
    for (int k = 0; k < kSortWaves; ++k) {
      const int c = hist[k * a.R + tid];
      hist[k * a.R + tid] = at;
      at += c;
    }
    if (lo + tid == a.V - 1) a.start[a.V] = at;
  }
  __syncthreads();
  for (int t = t0; t < t1; t += 64 * U) {
    long v[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int i = t + 64 * k + lane;
      v[k] = i < t1 ? (long)ids[i] : -1;
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const bool in = v[k] >= lo && v[k] < lo + n && v[k] != a.pad;
      const int bin = (int)v[k] - lo;
      each_bin(bin, in, [&](int b, unsigned long long same) {
        const int c = mine[b];
        if ((same >> lane) & 1) a.order[c + __popcll(same & ((1ull << lane) - 1))] = t + 64 * k + lane;
        mine[b] = c + __popcll(same);              // every lane stores the same value
      });
    }
  }
}

// ------------------------------------------------------------------ gradient rows
struct BwdArgs {
  const void* dout; long ldd;
  const int* start;
  const int* order;
  void* dtable; long ldt;
  int V, E;
  float scale;
  int accumulate;
};

// One wave = one table row x one slice of 64 VEC columns.
template <class T, int VEC>
__global__ __launch_bounds__(256) void embedding_bwd_rows_kernel(BwdArgs a) {
  typedef T V __attribute__((ext_vector_type(VEC)));
  const int lane = threadIdx.x & 63;
  const long v = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (v >= a.V) return;
  const int col = (blockIdx.y * 64 + lane) * VEC;
  const int s = a.start[v], e = a.start[v + 1];
  if (a.accumulate && s == e) return;
  if (col >= a.E) return;
  float acc[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
  const T* d = reinterpret_cast<const T*>(a.dout) + col;
  for (int j = s; j < e; ++j) {
    const V x = *reinterpret_cast<const V*>(d + (long)a.order[j] * a.ldd);
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] += (float)x[i];
  }
  V* o = reinterpret_cast<V*>(reinterpret_cast<T*>(a.dtable) + v * a.ldt + col);
  V y;
  if (a.accumulate) {
    const V old = *o;
#pragma unroll
    for (int i = 0; i < VEC; ++i) y[i] = (T)((float)old[i] + acc[i] * a.scale);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) y[i] = (T)(acc[i] * a.scale);
  }
  *o = y;
}

template <class T, int VEC>
int launch_rows(const BwdArgs& a, hipStream_t st) {
  const int slices = (a.E + 64 * VEC - 1) / (64 * VEC);
  hipLaunchKernelGGL((embedding_bwd_rows_kernel<T, VEC>), dim3((a.V + 3) / 4, slices), dim3(256), 0, st, a);
  DASA_CHECK_LAUNCH();
  return 0;
}

inline bool aligned16(const void* p, long ld, int elem) { return (((uintptr_t)p | (uintptr_t)(ld * elem)) & 15) == 0; }

template <class T>
int fwd_types(const LookupArgs& a, int64_t rows, int E, bool i64, hipStream_t st) {
  constexpr int N = Vec<T>::N;
  const bool vec = E % N == 0 && aligned16(a.table, a.ldt, sizeof(T)) && aligned16(a.out, a.ldo, sizeof(T));
  if (vec) return i64 ? launch_fwd<T, int64_t, N>(a, rows, E, st) : launch_fwd<T, int32_t, N>(a, rows, E, st);
  return i64 ? launch_fwd<T, int64_t, 1>(a, rows, E, st) : launch_fwd<T, int32_t, 1>(a, rows, E, st);
}

template <class T>
int bwd_types(const BwdArgs& a, hipStream_t st) {
  constexpr int N = Vec<T>::N;
  const bool vec = a.E % N == 0 && aligned16(a.dout, a.ldd, sizeof(T)) && aligned16(a.dtable, a.ldt, sizeof(T));
  return vec ? launch_rows<T, N>(a, st) : launch_rows<T, 1>(a, st);
}

inline int64_t round16(int64_t n) { return (n + 15) & ~(int64_t)15; }

}  // namespace

extern "C" int dasa_embedding_fwd(const void* table, int64_t ldt, const void* ids, int32_t ids_bytes, int64_t T,
                                  int32_t V, int32_t E, float scale, int32_t bf16, void* out, int64_t ldo,
                                  uint32_t* err, void* stream) {
  if (T < 0 || V < 0 || E < 0 || (ids_bytes != 4 && ids_bytes != 8)) return (int)hipErrorInvalidValue;
  if (T == 0 || E == 0) return 0;
  if (V == 0 || !table || !ids || !out || ldt < E || ldo < E) return (int)hipErrorInvalidValue;
  LookupArgs a{table, (long)ldt, ids, out, (long)ldo, 0, 0, V, scale, err};
  return bf16 ? fwd_types<__bf16>(a, T, E, ids_bytes == 8, (hipStream_t)stream)
              : fwd_types<float>(a, T, E, ids_bytes == 8, (hipStream_t)stream);
}

extern "C" int64_t dasa_embedding_bwd_workspace(int64_t T, int32_t V, int32_t E) {
  if (T < 0 || T >= (1LL << 31) || V < 0 || E < 0) return 0;
  return round16(((int64_t)V + 1) * 4) + round16(T * 4);
}

extern "C" int dasa_embedding_bwd(const void* dout, int64_t ldd, const void* ids, int32_t ids_bytes, int64_t T,
                                  int32_t V, int32_t E, float scale, int32_t padding_idx, int32_t bf16, void* dtable,
                                  int64_t ldt, int32_t accumulate, void* ws, int64_t ws_bytes, void* stream) {
  if (T < 0 || T >= (1LL << 31) - 65536 || V < 0 || E < 0 || (ids_bytes != 4 && ids_bytes != 8))
    return (int)hipErrorInvalidValue;
  if (V == 0 || E == 0) return 0;
  if (!dtable || ldt < E || !ws || ws_bytes < dasa_embedding_bwd_workspace(T, V, E)) return (int)hipErrorInvalidValue;
  if (T > 0 && (!ids || !dout || ldd < E)) return (int)hipErrorInvalidValue;
  int* start = reinterpret_cast<int*>(ws);
  int* order = reinterpret_cast<int*>(reinterpret_cast<char*>(ws) + round16(((int64_t)V + 1) * 4));
  hipStream_t st = (hipStream_t)stream;
  int G = (V + kMaxRange - 1) / kMaxRange;
  if (G < 256) G = V < 256 ? V : 256;
  const int R = (V + G - 1) / G;
  G = (V + R - 1) / R;
  SortArgs sa{ids, (int)T, V, R, padding_idx, start, order};
  const size_t lds = (size_t)kSortWaves * R * sizeof(int);
  if (ids_bytes == 8)
    hipLaunchKernelGGL(token_sort_kernel<int64_t>, dim3(G), dim3(64 * kSortWaves), lds, st, sa);
  else
    hipLaunchKernelGGL(token_sort_kernel<int32_t>, dim3(G), dim3(64 * kSortWaves), lds, st, sa);
  DASA_CHECK_LAUNCH();
  BwdArgs ba{dout, (long)ldd, start, order, dtable, (long)ldt, V, E, scale, accumulate};
  return bf16 ? bwd_types<__bf16>(ba, st) : bwd_types<float>(ba, st);
}
