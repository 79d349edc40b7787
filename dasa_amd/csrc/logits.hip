// Rules on the logits of one decoding step, before a token is chosen (Speaker.infer_batch, speaker.py:319-323):
// penalties for tokens the row has already emitted, biases, a grammar mask, and the greedy choice.
//
//   c = number of times v occurs in history[b, :len_b]
//   x = logit[b, v];  if c > 0:  x = (x > 0 ? x / r : x r) - f c - p
//   x = x + bias[v];  not allowed: x = -inf;  y = round(x);  choice_b = lowest index of the largest y (NaN largest)
//
// Every product, quotient and sum is one rounded fp32 operation in this order (no contraction), so the result does
// not depend on how a row is split over workgroups.
//
// A workgroup owns a slice of one row, 4 ITER tokens a thread: it asks for its logits, biases and mask words first,
// counts the row's history into LDS while they come (integer atomics: the counts do not depend on their order), and
// writes the slice. With one slice a row, the workgroup also makes the choice; else each slice leaves its best key
// and a second launch takes the best of them, one wave a row.
//
// Bound by latency at a decoding step's sizes: 20 x 992 fp32 with 120 ids a row 4.3 us, where an empty kernel takes 2.4.
// 64 x 30522 fp32, 1024 ids: 8.9 + 2.5 us (17 MB: 3.2 at a copy's rate); 16 x 128255 bf16 with a bias a row, 16384 ids:
// 13.8 + 3.0 (18 MB: 3.5), 2.4 of it the history that every slice reads.
#include "common.h"
#include "../../include/dasa_hip.h"

namespace {

// 16 B of a row whose start need not be aligned (an odd vocabulary): element-aligned vector accesses
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 b4u __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned u32u __attribute__((aligned(1)));
template <class T> struct V4;
template <> struct V4<float> { typedef f4u type; };
template <> struct V4<__bf16> { typedef b4u type; };

struct RulesArgs {
  const void* logits; long ld;
  void* out; long ldo;
  const void* history; long ldh; int L;
  const int* lengths;          // [B] or null: all L
  const float* rep; const float* pres; const float* freq;   // [B] or null: the numbers below
  float rep0, pres0, freq0;
  const float* bias; long ldb;         // row stride 0: shared
  const unsigned* bits; long ldbits;   // allowed tokens, one bit each; row stride 0: shared
  const unsigned char* bytes; long ldbytes;
  int64_t* choice;
  unsigned long long* best;    // [B][slices] keys when a row has several slices
  int V, slices;
};

// Order-preserving key of a value and its index: larger value first, NaN above all, -0 = +0, then the lower index.
__device__ __forceinline__ unsigned long long choice_key(float y, int v) {
  unsigned u;
  if (y != y) {
    u = 0xffffffffu;
  } else {
    u = __float_as_uint(y + 0.f);       // -0 -> +0
    u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  }
  return ((unsigned long long)u << 32) | (unsigned)~v;
}

__device__ __forceinline__ unsigned long long wave_best(unsigned long long k) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const unsigned long long y = __shfl_xor(k, o, 64);
    k = y > k ? y : k;
  }
  return k;
}

template <class T, class I, int ITER>
__global__ __launch_bounds__(1024) void logit_rules_kernel(RulesArgs a) {
#pragma clang fp contract(off)
  typedef typename V4<T>::type V;
  extern __shared__ int count[];        // [4 ITER threads] when there is a history
  __shared__ unsigned long long wbest[16];
  const int tid = threadIdx.x, lane = tid & 63, nt = blockDim.x, slice = 4 * ITER * nt;
  const int b = blockIdx.y, lo = blockIdx.x * slice, n = min(slice, a.V - lo);
  const T* x0 = reinterpret_cast<const T*>(a.logits) + (long)b * a.ld + lo;
  T* y0 = reinterpret_cast<T*>(a.out) + (long)b * a.ldo + lo;
  const float* bias = a.bias ? a.bias + (long)b * a.ldb + lo : nullptr;
  const unsigned* bits = a.bits ? a.bits + (long)b * a.ldbits + (lo >> 5) : nullptr;     // lo % 32 == 0
  const unsigned char* bytes = a.bytes ? a.bytes + (long)b * a.ldbytes + lo : nullptr;
  V x[ITER];
  f4u add[ITER];
  unsigned open[ITER];                  // the four tokens' bits
#pragma unroll
  for (int k = 0; k < ITER; ++k) {
    const int i = 4 * (tid + k * nt);
    add[k] = f4u{0.f, 0.f, 0.f, 0.f};
    open[k] = 15u;
    if (i + 4 <= n) {
      x[k] = *reinterpret_cast<const V*>(x0 + i);
      if (bias) add[k] = *reinterpret_cast<const f4u*>(bias + i);
      if (bits) open[k] = bits[i >> 5] >> (i & 31);
      if (bytes) open[k] = *reinterpret_cast<const u32u*>(bytes + i);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[k][e] = i + e < n ? x0[i + e] : (T)0.f;
      if (bias)
#pragma unroll
        for (int e = 0; e < 4; ++e) add[k][e] = i + e < n ? bias[i + e] : 0.f;
      if (bits && i < n) open[k] = bits[i >> 5] >> (i & 31);
      if (bytes) {
        open[k] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) open[k] |= i + e < n ? (unsigned)bytes[i + e] << (8 * e) : 0u;
      }
    }
  }
  const float r = a.rep ? a.rep[b] : a.rep0, p = a.pres ? a.pres[b] : a.pres0, f = a.freq ? a.freq[b] : a.freq0;
  if (a.history) {
    const I* h = reinterpret_cast<const I*>(a.history) + (long)b * a.ldh;
    const int len = a.lengths ? min(max(a.lengths[b], 0), a.L) : a.L;
    constexpr int U = 8;                // ids in flight
    long id[U];
    auto ask = [&](int at) {
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int i = at + k * nt + tid;
        id[k] = i < len ? (long)h[i] - lo : -1;
      }
    };
    ask(0);
#pragma unroll
    for (int k = 0; k < ITER; ++k) *reinterpret_cast<int4*>(count + 4 * (tid + k * nt)) = make_int4(0, 0, 0, 0);
    __syncthreads();
    for (int at = 0; at < len;) {
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (id[k] >= 0 && id[k] < n) atomicAdd(&count[id[k]], 1);
      at += U * nt;
      if (at < len) ask(at);
    }
    __syncthreads();
  }
  unsigned long long best = 0;
#pragma unroll
  for (int k = 0; k < ITER; ++k) {
    const int i = 4 * (tid + k * nt);
    int4 c = make_int4(0, 0, 0, 0);
    if (a.history) c = *reinterpret_cast<const int4*>(count + i);
    const int cc[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float v = (float)x[k][e];
      if (cc[e] > 0) {
        v = v > 0.f ? v / r : v * r;
        v = v - f * (float)cc[e];
        v = v - p;
      }
      if (bias) v = v + add[k][e];
      const bool o = bytes ? (open[k] >> (8 * e)) & 255u : (open[k] >> e) & 1u;
      x[k][e] = (T)(o ? v : -INFINITY);
    }
    if (i + 4 <= n) {
      *reinterpret_cast<V*>(y0 + i) = x[k];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < n) y0[i + e] = x[k][e];
    }
    if (a.choice)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned long long key = i + e < n ? choice_key((float)x[k][e], lo + i + e) : 0;
        best = key > best ? key : best;
      }
  }
  if (!a.choice) return;
  best = wave_best(best);
  if (lane == 0) wbest[tid >> 6] = best;
  __syncthreads();
  if (tid >= 64) return;
  best = wave_best(lane < nt / 64 ? wbest[lane] : 0);
  if (tid != 0) return;
  if (a.slices == 1) a.choice[b] = (int64_t)(unsigned)~(unsigned)best;
  else a.best[(long)b * a.slices + blockIdx.x] = best;
}

// The best of one row's slices: one wave a row.
__global__ __launch_bounds__(64) void logit_choice_kernel(const unsigned long long* best, int64_t* choice, int slices) {
  unsigned long long k = 0;
  for (int i = threadIdx.x; i < slices; i += 64) {
    const unsigned long long y = best[(long)blockIdx.x * slices + i];
    k = y > k ? y : k;
  }
  k = wave_best(k);
  if (threadIdx.x == 0) choice[blockIdx.x] = (int64_t)(unsigned)~(unsigned)k;
}

constexpr int kMostSize = 1 << 30;    // of V and L: index arithmetic adds slices to them in 32 bits

struct Shape {
  int iter, threads, slices;
};

// One slice a row up to 8192 tokens (4 or 8 a thread). Else slices of 8 tokens a thread, as wide as still gives every
// CU a workgroup (each reads the whole history). One workgroup a row up to 32768 tokens saves the second launch and
// loses more: 64 x 30522 fp32, 1024 ids, 16.5 us against 11.8.
inline Shape shape_of(int B, int V) {
  auto threads = [&](int iter) { return (V + 256 * iter - 1) / (256 * iter) * 64; };
  if (V <= 4096) return {1, threads(1), 1};
  if (V <= 8192) return {2, threads(2), 1};
  for (int nt = 1024;; nt /= 2) {
    const int s = (V + 8 * nt - 1) / (8 * nt);
    if ((long)B * s >= 256 || nt == 256) return {2, nt, s};
  }
}

template <class T, class I>
void launch(const RulesArgs& a, const Shape& s, int B, hipStream_t st) {
  const size_t lds = a.history ? (size_t)4 * s.iter * s.threads * sizeof(int) : 0;
  const dim3 grid(s.slices, B), block(s.threads);
  if (s.iter == 1) hipLaunchKernelGGL((logit_rules_kernel<T, I, 1>), grid, block, lds, st, a);
  else hipLaunchKernelGGL((logit_rules_kernel<T, I, 2>), grid, block, lds, st, a);
}

}  // namespace

extern "C" int64_t dasa_logit_rules_workspace(int32_t B, int32_t V) {
  if (B <= 0 || V <= 0 || V > kMostSize) return 0;
  const int s = shape_of(B, V).slices;
  return s > 1 ? (int64_t)B * s * 8 : 0;
}

extern "C" int dasa_logit_rules(const dasa_logit_rules_desc* d, void* ws, int64_t ws_bytes, void* stream) {
  if (!d || d->B < 0 || d->V < 0) return (int)hipErrorInvalidValue;
  if (d->B == 0) return 0;
  if (d->V == 0 || d->V > kMostSize || d->B > 65535 || d->L < 0 || d->L > kMostSize ||
      !d->logits || !d->out || d->ld < d->V || d->ldo < d->V)
    return (int)hipErrorInvalidValue;
  if (d->history && ((d->ids_bytes != 4 && d->ids_bytes != 8) || d->ldh < d->L)) return (int)hipErrorInvalidValue;
  if ((d->allowed_bits && d->allowed_bytes) || (d->bias && d->ldb != 0 && d->ldb < d->V) ||
      (d->allowed_bits && d->ldbits != 0 && d->ldbits < (d->V + 31) / 32) ||
      (d->allowed_bytes && d->ldbytes != 0 && d->ldbytes < d->V))
    return (int)hipErrorInvalidValue;
  const Shape sh = shape_of(d->B, d->V);
  const int slices = sh.slices;
  if (d->choice && slices > 1 && (!ws || !aligned16(ws) || ws_bytes < dasa_logit_rules_workspace(d->B, d->V)))
    return (int)hipErrorInvalidValue;
  RulesArgs a{};
  a.logits = d->logits; a.ld = d->ld; a.out = d->out; a.ldo = d->ldo;
  a.history = d->L > 0 ? d->history : nullptr; a.ldh = d->ldh; a.L = d->L; a.lengths = d->lengths;
  a.rep = d->repetition; a.pres = d->presence; a.freq = d->frequency;
  a.rep0 = d->repetition0; a.pres0 = d->presence0; a.freq0 = d->frequency0;
  a.bias = d->bias; a.ldb = d->ldb;
  a.bits = d->allowed_bits; a.ldbits = d->ldbits; a.bytes = d->allowed_bytes; a.ldbytes = d->ldbytes;
  a.choice = d->choice; a.best = reinterpret_cast<unsigned long long*>(ws);
  a.V = d->V; a.slices = slices;
  hipStream_t st = (hipStream_t)stream;
  const bool narrow = d->ids_bytes == 4;
  if (d->bf16) narrow ? launch<__bf16, int32_t>(a, sh, d->B, st) : launch<__bf16, int64_t>(a, sh, d->B, st);
  else narrow ? launch<float, int32_t>(a, sh, d->B, st) : launch<float, int64_t>(a, sh, d->B, st);
  DASA_CHECK_LAUNCH();
  if (d->choice && slices > 1) {
    hipLaunchKernelGGL(logit_choice_kernel, dim3(d->B), dim3(64), 0, st, a.best, a.choice, slices);
    DASA_CHECK_LAUNCH();
  }
  return 0;
}
