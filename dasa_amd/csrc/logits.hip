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
// A workgroup owns one row's slice of kSlice tokens: it counts the row's history into LDS (integer atomics: the
// counts do not depend on their order), then streams the slice once. With one slice a row, the workgroup also makes
// the choice; else each slice leaves its best key and one wave a row takes the best of them.
#include "common.h"
#include "../../include/dasa_hip.h"

namespace {

// 16 B of a row whose start need not be aligned (an odd vocabulary): element-aligned vector accesses
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 b4u __attribute__((ext_vector_type(4), aligned(2)));
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
  int V, slices, slice;
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

template <class T, class I>
__global__ __launch_bounds__(1024) void logit_rules_kernel(RulesArgs a) {
#pragma clang fp contract(off)
  typedef typename V4<T>::type V;
  extern __shared__ int count[];        // [slice] when there is a history
  __shared__ unsigned long long wbest[16];
  const int b = blockIdx.y, lo = blockIdx.x * a.slice, n = min(a.slice, a.V - lo);
  const int tid = threadIdx.x, lane = tid & 63, nt = blockDim.x;
  if (a.history) {
    for (int i = tid; i < a.slice; i += nt) count[i] = 0;
    __syncthreads();
    const I* h = reinterpret_cast<const I*>(a.history) + (long)b * a.ldh;
    const int len = a.lengths ? min(max(a.lengths[b], 0), a.L) : a.L;
    for (int i = tid; i < len; i += nt) {
      const long v = (long)h[i] - lo;
      if (v >= 0 && v < n) atomicAdd(&count[v], 1);
    }
    __syncthreads();
  }
  const float r = a.rep ? a.rep[b] : a.rep0, p = a.pres ? a.pres[b] : a.pres0, f = a.freq ? a.freq[b] : a.freq0;
  const T* x0 = reinterpret_cast<const T*>(a.logits) + (long)b * a.ld + lo;
  T* y0 = reinterpret_cast<T*>(a.out) + (long)b * a.ldo + lo;
  const float* bias = a.bias ? a.bias + (long)b * a.ldb + lo : nullptr;
  const unsigned* bits = a.bits ? a.bits + (long)b * a.ldbits : nullptr;
  const unsigned char* bytes = a.bytes ? a.bytes + (long)b * a.ldbytes + lo : nullptr;
  unsigned long long best = 0;
  auto rule = [&](float x, int c, float add, bool open) {
    if (c > 0) {
      x = x > 0.f ? x / r : x * r;
      x = x - f * (float)c;
      x = x - p;
    }
    if (bias) x = x + add;
    return (T)(open ? x : -INFINITY);
  };
  for (int i = 4 * tid; i < n; i += 4 * nt) {
    unsigned open = 15u;                 // lo and i are multiples of 4: the four bits share a word
    if (bits) open = (bits[(lo + i) >> 5] >> ((lo + i) & 31)) & 15u;
    if (i + 4 <= n) {
      V x = *reinterpret_cast<const V*>(x0 + i);
      f4u add = {0.f, 0.f, 0.f, 0.f};
      if (bias) add = *reinterpret_cast<const f4u*>(bias + i);
      int4 c = make_int4(0, 0, 0, 0);
      if (a.history) c = *reinterpret_cast<const int4*>(count + i);
      const int cc[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (bytes && !bytes[i + e]) open &= ~(1u << e);
        x[e] = rule((float)x[e], cc[e], add[e], (open >> e) & 1);
      }
      *reinterpret_cast<V*>(y0 + i) = x;
      if (a.choice) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned long long k = choice_key((float)x[e], lo + i + e);
          best = k > best ? k : best;
        }
      }
    } else {
      for (int e = 0; i + e < n; ++e) {
        const bool o = ((open >> e) & 1) && (!bytes || bytes[i + e]);
        const T y = rule((float)x0[i + e], a.history ? count[i + e] : 0, bias ? bias[i + e] : 0.f, o);
        y0[i + e] = y;
        const unsigned long long k = choice_key((float)y, lo + i + e);
        best = k > best ? k : best;
      }
    }
  }
  if (!a.choice) return;
  best = wave_best(best);
  if (lane == 0) wbest[tid >> 6] = best;
  __syncthreads();
  if (tid == 0) {
    for (int k = 1; k < nt / 64; ++k) best = wbest[k] > best ? wbest[k] : best;
    if (a.slices == 1) a.choice[b] = (int64_t)(unsigned)~(unsigned)best;
    else a.best[(long)b * a.slices + blockIdx.x] = best;
  }
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

constexpr int kSlice = 8192;     // tokens of one workgroup: 32 KB of counts

inline int slices_of(int B, int V) { (void)B; return (V + kSlice - 1) / kSlice; }

}  // namespace

extern "C" int64_t dasa_logit_rules_workspace(int32_t B, int32_t V) {
  if (B <= 0 || V <= 0) return 0;
  const int s = slices_of(B, V);
  return s > 1 ? (int64_t)B * s * 8 : 0;
}

extern "C" int dasa_logit_rules(const dasa_logit_rules_desc* d, void* ws, int64_t ws_bytes, void* stream) {
  if (!d || d->B < 0 || d->V < 0) return (int)hipErrorInvalidValue;
  if (d->B == 0) return 0;
  if (d->V == 0 || d->B > 65535 || d->L < 0 || !d->logits || !d->out || d->ld < d->V || d->ldo < d->V)
    return (int)hipErrorInvalidValue;
  if (d->history && ((d->ids_bytes != 4 && d->ids_bytes != 8) || d->ldh < d->L)) return (int)hipErrorInvalidValue;
  if ((d->allowed_bits && d->allowed_bytes) || (d->bias && d->ldb != 0 && d->ldb < d->V) ||
      (d->allowed_bits && d->ldbits != 0 && d->ldbits < (d->V + 31) / 32) ||
      (d->allowed_bytes && d->ldbytes != 0 && d->ldbytes < d->V))
    return (int)hipErrorInvalidValue;
  const int slices = slices_of(d->B, d->V);
  if (d->choice && slices > 1 && (!ws || ws_bytes < dasa_logit_rules_workspace(d->B, d->V)))
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
  a.slice = slices > 1 ? kSlice : ((d->V + 3) & ~3);
  const int work = d->V < a.slice ? d->V : a.slice;
  int nt = (((work + 3) / 4 + 63) / 64) * 64;
  if (a.history && nt < 256) nt = 256;
  if (nt > 1024) nt = 1024;
  const size_t lds = a.history ? (size_t)a.slice * sizeof(int) : 0;
  const dim3 grid(slices, d->B), block(nt);
  hipStream_t st = (hipStream_t)stream;
  if (d->bf16) {
    if (d->ids_bytes == 4) hipLaunchKernelGGL((logit_rules_kernel<__bf16, int32_t>), grid, block, lds, st, a);
    else hipLaunchKernelGGL((logit_rules_kernel<__bf16, int64_t>), grid, block, lds, st, a);
  } else {
    if (d->ids_bytes == 4) hipLaunchKernelGGL((logit_rules_kernel<float, int32_t>), grid, block, lds, st, a);
    else hipLaunchKernelGGL((logit_rules_kernel<float, int64_t>), grid, block, lds, st, a);
  }
  DASA_CHECK_LAUNCH();
  if (d->choice && slices > 1) {
    hipLaunchKernelGGL(logit_choice_kernel, dim3(d->B), dim3(64), 0, st, a.best, a.choice, slices);
    DASA_CHECK_LAUNCH();
  }
  return 0;
}
