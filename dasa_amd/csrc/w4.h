// Products of a few activation rows with 4-bit weights and group scales (the matrix-vector end of decoding):
//
//   y[m][n] = act( sum_k x[m][k] (q[n][k] - 8) s[n][k / g] + b[n] ) + beta y[m][n],    q in 0..15, g in {32, 64, 128}
//
// the nn.Linear of one word step (SpeakerDecoder: model.py:1066-1078) on weights that a program quantised once
// (dasa_w4_quantize / dasa_w4_layout).
//
// Mathematics: q - 8 is exact in bf16, and an fp32 activation is split exactly into three bf16 planes (x = hi + mid +
// lo by truncation), so every product on v_mfma_f32_16x16x32_bf16 is exact and only the fp32 accumulation rounds: the
// result has fp32 accuracy (bf16 activations need one plane). A group's sum is scaled once, in fp32, when the group
// ends. Below 2^-110 the lower planes are flushed (measured: 2^-23.7 of the value at 2^-110, 2^-7 at 2^-126); above 2^121
// a group's sum of up to 64 |x| can overflow before its scale.
//
// Layout: the weights are stored in the order in which lanes eat them. A 16-column x 128-deep block is 1 KB: lane l's
// 16 B are its column (l & 15)'s nibbles k = 32 j + 8 (l >> 4) + i of word j, nibble i — one global_load_dwordx4 per
// lane per block, no LDS, no shuffle. Nibbles are two's complement (q ^ 8), which v_cvt_off_f32_i4 turns into
// (q - 8) / 16; the 16 is multiplied back at the end.
//
// Two forms. Split: a workgroup owns 16 rows and NT column blocks, its waves take the 128-deep blocks of K in turn and
// their sums meet in LDS in wave order. Shared: the waves own column blocks and walk K together, so that more rows of
// x are split into planes and held in LDS once for all of them. K may be split over workgroups in both; a second
// launch then joins the sums in order. Every order is fixed by the shape: results are bitwise reproducible.
//
// What bounds it, measured: one row on a wide layer is its weights' bytes (1 x 32768 x 8192 bf16, group 128: 27.1 us for
// 138 MB = 5.1 TB/s, a large copy reaches 5.2); small layers are a launch (1 x 2048 x 256 fp32: 3.1 us, an empty kernel
// 2.4); 64 bf16 rows of a short K are the unpacking and the stores (64 x 30522 x 768: 10.4 us, of them 2.5 the stores);
// many fp32 rows are the three planes' matrix instructions (64 x 32768 x 8192: 108 us = 0.95 PFLOP/s of bf16 work).
#pragma once
#include "common.h"
#include "../../include/dasa_hip.h"

#include <type_traits>

namespace w4 {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

struct W4Args {
  const void* x; long ldx;
  const uint4* w;           // [N16][Kb][64 lanes] 16 B
  const void* scales;       // [N16][Kb][16][128 / g]
  const float* bias;
  void* y; long ldy;
  float beta;
  int act;
  int M, N, K, Kb, N16;
  int per;                  // 128-deep blocks of one K split
  float4* part;             // [splits][16-row tiles][N16][64] sums of a split, or null: one split
};

__device__ __forceinline__ float act_of(float v, int act) {
  switch (act) {
    case DASA_ACT_RELU: return v < 0.f ? 0.f : v;
    case DASA_ACT_GELU: return gelu_erf(v);
    case DASA_ACT_TANH: return tanhf(v);
    case DASA_ACT_SIGMOID: return sigmoidf_(v);
    default: return v;
  }
}

union Frag {
  unsigned u[4];
  bf16x8 v;
};

// eight two's-complement nibbles -> eight bf16 values (q - 8) / 16, element i = nibble i: one shift, eight converts
// (each from one byte of the word, whose low nibble counts), four merges of the high halves, which hold it all
__device__ __forceinline__ bf16x8 unpack8(unsigned w) {
  Frag f;
  unsigned h = w >> 4;
  asm("" : "+v"(h));      // kept: taking the odd nibbles out of w costs an instruction each (64 x 14336 x 4096: 22.3 us)
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const float e = __builtin_amdgcn_cvt_off_f32_i4((int)((w >> (8 * b)) & 255u));
    const float o = __builtin_amdgcn_cvt_off_f32_i4((int)((h >> (8 * b)) & 255u));
    f.u[b] = __builtin_amdgcn_perm(__float_as_uint(o), __float_as_uint(e), 0x07060302u);
  }
  return f.v;
}

// Eight consecutive activations of one row, as loaded (Raw) and as PL bf16 fragments. Rows start anywhere: element-
// aligned vectors. `left` <= 8 values exist; the rest are zeros.
template <class T> struct XFrag;
template <> struct XFrag<float> {
  static constexpr int PL = 3;
  typedef float V __attribute__((ext_vector_type(4), aligned(4)));
  struct Raw { float v[8]; };
  static __device__ __forceinline__ Raw load(const float* p) {
    const V a = reinterpret_cast<const V*>(p)[0], b = reinterpret_cast<const V*>(p)[1];
    return Raw{{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}};
  }
  static __device__ __forceinline__ Raw load_part(const float* p, int left) {
    Raw r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = i < left ? p[i] : 0.f;
    return r;
  }
  // x = p0 + p1 + p2, every plane a bf16 (truncated: 8 + 8 + 8 significand bits). A NaN stays one in every plane. An
  // infinity would leave inf - inf behind, so a fragment that holds one takes the guarded form.
  static __device__ __forceinline__ void planes(const Raw& r, bf16x8 (&f)[3]) {
    float m = fmaxf(fabsf(r.v[0]), fabsf(r.v[1]));
#pragma unroll
    for (int i = 2; i < 8; ++i) m = fmaxf(m, fabsf(r.v[i]));
    const bool inf = __any(m == INFINITY);
    Frag q[3];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      unsigned p0[2], p1[2], p2[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float x = r.v[2 * i + e];
        p0[e] = __float_as_uint(x);
        float d = x - __uint_as_float(p0[e] & 0xffff0000u);
        if (inf && fabsf(x) == INFINITY) d = 0.f;
        p1[e] = __float_as_uint(d);
        p2[e] = __float_as_uint(d - __uint_as_float(p1[e] & 0xffff0000u));
      }
      q[0].u[i] = __builtin_amdgcn_perm(p0[1], p0[0], 0x07060302u);
      q[1].u[i] = __builtin_amdgcn_perm(p1[1], p1[0], 0x07060302u);
      q[2].u[i] = __builtin_amdgcn_perm(p2[1], p2[0], 0x07060302u);
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) f[k] = q[k].v;
  }
};
template <> struct XFrag<__bf16> {
  static constexpr int PL = 1;
  typedef __bf16 V __attribute__((ext_vector_type(8), aligned(2)));
  struct Raw { V v; };
  static __device__ __forceinline__ Raw load(const __bf16* p) { return Raw{*reinterpret_cast<const V*>(p)}; }
  static __device__ __forceinline__ Raw load_part(const __bf16* p, int left) {
    Raw r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = i < left ? p[i] : (__bf16)0.f;
    return r;
  }
  static __device__ __forceinline__ void planes(const Raw& r, bf16x8 (&f)[1]) { f[0] = r.v; }
};

// The GPB scales of one column of one block, in their type: widening them where they are loaded would wait for them there
// (64 x 32768 x 8192, scales bf16: 61.1 us against 55.8).
template <class S, int GPB> struct Scales {
  typedef S V __attribute__((ext_vector_type(GPB)));
  V v;
  __device__ __forceinline__ void load(const void* scales, long at) { v = reinterpret_cast<const V*>(scales)[at]; }
  __device__ __forceinline__ float operator[](int g) const { return (float)v[g]; }
};
template <class S> struct Scales<S, 1> {
  S v;
  __device__ __forceinline__ void load(const void* scales, long at) { v = reinterpret_cast<const S*>(scales)[at]; }
  __device__ __forceinline__ float operator[](int) const { return (float)v; }
};

// four consecutive rows of one output column
template <class T>
__device__ __forceinline__ void epilogue(const W4Args& a, float4 s, int n, int row) {
  if (n >= a.N) return;
  const float b = a.bias ? a.bias[n] : 0.f;
  const float r[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (row + e >= a.M) continue;
    float v = 16.f * r[e];
    if (a.bias) v += b;
    v = act_of(v, a.act);
    T* o = reinterpret_cast<T*>(a.y) + (long)(row + e) * a.ldy + n;
    if (a.beta != 0.f) v += a.beta * (float)*o;
    *o = (T)v;
  }
}

// four consecutive columns of one output row
template <class T>
__device__ __forceinline__ void store4(const W4Args& a, float4 s, int row, int n) {
  typedef T V __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  typedef float F __attribute__((ext_vector_type(4), aligned(4)));
  const int left = a.N - n;
  if (left <= 0) return;
  T* o = reinterpret_cast<T*>(a.y) + (long)row * a.ldy + n;
  float r[4] = {s.x, s.y, s.z, s.w};
  float b[4] = {0.f, 0.f, 0.f, 0.f};
  if (a.bias) {
    if (left >= 4) {
      const F v = *reinterpret_cast<const F*>(a.bias + n);
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e] = v[e];
    } else {
      for (int e = 0; e < left; ++e) b[e] = a.bias[n + e];
    }
  }
  V v;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float y = 16.f * r[e];
    if (a.bias) y += b[e];
    y = act_of(y, a.act);
    if (a.beta != 0.f && e < left) y += a.beta * (float)o[e];
    v[e] = (T)y;
  }
  if (left >= 4) {
    *reinterpret_cast<V*>(o) = v;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) o[e] = v[e];
  }
}

// Split form. A workgroup owns 16 rows of x and NT blocks of 16 columns; its W waves take the 128-deep blocks of K in
// turn, straight from memory, and their sums meet in LDS in wave order. GPB = groups of a 128-deep block.
template <class T, class S, int NT, int GPB, int W>
__global__ __launch_bounds__(64 * W, 4) void w4_split_kernel(W4Args a) {
  typedef XFrag<T> X;
  constexpr int PL = X::PL;
  extern __shared__ float4 part[];          // [W][NT][64]
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int nt0 = blockIdx.x * NT, m0 = blockIdx.y * 16;
  const int c16 = lane & 15, kq = lane >> 4;
  floatx4 y[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) y[t] = floatx4{0.f, 0.f, 0.f, 0.f};
  // a row past the last repeats it: it only reaches output rows that are not stored
  const T* x = reinterpret_cast<const T*>(a.x) + (long)min(m0 + c16, a.M - 1) * a.ldx + kq * 8;
  long blk0[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) blk0[t] = (long)min(nt0 + t, a.N16 - 1) * a.Kb;

  const int k0 = blockIdx.z * a.per, k1 = min(k0 + a.per, a.Kb), full = min(k1, a.K / 128);
  auto block = [&](int kb, auto tail) {
    constexpr bool TAIL = decltype(tail)::value;
    uint4 wq[NT];
    Scales<S, GPB> sc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      wq[t] = a.w[(blk0[t] + kb) * 64 + lane];
      sc[t].load(a.scales, (blk0[t] + kb) * 16 + c16);
    }
    typename X::Raw raw[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = kb * 128 + j * 32;
      if constexpr (TAIL) raw[j] = X::load_part(x + k, a.K - k - kq * 8);
      else raw[j] = X::load(x + k);
    }
    // all loads of the block before its first product (1 x 32768 x 8192 bf16: 33.0 us without); fp32 rows' three planes
    // need the registers that this would hold (20 x 4096 x 2240: 10.8 us with, 10.0 without)
    if constexpr (PL == 1) __builtin_amdgcn_sched_barrier(0);
    floatx4 acc[NT];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      bf16x8 xf[PL];
      X::planes(raw[j], xf);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const bf16x8 wf = unpack8(j == 0 ? wq[t].x : j == 1 ? wq[t].y : j == 2 ? wq[t].z : wq[t].w);
        if (j % (4 / GPB) == 0) acc[t] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int p = PL - 1; p >= 0; --p)     // small planes first
          acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[p], wf, acc[t], 0, 0, 0);
        if (j % (4 / GPB) == 4 / GPB - 1)
#pragma unroll
          for (int i = 0; i < 4; ++i) y[t][i] += sc[t][j / (4 / GPB)] * acc[t][i];
      }
    }
  };
  for (int kb = k0 + w; kb < full; kb += W) block(kb, std::false_type{});
  if (full >= k0 && full < k1 && (full - k0) % W == w) block(full, std::true_type{});

#pragma unroll
  for (int t = 0; t < NT; ++t) part[(w * NT + t) * 64 + lane] = make_float4(y[t][0], y[t][1], y[t][2], y[t][3]);
  __syncthreads();
  for (int i = threadIdx.x; i < NT * 64; i += 64 * W) {
    float4 s = part[i];
#pragma unroll
    for (int k = 1; k < W; ++k) {
      const float4 v = part[k * NT * 64 + i];
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    const int l = i & 63, t = i >> 6;
    if (!a.part) epilogue<T>(a, s, (nt0 + t) * 16 + (l & 15), m0 + (l >> 4) * 4);
    else if (nt0 + t < a.N16) a.part[(((long)blockIdx.z * gridDim.y + blockIdx.y) * a.N16 + nt0 + t) * 64 + l] = s;
  }
}

constexpr int kShareWaves = 8;

// The form for more rows: the workgroup's waves own NT column blocks each and walk K together, so the activations'
// fragments are split into their planes once for the 8 NT blocks, in LDS (two buffers, one barrier a 128-deep block),
// where each wave reads them back in fragment order.
// TAIL: K ends inside a block (a branch at every load of x otherwise).
template <class T, class S, int MT, int NT, int GPB, bool TAIL>
__global__ __launch_bounds__(64 * kShareWaves, 2) void w4_shared_kernel(W4Args a) {
  typedef XFrag<T> X;
  // weights are asked for AHEAD - 1 blocks early (even: the two activation buffers keep their places over a turn of the
  // ring). Three early only pay for a long K with registers left (64 x 16384 x 4096 bf16 19.9 us against 21.6; 64 x 30522
  // x 768 bf16 11.0 against 9.9 with one, fp32 16.6 against 15.7)
  constexpr int AHEAD = X::PL == 1 && NT > 1 ? 4 : 2;
  constexpr int PL = X::PL, UNITS = MT * 4, PER = (UNITS + kShareWaves - 1) / kShareWaves;   // fragments a wave makes
  extern __shared__ float4 smem[];
  bf16x8* frag = reinterpret_cast<bf16x8*>(smem);       // [2][PL][4 steps][MT][64]
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int nt0 = (blockIdx.x * kShareWaves + w) * NT, m0 = blockIdx.y * (16 * MT);
  const int c16 = lane & 15, kq = lane >> 4;
  floatx4 y[NT][MT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m) y[t][m] = floatx4{0.f, 0.f, 0.f, 0.f};
  const int k0 = blockIdx.z * a.per, k1 = min(k0 + a.per, a.Kb);
  typename X::Raw raw[2][PER];           // activations two blocks ahead
  auto fetch = [&](int kb, typename X::Raw (&r)[PER]) {
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int f = u * kShareWaves + w;
      if (UNITS % kShareWaves && f >= UNITS) continue;
      const int m = f % MT, k = kb * 128 + (f / MT) * 32 + kq * 8;
      const T* p = reinterpret_cast<const T*>(a.x) + (long)min(m0 + m * 16 + c16, a.M - 1) * a.ldx + k;
      r[u] = !TAIL || kb * 128 + 128 <= a.K ? X::load(p) : X::load_part(p, a.K - k);
    }
  };
  auto put = [&](int buf, const typename X::Raw (&r)[PER]) {
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int f = u * kShareWaves + w;
      if (UNITS % kShareWaves && f >= UNITS) continue;
      bf16x8 q[PL];
      X::planes(r[u], q);
#pragma unroll
      for (int p = 0; p < PL; ++p) frag[((buf * PL + p) * UNITS + f) * 64 + lane] = q[p];
    }
  };
  uint4 wq[AHEAD][NT];
  Scales<S, GPB> sc[AHEAD][NT];
  auto weights = [&](int kb, uint4 (&q)[NT], Scales<S, GPB> (&s)[NT]) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const long b = (long)min(nt0 + t, a.N16 - 1) * a.Kb + kb;
      q[t] = a.w[b * 64 + lane];
      s[t].load(a.scales, b * 16 + c16);
    }
  };
  auto compute = [&](int buf, const uint4 (&q)[NT], const Scales<S, GPB> (&s)[NT]) {
    floatx4 acc[NT][MT];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      bf16x8 xf[MT][PL];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int p = 0; p < PL; ++p) xf[m][p] = frag[((buf * PL + p) * UNITS + j * MT + m) * 64 + lane];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const bf16x8 wf = unpack8(j == 0 ? q[t].x : j == 1 ? q[t].y : j == 2 ? q[t].z : q[t].w);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          if (j % (4 / GPB) == 0) acc[t][m] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int p = PL - 1; p >= 0; --p)
            acc[t][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[m][p], wf, acc[t][m], 0, 0, 0);
          if (j % (4 / GPB) == 4 / GPB - 1)
#pragma unroll
            for (int i = 0; i < 4; ++i) y[t][m][i] += s[t][j / (4 / GPB)] * acc[t][m][i];
        }
      }
    }
  };
  if (k0 < k1) {                          // blocks past the last are the last again: loads without branches
    fetch(k0, raw[0]);
    weights(k0, wq[0], sc[0]);
    fetch(min(k0 + 1, k1 - 1), raw[1]);
#pragma unroll
    for (int i = 1; i < AHEAD - 1; ++i) weights(min(k0 + i, k1 - 1), wq[i], sc[i]);
    put(0, raw[0]);
  }
  __syncthreads();
  for (int kb = k0; kb < k1; kb += AHEAD) {
#pragma unroll
    for (int h = 0; h < AHEAD; ++h) {
      if (kb + h >= k1) break;
      fetch(min(kb + h + 2, k1 - 1), raw[h & 1]);
      weights(min(kb + h + AHEAD - 1, k1 - 1), wq[(h + AHEAD - 1) % AHEAD], sc[(h + AHEAD - 1) % AHEAD]);
      compute(h & 1, wq[h], sc[h]);
      put((h & 1) ^ 1, raw[(h & 1) ^ 1]);
      __syncthreads();
    }
  }
  if (a.part) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int m = 0; m < MT; ++m)
        if (nt0 + t < a.N16)
          a.part[(((long)blockIdx.z * gridDim.y * MT + blockIdx.y * MT + m) * a.N16 + nt0 + t) * 64 + lane] =
              make_float4(y[t][m][0], y[t][m][1], y[t][m][2], y[t][m][3]);
    return;
  }
  // the sums through LDS, so that a row's columns leave in runs of four (a fragment holds four rows of one column:
  // stored from there, 64 x 30522 bf16 outputs took 4 us more)
  constexpr int COLS = kShareWaves * NT * 16, LD = COLS + 4;
  float* tile = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) tile[(m * 16 + kq * 4 + i) * LD + (w * NT + t) * 16 + c16] = y[t][m][i];
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * MT * (COLS / 4); i += 64 * kShareWaves) {
    const int r = i / (COLS / 4), c = (i % (COLS / 4)) * 4;
    if (m0 + r < a.M) store4<T>(a, *reinterpret_cast<const float4*>(tile + r * LD + c), m0 + r, blockIdx.x * COLS + c);
  }
}

// The splits of K joined in order: one thread = four output rows of one column.
template <class T>
__global__ __launch_bounds__(256) void w4_join_kernel(W4Args a, int splits, int tiles) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x, n = (long)tiles * a.N16 * 64;
  if (i >= n) return;
  float4 s = a.part[i];
  for (int k = 1; k < splits; ++k) {
    const float4 v = a.part[k * n + i];
    s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
  }
  const int l = (int)(i & 63);
  const long b = i >> 6;
  epilogue<T>(a, s, (int)(b % a.N16) * 16 + (l & 15), (int)(b / a.N16) * 16 + (l >> 4) * 4);
}

struct Plan {
  bool shared;   // which form
  int mt;        // 16-row tiles of a workgroup (split form: 1)
  int nt;        // column blocks of a workgroup (split form) or of a wave (shared form)
  int waves;     // of a workgroup
  int splits;    // of K over workgroups
};

template <class T>
int launch_join(const W4Args& a, int splits, int tiles, hipStream_t st) {
  if (!a.part) return 0;
  const long n = (long)tiles * a.N16 * 64;
  hipLaunchKernelGGL(w4_join_kernel<T>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, a, splits, tiles);
  DASA_CHECK_LAUNCH();
  return 0;
}

template <class T, class S, int MT, int NT>
int launch_shared(const W4Args& a, int g, int splits, hipStream_t st) {
  constexpr int cols = kShareWaves * NT;
  const dim3 grid((a.N16 + cols - 1) / cols, (a.M + 16 * MT - 1) / (16 * MT), splits), block(64 * kShareWaves);
  constexpr size_t frags = (size_t)2 * XFrag<T>::PL * 4 * MT * 64 * 16, tile = (size_t)16 * MT * (cols * 16 + 4) * 4;
  constexpr size_t lds = frags > tile ? frags : tile;
  auto go = [&](auto gpb) {
    constexpr int GPB = decltype(gpb)::value;
    if (a.K % 128) hipLaunchKernelGGL((w4_shared_kernel<T, S, MT, NT, GPB, true>), grid, block, lds, st, a);
    else hipLaunchKernelGGL((w4_shared_kernel<T, S, MT, NT, GPB, false>), grid, block, lds, st, a);
  };
  if (g == 32) go(std::integral_constant<int, 4>{});
  else if (g == 64) go(std::integral_constant<int, 2>{});
  else go(std::integral_constant<int, 1>{});
  DASA_CHECK_LAUNCH();
  return launch_join<T>(a, splits, (int)grid.y * MT, st);
}

template <class T, class S, int NT, int W>
int launch_split(const W4Args& a, int g, int splits, hipStream_t st) {
  const dim3 grid((a.N16 + NT - 1) / NT, (a.M + 15) / 16, splits), block(64 * W);
  constexpr size_t lds = (size_t)W * NT * 64 * 16;
  if (g == 32) hipLaunchKernelGGL((w4_split_kernel<T, S, NT, 4, W>), grid, block, lds, st, a);
  else if (g == 64) hipLaunchKernelGGL((w4_split_kernel<T, S, NT, 2, W>), grid, block, lds, st, a);
  else hipLaunchKernelGGL((w4_split_kernel<T, S, NT, 1, W>), grid, block, lds, st, a);
  DASA_CHECK_LAUNCH();
  return launch_join<T>(a, splits, (int)grid.y, st);
}

template <class T, class S>
int launch_plan(const W4Args& a, int g, const Plan& p, hipStream_t st) {
  if (p.shared) {
    if (p.mt == 4) return launch_shared<T, S, 4, 2>(a, g, p.splits, st);
    return p.nt == 2 ? launch_shared<T, S, 2, 2>(a, g, p.splits, st) : launch_shared<T, S, 2, 1>(a, g, p.splits, st);
  }
  if (p.nt == 4) return p.waves == 8 ? launch_split<T, S, 4, 8>(a, g, p.splits, st) : launch_split<T, S, 4, 16>(a, g, p.splits, st);
  if (p.nt == 2) return p.waves == 8 ? launch_split<T, S, 2, 8>(a, g, p.splits, st) : launch_split<T, S, 2, 16>(a, g, p.splits, st);
  return p.waves == 8 ? launch_split<T, S, 1, 8>(a, g, p.splits, st) : launch_split<T, S, 1, 16>(a, g, p.splits, st);
}

}  // namespace w4
