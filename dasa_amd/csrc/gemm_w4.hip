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
// ends.
//
// Layout: the weights are stored in the order in which lanes eat them. A 16-column x 128-deep block is 1 KB: lane l's
// 16 B are its column (l & 15)'s nibbles k = 32 j + 8 (l >> 4) + i of word j, nibble i — one global_load_dwordx4 per
// lane per block, no LDS, no shuffle. Nibbles are two's complement (q ^ 8), which v_cvt_off_f32_i4 turns into
// (q - 8) / 16; the 16 is multiplied back at the end.
//
// A workgroup of 4 waves owns NT blocks of 16 columns; the waves take the 128-deep blocks of K in turn and their sums
// meet in LDS in wave order (deterministic, one launch).
#include "common.h"
#include "../../include/dasa_hip.h"

#include <type_traits>

namespace {

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
  const unsigned h = w >> 4;
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

// the GPB scales of one column of one block
template <class S, int GPB>
__device__ __forceinline__ void load_scales(const void* scales, long at, float (&sc)[GPB]) {
  typedef S V __attribute__((ext_vector_type(GPB)));
  if constexpr (GPB == 1) {
    sc[0] = (float)reinterpret_cast<const S*>(scales)[at];
  } else {
    const V v = reinterpret_cast<const V*>(scales)[at];
#pragma unroll
    for (int g = 0; g < GPB; ++g) sc[g] = (float)v[g];
  }
}

// MT = 16-row tiles of x, NT = 16-column blocks of a workgroup, GPB = groups of a 128-deep block, W = waves
template <class T, class S, int MT, int NT, int GPB, int W>
__global__ __launch_bounds__(64 * W) void w4_kernel(W4Args a) {
  typedef XFrag<T> X;
  constexpr int PL = X::PL;
  extern __shared__ float4 part[];          // [W][NT][MT][64]
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int nt0 = blockIdx.x * NT, m0 = blockIdx.y * (16 * MT);
  const int c16 = lane & 15, kq = lane >> 4;
  floatx4 y[NT][MT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m) y[t][m] = floatx4{0.f, 0.f, 0.f, 0.f};
  // a row past the last repeats it: it only reaches output rows that are not stored
  const T* x[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
    x[m] = reinterpret_cast<const T*>(a.x) + (long)min(m0 + m * 16 + c16, a.M - 1) * a.ldx + kq * 8;
  long blk0[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) blk0[t] = (long)min(nt0 + t, a.N16 - 1) * a.Kb;

  auto block = [&](int kb, auto tail) {
    constexpr bool TAIL = decltype(tail)::value;
    uint4 wq[NT];
    float sc[NT][GPB];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      wq[t] = a.w[(blk0[t] + kb) * 64 + lane];
      load_scales<S, GPB>(a.scales, (blk0[t] + kb) * 16 + c16, sc[t]);
    }
    floatx4 acc[NT][MT];
    typename X::Raw raw[4][MT];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int k = kb * 128 + j * 32;
        if constexpr (TAIL) raw[j][m] = X::load_part(x[m] + k, a.K - k - kq * 8);
        else raw[j][m] = X::load(x[m] + k);
      }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      bf16x8 xf[MT][PL];
#pragma unroll
      for (int m = 0; m < MT; ++m) X::planes(raw[j][m], xf[m]);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const unsigned word = j == 0 ? wq[t].x : j == 1 ? wq[t].y : j == 2 ? wq[t].z : wq[t].w;
        const bf16x8 wf = unpack8(word);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          if (j % (4 / GPB) == 0) acc[t][m] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int p = PL - 1; p >= 0; --p)     // small planes first
            acc[t][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[m][p], wf, acc[t][m], 0, 0, 0);
          if (j % (4 / GPB) == 4 / GPB - 1) {
            const float s = sc[t][j / (4 / GPB)];
#pragma unroll
            for (int i = 0; i < 4; ++i) y[t][m][i] += s * acc[t][m][i];
          }
        }
      }
    }
  };
  const int full = a.K / 128;
  for (int kb = w; kb < full; kb += W) block(kb, std::false_type{});
  if (full < a.Kb && full % W == w) block(full, std::true_type{});

#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m)
      part[((w * NT + t) * MT + m) * 64 + lane] = make_float4(y[t][m][0], y[t][m][1], y[t][m][2], y[t][m][3]);
  __syncthreads();
  for (int i = threadIdx.x; i < NT * MT * 64; i += 64 * W) {
    float4 s = part[i];
#pragma unroll
    for (int k = 1; k < W; ++k) {
      const float4 v = part[k * NT * MT * 64 + i];
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    const int l = i & 63, m = (i >> 6) % MT, t = (i >> 6) / MT;
    const int n = (nt0 + t) * 16 + (l & 15), row = m0 + m * 16 + (l >> 4) * 4;
    if (n >= a.N) continue;
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
}

template <class T, class S, int MT, int NT, int W>
int launch_g(const W4Args& a, int g, hipStream_t st) {
  const dim3 grid((a.N16 + NT - 1) / NT, (a.M + 16 * MT - 1) / (16 * MT)), block(64 * W);
  const size_t lds = (size_t)W * NT * MT * 64 * 16;
  if (g == 32) hipLaunchKernelGGL((w4_kernel<T, S, MT, NT, 4, W>), grid, block, lds, st, a);
  else if (g == 64) hipLaunchKernelGGL((w4_kernel<T, S, MT, NT, 2, W>), grid, block, lds, st, a);
  else hipLaunchKernelGGL((w4_kernel<T, S, MT, NT, 1, W>), grid, block, lds, st, a);
  DASA_CHECK_LAUNCH();
  return 0;
}

#ifdef W4_TUNE
int g_nt = 1, g_w = 4;
template <class T, class S, int MT, int NT>
int launch_w(const W4Args& a, int g, hipStream_t st) {
  if (g_w == 4) return launch_g<T, S, MT, NT, 4>(a, g, st);
  if (g_w == 8) return launch_g<T, S, MT, NT, 8>(a, g, st);
  if constexpr (NT * MT <= 4) return launch_g<T, S, MT, NT, 16>(a, g, st);
  return 1;
}
template <class T, class S, int MT>
int launch_n(const W4Args& a, int g, hipStream_t st) {
  if (g_nt == 1) return launch_w<T, S, MT, 1>(a, g, st);
  if (g_nt == 2) return launch_w<T, S, MT, 2>(a, g, st);
  return launch_w<T, S, MT, 4>(a, g, st);
}
#else
template <class T, class S, int MT>
int launch_n(const W4Args& a, int g, hipStream_t st) {
  // two column blocks a workgroup once that still gives every CU one (halves the re-read of x)
  return a.N16 >= 512 ? launch_g<T, S, MT, 2, 4>(a, g, st) : launch_g<T, S, MT, 1, 4>(a, g, st);
}
#endif

template <class T, class S>
int launch_m(const W4Args& a, int g, hipStream_t st) {
  if (a.M <= 16) return launch_n<T, S, 1>(a, g, st);
  if (a.M <= 32) return launch_n<T, S, 2>(a, g, st);
  return launch_n<T, S, 4>(a, g, st);
}

// ------------------------------------------------------------------ layout and quantisation (once per weight)
struct LayoutArgs {
  const unsigned char* codes; long ldc;   // [N][ceil(K / 2)], the even k in the low nibble
  const void* scales; long lds_;          // [N][ceil(K / g)]
  unsigned* w; void* ws;
  int N, K, Kb, N16, g;
};

// One thread per 32-bit word of the tiled weights; the first threads of a block also place its scales.
template <class S>
__global__ __launch_bounds__(256) void w4_layout_kernel(LayoutArgs a) {
  const long blk = blockIdx.x;                        // (column block, K block)
  const int nt = (int)(blk / a.Kb), kb = (int)(blk % a.Kb);
  const int tid = threadIdx.x, l = tid >> 2, j = tid & 3;
  const int n = nt * 16 + (l & 15), k = kb * 128 + j * 32 + (l >> 4) * 8;
  unsigned word = 0;                                  // two's complement 0: padding adds nothing
  if (n < a.N) {
    for (int i = 0; i < 8 && k + i < a.K; ++i) {
      const unsigned c = (a.codes[(long)n * a.ldc + ((k + i) >> 1)] >> (4 * ((k + i) & 1))) & 15u;
      word |= (c ^ 8u) << (4 * i);
    }
  }
  a.w[blk * 256 + tid] = word;
  const int gpb = 128 / a.g, groups = (a.K + a.g - 1) / a.g;
  if (tid < gpb * 16) {
    const int nn = nt * 16 + tid / gpb, gi = kb * gpb + tid % gpb;
    const bool in = nn < a.N && gi < groups;
    reinterpret_cast<S*>(a.ws)[blk * gpb * 16 + tid] =
        in ? reinterpret_cast<const S*>(a.scales)[(long)nn * a.lds_ + gi] : (S)0.f;
  }
}

struct QuantArgs {
  const void* w; long ldw;
  unsigned char* codes; long ldc;
  void* scales; long lds_;
  int N, K, g;
};

// One thread per (row, group): s = max |w| / 7, q = clamp(rne(w / s), -8, 7) + 8; an all-zero group has s = 0, q = 8.
// The scale is rounded to its stored type first, so the codes are nearest to the values they will stand for.
template <class T, class S>
__global__ __launch_bounds__(256) void w4_quantize_kernel(QuantArgs a) {
  const int groups = (a.K + a.g - 1) / a.g;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long)a.N * groups) return;
  const int n = (int)(i / groups), gi = (int)(i % groups), k0 = gi * a.g, k1 = min(k0 + a.g, a.K);
  const T* w = reinterpret_cast<const T*>(a.w) + (long)n * a.ldw;
  float m = 0.f;
  for (int k = k0; k < k1; ++k) m = fmaxf(m, fabsf((float)w[k]));
  const S st = (S)(m / 7.f);
  reinterpret_cast<S*>(a.scales)[(long)n * a.lds_ + gi] = st;
  const float s = (float)st;
  for (int k = k0; k < k1; k += 2) {
    unsigned byte = 0x88u;
    for (int e = 0; e < 2 && k + e < k1; ++e) {
      int q = 0;
      if (s > 0.f) q = (int)fminf(fmaxf(rintf((float)w[k + e] / s), -8.f), 7.f);
      byte = (byte & ~(15u << (4 * e))) | ((unsigned)(q + 8) << (4 * e));
    }
    a.codes[(long)n * a.ldc + (k >> 1)] = (unsigned char)byte;
  }
}

inline bool group_ok(int g) { return g == 32 || g == 64 || g == 128; }

}  // namespace

extern "C" int64_t dasa_w4_weight_bytes(int32_t N, int32_t K) {
  if (N <= 0 || K <= 0) return 0;
  return (int64_t)((N + 15) / 16) * ((K + 127) / 128) * 1024;
}

extern "C" int64_t dasa_w4_scale_count(int32_t N, int32_t K, int32_t group) {
  if (N <= 0 || K <= 0 || !group_ok(group)) return 0;
  return (int64_t)((N + 15) / 16) * ((K + 127) / 128) * (128 / group) * 16;
}

extern "C" int dasa_w4_quantize(const void* W, int64_t ldw, int32_t w_bf16, int32_t N, int32_t K, int32_t group,
                                uint8_t* codes, int64_t ldc, void* scales, int64_t lds, int32_t scale_bf16,
                                void* stream) {
  if (N <= 0 || K <= 0 || !group_ok(group) || !W || !codes || !scales || ldw < K || ldc < (K + 1) / 2 ||
      lds < (K + group - 1) / group)
    return (int)hipErrorInvalidValue;
  QuantArgs a{W, (long)ldw, codes, (long)ldc, scales, (long)lds, N, K, group};
  const long total = (long)N * ((K + group - 1) / group);
  if ((total + 255) / 256 > 0x7fffffffL) return (int)hipErrorInvalidValue;
  const dim3 grid((unsigned)((total + 255) / 256)), block(256);
  hipStream_t st = (hipStream_t)stream;
  if (w_bf16 && scale_bf16) hipLaunchKernelGGL((w4_quantize_kernel<__bf16, __bf16>), grid, block, 0, st, a);
  else if (w_bf16) hipLaunchKernelGGL((w4_quantize_kernel<__bf16, float>), grid, block, 0, st, a);
  else if (scale_bf16) hipLaunchKernelGGL((w4_quantize_kernel<float, __bf16>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((w4_quantize_kernel<float, float>), grid, block, 0, st, a);
  DASA_CHECK_LAUNCH();
  return 0;
}

extern "C" int dasa_w4_layout(const uint8_t* codes, int64_t ldc, const void* scales, int64_t lds, int32_t scale_bf16,
                              int32_t N, int32_t K, int32_t group, void* weight, void* scale_tiles, void* stream) {
  if (N <= 0 || K <= 0 || !group_ok(group) || !codes || !scales || !weight || !scale_tiles || ldc < (K + 1) / 2 ||
      lds < (K + group - 1) / group)
    return (int)hipErrorInvalidValue;
  LayoutArgs a{codes, (long)ldc, scales, (long)lds, reinterpret_cast<unsigned*>(weight), scale_tiles, N, K,
               (K + 127) / 128, (N + 15) / 16, group};
  const long blocks = (long)a.N16 * a.Kb;
  if (blocks > 0x7fffffffL) return (int)hipErrorInvalidValue;
  if (scale_bf16)
    hipLaunchKernelGGL(w4_layout_kernel<__bf16>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(w4_layout_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a);
  DASA_CHECK_LAUNCH();
  return 0;
}

extern "C" int dasa_gemm_w4(const void* x, int64_t ldx, int32_t bf16, const void* weight, const void* scale_tiles,
                            int32_t scale_bf16, int32_t group, const float* bias, int32_t act, float beta, void* y,
                            int64_t ldy, int32_t M, int32_t N, int32_t K, void* stream) {
  if (M < 0 || N <= 0 || K <= 0 || !group_ok(group) || act < DASA_ACT_NONE || act > DASA_ACT_SIGMOID)
    return (int)hipErrorInvalidValue;
  if (M == 0) return 0;
  if (!x || !weight || !scale_tiles || !y || ldx < K || ldy < N || ((uintptr_t)weight & 15) || M > 65535 * 16)
    return (int)hipErrorInvalidValue;
  W4Args a{x, (long)ldx, reinterpret_cast<const uint4*>(weight), scale_tiles, bias, y, (long)ldy, beta, act, M, N, K,
           (K + 127) / 128, (N + 15) / 16};
  hipStream_t st = (hipStream_t)stream;
  if (bf16) return scale_bf16 ? launch_m<__bf16, __bf16>(a, group, st) : launch_m<__bf16, float>(a, group, st);
  return scale_bf16 ? launch_m<float, __bf16>(a, group, st) : launch_m<float, float>(a, group, st);
}
