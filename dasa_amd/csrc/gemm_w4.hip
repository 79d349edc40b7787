// Entry points of the 4-bit products (kernels: w4.h): the plan, the fp32 instantiations, and the layout and quantisation
// kernels that run once for a weight.
#include "w4.h"

#include <algorithm>

// gemm_w4_bf16.hip: the instantiations for bf16 activations
__attribute__((visibility("hidden"))) int dasa_w4_launch_bf16(const w4::W4Args& a, int group, const w4::Plan& p,
                                                              int scale_bf16, hipStream_t st);

namespace {

using w4::Plan;
using w4::W4Args;

// Which form and shape: measured over M = 1 .. 64, N = 992 .. 32768, K = 256 .. 8192 in both types (us). `units` counts
// column blocks times 16-row tiles.
//  * few units: the split form with each 16 rows a workgroup of their own. The weights come from cache for the second
//    rows; holding several row tiles in a workgroup instead leaves the chip emptier (20 x 4096 x 2240 fp32 8.4 against
//    11.4, 64 x 992 x 512 fp32 4.4 against 7.8). Column blocks of a workgroup: as many as still leave about one
//    workgroup a CU, since they share the activations' loads and their splitting into planes; up to eight bf16 rows,
//    which need no splitting, stop at two (1 x 30522 x 768 bf16 5.1 against 5.9, 16 rows 7.3 against 6.9; 32768 x 8192:
//    one row 30.0 against 30.9, 16 rows 43.0 against 33.9).
//  * many units and more than 16 rows: the shared form (64 x 30522 x 768 bf16 10.1 against 19.8). From 3500 units; a
//    short K, which the split form cannot deal to its waves, from 2500 (20 x 20000 x 640 bf16 6.1 against 7.8, but
//    33 x 16384 x 1024 fp32 13.3 against 10.8), a long one, which can be split over workgroups, from 1500 (33 x 8192 x
//    8192 fp32 32.3 against 39.2, but 64 x 4096 x 8192 fp32 17.6 against 14.5).
//    Two row tiles a workgroup, four where the weights are too many to read twice (64 x 12000 x 8192 bf16 24.7 against
//    30.0). Two column blocks a wave if that still fills five eighths of the chip (64 x 16384 x 1024 fp32 13.8 with one
//    against 17.5; 64 x 12000 x 8192 fp32 55.7 with two against 77.9), one for a short K of bf16 rows, where the loop is
//    mostly its start and end (33 x 32768 x 1024 bf16 11.5 against 13.3).
//  * K is split over workgroups, at the price of a second launch (2 us), only where a long K leaves too few of them
//    (1 x 1000 x 8192 fp32 7.7 against 13.4).
inline Plan plan_of(int M, int N, int K, int bf16) {
  Plan p{};
  const long tiles = (N + 15) / 16, Kb = (K + 127) / 128, rows = (M + 15) / 16, units = tiles * rows;
  p.mt = 1;
  p.nt = 1;
  p.waves = 8;
  p.splits = 1;
  if (rows > 1 && units >= (Kb >= 32 ? 1500 : Kb < 8 ? 2500 : 3500)) {
    p.shared = true;
    p.mt = rows > 2 && tiles * Kb >= 40000 ? 4 : 2;
    auto wgs = [&](int nt) { return (tiles + 8 * nt - 1) / (8 * nt) * ((rows + p.mt - 1) / p.mt); };
    auto splits = [&](int nt) { return (int)std::max(1L, std::min(256 / wgs(nt), Kb / 8)); };
    p.nt = p.mt == 4 || (wgs(2) * splits(2) >= 160 && (Kb >= 16 || !bf16)) ? 2 : 1;
    p.splits = splits(p.nt);
    return p;
  }
  if (Kb >= 48 && (!bf16 || rows > 1)) p.splits = (int)std::max(1L, std::min({Kb / 16, 4L, 1024 / units}));
  const long fill = units * p.splits;            // workgroups of one column block
  p.nt = fill < 384 ? 1 : fill < 640 || (bf16 && M <= 8) ? 2 : 4;
  p.waves = Kb > 8 && fill / p.nt <= 256 ? 16 : 8;
  return p;
}

// ------------------------------------------------------------------ layout and quantisation (once per weight)
struct LayoutArgs {
  const unsigned char* codes; long ldc;   // [N][ceil(K / 2)], the even k in the low nibble
  const void* scales; long lds_;          // [N][ceil(K / g)]
  unsigned* w; void* ws;
  int N, K, Kb, N16, g;
};

// Workgroup = 16 rows and four 128-deep blocks, whose codes are 256 B of a row: lines are read whole (32768 x 8192: 88 us
// with a block a workgroup). Thread = 32 codes of a row, four words of the layout, in which eight codes keep their order:
// code ^ 8 is the stored nibble. The first threads also place the blocks' scales.
template <class S>
__global__ __launch_bounds__(256) void w4_layout_kernel(LayoutArgs a) {
  typedef unsigned u4u __attribute__((ext_vector_type(4), aligned(1)));
  const int per = (a.Kb + 3) / 4;
  const int nt = (int)(blockIdx.x / per), kb0 = (int)(blockIdx.x % per) * 4;
  const int tid = threadIdx.x, c = tid >> 4, q = tid & 15, kb = kb0 + (q >> 2);
  const int n = nt * 16 + c, k = kb0 * 128 + q * 32;
  unsigned word[4] = {0, 0, 0, 0};                    // two's complement 0: padding adds nothing
  if (n < a.N) {
    const unsigned char* p = a.codes + (long)n * a.ldc + (k >> 1);
    if (k + 32 <= a.K) {
      const u4u v = *reinterpret_cast<const u4u*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) word[i] = v[i] ^ 0x88888888u;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        for (int e = 0; e < 8 && k + 8 * i + e < a.K; ++e)
          word[i] |= (((p[4 * i + (e >> 1)] >> (4 * (e & 1))) & 15u) ^ 8u) << (4 * e);
    }
  }
  if (kb < a.Kb) {
#pragma unroll
    for (int i = 0; i < 4; ++i) a.w[((long)nt * a.Kb + kb) * 256 + (i * 16 + c) * 4 + (q & 3)] = word[i];
  }
  const int gpb = 128 / a.g, groups = (a.K + a.g - 1) / a.g;
  for (int i = tid; i < 4 * gpb * 16; i += 256) {
    const int b = kb0 + i / (gpb * 16), j = i % (gpb * 16), nn = nt * 16 + j / gpb, gi = b * gpb + j % gpb;
    if (b >= a.Kb) continue;
    reinterpret_cast<S*>(a.ws)[((long)nt * a.Kb + b) * gpb * 16 + j] =
        nn < a.N && gi < groups ? reinterpret_cast<const S*>(a.scales)[(long)nn * a.lds_ + gi] : (S)0.f;
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
// Once for a weight, so left simple: the thread reads its group twice, a cache line a thread (32768 x 8192 fp32: 9.3 to
// 10.2 ms = 110 GB/s, where a large sum reads at 4.0 TB/s).
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

// N and K of a weight: index arithmetic adds blocks to them in 32 bits, and the layout has a workgroup of 256 threads for
// 16 x 512 values, of which a launch takes fewer than 2^32 (the products and the quantisation start fewer)
inline bool sizes_ok(int N, int K) {
  return N > 0 && K > 0 && N <= 1 << 30 && K <= 1 << 30 &&
         threads_fit((long)((N + 15) / 16) * ((K + 511) / 512), 256);
}
inline bool group_ok(int g) { return g == 32 || g == 64 || g == 128; }

}  // namespace

extern "C" int64_t dasa_w4_weight_bytes(int32_t N, int32_t K) {
  if (!sizes_ok(N, K)) return 0;
  return (int64_t)((N + 15) / 16) * ((K + 127) / 128) * 1024;
}

extern "C" int64_t dasa_w4_scale_count(int32_t N, int32_t K, int32_t group) {
  if (!sizes_ok(N, K) || !group_ok(group)) return 0;
  return (int64_t)((N + 15) / 16) * ((K + 127) / 128) * (128 / group) * 16;
}

extern "C" int dasa_w4_quantize(const void* W, int64_t ldw, int32_t w_bf16, int32_t N, int32_t K, int32_t group,
                                uint8_t* codes, int64_t ldc, void* scales, int64_t lds, int32_t scale_bf16,
                                void* stream) {
  if (!sizes_ok(N, K) || !group_ok(group) || !W || !codes || !scales || ldw < K || ldc < (K + 1) / 2 ||
      lds < (K + group - 1) / group)
    return (int)hipErrorInvalidValue;
  QuantArgs a{W, (long)ldw, codes, (long)ldc, scales, (long)lds, N, K, group};
  const long total = (long)N * ((K + group - 1) / group);
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
  if (!sizes_ok(N, K) || !group_ok(group) || !codes || !scales || !weight || !scale_tiles || !aligned16(weight) ||
      !aligned16(scale_tiles) || ldc < (K + 1) / 2 || lds < (K + group - 1) / group)
    return (int)hipErrorInvalidValue;
  LayoutArgs a{codes, (long)ldc, scales, (long)lds, reinterpret_cast<unsigned*>(weight), scale_tiles, N, K,
               (K + 127) / 128, (N + 15) / 16, group};
  const long blocks = (long)a.N16 * ((a.Kb + 3) / 4);
  if (scale_bf16)
    hipLaunchKernelGGL(w4_layout_kernel<__bf16>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(w4_layout_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a);
  DASA_CHECK_LAUNCH();
  return 0;
}

extern "C" int64_t dasa_gemm_w4_workspace(int32_t M, int32_t N, int32_t K, int32_t bf16) {
  if (M <= 0 || M > 65535 * 16 || !sizes_ok(N, K)) return 0;
  const Plan p = plan_of(M, N, K, bf16);
  if (p.splits <= 1) return 0;
  return (int64_t)p.splits * ((M + 16 * p.mt - 1) / (16 * p.mt)) * p.mt * ((N + 15) / 16) * 1024;
}

extern "C" int dasa_gemm_w4(const void* x, int64_t ldx, int32_t bf16, const void* weight, const void* scale_tiles,
                            int32_t scale_bf16, int32_t group, const float* bias, int32_t act, float beta, void* y,
                            int64_t ldy, int32_t M, int32_t N, int32_t K, void* ws, int64_t ws_bytes, void* stream) {
  if (M < 0 || !sizes_ok(N, K) || !group_ok(group) || act < DASA_ACT_NONE || act > DASA_ACT_SIGMOID)
    return (int)hipErrorInvalidValue;
  if (M == 0) return 0;
  if (!x || !weight || !scale_tiles || !y || ldx < K || ldy < N || !aligned16(weight) || !aligned16(scale_tiles) ||
      M > 65535 * 16)
    return (int)hipErrorInvalidValue;
  Plan p = plan_of(M, N, K, bf16);
  W4Args a{x, (long)ldx, reinterpret_cast<const uint4*>(weight), scale_tiles, bias, y, (long)ldy, beta, act, M, N, K,
           (K + 127) / 128, (N + 15) / 16, 0, nullptr};
  a.per = (a.Kb + p.splits - 1) / p.splits;
  if (p.splits > 1) {
    if (!ws || !aligned16(ws) || ws_bytes < dasa_gemm_w4_workspace(M, N, K, bf16)) return (int)hipErrorInvalidValue;
    a.part = reinterpret_cast<float4*>(ws);
  }
  hipStream_t st = (hipStream_t)stream;
  if (bf16) return dasa_w4_launch_bf16(a, group, p, scale_bf16, st);
  return scale_bf16 ? w4::launch_plan<float, __bf16>(a, group, p, st) : w4::launch_plan<float, float>(a, group, p, st);
}
