// The instantiations of the 4-bit products (w4.h) for bf16 activations; a file of their own, so both halves compile
// side by side.
#include "w4.h"

__attribute__((visibility("hidden"))) int dasa_w4_launch_bf16(const w4::W4Args& a, int group, const w4::Plan& p,
                                                              int scale_bf16, hipStream_t st) {
  return scale_bf16 ? w4::launch_plan<__bf16, __bf16>(a, group, p, st) : w4::launch_plan<__bf16, float>(a, group, p, st);
}
