// Differential attention on __bf16 elements (kernels: diff_attention.h; entry points: diff_attention.hip).
#include "diff_attention.h"

namespace is {
namespace da {

void run_bf16(const Args& a, bool backward, hipStream_t st) {
  const int width = class_of(a);
  if (width == 32) backward ? launch_bwd<__bf16, 32>(a, st) : launch_fwd<__bf16, 32>(a, st);
  else if (width == 64) backward ? launch_bwd<__bf16, 64>(a, st) : launch_fwd<__bf16, 64>(a, st);
  else if (width == 128) backward ? launch_bwd<__bf16, 128>(a, st) : launch_fwd<__bf16, 128>(a, st);
}

}  // namespace da
}  // namespace is
