// Differential attention on float elements (kernels: diff_attention.h; entry points: diff_attention.hip).
#include "diff_attention.h"

namespace is {
namespace da {

void run_f32(const Args& a, bool backward, hipStream_t st) {
  const int width = class_of(a);
  if (width == 32) backward ? launch_bwd<float, 32>(a, st) : launch_fwd<float, 32>(a, st);
  else if (width == 64) backward ? launch_bwd<float, 64>(a, st) : launch_fwd<float, 64>(a, st);
}

}  // namespace da
}  // namespace is
