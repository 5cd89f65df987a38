// Differential attention on float elements (kernels: diff_attention.h; entry points: diff_attention.hip).
#include "diff_attention.h"

namespace is {
namespace da {

void run_f32(const Args& a, bool backward, hipStream_t st) {
  const int width = class_of(a);
  if (!a.vec) launch<float, 64, false>(a, backward, st);
  else if (width == 32) launch<float, 32, true>(a, backward, st);
  else if (width == 64) launch<float, 64, true>(a, backward, st);
}

}  // namespace da
}  // namespace is
