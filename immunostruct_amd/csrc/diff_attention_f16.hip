// Differential attention on _Float16 elements (kernels: diff_attention.h; entry points: diff_attention.hip).
#include "diff_attention.h"

namespace is {
namespace da {

void run_f16(const Args& a, bool backward, hipStream_t st) {
  const int width = class_of(a);
  if (!a.vec) launch<_Float16, 128, false>(a, backward, st);
  else if (width == 32) launch<_Float16, 32, true>(a, backward, st);
  else if (width == 64) launch<_Float16, 64, true>(a, backward, st);
  else if (width == 128) launch<_Float16, 128, true>(a, backward, st);
}

}  // namespace da
}  // namespace is
