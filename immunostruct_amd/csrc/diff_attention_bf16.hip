// Differential attention on __bf16 elements (kernels: diff_attention.h; entry points: diff_attention.hip).
#include "diff_attention.h"

namespace is {
namespace da {

void run_bf16(const Args& a, bool backward, hipStream_t st) {
  const int width = class_of(a);
  if (!a.vec) launch<__bf16, 128, false>(a, backward, st);
  else if (width == 32) launch<__bf16, 32, true>(a, backward, st);
  else if (width == 64) launch<__bf16, 64, true>(a, backward, st);
  else if (width == 128) launch<__bf16, 128, true>(a, backward, st);
}

}  // namespace da
}  // namespace is
