// The forms of f8_linear with 16-bit outputs, in a unit of their own.
#include "fp4x_f8_forms.h"

namespace fp4x {

void launch_f8_dense(int form, dim3 grid, const F8Args& a, hipStream_t st) {
  launch_f8_form<false, false>(form, grid, a, st);
}

}  // namespace fp4x
