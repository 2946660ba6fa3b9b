// The largest tiles of w8a8_linear (fp4x_i8.h), in a unit of their own.
#include "fp4x_i8.h"

namespace fp4x {

void launch_i8_256x128(dim3 grid, const I8Args& a, hipStream_t st) { launch_i8_tile<256, 128, 4, 2, 3>(grid, a, st); }
void launch_i8_256x256(dim3 grid, const I8Args& a, hipStream_t st) { launch_i8_tile<256, 256, 2, 4, 2>(grid, a, st); }

}  // namespace fp4x
