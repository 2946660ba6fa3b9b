// The launches of f8_linear's forms (fp4x_f8.h), for a unit that fixes EX and B16.
#pragma once
#include "fp4x_f8.h"

namespace fp4x {

template <int F, bool EX, bool B16>
void launch_f8_one(dim3 grid, const F8Args& a, hipStream_t st) {
  if constexpr ((kF8Have[EX][B16] >> F & 1) == 0) return;
  else if constexpr (F == 0) hipLaunchKernelGGL((f8_ring_kernel<1, 1, 8, 2, EX, B16>), grid, dim3(512), 0, st, a);
  else if constexpr (F == 1) hipLaunchKernelGGL((f8_ring_kernel<1, 2, 4, 3, EX, B16>), grid, dim3(256), 0, st, a);
  else if constexpr (F == 2) hipLaunchKernelGGL((f8_ring_kernel<2, 2, 4, 2, EX, B16>), grid, dim3(256), 0, st, a);
  else if constexpr (F == 3) hipLaunchKernelGGL((f8_ring_kernel<2, 4, 4, 2, EX, B16>), grid, dim3(256), 0, st, a);
  else if constexpr (F == 4) launch_f8_tile<64, 64, 2, 2, 4, EX, B16>(grid, a, st);
  else if constexpr (F == 5) launch_f8_tile<64, 128, 2, 2, 3, EX, B16>(grid, a, st);
  else if constexpr (F == 6) launch_f8_tile<128, 128, 4, 2, 4, EX, B16>(grid, a, st);
  else if constexpr (F == 7) launch_f8_tile<128, 128, 2, 2, 2, EX, B16>(grid, a, st);
  else if constexpr (F == 8) launch_f8_tile<256, 128, 4, 2, 3, EX, B16>(grid, a, st);
  else launch_f8_tile<256, 256, 2, 4, 2, EX, B16>(grid, a, st);
}

template <bool EX, bool B16>
void launch_f8_form(int form, dim3 grid, const F8Args& a, hipStream_t st) {
  switch (form) {
    case 0: launch_f8_one<0, EX, B16>(grid, a, st); break;
    case 1: launch_f8_one<1, EX, B16>(grid, a, st); break;
    case 2: launch_f8_one<2, EX, B16>(grid, a, st); break;
    case 3: launch_f8_one<3, EX, B16>(grid, a, st); break;
    case 4: launch_f8_one<4, EX, B16>(grid, a, st); break;
    case 5: launch_f8_one<5, EX, B16>(grid, a, st); break;
    case 6: launch_f8_one<6, EX, B16>(grid, a, st); break;
    case 7: launch_f8_one<7, EX, B16>(grid, a, st); break;
    case 8: launch_f8_one<8, EX, B16>(grid, a, st); break;
    default: launch_f8_one<9, EX, B16>(grid, a, st);
  }
}

}  // namespace fp4x
