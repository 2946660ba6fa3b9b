// w8a8_linear: which form a size takes, its launch and the C entry points
// (kernels: fp4x_i8.h).
#include <string>

#include "fp4x_i8.h"
#include "../../include/fp4x.h"

namespace fp4x {

int device_cus();

// ------------------------------------------------------------------ choice
constexpr int64_t kI8MaxStride = (1 << 24) - 16;   // 256 rows within 32-bit offsets

// Forms are ranked by a + n (b + d k) us: n tiles fall to the busiest CU, each
// with k = ceil(K / 128) k-tiles.  a, b and d are fitted to 490 sizes (1 to 4096
// rows, 16 to 18000 columns, K from 64 to 10240, most of them drawn evenly over
// their logarithms; weights from HBM), and the form with the least estimate is
// taken.  Over the 608 sizes on record it takes 0.7% more than the fastest on
// average at 489 of the fit and 1.6% at 119 that the fit has not seen, 24% at
// most.  Leaving any one form out costs 0.1 to 4.5% on average and 19 to 104% at
// one size.  As a time the estimate of the chosen form is good to -6 .. +37% at
// 90% of the sizes, and up to 2.4 times too low where few rows wait for the
// weights' bytes, which it does not count.
struct I8Form { int bm, bn, slots, ring, stages; float a, b, d; };
constexpr I8Form kI8Forms[] = {
    {16, 16, 2, 1, 2, 2.14f, 0.53f, 0.028f}, {16, 32, 2, 1, 3, 2.13f, 0.57f, 0.061f},
    {16, 64, 2, 1, 2, 2.26f, 0.62f, 0.111f}, {32, 32, 2, 1, 2, 2.18f, 0.59f, 0.076f},
    {32, 64, 1, 1, 2, 1.32f, 2.20f, 0.144f}, {64, 64, 2, 0, 4, 2.67f, 0.77f, 0.276f},
    {64, 128, 2, 0, 3, 2.93f, 1.12f, 0.312f}, {128, 128, 1, 0, 4, 0.89f, 2.80f, 0.519f},
    {128, 128, 2, 0, 2, 3.00f, 1.72f, 0.583f}, {256, 128, 1, 0, 3, 2.43f, 4.24f, 0.855f},
    {256, 256, 1, 0, 2, 5.83f, 5.42f, 1.341f}};

template <int F>
static void launch_i8(I8Args a, hipStream_t st) {
  constexpr I8Form f = kI8Forms[F];
  a.mt = (a.M + f.bm - 1) / f.bm;
  a.nt = (a.N + f.bn - 1) / f.bn;
  a.gm = f.ring ? a.mt : 4;                        // 4 x 8 tiles of 256 x 256 are what the CUs of an XCD work on
  const int tiles = a.mt * a.nt, slots = f.slots * device_cus();
  // Several tiles per workgroup only where a tile has more k-tiles than the ring has stages: the scales of tile t + 2
  // take the place of tile t's when the last load of tile t + 1 is out, which is then behind a barrier that every wave
  // comes to after its part of tile t's epilogue.
  const dim3 grid(!f.ring && tiles > slots && (a.K + 127) / 128 > f.stages ? slots : tiles);
  if constexpr (F == 0) hipLaunchKernelGGL((i8_ring_kernel<1, 1, 8, 2>), grid, dim3(512), 0, st, a);
  else if constexpr (F == 1) hipLaunchKernelGGL((i8_ring_kernel<1, 2, 4, 3>), grid, dim3(256), 0, st, a);
  else if constexpr (F == 2) hipLaunchKernelGGL((i8_ring_kernel<1, 4, 4, 2>), grid, dim3(256), 0, st, a);
  else if constexpr (F == 3) hipLaunchKernelGGL((i8_ring_kernel<2, 2, 4, 2>), grid, dim3(256), 0, st, a);
  else if constexpr (F == 4) hipLaunchKernelGGL((i8_ring_kernel<2, 4, 4, 2>), grid, dim3(256), 0, st, a);
  else if constexpr (F == 5) launch_i8_tile<64, 64, 2, 2, 4>(grid, a, st);
  else if constexpr (F == 6) launch_i8_tile<64, 128, 2, 2, 3>(grid, a, st);
  else if constexpr (F == 7) launch_i8_tile<128, 128, 4, 2, 4>(grid, a, st);
  else if constexpr (F == 8) launch_i8_tile<128, 128, 2, 2, 2>(grid, a, st);
  else if constexpr (F == 9) launch_i8_256x128(grid, a, st);
  else launch_i8_256x256(grid, a, st);
}

static int choose_i8(int M, int N, int K) {
  const int cus = device_cus();
  const float k = (float)((K + 127) / 128);
  int best = 0;
  float least = 0.0f;
  for (int f = 0; f < (int)(sizeof(kI8Forms) / sizeof(kI8Forms[0])); ++f) {
    const I8Form& c = kI8Forms[f];
    const int64_t tiles = (int64_t)((M + c.bm - 1) / c.bm) * ((N + c.bn - 1) / c.bn);
    const float time = c.a + (float)((tiles + cus - 1) / cus) * (c.b + c.d * k);
    if (f == 0 || time < least) {
      least = time;
      best = f;
    }
  }
  return best;
}

}  // namespace fp4x

using namespace fp4x;

extern "C" {

int fp4x_w8a8_form(int M, int N, int K) { return M < 1 || N < 1 || K < 1 ? -1 : choose_i8(M, N, K); }

int fp4x_w8a8_linear(const void* xq, int64_t x_stride, const float* xs, const void* wq, int64_t w_stride,
                     const float* ws, const float* bias, void* out, int64_t out_stride, int out_dtype, int M, int N,
                     int K, void* stream) {
  const auto bad = [](const char* why) {
    set_error(std::string("w8a8_linear: ") + why);
    return FP4X_ERR_ARG;
  };
  if (M < 0 || N < 1 || K < 1 || K > 131071) return bad("need M >= 0, N >= 1 and 1 <= K <= 131071 (an int32 sum)");
  if (out_dtype != DT_BF16 && out_dtype != DT_F32 && out_dtype != DT_F16) return bad("out is bf16, fp32 or fp16");
  if (M > 1 << 24 || N > 1 << 24 || (int64_t)M * N > (int64_t)1 << 37) return bad("M and N go to 2^24, M N to 2^37");
  if (M == 0) return FP4X_OK;
  if (!xq || !xs || !wq || !ws || !out) return bad("null tensor");
  const auto al = [](const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  if (!al(xq, 16) || !al(wq, 16) || x_stride % 16 || w_stride % 16 || x_stride < K || w_stride < K)
    return bad("code rows must start on 16 bytes, with strides of at least K");
  if (x_stride > kI8MaxStride || w_stride > kI8MaxStride) return bad("row strides go to 2^24 - 16");
  if (!al(xs, 4) || !al(ws, 4) || !al(bias, 4) || !al(out, out_dtype == DT_F32 ? 4 : 2))
    return bad("scales, bias and output must be aligned to their element");
  if (out_stride < N && M > 1) return bad("output rows overlap");
  const I8Args a{static_cast<const int8_t*>(xq), x_stride, xs, static_cast<const int8_t*>(wq), w_stride, ws, bias, out,
                 out_dtype, out_stride, M, N, K, 0, 0, 0};
  hipStream_t st = (hipStream_t)stream;
  switch (choose_i8(M, N, K)) {
    case 0: launch_i8<0>(a, st); break;
    case 1: launch_i8<1>(a, st); break;
    case 2: launch_i8<2>(a, st); break;
    case 3: launch_i8<3>(a, st); break;
    case 4: launch_i8<4>(a, st); break;
    case 5: launch_i8<5>(a, st); break;
    case 6: launch_i8<6>(a, st); break;
    case 7: launch_i8<7>(a, st); break;
    case 8: launch_i8<8>(a, st); break;
    case 9: launch_i8<9>(a, st); break;
    default: launch_i8<10>(a, st);
  }
  return check_launch("w8a8_linear");
}

}  // extern "C"
