// f8_linear and f8_linear_experts: which form a size takes, its launch and the C
// entry points (kernels: fp4x_f8.h).
#include <string>

#include "fp4x_f8.h"
#include "../../include/fp4x.h"

namespace fp4x {

int device_cus();

// ------------------------------------------------------------------ choice
constexpr int64_t kF8MaxStride = (1 << 24) - 16;   // 256 rows within 32-bit offsets

struct F8Form { int bm, bn, slots, ring, stages; float a, b, d; };
constexpr F8Form kF8Forms[] = {
    {16, 16, 2, 1, 2, 2.14f, 0.53f, 0.028f}, {16, 32, 2, 1, 3, 2.13f, 0.57f, 0.061f},
    {16, 64, 2, 1, 2, 2.26f, 0.62f, 0.111f}, {32, 32, 2, 1, 2, 2.18f, 0.59f, 0.076f},
    {32, 64, 1, 1, 2, 1.32f, 2.20f, 0.144f}, {64, 64, 2, 0, 4, 2.67f, 0.77f, 0.276f},
    {64, 128, 2, 0, 3, 2.93f, 1.12f, 0.312f}, {128, 128, 1, 0, 4, 0.89f, 2.80f, 0.519f},
    {128, 128, 2, 0, 2, 3.00f, 1.72f, 0.583f}, {256, 128, 1, 0, 3, 2.43f, 4.24f, 0.855f},
    {256, 256, 1, 0, 2, 5.83f, 5.42f, 1.341f}};
constexpr int kF8Count = sizeof(kF8Forms) / sizeof(kF8Forms[0]);

static int f8_best(int K, bool b16, int64_t (*tiles)(const F8Form&, int64_t, int64_t, int64_t), int64_t M, int64_t N, int64_t E) {
  const int cus = device_cus();
  const float k = (float)((K + 127) / 128);
  int best = 0;
  float least = 0.0f;
  for (int f = 0; f < kF8Count - b16; ++f) {     // (the last form has no bf16 products)
    const F8Form& c = kF8Forms[f];
    const float time = c.a + (float)((tiles(c, M, N, E) + cus - 1) / cus) * (c.b + c.d * k);
    if (f == 0 || time < least) {
      least = time;
      best = f;
    }
  }
  return best;
}
static int choose_f8(int M, int N, int K, bool b16) {
  return f8_best(K, b16, [](const F8Form& c, int64_t M, int64_t N, int64_t) {
    return (M + c.bm - 1) / c.bm * ((N + c.bn - 1) / c.bn);
  }, M, N, 1);
}
// As if each expert that can have a row had the mean of the rows.
static int choose_f8_experts(int M, int N, int K, int E, bool b16) {
  return f8_best(K, b16, [](const F8Form& c, int64_t M, int64_t N, int64_t E) {
    const int64_t hit = std::min(M, E), rows = (M + hit - 1) / hit;
    return hit * ((rows + c.bm - 1) / c.bm) * ((N + c.bn - 1) / c.bn);
  }, M, N, E);
}

static int f8_fail(const char* what, const char* why) {
  set_error(std::string(what) + ": " + why);
  return FP4X_ERR_ARG;
}

// What both entry points ask of their arguments; 0 rows: nothing else is looked at.
static int f8_check(const char* what, const F8Args& a) {
  if (a.M < 0 || a.N < 1 || a.K < 1 || a.K > 1 << 24) return f8_fail(what, "need M >= 0, N >= 1 and 1 <= K <= 2^24");
  if (a.out_dtype != DT_BF16 && a.out_dtype != DT_F32 && a.out_dtype != DT_F16) return f8_fail(what, "out is bf16, fp32 or fp16");
  if (a.M > 1 << 24 || a.N > 1 << 24 || (int64_t)a.M * a.N > (int64_t)1 << 37) return f8_fail(what, "M and N go to 2^24, M N to 2^37");
  if (a.M == 0) return FP4X_OK;
  if (!a.x || !a.sx || !a.w || !a.sw || !a.out) return f8_fail(what, "null tensor");
  const auto al = [](const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  if (!al(a.x, 16) || !al(a.w, 16) || a.x_stride % 16 || a.w_stride % 16 || a.w_estride % 16 || a.x_stride < a.K || a.w_stride < a.K)
    return f8_fail(what, "code rows must start on 16 bytes, with strides of at least K");
  if (a.x_stride > kF8MaxStride || a.w_stride > kF8MaxStride) return f8_fail(what, "row strides go to 2^24 - 16");
  if (a.sx_m < 0 || a.sx_b < 0) return f8_fail(what, "a scale stride is negative");
  if (!al(a.sx, 4) || !al(a.sw, 4) || !al(a.bias, 4) || !al(a.out, a.out_dtype == DT_F32 ? 4 : 2))
    return f8_fail(what, "scales, bias and output must be aligned to their element");
  if (a.out_stride < a.N && a.M > 1) return f8_fail(what, "output rows overlap");
  return FP4X_OK;
}

}  // namespace fp4x

using namespace fp4x;

extern "C" {

int fp4x_f8_form(int M, int N, int K, int out_dtype) {
  return M < 1 || N < 1 || K < 1 ? -1 : choose_f8(M, N, K, out_dtype == DT_F32);
}

int fp4x_f8_linear(const void* xq, int64_t x_stride, const float* xs, int64_t xs_row, int64_t xs_block, const void* wq,
                   int64_t w_stride, const float* ws, const float* bias, void* out, int64_t out_stride, int out_dtype,
                   int M, int N, int K, void* stream) {
  F8Args a{static_cast<const uint8_t*>(xq), x_stride, xs, xs_row, xs_block, static_cast<const uint8_t*>(wq), w_stride,
           ws, bias, out, out_dtype, out_stride, M, N, K, 0, 0, 0, nullptr, nullptr, 1, M, 0};
  if (int rc = f8_check("f8_linear", a)) return rc;
  if (M == 0) return FP4X_OK;
  const bool b16 = out_dtype == DT_F32;
  const int form = choose_f8(M, N, K, b16);
  const F8Form& f = kF8Forms[form];
  a.mt = (M + f.bm - 1) / f.bm;
  a.nt = (N + f.bn - 1) / f.bn;
  a.gm = f.ring ? a.mt : 4;                        // 4 x 8 tiles of 256 x 256 are what the CUs of an XCD work on
  const int tiles = a.mt * a.nt, slots = f.slots * device_cus();
  // Several tiles per workgroup only where a tile has more k-tiles than the ring has stages: the bias of tile t + 2
  // takes the place of tile t's when the last load of tile t + 1 is out, which is then behind a barrier that every wave
  // comes to after its part of tile t's epilogue.
  const dim3 grid(!f.ring && tiles > slots && (K + 127) / 128 > f.stages ? slots : tiles);
  (b16 ? launch_f8_dense_b16 : launch_f8_dense)(form, grid, a, (hipStream_t)stream);
  return check_launch("f8_linear");
}

int fp4x_f8_experts_form(int P, int N, int K, int E, int out_dtype) {
  return P < 1 || N < 1 || K < 1 || E < 1 ? -1 : choose_f8_experts(P, N, K, E, out_dtype == DT_F32);
}

int fp4x_f8_linear_experts(const void* xq, int64_t x_stride, const float* xs, int64_t xs_row, int64_t xs_block, int X,
                           const int* tokens, const int* offsets, int E, const void* wq, int64_t w_stride,
                           int64_t w_expert, const float* ws, void* out, int64_t out_stride, int out_dtype, int P,
                           int N, int K, void* stream) {
  const char* what = "f8_linear_experts";
  F8Args a{static_cast<const uint8_t*>(xq), x_stride, xs, xs_row, xs_block, static_cast<const uint8_t*>(wq), w_stride,
           ws, nullptr, out, out_dtype, out_stride, P, N, K, 0, 0, 0, offsets, tokens, E, X, w_expert};
  if (E < 1 || E > kF8MaxExperts) return f8_fail(what, "1 to 4096 experts");
  if (int rc = f8_check(what, a)) return rc;
  if (P == 0) return FP4X_OK;
  if (!offsets || (reinterpret_cast<uintptr_t>(offsets) & 3) || (reinterpret_cast<uintptr_t>(tokens) & 3))
    return f8_fail(what, "null or misaligned offsets, or misaligned tokens");
  if (w_expert < 0) return f8_fail(what, "a weight's stride is negative");
  if (tokens) {
    if (X < 1) return f8_fail(what, "there are no rows to pick from");
    if ((int64_t)X * x_stride > (int64_t)UINT32_MAX) return f8_fail(what, "rows that are picked lie within 2^32 bytes");
  } else if (X < P) {
    return f8_fail(what, "fewer rows than the output has");
  }
  const bool b16 = out_dtype == DT_F32;
  const int form = choose_f8_experts(P, N, K, E, b16);
  const F8Form& f = kF8Forms[form];
  a.nt = (N + f.bn - 1) / f.bn;
  // every expert with a row may end in a tile of its own that is not full
  const int64_t hit = std::min(P, E), tiles = ((P - hit) / f.bm + hit) * a.nt;
  if (tiles > INT32_MAX) return f8_fail(what, "more than 2^31 - 1 tiles");
  (b16 ? launch_f8_experts_b16 : launch_f8_experts)(form, dim3((unsigned)tiles), a, (hipStream_t)stream);
  return check_launch(what);
}

}  // extern "C"
