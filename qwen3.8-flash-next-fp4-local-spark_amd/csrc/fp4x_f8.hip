// f8_linear and f8_linear_experts: which form a size takes, its launch and the C
// entry points (kernels: fp4x_f8.h).
#include <cmath>
#include <string>

#include "fp4x_f8.h"
#include "../../include/fp4x.h"

namespace fp4x {

int device_cus();

// ------------------------------------------------------------------ choice
constexpr int64_t kF8MaxStride = (1 << 24) - 16;   // 256 rows within 32-bit offsets
// A grid has fewer than 2^32 lanes, 256 a tile (forms of 512 have fewer tiles at every size that M N allows).
constexpr int64_t kF8MaxTiles = (1 << 24) - 8;

struct F8Form { int bm, bn, slots, ring, stages; };
constexpr F8Form kF8Shape[kF8Forms] = {{16, 16, 2, 1, 2},   {16, 32, 2, 1, 3},   {32, 32, 2, 1, 2},   {32, 64, 1, 1, 2},
                                       {64, 64, 2, 0, 4},   {64, 128, 2, 0, 3},  {128, 128, 1, 0, 4}, {128, 128, 2, 0, 2},
                                       {256, 128, 1, 0, 3}, {256, 256, 1, 0, 2}};

// Forms are ranked by a + n (b + d k): n tiles fall to a CU, each with k = ceil(K / 128) k-tiles, and the one with the least
// is taken.  a, b and d are fitted to 1,000 sizes (1 to 8192 rows, 16 to 18000 columns, K from 64 to 10240; 1 to 512 experts;
// most drawn evenly over their logarithms, weights from HBM), so that the form taken is near the fastest.  The fit is of the
// kernels before code rows started on lines and before 256 x 256 tiles over experts left out halves of their strips; over the
// 997 sizes that profiles/f8_forms.txt lists with the kernels as they are, the form taken is on average 0.4% slower (products,
// 16-bit outputs; 15% at most), 0.8% (fp32 outputs; 22%), 1.4% and 1.1% (over experts; 32% and 16%).  The estimate's values
// are no times: only their order counts.
struct F8Cost { float a, b, d; };
constexpr F8Cost kF8Cost[2][2][kF8Forms] = {
    {{{0.84f, 0.852f, 0.0396f}, {1.12f, 0.858f, 0.0582f}, {1.28f, 1.022f, 0.0661f}, {0.80f, 3.811f, 0.0805f},
      {2.28f, 1.213f, 0.2582f}, {4.64f, 1.748f, 0.2608f}, {0.34f, 6.016f, 0.3885f}, {9.13f, 0.812f, 0.3704f},
      {0.00f, 7.808f, 0.6867f}, {0.00f, 13.045f, 1.0335f}},
     {{0.91f, 1.241f, 0.0302f}, {1.23f, 1.373f, 0.0429f}, {1.32f, 1.652f, 0.0484f}, {}, {3.95f, 0.340f, 0.7088f},
      {5.22f, 2.532f, 0.4773f}, {}, {0.41f, 8.166f, 0.6476f}, {}, {}}},
    {{{}, {0.56f, 1.944f, 0.0740f}, {1.24f, 1.698f, 0.1402f}, {}, {4.23f, 0.710f, 0.3542f}, {4.51f, 0.720f, 0.4488f}, {},
      {5.20f, 0.951f, 0.5319f}, {}, {11.47f, 3.946f, 1.0354f}},
     {{}, {0.64f, 3.149f, 0.0408f}, {1.37f, 3.270f, 0.0583f}, {}, {6.15f, 0.601f, 1.1460f}, {11.16f, 0.760f, 0.5155f}, {},
      {12.76f, 1.004f, 0.6093f}, {}, {}}}};

// rows of tiles: for a form's height, how many.
template <class Rows>
static int f8_best(int ex, bool b16, int N, int K, Rows rows) {
  const float k = (float)((K + 127) / 128), cus = (float)device_cus();
  int best = -1;
  float least = 0.0f;
  for (int f = 0; f < kF8Forms; ++f) {
    if ((kF8Have[ex][b16] >> f & 1) == 0) continue;
    const F8Cost& c = kF8Cost[ex][b16][f];
    float n = rows(kF8Shape[f].bm) * (float)((N + kF8Shape[f].bn - 1) / kF8Shape[f].bn) / cus;
    if (!ex || n < 4.0f) n = std::ceil(n);         // whole rounds, where the number of tiles is known
    const float time = c.a + n * (c.b + c.d * k);
    if (best < 0 || time < least) {
      least = time;
      best = f;
    }
  }
  return best;
}
static int choose_f8(int M, int N, int K, bool b16) {
  return f8_best(0, b16, N, K, [&](int bm) { return (float)((M + bm - 1) / bm); });
}
// As if the pairs fell on the experts evenly: so many are hit, and a hit one's rows end half-way through a tile.  M is all that
// is known here: where part of the pairs have no expert (another rank's), it counts them too, and the tiles are too tall for the
// rows that are left.  4096 tokens x 8 over 512 experts of [1280 x 2560], 64 of them here (3,600 to 5,800 rows kept): 78 us with the
// whole list of tokens, 49 with the list cut to the rows kept, whose number the host must know for that.
static int choose_f8_experts(int M, int N, int K, int E, bool b16) {
  const float hit = E == 1 ? 1.0f : (float)E * (1.0f - std::exp(-(float)M / (float)E)), mean = (float)M / hit;
  return f8_best(1, b16, N, K, [&](int bm) { return hit * (mean <= 0.7f * (float)bm ? 1.0f : mean / (float)bm + 0.5f); });
}

static int f8_streams(int64_t M, int64_t N, int out_dtype) { return M * N * (out_dtype == DT_F32 ? 4 : 2) > 32 << 20; }

static int f8_fail(const char* what, const char* why) {
  set_error(std::string(what) + ": " + why);
  return FP4X_ERR_ARG;
}

// What both entry points ask of their arguments; 0 rows: nothing else is looked at.
static int f8_check(const char* what, const F8Args& a) {
  if (a.M < 0 || a.N < 1 || a.K < 1 || a.K > 131071) return f8_fail(what, "need M >= 0, N >= 1 and 1 <= K <= 131071");
  if (a.out_dtype != DT_BF16 && a.out_dtype != DT_F32 && a.out_dtype != DT_F16) return f8_fail(what, "out is bf16, fp32 or fp16");
  if (a.M > 1 << 24 || a.N > 1 << 24 || (int64_t)a.M * a.N > (int64_t)1 << 37) return f8_fail(what, "M and N go to 2^24, M N to 2^37");
  if (a.M == 0) return FP4X_OK;
  if (!a.x || !a.sx || !a.w || !a.sw || !a.out) return f8_fail(what, "null tensor");
  const auto al = [](const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  if (!al(a.x, 16) || !al(a.w, 16) || a.x_stride % 16 || a.w_stride % 16 || a.w_estride % 16 || a.x_stride < a.K || a.w_stride < a.K)
    return f8_fail(what, "code rows must start on 16 bytes, with strides of at least K");
  if (a.x_stride > kF8MaxStride || a.w_stride > kF8MaxStride) return f8_fail(what, "row strides go to 2^24 - 16");
  if (a.sx_m < 0 || a.sx_b < 0 || a.sx_m >= 1 << 22) return f8_fail(what, "scale strides are not negative, between rows below 2^22");
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
           ws, bias, out, out_dtype, out_stride, M, N, K, 0, 0, 0, f8_streams(M, N, out_dtype), nullptr, nullptr, 1, M, 0};
  if (int rc = f8_check("f8_linear", a)) return rc;
  if (M == 0) return FP4X_OK;
  const bool b16 = out_dtype == DT_F32;
  const int form = choose_f8(M, N, K, b16);
  const F8Form& f = kF8Shape[form];
  a.mt = (M + f.bm - 1) / f.bm;
  a.nt = (N + f.bn - 1) / f.bn;
  a.gm = f.ring ? a.mt : 4;                        // 4 x 8 tiles of 256 x 256 are what the CUs of an XCD work on
  const int tiles = a.mt * a.nt, slots = f.slots * device_cus();
  if (tiles >= kF8MaxTiles) return f8_fail("f8_linear", "2^24 tiles or more");
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
           ws, nullptr, out, out_dtype, out_stride, P, N, K, 0, 0, 0, f8_streams(P, N, out_dtype), offsets, tokens, E, X, w_expert};
  if (E < 1 || E > kF8MaxExperts) return f8_fail(what, "1 to 4096 experts");
  if (int rc = f8_check(what, a)) return rc;
  if (P == 0) return FP4X_OK;
  if (!offsets || (reinterpret_cast<uintptr_t>(offsets) & 3) || (reinterpret_cast<uintptr_t>(tokens) & 3))
    return f8_fail(what, "null or misaligned offsets, or misaligned tokens");
  if (w_expert < 0) return f8_fail(what, "a weight's stride is negative");
  if (tokens) {
    if (X < 1) return f8_fail(what, "there are no rows to pick from");
    if ((int64_t)X * x_stride > (int64_t)UINT32_MAX || (int64_t)X * xs_row * 4 > (int64_t)UINT32_MAX) return f8_fail(what, "rows that are picked, and their scales, lie within 2^32 bytes");
  } else if (X < P) {
    return f8_fail(what, "fewer rows than the output has");
  }
  const bool b16 = out_dtype == DT_F32;
  const int form = choose_f8_experts(P, N, K, E, b16);
  const F8Form& f = kF8Shape[form];
  a.nt = (N + f.bn - 1) / f.bn;
  // every expert with a row may end in a tile of its own that is not full
  const int64_t hit = std::min(P, E), tiles = ((P - hit) / f.bm + hit) * a.nt;
  // large tiles: a workgroup takes several, 34 at most (lane j of its waves holds the place of tile j)
  const int64_t slots = f.slots * device_cus(), grid = f.ring ? tiles : std::min(tiles, std::max(slots, (tiles + 31) / 32));
  if (grid >= kF8MaxTiles) return f8_fail(what, "2^24 tiles or more");
  (b16 ? launch_f8_experts_b16 : launch_f8_experts)(form, dim3((unsigned)((grid + 7) / 8 * 8)), a, (hipStream_t)stream);
  return check_launch(what);
}

}  // extern "C"
