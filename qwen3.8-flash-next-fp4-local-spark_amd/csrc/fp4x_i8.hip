// Products of 8-bit integers: out[m, n] = cast((sum_k x[m, k] w[n, k]) * sx[m]
// * sw[n] + b[n]), x int8 [M, K] with a scale per row (token), w int8 [N, K]
// with a scale per row (output channel), summed in int32: exact for K up to
// 131,071 (|x w| <= 2^14), so no order of the sum changes a result.
#include <algorithm>

#include "fp4x_kernels.h"
#include "../../include/fp4x.h"

namespace fp4x {

int device_cus();

typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2_a2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef __attribute__((address_space(3))) void* i8_lds_t;

struct I8Args {
  const int8_t* x;  int64_t x_stride;  const float* sx;
  const int8_t* w;  int64_t w_stride;  const float* sw;
  const float* bias;
  void* out;  int out_dtype;  int64_t out_stride;
  int M, N, K;
};

// Bytes [c * 16, c * 16 + 16) of a row with those from K on as zeros.
__device__ __forceinline__ i32x4_t keep_to(i32x4_t v, int c, int K) {
  const int n = K - c * 16;
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const int left = n - 4 * d;
    v[d] = left >= 4 ? v[d] : left <= 0 ? 0 : v[d] & (int)((1u << (8 * left)) - 1u);
  }
  return v;
}

// Four neighbouring columns [n, n + 4) of row m; columns from N on are left out.
__device__ __forceinline__ void i8_store4(const I8Args& a, int64_t m, int n, i32x4_t acc, float sx) {
  float v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int nj = n + j < a.N ? n + j : a.N - 1;
    v[j] = ((float)acc[j] * sx) * a.sw[nj];
    if (a.bias) v[j] = v[j] + a.bias[nj];
  }
  const int64_t at = m * a.out_stride + n;
  if (n + 4 > a.N) {
    for (int j = 0; j < 4 && n + j < a.N; ++j) store_out(a.out, at + j, a.out_dtype, v[j]);
  } else if (a.out_dtype == DT_F32) {
    *reinterpret_cast<u32x4_a4*>(static_cast<float*>(a.out) + at) = u32x4_a4{
        __float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
  } else {
    uint32_t p[2];
    if (a.out_dtype == DT_BF16) { p[0] = pack_bf16x2(v[0], v[1]); p[1] = pack_bf16x2(v[2], v[3]); }
    else {
#pragma unroll
      for (int j = 0; j < 2; ++j)
        p[j] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * j]) |
               (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * j + 1]) << 16;
    }
    *reinterpret_cast<u32x2_a2*>(static_cast<uint16_t*>(a.out) + at) = u32x2_a2{p[0], p[1]};
  }
}

// ------------------------------------------------------------------ few rows
// A workgroup owns 16 MT rows of x and 16 NT rows of w; its W waves split K,
// and each wave reads its operands straight into registers (lane (i, g): 16
// bytes of row i at chunk 4 u + g of unit u), U units of 64 values at a time.
// The waves' integer sums meet in LDS.
template <int MT, int NT, int U, bool TAIL>
struct I8Batch {
  i32x4_t x[U][MT], w[U][NT];
  // TAIL: units from `end` on and chunks from K on count as zeros (x is cleared; w reads the row's last chunk)
  __device__ __forceinline__ void load(const int8_t* const (&xr)[MT], const int8_t* const (&wr)[NT], int u, int end,
                                       int K, int g) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      int c = (u + j) * 4 + g;
      const int last = (K - 1) >> 4, cc = TAIL && c > last ? last : c;
#pragma unroll
      for (int t = 0; t < NT; ++t) w[j][t] = *reinterpret_cast<const i32x4_t*>(wr[t] + cc * 16);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        x[j][t] = *reinterpret_cast<const i32x4_t*>(xr[t] + cc * 16);
        if (TAIL) x[j][t] = keep_to(x[j][t], u + j < end ? c : 1 << 26, K);
      }
    }
  }
  __device__ __forceinline__ void mul(i32x4_t (&acc)[MT][NT]) const {
#pragma unroll
    for (int j = 0; j < U; ++j)
#pragma unroll
      for (int s = 0; s < MT; ++s)
#pragma unroll
        for (int t = 0; t < NT; ++t)
          acc[s][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[j][t], x[j][s], acc[s][t], 0, 0, 0);
  }
};

template <int MT, int NT, int W, int U>
__global__ __launch_bounds__(64 * W) void i8_rows_kernel(const I8Args a) {
  constexpr int LD = 16 * NT + 4;                  // (a row of sums starts on 16 bytes)
  __shared__ int sum[16 * MT * LD];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, i = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16 * MT;
  for (int e = t; e < 16 * MT * LD; e += 64 * W) sum[e] = 0;
  const int8_t *xr[MT], *wr[NT];
#pragma unroll
  for (int s = 0; s < MT; ++s) xr[s] = a.x + (int64_t)min(m0 + 16 * s + i, a.M - 1) * a.x_stride;
#pragma unroll
  for (int s = 0; s < NT; ++s) wr[s] = a.w + (int64_t)min(n0 + 16 * s + i, a.N - 1) * a.w_stride;
  const int units = (a.K + 63) >> 6, per = (units + W - 1) / W;
  const int u0 = wave * per, u1 = min(u0 + per, units);
  const int full = min(u1, a.K >> 6);              // units of this wave before one that K ends in
  i32x4_t acc[MT][NT];
#pragma unroll
  for (int s = 0; s < MT; ++s)
#pragma unroll
    for (int r = 0; r < NT; ++r) acc[s][r] = i32x4_t{0, 0, 0, 0};
  int u = u0;
  if (u + U <= full) {
    I8Batch<MT, NT, U, false> b;
    b.load(xr, wr, u, u1, a.K, g);
    for (u += U; u + U <= full; u += U) {
      I8Batch<MT, NT, U, false> c;
      c.load(xr, wr, u, u1, a.K, g);
      b.mul(acc);
      b = c;
    }
    b.mul(acc);
  }
  for (; u < u1; u += U) {
    I8Batch<MT, NT, U, true> b;
    b.load(xr, wr, u, u1, a.K, g);
    b.mul(acc);
  }
  __syncthreads();
#pragma unroll
  for (int s = 0; s < MT; ++s)
#pragma unroll
    for (int r = 0; r < NT; ++r)
#pragma unroll
      for (int j = 0; j < 4; ++j) atomicAdd(&sum[(16 * s + i) * LD + 16 * r + 4 * g + j], acc[s][r][j]);
  __syncthreads();
  for (int e = t; e < 16 * MT * 4 * NT; e += 64 * W) {
    const int m = e / (4 * NT), c = e % (4 * NT);
    if (m0 + m < a.M && n0 + 4 * c < a.N)
      i8_store4(a, m0 + m, n0 + 4 * c, *reinterpret_cast<const i32x4_t*>(&sum[m * LD + 4 * c]), a.sx[m0 + m]);
  }
}

// ------------------------------------------------------------------ many rows
// A workgroup owns BM rows of x and BN rows of w, and walks K in tiles of 128
// bytes through two LDS stages filled by direct loads: while one is multiplied
// the other is on its way.  Row r's 16-byte chunk c lies at chunk c ^ key of
// its 128 bytes, so that the 16 lanes that LDS serves together read different
// banks.  Wave (wm, wn) owns 32 MI rows of x and 32 NI of w; a weight block's
// MFMA row p holds weight row 16 ((p >> 2) & 1) + 4 (p >> 3) + (p & 3), which
// gives lane (m, h) the 16 neighbouring columns [16 h, 16 h + 16) of row m.
__device__ __forceinline__ int i8_perm(int p) { return 16 * ((p >> 2) & 1) + 4 * (p >> 3) + (p & 3); }
__device__ __forceinline__ int i8_unperm(int r) { return ((r >> 2) & 3) * 8 + ((r >> 4) & 1) * 4 + (r & 3); }

template <int BM, int BN, int WM, int WN>
struct I8Tile {
  static constexpr int T = 64 * WM * WN, W = WM * WN;
  static constexpr int MI = BM / WM / 32, NI = BN / WN / 32;
  static constexpr int STAGE = (BM + BN) * 128, NL = STAGE / 1024 / W;
  static_assert(MI * 32 * WM == BM && NI * 32 * WN == BN && NL * 1024 * W == STAGE && BM / 8 % NL == 0, "tile");
};

template <int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void i8_tile_kernel(const I8Args a, int mtiles, int ntiles) {
  using C = I8Tile<BM, BN, WM, WN>;
  __shared__ char st0[C::STAGE], st1[C::STAGE];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int m0 = blockIdx.x % mtiles * BM, n0 = blockIdx.x / mtiles * BN;
  // direct loads: item e covers LDS rows [8 e, 8 e + 8); the first BM rows are x's
  const int8_t* src[C::NL];
  int chunk[C::NL];
#pragma unroll
  for (int j = 0; j < C::NL; ++j) {
    const int e = wave * C::NL + j, r = e * 8 + (lane >> 3);
    const bool isx = e * 8 < BM;
    const int wr = r - BM, key = isx ? (r >> 1) & 7 : (i8_unperm(wr & 31) >> 1) & 7;
    chunk[j] = (lane & 7) ^ key;
    src[j] = isx ? a.x + (int64_t)min(m0 + r, a.M - 1) * a.x_stride : a.w + (int64_t)min(n0 + wr, a.N - 1) * a.w_stride;
    src[j] += chunk[j] * 16;
  }
  const int last = (a.K - 1) >> 4;
  const auto issue = [&](char* st, int kt) {
#pragma unroll
    for (int j = 0; j < C::NL; ++j) {
      const int over = kt * 8 + chunk[j] - last;   // chunks past the row's last one read that one
      const int8_t* p = src[j] + kt * 128 - (over > 0 ? over * 16 : 0);
      __builtin_amdgcn_global_load_lds(p, (i8_lds_t)(st + (wave * C::NL + j) * 1024), 16, 0, 0);
    }
  };
  const int wm = wave % WM, wn = wave / WM, i = lane & 31, h = lane >> 5;
  const int xkey = (i >> 1) & 7, xrow = wm * 32 * C::MI + i, wrow = BM + wn * 32 * C::NI + i8_perm(i);
  i32x16_t acc[C::MI][C::NI];
#pragma unroll
  for (int s = 0; s < C::MI; ++s)
#pragma unroll
    for (int r = 0; r < C::NI; ++r)
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[s][r][j] = 0;
  const auto step = [&](const char* st, int kt, bool tail) {
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      const int at = ((kk * 2 + h) ^ xkey) * 16;
      i32x4_t x[C::MI], w[C::NI];
#pragma unroll
      for (int r = 0; r < C::NI; ++r) w[r] = *reinterpret_cast<const i32x4_t*>(st + (wrow + 32 * r) * 128 + at);
#pragma unroll
      for (int s = 0; s < C::MI; ++s) {
        x[s] = *reinterpret_cast<const i32x4_t*>(st + (xrow + 32 * s) * 128 + at);
        if (tail) x[s] = keep_to(x[s], kt * 8 + kk * 2 + h, a.K);
      }
#pragma unroll
      for (int s = 0; s < C::MI; ++s)
#pragma unroll
        for (int r = 0; r < C::NI; ++r)
          acc[s][r] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[r], x[s], acc[s][r], 0, 0, 0);
    }
  };
  const int kts = (a.K + 127) >> 7, whole = a.K >> 7;
  issue(st0, 0);
  int kt = 0;
  for (; kt + 2 <= whole; kt += 2) {
    __syncthreads();
    if (kt + 1 < kts) issue(st1, kt + 1);
    step(st0, kt, false);
    __syncthreads();
    if (kt + 2 < kts) issue(st0, kt + 2);
    step(st1, kt + 1, false);
  }
  if (kt < kts) {                                  // one or two tiles, the last of which K may end in
    __syncthreads();
    if (kt + 1 < kts) issue(st1, kt + 1);
    step(st0, kt, true);
    if (kt + 1 < kts) {
      __syncthreads();
      step(st1, kt + 1, true);
    }
  }
#pragma unroll
  for (int s = 0; s < C::MI; ++s) {
    const int m = m0 + wm * 32 * C::MI + 32 * s + i;
    if (m < a.M) {
      const float sx = a.sx[m];
#pragma unroll
      for (int r = 0; r < C::NI; ++r)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int n = n0 + wn * 32 * C::NI + 32 * r + 16 * h + 4 * q;
          if (n < a.N)
            i8_store4(a, m, n, i32x4_t{acc[s][r][4 * q], acc[s][r][4 * q + 1], acc[s][r][4 * q + 2], acc[s][r][4 * q + 3]},
                      sx);
        }
    }
  }
}

template <int MT, int NT, int W, int U>
static void launch_i8_rows(const I8Args& a, hipStream_t st) {
  hipLaunchKernelGGL((i8_rows_kernel<MT, NT, W, U>), dim3((a.N + 16 * NT - 1) / (16 * NT), (a.M + 16 * MT - 1) / (16 * MT)),
                     dim3(64 * W), 0, st, a);
}
template <int BM, int BN, int WM, int WN>
static void launch_i8_tile(const I8Args& a, hipStream_t st) {
  const int mt = (a.M + BM - 1) / BM, nt = (a.N + BN - 1) / BN;
  hipLaunchKernelGGL((i8_tile_kernel<BM, BN, WM, WN>), dim3((unsigned)mt * nt), dim3(64 * WM * WN), 0, st, a, mt, nt);
}

}  // namespace fp4x

using namespace fp4x;

extern "C" {

int fp4x_w8a8_linear(const void* xq, int64_t x_stride, const float* xs, const void* wq, int64_t w_stride,
                     const float* ws, const float* bias, void* out, int64_t out_stride, int out_dtype, int M, int N,
                     int K, void* stream) {
  const auto bad = [](const char* why) {
    set_error(std::string("w8a8_linear: ") + why);
    return FP4X_ERR_ARG;
  };
  if (M < 0 || N < 1 || K < 1 || K > 131071) return bad("need M >= 0, N >= 1 and 1 <= K <= 131071 (an int32 sum)");
  if (out_dtype != DT_BF16 && out_dtype != DT_F32 && out_dtype != DT_F16) return bad("out is bf16, fp32 or fp16");
  if (M > 1 << 24 || N > 1 << 24) return bad("M and N go to 2^24");
  if (M == 0) return FP4X_OK;
  if (!xq || !xs || !wq || !ws || !out) return bad("null tensor");
  const auto al = [](const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  if (!al(xq, 16) || !al(wq, 16) || x_stride % 16 || w_stride % 16 || x_stride < K || w_stride < K)
    return bad("code rows must start on 16 bytes, with strides of at least K");
  if (!al(xs, 4) || !al(ws, 4) || !al(bias, 4) || !al(out, out_dtype == DT_F32 ? 4 : 2))
    return bad("scales, bias and output must be aligned to their element");
  if (out_stride < N && M > 1) return bad("output rows overlap");
  const I8Args a{static_cast<const int8_t*>(xq), x_stride, xs, static_cast<const int8_t*>(wq), w_stride, ws, bias, out,
                 out_dtype, out_stride, M, N, K};
  hipStream_t st = (hipStream_t)stream;
  if (M <= 16) launch_i8_rows<1, 1, 8, 4>(a, st);
  else if (M <= 64) launch_i8_rows<4, 2, 8, 2>(a, st);
  else launch_i8_tile<256, 256, 2, 4>(a, st);
  return check_launch("w8a8_linear");
}

}  // extern "C"
