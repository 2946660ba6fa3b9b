// Rows and weights in e4m3 with a scale per block of 128: the launches of the
// rows (kernel: fp4x_rowq.h), and the weights' kernel and C entry point.
#include <string>

#include "fp4x_rowq.h"

namespace fp4x {

// Lanes and chunks per lane as the other formats have them (launch_row_q8), but
// where that leaves a quarter of them or more without values: blocks need no more
// than 16 lanes, so rows may share a wave, and the fewest idle of 16, 32 and 64
// lanes are taken.  32768 rows of 640, gated, take 26 us on 16 lanes of 5 chunks
// (64 of 2: 37), 8192 of 1280 15.4 on 32 of 5 (128 of 2: 16.4), in calls in a row on
// one input (the former 28 to 30 where inputs change, 27.4 at the least in a trace).
// Elsewhere fewer lanes of more chunks lose: 4096 of 2560, normed, 38 on 64 of 5
// (192 of 2: 17).
template <int KIND, int TX, int TR, int TW>
static int launch_g128(RowArgs a, hipStream_t st) {
  const int chunks = (a.H + 7) / 8;
  const auto lanes = [&](int c) { return (chunks + 64 * c - 1) / (64 * c) * 64; };
  int C = 1;
  a.L = 4;
  if (chunks <= 32) {
    while (a.L < chunks) a.L <<= 1;
  } else {
    if (chunks > 1024 || (int64_t)a.M * (lanes(1) / 64) > 16 * device_cus())
      C = lanes(2) * 2 < lanes(3) * 3 || lanes(2) <= 256 || lanes(3) > 256 ? 2 : 3;
    if (lanes(C) > 1024) C = 4;
    a.L = lanes(C);
    if (C > 1 && 4 * (C * a.L - chunks) >= C * a.L)
      for (int L = 16; L <= 64; L *= 2) {
        const int c = (chunks + L - 1) / L;
        if (c <= 5 && c != 4 && c * L < C * a.L) {
          C = c;
          a.L = L;
        }
      }
  }
  const int threads = a.L <= 64 ? 256 : a.L;
  a.rpb = a.L <= 64 ? 256 / a.L : 1;
  const dim3 g((unsigned)std::min<int64_t>((a.M + (int64_t)a.rpb - 1) / a.rpb, 1 << 20)), b(threads);
  if (C == 1) hipLaunchKernelGGL((row_q8_kernel<true, 1024, KIND, TX, TR, TW, 1>), g, b, 0, st, a);
  else if (C == 2) hipLaunchKernelGGL((row_q8_kernel<true, 1024, KIND, TX, TR, TW, 2>), g, b, 0, st, a);
  else if (C == 3) hipLaunchKernelGGL((row_q8_kernel<true, 256, KIND, TX, TR, TW, 3>), g, b, 0, st, a);
  else if (C == 4) hipLaunchKernelGGL((row_q8_kernel<true, 1024, KIND, TX, TR, TW, 4>), g, b, 0, st, a);
  else hipLaunchKernelGGL((row_q8_kernel<true, 256, KIND, TX, TR, TW, 5>), g, b, 0, st, a);
  return check_launch("row_q8");
}
template <int TX>
static int launch_g128_norm(int tr, int tw, const RowArgs& a, hipStream_t st) {
  if (tr == DT_F32) return tw == DT_F32 ? launch_g128<ROW_NORM, TX, DT_F32, DT_F32>(a, st) : launch_g128<ROW_NORM, TX, DT_F32, TX>(a, st);
  return tw == DT_F32 ? launch_g128<ROW_NORM, TX, TX, DT_F32>(a, st) : launch_g128<ROW_NORM, TX, TX, TX>(a, st);
}
template <int KIND>
static int launch_g128_one(int t, const RowArgs& a, hipStream_t st) {
  if (t == DT_BF16) return launch_g128<KIND, DT_BF16, DT_BF16, DT_BF16>(a, st);
  if (t == DT_F16) return launch_g128<KIND, DT_F16, DT_F16, DT_F16>(a, st);
  return launch_g128<KIND, DT_F32, DT_F32, DT_F32>(a, st);
}
int launch_row_g128(int kind, int tx, int tr, int tw, const RowArgs& a, hipStream_t st) {
  if (kind == ROW_SILU) return launch_g128_one<ROW_SILU>(tx, a, st);
  if (kind == ROW_QUANT) return launch_g128_one<ROW_QUANT>(tx, a, st);
  if (tx == DT_BF16) return launch_g128_norm<DT_BF16>(tr, tw, a, st);
  if (tx == DT_F16) return launch_g128_norm<DT_F16>(tr, tw, a, st);
  return launch_g128<ROW_NORM, DT_F32, DT_F32, DT_F32>(a, st);
}

// A weight in e4m3 with a scale per 128 x 128 block (blocks at its ends may be
// smaller), [E, N, K]: the values of a block stay in the registers of one
// workgroup, 8 rows x 8 values per lane, between the maximum and the codes.  Bound
// by memory: [16384 x 2560] in bf16, 126 MB, takes 21.7 us (5.8 TB/s, its output
// still in the caches when it ends).
struct BlockArgs {
  const void* w;  int64_t w_row, w_expert;         // strides in elements
  uint8_t* q;  int64_t q_row, q_expert;            // strides in bytes
  float* s;
  int N, K, nb, kb;
  int64_t blocks;
};
template <int T>
__global__ __launch_bounds__(256) void block_q8_kernel(const BlockArgs a) {
  __shared__ float slot[4];
  const int t = threadIdx.x, r0 = t >> 4;
  for (int64_t b = blockIdx.x; b < a.blocks; b += gridDim.x) {
    const int64_t bn = b / a.kb;
    const int e = (int)(bn / a.nb), n0 = (int)(bn % a.nb) * 128, k0 = (int)(b % a.kb) * 128 + (t & 15) * 8;
    const int nk = min(max(a.K - k0, 0), 8);
    float f[8][8], m = 0.0f;
    Raw8<T> raw[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t at = e * a.w_expert + min(n0 + r0 + 16 * i, a.N - 1) * a.w_row + k0;
      if (nk == 8) raw[i].load(a.w, at);
      else raw[i].load_n(a.w, at, nk);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {                  // (rows past the end hold the last one's values)
      raw[i].get(f[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) m = __builtin_elementwise_maximum(m, fabsf(f[i][j]));
    }
    m = fold<8>(fold<4>(fold<2>(fold<1>(m, MaxF32()), MaxF32()), MaxF32()), MaxF32());
    m = fold<32>(fold<16>(m, MaxF32()), MaxF32());
    if ((t & 63) == 0) slot[t >> 6] = m;
    __syncthreads();
    m = slot[0];
#pragma unroll
    for (int i = 1; i < 4; ++i) m = __builtin_elementwise_maximum(m, slot[i]);
    const bool fin = m < __builtin_inff();
    const float s = e4m3_scale(m);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t lo, hi;
      e4m3_codes(f[i], s, fin && mid_range(s), lo, hi);
      if (!fin) lo = hi = 0;
      if (n0 + r0 + 16 * i < a.N) store_codes(a.q + e * a.q_expert + (n0 + r0 + 16 * i) * a.q_row + k0, lo, hi, nk);
    }
    if (t == 0) a.s[b] = fin ? s : __uint_as_float(0x7fc00000u);
    __syncthreads();                               // the slots are used again
  }
}

}  // namespace fp4x

using namespace fp4x;

extern "C" {

int fp4x_quantize_f8(const void* w, int64_t w_row, int64_t w_expert, int dtype, int E, int N, int K, void* q, int64_t q_row,
                     int64_t q_expert, float* s, void* stream) {
  const char* what = "quantize_f8";
  if (dtype != DT_BF16 && dtype != DT_F32 && dtype != DT_F16) return row_fail(what, "weights are bf16, fp16 or fp32");
  if (E < 0 || N < 0 || K < 1 || N > 1 << 24 || K > 1 << 24) return row_fail(what, "need E and N >= 0, K >= 1, N and K up to 2^24");
  if (E == 0 || N == 0) return FP4X_OK;
  if (!w || !q || !s) return row_fail(what, "null weight, codes or scales");
  if (!el_aligned(w, dtype) || (reinterpret_cast<uintptr_t>(s) & 3)) return row_fail(what, "weights and scales must be aligned to their element");
  if (w_row < 0 || w_expert < 0 || q_row < K || (E > 1 && q_expert < (N - 1) * q_row + K))
    return row_fail(what, "the code rows overlap, or a stride is negative");
  const int nb = (N + 127) / 128, kb = (K + 127) / 128;
  const BlockArgs a{w, w_row, w_expert, static_cast<uint8_t*>(q), q_row, q_expert, s, N, K, nb, kb, (int64_t)E * nb * kb};
  const dim3 grid((unsigned)std::min<int64_t>(a.blocks, 1 << 20));
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DT_BF16) hipLaunchKernelGGL((block_q8_kernel<DT_BF16>), grid, dim3(256), 0, st, a);
  else if (dtype == DT_F16) hipLaunchKernelGGL((block_q8_kernel<DT_F16>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((block_q8_kernel<DT_F32>), grid, dim3(256), 0, st, a);
  return check_launch(what);
}

}  // extern "C"
