// rms_norm_q8, silu_mul_q8 and quantize_q8: the launch of a size and the C entry
// points (kernel: fp4x_rowq.h).
#include <string>

#include "fp4x_rowq.h"

namespace fp4x {

// Lanes per row and chunks per lane.  Rows of up to 256 values share a wave.
// Few rows (their waves at one chunk per lane fit the CUs at 16 each) take one
// chunk per lane, the shortest chain: 3 rows of 2560, normed, 3.35 us (2
// chunks: 3.7).  More rows are bound by the bytes that a CU can have on their
// way, and take 2 chunks, or 3 where that leaves no more lanes idle and 2 would
// take more than 4 waves: 16384 rows of 2560, quantized, 26 us (1 chunk: 45, 3:
// 27); 4096 of 6144, gated, 26 (1: 31, 2: 30); 3333 of 12000, normed, 35 (2: 57;
// 1 does not fit a workgroup).  The rule is coarse for short rows: 8192 of 512,
// quantized, take 5.6 with a second chunk that only repeats the first one's last
// (1: 4.9), and 8192 of 1536, normed with a residual, 21.3 (3: 20.1).  Rows loaded
// ahead of the one that is reduced gained nothing.
template <int KIND, int TX, int TR, int TW>
static int launch_row_q8(RowArgs a, hipStream_t st) {
  if (a.fmt == ROW_G128) return launch_row_g128(KIND, TX, TR, TW, a, st);
  const int chunks = (a.H + 7) / 8;
  const auto lanes = [&](int c) { return (chunks + 64 * c - 1) / (64 * c) * 64; };
  int C = 1;
  a.L = 4;
  if (chunks <= 32) {
    while (a.L < chunks) a.L <<= 1;
  } else {
    if (chunks > 1024 || (int64_t)a.M * (lanes(1) / 64) > 16 * device_cus())
      C = lanes(2) * 2 < lanes(3) * 3 || lanes(2) <= 256 ? 2 : 3;
    if (lanes(C) > 1024) C = 4;
    a.L = lanes(C);
  }
  const int threads = a.L <= 64 ? 256 : a.L;
  a.rpb = a.L <= 64 ? 256 / a.L : 1;
  const unsigned grid = (unsigned)std::min<int64_t>((a.M + (int64_t)a.rpb - 1) / a.rpb, 1 << 20);
  const dim3 g(grid), b(threads);
  if (C == 1) hipLaunchKernelGGL((row_q8_kernel<false, 1024, KIND, TX, TR, TW, 1>), g, b, 0, st, a);
  else if (C == 2) hipLaunchKernelGGL((row_q8_kernel<false, 1024, KIND, TX, TR, TW, 2>), g, b, 0, st, a);
  else if (C == 3) hipLaunchKernelGGL((row_q8_kernel<false, 1024, KIND, TX, TR, TW, 3>), g, b, 0, st, a);
  else hipLaunchKernelGGL((row_q8_kernel<false, 1024, KIND, TX, TR, TW, 4>), g, b, 0, st, a);
  return check_launch("row_q8");
}

// M rows of n bytes, `step` bytes apart (0: one row read M times).
struct RowSpan {
  uintptr_t at;
  int64_t step, n, M;
  RowSpan(const void* p, int dt, int64_t stride, int H, int M_)
      : at(reinterpret_cast<uintptr_t>(p)), step(M_ > 1 ? stride * (dt == DT_F32 ? 4 : 2) : 0),
        n((int64_t)H * (dt == DT_F32 ? 4 : 2)), M(step ? M_ : 1) {}
  uintptr_t end() const { return at + (M - 1) * step + n; }
};
static bool same_rows(const RowSpan& a, const RowSpan& b) {
  return a.at == b.at && a.n == b.n && a.M == b.M && a.step == b.step;
}
// Whether a row of b shares a byte with a row of a, whose own rows do not overlap.
static bool meet(const RowSpan& a, const RowSpan& b) {
  if (a.end() <= b.at || b.end() <= a.at) return false;
  if (a.M > 1 && a.step == b.step) {               // every period is alike
    const RowSpan &p = a.at <= b.at ? a : b, &q = a.at <= b.at ? b : a;
    const int64_t d = (int64_t)(q.at - p.at) % a.step;
    return d < p.n || d + q.n > a.step;
  }
  for (int64_t i = 0; i < b.M; ++i) {
    const uintptr_t from = b.at + i * b.step, to = from + b.n;
    if (to <= a.at) continue;
    const int64_t j = a.M > 1 ? std::min<int64_t>(a.M - 1, (int64_t)(to - 1 - a.at) / a.step) : 0;
    if (a.at + j * a.step + a.n > from) return true;   // the last row of a that begins before b's row i ends
  }
  return false;
}
static bool known_dt(int dt) { return dt == DT_BF16 || dt == DT_F32 || dt == DT_F16; }

// What the three entry points share; 0 rows: nothing else is looked at.
static int row_check(const char* what, const RowArgs& a, int dtype) {
  if (!known_dt(dtype)) return row_fail(what, "rows are bf16, fp16 or fp32");
  if (a.M < 0 || a.H < 1 || a.H > kRowMaxH) return row_fail(what, "need M >= 0 and 1 <= H <= 32768");
  if (a.fmt != ROW_INT8 && a.fmt != ROW_E4M3 && a.fmt != ROW_MX8 && a.fmt != ROW_G128) return row_fail(what, "unknown format");
  if (a.fmt == ROW_MX8 && a.H % 32) return row_fail(what, "mx8 needs rows of a multiple of 32 values");
  if (a.M == 0) return FP4X_OK;
  if (!a.x || !a.q || !a.s) return row_fail(what, "null rows, codes or scales");
  if (!el_aligned(a.x, dtype) || (a.fmt != ROW_MX8 && (reinterpret_cast<uintptr_t>(a.s) & 3)))
    return row_fail(what, "rows and scales must be aligned to their element");
  if (a.x_stride < 0 || (a.M > 1 && a.q_stride < a.H)) return row_fail(what, "the code rows overlap, or a row stride is negative");
  return FP4X_OK;
}

}  // namespace fp4x

using namespace fp4x;

extern "C" {

int fp4x_rms_norm_q8(const void* x, int64_t x_stride, int dtype, const void* res, int64_t res_stride, int res_dtype,
                     const void* w, int w_dtype, float w_offset, double eps, int M, int H, int fmt, void* q,
                     int64_t q_stride, void* s, void* res_out, int64_t res_out_stride, void* normed,
                     int64_t normed_stride, void* stream) {
  RowArgs a{x, x_stride, res, res_stride, w, w_offset, eps, 1.0 / (H > 0 ? H : 1), M, H, fmt, 0, 0, static_cast<uint8_t*>(q), q_stride, s,
            res_out, res_out_stride, normed, normed_stride};
  const char* what = "rms_norm_q8";
  if (int rc = row_check(what, a, dtype)) return rc;
  if ((res_dtype != dtype && res_dtype != DT_F32) || (w_dtype != dtype && w_dtype != DT_F32))
    return row_fail(what, "the residual and the weight have the rows' type or are fp32");
  if (!(eps >= 0.0)) return row_fail(what, "eps must not be negative");
  if (M == 0) return FP4X_OK;
  if (!w || !el_aligned(w, w_dtype) || (res && !el_aligned(res, res_dtype)) ||
      (res_out && !el_aligned(res_out, res_dtype)) || (normed && !el_aligned(normed, dtype)))
    return row_fail(what, "null weight, or a tensor not aligned to its element");
  if (res_out && !res) return row_fail(what, "a residual output needs a residual");
  if (res_stride < 0 || (M > 1 && ((res_out && res_out_stride < H) || (normed && normed_stride < H))))
    return row_fail(what, "output rows overlap, or a row stride is negative");
  if (res_out) {                                   // workgroups read and write rows in no order: each its own only
    const RowSpan out(res_out, res_dtype, res_out_stride, H, M);
    for (const RowSpan& in : {RowSpan(x, dtype, x_stride, H, M), RowSpan(res, res_dtype, res_stride, H, M)})
      if (!same_rows(out, in) && meet(out, in))
        return row_fail(what, "the residual output overlaps an input whose rows it does not replace one for one");
    if (meet(out, RowSpan(w, w_dtype, 0, H, 1))) return row_fail(what, "the residual output overlaps the norm weight");
  }
  hipStream_t st = (hipStream_t)stream;
  const bool r32 = res_dtype == DT_F32, w32 = w_dtype == DT_F32;
  if (dtype == DT_F32) return launch_row_q8<ROW_NORM, DT_F32, DT_F32, DT_F32>(a, st);
  if (dtype == DT_BF16)
    return r32 ? (w32 ? launch_row_q8<ROW_NORM, DT_BF16, DT_F32, DT_F32>(a, st)
                      : launch_row_q8<ROW_NORM, DT_BF16, DT_F32, DT_BF16>(a, st))
               : (w32 ? launch_row_q8<ROW_NORM, DT_BF16, DT_BF16, DT_F32>(a, st)
                      : launch_row_q8<ROW_NORM, DT_BF16, DT_BF16, DT_BF16>(a, st));
  return r32 ? (w32 ? launch_row_q8<ROW_NORM, DT_F16, DT_F32, DT_F32>(a, st)
                    : launch_row_q8<ROW_NORM, DT_F16, DT_F32, DT_F16>(a, st))
             : (w32 ? launch_row_q8<ROW_NORM, DT_F16, DT_F16, DT_F32>(a, st)
                    : launch_row_q8<ROW_NORM, DT_F16, DT_F16, DT_F16>(a, st));
}

int fp4x_silu_mul_q8(const void* gate, int64_t gate_stride, const void* up, int64_t up_stride, int dtype, int M, int F,
                     int fmt, void* q, int64_t q_stride, void* s, void* stream) {
  RowArgs a{gate, gate_stride, up, up_stride, nullptr, 0.0f, 0.0, 0.0, M, F, fmt, 0, 0, static_cast<uint8_t*>(q), q_stride,
            s, nullptr, 0, nullptr, 0};
  const char* what = "silu_mul_q8";
  if (int rc = row_check(what, a, dtype)) return rc;
  if (M == 0) return FP4X_OK;
  if (!up || !el_aligned(up, dtype) || up_stride < 0) return row_fail(what, "null or misaligned up rows");
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DT_BF16) return launch_row_q8<ROW_SILU, DT_BF16, DT_BF16, DT_BF16>(a, st);
  if (dtype == DT_F16) return launch_row_q8<ROW_SILU, DT_F16, DT_F16, DT_F16>(a, st);
  return launch_row_q8<ROW_SILU, DT_F32, DT_F32, DT_F32>(a, st);
}

int fp4x_quantize_q8(const void* x, int64_t x_stride, int dtype, int M, int H, int fmt, void* q, int64_t q_stride,
                     void* s, void* stream) {
  RowArgs a{x, x_stride, nullptr, 0, nullptr, 0.0f, 0.0, 0.0, M, H, fmt, 0, 0, static_cast<uint8_t*>(q), q_stride, s,
            nullptr, 0, nullptr, 0};
  if (int rc = row_check("quantize_q8", a, dtype)) return rc;
  if (M == 0) return FP4X_OK;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DT_BF16) return launch_row_q8<ROW_QUANT, DT_BF16, DT_BF16, DT_BF16>(a, st);
  if (dtype == DT_F16) return launch_row_q8<ROW_QUANT, DT_F16, DT_F16, DT_F16>(a, st);
  return launch_row_q8<ROW_QUANT, DT_F32, DT_F32, DT_F32>(a, st);
}

}  // extern "C"
