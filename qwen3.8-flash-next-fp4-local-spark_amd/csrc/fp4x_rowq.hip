// Rows in 8 bits with scales: the root-mean-square norm with the residual's
// addition (rms_norm_q8), the gated activation (silu_mul_q8) and plain rows
// (quantize_q8).  A row v of H fp32 values ends in one of
//   int8  s = max(amax, 1e-12) / 127, q = rint(v / s), one fp32 s per row
//   e4m3  s = max(amax, 1e-12) / 448, q = e4m3fn(v / s), one fp32 s per row
//   mx8   per 32 values the exponent X = clamp(floor(log2 amax) - 8, -127,
//         127) as the byte X + 127, q = e4m3fn(v * 2^-X) saturating at 448
// with IEEE fp32 division and round half to even.  A row (mx8: a block of 32)
// that holds an infinity or a NaN gets the scale NaN (byte 255) and the codes
// 0 (mx8: NaN codes), so that one bad token stays one bad row.
//
// The norm: h = x + r in fp32, rounded once to r's type and written back as
// the residual; v = (h * rs) * (w + offset) with rs = fp32(1 / sqrt(mean(h^2)
// + eps)).  The squares are exact in fp64 and summed there, so rs does not
// depend on the order of the sum, but where it is within some 2e-16 of a border
// between two fp32 values, which lie 6e-8 to 1.2e-7 apart: a few rows in 10^9.
// Every later step is one rounded fp32 operation: codes are the same for every
// launch shape, and equal a plain evaluation's bit for bit.
//
// One pass: a row's values stay in registers between the sum, the maximum and
// the codes.  Lane l of a row's L lanes holds the chunks of 8 values l, l + L,
// ..; L is a power of two below a wave for short rows (several rows per wave),
// a multiple of 64 otherwise.  A row's last chunk is moved back to end at H
// and overlaps the one before: its duplicates are left out of the sum, are
// harmless to the maximum, and are stored twice with one value.  Loads and
// stores need only their element's alignment.
#include <algorithm>

#include "fp4x_kernels.h"
#include "../../include/fp4x.h"

namespace fp4x {

int device_cus();

enum RowKind : int { ROW_NORM, ROW_SILU, ROW_QUANT };
enum RowFmt : int { ROW_INT8, ROW_E4M3, ROW_MX8 };

struct RowArgs {
  const void* x;  int64_t x_stride;                // rows (the gate)
  const void* r;  int64_t r_stride;                // residual or null (the up rows)
  const void* w;  float w_off;  double eps, inv_h; // norm weight, 1 / H
  int M, H, fmt, L, rpb;                           // lanes per row, rows per workgroup
  uint8_t* q;  int64_t q_stride;
  void* s;
  void* h;  int64_t h_stride;                      // residual out or null
  void* y;  int64_t y_stride;                      // normed rows or null
};

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));

// Eight values of a type, as loaded.
template <int DT> struct Raw8 {
  u32x4_any v;
  __device__ void load(const void* p, int64_t i) {
    v = *reinterpret_cast<const u32x4_any*>(static_cast<const uint16_t*>(p) + i);
  }
  __device__ void load_n(const void* p, int64_t i, int n) {
    uint32_t d[4] = {0, 0, 0, 0};
    for (int j = 0; j < n; ++j) d[j >> 1] |= (uint32_t)static_cast<const uint16_t*>(p)[i + j] << (16 * (j & 1));
    v = u32x4_any{d[0], d[1], d[2], d[3]};
  }
  __device__ void get(float (&f)[8]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (DT == DT_BF16) { f[2 * j] = bf16_lo(v[j]); f[2 * j + 1] = bf16_hi(v[j]); }
      else { f[2 * j] = f16_to_f32((uint16_t)v[j]); f[2 * j + 1] = f16_to_f32((uint16_t)(v[j] >> 16)); }
    }
  }
};
template <> struct Raw8<DT_F32> {
  u32x4_any a, b;
  __device__ void load(const void* p, int64_t i) {
    const u32x4_any* g = reinterpret_cast<const u32x4_any*>(static_cast<const float*>(p) + i);
    a = g[0]; b = g[1];
  }
  __device__ void load_n(const void* p, int64_t i, int n) {
    uint32_t d[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int j = 0; j < n; ++j) d[j] = static_cast<const uint32_t*>(p)[i + j];
    a = u32x4_any{d[0], d[1], d[2], d[3]}; b = u32x4_any{d[4], d[5], d[6], d[7]};
  }
  __device__ void get(float (&f)[8]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) { f[j] = __uint_as_float(a[j]); f[4 + j] = __uint_as_float(b[j]); }
  }
};

template <int DT>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if constexpr (DT == DT_BF16) return pack_bf16x2(lo, hi);
  else return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)lo) |
              (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)hi) << 16;
}
// Stores f[0..8) rounded to a type; n < 8: the first n only.
template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t i, const float (&f)[8], int n) {
  if (n < 8) {
    for (int j = 0; j < n; ++j) store_out(p, i + j, DT, f[j]);
  } else if constexpr (DT == DT_F32) {
    u32x4_any* g = reinterpret_cast<u32x4_any*>(static_cast<float*>(p) + i);
    g[0] = u32x4_any{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
    g[1] = u32x4_any{__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7])};
  } else {
    *reinterpret_cast<u32x4_any*>(static_cast<uint16_t*>(p) + i) =
        u32x4_any{pack16<DT>(f[0], f[1]), pack16<DT>(f[2], f[3]), pack16<DT>(f[4], f[5]), pack16<DT>(f[6], f[7])};
  }
}
template <int DT>
__device__ __forceinline__ float round_to(float f) {
  return DT == DT_BF16 ? round_bf16(f) : DT == DT_F16 ? (float)(_Float16)f : f;
}

struct SumF64 { __device__ double operator()(double a, double b) const { return a + b; } };
struct MaxF32 { __device__ float operator()(float a, float b) const { return __builtin_elementwise_maximum(a, b); } };

// A value of the lane that is 1, 2, 4 or 8 lanes on within 16 (or, for 4 and
// 8, of one that holds the same: the reductions below come to it with quads,
// then groups of 8, alike), in registers.
template <int S>
__device__ __forceinline__ uint32_t lane_other(uint32_t v) {
  constexpr int ctrl = S == 1 ? 0xB1 : S == 2 ? 0x4E : S == 4 ? 0x141 : 0x140;
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xf, 0xf, true);
}
template <int S, class T, class Op>
__device__ __forceinline__ T fold(T v, Op op) {
  struct Words { uint32_t w[sizeof(T) / 4]; } a = __builtin_bit_cast(Words, v), b;
#pragma unroll
  for (unsigned i = 0; i < sizeof(T) / 4; ++i) {
    if constexpr (S <= 8) {
      b.w[i] = lane_other<S>(a.w[i]);
    } else if constexpr (S == 16) {                // every lane gets both rows' (halves') values
      const auto p = __builtin_amdgcn_permlane16_swap(a.w[i], a.w[i], false, false);
      a.w[i] = p[0];
      b.w[i] = p[1];
    } else {
      const auto p = __builtin_amdgcn_permlane32_swap(a.w[i], a.w[i], false, false);
      a.w[i] = p[0];
      b.w[i] = p[1];
    }
  }
  return op(__builtin_bit_cast(T, a), __builtin_bit_cast(T, b));
}

// All-reduce over a row's L lanes: a butterfly within a wave, then one over the
// waves' results through LDS (`slot`: a value per wave, used once between
// barriers; 0 is the operations' identity here).  With lane exchanges through
// LDS, the waves' results read one by one, and fp64 divisions, the norm of 3
// rows of 2560 took 4.2 us and that of 4096 24.6, and without them 3.35 and 22,
// both at one chunk per lane (two bring the latter to 18).
template <class T, class Op>
__device__ __forceinline__ T row_reduce(T v, int L, T* slot, Op op) {
  v = fold<2>(fold<1>(v, op), op);
  if (L > 4) v = fold<4>(v, op);
  if (L > 8) v = fold<8>(v, op);
  if (L > 16) v = fold<16>(v, op);
  if (L > 32) v = fold<32>(v, op);
  if (L > 64) {
    if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
    __syncthreads();
    const int i = threadIdx.x & 15;
    v = i < L >> 6 ? slot[i] : T(0);
    v = fold<8>(fold<4>(fold<2>(fold<1>(v, op), op), op), op);
  }
  return v;
}

// x * sigmoid(x) from an expf within an ulp.  v_rcp_f32 is within an ulp, and one
// correction of it is the rounded quotient for every d from 1 to 2^100 (gates
// above -69): all 2^23 mantissas of the 100 exponents were compared with 1 / d on
// gfx950 and none differed, where 11% of the reciprocals alone do; it is not a
// theorem (33 mantissas would miss if the reciprocal were an ulp off there).
// Below -69 the reciprocal is taken as it is; from about -87 down, where silu is
// under 2e-36 in magnitude, it is flushed and the result is 0.
__device__ __forceinline__ float silu_f32(float x) {
  const float d = 1.0f + expf(-x), r = __builtin_amdgcn_rcpf(d);
  return x * (d < 0x1p100f ? __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r) : r);
}

__device__ __forceinline__ uint32_t e4m3x4(const float* f) {
  int d = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], d, true);
}
__device__ __forceinline__ void store_codes(uint8_t* q, uint32_t lo, uint32_t hi, int n) {
  if (n >= 8) {
    *reinterpret_cast<u32x2_any*>(q) = u32x2_any{lo, hi};
  } else {
    for (int j = 0; j < n; ++j) q[j] = (uint8_t)((j < 4 ? lo : hi) >> (8 * (j & 3)));
  }
}

template <int KIND, int TX, int TR, int TW, int C>
__global__ __launch_bounds__(1024) void row_q8_kernel(const RowArgs a) {
  __shared__ double sum_slot[16];
  __shared__ float max_slot[16];
  const int t = threadIdx.x, L = a.L, l = L <= 64 ? t & (L - 1) : t, sub = L <= 64 ? t / L : 0;
  const int last = a.H - 8, n = a.H < 8 ? a.H : 8;
  const bool two = KIND == ROW_SILU || (KIND == ROW_NORM && a.r);
  int k[C];
  Raw8<TX> x[C];
  Raw8<TR> r[C];
  Raw8<TW> w[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int k0 = (c * L + l) * 8;
    k[c] = k0 < last ? k0 : last < 0 ? 0 : last;
  }
  const auto load = [&](int64_t rb) __attribute__((always_inline)) {
    const int64_t want = rb * a.rpb + sub, row = want < a.M ? want : a.M - 1;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int64_t xi = row * a.x_stride + k[c], ri = row * a.r_stride + k[c];
      if (C == 1 && n < 8) {
        x[c].load_n(a.x, xi, n);
        if (two) r[c].load_n(a.r, ri, n);
      } else {
        x[c].load(a.x, xi);
        if (two) r[c].load(a.r, ri);
      }
    }
  };
  if constexpr (KIND == ROW_NORM && C <= 3) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (C == 1 && n < 8) w[c].load_n(a.w, k[c], n);
      else w[c].load(a.w, k[c]);
    }
  }
  for (int64_t rb = blockIdx.x; rb * a.rpb < a.M; rb += gridDim.x) {
    const int64_t want = rb * a.rpb + sub, row = want < a.M ? want : a.M - 1;
    const bool live = want < a.M;
    load(rb);
    float f[C][8];
    double ss = 0.0;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      x[c].get(f[c]);
      float g[8];
      if (two) r[c].get(g);
      if constexpr (KIND == ROW_SILU) {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[c][j] = silu_f32(f[c][j]) * g[j];
      }
      if constexpr (KIND == ROW_NORM) {
        if (two) {
#pragma unroll
          for (int j = 0; j < 8; ++j) f[c][j] = round_to<TR>(f[c][j] + g[j]);
        }
        const int d = (c * L + l) * 8 - k[c];      // duplicates at the front of a chunk moved back
        if (d == 0) {
#pragma unroll
          for (int j = 0; j < 8; ++j) ss = __builtin_fma((double)f[c][j], (double)f[c][j], ss);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const double v = j >= d ? (double)f[c][j] : 0.0;
            ss = __builtin_fma(v, v, ss);
          }
        }
      }
    }
    if constexpr (KIND == ROW_NORM) {
      ss = row_reduce(ss, L, sum_slot, SumF64());
      const float rs = (float)rsqrt(ss * a.inv_h + a.eps);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const bool in = live && (c * L + l) * 8 < a.H;
        if (a.h && in) store8<TR>(a.h, row * a.h_stride + k[c], f[c], n);
        float g[8];
        if (C > 3) {
          asm volatile("" ::: "memory");           // one chunk's weights at a time
          w[c].load(a.w, k[c]);
        }
        w[c].get(g);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[c][j] = (f[c][j] * rs) * (g[j] + a.w_off);
        if (a.y && in) store8<TX>(a.y, row * a.y_stride + k[c], f[c], n);
      }
    }

    float m[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      m[c] = fabsf(f[c][0]);
#pragma unroll
      for (int j = 1; j < 8; ++j) m[c] = __builtin_elementwise_maximum(m[c], fabsf(f[c][j]));
    }
    if (a.fmt == ROW_MX8) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float b = m[c];                            // 4 lanes hold a block of 32
        b = fold<2>(fold<1>(b, MaxF32()), MaxF32());
        const bool fin = b < __builtin_inff();
        const int e = (int)(__float_as_uint(b) >> 23);
        const int X = e == 0 ? -127 : max(e - 127 - 8, -127);
        const float up = __uint_as_float((uint32_t)(127 - X) << 23);   // 2^-X, X in [-127, 119]
        float g[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = fminf(fmaxf(f[c][j] * up, -448.0f), 448.0f);
        uint32_t lo = e4m3x4(g), hi = e4m3x4(g + 4);
        if (!fin) lo = hi = 0x7f7f7f7fu;
        if (live && (c * L + l) * 8 < a.H) {
          store_codes(a.q + row * a.q_stride + k[c], lo, hi, 8);
          if ((l & 3) == 0) static_cast<uint8_t*>(a.s)[row * (a.H / 32) + k[c] / 32] = fin ? (uint8_t)(X + 127) : 255;
        }
      }
    } else {
      float amax = m[0];
#pragma unroll
      for (int c = 1; c < C; ++c) amax = __builtin_elementwise_maximum(amax, m[c]);
      amax = row_reduce(amax, L, max_slot, MaxF32());
      const bool fin = amax < __builtin_inff();
      const float s = fmaxf(amax, 1e-12f) / (a.fmt == ROW_INT8 ? 127.0f : 448.0f);
      // the rounded quotient from the reciprocal where every row of the wave allows it (a branch: the division that it
      // saves is 10 of 16 operations per value)
      const bool quick = __all(fin && mid_range(s));
      const float rc = 1.0f / s;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float g[8];
        if (quick) {
#pragma unroll
          for (int j = 0; j < 8; ++j) g[j] = exact_quot(f[c][j], s, rc);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) g[j] = f[c][j] / s;
        }
        uint32_t lo, hi;
        if (a.fmt == ROW_INT8) {
          uint32_t b[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) b[j] = __float_as_uint(g[j] + kRint);
          lo = perm_b32(perm_b32(b[3], b[2], 0x0c0c0400u), perm_b32(b[1], b[0], 0x0c0c0400u), 0x05040100u);
          hi = perm_b32(perm_b32(b[7], b[6], 0x0c0c0400u), perm_b32(b[5], b[4], 0x0c0c0400u), 0x05040100u);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) g[j] = copysignf(fminf(fabsf(g[j]), 448.0f), f[c][j]);   // -0 too
          lo = e4m3x4(g);
          hi = e4m3x4(g + 4);
        }
        if (!fin) lo = hi = 0;
        if (live && (c * L + l) * 8 < a.H) store_codes(a.q + row * a.q_stride + k[c], lo, hi, n);
      }
      if (live && l == 0) static_cast<float*>(a.s)[row] = fin ? s : __uint_as_float(0x7fc00000u);
    }
    if (L > 64) __syncthreads();                   // the slots are used again
  }
}

constexpr int kRowMaxH = 32768;                    // 1024 lanes of 4 chunks

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
  if (C == 1) hipLaunchKernelGGL((row_q8_kernel<KIND, TX, TR, TW, 1>), g, b, 0, st, a);
  else if (C == 2) hipLaunchKernelGGL((row_q8_kernel<KIND, TX, TR, TW, 2>), g, b, 0, st, a);
  else if (C == 3) hipLaunchKernelGGL((row_q8_kernel<KIND, TX, TR, TW, 3>), g, b, 0, st, a);
  else hipLaunchKernelGGL((row_q8_kernel<KIND, TX, TR, TW, 4>), g, b, 0, st, a);
  return check_launch("row_q8");
}

static int row_fail(const char* what, const char* why) {
  set_error(std::string(what) + ": " + why);
  return FP4X_ERR_ARG;
}
static bool el_aligned(const void* p, int dt) {
  return (reinterpret_cast<uintptr_t>(p) & (dt == DT_F32 ? 3 : 1)) == 0;
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
  if (a.fmt < ROW_INT8 || a.fmt > ROW_MX8) return row_fail(what, "unknown format");
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
