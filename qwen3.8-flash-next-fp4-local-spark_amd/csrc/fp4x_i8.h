// Products of 8-bit integers: out[m, n] = cast((sum_k x[m, k] w[n, k]) * sx[m]
// * sw[n] + b[n]), x int8 [M, K] with a scale per row (token), w int8 [N, K]
// with a scale per row (output channel), summed in int32: exact for K up to
// 131,071 (|x w| <= 2^14), so no order of the sum changes a result.
#pragma once
#include <algorithm>
#include <type_traits>

#include "fp4x_kernels.h"
#include "../../include/fp4x.h"

namespace fp4x {

typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2_a2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32_a2 __attribute__((aligned(2)));
typedef uint32_t u32x2_a4 __attribute__((ext_vector_type(2), aligned(4)));
typedef uint32_t u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef const __attribute__((address_space(3))) void* i8_lds_t;

struct I8Args {
  const int8_t* x;  int64_t x_stride;  const float* sx;
  const int8_t* w;  int64_t w_stride;  const float* sw;
  const float* bias;
  void* out;  int out_dtype;  int64_t out_stride;
  int M, N, K;
  int mt, nt, gm;                                  // tiles over M and N, tiles of M in a band
};

// Places of 1-D grids: consecutive workgroups go to the 8 XCDs in turn, each
// with its own L2, so XCD x takes one run of consecutive tiles.  Tiles are
// ordered in bands of gm tiles of M, M first: a run's tiles share rows of x
// and of w.
struct I8Run {
  int first, count;
  __device__ I8Run(int tiles, int xcd) : first(xcd * (tiles >> 3) + min(xcd, tiles & 7)),
                                         count((tiles >> 3) + (xcd < (tiles & 7))) {}
};
__device__ __forceinline__ void tile_place(int mt, int nt, int gm, int id, int bm, int bn, int& m0, int& n0) {
  int band = 0, r = id, h = mt;
  if (mt > gm) {
    const int per = gm * nt;
    band = id / per;
    r = id - band * per;
    h = min(gm, mt - band * gm);
  }
  // (no general division for the heights of a band and of few rows)
  const int n = h == 1 ? r : h == 2 ? r >> 1 : h == 3 ? (int)__umulhi(r, 0x55555556u) : h == 4 ? r >> 2 : r / h;
  m0 = (band * gm + r - n * h) * bm;
  n0 = n * bn;
}
__device__ __forceinline__ void i8_place(const I8Args& a, int id, int bm, int bn, int& m0, int& n0) {
  tile_place(a.mt, a.nt, a.gm, id, bm, bn, m0, n0);
}

// Direct loads to LDS: lane l's 16 (4) bytes at base + off land at lds + 16 l
// (4 l).  They are asm so that the compiler, which cannot tell which stage a
// load fills, puts no waits of its own before LDS reads: i8_wait and i8_sync
// are the only waits for them.  They have no output register.
__device__ __forceinline__ void i8_load16(uint32_t lds, uint32_t off, const void* base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "m0");
}
__device__ __forceinline__ void i8_load4(uint32_t lds, uint32_t off, const void* base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(off), "s"(base) : "m0");
}
// All but the newest V memory operations of this wave are done.
template <int V> __device__ __forceinline__ void i8_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(V) : "memory"); }
// The same, its LDS reads are done too, and every wave of the workgroup has come so far.
template <int V> __device__ __forceinline__ void i8_sync() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(V) : "memory");
}
__device__ __forceinline__ uint32_t i8_lds(const void* p) { return (uint32_t)(uintptr_t)(i8_lds_t)p; }

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

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)lo) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)hi) << 16;
}

// Scales and bias of four neighbouring columns [n, n + 4) of row m.
struct I8Scales {
  float sx, sw[4], b[4];
  __device__ __forceinline__ void load(const I8Args& a, int m, int n) {
    sx = a.sx[min(m, a.M - 1)];
    if (n + 4 <= a.N) {
      get(sw, a.sw + n);
      if (a.bias) get(b, a.bias + n);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int nj = min(n + j, a.N - 1);
        sw[j] = a.sw[nj];
        if (a.bias) b[j] = a.bias[nj];
      }
    }
  }
  static __device__ __forceinline__ void get(float (&f)[4], const float* p) {
    const u32x4_a4 v = *reinterpret_cast<const u32x4_a4*>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = __uint_as_float(v[j]);
  }
};
// Those columns of y; the ones from N on are left out.
__device__ __forceinline__ void i8_store4(const I8Args& a, int64_t m, int n, i32x4_t acc, const I8Scales& s) {
  float v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[j] = ((float)acc[j] * s.sx) * s.sw[j];
    if (a.bias) v[j] = v[j] + s.b[j];
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
      for (int j = 0; j < 2; ++j) p[j] = pack_f16x2(v[2 * j], v[2 * j + 1]);
    }
    *reinterpret_cast<u32x2_a2*>(static_cast<uint16_t*>(a.out) + at) = u32x2_a2{p[0], p[1]};
  }
}

// ------------------------------------------------------------------ small tiles
// A workgroup owns 16 MT rows of x and 16 NT rows of w; its W waves split K in
// units of 128 values.  Each wave brings its units through a ring of D stages
// of its own, so the loop has no barrier: a direct load takes 8 rows x 128
// bytes (whole cache lines), D - 1 units are on their way while one is used,
// and the waves' integer sums meet in LDS at the end.
//
// What bounds it: the bytes a CU can have on their way.  The same split with
// loads into registers (16 rows x 64 bytes a load, in the layout that the MFMA
// takes) took 14.3 us at 16 x [16384 x 2560] and 13.1 at 64 x [2560 x 6144];
// this takes 8.5 and 7.1 (weights from HBM).  Scales that are loaded after the
// sums, and sums through atomics on a cleared block of LDS, took 0.6 us more.
template <int MT, int NT, int W, int D>
__global__ __launch_bounds__(64 * W) void i8_ring_kernel(const I8Args a) {
  constexpr int R = 16 * (MT + NT), NL = R / 8, STAGE = R * 128;
  constexpr int LD = 16 * NT + 4;                  // (a row of sums starts on 16 bytes)
  constexpr int ITEMS = (64 * MT * NT + 64 * W - 1) / (64 * W);   // of four columns, per thread
  static_assert(D * STAGE >= 16 * MT * LD * 4, "the sums reuse the ring");
  __shared__ __attribute__((aligned(1024))) char lds[W * D * STAGE];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), i = lane & 15, g = lane >> 4;
  const I8Run run(a.mt * a.nt, blockIdx.x & 7);
  int m0, n0;
  i8_place(a, run.first + (blockIdx.x >> 3), 16 * MT, 16 * NT, m0, n0);
  const int units = (a.K + 127) >> 7, per = (units + W - 1) / W, u0 = wave * per;
  const int n = max(min(per, units - u0), 0);      // this wave's units
  const int tail = a.K & 127 ? units - 1 - u0 : -1;   // the one that K ends in, if any
  const int last = (a.K - 1) >> 4;
  // LDS row r holds chunk c of its 128 bytes at c ^ key: the 16 lanes that LDS serves together read different banks
  const int slot = lane & 7, lr = lane >> 3;
  uint32_t off[NL];
#pragma unroll
  for (int j = 0; j < NL; ++j) {
    const int r = j * 8 + lr, c = slot ^ ((r >> 1) & 7);
    if (j < 2 * MT) off[j] = (uint32_t)(min(m0 + r, a.M - 1) - m0) * (uint32_t)a.x_stride + c * 16;
    else off[j] = (uint32_t)(min(n0 + r - 16 * MT, a.N - 1) - n0) * (uint32_t)a.w_stride + c * 16;
  }
  const int8_t* xb = a.x + m0 * a.x_stride + u0 * 128;
  const int8_t* wb = a.w + n0 * a.w_stride + u0 * 128;
  const uint32_t base = i8_lds(lds) + wave * D * STAGE;
  const char* mine = lds + wave * D * STAGE;
  const auto issue = [&](int s, int u) __attribute__((always_inline)) {
    if (u == tail) {                               // chunks past the row's last one read that one
#pragma unroll
      for (int j = 0; j < NL; ++j) {
        const int c = slot ^ (((j * 8 + lr) >> 1) & 7), over = (u0 + u) * 8 + c - last;
        if (over > 0) off[j] -= over * 16;         // (its last use)
      }
    }
#pragma unroll
    for (int j = NL - 1; j >= 0; --j) i8_load16(base + s * STAGE + j * 1024, off[j], (j < 2 * MT ? xb : wb) + u * 128);
  };
  // the epilogue's scales, before the units: a wait for a unit is then one for them too
  I8Scales sc[ITEMS];
#pragma unroll
  for (int p = 0; p < ITEMS; ++p) {
    const int e = t + p * 64 * W;                  // (whole waves have an item or none)
    if (e < 64 * MT * NT) sc[p].load(a, m0 + e / (4 * NT), n0 + 4 * (e % (4 * NT)));
  }
  asm volatile("" ::: "memory");                   // not behind the units' loads, whose waits count what is newer
  i32x4_t acc[MT][NT];
#pragma unroll
  for (int s = 0; s < MT; ++s)
#pragma unroll
    for (int r = 0; r < NT; ++r) acc[s][r] = i32x4_t{0, 0, 0, 0};
#pragma unroll
  for (int d = 0; d < D; ++d)
    if (d < n) issue(d, d);
  int stage = 0;
  for (int u = 0; u < n; ++u) {
    if (u + D - 1 < n) i8_wait<(D - 1) * NL>();
    else i8_wait<0>();
    const char* st = mine + stage * STAGE;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      const int at = ((kk * 4 + g) ^ ((i >> 1) & 7)) * 16;
      i32x4_t x[MT], w[NT];
#pragma unroll
      for (int r = 0; r < NT; ++r) w[r] = *reinterpret_cast<const i32x4_t*>(st + (16 * MT + 16 * r + i) * 128 + at);
#pragma unroll
      for (int s = 0; s < MT; ++s) x[s] = *reinterpret_cast<const i32x4_t*>(st + (16 * s + i) * 128 + at);
      if (u == tail)
#pragma unroll
        for (int s = 0; s < MT; ++s) x[s] = keep_to(x[s], (u0 + u) * 8 + kk * 4 + g, a.K);
#pragma unroll
      for (int s = 0; s < MT; ++s)
#pragma unroll
        for (int r = 0; r < NT; ++r) acc[s][r] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[r], x[s], acc[s][r], 0, 0, 0);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the stage is read before it is filled again
    if (u + D < n) issue(stage, u + D);
    if (++stage == D) stage = 0;
  }
  // the wave's sums take the place of its ring
  int* sum = reinterpret_cast<int*>(lds + wave * D * STAGE);
#pragma unroll
  for (int s = 0; s < MT; ++s)
#pragma unroll
    for (int r = 0; r < NT; ++r) *reinterpret_cast<i32x4_t*>(&sum[(16 * s + i) * LD + 16 * r + 4 * g]) = acc[s][r];
  __syncthreads();
#pragma unroll
  for (int p = 0; p < ITEMS; ++p) {
    const int e = t + p * 64 * W, m = e / (4 * NT), c = e % (4 * NT);
    if (e < 64 * MT * NT && m0 + m < a.M && n0 + 4 * c < a.N) {
      i32x4_t v = i32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int q = 0; q < W; ++q) v += *reinterpret_cast<const i32x4_t*>(lds + q * D * STAGE + (m * LD + 4 * c) * 4);
      i8_store4(a, m0 + m, n0 + 4 * c, v, sc[p]);
    }
  }
}

// ------------------------------------------------------------------ large tiles
// A workgroup owns BM rows of x and BN rows of w at a time and walks K in
// k-tiles of 128 through S LDS stages filled by direct loads.  Wave (wm, wn)
// owns 32 MI rows of x and 32 NI of w.  A k-tile is four steps of 32: while a
// step's MFMAs run, the next step's operands are read into the other half of
// the registers, and the last step of a k-tile reads the first of the next, so
// there is one barrier per k-tile: behind it the next k-tile is whole in LDS
// and the current one is wholly in registers, and its stage is filled again.
//
// A workgroup takes several tiles, and its loads run S k-tiles ahead across
// them: a tile's epilogue runs while the next tile's first k-tiles come in,
// and its stores are not waited for until the ring needs a load that was
// issued after them (`drain`).
//
// Weight row NI p + r of a wave's 32 NI is row p of its block r, so a lane
// holds NI neighbouring columns of each of its rows of y, and a wave stores
// whole lines of 32 NI columns without a pass through LDS (16-byte pieces of
// 64 rows at once, as 16 columns of a row per lane would give, took 13 us more
// of 4096 x [16384 x 2560]).
//
// What bounds it at 4096 x [16384 x 2560] (256 x 256 tiles): 159 to 181 us among
// other work (2.2 to 1.9 POP/s), 151 (2.3) in a long row of the same call.  In
// copies that leave parts out, timed in such rows, the MFMAs alone take 100, with
// LDS reads 116, with the loads too 134, with the conversion 139, with the stores
// 147.  In cycles the parts overlap (12% between the first and the last), but the
// clock falls from 2.2 to 1.8 GHz as they add up: the power limit.  Consecutive
// MFMAs keep one operand for that reason.  A 4-wave form (128 x 128 per wave)
// takes 174 and more, 16 x 16 x 64 MFMAs 166, k-tiles of 64 in four stages 147
// (all without stores), where this takes 138; 16 waves take as long.  A K that
// ends inside a k-tile is code of its own (TAIL): the test for it in every step
// took 9 us more.
template <int BM, int BN, int WM, int WN, int S>
struct I8Tile {
  static constexpr int W = WM * WN, MI = BM / WM / 32, NI = BN / WN / 32;
  static constexpr int STAGE = (BM + BN) * 128, XL = BM / 8 / W, WL = BN / 8 / W, NL = XL + WL;   // 1 KB loads per wave
  static constexpr int SC = (BM + 2 * BN) * 4;     // a tile's scales and bias
  static constexpr int LDS = S * STAGE + 2 * SC;
  static constexpr int DRAIN = (S - 2) * NL + 16 * MI < 63 ? (S - 2) * NL + 16 * MI : 63;
  static_assert(MI * 32 * WM == BM && NI * 32 * WN == BN && XL * 8 * W == BM && WL * 8 * W == BN && BM % 64 == 0 &&
                BN % 64 == 0 && NI <= 2 && S >= 2, "tile");
};

template <int BM, int BN, int WM, int WN, int S, bool TAIL>
__global__ __launch_bounds__(64 * WM * WN, 1) void i8_tile_kernel(const I8Args a) {
  using C = I8Tile<BM, BN, WM, WN, S>;
  constexpr int MI = C::MI, NI = C::NI, NL = C::NL, NM = MI * NI, NR = MI + NI;
  __shared__ __attribute__((aligned(1024))) char lds[C::LDS];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int xcd = blockIdx.x & 7;
  const I8Run run(a.mt * a.nt, xcd);
  const int stride = (gridDim.x + 7 - xcd) >> 3;   // workgroups of this XCD
  const int first = run.first + (blockIdx.x >> 3), tiles = (run.count - (blockIdx.x >> 3) + stride - 1) / stride;
  const int kts = (a.K + 127) >> 7, V = tiles * kts;
  const int last = (a.K - 1) >> 4;                 // TAIL: K ends inside a k-tile

  // ---- the loads: k-tile lk of tile lt
  // LDS row r holds chunk c of its 128 bytes at c ^ key: the 16 lanes that LDS serves together read different banks
  const int slot = lane & 7, lr = lane >> 3;
  const uint32_t lbase = i8_lds(lds);
  int lt = 0, lk = 0, lm0, ln0;
  int pm0 = 0, pn0 = 0, pm1 = 0, pn1 = 0;          // places of an even and of an odd tile
  uint32_t off[NL];
  const int8_t *xb, *wb;
  const auto row_of = [&](int j) __attribute__((always_inline)) {   // LDS row of load j in its operand's half
    return ((j < C::XL ? wave * C::XL + j : wave * C::WL + j - C::XL) << 3) + lr;
  };
  const auto next_tile = [&]() __attribute__((always_inline)) {
    i8_place(a, first + lt * stride, BM, BN, lm0, ln0);
    if (lt & 1) {
      pm1 = lm0;
      pn1 = ln0;
    } else {
      pm0 = lm0;
      pn0 = ln0;
    }
#pragma unroll
    for (int j = 0; j < NL; ++j) {
      const int r = row_of(j), c = slot ^ ((r >> 1) & 7);
      if (j < C::XL) off[j] = (uint32_t)(min(lm0 + r, a.M - 1) - lm0) * (uint32_t)a.x_stride + c * 16;
      else {
        const int wr = (r & -(32 * NI)) + NI * (r & 31) + (r >> 5) % NI;
        off[j] = (uint32_t)(min(ln0 + wr, a.N - 1) - ln0) * (uint32_t)a.w_stride + c * 16;
      }
    }
    xb = a.x + lm0 * a.x_stride;
    wb = a.w + ln0 * a.w_stride;
    // its scales and bias, before its first k-tile, so they are there when that is
    for (int e = wave; e < (BM + 2 * BN) / 64; e += C::W) {
      const int r = e * 64 + lane;
      const uint32_t to = lbase + S * C::STAGE + (lt & 1) * C::SC + e * 256;
      if (e < BM / 64) i8_load4(to, min(lm0 + r, a.M - 1) * 4, a.sx);
      else if (e < (BM + BN) / 64) i8_load4(to, min(ln0 + r - BM, a.N - 1) * 4, a.sw);
      else if (a.bias) i8_load4(to, min(ln0 + r - BM - BN, a.N - 1) * 4, a.bias);
    }
  };
  const auto clamp_tail = [&]() __attribute__((always_inline)) {   // chunks past a row's last one read that one
#pragma unroll
    for (int j = 0; j < NL; ++j) {
      const int over = lk * 8 + (slot ^ ((row_of(j) >> 1) & 7)) - last;
      if (over > 0) off[j] -= over * 16;
    }
  };
  const auto load = [&](int j, int so) __attribute__((always_inline)) {
    if (j < C::XL) i8_load16(lbase + so + (wave * C::XL + j) * 1024, off[j], xb + lk * 128);
    else i8_load16(lbase + so + BM * 128 + (wave * C::WL + j - C::XL) * 1024, off[j], wb + lk * 128);
  };
  const auto advance = [&]() __attribute__((always_inline)) {
    if (++lk == kts) {
      lk = 0;
      if (++lt < tiles) next_tile();
    }
    if (TAIL && lk == kts - 1) clamp_tail();       // (next_tile sets the offsets anew)
  };

  // ---- the products
  const int wm = wave % WM, wn = wave / WM, i = lane & 31, h = lane >> 5;
  const int key = (i >> 1) & 7, xrow = wm * 32 * MI + i, wrow = BM + wn * 32 * NI + i;
  i32x16_t acc[MI][NI];
  const auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < MI; ++s)
#pragma unroll
      for (int r = 0; r < NI; ++r)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[s][r][j] = 0;
  };
  i32x4_t x[2][MI], w[2][NI];
  const auto read = [&](int q, int so, int kk, int b) __attribute__((always_inline)) {
    const int at = ((kk * 2 + h) ^ key) * 16;
    if (q < NI) w[b][q] = *reinterpret_cast<const i32x4_t*>(lds + so + (wrow + 32 * q) * 128 + at);
    else x[b][q - NI] = *reinterpret_cast<const i32x4_t*>(lds + so + (xrow + 32 * (q - NI)) * 128 + at);
  };
  int ek = 0;                                      // the k-tile that is multiplied
  // Step kk on operands b = kk & 1; with `more` those of the next step (stage so) are read, and with `fill` the
  // loads of the stage that the barrier freed are issued.
  const auto step = [&](int kk, bool more, int so, bool fill, int fo) __attribute__((always_inline)) {
    const int b = kk & 1;
    int q = 0, j = 0;
    if (TAIL && ek == kts - 1) {
#pragma unroll
      for (int s = 0; s < MI; ++s) x[b][s] = keep_to(x[b][s], ek * 8 + kk * 2 + h, a.K);
    }
#pragma unroll
    for (int e = 0; e < NM; ++e) {
      if (more)
        while (q < NR && (e == NM - 1 || q * NM <= e * NR)) read(q++, so, (kk + 1) & 3, b ^ 1);
      if (fill)
        while (j < NL && (e == NM - 1 || j * NM <= e * NL)) load(j++, fo);
      const int es = e / NI, er = es & 1 ? NI - 1 - e % NI : e % NI;
      acc[es][er] = __builtin_amdgcn_mfma_i32_32x32x32_i8(x[b][es], w[b][er], acc[es][er], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);           // this order of loads, reads and MFMAs
    }
  };

  // ---- a tile's end
  int et = 0, drain = 0;
  const auto put = [&](auto dt, bool full, int em0, int n, const float* sc, const float (&sw)[NI], const float (&bs)[NI])
      __attribute__((always_inline)) {
    constexpr int DT = decltype(dt)::value;
#pragma unroll
    for (int s = 0; s < MI; ++s)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int ml = wm * 32 * MI + 32 * s + 8 * q + 4 * h;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const float sx = sc[ml + d];
          float v[NI];
#pragma unroll
          for (int r = 0; r < NI; ++r) {
            v[r] = ((float)acc[s][r][4 * q + d] * sx) * sw[r];
            if (a.bias) v[r] = v[r] + bs[r];
          }
          const int m = em0 + ml + d;
          const int64_t at = m * a.out_stride + n;
          if (!full) {
#pragma unroll
            for (int r = 0; r < NI; ++r)
              if (m < a.M && n + r < a.N) store_out(a.out, at + r, DT, v[r]);
          } else if constexpr (NI == 1) {
            store_out(a.out, at, DT, v[0]);
          } else if constexpr (DT == DT_F32) {
            *reinterpret_cast<u32x2_a4*>(static_cast<float*>(a.out) + at) =
                u32x2_a4{__float_as_uint(v[0]), __float_as_uint(v[1])};
          } else {
            *reinterpret_cast<u32_a2*>(static_cast<uint16_t*>(a.out) + at) =
                DT == DT_BF16 ? pack_bf16x2(v[0], v[1]) : pack_f16x2(v[0], v[1]);
          }
        }
      }
  };
  const auto finish = [&]() __attribute__((always_inline)) {
    asm volatile("" ::: "memory");                 // the stores come after the loads of this k-tile
    const int em0 = et & 1 ? pm1 : pm0, en0 = et & 1 ? pn1 : pn0;
    const float* sc = reinterpret_cast<const float*>(lds + S * C::STAGE + (et & 1) * C::SC);
    const int nl = wn * 32 * NI + NI * i, n = en0 + nl;
    float sw[NI], bs[NI];
#pragma unroll
    for (int r = 0; r < NI; ++r) {
      sw[r] = sc[BM + nl + r];
      bs[r] = a.bias ? sc[BM + BN + nl + r] : 0.0f;
    }
    const bool full = em0 + BM <= a.M && en0 + BN <= a.N;
    const auto go = [&](auto dt) __attribute__((always_inline)) {
      if (full) put(dt, true, em0, n, sc, sw, bs);
      else put(dt, false, em0, n, sc, sw, bs);
    };
    if (a.out_dtype == DT_BF16) go(std::integral_constant<int, DT_BF16>());
    else if (a.out_dtype == DT_F16) go(std::integral_constant<int, DT_F16>());
    else go(std::integral_constant<int, DT_F32>());
    // 16 MI stores, all newer than the loads of the next S - 1 k-tiles (a tile that ends at M or N may store less)
    drain = full ? S - 1 : 0;
    ++et;
    asm volatile("" ::: "memory");
  };

  next_tile();
  if (TAIL && kts == 1) clamp_tail();
#pragma unroll
  for (int d = 0; d < S; ++d)
    if (d < V) {
#pragma unroll
      for (int j = 0; j < NL; ++j) load(j, d * C::STAGE);
      advance();
    }
  if (V >= S) i8_sync<(S - 1) * NL>();
  else i8_sync<0>();
  clear();
#pragma unroll
  for (int q = 0; q < NR; ++q) read(q, 0, 0, 0);
#pragma unroll
  for (int kk = 0; kk < 3; ++kk) step(kk, true, 0, false, 0);
  int so = 0, v = 0;
  // Here the last step of k-tile v is to come; k-tiles up to v + S - 1 are on their way.
  for (; v + S < V; ++v) {
    if (drain > 0) {
      i8_sync<C::DRAIN>();
      --drain;
    } else {
      i8_sync<(S - 2) * NL>();
    }
    const int nx = so + C::STAGE == S * C::STAGE ? 0 : so + C::STAGE;
    step(3, true, nx, true, so);
    if (++ek == kts) {
      finish();
      clear();
      ek = 0;
    }
#pragma unroll
    for (int kk = 0; kk < 3; ++kk) step(kk, true, nx, false, 0);
    advance();
    so = nx;
  }
  for (; v + 1 < V; ++v) {
    i8_sync<0>();
    const int nx = so + C::STAGE == S * C::STAGE ? 0 : so + C::STAGE;
    step(3, true, nx, false, 0);
    if (++ek == kts) {
      finish();
      clear();
      ek = 0;
    }
#pragma unroll
    for (int kk = 0; kk < 3; ++kk) step(kk, true, nx, false, 0);
    so = nx;
  }
  step(3, false, 0, false, 0);
  finish();
}

template <int BM, int BN, int WM, int WN, int S>
void launch_i8_tile(dim3 grid, const I8Args& a, hipStream_t st) {
  const dim3 threads(64 * WM * WN);
  if (a.K & 127) hipLaunchKernelGGL((i8_tile_kernel<BM, BN, WM, WN, S, true>), grid, threads, 0, st, a);
  else hipLaunchKernelGGL((i8_tile_kernel<BM, BN, WM, WN, S, false>), grid, threads, 0, st, a);
}

// 256 x 128 and 256 x 256 tiles (fp4x_i8_large.hip: half of the compilation).
void launch_i8_256x128(dim3 grid, const I8Args& a, hipStream_t st);
void launch_i8_256x256(dim3 grid, const I8Args& a, hipStream_t st);

}  // namespace fp4x
