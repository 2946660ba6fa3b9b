// Products of 8-bit floats with a scale per block of 128:
//   out[m, n] = cast(sum_b (sum_{k in b} x[m, k] w[n, k]) * (sx[m, b] * sw[n / 128, b]) + bias[n])
// x e4m3 [M, K] with a scale per row and 128 values, w e4m3 [N, K] with a scale
// per 128 x 128 block.  A block's sum is one v_mfma_f32_16x16x128_f8f6f4 per 16
// x 16 outputs, which starts at 0; it is scaled and added to the outputs' fp32
// sums by fma in the order of the blocks.
//
// That instruction adds eight neighbouring products at a time, each cut to 2^-13
// of the power of two of the largest (measured; v_mfma_f32_16x16x32_fp8_fp8 does
// the same).  On average over normal values that is 1.5e-5 of a block's sum.  At
// worst it is 7 2^-13 = 8.5e-4 of the largest product of each eight: of the sum of
// magnitudes, so there is no bound relative to a result that cancels, and more
// than half a step of fp16 (4.9e-4; bf16 3.9e-3).  16-bit outputs take it all the
// same, since codes of e4m3 are themselves off by up to 2^-4 and exact products
// run at half of the rate.  For fp32 outputs (B16) both operands are turned into
// bf16, which holds every e4m3 value, and multiplied exactly.
//
// The same over experts: rows [off[e], off[e + 1]) of the output are products
// with expert e's weight, their rows of x picked by an index or lying in order.
#pragma once
#include "fp4x_i8.h"

namespace fp4x {

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));

struct F8Args {
  const uint8_t* x;  int64_t x_stride;  const float* sx;  int64_t sx_m, sx_b;   // scales' strides: row, block
  const uint8_t* w;  int64_t w_stride;  const float* sw;
  const float* bias;
  void* out;  int out_dtype;  int64_t out_stride;
  int M, N, K;
  int mt, nt, gm;                                  // tiles over M and N, tiles of M in a band
  int stream;                                      // large tiles: the output passes by the L2
  // experts
  const int *offsets, *tokens;                     // [E + 1]; rows of x or null
  int E, X;                                        // X: rows of x
  int64_t w_estride;
};

constexpr int kF8MaxExperts = 4096;                // 64 lanes of 64

// A tile: rows [m0, m_end) of the output and columns from n0, with the weight of expert e.
struct F8Place { int m0, m_end, n0, e; };

// Inclusive sum over the wave's lanes.
__device__ __forceinline__ int wave_sum_to(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);   // row_shr
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);   // row_bcast:31 into rows 2 and 3
  return v;
}

// A workgroup's tiles among the experts': expert by expert, the tiles of its rows
// per BN columns.  An XCD takes a run of consecutive tiles, in rounds of one per
// workgroup; a round is dealt one workgroup on from the round before, so that an
// expert's last tiles, which may hold a few rows only, do not all fall to some.
// Every wave finds them by itself: a lane sums the tiles of E / 64 experts, a scan
// gives the total, and then lane j looks its workgroup's tile j up, among the
// lanes' sums and then among the experts of one lane.  Offsets that do not rise,
// or leave the output's rows, give empty experts.  Returns the number of tiles,
// which the grid keeps to 64 at most; lane j < that holds tile j's place.
template <int BM, int BN>
__device__ __forceinline__ int f8_expert_tiles(const F8Args& a, F8Place& p) {
  const int lane = threadIdx.x & 63, per = (a.E + 63) >> 6;
  const auto at = [&](int e) __attribute__((always_inline)) { return min(max(a.offsets[min(e, a.E)], 0), a.M); };
  int sum = 0;
  for (int b = 0; b < per; b += 8) {
    int o[9];
#pragma unroll
    for (int i = 0; i < 9; ++i) o[i] = at(lane * per + min(b + i, per));
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += (max(o[i + 1] - o[i], 0) + BM - 1) / BM;
  }
  const int upto = wave_sum_to(sum), hit = min(a.M, a.E);   // (rising offsets stay within the bound by themselves)
  const int total = min(__builtin_amdgcn_readlane(upto, 63), (a.M - hit) / BM + hit) * a.nt;
  const int xcd = blockIdx.x & 7, stride = (gridDim.x + 7 - xcd) >> 3, own = blockIdx.x >> 3;
  const I8Run run(total, xcd);
  const int rounds = run.count / stride, rest = run.count - rounds * stride;
  const int tiles = rounds + ((own + rounds) % stride < rest);
  const int t = run.first + min(lane * stride + (own + lane) % stride, max(run.count - 1, 0));
  const int mt = t / a.nt;                         // the tile's place if every expert had one column
  int l = 0;
#pragma unroll
  for (int h = 32; h; h >>= 1)
    if (__shfl(upto, l + h - 1) <= mt) l += h;
  int begin = __shfl(upto - sum, l), found = 0, many = 1;
  p = F8Place{0, 0, 0, 0};
  for (int b = 0; b < per; b += 8) {
    int o[9];
#pragma unroll
    for (int i = 0; i < 9; ++i) o[i] = at(l * per + min(b + i, per));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int n = (max(o[i + 1] - o[i], 0) + BM - 1) / BM;
      if (mt >= begin && mt < begin + n) {
        p.e = l * per + b + i;
        p.m0 = o[i];
        p.m_end = o[i + 1];
        found = begin;
        many = n;
      }
      begin += n;
    }
  }
  const int r = t - found * a.nt, n = r / many;
  p.m0 += (r - n * many) * BM;
  p.n0 = n * BN;
  return tiles;
}
// The same for one tile per workgroup, which the lanes look up together: the second time each takes an expert (24 rows of
// 512 experts on 16 x 32 tiles took 1.1 us more with the function above).
template <int BM, int BN>
__device__ __forceinline__ bool f8_expert_tile(const F8Args& a, F8Place& p) {
  const int lane = threadIdx.x & 63, per = (a.E + 63) >> 6;
  const auto at = [&](int e) __attribute__((always_inline)) { return min(max(a.offsets[min(e, a.E)], 0), a.M); };
  int sum = 0;
  for (int b = 0; b < per; b += 8) {
    int o[9];
#pragma unroll
    for (int i = 0; i < 9; ++i) o[i] = at(lane * per + min(b + i, per));
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += (max(o[i + 1] - o[i], 0) + BM - 1) / BM;
  }
  const int upto = wave_sum_to(sum);
  const I8Run run(__builtin_amdgcn_readlane(upto, 63) * a.nt, blockIdx.x & 7);
  if ((int)(blockIdx.x >> 3) >= run.count) return false;
  const int t = run.first + (blockIdx.x >> 3), mt = t / a.nt;
  const int l = __builtin_ctzll(__ballot(upto > mt)), before = __builtin_amdgcn_readlane(upto - sum, l);
  const int e = l * per + min(lane, per), lo = at(e), hi = at(lane < per ? e + 1 : e);
  const int tiles = (max(hi - lo, 0) + BM - 1) / BM, to = before + wave_sum_to(tiles);
  const int i = __builtin_ctzll(__ballot(to > mt));
  const int own = __builtin_amdgcn_readlane(tiles, i), first = __builtin_amdgcn_readlane(to, i) - own;
  const int r = t - first * a.nt, n = own == 1 ? r : r / own;
  p = F8Place{__builtin_amdgcn_readlane(lo, i) + (r - n * own) * BM, __builtin_amdgcn_readlane(hi, i), n * BN, l * per + i};
  return true;
}
__device__ __forceinline__ F8Place f8_place_of(const F8Place& p, int j) {   // lane j's, for all
  return F8Place{__builtin_amdgcn_readlane(p.m0, j), __builtin_amdgcn_readlane(p.m_end, j), __builtin_amdgcn_readlane(p.n0, j),
                 __builtin_amdgcn_readlane(p.e, j)};
}

// Direct load of 4 bytes per lane, each from an address of its own, to lds + 4 lane.
__device__ __forceinline__ void f8_load4(uint32_t lds, const void* p) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds), "v"(p) : "m0");
}

// A lane's 32 bytes of a row's k-tile of 128: its chunks of 16 g and 4 + g.
// The MFMA pairs a lane's bytes of both operands whatever their place in K.
__device__ __forceinline__ i32x8_t f8_cat(i32x4_t a, i32x4_t b) {
  return i32x8_t{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}
__device__ __forceinline__ i32x8_t f8_keep(i32x8_t v, int c0, int K) {   // bytes from K on as zeros
  const i32x4_t a = keep_to(i32x4_t{v[0], v[1], v[2], v[3]}, c0, K), b = keep_to(i32x4_t{v[4], v[5], v[6], v[7]}, c0 + 4, K);
  return f8_cat(a, b);
}
// What the matrix cores take of those bytes: themselves, or as bf16.
template <bool B16> struct F8Frag {
  i32x8_t v;
  __device__ __forceinline__ void set(i32x8_t raw) { v = raw; }
};
template <> struct F8Frag<true> {
  u32x4_t v[4];
  __device__ __forceinline__ void set(i32x8_t raw) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
      v[c] = u32x4_t{fp8x2_to_bf16x2<false>(raw[2 * c], 1.0f), fp8x2_to_bf16x2<true>(raw[2 * c], 1.0f),
                     fp8x2_to_bf16x2<false>(raw[2 * c + 1], 1.0f), fp8x2_to_bf16x2<true>(raw[2 * c + 1], 1.0f)};
  }
};
template <bool B16>
__device__ __forceinline__ f32x4_t f8_block(const F8Frag<B16>& w, const F8Frag<B16>& x) {
  f32x4_t d = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  if constexpr (B16) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
      d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, w.v[c]), __builtin_bit_cast(bf16x8_t, x.v[c]), d, 0, 0, 0);
  } else {
    d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, x.v, d, 0, 0, 0, 0, 0, 0);
  }
  return d;
}

// Four neighbouring columns of a row; those from N on are left out.
__device__ __forceinline__ void f8_store4(const F8Args& a, int64_t m, int n, const float (&v)[4]) {
  const int64_t at = m * a.out_stride + n;
  if (n + 4 > a.N) {
    for (int j = 0; j < 4 && n + j < a.N; ++j) store_out(a.out, at + j, a.out_dtype, v[j]);
  } else if (a.out_dtype == DT_F32) {
    *reinterpret_cast<u32x4_a4*>(static_cast<float*>(a.out) + at) = u32x4_a4{
        __float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
  } else {
    const bool b = a.out_dtype == DT_BF16;
    *reinterpret_cast<u32x2_a2*>(static_cast<uint16_t*>(a.out) + at) =
        u32x2_a2{b ? pack_bf16x2(v[0], v[1]) : pack_f16x2(v[0], v[1]), b ? pack_bf16x2(v[2], v[3]) : pack_f16x2(v[2], v[3])};
  }
}

// 16 bytes of the output.  One that is larger than the 32 MB of the XCDs' L2 passes by it: it would push out the rows of x
// and w that the next tiles share (4096 x [16384 x 2560] took 175 us so, 163 with these stores).  Below that the next
// launch finds its input in the caches.  The store is asm because the compiler merges the two into a plain one; so it brings the two
// wait states that lie between a store of more than 64 bits and the next VALU write of its data (the compiler sees no store here).
template <class V>
__device__ __forceinline__ void f8_put(V* at, V v, int stream) {
  if (stream) asm volatile("global_store_dwordx4 %0, %1, off nt\n\ts_nop 1" ::"v"(at), "v"(v) : "memory");
  else *at = v;
}

// ------------------------------------------------------------------ small tiles
// A workgroup owns 16 MT rows of x and 16 NT rows of w; its W waves split K in
// units of 128 values, a block of scales each, and bring them through rings of
// their own by direct loads of whole cache lines, as the int8 product's small
// tiles do.  A unit's scales come with it (one more load: 16 MT of x, one of w,
// whose 16 NT rows lie in one block).  The waves' fp32 sums meet in LDS in the
// waves' order.
//
// Bound by the weight's bytes or by latency: 6 rows by [11316 x 9088], 103 MB, take
// 19.3 us (5.3 TB/s; a large copy moves 5.1), 3 rows by [2560 x 640] 3.3.  K is
// split over the W waves of a workgroup, D units of each on their way, and not over
// workgroups, whose sums would take a second pass over memory.
template <int MT, int NT, int W, int D, bool EX, bool B16>
__global__ __launch_bounds__(64 * W, 2) void f8_ring_kernel(const F8Args a) {
  constexpr int R = 16 * (MT + NT), NL = R / 8, STAGE = R * 128 + 256;
  constexpr int LD = 16 * NT + 4;                  // (a row of sums starts on 16 bytes)
  constexpr int ITEMS = (64 * MT * NT + 64 * W - 1) / (64 * W);   // of four columns, per thread
  static_assert(D * STAGE >= 16 * MT * LD * 4, "the sums reuse the ring");
  __shared__ __attribute__((aligned(1024))) char lds[W * D * STAGE];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), i = lane & 15, g = lane >> 4;
  F8Place p{0, a.M, 0, 0};
  if constexpr (EX) {
    if (!f8_expert_tile<16 * MT, 16 * NT>(a, p)) return;
  } else {
    const I8Run run(a.mt * a.nt, blockIdx.x & 7);
    tile_place(a.mt, a.nt, a.gm, run.first + (blockIdx.x >> 3), 16 * MT, 16 * NT, p.m0, p.n0);
  }
  const int units = (a.K + 127) >> 7, per = (units + W - 1) / W, u0 = wave * per;
  const int n = max(min(per, units - u0), 0);      // this wave's units
  const int tail = a.K & 127 ? units - 1 - u0 : -1;   // the one that K ends in, if any
  const int last = (a.K - 1) >> 4;
  const bool pick = EX && a.tokens;
  const auto x_row = [&](int r) __attribute__((always_inline)) {   // row of x of row r of the tile
    const int m = min(p.m0 + r, p.m_end - 1);
    return pick ? min(max(a.tokens[m], 0), a.X - 1) : m;
  };
  // LDS row r holds chunk c of its 128 bytes at c ^ key: the 16 lanes that LDS serves together read different banks
  const int slot = lane & 7, lr = lane >> 3;
  uint32_t off[NL];
#pragma unroll
  for (int j = 0; j < NL; ++j) {
    const int r = j * 8 + lr, c = slot ^ ((r >> 1) & 7);
    if (j < 2 * MT) off[j] = (uint32_t)(x_row(r) - (pick ? 0 : p.m0)) * (uint32_t)a.x_stride + c * 16;
    else off[j] = (uint32_t)(min(p.n0 + r - 16 * MT, a.N - 1) - p.n0) * (uint32_t)a.w_stride + c * 16;
  }
  const uint8_t* xb = a.x + (pick ? 0 : p.m0 * a.x_stride) + u0 * 128;
  const uint8_t* wb = a.w + p.e * a.w_estride + p.n0 * a.w_stride + u0 * 128;
  const int64_t sw_row = (int64_t)p.e * ((a.N + 127) >> 7) + (p.n0 >> 7);
  const float* sp = lane < 16 * MT ? a.sx + x_row(lane) * a.sx_m + u0 * a.sx_b : a.sw + sw_row * units + u0;
  const int64_t step = lane < 16 * MT ? a.sx_b : 1;
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
    f8_load4(base + s * STAGE + R * 128, sp);
    sp += step;
  };
  float bias[ITEMS][4];                            // before the units: a wait for a unit is then one for them too
#pragma unroll
  for (int q = 0; q < ITEMS; ++q) {
    const int e = t + q * 64 * W, c = p.n0 + 4 * (e % (4 * NT));
#pragma unroll
    for (int j = 0; j < 4; ++j) bias[q][j] = !EX && a.bias ? a.bias[min(c + j, a.N - 1)] : 0.0f;
  }
  asm volatile("" ::: "memory");                   // not behind the units' loads, whose waits count what is newer
  f32x4_t acc[MT][NT];
#pragma unroll
  for (int s = 0; s < MT; ++s)
#pragma unroll
    for (int r = 0; r < NT; ++r) acc[s][r] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int d = 0; d < D; ++d)
    if (d < n) issue(d, d);
  int stage = 0;
  for (int u = 0; u < n; ++u) {
    if (u + D - 1 < n) i8_wait<(D - 1) * (NL + 1)>();
    else i8_wait<0>();
    const char* st = mine + stage * STAGE;
    const auto read = [&](int row) __attribute__((always_inline)) {
      const int key = (i >> 1) & 7;
      const char* at = st + (row + i) * 128;
      return f8_cat(*reinterpret_cast<const i32x4_t*>(at + (g ^ key) * 16),
                    *reinterpret_cast<const i32x4_t*>(at + ((4 + g) ^ key) * 16));
    };
    i32x8_t x[MT], w[NT];
#pragma unroll
    for (int r = 0; r < NT; ++r) w[r] = read(16 * MT + 16 * r);
#pragma unroll
    for (int s = 0; s < MT; ++s) x[s] = read(16 * s);
    const float* sc = reinterpret_cast<const float*>(st + R * 128);
    float f[MT];
#pragma unroll
    for (int s = 0; s < MT; ++s) f[s] = sc[16 * s + i] * sc[16 * MT];
    if (u == tail) {                               // (both operands: bytes past K may be NaN codes)
#pragma unroll
      for (int s = 0; s < MT; ++s) x[s] = f8_keep(x[s], (u0 + u) * 8 + g, a.K);
#pragma unroll
      for (int r = 0; r < NT; ++r) w[r] = f8_keep(w[r], (u0 + u) * 8 + g, a.K);
    }
    F8Frag<B16> wf[NT];
#pragma unroll
    for (int r = 0; r < NT; ++r) wf[r].set(w[r]);
#pragma unroll
    for (int s = 0; s < MT; ++s) {
      F8Frag<B16> xf;
      xf.set(x[s]);
#pragma unroll
      for (int r = 0; r < NT; ++r) {
        const f32x4_t b = f8_block(wf[r], xf);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[s][r][j] = __builtin_fmaf(b[j], f[s], acc[s][r][j]);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the stage is read before it is filled again
    if (u + D < n) issue(stage, u + D);
    if (++stage == D) stage = 0;
  }
  // the wave's sums take the place of its ring
  float* sum = reinterpret_cast<float*>(lds + wave * D * STAGE);
#pragma unroll
  for (int s = 0; s < MT; ++s)
#pragma unroll
    for (int r = 0; r < NT; ++r) *reinterpret_cast<f32x4_t*>(&sum[(16 * s + i) * LD + 16 * r + 4 * g]) = acc[s][r];
  __syncthreads();
#pragma unroll
  for (int q = 0; q < ITEMS; ++q) {
    const int e = t + q * 64 * W, m = e / (4 * NT), c = e % (4 * NT);
    if (e < 64 * MT * NT && p.m0 + m < p.m_end && p.n0 + 4 * c < a.N) {
      f32x4_t v = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < W; ++k) v += *reinterpret_cast<const f32x4_t*>(lds + k * D * STAGE + (m * LD + 4 * c) * 4);
      const float y[4] = {v[0] + bias[q][0], v[1] + bias[q][1], v[2] + bias[q][2], v[3] + bias[q][3]};
      f8_store4(a, p.m0 + m, p.n0 + 4 * c, y);
    }
  }
}

// ------------------------------------------------------------------ large tiles
// A workgroup owns BM rows of x and BN rows of w at a time and walks K in
// k-tiles of 128, a block of scales each, through S LDS stages filled by direct
// loads.  Wave (wm, wn) owns 16 MS rows of x and 16 NS of w.  A k-tile is MS
// steps, one per strip of 16 rows of x, of NS MFMAs; during a step the next
// strip is read, and in the last one, behind the k-tile's only barrier, the
// first of the next k-tile and its rows of w, each once its last MFMA is issued.
// A block's sum is scaled and added two MFMAs later, in the shadow of the next.
//
// 4096 x [16384 x 2560] (256 x 256 tiles) takes 155 to 165 us in calls in a row,
// 2.1 to 2.2 PFLOP/s (158 to 193 in a trace).
// With parts of it left out (copies of the kernel): the MFMAs alone 110, with the
// scaling 120, with the reads of LDS 127, with the loads 145, with the stores 160.
// So it is bound by the matrix cores, and what is not under them is a tile's end
// and start (a tile has 20 k-tiles).  4096 tokens x 8 over 128 experts of [2560 x
// 640] (five k-tiles a tile) takes 98 to 99 us on one input and 110 to 117 where
// inputs change (115 to 124 in a trace); its bytes are 78 us' worth.  A third of
// its tiles' rows are none; MFMAs of such strips are left out, by wave and, in 256 x
// 256 tiles, by half a wave's strips, with one wave of each half on a SIMD (whole
// waves, both of a SIMD in one half: 116 us beside 110; strip by strip the registers
// spill).
// No gain from wave priorities, loads into L2 ahead, spread or bunched loads, later
// waits, workgroups that start apart, other bands (gm) of tiles, scale blocks an
// odd number of lines apart, or a tile's stores under the next one's first MFMAs.
//
// Weight rows are dealt to the MFMA's rows so that a lane holds 4 NS
// neighbouring columns of each of its rows of y.
template <int BM, int BN, int WM, int WN, int S>
struct F8Tile {
  static constexpr int W = WM * WN, MS = BM / WM / 16, NS = BN / WN / 16;
  static constexpr int SCALES = BM + 64;           // of x, then of w (a block each)
  static constexpr int STAGE = (BM + BN) * 128 + SCALES * 4, XL = BM / 8 / W, WL = BN / 8 / W, NL = XL + WL + 1;
  static constexpr int LDS = S * STAGE + 2 * BN * 4;   // and the bias of two tiles
  static constexpr int DRAIN = (S - 2) * NL + MS * NS / 2 < 63 ? (S - 2) * NL + MS * NS / 2 : 63;
  static_assert(MS * 16 * WM == BM && NS * 16 * WN == BN && XL * 8 * W == BM && WL * 8 * W == BN && BM % 64 == 0 &&
                BN % 64 == 0 && (128 % (16 * NS)) == 0 && MS % 2 == 0 && MS * NS % 4 == 0 && NS % 2 == 0 && S >= 2 &&
                W > BM / 64, "tile");
};

template <int BM, int BN, int WM, int WN, int S, bool EX, bool B16>
__global__ __launch_bounds__(64 * WM * WN, 2) void f8_tile_kernel(const F8Args a) {
  using C = F8Tile<BM, BN, WM, WN, S>;
  constexpr int MS = C::MS, NS = C::NS, NL = C::NL;
  __shared__ __attribute__((aligned(1024))) char lds[C::LDS];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  F8Place all;                                     // EX: lane j holds tile j's
  int first = 0, stride = 1, tiles = 1;
  if constexpr (EX) {
    tiles = f8_expert_tiles<BM, BN>(a, all);
    if (tiles < 1) return;
  } else {
    const int xcd = blockIdx.x & 7;
    const I8Run run(a.mt * a.nt, xcd);
    stride = (gridDim.x + 7 - xcd) >> 3;           // workgroups of this XCD
    first = run.first + (blockIdx.x >> 3);
    tiles = (run.count - (blockIdx.x >> 3) + stride - 1) / stride;
  }
  const int kts = (a.K + 127) >> 7, V = tiles * kts;
  const int last = (a.K - 1) >> 4;
  const bool tail = a.K & 127;                     // K ends inside a k-tile
  const bool pick = EX && a.tokens;

  // The lane, where what is computed from it is not to be kept in registers through the loop over K (the 256 x 256 tiles
  // have none left; a value that is spilled there is loaded again behind a wait for every load on its way).
  const auto lane_here = [&]() __attribute__((always_inline)) {
    int l = lane;
    asm volatile("" : "+v"(l));
    return l;
  };

  // ---- the loads: k-tile lk of tile lt
  // LDS row r holds chunk c of its 128 bytes at c ^ key: the 16 lanes that LDS serves together read different banks
  const uint32_t lbase = i8_lds(lds);
  int lt = 0, lk = 0;
  F8Place lp{0, a.M, 0, 0};
  int pm0 = 0, pn0 = 0, pm1 = 0, pn1 = 0;          // places of an even and of an odd tile
  uint32_t off[NL - 1];
  const uint8_t *xb, *wb;
  uint32_t soff;                                   // the scale that this lane brings of each k-tile
  const float* sb;
  const int64_t sstep = wave < BM / 64 ? a.sx_b : 1;
  const auto row_of = [&](int j, int l) __attribute__((always_inline)) {   // LDS row of load j in its operand's half
    return ((j < C::XL ? wave * C::XL + j : wave * C::WL + j - C::XL) << 3) + (l >> 3);
  };
  const auto x_row = [&](int r) __attribute__((always_inline)) {    // row of x of row r of the tile
    const int m = min(lp.m0 + r, lp.m_end - 1);
    return pick ? min(max(a.tokens[m], 0), a.X - 1) : m;
  };
  const auto next_tile = [&]() __attribute__((always_inline)) {
    if constexpr (EX) {
      lp = f8_place_of(all, lt);
    } else {
      tile_place(a.mt, a.nt, a.gm, first + lt * stride, BM, BN, lp.m0, lp.n0);
      if (lt & 1) {
        pm1 = lp.m0;
        pn1 = lp.n0;
      } else {
        pm0 = lp.m0;
        pn0 = lp.n0;
      }
    }
    const int l = lane_here();
#pragma unroll
    for (int j = 0; j < NL - 1; ++j) {
      const int r = row_of(j, l), c = (l & 7) ^ ((r >> 1) & 7);
      if (j < C::XL) off[j] = (uint32_t)(x_row(r) - (pick ? 0 : lp.m0)) * (uint32_t)a.x_stride + c * 16;
      else {
        const int wr = (r & -(16 * NS)) + ((r & 15) >> 2) * (4 * NS) + ((r >> 4) % NS) * 4 + (r & 3);
        off[j] = (uint32_t)(min(lp.n0 + wr, a.N - 1) - lp.n0) * (uint32_t)a.w_stride + c * 16;
      }
    }
    xb = a.x + (pick ? 0 : lp.m0 * a.x_stride);
    wb = a.w + lp.e * a.w_estride + lp.n0 * a.w_stride;
    const int nbs = (a.N + 127) >> 7;
    if (wave < BM / 64) {
      soff = (uint32_t)(x_row(wave * 64 + l) - (pick ? 0 : lp.m0)) * (uint32_t)a.sx_m * 4;
      sb = a.sx + (pick ? 0 : lp.m0 * a.sx_m);
    } else {                                       // (several waves bring the same values)
      soff = min(l, nbs - 1 - (lp.n0 >> 7)) * kts * 4;
      sb = a.sw + ((int64_t)lp.e * nbs + (lp.n0 >> 7)) * kts;
    }
    // its bias, before its first k-tile, so it is there when that is
    if (!EX && a.bias)
      for (int e = wave; e < BN / 64; e += C::W)
        i8_load4(__builtin_amdgcn_readfirstlane(lbase + S * C::STAGE + (lt & 1) * BN * 4 + e * 256), min(lp.n0 + e * 64 + l, a.N - 1) * 4, a.bias);
  };
  const auto clamp_tail = [&]() __attribute__((always_inline)) {   // chunks past a row's last one read that one
    const int l = lane_here();
#pragma unroll
    for (int j = 0; j < NL - 1; ++j) {
      const int over = lk * 8 + ((l & 7) ^ ((row_of(j, l) >> 1) & 7)) - last;
      if (over > 0) off[j] -= over * 16;
    }
  };
  const auto load = [&](int j, int so) __attribute__((always_inline)) {
    const auto to = [&](int at) { return __builtin_amdgcn_readfirstlane(lbase + so + at); };   // (scalars, for the asm)
    const int k = __builtin_amdgcn_readfirstlane(lk);
    if (j < C::XL) i8_load16(to((wave * C::XL + j) * 1024), off[j], xb + k * 128);
    else if (j < NL - 1) i8_load16(to(BM * 128 + (wave * C::WL + j - C::XL) * 1024), off[j], wb + k * 128);
    else i8_load4(to((BM + BN) * 128 + min(wave, BM / 64) * 256), soff, sb + k * sstep);
  };
  const auto advance = [&]() __attribute__((always_inline)) {
    if (++lk == kts) {
      lk = 0;
      if (++lt < tiles) next_tile();
    }
    if (tail && lk == kts - 1) clamp_tail();       // (next_tile sets the offsets anew)
  };

  // Zeros in place of what lies past K in a tile's last k-tile: both operands', since those bytes may be NaN codes.
  // (In LDS, behind a barrier of its own: masks in registers would not fit beside 256 x 256 sums.)
  const auto cut = [&](int so) __attribute__((always_inline)) {
    for (int r = wave * 64 + lane_here(); r < BM + BN; r += 64 * C::W)
      for (int c = (a.K & 127) >> 4; c < 8; ++c) {
        i32x4_t* at = reinterpret_cast<i32x4_t*>(lds + so + r * 128 + ((c ^ ((r >> 1) & 7)) * 16));
        *at = keep_to(*at, c, a.K & 127);
      }
    i8_sync<63>();
  };

  // ---- the products
  // Over experts a tile's upper rows may be all there are: with two waves to a SIMD each has one of its upper half.
  constexpr bool DEAL = EX && C::W == 8;
  const int wm = DEAL ? wave / WN : wave % WM, wn = DEAL ? wave % WN : wave / WM, i = lane & 15, g = lane >> 4, key = (i >> 1) & 7;
  // a lane's chunks of the first strip of x, and how far on the first one of w is
  const int c0 = (wm * 16 * MS + i) * 128 + (g ^ key) * 16, c1 = (wm * 16 * MS + i) * 128 + ((4 + g) ^ key) * 16;
  const int w_on = (BM + wn * 16 * NS - wm * 16 * MS) * 128;
  const int sx_at = (BM + BN) * 128 + (wm * 16 * MS + i) * 4, sw_at = (BM + BN) * 128 + BM * 4 + (wn * 16 * NS / 128) * 4;
  f32x4_t acc[MS][NS], part[4];
  i32x8_t x[2], w[NS];
  F8Frag<B16> wf[NS];
  float f[2], sx, sw;                              // f: both scales of a strip, of the next one still apart
  const auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < MS; ++s)
#pragma unroll
      for (int r = 0; r < NS; ++r) acc[s][r] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    part[2] = part[3] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};   // nothing waits to be added
    f[1] = 0.0f;
  };
  const auto fetch = [&](int so, int strip) __attribute__((always_inline)) {   // of x; of w: so + w_on
    return f8_cat(*reinterpret_cast<const i32x4_t*>(lds + so + c0 + strip * 2048),
                  *reinterpret_cast<const i32x4_t*>(lds + so + c1 + strip * 2048));
  };
  const auto scale = [&](int so, int s) __attribute__((always_inline)) {
    return *reinterpret_cast<const float*>(lds + so + sx_at + 64 * s);
  };
  int ek = 0, et = 0;                              // the k-tile that is multiplied, and its tile
  // EX: whether the tile has rows for this wave; where it owns eight strips, for how many of none, half or all.
  constexpr bool HALVES = EX && MS >= 8;
  std::conditional_t<HALVES, int, bool> busy = HALVES ? MS : 1;
  const auto look = [&]() __attribute__((always_inline)) {
    if constexpr (EX) {
      const F8Place ep = f8_place_of(all, min(et, tiles - 1));
      const int rows = ep.m_end - ep.m0 - wm * 16 * MS;
      if constexpr (HALVES) busy = rows <= 0 ? 0 : rows <= 8 * MS ? MS / 2 : MS;
      else busy = ep.m0 + wm * 16 * MS < ep.m_end;
    }
  };
  const auto add = [&](int e) __attribute__((always_inline)) {   // block e of a k-tile into its sums
    const int s = e / NS, r = e % NS;
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[s][r][j] = __builtin_fmaf(part[e & 3][j], f[s & 1], acc[s][r][j]);
    asm volatile("" : "+v"(acc[s][r]));            // here, not sunk to a later block with its part kept until then
  };
  const auto first_of = [&](int so) __attribute__((always_inline)) {   // a k-tile's first reads
#pragma unroll
    for (int r = 0; r < NS; ++r) w[r] = fetch(so + w_on, r);
    x[0] = fetch(so, 0);
    sx = scale(so, 0);
    sw = *reinterpret_cast<const float*>(lds + so + sw_at);
  };
  // Step s of a k-tile in stage so.  In the last step `more` reads from the next stage `nx`, and `fill` issues the loads
  // of the stage that the barrier freed.  The order is pinned: an MFMA, then what does not wait for it.
  // Strips that the tile has no rows for are left out, but for the wave's part in the loads.
  const auto step = [&](int s, int so, bool more, int nx, bool fill) __attribute__((always_inline)) {
    const bool end = s == MS - 1;
    if (EX && (HALVES && s >= MS / 2 ? busy != MS : !busy)) {
      if (HALVES && s == MS / 2 && busy) {
        add(s * NS - 2);
        add(s * NS - 1);
      }
      if (fill)
#pragma unroll
        for (int j = 0; j < NL; ++j) load(j, so);
      if (end && more) first_of(nx);
      return;
    }
    F8Frag<B16> xf;
    xf.set(x[s & 1]);
    int j = 0;
#pragma unroll
    for (int r = 0; r < NS; ++r) {
      const int e = s * NS + r;
      if (!B16 || s == 0) wf[r].set(w[r]);
      part[e & 3] = f8_block(wf[r], xf);
      if (!end) __builtin_amdgcn_sched_barrier(0);
      if (r == 0 && !end) x[(s + 1) & 1] = fetch(so, s + 1);
      if (r == 0 && end && more) x[0] = fetch(nx, 0);
      if (end && more) w[r] = fetch(nx + w_on, r);
      add(e < 2 ? e - 2 + MS * NS : e - 2);
      if (r == 1) {                                // the strip before is done with its scales
        f[s & 1] = sx * sw;
        if (!end) sx = scale(so, s + 1);
        if (end && more) {
          sx = scale(nx, 0);
          sw = *reinterpret_cast<const float*>(lds + nx + sw_at);
        }
      }
      if (fill)
        while (j < NL && (r == NS - 1 || j * NS <= r * NL)) load(j++, so);
      if (!end) {
        __builtin_amdgcn_sched_barrier(0);
      } else {
        __builtin_amdgcn_sched_group_barrier(0x008, B16 ? 4 : 1, 0);
        if (more) {
          if (r < 2) __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
          else __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        if (r == 1) __builtin_amdgcn_sched_group_barrier(0x002, 5, 0);
        else __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
      }
    }
  };

  // ---- a tile's end
  int drain = 0;
  // A lane's 4 NS columns of a row are NP pieces of 16 bytes.  The four lanes of a row exchange theirs (rows of 16 lanes,
  // then halves of the wave), so that a store would write 64 bytes of each of 16 rows, and then the halves of 8 rows: a
  // store writes whole lines of 8 rows where those start on one (NP 1: 64 bytes of 16).
  const auto put = [&](auto dt, int l, const F8Place& ep, int n0, const float (&bs)[4 * NS]) __attribute__((always_inline)) {
    constexpr int DT = decltype(dt)::value, PER = DT == DT_F32 ? 4 : 8, NP = 4 * NS / PER;
#pragma unroll
    for (int s = 0; s < MS; ++s) {
      if (HALVES && s >= MS / 2 && busy != MS) break;
      uint32_t d[NP][4];
#pragma unroll
      for (int q = 0; q < NP; ++q)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int c = PER * q + PER / 4 * k;
          const float lo = acc[s][c >> 2][c & 3] + bs[c];
          if constexpr (DT == DT_F32) {
            d[q][k] = __float_as_uint(lo);
          } else {
            const float hi = acc[s][c >> 2][(c & 3) + 1] + bs[c + 1];
            d[q][k] = DT == DT_BF16 ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
          }
        }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int q = 0; q + 1 < NP; q += 2) {
          const auto v = __builtin_amdgcn_permlane16_swap(d[q][k], d[q + 1][k], false, false);
          d[q][k] = v[0];
          d[q + 1][k] = v[1];
        }
#pragma unroll
        for (int q = 0; q < NP / 2; ++q) {
          const auto v = __builtin_amdgcn_permlane32_swap(d[q][k], d[q + NP / 2][k], false, false);
          d[q][k] = v[0];
          d[q + NP / 2][k] = v[1];
        }
#pragma unroll
        for (int q = 0; q + 1 < NP; q += 2) {      // lanes 8 to 15 of 16 <-> lanes 0 to 7, of the other piece
          const int u = (int)d[q][k], v = (int)d[q + 1][k];
          d[q][k] = (uint32_t)__builtin_amdgcn_update_dpp(u, v, 0x128, 0xf, 0xc, false);
          d[q + 1][k] = (uint32_t)__builtin_amdgcn_update_dpp(v, u, 0x128, 0xf, 0x3, false);
        }
      }
#pragma unroll
      for (int q = 0; q < NP; ++q) {
        const int row = NP == 1 ? l & 15 : 8 * (q & 1) + (l & 7), piece = NP == 1 ? l >> 4 : 8 * (q >> 1) + (l >> 1 & 4) + (l >> 4);
        const int m = ep.m0 + wm * 16 * MS + 16 * s + row, n = n0 + piece * PER;
        if (m < ep.m_end) {
          const int64_t at = m * a.out_stride + n;
          if (n + PER > a.N) {
            for (int k = 0; k < PER && n + k < a.N; ++k) {
              if constexpr (DT == DT_F32) static_cast<uint32_t*>(a.out)[at + k] = k < 2 ? (k ? d[q][1] : d[q][0]) : d[q][2];
              else static_cast<uint16_t*>(a.out)[at + k] = (uint16_t)((k < 2 ? d[q][0] : k < 4 ? d[q][1] : k < 6 ? d[q][2] : d[q][3]) >> (16 * (k & 1)));
            }
          } else if constexpr (DT == DT_F32) {
            f8_put(reinterpret_cast<u32x4_a4*>(static_cast<float*>(a.out) + at), u32x4_a4{d[q][0], d[q][1], d[q][2], d[q][3]}, a.stream);
          } else {
            f8_put(reinterpret_cast<u32x4_a2*>(static_cast<uint16_t*>(a.out) + at), u32x4_a2{d[q][0], d[q][1], d[q][2], d[q][3]}, a.stream);
          }
        }
      }
    }
  };
  const auto finish = [&]() __attribute__((always_inline)) {
    if (EX && !busy) {
      drain = 0;
      ++et;
      return;
    }
    add(MS * NS - 2);
    add(MS * NS - 1);
    asm volatile("" ::: "memory");                 // the stores come after the loads of this k-tile
    F8Place ep{et & 1 ? pm1 : pm0, a.M, et & 1 ? pn1 : pn0, 0};
    if constexpr (EX) ep = f8_place_of(all, et);
    const float* bp = reinterpret_cast<const float*>(lds + S * C::STAGE + (et & 1) * BN * 4);
    const int l = lane_here(), nl = wn * 16 * NS, n0 = ep.n0 + nl;
    float bs[4 * NS] = {};
    if (!EX && a.bias)
#pragma unroll
      for (int q = 0; q < 4 * NS; ++q) bs[q] = bp[nl + 4 * NS * (l >> 4) + q];
    if constexpr (B16) put(std::integral_constant<int, DT_F32>(), l, ep, n0, bs);
    else if (a.out_dtype == DT_BF16) put(std::integral_constant<int, DT_BF16>(), l, ep, n0, bs);
    else put(std::integral_constant<int, DT_F16>(), l, ep, n0, bs);
    // at least MS NS / 2 stores, all newer than the loads of the next S - 1 k-tiles (a tile that ends at M or N may store less)
    drain = ep.m0 + BM <= ep.m_end && ep.n0 + BN <= a.N ? S - 1 : 0;
    ++et;
    asm volatile("" ::: "memory");
  };

  next_tile();
  if (tail && kts == 1) clamp_tail();
#pragma unroll
  for (int d = 0; d < S; ++d)
    if (d < V) {
#pragma unroll
      for (int j = 0; j < NL; ++j) load(j, d * C::STAGE);
      advance();
    }
  if (V >= S) i8_sync<(S - 1) * NL>();
  else i8_sync<0>();
  if (tail && kts == 1) cut(0);
  clear();
  look();
  first_of(0);
#pragma unroll
  for (int s = 0; s < MS - 1; ++s) step(s, 0, true, 0, false);
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
    if (tail && (ek + 2 == kts || kts == 1)) cut(nx);
    step(MS - 1, so, true, nx, true);
    if (++ek == kts) {
      finish();
      clear();
      look();
      ek = 0;
    }
#pragma unroll
    for (int s = 0; s < MS - 1; ++s) step(s, nx, true, 0, false);
    advance();
    so = nx;
  }
  for (; v + 1 < V; ++v) {
    i8_sync<0>();
    const int nx = so + C::STAGE == S * C::STAGE ? 0 : so + C::STAGE;
    if (tail && (ek + 2 == kts || kts == 1)) cut(nx);
    step(MS - 1, so, true, nx, false);
    if (++ek == kts) {
      finish();
      clear();
      look();
      ek = 0;
    }
#pragma unroll
    for (int s = 0; s < MS - 1; ++s) step(s, nx, true, 0, false);
    so = nx;
  }
  step(MS - 1, so, false, 0, false);
  finish();
}

template <int BM, int BN, int WM, int WN, int S, bool EX, bool B16>
void launch_f8_tile(dim3 grid, const F8Args& a, hipStream_t st) {
  const dim3 threads(64 * WM * WN);
  hipLaunchKernelGGL((f8_tile_kernel<BM, BN, WM, WN, S, EX, B16>), grid, threads, 0, st, a);
}

// The forms: 0 to 3 small tiles, 4 to 9 large ones; and which of them there are, plain and over experts, for 16-bit and (B16)
// fp32 outputs.  One is left out where the others cost less than 1% more without it (the sizes are fp4x_f8.hip's); 256 x 256
// tiles have no room for bf16 operands beside their sums.
constexpr int kF8Forms = 10;
constexpr uint32_t kF8Have[2][2] = {{0x3ff, 0x0b7}, {0x2b6, 0x0b6}};   // [experts][B16], bit f: form f

// The launch of each form (fp4x_f8_forms.h), in units of their own.
void launch_f8_dense(int form, dim3 grid, const F8Args& a, hipStream_t st);
void launch_f8_dense_b16(int form, dim3 grid, const F8Args& a, hipStream_t st);
void launch_f8_experts(int form, dim3 grid, const F8Args& a, hipStream_t st);
void launch_f8_experts_b16(int form, dim3 grid, const F8Args& a, hipStream_t st);

}  // namespace fp4x
