// Tokens sorted by expert and back: expert_sort, expert_rows, expert_combine and
// its gradient.
//
// A router gives each of T tokens k experts' ids.  The T k pairs, sorted by
// expert and within one by their place (token by token), are the rows of the
// experts' products: offsets[e] is where expert e's rows begin, tokens[s] the
// token of row s, slots[t, j] the row of pair (t, j).  Pairs whose id is no
// expert (negative, or another rank's) have slot -1 and no row; the rows behind
// the last expert's have token -1.
//
// Rows:     r[s] = x[tokens[s]]
// Combine:  out[t] = sum_j w[t, j] y[slots[t, j]]  (fp32, j in order)
// Gradient: dy[slots[t, j]] = w[t, j] dout[t],  dw[t, j] = dout[t] . y[slots[t, j]]
// and the gradient of the rows is the combine without weights.  No atomic decides
// an order: every result is the same in every run.
#include <algorithm>
#include <climits>
#include <string>

#include "fp4x_f8.h"
#include "../../include/fp4x.h"

namespace fp4x {

static int ex_fail(const char* what, const char* why) {
  set_error(std::string(what) + ": " + why);
  return FP4X_ERR_ARG;
}

// ------------------------------------------------------------------ sort
// A counting sort.  A workgroup takes a chunk of consecutive pairs, each of its W
// counting waves a run of that, 256 at a time, four ids per lane: counts per wave
// and expert in LDS, their sums over the waves before (a thread per expert), and
// then every wave gives its pairs, 64 at a time, the next places of their experts;
// within the 64 a pair's place is the number of lanes before it with the same id.
//
// Up to 256 W pairs one workgroup does all, and its ids stay in registers between
// the two passes.  Above, a first launch counts per chunk, and in the second each
// workgroup adds up the chunks before its own and the totals (at most kSortChunks
// of E counts, from L2).
//
// Bound by latency, not by its 24 bytes per pair: 24 pairs of 512 experts take 2.8
// us, 32008 of 256 experts 9.3 to 10.5 in two launches (in a trace 3.8 + 6.0 at the
// least), where the bytes are 0.2: a kernel's start and reads that wait for each
// other (ids, the chunks' counts).  Every workgroup reads all chunks' counts, 256 E at
// the most: 2^20 pairs take 26 us with 512 experts and 75 with 4096, where that is 1
// GB from the L2 and the pairs' bytes are 5 us' worth.
constexpr int kSortOne = 4096, kSortChunks = 256;

struct SortArgs {
  const void* ids;  int wide;  int64_t row;        // int64 or int32, elements between tokens
  int P, k, E, rounds, chunks;                     // rounds of 256 pairs per wave and chunk
  int* hist;                                       // [chunks][E]
  int *offsets, *tokens, *slots;
};

struct SortRun {                                   // a wave's pairs [p0, p1)
  int p0, p1;
  __device__ SortRun(const SortArgs& a, int W) {
    const int wave = threadIdx.x >> 6;
    const int64_t lo = ((int64_t)blockIdx.x * W + wave) * 256 * a.rounds;
    p0 = wave < W ? (int)min(lo, (int64_t)a.P) : a.P;
    p1 = wave < W ? (int)min(lo + 256 * a.rounds, (int64_t)a.P) : a.P;
  }
};
// Ids of pairs p, p + 64, .. (E: none, or past p1).
__device__ __forceinline__ void sort_ids(const SortArgs& a, int p, int p1, int (&id)[4]) {
  int64_t v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int q = p + 64 * i;
    v[i] = -1;
    if (q < p1) {
      int64_t at = q;
      if (a.row != a.k) at = (unsigned)q / (unsigned)a.k * a.row + (unsigned)q % (unsigned)a.k;
      v[i] = a.wide ? static_cast<const int64_t*>(a.ids)[at] : static_cast<const int*>(a.ids)[at];
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) id[i] = v[i] >= 0 && v[i] < a.E ? (int)v[i] : a.E;
}
template <int W>
__device__ __forceinline__ void sort_count(const SortArgs& a, const SortRun& run, int* cnt, int (&id)[4]) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  sort_ids(a, run.p0 + lane, run.p1, id);          // on their way while the counts are cleared
  for (int i = threadIdx.x; i < W * a.E; i += blockDim.x) cnt[i] = 0;
  __syncthreads();
  for (int r = 0; run.p0 + r * 256 < run.p1; ++r) {
    if (r) sort_ids(a, run.p0 + r * 256 + lane, run.p1, id);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (id[i] < a.E) atomicAdd(&cnt[wave * a.E + id[i]], 1);
  }
  __syncthreads();
}

template <int W>
__global__ __launch_bounds__(1024) void sort_count_kernel(const SortArgs a) {
  extern __shared__ int cnt[];
  const SortRun run(a, W);
  int id[4];
  sort_count<W>(a, run, cnt, id);
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
    int n = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) n += cnt[w * a.E + e];
    a.hist[(int64_t)blockIdx.x * a.E + e] = n;
  }
}

template <int W>
__global__ __launch_bounds__(1024) void sort_place_kernel(const SortArgs a) {
  extern __shared__ int cnt[];
  __shared__ int wave_total[16];
  const SortRun run(a, W);
  int id[4];
  sort_count<W>(a, run, cnt, id);
  const int t = threadIdx.x, wave = t >> 6, lane = t & 63, waves = blockDim.x >> 6;
  int carry = 0;
  for (int e0 = 0; e0 < a.E; e0 += blockDim.x) {
    const int e = e0 + t;
    int before = 0, total = 0, n[W] = {};
    if (e < a.E) {
#pragma unroll
      for (int w = 0; w < W; ++w) n[w] = cnt[w * a.E + e];
      if (a.chunks == 1) {
#pragma unroll
        for (int w = 0; w < W; ++w) total += n[w];
      } else {
#pragma unroll 8
        for (int c = 0; c < a.chunks; ++c) {
          const int m = a.hist[(int64_t)c * a.E + e];
          total += m;
          if (c < (int)blockIdx.x) before += m;
        }
      }
    }
    const int upto = wave_sum_to(total);
    if (lane == 63) wave_total[wave] = upto;
    __syncthreads();
    const int of = lane < waves ? wave_total[lane] : 0, to = wave_sum_to(of);   // the waves' totals, on every wave's lanes
    const int base = carry + __builtin_amdgcn_readlane(to - of, __builtin_amdgcn_readfirstlane(wave)) + upto - total;
    carry += __builtin_amdgcn_readlane(to, 63);
    if (e < a.E) {
      if (blockIdx.x == 0) a.offsets[e] = base;    // where expert e begins
      int at = base + before;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        cnt[w * a.E + e] = at;
        at += n[w];
      }
    }
    __syncthreads();
  }
  if (blockIdx.x == 0 && t == 0) a.offsets[a.E] = carry;
  volatile int* next = cnt + wave * a.E;           // (a wave's LDS operations are done in order)
  const int bits = 32 - __builtin_clz(a.E);
  for (int r = 0; run.p0 + r * 256 < run.p1; ++r) {
    if (a.rounds > 1) sort_ids(a, run.p0 + r * 256 + lane, run.p1, id);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = run.p0 + r * 256 + 64 * i + lane;
      if (p - lane >= run.p1) break;
      const bool has = id[i] < a.E;
      uint64_t same = __ballot(has);
      for (int b = 0; b < bits; ++b) {
        const uint64_t m = __ballot(has && (id[i] >> b & 1));
        same &= id[i] >> b & 1 ? m : ~m;
      }
      const int rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(same >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)same, 0));
      if (has) {
        const int at = next[id[i]];
        if (rank == 0) next[id[i]] = at + __popcll(same);
        a.tokens[at + rank] = (int)((unsigned)p / (unsigned)a.k);
        a.slots[p] = at + rank;
      } else if (p < run.p1) {
        a.slots[p] = -1;
      }
    }
  }
  for (int64_t s = carry + (int64_t)blockIdx.x * blockDim.x + t; s < a.P; s += (int64_t)gridDim.x * blockDim.x) a.tokens[s] = -1;
}

// Chunks of W waves: few where few pairs leave few counts to clear and to add; 16 where one launch is enough (4800 pairs in one
// launch of two rounds take 9.6 to 11.3 us, in two launches 7.7 to 8.8) or the chunks' counts take longer to add than the waves'
// (320000 pairs of 256 experts 15.2 us, 16.0 with 8 waves and 21.2 with 4); 8 between (32768 of 512: 9.3; 10.9 with 16, 9.5 with 4),
// and where 16 would not fit the LDS.
struct SortPlan {
  int W, rounds, chunks;
  SortPlan(int64_t P, int E) : W(P <= 256 ? 1 : P <= 1024 ? 4 : E <= 2048 && (P <= kSortOne || P > 1 << 18) ? 16 : 8), rounds(1), chunks(1) {
    if (P > kSortOne || P > 256 * W) {
      rounds = (int)((P + (int64_t)kSortChunks * 256 * W - 1) / ((int64_t)kSortChunks * 256 * W));
      chunks = (int)((P + (int64_t)256 * W * rounds - 1) / ((int64_t)256 * W * rounds));
    }
  }
};
template <int W>
static int launch_sort(const SortArgs& a, hipStream_t st) {
  const int lds = W * a.E * (int)sizeof(int);
  const dim3 grid(a.chunks), threads(std::max(64 * W, std::min(1024, (a.E + 63) / 64 * 64)));
  if (lds + 16 * (int)sizeof(int) > 64 * 1024)     // sort_place's wave_total is beside it
    for (const void* f : {reinterpret_cast<const void*>(sort_count_kernel<W>), reinterpret_cast<const void*>(sort_place_kernel<W>)})
      if (hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) return check_launch("expert_sort");
  if (a.chunks > 1) hipLaunchKernelGGL((sort_count_kernel<W>), grid, threads, lds, st, a);
  hipLaunchKernelGGL((sort_place_kernel<W>), grid, threads, lds, st, a);
  return check_launch("expert_sort");
}

// ------------------------------------------------------------------ rows
// Bytes are copied as they are, 16 at a time, the last 16 of a row again where
// its length is no multiple.  A wave takes a part of a row, 4 KB at most, by C
// loads that are on their way together.
//
// Experts share tokens: each row of x is read k times, by rows of the output that
// lie far apart.  So where that is twice or more, and the output is larger than the
// L2, an XCD (workgroups go to the eight in turn) takes the rows whose tokens are in
// its eighth of x, which its L2 keeps, and the output passes by: for each kRowGroup
// rows, each XCD has a wave that copies its own of them.  32768 rows of 4096 tokens,
// 2560 in bf16, take 29.5 to 30 us over three inputs in turn (189 MB at 6.3 TB/s; 27
// on one input; 48 without this, 62 with stores that stay in L2, 36 with groups of 8,
// 42 with 2), 131072 of 1024 52 (78), 16384 of 8192 tokens and 5120 values 52 (57).
constexpr int kRowPart = 4096, kRowGroup = 4;
typedef uint32_t u32x4_b __attribute__((ext_vector_type(4), aligned(1)));

struct RowsArgs {
  const uint8_t* x;  int64_t x_stride;             // bytes
  const int* tokens;
  uint8_t* out;  int64_t out_stride;
  int T, P, parts, part;                           // parts of a row, bytes of one (a multiple of 128, the last may be shorter)
  int64_t bytes;
};
template <int C, bool STREAM>
__device__ __forceinline__ void copy_row(const RowsArgs& a, int lane, int64_t s, int tok, int part) {
  const int64_t b0 = (int64_t)part * a.part;
  const int n = (int)min(a.bytes - b0, (int64_t)a.part);
  const bool has = tok >= 0 && tok < a.T;
  const uint8_t* from = a.x + (int64_t)(has ? tok : 0) * a.x_stride + b0;
  uint8_t* to = a.out + s * a.out_stride + b0;
  if (n < 16) {
    if (lane < n) to[lane] = has ? from[lane] : 0;
    return;
  }
  const int b = lane * 16;
  u32x4_b v[C];
  if (has) {
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] = *reinterpret_cast<const u32x4_b*>(from + min(b + i * 1024, n - 16));
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] = u32x4_b{0, 0, 0, 0};
  }
#pragma unroll
  for (int i = 0; i < C; ++i) {
    u32x4_b* p = reinterpret_cast<u32x4_b*>(to + min(b + i * 1024, n - 16));
    if (b + i * 1024 < n) {
      if constexpr (STREAM) __builtin_nontemporal_store(v[i], p);
      else *p = v[i];
    }
  }
}
template <int C>
__global__ __launch_bounds__(256) void expert_rows_kernel(const RowsArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t waves = (int64_t)gridDim.x * 4, items = (int64_t)a.P * a.parts;
  for (int64_t it = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); it < items; it += waves) {
    const int64_t s = it / a.parts;
    copy_row<C, false>(a, lane, s, a.tokens[s], (int)(it - s * a.parts));
  }
}
template <int C>
__global__ __launch_bounds__(256) void expert_rows_large_kernel(const RowsArgs a) {
  const int lane = threadIdx.x & 63, xcd = blockIdx.x & 7;
  const int lo = (int)((int64_t)a.T * xcd >> 3), hi = (int)((int64_t)a.T * (xcd + 1) >> 3);
  const int64_t waves = (int64_t)(gridDim.x >> 3) * 4;   // (the grid is a multiple of 8)
  const int64_t items = ((int64_t)a.P + kRowGroup - 1) / kRowGroup * a.parts;
  for (int64_t it = (int64_t)(blockIdx.x >> 3) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); it < items; it += waves) {
    const int64_t g = it / a.parts, s = g * kRowGroup + lane;
    const bool in = lane < kRowGroup && s < a.P;
    const int tok = in ? a.tokens[s] : -1;
    const bool none = tok < 0 || tok >= a.T;       // zeros: dealt by their place
    uint64_t mine = __ballot(in && (none ? ((int)s & 7) == xcd : tok >= lo && tok < hi));
    while (mine) {
      const int l = __builtin_ctzll(mine);
      mine &= mine - 1;
      copy_row<C, true>(a, lane, g * kRowGroup + l, __builtin_amdgcn_readlane(tok, l), (int)(it - g * a.parts));
    }
  }
}
template <int C>
static void launch_rows(const RowsArgs& a, bool large, hipStream_t st) {
  if (large) {
    const int64_t waves = ((int64_t)a.P + kRowGroup - 1) / kRowGroup * a.parts;   // on each XCD
    hipLaunchKernelGGL((expert_rows_large_kernel<C>), dim3((unsigned)std::min<int64_t>((waves + 3) / 4, 1 << 17) * 8), dim3(256), 0, st, a);
  } else {
    hipLaunchKernelGGL((expert_rows_kernel<C>), dim3((unsigned)std::min<int64_t>(((int64_t)a.P * a.parts + 3) / 4, 1 << 20)), dim3(256), 0, st, a);
  }
}

// ------------------------------------------------------------------ combine
typedef uint32_t u32x4_e __attribute__((ext_vector_type(4), aligned(2)));

template <int DT> struct Vec8;                     // eight values of a type, as loaded
template <> struct Vec8<DT_F32> {
  u32x4_e a, b;
  __device__ void load(const void* p, int64_t i) {
    const u32x4_e* g = reinterpret_cast<const u32x4_e*>(static_cast<const float*>(p) + i);
    a = g[0];
    b = g[1];
  }
  __device__ float get(int j) const { return __uint_as_float(j < 4 ? a[j] : b[j - 4]); }
};
template <int DT> struct Vec8 {
  u32x4_e v;
  __device__ void load(const void* p, int64_t i) { v = *reinterpret_cast<const u32x4_e*>(static_cast<const uint16_t*>(p) + i); }
  __device__ float get(int j) const {
    const uint32_t d = v[j >> 1];
    if constexpr (DT == DT_BF16) return j & 1 ? bf16_hi(d) : bf16_lo(d);
    else return f16_to_f32((uint16_t)(j & 1 ? d >> 16 : d));
  }
};
// Eight values; STREAM: they pass by the L2.
template <bool STREAM>
__device__ __forceinline__ void put4(u32x4_e* p, u32x4_e v) {
  if constexpr (STREAM) __builtin_nontemporal_store(v, p);
  else *p = v;
}
template <int DT, bool STREAM>
__device__ __forceinline__ void put8(void* p, int64_t i, const float (&f)[8]) {
  if constexpr (DT == DT_F32) {
    u32x4_e* g = reinterpret_cast<u32x4_e*>(static_cast<float*>(p) + i);
    put4<STREAM>(g, u32x4_e{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])});
    put4<STREAM>(g + 1, u32x4_e{__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7])});
  } else {
    uint32_t d[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      d[j] = DT == DT_BF16 ? pack_bf16x2(f[2 * j], f[2 * j + 1]) : pack_f16x2(f[2 * j], f[2 * j + 1]);
    put4<STREAM>(reinterpret_cast<u32x4_e*>(static_cast<uint16_t*>(p) + i), u32x4_e{d[0], d[1], d[2], d[3]});
  }
}
template <int DT>
__device__ __forceinline__ float get1(const void* p, int64_t i) {
  if constexpr (DT == DT_F32) return static_cast<const float*>(p)[i];
  else if constexpr (DT == DT_BF16) return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
  else return f16_to_f32(static_cast<const uint16_t*>(p)[i]);
}
__device__ __forceinline__ float weight_at(const void* w, int dt, int64_t i) {
  return dt == DT_F32 ? get1<DT_F32>(w, i) : dt == DT_BF16 ? get1<DT_BF16>(w, i) : get1<DT_F16>(w, i);
}

struct CombineArgs {
  const void* y;  int64_t y_stride;
  const int* slots;
  const void* w;  int w_dtype;                     // [T, k] or null
  void* out;  int64_t out_stride;
  int T, k, P, H, parts;                           // parts: waves per token
};

// A wave takes 512 values of a token, eight per lane, and its k rows B at a time, whose loads are on their way together (B 8
// for two rows left registers for 5 waves per SIMD: 20000 tokens of 2 rows of 700 took 34 us).  The last lanes of a row are
// moved back to end at H.  Sums are fp32 by fma, rounded once.  Bound by the reads: 4096 tokens of 8 rows of 2560 in bf16,
// 189 MB, take 40 us (4.8 TB/s); 3 tokens 3.0 (latency).
template <int DT, int B, bool STREAM>
__global__ __launch_bounds__(256) void expert_combine_kernel(const CombineArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t waves = (int64_t)gridDim.x * 4, items = (int64_t)a.T * a.parts;
  for (int64_t it = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); it < items; it += waves) {
    const int64_t t = it / a.parts;
    const int h0 = ((int)(it - t * a.parts) * 64 + lane) * 8;
    const int* slots = a.slots + t * a.k;
    if (a.H < 8) {
      if (lane < a.H) {
        float acc = 0.0f;
        for (int j = 0; j < a.k; ++j) {
          const int s = slots[j];
          if (s >= 0 && s < a.P)
            acc = __builtin_fmaf(a.w ? weight_at(a.w, a.w_dtype, t * a.k + j) : 1.0f, get1<DT>(a.y, s * a.y_stride + lane), acc);
        }
        store_out(a.out, t * a.out_stride + lane, DT, acc);
      }
      continue;
    }
    const int h = min(h0, a.H - 8);
    float acc[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    for (int j0 = 0; j0 < a.k; j0 += B) {
      Vec8<DT> v[B];
      float w[B];
      bool has[B];
#pragma unroll
      for (int j = 0; j < B; ++j) {
        const int at = min(j0 + j, a.k - 1), s = slots[at];
        has[j] = j0 + j < a.k && s >= 0 && s < a.P;
        if (has[j]) v[j].load(a.y, s * a.y_stride + h);
        w[j] = a.w ? weight_at(a.w, a.w_dtype, t * a.k + at) : 1.0f;
      }
#pragma unroll
      for (int j = 0; j < B; ++j)
        if (has[j])
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[i] = __builtin_fmaf(w[j], v[j].get(i), acc[i]);
    }
    if (h0 < a.H) put8<DT, STREAM>(a.out, t * a.out_stride + h, acc);
  }
}

// Where y does not stay in the 32 MB of the XCDs' L2, neither do the results: they would push out what other waves are about
// to read (4096 tokens of 8 rows of 2560 in bf16: the sum 43.0 us so, 39.7 with stores that pass by; the gradient 78 and
// 76, when its workgroups that clear rows took 3 us more).
static bool ex_streams(int64_t P, int64_t H, int dt) { return P * H * (dt == DT_F32 ? 4 : 2) > 32 << 20; }

template <int DT, bool STREAM>
static void launch_combine_as(const CombineArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)std::min<int64_t>(((int64_t)a.T * a.parts + 3) / 4, 1 << 20));
  if (a.k <= 2) hipLaunchKernelGGL((expert_combine_kernel<DT, 2, STREAM>), grid, dim3(256), 0, st, a);
  else if (a.k <= 4) hipLaunchKernelGGL((expert_combine_kernel<DT, 4, STREAM>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((expert_combine_kernel<DT, 8, STREAM>), grid, dim3(256), 0, st, a);
}
template <int DT>
static void launch_combine(const CombineArgs& a, hipStream_t st) {
  if (ex_streams(a.P, a.H, DT)) launch_combine_as<DT, true>(a, st);
  else launch_combine_as<DT, false>(a, st);
}

// ------------------------------------------------------------------ its gradient
constexpr int kGradTop = 128, kGradTail = 64;      // pairs per token; rows that a workgroup of the second role looks at, one per lane

struct GradArgs {
  const void* d;  int64_t d_stride;                // dout
  const void* y;  int64_t y_stride;
  const int *slots, *tokens;
  const void* w;  int w_dtype;
  void* dy;  int64_t dy_stride;
  void* dw;
  int T, k, P, H;
};

// A sum over the wave, in a fixed order: within 16 lanes, then of the four 16s, in lane 63's place.
__device__ __forceinline__ float wave_total(float v) {
  const auto other = [](float x, auto ctrl, auto rows) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
  };
  using std::integral_constant;
  v += other(v, integral_constant<int, 0x111>(), integral_constant<int, 0xf>());
  v += other(v, integral_constant<int, 0x112>(), integral_constant<int, 0xf>());
  v += other(v, integral_constant<int, 0x114>(), integral_constant<int, 0xf>());
  v += other(v, integral_constant<int, 0x118>(), integral_constant<int, 0xf>());
  v += other(v, integral_constant<int, 0x142>(), integral_constant<int, 0xa>());
  v += other(v, integral_constant<int, 0x143>(), integral_constant<int, 0xc>());
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// A workgroup takes a token: its row of dout stays in registers, C chunks of
// eight values per lane, while its k rows of y go by, so that y is read and dy
// written once for both gradients.  A wave's sum of the products has a fixed
// order, and the waves' are added in theirs.  Workgroups past the tokens clear the
// rows that no pair has: those whose token is none, or has no slot that is the row.
// A lane looks through the slots of one row's token, so 64 rows are known after a
// few loads on their way together (4096 tokens of 8 rows of 2560 take 74 us, by the
// tokens alone and one row after the other 77; 100 rows of 512 191 and 181, for the
// slots' bytes, and 200 with those dealt over a wave's lanes).  Bound by memory:
// 4096 tokens of 8 rows of 2560 in bf16, 357 MB, take 57 us after the sum of the
// same y and 74 over three sets of rows in turn (6.3 and 4.8 TB/s; a large copy 5.1).
// Where pairs are dropped, rows are cleared in more time than their bytes take, one
// after the other and an element per lane: half of the pairs 74 us, seven eighths 57
// (their bytes 54 and 41).
template <int DT, int C, bool STREAM>
__global__ __launch_bounds__(1024) void expert_grad_kernel(const GradArgs a) {
  __shared__ float sum[16][kGradTop];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), W = blockDim.x >> 6;
  if ((int)blockIdx.x >= a.T) {
    __shared__ uint64_t none_of;
    static_assert(kGradTail == 64, "a lane per row");
    const int64_t s0 = (int64_t)(blockIdx.x - a.T) * kGradTail;
    if (wave == 0) {
      const int64_t s = s0 + lane;
      const int tok = s < a.P ? a.tokens[s] : -1;
      bool none = s < a.P;
      if (tok >= 0 && tok < a.T)                   // a pair may have been taken out after the sort: its slot is -1
#pragma unroll 8
        for (int j = 0; j < a.k; ++j) none &= a.slots[(int64_t)tok * a.k + j] != (int)s;
      const uint64_t rows = __ballot(none);
      if (lane == 0) none_of = rows;
    }
    __syncthreads();
    for (uint64_t rows = none_of; rows; rows &= rows - 1) {
      const int64_t s = s0 + __builtin_ctzll(rows);
      for (int h = t; h < a.H; h += blockDim.x) store_out(a.dy, s * a.dy_stride + h, DT, 0.0f);
    }
    return;
  }
  const int64_t tok = blockIdx.x;
  const int* slots = a.slots + tok * a.k;
  if (a.H < 8) {                                   // (one wave)
    const float d = lane < a.H ? get1<DT>(a.d, tok * a.d_stride + lane) : 0.0f;
    for (int j = 0; j < a.k; ++j) {
      const int s = slots[j];
      const bool has = s >= 0 && s < a.P;
      float v = 0.0f;
      if (has && lane < a.H) {
        v = d * get1<DT>(a.y, s * a.y_stride + lane);
        store_out(a.dy, s * a.dy_stride + lane, DT, weight_at(a.w, a.w_dtype, tok * a.k + j) * d);
      }
      v = group_allreduce(v, 64);
      if (lane == 0) store_out(a.dw, tok * a.k + j, a.w_dtype, v);
    }
    return;
  }
  int h[C];
  bool in[C];
  Vec8<DT> d[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int h0 = (c * (int)blockDim.x + t) * 8;
    in[c] = h0 < a.H;
    h[c] = min(h0, a.H - 8);
    d[c].load(a.d, tok * a.d_stride + h[c]);
  }
  constexpr int B = C == 1 ? 4 : C == 2 ? 2 : 1;   // rows whose loads are on their way together
  for (int j0 = 0; j0 < a.k; j0 += B) {
    Vec8<DT> v[B][C];
    int s[B];
    float dot[B], w[B];
#pragma unroll
    for (int j = 0; j < B; ++j) {
      const int at = min(j0 + j, a.k - 1);
      s[j] = slots[at];
      if (j0 + j >= a.k || s[j] >= a.P) s[j] = -1;
      w[j] = weight_at(a.w, a.w_dtype, tok * a.k + at);
      if (s[j] >= 0)
#pragma unroll
        for (int c = 0; c < C; ++c) v[j][c].load(a.y, s[j] * a.y_stride + h[c]);
    }
#pragma unroll
    for (int j = 0; j < B; ++j) {
      dot[j] = 0.0f;
      if (s[j] >= 0)
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const int dup = (c * (int)blockDim.x + t) * 8 - h[c];   // values that the chunk before has, of one moved back
          float g[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            g[i] = w[j] * d[c].get(i);
            if (in[c] && i >= dup) dot[j] = __builtin_fmaf(d[c].get(i), v[j][c].get(i), dot[j]);
          }
          if (in[c]) put8<DT, STREAM>(a.dy, s[j] * a.dy_stride + h[c], g);
        }
    }
#pragma unroll
    for (int j = 0; j < B; ++j) {
      const float total = wave_total(dot[j]);
      if (lane == 0 && j0 + j < a.k) sum[wave][j0 + j] = total;
    }
  }
  __syncthreads();
  for (int j = t; j < a.k; j += blockDim.x) {
    float v = sum[0][j];
    for (int q = 1; q < W; ++q) v += sum[q][j];
    store_out(a.dw, tok * a.k + j, a.w_dtype, v);
  }
}

template <int DT, bool STREAM>
static int launch_grad_as(const GradArgs& a, hipStream_t st) {
  const int chunks = (a.H + 7) / 8, C = chunks <= 1024 ? 1 : chunks <= 2048 ? 2 : 4;
  const int threads = std::min(1024, ((chunks + C - 1) / C + 63) / 64 * 64);
  const int64_t groups = a.T + (a.P + (int64_t)kGradTail - 1) / kGradTail;
  if (groups * threads > (int64_t)UINT32_MAX) return ex_fail("expert_combine_grad", "tokens times the lanes of a row pass 2^32");
  const dim3 grid((unsigned)groups);
  if (C == 1) hipLaunchKernelGGL((expert_grad_kernel<DT, 1, STREAM>), grid, dim3(threads), 0, st, a);
  else if (C == 2) hipLaunchKernelGGL((expert_grad_kernel<DT, 2, STREAM>), grid, dim3(threads), 0, st, a);
  else hipLaunchKernelGGL((expert_grad_kernel<DT, 4, STREAM>), grid, dim3(threads), 0, st, a);
  return check_launch("expert_combine_grad");
}
template <int DT>
static int launch_grad(const GradArgs& a, hipStream_t st) {
  return ex_streams(a.P, a.H, DT) ? launch_grad_as<DT, true>(a, st) : launch_grad_as<DT, false>(a, st);
}

static bool ex_dt(int dt) { return dt == DT_BF16 || dt == DT_F32 || dt == DT_F16; }
static bool ex_al(const void* p, int dt) { return (reinterpret_cast<uintptr_t>(p) & (dt == DT_F32 ? 3 : 1)) == 0; }
static bool al4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

}  // namespace fp4x

using namespace fp4x;

extern "C" {

int64_t fp4x_expert_sort_workspace(int64_t T, int k, int E) {
  if (T < 1 || k < 1 || E < 1) return 0;
  const SortPlan plan(T * k, E);
  return plan.chunks == 1 ? 0 : (int64_t)plan.chunks * E * (int64_t)sizeof(int);
}

int fp4x_expert_sort(const void* ids, int wide, int64_t row, int64_t T, int k, int E, int* offsets, int* tokens,
                     int* slots, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "expert_sort";
  if (T < 0 || k < 1 || k > 1 << 20 || E < 1 || E > kF8MaxExperts) return ex_fail(what, "need T >= 0, 1 <= k <= 2^20 and 1 to 4096 experts");
  if (T > (1 << 30) / k) return ex_fail(what, "more than 2^30 pairs");
  if (!offsets || !al4(offsets)) return ex_fail(what, "null or misaligned offsets");
  if (T && (!ids || !tokens || !slots)) return ex_fail(what, "null ids, tokens or slots");
  if ((reinterpret_cast<uintptr_t>(ids) & (wide ? 7 : 3)) || !al4(tokens) || !al4(slots))
    return ex_fail(what, "tensors must be aligned to their element");
  if (row < 0) return ex_fail(what, "a stride is negative");
  const int64_t need = fp4x_expert_sort_workspace(T, k, E);
  if (need && (!workspace || workspace_bytes < need || !al4(workspace))) return ex_fail(what, "the workspace is too small, null or misaligned");
  const int P = (int)(T * k);
  const SortPlan plan(P, E);
  const SortArgs a{ids, wide ? 1 : 0, row, P, k, E, plan.rounds, plan.chunks, static_cast<int*>(workspace), offsets, tokens, slots};
  hipStream_t st = (hipStream_t)stream;
  if (plan.W == 1) return launch_sort<1>(a, st);
  if (plan.W == 4) return launch_sort<4>(a, st);
  if (plan.W == 8) return launch_sort<8>(a, st);
  return launch_sort<16>(a, st);
}

int fp4x_expert_rows(const void* x, int64_t x_stride, int elem, int T, const int* tokens, int P, int H, void* out,
                     int64_t out_stride, void* stream) {
  const char* what = "expert_rows";
  if (T < 0 || P < 0 || H < 1 || (elem != 1 && elem != 2 && elem != 4)) return ex_fail(what, "need T and P >= 0, H >= 1 and elements of 1, 2 or 4 bytes");
  if (P == 0) return FP4X_OK;
  if ((!x && T) || !tokens || !out || !al4(tokens)) return ex_fail(what, "null tensor, or misaligned tokens");
  if (x_stride < 0 || (P > 1 && out_stride < H)) return ex_fail(what, "output rows overlap, or a stride is negative");
  const int64_t bytes = (int64_t)H * elem;
  const int64_t parts = (bytes + kRowPart - 1) / kRowPart;
  const int part = (int)(((bytes + parts - 1) / parts + 127) & -128);
  const RowsArgs a{static_cast<const uint8_t*>(x), x_stride * elem, tokens, static_cast<uint8_t*>(out), out_stride * elem,
                   T, P, (int)parts, part, bytes};
  hipStream_t st = (hipStream_t)stream;
  const bool large = P / 2 >= T && T >= 8 && P * bytes > 32 << 20;
  if (part <= 1024) launch_rows<1>(a, large, st);
  else if (part <= 2048) launch_rows<2>(a, large, st);
  else if (part <= 3 * 1024) launch_rows<3>(a, large, st);
  else launch_rows<4>(a, large, st);
  return check_launch(what);
}

int fp4x_expert_combine(const void* y, int64_t y_stride, int dtype, int P, const int* slots, const void* w, int w_dtype,
                        void* out, int64_t out_stride, int T, int k, int H, void* stream) {
  const char* what = "expert_combine";
  if (!ex_dt(dtype) || (w && !ex_dt(w_dtype))) return ex_fail(what, "rows and weights are bf16, fp16 or fp32");
  // a step of the loops over k and over a row's parts stays within an int
  constexpr int kMost = INT_MAX - 511;
  if (T < 0 || k < 1 || P < 0 || H < 1 || k > kMost || H > kMost) return ex_fail(what, "need T and P >= 0, k and H from 1 to 2^31 - 512");
  if (T == 0) return FP4X_OK;
  if ((!y && P) || !slots || !out || !al4(slots) || !ex_al(y, dtype) || !ex_al(out, dtype) || (w && !ex_al(w, w_dtype)))
    return ex_fail(what, "null tensor, or one that is not aligned to its element");
  if (y_stride < 0 || (T > 1 && out_stride < H)) return ex_fail(what, "output rows overlap, or a stride is negative");
  const int parts = (H + 511) / 512;
  const CombineArgs a{y, y_stride, slots, w, w_dtype, out, out_stride, T, k, P, H, parts};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DT_BF16) launch_combine<DT_BF16>(a, st);
  else if (dtype == DT_F16) launch_combine<DT_F16>(a, st);
  else launch_combine<DT_F32>(a, st);
  return check_launch(what);
}

int fp4x_expert_combine_grad(const void* dout, int64_t dout_stride, const void* y, int64_t y_stride, int dtype, int P,
                             const int* slots, const int* tokens, const void* w, int w_dtype, void* dy,
                             int64_t dy_stride, void* dw, int T, int k, int H, void* stream) {
  const char* what = "expert_combine_grad";
  if (!ex_dt(dtype) || !ex_dt(w_dtype)) return ex_fail(what, "rows and weights are bf16, fp16 or fp32");
  if (T < 0 || k < 1 || k > kGradTop || P < 0 || H < 1 || H > 32768)
    return ex_fail(what, "need T and P >= 0, 1 <= k <= 128 and 1 <= H <= 32768");
  if (T == 0 && P == 0) return FP4X_OK;
  if ((T && (!dout || !slots || !w || !dw)) || (P && (!y || !tokens || !dy))) return ex_fail(what, "null tensor");
  if (!al4(slots) || !al4(tokens) || !ex_al(dout, dtype) || !ex_al(y, dtype) || !ex_al(dy, dtype) || !ex_al(w, w_dtype) ||
      !ex_al(dw, w_dtype))
    return ex_fail(what, "tensors must be aligned to their element");
  if (dout_stride < 0 || y_stride < 0 || (P > 1 && dy_stride < H)) return ex_fail(what, "output rows overlap, or a stride is negative");
  const GradArgs a{dout, dout_stride, y, y_stride, slots, tokens, w, w_dtype, dy, dy_stride, dw, T, k, P, H};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DT_BF16) return launch_grad<DT_BF16>(a, st);
  if (dtype == DT_F16) return launch_grad<DT_F16>(a, st);
  return launch_grad<DT_F32>(a, st);
}

}  // extern "C"
