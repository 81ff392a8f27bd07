// Expert products with 4-bit weights: out[t] = sum over t's entries (expert e, score s) of
// s * W2_e (silu(W1_e^gate x_t) * (W1_e^up x_t)), x and out bf16, the weights 4-bit codes with a scale
// per group of input columns.
//
// The format and the layout are described in int4.cuh.  This file: preparing and expanding the weights,
// and the layer for few tokens (int4_wide.cu has it for many).
#include <type_traits>

#include "int4.cuh"

namespace smb {

namespace {

// ---------------------------------------------------------------------------------------------
// preparation

__device__ __forceinline__ int int4_source_row(int p, int N, int concat) {
  return concat ? (p & 1 ? N / 2 + (p >> 1) : p >> 1) : p;
}

// Smallest 5-significant-bit number >= amax / 7, at least 2^-126; 0 for amax = 0, NaN for one that is
// not finite (such a group's products become NaN instead of hiding it).
__device__ __forceinline__ float int4_scale_of(float amax) {
  if (amax == 0.0f) return 0.0f;
  if (!(amax < __int_as_float(0x7f800000))) return __int_as_float(0x7fffffff);
  float s = __uint_as_float(__float_as_uint(__fdiv_rn(amax, 7.0f)) & 0xFFF80000u);
  if (__fmul_rn(7.0f, s) < amax) s = __uint_as_float(__float_as_uint(s) + 0x80000u);  // 7 s is exact
  return fmaxf(s, 1.1754944e-38f);
}

// One warp per (16-row tile, 128-column block).
constexpr int kPrepWarps = 8;

__global__ void __launch_bounds__(32 * kPrepWarps)
    weight_prep_int4_kernel(const __nv_bfloat16* __restrict__ w, int E, int N, int K, int group, int concat,
                            int n_tiles, int k_blocks, uint8_t* __restrict__ wq, __nv_bfloat16* __restrict__ ws) {
  __shared__ __align__(16) uint32_t s_word[kPrepWarps][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long item = static_cast<long long>(blockIdx.x) * kPrepWarps + warp;
  if (item >= static_cast<long long>(E) * n_tiles * k_blocks) return;
  const int kb = static_cast<int>(item % k_blocks);
  const long long et = item / k_blocks;  // expert * n_tiles + tile
  const int tile = static_cast<int>(et % n_tiles), e = static_cast<int>(et / n_tiles);
  const int c = lane & 15;               // 8 columns 8 c .. of the block
  const int k0 = kb * 128 + 8 * c;
  const int gpb = 128 / group, lanes_per_group = group / 8;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 2 * i + (lane >> 4);
    const int p = tile * 16 + r;
    float v[8];
    if (p < N && k0 < K) {  // K % 8 == 0: a piece of 8 columns lies inside or outside as a whole
      const size_t row = static_cast<size_t>(e) * N + int4_source_row(p, N, concat);
      const uint4 raw = *reinterpret_cast<const uint4*>(w + row * K + k0);
      const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(u[j] << 16);
        v[2 * j + 1] = __uint_as_float(u[j] & 0xFFFF0000u);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.0f;
    }
    float amax = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = isfinite(v[j]) ? fmaxf(amax, fabsf(v[j])) : __int_as_float(0x7f800000);
    for (int o = 1; o < lanes_per_group; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const float s = int4_scale_of(amax);
    uint32_t word = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int q = s > 0.0f ? static_cast<int>(rintf(__fdiv_rn(v[j], s))) : 0;
      word |= static_cast<uint32_t>(q + 8) << (4 * (j >> 1) + 16 * (j & 1));
    }
    word = __funnelshift_l(word, word, 3);
    const int h = c >> 3, blk = (c >> 2) & 1, t = c & 3;
    s_word[warp][h * 128 + (4 * (r & 7) + t) * 4 + 2 * blk + (r >> 3)] = word;
    if (c % lanes_per_group == 0)
      ws[(et * k_blocks + kb) * gpb * 16 + ((r & 7) * gpb + c / lanes_per_group) * 2 + (r >> 3)] =
          __float2bfloat16_rn(s);
  }
  __syncwarp();
  uint4* dst = reinterpret_cast<uint4*>(wq + (et * k_blocks + kb) * 1024);
  const uint4* src = reinterpret_cast<const uint4*>(s_word[warp]);
  dst[lane] = src[lane];
  dst[32 + lane] = src[32 + lane];
}

// The bf16 weights that the 4-bit form stands for (exact), [E, N, K] in the caller's row order.
__global__ void __launch_bounds__(32 * kPrepWarps)
    int4_expand_kernel(const uint8_t* __restrict__ wq, const __nv_bfloat16* __restrict__ ws, int E, int N, int K,
                       int group, int concat, int n_tiles, int k_blocks, __nv_bfloat16* __restrict__ w) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long item = static_cast<long long>(blockIdx.x) * kPrepWarps + warp;
  if (item >= static_cast<long long>(E) * n_tiles * k_blocks) return;
  const int kb = static_cast<int>(item % k_blocks);
  const long long et = item / k_blocks;
  const int tile = static_cast<int>(et % n_tiles), e = static_cast<int>(et / n_tiles);
  const int c = lane & 15;
  const int k0 = kb * 128 + 8 * c;
  const int gpb = 128 / group, lanes_per_group = group / 8;
  const uint32_t* words = reinterpret_cast<const uint32_t*>(wq + (et * k_blocks + kb) * 1024);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 2 * i + (lane >> 4);
    const int p = tile * 16 + r;
    if (p >= N || k0 >= K) continue;
    const int h = c >> 3, blk = (c >> 2) & 1, t = c & 3;
    const uint32_t stored = words[h * 128 + (4 * (r & 7) + t) * 4 + 2 * blk + (r >> 3)];
    const uint32_t word = __funnelshift_r(stored, stored, 3);
    const float s = __bfloat162float(
        ws[(et * k_blocks + kb) * gpb * 16 + ((r & 7) * gpb + c / lanes_per_group) * 2 + (r >> 3)]);
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      o[j] = pack_bf16x2_rn(s * static_cast<float>(static_cast<int>((word >> (4 * j)) & 15u) - 8),
                            s * static_cast<float>(static_cast<int>((word >> (4 * j + 16)) & 15u) - 8));
    const size_t row = static_cast<size_t>(e) * N + int4_source_row(p, N, concat);
    *reinterpret_cast<uint4*>(w + row * K + k0) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// ---------------------------------------------------------------------------------------------
// products

__device__ __forceinline__ void mma_bf16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr int kMvWarps = 8;
constexpr int kMvThreads = 32 * kMvWarps;

// ---------------------------------------------------------------------------------------------
// Few tokens.  Two launches: the up projection and the down projection with the sum over a token's
// experts.  Both read each weight of an active expert once:
//   - every warp streams row tiles of its own (MT x 16 rows) through a ring of kDepth column blocks in
//     shared memory, filled by 16-byte asynchronous copies ahead of the products, across the end of one
//     tile and the start of the next; a lane reads back only what it copied itself, so the ring needs no
//     barrier;
//   - there is no routing pass: every CTA makes the list of active experts and their entries itself from
//     the (few) expert ids;
//   - the down kernel starts while the up kernel drains (programmatic dependent launch) and has its first
//     weights on the way before it waits for the intermediate.
// The m16n8k16 tensor core product takes 8 tokens as its 8 columns; with one token 7/8 of its work is
// thrown away, but it still keeps up with the memory, which the plain FMA units would not beyond 2 tokens.
// What it spends its time on: turning 2048 codes into bf16 takes a warp 56 integer instructions, which an SM
// issues at half rate (28 cycles of it), 32 packed bf16 ones and some 25 for the ring, against 44 cycles that
// their bytes take at the HBM rate.  Neither unit is full: at 8 tokens of 4096 x 1024 (64 experts) the up kernel
// issues in 60% of the cycles with its integer pipe at 57% and DRAM at 35%, the down kernel in 44% (40%, 25%);
// the rest is latency.  8 tokens of 4096 x 1024 with 128 experts take 103 us, one token 26 us.  Scaling the
// groups' sums instead of the weights is up to 5% faster (groups of 64: 102 us against 106) but wrong for large
// x, see use_stage.  Registers instead of the shared-memory ring, and a block of x without the read-ahead,
// measured slower.

constexpr int kSmMaxEntries = 256;  // their down results are kept in shared memory (128 bytes an entry)

// Active experts (slots, ascending) of the entries and their flat entries, slot s owning
// list[beg[s]] .. list[beg[s + 1]).  The order inside a slot does not matter: an entry's values do not
// depend on the column it has in a product.  Shared memory: cnt [E], act / beg / list as sized below.
struct SmallPlan {
  uint16_t act[kSmMaxEntries];
  uint16_t beg[kSmMaxEntries + 2];
  uint16_t list[kSmMaxEntries];
  int32_t scan[2][kMvWarps];
};

__device__ __forceinline__ int small_plan(const int32_t* __restrict__ experts, int n, int E, int32_t* cnt, SmallPlan& p,
                                          int32_t* freq_out, int* err) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (freq_out)
    for (int e = tid; e < E; e += kMvThreads) freq_out[e] = 0;
  if (n <= 32) {  // one warp finds equal experts by matching; slots in the order of first appearance
    __syncthreads();  // freq_out is zero
    if (warp == 0) {
      int e = lane < n ? experts[lane] : -1;
      const bool ok = e >= 0 && e < E;
      if (lane < n && !ok && freq_out && err) atomicCAS(err, 0, kErrBadExpert);
      const uint32_t same = __match_any_sync(0xffffffffu, ok ? e : -1);
      const uint32_t below = (1u << lane) - 1u;
      const bool first = ok && (same & below) == 0;
      const uint32_t firsts = __ballot_sync(0xffffffffu, first);
      const int c = first ? __popc(same) : 0;
      int inc = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      const int beg = __shfl_sync(0xffffffffu, inc - c, ok ? __ffs(same) - 1 : 0);
      if (first) {
        const int s = __popc(firsts & below);
        p.act[s] = static_cast<uint16_t>(e);
        p.beg[s] = static_cast<uint16_t>(beg);
        if (freq_out) freq_out[e] = c;
      }
      if (ok) p.list[beg + __popc(same & below)] = static_cast<uint16_t>(lane);
      if (lane == 31) {
        p.beg[__popc(firsts)] = static_cast<uint16_t>(inc);
        p.scan[0][0] = __popc(firsts);
      }
    }
    __syncthreads();
    return p.scan[0][0];
  }
  for (int e = tid; e < E; e += kMvThreads) cnt[e] = 0;
  __syncthreads();
  for (int f = tid; f < n; f += kMvThreads) {
    const int e = experts[f];
    if (e >= 0 && e < E)
      atomicAdd(&cnt[e], 1);
    else if (freq_out && err)
      atomicCAS(err, 0, kErrBadExpert);
  }
  __syncthreads();
  const int per = (E + kMvThreads - 1) / kMvThreads;
  const int e0 = min(E, tid * per), e1 = min(E, e0 + per);
  int a = 0, c = 0;
  for (int e = e0; e < e1; ++e) {
    const int v = cnt[e];
    a += v > 0;
    c += v;
    if (freq_out) freq_out[e] = v;
  }
  int ia = a, ic = c;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int ya = __shfl_up_sync(0xffffffffu, ia, o), yc = __shfl_up_sync(0xffffffffu, ic, o);
    if (lane >= o) {
      ia += ya;
      ic += yc;
    }
  }
  if (lane == 31) {
    p.scan[0][warp] = ia;
    p.scan[1][warp] = ic;
  }
  __syncthreads();
  ia -= a;
  ic -= c;
  int slots = 0;
#pragma unroll
  for (int w = 0; w < kMvWarps; ++w) {
    const int sa = p.scan[0][w], sc = p.scan[1][w];
    if (w < warp) {
      ia += sa;
      ic += sc;
    }
    slots += sa;
  }
  for (int e = e0; e < e1; ++e) {
    const int v = cnt[e];
    if (v == 0) continue;
    p.act[ia] = static_cast<uint16_t>(e);
    p.beg[ia] = static_cast<uint16_t>(ic);
    cnt[e] = ic;  // becomes the next free place of e's list
    ++ia;
    ic += v;
  }
  if (tid == kMvThreads - 1) p.beg[slots] = static_cast<uint16_t>(ic);
  __syncthreads();
  for (int f = tid; f < n; f += kMvThreads) {
    const int e = experts[f];
    if (e >= 0 && e < E) p.list[atomicAdd(&cnt[e], 1)] = static_cast<uint16_t>(f);
  }
  __syncthreads();
  return slots;
}

struct SmallArgs {
  const uint8_t* wq;
  const __nv_bfloat16* ws;
  int N, K, n_tiles, k_blocks;  // prepared rows N, input columns K
  const int32_t* experts;
  const int32_t* tokens;  // explicit lists, else null: token f / topk
  int n_entries, topk, T, E;
  const __nv_bfloat16* x;  // up: tokens [T, K]; down: the intermediate [entries, K]
  const float* scores;
  __nv_bfloat16* a;    // up output [entries, N / 2]
  __nv_bfloat16* out;  // down output [T, N]
  int32_t* freq;
  int ksplit;  // parts of the columns of a tile, one warp each
  int* err;
};

// The intermediate is written by the grid this one overlaps with: not through the read-only path.
__device__ __forceinline__ uint4 ld_plain(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// A warp's ring: kDepth stages of one column block of MT row tiles, lane l's 16-byte piece h of tile m at
// (2 m + h) * 512 + 16 l, then its scales (GPB words) at MT * 1024 + m * 128 GPB + 4 GPB l.
constexpr int kDepth = 4;
template <int MT, int GPB>
constexpr int kStage = MT * (1024 + 128 * GPB);

// src: the lane's piece of the block in the first tile's codes, sc: its scales.  Tiles beyond the `tiles`
// that are left repeat the first; their results are dropped.
template <int MT, int GPB>
__device__ __forceinline__ void fill_stage(uint32_t stage, const uint8_t* src, const __nv_bfloat16* sc, int tiles,
                                           int k_blocks) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const size_t at = m < tiles ? static_cast<size_t>(m) * k_blocks : 0;
    const uint8_t* q = src + at * 1024;
    const __nv_bfloat16* s = sc + at * (GPB * 16);
    cp_async16(stage + 1024 * m + 16 * lane, q);
    cp_async16(stage + 1024 * m + 512 + 16 * lane, q + 512);
    const uint32_t sd = stage + 1024 * MT + 128 * GPB * m + 4 * GPB * lane;
    if constexpr (GPB == 4)
      cp_async16(sd, s);
    else
      cp_async_small<4 * GPB>(sd, s);
  }
}

// Values 8 t .. 8 t + 7 of the four 32-column pieces of block b of a token's row, zero beyond K.
template <bool kUp>
__device__ __forceinline__ void load_x(uint4 (&x)[4], const __nv_bfloat16* xrow, int b, int K) {
  const int k = b * 128 + 8 * (threadIdx.x & 3);
  const bool whole = (b + 1) * 128 <= K;
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    x[s] = make_uint4(0, 0, 0, 0);
    if (whole || k + 32 * s < K)
      x[s] = kUp ? __ldg(reinterpret_cast<const uint4*>(xrow + k + 32 * s)) : ld_plain(xrow + k + 32 * s);
  }
}

// One stage's products.  The weights enter them with their scale, as exact bf16 numbers: taking the codes' offset
// from a sum of (16 + n) x afterwards would leave an error of 24 |x| in it, whatever the code, and overflow where
// the sum itself does not.
template <int MT, int GPB>
__device__ __forceinline__ void use_stage(const Int4Magic& magic, uint32_t stage, const uint4 (&x)[4],
                                          float (&acc)[MT][4]) {
  const int lane = threadIdx.x & 31;
  uint4 q[MT];
  uint32_t s2[MT][GPB];
  __nv_bfloat162 sl[MT], sh[MT], ml[MT], mh[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const uint32_t a = stage + 1024 * MT + 128 * GPB * m + 4 * GPB * lane;
    if constexpr (GPB == 4) {
      const uint4 v = lds128(a);
      s2[m][0] = v.x;
      s2[m][1] = v.y;
      s2[m][2] = v.z;
      s2[m][3] = v.w;
    } else {
#pragma unroll
      for (int i = 0; i < GPB; ++i) s2[m][i] = lds32(a + 4 * i);
    }
  }
#pragma unroll
  for (int s = 0; s < 4; ++s) {  // 32 columns each
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (s % (4 / GPB) == 0) {  // a group's first columns
        const uint32_t w = s2[m][s / (4 / GPB)];
        sl[m] = int4_scale2(w, 0);
        sh[m] = int4_scale2(w, 1);
        ml[m] = int4_m24(sl[m]);
        mh[m] = int4_m24(sh[m]);
      }
      if (s % 2 == 0) q[m] = lds128(stage + 1024 * m + 256 * s + 16 * lane);
      const uint32_t wl = s & 1 ? q[m].z : q[m].x, wh = s & 1 ? q[m].w : q[m].y;
      uint32_t lo[4], hi[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        lo[i] = int4_scaled(magic, wl, i, sl[m], ml[m]);
        hi[i] = int4_scaled(magic, wh, i, sh[m], mh[m]);
      }
      mma_bf16_16816(acc[m], lo[0], hi[0], lo[1], hi[1], x[s].x, x[s].y);
      mma_bf16_16816(acc[m], lo[2], hi[2], lo[3], hi[3], x[s].z, x[s].w);
    }
  }
}

// A warp's stream: items first, first + step, ... < count; decode(item) gives (slot, tile, columns part).
// Tokens of an item come in chunks of 8 columns, each a pass over the item's blocks.  Calls
// done(tile, part, beg, n, acc) after each pass; before_x() once after the first copies have been issued.
template <int MT, int GPB, bool kUp, typename Decode, typename Done, typename BeforeX>
__device__ __forceinline__ void stream_items(const SmallArgs& p, const SmallPlan& pl, uint32_t ring, int first,
                                             int step, int count, Decode decode, BeforeX before_x, Done done) {
  const int g = (threadIdx.x & 31) >> 2;
  const Int4Magic magic;
  // the copies' position: item, blocks left of this pass, passes' tokens left, addresses
  int l_item = first, l_left = 0, l_tokens = 0, l_tiles = 0;
  const uint8_t* l_src = nullptr;
  const __nv_bfloat16* l_sc = nullptr;
  uint32_t l_stage = 0, u_stage = 0;
  const int lane = threadIdx.x & 31;
  auto bounds = [&](int part, int& b0, int& b1) {
    b0 = part * p.k_blocks / p.ksplit;
    b1 = (part + 1) * p.k_blocks / p.ksplit;
  };
  auto open = [&](bool next_pass) {
    if (l_item >= count) return;
    int slot, tile, part, b0, b1;
    decode(l_item, slot, tile, part);
    bounds(part, b0, b1);
    if (!next_pass) l_tokens = pl.beg[slot + 1] - pl.beg[slot];
    const size_t blk = (static_cast<size_t>(pl.act[slot]) * p.n_tiles + tile) * p.k_blocks + b0;
    l_src = p.wq + blk * 1024 + 16 * lane;
    l_sc = p.ws + blk * (GPB * 16) + (lane >> 2) * (GPB * 2);
    l_tiles = p.n_tiles - tile;
    l_left = b1 - b0;
  };
  auto fill = [&] {
    if (l_item < count) {
      fill_stage<MT, GPB>(ring + l_stage * kStage<MT, GPB>, l_src, l_sc, l_tiles, p.k_blocks);
      if (++l_stage == kDepth) l_stage = 0;
      l_src += 1024;
      l_sc += GPB * 16;
      if (--l_left == 0) {
        l_tokens -= 8;
        const bool again = l_tokens > 0;
        if (!again) l_item += step;
        open(again);
      }
    }
    cp_async_commit();
  };
  open(false);
#pragma unroll
  for (int d = 0; d < kDepth - 1; ++d) fill();
  before_x();
  for (int item = first; item < count; item += step) {
    int slot, tile, part, b0, b1;
    decode(item, slot, tile, part);
    bounds(part, b0, b1);
    const int end = pl.beg[slot + 1];
    for (int beg = pl.beg[slot]; beg < end; beg += 8) {
      const int n = min(end - beg, 8);
      // columns without a token repeat another's row (any row serves); their results are dropped
      const int f = pl.list[beg + min(g, n - 1)];
      const __nv_bfloat16* xrow;
      if (kUp) {
        int tok = p.tokens ? p.tokens[f] : f / p.topk;
        if (tok < 0 || tok >= p.T) {
          if (p.err) atomicCAS(p.err, 0, kErrBadToken);
          tok = 0;  // the entry belongs to no token of the output: its results are not summed anywhere
        }
        xrow = p.x + static_cast<size_t>(tok) * p.K;
      } else {
        xrow = p.x + static_cast<size_t>(f) * p.K;
      }
      float acc[MT][4];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][i] = 0.0f;
      uint4 next[4];
      load_x<kUp>(next, xrow, b0, p.K);
      for (int b = b0; b < b1; ++b) {
        uint4 x[4];  // the next block's x is under way during this one's products
#pragma unroll
        for (int s = 0; s < 4; ++s) x[s] = next[s];
        if (b + 1 < b1) load_x<kUp>(next, xrow, b + 1, p.K);
        fill();  // the stage freed by the block before
        cp_async_wait<kDepth - 1>();
        use_stage<MT, GPB>(magic, ring + u_stage * kStage<MT, GPB>, x, acc);
        if (++u_stage == kDepth) u_stage = 0;
      }
      done(tile, part, beg, n, acc);
    }
  }
}

// Up projection and SwiGLU: a persistent grid, item = (slot, MT row tiles).  With ksplit > 1 (few items)
// adjacent warps of a CTA share a tile's columns and their sums meet in shared memory.
template <int MT, int GPB>
__global__ void __launch_bounds__(kMvThreads, 2) small_up_kernel(const SmallArgs p) {
  extern __shared__ __align__(16) uint8_t s_dyn[];  // rings, counts [E]
  __shared__ SmallPlan pl;
  __shared__ float s_part[kMvWarps][8][16 * MT + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(s_dyn) + warp * kDepth * kStage<MT, GPB>;
  int32_t* s_cnt = reinterpret_cast<int32_t*>(s_dyn + kMvWarps * kDepth * kStage<MT, GPB>);
  pdl_launch();
  const int slots = small_plan(p.experts, p.n_entries, p.E, s_cnt, pl, blockIdx.x == 0 ? p.freq : nullptr, p.err);
  const int tiles = (p.n_tiles + MT - 1) / MT, half = p.N / 2;
  auto decode = [&](int item, int& slot, int& tile, int& part) {
    part = item % p.ksplit;
    const int i = item / p.ksplit;
    slot = i / tiles;
    tile = (i - slot * tiles) * MT;
  };
  const int count = slots * tiles * p.ksplit, step = gridDim.x * kMvWarps;
  auto store = [&](int f, int col, float v) {
    if (col < half) p.a[static_cast<size_t>(f) * half + col] = __float2bfloat16_rn(v);
  };
  if (p.ksplit == 1) {
    stream_items<MT, GPB, true>(
        p, pl, ring, blockIdx.x * kMvWarps + warp, step, count, decode, [] {},
        [&](int tile, int, int beg, int n, float (&acc)[MT][4]) {
          // rows 2 r are gates, rows 2 r + 1 ups: lanes of even g finish row g's pair, their partners
          // (lane ^ 4) row (g - 1) + 8's
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            const bool odd = g & 1;
            const float r0 = __shfl_xor_sync(0xffffffffu, odd ? acc[m][0] : acc[m][2], 4);
            const float r1 = __shfl_xor_sync(0xffffffffu, odd ? acc[m][1] : acc[m][3], 4);
            const float v0 = odd ? silu_mul(r0, acc[m][2]) : silu_mul(acc[m][0], r0);
            const float v1 = odd ? silu_mul(r1, acc[m][3]) : silu_mul(acc[m][1], r1);
            const int col = (tile + m) * 8 + (odd ? 4 : 0) + (g >> 1), i = 2 * t;
            if (i < n) store(pl.list[beg + i], col, v0);
            if (i + 1 < n) store(pl.list[beg + i + 1], col, v1);
          }
        });
    return;
  }
  // every warp of the CTA takes the same number of rounds, one item (and one chunk of tokens) each
  for (int r = blockIdx.x * kMvWarps; r < count; r += step) {
    stream_items<MT, GPB, true>(
        p, pl, ring, r + warp, count, min(count, r + kMvWarps), decode, [] {},
        [&](int, int, int, int, float (&acc)[MT][4]) {
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) s_part[warp][2 * t + (i & 1)][16 * m + g + 8 * (i >> 1)] = acc[m][i];
        });
    __syncthreads();
    int slot, tile, part;
    if (r + warp < count) {
      decode(r + warp, slot, tile, part);
      const int beg = pl.beg[slot], n = pl.beg[slot + 1] - beg;
      for (int o = part * 32 + lane; o < n * 8 * MT; o += p.ksplit * 32) {
        const int i = o / (8 * MT), row = o % (8 * MT);
        float gate = 0.0f, up = 0.0f;
        for (int k = 0; k < p.ksplit; ++k) {
          gate += s_part[warp - part + k][i][2 * row];
          up += s_part[warp - part + k][i][2 * row + 1];
        }
        store(pl.list[beg + i], tile * 8 + row, silu_mul(gate, up));
      }
    }
    __syncthreads();
  }
}

// Down projection and the sum over each token's entries: a cluster owns MT row tiles for all active
// experts, whose (slot, columns part) items its warps take in turn.  Every entry's result is written
// once, into the first CTA's shared memory, and a token's entries are then added in entry order.
template <int MT, int GPB>
__global__ void __launch_bounds__(kMvThreads, 2) small_down_kernel(const SmallArgs p) {
  // rings, counts [E], the results [ksplit][entries][16 MT] of the cluster
  extern __shared__ __align__(16) uint8_t s_dyn[];
  __shared__ SmallPlan pl;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(s_dyn) + warp * kDepth * kStage<MT, GPB>;
  int32_t* s_cnt = reinterpret_cast<int32_t*>(s_dyn + kMvWarps * kDepth * kStage<MT, GPB>);
  float* s_y = reinterpret_cast<float*>(s_cnt + p.E);
  uint32_t rank, csize;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(csize));
  const int slots = small_plan(p.experts, p.n_entries, p.E, s_cnt, pl, nullptr, p.err);
  const int tile0 = static_cast<int>(blockIdx.x / csize) * MT;
  uint32_t y0;  // the first CTA's results, as seen from this one
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(y0) : "r"(smem_u32(s_y)));
  // the first CTA has started (its shared memory may be written)
  asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  stream_items<MT, GPB, false>(
      p, pl, ring, static_cast<int>(rank) * kMvWarps + warp, static_cast<int>(csize) * kMvWarps, slots * p.ksplit,
      [&](int item, int& slot, int& tile, int& part) {
        slot = item / p.ksplit;
        part = item - slot * p.ksplit;
        tile = tile0;
      },
      [] { pdl_wait(); },
      [&](int, int part, int beg, int n, float (&acc)[MT][4]) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int c = 2 * t + (i & 1);
            if (c < n) {
              const uint32_t at = (part * p.n_entries + pl.list[beg + c]) * (16 * MT) + 16 * m + g + 8 * (i >> 1);
              asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(y0 + 4 * at), "f"(acc[m][i]) : "memory");
            }
          }
      });
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (rank != 0) return;
  for (int o = threadIdx.x; o < p.T * 16 * MT; o += kMvThreads) {
    const int tok = o / (16 * MT), row = o % (16 * MT);
    const int col = tile0 * 16 + row;
    if (col >= p.N) continue;
    int f0 = tok * p.topk, f1 = f0 + p.topk;
    if (p.tokens) {  // sorted list: first entry of tok and of tok + 1
      int lo = 0, hi = p.n_entries;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (p.tokens[mid] < tok)
          lo = mid + 1;
        else
          hi = mid;
      }
      f0 = lo;
      f1 = f0;
      while (f1 < p.n_entries && p.tokens[f1] == tok) ++f1;
    }
    float v = 0.0f;
    for (int f = f0; f < f1; ++f) {
      const int e = p.experts[f];
      if (e < 0 || e >= p.E) continue;
      float y = 0.0f;
      for (int k = 0; k < p.ksplit; ++k) y += s_y[(k * p.n_entries + f) * (16 * MT) + row];
      v = fmaf(p.scores[f], y, v);
    }
    p.out[static_cast<size_t>(tok) * p.N + col] = __float2bfloat16_rn(v);
  }
}

}  // namespace

int int4_row_tiles(int N) { return ceil_div(N, 16); }
int int4_col_blocks(int K) { return ceil_div(K, 128); }

cudaError_t launch_weight_prep_int4(const void* w, int E, int N, int K, int group, int concat, uint8_t* wq, void* ws,
                                    cudaStream_t st) {
  const int nt = int4_row_tiles(N), kb = int4_col_blocks(K);
  const long long items = static_cast<long long>(E) * nt * kb;
  weight_prep_int4_kernel<<<static_cast<unsigned>((items + kPrepWarps - 1) / kPrepWarps), 32 * kPrepWarps, 0, st>>>(
      static_cast<const __nv_bfloat16*>(w), E, N, K, group, concat, nt, kb, wq, static_cast<__nv_bfloat16*>(ws));
  return cudaGetLastError();
}

cudaError_t launch_int4_expand(const uint8_t* wq, const void* ws, int E, int N, int K, int group, int concat, void* w,
                               cudaStream_t st) {
  const int nt = int4_row_tiles(N), kb = int4_col_blocks(K);
  const long long items = static_cast<long long>(E) * nt * kb;
  int4_expand_kernel<<<static_cast<unsigned>((items + kPrepWarps - 1) / kPrepWarps), 32 * kPrepWarps, 0, st>>>(
      wq, static_cast<const __nv_bfloat16*>(ws), E, N, K, group, concat, nt, kb, static_cast<__nv_bfloat16*>(w));
  return cudaGetLastError();
}

namespace {

// A kernel's limit of dynamic shared memory is one value for all threads of the process: it is set to the most
// that any call of the instantiation takes, never to one call's own need, which a call beside it could lower
// before the launch.
constexpr int kSmMaxExperts = 4096;
constexpr int kSmResultBytes = 64 * 1024;  // results of a down cluster
template <int MT, int GPB>
constexpr int kSmUpBytes = kMvWarps * kDepth * kStage<MT, GPB> + kSmMaxExperts * 4;
template <int MT, int GPB>
constexpr int kSmDownBytes = kSmUpBytes<MT, GPB> + kSmResultBytes;

template <int MT, int GPB>
cudaError_t launch_small_up(SmallArgs p, cudaStream_t st) {
  const int tiles = ceil_div(p.n_tiles, MT);
  const int slots = p.E < p.n_entries ? p.E : p.n_entries;
  auto kern = small_up_kernel<MT, GPB>;
  const int smem = kMvWarps * kDepth * kStage<MT, GPB> + p.E * 4;
  if (smem > kSmUpBytes<MT, GPB>) return cudaErrorInvalidValue;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmUpBytes<MT, GPB>);
  if (e != cudaSuccess) return e;
  int occ = 0;
  e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, kern, kMvThreads, smem);
  if (e != cudaSuccess) return e;
  const long long most = static_cast<long long>(gemm_grid_sms()) * (occ > 0 ? occ : 1);
  // few items: split their columns while that leaves one item a warp (an expert must fit one chunk)
  p.ksplit = 1;
  while (p.n_entries <= 8 && p.ksplit < kMvWarps && 2 * p.ksplit <= p.k_blocks &&
         static_cast<long long>(slots) * tiles * 2 * p.ksplit <= most * kMvWarps)
    p.ksplit *= 2;
  const long long ctas = ceil_div(static_cast<long long>(slots) * tiles * p.ksplit, kMvWarps);
  kern<<<static_cast<unsigned>(ctas < most ? ctas : most), kMvThreads, smem, st>>>(p);
  return cudaGetLastError();
}

template <int MT, int GPB>
cudaError_t launch_small_down(SmallArgs p, cudaStream_t st) {
  const int tiles = ceil_div(p.n_tiles, MT);
  const int slots = p.E < p.n_entries ? p.E : p.n_entries;
  int cluster = 1;  // CTAs that share a row tile's experts, so that narrow outputs still fill the SMs
  while (cluster < 8 && tiles * cluster < 200 && slots > 8 * cluster) cluster *= 2;
  p.ksplit = 1;
  while (slots * p.ksplit < kMvWarps * cluster && 2 * p.ksplit <= p.k_blocks && p.ksplit < kMvWarps &&
         2 * p.ksplit * p.n_entries * 64 * MT <= kSmResultBytes)
    p.ksplit *= 2;
  const int smem = kMvWarps * kDepth * kStage<MT, GPB> + p.E * 4 + p.ksplit * p.n_entries * 16 * MT * 4;
  static_assert(kSmMaxEntries * 64 * MT <= kSmResultBytes && kSmDownBytes<MT, GPB> <= 232448 - 4096,
                "shared memory budget");
  if (smem > kSmDownBytes<MT, GPB>) return cudaErrorInvalidValue;
  auto kern = small_down_kernel<MT, GPB>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmDownBytes<MT, GPB>);
  if (e != cudaSuccess) return e;
  return launch_dependent(kern, dim3(tiles * cluster), kMvThreads, smem, cluster, st, p);
}

template <int MT>
cudaError_t launch_small(const SmallArgs& u, int group1, const SmallArgs& d, int group2, cudaStream_t st) {
  cudaError_t e = group1 == 32   ? launch_small_up<MT, 4>(u, st)
                  : group1 == 64 ? launch_small_up<MT, 2>(u, st)
                                 : launch_small_up<MT, 1>(u, st);
  if (e != cudaSuccess) return e;
  return group2 == 32   ? launch_small_down<MT, 4>(d, st)
         : group2 == 64 ? launch_small_down<MT, 2>(d, st)
                        : launch_small_down<MT, 1>(d, st);
}

}  // namespace

// Row tiles of a warp's item (4096 x 1024, 128 experts, groups of 128, us with 1 / 2 / 4): one token 23 / 26 / 28,
// 2 tokens 39 / 36 / 55, 4 tokens 70 / 61 / 70, 8 tokens 109 / 105 / 128.
constexpr int kMT = 2;

// Up to 8 tokens an expert's tokens fit the 8 columns of a product and nothing is read twice; beyond, that
// depends on the routing (before its weights were scaled ahead of the products, 4096 x 1024, 128 experts, us, this /
// the other: 16 tokens even 142 / 162, Zipf 115 / 109; 24 tokens 180 / 193 and 180 / 135).  With groups of 64 or
// 128 this path is then the faster one or within 8% of it (us, this / the other, groups of 128: 1, 4 and 8 tokens
// of 4096 x 1024 26 / 38, 61 / 75, 103 / 105; of 2048 x 768 16 / 27, 32 / 43, 48 / 56; of 7168 x 2048 with 64
// experts 56 / 67, 189 / 189, 272 / 269; groups of 64: 64 / 73 and 107 / 103 at 4 and 8 tokens of 4096 x 1024,
// 200 / 185 and 295 / 281 of 7168 x 2048).  Groups of 32 cost its warps more scales: the other path wins from about
// 2 10^8 weights a matrix on (4096 x 1024 at 4, 6 and 8 tokens, 1.3, 2.0 and 2.7 10^8: 72 / 76, 98 / 97, 119 / 106;
// 7168 x 2048 at 1, 2 and 4, 1.2, 2.3 and 4.7 10^8: 66 / 67, 118 / 114, 222 / 202).
bool int4_small(const Int4Args& p) {
  if (p.T > 8 || p.n_entries > kSmMaxEntries) return false;
  const size_t weights = static_cast<size_t>(p.n_entries < p.E ? p.n_entries : p.E) * p.H * p.I;
  return (p.group1 > 32 && p.group2 > 32) || weights <= (size_t{3} << 26);
}

cudaError_t launch_int4_small(const Int4Args& p, cudaStream_t st) {
  SmallArgs u{};
  u.wq = p.w1q;
  u.ws = static_cast<const __nv_bfloat16*>(p.w1s);
  u.N = 2 * p.I;
  u.K = p.H;
  u.n_tiles = int4_row_tiles(u.N);
  u.k_blocks = int4_col_blocks(u.K);
  u.experts = p.experts;
  u.tokens = p.tokens;
  u.n_entries = p.n_entries;
  u.topk = p.K;
  u.T = p.T;
  u.E = p.E;
  u.x = static_cast<const __nv_bfloat16*>(p.x);
  u.a = static_cast<__nv_bfloat16*>(p.a);
  u.freq = p.freq;
  u.err = p.err;
  SmallArgs d = u;
  d.wq = p.w2q;
  d.ws = static_cast<const __nv_bfloat16*>(p.w2s);
  d.N = p.H;
  d.K = p.I;
  d.n_tiles = int4_row_tiles(d.N);
  d.k_blocks = int4_col_blocks(d.K);
  d.x = u.a;
  d.scores = p.scores;
  d.out = static_cast<__nv_bfloat16*>(p.out);
  return launch_small<kMT>(u, p.group1, d, p.group2, st);
}

}  // namespace smb
