// Expert products with 4-bit weights: out[t] = sum over t's entries (expert e, score s) of
// s * W2_e (silu(W1_e^gate x_t) * (W1_e^up x_t)), x and out bf16, the weights 4-bit codes with a scale
// per group of input columns.
//
// Format.  w[n, k] = q[n, k] * s[n, k / group], q in [-7, 7], group 32, 64 or 128.  The scale is the
// smallest number of 5 significant bits (at least 2^-126) that is >= amax / 7 of its group, so
// q (3 bits) times s (5 bits) has at most 8 significant bits: every weight is exactly a bf16 number.
// Taking 5 bits instead of bf16's 8 widens the step by 3% at most; in exchange the codes can be scaled
// before or after the products, on any path, without a rounding of their own.
//
// Layout (int4_tile_bytes / int4_scales of them per expert).  Rows come in tiles of 16, columns in
// blocks of 128 (both padded with zero weights).  A block of a tile is 2 x 512 bytes; in the half h,
// lane l = 4 g + t of a warp owns 16 bytes = 4 words: row g and row g + 8 of the columns
// 64 h + 8 t .. + 7, then of the columns 64 h + 32 + 8 t .. + 7.  Nibble i of a word holds the code + 8
// of column 2 i, nibble i + 4 that of column 2 i + 1, so (word >> 4 i) & 0x000F000F is a pair of
// neighbours in the halves of a register.  A column block's order inside the product does not matter
// as long as x is read the same way: lane l reads 8 consecutive values of x (16 bytes) for each word
// pair, and two m16n8k16 products consume them.  Scales are [tile][group][16] bf16, row g at 2 g, row
// g + 8 at 2 g + 1.  A GLU weight's prepared row 2 j is gate row j and 2 j + 1 up row j (the
// interleaved order; a concatenated w1 is re-ordered when it is prepared).
#include "common.cuh"
#include "sonic_internal.h"

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
    const int h = c >> 3, blk = (c >> 2) & 1, t = c & 3;
    s_word[warp][h * 128 + (4 * (r & 7) + t) * 4 + 2 * blk + (r >> 3)] = word;
    if (c % lanes_per_group == 0)
      ws[((et * k_blocks + kb) * gpb + c / lanes_per_group) * 16 + 2 * (r & 7) + (r >> 3)] = __float2bfloat16_rn(s);
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
    const uint32_t word = words[h * 128 + (4 * (r & 7) + t) * 4 + 2 * blk + (r >> 3)];
    const float s = __bfloat162float(
        ws[((et * k_blocks + kb) * gpb + c / lanes_per_group) * 16 + 2 * (r & 7) + (r >> 3)]);
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

// Codes of word `w`, pair i (columns 2 i, 2 i + 1), as two bf16: 0x4300 is 128, whose last mantissa bit
// is worth 1, so 0x4300 | n is 128 + n, and subtracting 136 leaves q = n - 8 exactly.
__device__ __forceinline__ uint32_t int4_pair(uint32_t w, int i) {
  const uint32_t u = ((w >> (4 * i)) & 0x000F000Fu) | 0x43004300u;
  const uint32_t off = 0x43084308u;
  __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), *reinterpret_cast<const __nv_bfloat162*>(&off));
  return *reinterpret_cast<uint32_t*>(&r);
}

__device__ __forceinline__ void mma_bf16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr int kMvWarps = 8;
constexpr int kMvThreads = 32 * kMvWarps;

// acc[j][.] += rows of one tile times the tokens of n-tile j, over the column blocks [b0, b1).
// wq: the tile's first block; sc: its scales; xrow[j]: this lane's token of n-tile j (null: none).
template <int NT>
__device__ __forceinline__ void mv_tile(const uint8_t* __restrict__ wq, const __nv_bfloat16* __restrict__ sc, int group,
                                        int K, int b0, int b1, const __nv_bfloat16* const (&xrow)[NT],
                                        float (&acc)[NT][4]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  for (int b = b0; b < b1; ++b) {
    uint4 q[2];
    q[0] = __ldg(reinterpret_cast<const uint4*>(wq + static_cast<size_t>(b) * 1024) + lane);
    q[1] = __ldg(reinterpret_cast<const uint4*>(wq + static_cast<size_t>(b) * 1024) + 32 + lane);
    const int gpb = 128 / group;
    float part[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) part[j][i] = 0.0f;
#pragma unroll
    for (int s = 0; s < 4; ++s) {  // 32 columns each
      const uint4 qh = q[s >> 1];
      const uint32_t lo = s & 1 ? qh.z : qh.x, hi = s & 1 ? qh.w : qh.y;
      const int k = b * 128 + 32 * s + 8 * t;
      uint32_t a[4], c[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = int4_pair(lo, i);
        c[i] = int4_pair(hi, i);
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        uint4 xv = make_uint4(0, 0, 0, 0);
        if (xrow[j] && k < K) xv = __ldg(reinterpret_cast<const uint4*>(xrow[j] + k));
        mma_bf16_16816(part[j], a[0], c[0], a[1], c[1], xv.x, xv.y);
        mma_bf16_16816(part[j], a[2], c[2], a[3], c[3], xv.z, xv.w);
      }
      if (((s + 1) * 32) % group == 0) {  // end of a group: its sums times the rows' scales
        const uint32_t s2 = __ldg(reinterpret_cast<const uint32_t*>(
                                      sc + (static_cast<size_t>(b) * gpb + (s * 32) / group) * 16) + g);
        const float slo = __uint_as_float(s2 << 16), shi = __uint_as_float(s2 & 0xFFFF0000u);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          acc[j][0] = fmaf(slo, part[j][0], acc[j][0]);
          acc[j][1] = fmaf(slo, part[j][1], acc[j][1]);
          acc[j][2] = fmaf(shi, part[j][2], acc[j][2]);
          acc[j][3] = fmaf(shi, part[j][3], acc[j][3]);
#pragma unroll
          for (int i = 0; i < 4; ++i) part[j][i] = 0.0f;
        }
      }
    }
  }
}

struct MvArgs {
  const uint8_t* wq;
  const __nv_bfloat16* ws;
  int group, N, K, n_tiles, k_blocks;  // prepared rows N, input columns K
  const int32_t* freq;
  const int32_t* off;
  const int32_t* s_scatter;   // flat entry of a sorted position
  const int32_t* x_gather;    // token of a sorted position
  const __nv_bfloat16* x;     // up: tokens [T, K]; down: the intermediate [entries, K] in sorted order
  int T;
  const float* scores;        // down: by flat entry
  __nv_bfloat16* a;           // up output [entries, N / 2], sorted order
  float* y;                   // down output [entries, N] fp32, by flat entry, times the score
  int* err;
};

// Tokens [c0, c0 + 8 NT) of expert e with one 16-row tile: the 8 warps split the columns, the sums meet
// in shared memory.
template <bool kUp, int NT>
__device__ __forceinline__ void mv_chunk(const MvArgs& p, int e, int tile, int c0, int n, float* s_red) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int base = p.off[e] + c0;
  const __nv_bfloat16* xrow[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int i = 8 * j + g;
    xrow[j] = nullptr;
    if (i < n) {
      if (kUp) {
        const int tok = p.x_gather[base + i];
        if (tok >= 0 && tok < p.T)
          xrow[j] = p.x + static_cast<size_t>(tok) * p.K;
        else
          atomicCAS(p.err, 0, kErrBadToken);
      } else {
        xrow[j] = p.x + static_cast<size_t>(base + i) * p.K;
      }
    }
  }
  float acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[j][i] = 0.0f;
  const size_t et = static_cast<size_t>(e) * p.n_tiles + tile;
  mv_tile<NT>(p.wq + et * p.k_blocks * 1024, p.ws + et * p.k_blocks * (128 / p.group) * 16, p.group, p.K,
              warp * p.k_blocks / kMvWarps, (warp + 1) * p.k_blocks / kMvWarps, xrow, acc);
  constexpr int kLd = 8 * NT + 1;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    float* d = s_red + warp * 16 * kLd + 8 * j + 2 * t;
    d[g * kLd] = acc[j][0];
    d[g * kLd + 1] = acc[j][1];
    d[(g + 8) * kLd] = acc[j][2];
    d[(g + 8) * kLd + 1] = acc[j][3];
  }
  __syncthreads();
  auto total = [&](int row, int i) {
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < kMvWarps; ++w) v += s_red[w * 16 * kLd + row * kLd + i];
    return v;
  };
  if (kUp) {
    for (int o = threadIdx.x; o < 8 * n; o += kMvThreads) {
      const int i = o >> 3, r = o & 7;
      const int col = tile * 8 + r;
      if (col >= p.N / 2) continue;
      const float gate = total(2 * r, i), up = total(2 * r + 1, i);
      p.a[static_cast<size_t>(base + i) * (p.N / 2) + col] = __float2bfloat16_rn(gate / (1.0f + __expf(-gate)) * up);
    }
  } else {
    for (int o = threadIdx.x; o < 16 * n; o += kMvThreads) {
      const int i = o >> 4, r = o & 15;
      const int col = tile * 16 + r;
      if (col >= p.N) continue;
      const int f = p.s_scatter[base + i];
      p.y[static_cast<size_t>(f) * p.N + col] = p.scores[f] * total(r, i);
    }
  }
}

template <bool kUp>
__global__ void __launch_bounds__(kMvThreads) mv_kernel(const MvArgs p) {
  __shared__ float s_red[kMvWarps * 16 * 33];
  const int e = blockIdx.y, tile = blockIdx.x;
  const int n_e = p.freq[e];
  for (int c0 = 0; c0 < n_e; c0 += 32) {
    const int n = min(32, n_e - c0);
    if (n <= 8)
      mv_chunk<kUp, 1>(p, e, tile, c0, n, s_red);
    else if (n <= 16)
      mv_chunk<kUp, 2>(p, e, tile, c0, n, s_red);
    else
      mv_chunk<kUp, 4>(p, e, tile, c0, n, s_red);
  }
}

// out[t] = sum of the rows y[f] of t's entries, f in [t K, (t + 1) K) or [tok_off[t], tok_off[t + 1]),
// in entry order, rounded once.  Entries whose expert or token was rejected have no row.
__global__ void __launch_bounds__(256)
    int4_combine_kernel(const float* __restrict__ y, int T, int H, int K, const int32_t* __restrict__ tok_off,
                        const int32_t* __restrict__ experts, int E, __nv_bfloat16* __restrict__ out) {
  const int t = blockIdx.y;
  const int c = (blockIdx.x * blockDim.x + threadIdx.x) * 4;
  if (c >= H) return;
  const int f0 = tok_off ? tok_off[t] : t * K, f1 = tok_off ? tok_off[t + 1] : (t + 1) * K;
  float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int f = f0; f < f1; ++f) {
    const int e = experts[f];
    if (e < 0 || e >= E) continue;
    const float4 v = *reinterpret_cast<const float4*>(y + static_cast<size_t>(f) * H + c);
    s.x += v.x;
    s.y += v.y;
    s.z += v.z;
    s.w += v.w;
  }
  *reinterpret_cast<uint2*>(out + static_cast<size_t>(t) * H + c) =
      make_uint2(pack_bf16x2_rn(s.x, s.y), pack_bf16x2_rn(s.z, s.w));
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

cudaError_t launch_int4_experts(const Int4Args& p, cudaStream_t st) {
  MvArgs u{};
  u.wq = p.w1q;
  u.ws = static_cast<const __nv_bfloat16*>(p.w1s);
  u.group = p.group1;
  u.N = 2 * p.I;
  u.K = p.H;
  u.n_tiles = int4_row_tiles(u.N);
  u.k_blocks = int4_col_blocks(u.K);
  u.freq = p.freq;
  u.off = p.off;
  u.s_scatter = p.s_scatter;
  u.x_gather = p.x_gather;
  u.x = static_cast<const __nv_bfloat16*>(p.x);
  u.T = p.T;
  u.a = static_cast<__nv_bfloat16*>(p.a);
  u.err = p.err;
  MvArgs d = u;
  d.wq = p.w2q;
  d.ws = static_cast<const __nv_bfloat16*>(p.w2s);
  d.group = p.group2;
  d.N = p.H;
  d.K = p.I;
  d.n_tiles = int4_row_tiles(d.N);
  d.k_blocks = int4_col_blocks(d.K);
  d.x = u.a;
  d.scores = p.scores;
  d.y = p.y;
  mv_kernel<true><<<dim3(u.n_tiles, p.E), kMvThreads, 0, st>>>(u);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  mv_kernel<false><<<dim3(d.n_tiles, p.E), kMvThreads, 0, st>>>(d);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  for (int t0 = 0; t0 < p.T; t0 += 32768) {  // grid.y limit
    const int n = p.T - t0 < 32768 ? p.T - t0 : 32768;
    int4_combine_kernel<<<dim3(ceil_div(p.H, 1024), n), 256, 0, st>>>(
        p.y + (p.tok_off ? 0 : static_cast<size_t>(t0) * p.K * p.H), n, p.H, p.K,
        p.tok_off ? p.tok_off + t0 : nullptr, p.experts + (p.tok_off ? 0 : static_cast<size_t>(t0) * p.K), p.E,
        static_cast<__nv_bfloat16*>(p.out) + static_cast<size_t>(t0) * p.H);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace smb
