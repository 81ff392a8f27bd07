// Switch balance loss of the router (reference sonicmoe/moe.py:263-276), its per-expert counts and its
// gradient.
//
//   p[t, :] = softmax(logits[t, :]),  P_e = sum_t p[t, e] over the tokens that count, n = sum_e P_e,
//   f_e = entries routed to expert e, F = sum_e f_e,      loss = E * sum_e (P_e / n) (f_e / F)
//   dloss/dlogits[t, e] = p[t, e] (c_e - sum_j p[t, j] c_j),   c_e = (E f_e - F) / (F n)
//
// (sum_e p[t, e] = 1, so neither the normalisation of P by n nor a constant added to c changes the
// gradient; taking E f_e - F in 64 bits, where whole counts are exact, instead of E f_e keeps c free of the
// cancellation that a nearly balanced routing would otherwise bring.)
//
// switch_loss_kernel        one pass over the logits: softmax of each row in registers, its columns
//                           summed per thread, over the CTA and over a cluster of 8 CTAs; counts of the
//                           top-k indices beside it.
// switch_loss_finish_kernel adds the clusters' sums in a fixed order (no floating-point atomics: the loss
//                           is the same bits every time) and forms the loss and c.
// switch_loss_bwd_kernel    reads the logits once more, recomputes the softmax, writes the gradient.
//
// 131072 x 256 bf16: forward with counts 35 us, backward 27 us, against 11 and 21 us for their bytes.  The
// backward is bound by its instructions (76% of the issue slots; 151 a row of 256 for a warp, so operations
// go in pairs and a maximum in one instruction), the forward by the latency of a row's two reductions
// (54%), hence two rows a warp and the next two on the way.  Up to a few thousand tokens it is the launches:
// one CTA 4 us, two kernels 10 us.
#include "common.cuh"
#include "sonic_internal.h"

namespace smb {

namespace {

constexpr int kSlThreads = 256;
constexpr int kSlCluster = 8;       // CTAs of the forward that add their sums before they write them
constexpr int kSlMaxParts = 4 * 18;  // clusters at most: 4 CTAs per SM (5 or 6: 131072 x 256 37 us against 35)
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_f32(float v, float* p) { *p = v; }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16* p) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f32(float v, __half* p) { *p = __float2half_rn(v); }

// 8 consecutive values as loaded; vec: how many of them one aligned access may cover (8, 4 or 1).
template <typename InT>
struct Raw8 {
  alignas(16) InT v[8];
};
template <typename InT>
__device__ __forceinline__ void load8(const InT* __restrict__ src, int vec, int n, Raw8<InT>& raw) {
  if (vec >= 4 && n >= 8) {
    if constexpr (sizeof(InT) == 4) {
      *reinterpret_cast<uint4*>(raw.v) = __ldg(reinterpret_cast<const uint4*>(src));
      *reinterpret_cast<uint4*>(raw.v + 4) = __ldg(reinterpret_cast<const uint4*>(src + 4));
    } else if (vec == 8) {
      *reinterpret_cast<uint4*>(raw.v) = __ldg(reinterpret_cast<const uint4*>(src));
    } else {
      *reinterpret_cast<uint2*>(raw.v) = __ldg(reinterpret_cast<const uint2*>(src));
      *reinterpret_cast<uint2*>(raw.v + 4) = __ldg(reinterpret_cast<const uint2*>(src + 4));
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (j < n)
      raw.v[j] = src[j];
    else
      from_f32(-__int_as_float(0x7f800000), &raw.v[j]);
  }
}

template <typename InT>
__device__ __forceinline__ void store8(InT* __restrict__ dst, int vec, int n, const float* v) {
  alignas(16) InT raw[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) from_f32(v[j], &raw[j]);
  if (vec >= 4 && n >= 8) {
    if constexpr (sizeof(InT) == 4) {
      reinterpret_cast<uint4*>(dst)[0] = *reinterpret_cast<uint4*>(raw);
      reinterpret_cast<uint4*>(dst)[1] = *reinterpret_cast<uint4*>(raw + 4);
    } else if (vec == 8) {
      *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<uint4*>(raw);
    } else {
      reinterpret_cast<uint2*>(dst)[0] = *reinterpret_cast<uint2*>(raw);
      reinterpret_cast<uint2*>(dst)[1] = *reinterpret_cast<uint2*>(raw + 4);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < n) dst[j] = raw[j];
}

// Two fp32 operations in one instruction, each half rounded as the scalar operation would.
__device__ __forceinline__ unsigned long long f2_bits(float2 v) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
  return r;
}
__device__ __forceinline__ float2 f2_of(unsigned long long b) {
  float2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(b));
  return v;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)));
  return f2_of(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)));
  return f2_of(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)), "l"(f2_bits(c)));
  return f2_of(r);
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// N reductions at once over the L lanes that share a row: lanes of one warp (L <= 32) or the whole CTA,
// whose partial results go through s_red [N * L / 32].  Every thread of the group gets the results.
template <int L, bool kMax, int N>
__device__ __forceinline__ void row_reduce(float (&x)[N], float* s_red) {
  if constexpr (L >= 32 && kMax) {  // one instruction for a warp's maximum
#pragma unroll
    for (int n = 0; n < N; ++n) asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(x[n]) : "f"(x[n]));
  } else {
#pragma unroll
    for (int o = (L < 32 ? L : 32) / 2; o >= 1; o >>= 1)
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const float y = __shfl_xor_sync(0xffffffffu, x[n], o);
        x[n] = kMax ? fmaxf(x[n], y) : x[n] + y;
      }
  }
  if constexpr (L > 32) {
    __syncthreads();
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int n = 0; n < N; ++n) s_red[n * (L / 32) + (threadIdx.x >> 5)] = x[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
      x[n] = s_red[n * (L / 32)];
#pragma unroll
      for (int w = 1; w < L / 32; ++w) {
        const float y = s_red[n * (L / 32) + w];
        x[n] = kMax ? fmaxf(x[n], y) : x[n] + y;
      }
    }
  }
}

// R rows held as 8 * C values a lane: v becomes exp2(log2e (x - max)), s the lane's sum of it.  The
// maximum is subtracted before the scaling, so that a row of the type's lowest values does not overflow.
// A row whose maximum is not finite (all -inf, or +inf or NaN in it) gives NaN, as a softmax does.
template <int L, int C, int R>
__device__ __forceinline__ void exp_rows(float2 (&v)[R][4 * C], float (&s)[R], float* s_red) {
  float mx[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    mx[j] = fmaxf(v[j][0].x, v[j][0].y);
#pragma unroll
    for (int i = 1; i < 4 * C; ++i) mx[j] = fmaxf(mx[j], fmaxf(v[j][i].x, v[j][i].y));
  }
  row_reduce<L, true, R>(mx, s_red);
#pragma unroll
  for (int j = 0; j < R; ++j) {
    float2 s2 = both(0.0f);
#pragma unroll
    for (int i = 0; i < 4 * C; ++i) {
      const float2 t = mul2(add2(v[j][i], both(-mx[j])), both(kLog2e));
      v[j][i] = make_float2(ex2(t.x), ex2(t.y));
      s2 = add2(s2, v[j][i]);
    }
    s[j] = s2.x + s2.y;
  }
}
// 1 / s of a row's sum, 1 <= s <= E: within two units in the last place.
__device__ __forceinline__ float row_inv(float s) { return __fdividef(1.0f, s); }

// Rows that a group takes at once: two, where the registers allow it, keep twice the loads on the way and
// fill the latencies of one row's reductions with the other's (131072 x 256: forward 35 us against 39,
// backward 27 against 31).  An fp32 row of a whole warp has as many bytes by itself (42 us against 47).
template <typename InT, int L, int C>
constexpr int kRows = C == 1 && (sizeof(InT) == 2 || L < 32) ? 2 : 1;

// Lane layout: group lane l holds columns 8 l + 8 L c + (0..7), c < C; E <= 8 L C.  A row that does not
// count is not read (zeros stand in).
template <typename InT, int L, int C>
__device__ __forceinline__ void load_row(const InT* __restrict__ row, bool on, int E, int vec, int gl,
                                         Raw8<InT> (&raw)[C]) {
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (on) {
      load8<InT>(row + 8 * gl + 8 * L * c, vec, E - 8 * gl - 8 * L * c, raw[c]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) from_f32(0.0f, &raw[c].v[j]);
    }
  }
}
template <typename InT, int C>
__device__ __forceinline__ void row_f32(const Raw8<InT> (&raw)[C], float2 (&v)[4 * C]) {
#pragma unroll
  for (int i = 0; i < 4 * C; ++i)
    v[i] = make_float2(to_f32(raw[i / 4].v[2 * i % 8]), to_f32(raw[i / 4].v[2 * i % 8 + 1]));
}

__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return static_cast<int>(r);
}
// The 32-bit word at this CTA's shared address `p`, in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t ld_cluster(const void* p, int rank) {
  uint32_t a, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

// Counts as given: whole numbers, or fractions and averages of counts.
struct Counts {
  const void* p;
  int type;  // CountType
  __device__ __forceinline__ double at(int e) const {
    switch (type) {
      case kCountI32:
        return static_cast<const int32_t*>(p)[e];
      case kCountI64:
        return static_cast<double>(static_cast<const long long*>(p)[e]);
      case kCountF32:
        return static_cast<const float*>(p)[e];
      default:
        return static_cast<const double*>(p)[e];
    }
  }
};

// The threads' x and f summed over the CTA, in a fixed order; every thread gets the sums.
struct FinishSums {
  float x[32];
  double f[32];
};
__device__ __forceinline__ void block_sums(float& x, double& f, FinishSums& sm) {
  __syncthreads();
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    x += __shfl_xor_sync(0xffffffffu, x, o);
    f += __shfl_xor_sync(0xffffffffu, f, o);
  }
  if ((threadIdx.x & 31) == 0) {
    sm.x[threadIdx.x >> 5] = x;
    sm.f[threadIdx.x >> 5] = f;
  }
  __syncthreads();
  x = 0.0f;
  f = 0.0;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) {
    x += sm.x[w];
    f += sm.f[w];
  }
}

// P (column sums) and f (counts) of the CTA's experts e0 .. e0 + n_own - 1 -> loss, c, counts; s_p and, unless it
// is null, s_f lie in shared memory, other counts are those given.  kClustered: the CTAs of a cluster hold the
// experts between them.
template <bool kClustered>
__device__ void finish(const float* s_p, const int32_t* s_f, const Counts& given, int E, int e0, int n_own,
                       float* __restrict__ loss, float* __restrict__ coef, int32_t* __restrict__ freq_out) {
  __shared__ FinishSums s_sums;
  __shared__ float s_x[2];  // the CTA's sum of P, its part of the loss
  __shared__ double s_count;  // its sum of f
  auto count = [&](int e) { return s_f ? static_cast<double>(s_f[e]) : given.at(e0 + e); };
  float n = 0.0f;
  double F = 0.0;
  for (int e = threadIdx.x; e < n_own; e += blockDim.x) {
    n += s_p[e];
    F += count(e);
  }
  block_sums(n, F, s_sums);
  if constexpr (kClustered) {
    if (threadIdx.x == 0) {
      s_x[0] = n;
      s_count = F;
    }
    cluster_sync();
    n = 0.0f;
    F = 0.0;
#pragma unroll
    for (int k = 0; k < kSlCluster; ++k) {
      n += __uint_as_float(ld_cluster(&s_x[0], k));
      const uint32_t* half = reinterpret_cast<const uint32_t*>(&s_count);
      F += __hiloint2double(ld_cluster(half + 1, k), ld_cluster(half, k));
    }
  }
  // no token counts, or no entry: the loss and the gradient are 0 (a NaN sum stays NaN)
  const float inv_n = n == 0.0f ? 0.0f : 1.0f / n;
  const float inv_f = F == 0.0 ? 0.0f : 1.0f / static_cast<float>(F);
  float l = 0.0f;
  for (int e = threadIdx.x; e < n_own; e += blockDim.x) {
    const double f = count(e);
    l += (s_p[e] * inv_n) * (static_cast<float>(f) * inv_f);
    coef[e0 + e] = static_cast<float>(f * E - F) * inv_f * inv_n;
    if (freq_out) freq_out[e0 + e] = static_cast<int32_t>(f);
  }
  double none = 0.0;
  block_sums(l, none, s_sums);
  if constexpr (kClustered) {
    if (threadIdx.x == 0) s_x[1] = l;
    cluster_sync();
    if (cluster_rank() == 0) {
      l = 0.0f;
#pragma unroll
      for (int k = 0; k < kSlCluster; ++k) l += __uint_as_float(ld_cluster(&s_x[1], k));
      if (threadIdx.x == 0) *loss = l * static_cast<float>(E);
    }
    cluster_sync();  // nobody's shared memory goes away while it is read
  } else {
    if (threadIdx.x == 0) *loss = l * static_cast<float>(E);
  }
}

// Dynamic shared memory: column sums [kSlThreads / max(L, 32)][E] (one copy per warp, or one), counts [E].
template <typename InT, int L, int C>
__global__ void __launch_bounds__(kSlThreads)
    switch_loss_kernel(const InT* __restrict__ logits, int T, int E, int vec, const uint8_t* __restrict__ mask,
                       const int32_t* __restrict__ idx, int K, const Counts given, float* __restrict__ part_p,
                       int32_t* __restrict__ part_f, float* __restrict__ loss, float* __restrict__ coef, int32_t* __restrict__ freq_out, int* __restrict__ err) {
  constexpr int kGroups = kSlThreads / L;               // rows of a CTA's step
  constexpr int kCopies = L < 32 ? kSlThreads / 32 : kGroups;
  extern __shared__ float s_dyn[];
  __shared__ float s_red[16 * kRows<InT, L, C>];
  float* s_p = s_dyn;
  int32_t* s_f = reinterpret_cast<int32_t*>(s_dyn + static_cast<size_t>(kCopies) * E);
  const int gl = threadIdx.x % L, grp = threadIdx.x / L;
  pdl_launch();
  if (idx)
    for (int e = threadIdx.x; e < E; e += kSlThreads) s_f[e] = 0;
  float2 acc2[4 * C];
#pragma unroll
  for (int i = 0; i < 4 * C; ++i) acc2[i] = both(0.0f);
  // every group takes the same number of rows, so that the shuffles and barriers below are uniform; the
  // next rows are under way while some are reduced
  constexpr int R = kRows<InT, L, C>;
  const long long stride = static_cast<long long>(gridDim.x) * kGroups;
  auto counts = [&](long long r) { return r < T && (!mask || mask[r]); };
  long long r = static_cast<long long>(blockIdx.x) * kGroups + grp;
  Raw8<InT> next[R][C];
  bool on_next[R];
  auto load = [&] {
#pragma unroll
    for (int j = 0; j < R; ++j) on_next[j] = counts(r + j * stride);
#pragma unroll
    for (int j = 0; j < R; ++j) load_row<InT, L, C>(logits + (r + j * stride) * E, on_next[j], E, vec, gl, next[j]);
  };
  load();
  for (long long r0 = static_cast<long long>(blockIdx.x) * kGroups; r0 < T; r0 += R * stride) {
    float2 v[R][4 * C];
    bool on[R];
    float sum[R];
#pragma unroll
    for (int j = 0; j < R; ++j) {
      row_f32<InT, C>(next[j], v[j]);
      on[j] = on_next[j];
    }
    r += R * stride;
    load();
    exp_rows<L, C, R>(v, sum, s_red);
    row_reduce<L, false, R>(sum, s_red);
#pragma unroll
    for (int j = 0; j < R; ++j)
      if (on[j]) {
        const float2 inv = both(row_inv(sum[j]));
#pragma unroll
        for (int i = 0; i < 4 * C; ++i) acc2[i] = fma2(v[j][i], inv, acc2[i]);
      }
  }
  float acc[8 * C];
#pragma unroll
  for (int i = 0; i < 4 * C; ++i) {
    acc[2 * i] = acc2[i].x;
    acc[2 * i + 1] = acc2[i].y;
  }
  // rows of one warp first (lanes that hold the same columns), then the warps through shared memory
  if constexpr (L < 32) {
#pragma unroll
    for (int o = 16; o >= L; o >>= 1)
#pragma unroll
      for (int i = 0; i < 8 * C; ++i) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
  }
  if (L >= 32 || (threadIdx.x & 31) < L) {
    float* dst = s_p + static_cast<size_t>(L < 32 ? threadIdx.x / 32 : grp) * E;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int e = 8 * gl + 8 * L * c + j;
        if (e < E) dst[e] = acc[8 * c + j];
      }
  }
  __syncthreads();
  if (idx) {
    const int n = T * K;
    for (int i = blockIdx.x * kSlThreads + threadIdx.x; i < n; i += gridDim.x * kSlThreads) {
      if (mask && !mask[i / K]) continue;
      const int e = idx[i];
      if (e >= 0 && e < E)
        atomicAdd(&s_f[e], 1);
      else
        atomicCAS(err, 0, kErrBadExpert);
    }
    __syncthreads();
  }
  for (int e = threadIdx.x; e < E; e += kSlThreads) {
    float p = s_p[e];
    for (int k = 1; k < kCopies; ++k) p += s_p[static_cast<size_t>(k) * E + e];
    s_p[e] = p;
  }
  if (gridDim.x == 1) {
    __syncthreads();
    finish<false>(s_p, idx ? s_f : nullptr, given, E, 0, E, loss, coef, freq_out);
    return;
  }
  // the cluster's CTAs each add an eighth of the columns over all 8
  cluster_sync();
  const int rank = blockIdx.x % kSlCluster;
  const size_t part = static_cast<size_t>(blockIdx.x / kSlCluster) * E;
  for (int e = rank * kSlThreads + threadIdx.x; e < E; e += kSlCluster * kSlThreads) {
    float p = 0.0f;
    int f = 0;
#pragma unroll
    for (int k = 0; k < kSlCluster; ++k) {
      p += __uint_as_float(ld_cluster(&s_p[e], k));
      if (idx) f += static_cast<int>(ld_cluster(&s_f[e], k));
    }
    part_p[part + e] = p;
    if (idx) part_f[part + e] = f;
  }
  cluster_sync();  // nobody's shared memory goes away while it is read
}

// The clusters' sums: `slices` groups of threads each add every slices-th part, then the groups are added in
// order.  Up to 256 experts one CTA does it; more are shared by the CTAs of a cluster, since the chain of
// loads would take longer than its barriers (forward, us, one CTA / a cluster: 20000 x 4096 138 / 82, 65536 x
// 512 37 / 34, 131072 x 256 35 / 35, 32768 x 128 14 / 16).
constexpr int kFinThreads = 1024;
constexpr int kFinOneCta = 256;

template <bool kClustered>
__global__ void __launch_bounds__(kFinThreads)
    switch_loss_finish_kernel(const float* __restrict__ part_p, const int32_t* __restrict__ part_f, int parts, int E,
                              int slices, const Counts given, float* __restrict__ loss, float* __restrict__ coef,
                              int32_t* __restrict__ freq_out) {
  __shared__ float s_p[kFinThreads];
  __shared__ int32_t s_f[kFinThreads];
  const int own = kClustered ? (E + kSlCluster - 1) / kSlCluster : E;  // slices * own <= kFinThreads
  const int e0 = kClustered ? min(E, cluster_rank() * own) : 0, n_own = min(own, E - e0);
  const int sl = threadIdx.x / own, c = threadIdx.x - sl * own;
  pdl_wait();
  if (sl < slices && c < n_own) {
    float p = 0.0f;
    int f = 0;
#pragma unroll 12
    for (int k = sl; k < parts; k += slices) {
      p += part_p[static_cast<size_t>(k) * E + e0 + c];
      if (part_f) f += part_f[static_cast<size_t>(k) * E + e0 + c];
    }
    s_p[threadIdx.x] = p;
    s_f[threadIdx.x] = f;
  }
  __syncthreads();
  if (threadIdx.x < n_own) {
    float p = s_p[threadIdx.x];
    int f = s_f[threadIdx.x];
    for (int k = 1; k < slices; ++k) {
      p += s_p[k * own + threadIdx.x];
      f += s_f[k * own + threadIdx.x];
    }
    s_p[threadIdx.x] = p;
    s_f[threadIdx.x] = f;
  }
  __syncthreads();
  finish<kClustered>(s_p, part_f ? s_f : nullptr, given, E, e0, n_own, loss, coef, freq_out);
}

template <typename InT, int L, int C>
__global__ void __launch_bounds__(kSlThreads)
    switch_loss_bwd_kernel(const InT* __restrict__ logits, int T, int E, int vec, const uint8_t* __restrict__ mask,
                           const float* __restrict__ coef, const float* __restrict__ dloss,
                           InT* __restrict__ dlogits) {
  constexpr int kGroups = kSlThreads / L;
  __shared__ float s_red[16 * kRows<InT, L, C>];
  const int gl = threadIdx.x % L, grp = threadIdx.x / L;
  const float g = *dloss;
  float2 c[4 * C];
#pragma unroll
  for (int i = 0; i < 4 * C; ++i) {
    const int e = 8 * gl + 8 * L * (i / 4) + 2 * (i % 4);
    c[i] = make_float2(e < E ? coef[e] : 0.0f, e + 1 < E ? coef[e + 1] : 0.0f);
  }
  constexpr int R = kRows<InT, L, C>;
  const long long stride = static_cast<long long>(gridDim.x) * kGroups;
  auto counts = [&](long long r) { return r < T && (!mask || mask[r]); };
  long long r = static_cast<long long>(blockIdx.x) * kGroups + grp;
  Raw8<InT> next[R][C];
  bool on_next[R];
  auto load = [&](long long at) {
#pragma unroll
    for (int j = 0; j < R; ++j) on_next[j] = counts(at + j * stride);
#pragma unroll
    for (int j = 0; j < R; ++j) load_row<InT, L, C>(logits + (at + j * stride) * E, on_next[j], E, vec, gl, next[j]);
  };
  load(r);
  for (long long r0 = static_cast<long long>(blockIdx.x) * kGroups; r0 < T; r0 += R * stride, r += R * stride) {
    float2 v[R][4 * C];
    bool on[R];
    float sum[R], sums[2 * R];  // the rows' sums, then their products with c
#pragma unroll
    for (int j = 0; j < R; ++j) {
      row_f32<InT, C>(next[j], v[j]);
      on[j] = on_next[j];
    }
    load(r + R * stride);
    exp_rows<L, C, R>(v, sum, s_red);
#pragma unroll
    for (int j = 0; j < R; ++j) {
      float2 d = both(0.0f);
#pragma unroll
      for (int i = 0; i < 4 * C; ++i) d = fma2(v[j][i], c[i], d);
      sums[j] = sum[j];
      sums[R + j] = d.x + d.y;
    }
    row_reduce<L, false, 2 * R>(sums, s_red);
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const long long row = r + j * stride;
      if (row >= T) continue;
      float w[8 * C];
      if (on[j]) {
        const float inv = row_inv(sums[j]);
        const float2 gi = both(g * inv), dot = both(-sums[R + j] * inv);
#pragma unroll
        for (int i = 0; i < 4 * C; ++i) {
          const float2 o = mul2(mul2(v[j][i], gi), add2(c[i], dot));
          w[2 * i] = o.x;
          w[2 * i + 1] = o.y;
        }
      } else {  // a token that does not count gets a gradient of exactly 0, whatever its logits hold
#pragma unroll
        for (int i = 0; i < 8 * C; ++i) w[i] = 0.0f;
      }
#pragma unroll
      for (int k = 0; k < C; ++k)
        store8<InT>(dlogits + row * E + 8 * gl + 8 * L * k, vec, E - 8 * gl - 8 * L * k, w + 8 * k);
    }
  }
}

// Aligned accesses of a row's 8-value pieces: 8, 4 or 1 values at a time.
int vec_of(const void* p, int E, int esize) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p);
  if (esize == 4) return E % 4 == 0 && a % 16 == 0 ? 4 : 1;
  if (E % 8 == 0 && a % 16 == 0) return 8;
  return E % 4 == 0 && a % 8 == 0 ? 4 : 1;
}

struct SlArgs {
  const void* logits;
  int T, E;
  const uint8_t* mask;
  const int32_t* idx;
  int K;
  Counts given;
  float* part_p;
  int32_t* part_f;
  float* loss;
  float* coef;
  int32_t* freq_out;
  int* err;
  const float* dloss;
  void* dlogits;
  int grid;
};

template <typename InT, int L, int C>
cudaError_t launch_lc(const SlArgs& a, bool bwd, cudaStream_t st) {
  const InT* x = static_cast<const InT*>(a.logits);
  if (bwd) {
    int vec = vec_of(a.logits, a.E, sizeof(InT));
    const int v2 = vec_of(a.dlogits, a.E, sizeof(InT));
    vec = v2 < vec ? v2 : vec;
    switch_loss_bwd_kernel<InT, L, C><<<a.grid, kSlThreads, 0, st>>>(x, a.T, a.E, vec, a.mask, a.coef, a.dloss,
                                                                      static_cast<InT*>(a.dlogits));
    return cudaGetLastError();
  }
  constexpr int kCopies = L < 32 ? kSlThreads / 32 : kSlThreads / L;
  const int smem = (kCopies + 1) * a.E * 4;
  auto kern = switch_loss_kernel<InT, L, C>;
  const int vec = vec_of(a.logits, a.E, sizeof(InT));
  cudaError_t e;
  if (a.grid == 1) {
    kern<<<1, kSlThreads, smem, st>>>(x, a.T, a.E, vec, a.mask, a.idx, a.K, a.given, a.part_p, a.part_f, a.loss, a.coef,
                                      a.freq_out, a.err);
    return cudaGetLastError();
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.grid * kSlCluster);
  cfg.blockDim = dim3(kSlThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = kSlCluster;
  at.val.clusterDim.y = 1;
  at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kern, x, a.T, a.E, vec, a.mask, a.idx, a.K, a.given, a.part_p, a.part_f, a.loss, a.coef,
                         a.freq_out, a.err);
  if (e != cudaSuccess) return e;
  const bool one = a.E <= kFinOneCta;
  const int ctas = one ? 1 : kSlCluster, slices = kFinThreads / ceil_div(a.E, ctas);
  return launch_dependent(one ? switch_loss_finish_kernel<false> : switch_loss_finish_kernel<true>, dim3(ctas),
                          kFinThreads, 0, ctas, st, a.part_p, a.idx ? a.part_f : nullptr, a.grid, a.E,
                          slices < 32 ? slices : 32, a.given, a.loss, a.coef, a.freq_out);
}

// Lanes per row: as many as hold the row at 8 values each, up to a warp; wider rows take 16 or 32
// values a lane, and beyond 1024 experts a whole CTA shares the row.
int lanes_of(int E) { return E <= 32 ? 4 : E <= 64 ? 8 : E <= 128 ? 16 : E <= 1024 ? 32 : kSlThreads; }

template <typename InT>
cudaError_t launch_t(const SlArgs& a, bool bwd, cudaStream_t st) {
  if (a.E <= 32) return launch_lc<InT, 4, 1>(a, bwd, st);
  if (a.E <= 64) return launch_lc<InT, 8, 1>(a, bwd, st);
  if (a.E <= 128) return launch_lc<InT, 16, 1>(a, bwd, st);
  if (a.E <= 256) return launch_lc<InT, 32, 1>(a, bwd, st);
  if (a.E <= 512) return launch_lc<InT, 32, 2>(a, bwd, st);
  if (a.E <= 1024) return launch_lc<InT, 32, 4>(a, bwd, st);
  return launch_lc<InT, kSlThreads, 2>(a, bwd, st);
}

cudaError_t launch(const SlArgs& a, int dtype, bool bwd, cudaStream_t st) {
  switch (dtype) {
    case kDtypeBF16:
      return launch_t<__nv_bfloat16>(a, bwd, st);
    case kDtypeF16:
      return launch_t<__half>(a, bwd, st);
    default:
      return launch_t<float>(a, bwd, st);
  }
}

}  // namespace

// Rows of the partial sums: one CTA does it all where that takes at most 8 steps, else clusters of 8.
int switch_loss_parts(int T, int E) {
  const int ctas = ceil_div(T, 8 * (kSlThreads / lanes_of(E)));
  const int want = ceil_div(ctas, kSlCluster);
  return ctas <= 1 ? 1 : want < 2 ? 2 : want > kSlMaxParts ? kSlMaxParts : want;
}

cudaError_t launch_switch_loss(const void* logits, int dtype, int T, int E, const uint8_t* mask, const int32_t* idx,
                               int K, const void* counts, int count_type, float* part_p, int32_t* part_f, float* loss,
                               float* coef, int32_t* freq_out, int* err, cudaStream_t st) {
  SlArgs a{logits, T, E, mask, idx, K, Counts{counts, count_type}, part_p, part_f, loss, coef, freq_out, err, nullptr, nullptr,
           switch_loss_parts(T, E)};
  return launch(a, dtype, false, st);
}

cudaError_t launch_switch_loss_bwd(const void* logits, int dtype, int T, int E, const uint8_t* mask,
                                   const float* coef, const float* dloss, void* dlogits, cudaStream_t st) {
  if (T == 0) return cudaSuccess;
  SlArgs a{};
  a.logits = logits;
  a.T = T;
  a.E = E;
  a.mask = mask;
  a.coef = const_cast<float*>(coef);
  a.dloss = dloss;
  a.dlogits = dlogits;
  const int rows = kSlThreads / lanes_of(E);
  const int want = ceil_div(T, rows);
  a.grid = want > 8 * 148 ? 8 * 148 : want;
  return launch(a, dtype, true, st);
}

}  // namespace smb
