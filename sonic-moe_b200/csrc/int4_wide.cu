// Expert products with 4-bit weights for many tokens (format and layout: int4.cuh; few tokens: int4.cu).
//
// Grouped GEMMs on tcgen05 whose first operand is the weight: D[256 rows, tokens] = W[256, K] x[tokens, K]^T.
// The codes go from global memory through shared memory into registers, become bf16 there (exact, scale
// included) and are stored to tensor memory, from where the MMA reads its A operand; x comes through TMA
// into 128-byte-swizzled shared memory.  Keeping A out of shared memory is what makes this bound by the
// weights' bytes rather than by shared memory: at 64 tokens a 128 x 128 step moves 8 KB of codes, and
// writing its 32 KB of bf16 to shared memory and reading it back would take twice as long as HBM does.
//
// The columns inside a block of 32 are permuted on the way (both operands alike, the product does not
// see it): a lane of a dequantising warp holds 8 consecutive columns as 4 pairs, and the 16-lane x
// 128-bit store to tensor memory takes one pair of each of 4 lanes, so column 8 t + 2 i + e sits at
// place 8 i + 2 t + e.  x is gathered into expert order and permuted by wide_gather_kernel; the up
// projection writes its intermediate in that order.
//
// Roles per CTA (736 threads, one CTA per SM):
//   warps 0-15   dequantise; a group of 4 has one half of the rows and every other step of 128 columns,
//                its warp w rows 32 (w % 4) .. + 31 of the half
//   warps 16-19  epilogue: rows 32 (w % 4) .. of the accumulators of the two halves
//   warp 20      TMA producer of x
//   warps 21-22  MMA issuers, one for each half of the rows (21 allocates tensor memory)
// An issuer's waits and its commit cost it some hundred cycles a step whatever they guard, as long as its
// 8 MMAs of 64 tokens take (32 cycles each, measured).  So a step has 128 columns and the halves have an
// issuer each, whose work the tensor core interleaves.  An item has 256 rows because x, which every row
// tile reads from L2, otherwise costs an SM twice the bytes of the weights (64 tokens: 16 KB a step
// against 8 KB).
// Work items (expert, 256 rows, up to kN of its tokens), rows fastest, static round robin; the items of
// an expert's token chunks follow each other, so their second reading of the weights is from L2.  kN is
// 64 or 128; 128 halves the dequantising per token, 64 leaves room for a third stage of weights in tensor
// memory.
// What it spends its time on (512 tokens, 64 experts of 4096 x 1024): the dequantising warps.  Per SM a step of 256
// rows takes about 1000 cycles, against 790 for its bytes at the HBM rate and 512 for its MMAs; 7 of the 11
// instructions for 8 weights are integer ones, which an SM issues at half rate (448 cycles of the step).
// The schedulers issue in 62% of the cycles, the integer pipe is busy in 57% of them: no unit is full, the warps
// also wait for their stores to tensor memory.  24 dequantising warps
// gain nothing (16 tokens 167 against 163 us, 64 tokens 235 against 228).
// Fetching the codes by bulk copies from a warp of their own instead of per-lane copies, which takes a
// tenth of the instructions away but adds a barrier wait to every step, measured 117 us against 104 (up
// projection); double-buffered accumulators instead of the third stage of weights 239 against 228 us
// (64 tokens, 128 experts).
// Every wait is bounded; after a time-out the kernel records an error, drains and returns.
#include "int4.cuh"

namespace smb {

namespace {

constexpr int kWdDeqWarps = 16;
constexpr int kWdThreads = 32 * (kWdDeqWarps + 7);

template <int kN>  // tokens of an item at most
struct WdShape {
  static constexpr uint32_t kTmemA = 2 * kN;  // accumulators of the two halves below, stages of A from here
  static constexpr int kAStages = (512 - 2 * kN) / 128;
  static constexpr int kBHalf = kN * 128;  // 64 columns of x
  static constexpr int kBStage = 2 * kBHalf;
  static constexpr int kStages = 98304 / kBStage;  // 128-column steps of x in shared memory
};

template <int GPB>
struct WdRing {
  static constexpr int kStage = 2 * (1024 + 128 * GPB);  // a step of 2 row tiles, GPB scale words a lane
  // steps of codes in flight per dequantising warp: what fits beside x and 4096 experts' prefix
  static constexpr int kDepth = GPB == 1 ? 3 : 2;
  static constexpr int kBytes = kWdDeqWarps * kDepth * kStage;
};

struct WdArgs {
  const uint8_t* wq;
  const __nv_bfloat16* ws;
  int N, n_tiles, k_blocks;  // prepared rows, their 16-row tiles, column blocks
  int E, m_tiles;
  const int32_t* freq;
  const int32_t* off;
  __nv_bfloat16* a;  // up output [entries, a_ld], sorted order, permuted columns, zero beyond N / 2
  int a_ld;
  float* y;  // down output [entries, N], sorted order
  int* stop;  // 0, or the code of a wait of this call that gave up
  int* err;   // the caller's error word, which only learns of such a wait
};

struct WdItem {
  int e, mt, base, n;
};

__device__ __forceinline__ void tc_mma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// kind::f16 instruction descriptor: bf16 x bf16 -> f32, both operands K-major.
__device__ __forceinline__ uint32_t wd_idesc(int n) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (8u << 24);
}
// 16 lanes x 32 columns: lane 4 g + t of the warp gives columns 4 c + t of rows g (r[2 c]) and g + 8 (r[2 c + 1]).
__device__ __forceinline__ void tmem_st_16x32(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}\n" : "=r"(p));
  return p != 0;
}
// A wait of a whole warp, with one answer for all its lanes.  A wait gives up once *stop is set, so that word
// is this call's own: a routing entry that was rejected, or an error of an earlier call in the caller's word,
// must not end the waits of a call that is all right.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* stop, int where) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, stop, where));
}

// Tokens of one of an expert's ceil(n / kN) chunks: the equal share rounded up to whole 16s, and what is left for
// the last (193 tokens in chunks of 64: 64, 64, 64 and 1).
__device__ __forceinline__ int wd_share(int n, int chunks) { return ((n + chunks - 1) / chunks + 15) & ~15; }

// Place of column k (< 32) of a block of 32 in the permuted order.
__device__ __forceinline__ int wd_place(int k) { return 8 * ((k >> 1) & 3) + 2 * (k >> 3) + (k & 1); }

template <bool kUp, int kN, int GPB>
__global__ void __launch_bounds__(kWdThreads, 1)
    wide_kernel(const __grid_constant__ CUtensorMap tmap_x16, const __grid_constant__ CUtensorMap tmap_x64,
                const WdArgs p) {
  using Shape = WdShape<kN>;
  constexpr int kStages = Shape::kStages;
  extern __shared__ uint8_t smem_raw[];
  // step n, half h: full_a[h][n % kA] the weights are there, full_b[n % kStages] x is, done[h][n % kStages] the
  // MMAs have read both
  constexpr int kA = Shape::kAStages;
  __shared__ uint64_t full_a[2][kA], full_b[kStages], done[2][kStages], tfull, tempty, drain[2];
  __shared__ uint32_t tmem_holder;
  __shared__ int32_t s_warp[kWdThreads / 32];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  uint8_t* rings = smem + kStages * Shape::kBStage;
  int32_t* pre = reinterpret_cast<int32_t*>(rings + WdRing<GPB>::kBytes);  // [E + 1] chunks before each expert
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int s = 0; s < kA; ++s)
      for (int h = 0; h < 2; ++h) mbar_init(&full_a[h][s], 4);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_b[s], 1);
      mbar_init(&done[0][s], 1);
      mbar_init(&done[1][s], 1);
    }
    mbar_init(&tfull, 2);
    mbar_init(&tempty, 4);
    mbar_init(&drain[0], 1);
    mbar_init(&drain[1], 1);
    fence_mbar_init();
    prefetch_tmap(&tmap_x16);
    prefetch_tmap(&tmap_x64);
  }
  if (warp == kWdDeqWarps + 5) {
    tmem_alloc(&tmem_holder, 512);
    tmem_relinquish();
  }
  pdl_launch();
  pdl_wait();
  {  // chunks of kN tokens per expert, exclusive prefix
    const int per = (p.E + kWdThreads - 1) / kWdThreads;
    const int e0 = min(p.E, tid * per), e1 = min(p.E, e0 + per);
    int c = 0;
    for (int e = e0; e < e1; ++e) c += (p.freq[e] + kN - 1) / kN;
    int inc = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    int run = inc - c;
    for (int w = 0; w < warp; ++w) run += s_warp[w];
    for (int e = e0; e < e1; ++e) {
      pre[e] = run;
      run += (p.freq[e] + kN - 1) / kN;
    }
    if (tid == kWdThreads - 1) pre[p.E] = run;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_holder;
  const int items = pre[p.E] * p.m_tiles;
  auto item_of = [&](int i) {
    WdItem it;
    const int c = i / p.m_tiles;
    it.mt = i - c * p.m_tiles;
    int lo = 0, hi = p.E;  // pre[lo] <= c < pre[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= c)
        lo = mid;
      else
        hi = mid;
    }
    it.e = lo;
    const int n = p.freq[lo], share = wd_share(n, pre[lo + 1] - pre[lo]);
    const int done = (c - pre[lo]) * share;
    it.base = p.off[lo] + done;
    it.n = min(share, n - done);
    return it;
  };

  if (warp < kWdDeqWarps) {
    // ---------------------------------------------------------------- dequantise
    // Steps are numbered through all items of the CTA; a group takes every other one.  A parity wait may
    // not fall two phases behind its barrier; here it cannot, since the wait for a step's MMAs implies that
    // every earlier use of the barriers is over.
    constexpr int kStage = WdRing<GPB>::kStage, kDepth = WdRing<GPB>::kDepth;
    const Int4Magic magic;
    const int quarter = warp & 3, half = (warp >> 2) & 1, odd = warp >> 3, g = lane >> 2;
    const uint32_t ring = smem_u32(rings) + warp * kDepth * kStage;
    int l_item = blockIdx.x, l_b = odd, l_stage = 0, u_stage = 0;
    const uint8_t* l_src[2] = {};
    const __nv_bfloat16* l_sc[2] = {};
    bool l_on[2] = {};
    auto open = [&] {  // the item of block l_b
      const int skip = l_b / p.k_blocks;
      l_item += skip * gridDim.x;
      l_b -= skip * p.k_blocks;
      if (l_item >= items) return;
      const WdItem it = item_of(l_item);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int tile = it.mt * 16 + 8 * half + 2 * quarter + j;
        l_on[j] = tile < p.n_tiles;
        const size_t blk = (static_cast<size_t>(it.e) * p.n_tiles + (l_on[j] ? tile : 0)) * p.k_blocks + l_b;
        l_src[j] = p.wq + blk * 1024 + 16 * lane;
        l_sc[j] = p.ws + blk * (GPB * 16) + g * (GPB * 2);
      }
    };
    auto fill = [&] {
      if (l_item < items) {
        const uint32_t st = ring + l_stage * kStage;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t sd = st + 2048 + j * 128 * GPB + 4 * GPB * lane;
          if (l_on[j]) {
            cp_async16(st + 1024 * j + 16 * lane, l_src[j]);
            cp_async16(st + 1024 * j + 512 + 16 * lane, l_src[j] + 512);
            if constexpr (GPB == 4)
              cp_async16(sd, l_sc[j]);
            else
              cp_async_small<4 * GPB>(sd, l_sc[j]);
          } else {  // rows past the last tile: any codes, scale 0
#pragma unroll
            for (int i = 0; i < GPB; ++i) asm volatile("st.shared.u32 [%0], %1;" ::"r"(sd + 4 * i), "r"(0) : "memory");
          }
          l_src[j] += 2 * 1024;
          l_sc[j] += 2 * GPB * 16;
        }
        if (++l_stage == kDepth) l_stage = 0;
        l_b += 2;
        if (l_b >= p.k_blocks) open();
      }
      cp_async_commit();
    };
    open();
#pragma unroll
    for (int d = 0; d < kDepth - 1; ++d) fill();
    const int my_items = (items - static_cast<int>(blockIdx.x) + static_cast<int>(gridDim.x) - 1) /
                         static_cast<int>(gridDim.x);
    const int total = my_items * p.k_blocks;  // steps of this CTA
    const uint32_t lanes = tmem + Shape::kTmemA + 64 * half + (static_cast<uint32_t>(32 * quarter) << 16);
    bool ok = true;
    for (int step = odd; step < total; step += 2) {
      const int sa = step % kA;  // stage of tensor memory
      fill();  // the stage freed by the step before
      cp_async_wait<kDepth - 1>();
      const uint32_t st = ring + u_stage * kStage;
      if (++u_stage == kDepth) u_stage = 0;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t sw[GPB];
#pragma unroll
        for (int i = 0; i < GPB; ++i) sw[i] = lds32(st + 2048 + j * 128 * GPB + 4 * GPB * lane + 4 * i);
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // 64 columns
          const uint4 q = lds128(st + 1024 * j + 512 * h + 16 * lane);
          const uint32_t w[4] = {q.x, q.y, q.z, q.w};
          uint32_t r[16];
#pragma unroll
          for (int k = 0; k < 2; ++k) {  // 32 columns
            const uint32_t s = sw[(2 * h + k) * GPB / 4];
            const __nv_bfloat162 sl = int4_scale2(s, 0), sh = int4_scale2(s, 1);
            const __nv_bfloat162 ml = int4_m24(sl), mh = int4_m24(sh);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              r[2 * (4 * k + c)] = int4_scaled(magic, w[2 * k], c, sl, ml);
              r[2 * (4 * k + c) + 1] = int4_scaled(magic, w[2 * k + 1], c, sh, mh);
            }
          }
          if (ok && j == 0 && h == 0) {  // the MMAs of the stage's last step
            if (step >= kA)
              ok = warp_wait(&done[half][(step - kA) % kStages], ((step - kA) / kStages) & 1, p.stop,
                             kErrTimeoutProducer);
            tc_fence_after();
          }
          if (ok) tmem_st_16x32(lanes + 128 * sa + (static_cast<uint32_t>(16 * j) << 16) + 32 * h, r);
        }
      }
      if (!ok) break;
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full_a[half][sa]);
    }
    cp_async_wait<0>();
  } else if (warp < kWdDeqWarps + 4) {
    // ---------------------------------------------------------------- epilogue
    const int quarter = warp & 3;
    int li = 0;
    for (int i = blockIdx.x; i < items; i += gridDim.x, ++li) {
      const WdItem it = item_of(i);
      if (!warp_wait(&tfull, li & 1, p.stop, kErrTimeoutEpilogue)) break;
      tc_fence_after();
      const int pieces = (it.n + 31) / 32;
      for (int piece = 0; piece < 2 * pieces; ++piece) {  // half of the rows, 32 tokens
        const int half = piece >= pieces, c0 = 32 * (piece - half * pieces);
        uint32_t v[32];
        tmem_ld32(tmem + half * kN + c0 + (static_cast<uint32_t>(32 * quarter) << 16), v);
        tmem_ld_wait();
        const int n = min(32, it.n - c0);
        if (kUp) {
          // even lanes hold gates, odd lanes the ups of the same output column: a pair finishes two tokens
          const bool odd = lane & 1;
          const int col = it.mt * 128 + half * 64 + quarter * 16 + (lane >> 1);
          __nv_bfloat16* dst =
              p.a + static_cast<size_t>(it.base + c0 + (odd ? 1 : 0)) * p.a_ld + (col & ~31) + wd_place(col & 31);
#pragma unroll
          for (int c = 0; c < 32; c += 2, dst += 2 * p.a_ld) {
            const float v0 = __uint_as_float(v[c]), v1 = __uint_as_float(v[c + 1]);
            const float o = __shfl_xor_sync(0xffffffffu, odd ? v0 : v1, 1);
            const float r = odd ? silu_mul(o, v1) : silu_mul(v0, o);
            if (c + (odd ? 1 : 0) < n) *dst = __float2bfloat16_rn(r);
          }
        } else {
          const int row = it.mt * 256 + half * 128 + quarter * 32 + lane;
          float* dst = p.y + static_cast<size_t>(it.base + c0) * p.N + row;
          if (row < p.N) {
#pragma unroll
            for (int c = 0; c < 32; ++c, dst += p.N)
              if (c < n) *dst = __uint_as_float(v[c]);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty);
    }
  } else if (warp == kWdDeqWarps + 4) {
    // ---------------------------------------------------------------- TMA producer of x
    if (lane == 0) {
      const uint64_t policy = policy_evict_last();  // every row tile of the expert reads it
      int step = 0;
      bool ok = true;
      for (int i = blockIdx.x; ok && i < items; i += gridDim.x) {
        const WdItem it = item_of(i);
        // boxes of 64 rows, or with fewer tokens of 16 (rows past the item's are not used)
        const int rows = it.n > 48 ? 64 : 16, boxes = (it.n + rows - 1) / rows;
        const CUtensorMap* map = it.n > 48 ? &tmap_x64 : &tmap_x16;
        for (int k = 0; k < p.k_blocks; ++k, ++step) {
          const int s = step % kStages;
          const uint32_t ph = ((step / kStages) & 1) ^ 1;
          if (!mbar_wait(&done[0][s], ph, p.stop, kErrTimeoutProducer) ||
              !mbar_wait(&done[1][s], ph, p.stop, kErrTimeoutProducer)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&full_b[s], 2 * boxes * rows * 128);
          for (int h = 0; h < 2; ++h)
            for (int r = 0; r < boxes; ++r)
              tma_load_2d(smem + s * Shape::kBStage + h * Shape::kBHalf + r * rows * 128, map, &full_b[s],
                          k * 128 + h * 64, it.base + rows * r, policy);
        }
      }
      // let the loads already issued land before shared memory goes away: an issuer that gave up has not
      // waited for them
      for (int j = max(0, step - kStages); j < step; ++j)
        mbar_wait_ns(&full_b[j % kStages], (j / kStages) & 1, 50000000ull);
    }
  } else {
    // ---------------------------------------------------------------- MMA issuers
    // The whole warp walks the loop, so that the operands of the MMAs are known to be uniform; one
    // elected lane issues.
    const int half = warp - (kWdDeqWarps + 5);
    int step = 0, li = 0;
    bool ok = true;
    for (int i = blockIdx.x; ok && i < items; i += gridDim.x, ++li) {
      const int n = __shfl_sync(0xffffffffu, item_of(i).n, 0);
      const uint32_t idesc = wd_idesc((n + 15) & ~15);
      if (!warp_wait(&tempty, (li & 1) ^ 1, p.stop, kErrTimeoutMma)) break;
      tc_fence_after();
      const uint32_t d = tmem + half * kN;
      for (int k = 0; k < p.k_blocks; ++k, ++step) {
        const int s = step % kStages, g = step % kA;
        if (!warp_wait(&full_b[s], (step / kStages) & 1, p.stop, kErrTimeoutMma) ||
            !warp_wait(&full_a[half][g], (step / kA) & 1, p.stop, kErrTimeoutMma)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint64_t bd = sdesc_sw128(smem_u32(smem + s * Shape::kBStage));
        const uint32_t a = tmem + Shape::kTmemA + 128 * g + 64 * half;
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)  // 16 columns per MMA: 8 columns of A, 32 bytes of B
            tc_mma_bf16_ts(d, a + 8 * kk, bd + (kk >> 2) * (Shape::kBHalf >> 4) + 2 * (kk & 3), idesc,
                           (k | kk) != 0 ? 1u : 0u);
          tc_commit(&done[half][s]);
        }
        __syncwarp();
      }
      if (ok && elect_one()) tc_commit(&tfull);
      __syncwarp();
    }
    if (elect_one()) {
      tc_commit(&drain[half]);  // every MMA has finished before tensor memory is freed
      mbar_wait_ns(&drain[half], 0, 100000000ull);
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kWdDeqWarps + 5) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (tid == 0) {  // a wait that gave up leaves rows unwritten: it outranks a rejected entry
    const int code = *reinterpret_cast<volatile int*>(p.stop);
    if (code != 0) atomicExch(p.err, code);
  }
}

// Routing plan of few entries (kPlanMaxEntries) and experts (kPlanMaxExperts) in one CTA: counts, offsets,
// an expert order (s_rev: place of an entry, x_gather: token of a place) and, for explicit lists, the
// entries of each token.  The order of an expert's entries is that of shared-memory atomics: it decides
// which column of a product an entry takes, and no column's value depends on that.  (For more entries,
// the tiled kernels of router.cu.)
constexpr int kPlanMaxEntries = 16384, kPlanMaxExperts = 1024;

template <int kPer>  // entries of a thread
__global__ void __launch_bounds__(1024)
    wide_plan_kernel(const int32_t* __restrict__ experts, const int32_t* __restrict__ tokens, int n, int T, int K, int E,
                     int32_t* __restrict__ freq, int32_t* __restrict__ off, int32_t* __restrict__ s_rev,
                     int32_t* __restrict__ x_gather, int32_t* __restrict__ tok_off, int* err, int* stop) {
  __shared__ int32_t s_cnt[kPlanMaxExperts], s_sum[32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_launch();
  int e[kPer], rank[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) e[i] = tid + 1024 * i < n ? experts[tid + 1024 * i] : -1;
  s_cnt[tid] = 0;
  if (tid == 0) *stop = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (e[i] >= 0 && e[i] < E) {
      rank[i] = atomicAdd(&s_cnt[e[i]], 1);
    } else {
      if (tid + 1024 * i < n) atomicCAS(err, 0, kErrBadExpert);
      e[i] = -1;
    }
  }
  __syncthreads();
  const int count = s_cnt[tid];  // zero beyond E
  int inc = count;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  if (lane == 31) s_sum[warp] = inc;
  __syncthreads();
  int base = inc - count;
  for (int w = 0; w < warp; ++w) base += s_sum[w];
  s_cnt[tid] = base;
  if (tid < E) {
    freq[tid] = count;
    off[tid] = base;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int f = tid + 1024 * i;
    if (e[i] >= 0) {
      const int pos = s_cnt[e[i]] + rank[i];
      s_rev[f] = pos;
      x_gather[pos] = tokens ? tokens[f] : f / K;
    }
  }
  if (tokens)
    for (int t = tid; t <= T; t += 1024) {  // first entry of token t (the list is sorted)
      int lo = 0, hi = n;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (tokens[mid] < t)
          lo = mid + 1;
        else
          hi = mid;
      }
      tok_off[t] = lo;
    }
}

// x rows in expert order with permuted columns: xs[pos][32 b + wd_place(k)] = x[token(pos)][32 b + k], zero
// beyond K.  Thread t of a quad reads columns 8 t .. + 7 of a block (4 pairs) and the quad transposes its
// 4 x 4 pairs, so that both sides move whole 64-byte blocks per quad.
__global__ void __launch_bounds__(256)
    wide_gather_kernel(const __nv_bfloat16* __restrict__ x, int T, int K, const int32_t* __restrict__ x_gather,
                       const int32_t* __restrict__ freq, const int32_t* __restrict__ off, int E, int blocks,
                       __nv_bfloat16* __restrict__ xs, int* err) {
  pdl_launch();
  pdl_wait();
  const int total = off[E - 1] + freq[E - 1];  // entries that were not rejected
  const int pos = blockIdx.x;
  if (pos >= total) return;
  const int tok = x_gather[pos];
  const bool ok = tok >= 0 && tok < T;
  if (!ok && threadIdx.x == 0) atomicCAS(err, 0, kErrBadToken);
  const int t = threadIdx.x & 3;
  for (int b0 = 0; b0 < blocks; b0 += 64) {  // whole quads stay together for the shuffles
    const int b = b0 + (threadIdx.x >> 2);
    const int k = 32 * b + 8 * t;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (ok && k < K) v = __ldg(reinterpret_cast<const uint4*>(x + static_cast<size_t>(tok) * K + k));
    // first swap the 2 x 2 blocks between t and t ^ 2, then within them between t and t ^ 1
    const bool hi = t & 2, odd = t & 1;
    const uint32_t s0 = __shfl_xor_sync(0xffffffffu, hi ? v.x : v.z, 2), s1 = __shfl_xor_sync(0xffffffffu, hi ? v.y : v.w, 2);
    if (hi) {
      v.x = s0;
      v.y = s1;
    } else {
      v.z = s0;
      v.w = s1;
    }
    const uint32_t r0 = __shfl_xor_sync(0xffffffffu, odd ? v.x : v.y, 1), r1 = __shfl_xor_sync(0xffffffffu, odd ? v.z : v.w, 1);
    if (odd) {
      v.x = r0;
      v.z = r1;
    } else {
      v.y = r0;
      v.w = r1;
    }
    if (b < blocks) *reinterpret_cast<uint4*>(xs + (static_cast<size_t>(pos) * blocks + b) * 32 + 8 * t) = v;
  }
}

// out[t] = sum over t's entries f, [t K, (t + 1) K) or [tok_off[t], tok_off[t + 1]), of scores[f] times
// the row y[s_rev[f]], in entry order, rounded once.  Entries whose expert was rejected have no row.  A
// warp's lanes look up 8 entries at a time, then all their rows are on the way together.
__global__ void __launch_bounds__(256)
    wide_combine_kernel(const float* __restrict__ y, int T, int H, int K, const int32_t* __restrict__ tok_off,
                        const int32_t* __restrict__ experts, const float* __restrict__ scores,
                        const int32_t* __restrict__ s_rev, int E, __nv_bfloat16* __restrict__ out) {
  pdl_wait();
  const int t = blockIdx.y, lane = threadIdx.x & 31;
  const int c = (blockIdx.x * blockDim.x + threadIdx.x) * 4;
  const int f0 = tok_off ? tok_off[t] : t * K, f1 = tok_off ? tok_off[t + 1] : (t + 1) * K;
  const float* col = y + (c < H ? c : 0);
  float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int f = f0; f < f1; f += 8) {
    int row = -1;
    float w = 0.0f;
    if (lane < 8 && f + lane < f1) {
      const int e = experts[f + lane];
      if (e >= 0 && e < E) row = s_rev[f + lane];
      w = scores[f + lane];
    }
    float4 v[8];
    float ws[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int r = __shfl_sync(0xffffffffu, row, k);
      ws[k] = __shfl_sync(0xffffffffu, w, k);
      v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (r >= 0)
        v[k] = __ldcs(reinterpret_cast<const float4*>(col + static_cast<size_t>(r) * H));
      else
        ws[k] = 0.0f;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      s.x = fmaf(ws[k], v[k].x, s.x);
      s.y = fmaf(ws[k], v[k].y, s.y);
      s.z = fmaf(ws[k], v[k].z, s.z);
      s.w = fmaf(ws[k], v[k].w, s.w);
    }
  }
  if (c < H)
    *reinterpret_cast<uint2*>(out + static_cast<size_t>(t) * H + c) =
        make_uint2(pack_bf16x2_rn(s.x, s.y), pack_bf16x2_rn(s.z, s.w));
}

template <bool kUp, int kN, int GPB>
cudaError_t launch_wide(const CUtensorMap& t16, const CUtensorMap& t64, const WdArgs& p, int grid, cudaStream_t st) {
  constexpr int kFixed = 1024 + WdShape<kN>::kStages * WdShape<kN>::kBStage + WdRing<GPB>::kBytes;
  constexpr int kMost = kFixed + 4097 * 4;  // set for every call alike: the limit is the whole process's
  static_assert(kMost <= 232448 - 1024, "shared memory budget");
  const int smem = kFixed + (p.E + 1) * 4;
  if (smem > kMost) return cudaErrorInvalidValue;
  auto kern = wide_kernel<kUp, kN, GPB>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
  if (e != cudaSuccess) return e;
  return launch_dependent(kern, dim3(grid), kWdThreads, smem, 1, st, t16, t64, p);
}

template <bool kUp, int kN>
cudaError_t launch_wide(WdArgs p, const void* x, int ld, int n_entries, int group, cudaStream_t st) {
  CUtensorMap t16, t64;
  const uint64_t inner = static_cast<uint64_t>(ld), rows = static_cast<uint64_t>(n_entries);
  if (!encode_tmap_2d(&t16, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, x, inner, rows, 64, 16, true) ||
      !encode_tmap_2d(&t64, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, x, inner, rows, 64, 64, true))
    return cudaErrorInvalidValue;
  const long long most = (n_entries / kN + static_cast<long long>(p.E < n_entries ? p.E : n_entries)) * p.m_tiles;
  const int sms = gemm_grid_sms();
  const int grid = most < sms ? static_cast<int>(most) : sms;
  return group == 32   ? launch_wide<kUp, kN, 4>(t16, t64, p, grid, st)
         : group == 64 ? launch_wide<kUp, kN, 2>(t16, t64, p, grid, st)
                       : launch_wide<kUp, kN, 1>(t16, t64, p, grid, st);
}

}  // namespace

int int4_padded(int K) { return int4_col_blocks(K) * 128; }

bool int4_plan_fits(int n_entries, int E) { return n_entries <= kPlanMaxEntries && E <= kPlanMaxExperts; }

cudaError_t launch_int4_plan(const int32_t* experts, const int32_t* tokens, int n, int T, int K, int E, int32_t* freq,
                             int32_t* off, int32_t* s_rev, int32_t* x_gather, int32_t* tok_off, int* err,
                             int* stop, cudaStream_t st) {
  auto kern = n <= 1024 ? wide_plan_kernel<1> : n <= 4096 ? wide_plan_kernel<4> : wide_plan_kernel<16>;
  kern<<<1, 1024, 0, st>>>(experts, tokens, n, T, K, E, freq, off, s_rev, x_gather, tok_off, err, stop);
  return cudaGetLastError();
}

cudaError_t launch_int4_wide(const Int4Args& p, cudaStream_t st) {
  const int blocks = int4_padded(p.H) / 32;
  cudaError_t e = launch_dependent(
      wide_gather_kernel, dim3(p.n_entries), 256, 0, 1, st, static_cast<const __nv_bfloat16*>(p.x), p.T, p.H,
      p.x_gather, p.freq, p.off, p.E, blocks, static_cast<__nv_bfloat16*>(p.xs), p.err);
  if (e != cudaSuccess) return e;
  WdArgs u{};
  u.wq = p.w1q;
  u.ws = static_cast<const __nv_bfloat16*>(p.w1s);
  u.N = 2 * p.I;
  u.n_tiles = int4_row_tiles(u.N);
  u.k_blocks = int4_col_blocks(p.H);
  u.E = p.E;
  u.m_tiles = int4_padded(p.I) / 128;  // 256 rows make 128 columns; the padding is written too (zeros)
  u.freq = p.freq;
  u.off = p.off;
  u.a = static_cast<__nv_bfloat16*>(p.a);
  u.a_ld = int4_padded(p.I);
  u.y = p.y;
  u.stop = p.stop;
  u.err = p.err;
  WdArgs d = u;
  d.wq = p.w2q;
  d.ws = static_cast<const __nv_bfloat16*>(p.w2s);
  d.N = p.H;
  d.n_tiles = int4_row_tiles(d.N);
  d.k_blocks = int4_col_blocks(p.I);
  d.m_tiles = ceil_div(d.N, 256);
  // Items of 128 tokens once the experts have 32 on average.  4096 x 1024, 128 experts, us with 128 / 64: 512
  // tokens even 280 / 278, Zipf 292 / 314; 1024 tokens 327 / 400 and 373 / 418; 256 tokens 245 / 246 and 259 /
  // 267.  2048 x 768: 512 tokens 138 / 135 and 139 / 145, 256 tokens 120 / 122 and 122 / 121.  A layer with
  // fewer items than SMs loses its share of them (40 experts of 1000 x 408, 512 tokens: 45 / 43).
  const bool many = p.n_entries >= 32 * p.E;
  e = many ? launch_wide<true, 128>(u, p.xs, int4_padded(p.H), p.n_entries, p.group1, st)
           : launch_wide<true, 64>(u, p.xs, int4_padded(p.H), p.n_entries, p.group1, st);
  if (e != cudaSuccess) return e;
  e = many ? launch_wide<false, 128>(d, p.a, u.a_ld, p.n_entries, p.group2, st)
           : launch_wide<false, 64>(d, p.a, u.a_ld, p.n_entries, p.group2, st);
  if (e != cudaSuccess) return e;
  for (int t0 = 0; t0 < p.T; t0 += 32768) {  // grid.y limit
    const int n = p.T - t0 < 32768 ? p.T - t0 : 32768;
    const size_t f0 = p.tok_off ? 0 : static_cast<size_t>(t0) * p.K;
    e = launch_dependent(
        wide_combine_kernel, dim3(ceil_div(p.H, 1024), n), 256, 0, 1, st, p.y, n, p.H, p.K,
        p.tok_off ? p.tok_off + t0 : nullptr, p.experts + f0, p.scores + f0, p.s_rev + f0, p.E,
        static_cast<__nv_bfloat16*>(p.out) + static_cast<size_t>(t0) * p.H);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace smb
