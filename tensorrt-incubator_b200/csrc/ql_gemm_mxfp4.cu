// Block-scaled MXFP4 product on the 5th-generation tensor cores (sm_100a only):
//     Y[m,n] = sum over blocks b of 2^(ea[m,b] + eb[n,b]) * sum over k in b of qa[m,k] qb[n,k]
// with qa, qb in e2m1 and the e8m0 block scales of quantize_mxfp4 (blocks of 32 along K).  The tensor core applies the
// scales itself (tcgen05.mma kind::mxf4.block_scale, scales read from tensor memory) and accumulates in f32; the result is
// rounded once.  One MMA consumes 64 values of K, two blocks, so a 32-bit cell of tensor memory holds the scales of two
// MMAs; which half an MMA uses is a field of its instruction descriptor.
//
// The tensor core wants the scales of 128 rows as 4 columns of 32 lanes (row r in lane r % 32, column r / 32), repeated in
// all four lane quarters of tensor memory.  The operands' scales are row-major, a row's bytes in a line.  The NVFP4 kernel
// re-orders them in a kernel of its own and copies them from shared to tensor memory with tcgen05.cp, one 32-bit cell a
// cycle and quarter, which is what bounds it.  Here four warps (one per quarter) take the bytes of "their" rows into
// registers in the layout they already need -- lane l holds rows l, l + 32, ... -- and store them with tcgen05.st, 32 lanes
// a cycle: no re-ordering pass and no copy instructions between the MMAs.
//
// Two kernels:
//   split   few output tiles (decoding, short prompts): the weights are the 128-row operand and up to 128 tokens the other;
//           a cluster of up to 8 CTAs shares the K axis of one tile and adds its parts through distributed shared memory,
//           in rank order (the same bits on every run).
//   tiles   many output tiles: one persistent CTA per SM on 128 x 224 tiles.
// Every wait is bounded, as in the other tensor-core kernels.
#include <cuda.h>
#include <string.h>

#include "ql_common.cuh"
#include "ql_tc_common.cuh"

namespace ql {
namespace {

constexpr int kKStep = 256;           // values of K per pipeline stage: 128 bytes of e2m1
constexpr int kScaleBytes = 8;        // scales of one row and k step
constexpr int MX_A_BYTES = BM * BK_BYTES;

struct MxArgs {
  void *Y;
  const uint8_t *sfa, *sfb; // row-major scales of the 128-row operand and of the other one
  int y_dtype;
  int M, N;                 // rows of Y (tokens), columns of Y
  int kb;                   // blocks (scale bytes) per row
  int num_ks;
  int tiles_a, tiles_b;     // tiles over the 128-row operand's rows and over the other's
  int *status;
};

__device__ __forceinline__ void mx_mma(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.block32 [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
               ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
               : "memory");
}
// e2m1 operands (format 1), both K-major, e8m0 scales (bit 23), N >> 3 at bit 17, M >> 4 at bit 24, dense K = 64; the byte
// offset (0 or 2) of the scales within their cells at bits 29 (A) and 4 (B)
template <int N> __device__ __forceinline__ uint32_t mx_idesc(uint32_t byte) {
  return 1u << 7 | 1u << 10 | (uint32_t)(N >> 3) << 17 | 1u << 23 | (uint32_t)(BM >> 4) << 24 | byte << 29 | byte << 4;
}
__device__ __forceinline__ void tmem_store_4(uint32_t taddr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// A warp's wait with one answer for all lanes: what follows is executed by the whole warp or by none of it.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag, int *status, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, code));
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// the four MMAs of one k step
template <int N>
__device__ __forceinline__ void mx_k_step(uint32_t tmem_d, uint32_t a_addr, uint32_t b_addr, uint32_t t_sfa, uint32_t t_sfb, int sfb_cols, bool first) {
  const uint64_t adesc = make_smem_desc(a_addr), bdesc = make_smem_desc(b_addr);
#pragma unroll
  for (int j = 0; j < 4; j++) // 64 values = 32 bytes of K each; two MMAs share one set of scale cells
    mx_mma(tmem_d, adesc + 2 * j, bdesc + 2 * j, mx_idesc<N>((j & 1) * 2), t_sfa + 4 * (j >> 1), t_sfb + sfb_cols * (j >> 1), (first && j == 0) ? 0u : 1u);
}

template <typename OutT> __device__ __forceinline__ void store_y(void *Y, size_t i, float v) { static_cast<OutT *>(Y)[i] = FloatIO<OutT>::from_f32(v); }
__device__ __forceinline__ void store_y(void *Y, int dtype, size_t i, float v) {
  if (dtype == QL_F32) store_y<float>(Y, i, v);
  else if (dtype == QL_F16) store_y<__half>(Y, i, v);
  else store_y<__nv_bfloat16>(Y, i, v);
}

// The 8 scale bytes of one row and k step (zeros beyond the row's end and beyond the operand).
__device__ __forceinline__ uint2 load_row_scales(const uint8_t *sf, int row, int rows, int kb, int ks, int vec) {
  uint2 v = make_uint2(0u, 0u);
  if (row >= rows) return v;
  const int b0 = ks * kScaleBytes;
  const uint8_t *p = sf + (size_t)row * kb + b0;
  if (vec == 8) return __ldg(reinterpret_cast<const uint2 *>(p));
  if (vec == 4) {
    v.x = __ldg(reinterpret_cast<const uint32_t *>(p));
    if (b0 + 4 < kb) v.y = __ldg(reinterpret_cast<const uint32_t *>(p) + 1);
    return v;
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if (b0 + i < kb) v.x |= (uint32_t)__ldg(p + i) << (8 * i);
    if (b0 + 4 + i < kb) v.y |= (uint32_t)__ldg(p + 4 + i) << (8 * i);
  }
  return v;
}

// ------------------------------------------------------------------------------------------------------------------
// split kernel: 128 rows of the weights x TN tokens, K over the CTAs of a cluster
// ------------------------------------------------------------------------------------------------------------------
constexpr int kSplitThreads = 192;
constexpr int kMaxSplit = 8;

template <int TN> struct SplitSmem {
  static constexpr int kStages = 4;
  static constexpr int kStageBytes = MX_A_BYTES + TN * BK_BYTES;
  static constexpr int kTiles = kStages * kStageBytes;
  static_assert(TN * BM * 4 <= kTiles && kStageBytes % 1024 == 0, "the partial sums reuse the ring");
  static constexpr int kBarriers = kTiles; // full[S], empty[S], sfull[2], sempty[2], tfull
  static constexpr int kTmemPtr = kBarriers + (2 * kStages + 5) * 8;
  static constexpr int kAbort = kTmemPtr + 4;
  static constexpr int kDynamic = kAbort + 4 + 1024;
};

template <int TN>
__global__ void __launch_bounds__(kSplitThreads)
gemm_mxfp4_split_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const MxArgs args, int split, int vec_a, int vec_b) {
  using L = SplitSmem<TN>;
  constexpr int ST = L::kStages;
  constexpr uint32_t kSfCol0 = TN;                         // two slots of 16 columns: 8 of the weights' scales, 8 of the tokens'
  constexpr uint32_t kTmemCols = TN + 32 <= 64 ? 64 : (TN + 32 <= 128 ? 128 : 256);
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t smem_base = smem_u32(smem), bar_base = smem_base + L::kBarriers;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (ST + s); };
  auto sfull_bar = [&](int s) { return bar_base + 8u * (2 * ST + s); };
  auto sempty_bar = [&](int s) { return bar_base + 8u * (2 * ST + 2 + s); };
  const uint32_t tfull_bar = bar_base + 8u * (2 * ST + 4);
  volatile uint32_t *tmem_ptr_smem = reinterpret_cast<volatile uint32_t *>(smem + L::kTmemPtr);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::kAbort);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % split, tile = blockIdx.x / split;
  const int wt = tile % args.tiles_a, xt = tile / args.tiles_a;
  const int ks0 = (int)((long long)args.num_ks * rank / split), ks1 = (int)((long long)args.num_ks * (rank + 1) / split);

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; s++) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int s = 0; s < 2; s++) {
      mbar_init(sfull_bar(s), 4);
      mbar_init(sempty_bar(s), 1);
    }
    mbar_init(tfull_bar, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void *)tmem_ptr_smem)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_ptr_smem;

  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int issued = 0;
      bool ok = true;
      for (int ks = ks0; ks < ks1; ks++) {
        if (!mbar_wait(empty_bar(stage), phase ^ 1, abort_flag, args.status, ST_TIMEOUT_EMPTY)) { ok = false; break; }
        const uint32_t a_dst = smem_base + stage * L::kStageBytes;
        mbar_expect_tx(full_bar(stage), L::kStageBytes);
        tma_load_2d(a_dst, &map_w, full_bar(stage), ks * BK_BYTES, wt * BM); // coordinates in bytes of packed e2m1
        tma_load_2d(a_dst + MX_A_BYTES, &map_x, full_bar(stage), ks * BK_BYTES, xt * TN);
        issued++;
        if (++stage == ST) { stage = 0; phase ^= 1; }
      }
      if (!ok) { // let the loads in flight land before the shared memory goes away
        const int pending = issued < ST ? issued : ST;
        for (int i = 0; i < pending; i++) {
          stage = (stage == 0) ? ST - 1 : stage - 1;
          if (stage == ST - 1) phase ^= 1;
          const long long t0 = clock64();
          while (!mbar_try_wait(full_bar(stage), phase) && clock64() - t0 < kWaitLimitCycles) {}
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issue
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int ks = ks0; ks < ks1; ks++) {
        const int it = ks - ks0, slot = it & 1;
        if (!mbar_wait(full_bar(stage), phase, abort_flag, args.status, ST_TIMEOUT_FULL)) break;
        if (!mbar_wait(sfull_bar(slot), (it >> 1) & 1, abort_flag, args.status, ST_TIMEOUT_FULL)) break;
        tc_fence_after();
        const uint32_t a_addr = smem_base + stage * L::kStageBytes, t_sf = tmem_base + kSfCol0 + 16 * slot;
        mx_k_step<TN>(tmem_base, a_addr, a_addr + MX_A_BYTES, t_sf, t_sf + 8, 4, it == 0);
        tc_commit(empty_bar(stage));
        tc_commit(sempty_bar(slot));
        if (++stage == ST) { stage = 0; phase ^= 1; }
      }
      tc_commit(tfull_bar);
      // every MMA issued above is done with shared and tensor memory before this thread goes on, after an abort too
      const long long t0 = clock64();
      while (!mbar_try_wait(tfull_bar, 0)) {
        if (clock64() - t0 > kWaitLimitCycles) { atomicCAS(args.status, 0, ST_TIMEOUT_DRAIN); break; }
      }
    }
  } else {
    // ------------------------------------------------------------------ scales, then the accumulator (warps 2..5)
    const int quad = warp & 3;
    const uint32_t quarter = (uint32_t)(quad * 32) << 16;
    constexpr int XR = TN <= 32 ? 1 : TN / 32; // rows of the token operand a lane carries
    uint2 a[4], b[XR];
    auto fetch = [&](int ks) {
#pragma unroll
      for (int c = 0; c < 4; c++) a[c] = load_row_scales(args.sfa, wt * BM + c * 32 + lane, args.N, args.kb, ks, vec_a);
#pragma unroll
      for (int c = 0; c < XR; c++) {
        const int r = c * 32 + lane;
        b[c] = r < TN ? load_row_scales(args.sfb, xt * TN + r, args.M, args.kb, ks, vec_b) : make_uint2(0u, 0u);
      }
    };
    if (ks0 < ks1) fetch(ks0);
    for (int ks = ks0; ks < ks1; ks++) {
      const int it = ks - ks0, slot = it & 1;
      uint2 pa[4], pb[4];
#pragma unroll
      for (int c = 0; c < 4; c++) {
        pa[c] = a[c];
        pb[c] = c < XR ? b[c < XR ? c : 0] : make_uint2(0u, 0u);
      }
      if (ks + 1 < ks1) fetch(ks + 1); // in flight while this step's slot is waited for
      if (!warp_wait(sempty_bar(slot), ((it >> 1) & 1) ^ 1, abort_flag, args.status, ST_TIMEOUT_EMPTY)) break;
      const uint32_t t = tmem_base + quarter + kSfCol0 + 16 * slot;
      tmem_store_4(t, pa[0].x, pa[1].x, pa[2].x, pa[3].x);
      tmem_store_4(t + 4, pa[0].y, pa[1].y, pa[2].y, pa[3].y);
      tmem_store_4(t + 8, pb[0].x, pb[1].x, pb[2].x, pb[3].x);
      tmem_store_4(t + 12, pb[0].y, pb[1].y, pb[2].y, pb[3].y);
      tmem_store_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(sfull_bar(slot));
    }
    warp_wait(tfull_bar, 0, abort_flag, args.status, ST_TIMEOUT_TMEM_FULL);
    tc_fence_after();
    // lane = row of the weights = column of Y, so a warp's store of one token is contiguous
    const int n = wt * BM + quad * 32 + lane;
    float *part = reinterpret_cast<float *>(smem); // [TN][128]: the ring is free once the MMAs are done
#pragma unroll 1
    for (int c = 0; c < TN / 16; c++) {
      uint32_t r[16];
      tmem_load_16(tmem_base + quarter + c * 16, r);
      if (split > 1) {
#pragma unroll
        for (int j = 0; j < 16; j++) part[(c * 16 + j) * BM + quad * 32 + lane] = __uint_as_float(r[j]);
      } else if (n < args.N) {
        const int m = xt * TN + c * 16;
#pragma unroll
        for (int j = 0; j < 16; j++)
          if (m + j < args.M) store_y(args.Y, args.y_dtype, (size_t)(m + j) * args.N + n, __uint_as_float(r[j]));
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (split > 1) {
    cluster_sync_all(); // every CTA's partial sums are in its shared memory
    const int t0 = TN * rank / split, t1 = TN * (rank + 1) / split;
    for (int i = threadIdx.x; i < (t1 - t0) * BM; i += kSplitThreads) {
      const int t = t0 + i / BM, row = i % BM;
      const int m = xt * TN + t, n = wt * BM + row;
      if (m >= args.M || n >= args.N) continue;
      const uint32_t local = smem_base + (uint32_t)(t * BM + row) * 4u;
      float p[kMaxSplit], v = 0.f;
#pragma unroll
      for (int s = 0; s < kMaxSplit; s++)
        if (s < split) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(p[s]) : "r"(map_to_cta(local, (uint32_t)s)));
#pragma unroll
      for (int s = 0; s < kMaxSplit; s++)
        if (s < split) v += p[s];
      store_y(args.Y, args.y_dtype, (size_t)m * args.N + n, v);
    }
    cluster_sync_all(); // a CTA's shared memory stays until its partners have read it
  }
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
  }
}

// ------------------------------------------------------------------------------------------------------------------
// tiles kernel: persistent, 128 x 224
// ------------------------------------------------------------------------------------------------------------------
constexpr int TBN = 224;            // widest tile whose two accumulators leave room for two slots of scales
constexpr int kTileThreads = 320;   // producer, MMA, four epilogue warps, four scale warps
constexpr int TSTAGES = 4;
constexpr int T_STAGE_BYTES = MX_A_BYTES + TBN * BK_BYTES;
constexpr int kScSteps = 4;         // k steps whose scales travel together: 32 bytes, a whole sector, of every row
constexpr int T_SC_ROWS = BM + TBN;
constexpr int T_SC_BYTES = T_SC_ROWS * 32;
struct TileSmem {
  static constexpr int kScales = TSTAGES * T_STAGE_BYTES;
  static constexpr int kBarriers = kScales + 2 * T_SC_BYTES; // full[S], empty[S], tfull[2], tempty[2], scfull[2], scempty[2], sfull[2], sempty[2], drain
  static constexpr int kTmemPtr = kBarriers + (2 * TSTAGES + 13) * 8;
  static constexpr int kAbort = kTmemPtr + 4;
  static constexpr int kDynamic = kAbort + 4 + 1024;
};
static_assert(TileSmem::kDynamic <= 232448 && T_STAGE_BYTES % 1024 == 0 && T_SC_BYTES % 128 == 0, "tile shape");

// 32 columns of one accumulator row, rounded to y's type and stored
template <typename OutT>
__device__ __forceinline__ void mx_store_chunk(OutT *Y, const uint32_t (&r)[32], int m, int n, int N, bool vec) {
  OutT *y = Y + (size_t)m * (size_t)N + n;
  if (vec && n + 32 <= N) {
    if constexpr (sizeof(OutT) == 4) {
#pragma unroll
      for (int j = 0; j < 32; j += 4) __stcs(reinterpret_cast<uint4 *>(y + j), make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]));
    } else {
      auto two = [&](int j) { return pack2<OutT>(__uint_as_float(r[j]), __uint_as_float(r[j + 1])); };
#pragma unroll
      for (int j = 0; j < 32; j += 8) __stcs(reinterpret_cast<uint4 *>(y + j), make_uint4(two(j), two(j + 2), two(j + 4), two(j + 6)));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; j++)
      if (n + j < N) y[j] = FloatIO<OutT>::from_f32(__uint_as_float(r[j]));
  }
}

__global__ void __launch_bounds__(kTileThreads, 1)
gemm_mxfp4_tiles_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_sa,
                        const __grid_constant__ CUtensorMap map_sb, const MxArgs args) {
  using L = TileSmem;
  constexpr uint32_t kTmemCols = 512; // 2 x 224 accumulator columns, then two slots of 32: 8 columns of A's scales, 16 of B's
  constexpr uint32_t kSfCol0 = 2 * TBN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t smem_base = smem_u32(smem), bar_base = smem_base + L::kBarriers;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (TSTAGES + s); };
  auto tfull_bar = [&](int b) { return bar_base + 8u * (2 * TSTAGES + b); };
  auto tempty_bar = [&](int b) { return bar_base + 8u * (2 * TSTAGES + 2 + b); };
  auto scfull_bar = [&](int b) { return bar_base + 8u * (2 * TSTAGES + 4 + b); };
  auto scempty_bar = [&](int b) { return bar_base + 8u * (2 * TSTAGES + 6 + b); };
  auto sfull_bar = [&](int b) { return bar_base + 8u * (2 * TSTAGES + 8 + b); };
  auto sempty_bar = [&](int b) { return bar_base + 8u * (2 * TSTAGES + 10 + b); };
  const uint32_t drain_bar = bar_base + 8u * (2 * TSTAGES + 12);
  volatile uint32_t *tmem_ptr_smem = reinterpret_cast<volatile uint32_t *>(smem + L::kTmemPtr);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::kAbort);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int num_tiles = args.tiles_a * args.tiles_b;

  if (threadIdx.x == 0) {
    for (int s = 0; s < TSTAGES; s++) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; b++) {
      mbar_init(tfull_bar(b), 1);
      mbar_init(tempty_bar(b), 4);
      mbar_init(scfull_bar(b), 1);
      mbar_init(scempty_bar(b), 4);
      mbar_init(sfull_bar(b), 4);
      mbar_init(sempty_bar(b), 1);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void *)tmem_ptr_smem)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_ptr_smem;

  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    if (lane == 0) {
      int stage = 0, sc = 0;
      uint32_t phase = 0, sc_phase = 0;
      long long issued = 0, sc_issued = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x) {
        const int mt = tile % args.tiles_a, nt = tile / args.tiles_a; // row tiles of one column tile run side by side: B stays in L2
        for (int ks = 0; ks < args.num_ks; ks++) {
          if (ks % kScSteps == 0) {
            if (!mbar_wait(scempty_bar(sc), sc_phase ^ 1, abort_flag, args.status, ST_TIMEOUT_EMPTY)) { ok = false; break; }
            const uint32_t dst = smem_base + L::kScales + sc * T_SC_BYTES;
            mbar_expect_tx(scfull_bar(sc), T_SC_BYTES);
            tma_load_2d(dst, &map_sa, scfull_bar(sc), ks * kScaleBytes, mt * BM);
            tma_load_2d(dst + BM * 32, &map_sb, scfull_bar(sc), ks * kScaleBytes, nt * TBN);
            sc_issued++;
            if (++sc == 2) { sc = 0; sc_phase ^= 1; }
          }
          if (!mbar_wait(empty_bar(stage), phase ^ 1, abort_flag, args.status, ST_TIMEOUT_EMPTY)) { ok = false; break; }
          const uint32_t a_dst = smem_base + stage * T_STAGE_BYTES;
          mbar_expect_tx(full_bar(stage), T_STAGE_BYTES);
          tma_load_2d(a_dst, &map_a, full_bar(stage), ks * BK_BYTES, mt * BM); // coordinates in bytes of packed e2m1
          tma_load_2d(a_dst + MX_A_BYTES, &map_b, full_bar(stage), ks * BK_BYTES, nt * TBN);
          issued++;
          if (++stage == TSTAGES) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok) { // let the loads in flight land before the shared memory goes away
        const long long pending = issued < TSTAGES ? issued : TSTAGES, sc_pending = sc_issued < 2 ? sc_issued : 2;
        for (long long i = 0; i < pending; i++) {
          stage = (stage == 0) ? TSTAGES - 1 : stage - 1;
          if (stage == TSTAGES - 1) phase ^= 1;
          const long long t0 = clock64();
          while (!mbar_try_wait(full_bar(stage), phase) && clock64() - t0 < kWaitLimitCycles) {}
        }
        for (long long i = 0; i < sc_pending; i++) {
          sc ^= 1;
          if (sc == 1) sc_phase ^= 1;
          const long long t0 = clock64();
          while (!mbar_try_wait(scfull_bar(sc), sc_phase) && clock64() - t0 < kWaitLimitCycles) {}
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issue
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int it = 0;
      long long step = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x, it++) {
        const int buf = it & 1;
        if (!mbar_wait(tempty_bar(buf), ((it >> 1) & 1) ^ 1, abort_flag, args.status, ST_TIMEOUT_TMEM_EMPTY)) { ok = false; break; }
        for (int ks = 0; ks < args.num_ks; ks++, step++) {
          const int slot = (int)(step & 1);
          if (!mbar_wait(full_bar(stage), phase, abort_flag, args.status, ST_TIMEOUT_FULL)) { ok = false; break; }
          if (!mbar_wait(sfull_bar(slot), (uint32_t)((step >> 1) & 1), abort_flag, args.status, ST_TIMEOUT_FULL)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a_addr = smem_base + stage * T_STAGE_BYTES, t_sf = tmem_base + kSfCol0 + 32 * slot;
          mx_k_step<TBN>(tmem_base + (uint32_t)(buf * TBN), a_addr, a_addr + MX_A_BYTES, t_sf, t_sf + 8, 8, ks == 0);
          tc_commit(empty_bar(stage));
          tc_commit(sempty_bar(slot));
          if (++stage == TSTAGES) { stage = 0; phase ^= 1; }
        }
        if (ok) tc_commit(tfull_bar(buf));
      }
      tc_commit(drain_bar); // every MMA issued above has to finish before tensor memory is released
      const long long t0 = clock64();
      while (!mbar_try_wait(drain_bar, 0)) {
        if (clock64() - t0 > kWaitLimitCycles) { atomicCAS(args.status, 0, ST_TIMEOUT_DRAIN); break; }
      }
    }
  } else if (warp >= 6) {
    // ------------------------------------------------------------------ scales (warps 6..9, one per quarter of the lanes)
    const uint32_t quarter = (uint32_t)((warp & 3) * 32) << 16;
    int sc = 0;
    uint32_t sc_phase = 0;
    long long step = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x) {
      for (int ks = 0; ks < args.num_ks && ok; ks += kScSteps) {
        if (!warp_wait(scfull_bar(sc), sc_phase, abort_flag, args.status, ST_TIMEOUT_FULL)) { ok = false; break; }
        uint32_t w[T_SC_ROWS / 32][8]; // rows lane, lane + 32, ... : the words of four k steps
        const uint8_t *src = smem + L::kScales + sc * T_SC_BYTES + lane * 32;
#pragma unroll
        for (int c = 0; c < T_SC_ROWS / 32; c++) {
          const uint4 lo = *reinterpret_cast<const uint4 *>(src + c * 1024), hi = *reinterpret_cast<const uint4 *>(src + c * 1024 + 16);
          w[c][0] = lo.x, w[c][1] = lo.y, w[c][2] = lo.z, w[c][3] = lo.w;
          w[c][4] = hi.x, w[c][5] = hi.y, w[c][6] = hi.z, w[c][7] = hi.w;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(scempty_bar(sc));
        if (++sc == 2) { sc = 0; sc_phase ^= 1; }
#pragma unroll
        for (int q = 0; q < kScSteps; q++) {
          if (ok && ks + q < args.num_ks) {
            const int slot = (int)(step & 1);
            if (!warp_wait(sempty_bar(slot), (uint32_t)((step >> 1) & 1) ^ 1u, abort_flag, args.status, ST_TIMEOUT_EMPTY)) ok = false;
            if (ok) {
              const uint32_t t = tmem_base + quarter + kSfCol0 + 32 * slot;
#pragma unroll
              for (int j = 0; j < 2; j++) { // two MMAs' worth of cells: A's rows, B's first 128 rows, B's last 96
                tmem_store_4(t + 4 * j, w[0][2 * q + j], w[1][2 * q + j], w[2][2 * q + j], w[3][2 * q + j]);
                tmem_store_4(t + 8 + 8 * j, w[4][2 * q + j], w[5][2 * q + j], w[6][2 * q + j], w[7][2 * q + j]);
                tmem_store_4(t + 12 + 8 * j, w[8][2 * q + j], w[9][2 * q + j], w[10][2 * q + j], 0u);
              }
              tmem_store_wait();
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(sfull_bar(slot));
              step++;
            }
          }
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ epilogue (warps 2..5)
    const int quad = warp & 3;
    const bool vec = (reinterpret_cast<uintptr_t>(args.Y) & 15) == 0 && args.N % (args.y_dtype == QL_F32 ? 4 : 8) == 0;
    int it = 0;
    for (int tile = blockIdx.x; tile < num_tiles; tile += gridDim.x, it++) {
      const int buf = it & 1;
      const int mt = tile % args.tiles_a, nt = tile / args.tiles_a;
      if (!warp_wait(tfull_bar(buf), (it >> 1) & 1, abort_flag, args.status, ST_TIMEOUT_TMEM_FULL)) break;
      tc_fence_after();
      const int m = mt * BM + quad * 32 + lane;
      const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(buf * TBN);
#pragma unroll 1
      for (int c = 0; c < TBN / 32; c++) {
        uint32_t r[32];
        tmem_load_32(taddr + c * 32, r);
        const int n = nt * TBN + c * 32;
        if (m < args.M && n < args.N) {
          if (args.y_dtype == QL_F32) mx_store_chunk(static_cast<float *>(args.Y), r, m, n, args.N, vec);
          else if (args.y_dtype == QL_F16) mx_store_chunk(static_cast<__half *>(args.Y), r, m, n, args.N, vec);
          else mx_store_chunk(static_cast<__nv_bfloat16 *>(args.Y), r, m, n, args.N, vec);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(tempty_bar(buf));
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
  }
}

// Row-major scales with rows padded to `pitch` bytes (zeros), so that the copy engine can address them: both operands.
__global__ void __launch_bounds__(256) mx_pad_scales_kernel(const uint8_t *__restrict__ a, int64_t rows_a, const uint8_t *__restrict__ b, int64_t rows_b, int kb, int pitch,
                                                            uint32_t *__restrict__ out) {
  const int64_t words = (rows_a + rows_b) * (pitch / 4);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / (pitch / 4);
    const int b0 = (int)(i % (pitch / 4)) * 4;
    const uint8_t *p = row < rows_a ? a + row * kb : b + (row - rows_a) * kb;
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (b0 + j < kb) w |= (uint32_t)p[b0 + j] << (8 * j);
    out[i] = w;
  }
}

int check_mx_operand(const char *op, const char *name, const ql_tensor *d, const ql_tensor *s) {
  if (!d || !s) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: %s is null", op, name);
  if (d->dtype != QL_F4E2M1 || s->dtype != QL_F8E8M0) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: %s: data must be f4E2M1FN and scales f8E8M0FNU", op, name);
  if (d->rank != 2 || s->rank != 2) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: %s: data and scales must be 2-D", op, name);
  if (d->shape[0] < 0 || d->shape[1] < 0) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: %s: negative dimension", op, name);
  if (d->shape[1] % 32 != 0 || s->shape[0] != d->shape[0] || s->shape[1] != d->shape[1] / 32)
    return set_error(QL_ERR_INVALID_ARGUMENT, "%s: %s: scales must hold one entry per block of 32 along the last dimension", op, name);
  if (numel(d) > 0 && (!d->data || !s->data)) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: %s has no data pointer", op, name);
  return QL_OK;
}

template <typename K> int allow_smem(K kern, int bytes, bool (&configured)[64]) {
  int dev = 0;
  QL_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    QL_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  return QL_OK;
}

int scale_vec(const uint8_t *p, int kb) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p) | (uintptr_t)kb;
  return a % 8 == 0 ? 8 : (a % 4 == 0 ? 4 : 1);
}

// args: the weights are operand a here
template <int TN> int launch_split(const void *w, const void *x, MxArgs args, int64_t K, cudaStream_t st) {
  using L = SplitSmem<TN>;
  static bool configured[64] = {false};
  int rc = allow_smem(gemm_mxfp4_split_kernel<TN>, L::kDynamic, configured);
  if (rc != QL_OK) return rc;
  CUtensorMap mw, mx;
  if ((rc = make_map(&mw, KIND_F8, w, args.N, K / 2, BM)) != QL_OK) return rc;
  if ((rc = make_map(&mx, KIND_F8, x, args.M, K / 2, TN)) != QL_OK) return rc;
  args.tiles_a = (args.N + BM - 1) / BM;
  args.tiles_b = (args.M + TN - 1) / TN;
  const int64_t tiles = (int64_t)args.tiles_a * args.tiles_b;
  // K is shared by more CTAs while the machine is not full and every CTA keeps two k steps
  int split = 1;
  while (split < kMaxSplit && tiles * split < 2ll * sm_count() && args.num_ks / (2 * split) >= 2) split *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * split), 1, 1);
  cfg.blockDim = dim3(kSplitThreads, 1, 1);
  cfg.dynamicSmemBytes = L::kDynamic;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)split, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  QL_CUDA_TRY(cudaLaunchKernelEx(&cfg, gemm_mxfp4_split_kernel<TN>, mw, mx, args, split, scale_vec(args.sfa, args.kb), scale_vec(args.sfb, args.kb)));
  count_launches(1);
  return QL_OK;
}

int launch_tiles(const void *a, const void *b, MxArgs args, int64_t K, cudaStream_t st) {
  static bool configured[64] = {false};
  int rc = allow_smem(gemm_mxfp4_tiles_kernel, TileSmem::kDynamic, configured);
  if (rc != QL_OK) return rc;
  CUtensorMap ma, mb, msa, msb;
  if ((rc = make_map(&ma, KIND_F8, a, args.M, K / 2, BM)) != QL_OK) return rc;
  if ((rc = make_map(&mb, KIND_F8, b, args.N, K / 2, TBN)) != QL_OK) return rc;
  // the copy engine takes rows of whole 16-byte units from a 16-byte aligned base; other scales are padded first
  uint8_t *scratch = nullptr;
  int pitch = args.kb;
  if (args.kb % 16 != 0 || !aligned16(args.sfa) || !aligned16(args.sfb)) {
    pitch = (args.kb + 15) / 16 * 16;
    keep_scratch_pool_warm();
    QL_CUDA_TRY(cudaMallocAsync(&scratch, (size_t)((int64_t)args.M + args.N) * pitch, st));
    const int64_t words = ((int64_t)args.M + args.N) * (pitch / 4), blocks = (words + 255) / 256, cap = (int64_t)sm_count() * 16;
    mx_pad_scales_kernel<<<(unsigned)(blocks < cap ? blocks : cap), 256, 0, st>>>(args.sfa, args.M, args.sfb, args.N, args.kb, pitch, reinterpret_cast<uint32_t *>(scratch));
    count_launches(1);
    args.sfa = scratch;
    args.sfb = scratch + (int64_t)args.M * pitch;
  }
  if ((rc = make_map_bytes(&msa, args.sfa, args.M, pitch, 32, BM)) == QL_OK && (rc = make_map_bytes(&msb, args.sfb, args.N, pitch, 32, TBN)) == QL_OK) {
    args.tiles_a = (args.M + BM - 1) / BM;
    args.tiles_b = (args.N + TBN - 1) / TBN;
    const int64_t tiles = (int64_t)args.tiles_a * args.tiles_b;
    gemm_mxfp4_tiles_kernel<<<(unsigned)(tiles < sm_count() ? tiles : sm_count()), kTileThreads, TileSmem::kDynamic, st>>>(ma, mb, msa, msb, args);
    count_launches(1);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) rc = cuda_error(e, "gemm_mxfp4_tiles_kernel");
  }
  if (scratch) {
    const cudaError_t e = cudaFreeAsync(scratch, st);
    if (rc == QL_OK && e != cudaSuccess) return cuda_error(e, "cudaFreeAsync");
  }
  return rc;
}

} // namespace
} // namespace ql

using namespace ql;

extern "C" int ql_gemm_mxfp4(const ql_tensor *a, const ql_tensor *a_scales, const ql_tensor *b, const ql_tensor *b_scales, ql_tensor *y, void *stream) {
  const char *op = "gemm_mxfp4";
  int rc;
  if ((rc = check_mx_operand(op, "a", a, a_scales)) != QL_OK) return rc;
  if ((rc = check_mx_operand(op, "b", b, b_scales)) != QL_OK) return rc;
  if (!y || y->rank != 2 || !is_float_dtype(y->dtype)) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: y must be a 2-D f32, f16 or bf16 tensor", op);
  const int64_t M = a->shape[0], K = a->shape[1], N = b->shape[0];
  if (b->shape[1] != K) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: inner dimensions differ (%lld vs %lld)", op, (long long)K, (long long)b->shape[1]);
  if (y->shape[0] != M || y->shape[1] != N) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: y must be [M,N] = [%lld,%lld]", op, (long long)M, (long long)N);
  if (M == 0 || N == 0) return QL_OK;
  if (!y->data) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: y has no data pointer", op);
  if (K == 0) return set_error(QL_ERR_UNSUPPORTED, "%s: needs a non-zero K", op);
  if (!aligned16(a->data) || !aligned16(b->data)) return set_error(QL_ERR_UNSUPPORTED, "%s: needs 16-byte aligned operands", op);
  if (reinterpret_cast<uintptr_t>(y->data) % (y->dtype == QL_F32 ? 4 : 2)) return set_error(QL_ERR_UNSUPPORTED, "%s: y is not aligned to its type", op);
  if (M > (1 << 30) || N > (1 << 30) || K > (1 << 30)) return set_error(QL_ERR_UNSUPPORTED, "%s: dimension too large", op);
  cudaStream_t st = (cudaStream_t)stream;

  MxArgs args;
  args.Y = y->data;
  args.y_dtype = y->dtype;
  args.M = (int)M;
  args.N = (int)N;
  args.kb = (int)(K / 32);
  args.num_ks = (int)((K + kKStep - 1) / kKStep);
  args.tiles_a = args.tiles_b = 0;
  args.status = device_status_word();
  if (!args.status) return set_error(QL_ERR_CUDA, "%s: could not allocate the device status word", op);
  const int64_t tiles = ((M + BM - 1) / BM) * ((N + TBN - 1) / TBN);
  if (tiles >= (1ll << 30)) return set_error(QL_ERR_UNSUPPORTED, "%s: too many output tiles", op);
  if (M > 128 && tiles >= sm_count()) {
    args.sfa = static_cast<const uint8_t *>(a_scales->data);
    args.sfb = static_cast<const uint8_t *>(b_scales->data);
    return launch_tiles(a->data, b->data, args, K, st);
  }
  args.sfa = static_cast<const uint8_t *>(b_scales->data); // the weights are the 128-row operand
  args.sfb = static_cast<const uint8_t *>(a_scales->data);
  if (M <= 16) return launch_split<16>(b->data, a->data, args, K, st);
  if (M <= 32) return launch_split<32>(b->data, a->data, args, K, st);
  if (M <= 64) return launch_split<64>(b->data, a->data, args, K, st);
  return launch_split<128>(b->data, a->data, args, K, st);
}
