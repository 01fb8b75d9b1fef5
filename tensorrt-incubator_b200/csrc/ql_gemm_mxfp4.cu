// Block-scaled MXFP4 product on the 5th-generation tensor cores (sm_100a only):
//     Y[m,n] = sum over blocks b of 2^(ea[m,b] + eb[n,b]) * sum over k in b of qa[m,k] qb[n,k]
// with qa, qb in e2m1 and the e8m0 block scales of quantize_mxfp4 (blocks of 32 along K).  The tensor core applies the
// scales itself (tcgen05.mma kind::mxf4.block_scale, scales read from tensor memory) and accumulates in f32; the result is
// rounded once.  One MMA consumes 64 values of K, two blocks, so a 32-bit cell of tensor memory holds the scales of two
// MMAs; which half an MMA uses is a field of its instruction descriptor.
//
// The tensor core wants the scales of 128 rows as 4 columns of 32 lanes (row r in lane r % 32, column r / 32), repeated in
// all four lane quarters of tensor memory.  The operands' scales are row-major, a row's bytes in a line.  The NVFP4 kernel
// re-orders them in a kernel of its own and copies them from shared to tensor memory between its MMAs.  Here four warps (one
// per quarter; two such sets in the tiles kernel) take the bytes of "their" rows into registers in the layout they already
// need -- lane l holds rows l, l + 32, ... -- and store them with tcgen05.st: no re-ordering pass and no copy instructions
// between the MMAs.
//
// Two kernels:
//   split   few output tiles (decoding, short prompts): the weights are the 128-row operand and up to 128 tokens the other;
//           a cluster of up to 8 CTAs shares the K axis of one tile and adds its parts through distributed shared memory,
//           in rank order (the same bits on every run).
//   tiles   many output tiles, persistent: one CTA per SM on 128 x 208 tiles, or CTA pairs on 256 x 208 tiles (x 112 where the wider
//           ones would leave SMs without work).  In a pair
//           (tcgen05.mma.cta_group::2, issued by its leader) each CTA holds its own 128 rows of A and half of the B tile, so
//           per MMA it reads 232 rows of operands from shared memory instead of 336; the scales of all 208 columns are needed
//           by both.  Y leaves by bulk tensor stores of 32 columns (4096 x 8192 x 512 24 us, 39 with each lane
//           storing its row).
// Every wait is bounded, as in the other tensor-core kernels.
#include <cuda.h>
#include <string.h>

#include "ql_common.cuh"
#include "ql_tc_common.cuh"
#include "ql_together.cuh"

namespace ql {
namespace {

constexpr int kKStep = 256;           // values of K per pipeline stage: 128 bytes of e2m1
constexpr int kScaleBytes = 8;        // scales of one row and k step
constexpr int kSplitOnly = 32;        // up to so many tokens the split kernel is always the one
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

template <bool PAIR>
__device__ __forceinline__ void mx_mma(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  if constexpr (PAIR)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.block32 [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
                 ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
                 : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.block32 [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
                 ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
                 : "memory");
}
// e2m1 operands (format 1), both K-major, e8m0 scales (bit 23), N >> 3 at bit 17, M >> 4 at bit 24, dense K = 64; the byte
// offset (0 or 2) of the scales within their cells at bits 29 (A) and 4 (B)
template <int M, int N> __device__ __forceinline__ uint32_t mx_idesc(uint32_t byte) {
  return 1u << 7 | 1u << 10 | (uint32_t)(N >> 3) << 17 | 1u << 23 | (uint32_t)(M >> 4) << 24 | byte << 29 | byte << 4;
}
__device__ __forceinline__ void tmem_store_4(uint32_t taddr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void tmem_store_16(uint32_t taddr, uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t e, uint32_t f, uint32_t g, uint32_t h, uint32_t i, uint32_t j,
                                              uint32_t k, uint32_t l, uint32_t m, uint32_t n, uint32_t o, uint32_t p) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
               ::"r"(taddr), "r"(a), "r"(b), "r"(c), "r"(d), "r"(e), "r"(f), "r"(g), "r"(h), "r"(i), "r"(j), "r"(k), "r"(l), "r"(m), "r"(n), "r"(o), "r"(p)
               : "memory");
}
// A look at a barrier, without waiting
__device__ __forceinline__ bool mbar_test_wait(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0;
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// MMA j (0..3) of a k step, issued by one lane of a converged warp: 64 values = 32 bytes of K; two MMAs share one set of
// scale cells.
template <int N, bool PAIR>
__device__ __forceinline__ void mx_k_mma(int j, uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t t_sfa, uint32_t t_sfb, int sfb_cols, uint32_t accumulate) {
  mx_mma<PAIR>(tmem_d, adesc + 2 * j, bdesc + 2 * j, mx_idesc<PAIR ? 2 * BM : BM, N>((j & 1) * 2), t_sfa + 4 * (j >> 1), t_sfb + sfb_cols * (j >> 1), accumulate);
}

template <typename OutT> __device__ __forceinline__ void store_y(void *Y, size_t i, float v) { static_cast<OutT *>(Y)[i] = FloatIO<OutT>::from_f32(v); }
__device__ __forceinline__ void store_y(void *Y, int dtype, size_t i, float v) {
  if (dtype == QL_F32) store_y<float>(Y, i, v);
  else if (dtype == QL_F16) store_y<__half>(Y, i, v);
  else store_y<__nv_bfloat16>(Y, i, v);
}

__device__ __forceinline__ uint32_t ldg32_if(const void *p, bool on) {
  uint32_t v;
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\tmov.b32 %0, 0;\n\t@p ld.global.nc.b32 %0, [%1];\n\t}" : "=r"(v) : "l"(p), "r"((int)on));
  return v;
}
// up to four neighbouring values of y
__device__ __forceinline__ void store_y4(const MxArgs &args, size_t i, const float4 &v, int n, bool vec) {
  if (vec && args.y_dtype == QL_F32) *reinterpret_cast<float4 *>(static_cast<float *>(args.Y) + i) = v;
  else if (vec && args.y_dtype == QL_F16) *reinterpret_cast<uint2 *>(static_cast<__half *>(args.Y) + i) = make_uint2(pack2<__half>(v.x, v.y), pack2<__half>(v.z, v.w));
  else if (vec) *reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(args.Y) + i) = make_uint2(pack2<__nv_bfloat16>(v.x, v.y), pack2<__nv_bfloat16>(v.z, v.w));
  else {
    const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (j < n) store_y(args.Y, args.y_dtype, i + j, f[j]);
  }
}

__device__ __forceinline__ uint32_t ldg8_if(const void *p, bool on) {
  uint32_t v;
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\tmov.b32 %0, 0;\n\t@p ld.global.nc.u8 %0, [%1];\n\t}" : "=r"(v) : "l"(p), "r"((int)on));
  return v;
}
// The barrier of the 128 threads that hand scales over (warps as wholes, converged): do all of them go on?
__device__ __forceinline__ bool all_of_128(bool go) {
  uint32_t all;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbar.red.and.pred q, 1, 128, p;\n\tselp.b32 %0, 1, 0, q;\n\t}" : "=r"(all) : "r"((int)go) : "memory");
  return all != 0;
}
// The scale bytes of four k steps of one row: the first `n` of 32 bytes from p on, zeros beyond.  Loading and shifting are
// apart, so that the loads of several rows are in flight together, and the loads are predicated, not branched around: a
// branch or a use between them makes each wait for the one before.
// WIDE: rows lie on multiples of 8 bytes.  Else only the operand does, on a multiple of 4: the aligned words that hold the
// bytes are read, and of a word that reaches beyond the operand (`left` bytes from p on) just the bytes inside.
template <bool WIDE> struct RowScales {
  uint32_t r[WIDE ? 8 : 9];
  int n, off;
  __device__ __forceinline__ void load(const uint8_t *p, int n_, long long left) {
    n = n_;
    off = WIDE ? 0 : (int)(reinterpret_cast<uintptr_t>(p) & 3);
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < 8; i += 2)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.lt.s32 p, %3, %4;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\t@p ld.global.nc.v2.b32 {%0, %1}, [%2];\n\t}"
            : "=r"(r[i]), "=r"(r[i + 1])
            : "l"(p + 4 * i), "r"(4 * i), "r"(n));
    } else {
      const uint8_t *q = p - off;
      const int inside = left > 64 ? 64 : (int)left + off; // bytes of the operand from q on
#pragma unroll
      for (int i = 0; i < 9; i++) r[i] = ldg32_if(q + 4 * i, 4 * i < n + off && 4 * i + 4 <= inside);
      const int cut = inside & ~3; // the word that reaches beyond, if it is wanted
      const bool wanted = cut < 36 && cut < n + off;
#pragma unroll
      for (int j = 0; j < 3; j++) {
        uint32_t v = ldg8_if(q + cut + j, wanted && cut + j < inside) << (8 * j);
#pragma unroll
        for (int i = 0; i < 9; i++)
          if (4 * i == cut && wanted) r[i] |= v;
      }
    }
  }
  __device__ __forceinline__ uint32_t word(int i) const {
    if constexpr (WIDE) return r[i];
    const uint32_t w = __funnelshift_r(r[i], r[i + 1], 8 * off);
    const int here = n - 4 * i; // valid bytes of this word
    return here >= 4 ? w : (here <= 0 ? 0u : w & ((1u << (8 * here)) - 1u));
  }
};

// ------------------------------------------------------------------------------------------------------------------
// split kernel: 128 rows of the weights x TN tokens, K over the CTAs of a cluster
// ------------------------------------------------------------------------------------------------------------------
constexpr int kSplitThreads = 192;
constexpr int kMaxSplit = 8;
constexpr int kFetchSteps = 4;      // k steps whose scales travel together: 32 bytes, a whole sector, of every row
constexpr int kScPitch = 40;

constexpr int kSplitSlots = 2;      // groups of k steps whose scales lie in tensor memory at once
constexpr int kSplitMaxStages = 16;

// Fixed parts first, then the ring: `stages` of (rows of the weights rounded up to 8) + TN rows of 128 bytes.  The MMA reads
// 128 rows of the first operand whatever `rows` is; what it reads beyond them (other stages, the slack behind the last one)
// ends up in accumulator rows nobody looks at.
template <int TN> struct SplitSmem {
  static constexpr int kParts = 0;                         // partial sums of this CTA's tokens, [split][TN / split][128]
  static constexpr int kScales = kParts + TN * BM * 4;     // two groups of four k steps' scales
  static constexpr int kScaleGroup = (BM + TN) * kScPitch;
  static constexpr int kBarriers = kScales + 2 * kScaleGroup; // full[16], empty[16], sfull[2], sempty[2], tfull
  static constexpr int kTmemPtr = kBarriers + (2 * kSplitMaxStages + 2 * kSplitSlots + 1) * 8;
  static constexpr int kAbort = kTmemPtr + 4;
  static constexpr int kRing = (kAbort + 4 + 1023) / 1024 * 1024;
  static constexpr int stage_bytes(int rows) { return ((rows + 7) / 8 * 8 + TN) * BK_BYTES; }
  // At least half of an SM's shared memory, as it takes half of its tensor memory: what fits beside it then finds the columns it
  // needs.  A CTA waiting for columns while its cluster partners wait for it could wait for good.
  static constexpr int kHalf = 232448 / 2 - 2048;
  static constexpr int total(int rows, int stages) {
    const int n = kRing + stages * stage_bytes(rows) + MX_A_BYTES + 1024;
    return n < kHalf ? kHalf : n;
  }
};

template <int TN, bool WIDE>
__global__ void __launch_bounds__(kSplitThreads)
gemm_mxfp4_split_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const MxArgs args, int rows, int stages, int split_log2) {
  using L = SplitSmem<TN>;
  constexpr int ST = kSplitMaxStages, SL = kSplitSlots;
  const int stage_bytes = L::stage_bytes(rows), b_off = stage_bytes - TN * BK_BYTES;
  constexpr int TN_LOG2 = TN == 16 ? 4 : (TN == 32 ? 5 : (TN == 64 ? 6 : 7));
  constexpr uint32_t kSfCol0 = TN;                         // two slots of four k steps, 16 columns each: 8 of the weights' scales, 8 of the tokens'
  constexpr uint32_t kSlotCols = 16 * kFetchSteps, kTmemCols = 256;
  static_assert(kSfCol0 + SL * kSlotCols <= kTmemCols, "tensor memory");
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t smem_base = smem_u32(smem), bar_base = smem_base + L::kBarriers;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (ST + s); };
  auto sfull_bar = [&](int s) { return bar_base + 8u * (2 * ST + s); };
  auto sempty_bar = [&](int s) { return bar_base + 8u * (2 * ST + SL + s); };
  const uint32_t tfull_bar = bar_base + 8u * (2 * ST + 2 * SL);
  volatile uint32_t *tmem_ptr_smem = reinterpret_cast<volatile uint32_t *>(smem + L::kTmemPtr);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::kAbort);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int split = 1 << split_log2;
  const int rank = blockIdx.x & (split - 1), tile = blockIdx.x >> split_log2;
  const int wt = tile % args.tiles_a, xt = tile / args.tiles_a;
  const int ks0 = (int)((long long)args.num_ks * rank / split), ks1 = (int)((long long)args.num_ks * (rank + 1) / split);

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; s++) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int s = 0; s < SL; s++) {
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
  if (split > 1) cluster_arrive(); // waited for before the first store into a partner: the partner has started by then
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_ptr_smem, 0);

  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    int stage = 0, issued = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int ks = ks0; ks < ks1; ks++) {
      if (!warp_wait(empty_bar(stage), phase ^ 1, abort_flag, args.status, ST_TIMEOUT_EMPTY)) { ok = false; break; }
      if (elect_one()) {
        const uint32_t a_dst = smem_base + L::kRing + stage * stage_bytes;
        mbar_expect_tx(full_bar(stage), (uint32_t)(rows + TN) * BK_BYTES);
        tma_load_2d(a_dst, &map_w, full_bar(stage), ks * BK_BYTES, wt * rows); // coordinates in bytes of packed e2m1
        tma_load_2d(a_dst + b_off, &map_x, full_bar(stage), ks * BK_BYTES, xt * TN);
      }
      __syncwarp();
      issued++;
      if (++stage == stages) { stage = 0; phase ^= 1; }
    }
    if (!ok) { // let the loads in flight land before the shared memory goes away
      const int pending = issued < stages ? issued : stages;
      for (int i = 0; i < pending; i++) {
        stage = (stage == 0) ? stages - 1 : stage - 1;
        if (stage == stages - 1) phase ^= 1;
        bounded_wait(full_bar(stage), phase);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issue
    int stage = 0;
    uint32_t phase = 0;
    for (int ks = ks0; ks < ks1; ks++) {
      const int it = ks - ks0, group = it / kFetchSteps, slot = group & 1, q = it % kFetchSteps;
      if (q == 0 && !warp_wait(sfull_bar(slot), (group >> 1) & 1, abort_flag, args.status, ST_TIMEOUT_FULL)) break;
      if (!warp_wait(full_bar(stage), phase, abort_flag, args.status, ST_TIMEOUT_FULL)) break;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t a_addr = smem_base + L::kRing + stage * stage_bytes, t_sf = tmem_base + kSfCol0 + slot * kSlotCols + 16 * q;
        const uint64_t adesc = make_smem_desc(a_addr), bdesc = make_smem_desc(a_addr + b_off);
#pragma unroll
        for (int j = 0; j < 4; j++) mx_k_mma<TN, false>(j, tmem_base, adesc, bdesc, t_sf, t_sf + 8, 4, (it | j) != 0 ? 1u : 0u);
        tc_commit(empty_bar(stage));
        if (q == kFetchSteps - 1) tc_commit(sempty_bar(slot));
      }
      __syncwarp();
      if (++stage == stages) { stage = 0; phase ^= 1; }
    }
    // every MMA issued above is done with shared and tensor memory before this warp goes on, after an abort too
    if (elect_one()) tc_commit(tfull_bar);
    __syncwarp();
    if (!bounded_wait(tfull_bar, 0) && lane == 0) atomicCAS(args.status, 0, ST_TIMEOUT_DRAIN);
  } else {
    // ------------------------------------------------------------------ scales, then the accumulator (warps 2..5)
    const int quad = warp & 3;
    const uint32_t quarter = (uint32_t)(quad * 32) << 16;
    // The 128 threads fetch four k steps of scales together, a row each, two groups ahead; they hand them over through
    // shared memory (rows 40 bytes apart: conflict-free both ways), and each warp stores the rows its lanes hold, one
    // hand-over to the MMA thread per group.  (Each warp loading all rows for itself is four times the L1 look-ups, one per
    // row and step: 1 us per k step at TN = 128.  A hand-over per k step: 0.4 us per step, a latency.)
    constexpr int XR = TN <= 32 ? 1 : TN / 32; // rows of the token operand a lane carries
    const int tid = quad * 32 + lane;
    RowScales<WIDE> a[2], b[2];
    const long long row_a = (long long)wt * rows + tid, row_b = (long long)xt * TN + tid;
    const bool has_a = tid < rows && row_a < args.N, has_b = tid < TN && row_b < args.M;
    auto fetch = [&](int ks, RowScales<WIDE> &fa, RowScales<WIDE> &fb) {
      const int b0 = ks * kScaleBytes, n = min(args.kb, ks1 * kScaleBytes) - b0;
      const long long at_a = has_a ? row_a * args.kb + b0 : 0, at_b = has_b ? row_b * args.kb + b0 : 0;
      fa.load(args.sfa + at_a, has_a ? n : 0, (long long)args.N * args.kb - at_a);
      fb.load(args.sfb + at_b, has_b ? n : 0, (long long)args.M * args.kb - at_b);
    };
    auto meet = [&](auto slot, int, bool go) { // this thread's rows, then the barrier behind which all rows are there
      uint8_t *buf = smem + L::kScales + slot * L::kScaleGroup;
#pragma unroll
      for (int q = 0; q < kFetchSteps; q++) {
        *reinterpret_cast<uint2 *>(buf + tid * kScPitch + q * 8) = make_uint2(a[slot].word(2 * q), a[slot].word(2 * q + 1));
        if (tid < TN) *reinterpret_cast<uint2 *>(buf + (BM + tid) * kScPitch + q * 8) = make_uint2(b[slot].word(2 * q), b[slot].word(2 * q + 1));
      }
      return all_of_128(go);
    };
    auto take = [&](auto slot, int group) {
      const uint8_t *buf = smem + L::kScales + slot * L::kScaleGroup;
      fetch(ks0 + (group + 2) * kFetchSteps, a[slot], b[slot]);
      if (!warp_wait(sempty_bar(slot), ((group >> 1) & 1) ^ 1u, abort_flag, args.status, ST_TIMEOUT_EMPTY)) return false;
      const uint32_t t = tmem_base + quarter + kSfCol0 + slot * kSlotCols;
#pragma unroll
      for (int q = 0; q < kFetchSteps; q++) {
        uint2 pa[4], pb[4];
#pragma unroll
        for (int c = 0; c < 4; c++) {
          pa[c] = *reinterpret_cast<const uint2 *>(buf + (c * 32 + lane) * kScPitch + q * 8);
          pb[c] = make_uint2(0u, 0u);
          if (c < XR && c * 32 + lane < TN) pb[c] = *reinterpret_cast<const uint2 *>(buf + (BM + c * 32 + lane) * kScPitch + q * 8);
        }
        tmem_store_4(t + 16 * q, pa[0].x, pa[1].x, pa[2].x, pa[3].x);
        tmem_store_4(t + 16 * q + 4, pa[0].y, pa[1].y, pa[2].y, pa[3].y);
        tmem_store_4(t + 16 * q + 8, pb[0].x, pb[1].x, pb[2].x, pb[3].x);
        tmem_store_4(t + 16 * q + 12, pb[0].y, pb[1].y, pb[2].y, pb[3].y);
      }
      tmem_store_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(sfull_bar(slot));
      return true;
    };
    fetch(ks0, a[0], b[0]);
    fetch(ks0 + kFetchSteps, a[1], b[1]);
    steps_together((ks1 - ks0 + kFetchSteps - 1) / kFetchSteps, meet, take);
    warp_wait(tfull_bar, 0, abort_flag, args.status, ST_TIMEOUT_TMEM_FULL);
    tc_fence_after();
    // lane = row of the weights = column of Y, so a warp's store of one token is contiguous
    const int row = quad * 32 + lane, n = row < rows ? wt * rows + row : args.N;
    const int tokens = min(TN, args.M - xt * TN), per_log2 = TN_LOG2 - split_log2, per = 1 << per_log2; // CTA o adds up tokens [o * per, (o + 1) * per)
    if (split > 1) cluster_wait();
#pragma unroll 1
    for (int c = 0; c < TN / 16; c++) {
      if (c * 16 >= tokens) break;
      uint32_t r[16];
      tmem_load_16(tmem_base + quarter + c * 16, r);
      if (split > 1) {
#pragma unroll
        for (int j = 0; j < 16; j++) {
          const int t = c * 16 + j;
          if (t < tokens) {
            const uint32_t local = smem_base + (uint32_t)(L::kParts + ((rank * per + (t & (per - 1))) * BM + row) * 4);
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(map_to_cta(local, (uint32_t)(t >> per_log2))), "f"(__uint_as_float(r[j])) : "memory");
          }
        }
      } else if (n < args.N) {
        const int m = xt * TN + c * 16;
#pragma unroll
        for (int j = 0; j < 16; j++)
          if (m + j < args.M) store_y(args.Y, args.y_dtype, (size_t)(m + j) * args.N + n, __uint_as_float(r[j]));
      }
    }
    tc_fence_before();
  }
  if (split > 1) {
    if (warp < 2) cluster_wait();
    __syncwarp();
    cluster_sync_all(); // every part has arrived
    const int per = TN >> split_log2, t0 = rank * per, t1 = min(t0 + per, args.M - xt * TN);
    // four neighbouring columns of Y a thread: rows is a multiple of 4
    const float4 *parts = reinterpret_cast<const float4 *>(smem + L::kParts);
    const bool vec = args.N % 4 == 0 && (reinterpret_cast<uintptr_t>(args.Y) & 15) == 0;
    for (int i = threadIdx.x; i < (t1 - t0) * (BM / 4); i += kSplitThreads) {
      const int row = i % (BM / 4) * 4, n = wt * rows + row;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int p = 0; p < kMaxSplit; p++) {
        if (p < split) {
          const float4 w = parts[p * per * (BM / 4) + i];
          v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
        }
      }
      if (row < rows && n < args.N) store_y4(args, (size_t)(xt * TN + t0 + i / (BM / 4)) * args.N + n, v, vec ? 4 : min(4, args.N - n), vec);
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
  }
}

// ------------------------------------------------------------------------------------------------------------------
// tiles kernel: persistent, 128 x 208 or 128 x 112, or twice the rows by CTA pairs
// ------------------------------------------------------------------------------------------------------------------
// TBN, columns of a tile: 208 leaves tensor memory, beside two accumulators, 96 columns: four slots of the scales of one k step.  A slot is free
// when the MMAs of its step are done, and refilled (the commit, the wait, the stores, the arrival at the pair's leader) about
// 1100 cycles later: three steps (416 cycles each) hide that.  Two slots of two steps, the stage in between hiding it: 8192 x
// 28672 x 8192 765 us, 715 now.  With 224 columns there is room for two slots of one step.
constexpr int kTileThreads = 448;   // producer, MMA, four epilogue warps, two sets of four scale warps
constexpr int kScSteps = 4;         // k steps whose scales travel together: 32 bytes, a whole sector, of every row
constexpr int kStageSteps = 2;      // k steps of one stage
constexpr int kSlots = 4;           // of one k step: 8 columns of A's scales, then 16 (8) of B's: 8 (4) per pair of MMAs, 6.5 (3.5) used
template <bool PAIR, int TBN> struct TileSmem {
  static constexpr int kScRows = BM + TBN, kScLanes = (kScRows + 31) / 32; // rows of scales, and of them those a lane carries
  static constexpr int kScBytes = kScLanes * 32 * 32;                      // with room for the last lanes' rows past the tile
  static constexpr int kCellsB = (TBN + 31) / 32, kColsB = kCellsB > 4 ? 8 : 4;
  static constexpr int kSlotCols = 8 + 2 * kColsB;
  static constexpr int kStages = (PAIR ? 3 : 2) + (TBN <= 128 ? 1 : 0); // of two k steps: half as many barriers to look at and to signal as with one
  static constexpr int kRowsB = PAIR ? TBN / 2 : TBN;                     // rows of the B tile one CTA holds
  static constexpr int kTileB = kRowsB * BK_BYTES;
  static constexpr int kStageBytes = kStageSteps * (MX_A_BYTES + kTileB);  // A's tiles, then B's
  static constexpr int kScales = kStages * kStageBytes;
  static constexpr int kStaging = kScales + 2 * kScBytes;  // the epilogue's, 4096 bytes a warp
  static constexpr int kBarriers = kStaging + 4 * 4096; // full[S], empty[S], tfull[2], tempty[2], scfull[2], scempty[2], sfull[4], sempty[4], drain
  static constexpr int kTmemPtr = kBarriers + (2 * kStages + 9 + 2 * kSlots) * 8;
  static constexpr int kAbort = kTmemPtr + 4;
  static constexpr int kDynamic = kAbort + 4 + 1024;
  static_assert(kDynamic <= 232448 && kStageBytes % 1024 == 0 && kScBytes % 1024 == 0, "tile shape");
};

// A tile's last 16 columns, or the `cols` (a multiple of the 16-byte piece) of them that Y has, of one row a lane, rounded to y's type
template <typename OutT>
__device__ __forceinline__ void mx_store_chunk(OutT *y, const uint32_t (&r)[32], int cols) {
  if constexpr (sizeof(OutT) == 4) {
#pragma unroll
    for (int j = 0; j < 16; j += 4)
      if (j < cols) __stcs(reinterpret_cast<uint4 *>(y + j), make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]));
  } else {
    auto two = [&](int j) { return pack2<OutT>(__uint_as_float(r[j]), __uint_as_float(r[j + 1])); };
#pragma unroll
    for (int j = 0; j < 16; j += 8)
      if (j < cols) __stcs(reinterpret_cast<uint4 *>(y + j), make_uint4(two(j), two(j + 2), two(j + 4), two(j + 6)));
  }
}
// TURNED: 32 rows of Y, a lane its column of them, so that a warp's store is a row's run of 32 columns
template <typename OutT>
__device__ __forceinline__ void mx_store_turned(OutT *y, const uint32_t (&r)[32], int rows, size_t pitch) {
#pragma unroll
  for (int j = 0; j < 32; j++)
    if (j < rows) y[(size_t)j * pitch] = FloatIO<OutT>::from_f32(__uint_as_float(r[j]));
}

// TURNED: operand a are the weights and operand b the activations (args.M, args.N: rows of a and b; Y is [N, M]).  For rows of
// Y that are no multiple of 16 bytes, where a lane that holds a row of Y could only store it value by value, far apart:
// 4571 x 5597 x 160 takes 39 us turned, 88 through a staging buffer in shared memory.
template <bool PAIR, bool TURNED, int TBN>
__global__ void __launch_bounds__(kTileThreads, 1)
gemm_mxfp4_tiles_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_sa,
                        const __grid_constant__ CUtensorMap map_sb, const __grid_constant__ CUtensorMap map_y, const MxArgs args) {
  using L = TileSmem<PAIR, TBN>;
  constexpr int TSTAGES = L::kStages;
  constexpr uint32_t kTmemCols = 512; // two accumulators, four slots of scales
  static_assert(2 * TBN + kSlots * L::kSlotCols <= 512, "tensor memory");
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
  auto sempty_bar = [&](int b) { return bar_base + 8u * (2 * TSTAGES + 8 + kSlots + b); };
  const uint32_t drain_bar = bar_base + 8u * (2 * TSTAGES + 8 + 2 * kSlots);
  volatile uint32_t *tmem_ptr_smem = reinterpret_cast<volatile uint32_t *>(smem + L::kTmemPtr);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::kAbort);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int num_tiles = args.tiles_a * args.tiles_b; // tiles_a counts 256 rows for a pair
  const uint32_t rank = PAIR ? cluster_ctarank() : 0;
  const int first_tile = PAIR ? blockIdx.x >> 1 : blockIdx.x, tile_stride = PAIR ? gridDim.x >> 1 : gridDim.x;
  const int row_tile = PAIR ? 2 : 1; // this CTA's rows are the 128-row tile row_tile * mt + rank
  auto arrive_leader = [&](uint32_t bar) { // the pair's leader owns what the MMAs wait for
    if (PAIR) mbar_arrive_remote(map_to_cta(bar, 0));
    else mbar_arrive(bar);
  };
  auto commit_all = [&](uint32_t bar) { // to the same barrier of both CTAs
    if (PAIR)
      tc_commit_both(bar);
    else
      tc_commit(bar);
  };
  auto tell_partner = [&]() {
    if (PAIR && lane == 0) signal_partner_abort(smem_u32((const void *)abort_flag), rank);
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < TSTAGES; s++) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; b++) {
      mbar_init(tfull_bar(b), 1);
      mbar_init(tempty_bar(b), PAIR ? 8 : 4);
      mbar_init(scfull_bar(b), 1);
      mbar_init(scempty_bar(b), 8); // both sets of scale warps
    }
    for (int b = 0; b < kSlots; b++) {
      mbar_init(sfull_bar(b), PAIR ? 8 : 4);
      mbar_init(sempty_bar(b), 1);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void *)tmem_ptr_smem)), "r"(kTmemCols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void *)tmem_ptr_smem)), "r"(kTmemCols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all(); // the partner's barriers exist before anything is signalled across the pair
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_ptr_smem, 0);

  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    int stage = 0, sc = 0;
    uint32_t phase = 0, sc_phase = 0;
    long long issued = 0, sc_issued = 0;
    bool ok = true;
    for (int tile = first_tile; tile < num_tiles && ok; tile += tile_stride) {
      const int mt = tile % args.tiles_a, nt = tile / args.tiles_a; // row tiles of one column tile run side by side: B stays in L2
      for (int ks = 0; ks < args.num_ks; ks += kStageSteps) { // a second step beyond K is loaded as zeros
        if (ks % kScSteps == 0) {
          if (!warp_wait(scempty_bar(sc), sc_phase ^ 1, abort_flag, args.status, ST_TIMEOUT_EMPTY)) { ok = false; break; }
          if (sc_issued == 0) wait_for_results(); // of the kernel that pads the scales
          if (elect_one()) {
            const uint32_t dst = smem_base + L::kScales + sc * L::kScBytes;
            mbar_expect_tx(scfull_bar(sc), L::kScRows * 32);
            tma_load_2d(dst, &map_sa, scfull_bar(sc), ks * kScaleBytes, (row_tile * mt + rank) * BM);
            tma_load_2d(dst + BM * 32, &map_sb, scfull_bar(sc), ks * kScaleBytes, nt * TBN);
          }
          __syncwarp();
          sc_issued++;
          if (++sc == 2) { sc = 0; sc_phase ^= 1; }
        }
        if (!warp_wait(empty_bar(stage), phase ^ 1, abort_flag, args.status, ST_TIMEOUT_EMPTY)) { ok = false; break; }
        if (elect_one()) {
          const uint32_t a_dst = smem_base + stage * L::kStageBytes, b_dst = a_dst + kStageSteps * MX_A_BYTES;
          const uint32_t bar = PAIR ? map_to_cta(full_bar(stage), 0) : full_bar(stage); // a pair's bytes all land on the leader's barrier
          if (rank == 0) mbar_expect_tx(full_bar(stage), (PAIR ? 2 : 1) * L::kStageBytes);
#pragma unroll
          for (int q = 0; q < kStageSteps; q++) { // coordinates in bytes of packed e2m1
            const int x = (ks + q) * BK_BYTES;
            if (PAIR) {
              tma_load_2d_pair(a_dst + q * MX_A_BYTES, &map_a, bar, x, (2 * mt + rank) * BM);
              tma_load_2d_pair(b_dst + q * L::kTileB, &map_b, bar, x, nt * TBN + rank * L::kRowsB);
            } else {
              tma_load_2d(a_dst + q * MX_A_BYTES, &map_a, bar, x, mt * BM);
              tma_load_2d(b_dst + q * L::kTileB, &map_b, bar, x, nt * TBN);
            }
          }
        }
        __syncwarp();
        issued++;
        if (++stage == TSTAGES) { stage = 0; phase ^= 1; }
      }
    }
    if (!ok) { // let the loads in flight land before the shared memory goes away
      tell_partner();
      const long long pending = issued < TSTAGES ? issued : TSTAGES, sc_pending = sc_issued < 2 ? sc_issued : 2;
      for (long long i = 0; i < pending && rank == 0; i++) { // a pair's loads complete on its leader's barriers
        stage = (stage == 0) ? TSTAGES - 1 : stage - 1;
        if (stage == TSTAGES - 1) phase ^= 1;
        bounded_wait(full_bar(stage), phase);
      }
      for (long long i = 0; i < sc_pending; i++) {
        sc ^= 1;
        if (sc == 1) sc_phase ^= 1;
        bounded_wait(scfull_bar(sc), sc_phase);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issue (a pair's leader)
    // The tensor core takes the next MMA when it starts the one before, so whatever this warp does between two MMAs has one
    // MMA's time (104 cycles) to hide in.  A look at a barrier takes about 80: the ones for the next stage and slot go between
    // the MMAs of this one, and only what was not ready then is waited for.  (Both waits ahead of the MMAs left the tensor
    // core idle for half of every k step.)
    if (rank == 0) {
      const bool leader = elect_one();
      int stage = 0, it = 0;
      uint32_t phase = 0, half = 0; // half: slots used so far
      bool ok = true, data_ready = false, scales_ready = false;
      for (int tile = first_tile; tile < num_tiles && ok; tile += tile_stride, it++) {
        const int buf = it & 1;
        if (!warp_wait(tempty_bar(buf), ((it >> 1) & 1) ^ 1, abort_flag, args.status, ST_TIMEOUT_TMEM_EMPTY)) { ok = false; break; }
        const uint32_t tmem_d = tmem_base + (uint32_t)(buf * TBN);
        for (int ks = 0; ks < args.num_ks; ks += kStageSteps) {
          const int slot = (int)(half & 1) * kStageSteps; // of the first step; the second has the next one
          const uint32_t parity = (half >> 1) & 1;
          if (!scales_ready && !warp_wait(sfull_bar(slot), parity, abort_flag, args.status, ST_TIMEOUT_FULL)) { ok = false; break; }
          if (!data_ready && !warp_wait(full_bar(stage), phase, abort_flag, args.status, ST_TIMEOUT_FULL)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a_addr = smem_base + stage * L::kStageBytes, t_sfa = tmem_base + kSfCol0 + L::kSlotCols * slot, t_sfb = t_sfa + 8;
          const uint64_t adesc = make_smem_desc(a_addr), bdesc = make_smem_desc(a_addr + kStageSteps * MX_A_BYTES);
          const int cur = stage;
          if (++stage == TSTAGES) { stage = 0; phase ^= 1; }
          half++;
          auto mma = [&](int q, int j) {
            mx_k_mma<TBN, PAIR>(j, tmem_d, adesc + q * (MX_A_BYTES >> 4), bdesc + q * (L::kTileB >> 4), t_sfa + q * L::kSlotCols, t_sfb + q * L::kSlotCols, L::kColsB, (ks | q | j) != 0 ? 1u : 0u);
          };
          if (leader) {
#pragma unroll
            for (int j = 0; j < 3; j++) mma(0, j);
          }
          __syncwarp();
          const bool second_ready = __all_sync(0xffffffffu, mbar_test_wait(sfull_bar(slot + 1), parity));
          if (leader) {
            mma(0, 3);
            commit_all(sempty_bar(slot));
          }
          __syncwarp();
          if (!second_ready && !warp_wait(sfull_bar(slot + 1), parity, abort_flag, args.status, ST_TIMEOUT_FULL)) { ok = false; break; }
          tc_fence_after();
          if (leader) mma(1, 0);
          __syncwarp();
          data_ready = __all_sync(0xffffffffu, mbar_test_wait(full_bar(stage), phase));
          if (leader) {
            mma(1, 1);
            mma(1, 2);
          }
          __syncwarp();
          scales_ready = __all_sync(0xffffffffu, mbar_test_wait(sfull_bar((int)(half & 1) * kStageSteps), (half >> 1) & 1));
          if (leader) {
            mma(1, 3);
            commit_all(sempty_bar(slot + 1));
            commit_all(empty_bar(cur));
            if (ks + kStageSteps >= args.num_ks) commit_all(tfull_bar(buf));
          }
          __syncwarp();
        }
      }
      if (!ok) tell_partner();
      if (elect_one()) { // every MMA issued above has to finish before tensor memory is released
        if (PAIR) tc_commit_pair(map_to_cta(drain_bar, 0));
        else tc_commit(drain_bar);
      }
      __syncwarp();
      if (!bounded_wait(drain_bar, 0) && lane == 0) atomicCAS(args.status, 0, ST_TIMEOUT_DRAIN);
    }
  } else if (warp >= 6) {
    // ------------------------------------------------------------------ scales (warps 6..13, two for each quarter of the lanes)
    // The two sets take stages in turn, each with the two slots that are its own.
    const uint32_t quarter = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t set = warp >= 10 ? 1 : 0;
    uint32_t half = 0; // stages so far
    bool ok = true;
    const int groups = (args.num_ks + kScSteps - 1) / kScSteps; // of four k steps, in a tile
    auto hand_over = [&](int ks, int sc, uint32_t sc_phase) {
      ok = warp_wait(scfull_bar(sc), sc_phase, abort_flag, args.status, ST_TIMEOUT_FULL);
      if (!ok) return;
      const uint8_t *buf = smem + L::kScales + sc * L::kScBytes;
      uint32_t w[L::kScLanes][4]; // rows lane, lane + 32, ... : the words of two k steps
      int h = 0;                 // the stage of this group that is this set's, if there is one
      while (h < kScSteps / kStageSteps && ks + h * kStageSteps < args.num_ks && ((half + h) & 1) != set) h++;
      const bool mine = h < kScSteps / kStageSteps && ks + h * kStageSteps < args.num_ks;
      const uint32_t parity = ((half + h) >> 1 & 1) ^ 1u;
      half += min((args.num_ks - ks + kStageSteps - 1) / kStageSteps, kScSteps / kStageSteps);
      if (mine) {
        // 32-byte rows as the copy engine's 32-byte swizzle leaves them: a row's halves changed places in rows 4 to 7 of 8, so that
        // eight lanes' 16 bytes cover all banks
        const uint8_t *row = buf + lane * 32 + ((16 * h) ^ ((lane & 4) << 2));
#pragma unroll
        for (int c = 0; c < L::kScLanes; c++) {
          const uint4 v = *reinterpret_cast<const uint4 *>(row + c * 1024);
          w[c][0] = v.x, w[c][1] = v.y, w[c][2] = v.z, w[c][3] = v.w;
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(scempty_bar(sc));
      if (!mine) return;
#pragma unroll
      for (int q = 0; q < kStageSteps; q++) {
        const int slot = (int)set * kStageSteps + q;
        ok = warp_wait(sempty_bar(slot), parity, abort_flag, args.status, ST_TIMEOUT_EMPTY);
        if (!ok) return;
        // for each pair of MMAs (word j): four cells of A's rows, seven (four) of B's
        const uint32_t t = tmem_base + quarter + kSfCol0 + L::kSlotCols * slot;
        auto v = [&](int c, int j) { return w[c][2 * q + j]; };
        tmem_store_4(t, v(0, 0), v(1, 0), v(2, 0), v(3, 0));
        tmem_store_4(t + 4, v(0, 1), v(1, 1), v(2, 1), v(3, 1));
        if constexpr (L::kCellsB == 7) {
          tmem_store_16(t + 8, v(4, 0), v(5, 0), v(6, 0), v(7, 0), v(8, 0), v(9, 0), v(10, 0), 0u, v(4, 1), v(5, 1), v(6, 1), v(7, 1), v(8, 1), v(9, 1), v(10, 1), 0u);
        } else {
          static_assert(L::kCellsB == 4, "cells of B's scales");
          tmem_store_4(t + 8, v(4, 0), v(5, 0), v(6, 0), v(7, 0));
          tmem_store_4(t + 12, v(4, 1), v(5, 1), v(6, 1), v(7, 1));
        }
        tmem_store_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_leader(sfull_bar(slot));
      }
    };
    const int mine = first_tile < num_tiles ? (num_tiles - first_tile + tile_stride - 1) / tile_stride : 0;
    const long long total = (long long)mine * groups;
    int group = 0;
    uint32_t sc_phase = 0;
    for (long long i = 0; i < total && ok; i += 2, sc_phase ^= 1) {
      hand_over(group * kScSteps, 0, sc_phase);
      if (++group == groups) group = 0;
      if (ok && i + 1 < total) hand_over(group * kScSteps, 1, sc_phase);
      if (++group == groups) group = 0;
    }
    if (!ok) tell_partner();
  } else {
    // ------------------------------------------------------------------ epilogue (warps 2..5)
    const int quad = warp & 3;
    const bool wide = args.y_dtype == QL_F32;
    Parked out{smem + L::kStaging + quad * 4096};
    int it = 0, b = 0; // b: the staging buffer whose turn it is
    for (int tile = first_tile; tile < num_tiles; tile += tile_stride, it++) {
      const int buf = it & 1;
      const int mt = tile % args.tiles_a, nt = tile / args.tiles_a;
      if (!warp_wait(tfull_bar(buf), (it >> 1) & 1, abort_flag, args.status, ST_TIMEOUT_TMEM_FULL)) { tell_partner(); break; }
      tc_fence_after();
      const int m0 = (row_tile * mt + (int)rank) * BM + quad * 32, m = m0 + lane;
      const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(buf * TBN);
#pragma unroll 1
      for (int c = 0; c < (TBN + 31) / 32; c++) {
        const int n = nt * TBN + c * 32, cols = min(min(args.N, nt * TBN + TBN) - n, 32);
        if (m0 >= args.M || cols <= 0) break; // nothing left to store
        uint32_t r[32];
        tmem_load_32(taddr + c * 32, r); // of the last chunk half the columns are the next accumulator's, or scales: not stored
        if (!TURNED && c < TBN / 32) { // rows of 64 bytes in two buffers, of 128 (f32) in the room of both
          auto put16 = [&](auto type) {
            using OutT = decltype(type);
            auto two = [&](int j) { return pack2<OutT>(__uint_as_float(r[j]), __uint_as_float(r[j + 1])); };
#pragma unroll
            for (int j = 0; j < 32; j += 8) out.put64(b, lane, j >> 3, make_uint4(two(j), two(j + 2), two(j + 4), two(j + 6)));
          };
          if (wide) {
            out.reusable<0>(lane);
#pragma unroll
            for (int j = 0; j < 32; j += 4) out.put(0, lane, j >> 2, make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]));
            out.send(0, &map_y, lane, n, m0);
          } else {
            out.reusable<1>(lane);
            if (args.y_dtype == QL_F16) put16(__half());
            else put16(__nv_bfloat16());
            out.send64(b, &map_y, lane, n, m0);
            b ^= 1;
          }
        } else if (m < args.M) { // the tile's last 16 columns, or TURNED
          const size_t at = TURNED ? (size_t)n * (size_t)args.M + m : (size_t)m * (size_t)args.N + n;
          auto store = [&](auto *y) {
            if constexpr (TURNED) mx_store_turned(y, r, cols, (size_t)args.M);
            else mx_store_chunk(y, r, cols);
          };
          if (wide) store(static_cast<float *>(args.Y) + at);
          else if (args.y_dtype == QL_F16) store(static_cast<__half *>(args.Y) + at);
          else store(static_cast<__nv_bfloat16 *>(args.Y) + at);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_leader(tempty_bar(buf));
    }
    if (!TURNED) out.finish(lane);
  }

  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all(); // neither CTA may leave while the pair's MMAs or barriers can still touch it
  if (warp == 1) {
    tc_fence_after();
    if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
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

bool scales_on_multiple(const MxArgs &args, int of) {
  return ((reinterpret_cast<uintptr_t>(args.sfa) | reinterpret_cast<uintptr_t>(args.sfb) | (uintptr_t)args.kb) & (uintptr_t)(of - 1)) == 0;
}

// Clusters of 2^log2 CTAs that the device holds at once at one CTA per SM (a part of the machine with a number of SMs that is
// no multiple of the cluster leaves some idle: 148, 74, 33, 15 on B200).
template <int TN, bool WIDE> int resident_clusters(int log2) {
  static int cached[64][4] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 1;
  int &n = cached[dev][log2];
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(2 * sm_count() << log2), 1, 1);
    cfg.blockDim = dim3(kSplitThreads, 1, 1);
    cfg.dynamicSmemBytes = 232448;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 1u << log2, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int got = 0;
    if (cudaOccupancyMaxActiveClusters(&got, gemm_mxfp4_split_kernel<TN, WIDE>, &cfg) != cudaSuccess || got < 1) {
      cudaGetLastError();
      got = sm_count() >> log2;
    }
    n = got;
  }
  return n;
}

struct SplitPlan {
  int co, log2, rows, stages;
  double us;
};

// How to cut a product of few tiles: `rows` of the weights per CTA, 2^log2 CTAs sharing K, `co` CTAs per SM.  The estimate
// of each choice's time comes from measurements on B200 (graph-replayed calls, cold weights): 3.3 us fixed; per k step
// 0.33 us, 0.0029 us more for every token row beyond 16, or what one SM's share of memory bandwidth (48 KB/us) takes;
// 1.2 us + 0.033 us per token row to add up the parts of a cluster, or half of that to store more than 32 tokens.  Examples (us; M, N, K):
//   1 x 28672 x 8192    100 rows, 2 CTAs per SM 23.5   |  128 rows, 1 per SM (two waves) 30.8  |  K over 4 CTAs 31.5
//   1 x 4096 x 4096     128 rows, K over 4 CTAs 6.4    |  28 rows, K whole 9.4
//   24 x 4096 x 11008   128 rows, K over 4 CTAs 11.0   |  28 rows, K whole 18.3
// Rows are spread so that one wave of CTAs covers the weights: an MMA's rows beyond them cost nothing here, a second wave
// does.
template <int TN, bool WIDE> SplitPlan plan_split(int M, int N, int num_ks) {
  using L = SplitSmem<TN>;
  const int64_t tiles_x = (M + TN - 1) / TN;
  SplitPlan best = {1, 0, BM, 1, 1e30};
  for (int co = 1; co <= (TN <= 32 ? 2 : 1); co++) {
    for (int log2 = 0; log2 < 4 && (log2 == 0 || num_ks >= (2 << log2)); log2++) {
      const int fit = resident_clusters<TN, WIDE>(log2) * co;
      const int64_t per_x = fit / tiles_x, want = per_x < 1 ? BM : (N + per_x - 1) / per_x;
      const int rows = ((int)(want > BM ? BM : (want < 16 ? 16 : want)) + 3) / 4 * 4;
      const int64_t tiles = (int64_t)((N + rows - 1) / rows) * tiles_x, waves = (tiles + fit - 1) / fit;
      const int steps = (num_ks + (1 << log2) - 1) >> log2;
      const double latency = 0.33 + 0.0029 * (TN - 16), bandwidth = (double)(rows + TN) * BK_BYTES * co / 48e3;
      const double join = log2 ? 1.2 + 0.033 * TN : (TN >= 64 ? 1.2 + 0.016 * TN : 0.0);
      const double us = (double)waves * (3.3 + 0.5 * (co - 1) + join + steps * (latency > bandwidth ? latency : bandwidth));
      if (us < best.us) {
        int stages = (232448 / co - 2048 - (L::kRing + MX_A_BYTES + 1024)) / L::stage_bytes(rows);
        stages = stages > kSplitMaxStages ? kSplitMaxStages : stages;
        best = {co, log2, rows, stages > steps ? steps : stages, us};
      }
    }
  }
  return best;
}

// args: the weights are operand a here
template <int TN, bool WIDE> int launch_split_as(const void *w, const void *x, MxArgs args, int64_t K, const SplitPlan &plan, cudaStream_t st) {
  using L = SplitSmem<TN>;
  auto kern = gemm_mxfp4_split_kernel<TN, WIDE>;
  int rc;
  args.tiles_a = (args.N + plan.rows - 1) / plan.rows;
  args.tiles_b = (args.M + TN - 1) / TN;
  CUtensorMap mw, mx;
  if ((rc = encode_map(&mw, KIND_F8, w, args.N, K / 2, plan.rows)) != QL_OK) return rc;
  if ((rc = encode_map(&mx, KIND_F8, x, args.M, K / 2, TN)) != QL_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(((int64_t)args.tiles_a * args.tiles_b) << plan.log2), 1, 1);
  cfg.blockDim = dim3(kSplitThreads, 1, 1);
  cfg.dynamicSmemBytes = L::total(plan.rows, plan.stages);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 1u << plan.log2, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  QL_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, mw, mx, args, plan.rows, plan.stages, plan.log2));
  count_launches(1);
  return QL_OK;
}
// Runs the split kernel where its estimate is below `limit_us`, else says so in *ran.
template <int TN> int launch_split(const void *w, const void *x, const MxArgs &args, int64_t K, double limit_us, bool *ran, cudaStream_t st) {
  const bool wide = scales_on_multiple(args, 8);
  // the occupancy query needs the kernels' shared-memory limit raised first
  static bool configured_f[64] = {false}, configured_g[64] = {false};
  int rc = wide ? allow_smem(gemm_mxfp4_split_kernel<TN, true>, 232448, configured_f) : allow_smem(gemm_mxfp4_split_kernel<TN, false>, 232448, configured_g);
  if (rc != QL_OK) return rc;
  const SplitPlan plan = wide ? plan_split<TN, true>(args.M, args.N, args.num_ks) : plan_split<TN, false>(args.M, args.N, args.num_ks);
  *ran = plan.us <= limit_us;
  if (!*ran) return QL_OK;
  return wide ? launch_split_as<TN, true>(w, x, args, K, plan, st) : launch_split_as<TN, false>(w, x, args, K, plan, st);
}

// Rows of scale bytes, `pitch` bytes apart and zero-padded, of both operands: 16 bytes a thread, from the aligned words that hold
// them (the operands lie on multiples of 4); a word that reaches beyond its operand is read byte by byte.
__global__ void __launch_bounds__(256) mx_pad_scales_kernel(const uint8_t *__restrict__ a, int rows_a, const uint8_t *__restrict__ b, int rows_b, int kb, int units,
                                                            uint4 *__restrict__ out) {
  dependents_may_start();
  const int unit = blockIdx.x * 32 + threadIdx.x % 32, b0 = unit * 16; // a warp takes 512 bytes of a row, a block eight rows
  if (unit >= units) return;
  for (int64_t row = (int64_t)blockIdx.y * 8 + threadIdx.x / 32; row < (int64_t)rows_a + rows_b; row += (int64_t)gridDim.y * 8) {
    const bool first = row < rows_a;
    const int64_t at = (first ? row : row - rows_a) * kb + b0, left = (int64_t)(first ? rows_a : rows_b) * kb - at; // bytes of the operand from here on
    const uint8_t *p = (first ? a : b) + at;
    const int off = (int)(at & 3), valid = min(16, kb - b0); // of the unit
    const uint8_t *q = p - off;
    uint32_t r[5];
#pragma unroll
    for (int i = 0; i < 5; i++) r[i] = ldg32_if(q + 4 * i, 4 * i < valid + off && 4 * i + 4 <= left + off);
    if (left + off < 4 * ((valid + off + 3) / 4)) { // the operand's last row
#pragma unroll
      for (int j = 0; j < 20; j++)
        if (j >= (int)((left + off) & ~3) && j < left + off) r[j / 4] |= (uint32_t)__ldg(q + j) << (8 * (j % 4));
    }
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int here = valid - 4 * i;
      w[i] = __funnelshift_r(r[i], r[i + 1], 8 * off) & (here >= 4 ? 0xFFFFFFFFu : (here <= 0 ? 0u : (1u << (8 * here)) - 1u));
    }
    out[row * units + unit] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// The copy engine takes rows of whole 16-byte units from a 16-byte aligned base.  Other scales are copied into such rows first
// (in the caller's workspace): 2000 x 4096 x 11008 47.5 us, against 45.7 at K = 11264; 150 with the scale warps loading them.
int padded_pitch(int64_t kb) { return (int)((kb + 15) / 16 * 16); }
bool needs_padding(const MxArgs &args) { return args.kb % 16 != 0 || !aligned16(args.sfa) || !aligned16(args.sfb); }
int64_t padded_bytes(int64_t M, int64_t N, int64_t kb) { return (M + N) * padded_pitch(kb); }

// scales [rows, pitch] as bytes, box = [box_rows, 32 bytes], 32-byte swizzle
int encode_map_scales(CUtensorMap *map, const uint8_t *ptr, int64_t rows, int64_t pitch, int box_rows) {
  EncodeTiledFn enc;
  const int rc = get_encode_fn(&enc);
  if (rc != QL_OK) return rc;
  cuuint64_t dims[2] = {(cuuint64_t)pitch, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)pitch};
  cuuint32_t box[2] = {32, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_32B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(QL_ERR_CUDA, "cuTensorMapEncodeTiled (scales) failed with code %d", (int)r);
  return QL_OK;
}

// args: operands a and b as the kernel takes them (TURNED: the weights first)
template <bool PAIR, bool TURNED, int TBN> int launch_tiles(const void *a, const void *b, MxArgs args, int64_t K, void *workspace, cudaStream_t st) {
  using L = TileSmem<PAIR, TBN>;
  static bool configured[64] = {false};
  int rc = allow_smem(gemm_mxfp4_tiles_kernel<PAIR, TURNED, TBN>, L::kDynamic, configured);
  if (rc != QL_OK) return rc;
  int pitch = args.kb;
  const bool padding = needs_padding(args);
  if (padding) {
    pitch = padded_pitch(args.kb);
    const int units = pitch / 16;
    const int64_t row_blocks = ((int64_t)args.M + args.N + 7) / 8;
    const dim3 grid((unsigned)((units + 31) / 32), (unsigned)(row_blocks < 65535 ? row_blocks : 65535));
    mx_pad_scales_kernel<<<grid, 256, 0, st>>>(args.sfa, args.M, args.sfb, args.N, args.kb, units, static_cast<uint4 *>(workspace));
    count_launches(1);
    QL_CUDA_TRY(cudaGetLastError());
    args.sfa = static_cast<const uint8_t *>(workspace);
    args.sfb = args.sfa + (int64_t)args.M * pitch;
  }
  CUtensorMap ma, mb, msa, msb, my;
  if ((rc = encode_map(&ma, KIND_F8, a, args.M, K / 2, BM)) != QL_OK) return rc;
  if ((rc = encode_map(&mb, KIND_F8, b, args.N, K / 2, L::kRowsB)) != QL_OK) return rc;
  if ((rc = encode_map_scales(&msa, args.sfa, args.M, pitch, BM)) != QL_OK) return rc;
  if ((rc = encode_map_scales(&msb, args.sfb, args.N, pitch, TBN)) != QL_OK) return rc;
  my = ma; // TURNED: not used
  if (!TURNED && (rc = args.y_dtype == QL_F32 ? encode_map_out(&my, QL_F32, args.Y, args.M, args.N, args.N) : encode_map_narrow(&my, args.y_dtype, args.Y, args.M, args.N)) != QL_OK)
    return rc;
  args.tiles_a = (args.M + (PAIR ? 2 : 1) * BM - 1) / ((PAIR ? 2 : 1) * BM);
  args.tiles_b = (args.N + TBN - 1) / TBN;
  const int64_t tiles = (int64_t)args.tiles_a * args.tiles_b;
  const int units = PAIR ? sm_count() / 2 : sm_count();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((PAIR ? 2 : 1) * (tiles < units ? tiles : units)), 1, 1);
  cfg.blockDim = dim3(kTileThreads, 1, 1);
  cfg.dynamicSmemBytes = L::kDynamic;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = PAIR ? 2 : 1, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization; // it starts while the scales are being padded
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = padding ? 2 : 1;
  QL_CUDA_TRY(cudaLaunchKernelEx(&cfg, gemm_mxfp4_tiles_kernel<PAIR, TURNED, TBN>, ma, mb, msa, msb, my, args));
  count_launches(1);
  return QL_OK;
}
template <bool TURNED> int launch_tiles_as(bool pairs, bool narrow, const void *a, const void *b, const MxArgs &args, int64_t K, void *workspace, cudaStream_t st) {
  if (pairs) return narrow ? launch_tiles<true, TURNED, 112>(a, b, args, K, workspace, st) : launch_tiles<true, TURNED, 208>(a, b, args, K, workspace, st);
  return narrow ? launch_tiles<false, TURNED, 112>(a, b, args, K, workspace, st) : launch_tiles<false, TURNED, 208>(a, b, args, K, workspace, st);
}

} // namespace
} // namespace ql

using namespace ql;

extern "C" int ql_gemm_mxfp4_workspace(const ql_tensor *a, const ql_tensor *a_scales, const ql_tensor *b, const ql_tensor *b_scales, int64_t *bytes) {
  const char *op = "gemm_mxfp4_workspace";
  int rc;
  if ((rc = check_mx_operand(op, "a", a, a_scales)) != QL_OK) return rc;
  if ((rc = check_mx_operand(op, "b", b, b_scales)) != QL_OK) return rc;
  if (!bytes) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: no place for the size", op);
  const int64_t M = a->shape[0], N = b->shape[0], kb = a->shape[1] / 32;
  const bool rows16 = kb % 16 == 0 && aligned16(a_scales->data) && aligned16(b_scales->data);
  *bytes = rows16 || M <= kSplitOnly || N == 0 ? 0 : padded_bytes(M, N, kb);
  return QL_OK;
}

extern "C" int ql_gemm_mxfp4(const ql_tensor *a, const ql_tensor *a_scales, const ql_tensor *b, const ql_tensor *b_scales, ql_tensor *y, void *workspace, int64_t workspace_bytes,
                             void *stream) {
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
  if ((reinterpret_cast<uintptr_t>(a_scales->data) | reinterpret_cast<uintptr_t>(b_scales->data)) & 3) return set_error(QL_ERR_UNSUPPORTED, "%s: needs 4-byte aligned scales", op);
  if (reinterpret_cast<uintptr_t>(y->data) % (y->dtype == QL_F32 ? 4 : 2)) return set_error(QL_ERR_UNSUPPORTED, "%s: y is not aligned to its type", op);
  if (M > (1 << 30) || N > (1 << 30) || K > (1 << 30)) return set_error(QL_ERR_UNSUPPORTED, "%s: dimension too large", op);
  int64_t need = 0;
  if ((rc = ql_gemm_mxfp4_workspace(a, a_scales, b, b_scales, &need)) != QL_OK) return rc;
  if (need > 0 && (!workspace || workspace_bytes < need))
    return set_error(QL_ERR_INVALID_ARGUMENT, "%s: needs a workspace of %lld bytes, got %lld", op, (long long)need, (long long)(workspace ? workspace_bytes : 0));
  if (need > 0 && !aligned16(workspace)) return set_error(QL_ERR_UNSUPPORTED, "%s: the workspace must be 16-byte aligned", op);
  if (overlap(y, a) || overlap(y, a_scales) || overlap(y, b) || overlap(y, b_scales)) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: y must not overlap an operand", op);
  const ql_tensor scratch = workspace_view(workspace, need);
  if (overlap(&scratch, y) || overlap(&scratch, a) || overlap(&scratch, a_scales) || overlap(&scratch, b) || overlap(&scratch, b_scales))
    return set_error(QL_ERR_INVALID_ARGUMENT, "%s: the workspace must not overlap y or an operand", op);
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
  // Pairs of the tiles kernel take 6.7 us and 0.29 us per tile and k step, with tiles of 112 columns 5.6 and 0.243; its single CTAs
  // 6.0 and 0.43, or 4.0 and 0.36; a tile at least the 2.2 (1.7) us that storing it takes beside the next; 3 more where scales are
  // padded, half of them the host's.  The split kernel takes what plan_split says.  Up to 32 tokens the tiles are mostly padding
  // and the split kernel is the better one throughout; up to 128 rows of the first operand a pair's second half would be.  us,
  // split and tiles: 128 x 1928 x 4736 11.8, 14.1; 534 x 1617 x 768 8.4, 8.7; 356 x 4440 x 5088 19.4, 16.2; 458 x 11848 x 480 23.8, 13.5.
  // Tiles of 208 and of 112 columns: 512 x 4096 x 4096 11.9, 10.0; 4490 x 384 x 22528 32.5, 26.9; 70 x 9000 x 4096 12.9, 9.7;
  // 2048 x 1024 x 4096 11.5, 12.7; 1403 x 7344 x 768 14.5, 16.9; 4096 x 4096 x 8192 55, 68.5.  Single CTAs and pairs: 128 x 28672 x
  // 8192 28.0, 32; 8192 x 28672 x 8192 920, 720.
  const bool turned = N % (y->dtype == QL_F32 ? 4 : 8) != 0 || !aligned16(y->data);
  const int64_t R = turned ? N : M, C = turned ? M : N; // rows of the tiles kernel's operands
  const bool pairs = R > BM;
  const int64_t row_tiles = pairs ? (R + 2 * BM - 1) / (2 * BM) : (R + BM - 1) / BM, units = pairs ? sm_count() / 2 : sm_count();
  if (row_tiles * ((C + 111) / 112) >= (1ll << 30)) return set_error(QL_ERR_UNSUPPORTED, "%s: too many output tiles", op);
  auto tiles_us = [&](int width, double fixed, double step, double store) {
    const int64_t tiles = row_tiles * ((C + width - 1) / width);
    const double main_us = step * args.num_ks, store_us = C < width ? store * C / width : store; // of a tile, one beside the other
    return fixed + (need > 0 ? 3.0 : 0.0) + (double)((tiles + units - 1) / units) * (main_us > store_us ? main_us : store_us);
  };
  const double wide_us = tiles_us(208, pairs ? 6.7 : 6.0, pairs ? 0.29 : 0.43, 2.2), narrow_us = tiles_us(112, pairs ? 5.6 : 4.0, pairs ? 0.243 : 0.36, 1.7);
  const bool narrow = narrow_us < wide_us;
  const double limit_us = M <= kSplitOnly ? 1e30 : (narrow ? narrow_us : wide_us);
  args.sfa = static_cast<const uint8_t *>(b_scales->data); // the weights are the 128-row operand of the split kernel
  args.sfb = static_cast<const uint8_t *>(a_scales->data);
  bool ran = false;
  rc = M <= 16   ? launch_split<16>(b->data, a->data, args, K, limit_us, &ran, st)
       : M <= 32 ? launch_split<32>(b->data, a->data, args, K, limit_us, &ran, st)
       : M <= 64 ? launch_split<64>(b->data, a->data, args, K, limit_us, &ran, st)
                 : launch_split<128>(b->data, a->data, args, K, limit_us, &ran, st);
  if (rc != QL_OK || ran) return rc;
  if (turned) {
    args.M = (int)N, args.N = (int)M;
    return launch_tiles_as<true>(pairs, narrow, b->data, a->data, args, K, workspace, st);
  }
  args.sfa = static_cast<const uint8_t *>(a_scales->data);
  args.sfb = static_cast<const uint8_t *>(b_scales->data);
  return launch_tiles_as<false>(pairs, narrow, a->data, b->data, args, K, workspace, st);
}
