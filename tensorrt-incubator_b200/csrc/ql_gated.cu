// Gated projection of a feed-forward block in 16 bits and its backward pass (sm_100a only):
//     H = act(G) * U,   G = X Wg^T,  U = X Wu^T          X [M,K], Wg and Wu [I,K], H [M,I]; act: silu, gelu, gelu_tanh, relu
//     dG = dH * U * act'(G),  dU = dH * act(G),  dX = dG Wg + dU Wu,  dWg = dG^T X,  dWu = dU^T X
// the unquantized counterpart of the fp8 block's gate/up projection (ql_gemm_fp8_swiglu), weights as they are stored.
//
// Forward: both projections are one product with the gate rows as one half of the B operand and the up rows as the other;
// activation and product are formed from the f32 accumulators, and H is rounded once.  G and U never reach memory.
// Of few tokens dG and dU are kept as the sum of two values of the operands' type, the rounded one and the rounding's remainder,
// and the second products take both: the rows of the remainders go where a pair's 256 rows would be empty, and another step
// over the tokens hides behind writing the weights' gradients.  The gradients' error is then their last rounding's alone.  With
// many tokens the rounding of dG and dU stays, for the second products would take twice as long: it is of the last one's size
// (sqrt 2 of it in all), being averaged over many values.
//
// Backward: nothing of size M x I is kept from the forward pass.  A first kernel repeats the two projections and forms dG and
// dU in its epilogue from the f32 accumulators and dH; both are rounded to the operands' type (f16: times a power of two), being
// the operands of the second kernel, which computes dX and both weight gradients in one launch.  Keeping G and U in 16 bits would save the third
// of the backward pass that repeats them and would add their two roundings to the one of dG and dU.
//
// Kernels:
//   gated_split     few tokens (decoding): the weights are the 128-row operand (gate rows, then up rows of the same channels),
//                   up to 128 tokens the other; a cluster of CTAs shares K and adds its parts in rank order through
//                   distributed shared memory.  Bound by reading the weights once.
//                   (each runs a second time where f16 needs another power of two, see kRanged)
//   gated_pair      many tokens: persistent CTA pairs (cta_group::2) on 256 tokens x 128 (or 64) channels, six stages; CTA 0
//                   of a pair loads the gate rows, CTA 1 the up rows, so each holds half of the B tile.  Bound by the tensor
//                   cores; small problems by what comes before the first MMA and after the last.
//   gated_grads     the second products, persistent CTA pairs on 256 x 256 tiles.  dX reads dG, dU along their rows (K-major)
//                   and the weights across (MN-major); the weight gradients read both operands across.  All through the
//                   same 128-byte-swizzled tiles: for an operand whose rows run along the reduction a tile is 64 rows of
//                   128 bytes per 64 columns, and the descriptor says so.  No operand is transposed in memory.
//   grads_reduce    adds the f32 parts of units whose reduction was cut, in a fixed order.
// Every wait is bounded, as in the other tensor-core kernels.
#include <cuda.h>
#include <string.h>

#include <type_traits>

#include "ql_common.cuh"
#include "ql_gated_plan.cuh"
#include "ql_tc_common.cuh"

namespace ql {
namespace {

enum { ACT_SILU = 0, ACT_GELU = 1, ACT_GELU_TANH = 2, ACT_RELU = 3 };

// Phi(z), the normal distribution, and e = exp(-z^2 / 2).  For a = |z| the tail is Phi(-a) = e M(a) with M the Mills ratio over
// sqrt(2 pi), which is smooth and here a polynomial of degree 7 in 1 / (1 + a / 4), fitted by reweighted least squares to
// the smallest relative error on [0, 13]: 5e-7.  Rounding z^2 / 2 adds up to 2^-24 z^2 / 2 and the fast exponential its 2 + 0.59 z^2
// units of 2^-23: below 5e-6 in all for |z| <= 6 and 2e-5 at 13, so the tails keep their digits where 1 + erf would cancel.  A third of erfcf's instructions: with it the epilogue bounded small K (6606 x 21984 x 792 with both gradients 1.82 ms,
// 1.47 now, as silu).
__device__ __forceinline__ float normal_cdf(float z, float &e) {
  e = __expf(-0.5f * z * z);
  const float t = __fdividef(1.f, fmaf(0.25f, fabsf(z), 1.f));
  float m = -0.0926494300365448f;
  m = fmaf(m, t, 0.3499186933040619f);
  m = fmaf(m, t, -0.2896791994571686f);
  m = fmaf(m, t, 0.31156009435653687f);
  m = fmaf(m, t, 0.002527108183130622f);
  m = fmaf(m, t, 0.12122871726751328f);
  m = fmaf(m, t, 0.09694066643714905f);
  m = fmaf(m, t, 0.00015359123062808067f);
  const float tail = e * m;
  return z < 0.f ? tail : 1.f - tail;
}

// act(z).  The fast exponential is off by 2 + 1.17 |x| units of 2^-23 for e^x, the fast division by two: far below the 16-bit
// rounding that follows (2^-12 at the least) while the result is not tiny; at z = -80 it is 1e-5.  A divisor beyond 2^126 gives 0:
// silu below z = -87.3, where it is -z e^z < 2^-119, and likewise gelu_tanh.
template <int ACT> __device__ __forceinline__ float act_value(float z) {
  if constexpr (ACT == ACT_SILU) return __fdividef(z, 1.f + __expf(-z));
  else if constexpr (ACT == ACT_GELU) { float e; return z * normal_cdf(z, e); }
  else if constexpr (ACT == ACT_GELU_TANH) return __fdividef(z, 1.f + __expf(-1.5957691f * (z + 0.044715f * z * z * z))); // (1 + tanh y) / 2 = 1 / (1 + e^-2y)
  else return z < 0.f ? 0.f : z; // a NaN stays one
}
// act(z) and act'(z)
template <int ACT> __device__ __forceinline__ void act_both(float z, float &a, float &d) {
  if constexpr (ACT == ACT_SILU) {
    const float s = __fdividef(1.f, 1.f + __expf(-z));
    a = z * s;
    d = s * (1.f + z * (1.f - s));
  } else if constexpr (ACT == ACT_GELU) {
    float e;
    const float c = normal_cdf(z, e);
    a = z * c;
    d = c + z * 0.39894228f * e;
  } else if constexpr (ACT == ACT_GELU_TANH) {
    const float s = __fdividef(1.f, 1.f + __expf(-1.5957691f * (z + 0.044715f * z * z * z)));
    a = z * s;
    const float b = fminf(fmaxf(z, -32.f), 32.f); // beyond, s (1 - s) is 0 in f32, and z^2 need not be finite; a NaN is s's too
    d = s + b * s * (1.f - s) * 1.5957691f * (1.f + 0.134145f * b * b);
  } else {
    a = z < 0.f ? 0.f : z;
    d = z > 0.f ? 1.f : a; // 0, or z's NaN
  }
}
// f(activation as a template argument), chosen once for a whole chunk of values
template <typename F> __device__ __forceinline__ void with_act(int act, F &&f) {
  switch (act) {
  case ACT_SILU: f(std::integral_constant<int, ACT_SILU>{}); break;
  case ACT_GELU: f(std::integral_constant<int, ACT_GELU>{}); break;
  case ACT_GELU_TANH: f(std::integral_constant<int, ACT_GELU_TANH>{}); break;
  default: f(std::integral_constant<int, ACT_RELU>{}); break;
  }
}

// What rounding v to T leaves; 0 where that is an infinity.
template <typename T> __device__ __forceinline__ float remainder_of(float v) {
  const float h = FloatIO<T>::to_f32(FloatIO<T>::from_f32(v));
  return fabsf(h) == INFINITY ? 0.f : v - h;
}

// dG and dU in f16 are held times a power of two, undone in f32 where the second products leave their accumulators: f16 ends at
// 65504, and below 2^-14 its digits fade, while gradients come in every size.  The first stage multiplies dH by 2^6 and notes the
// largest finite magnitude it then met, before rounding; where that is not between 2^2 and 65504 it is run again (the launch is
// there on every call and ends at once otherwise) with the power that takes it to 2^14 .. 2^15.  So digits are lost below 2^-16
// of the largest value at the earliest.  bf16 has f32's range and none of this.
// Beside one launch without any of it: 16 x 2744 x 1032 22.0 us, 24.4 with the second launch, 31 where it runs; 77 x 2744 x 1032
// 23.6, 26.5 and 35; 128 x 11008 x 4096 133, 136 and 185; 512 x 2744 x 1032 43, 45 and 56; 4096 x 11008 x 4096 1.66, 1.69 and 2.17 ms.
// Noting the largest takes 0.3 to 0.7 of the 2.5 us, the launch the rest.  An exponent from the largest |dH| alone would need no
// second run but for gates and projections far from 1, where it would be as wrong as none.
template <typename T> constexpr bool kRanged = FloatIO<T>::kDtype == QL_F16;
constexpr int kFirstExponent = 6;
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// The largest of what the first stage's CTAs met, for every lane of a warp; bits of floats that are not negative order as these do.
__device__ __forceinline__ float largest_of(const float *largest, int n, int lane) {
  uint32_t m = 0;
#pragma unroll 8
  for (int i = lane; i < n; i += 32) m = max(m, __float_as_uint(largest[i]));
  return __uint_as_float(__reduce_max_sync(0xffffffffu, m));
}
__device__ __forceinline__ bool first_exponent_fits(float largest) { return largest == 0.f || (largest >= 4.f && largest <= 65504.f); }
__device__ __forceinline__ int range_exponent(float largest) {
  // 60 at the most: beyond, every gradient is 0 in f16, and a product on the way would leave f32's range
  return first_exponent_fits(largest) ? kFirstExponent : min(kFirstExponent + 14 + 127 - (int)(__float_as_uint(largest) >> 23), 60);
}
// The larger of `top` and the values' magnitudes, a NaN or an infinity aside
template <int N> __device__ __forceinline__ float finite_top(float top, const uint32_t (&bits)[N]) {
  auto magnitude = [&](int i) { return fabsf(__uint_as_float(bits[i])); };
  float all = 0.f;
#pragma unroll
  for (int i = 0; i < N; i++) all = fmaxf(all, magnitude(i)); // passes over a NaN
  if (all < INFINITY) return fmaxf(top, all);
#pragma unroll
  for (int i = 0; i < N; i++) top = fmaxf(top, magnitude(i) < INFINITY ? magnitude(i) : 0.f);
  return top;
}

template <typename T> constexpr uint32_t kTypeBits = FloatIO<T>::kDtype == QL_BF16 ? (1u << 7 | 1u << 10) : 0u; // operand formats of kind::f16

// Instruction descriptor of kind::f16: f32 accumulation, N >> 3 at bit 17, M >> 4 at bit 24, operand A (bit 15) or B (bit 16)
// MN-major.
template <typename T> __device__ __forceinline__ uint32_t f16_idesc(int m, int n, bool a_mn, bool b_mn) {
  return 1u << 4 | kTypeBits<T> | (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24 | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u);
}
// Descriptor of an MN-major tile as [64-column groups][64 rows of 128 bytes], 128-byte swizzle: 64 columns further on is 8192
// bytes (leading byte offset), 8 rows of the reduction further on is 1024 (stride byte offset).
__device__ __forceinline__ uint64_t make_mn_desc(uint32_t addr) {
  uint64_t d = 0;
  d |= (uint64_t)((addr >> 4) & 0x3FFF);
  d |= (uint64_t)(8192 >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
__device__ __forceinline__ void mma_f16_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
               : "memory");
}

constexpr int G_TILE = 128 * BK_BYTES;      // 16 KiB: one CTA's half of an operand tile, 128 rows x 64 values or 64 x 128
constexpr int G_STAGE = 2 * G_TILE;
constexpr int G_STAGES = 6;
constexpr int kEpilogueWarps = 8;           // two for each quarter of tensor memory's lanes, which take 32 columns in turn
constexpr int kPairThreads = 64 + 32 * kEpilogueWarps; // producer, MMA, epilogue
constexpr int G_N = 256;                    // columns of the pair's accumulator

struct PairSmem {
  static constexpr int kStaging = G_STAGES * G_STAGE;       // the epilogue's, 4096 bytes a warp
  static constexpr int kBarriers = kStaging + kEpilogueWarps * 4096; // full[S], empty[S], tfull[2], tempty[2], drain
  static constexpr int kTmemPtr = kBarriers + (2 * G_STAGES + 5) * 8;
  static constexpr int kAbort = kTmemPtr + 4;
  static constexpr int kLargest = kAbort + 4; // kRanged
  static constexpr int kDynamic = kLargest + 4 + 1024;
};
static_assert(PairSmem::kDynamic <= 232448, "shared memory");

// The backward pass's kernels are launched as soon as all CTAs of the one before have started: they set up barriers and tensor
// memory where an SM is free, and wait here for its results.  dependents_may_start() comes at the start of a kernel; nothing is
// written before the wait, and the first kernel of a call is launched in the stream's order.  77 x 2744 x 1032 27.2 us, 29.1
// with each launched when the one before has ended.
// What the two pair kernels share: barriers, tensor memory, the ring.  Both CTAs' loads complete on the leader's barriers.
struct Pair {
  uint8_t *smem;
  uint32_t base, bars, tmem, rank;
  volatile int *abort_flag;
  int *status;
  int warp, lane;
  __device__ __forceinline__ uint32_t full(int s) const { return bars + 8u * s; }
  __device__ __forceinline__ uint32_t empty(int s) const { return bars + 8u * (G_STAGES + s); }
  __device__ __forceinline__ uint32_t tfull(int b) const { return bars + 8u * (2 * G_STAGES + b); }
  __device__ __forceinline__ uint32_t tempty(int b) const { return bars + 8u * (2 * G_STAGES + 2 + b); }
  __device__ __forceinline__ float *largest() const { return reinterpret_cast<float *>(smem + PairSmem::kLargest); }
  __device__ __forceinline__ uint32_t drain() const { return bars + 8u * (2 * G_STAGES + 4); }

  __device__ __forceinline__ void start(uint8_t *raw, int *status_) {
    smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    base = smem_u32(smem);
    bars = base + PairSmem::kBarriers;
    abort_flag = reinterpret_cast<volatile int *>(smem + PairSmem::kAbort);
    status = status_;
    warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    lane = threadIdx.x & 31;
    rank = cluster_ctarank();
    volatile uint32_t *tmem_ptr = reinterpret_cast<volatile uint32_t *>(smem + PairSmem::kTmemPtr);
    if (threadIdx.x == 0) {
      for (int s = 0; s < G_STAGES; s++) {
        mbar_init(full(s), 1);
        mbar_init(empty(s), 1);
      }
      for (int b = 0; b < 2; b++) {
        mbar_init(tfull(b), 1);
        mbar_init(tempty(b), 2 * kEpilogueWarps); // of both CTAs of the pair
      }
      mbar_init(drain(), 1);
      *abort_flag = 0;
      *largest() = 0.f;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32((const void *)tmem_ptr)) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all(); // the partner's barriers exist before anything is signalled across the pair
    tc_fence_after();
    tmem = __shfl_sync(0xffffffffu, *tmem_ptr, 0);
  }
  __device__ __forceinline__ void end() {
    tc_fence_before();
    __syncthreads();
    cluster_sync_all(); // neither CTA may leave while the pair's MMAs or barriers can still touch it
    if (warp == 1) {
      tc_fence_after();
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
  }
  // after a failed wait of the producer: tells the partner, and lets what this ring still expects land
  __device__ __forceinline__ void producer_gives_up(int stage, uint32_t phase, long long issued) {
    if (lane == 0) signal_partner_abort(smem_u32((const void *)abort_flag), rank);
    if (rank != 0) return;
    const long long pending = issued < G_STAGES ? issued : G_STAGES;
    for (long long i = 0; i < pending; i++) {
      stage = (stage == 0) ? G_STAGES - 1 : stage - 1;
      if (stage == G_STAGES - 1) phase ^= 1;
      bounded_wait(full(stage), phase);
    }
  }
  __device__ __forceinline__ void drain_mmas() {
    if (elect_one()) tc_commit_pair(map_to_cta(drain(), 0));
    __syncwarp();
    if (!bounded_wait(drain(), 0) && lane == 0) atomicCAS(status, 0, ST_TIMEOUT_DRAIN);
  }
};

// ------------------------------------------------------------------------------------------------------------------
// the two projections of many tokens: forward (H), or dG and dU
// ------------------------------------------------------------------------------------------------------------------
struct ProjArgs {
  const void *dh; // backward: [M, I]
  int M, I, K;
  int act;
  int layers; // backward: of dG and dU, 2 with the remainders
  float *largest;    // backward, kRanged: what each CTA of the first run met
  int again;         // this is the second run, of as many CTAs
  int num_kb; // steps of 64 values of K
  int tiles_m, tiles_n, group_m;
  int *status;
};

// C channels to a tile
template <typename T, bool BACKWARD, int C>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
gated_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_gate, const __grid_constant__ CUtensorMap map_up,
                  const __grid_constant__ CUtensorMap map_out, const __grid_constant__ CUtensorMap map_out2, const ProjArgs args) {
  extern __shared__ uint8_t smem_raw[];
  Pair p;
  if (BACKWARD) dependents_may_start();
  constexpr bool RANGED = BACKWARD && kRanged<T>;
  float scale = pow2(kFirstExponent);
  if (RANGED && args.again) {
    wait_for_results();
    const float seen = largest_of(args.largest, gridDim.x, threadIdx.x & 31);
    if (first_exponent_fits(seen)) return; // all CTAs alike
    scale = pow2(range_exponent(seen));
  }
  p.start(smem_raw, args.status);
  const int cluster_id = blockIdx.x >> 1, num_clusters = gridDim.x >> 1, num_tiles = args.tiles_m * args.tiles_n;

  if (p.warp == 0) {
    // ------------------------------------------------------------------ producer (both CTAs)
    int stage = 0;
    uint32_t phase = 0;
    long long issued = 0;
    bool ok = true;
    const CUtensorMap *map_w = p.rank == 0 ? &map_gate : &map_up;
    for (int tile = cluster_id; tile < num_tiles && ok; tile += num_clusters) {
      int mt, nt;
      band_coords(tile, args.tiles_m, args.tiles_n, args.group_m, &mt, &nt);
      const int m0 = mt * 256 + (int)p.rank * 128, n0 = nt * C;
      for (int kb = 0; kb < args.num_kb; kb++) {
        if (!warp_wait(p.empty(stage), phase ^ 1, p.abort_flag, p.status, ST_TIMEOUT_EMPTY)) { ok = false; break; }
        if (elect_one()) {
          const uint32_t dst = p.base + stage * G_STAGE, bar = map_to_cta(p.full(stage), 0);
          if (p.rank == 0) mbar_expect_tx(p.full(stage), 2 * (G_TILE + C * BK_BYTES));
          tma_load_2d_pair(dst, &map_x, bar, kb * 64, m0);
          tma_load_2d_pair(dst + G_TILE, map_w, bar, kb * 64, n0);
        }
        __syncwarp();
        issued++;
        if (++stage == G_STAGES) { stage = 0; phase ^= 1; }
      }
    }
    if (!ok) p.producer_gives_up(stage, phase, issued);
  } else if (p.warp == 1) {
    // ------------------------------------------------------------------ MMA issue (leader only)
    if (p.rank == 0) {
      const uint32_t idesc = f16_idesc<T>(256, 2 * C, false, false);
      int stage = 0, it = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = cluster_id; tile < num_tiles && ok; tile += num_clusters, it++) {
        const int buf = it & 1;
        if (!warp_wait(p.tempty(buf), ((it >> 1) & 1) ^ 1, p.abort_flag, p.status, ST_TIMEOUT_TMEM_EMPTY)) { ok = false; break; }
        for (int kb = 0; kb < args.num_kb; kb++) {
          if (!warp_wait(p.full(stage), phase, p.abort_flag, p.status, ST_TIMEOUT_FULL)) { ok = false; break; }
          tc_fence_after();
          if (elect_one()) {
            const uint32_t a = p.base + stage * G_STAGE;
            const uint64_t adesc = make_smem_desc(a), bdesc = make_smem_desc(a + G_TILE);
#pragma unroll
            for (int k = 0; k < 4; k++) mma_f16_pair(p.tmem + (uint32_t)(buf * G_N), adesc + 2 * k, bdesc + 2 * k, idesc, (kb | k) != 0 ? 1u : 0u);
            tc_commit_both(p.empty(stage));
            if (kb == args.num_kb - 1) {
              tc_commit_both(p.tfull(buf));
            }
          }
          __syncwarp();
          if (++stage == G_STAGES) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok && p.lane == 0) signal_partner_abort(smem_u32((const void *)p.abort_flag), p.rank);
      p.drain_mmas();
    }
  } else {
    // ------------------------------------------------------------------ epilogue (warps 2..9, both CTAs)
    const int quad = p.warp & 3, turn = (p.warp - 2) >> 2, lane = p.lane;
    Parked out{p.smem + PairSmem::kStaging + (p.warp - 2) * 4096};
    int it = 0, b = 0; // b: the staging buffer whose turn it is (forward)
    bool ok = true;
    float top = 0.f;
    uint4 ahead[4]; // dH of this warp's next chunk, of the next tile after a tile's last one: on its way while the one before is worked on
    auto fetch = [&](int tile, int c) {
      if (tile >= num_tiles) return;
      int mt, nt;
      band_coords(tile, args.tiles_m, args.tiles_n, args.group_m, &mt, &nt);
      const int m = mt * 256 + (int)p.rank * 128 + quad * 32 + lane, n = nt * C + c * 32;
      const T *row = static_cast<const T *>(args.dh) + (size_t)m * (size_t)args.I + n;
#pragma unroll
      for (int j = 0; j < 4; j++) ahead[j] = m < args.M && n + 8 * j < args.I ? __ldcs(reinterpret_cast<const uint4 *>(row) + j) : make_uint4(0u, 0u, 0u, 0u);
    };
    if constexpr (BACKWARD) fetch(cluster_id, turn);
    for (int tile = cluster_id; tile < num_tiles; tile += num_clusters, it++) {
      const int buf = it & 1;
      int mt, nt;
      band_coords(tile, args.tiles_m, args.tiles_n, args.group_m, &mt, &nt);
      const int m0 = mt * 256 + (int)p.rank * 128 + quad * 32;
      ok = warp_wait(p.tfull(buf), (it >> 1) & 1, p.abort_flag, p.status, ST_TIMEOUT_TMEM_FULL);
      if (!ok) break;
      tc_fence_after();
      const uint32_t taddr = p.tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(buf * G_N);
#pragma unroll 1
      for (int c = turn; c < C / 32; c += 2) { // 32 channels: gate in columns 32 c, up in columns C + 32 c
        const int n = nt * C + c * 32;
        uint4 dh[4];
        if constexpr (BACKWARD) {
#pragma unroll
          for (int j = 0; j < 4; j++) dh[j] = ahead[j];
          if (c + 2 < C / 32) fetch(tile, c + 2);
          else fetch(tile + num_clusters, turn);
        }
        if (m0 >= args.M || n >= args.I) continue; // nothing to store
        uint32_t g[32], u[32];
        tmem_load_32(taddr + c * 32, g);
        tmem_load_32(taddr + C + c * 32, u);
        if constexpr (!BACKWARD) {
          with_act(args.act, [&](auto act) {
#pragma unroll
            for (int j = 0; j < 32; j++) g[j] = __float_as_uint(act_value<decltype(act)::value>(__uint_as_float(g[j])) * __uint_as_float(u[j]));
          });
          auto two = [&](int j) { return pack2<T>(__uint_as_float(g[j]), __uint_as_float(g[j + 1])); };
          out.reusable<1>(lane);
#pragma unroll
          for (int j = 0; j < 32; j += 8) out.put64(b, lane, j >> 3, make_uint4(two(j), two(j + 2), two(j + 4), two(j + 6)));
          out.send64(b, &map_out, lane, n, m0);
          b ^= 1;
        } else {
          const T *d = reinterpret_cast<const T *>(dh);
          with_act(args.act, [&](auto act) {
#pragma unroll
            for (int j = 0; j < 32; j++) {
              float a, da;
              const float dv = FloatIO<T>::to_f32(d[j]) * (RANGED ? scale : 1.f);
              act_both<decltype(act)::value>(__uint_as_float(g[j]), a, da);
              g[j] = __float_as_uint(dv * __uint_as_float(u[j]) * da);
              u[j] = __float_as_uint(dv * a);
            }
          });
          if constexpr (RANGED) {
            top = finite_top(top, g);
            top = finite_top(top, u);
          }
          auto two = [&](const uint32_t (&v)[32], int j) { return pack2<T>(__uint_as_float(v[j]), __uint_as_float(v[j + 1])); };
          for (int layer = 0; layer < args.layers; layer++) {
            if (layer > 0) {
#pragma unroll
              for (int j = 0; j < 32; j++) {
                g[j] = __float_as_uint(remainder_of<T>(__uint_as_float(g[j])));
                u[j] = __float_as_uint(remainder_of<T>(__uint_as_float(u[j])));
              }
            }
            out.reusable<0>(lane); // both buffers: dG in one, dU in the other
#pragma unroll
            for (int j = 0; j < 32; j += 8) {
              out.put64(0, lane, j >> 3, make_uint4(two(g, j), two(g, j + 2), two(g, j + 4), two(g, j + 6)));
              out.put64(1, lane, j >> 3, make_uint4(two(u, j), two(u, j + 2), two(u, j + 4), two(u, j + 6)));
            }
            out.send_layer(0, &map_out, lane, n, m0, layer);
            out.send_layer(2048, &map_out2, lane, n, m0, layer);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(map_to_cta(p.tempty(buf), 0)); // the leader owns the accumulator hand-over
    }
    out.finish(lane);
    if (RANGED) {
      const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
      if (lane == 0) atomicMax(reinterpret_cast<uint32_t *>(p.largest()), bits);
    }
    if (!ok && lane == 0) signal_partner_abort(smem_u32((const void *)p.abort_flag), p.rank);
  }
  p.end();
  if (RANGED && !args.again && threadIdx.x == 0) args.largest[blockIdx.x] = *p.largest();
}

// ------------------------------------------------------------------------------------------------------------------
// dX and both weight gradients
// ------------------------------------------------------------------------------------------------------------------
// Maps: d*_k see dG / dU as tiles of 128 rows x 64 columns (K-major), d*_mn, w*_mn, x_mn as 64 rows x 64 columns.
template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
gated_grads_kernel(const __grid_constant__ CUtensorMap map_dg_k, const __grid_constant__ CUtensorMap map_du_k, const __grid_constant__ CUtensorMap map_dg_mn,
                   const __grid_constant__ CUtensorMap map_du_mn, const __grid_constant__ CUtensorMap map_wg_mn, const __grid_constant__ CUtensorMap map_wu_mn,
                   const __grid_constant__ CUtensorMap map_x_mn, const __grid_constant__ CUtensorMap map_dx, const __grid_constant__ CUtensorMap map_dwg,
                   const __grid_constant__ CUtensorMap map_dwu, const GradArgs args) {
  extern __shared__ uint8_t smem_raw[];
  Pair p;
  dependents_may_start();
  p.start(smem_raw, args.status);
  wait_for_results();
  const int cluster_id = blockIdx.x >> 1, num_clusters = gridDim.x >> 1;
  Unit u;

  if (p.warp == 0) {
    // ------------------------------------------------------------------ producer (both CTAs)
    int stage = 0;
    uint32_t phase = 0;
    long long issued = 0;
    bool ok = true;
    const int half_steps = args.x_steps / 2; // steps of the gate's channels
    for (int j = 0; ok && get_unit(args, cluster_id, num_clusters, j, &u); j++) {
      const int r0 = u.row0 + (int)p.rank * 128, c0 = u.col0 + (int)p.rank * 128;
      for (int s = u.step0; s < u.step1; s++) {
        if (!warp_wait(p.empty(stage), phase ^ 1, p.abort_flag, p.status, ST_TIMEOUT_EMPTY)) { ok = false; break; }
        if (elect_one()) {
          const uint32_t a = p.base + stage * G_STAGE, b = a + G_TILE, bar = map_to_cta(p.full(stage), 0);
          if (p.rank == 0) mbar_expect_tx(p.full(stage), 2 * G_STAGE);
          if (u.is_x) {
            const bool up = s >= half_steps;
            const int i0 = (up ? s - half_steps : s) * 64;
            if (args.layers == 2) tma_load_3d_pair(a, up ? &map_du_k : &map_dg_k, bar, i0, 0, (int)p.rank);
            else tma_load_3d_pair(a, up ? &map_du_k : &map_dg_k, bar, i0, r0, 0);
            const CUtensorMap *w = up ? &map_wu_mn : &map_wg_mn;
            tma_load_2d_pair(b, w, bar, c0, i0);
            tma_load_2d_pair(b + 8192, w, bar, c0 + 64, i0);
          } else {
            const CUtensorMap *d = u.up ? &map_du_mn : &map_dg_mn;
            const int layer = args.layers == 2 ? s & 1 : 0, m = (args.layers == 2 ? s >> 1 : s) * 64;
            tma_load_3d_pair(a, d, bar, r0, m, layer);
            tma_load_3d_pair(a + 8192, d, bar, r0 + 64, m, layer);
            tma_load_2d_pair(b, &map_x_mn, bar, c0, m);
            tma_load_2d_pair(b + 8192, &map_x_mn, bar, c0 + 64, m);
          }
        }
        __syncwarp();
        issued++;
        if (++stage == G_STAGES) { stage = 0; phase ^= 1; }
      }
    }
    if (!ok) p.producer_gives_up(stage, phase, issued);
  } else if (p.warp == 1) {
    // ------------------------------------------------------------------ MMA issue (leader only)
    if (p.rank == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int j = 0; ok && get_unit(args, cluster_id, num_clusters, j, &u); j++) {
        const int buf = j & 1;
        const uint32_t idesc = f16_idesc<T>(256, G_N, !u.is_x, true);
        if (!warp_wait(p.tempty(buf), ((j >> 1) & 1) ^ 1, p.abort_flag, p.status, ST_TIMEOUT_TMEM_EMPTY)) { ok = false; break; }
        for (int s = u.step0; s < u.step1; s++) {
          if (!warp_wait(p.full(stage), phase, p.abort_flag, p.status, ST_TIMEOUT_FULL)) { ok = false; break; }
          tc_fence_after();
          if (elect_one()) {
            const uint32_t a = p.base + stage * G_STAGE;
            // 16 values of the reduction further on: 32 bytes along a row, or 16 rows of 128 bytes
            const uint64_t adesc = u.is_x ? make_smem_desc(a) : make_mn_desc(a), bdesc = make_mn_desc(a + G_TILE);
            const uint64_t astep = u.is_x ? 2 : 128;
#pragma unroll
            for (int k = 0; k < 4; k++) mma_f16_pair(p.tmem + (uint32_t)(buf * G_N), adesc + astep * k, bdesc + 128 * k, idesc, (s > u.step0 || k) ? 1u : 0u);
            tc_commit_both(p.empty(stage));
            if (s == u.step1 - 1) {
              tc_commit_both(p.tfull(buf));
            }
          }
          __syncwarp();
          if (++stage == G_STAGES) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok && p.lane == 0) signal_partner_abort(smem_u32((const void *)p.abort_flag), p.rank);
      p.drain_mmas();
    }
  } else {
    // ------------------------------------------------------------------ epilogue (warps 2..9, both CTAs)
    const int quad = p.warp & 3, turn = (p.warp - 2) >> 2, lane = p.lane;
    Parked out{p.smem + PairSmem::kStaging + (p.warp - 2) * 4096};
    bool ok = true;
    float back = 1.f; // what dG and dU were multiplied by, undone
    if constexpr (kRanged<T>) back = pow2(-range_exponent(largest_of(args.largest, args.num_largest, lane)));
    for (int j = 0; get_unit(args, cluster_id, num_clusters, j, &u); j++) {
      const int buf = j & 1;
      ok = warp_wait(p.tfull(buf), (j >> 1) & 1, p.abort_flag, p.status, ST_TIMEOUT_TMEM_FULL);
      if (!ok) break;
      tc_fence_after();
      const bool stacked = u.is_x && args.layers == 2; // this CTA has the rounded values' rows, or the remainders'
      const int r0 = u.row0 + (stacked ? 0 : (int)p.rank * 128) + quad * 32;
      const uint32_t taddr = p.tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(buf * G_N);
      const bool parts = (u.is_x ? args.x_parts : args.w_parts) != nullptr; // f32, a layer for each part of the sum
      const int layer = stacked ? 2 * u.part + (int)p.rank : (u.is_x ? u.part : 2 * u.part + (u.up ? 1 : 0));
      const CUtensorMap *map = u.is_x ? &map_dx : (u.up && !parts ? &map_dwu : &map_dwg);
      out.reusable<0>(lane); // a part takes the room of both 16-bit buffers
      int b = 0;             // the buffer whose turn it is
#pragma unroll 1
      for (int c = turn; c < G_N / 32; c += 2) {
        const int n = u.col0 + c * 32;
        if (r0 >= (u.is_x ? args.M : args.I) || n >= args.K) break; // nothing left to store
        uint32_t v[32];
        tmem_load_32(taddr + c * 32, v);
        if constexpr (kRanged<T>) {
#pragma unroll
          for (int i = 0; i < 32; i++) v[i] = __float_as_uint(__uint_as_float(v[i]) * back);
        }
        if (parts) {
          out.reusable<0>(lane);
#pragma unroll
          for (int i = 0; i < 32; i += 4) out.put(0, lane, i >> 2, make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]));
          out.send_layer(0, map, lane, n, r0, layer);
        } else {
          auto two = [&](int i) { return pack2<T>(__uint_as_float(v[i]), __uint_as_float(v[i + 1])); };
          out.reusable<1>(lane);
#pragma unroll
          for (int i = 0; i < 32; i += 8) out.put64(b, lane, i >> 3, make_uint4(two(i), two(i + 2), two(i + 4), two(i + 6)));
          out.send64(b, map, lane, n, r0);
          b ^= 1;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(map_to_cta(p.tempty(buf), 0));
    }
    out.finish(lane);
    if (!ok && lane == 0) signal_partner_abort(smem_u32((const void *)p.abort_flag), p.rank);
  }
  p.end();
}

// out[i] = sum over p of parts[p][i]; the first values are dX's, then come dWg's and dWu's.  1 << slices_log2 threads share four
// neighbouring values where there are few of them and many parts: thread s adds parts s, s + slices, ... and the sums are
// added in the order of s, so that the result is the same on every run.
constexpr int kReduceThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kReduceThreads) grads_reduce_kernel(const float4 *__restrict__ x_parts, int x_split, T *__restrict__ dx, int64_t nx4,
                                                                      const float4 *__restrict__ w_parts, int w_split, T *__restrict__ dwg, T *__restrict__ dwu, int64_t nw4,
                                                                      int slices_log2) {
  __shared__ float4 sums[kReduceThreads];
  const int per_log2 = 8 - slices_log2, at = threadIdx.x & ((1 << per_log2) - 1), slice = threadIdx.x >> per_log2, slices = 1 << slices_log2;
  const int64_t n = (x_parts ? nx4 : 0) + (w_parts ? 2 * nw4 : 0);
  wait_for_results();
  for (int64_t first = (int64_t)blockIdx.x << per_log2; first < n; first += (int64_t)gridDim.x << per_log2) {
    const int64_t i = first + at;
    const bool is_x = x_parts && i < nx4;
    const int64_t j = is_x ? i : i - (x_parts ? nx4 : 0);
    const float4 *src = is_x ? x_parts + j : w_parts + j;
    const int64_t stride = is_x ? nx4 : 2 * nw4;
    const int split = i < n ? (is_x ? x_split : w_split) : 0;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p = slice; p < split; p += slices) {
      const float4 w = __ldcs(src + p * stride);
      v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
    }
    if (slices > 1) {
      __syncthreads(); // the sums of the round before have been read
      sums[threadIdx.x] = v;
      __syncthreads();
      if (slice != 0) continue;
      for (int s = 1; s < slices; s++) {
        const float4 w = sums[(s << per_log2) + at];
        v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
      }
    }
    if (i >= n) continue;
    T *out = is_x ? dx : (j < nw4 ? dwg : dwu);
    reinterpret_cast<uint2 *>(out)[is_x || j < nw4 ? j : j - nw4] = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
  }
}

// ------------------------------------------------------------------------------------------------------------------
// few tokens: the weights as the 128-row operand, K over the CTAs of a cluster
// ------------------------------------------------------------------------------------------------------------------
template <bool WIDE> constexpr int kSplitThreads = WIDE ? 320 : 192; // producer, MMA, four or eight warps on the accumulators
constexpr int kSplitMaxStages = 16;
constexpr int kMaxSplit = 8;

struct SplitArgs {
  const void *dh; // backward: [M, I]
  void *out, *out2; // H, or dG and dU, [layers][M][I]
  int M, I;
  int act, layers;
  float *largest; // as in ProjArgs
  int again;
  int num_kb;
  int tiles_c; // tiles of channels
  int *status;
};

// Fixed parts first, then the ring: `stages` of (channels rounded up to 8) gate rows, as many up rows and TN tokens of 128
// bytes each.  The MMA reads 128 rows whatever there is of them; the rest lands in accumulator rows nobody looks at.
template <int TN, bool WIDE> struct SplitSmem {
  static constexpr int kParts = 0;                                      // this CTA's tokens, [split][TN / split][128]
  static constexpr int kBarriers = kParts + (WIDE ? 0 : TN * BM * 4); // full[16], empty[16], tfull
  static constexpr int kTmemPtr = kBarriers + (2 * kSplitMaxStages + 1) * 8;
  static constexpr int kAbort = kTmemPtr + 4;
  static constexpr int kLargest = kAbort + 4;
  static constexpr int kRing = (kLargest + 4 + 1023) / 1024 * 1024;
  static constexpr int stage_bytes(int channels) { return ((channels + 7) / 8 * 16 + TN) * BK_BYTES; }
  static constexpr int total(int channels, int stages) { return kRing + stages * stage_bytes(channels) + BM * BK_BYTES + 1024; }
};

// WIDE: up to 128 channels, gate and up rows each as a 128-row operand with an accumulator of its own; a lane then holds both of
// its channel, and nothing is shared out.  For 33 to 128 tokens, where one wave of CTAs has to take more than 64 channels each to
// read the weights once.
template <typename T, int TN, bool BACKWARD, bool WIDE>
__global__ void __launch_bounds__(kSplitThreads<WIDE>)
gated_split_kernel(const __grid_constant__ CUtensorMap map_gate, const __grid_constant__ CUtensorMap map_up, const __grid_constant__ CUtensorMap map_x,
                   const SplitArgs args, int channels, int stages, int split_log2) {
  using L = SplitSmem<TN, WIDE>;
  constexpr int TN_LOG2 = TN == 16 ? 4 : (TN == 32 ? 5 : (TN == 64 ? 6 : 7));
  constexpr uint32_t kTmemCols = WIDE ? 2 * TN : (TN < 32 ? 32 : TN);
  const int c8 = (channels + 7) / 8 * 8, stage_bytes = L::stage_bytes(channels), x_off = stage_bytes - TN * BK_BYTES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t smem_base = smem_u32(smem), bar_base = smem_base + L::kBarriers;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (kSplitMaxStages + s); };
  const uint32_t tfull_bar = bar_base + 8u * (2 * kSplitMaxStages);
  volatile uint32_t *tmem_ptr_smem = reinterpret_cast<volatile uint32_t *>(smem + L::kTmemPtr);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::kAbort);
  float *largest = reinterpret_cast<float *>(smem + L::kLargest);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int split = 1 << split_log2;
  const int rank = blockIdx.x & (split - 1), tile = blockIdx.x >> split_log2;
  const int ct = tile % args.tiles_c, xt = tile / args.tiles_c;
  const int kb0 = (int)((long long)args.num_kb * rank / split), kb1 = (int)((long long)args.num_kb * (rank + 1) / split);

  if (BACKWARD) dependents_may_start();
  constexpr bool RANGED = BACKWARD && kRanged<T>;
  float scale = pow2(kFirstExponent), top = 0.f;
  if (RANGED && args.again) {
    wait_for_results();
    const float seen = largest_of(args.largest, gridDim.x, lane);
    if (first_exponent_fits(seen)) return; // all CTAs alike
    scale = pow2(range_exponent(seen));
  }
  auto met = [&](float vg, float vu) { // values of dG and dU
    const float m = fmaxf(fabsf(vg), fabsf(vu));
    if constexpr (RANGED) top = fmaxf(top, m < INFINITY ? m : fminf(fabsf(vg), fabsf(vu)) < INFINITY ? fminf(fabsf(vg), fabsf(vu)) : 0.f);
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; s++) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(tfull_bar, 1);
    *abort_flag = 0;
    *largest = 0.f;
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
    for (int kb = kb0; kb < kb1; kb++) {
      if (!warp_wait(empty_bar(stage), phase ^ 1, abort_flag, args.status, ST_TIMEOUT_EMPTY)) { ok = false; break; }
      if (elect_one()) {
        const uint32_t dst = smem_base + L::kRing + stage * stage_bytes;
        mbar_expect_tx(full_bar(stage), (uint32_t)(2 * channels + TN) * BK_BYTES);
        tma_load_2d(dst, &map_gate, full_bar(stage), kb * 64, ct * channels);
        tma_load_2d(dst + c8 * BK_BYTES, &map_up, full_bar(stage), kb * 64, ct * channels);
        tma_load_2d(dst + x_off, &map_x, full_bar(stage), kb * 64, xt * TN);
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
    const uint32_t idesc = f16_idesc<T>(BM, TN, false, false);
    int stage = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; kb++) {
      if (!warp_wait(full_bar(stage), phase, abort_flag, args.status, ST_TIMEOUT_FULL)) break;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t a = smem_base + L::kRing + stage * stage_bytes;
        const uint64_t adesc = make_smem_desc(a), bdesc = make_smem_desc(a + x_off);
#pragma unroll
        for (int k = 0; k < 4; k++) {
          tc_mma<KIND_F16>(tmem_base, adesc + 2 * k, bdesc + 2 * k, idesc, (kb > kb0 || k) ? 1u : 0u);
          if (WIDE) tc_mma<KIND_F16>(tmem_base + TN, make_smem_desc(a + c8 * BK_BYTES) + 2 * k, bdesc + 2 * k, idesc, (kb > kb0 || k) ? 1u : 0u);
        }
        tc_commit(empty_bar(stage));
      }
      __syncwarp();
      if (++stage == stages) { stage = 0; phase ^= 1; }
    }
    // every MMA issued above is done with shared and tensor memory before this warp goes on, after an abort too
    if (elect_one()) tc_commit(tfull_bar);
    __syncwarp();
    if (!bounded_wait(tfull_bar, 0) && lane == 0) atomicCAS(args.status, 0, ST_TIMEOUT_DRAIN);
    if (split > 1) cluster_wait();
  } else if (WIDE) {
    // ------------------------------------------------------------------ the accumulators (warps 2..9): a channel a lane, every
    // other 16 tokens a warp
    const int quad = warp & 3, row = quad * 32 + lane, ch = ct * channels + row;
    const bool mine = row < channels && ch < args.I;
    const T *dh = static_cast<const T *>(args.dh);
    T *out = static_cast<T *>(args.out), *out2 = static_cast<T *>(args.out2);
    warp_wait(tfull_bar, 0, abort_flag, args.status, ST_TIMEOUT_TMEM_FULL);
    tc_fence_after();
    const int tokens = min(TN, args.M - xt * TN);
    with_act(args.act, [&](auto act) {
#pragma unroll 1
      for (int c = (warp - 2) >> 2; c * 16 < tokens && quad * 32 < channels; c += 2) {
        uint32_t g[16], u[16];
        float d[16];
        const size_t at = (size_t)(xt * TN + c * 16) * (size_t)args.I + ch;
        if constexpr (BACKWARD) {
#pragma unroll
          for (int j = 0; j < 16; j++) d[j] = mine && c * 16 + j < tokens ? FloatIO<T>::to_f32(dh[at + (size_t)j * (size_t)args.I]) * (RANGED ? scale : 1.f) : 0.f;
        }
        tmem_load_16(tmem_base + ((uint32_t)(quad * 32) << 16) + c * 16, g);
        tmem_load_16(tmem_base + ((uint32_t)(quad * 32) << 16) + TN + c * 16, u);
#pragma unroll
        for (int j = 0; j < 16; j++) {
          const float z = __uint_as_float(g[j]), up = __uint_as_float(u[j]);
          const bool on = mine && c * 16 + j < tokens;
          if constexpr (BACKWARD) {
            float a, da;
            act_both<decltype(act)::value>(z, a, da);
            if (on) {
              const size_t i = at + (size_t)j * (size_t)args.I;
              const float vg = d[j] * up * da, vu = d[j] * a;
              met(vg, vu);
              out[i] = FloatIO<T>::from_f32(vg);
              out2[i] = FloatIO<T>::from_f32(vu);
              if (args.layers == 2) {
                out[i + (size_t)args.M * (size_t)args.I] = FloatIO<T>::from_f32(remainder_of<T>(vg));
                out2[i + (size_t)args.M * (size_t)args.I] = FloatIO<T>::from_f32(remainder_of<T>(vu));
              }
            }
          } else {
            const float h = act_value<decltype(act)::value>(z) * up;
            if (on) out[at + (size_t)j * (size_t)args.I] = FloatIO<T>::from_f32(h);
          }
        }
      }
    });
    tc_fence_before();
  } else {
    // ------------------------------------------------------------------ the accumulator (warps 2..5)
    const int quad = warp & 3, row = quad * 32 + lane;
    warp_wait(tfull_bar, 0, abort_flag, args.status, ST_TIMEOUT_TMEM_FULL);
    tc_fence_after();
    const int tokens = min(TN, args.M - xt * TN), per_log2 = TN_LOG2 - split_log2, per = 1 << per_log2; // CTA o adds up tokens [o * per, (o + 1) * per)
    if (split > 1) cluster_wait();
#pragma unroll 1
    for (int c = 0; c < TN / 16; c++) {
      if (c * 16 >= tokens) break;
      uint32_t r[16];
      tmem_load_16(tmem_base + ((uint32_t)(quad * 32) << 16) + c * 16, r);
#pragma unroll
      for (int j = 0; j < 16; j++) {
        const int t = c * 16 + j;
        if (t < tokens) {
          const uint32_t local = smem_base + (uint32_t)(L::kParts + ((rank * per + (t & (per - 1))) * BM + row) * 4);
          if (split > 1) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(map_to_cta(local, (uint32_t)(t >> per_log2))), "f"(__uint_as_float(r[j])) : "memory");
          else asm volatile("st.shared.f32 [%0], %1;" ::"r"(local), "f"(__uint_as_float(r[j])) : "memory");
        }
      }
    }
    tc_fence_before();
  }
  if (split > 1 && warp == 0) cluster_wait();
  __syncthreads();
  if (split > 1) cluster_sync_all(); // every part has arrived
  if constexpr (!WIDE) {
    constexpr int kThreads = kSplitThreads<WIDE>;
    const int per = TN >> split_log2, t0 = rank * per, t1 = min(t0 + per, args.M - xt * TN);
    const float *parts = reinterpret_cast<const float *>(smem + L::kParts);
    T *out = static_cast<T *>(args.out), *out2 = static_cast<T *>(args.out2);
    const int here = min(channels, args.I - ct * channels), items = (t1 - t0) * here;
    with_act(args.act, [&](auto act) {
      constexpr int U = BACKWARD ? 4 : 1; // values a thread works on at once, where it has dH to wait for
      for (int i0 = threadIdx.x; i0 < items; i0 += U * kThreads) {
        float g[U], u[U], d[U];
        size_t at[U];
#pragma unroll
        for (int k = 0; k < U; k++) {
          const int i = min(i0 + k * kThreads, items - 1), t = i / here, ch = i - t * here;
          at[k] = (size_t)(xt * TN + t0 + t) * (size_t)args.I + ct * channels + ch;
          if constexpr (BACKWARD) d[k] = FloatIO<T>::to_f32(static_cast<const T *>(args.dh)[at[k]]) * (RANGED ? scale : 1.f);
          g[k] = u[k] = 0.f;
#pragma unroll
          for (int p = 0; p < kMaxSplit; p++) {
            if (p < split) {
              g[k] += parts[(p * per + t) * BM + ch];
              u[k] += parts[(p * per + t) * BM + c8 + ch];
            }
          }
        }
#pragma unroll
        for (int k = 0; k < U; k++) {
          if (i0 + k * kThreads >= items) break;
          if constexpr (BACKWARD) {
            float a, da;
            act_both<decltype(act)::value>(g[k], a, da);
            const float vg = d[k] * u[k] * da, vu = d[k] * a;
            met(vg, vu);
            out[at[k]] = FloatIO<T>::from_f32(vg);
            out2[at[k]] = FloatIO<T>::from_f32(vu);
            if (args.layers == 2) {
              out[at[k] + (size_t)args.M * (size_t)args.I] = FloatIO<T>::from_f32(remainder_of<T>(vg));
              out2[at[k] + (size_t)args.M * (size_t)args.I] = FloatIO<T>::from_f32(remainder_of<T>(vu));
            }
          } else {
            out[at[k]] = FloatIO<T>::from_f32(act_value<decltype(act)::value>(g[k]) * u[k]);
          }
        }
      }
    });
  }
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
  }
  if (RANGED && !args.again) {
    __syncwarp();
    const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
    if (lane == 0) atomicMax(reinterpret_cast<uint32_t *>(largest), bits);
    __syncthreads();
    if (threadIdx.x == 0) args.largest[blockIdx.x] = *largest;
  }
}

// ----------------------------------------------------------------------------------------------
// host side
// ----------------------------------------------------------------------------------------------
template <typename T> constexpr int kMapKind = FloatIO<T>::kDtype == QL_BF16 ? KIND_BF16 : KIND_F16;

// 16-bit operand [layers, rows, cols], box = [box_rows, 64 columns], 128-byte swizzle: encode_map's with layers
int encode_map_layers(CUtensorMap *map, int dtype, const void *ptr, int64_t layers, int64_t rows, int64_t cols, int box_rows) {
  EncodeTiledFn enc;
  const int rc = get_encode_fn(&enc);
  if (rc != QL_OK) return rc;
  cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)layers};
  cuuint64_t strides[2] = {(cuuint64_t)cols * 2, (cuuint64_t)(rows * cols) * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = enc(map, dtype == QL_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(ptr), dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(QL_ERR_CUDA, "cuTensorMapEncodeTiled (layers) failed with code %d", (int)r);
  return QL_OK;
}

template <typename K> int resident(K kern, int threads, int smem, int cluster) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * sm_count() * cluster), 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)cluster, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n < 1) {
    cudaGetLastError();
    n = sm_count() / cluster;
  }
  return n;
}
// clusters (of `cluster` CTAs, one CTA per SM) of a kernel the current device holds at once; asked once
template <typename K> int resident_cached(K kern, int threads, int smem, int cluster, int (&cache)[64]) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return sm_count() / cluster;
  if (cache[dev] == 0) cache[dev] = resident(kern, threads, smem, cluster);
  return cache[dev];
}

// A band of rows of A stays L2-resident: about 32 MiB of it, four row tiles of 256 at the least.  4096 x 28672 x 8192: bands
// of 16, 32, 64 and 128 MiB 3.00, 2.78, 2.81 and 2.83 ms; 4096 x 11008 x 4096: 522, 501, 504 and 509 us.
int band(int64_t row_bytes, int tiles_m) {
  int64_t g = (32ll << 20) / (256 * row_bytes);
  g = g < 4 ? 4 : g;
  return (int)(g > tiles_m ? (tiles_m < 1 ? 1 : tiles_m) : g);
}

struct SplitPlan {
  int co, log2, channels, stages;
  double us;
};

template <typename T, int TN, bool BACKWARD, bool WIDE> int allow_split() {
  static bool configured[64] = {false};
  return allow_smem(gated_split_kernel<T, TN, BACKWARD, WIDE>, 232448, configured);
}
template <typename T, bool BACKWARD, int C> int allow_pair() {
  static bool configured[64] = {false};
  return allow_smem(gated_pair_kernel<T, BACKWARD, C>, PairSmem::kDynamic, configured);
}
template <typename T, bool BACKWARD, int C> int resident_pairs() {
  static int cache[64] = {0};
  return resident_cached(gated_pair_kernel<T, BACKWARD, C>, kPairThreads, PairSmem::kDynamic, 2, cache);
}

// (the occupancy query needs allow_split first)
template <typename T, int TN, bool BACKWARD> SplitPlan plan_split(int M, int I, int num_kb) {
  using L = SplitSmem<TN, false>;
  static int cache[4][64] = {};
  const int64_t tiles_x = (M + TN - 1) / TN;
  SplitPlan best = {1, 0, 64, 1, 1e30};
  for (int co = 1; co <= (TN <= 32 ? 2 : 1); co++) {
    for (int log2 = 0; log2 < 4 && (log2 == 0 || num_kb >= (4 << log2)); log2++) {
      const int fit = resident_cached(gated_split_kernel<T, TN, BACKWARD, false>, kSplitThreads<false>, 232448, 1 << log2, cache[log2]) * co;
      const int64_t per_x = fit / tiles_x, want = per_x < 1 ? 64 : (I + per_x - 1) / per_x;
      const int channels = (int)(want > 64 ? 64 : (want < 8 ? 8 : want));
      const int64_t tiles = (int64_t)((I + channels - 1) / channels) * tiles_x, waves = (tiles + fit - 1) / fit;
      const int steps = (num_kb + (1 << log2) - 1) >> log2;
      const double latency = 0.2 + 0.0029 * (TN - 16), bandwidth = (double)(2 * channels + TN) * BK_BYTES * co / 48e3;
      const double epilogue = TN / 64.0 + 0.0014 * ((M < TN ? M : TN) * channels >> log2);
      const double us = (double)waves * (3.3 + 0.5 * (co - 1) + epilogue + (log2 ? 1.2 + 0.015 * TN : 0.0) + steps * (latency > bandwidth ? latency : bandwidth));
      if (us < best.us) {
        int stages = (232448 / co - 2048 - L::total(channels, 0)) / L::stage_bytes(channels);
        stages = stages > kSplitMaxStages ? kSplitMaxStages : stages;
        best = {co, log2, channels, stages > steps ? steps : stages, us};
      }
    }
  }
  return best;
}

// WIDE: as many channels a CTA as let one wave cover them, K whole, one CTA per SM.  5.3 us, 0.03 us per token to store, and per
// step of 64 values of K 0.30 us for its eight MMAs, or the weights' time at an SM's share of memory bandwidth.
template <int TN> SplitPlan plan_wide(int M, int I, int num_kb) {
  const int64_t fit = sm_count(), want = (I + fit - 1) / fit;
  const int channels = (int)(want > BM ? BM : (want < 8 ? 8 : want));
  const int64_t tiles = (I + channels - 1) / channels, waves = (tiles + fit - 1) / fit;
  const double memory = 2.0 * channels * BK_BYTES / 41.5e3, step = memory > 0.30 ? memory : 0.30;
  int stages = (232448 - 2048 - SplitSmem<TN, true>::total(channels, 0)) / SplitSmem<TN, true>::stage_bytes(channels);
  stages = stages > kSplitMaxStages ? kSplitMaxStages : stages;
  return {1, 0, channels, stages > num_kb ? num_kb : stages, (double)waves * (5.3 + 0.03 * M + num_kb * step)};
}

// The first stage: its operands, and by which kernel it is done.
struct Projection {
  const void *x, *wg, *wu, *dh;
  void *out, *out2;  // H, or dG and dU
  float *largest;    // as in ProjArgs
  int M, I, K, act;
};
struct Choice {
  int tokens;   // of the split kernels' tile; 0: pairs
  bool wide;    // split kernel
  int channels; // of the pairs' tile
  SplitPlan split;
  int ctas;
};

// Backward, kRanged: launched twice, the second time to be run where the first one's exponent did not fit.
template <typename T, bool BACKWARD, int C> int launch_pair(const Projection &p, const Choice &choice, cudaStream_t st) {
  auto kern = gated_pair_kernel<T, BACKWARD, C>;
  int rc = allow_pair<T, BACKWARD, C>();
  if (rc != QL_OK) return rc;
  ProjArgs a;
  a.dh = p.dh;
  a.M = p.M, a.I = p.I, a.K = p.K, a.act = p.act;
  a.layers = grad_layers(p.M, p.I, p.K);
  a.largest = p.largest;
  a.num_kb = (p.K + 63) / 64;
  a.tiles_m = (p.M + 255) / 256;
  a.tiles_n = (p.I + C - 1) / C;
  a.group_m = band((int64_t)p.K * 2, a.tiles_m);
  a.status = device_status_word();
  if (!a.status) return set_error(QL_ERR_CUDA, "gated_linear: could not allocate the device status word");
  CUtensorMap mx, mg, mu, mo, mo2;
  const int kind = kMapKind<T>, dtype = FloatIO<T>::kDtype;
  if ((rc = encode_map(&mx, kind, p.x, p.M, p.K, 128)) != QL_OK) return rc;
  if ((rc = encode_map(&mg, kind, p.wg, p.I, p.K, C)) != QL_OK) return rc;
  if ((rc = encode_map(&mu, kind, p.wu, p.I, p.K, C)) != QL_OK) return rc;
  if ((rc = encode_map_narrow(&mo, dtype, p.out, p.M, p.I, BACKWARD ? a.layers : 0)) != QL_OK) return rc;
  mo2 = mo; // forward: not used
  if (BACKWARD && (rc = encode_map_narrow(&mo2, dtype, p.out2, p.M, p.I, a.layers)) != QL_OK) return rc;
  for (a.again = 0; a.again < (BACKWARD && kRanged<T> ? 2 : 1); a.again++) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)choice.ctas, 1, 1);
    cfg.blockDim = dim3(kPairThreads, 1, 1);
    cfg.dynamicSmemBytes = PairSmem::kDynamic;
    cfg.stream = st;
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &early;
    cfg.numAttrs = a.again;
    QL_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, mx, mg, mu, mo, mo2, a));
    count_launches(1);
  }
  return QL_OK;
}
template <typename T, int TN, bool BACKWARD, bool WIDE> int launch_split(const Projection &p, const Choice &choice, cudaStream_t st) {
  using L = SplitSmem<TN, WIDE>;
  int rc = allow_split<T, TN, BACKWARD, WIDE>();
  if (rc != QL_OK) return rc;
  const SplitPlan &plan = choice.split;
  SplitArgs a;
  a.dh = p.dh, a.out = p.out, a.out2 = p.out2;
  a.M = p.M, a.I = p.I, a.act = p.act, a.layers = grad_layers(p.M, p.I, p.K);
  a.largest = p.largest;
  a.num_kb = (p.K + 63) / 64;
  a.tiles_c = (p.I + plan.channels - 1) / plan.channels;
  a.status = device_status_word();
  if (!a.status) return set_error(QL_ERR_CUDA, "gated_linear: could not allocate the device status word");
  CUtensorMap mg, mu, mx;
  const int kind = kMapKind<T>;
  if ((rc = encode_map(&mg, kind, p.wg, p.I, p.K, plan.channels)) != QL_OK) return rc;
  if ((rc = encode_map(&mu, kind, p.wu, p.I, p.K, plan.channels)) != QL_OK) return rc;
  if ((rc = encode_map(&mx, kind, p.x, p.M, p.K, TN)) != QL_OK) return rc;
  for (a.again = 0; a.again < (BACKWARD && kRanged<T> ? 2 : 1); a.again++) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)choice.ctas, 1, 1);
    cfg.blockDim = dim3(kSplitThreads<WIDE>, 1, 1);
    cfg.dynamicSmemBytes = L::total(plan.channels, plan.stages);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1u << plan.log2, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1 + a.again;
    QL_CUDA_TRY(cudaLaunchKernelEx(&cfg, gated_split_kernel<T, TN, BACKWARD, WIDE>, mg, mu, mx, a, plan.channels, plan.stages, plan.log2));
    count_launches(1);
  }
  return QL_OK;
}

// The two projections, by whichever kernel is estimated the faster: pairs take 7.2 us and 0.28 us per tile of 128 channels and 64
// values of K, or 5.2 and 0.23 per tile of 64 channels (half the MMAs and half the epilogue, but as many rows of X to load), or
// what a wave's weights take at 6 TB/s, and 0.3 (0.8) for every further tile; the split kernels what plan_split and plan_wide say.  Up to 32 tokens a pair's 256 rows
// are mostly padding.  Forward, us (M x I x K):
//   256 x 512 x 4096    split 14.4, pairs 24.9     |  2314 x 80 x 6296  split 24.8, pairs 38.8
//   211 x 2744 x 1032   split 20.9, pairs 13.3, of 64 channels 10.5  |  256 x 9472 x 4096  pairs 36.1, of 64 channels 41.7
//   128 x 11008 x 4096  pairs 50.1, wide split 39.4  |  64 x 11008 x 4096  pairs 50.1, wide split 36.0
//   128 x 9472 x 2048   pairs 19.8, wide split 21.9  |  512 x 2368 x 4096  pairs 25.9, of 64 channels 20.9
template <typename T, bool BACKWARD> Choice choose(int M, int I, int K) {
  const int num_kb = (K + 63) / 64;
  auto pairs_us = [&](int c, double fixed, double step, double next) {
    const int64_t pairs = sm_count() / 2, rows = (M + 255) / 256, tiles = rows * ((I + c - 1) / c), rest = tiles % pairs;
    const double bytes = 2.0 * c * BK_BYTES / (double)rows; // of weights from memory, per step and pair; other row tiles find them in L2
    auto wave = [&](int64_t n) { return n == 0 ? 0.0 : (step > bytes * (double)n / 6e6 ? step : bytes * (double)n / 6e6); };
    return fixed + next * (double)((tiles - 1) / pairs) + num_kb * ((double)(tiles / pairs) * wave(pairs) + wave(rest));
  };
  const double full_us = pairs_us(128, 7.2, 0.28, 0.3), narrow_us = pairs_us(64, 5.2, 0.23, 0.8);
  const bool narrow = narrow_us < full_us;
  const double pair_us = M <= 32 ? 1e30 : (narrow ? narrow_us : full_us);
  Choice ch = {};
  // the split kernel of TN tokens, where its estimate is no larger than `limit_us`
  auto split = [&](auto tn, auto wide, double limit_us) {
    constexpr int TN = decltype(tn)::value;
    constexpr bool WIDE = decltype(wide)::value;
    allow_split<T, TN, BACKWARD, WIDE>(); // where it fails, so does the launch
    if constexpr (WIDE) ch.split = plan_wide<TN>(M, I, num_kb);
    else ch.split = plan_split<T, TN, BACKWARD>(M, I, num_kb);
    ch.tokens = ch.split.us <= limit_us ? TN : 0, ch.wide = WIDE;
    ch.ctas = (int)(((int64_t)((I + ch.split.channels - 1) / ch.split.channels) * ((M + TN - 1) / TN)) << ch.split.log2);
    return ch.tokens != 0;
  };
  auto either = [&](auto tn) { // split or wide
    const double wide_us = M <= 128 ? plan_wide<decltype(tn)::value>(M, I, num_kb).us : 1e30;
    return split(tn, std::false_type{}, pair_us < wide_us ? pair_us : wide_us) || (M <= 128 && split(tn, std::true_type{}, pair_us));
  };
  if (M <= 16) split(std::integral_constant<int, 16>{}, std::false_type{}, pair_us);
  else if (M <= 32) split(std::integral_constant<int, 32>{}, std::false_type{}, pair_us);
  else if (M <= 64) either(std::integral_constant<int, 64>{});
  else either(std::integral_constant<int, 128>{});
  if (ch.tokens == 0) {
    ch.channels = narrow ? 64 : 128;
    (void)(narrow ? allow_pair<T, BACKWARD, 64>() : allow_pair<T, BACKWARD, 128>());
    const int tiles = ((M + 255) / 256) * ((I + ch.channels - 1) / ch.channels);
    const int pairs = narrow ? resident_pairs<T, BACKWARD, 64>() : resident_pairs<T, BACKWARD, 128>();
    ch.ctas = 2 * (tiles < pairs ? tiles : pairs);
  }
  return ch;
}
template <typename T, bool BACKWARD> int project(const Projection &p, const Choice &ch, cudaStream_t st) {
  switch (ch.tokens) {
  case 16: return launch_split<T, 16, BACKWARD, false>(p, ch, st);
  case 32: return launch_split<T, 32, BACKWARD, false>(p, ch, st);
  case 64: return ch.wide ? launch_split<T, 64, BACKWARD, true>(p, ch, st) : launch_split<T, 64, BACKWARD, false>(p, ch, st);
  case 128: return ch.wide ? launch_split<T, 128, BACKWARD, true>(p, ch, st) : launch_split<T, 128, BACKWARD, false>(p, ch, st);
  default: return ch.channels == 64 ? launch_pair<T, BACKWARD, 64>(p, ch, st) : launch_pair<T, BACKWARD, 128>(p, ch, st);
  }
}

// f32 [layers, rows, cols], box = [1, 32 rows, 32 columns], 128-byte swizzle: a store is clipped at its own layer's edges
int encode_map_parts(CUtensorMap *map, const float *ptr, int64_t layers, int64_t rows, int64_t cols) {
  EncodeTiledFn enc;
  const int rc = get_encode_fn(&enc);
  if (rc != QL_OK) return rc;
  cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)layers};
  cuuint64_t strides[2] = {(cuuint64_t)cols * 4, (cuuint64_t)(rows * cols) * 4};
  cuuint32_t box[3] = {32, 32, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<float *>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(QL_ERR_CUDA, "cuTensorMapEncodeTiled (parts) failed with code %d", (int)r);
  return QL_OK;
}

int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }

template <typename T> int grad_pairs() {
  static bool configured[64] = {false};
  static int cache[64] = {0};
  if (allow_smem(gated_grads_kernel<T>, PairSmem::kDynamic, configured) != QL_OK) return sm_count() / 2;
  return resident_cached(gated_grads_kernel<T>, kPairThreads, PairSmem::kDynamic, 2, cache);
}
int pairs_of(int dtype) { return dtype == QL_BF16 ? grad_pairs<__nv_bfloat16>() : grad_pairs<__half>(); }

// A backward call: the first stage's kernel, the second's plan, and where things lie in the workspace.
struct BackwardPlan {
  Choice first;
  GradPlan grads;
  int64_t mi, x_parts, w_parts, largest, bytes; // offsets; dG at 0, dU at mi
};
BackwardPlan plan_backward(int dtype, int M, int I, int K, bool want_x, bool want_w) {
  BackwardPlan p;
  p.first = dtype == QL_BF16 ? choose<__nv_bfloat16, true>(M, I, K) : choose<__half, true>(M, I, K);
  p.grads = plan_grads(M, I, K, want_x, want_w, pairs_of(dtype));
  p.mi = align256((int64_t)p.grads.a.layers * M * I * 2);
  p.x_parts = 2 * p.mi;
  p.w_parts = p.x_parts + align256(p.grads.x_part_floats * 4);
  p.largest = p.w_parts + align256(p.grads.w_part_floats * 4);
  p.bytes = p.largest + (dtype == QL_F16 ? align256((int64_t)p.first.ctas * 4) : 0);
  return p;
}

template <typename T>
int backward(const void *dh, const void *x, const void *wg, const void *wu, void *dx, void *dwg, void *dwu, int M, int I, int K, int act, uint8_t *ws, const BackwardPlan &plan,
             cudaStream_t st) {
  void *dg = ws, *du = ws + plan.mi;
  float *largest = reinterpret_cast<float *>(ws + plan.largest);
  int rc = project<T, true>({x, wg, wu, dh, dg, du, largest, M, I, K, act}, plan.first, st);
  if (rc != QL_OK) return rc;
  GradArgs a = plan.grads.a;
  a.status = device_status_word();
  if (plan.grads.x_part_floats) a.x_parts = reinterpret_cast<float *>(ws + plan.x_parts);
  if (plan.grads.w_part_floats) a.w_parts = reinterpret_cast<float *>(ws + plan.w_parts);
  a.largest = largest, a.num_largest = plan.first.ctas;
  const int x_layers = a.x_split * a.layers;
  CUtensorMap dgk, duk, dgm, dum, wgm, wum, xm, mx, mg, mu;
  const int kind = kMapKind<T>, dtype = FloatIO<T>::kDtype;
  if ((rc = encode_map_layers(&dgk, dtype, dg, a.layers, M, I, 128)) != QL_OK) return rc;
  if ((rc = encode_map_layers(&duk, dtype, du, a.layers, M, I, 128)) != QL_OK) return rc;
  if ((rc = encode_map_layers(&dgm, dtype, dg, a.layers, M, I, 64)) != QL_OK) return rc;
  if ((rc = encode_map_layers(&dum, dtype, du, a.layers, M, I, 64)) != QL_OK) return rc;
  if ((rc = encode_map(&wgm, kind, wg, I, K, 64)) != QL_OK) return rc;
  if ((rc = encode_map(&wum, kind, wu, I, K, 64)) != QL_OK) return rc;
  if ((rc = encode_map(&xm, kind, x, M, K, 64)) != QL_OK) return rc;
  mx = mg = mu = xm; // what is not wanted is not written
  if (a.x_parts) rc = encode_map_parts(&mx, a.x_parts, x_layers, M, K);
  else if (dx) rc = encode_map_narrow(&mx, dtype, dx, M, K);
  if (rc != QL_OK) return rc;
  if (a.w_parts) rc = encode_map_parts(&mg, a.w_parts, 2 * a.w_split, I, K);
  else if (dwg && (rc = encode_map_narrow(&mg, dtype, dwg, I, K)) == QL_OK) rc = encode_map_narrow(&mu, dtype, dwu, I, K);
  if (rc != QL_OK) return rc;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * plan.grads.clusters), 1, 1);
  cfg.blockDim = dim3(kPairThreads, 1, 1);
  cfg.dynamicSmemBytes = PairSmem::kDynamic;
  cfg.stream = st;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  QL_CUDA_TRY(cudaLaunchKernelEx(&cfg, gated_grads_kernel<T>, dgk, duk, dgm, dum, wgm, wum, xm, mx, mg, mu, a));
  count_launches(1);
  if (a.x_parts || a.w_parts) {
    const int64_t nx4 = (int64_t)M * K / 4, nw4 = (int64_t)I * K / 4, n = (a.x_parts ? nx4 : 0) + (a.w_parts ? 2 * nw4 : 0);
    const int split = a.x_parts && a.w_parts ? (x_layers > a.w_split ? x_layers : a.w_split) : (a.x_parts ? x_layers : a.w_split);
    const int64_t room = (int64_t)sm_count() * 2048; // threads the device holds
    int slices_log2 = 0;
    while (slices_log2 < 3 && (2 << slices_log2) <= split && (n << (slices_log2 + 1)) <= room) slices_log2++;
    const int64_t per = kReduceThreads >> slices_log2, blocks = (n + per - 1) / per, cap = room / kReduceThreads;
    cfg.gridDim = dim3((unsigned)(blocks < cap ? blocks : cap), 1, 1);
    cfg.blockDim = dim3(kReduceThreads, 1, 1);
    cfg.dynamicSmemBytes = 0;
    QL_CUDA_TRY(cudaLaunchKernelEx(&cfg, grads_reduce_kernel<T>, reinterpret_cast<const float4 *>(a.x_parts), x_layers, static_cast<T *>(dx), nx4,
                                   reinterpret_cast<const float4 *>(a.w_parts), a.w_split, static_cast<T *>(dwg), static_cast<T *>(dwu), nw4, slices_log2));
    count_launches(1);
  }
  return QL_OK;
}

// Shapes and types of x [M,K], the two weights [I,K] and a matrix [M,I].
int check_gated(const char *op, const ql_tensor *x, const ql_tensor *wg, const ql_tensor *wu, const ql_tensor *h, const char *h_name, int act) {
  const ql_tensor *t[4] = {x, wg, wu, h};
  const char *name[4] = {"x", "w_gate", "w_up", h_name};
  for (int i = 0; i < 4; i++) {
    if (!t[i]) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: %s is null", op, name[i]);
    if (t[i]->rank != 2 || t[i]->shape[0] < 0 || t[i]->shape[1] < 0) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: %s must be a 2-D tensor", op, name[i]);
    if (t[i]->dtype != QL_F16 && t[i]->dtype != QL_BF16) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: %s must be f16 or bf16", op, name[i]);
    if (t[i]->dtype != x->dtype) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: %s and x must be of one type", op, name[i]);
    if (t[i]->shape[0] > (1 << 30) || t[i]->shape[1] > (1 << 30)) return set_error(QL_ERR_UNSUPPORTED, "%s: dimension of %s too large", op, name[i]);
  }
  if (act < ACT_SILU || act > ACT_RELU) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: unknown activation %d", op, act);
  const int64_t M = x->shape[0], K = x->shape[1], I = wg->shape[0];
  if (wg->shape[1] != K || wu->shape[0] != I || wu->shape[1] != K)
    return set_error(QL_ERR_INVALID_ARGUMENT, "%s: w_gate and w_up must both be [I,K] with K = %lld", op, (long long)K);
  if (h->shape[0] != M || h->shape[1] != I) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: %s must be [M,I] = [%lld,%lld]", op, h_name, (long long)M, (long long)I);
  for (int i = 0; i < 4; i++) {
    if (numel(t[i]) > 0 && !t[i]->data) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: %s has no data pointer", op, name[i]);
    if (!aligned16(t[i]->data)) return set_error(QL_ERR_UNSUPPORTED, "%s: %s must be 16-byte aligned", op, name[i]);
  }
  if (K % 8 != 0 || I % 8 != 0) return set_error(QL_ERR_UNSUPPORTED, "%s: needs K (%lld) and I (%lld) to be multiples of 8", op, (long long)K, (long long)I);
  return QL_OK;
}

} // namespace
} // namespace ql

using namespace ql;

extern "C" int ql_gated_linear(const ql_tensor *x, const ql_tensor *w_gate, const ql_tensor *w_up, int32_t activation, ql_tensor *h, void *stream) {
  const char *op = "gated_linear";
  const int rc = check_gated(op, x, w_gate, w_up, h, "h", activation);
  if (rc != QL_OK) return rc;
  const int M = (int)x->shape[0], K = (int)x->shape[1], I = (int)w_gate->shape[0];
  cudaStream_t st = (cudaStream_t)stream;
  if (M == 0 || I == 0) return QL_OK;
  if (overlap(h, x) || overlap(h, w_gate) || overlap(h, w_up)) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: h must not overlap an operand", op);
  if (K == 0) { // act(0) * 0
    QL_CUDA_TRY(cudaMemsetAsync(h->data, 0, (size_t)numel(h) * 2, st));
    return QL_OK;
  }
  const Projection p = {x->data, w_gate->data, w_up->data, nullptr, h->data, nullptr, nullptr, M, I, K, activation};
  return x->dtype == QL_BF16 ? project<__nv_bfloat16, false>(p, choose<__nv_bfloat16, false>(M, I, K), st) : project<__half, false>(p, choose<__half, false>(M, I, K), st);
}

extern "C" int ql_gated_linear_backward_workspace(const ql_tensor *x, const ql_tensor *w_gate, int32_t want_dx, int32_t want_dw, int64_t *bytes) {
  const char *op = "gated_linear_backward_workspace";
  if (!x || !w_gate || !bytes || x->rank != 2 || w_gate->rank != 2) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: needs x [M,K], w_gate [I,K] and a place for the size", op);
  const int64_t M = x->shape[0], K = x->shape[1], I = w_gate->shape[0];
  if (M < 0 || K < 0 || I < 0 || M > (1 << 30) || K > (1 << 30) || I > (1 << 30)) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: bad shape", op);
  *bytes = 0;
  if (M == 0 || K == 0 || I == 0) return QL_OK;
  *bytes = plan_backward(x->dtype, (int)M, (int)I, (int)K, want_dx != 0, want_dw != 0).bytes;
  return QL_OK;
}

extern "C" int ql_gated_linear_backward(const ql_tensor *grad, const ql_tensor *x, const ql_tensor *w_gate, const ql_tensor *w_up, int32_t activation, ql_tensor *dx,
                                        ql_tensor *dw_gate, ql_tensor *dw_up, void *workspace, int64_t workspace_bytes, void *stream) {
  const char *op = "gated_linear_backward";
  int rc = check_gated(op, x, w_gate, w_up, grad, "grad", activation);
  if (rc != QL_OK) return rc;
  if ((dw_gate == nullptr) != (dw_up == nullptr)) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: dw_gate and dw_up go together", op);
  const ql_tensor *out[3] = {dx, dw_gate, dw_up}, *like[3] = {x, w_gate, w_up};
  const char *name[3] = {"dx", "dw_gate", "dw_up"};
  for (int i = 0; i < 3; i++) {
    if (!out[i]) continue;
    if (out[i]->dtype != x->dtype || out[i]->rank != 2 || out[i]->shape[0] != like[i]->shape[0] || out[i]->shape[1] != like[i]->shape[1])
      return set_error(QL_ERR_INVALID_ARGUMENT, "%s: %s must have the type and shape of what it is the gradient of", op, name[i]);
    if (numel(out[i]) > 0 && !out[i]->data) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: %s has no data pointer", op, name[i]);
    if (!aligned16(out[i]->data)) return set_error(QL_ERR_UNSUPPORTED, "%s: %s must be 16-byte aligned", op, name[i]);
  }
  const int M = (int)x->shape[0], K = (int)x->shape[1], I = (int)w_gate->shape[0];
  cudaStream_t st = (cudaStream_t)stream;
  if (M == 0 || I == 0 || K == 0) { // sums over nothing
    for (int i = 0; i < 3; i++)
      if (out[i] && numel(out[i]) > 0) QL_CUDA_TRY(cudaMemsetAsync(out[i]->data, 0, (size_t)numel(out[i]) * 2, st));
    return QL_OK;
  }
  if (!dx && !dw_gate) return QL_OK;
  const BackwardPlan plan = plan_backward(x->dtype, M, I, K, dx != nullptr, dw_gate != nullptr);
  if (!workspace || workspace_bytes < plan.bytes)
    return set_error(QL_ERR_INVALID_ARGUMENT, "%s: needs a workspace of %lld bytes, got %lld", op, (long long)plan.bytes, (long long)(workspace ? workspace_bytes : 0));
  if (reinterpret_cast<uintptr_t>(workspace) & 255) return set_error(QL_ERR_UNSUPPORTED, "%s: the workspace must be 256-byte aligned", op);
  const ql_tensor *in[4] = {grad, x, w_gate, w_up};
  const ql_tensor scratch = workspace_view(workspace, plan.bytes);
  for (int i = 0; i < 4; i++)
    if (overlap(&scratch, in[i]) || (i < 3 && overlap(&scratch, out[i]))) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: the workspace must not overlap an operand or a gradient", op);
  for (int i = 0; i < 3; i++) {
    for (int j = 0; j < 4; j++)
      if (overlap(out[i], in[j])) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: %s must not overlap an operand", op, name[i]);
    for (int j = 0; j < i; j++)
      if (overlap(out[i], out[j])) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: %s and %s must not overlap", op, name[j], name[i]);
  }
  if (!device_status_word()) return set_error(QL_ERR_CUDA, "%s: could not allocate the device status word", op);
  void *p[3] = {dx ? dx->data : nullptr, dw_gate ? dw_gate->data : nullptr, dw_up ? dw_up->data : nullptr};
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  return x->dtype == QL_BF16 ? backward<__nv_bfloat16>(grad->data, x->data, w_gate->data, w_up->data, p[0], p[1], p[2], M, I, K, activation, ws, plan, st)
                             : backward<__half>(grad->data, x->data, w_gate->data, w_up->data, p[0], p[1], p[2], M, I, K, activation, ws, plan, st);
}
