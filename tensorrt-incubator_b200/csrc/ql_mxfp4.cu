// MXFP4 (the OCP microscaling format: e2m1 data, one e8m0 scale per block of 32 along the last axis): quantize and its
// inverse.  With m = max|block| the scale is 2^(floor(log2 m) - 2) -- the largest power of two for which m lands on e2m1's
// top binade [4, 8) -- and the data are x / scale, rounded half to even and saturated at 6.  For a normal f32 m the biased
// exponent of m, less 2, IS the scale's byte; zeros and subnormal m clamp to byte 0 (2^-127), infinities and NaN to 0xFF.
// x / scale is a multiplication by 2^(127 - byte), exact in f32 unless the quotient is far below e2m1's smallest step, so
// the only rounding is the conversion's.
//
// Both kernels are streams: 2 (or 4) bytes in and 17/32 out per value, and the reverse.  Four lanes share a block, eight
// values each: a 16-bit lane moves 16 bytes in and 4 out (an f32 lane 32 and 4), so every warp access is contiguous, and
// the block maximum is two shuffles.  One thread per block (as NVFP4's blocks of 16 have it) would read with a stride of 64
// or 128 bytes between lanes.
#include "ql_common.cuh"

namespace ql {
namespace {

constexpr int kMxThreads = 256;
constexpr int kMxBlock = 32;

// Eight floating-point values as they lie in memory.
template <typename T> struct Raw8 { uint4 w[sizeof(T) / 2]; };

template <typename T> __device__ __forceinline__ Raw8<T> load_raw8(const T *p) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; i++) r.w[i] = __ldcs(reinterpret_cast<const uint4 *>(p) + i);
  return r;
}
// f32 bit pattern of the largest magnitude (NaN patterns are the largest of all)
__device__ __forceinline__ uint32_t absmax_bits(const Raw8<float> &r) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const uint32_t w[4] = {r.w[i].x, r.w[i].y, r.w[i].z, r.w[i].w};
#pragma unroll
    for (int j = 0; j < 4; j++) m = max(m, w[j] & 0x7FFFFFFFu);
  }
  return m;
}
template <typename T> __device__ __forceinline__ uint32_t absmax_bits16(const Raw8<T> &r) {
  // 16-bit magnitudes order like their patterns, two at a time
  const uint32_t a = __vmaxu2(r.w[0].x & 0x7FFF7FFFu, r.w[0].y & 0x7FFF7FFFu), b = __vmaxu2(r.w[0].z & 0x7FFF7FFFu, r.w[0].w & 0x7FFF7FFFu);
  const uint32_t c = __vmaxu2(a, b);
  return max(c & 0xFFFFu, c >> 16);
}
__device__ __forceinline__ uint32_t absmax_bits(const Raw8<__nv_bfloat16> &r) { return absmax_bits16(r) << 16; }
__device__ __forceinline__ uint32_t absmax_bits(const Raw8<__half> &r) {
  return __float_as_uint(__half2float(__ushort_as_half((unsigned short)absmax_bits16(r))));
}

__device__ __forceinline__ uint32_t e2m1x2(float lo, float hi) {
  uint32_t r;
  asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %2, %1;\n\tcvt.u32.u8 %0, t;\n\t}" : "=r"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 e2m1x2_to_f32(uint32_t byte) {
  uint32_t h2;
  asm("{\n\t.reg .b8 t;\n\tcvt.u8.u32 t, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}" : "=r"(h2) : "r"(byte));
  return __half22float2(*reinterpret_cast<__half2 *>(&h2));
}
// 2^(byte - 127); byte 0 is the subnormal 2^-127, 0xFF is NaN
__device__ __forceinline__ float e8m0_to_f32(uint32_t byte) {
  const uint32_t bits = byte == 0 ? 0x00400000u : (byte == 0xFFu ? 0x7FC00000u : byte << 23);
  return __uint_as_float(bits);
}

constexpr int kMxUnroll = 4; // groups of eight values a thread has in flight

// n8 = number of groups of eight values (a multiple of four: whole blocks)
template <typename InT>
__global__ void __launch_bounds__(kMxThreads) mxfp4_quantize_kernel(const InT *__restrict__ x, uint32_t *__restrict__ q, uint8_t *__restrict__ scales, int64_t n8) {
  const int64_t per_pass = (int64_t)gridDim.x * kMxThreads * kMxUnroll;
  for (int64_t base = (int64_t)blockIdx.x * kMxThreads * kMxUnroll; base < n8; base += per_pass) {
    Raw8<InT> raw[kMxUnroll];
#pragma unroll
    for (int u = 0; u < kMxUnroll; u++) {
      const int64_t i = base + u * kMxThreads + threadIdx.x;
      if (i < n8) raw[u] = load_raw8(x + i * 8);
      else raw[u] = Raw8<InT>{};
    }
#pragma unroll
    for (int u = 0; u < kMxUnroll; u++) {
      const int64_t i = base + u * kMxThreads + threadIdx.x;
      uint32_t m = absmax_bits(raw[u]);
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
      const uint32_t e = m >> 23;
      const uint32_t byte = e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
      const float inv = e == 255u ? 0.f : __uint_as_float((254u - byte) << 23);
      const InT *v = reinterpret_cast<const InT *>(&raw[u]);
      uint32_t w = 0;
#pragma unroll
      for (int j = 0; j < 8; j += 2) w |= e2m1x2(FloatIO<InT>::to_f32(v[j]) * inv, FloatIO<InT>::to_f32(v[j + 1]) * inv) << (4 * j);
      if (e == 255u) w = 0; // infinity * 0 would be NaN, which the conversion turns into 6
      if (i < n8) {
        q[i] = w;
        if ((threadIdx.x & 3) == 0) scales[i >> 2] = (uint8_t)byte;
      }
    }
  }
}

template <typename OutT>
__global__ void __launch_bounds__(kMxThreads) mxfp4_dequantize_kernel(const uint32_t *__restrict__ q, const uint8_t *__restrict__ scales, OutT *__restrict__ y, int64_t n8) {
  const int64_t per_pass = (int64_t)gridDim.x * kMxThreads * kMxUnroll;
  for (int64_t base = (int64_t)blockIdx.x * kMxThreads * kMxUnroll; base < n8; base += per_pass) {
    uint32_t w[kMxUnroll], s[kMxUnroll];
#pragma unroll
    for (int u = 0; u < kMxUnroll; u++) {
      const int64_t i = base + u * kMxThreads + threadIdx.x;
      w[u] = s[u] = 0;
      if (i < n8) {
        w[u] = __ldcs(q + i);
        s[u] = scales[i >> 2];
      }
    }
#pragma unroll
    for (int u = 0; u < kMxUnroll; u++) {
      const int64_t i = base + u * kMxThreads + threadIdx.x;
      const float f = e8m0_to_f32(s[u]);
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const float2 p = e2m1x2_to_f32((w[u] >> (4 * j)) & 0xFFu);
        v[j] = p.x * f;
        v[j + 1] = p.y * f;
      }
      if (i < n8) store_vec_f32<OutT, 8>(y + i * 8, v);
    }
  }
}

// `x` is the floating-point side [..., K], `q` the e2m1 side, `s` the e8m0 scales
int check_mxfp4(const char *op, const ql_tensor *x, const ql_tensor *q, const ql_tensor *s) {
  if (!x || !q || !s) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: null tensor", op);
  if (!is_float_dtype(x->dtype)) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: the floating-point tensor must be f32, f16 or bf16", op);
  if (q->dtype != QL_F4E2M1 || s->dtype != QL_F8E8M0) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: data must be f4E2M1FN and scales f8E8M0FNU", op);
  if (x->rank < 1 || x->rank > QL_MAX_RANK || q->rank != x->rank || s->rank != x->rank)
    return set_error(QL_ERR_INVALID_ARGUMENT, "%s: input, result and scales must have the same rank (1..%d)", op, QL_MAX_RANK);
  for (int i = 0; i < x->rank; i++) {
    if (x->shape[i] < 0) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: negative dimension", op);
    if (q->shape[i] != x->shape[i]) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: data and floating-point tensor differ in shape", op);
    const bool last = i == x->rank - 1;
    if (last && x->shape[i] % kMxBlock != 0) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: the last dimension must be divisible by %d.", op, kMxBlock);
    if (s->shape[i] != (last ? x->shape[i] / kMxBlock : x->shape[i]))
      return set_error(QL_ERR_INVALID_ARGUMENT, "%s: scales must have one entry per block of %d along the last axis", op, kMxBlock);
  }
  if (numel(x) > 0 && (!x->data || !q->data || !s->data)) return set_error(QL_ERR_INVALID_ARGUMENT, "%s: tensor without data", op);
  if (!aligned16(x->data) || (reinterpret_cast<uintptr_t>(q->data) & 3))
    return set_error(QL_ERR_UNSUPPORTED, "%s: buffers must be 16-byte (data: 4-byte) aligned", op);
  return QL_OK;
}

unsigned mx_grid(int64_t n8) {
  const int64_t per = (int64_t)kMxThreads * kMxUnroll, blocks = (n8 + per - 1) / per, cap = (int64_t)sm_count() * 8;
  return (unsigned)(blocks < cap ? blocks : cap);
}

} // namespace
} // namespace ql

using namespace ql;

extern "C" int ql_quantize_mxfp4(const ql_tensor *input, ql_tensor *data, ql_tensor *scales, void *stream) {
  const int rc = check_mxfp4("quantize_mxfp4", input, data, scales);
  if (rc != QL_OK) return rc;
  const int64_t n8 = numel(input) / 8;
  if (n8 == 0) return QL_OK;
  if (overlap(data, input) || overlap(scales, input) || overlap(data, scales)) return set_error(QL_ERR_INVALID_ARGUMENT, "quantize_mxfp4: input and results must not overlap");
  cudaStream_t st = (cudaStream_t)stream;
  uint32_t *q = static_cast<uint32_t *>(data->data);
  uint8_t *s = static_cast<uint8_t *>(scales->data);
  if (input->dtype == QL_F32) mxfp4_quantize_kernel<float><<<mx_grid(n8), kMxThreads, 0, st>>>(static_cast<const float *>(input->data), q, s, n8);
  else if (input->dtype == QL_F16) mxfp4_quantize_kernel<__half><<<mx_grid(n8), kMxThreads, 0, st>>>(static_cast<const __half *>(input->data), q, s, n8);
  else mxfp4_quantize_kernel<__nv_bfloat16><<<mx_grid(n8), kMxThreads, 0, st>>>(static_cast<const __nv_bfloat16 *>(input->data), q, s, n8);
  count_launches(1);
  QL_CUDA_TRY(cudaGetLastError());
  return QL_OK;
}

extern "C" int ql_dequantize_mxfp4(const ql_tensor *data, const ql_tensor *scales, ql_tensor *output, void *stream) {
  const int rc = check_mxfp4("dequantize_mxfp4", output, data, scales);
  if (rc != QL_OK) return rc;
  const int64_t n8 = numel(output) / 8;
  if (n8 == 0) return QL_OK;
  if (overlap(output, data) || overlap(output, scales)) return set_error(QL_ERR_INVALID_ARGUMENT, "dequantize_mxfp4: output must not overlap data or scales");
  cudaStream_t st = (cudaStream_t)stream;
  const uint32_t *q = static_cast<const uint32_t *>(data->data);
  const uint8_t *s = static_cast<const uint8_t *>(scales->data);
  if (output->dtype == QL_F32) mxfp4_dequantize_kernel<float><<<mx_grid(n8), kMxThreads, 0, st>>>(q, s, static_cast<float *>(output->data), n8);
  else if (output->dtype == QL_F16) mxfp4_dequantize_kernel<__half><<<mx_grid(n8), kMxThreads, 0, st>>>(q, s, static_cast<__half *>(output->data), n8);
  else mxfp4_dequantize_kernel<__nv_bfloat16><<<mx_grid(n8), kMxThreads, 0, st>>>(q, s, static_cast<__nv_bfloat16 *>(output->data), n8);
  count_launches(1);
  QL_CUDA_TRY(cudaGetLastError());
  return QL_OK;
}
