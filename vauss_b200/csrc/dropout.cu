// Dropout from a counter-based generator; the backward pass is the same call
// on the gradient.
//
// One read and one write of the values: the generator's arithmetic (about 50
// instructions per group of eight values, and 3 per value to decide) has to hide
// behind the copy.
#include "norm.cuh"

namespace {

using namespace vs;

// 16-byte aligned buffers; GROUPS whole groups in flight per thread, a CTA's
// worth apart (3M x 48 f16: two 83 us, 105 % of the copy rate, one 91 us, four
// 84 us).  The values after the last whole group are the first CTA's.
template <typename T, int GROUPS>
__global__ void __launch_bounds__(256) dropout_kernel(uint64_t count, const T* x, T* y,
                                                      const __grid_constant__ Dropout d) {
  constexpr int W = sizeof(T) / 2;  // 16-byte pieces of a group
  const uint64_t groups = count / 8;
  if (blockIdx.x == 0 && threadIdx.x < (count & 7u)) {
    const uint64_t i = groups * 8 + threadIdx.x;
    y[i] = from_f32<T>(keep_at(d, i) ? to_f32(x[i]) * d.scale : 0.0f);
  }
  const uint64_t first = (uint64_t)blockIdx.x * (256 * GROUPS) + threadIdx.x;
  uint4 q[GROUPS][W];
#pragma unroll
  for (int k = 0; k < GROUPS; ++k) {
    if (first + k * 256 < groups) {
#pragma unroll
      for (int i = 0; i < W; ++i) q[k][i] = reinterpret_cast<const uint4*>(x)[(first + k * 256) * W + i];
    }
  }
#pragma unroll
  for (int k = 0; k < GROUPS; ++k) {
    const uint64_t g = first + k * 256;
    if (g >= groups) return;
    const Words words = philox(d, g);
    T* t = reinterpret_cast<T*>(q[k]);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = keeps(words, j, d.limit) ? to_f32(t[j]) * d.scale : 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = from_f32<T>(v[j]);
#pragma unroll
    for (int i = 0; i < W; ++i) reinterpret_cast<uint4*>(y)[g * W + i] = q[k][i];
  }
}

// Any alignment: the values of one group per thread, one by one.
template <typename T>
__global__ void __launch_bounds__(256) dropout_plain_kernel(uint64_t count, const T* x, T* y,
                                                            const __grid_constant__ Dropout d) {
  const uint64_t groups = (count + 7) / 8;
  for (uint64_t g = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; g < groups;
       g += (uint64_t)gridDim.x * blockDim.x) {
    const Words w = philox(d, g);
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      const uint64_t i = g * 8 + j;
      if (i < count) y[i] = from_f32<T>(keeps(w, j, d.limit) ? to_f32(x[i]) * d.scale : 0.0f);
    }
  }
}

}  // namespace

vs_status vs_make_dropout(vs_ctx* ctx, const char* what, double p, uint64_t seed, uint64_t offset, vs::Dropout* out) {
  if (!(p >= 0.0 && p <= 1.0)) return vs_fail(ctx, VS_ERR_INVALID, "%s: p = %g is not in [0, 1]", what, p);
  uint32_t t = (uint32_t)(p * 65536.0 + 0.5);
  if (p < 1.0 && t > 65535u) t = 65535u;  // only p = 1 drops everything
  out->threshold = t;
  out->limit = (uint32_t)(((uint64_t)t << 16) - 1);
  out->scale = t < 65536u ? (float)(65536.0 / (65536.0 - t)) : 0.0f;
  out->offset[0] = (uint32_t)offset;
  out->offset[1] = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
  for (int r = 0; r < 10; ++r) {
    out->keys[r][0] = k0;
    out->keys[r][1] = k1;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return VS_OK;
}

extern "C" VS_API vs_status vs_dropout(vs_ctx* ctx, uint64_t count, int32_t dtype, const void* x, double p,
                                       uint64_t seed, uint64_t offset, void* y) {
  if (!ctx) return VS_ERR_INVALID;
  if (!vs_dtype_valid(dtype)) return vs_fail(ctx, VS_ERR_UNSUPPORTED, "dropout: element type %d", dtype);
  if (count && (!x || !y)) return vs_fail(ctx, VS_ERR_INVALID, "dropout: null buffer");
  if (((uintptr_t)x | (uintptr_t)y) & (vs_dtype_size(dtype) - 1))
    return vs_fail(ctx, VS_ERR_INVALID, "dropout: buffers must be aligned to their element");
  if (count > (1ull << 60)) return vs_fail(ctx, VS_ERR_CAPACITY, "dropout: %llu values", (unsigned long long)count);
  vs::Dropout d;
  VS_TRY(vs_make_dropout(ctx, "dropout", p, seed, offset, &d));
  if (count == 0) return VS_OK;
  VS_CUDA(ctx, cudaSetDevice(ctx->device));
  if (d.threshold == 0) {  // everything is kept as it is
    if (x == y) return VS_OK;
    return vs_cuda(ctx, cudaMemcpyAsync(y, x, count * vs_dtype_size(dtype), cudaMemcpyDeviceToDevice, ctx->stream),
                   "dropout");
  }
  return vs_with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    constexpr int GROUPS = 2;
    const uint64_t blocks = (count / 8 + 256 * GROUPS - 1) / (256 * GROUPS);
    if ((((uintptr_t)x | (uintptr_t)y) & 15u) == 0 && blocks <= 0x7fffffffull) {
      dropout_kernel<T, GROUPS><<<blocks ? (uint32_t)blocks : 1, 256, 0, ctx->stream>>>(count, (const T*)x, (T*)y, d);
    } else {
      const uint64_t want = ((count + 7) / 8 + 255) / 256;
      dropout_plain_kernel<T><<<(uint32_t)(want < B200_SMS * 64 ? want : B200_SMS * 64), 256, 0, ctx->stream>>>(
          count, (const T*)x, (T*)y, d);
    }
    ++ctx->launches;
    return vs_cuda(ctx, cudaGetLastError(), "dropout launch");
  });
}
