// Dropout from a counter-based generator; the backward pass is the same call
// on the gradient.
#include "rows.cuh"

namespace {

using namespace vs;

template <typename T>
__global__ void __launch_bounds__(256) dropout_kernel(uint64_t count, const T* x, T* y, const Dropout d) {
  const uint64_t groups = (count + 7) / 8;
  for (uint64_t g = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; g < groups;
       g += (uint64_t)gridDim.x * blockDim.x) {
    const Words w = philox(d, g);
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      const uint64_t i = g * 8 + j;
      if (i < count) y[i] = from_f32<T>(dropped(to_f32(x[i]), (d.threshold == 0 || keeps(w, j, d.limit)), d.scale));
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
  const uint64_t blocks = ((count + 7) / 8 + 255) / 256;
  const uint32_t grid = (uint32_t)(blocks < 148 * 64 ? blocks : 148 * 64);
  return vs_with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    dropout_kernel<T><<<grid, 256, 0, ctx->stream>>>(count, (const T*)x, (T*)y, d);
    ++ctx->launches;
    return vs_cuda(ctx, cudaGetLastError(), "dropout launch");
  });
}
