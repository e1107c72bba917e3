// What the row operators (dropout, layer norm and the two joined) share:
// element types, the counter-based generator, row reductions.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "vs_internal.cuh"

namespace vs {

// Values are read and written in T and computed in f32.
template <typename T> VSD float to_f32(T v);
template <> VSD float to_f32<float>(float v) { return v; }
template <> VSD float to_f32<__half>(__half v) { return __half2float(v); }
template <> VSD float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> VSD T from_f32(float v);
template <> VSD float from_f32<float>(float v) { return v; }
template <> VSD __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> VSD __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Layer-norm weights may be f32 beside narrower rows; their type is a run-time
// value, since each CTA reads them once.
struct Weights {
  const void* weight;  // NULL: ones
  const void* bias;    // NULL: zeros
  int32_t dtype;       // vs_dtype
};
VSD float load_as(const void* p, int32_t dtype, uint64_t i) {
  if (dtype == VS_F32) return static_cast<const float*>(p)[i];
  if (dtype == VS_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
VSD void store_as(void* p, int32_t dtype, uint64_t i, float v) {
  if (dtype == VS_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == VS_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// Dropout's mask is a function of the value's index and is never stored.
// The generator is Philox 4x32 with ten rounds (Salmon, Moraes, Dror, Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", 2011): counter (group,
// offset), key seed.  One call gives four words, eight 16-bit numbers, for the
// eight values of a group (index / 8), so a value costs an eighth of a call.
// A value is kept when its number is at least `threshold`, that is with
// probability (65536 - threshold) / 65536, and scaled by the inverse of that
// probability: p is rounded to a multiple of 2^-16 and the expectation stays
// exact for the rounded p.
struct Dropout {
  uint32_t keys[10][2];  // the key of each round
  uint32_t offset[2];
  uint32_t threshold;    // 0: nothing is dropped, 65536: everything
  uint32_t limit;        // 65536 threshold - 1, for `keeps` where the threshold is not 0
  float scale;
};

struct Words { uint32_t w[4]; };

VSD Words philox(const Dropout& d, uint64_t group) {
  uint32_t c0 = (uint32_t)group, c1 = (uint32_t)(group >> 32), c2 = d.offset[0], c3 = d.offset[1];
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0;
    const uint64_t b = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ d.keys[r][0];
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ d.keys[r][1];
    c3 = (uint32_t)a;
  }
  return {{c0, c1, c2, c3}};
}

// Whether the value with half-word `lane` (low half first) is kept: its number,
// moved into a word's upper half, is above `limit` = 65536 threshold - 1, which
// no number is when the threshold is 65536.
VSD bool keeps(const Words& w, uint32_t lane, uint32_t limit) {
  return (lane & 1 ? w.w[lane >> 1] : w.w[lane >> 1] << 16) > limit;
}
// One value's decision on its own.
VSD bool keep_at(const Dropout& d, uint64_t index) {
  const Words w = philox(d, index >> 3);
  const uint32_t j = (uint32_t)index & 7u;
  const uint32_t word = j < 4 ? (j < 2 ? w.w[0] : w.w[1]) : (j < 6 ? w.w[2] : w.w[3]);
  return (j & 1 ? word : word << 16) > d.limit;
}
// A dropped value gives zero whatever it holds (NaN and infinities too).
VSD float dropped(float v, bool keep, float scale) { return keep ? v * scale : 0.0f; }

VSD float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// The sum over a CTA, the same in every thread; `scratch` holds 33 floats.
VSD float block_sum(float v, float* scratch) {
  v = warp_sum(v);
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, warps = (blockDim.x + 31u) >> 5;
  __syncthreads();
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  if (warp == 0) {
    const float s = warp_sum(lane < warps ? scratch[lane] : 0.0f);
    if (lane == 0) scratch[32] = s;
  }
  __syncthreads();
  return scratch[32];
}

}  // namespace vs

// Calls fn with a value of the element type's C++ type.
template <typename F> vs_status vs_with_dtype(int32_t dtype, F fn) {
  if (dtype == VS_F32) return fn(float{});
  if (dtype == VS_F16) return fn(__half{});
  return fn(__nv_bfloat16{});
}

inline size_t vs_dtype_size(int32_t dtype) { return dtype == VS_F32 ? 4 : 2; }
inline bool vs_dtype_valid(int32_t dtype) { return dtype == VS_F32 || dtype == VS_F16 || dtype == VS_BF16; }

// Checks p and lays out the generator's round keys.
vs_status vs_make_dropout(vs_ctx* ctx, const char* what, double p, uint64_t seed, uint64_t offset, vs::Dropout* out);
