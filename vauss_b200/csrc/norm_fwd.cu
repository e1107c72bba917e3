// Streaming forward layer norm, alone or joined with the dropout and residual
// sum before it, for contiguous rows.
//
// The work is one read and one write of the rows, so the kernels keep bulk
// copies in flight all the time: each worker (a warp, or a CTA for rows over
// 512 values) owns a ring of shared-memory slots that one thread refills with
// cp.async.bulk, and holds its row in registers for the two sums (mean, then
// squares about it).  A lane's columns are the same for every row, so weights
// stay in registers too.
#include <atomic>

#include "norm.cuh"

namespace {

using namespace vs;

// CTAs of the warp kernel on an SM, by the values a lane holds: the registers
// they need fix it.
constexpr int warp_ctas(int elems) { return elems == 16 ? 4 : 7; }

struct FwdArgs {
  uint64_t rows, tiles;
  uint32_t cols, tile_rows, lanes, slot, bits, stages;
  const void *x, *residual;
  Weights w;
  float eps;
  void *y, *z;
  float *mean, *rstd;
  uint32_t* err;
};

// One warp per tile of rows, `lanes` lanes per row, VEC x K values per lane.
// Rows of whole 16-byte vectors are written from registers; others go back
// into their slot and out by a bulk store, so that no access is narrower than
// its run of bytes.
template <typename T, int VEC, int K, bool kJoin>
__global__ void __launch_bounds__(NORM_WARPS * 32, warp_ctas(VEC * K))
    norm_fwd_warp_kernel(const FwdArgs a, const __grid_constant__ Dropout d) {
  constexpr int E = VEC * K;
  constexpr uint32_t NIN = kJoin ? 2 : 1;
  constexpr bool kDirect = VEC * sizeof(T) == 16;
  constexpr bool kBits = kJoin && VEC != 8;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) uint64_t bars[NORM_WARPS][NORM_STAGES];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  unsigned char* ring = smem + (size_t)warp * (NORM_STAGES * NIN * a.slot + a.bits);
  unsigned char* bits = ring + NORM_STAGES * NIN * a.slot;
  uint64_t* full = bars[warp];
  const uint64_t total = a.rows * a.cols * sizeof(T);
  const uint64_t step = (uint64_t)gridDim.x * NORM_WARPS;
  const uint64_t first = (uint64_t)blockIdx.x * NORM_WARPS + warp;

  auto tile_span = [&](uint64_t tile) {
    const uint64_t r0 = tile * a.tile_rows;
    const uint64_t r1 = r0 + a.tile_rows < a.rows ? r0 + a.tile_rows : a.rows;
    return span_of(r0 * a.cols * sizeof(T), r1 * a.cols * sizeof(T), total);
  };
  auto refill = [&](uint64_t tile, uint32_t slot) {  // lane 0
    const Span s = tile_span(tile);
    mbar_expect(&full[slot], s.bytes * NIN);
    span_load(s, ring + slot * NIN * a.slot, a.x, &full[slot]);
    if (kJoin) span_load(s, ring + (slot * NIN + 1) * a.slot, a.residual, &full[slot]);
  };
  if (lane == 0) {
    for (uint32_t k = 0; k < NORM_STAGES; ++k) mbar_init(&full[k], 1);
    mbar_init_fence();
    for (uint32_t k = 0; k < NORM_STAGES; ++k)
      if (first + k * step < a.tiles) refill(first + k * step, k);
  }
  const uint32_t lanes = a.lanes, sub = lane / lanes, at = lane % lanes, per_pass = 32 / lanes;
  float w[E], b[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const uint32_t c = (at + lanes * (e / VEC)) * VEC + e % VEC;
    w[e] = c < a.cols && a.w.weight ? load_as(a.w.weight, a.w.dtype, c) : 1.0f;
    b[e] = c < a.cols && a.w.bias ? load_as(a.w.bias, a.w.dtype, c) : 0.0f;
  }
  const float n = (float)a.cols, inv = 1.0f / n;
  __syncwarp();

  uint32_t slot = 0, parity = 0;
  uint64_t left = 0;  // first tile whose copies have not been waited for
  bool ok = true;
  for (uint64_t tile = first; tile < a.tiles; tile += step) {
    ok = __all_sync(0xffffffffu, mbar_wait(&full[slot], parity));
    left = tile;
    if (!ok) break;
    unsigned char* in = ring + slot * NIN * a.slot;
    unsigned char* res = in + a.slot;
    const Span s = tile_span(tile);
    const uint64_t r0 = tile * a.tile_rows;
    const uint32_t rows = a.rows - r0 < a.tile_rows ? (uint32_t)(a.rows - r0) : a.tile_rows;
    if (span_has_tail(s)) {
      span_tail<T>(s, in, a.x, lane, 32);
      if (kJoin) span_tail<T>(s, res, a.residual, lane, 32);
      __syncwarp();
    }
    const uint64_t i0 = r0 * a.cols;
    if (kBits && d.threshold) {
      const uint64_t g0 = i0 >> 3, g1 = (i0 + (uint64_t)rows * a.cols + 7) >> 3;
      for (uint64_t g = g0 + lane; g < g1; g += 32) bits[g - g0] = (unsigned char)keep_bits(philox(d, g), d.threshold);
      __syncwarp();
    }
    for (uint32_t p = 0; p < rows; p += per_pass) {
      const bool live = p + sub < rows;
      const uint32_t r = live ? p + sub : rows - 1;
      T* xr = reinterpret_cast<T*>(in + s.shift) + r * a.cols;
      T* rr = reinterpret_cast<T*>(res + s.shift) + r * a.cols;
      float v[E];
      float sum = 0.0f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const uint32_t c = (at + lanes * k) * VEC;
        float* vk = v + k * VEC;
        if (c < a.cols) {
          load_vec<VEC>(xr + c, vk);
          if (kJoin) {
            if (d.threshold) {
              if (VEC == 8) {
                const Words words = philox(d, (i0 + (uint64_t)r * a.cols + c) >> 3);
#pragma unroll
                for (int j = 0; j < VEC; ++j) vk[j] = dropped(vk[j], keeps(words, j, d.threshold), d.scale);
              } else {
                const uint32_t e0 = ((uint32_t)i0 & 7u) + r * a.cols + c;
                const uint32_t kept = bits[e0 >> 3] >> (e0 & 7u);
#pragma unroll
                for (int j = 0; j < VEC; ++j) vk[j] = dropped(vk[j], kept >> j & 1u, d.scale);
              }
            }
            float rv[VEC];
            load_vec<VEC>(rr + c, rv);
#pragma unroll
            for (int j = 0; j < VEC; ++j) vk[j] = to_f32(from_f32<T>(vk[j] + rv[j]));
          }
#pragma unroll
          for (int j = 0; j < VEC; ++j) sum += vk[j];
        }
      }
      const float m = quotient(lanes_sum(sum, lanes), n, inv);
      float sq = 0.0f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if ((at + lanes * k) * VEC < a.cols) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float e = v[k * VEC + j] - m;
            sq = fmaf(e, e, sq);
          }
        }
      }
      const float q = rsqrtf(fmaf(lanes_sum(sq, lanes), inv, a.eps));
      if (!kDirect) __syncwarp();  // a row beyond the tile stands for the last one, which is read before it is written
      if (live) {
        T* yr = kDirect ? static_cast<T*>(a.y) + i0 + (uint64_t)r * a.cols : xr;
        T* zr = kDirect ? static_cast<T*>(a.z) + i0 + (uint64_t)r * a.cols : rr;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const uint32_t c = (at + lanes * k) * VEC;
          if (c < a.cols) {
            float* vk = v + k * VEC;
            if (kJoin) store_vec<VEC>(zr + c, vk);
            float o[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) o[j] = fmaf((vk[j] - m) * q, w[k * VEC + j], b[k * VEC + j]);
            store_vec<VEC>(yr + c, o);
          }
        }
        if (at == 0) {
          if (a.mean) a.mean[r0 + r] = m;
          if (a.rstd) a.rstd[r0 + r] = q;
        }
      }
    }
    if (kDirect) {
      __syncwarp();
      if (lane == 0 && tile + NORM_STAGES * step < a.tiles) refill(tile + NORM_STAGES * step, slot);
    } else {
      proxy_fence();
      __syncwarp();
      span_store<T>(s, in, a.y, lane);
      if (kJoin) span_store<T>(s, res, a.z, lane);
      if (lane == 0) {
        bulk_commit();
        // the slot before this one has been read out by now: it is filled again
        bulk_wait_read<1>();
        if (tile != first && tile + (NORM_STAGES - 1) * step < a.tiles)
          refill(tile + (NORM_STAGES - 1) * step, slot == 0 ? NORM_STAGES - 1 : slot - 1);
      }
      __syncwarp();
    }
    if (++slot == NORM_STAGES) {
      slot = 0;
      parity ^= 1;
    }
  }
  if (!ok) {  // a copy did not land in time: report, and let those in flight end
    if (lane == 0) atomicOr(a.err, VS_DERR_WAIT);
    for (uint32_t k = 0; k < NORM_STAGES && left + k * step < a.tiles; ++k) {
      mbar_wait(&full[slot], parity);
      if (++slot == NORM_STAGES) {
        slot = 0;
        parity ^= 1;
      }
    }
  }
  if (!kDirect && lane == 0) bulk_wait<0>();
}

// One CTA per row of more than 512 values; the row's slot is free again once
// every thread holds its part, which the first sum's barrier tells.
template <typename T, int VEC, int K, bool kJoin>
__global__ void __launch_bounds__(NORM_FWD_THREADS)
    norm_fwd_cta_kernel(const FwdArgs a, const __grid_constant__ Dropout d) {
  constexpr int E = VEC * K;
  constexpr uint32_t NIN = kJoin ? 2 : 1;
  constexpr bool kBits = kJoin && VEC != 8;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) uint64_t full[NORM_STAGES];
  __shared__ float red[2][NORM_FWD_THREADS / 32];
  __shared__ uint32_t late;
  unsigned char* bits = smem + a.stages * NIN * a.slot;  // two rows' keep bits
  const uint32_t tid = threadIdx.x, threads = blockDim.x, warps = threads >> 5;
  const uint64_t total = a.rows * a.cols * sizeof(T);

  auto row_span = [&](uint64_t r) { return span_of(r * a.cols * sizeof(T), (r + 1) * a.cols * sizeof(T), total); };
  auto refill = [&](uint64_t r, uint32_t slot) {  // thread 0
    const Span s = row_span(r);
    mbar_expect(&full[slot], s.bytes * NIN);
    span_load(s, smem + slot * NIN * a.slot, a.x, &full[slot]);
    if (kJoin) span_load(s, smem + (slot * NIN + 1) * a.slot, a.residual, &full[slot]);
  };
  auto fill_bits = [&](uint64_t r, uint32_t half) {
    const uint64_t i0 = r * a.cols, g0 = i0 >> 3, g1 = (i0 + a.cols + 7) >> 3;
    for (uint64_t g = g0 + tid; g < g1; g += threads)
      bits[half * (a.bits / 2) + (g - g0)] = (unsigned char)keep_bits(philox(d, g), d.threshold);
  };
  auto cta_sum = [&](float v, float* part) {
    v = warp_sum(v);
    if ((tid & 31u) == 0) part[tid >> 5] = v;
    __syncthreads();
    float s = part[0];
    for (uint32_t k = 1; k < warps; ++k) s += part[k];
    return s;
  };
  if (tid == 0) {
    late = 0;
    for (uint32_t k = 0; k < a.stages; ++k) mbar_init(&full[k], 1);
    mbar_init_fence();
    for (uint32_t k = 0; k < a.stages; ++k)
      if (blockIdx.x + (uint64_t)k * gridDim.x < a.rows) refill(blockIdx.x + (uint64_t)k * gridDim.x, k);
  }
  float w[E], b[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const uint32_t c = (tid + threads * (e / VEC)) * VEC + e % VEC;
    w[e] = c < a.cols && a.w.weight ? load_as(a.w.weight, a.w.dtype, c) : 1.0f;
    b[e] = c < a.cols && a.w.bias ? load_as(a.w.bias, a.w.dtype, c) : 0.0f;
  }
  if (kBits && d.threshold) fill_bits(blockIdx.x, 0);
  const float n = (float)a.cols, inv = 1.0f / n;
  __syncthreads();

  uint32_t slot = 0, parity = 0, half = 0;
  for (uint64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    if (!mbar_wait(&full[slot], parity)) late = 1;
    unsigned char* in = smem + slot * NIN * a.slot;
    unsigned char* res = in + a.slot;
    const Span s = row_span(r);
    if (span_has_tail(s)) {
      span_tail<T>(s, in, a.x, tid, threads);
      if (kJoin) span_tail<T>(s, res, a.residual, tid, threads);
      __syncthreads();
    }
    const uint64_t i0 = r * a.cols;
    const T* xr = reinterpret_cast<const T*>(in + s.shift);
    const T* rr = reinterpret_cast<const T*>(res + s.shift);
    float v[E];
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const uint32_t c = (tid + threads * k) * VEC;
      float* vk = v + k * VEC;
      if (c < a.cols) {
        load_vec<VEC>(xr + c, vk);
        if (kJoin) {
          if (d.threshold) {
            if (VEC == 8) {
              const Words words = philox(d, (i0 + c) >> 3);
#pragma unroll
              for (int j = 0; j < VEC; ++j) vk[j] = dropped(vk[j], keeps(words, j, d.threshold), d.scale);
            } else {
              const uint32_t e0 = ((uint32_t)i0 & 7u) + c;
              const uint32_t kept = bits[half * (a.bits / 2) + (e0 >> 3)] >> (e0 & 7u);
#pragma unroll
              for (int j = 0; j < VEC; ++j) vk[j] = dropped(vk[j], kept >> j & 1u, d.scale);
            }
          }
          float rv[VEC];
          load_vec<VEC>(rr + c, rv);
#pragma unroll
          for (int j = 0; j < VEC; ++j) vk[j] = to_f32(from_f32<T>(vk[j] + rv[j]));
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum += vk[j];
      }
    }
    const float m = quotient(cta_sum(sum, red[0]), n, inv);
    if (late) break;  // uniform: set before the barrier, never cleared
    if (tid == 0 && r + (uint64_t)a.stages * gridDim.x < a.rows) refill(r + (uint64_t)a.stages * gridDim.x, slot);
    half ^= 1;
    if (kBits && d.threshold && r + gridDim.x < a.rows) fill_bits(r + gridDim.x, half);
    float sq = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if ((tid + threads * k) * VEC < a.cols) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float e = v[k * VEC + j] - m;
          sq = fmaf(e, e, sq);
        }
      }
    }
    const float q = rsqrtf(fmaf(cta_sum(sq, red[1]), inv, a.eps));
    T* yr = static_cast<T*>(a.y) + i0;
    T* zr = static_cast<T*>(a.z) + i0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const uint32_t c = (tid + threads * k) * VEC;
      if (c < a.cols) {
        float* vk = v + k * VEC;
        if (kJoin) store_vec<VEC>(zr + c, vk);
        float o[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] = fmaf((vk[j] - m) * q, w[k * VEC + j], b[k * VEC + j]);
        store_vec<VEC>(yr + c, o);
      }
    }
    if (tid == 0) {
      if (a.mean) a.mean[r] = m;
      if (a.rstd) a.rstd[r] = q;
    }
    if (++slot == a.stages) {
      slot = 0;
      parity ^= 1;
    }
  }
  if (late && tid == 0) {  // as in the warp kernel
    atomicOr(a.err, VS_DERR_WAIT);
    for (uint32_t k = 0; k < a.stages; ++k) mbar_wait(&full[(slot + k) % a.stages], parity ^ (slot + k >= a.stages));
  }
}

// Launches `kernel` with `per_sm` CTAs on each SM, at most `most`.
template <typename Kernel>
vs_status launch_full(vs_ctx* ctx, Kernel kernel, std::atomic<uint64_t>& ready, uint32_t threads, uint32_t per_sm,
                      size_t smem, uint64_t most, const FwdArgs& a, const Dropout& d) {
  const uint64_t bit = 1ull << (ctx->device & 63);
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    VS_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)NORM_MAX_SMEM));
    ready.fetch_or(bit);
  }
  const uint64_t grid = (uint64_t)per_sm * B200_SMS;
  kernel<<<(uint32_t)(grid < most ? grid : most), threads, smem, ctx->stream>>>(a, d);
  ++ctx->launches;
  return vs_cuda(ctx, cudaGetLastError(), "norm launch");
}

template <typename T, int VEC, int K, bool kJoin>
vs_status run_warp(vs_ctx* ctx, const NormFwd& f) {
  static std::atomic<uint64_t> ready{0};
  constexpr uint32_t NIN = kJoin ? 2 : 1;
  FwdArgs a{};
  a.rows = f.s.rows;
  a.cols = f.s.cols;
  const uint32_t chunks = (a.cols + VEC - 1) / VEC;
  a.lanes = 1;
  while (a.lanes * K < chunks) a.lanes *= 2;
  const uint32_t per_pass = 32 / a.lanes, row_bytes = a.cols * sizeof(T);
  // about 2 KB of copies per slot, in whole passes; fewer where that would
  // leave warps without rows
  uint32_t passes = 2048 / NIN / (row_bytes * per_pass);
  const uint64_t share = (uint64_t)B200_SMS * warp_ctas(VEC * K) * NORM_WARPS * per_pass;
  const uint64_t even = (a.rows + share - 1) / share;
  if (passes > even) passes = (uint32_t)even;
  if (passes < 1) passes = 1;
  a.tile_rows = passes * per_pass;
  a.tiles = (a.rows + a.tile_rows - 1) / a.tile_rows;
  a.slot = (a.tile_rows * row_bytes + 30u) & ~15u;
  a.bits = kJoin && VEC != 8 ? (a.tile_rows * a.cols / 8 + 2 + 15) & ~15u : 0;
  a.x = f.x; a.residual = f.residual; a.w = f.w; a.eps = f.eps; a.y = f.y; a.z = f.z; a.mean = f.mean; a.rstd = f.rstd;
  a.err = ctx->d_err;
  const size_t smem = (size_t)NORM_WARPS * (NORM_STAGES * NIN * a.slot + a.bits);
  return launch_full(ctx, norm_fwd_warp_kernel<T, VEC, K, kJoin>, ready, NORM_WARPS * 32, warp_ctas(VEC * K), smem,
                     (a.tiles + NORM_WARPS - 1) / NORM_WARPS, a, f.d);
}

template <typename T, int VEC, int K, bool kJoin>
vs_status run_cta(vs_ctx* ctx, const NormFwd& f, bool* taken) {
  static std::atomic<uint64_t> ready{0};
  constexpr uint32_t NIN = kJoin ? 2 : 1;
  FwdArgs a{};
  a.rows = f.s.rows;
  a.cols = f.s.cols;
  const uint32_t chunks = (a.cols + VEC - 1) / VEC;
  const uint32_t threads = ((chunks + K - 1) / K + 31) & ~31u;
  if (threads > NORM_FWD_THREADS) return VS_OK;
  a.slot = (a.cols * (uint32_t)sizeof(T) + 30u) & ~15u;
  a.bits = kJoin && VEC != 8 ? 2 * ((a.cols / 8 + 2 + 15) & ~15u) : 0;
  a.stages = NORM_STAGES;
  while (a.stages > 2 && a.stages * NIN * a.slot * (NORM_FWD_THREADS / threads) > 200 * 1024) --a.stages;
  a.x = f.x; a.residual = f.residual; a.w = f.w; a.eps = f.eps; a.y = f.y; a.z = f.z; a.mean = f.mean; a.rstd = f.rstd;
  a.err = ctx->d_err;
  *taken = true;
  return launch_full(ctx, norm_fwd_cta_kernel<T, VEC, K, kJoin>, ready, threads,
                     NORM_FWD_THREADS / threads,
                     (size_t)a.stages * NIN * a.slot + a.bits, a.rows, a, f.d);
}

// Few values per lane where a warp's lanes still cover the row (fewer
// registers, more rows per pass), NORM_ELEMS otherwise.
template <typename T, int VEC, int KS, bool kJoin> vs_status run_vec(vs_ctx* ctx, const NormFwd& f, bool* taken) {
  constexpr int KL = NORM_ELEMS / VEC;
  *taken = true;
  if (f.s.cols <= 32 * VEC * KS) return run_warp<T, VEC, KS, kJoin>(ctx, f);
  if (f.s.cols <= 32 * VEC * KL) return run_warp<T, VEC, KL, kJoin>(ctx, f);
  *taken = false;
  return run_cta<T, VEC, KL, kJoin>(ctx, f, taken);
}

template <typename T, bool kJoin> vs_status run(vs_ctx* ctx, const NormFwd& f, bool* taken) {
  constexpr int V = 16 / sizeof(T);
  if (f.s.cols % V == 0) return run_vec<T, V, 1, kJoin>(ctx, f, taken);
  if (sizeof(T) == 2 && f.s.cols % 2 == 0) return run_vec<T, 2, 2, kJoin>(ctx, f, taken);
  return run_vec<T, 1, 4, kJoin>(ctx, f, taken);
}

}  // namespace

vs_status norm_stream_forward(vs_ctx* ctx, int32_t dtype, bool join, const NormFwd& f, bool* taken) {
  *taken = false;
  return vs_with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    return join ? run<T, true>(ctx, f, taken) : run<T, false>(ctx, f, taken);
  });
}
