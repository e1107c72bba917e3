// Streaming backward layer norm, alone or joined with the residual sum and the
// dropout, for contiguous rows; the workers and their rings are those of the
// forward (norm_fwd.cu).
//
// A lane's columns are the same for every row, so the weight's and the bias's
// gradients grow in registers over all rows of a worker; a CTA then leaves one
// partial sum per column and a second kernel adds the CTAs' in a fixed order.
#include <atomic>

#include "norm.cuh"

namespace {

using namespace vs;

// As in the forward.
constexpr int warp_ctas(int elems) { return elems == 16 ? 3 : 5; }

struct BwdArgs {
  uint64_t rows, tiles;
  uint32_t cols, tile_rows, lanes, slot, stat_slot, bits, stages, inputs;
  const void *dy, *z, *dz;
  Weights w;
  const float *mean, *rstd;
  void *dx, *dresidual;
  float* partial;  // [CTA][2][cols], NULL when no weight gradient is wanted
  uint32_t* err;
};

// t = q (g - s1 - h s2) (+ dz) of VEC values, and the columns' sums.
template <int VEC> VSD void accumulate(const float* dy, const float* h, float* dw, float* db) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    dw[j] = fmaf(dy[j], h[j], dw[j]);
    db[j] += dy[j];
  }
}

template <typename T, int VEC, int K, bool kJoin>
__global__ void __launch_bounds__(NORM_WARPS * 32, warp_ctas(VEC * K))
    norm_bwd_warp_kernel(const BwdArgs a, const __grid_constant__ Dropout d) {
  constexpr int E = VEC * K;
  constexpr bool kDirect = VEC * sizeof(T) == 16;
  constexpr bool kBits = kJoin && VEC != 8;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) uint64_t bars[NORM_WARPS][NORM_STAGES];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint32_t stage = a.inputs * a.slot + 2 * a.stat_slot;  // dy, z, (dz), mean, rstd
  unsigned char* ring = smem + (size_t)warp * (a.stages * stage + a.bits);
  unsigned char* bits = ring + a.stages * stage;
  uint64_t* full = bars[warp];
  const uint64_t total = a.rows * a.cols * sizeof(T);
  const uint64_t step = (uint64_t)gridDim.x * NORM_WARPS;
  const uint64_t first = (uint64_t)blockIdx.x * NORM_WARPS + warp;

  auto rows_of = [&](uint64_t tile) {
    const uint64_t left = a.rows - tile * a.tile_rows;
    return left < a.tile_rows ? (uint32_t)left : a.tile_rows;
  };
  auto tile_span = [&](uint64_t tile) {
    const uint64_t r0 = tile * a.tile_rows;
    return span_of(r0 * a.cols * sizeof(T), (r0 + rows_of(tile)) * a.cols * sizeof(T), total);
  };
  auto stat_span = [&](uint64_t tile) {
    const uint64_t r0 = tile * a.tile_rows;
    return span_of(r0 * 4, (r0 + rows_of(tile)) * 4, a.rows * 4);
  };
  auto refill = [&](uint64_t tile, uint32_t slot) {  // lane 0
    const Span s = tile_span(tile), t = stat_span(tile);
    unsigned char* to = ring + slot * stage;
    mbar_expect(&full[slot], s.bytes * a.inputs + t.bytes * 2);
    span_load(s, to, a.dy, &full[slot]);
    span_load(s, to + a.slot, a.z, &full[slot]);
    if (kJoin && a.inputs == 3) span_load(s, to + 2 * a.slot, a.dz, &full[slot]);
    span_load(t, to + a.inputs * a.slot, a.mean, &full[slot]);
    span_load(t, to + a.inputs * a.slot + a.stat_slot, a.rstd, &full[slot]);
  };
  if (lane == 0) {
    for (uint32_t k = 0; k < a.stages; ++k) mbar_init(&full[k], 1);
    mbar_init_fence();
    for (uint32_t k = 0; k < a.stages; ++k)
      if (first + k * step < a.tiles) refill(first + k * step, k);
  }
  const uint32_t lanes = a.lanes, sub = lane / lanes, at = lane % lanes, per_pass = 32 / lanes;
  float w[E], dw[E], db[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const uint32_t c = (at + lanes * (e / VEC)) * VEC + e % VEC;
    w[e] = c < a.cols && a.w.weight ? load_as(a.w.weight, a.w.dtype, c) : 1.0f;
    dw[e] = db[e] = 0.0f;
  }
  const float n = (float)a.cols, inv = 1.0f / n;
  __syncwarp();

  uint32_t slot = 0, parity = 0;
  uint64_t left = 0;
  bool ok = true;
  for (uint64_t tile = first; tile < a.tiles; tile += step) {
    ok = __all_sync(0xffffffffu, mbar_wait(&full[slot], parity));
    left = tile;
    if (!ok) break;
    unsigned char* gbuf = ring + slot * stage;
    unsigned char* zbuf = gbuf + a.slot;
    unsigned char* rbuf = zbuf + a.slot;  // dz, where there is one
    unsigned char* mbuf = gbuf + a.inputs * a.slot;
    const Span s = tile_span(tile), st = stat_span(tile);
    const uint64_t r0 = tile * a.tile_rows, i0 = r0 * a.cols;
    const uint32_t rows = rows_of(tile);
    if (span_has_tail(s) || span_has_tail(st)) {
      span_tail<T>(s, gbuf, a.dy, lane, 32);
      span_tail<T>(s, zbuf, a.z, lane, 32);
      if (kJoin && a.inputs == 3) span_tail<T>(s, rbuf, a.dz, lane, 32);
      span_tail<float>(st, mbuf, a.mean, lane, 32);
      span_tail<float>(st, mbuf + a.stat_slot, a.rstd, lane, 32);
      __syncwarp();
    }
    const float* ms = reinterpret_cast<const float*>(mbuf + st.shift);
    const float* qs = reinterpret_cast<const float*>(mbuf + a.stat_slot + st.shift);
    if (kBits && d.threshold) {
      const uint64_t g0 = i0 >> 3, g1 = (i0 + (uint64_t)rows * a.cols + 7) >> 3;
      for (uint64_t g = g0 + lane; g < g1; g += 32) bits[g - g0] = (unsigned char)keep_bits(philox(d, g), d.threshold);
      __syncwarp();
    }
    for (uint32_t p = 0; p < rows; p += per_pass) {
      const bool live = p + sub < rows;
      const uint32_t r = live ? p + sub : rows - 1;
      T* gr = reinterpret_cast<T*>(gbuf + s.shift) + r * a.cols;
      T* zr = reinterpret_cast<T*>(zbuf + s.shift) + r * a.cols;
      T* dr = reinterpret_cast<T*>(rbuf + s.shift) + r * a.cols;
      const float m = ms[r], q = qs[r];
      float g[E], h[E];
      float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const uint32_t c = (at + lanes * k) * VEC;
        if (c < a.cols) {
          float *gk = g + k * VEC, *hk = h + k * VEC;
          load_vec<VEC>(gr + c, gk);
          load_vec<VEC>(zr + c, hk);
#pragma unroll
          for (int j = 0; j < VEC; ++j) hk[j] = (hk[j] - m) * q;
          if (live) accumulate<VEC>(gk, hk, dw + k * VEC, db + k * VEC);
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            gk[j] *= w[k * VEC + j];
            s1 += gk[j];
            s2 = fmaf(gk[j], hk[j], s2);
          }
        }
      }
      s1 = quotient(lanes_sum(s1, lanes), n, inv);
      s2 = quotient(lanes_sum(s2, lanes), n, inv);
      if (!kDirect) __syncwarp();  // rows beyond the tile read the last one before it is written
      if (live) {
        T* dxr = kDirect ? static_cast<T*>(a.dx) + i0 + (uint64_t)r * a.cols : gr;
        T* drr = kDirect ? static_cast<T*>(a.dresidual) + i0 + (uint64_t)r * a.cols : zr;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const uint32_t c = (at + lanes * k) * VEC;
          if (c < a.cols) {
            float* gk = g + k * VEC;
#pragma unroll
            for (int j = 0; j < VEC; ++j) gk[j] = q * (gk[j] - s1 - h[k * VEC + j] * s2);
            if (kJoin) {
              if (a.inputs == 3) {
                float rv[VEC];
                load_vec<VEC>(dr + c, rv);
#pragma unroll
                for (int j = 0; j < VEC; ++j) gk[j] += rv[j];
              }
              store_vec<VEC>(drr + c, gk);
              if (d.threshold) {
                if (VEC == 8) {
                  const Words words = philox(d, (i0 + (uint64_t)r * a.cols + c) >> 3);
#pragma unroll
                  for (int j = 0; j < VEC; ++j) gk[j] = dropped(gk[j], keeps(words, j, d.threshold), d.scale);
                } else {
                  const uint32_t e0 = ((uint32_t)i0 & 7u) + r * a.cols + c;
                  const uint32_t kept = bits[e0 >> 3] >> (e0 & 7u);
#pragma unroll
                  for (int j = 0; j < VEC; ++j) gk[j] = dropped(gk[j], kept >> j & 1u, d.scale);
                }
              }
            }
            store_vec<VEC>(dxr + c, gk);
          }
        }
      }
    }
    if (kDirect) {
      __syncwarp();
      if (lane == 0 && tile + a.stages * step < a.tiles) refill(tile + a.stages * step, slot);
    } else {
      proxy_fence();
      __syncwarp();
      span_store<T>(s, gbuf, a.dx, lane);
      if (kJoin) span_store<T>(s, zbuf, a.dresidual, lane);
      if (lane == 0) {
        bulk_commit();
        bulk_wait_read<1>();
        if (tile != first && tile + (a.stages - 1) * step < a.tiles)
          refill(tile + (a.stages - 1) * step, slot == 0 ? a.stages - 1 : slot - 1);
      }
      __syncwarp();
    }
    if (++slot == a.stages) {
      slot = 0;
      parity ^= 1;
    }
  }
  if (!ok) {  // a copy did not land in time: report, and let those in flight end
    if (lane == 0) atomicOr(a.err, VS_DERR_WAIT);
    for (uint32_t k = 0; k < a.stages && left + k * step < a.tiles; ++k) {
      mbar_wait(&full[slot], parity);
      if (++slot == a.stages) {
        slot = 0;
        parity ^= 1;
      }
    }
  }
  if (!kDirect && lane == 0) bulk_wait<0>();
  if (!a.partial) return;
  // lanes with the same columns, then the warps, in order
  __syncthreads();
#pragma unroll
  for (int e = 0; e < E; ++e) {
    for (uint32_t o = lanes; o < 32; o <<= 1) {
      dw[e] += __shfl_xor_sync(0xffffffffu, dw[e], o);
      db[e] += __shfl_xor_sync(0xffffffffu, db[e], o);
    }
  }
  float* red = reinterpret_cast<float*>(smem);  // [warp][2][cols]
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const uint32_t c = (at + lanes * (e / VEC)) * VEC + e % VEC;
    if (sub == 0 && c < a.cols) {
      red[warp * 2 * a.cols + c] = dw[e];
      red[(warp * 2 + 1) * a.cols + c] = db[e];
    }
  }
  __syncthreads();
  for (uint32_t c = threadIdx.x; c < 2 * a.cols; c += NORM_WARPS * 32) {
    float v = red[c];
    for (uint32_t k = 1; k < NORM_WARPS; ++k) v += red[k * 2 * a.cols + c];
    a.partial[(uint64_t)blockIdx.x * 2 * a.cols + c] = v;
  }
}

template <typename T, int VEC, int K, bool kJoin>
__global__ void __launch_bounds__(NORM_BWD_THREADS)
    norm_bwd_cta_kernel(const BwdArgs a, const __grid_constant__ Dropout d) {
  constexpr int E = VEC * K;
  constexpr bool kBits = kJoin && VEC != 8;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) uint64_t full[NORM_STAGES];
  __shared__ float2 red[2][NORM_BWD_THREADS / 32];
  __shared__ uint32_t late[2];
  const uint32_t stage = a.inputs * a.slot;
  unsigned char* bits = smem + a.stages * stage;  // two rows' keep bits
  const uint32_t tid = threadIdx.x, threads = blockDim.x, warps = threads >> 5;
  const uint64_t total = a.rows * a.cols * sizeof(T);

  auto row_span = [&](uint64_t r) { return span_of(r * a.cols * sizeof(T), (r + 1) * a.cols * sizeof(T), total); };
  auto refill = [&](uint64_t r, uint32_t slot) {  // thread 0
    const Span s = row_span(r);
    unsigned char* to = smem + slot * stage;
    mbar_expect(&full[slot], s.bytes * a.inputs);
    span_load(s, to, a.dy, &full[slot]);
    span_load(s, to + a.slot, a.z, &full[slot]);
    if (kJoin && a.inputs == 3) span_load(s, to + 2 * a.slot, a.dz, &full[slot]);
  };
  if (tid == 0) {
    late[0] = late[1] = 0;
    for (uint32_t k = 0; k < a.stages; ++k) mbar_init(&full[k], 1);
    mbar_init_fence();
    for (uint32_t k = 0; k < a.stages; ++k)
      if (blockIdx.x + (uint64_t)k * gridDim.x < a.rows) refill(blockIdx.x + (uint64_t)k * gridDim.x, k);
  }
  float w[E], dw[E], db[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const uint32_t c = (tid + threads * (e / VEC)) * VEC + e % VEC;
    w[e] = c < a.cols && a.w.weight ? load_as(a.w.weight, a.w.dtype, c) : 1.0f;
    dw[e] = db[e] = 0.0f;
  }
  const float n = (float)a.cols, inv = 1.0f / n;
  float m_next = a.mean[blockIdx.x], q_next = a.rstd[blockIdx.x];
  __syncthreads();

  uint32_t slot = 0, parity = 0, half = 0;
  bool stop = false;
  for (uint64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const float m = m_next, q = q_next;
    if (r + gridDim.x < a.rows) {  // the next row's statistics travel while this row is worked on
      m_next = a.mean[r + gridDim.x];
      q_next = a.rstd[r + gridDim.x];
    }
    if (!mbar_wait(&full[slot], parity)) late[half] = 1;
    unsigned char* gbuf = smem + slot * stage;
    unsigned char* zbuf = gbuf + a.slot;
    unsigned char* rbuf = zbuf + a.slot;
    const Span s = row_span(r);
    if (span_has_tail(s)) {
      span_tail<T>(s, gbuf, a.dy, tid, threads);
      span_tail<T>(s, zbuf, a.z, tid, threads);
      if (kJoin && a.inputs == 3) span_tail<T>(s, rbuf, a.dz, tid, threads);
      __syncthreads();
    }
    const uint64_t i0 = r * a.cols;
    if (kBits && d.threshold) {
      const uint64_t g0 = i0 >> 3, g1 = (i0 + a.cols + 7) >> 3;
      for (uint64_t k = g0 + tid; k < g1; k += threads)
        bits[half * (a.bits / 2) + (k - g0)] = (unsigned char)keep_bits(philox(d, k), d.threshold);
    }
    const T* gr = reinterpret_cast<const T*>(gbuf + s.shift);
    const T* zr = reinterpret_cast<const T*>(zbuf + s.shift);
    const T* dr = reinterpret_cast<const T*>(rbuf + s.shift);
    float g[E], h[E];
    __align__(16) T rv[kJoin ? E : 1];  // dz, held in its own type
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const uint32_t c = (tid + threads * k) * VEC;
      if (c < a.cols) {
        float *gk = g + k * VEC, *hk = h + k * VEC;
        load_vec<VEC>(gr + c, gk);
        load_vec<VEC>(zr + c, hk);
        if constexpr (kJoin) {
          using W = typename Word<VEC * sizeof(T)>::type;
          if (a.inputs == 3) *reinterpret_cast<W*>(rv + k * VEC) = *reinterpret_cast<const W*>(dr + c);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) hk[j] = (hk[j] - m) * q;
        accumulate<VEC>(gk, hk, dw + k * VEC, db + k * VEC);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          gk[j] *= w[k * VEC + j];
          s1 += gk[j];
          s2 = fmaf(gk[j], hk[j], s2);
        }
      }
    }
    s1 = warp_sum(s1);
    s2 = warp_sum(s2);
    if ((tid & 31u) == 0) red[half][tid >> 5] = make_float2(s1, s2);
    __syncthreads();
    // every thread holds its part of the row: the slot is free.  `late` and
    // `red` alternate between two rows, so one barrier per row is enough.
    stop = late[half] != 0;
    if (stop) break;
    if (tid == 0 && r + (uint64_t)a.stages * gridDim.x < a.rows) refill(r + (uint64_t)a.stages * gridDim.x, slot);
    s1 = red[half][0].x;
    s2 = red[half][0].y;
    for (uint32_t k = 1; k < warps; ++k) {
      s1 += red[half][k].x;
      s2 += red[half][k].y;
    }
    s1 = quotient(s1, n, inv);
    s2 = quotient(s2, n, inv);
    T* dxr = static_cast<T*>(a.dx) + i0;
    T* drr = static_cast<T*>(a.dresidual) + i0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const uint32_t c = (tid + threads * k) * VEC;
      if (c < a.cols) {
        float* gk = g + k * VEC;
#pragma unroll
        for (int j = 0; j < VEC; ++j) gk[j] = q * (gk[j] - s1 - h[k * VEC + j] * s2);
        if constexpr (kJoin) {
          if (a.inputs == 3) {
            float rf[VEC];
            load_vec<VEC>(rv + k * VEC, rf);
#pragma unroll
            for (int j = 0; j < VEC; ++j) gk[j] += rf[j];
          }
          store_vec<VEC>(drr + c, gk);
          if (d.threshold) {
            if (VEC == 8) {
              const Words words = philox(d, (i0 + c) >> 3);
#pragma unroll
              for (int j = 0; j < VEC; ++j) gk[j] = dropped(gk[j], keeps(words, j, d.threshold), d.scale);
            } else {
              const uint32_t e0 = ((uint32_t)i0 & 7u) + c;
              const uint32_t kept = bits[half * (a.bits / 2) + (e0 >> 3)] >> (e0 & 7u);
#pragma unroll
              for (int j = 0; j < VEC; ++j) gk[j] = dropped(gk[j], kept >> j & 1u, d.scale);
            }
          }
        }
        store_vec<VEC>(dxr + c, gk);
      }
    }
    half ^= 1;
    if (++slot == a.stages) {
      slot = 0;
      parity ^= 1;
    }
  }
  if (stop && tid == 0) {
    atomicOr(a.err, VS_DERR_WAIT);
    for (uint32_t k = 0; k < a.stages; ++k) mbar_wait(&full[(slot + k) % a.stages], parity ^ (slot + k >= a.stages));
  }
  if (!a.partial) return;
  float* out = a.partial + (uint64_t)blockIdx.x * 2 * a.cols;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const uint32_t c = (tid + threads * k) * VEC;
    if (c < a.cols) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        out[c + j] = dw[k * VEC + j];
        out[a.cols + c + j] = db[k * VEC + j];
      }
    }
  }
}

// Launches `kernel` with `per_sm` CTAs on each SM, at most
// `most`, and then adds up their column sums.
template <typename Kernel>
vs_status launch_full(vs_ctx* ctx, Kernel kernel, std::atomic<uint64_t>& ready, uint32_t threads, uint32_t per_sm,
                      size_t smem, uint64_t most, BwdArgs& a, const NormBwd& f) {
  const uint64_t bit = 1ull << (ctx->device & 63);
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    VS_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)NORM_MAX_SMEM));
    ready.fetch_or(bit);
  }
  const uint64_t full = (uint64_t)per_sm * B200_SMS;
  const uint32_t grid = (uint32_t)(full < most ? full : most);
  const bool sums = f.dweight || f.dbias;
  // from the stream-ordered pool: calls of one ctx on several streams do not share it
  if (sums) VS_CUDA(ctx, cudaMallocAsync((void**)&a.partial, (size_t)grid * 2 * a.cols * 4, ctx->stream));
  kernel<<<grid, threads, smem, ctx->stream>>>(a, f.d);
  ++ctx->launches;
  vs_status st = vs_cuda(ctx, cudaGetLastError(), "norm backward launch");
  if (sums) {
    if (st == VS_OK) st = norm_join_partials(ctx, a.cols, grid, a.partial, f.wdtype, f.dweight, f.dbias);
    VS_CUDA(ctx, cudaFreeAsync(a.partial, ctx->stream));
  }
  return st;
}

template <typename T> BwdArgs common_args(vs_ctx* ctx, const NormBwd& f) {
  BwdArgs a{};
  a.rows = f.s.rows;
  a.cols = f.s.cols;
  a.inputs = f.dz ? 3 : 2;
  a.dy = f.dy; a.z = f.z; a.dz = f.dz; a.w = f.w; a.mean = f.mean; a.rstd = f.rstd;
  a.dx = f.dx; a.dresidual = f.dresidual;
  a.err = ctx->d_err;
  return a;
}

template <typename T, int VEC, int K, bool kJoin> vs_status run_warp(vs_ctx* ctx, const NormBwd& f) {
  static std::atomic<uint64_t> ready{0};
  BwdArgs a = common_args<T>(ctx, f);
  const uint32_t chunks = (a.cols + VEC - 1) / VEC;
  a.lanes = 1;
  while (a.lanes * K < chunks) a.lanes *= 2;
  const uint32_t per_pass = 32 / a.lanes, row_bytes = a.cols * sizeof(T);
  // About 1 KB of copies per slot and input, otherwise as in the forward.  The
  // same for the plain and the joined kernel, so that their weight gradients
  // are the same sums in the same order.
  uint32_t passes = 1024 / (row_bytes * per_pass);
  const uint64_t share = (uint64_t)B200_SMS * warp_ctas(VEC * K) * NORM_WARPS * per_pass;
  const uint64_t even = (a.rows + share - 1) / share;
  if (passes > even) passes = (uint32_t)even;
  if (passes < 1) passes = 1;
  a.tile_rows = passes * per_pass;
  a.tiles = (a.rows + a.tile_rows - 1) / a.tile_rows;
  a.slot = (a.tile_rows * row_bytes + 30u) & ~15u;
  a.stat_slot = (a.tile_rows * 4 + 30u) & ~15u;
  a.bits = kJoin && VEC != 8 ? (a.tile_rows * a.cols / 8 + 2 + 15) & ~15u : 0;
  const uint32_t stage = a.inputs * a.slot + 2 * a.stat_slot;
  a.stages = NORM_STAGES;
  while (a.stages > 3 && warp_ctas(VEC * K) * NORM_WARPS * (a.stages * stage + a.bits) > NORM_MAX_SMEM - 16 * 1024) --a.stages;
  size_t smem = (size_t)NORM_WARPS * (a.stages * stage + a.bits);
  const size_t sums = (size_t)NORM_WARPS * 2 * a.cols * 4;
  if (smem < sums) smem = sums;
  return launch_full(ctx, norm_bwd_warp_kernel<T, VEC, K, kJoin>, ready, NORM_WARPS * 32, warp_ctas(VEC * K), smem,
                     (a.tiles + NORM_WARPS - 1) / NORM_WARPS, a, f);
}

template <typename T, int VEC, int K, bool kJoin> vs_status run_cta(vs_ctx* ctx, const NormBwd& f, bool* taken) {
  static std::atomic<uint64_t> ready{0};
  BwdArgs a = common_args<T>(ctx, f);
  const uint32_t chunks = (a.cols + VEC - 1) / VEC;
  const uint32_t threads = ((chunks + K - 1) / K + 31) & ~31u;
  if (threads > NORM_BWD_THREADS) return VS_OK;
  a.slot = (a.cols * (uint32_t)sizeof(T) + 30u) & ~15u;
  a.bits = kJoin && VEC != 8 ? 2 * ((a.cols / 8 + 2 + 15) & ~15u) : 0;
  a.stages = NORM_STAGES;
  while (a.stages > 2 && a.stages * a.inputs * a.slot * (NORM_BWD_THREADS / threads) > 200 * 1024) --a.stages;
  *taken = true;
  return launch_full(ctx, norm_bwd_cta_kernel<T, VEC, K, kJoin>, ready, threads,
                     NORM_BWD_THREADS / threads,
                     (size_t)a.stages * a.inputs * a.slot + a.bits, a.rows, a, f);
}

template <typename T, int VEC, int KS, bool kJoin> vs_status run_vec(vs_ctx* ctx, const NormBwd& f, bool* taken) {
  constexpr int KL = NORM_ELEMS / VEC;
  *taken = true;
  if (f.s.cols <= 32 * VEC * KS) return run_warp<T, VEC, KS, kJoin>(ctx, f);
  if (f.s.cols <= 32 * VEC * KL) return run_warp<T, VEC, KL, kJoin>(ctx, f);
  *taken = false;
  return run_cta<T, VEC, KL, kJoin>(ctx, f, taken);
}

template <typename T, bool kJoin> vs_status run(vs_ctx* ctx, const NormBwd& f, bool* taken) {
  constexpr int V = 16 / sizeof(T);
  if (f.s.cols % V == 0) return run_vec<T, V, 1, kJoin>(ctx, f, taken);
  if (sizeof(T) == 2 && f.s.cols % 2 == 0) return run_vec<T, 2, 2, kJoin>(ctx, f, taken);
  return run_vec<T, 1, 4, kJoin>(ctx, f, taken);
}

}  // namespace

vs_status norm_stream_backward(vs_ctx* ctx, int32_t dtype, bool join, const NormBwd& f, bool* taken) {
  *taken = false;
  return vs_with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    return join ? run<T, true>(ctx, f, taken) : run<T, false>(ctx, f, taken);
  });
}
