// Streaming backward layer norm, alone or joined with the residual sum and the
// dropout, for short contiguous rows; the warps and their rings are those of the
// forward (norm_fwd.cu).
//
// A lane's columns are the same for every row, so the weight's and the bias's
// gradients grow in registers over all rows of a warp; a CTA then leaves one
// partial sum per column and a second kernel adds the CTAs' in a fixed order.
#include <atomic>

#include "norm.cuh"

namespace {

using namespace vs;

// As in the forward: f32 rows of 256 reach 94 % of the copy rate with 8 warps
// and 85 % with 12; bf16 rows of 256 93 % with 12 warps of 16 values a lane and
// slots of 3 KB, 80 % with 8 warps of 32 values.
template <typename T, int VEC, int K> constexpr int warp_ctas() {
  if (VEC * K <= 8) return 5;
  if (VEC * K > 20) return 2;
  return VEC * sizeof(T) == 16 && sizeof(T) == 4 ? 2 : 3;
}
// Bytes of a slot and input; `pass` bytes of rows go through a warp at once.  f32 rows
// 2 KB, 16-bit rows 3 KB (share of the copy rate at 48 columns 73 %, in 2 KB 63 %, at
// 128 columns 83 and 81 %, at 256 columns 86 and 79 %), but 2 KB for rows of 64 to 128
// bytes whose passes fill that without a rest (32 columns 76 %, in 3 KB 72 %, joined 81
// and 75 %, joined without a mask 73 and 73 %; 64 columns 81 and 78 %).  Shorter rows, a
// lane each: 16 columns 66 %, in 2 KB 64 %; 8 columns 60 and 67 %, joined 63 and 70 %, but
// without a mask 79 and 67 %.  Rows that are not whole vectors and over 1.5 KB go two to a
// slot (780 bf16 columns 68 %, one to a slot 47 %; shorter ones lose by slots of 4 KB, 460
// columns 59 and 54 %).
template <typename T, int VEC> constexpr uint32_t warp_slot(uint32_t row_bytes, uint32_t pass) {
  if (VEC * sizeof(T) != 16) return row_bytes > 1536 ? 4096 : 3072;
  return sizeof(T) == 4 || (row_bytes >= 64 && row_bytes <= 128 && 2048 % pass == 0) ? 2048 : 3072;
}

// Whether a lane's values are few enough for a second set of sums: those of a tile.
// Narrow rows need it: at one column a lane has 1055 rows of a call of 100M, and 256 of
// them to a CTA make so many CTAs that 16M x 3 f32 takes 10 % longer.
template <int VEC, int K> constexpr bool sums_twice = VEC * K <= 6;

struct BwdArgs {
  uint64_t rows;
  uint32_t cols, tile_rows, log_lanes, slot, stat_slot, bits, stages, inputs;
  const void *dy, *z, *dz;
  Weights w;
  const float *mean, *rstd;
  void *dx, *dresidual;
  float* partial;  // [CTA][2][cols], NULL when no weight gradient is wanted
  uint32_t* err;
};

// Whole-vector rows are written from registers, others through their slots, as
// in the forward.
template <typename T, int VEC, int K, bool kJoin>
__global__ void __launch_bounds__(NORM_WARPS * 32, warp_ctas<T, VEC, K>())
    norm_bwd_kernel(const BwdArgs a, const __grid_constant__ Dropout d) {
  using P = Part<T, VEC, K>;
  using R = typename P::R;
  constexpr int PAIRS = P::PAIRS;
  constexpr bool kDirect = P::kVector;
  constexpr bool kBits = kJoin && VEC != 8;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) uint64_t bars[NORM_WARPS][NORM_STAGES];
  __shared__ uint32_t gave_up[NORM_WARPS];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint32_t lanes = 1u << a.log_lanes, sub = lane >> a.log_lanes, per_pass = 32u >> a.log_lanes;
  const P part(lane & (lanes - 1), lanes, sub, a.cols);
  const uint32_t stage = a.inputs * a.slot + 2 * a.stat_slot;  // dy, z, (dz), mean, rstd
  unsigned char* ring = smem + (size_t)warp * (a.stages * stage + a.bits);
  uint32_t* bits = reinterpret_cast<uint32_t*>(ring + a.stages * stage);
  uint64_t* full = bars[warp];

  const uint64_t first = (uint64_t)blockIdx.x * NORM_WARPS + warp, step = (uint64_t)gridDim.x * NORM_WARPS;
  const uint32_t tile_bytes = a.tile_rows * a.cols * (uint32_t)sizeof(T);
  const uint64_t total = a.rows * a.cols * sizeof(T), step_bytes = step * tile_bytes;
  const uint64_t step_rows = step * a.tile_rows;
  uint64_t begin = first * tile_bytes;
  uint64_t load_at = begin, load_row = first * a.tile_rows;
  auto span_at = [&](uint64_t b) {
    const uint64_t end = total - b < tile_bytes ? total : b + tile_bytes;
    return kDirect ? Span{b, end, b, (uint32_t)(end - b), 0} : span_of(b, end, total);
  };
  auto stat_at = [&](uint64_t r) {
    const uint64_t end = a.rows - r < a.tile_rows ? a.rows : r + a.tile_rows;
    return span_of(r * 4, end * 4, a.rows * 4);
  };
  auto refill = [&](uint32_t slot) {
    if (load_at < total) {
      const Span s = span_at(load_at), t = stat_at(load_row);
      unsigned char* to = ring + slot * stage;
      mbar_expect(&full[slot], s.bytes * a.inputs + t.bytes * 2);
      span_load(s, to, a.dy, &full[slot]);
      span_load(s, to + a.slot, a.z, &full[slot]);
      if (kJoin && a.inputs == 3) span_load(s, to + 2 * a.slot, a.dz, &full[slot]);
      span_load(t, to + a.inputs * a.slot, a.mean, &full[slot]);
      span_load(t, to + a.inputs * a.slot + a.stat_slot, a.rstd, &full[slot]);
    }
    load_at += step_bytes;
    load_row += step_rows;
  };
  if (lane == 0) {
    for (uint32_t k = 0; k < a.stages; ++k) mbar_init(&full[k], 1);
    mbar_init_fence();
    for (uint32_t k = 0; k < a.stages; ++k) refill(k);
  }
  float2 w[PAIRS], dw[PAIRS], db[PAIRS];
  part.weights(a.w.weight, a.w.dtype, 1.0f, w);
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) dw[i] = db[i] = both(0.0f);
  // where registers allow, a tile's rows are added up and then their sum to the others'
  constexpr bool kTwice = sums_twice<VEC, K>;
  float2 tile_w[kTwice ? PAIRS : 1], tile_b[kTwice ? PAIRS : 1];
  const float n = (float)a.cols, inv = 1.0f / n;
  __syncwarp();

  launch_next();
  uint32_t slot = 0, parity = 0;
  bool ok = true;
  uint64_t row0 = first * a.tile_rows;
  for (; row0 < a.rows; row0 += step_rows, begin += step_bytes) {
    ok = __all_sync(0xffffffffu, mbar_wait(&full[slot], parity));
    if (!ok) break;
    unsigned char* gbuf = ring + slot * stage;
    unsigned char* zbuf = gbuf + a.slot;
    unsigned char* rbuf = zbuf + a.slot;  // dz, where there is one
    unsigned char* mbuf = gbuf + a.inputs * a.slot;
    const uint32_t rows = a.rows - row0 < a.tile_rows ? (uint32_t)(a.rows - row0) : a.tile_rows;
    const uint64_t i0 = begin / sizeof(T);
    const uint32_t shift = kDirect ? 0 : (uint32_t)begin & 15u;
    // the buffers' last 16-byte pieces, where they are not whole
    if (a.rows - row0 < a.tile_rows + 4u || (!kDirect && total - begin < tile_bytes + 16u)) {
      const Span s = span_at(begin), st = stat_at(row0);
      span_tail<T>(s, gbuf, a.dy, lane, 32);
      span_tail<T>(s, zbuf, a.z, lane, 32);
      if (kJoin && a.inputs == 3) span_tail<T>(s, rbuf, a.dz, lane, 32);
      span_tail<float>(st, mbuf, a.mean, lane, 32);
      span_tail<float>(st, mbuf + a.stat_slot, a.rstd, lane, 32);
      __syncwarp();
    }
    const uint32_t stat_shift = (uint32_t)row0 * 4 & 15u;
    const float* ms = reinterpret_cast<const float*>(mbuf + stat_shift);
    const float* qs = reinterpret_cast<const float*>(mbuf + a.stat_slot + stat_shift);
    if (kBits && d.threshold) {
      fill_bits(d, i0, rows * a.cols, bits, lane, 32);
      __syncwarp();
    }
    if constexpr (kTwice) {
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) tile_w[i] = tile_b[i] = both(0.0f);
    }
    for (uint32_t p = 0; p < rows; p += per_pass) {
      // a lane beyond the tile's rows computes its last row and leaves nothing
      const bool live = p + sub < rows;
      const uint32_t r = live ? p + sub : rows - 1, r_at = r * a.cols;
      T* gr = reinterpret_cast<T*>(gbuf + shift) + r_at;
      T* zr = reinterpret_cast<T*>(zbuf + shift) + r_at;
      const T* dr = reinterpret_cast<const T*>(rbuf + shift) + r_at;
      const float m = ms[r], q = qs[r];
      float2 g[PAIRS], h[PAIRS];
      R t[PAIRS], res[PAIRS];
      part.load(gr, t);
      part.clear(t);
      if (p + per_pass > rows && !live) {  // the first test is the same for all
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) t[i] = R{};
      }
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) g[i] = part.value(t, i);
      part.load(zr, t);
      if (!kDirect) part.clear(t);
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) h[i] = mul2(add2(part.value(t, i), both(-m)), both(q));
      if (kJoin && a.inputs == 3) part.load(dr, res);
      float2 s1 = both(0.0f), s2 = both(0.0f);
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {  // g is zero for values that are not the row's
        if constexpr (kTwice) {
          tile_w[i] = fma2(g[i], h[i], tile_w[i]);
          tile_b[i] = add2(tile_b[i], g[i]);
        } else {
          dw[i] = fma2(g[i], h[i], dw[i]);
          db[i] = add2(db[i], g[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        g[i] = mul2(g[i], w[i]);
        s1 = add2(s1, g[i]);
        s2 = fma2(g[i], h[i], s2);
      }
      float m1 = s1.x + s1.y, m2 = s2.x + s2.y;
      m1 = lanes_sum(m1, lanes);
      m2 = lanes_sum(m2, lanes);
      m1 = quotient(m1, n, inv);
      m2 = quotient(m2, n, inv);
      if (!kDirect) __syncwarp();  // the last row is read by all before it is written
      if (live) {
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) g[i] = mul2(fma2(h[i], both(-m2), add2(g[i], both(-m1))), both(q));
        if (kJoin) {
          if (a.inputs == 3) {
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) g[i] = add2(g[i], part.value(res, i));
          }
#pragma unroll
          for (int i = 0; i < PAIRS; ++i) part.set(t, i, g[i]);
          part.store(kDirect ? static_cast<T*>(a.dresidual) + i0 + r_at : zr, t);
          if (d.threshold) drop_part(part, g, i0 + r_at, d, bits, ((uint32_t)i0 & 7u) + r_at);
        }
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) part.set(t, i, g[i]);
        part.store(kDirect ? static_cast<T*>(a.dx) + i0 + r_at : gr, t);
      }
    }
    if constexpr (kTwice) {
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        dw[i] = add2(dw[i], tile_w[i]);
        db[i] = add2(db[i], tile_b[i]);
      }
    }
    if (kDirect) {
      // every lane has its part of the tile in registers
      __syncwarp();
      if (lane == 0) refill(slot);
    } else {
      proxy_fence();
      __syncwarp();
      const Span s = span_at(begin);
      span_store<T>(s, gbuf, a.dx, lane);
      if (kJoin) span_store<T>(s, zbuf, a.dresidual, lane);
      if (lane == 0) {
        bulk_commit();
        bulk_wait_read<1>();
        if (row0 != first * a.tile_rows) refill(slot == 0 ? a.stages - 1 : slot - 1);
      }
      __syncwarp();
    }
    if (++slot == a.stages) {
      slot = 0;
      parity ^= 1;
    }
  }
  if (!ok && lane == 0) {  // a copy did not land in time: report, and wait for those in flight, as long again each
    atomicOr(a.err, VS_DERR_WAIT);
    for (uint32_t k = 0; k < a.stages && row0 < a.rows; ++k, row0 += step_rows) {
      mbar_wait(&full[slot], parity);
      if (++slot == a.stages) {
        slot = 0;
        parity ^= 1;
      }
    }
  }
  if (!kDirect && lane == 0) bulk_wait<0>();
  if (!a.partial) return;

  float* out = a.partial + (uint64_t)blockIdx.x * 2 * a.cols;
  // lanes with the same columns (their runs turned differently), then the
  // warps, each in order, through the rings' memory; where a warp gave up, whose copies
  // may still be on their way there, the sums are marked invalid
  if (lane == 0) gave_up[warp] = ok ? 0u : 1u;
  __syncthreads();
  float* sums = reinterpret_cast<float*>(smem);  // [warp][2][cols]
  float* mine = sums + warp * 2 * a.cols;
  for (uint32_t k = 0; k < per_pass; ++k) {
    if (sub == k) {
#pragma unroll
      for (int e = 0; e < P::E; ++e) {
        const uint32_t c = part.col(e / VEC) + e % VEC;
        if (part.has(e / VEC)) {
          const float pw = (&dw[e / 2].x)[e % 2], pb = (&db[e / 2].x)[e % 2];
          mine[c] = k ? mine[c] + pw : pw;
          mine[a.cols + c] = k ? mine[a.cols + c] + pb : pb;
        }
      }
    }
    __syncwarp();
  }
  __syncthreads();
  for (uint32_t c = threadIdx.x; c < 2 * a.cols; c += NORM_WARPS * 32) {
    float v = sums[c];
    uint32_t late = gave_up[0];
    for (uint32_t k = 1; k < NORM_WARPS; ++k) {
      v += sums[k * 2 * a.cols + c];
      late |= gave_up[k];
    }
    out[c] = late ? nan_value() : v;
  }
}

// Leaves *taken as it is where the slots do not fit.
template <typename T, int VEC, int K, bool kJoin> vs_status run_kernel(vs_ctx* ctx, const NormBwd& f, bool* taken) {
  static std::atomic<uint64_t> ready{0};
  auto kernel = norm_bwd_kernel<T, VEC, K, kJoin>;
  const uint64_t bit = 1ull << (ctx->device & 63);
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    VS_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)NORM_MAX_SMEM));
    ready.fetch_or(bit);
  }
  BwdArgs a{};
  a.rows = f.s.rows;
  a.cols = f.s.cols;
  a.inputs = f.dz ? 3 : 2;
  const uint32_t chunks = (a.cols + VEC - 1) / VEC, row_bytes = a.cols * (uint32_t)sizeof(T);
  uint32_t per_sm = warp_ctas<T, VEC, K>();
  while ((1u << a.log_lanes) * K < chunks) ++a.log_lanes;
  // As in the forward, and the same for the plain and the joined kernel, so
  // that their weight gradients are the same sums in the same order.
  const uint32_t per_pass = 32u >> a.log_lanes;
  const uint32_t pass = row_bytes * per_pass;
  uint32_t passes = warp_slot<T, VEC>(row_bytes, pass) / pass;
  const uint64_t share = (uint64_t)B200_SMS * per_sm * NORM_WARPS * per_pass;
  const uint64_t even = (a.rows + share - 1) / share;
  if (passes > even) passes = (uint32_t)even;
  a.tile_rows = (passes < 1 ? 1 : passes) * per_pass;
  a.slot = (a.tile_rows * row_bytes + 30u) & ~15u;
  a.stat_slot = (a.tile_rows * 4 + 30u) & ~15u;
  a.bits = VEC != 8 ? ((a.tile_rows * a.cols / 8 + 2 + 15) & ~15u) : 0;
  // Slots and CTAs as in the forward, the CTAs as for the joined kernel's three
  // inputs; the rings' memory also takes the warps' column sums.
  constexpr uint32_t least = Part<T, VEC, K>::kVector ? 1 : 2;
  const uint32_t sums = NORM_WARPS * 2 * a.cols * 4;
  auto bytes = [&](uint32_t inputs, uint32_t stages) {
    const uint32_t rings = NORM_WARPS * (stages * (inputs * a.slot + 2 * a.stat_slot) + a.bits);
    return (rings < sums ? sums : rings) + NORM_PADDING;
  };
  auto room = [&] { return NORM_MAX_SMEM / per_sm - 1024; };
  while (per_sm > 1 && bytes(3, 2) > room()) --per_sm;
  if (bytes(3, least) > room()) return VS_OK;
  a.stages = Part<T, VEC, K>::kVector ? 2 : 3;
  while (a.stages > least && bytes(a.inputs, a.stages) > room()) --a.stages;
  *taken = true;
  a.dy = f.dy; a.z = f.z; a.dz = f.dz; a.w = f.w; a.mean = f.mean; a.rstd = f.rstd;
  a.dx = f.dx; a.dresidual = f.dresidual;
  a.err = ctx->d_err;
  const uint64_t most = ((a.rows + a.tile_rows - 1) / a.tile_rows + NORM_WARPS - 1) / NORM_WARPS;
  const uint64_t once = (uint64_t)per_sm * B200_SMS;
  // A warp's rows at most.  Another wave of warps costs about 20 us (12.5M x 8 bf16 139 us,
  // in two waves 162), so lanes of many values take four times the chain.
  const uint64_t chain = NORM_CHAIN * (sums_twice<VEC, K> ? a.tile_rows : 4 * per_pass);
  const uint64_t all = once * (a.rows / (once * NORM_WARPS * chain) + 1);
  const uint32_t grid = (uint32_t)(all < most ? all : most);
  const bool want = f.dweight || f.dbias;
  NormScratch scratch;
  if (want) VS_TRY(norm_scratch_begin(ctx, (size_t)grid * 2 * a.cols, &scratch));
  a.partial = scratch.p;
  kernel<<<grid, NORM_WARPS * 32, bytes(a.inputs, a.stages), ctx->stream>>>(a, f.d);
  ++ctx->launches;
  vs_status st = vs_cuda(ctx, cudaGetLastError(), "norm backward launch");
  if (want) {
    if (st == VS_OK) st = norm_join_partials(ctx, a.cols, grid, a.partial, f.wdtype, f.dweight, f.dbias);
    const vs_status end = norm_scratch_end(ctx, scratch);
    if (st == VS_OK) st = end;
  }
  return st;
}

// As in the forward, with up to 3 vectors of 8 or 4 of 4 values per lane.
template <typename T, bool kJoin> vs_status run_vectors(vs_ctx* ctx, const NormBwd& f, bool* taken) {
  constexpr int V = 16 / sizeof(T);
  const uint32_t chunks = f.s.cols / V;
  switch ((sizeof(T) == 4 ? norm_fit(chunks, V, {1, 2, 3, 4}) : norm_fit(chunks, V, {1, 2, 3})).k) {
    case 1: return run_kernel<T, V, 1, kJoin>(ctx, f, taken);
    case 2: return run_kernel<T, V, 2, kJoin>(ctx, f, taken);
    case 3: return run_kernel<T, V, 3, kJoin>(ctx, f, taken);
    case 4:
      if constexpr (sizeof(T) == 4) return run_kernel<T, V, 4, kJoin>(ctx, f, taken);
  }
  return VS_OK;
}

// Runs of four where they cost less than runs of two (64M bf16 values in 300 columns
// 71 %, in runs of two 57 %; 100 columns in runs of two 62 %, of four 52 %), but on one
// lane up to 16 values only (12 columns 63 %, in runs of two 53 %; 20 columns, 3.2M rows
// 59 and 69 %, 200k rows 41 and 23 us, since the lanes' column sums are added one lane
// after another).  28 values a lane leave registers for two CTAs only, so they are for
// rows that nothing else holds (700 columns 62 %, a CTA per row 43 %; 28 columns 57 %,
// 14 values on two lanes 70 %); so are 22 to 30 in runs of two (750 columns 60 and 45 %,
// 902 columns 66 and 53 %; joined 902 columns 47 and 50 %, which the plain rows' choice
// decides).
template <typename T, bool kJoin> vs_status run_blocks(vs_ctx* ctx, const NormBwd& f, bool* taken) {
  if constexpr (sizeof(T) == 2) {
    const uint32_t cols = f.s.cols;
    const NormFit two = cols % 2 == 0 ? norm_fit(cols / 2, 2, {3, 5, 7, 9}) : NormFit{0, ~0u};
    if (cols % 4 == 0) {
      const NormFit four = norm_fit(cols / 4, 4, {3, 5});
      if (four.k == 0 && two.k == 0 && norm_fit(cols / 4, 4, {7}).k) return run_kernel<T, 4, 7, kJoin>(ctx, f, taken);
      if (four.cost < two.cost && (cols <= 16 || cols > 4 * 5))
        return four.k == 3 ? run_kernel<T, 4, 3, kJoin>(ctx, f, taken) : run_kernel<T, 4, 5, kJoin>(ctx, f, taken);
    }
    if (cols % 2 == 0) {
      switch (two.k) {
        case 3: return run_kernel<T, 2, 3, kJoin>(ctx, f, taken);
        case 5: return run_kernel<T, 2, 5, kJoin>(ctx, f, taken);
        case 7: return run_kernel<T, 2, 7, kJoin>(ctx, f, taken);
        case 9: return run_kernel<T, 2, 9, kJoin>(ctx, f, taken);
      }
      switch (norm_fit(f.s.cols / 2, 2, {11, 13, 15}).k) {
        case 11: return run_kernel<T, 2, 11, kJoin>(ctx, f, taken);
        case 13: return run_kernel<T, 2, 13, kJoin>(ctx, f, taken);
        case 15: return run_kernel<T, 2, 15, kJoin>(ctx, f, taken);
      }
      return VS_OK;
    }
  }
  switch (norm_fit(f.s.cols, 1, {5, 9, 11, 15}).k) {
    case 5: return run_kernel<T, 1, 5, kJoin>(ctx, f, taken);
    case 9: return run_kernel<T, 1, 9, kJoin>(ctx, f, taken);
    case 11: return run_kernel<T, 1, 11, kJoin>(ctx, f, taken);
    case 15: return run_kernel<T, 1, 15, kJoin>(ctx, f, taken);
  }
  return VS_OK;
}

template <typename T, bool kJoin> vs_status run(vs_ctx* ctx, const NormBwd& f, bool* taken) {
  if (f.s.cols % (16 / sizeof(T)) == 0) return run_vectors<T, kJoin>(ctx, f, taken);
  return run_blocks<T, kJoin>(ctx, f, taken);
}

}  // namespace

vs_status norm_tile_backward(vs_ctx* ctx, int32_t dtype, bool join, const NormBwd& f, bool* taken) {
  *taken = false;
  return vs_with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    return join ? run<T, true>(ctx, f, taken) : run<T, false>(ctx, f, taken);
  });
}
