// Streaming forward layer norm, alone or joined with the dropout and residual
// sum before it, for short contiguous rows.
//
// The work is one read and one write of the rows, so the kernels keep bulk
// copies in flight all the time: each warp owns a ring of shared-memory slots, a
// tile of rows each, that one lane refills with cp.async.bulk, and its lanes hold
// rows in registers for the two sums (mean, then squares about it).  A lane's
// columns are the same for every row, so the weights stay in registers too.
#include <atomic>

#include "norm.cuh"

namespace {

using namespace vs;

// CTAs on an SM, and the bytes of one slot and input.  Two
// things meet here.  Every byte in flight beyond what hides the latency only
// queues in front of the DRAM and costs throughput (f32 rows of 256, two slots
// of 2 KB a warp: 12 warps 97 % of the copy rate, 16 warps 86 %; joined, two
// inputs: 8 warps 96 %, 12 warps 83 %), while 16-bit rows need the warps'
// arithmetic (bf16 rows of 64, 16 values a lane: 16 warps 91 %, 12 warps 87 %;
// of 512, 32 values a lane: 12 warps 92 %).  Slots that are written back need
// longer runs (59 f32: 4 KB 97 %, 2 KB 80 %).
template <typename T, int VEC, int K, bool kJoin> constexpr int warp_ctas() {
  if (VEC * K <= 8) return 6;
  if (VEC * sizeof(T) == 16 && sizeof(T) == 4) return kJoin ? 2 : 3;
  return VEC * K > 20 || sizeof(T) == 4 ? 3 : 4;
}
// One input's long ones run in slots of 6 KB (750 bf16 columns 71 %, 4 KB 60 %; 450
// columns 58 and 66 %; joined, 602 columns 47 and 52 %).
template <typename T, int VEC, bool kJoin> constexpr uint32_t warp_slot(uint32_t row_bytes) {
  if (VEC * sizeof(T) == 16) return 2048;
  return !kJoin && row_bytes > 1000 ? 6144 : 4096;
}

struct FwdArgs {
  uint64_t rows;
  uint32_t cols, tile_rows, log_lanes, slot, bits, stages;
  const void *x, *residual;
  Weights w;
  float eps;
  void *y, *z;
  float *mean, *rstd;
  uint32_t* err;
};

// Rows of whole 16-byte vectors are written from registers; others go back into
// their slot and out by a bulk store, so that no access is narrower than its
// run of bytes.
template <typename T, int VEC, int K, bool kJoin>
__global__ void __launch_bounds__(NORM_WARPS * 32, warp_ctas<T, VEC, K, kJoin>())
    norm_fwd_kernel(const FwdArgs a, const __grid_constant__ Dropout d) {
  using P = Part<T, VEC, K>;
  using R = typename P::R;
  constexpr int PAIRS = P::PAIRS;
  constexpr bool kDirect = P::kVector;
  constexpr bool kBits = kJoin && VEC != 8;
  constexpr uint32_t NIN = kJoin ? 2 : 1;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) uint64_t bars[NORM_WARPS][NORM_STAGES];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint32_t lanes = 1u << a.log_lanes, sub = lane >> a.log_lanes, per_pass = 32u >> a.log_lanes;
  const P part(lane & (lanes - 1), lanes, sub, a.cols);
  unsigned char* ring = smem + (size_t)warp * (a.stages * NIN * a.slot + a.bits);
  uint32_t* bits = reinterpret_cast<uint32_t*>(ring + a.stages * NIN * a.slot);
  uint64_t* full = bars[warp];

  const uint64_t first = (uint64_t)blockIdx.x * NORM_WARPS + warp, step = (uint64_t)gridDim.x * NORM_WARPS;
  const uint32_t tile_bytes = a.tile_rows * a.cols * (uint32_t)sizeof(T);
  const uint64_t total = a.rows * a.cols * sizeof(T), step_bytes = step * tile_bytes;
  uint64_t begin = first * tile_bytes;  // of the tile at hand
  uint64_t load_at = begin;             // of the tile to be copied next (lane 0's)
  auto span_at = [&](uint64_t b) {
    const uint64_t end = total - b < tile_bytes ? total : b + tile_bytes;
    return kDirect ? Span{b, end, b, (uint32_t)(end - b), 0} : span_of(b, end, total);
  };
  auto refill = [&](uint32_t slot) {
    if (load_at < total) {
      const Span s = span_at(load_at);
      unsigned char* to = ring + slot * NIN * a.slot;
      mbar_expect(&full[slot], s.bytes * NIN);
      span_load(s, to, a.x, &full[slot]);
      if (kJoin) span_load(s, to + a.slot, a.residual, &full[slot]);
    }
    load_at += step_bytes;
  };
  if (lane == 0) {
    for (uint32_t k = 0; k < a.stages; ++k) mbar_init(&full[k], 1);
    mbar_init_fence();
    for (uint32_t k = 0; k < a.stages; ++k) refill(k);
  }
  float2 w[PAIRS], b[PAIRS];
  part.weights(a.w.weight, a.w.dtype, 1.0f, w);
  part.weights(a.w.bias, a.w.dtype, 0.0f, b);
  const float n = (float)a.cols, inv = 1.0f / n;
  __syncwarp();

  uint32_t slot = 0, parity = 0;
  bool ok = true;
  uint64_t row0 = first * a.tile_rows;
  for (; row0 < a.rows; row0 += step * a.tile_rows, begin += step_bytes) {
    ok = __all_sync(0xffffffffu, mbar_wait(&full[slot], parity));
    if (!ok) break;
    unsigned char* in = ring + slot * NIN * a.slot;
    unsigned char* res = in + a.slot;
    const uint32_t rows = a.rows - row0 < a.tile_rows ? (uint32_t)(a.rows - row0) : a.tile_rows;
    const uint64_t i0 = begin / sizeof(T);
    const uint32_t shift = kDirect ? 0 : (uint32_t)begin & 15u;
    if (!kDirect && total - begin < tile_bytes + 16u) {  // the last 16-byte piece, where it is not whole
      const Span s = span_at(begin);
      span_tail<T>(s, in, a.x, lane, 32);
      if (kJoin) span_tail<T>(s, res, a.residual, lane, 32);
      __syncwarp();
    }
    if (kBits && d.threshold) {
      fill_bits(d, i0, rows * a.cols, bits, lane, 32);
      __syncwarp();
    }
    for (uint32_t p = 0; p < rows; p += per_pass) {
      // a lane beyond the tile's rows computes its last row and writes nothing
      const bool live = p + sub < rows;
      const uint32_t r = live ? p + sub : rows - 1, r_at = r * a.cols;
      T* xr = reinterpret_cast<T*>(in + shift) + r_at;
      T* rr = reinterpret_cast<T*>(res + shift) + r_at;
      float2 v[PAIRS];
      R t[PAIRS];
      part.load(xr, t);
      part.clear(t);
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) v[i] = part.value(t, i);
      if (kJoin) {
        if (d.threshold) drop_part(part, v, i0 + r_at, d, bits, ((uint32_t)i0 & 7u) + r_at);
        part.load(rr, t);
        part.clear(t);
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
          part.set(t, i, add2(v[i], part.value(t, i)));  // z, rounded as it is stored
          v[i] = part.value(t, i);
        }
      }
      float2 s = both(0.0f);
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) s = add2(v[i], s);
      float m = s.x + s.y;
      m = quotient(lanes_sum(m, lanes), n, inv);
      part.subtract(v, m);
      s = both(0.0f);
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) s = fma2(v[i], v[i], s);
      float q = s.x + s.y;
      q = rsqrtf(fmaf(lanes_sum(q, lanes), inv, a.eps));
      if (!kDirect) __syncwarp();  // the last row is read by all before it is written
      if (live) {
        if (kJoin) part.store(kDirect ? static_cast<T*>(a.z) + i0 + r_at : rr, t);
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) part.set(t, i, fma2(mul2(v[i], both(q)), w[i], b[i]));
        part.store(kDirect ? static_cast<T*>(a.y) + i0 + r_at : xr, t);
        if (part.at == 0) {
          if (a.mean) a.mean[row0 + r] = m;
          if (a.rstd) a.rstd[row0 + r] = q;
        }
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
      span_store<T>(s, in, a.y, lane);
      if (kJoin) span_store<T>(s, res, a.z, lane);
      if (lane == 0) {
        bulk_commit();
        // the slot before this one has been read out by now: it is filled again
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
    for (uint32_t k = 0; k < a.stages && row0 < a.rows; ++k, row0 += step * a.tile_rows) {
      mbar_wait(&full[slot], parity);
      if (++slot == a.stages) {
        slot = 0;
        parity ^= 1;
      }
    }
  }
  if (!kDirect && lane == 0) bulk_wait<0>();
}

// Leaves *taken as it is where the slots do not fit.
template <typename T, int VEC, int K, bool kJoin> vs_status run_kernel(vs_ctx* ctx, const NormFwd& f, bool* taken) {
  static std::atomic<uint64_t> ready{0};
  constexpr uint32_t NIN = kJoin ? 2 : 1;
  auto kernel = norm_fwd_kernel<T, VEC, K, kJoin>;
  const uint64_t bit = 1ull << (ctx->device & 63);
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    VS_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)NORM_MAX_SMEM));
    ready.fetch_or(bit);
  }
  FwdArgs a{};
  a.rows = f.s.rows;
  a.cols = f.s.cols;
  const uint32_t chunks = (a.cols + VEC - 1) / VEC, row_bytes = a.cols * (uint32_t)sizeof(T);
  uint32_t per_sm = warp_ctas<T, VEC, K, kJoin>();
  while ((1u << a.log_lanes) * K < chunks) ++a.log_lanes;
  // whole passes per slot; fewer where that would leave warps without rows
  const uint32_t per_pass = 32u >> a.log_lanes;
  uint32_t passes = warp_slot<T, VEC, kJoin>(row_bytes) / (row_bytes * per_pass);
  const uint64_t share = (uint64_t)B200_SMS * per_sm * NORM_WARPS * per_pass;
  const uint64_t even = (a.rows + share - 1) / share;
  if (passes > even) passes = (uint32_t)even;
  a.tile_rows = (passes < 1 ? 1 : passes) * per_pass;
  a.slot = (a.tile_rows * row_bytes + 30u) & ~15u;
  a.bits = kJoin && VEC != 8 ? (a.tile_rows * a.cols / 8 + 2 + 15) & ~15u : 0;
  // Two slots: one being worked on, one on its way, and a third where slots are
  // written back (59 f32 columns: two 69 %, three 89 %); fewer CTAs where the SM's
  // shared memory does not hold theirs.  A slot that is written back needs at
  // least another beside it.
  constexpr uint32_t least = Part<T, VEC, K>::kVector ? 1 : 2;
  auto bytes = [&](uint32_t stages) { return NORM_WARPS * (stages * NIN * a.slot + a.bits) + NORM_PADDING; };
  auto room = [&] { return NORM_MAX_SMEM / per_sm - 1024; };
  while (per_sm > 1 && bytes(2) > room()) --per_sm;
  a.stages = Part<T, VEC, K>::kVector ? 2 : 3;
  while (a.stages > least && bytes(a.stages) > room()) --a.stages;
  if (bytes(a.stages) > room()) return VS_OK;
  *taken = true;
  a.x = f.x; a.residual = f.residual; a.w = f.w; a.eps = f.eps; a.y = f.y; a.z = f.z; a.mean = f.mean; a.rstd = f.rstd;
  a.err = ctx->d_err;
  const uint64_t most = ((a.rows + a.tile_rows - 1) / a.tile_rows + NORM_WARPS - 1) / NORM_WARPS;
  const uint64_t grid = (uint64_t)per_sm * B200_SMS;
  kernel<<<(uint32_t)(grid < most ? grid : most), NORM_WARPS * 32, bytes(a.stages), ctx->stream>>>(a, f.d);
  ++ctx->launches;
  return vs_cuda(ctx, cudaGetLastError(), "norm launch");
}

// Up to 4 vectors per lane.
template <typename T, bool kJoin> vs_status run_vectors(vs_ctx* ctx, const NormFwd& f, bool* taken) {
  constexpr int V = 16 / sizeof(T);
  const uint32_t chunks = f.s.cols / V;
  switch (norm_fit(chunks, V, {1, 2, 3, 4}).k) {
    case 1: return run_kernel<T, V, 1, kJoin>(ctx, f, taken);
    case 2: return run_kernel<T, V, 2, kJoin>(ctx, f, taken);
    case 3: return run_kernel<T, V, 3, kJoin>(ctx, f, taken);
    case 4: return run_kernel<T, V, 4, kJoin>(ctx, f, taken);
  }
  return VS_OK;
}

// Blocks of K runs, K odd (bf16 rows of 250: 16 lanes of 18 values 77 % of the copy
// rate, 32 lanes of 14 values 47 %; of 170: 16 lanes of 14 values 63 %, 32 lanes of 6
// values 47 %).  Runs as wide as the columns allow: 64M bf16 values in 300 columns in
// runs of four 82 %, of two 57 %, in 100 columns 70 and 65 %; where a lane holds a row
// on its own it depends on their number (20 columns, 3.2M rows 53 us, in runs of two 49,
// 200k rows 6.4 and 7.3; joined, 3.2M rows 112 and 130).  16-bit rows that more values a
// lane hold go with those rather than with a CTA each (602 columns 65 and 38 %; 31 values
// a lane for 801 columns 48 and 49 %, so not those), but 23 values a lane and more, a row
// to a warp, only where each warp has enough of them to be busy: 750 columns, 4800 rows
// 8.8 us and 8.9 with a CTA each, 1200 rows 6.0 and 5.2, 38400 rows 32 and 41; joined
// 4800 rows 16.3 and 13.9, 38400 rows 71 and 77.  Multiples of four that runs of four do
// not hold go by runs of two from twice as many rows on, where there is one input (924
// columns, 69k rows 55 and 69 us, 38400 rows 35 and 40, 19200 rows 23.1 and 21.7; joined,
// 38400 rows 78 and 77).
constexpr uint64_t NORM_MANY = (uint64_t)B200_SMS * 3 * NORM_WARPS * 8;  // rows: 8 for each warp
template <typename T, bool kJoin> vs_status run_blocks(vs_ctx* ctx, const NormFwd& f, bool* taken) {
  const bool many = f.s.rows >= NORM_MANY;
  if constexpr (sizeof(T) == 2) {
    if (f.s.cols % 4 == 0) {
      switch (norm_fit(f.s.cols / 4, 4, {3, 5, 7}).k) {
        case 3: return run_kernel<T, 4, 3, kJoin>(ctx, f, taken);
        case 5: return run_kernel<T, 4, 5, kJoin>(ctx, f, taken);
        case 7:
          if (f.s.cols > 640 && !many) return VS_OK;
          return run_kernel<T, 4, 7, kJoin>(ctx, f, taken);
      }
      if (kJoin || f.s.rows < 2 * NORM_MANY) return VS_OK;
    }
    if (f.s.cols % 2 == 0) {
      switch (norm_fit(f.s.cols / 2, 2, {3, 5, 7, 9}).k) {
        case 3: return run_kernel<T, 2, 3, kJoin>(ctx, f, taken);
        case 5: return run_kernel<T, 2, 5, kJoin>(ctx, f, taken);
        case 7: return run_kernel<T, 2, 7, kJoin>(ctx, f, taken);
        case 9: return run_kernel<T, 2, 9, kJoin>(ctx, f, taken);
      }
      switch (norm_fit(f.s.cols / 2, 2, {11, 15}).k) {
        case 11: return run_kernel<T, 2, 11, kJoin>(ctx, f, taken);
        case 15:
          if (many) return run_kernel<T, 2, 15, kJoin>(ctx, f, taken);
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
  if constexpr (sizeof(T) == 2) {
    if (many && norm_fit(f.s.cols, 1, {23}).k) return run_kernel<T, 1, 23, kJoin>(ctx, f, taken);
  }
  return VS_OK;
}

template <typename T, bool kJoin> vs_status run(vs_ctx* ctx, const NormFwd& f, bool* taken) {
  if (f.s.cols % (16 / sizeof(T)) == 0) return run_vectors<T, kJoin>(ctx, f, taken);
  return run_blocks<T, kJoin>(ctx, f, taken);
}

}  // namespace

vs_status norm_tile_forward(vs_ctx* ctx, int32_t dtype, bool join, const NormFwd& f, bool* taken) {
  *taken = false;
  return vs_with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    return join ? run<T, true>(ctx, f, taken) : run<T, false>(ctx, f, taken);
  });
}
