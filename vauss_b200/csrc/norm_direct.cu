// Direct layer norm, forward and backward, alone or joined: the rows go from
// global memory straight into registers.  For calls too small to fill a ring,
// where only latency counts, and for rows that bulk copies cannot take (strides,
// odd alignment).  A warp's lanes share rows of up to 32 * VEC * K values, longer
// rows take a CTA each; a thread's columns are the same for every row.
#include <initializer_list>

#include "norm.cuh"

namespace {

using namespace vs;

// Warps of a CTA whose warps work on their own.  The backward's leave their sums
// together, so that few CTAs' sums are left to be added.
constexpr uint32_t FWD_WARPS = 4, BWD_WARPS = 16;
// threads of a CTA by the values each one holds
constexpr uint32_t direct_threads(int elems) { return elems > 8 ? 512 : 1024; }
// The sums of up to this many CTAs are added by the last one to leave its own,
// which saves the launch of another kernel: a call of 500 x 64 bf16 (8 CTAs) takes
// 9.0 us instead of 11.6; with 148 CTAs the one CTA's reads take longer than the
// launch (20k x 64 f16 12.3 us instead of 10.9).
constexpr uint32_t FOLD_CTAS = 64, FOLD_GROUPS = 32;

template <typename T, int VEC, int K, bool kJoin, bool kCta>
__global__ void __launch_bounds__(kCta ? direct_threads(VEC * K) : FWD_WARPS * 32)
    norm_direct_fwd_kernel(const NormFwd a, uint32_t log_lanes, const __grid_constant__ Dropout d) {
  using P = Part<T, VEC, K, true>;
  constexpr int PAIRS = P::PAIRS;
  __shared__ __align__(16) float red[2][kCta ? NORM_MAX_WARPS : 4];
  const uint32_t id = kCta ? threadIdx.x : threadIdx.x & 31u, warps = blockDim.x >> 5;
  const uint32_t lanes = kCta ? blockDim.x : 1u << log_lanes;
  const uint32_t sub = kCta ? 0 : id >> log_lanes, per_pass = kCta ? 1 : 32u >> log_lanes;
  const P part(kCta ? id : id & (lanes - 1), lanes, sub, a.s.cols);
  const uint64_t step = (uint64_t)gridDim.x * (kCta ? 1 : FWD_WARPS) * per_pass;
  const float n = (float)a.s.cols, inv = 1.0f / n;
  float2 w[PAIRS], b[PAIRS];
  bool ready = false;
  if (kCta) {
    for (uint32_t k = id; k < 2 * NORM_MAX_WARPS; k += blockDim.x) (&red[0][0])[k] = 0.0f;
    __syncthreads();
  }
  for (uint64_t r0 = ((uint64_t)blockIdx.x * (kCta ? 1 : FWD_WARPS) + (kCta ? 0 : threadIdx.x >> 5)) * per_pass;
       r0 < a.s.rows; r0 += step) {
    // a lane beyond the last row computes that row and writes nothing
    const bool live = r0 + sub < a.s.rows;
    const uint64_t r = live ? r0 + sub : a.s.rows - 1;
    float2 v[PAIRS];
    typename P::R t[PAIRS], u[PAIRS];
    part.load(static_cast<const T*>(a.x) + r * a.x_stride, t);
    if (kJoin) part.load(static_cast<const T*>(a.residual) + r * a.residual_stride, u);
    if (!ready) {  // after the first row's loads, so that they travel together
      part.weights(a.w.weight, a.w.dtype, 1.0f, w);
      part.weights(a.w.bias, a.w.dtype, 0.0f, b);
      ready = true;
    }
    part.clear(t);
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) v[i] = part.value(t, i);
    if (kJoin) {
      if (d.threshold) drop_runs(part, v, r * a.s.cols, d);
      part.clear(u);
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        part.set(t, i, add2(v[i], part.value(u, i)));  // z, rounded as it is stored
        v[i] = part.value(t, i);
      }
    }
    float2 s = both(0.0f);
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) s = add2(v[i], s);
    float m = s.x + s.y;
    m = quotient(kCta ? cta_sum(m, red[0], warps) : lanes_sum(m, lanes), n, inv);
    part.subtract(v, m);
    s = both(0.0f);
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) s = fma2(v[i], v[i], s);
    float q = s.x + s.y;
    q = rsqrtf(fmaf(kCta ? cta_sum(q, red[1], warps) : lanes_sum(q, lanes), inv, a.eps));
    if (!kCta) __syncwarp();  // the last row is read by all before it is written
    if (live) {
      if (kJoin) part.store(static_cast<T*>(a.z) + r * a.s.cols, t);
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) part.set(t, i, fma2(mul2(v[i], both(q)), w[i], b[i]));
      part.store(static_cast<T*>(a.y) + r * a.s.cols, t);
      if (part.at == 0) {
        if (a.mean) a.mean[r] = m;
        if (a.rstd) a.rstd[r] = q;
      }
    }
  }
}

template <typename T, int VEC, int K, bool kJoin, bool kCta>
__global__ void __launch_bounds__(kCta ? direct_threads(VEC * K) : BWD_WARPS * 32)
    norm_direct_bwd_kernel(const NormBwd a, uint32_t log_lanes, const __grid_constant__ Dropout d, float* partial,
                           uint32_t* ticket) {
  // One CTA's column sums are the weight gradients; several leave theirs in
  // `partial`, and with a `ticket` the last one adds them up.
  const bool alone = gridDim.x == 1;
  using P = Part<T, VEC, K, true>;
  constexpr int PAIRS = P::PAIRS;
  __shared__ __align__(16) float red[2][2][kCta ? NORM_MAX_WARPS : 4];
  extern __shared__ __align__(16) float sums[];  // [warp][2][cols], the lanes' column sums
  const uint32_t id = kCta ? threadIdx.x : threadIdx.x & 31u, warps = blockDim.x >> 5;
  const uint32_t lanes = kCta ? blockDim.x : 1u << log_lanes;
  const uint32_t sub = kCta ? 0 : id >> log_lanes, per_pass = kCta ? 1 : 32u >> log_lanes;
  const P part(kCta ? id : id & (lanes - 1), lanes, sub, a.s.cols);
  const uint64_t step = (uint64_t)gridDim.x * (kCta ? 1 : BWD_WARPS) * per_pass;
  const float n = (float)a.s.cols, inv = 1.0f / n;
  float2 w[PAIRS], dw[PAIRS], db[PAIRS];
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) dw[i] = db[i] = both(0.0f);
  if (!alone && !ticket) launch_next();
  bool ready = false;
  uint32_t half = 0;
  if (kCta) {
    for (uint32_t k = id; k < 4 * NORM_MAX_WARPS; k += blockDim.x) (&red[0][0][0])[k] = 0.0f;
    __syncthreads();
  }
  for (uint64_t r0 = ((uint64_t)blockIdx.x * (kCta ? 1 : BWD_WARPS) + (kCta ? 0 : threadIdx.x >> 5)) * per_pass;
       r0 < a.s.rows; r0 += step) {
    const bool live = r0 + sub < a.s.rows;
    const uint64_t r = live ? r0 + sub : a.s.rows - 1;
    float2 g[PAIRS], h[PAIRS];
    typename P::R t[PAIRS], u[PAIRS], res[PAIRS];
    const float m = a.mean[r], q = a.rstd[r];
    part.load(static_cast<const T*>(a.dy) + r * a.dy_stride, t);
    part.load(static_cast<const T*>(a.z) + r * a.z_stride, u);
    if (kJoin && a.dz) part.load(static_cast<const T*>(a.dz) + r * a.dz_stride, res);
    if (!ready) {
      part.weights(a.w.weight, a.w.dtype, 1.0f, w);
      ready = true;
    }
    part.clear(t);
    if (!live) {
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) t[i] = typename P::R{};
    }
    float2 s1 = both(0.0f), s2 = both(0.0f);
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {  // g is zero for values that are not the row's
      g[i] = part.value(t, i);
      h[i] = mul2(add2(part.value(u, i), both(-m)), both(q));
      dw[i] = fma2(g[i], h[i], dw[i]);
      db[i] = add2(db[i], g[i]);
      g[i] = mul2(g[i], w[i]);
      s1 = add2(s1, g[i]);
      s2 = fma2(g[i], h[i], s2);
    }
    float m1 = s1.x + s1.y, m2 = s2.x + s2.y;
    if (kCta) {
      m1 = warp_sum2(m1, m2);
      if ((id & 15u) == 0) red[half][id >> 4 & 1u][id >> 5] = m1;
      __syncthreads();  // `red` alternates between two rows, so one barrier per row is enough
      m1 = parts_sum(red[half][0], warps);
      m2 = parts_sum(red[half][1], warps);
      half ^= 1;
    } else {
      m1 = lanes_sum(m1, lanes);
      m2 = lanes_sum(m2, lanes);
    }
    m1 = quotient(m1, n, inv);
    m2 = quotient(m2, n, inv);
    if (!kCta) __syncwarp();  // as in the forward
    if (live) {
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) g[i] = mul2(fma2(h[i], both(-m2), add2(g[i], both(-m1))), both(q));
      if (kJoin) {
        if (a.dz) {
#pragma unroll
          for (int i = 0; i < PAIRS; ++i) g[i] = add2(g[i], part.value(res, i));
        }
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) part.set(t, i, g[i]);
        part.store(static_cast<T*>(a.dresidual) + r * a.s.cols, t);
        if (d.threshold) drop_runs(part, g, r * a.s.cols, d);
      }
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) part.set(t, i, g[i]);
      part.store(static_cast<T*>(a.dx) + r * a.s.cols, t);
    }
  }
  if (!partial && !(alone && (a.dweight || a.dbias))) return;
  float* out = partial + (uint64_t)blockIdx.x * 2 * a.s.cols;
  auto leave = [&](uint32_t which, uint32_t c, float v) {
    if (!alone) out[which * a.s.cols + c] = v;
    else if (void* to = which ? a.dbias : a.dweight) store_as(to, a.wdtype, c, v);
  };
  if (kCta) {
    // whole 16-byte pieces where they fit
    float* to0 = alone ? static_cast<float*>(a.dweight) : out;
    float* to1 = alone ? static_cast<float*>(a.dbias) : out + a.s.cols;
    if (VEC % 4 == 0 && (!alone || (a.wdtype == VS_F32 && (((uintptr_t)to0 | (uintptr_t)to1) & 15u) == 0))) {
#pragma unroll
      for (int i = 0; i + 1 < PAIRS; i += 2) {
        const int k = 2 * i / VEC;
        if (!part.has(k)) continue;
        const uint32_t c = part.col(k) + 2 * i % VEC;
        if (to0) *reinterpret_cast<float4*>(to0 + c) = make_float4(dw[i].x, dw[i].y, dw[i + 1].x, dw[i + 1].y);
        if (to1) *reinterpret_cast<float4*>(to1 + c) = make_float4(db[i].x, db[i].y, db[i + 1].x, db[i + 1].y);
      }
      return;
    }
#pragma unroll
    for (int e = 0; e < P::E; ++e) {
      if (!part.has(e / VEC)) continue;
      const uint32_t c = part.col(e / VEC) + e % VEC;
      leave(0, c, (&dw[e / 2].x)[e % 2]);
      leave(1, c, (&db[e / 2].x)[e % 2]);
    }
    return;
  }
  // lanes with the same columns, then the warps, each in order
  float* mine = sums + (threadIdx.x >> 5) * 2 * a.s.cols;
  for (uint32_t k = 0; k < per_pass; ++k) {
    if (sub == k) {
#pragma unroll
      for (int e = 0; e < P::E; ++e) {
        if (!part.has(e / VEC)) continue;
        const uint32_t c = part.col(e / VEC) + e % VEC;
        const float pw = (&dw[e / 2].x)[e % 2], pb = (&db[e / 2].x)[e % 2];
        mine[c] = k ? mine[c] + pw : pw;
        mine[a.s.cols + c] = k ? mine[a.s.cols + c] + pb : pb;
      }
    }
    __syncwarp();
  }
  __syncthreads();
  const uint32_t pieces = (2 * a.s.cols + 3) / 4;  // of 16 bytes, in which the last CTA reads
  if (ticket) out = partial + (uint64_t)blockIdx.x * 4 * pieces;
  for (uint32_t c = threadIdx.x; c < 2 * a.s.cols; c += BWD_WARPS * 32) {
    float v = sums[c];
    for (uint32_t k = 1; k < BWD_WARPS; ++k) v += sums[k * 2 * a.s.cols + c];
    if (ticket) out[c] = v;
    else leave(c >= a.s.cols, c >= a.s.cols ? c - a.s.cols : c, v);
  }
  if (!ticket) return;
  __shared__ bool last;
  __threadfence();  // the sums are written before the ticket is drawn
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(ticket, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  // groups of threads take every groups-th CTA's sums, 16 bytes a thread; then the
  // groups' sums are added in order
  const uint32_t fit = BWD_WARPS * 32 / pieces, groups = fit < FOLD_GROUPS ? fit : FOLD_GROUPS;
  const uint32_t group = threadIdx.x / pieces, piece = threadIdx.x % pieces;
  if (group < groups) {
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const float4* from = reinterpret_cast<const float4*>(partial) + piece;
#pragma unroll 4
    for (uint32_t k = group; k < gridDim.x; k += groups) {
      const float4 v = __ldcg(from + (uint64_t)k * pieces);
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    reinterpret_cast<float4*>(sums)[group * pieces + piece] = s;
  }
  __syncthreads();
  for (uint32_t c = threadIdx.x; c < 2 * a.s.cols; c += BWD_WARPS * 32) {
    float v = sums[c];
    for (uint32_t k = 1; k < groups; ++k) v += sums[k * 4 * pieces + c];
    const uint32_t which = c >= a.s.cols;
    if (void* to = which ? a.dbias : a.dweight) store_as(to, a.wdtype, which ? c - a.s.cols : c, v);
  }
  if (threadIdx.x == 0) *ticket = 0;  // for the next call
}

// The launch of one shape: a CTA per row of `threads`, or warps.
struct Shape {
  uint32_t grid, threads, log_lanes;
};
// `alone`: up to this many rounds of rows stay on one CTA (a second launch costs
// about 3 us of the host and of the GPU, a round about 1 us).  No CTA takes more than
// `chain` rounds.
template <int VEC, int K, bool kCta>
Shape shape_of(const NormShape& s, uint32_t warps, uint32_t alone, uint64_t chain) {
  const uint32_t chunks = (s.cols + VEC - 1) / VEC;
  Shape l{0, warps * 32, 0};
  uint64_t most = s.rows;
  if (kCta) {
    l.threads = ((chunks + K - 1) / K + 31) & ~31u;
  } else {
    while ((1u << l.log_lanes) * K < chunks) ++l.log_lanes;
    const uint32_t rows = warps * (32u >> l.log_lanes);
    most = (s.rows + rows - 1) / rows;
  }
  uint64_t room = (uint64_t)B200_SMS * (l.threads >= 512 ? 1 : 512 / l.threads);
  room *= most / (room * chain) + 1;
  l.grid = most <= alone ? 1 : (uint32_t)(room < most ? room : most);
  return l;
}

template <typename T, int VEC, int K, bool kJoin, bool kCta> vs_status launch(vs_ctx* ctx, const NormFwd& f) {
  const Shape l = shape_of<VEC, K, kCta>(f.s, FWD_WARPS, 1, ~0u);
  norm_direct_fwd_kernel<T, VEC, K, kJoin, kCta><<<l.grid, l.threads, 0, ctx->stream>>>(f, l.log_lanes, f.d);
  ++ctx->launches;
  return vs_cuda(ctx, cudaGetLastError(), "norm launch");
}
template <typename T, int VEC, int K, bool kJoin, bool kCta> vs_status launch(vs_ctx* ctx, const NormBwd& f) {
  const Shape l = shape_of<VEC, K, kCta>(f.s, BWD_WARPS, 4, NORM_CHAIN);
  const bool want = (f.dweight || f.dbias) && l.grid > 1;
  NormScratch scratch;
  if (want) VS_TRY(norm_scratch_begin(ctx, (size_t)l.grid * (2 * f.s.cols + 3), &scratch));
  const bool fold = want && !kCta && l.grid <= FOLD_CTAS;
  size_t smem = kCta ? 0 : BWD_WARPS * 2 * f.s.cols * 4;
  if (fold && smem < BWD_WARPS * 32 * 16) smem = BWD_WARPS * 32 * 16;
  norm_direct_bwd_kernel<T, VEC, K, kJoin, kCta><<<l.grid, l.threads, smem, ctx->stream>>>(
      f, l.log_lanes, f.d, scratch.p, fold ? scratch.ticket : nullptr);
  ++ctx->launches;
  vs_status st = vs_cuda(ctx, cudaGetLastError(), "norm backward launch");
  if (want) {
    if (st == VS_OK && !fold) st = norm_join_partials(ctx, f.s.cols, l.grid, scratch.p, f.wdtype, f.dweight, f.dbias);
    const vs_status end = norm_scratch_end(ctx, scratch);
    if (st == VS_OK) st = end;
  }
  return st;
}

// KS runs per thread while a CTA of 1024 can hold the row (the shortest chain of
// work per thread), KL beyond, with 512 threads.
template <typename T, int VEC, int KS, int KL, bool kJoin, typename F>
vs_status pick(vs_ctx* ctx, const F& f, bool* taken) {
  *taken = true;
  if (f.s.cols <= 32 * VEC * KS) return launch<T, VEC, KS, kJoin, false>(ctx, f);
  if (f.s.cols <= direct_threads(VEC * KS) * VEC * KS) return launch<T, VEC, KS, kJoin, true>(ctx, f);
  if (f.s.cols <= direct_threads(VEC * KL) * VEC * KL) return launch<T, VEC, KL, kJoin, true>(ctx, f);
  *taken = false;
  return VS_OK;
}

// Whether 16-byte vectors fit the buffers and strides (0 passes).
template <typename T>
bool vectors(uint32_t cols, std::initializer_list<uint64_t> strides, std::initializer_list<const void*> buffers) {
  bool fit = cols % (16 / sizeof(T)) == 0;
  for (uint64_t s : strides) fit = fit && s % (16 / sizeof(T)) == 0;
  for (const void* p : buffers) fit = fit && ((uintptr_t)p & 15u) == 0;
  return fit;
}

}  // namespace

vs_status norm_direct_forward(vs_ctx* ctx, int32_t dtype, bool join, const NormFwd& f, bool* taken) {
  return vs_with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    constexpr int V = 16 / sizeof(T);
    if (vectors<T>(f.s.cols, {f.x_stride, f.residual_stride}, {f.x, f.residual, f.y, f.z}))
      return join ? pick<T, V, 1, 32 / V, true>(ctx, f, taken) : pick<T, V, 1, 32 / V, false>(ctx, f, taken);
    return join ? pick<T, 1, 4, 16, true>(ctx, f, taken) : pick<T, 1, 4, 16, false>(ctx, f, taken);
  });
}

vs_status norm_direct_backward(vs_ctx* ctx, int32_t dtype, bool join, const NormBwd& f, bool* taken) {
  return vs_with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    constexpr int V = 16 / sizeof(T);
    if (vectors<T>(f.s.cols, {f.dy_stride, f.dz_stride, f.z_stride}, {f.dy, f.dz, f.z, f.dx, f.dresidual}))
      return join ? pick<T, V, 1, 16 / V, true>(ctx, f, taken) : pick<T, V, 1, 16 / V, false>(ctx, f, taken);
    return join ? pick<T, 1, 4, 16, true>(ctx, f, taken) : pick<T, 1, 4, 16, false>(ctx, f, taken);
  });
}
