// Streaming layer norm, forward and backward, alone or joined, for long
// contiguous rows: a CTA per row, a ring of two slots filled by bulk copies.
//
// Any width runs on 16-byte vectors.  The grid is a multiple of the values in a
// vector, so all rows of one CTA start at the same place within a vector; the
// threads deal out the whole aligned vectors of the row, and where its ends are
// ragged one more warp takes the few values before the first and behind the last
// of them, a lane each.  A thread's columns are the same for every row, so weights
// and weight gradients stay with it.
#include <atomic>
#include <type_traits>

#include "norm.cuh"

namespace {

using namespace vs;

// Threads that an SM holds of the forward and of the backward by the values each
// one holds: their registers fix it.
template <typename T, int K, bool kJoin> constexpr uint32_t row_fwd() {
  return K * (16 / sizeof(T)) <= 16 ? 768 : kJoin ? 384 : 512;
}
template <typename T, int K> constexpr uint32_t row_bwd() { return K * (16 / sizeof(T)) <= 16 ? 512 : 384; }

struct RowArgs {
  uint64_t rows;
  uint32_t cols, slot, stages, inputs, ragged;  // ragged: 1 where the last warp takes the rows' ends
  const void* in[3];  // x, residual; or dy, z, dz
  Weights w;
  float eps;
  void *out0, *out1;  // y, z; or dx, dresidual
  float *mean, *rstd;
  float* partial;  // [CTA][2][cols], NULL when no weight gradient is wanted
  uint32_t* err;
};

// Where a CTA's rows lie: `shift` values into their first vector, with `lead`
// values before the first whole vector and `vectors` of those.
template <typename T> struct RowPlace {
  static constexpr uint32_t V = 16 / sizeof(T);
  uint32_t shift, lead, vectors;
  VSD explicit RowPlace(uint32_t cols) {
    shift = (uint32_t)((uint64_t)blockIdx.x * cols % V);
    lead = (V - shift) % V;
    vectors = cols > lead ? (cols - lead) / V : 0;
  }
};

// The sums over a CTA whose warps are in two different loops.
VSD void row_sync() { asm volatile("barrier.sync.aligned 1, %0;" ::"r"(blockDim.x) : "memory"); }
VSD float row_sum(float v, float* part, uint32_t warps) {
  v = warp_sum(v);
  if ((threadIdx.x & 31u) == 0) part[threadIdx.x >> 5] = v;
  row_sync();
  return parts_sum(part, warps);
}

// A thread's K vectors.
template <typename T, int K> struct RowPart {
  static constexpr int V = 16 / sizeof(T);
  static constexpr int E = V * K;
  static constexpr int PAIRS = E / 2;
  using R = typename Raw<T, V>::type;
  static constexpr int WORDS = 16 / sizeof(R);  // pairs of a vector
  uint32_t at, threads, lead, vectors;

  VSD bool has(int k) const { return at + k * threads < vectors; }
  VSD uint32_t col(int k) const { return lead + (at + k * threads) * V; }
  // the vectors of a row whose first value lies at `row` in shared memory, the 16
  // zero bytes at `zeros` for those beyond it
  VSD void load(uint32_t row, uint32_t zeros, R* t) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const uint4 q = lds16(has(k) ? row + col(k) * (uint32_t)sizeof(T) : zeros);
      if constexpr (WORDS == 4) {
        t[k * 4] = q.x; t[k * 4 + 1] = q.y; t[k * 4 + 2] = q.z; t[k * 4 + 3] = q.w;
      } else {
        t[k * 2] = make_float2(__uint_as_float(q.x), __uint_as_float(q.y));
        t[k * 2 + 1] = make_float2(__uint_as_float(q.z), __uint_as_float(q.w));
      }
    }
  }
  VSD void store(T* row, const R* t) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!has(k)) continue;
      uint4 q;
      if constexpr (WORDS == 4) q = make_uint4(t[k * 4], t[k * 4 + 1], t[k * 4 + 2], t[k * 4 + 3]);
      else q = make_uint4(__float_as_uint(t[k * 2].x), __float_as_uint(t[k * 2].y), __float_as_uint(t[k * 2 + 1].x),
                          __float_as_uint(t[k * 2 + 1].y));
      *reinterpret_cast<uint4*>(row + col(k)) = q;
    }
  }
  VSD float2 value(const R* t, int i) const { return unpack(static_cast<const T*>(nullptr), t[i]); }
  VSD void set(R* t, int i, float2 v) const { pack(static_cast<const T*>(nullptr), v, t[i]); }
  // v - m for the row's values, zero for the others (which hold zero)
  VSD void subtract(float2* v, float m) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float2 s = both(has(k) ? -m : 0.0f);
#pragma unroll
      for (int i = k * V / 2; i < (k + 1) * V / 2; ++i) v[i] = add2(v[i], s);
    }
  }
  VSD void weights(const void* p, int32_t dtype, float other, float2* w) const {
    if (p && dtype == VS_F32 && ((uintptr_t)(static_cast<const float*>(p) + lead) & 15u) == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int j = 0; j < V; j += 4) {
          const float4 q = has(k) ? *reinterpret_cast<const float4*>(static_cast<const float*>(p) + col(k) + j)
                                  : make_float4(other, other, other, other);
          w[(k * V + j) / 2] = make_float2(q.x, q.y);
          w[(k * V + j) / 2 + 1] = make_float2(q.z, q.w);
        }
      }
      return;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) (&w[e / 2].x)[e % 2] = p && has(e / V) ? load_as(p, dtype, col(e / V) + e % V) : other;
  }
  // Dropout of the values; i0 is the index of the row's first one.
  VSD void drop(float2* v, uint64_t i0, const Dropout& d) const {
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) v[i] = mul2(v[i], both(d.scale));
    float* f = reinterpret_cast<float*>(v);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const uint64_t e = i0 + col(k);
      const Words words = run_words<V>(d, e);
#pragma unroll
      for (int j = 0; j < V; ++j) f[k * V + j] = keeps(words, j, d.limit) ? f[k * V + j] : 0.0f;
    }
  }
};

// The ring of one CTA.
template <typename T> struct RowRing {
  const RowArgs& a;
  unsigned char* slots;
  uint64_t* full;
  uint32_t base;  // the first slot's row in shared memory, `shift` values into the slot
  uint64_t total, row_bytes, load_at;  // load_at: where the next row to be copied begins (thread 0's)
  VSD RowRing(const RowArgs& a_, unsigned char* s, uint64_t* f, uint32_t shift)
      : a(a_), slots(s), full(f), base(smem_u32(s) + shift * (uint32_t)sizeof(T)) {
    row_bytes = (uint64_t)a.cols * sizeof(T);
    total = a.rows * row_bytes;
    load_at = blockIdx.x * row_bytes;
  }
  VSD uint32_t row(uint32_t slot, uint32_t input) const { return base + (slot * a.inputs + input) * a.slot; }
  VSD void refill(uint32_t slot) {
    if (load_at < total) {
      const Span s = span_of(load_at, load_at + row_bytes, total);
      mbar_expect(&full[slot], s.bytes * a.inputs);
      for (uint32_t k = 0; k < a.inputs; ++k) span_load(s, slots + (slot * a.inputs + k) * a.slot, a.in[k], &full[slot]);
    }
    load_at += gridDim.x * row_bytes;
  }
  VSD void start() {
    for (uint32_t k = 0; k < a.stages; ++k) mbar_init(&full[k], 1);
    mbar_init_fence();
    for (uint32_t k = 0; k < a.stages; ++k) refill(k);
  }
  // A single value of a row that begins at byte `begin`; the buffers' last,
  // unwhole 16 bytes are not copied.
  VSD float single(uint32_t slot, uint32_t input, uint64_t begin, uint32_t c) const {
    const uint64_t at = begin + c * sizeof(T);
    if (at >= (total & ~15ull)) return to_f32(static_cast<const T*>(a.in[input])[at / sizeof(T)]);
    return lds_value<T>(row(slot, input) + c * (uint32_t)sizeof(T));
  }
  // After a copy that did not land in time: report it and wait for those in flight, as
  // long again for each.
  VSD void give_up(uint32_t slot, uint32_t parity, uint64_t row) const {
    atomicOr(a.err, VS_DERR_WAIT);
    for (uint32_t k = 0; k < a.stages && row < a.rows; ++k, row += gridDim.x) {
      mbar_wait(&full[slot], parity);
      if (++slot == a.stages) {
        slot = 0;
        parity ^= 1;
      }
    }
  }
};

// The ragged ends' warp: its lane's column, or none.
template <typename T> VSD bool end_column(const RowPlace<T>& place, uint32_t cols, uint32_t* c) {
  const uint32_t lane = threadIdx.x & 31u;
  *c = lane < 16 ? lane : place.lead + place.vectors * RowPlace<T>::V + (lane - 16);
  return lane < 16 ? lane < place.lead && lane < cols : *c < cols;
}

template <typename T, int K, bool kJoin>
__global__ void __launch_bounds__(row_fwd<T, K, kJoin>()) norm_row_fwd_kernel(const RowArgs a, const __grid_constant__ Dropout d) {
  using P = RowPart<T, K>;
  constexpr int PAIRS = P::PAIRS;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) uint64_t full[NORM_STAGES];
  __shared__ __align__(16) float red[2][NORM_MAX_WARPS];
  __shared__ uint4 zeros;
  __shared__ uint32_t late;
  const uint32_t tid = threadIdx.x, warps = blockDim.x >> 5;
  const RowPlace<T> place(a.cols);
  RowRing<T> ring(a, smem, full, place.shift);
  for (uint32_t k = tid; k < 2 * NORM_MAX_WARPS; k += blockDim.x) (&red[0][0])[k] = 0.0f;
  if (tid == 0) {
    late = 0;
    zeros = make_uint4(0, 0, 0, 0);
    ring.start();
  }
  __syncthreads();
  const float n = (float)a.cols, inv = 1.0f / n;
  T *y = static_cast<T*>(a.out0), *z = static_cast<T*>(a.out1);
  uint32_t slot = 0, parity = 0;
  uint64_t row = blockIdx.x, begin = row * ring.row_bytes;
  const uint64_t step = gridDim.x * ring.row_bytes;

  if (a.ragged && tid >> 5 == warps - 1) {
    uint32_t c;
    const bool mine = end_column(place, a.cols, &c);
    const float w = mine && a.w.weight ? load_as(a.w.weight, a.w.dtype, c) : 1.0f;
    const float b = mine && a.w.bias ? load_as(a.w.bias, a.w.dtype, c) : 0.0f;
    for (; row < a.rows; row += gridDim.x, begin += step) {
      if (!mbar_wait(&full[slot], parity)) late = 1;
      const uint64_t at = begin / sizeof(T) + c;
      float v = 0.0f;
      if (mine) {
        v = ring.single(slot, 0, begin, c);
        if (kJoin) {
          if (d.threshold) v = dropped(v, keep_at(d, at), d.scale);
          v = to_f32(from_f32<T>(v + ring.single(slot, 1, begin, c)));
        }
      }
      const float m = quotient(row_sum(v, red[0], warps), n, inv);
      const bool stop = late;
      const float e = mine ? v - m : 0.0f;
      const float q = rsqrtf(fmaf(row_sum(e * e, red[1], warps), inv, a.eps));
      if (stop) return;
      if (mine) {
        if (kJoin) z[at] = from_f32<T>(v);
        y[at] = from_f32<T>(fmaf(e * q, w, b));
      }
      if (++slot == a.stages) {
        slot = 0;
        parity ^= 1;
      }
    }
    return;
  }

  const P part{tid, blockDim.x - 32 * a.ragged, place.lead, place.vectors};
  float2 w[PAIRS], b[PAIRS];
  part.weights(a.w.weight, a.w.dtype, 1.0f, w);
  part.weights(a.w.bias, a.w.dtype, 0.0f, b);
  bool ok = true;
  for (; row < a.rows; row += gridDim.x, begin += step) {
    if (!mbar_wait(&full[slot], parity)) late = 1;
    const uint64_t i0 = begin / sizeof(T);
    float2 v[PAIRS];
    typename P::R t[PAIRS];
    part.load(ring.row(slot, 0), smem_u32(&zeros), t);
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) v[i] = part.value(t, i);
    if (kJoin) {
      if (d.threshold) part.drop(v, i0, d);
      part.load(ring.row(slot, 1), smem_u32(&zeros), t);
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        part.set(t, i, add2(v[i], part.value(t, i)));  // z, rounded as it is stored
        v[i] = part.value(t, i);
      }
    }
    float2 s = both(0.0f);
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) s = add2(s, v[i]);
    const float m = quotient(row_sum(s.x + s.y, red[0], warps), n, inv);
    ok = !late;  // between two barriers: the same for all
    part.subtract(v, m);
    s = both(0.0f);
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) s = fma2(v[i], v[i], s);
    const float q = rsqrtf(fmaf(row_sum(s.x + s.y, red[1], warps), inv, a.eps));
    if (!ok) break;
    if (tid == 0) ring.refill(slot);  // every thread has its part in registers
    if (kJoin) part.store(z + i0, t);
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) part.set(t, i, fma2(mul2(v[i], both(q)), w[i], b[i]));
    part.store(y + i0, t);
    if (tid == 0) {
      if (a.mean) a.mean[row] = m;
      if (a.rstd) a.rstd[row] = q;
    }
    if (++slot == a.stages) {
      slot = 0;
      parity ^= 1;
    }
  }
  if (!ok && tid == 0) ring.give_up(slot, parity, row);
}

template <typename T, int K, bool kJoin>
__global__ void __launch_bounds__(row_bwd<T, K>()) norm_row_bwd_kernel(const RowArgs a, const __grid_constant__ Dropout d) {
  using P = RowPart<T, K>;
  constexpr int PAIRS = P::PAIRS;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) uint64_t full[NORM_STAGES];
  __shared__ __align__(16) float red[2][2][NORM_MAX_WARPS];
  __shared__ uint4 zeros;
  __shared__ uint32_t late[2];
  const uint32_t tid = threadIdx.x, warps = blockDim.x >> 5;
  const RowPlace<T> place(a.cols);
  RowRing<T> ring(a, smem, full, place.shift);
  for (uint32_t k = tid; k < 4 * NORM_MAX_WARPS; k += blockDim.x) (&red[0][0][0])[k] = 0.0f;
  if (tid == 0) {
    late[0] = late[1] = 0;
    zeros = make_uint4(0, 0, 0, 0);
    ring.start();
  }
  __syncthreads();
  launch_next();
  const float n = (float)a.cols, inv = 1.0f / n;
  T *dx = static_cast<T*>(a.out0), *dres = static_cast<T*>(a.out1);
  float* out = a.partial ? a.partial + (uint64_t)blockIdx.x * 2 * a.cols : nullptr;
  uint32_t slot = 0, parity = 0, half = 0;
  uint64_t row = blockIdx.x, begin = row * ring.row_bytes;
  const uint64_t step = gridDim.x * ring.row_bytes;
  float m_next = a.mean[row], q_next = a.rstd[row];
  // the next row's statistics travel while a row is worked on
  auto statistics = [&](float* m, float* q) {
    *m = m_next;
    *q = q_next;
    if (row + gridDim.x < a.rows) {
      m_next = a.mean[row + gridDim.x];
      q_next = a.rstd[row + gridDim.x];
    }
  };
  // the row's two sums; `red` and `late` alternate between two rows, so one barrier per row is enough
  auto sums = [&](float s1, float s2, float* m1, float* m2) {
    const float s = warp_sum2(s1, s2);
    if ((tid & 15u) == 0) red[half][tid >> 4 & 1u][tid >> 5] = s;
    row_sync();
    *m1 = quotient(parts_sum(red[half][0], warps), n, inv);
    *m2 = quotient(parts_sum(red[half][1], warps), n, inv);
    const bool good = !late[half];
    half ^= 1;
    return good;
  };

  if (a.ragged && tid >> 5 == warps - 1) {
    uint32_t c;
    const bool mine = end_column(place, a.cols, &c);
    const float w = mine && a.w.weight ? load_as(a.w.weight, a.w.dtype, c) : 1.0f;
    float dw = 0.0f, db = 0.0f;
    for (; row < a.rows; row += gridDim.x, begin += step) {
      float m, q, m1, m2;
      statistics(&m, &q);
      if (!mbar_wait(&full[slot], parity)) late[half] = 1;
      const uint64_t at = begin / sizeof(T) + c;
      const float dy = mine ? ring.single(slot, 0, begin, c) : 0.0f;
      const float h = mine ? (ring.single(slot, 1, begin, c) - m) * q : 0.0f;
      const float res = mine && a.inputs == 3 ? ring.single(slot, 2, begin, c) : 0.0f;
      dw = fmaf(dy, h, dw);
      db += dy;
      if (!sums(dy * w, dy * w * h, &m1, &m2)) return;
      if (mine) {
        const float t = q * fmaf(h, -m2, dy * w - m1) + res;
        if (kJoin) dres[at] = from_f32<T>(t);
        dx[at] = from_f32<T>(kJoin && d.threshold ? dropped(t, keep_at(d, at), d.scale) : t);
      }
      if (++slot == a.stages) {
        slot = 0;
        parity ^= 1;
      }
    }
    if (out && mine) {
      out[c] = dw;
      out[a.cols + c] = db;
    }
    return;
  }

  const P part{tid, blockDim.x - 32 * a.ragged, place.lead, place.vectors};
  // the weights, each thread's own at places of its own
  const uint32_t ws = smem_u32(smem) + a.stages * a.inputs * a.slot + tid * 16, ws_step = blockDim.x * 16;
  float2 dw[PAIRS], db[PAIRS];
  part.weights(a.w.weight, a.w.dtype, 1.0f, dw);
#pragma unroll
  for (int i = 0; i < PAIRS; i += 2)
    sts16(ws + i / 2 * ws_step, make_uint4(__float_as_uint(dw[i].x), __float_as_uint(dw[i].y),
                                           __float_as_uint(dw[i + 1].x), __float_as_uint(dw[i + 1].y)));
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) dw[i] = db[i] = both(0.0f);
  bool ok = true;
  for (; row < a.rows; row += gridDim.x, begin += step) {
    float m, q, m1, m2;
    statistics(&m, &q);
    if (!mbar_wait(&full[slot], parity)) late[half] = 1;
    const uint64_t i0 = begin / sizeof(T);
    typename P::R t[PAIRS], res[kJoin ? PAIRS : 1];
    float2 g[PAIRS], h[PAIRS];
    part.load(ring.row(slot, 0), smem_u32(&zeros), t);
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) g[i] = part.value(t, i);
    part.load(ring.row(slot, 1), smem_u32(&zeros), t);
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) h[i] = mul2(add2(part.value(t, i), both(-m)), both(q));
    if constexpr (kJoin)
      if (a.inputs == 3) part.load(ring.row(slot, 2), smem_u32(&zeros), res);
    float2 s1 = both(0.0f), s2 = both(0.0f);
#pragma unroll
    for (int i = 0; i < PAIRS; i += 2) {  // g is zero for values that are not the row's
      const uint4 w = lds16(ws + i / 2 * ws_step);
#pragma unroll
      for (int j = i; j < i + 2; ++j) {
        dw[j] = fma2(g[j], h[j], dw[j]);
        db[j] = add2(db[j], g[j]);
        g[j] = mul2(g[j], j > i ? make_float2(__uint_as_float(w.z), __uint_as_float(w.w))
                                     : make_float2(__uint_as_float(w.x), __uint_as_float(w.y)));
        s1 = add2(s1, g[j]);
        s2 = fma2(g[j], h[j], s2);
      }
    }
    ok = sums(s1.x + s1.y, s2.x + s2.y, &m1, &m2);
    if (!ok) break;
    if (tid == 0) ring.refill(slot);  // every thread has its part in registers
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) g[i] = mul2(fma2(h[i], both(-m2), add2(g[i], both(-m1))), both(q));
    if constexpr (kJoin) {
      if (a.inputs == 3) {
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) g[i] = add2(g[i], part.value(res, i));
      }
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) part.set(t, i, g[i]);
      part.store(dres + i0, t);
      if (d.threshold) part.drop(g, i0, d);
    }
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) part.set(t, i, g[i]);
    part.store(dx + i0, t);
    if (++slot == a.stages) {
      slot = 0;
      parity ^= 1;
    }
  }
  if (!ok && tid == 0) ring.give_up(slot, parity, row);
  if (!out) return;
  if (!ok) {  // the sums are marked invalid, those of the ends' warp too, which has left
    for (uint32_t c = tid; c < 2 * a.cols; c += part.threads) out[c] = nan_value();
    return;
  }
  if (a.cols % 4 == 0 && place.lead % 4 == 0) {  // whole 16-byte pieces: single values would cost the L2 a write each
#pragma unroll
    for (int i = 0; i < PAIRS; i += 2) {
      const int k = 2 * i / P::V;
      if (!part.has(k)) continue;
      float* to = out + part.col(k) + 2 * i % P::V;
      *reinterpret_cast<float4*>(to) = make_float4(dw[i].x, dw[i].y, dw[i + 1].x, dw[i + 1].y);
      *reinterpret_cast<float4*>(to + a.cols) = make_float4(db[i].x, db[i].y, db[i + 1].x, db[i + 1].y);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < P::E; ++e) {
    if (!part.has(e / P::V)) continue;
    const uint32_t c = part.col(e / P::V) + e % P::V;
    out[c] = (&dw[e / 2].x)[e % 2];
    out[a.cols + c] = (&db[e / 2].x)[e % 2];
  }
}

// Threads of a CTA.
template <typename T, int K> uint32_t row_threads(uint32_t cols) {
  constexpr uint32_t V = 16 / sizeof(T);
  return ((cols / V + K - 1) / K + 31) / 32 * 32 + (cols % V ? 32 : 0);
}

// Grid and slots of a shape; `held` bytes per thread stand beside the ring (of the
// backward, whose threads add up NORM_CHAIN rows each at most), and the grid is that of
// CTAs of `grid_threads` threads of `sm_threads` with `inputs` inputs.  CTAs beyond what
// keeps `flight` bytes on their way only queue at the DRAM: one input, f32 rows of 1024,
// 6 CTAs 95 % of the copy rate, 8 CTAs 85 %; two inputs, bf16 rows of 4096, 3 CTAs 96 %,
// 4 CTAs 76 %.  False where the slots do not fit.
template <typename T>
bool lay_out(RowArgs* a, uint32_t threads, uint32_t grid_threads, uint32_t sm_threads, uint32_t inputs, uint32_t held,
             uint32_t* grid, size_t* smem) {
  constexpr uint32_t V = 16 / sizeof(T);
  if (threads > sm_threads || grid_threads > sm_threads) return false;
  a->ragged = a->cols % V != 0;
  a->slot = (a->cols * (uint32_t)sizeof(T) + 30u) & ~15u;
  const uint32_t flight = (inputs > 1 ? 96 : sizeof(T) == 4 ? 48 : 64) * 1024, each = 2 * inputs * a->slot;
  uint32_t per_sm = sm_threads / grid_threads;
  if (per_sm > (flight + each - 1) / each) per_sm = (flight + each - 1) / each;
  auto bytes = [&](uint32_t in, uint32_t stages) { return stages * in * a->slot + threads * held; };
  auto room = [&] { return NORM_MAX_SMEM / per_sm - 1024; };
  while (per_sm > 1 && bytes(inputs, 2) > room()) --per_sm;
  if (bytes(inputs, 1) > room()) return false;
  a->stages = bytes(a->inputs, 2) <= room() ? 2 : 1;
  *smem = bytes(a->inputs, a->stages);
  const uint64_t once = (uint64_t)per_sm * B200_SMS / V * V;
  const uint64_t full = held ? once * (a->rows / (once * NORM_CHAIN) + 1) : once;
  *grid = (uint32_t)(a->rows < full ? a->rows : full);
  return true;
}

template <typename Kernel>
vs_status allow_smem(vs_ctx* ctx, Kernel kernel, std::atomic<uint64_t>& ready) {
  const uint64_t bit = 1ull << (ctx->device & 63);
  if (ready.load(std::memory_order_relaxed) & bit) return VS_OK;
  VS_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)NORM_MAX_SMEM));
  ready.fetch_or(bit);
  return VS_OK;
}

template <typename T, int K, bool kJoin> vs_status run(vs_ctx* ctx, const NormFwd& f, bool* taken) {
  static std::atomic<uint64_t> ready{0};
  RowArgs a{};
  a.rows = f.s.rows;
  a.cols = f.s.cols;
  a.inputs = kJoin ? 2 : 1;
  a.in[0] = f.x; a.in[1] = f.residual; a.w = f.w; a.eps = f.eps; a.out0 = f.y; a.out1 = f.z;
  a.mean = f.mean; a.rstd = f.rstd; a.err = ctx->d_err;
  const uint32_t threads = row_threads<T, K>(a.cols);
  uint32_t grid;
  size_t smem;
  if (!lay_out<T>(&a, threads, threads, row_fwd<T, K, kJoin>(), a.inputs, 0, &grid, &smem)) return VS_OK;
  auto kernel = norm_row_fwd_kernel<T, K, kJoin>;
  VS_TRY(allow_smem(ctx, kernel, ready));
  *taken = true;
  kernel<<<grid, threads, smem, ctx->stream>>>(a, f.d);
  ++ctx->launches;
  return vs_cuda(ctx, cudaGetLastError(), "norm launch");
}

template <typename T, int K, int KG, bool kJoin> vs_status run(vs_ctx* ctx, const NormBwd& f, bool* taken) {
  static std::atomic<uint64_t> ready{0};
  RowArgs a{};
  a.rows = f.s.rows;
  a.cols = f.s.cols;
  a.inputs = f.dz ? 3 : 2;
  a.in[0] = f.dy; a.in[1] = f.z; a.in[2] = f.dz; a.w = f.w; a.out0 = f.dx; a.out1 = f.dresidual;
  a.mean = const_cast<float*>(f.mean); a.rstd = const_cast<float*>(f.rstd); a.err = ctx->d_err;
  // the grid is the joined kernel's for both, so that they add up the same sums
  const uint32_t threads = row_threads<T, K>(a.cols);
  uint32_t grid;
  size_t smem;
  if (!lay_out<T>(&a, threads, row_threads<T, KG>(a.cols), row_bwd<T, K>(), 3, RowPart<T, K>::E * 4, &grid, &smem)) return VS_OK;
  auto kernel = norm_row_bwd_kernel<T, K, kJoin>;
  VS_TRY(allow_smem(ctx, kernel, ready));
  *taken = true;
  const bool want = f.dweight || f.dbias;
  NormScratch scratch;
  if (want) VS_TRY(norm_scratch_begin(ctx, (size_t)grid * 2 * a.cols, &scratch));
  a.partial = scratch.p;
  kernel<<<grid, threads, smem, ctx->stream>>>(a, f.d);
  ++ctx->launches;
  vs_status st = vs_cuda(ctx, cudaGetLastError(), "norm backward launch");
  if (want) {
    if (st == VS_OK) st = norm_join_partials(ctx, a.cols, grid, a.partial, f.wdtype, f.dweight, f.dbias);
    const vs_status end = norm_scratch_end(ctx, scratch);
    if (st == VS_OK) st = end;
  }
  return st;
}

// Values per thread: 32 make fewer instructions per value, 16 more warps.  Forward,
// bf16 rows of 4096: 32 values 92 %, 16 values 74 % of the copy rate, of 1544 75 and 63 %
// (from there on 16 values take more than 96 threads), of 1536 75 and 80 %, f16 rows of
// 1030, whose ends take a warp, 51 and 60 %.  Plain f32 rows of 1536 82 and 89 %, of 4096
// 90 and 93 %, of 12288 91 and 93 %; joined ones, whose vectors need a generator call
// each, of 1536 80 and 81 %, of 2049 83 and 72 %, of 4096 94 and 86 %.
template <typename T, bool kJoin> vs_status pick(vs_ctx* ctx, const NormFwd& f, bool* taken) {
  constexpr int V = 16 / sizeof(T);
  const uint32_t most = sizeof(T) == 2 ? 1543 : kJoin ? 2047 : ~0u;  // columns for 16 values
  if (f.s.cols <= most) VS_TRY((run<T, 16 / V, kJoin>(ctx, f, taken)));
  if (!*taken) VS_TRY((run<T, 32 / V, kJoin>(ctx, f, taken)));
  // beside their ends' warp, 16 values a thread hold 512 columns more of joined rows
  if (kJoin && !*taken && f.s.cols > most) VS_TRY((run<T, 16 / V, kJoin>(ctx, f, taken)));
  return VS_OK;
}
// Backward: bf16 rows of 4096, joined, 17k of them, 16 values 83 %, 32 values 51 %; the
// joined f32 kernel holds 8 where it can (8192 x 4096 93 %, 32 values 42 %).
template <typename T, bool kJoin> vs_status pick(vs_ctx* ctx, const NormBwd& f, bool* taken) {
  constexpr int V = 16 / sizeof(T), S = 16 / V, L = 32 / V;
  if constexpr (sizeof(T) == 4) VS_TRY((run<T, kJoin ? 2 : S, 2, kJoin>(ctx, f, taken)));
  if (!*taken) VS_TRY((run<T, S, S, kJoin>(ctx, f, taken)));
  if (!*taken) VS_TRY((run<T, L, L, kJoin>(ctx, f, taken)));
  return VS_OK;
}

}  // namespace

vs_status norm_row_forward(vs_ctx* ctx, int32_t dtype, bool join, const NormFwd& f, bool* taken) {
  return vs_with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    return join ? pick<T, true>(ctx, f, taken) : pick<T, false>(ctx, f, taken);
  });
}
vs_status norm_row_backward(vs_ctx* ctx, int32_t dtype, bool join, const NormBwd& f, bool* taken) {
  return vs_with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    return join ? pick<T, true>(ctx, f, taken) : pick<T, false>(ctx, f, taken);
  });
}
