// Layer norm over rows and its gradient, alone or joined with the dropout and
// the residual sum before it (z = residual + dropout(x), y = layer norm of z).
//
//   forward   m = mean z, v = mean (z - m)^2, q = 1 / sqrt(v + eps),
//             y = (z - m) q w + b
//   backward  h = (z - m) q, g = dy w,
//             t = q (g - mean g - h mean(g h)) (+ dz),
//             dresidual = t, dx = dropout(t), dw = sum_rows dy h, db = sum_rows dy
#include <initializer_list>
#include <type_traits>

#include "norm.cuh"

namespace {

using namespace vs;

using Shape = NormShape;

// One CTA per row, three passes over it: any width, stride and alignment, for rows
// that the other kernels do not hold.  The later passes read what the first left in
// L1 and L2; three CTAs an SM (40 registers) hide more of that than two (2000 rows of
// 30001 f32 134 and 155 us, 55 and 47 % of the copy rate).  The
// mean is a quotient, not a product with 1 / cols, so that a constant row whose
// sum is exact has a variance of exactly zero.
//
// A row goes in 16-byte vectors where all its buffers begin alike within 16 bytes, its
// ends and other rows value by value; each pass deals the same values to the same
// thread, so that a pass may read what the thread wrote or overwrite what it read.
constexpr uint32_t ROW_THREADS = 512;
template <typename T> struct RowSplit {
  static constexpr uint32_t V = 16 / sizeof(T);
  uint32_t lead, end, cols;  // whole vectors of [lead, end)
  VSD RowSplit(uint32_t cols_, const void* p, uint32_t differ) : cols(cols_) {
    const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(p) & 15u);
    lead = (16 - off) % 16 / sizeof(T);
    if (lead > cols || (differ & 15u)) lead = cols;
    end = lead + (cols - lead) / V * V;
  }
  // fn(c, number of values from c on)
  template <typename F> VSD void each(F fn) const {
#pragma unroll 2
    for (uint32_t c = lead + threadIdx.x * V; c < end; c += ROW_THREADS * V) fn(c, std::integral_constant<uint32_t, V>());
    for (uint32_t k = threadIdx.x; k < lead + (cols - end); k += ROW_THREADS)
      fn(k < lead ? k : end + (k - lead), std::integral_constant<uint32_t, 1>());
  }
};
VSD uint32_t differ(const void* a, const void* b) {
  return (uint32_t)(reinterpret_cast<uintptr_t>(a) ^ reinterpret_cast<uintptr_t>(b));
}
template <uint32_t N, typename T> VSD void row_load(const T* p, float* v) {
  alignas(16) T t[N];
  if constexpr (N > 1) *reinterpret_cast<uint4*>(t) = *reinterpret_cast<const uint4*>(p);
  else t[0] = p[0];
#pragma unroll
  for (uint32_t j = 0; j < N; ++j) v[j] = to_f32(t[j]);
}
template <uint32_t N, typename T> VSD void row_store(T* p, const float* v) {
  alignas(16) T t[N];
#pragma unroll
  for (uint32_t j = 0; j < N; ++j) t[j] = from_f32<T>(v[j]);
  if constexpr (N > 1) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(t);
  else p[0] = t[0];
}
template <uint32_t N> VSD void row_weights(const void* p, int32_t dtype, uint32_t c, float other, float* v) {
  const float* f = static_cast<const float*>(p) + c;
  if (N > 1 && p && dtype == VS_F32 && (reinterpret_cast<uintptr_t>(f) & 15u) == 0) {
#pragma unroll
    for (uint32_t j = 0; j < N; j += 4) {
      const float4 q = *reinterpret_cast<const float4*>(f + j);
      v[j] = q.x; v[j + 1] = q.y; v[j + 2] = q.z; v[j + 3] = q.w;
    }
    return;
  }
#pragma unroll
  for (uint32_t j = 0; j < N; ++j) v[j] = p ? load_as(p, dtype, c + j) : other;
}
template <uint32_t N> VSD void row_drop(const Dropout& d, uint64_t i, float* v) {
  if (!d.threshold) return;
  if (N > 1 && i % N == 0) {
    const Words words = run_words<N>(d, i);
#pragma unroll
    for (uint32_t j = 0; j < N; ++j) v[j] = dropped(v[j], keeps(words, j, d.limit), d.scale);
    return;
  }
#pragma unroll
  for (uint32_t j = 0; j < N; ++j) v[j] = dropped(v[j], keep_at(d, i + j), d.scale);
}

template <typename T, bool kJoin>
__global__ void __launch_bounds__(ROW_THREADS, 3) norm_fwd_rows_kernel(Shape s, Mat<const T> x, Mat<const T> residual,
                                                                    Weights wt, float eps, const Dropout d, T* y, T* z,
                                                                    float* mean, float* rstd) {
  __shared__ float scratch[33];
  const float cols = (float)s.cols;
  for (uint64_t r = blockIdx.x; r < s.rows; r += gridDim.x) {
    const T *in = x.row(r), *res = kJoin ? residual.row(r) : nullptr;
    T* out = y + r * s.cols;
    T* zr = kJoin ? z + r * s.cols : nullptr;
    const RowSplit<T> split(s.cols, in, differ(in, out) | (kJoin ? differ(in, zr) | differ(in, res) : 0));
    float sum = 0.0f;
    split.each([&](uint32_t c, auto n) {
      constexpr uint32_t N = decltype(n)::value;
      float v[N];
      row_load<N>(in + c, v);
      if constexpr (kJoin) {
        row_drop<N>(d, r * s.cols + c, v);
        float e[N];
        row_load<N>(res + c, e);
#pragma unroll
        for (uint32_t j = 0; j < N; ++j) v[j] = to_f32(from_f32<T>(e[j] + v[j]));
        row_store<N>(zr + c, v);
      }
#pragma unroll
      for (uint32_t j = 0; j < N; ++j) sum += v[j];
    });
    const T* src = kJoin ? zr : in;
    const float m = block_sum(sum, scratch) / cols;
    float sq = 0.0f;
    split.each([&](uint32_t c, auto n) {
      constexpr uint32_t N = decltype(n)::value;
      float v[N];
      row_load<N>(src + c, v);
#pragma unroll
      for (uint32_t j = 0; j < N; ++j) sq = fmaf(v[j] - m, v[j] - m, sq);
    });
    const float q = rsqrtf(block_sum(sq, scratch) / cols + eps);
    split.each([&](uint32_t c, auto n) {
      constexpr uint32_t N = decltype(n)::value;
      float v[N], w[N], b[N];
      row_load<N>(src + c, v);
      row_weights<N>(wt.weight, wt.dtype, c, 1.0f, w);
      row_weights<N>(wt.bias, wt.dtype, c, 0.0f, b);
#pragma unroll
      for (uint32_t j = 0; j < N; ++j) v[j] = fmaf((v[j] - m) * q, w[j], b[j]);
      row_store<N>(out + c, v);
    });
    if (threadIdx.x == 0) {
      if (mean) mean[r] = m;
      if (rstd) rstd[r] = q;
    }
  }
}

template <typename T, bool kJoin>
__global__ void __launch_bounds__(ROW_THREADS, 3) norm_bwd_rows_kernel(Shape s, Mat<const T> dy, Mat<const T> dz,
                                                                    Mat<const T> z, Weights wt, const float* mean,
                                                                    const float* rstd, const Dropout d, T* dx,
                                                                    T* dresidual) {
  __shared__ float scratch[33];
  const float cols = (float)s.cols;
  launch_next();
  for (uint64_t r = blockIdx.x; r < s.rows; r += gridDim.x) {
    const float m = mean[r], q = rstd[r];
    const T *gy = dy.row(r), *zr = z.row(r), *gz = kJoin && dz.p ? dz.row(r) : nullptr;
    T *out = dx + r * s.cols, *res = kJoin ? dresidual + r * s.cols : nullptr;
    const RowSplit<T> split(s.cols, gy, differ(gy, zr) | differ(gy, out) | (kJoin ? differ(gy, res) : 0) |
                                            (gz ? differ(gy, gz) : 0));
    float sg = 0.0f, sgh = 0.0f;
    split.each([&](uint32_t c, auto n) {
      constexpr uint32_t N = decltype(n)::value;
      float g[N], h[N], w[N];
      row_load<N>(gy + c, g);
      row_load<N>(zr + c, h);
      row_weights<N>(wt.weight, wt.dtype, c, 1.0f, w);
#pragma unroll
      for (uint32_t j = 0; j < N; ++j) {
        const float e = g[j] * w[j];
        sg += e;
        sgh = fmaf(e, (h[j] - m) * q, sgh);
      }
    });
    sg = block_sum(sg, scratch) / cols;
    sgh = block_sum(sgh, scratch) / cols;
    split.each([&](uint32_t c, auto n) {
      constexpr uint32_t N = decltype(n)::value;
      float g[N], h[N], w[N];
      row_load<N>(gy + c, g);
      row_load<N>(zr + c, h);
      row_weights<N>(wt.weight, wt.dtype, c, 1.0f, w);
#pragma unroll
      for (uint32_t j = 0; j < N; ++j) g[j] = q * (g[j] * w[j] - sg - (h[j] - m) * q * sgh);
      if constexpr (kJoin) {
        if (gz) {
          row_load<N>(gz + c, h);
#pragma unroll
          for (uint32_t j = 0; j < N; ++j) g[j] += h[j];
        }
        row_store<N>(res + c, g);
        row_drop<N>(d, r * s.cols + c, g);
      }
      row_store<N>(out + c, g);
    });
  }
}

// Column sums of a strip of rows: partial[strip][0] = sum dy h, [1] = sum dy.
// 32 x 8 threads of four columns each (bf16 rows of 16384, the whole backward 308 us,
// one column each 516); each thread's rows are summed in order, then the eight in
// order, so the result does not depend on timing.
constexpr uint32_t COLS_EACH = 4, COLS_WIDE = 32 * COLS_EACH;  // columns of a thread and of a CTA
template <typename T>
__global__ void __launch_bounds__(256) norm_cols_kernel(Shape s, Mat<const T> dy, Mat<const T> z, const float* mean,
                                                        const float* rstd, uint64_t strip, float* partial) {
  __shared__ float sw[8][COLS_WIDE], sb[8][COLS_WIDE];
  const uint64_t c0 = (uint64_t)blockIdx.x * COLS_WIDE + threadIdx.x;
  const uint64_t r0 = blockIdx.y * strip;
  const uint64_t r1 = r0 + strip < s.rows ? r0 + strip : s.rows;
  float w[COLS_EACH], b[COLS_EACH];
#pragma unroll
  for (uint32_t j = 0; j < COLS_EACH; ++j) w[j] = b[j] = 0.0f;
#pragma unroll 2
  for (uint64_t r = r0 + threadIdx.y; r < r1; r += 8) {
    const T *g = dy.row(r) + c0, *v = z.row(r) + c0;
    const float m = mean[r], q = rstd[r];
#pragma unroll
    for (uint32_t j = 0; j < COLS_EACH; ++j) {
      if (c0 + 32 * j >= s.cols) continue;
      const float e = to_f32(g[32 * j]);
      w[j] = fmaf(e, (to_f32(v[32 * j]) - m) * q, w[j]);
      b[j] += e;
    }
  }
#pragma unroll
  for (uint32_t j = 0; j < COLS_EACH; ++j) {
    sw[threadIdx.y][threadIdx.x + 32 * j] = w[j];
    sb[threadIdx.y][threadIdx.x + 32 * j] = b[j];
  }
  __syncthreads();
  const uint32_t k = threadIdx.y * 32 + threadIdx.x;
  const uint64_t c = (uint64_t)blockIdx.x * COLS_WIDE + k;
  if (k < COLS_WIDE && c < s.cols) {
    float tw = 0.0f, tb = 0.0f;
    for (uint32_t y = 0; y < 8; ++y) {
      tw += sw[y][k];
      tb += sb[y][k];
    }
    float* out = partial + (uint64_t)blockIdx.y * 2 * s.cols;
    out[c] = tw;
    out[s.cols + c] = tb;
  }
}

// dw and db from `strips` partial sums [strips][2][cols]: a CTA takes 32 columns
// of one of the two, GROUPS groups of 8 threads take every GROUPS-th strip's
// 16-byte pieces of them, and the groups' sums are added in a fixed order.
template <uint32_t GROUPS>
__global__ void __launch_bounds__(GROUPS * 8) norm_join_kernel(uint32_t cols, uint32_t strips, const float* partial,
                                                         int32_t dtype, void* dweight, void* dbias) {
  __shared__ float4 part[GROUPS][9];
  const uint32_t piece = threadIdx.x & 7u, group = threadIdx.x >> 3;
  const uint32_t c = blockIdx.x * 32 + piece * 4;
  const float* from = partial + (uint64_t)blockIdx.y * cols + c;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the sums' kernel has ended and its writes are visible
  float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (cols % 4 == 0) {
    if (c < cols) {
#pragma unroll 4
      for (uint32_t k = group; k < strips; k += GROUPS) {
        const float4 v = *reinterpret_cast<const float4*>(from + (uint64_t)k * 2 * cols);
        s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
      }
    }
  } else {
#pragma unroll 2
    for (uint32_t k = group; k < strips; k += GROUPS) {
      const float* p = from + (uint64_t)k * 2 * cols;
      if (c < cols) s.x += p[0];
      if (c + 1 < cols) s.y += p[1];
      if (c + 2 < cols) s.z += p[2];
      if (c + 3 < cols) s.w += p[3];
    }
  }
  part[group][piece] = s;
  __syncthreads();
  // a warp per column
  const uint32_t lane = threadIdx.x & 31u;
  void* out = blockIdx.y ? dbias : dweight;
  for (uint32_t col = threadIdx.x >> 5; col < 32; col += GROUPS / 4) {
    float v = 0.0f;
#pragma unroll
    for (uint32_t k = lane; k < GROUPS; k += 32) v += reinterpret_cast<const float*>(&part[k][col >> 2])[col & 3u];
    v = warp_sum(v);
    if (lane == 0 && blockIdx.x * 32 + col < cols && out) store_as(out, dtype, blockIdx.x * 32 + col, v);
  }
}

// What every entry point checks of its shape.
vs_status check_shape(vs_ctx* ctx, const char* what, uint64_t rows, uint32_t cols, int32_t dtype, int32_t wdtype) {
  if (!vs_dtype_valid(dtype)) return vs_fail(ctx, VS_ERR_UNSUPPORTED, "%s: element type %d", what, dtype);
  if (wdtype != VS_F32 && wdtype != dtype)
    return vs_fail(ctx, VS_ERR_UNSUPPORTED, "%s: weights of type %d beside rows of type %d (f32 or the rows' type)",
                   what, wdtype, dtype);
  if (cols == 0) return vs_fail(ctx, VS_ERR_INVALID, "%s: rows without columns", what);
  if (cols > 0x7fffffffu || rows > (1ull << 60) / cols)
    return vs_fail(ctx, VS_ERR_CAPACITY, "%s: %llu rows of %u columns", what, (unsigned long long)rows, cols);
  return VS_OK;
}

// An input's buffer; a stride of 0 stands for `cols`.
template <typename T>
vs_status check_in(vs_ctx* ctx, const char* what, const char* name, Shape s, const void* p, uint64_t stride,
                   Mat<const T>* out) {
  if (stride == 0) stride = s.cols;
  if (!p && s.rows) return vs_fail(ctx, VS_ERR_INVALID, "%s: null %s", what, name);
  if (stride < s.cols || (s.rows > 1 && stride > (1ull << 60) / s.rows))
    return vs_fail(ctx, VS_ERR_INVALID, "%s: %s rows %llu apart, %u wide", what, name, (unsigned long long)stride, s.cols);
  if ((uintptr_t)p & (sizeof(T) - 1)) return vs_fail(ctx, VS_ERR_INVALID, "%s: %s is not aligned to its element", what, name);
  *out = {static_cast<const T*>(p), stride};
  return VS_OK;
}

vs_status check_ptr(vs_ctx* ctx, const char* what, const char* name, const void* p, size_t align, bool needed) {
  if (needed && !p) return vs_fail(ctx, VS_ERR_INVALID, "%s: null %s", what, name);
  if ((uintptr_t)p & (align - 1)) return vs_fail(ctx, VS_ERR_INVALID, "%s: %s is not aligned to its element", what, name);
  return VS_OK;
}

// Whether the streaming kernels can take the rows: contiguous, on 16-byte
// aligned buffers (NULL passes).
bool vector_rows(Shape s, std::initializer_list<uint64_t> strides, std::initializer_list<const void*> buffers) {
  for (uint64_t stride : strides)
    if (stride != s.cols && s.rows > 1) return false;
  for (const void* p : buffers)
    if ((uintptr_t)p & 15u) return false;
  return true;
}

uint32_t row_grid(uint64_t rows) { return (uint32_t)(rows < 0x7fffffffull ? rows : 0x7fffffffull); }

template <typename T, bool kJoin>
vs_status norm_forward(vs_ctx* ctx, const char* what, int32_t dtype, Shape s, const void* x, uint64_t x_stride, const void* residual,
                       uint64_t residual_stride, Weights wt, float eps, const Dropout& d, void* y, void* z,
                       float* mean, float* rstd) {
  Mat<const T> mx, mr{};
  VS_TRY(check_in<T>(ctx, what, "x", s, x, x_stride, &mx));
  if (kJoin) VS_TRY(check_in<T>(ctx, what, "residual", s, residual, residual_stride, &mr));
  VS_TRY(check_ptr(ctx, what, "y", y, sizeof(T), s.rows > 0));
  if (kJoin) VS_TRY(check_ptr(ctx, what, "z", z, sizeof(T), s.rows > 0));
  VS_TRY(check_ptr(ctx, what, "mean", mean, 4, false));
  VS_TRY(check_ptr(ctx, what, "rstd", rstd, 4, false));
  VS_TRY(check_ptr(ctx, what, "weight", wt.weight, vs_dtype_size(wt.dtype), false));
  VS_TRY(check_ptr(ctx, what, "bias", wt.bias, vs_dtype_size(wt.dtype), false));
  // a row's statistics are written while other rows still read the weights
  for (const float* stat : {mean, rstd})
    if (stat && (stat == wt.weight || stat == wt.bias))
      return vs_fail(ctx, VS_ERR_INVALID, "%s: mean and rstd cannot share the weight's or the bias's buffer", what);
  if (!(eps >= 0.0f) || eps > 3e38f) return vs_fail(ctx, VS_ERR_INVALID, "%s: eps = %g", what, (double)eps);
  if (s.rows == 0) return VS_OK;
  VS_CUDA(ctx, cudaSetDevice(ctx->device));
  const NormFwd f{s, x, residual, mx.stride, mr.stride, wt, eps, d, y, z, mean, rstd};
  const bool stream = vector_rows(s, {mx.stride, kJoin ? mr.stride : mx.stride}, {x, residual, y, z});
  bool taken = false;
  if (stream) VS_TRY(norm_tile_forward(ctx, dtype, kJoin, f, &taken));
  if (stream && !taken) VS_TRY(norm_row_forward(ctx, dtype, kJoin, f, &taken));
  if (!taken) VS_TRY(norm_direct_forward(ctx, dtype, kJoin, f, &taken));
  if (taken) return VS_OK;
  norm_fwd_rows_kernel<T, kJoin><<<row_grid(s.rows), ROW_THREADS, 0, ctx->stream>>>(s, mx, mr, wt, eps, d, (T*)y, (T*)z, mean,
                                                                            rstd);
  ++ctx->launches;
  return vs_cuda(ctx, cudaGetLastError(), "norm launch");
}

template <typename T, bool kJoin>
vs_status norm_backward(vs_ctx* ctx, const char* what, int32_t dtype, Shape s, const void* dy, uint64_t dy_stride, const void* dz,
                        uint64_t dz_stride, const void* z, uint64_t z_stride, Weights wt, const float* mean,
                        const float* rstd, const Dropout& d, void* dx, void* dresidual, void* dweight, void* dbias) {
  Mat<const T> mdy, mdz{}, mz;
  VS_TRY(check_in<T>(ctx, what, "dy", s, dy, dy_stride, &mdy));
  if (kJoin && dz) VS_TRY(check_in<T>(ctx, what, "dz", s, dz, dz_stride, &mdz));
  VS_TRY(check_in<T>(ctx, what, kJoin ? "z" : "x", s, z, z_stride, &mz));
  VS_TRY(check_ptr(ctx, what, "mean", mean, 4, s.rows > 0));
  VS_TRY(check_ptr(ctx, what, "rstd", rstd, 4, s.rows > 0));
  VS_TRY(check_ptr(ctx, what, "dx", dx, sizeof(T), s.rows > 0));
  if (kJoin) VS_TRY(check_ptr(ctx, what, "dresidual", dresidual, sizeof(T), s.rows > 0));
  VS_TRY(check_ptr(ctx, what, "weight", wt.weight, vs_dtype_size(wt.dtype), false));
  VS_TRY(check_ptr(ctx, what, "dweight", dweight, vs_dtype_size(wt.dtype), false));
  VS_TRY(check_ptr(ctx, what, "dbias", dbias, vs_dtype_size(wt.dtype), false));
  VS_CUDA(ctx, cudaSetDevice(ctx->device));
  if (s.rows == 0) {
    if (dweight) VS_CUDA(ctx, cudaMemsetAsync(dweight, 0, s.cols * vs_dtype_size(wt.dtype), ctx->stream));
    if (dbias) VS_CUDA(ctx, cudaMemsetAsync(dbias, 0, s.cols * vs_dtype_size(wt.dtype), ctx->stream));
    return VS_OK;
  }
  const NormBwd f{s, dy, kJoin ? dz : nullptr, z, mdy.stride, mdz.stride, mz.stride, wt, mean, rstd, d, dx, dresidual,
                  wt.dtype, dweight, dbias};
  const bool stream = vector_rows(s, {mdy.stride, mz.stride, kJoin && dz ? mdz.stride : mz.stride},
                                  {dy, dz, z, dx, dresidual, mean, rstd});
  // Small calls leave fewer CTAs' sums to join when they run direct: 20k x 64 f16
  // (8 MB of the plain kernel's traffic, which decides for the joined one too, so
  // that both add up the same sums) 17 and 25 us, 1000 x 4096 bf16 (25 MB) 23 and
  // 25 us, 2000 x 4096 35 and 29 us.
  const bool small = (double)s.rows * s.cols * sizeof(T) * 3 < 16e6;
  bool taken = false;
  if (stream && !small) VS_TRY(norm_tile_backward(ctx, dtype, kJoin, f, &taken));
  if (stream && !small && !taken) VS_TRY(norm_row_backward(ctx, dtype, kJoin, f, &taken));
  if (!taken) VS_TRY(norm_direct_backward(ctx, dtype, kJoin, f, &taken));
  if (!taken && stream && small) VS_TRY(norm_row_backward(ctx, dtype, kJoin, f, &taken));
  if (taken) return VS_OK;
  // The column sums read dy, which dx may overwrite, so they come before the rows; dx
  // reads the weight, which dweight may overwrite, so the sums are joined after them.
  const bool want = dweight || dbias;
  const uint32_t col_blocks = (s.cols + COLS_WIDE - 1) / COLS_WIDE;
  uint64_t even = 1184 / col_blocks + 1;  // CTAs for every SM, and no thread with more than NORM_CHAIN rows
  if (even < s.rows / (8 * NORM_CHAIN) + 1) even = s.rows / (8 * NORM_CHAIN) + 1;
  const uint64_t most = (s.rows + 15) / 16;
  const uint32_t strips = (uint32_t)(even < most ? even : most);
  NormScratch scratch;
  vs_status st = VS_OK;
  if (want) {
    VS_TRY(norm_scratch_begin(ctx, (size_t)strips * 2 * s.cols, &scratch));
    norm_cols_kernel<T><<<dim3(col_blocks, strips), dim3(32, 8), 0, ctx->stream>>>(
        s, mdy, mz, mean, rstd, (s.rows + strips - 1) / strips, scratch.p);
    ++ctx->launches;
    st = vs_cuda(ctx, cudaGetLastError(), "norm column sums launch");
  }
  if (st == VS_OK) {
    norm_bwd_rows_kernel<T, kJoin><<<row_grid(s.rows), ROW_THREADS, 0, ctx->stream>>>(s, mdy, mdz, mz, wt, mean, rstd, d,
                                                                              (T*)dx, (T*)dresidual);
    ++ctx->launches;
    st = vs_cuda(ctx, cudaGetLastError(), "norm backward launch");
  }
  if (want) {
    if (st == VS_OK) st = norm_join_partials(ctx, s.cols, strips, scratch.p, wt.dtype, dweight, dbias);
    const vs_status end = norm_scratch_end(ctx, scratch);
    if (st == VS_OK) st = end;
  }
  return st;
}

}  // namespace

vs_status norm_join_partials(vs_ctx* ctx, uint32_t cols, uint32_t strips, const float* partial, int32_t dtype,
                             void* dweight, void* dbias) {
  // launched beside the kernel that writes the sums, which it waits for: its
  // launch is over by then
  cudaLaunchConfig_t config{};
  config.gridDim = dim3((cols + 31) / 32, 2);
  const bool few = strips <= 128;
  config.blockDim = dim3(few ? 256 : 1024);
  config.stream = ctx->stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  VS_CUDA(ctx, cudaLaunchKernelEx(&config, few ? norm_join_kernel<32> : norm_join_kernel<128>, cols, strips, partial,
                                  dtype, dweight, dbias));
  ++ctx->launches;
  return VS_OK;
}

// Calls on one stream follow one another, so each stream has one buffer (the
// first NORM_STREAMS that call).  A call being captured into a graph gets memory of
// the graph's own, since the graph may run beside other calls.
vs_status norm_scratch_begin(vs_ctx* ctx, size_t floats, NormScratch* out) {
  const size_t bytes = 16 + floats * 4;  // the ticket, then the floats
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  VS_CUDA(ctx, cudaStreamIsCapturing(ctx->stream, &capture));
  uint32_t k = 0;
  out->pooled = capture != cudaStreamCaptureStatusNone;
  if (!out->pooled) {
    VS_CUDA(ctx, cudaStreamGetId(ctx->stream, &id));  // not while capturing: it ends the capture
    while (k < ctx->norm_streams && ctx->norm_stream[k] != id) ++k;
    out->pooled = k == vs_ctx::NORM_STREAMS;
  }
  void* at = nullptr;
  bool fresh = true;
  if (out->pooled) {
    VS_CUDA(ctx, cudaMallocAsync(&at, bytes, ctx->stream));
  } else {
    if (k == ctx->norm_streams) ctx->norm_stream[ctx->norm_streams++] = id;
    const size_t before = ctx->norm_sums[k].bytes;
    VS_TRY(vs_ensure(ctx, ctx->norm_sums[k], bytes));
    at = ctx->norm_sums[k].ptr;
    fresh = ctx->norm_sums[k].bytes != before;
  }
  out->ticket = static_cast<uint32_t*>(at);
  out->p = static_cast<float*>(at) + 4;
  return fresh ? vs_cuda(ctx, cudaMemsetAsync(at, 0, 16, ctx->stream), "norm scratch") : VS_OK;
}
vs_status norm_scratch_end(vs_ctx* ctx, const NormScratch& scratch) {
  return scratch.pooled ? vs_cuda(ctx, cudaFreeAsync(scratch.ticket, ctx->stream), "norm scratch") : VS_OK;
}

extern "C" {

VS_API vs_status vs_layer_norm(vs_ctx* ctx, uint64_t rows, uint32_t cols, int32_t dtype, int32_t weight_dtype,
                               const void* x, uint64_t x_stride, const void* weight, const void* bias, float eps,
                               void* y, float* mean, float* rstd) {
  if (!ctx) return VS_ERR_INVALID;
  VS_TRY(check_shape(ctx, "layer_norm", rows, cols, dtype, weight_dtype));
  return vs_with_dtype(dtype, [&](auto tag) {
    return norm_forward<decltype(tag), false>(ctx, "layer_norm", dtype, {rows, cols}, x, x_stride, nullptr, 0,
                                              {weight, bias, weight_dtype}, eps, vs::Dropout{}, y, nullptr, mean,
                                              rstd);
  });
}

VS_API vs_status vs_layer_norm_backward(vs_ctx* ctx, uint64_t rows, uint32_t cols, int32_t dtype,
                                        int32_t weight_dtype, const void* dy, uint64_t dy_stride, const void* x,
                                        uint64_t x_stride, const void* weight, const float* mean, const float* rstd,
                                        void* dx, void* dweight, void* dbias) {
  if (!ctx) return VS_ERR_INVALID;
  VS_TRY(check_shape(ctx, "layer_norm_backward", rows, cols, dtype, weight_dtype));
  return vs_with_dtype(dtype, [&](auto tag) {
    return norm_backward<decltype(tag), false>(ctx, "layer_norm_backward", dtype, {rows, cols}, dy, dy_stride, nullptr, 0, x,
                                               x_stride, {weight, nullptr, weight_dtype}, mean, rstd, vs::Dropout{},
                                               dx, nullptr, dweight, dbias);
  });
}

VS_API vs_status vs_dropout_add_norm(vs_ctx* ctx, uint64_t rows, uint32_t cols, int32_t dtype, int32_t weight_dtype,
                                     const void* x, uint64_t x_stride, const void* residual, uint64_t residual_stride,
                                     const void* weight, const void* bias, double p, uint64_t seed, uint64_t offset,
                                     float eps, void* y, void* z, float* mean, float* rstd) {
  if (!ctx) return VS_ERR_INVALID;
  VS_TRY(check_shape(ctx, "dropout_add_norm", rows, cols, dtype, weight_dtype));
  vs::Dropout d;
  VS_TRY(vs_make_dropout(ctx, "dropout_add_norm", p, seed, offset, &d));
  return vs_with_dtype(dtype, [&](auto tag) {
    return norm_forward<decltype(tag), true>(ctx, "dropout_add_norm", dtype, {rows, cols}, x, x_stride, residual,
                                             residual_stride, {weight, bias, weight_dtype}, eps, d, y, z, mean, rstd);
  });
}

VS_API vs_status vs_dropout_add_norm_backward(vs_ctx* ctx, uint64_t rows, uint32_t cols, int32_t dtype,
                                              int32_t weight_dtype, const void* dy, uint64_t dy_stride,
                                              const void* dz, uint64_t dz_stride, const void* z, uint64_t z_stride,
                                              const void* weight, const float* mean, const float* rstd, double p,
                                              uint64_t seed, uint64_t offset, void* dx, void* dresidual,
                                              void* dweight, void* dbias) {
  if (!ctx) return VS_ERR_INVALID;
  VS_TRY(check_shape(ctx, "dropout_add_norm_backward", rows, cols, dtype, weight_dtype));
  vs::Dropout d;
  VS_TRY(vs_make_dropout(ctx, "dropout_add_norm_backward", p, seed, offset, &d));
  return vs_with_dtype(dtype, [&](auto tag) {
    return norm_backward<decltype(tag), true>(ctx, "dropout_add_norm_backward", dtype, {rows, cols}, dy, dy_stride, dz,
                                              dz_stride, z, z_stride, {weight, nullptr, weight_dtype}, mean, rstd, d,
                                              dx, dresidual, dweight, dbias);
  });
}

}  // extern "C"
