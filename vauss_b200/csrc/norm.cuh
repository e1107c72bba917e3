// The layer-norm kernels' shared pieces: shapes, the bulk-copy ring that feeds
// the streaming kernels, and the launchers norm.cu chooses between.
#pragma once

#include <initializer_list>

#include "rows.cuh"

namespace vs {

// Rows of `cols` values that start `stride` values apart.
template <typename T> struct Mat {
  T* p;
  uint64_t stride;
  VSD T* row(uint64_t r) const { return p + r * stride; }
};

struct NormShape {
  uint64_t rows;
  uint32_t cols;
};

// ---- bulk copies into shared memory ---------------------------------------
VSD uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
VSD void mbar_init(uint64_t* b, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(b)), "r"(count) : "memory");
}
VSD void mbar_init_fence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
VSD void mbar_expect(uint64_t* b, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(b)), "r"(bytes) : "memory");
}
VSD bool mbar_try(uint64_t* b, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(b)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Waits for a copy to land; false after a second without it.  The caller then sets
// the device error word and ends, so what it had yet to write is undefined; the column
// sums of its CTA become NaN.
constexpr uint64_t COPY_WAIT_NS = 1000000000ull;
constexpr uint32_t COPY_SPIN_LIMIT = 1u << 26;  // backstop on the iteration count
VSD uint64_t copy_clock_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}
VSD bool mbar_wait(uint64_t* b, uint32_t parity) {
  if (mbar_try(b, parity)) return true;
  const uint64_t t0 = copy_clock_ns();
  for (uint32_t spins = 0; spins < COPY_SPIN_LIMIT && copy_clock_ns() - t0 < COPY_WAIT_NS; ++spins)
    if (mbar_try(b, parity)) return true;
  return false;
}
// dst, src 16-byte aligned, bytes a multiple of 16
VSD void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
VSD void bulk_store(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(src)),
               "r"(bytes)
               : "memory");
}
VSD void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// all but the newest `N` groups of stores have been read out of shared memory
template <int N> VSD void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }
template <int N> VSD void bulk_wait() { asm volatile("cp.async.bulk.wait_group %0;" ::"n"(N) : "memory"); }
VSD void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Loads and stores by shared-memory address.
VSD uint4 lds16(uint32_t at) {
  uint4 q;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w) : "r"(at));
  return q;
}
VSD void sts16(uint32_t at, uint4 q) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(q.x), "r"(q.y), "r"(q.z), "r"(q.w) : "memory");
}
template <typename T> VSD float lds_value(uint32_t at) {
  if constexpr (sizeof(T) == 4) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at));
    return v;
  } else {
    unsigned short v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at));
    return to_f32(reinterpret_cast<const T&>(v));
  }
}

// A run [begin, end) of bytes of a 16-byte aligned buffer of `total` bytes, as
// bulk copies see it: they move the aligned pieces that cover the run, [lo, hi);
// where the buffer's last piece is not whole, its bytes [hi, end) are copied by
// hand.  In shared memory the run starts `shift` bytes into its slot.
struct Span {
  uint64_t begin, end, lo;
  uint32_t bytes;  // hi - lo
  uint32_t shift;
};
VSD Span span_of(uint64_t begin, uint64_t end, uint64_t total) {
  Span s;
  s.begin = begin;
  s.end = end;
  s.lo = begin & ~15ull;
  uint64_t hi = (end + 15) & ~15ull;
  if (hi > (total & ~15ull)) hi = total & ~15ull;
  s.bytes = hi > s.lo ? (uint32_t)(hi - s.lo) : 0;
  s.shift = (uint32_t)begin & 15u;
  return s;
}

VSD void span_load(const Span& s, void* slot, const void* base, uint64_t* bar) {
  if (s.bytes) bulk_load(slot, static_cast<const char*>(base) + s.lo, s.bytes, bar);
}
// The bytes the bulk copy left out, by `threads` threads; the caller
// synchronises them.
template <typename U>
VSD void span_tail(const Span& s, void* slot, const void* base, uint32_t thread, uint32_t threads) {
  uint64_t at = s.lo + s.bytes;
  if (at < s.begin) at = s.begin;
  for (uint64_t i = at / sizeof(U) + thread; i < s.end / sizeof(U); i += threads)
    reinterpret_cast<U*>(static_cast<char*>(slot) + (i * sizeof(U) - s.lo))[0] = static_cast<const U*>(base)[i];
}
// Writes the run back: whole 16-byte pieces by one thread's bulk store, the
// ragged ends (which belong to neighbouring runs too) value by value.
template <typename U> VSD void span_store(const Span& s, const void* slot, void* base, uint32_t lane) {
  const uint64_t a = (s.begin + 15) & ~15ull, b = s.end & ~15ull;
  if (lane == 0 && a < b)
    bulk_store(static_cast<char*>(base) + a, static_cast<const char*>(slot) + (a - s.lo), (uint32_t)(b - a));
  if (a == s.begin && b == s.end) return;
  const uint64_t head = a < s.end ? a : s.end;
  for (uint64_t i = s.begin / sizeof(U) + lane; i < head / sizeof(U); i += 32)
    static_cast<U*>(base)[i] = reinterpret_cast<const U*>(static_cast<const char*>(slot) + (i * sizeof(U) - s.lo))[0];
  const uint64_t tail = b > head ? b : head;
  for (uint64_t i = tail / sizeof(U) + lane; i < s.end / sizeof(U); i += 32)
    static_cast<U*>(base)[i] = reinterpret_cast<const U*>(static_cast<const char*>(slot) + (i * sizeof(U) - s.lo))[0];
}

VSD float nan_value() { return __uint_as_float(0x7fc00000u); }

// Two f32 operations in one instruction.
VSD unsigned long long bits2(float2 a) { return reinterpret_cast<unsigned long long&>(a); }
VSD float2 add2(float2 a, float2 b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)));
  return reinterpret_cast<float2&>(r);
}
VSD float2 mul2(float2 a, float2 b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)));
  return reinterpret_cast<float2&>(r);
}
VSD float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
  return reinterpret_cast<float2&>(r);
}
VSD float2 both(float v) { return make_float2(v, v); }

// ---- pairs of values as they lie in memory ----------------------------------
// Two neighbouring values: one word for 16-bit types, or two where every value
// is read on its own (VEC = 1).
template <typename T, int VEC> struct Raw { using type = uint32_t; };
template <int VEC> struct Raw<float, VEC> { using type = float2; };
template <> struct Raw<__half, 1> { using type = uint2; };
template <> struct Raw<__nv_bfloat16, 1> { using type = uint2; };

VSD float2 unpack(const __half*, uint32_t u) { return __half22float2(reinterpret_cast<const __half2&>(u)); }
VSD float2 unpack(const __half*, uint2 u) {
  return make_float2(__half2float(__ushort_as_half((unsigned short)u.x)),
                     __half2float(__ushort_as_half((unsigned short)u.y)));
}
VSD float2 unpack(const __nv_bfloat16*, uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
VSD float2 unpack(const __nv_bfloat16*, uint2 u) {
  return make_float2(__uint_as_float(u.x << 16), __uint_as_float(u.y << 16));
}
VSD float2 unpack(const float*, float2 u) { return u; }
VSD void pack(const float*, float2 v, float2& u) { u = v; }
VSD void pack(const __half*, float2 v, uint32_t& u) {
  const __half2 h = __float22half2_rn(v);
  u = reinterpret_cast<const uint32_t&>(h);
}
VSD void pack(const __nv_bfloat16*, float2 v, uint32_t& u) {
  const __nv_bfloat162 h = __float22bfloat162_rn(v);
  u = reinterpret_cast<const uint32_t&>(h);
}
template <typename T> VSD void pack(const T* t, float2 v, uint2& u) {
  uint32_t both_values;
  pack(t, v, both_values);
  u = make_uint2(both_values, both_values >> 16);  // the first value is read and stored by its lower half
}
VSD float keep_if(float v, uint32_t mask) { return __uint_as_float(__float_as_uint(v) & mask); }

// The values of a row that one thread holds: K runs of VEC.  `kSpread` deals
// them out run by run, so that a warp's accesses are contiguous; where K is even
// the runs' order turns with the row's place in the warp, which keeps the rows'
// like runs off each other's shared-memory banks; a run beyond the row reads the
// row's first one.  Otherwise a thread holds a block of K runs, K odd, so that a
// warp's narrow accesses to shared memory fall into different banks and every
// offset is a constant; there a run beyond the row reads what lies behind it (the
// next row, or the slot's padding).  Where a row does not fill a warp's lanes such
// values are cleared before they are used.
constexpr uint32_t NORM_PADDING = 128;  // bytes behind the last slot that such reads may reach
template <typename T, int VEC, int K, bool kSpread = VEC * sizeof(T) == 16> struct Part {
  static constexpr int E = VEC * K;
  static constexpr int RUNS = K;
  static constexpr int PAIRS = (E + 1) / 2;
  static constexpr bool kVector = VEC * sizeof(T) == 16;
  using R = typename Raw<T, VEC>::type;
  uint32_t at, lanes, sub;
  bool full;                      // the same for a warp
  uint32_t off[kSpread ? K : 1];  // where the runs are read
  uint32_t have;                  // the runs that are the row's, as bits (spread) or their number (blocks)
  static constexpr bool kMasks = K <= 16;
  uint32_t masks[kMasks ? K : 1];  // all ones for the row's runs, where registers allow

  VSD Part(uint32_t at_, uint32_t lanes_, uint32_t sub_, uint32_t cols) : at(at_), lanes(lanes_), sub(sub_), have(0) {
#pragma unroll
    for (int k = 0; k < K; ++k) have += col(k) < cols ? (kSpread ? 1u << k : 1u) : 0u;
    full = __all_sync(0xffffffffu, have == (kSpread ? (1u << K) - 1 : (uint32_t)K));
    if constexpr (kMasks) {
#pragma unroll
      for (int k = 0; k < K; ++k) masks[k] = has(k) ? 0xffffffffu : 0u;
    }
    if constexpr (kSpread) {
#pragma unroll
      for (int k = 0; k < K; ++k) off[k] = has(k) ? col(k) : 0;
    } else {
      // a thread wholly beyond the row reads what the row's last thread reads
      const uint32_t last = (cols - 1) / E;
      off[0] = (at < last ? at : last) * E;
    }
  }
  VSD uint32_t col(int k) const {
    if (kSpread) return (at + lanes * (K % 2 ? k : (k + sub) % K)) * VEC;
    return (at * K + k) * VEC;
  }
  VSD bool has(int k) const { return kSpread ? have >> k & 1u : k < (int)have; }
  VSD uint32_t mask(int k) const {
    if constexpr (kMasks) return masks[k];
    else return has(k) ? 0xffffffffu : 0u;
  }
  // where run k is read, from the row's start
  VSD uint32_t from(int k) const { return kSpread ? off[kSpread ? k : 0] : off[0] + k * VEC; }
  VSD void load(const T* row, R* t) const {
    if constexpr (kVector) {
      constexpr int W = 16 / sizeof(R);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const uint4 q = *reinterpret_cast<const uint4*>(row + from(k));
        if constexpr (W == 4) {
          t[k * W] = q.x; t[k * W + 1] = q.y; t[k * W + 2] = q.z; t[k * W + 3] = q.w;
        } else {
          t[k * W] = make_float2(__uint_as_float(q.x), __uint_as_float(q.y));
          t[k * W + 1] = make_float2(__uint_as_float(q.z), __uint_as_float(q.w));
        }
      }
    } else if constexpr (VEC == 4 && sizeof(T) == 2) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const uint2 q = *reinterpret_cast<const uint2*>(row + from(k));
        t[2 * k] = q.x;
        t[2 * k + 1] = q.y;
      }
    } else if constexpr (VEC == 2 && sizeof(T) == 2) {
#pragma unroll
      for (int k = 0; k < K; ++k) t[k] = *reinterpret_cast<const uint32_t*>(row + from(k));
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if constexpr (sizeof(T) == 2) (&t[k / 2].x)[k % 2] = *reinterpret_cast<const uint16_t*>(row + from(k));
        else (&t[k / 2].x)[k % 2] = *reinterpret_cast<const float*>(row + from(k));
      }
      if constexpr (E % 2 == 1) t[E / 2].y = 0;
    }
  }
  VSD void store(T* row, const R* t) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!has(k)) continue;
      if constexpr (kVector) {
        constexpr int W = 16 / sizeof(R);
        uint4 q;
        if constexpr (W == 4) q = make_uint4(t[k * W], t[k * W + 1], t[k * W + 2], t[k * W + 3]);
        else q = make_uint4(__float_as_uint(t[k * W].x), __float_as_uint(t[k * W].y), __float_as_uint(t[k * W + 1].x),
                            __float_as_uint(t[k * W + 1].y));
        *reinterpret_cast<uint4*>(row + from(k)) = q;
      } else if constexpr (VEC == 4 && sizeof(T) == 2) {
        *reinterpret_cast<uint2*>(row + from(k)) = make_uint2(t[2 * k], t[2 * k + 1]);
      } else if constexpr (VEC == 2 && sizeof(T) == 2) {
        *reinterpret_cast<uint32_t*>(row + from(k)) = t[k];
      } else if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint16_t*>(row + from(k)) = (uint16_t)(&t[k / 2].x)[k % 2];
      } else {
        *reinterpret_cast<float*>(row + from(k)) = (&t[k / 2].x)[k % 2];
      }
    }
  }
  // A [cols] vector of weights, `other` where there is none.
  VSD void weights(const void* p, int32_t dtype, float other, float2* w) const {
    if constexpr (kSpread && VEC % 4 == 0) {
      if (p && dtype == VS_F32 && ((uintptr_t)p & 15u) == 0) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
          for (int j = 0; j < VEC; j += 4) {
            const float4 q = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + from(k) + j);
            w[(k * VEC + j) / 2] = make_float2(q.x, q.y);
            w[(k * VEC + j) / 2 + 1] = make_float2(q.z, q.w);
          }
        }
        return;
      }
    }
#pragma unroll
    for (int e = 0; e < 2 * PAIRS; ++e)
      (&w[e / 2].x)[e % 2] =
          e < E && p && has(e / VEC) ? load_as(p, dtype, col(e / VEC) + e % VEC) : other;
  }
  // Zero for the values that are not the row's.
  VSD void clear(R* t) const {
    if (full) return;
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      const uint32_t mx = mask(2 * i / VEC), my = 2 * i + 1 < E ? mask((2 * i + 1) / VEC) : 0;
      if constexpr (sizeof(T) == 4) {
        t[i].x = keep_if(t[i].x, mx);
        t[i].y = keep_if(t[i].y, my);
      } else if constexpr (VEC == 1) {
        t[i].x &= mx;
        t[i].y &= my;
      } else {
        t[i] &= mx;
      }
    }
  }
  VSD float2 value(const R* t, int pair) const { return unpack(static_cast<const T*>(nullptr), t[pair]); }
  VSD void set(R* t, int pair, float2 v) const { pack(static_cast<const T*>(nullptr), v, t[pair]); }
  // v - m for the row's values, zero for the others (which hold zero)
  VSD void subtract(float2* v, float m) const {
    if (full) {
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) v[i] = add2(v[i], 2 * i + 1 < E ? both(-m) : make_float2(-m, 0.0f));
    } else {
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        const float x = keep_if(-m, mask(2 * i / VEC));
        const float y = 2 * i + 1 >= E ? 0.0f : VEC > 1 ? x : keep_if(-m, mask((2 * i + 1) / VEC));
        v[i] = add2(v[i], make_float2(x, y));
      }
    }
  }
};

// Lets the kernel that joins the column sums be launched; it waits by itself.
VSD void launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// The sum over groups of `lanes` (a power of two) neighbouring lanes.
VSD float lanes_sum(float v, uint32_t lanes) {
#pragma unroll
  for (uint32_t o = 16; o > 0; o >>= 1)
    if (o < lanes) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// sum / n with inv = 1 / n rounded correctly, for a whole n below 2^16 (the columns of a
// row): the correction of a quotient by its remainder that P. Markstein describes
// ("Computation of elementary functions on the IBM RISC System/6000 processor", 1990).
// q is within two units of its last place, and the remainder is a multiple of one unit,
// since n is whole, and below 2^18 of them, so the fma gives it exactly; sum / n lies at
// least 1 / 2n of a unit from the middle between two f32 values, far more than the rounded
// inverse leaves in the second fma.  So the result is the correctly rounded quotient
// wherever that is a normal number; an infinite one stays as it is.
VSD float quotient(float sum, float n, float inv) {
  const float q = sum * inv;
  const float r = fmaf(fmaf(-q, n, sum), inv, q);
  return fabsf(q) <= 3.402823466e38f ? r : q;
}

// The keep decisions of one group as bits.
VSD uint32_t keep_bits(const Words& w, uint32_t limit) {
  uint32_t bits = 0;
#pragma unroll
  for (uint32_t j = 0; j < 8; ++j) bits |= (keeps(w, j, limit) ? 1u : 0u) << j;
  return bits;
}

// The numbers of a run of four or eight values from index e, a multiple of the
// run: the first words, where a run of four is a group's second half.
template <int VEC> VSD Words run_words(const Dropout& d, uint64_t e) {
  Words w = philox(d, e >> 3);
  if (VEC == 4 && (e & 4u)) {
    w.w[0] = w.w[2];
    w.w[1] = w.w[3];
  }
  return w;
}

// Dropout of a thread's values, decided one run at a time.
template <typename P> VSD void drop_runs(const P& part, float2* v, uint64_t i0, const Dropout& d) {
  constexpr int VEC = P::E / P::RUNS;
#pragma unroll
  for (int i = 0; i < P::PAIRS; ++i) v[i] = mul2(v[i], both(d.scale));
  float* f = reinterpret_cast<float*>(v);
#pragma unroll
  for (int k = 0; k < P::RUNS; ++k) {
    const uint64_t e = i0 + part.from(k);
    if constexpr (VEC == 1) {
      f[k] = keep_at(d, e) ? f[k] : 0.0f;
    } else {
      const Words words = run_words<VEC>(d, e);
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[k * VEC + j] = keeps(words, j, d.limit) ? f[k * VEC + j] : 0.0f;
    }
  }
}

// Dropout of a thread's values: v holds pairs, i0 is the row's first index.
// Runs of eight are groups of the generator; for others the decisions have been
// left in `bits`, the row's first at bit `at`.
template <typename T, int VEC, int K>
VSD void drop_part(const Part<T, VEC, K>& part, float2* v, uint64_t i0, const Dropout& d, const uint32_t* bits,
                   uint32_t at) {
  const float2 scale = both(d.scale);
#pragma unroll
  for (int i = 0; i < part.PAIRS; ++i) v[i] = mul2(v[i], scale);
  float* f = reinterpret_cast<float*>(v);
  if constexpr (VEC == 8) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const Words words = philox(d, (i0 + part.off[k]) >> 3);
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[k * VEC + j] = keeps(words, j, d.limit) ? f[k * VEC + j] : 0.0f;
    }
  } else if constexpr (part.kVector) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const uint32_t e = at + part.off[k];
      const uint32_t kept = reinterpret_cast<const unsigned char*>(bits)[e >> 3] >> (e & 7u);
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[k * VEC + j] = kept >> j & 1u ? f[k * VEC + j] : 0.0f;
    }
  } else {  // a block of at most 32 values
    const uint32_t e = at + part.off[0];
    const uint32_t kept = __funnelshift_r(bits[e >> 5], bits[(e >> 5) + 1], e & 31u);
#pragma unroll
    for (int j = 0; j < part.E; ++j) f[j] = kept >> j & 1u ? f[j] : 0.0f;
  }
}
// Leaves the decisions of indices [i0, i0 + count) for drop_part, the first at bit i0 & 7.
VSD void fill_bits(const Dropout& d, uint64_t i0, uint32_t count, uint32_t* bits, uint32_t id, uint32_t members) {
  const uint64_t g0 = i0 >> 3;
  const uint32_t groups = (((uint32_t)i0 & 7u) + count + 7) >> 3;
  for (uint32_t g = id; g < groups; g += members)
    reinterpret_cast<unsigned char*>(bits)[g] = (unsigned char)keep_bits(philox(d, g0 + g), d.limit);
}

// The sum over a CTA, the same in every thread; `part` holds a value per warp,
// with zeros up to a multiple of four, and is free for the next use after
// another barrier.
constexpr uint32_t NORM_MAX_WARPS = 32;
VSD float parts_sum(const float* part, uint32_t warps) {
  const float4* p = reinterpret_cast<const float4*>(part);
  float4 s = p[0];
  for (uint32_t k = 1; k < (warps + 3) / 4; ++k) {
    const float4 q = p[k];
    s.x += q.x;
    s.y += q.y;
    s.z += q.z;
    s.w += q.w;
  }
  return (s.x + s.y) + (s.z + s.w);
}
VSD float cta_sum(float v, float* part, uint32_t warps) {
  v = warp_sum(v);
  if ((threadIdx.x & 31u) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  return parts_sum(part, warps);
}

constexpr uint32_t NORM_WARPS = 4;   // warps of a CTA whose warps work on their own
constexpr uint32_t NORM_STAGES = 4;  // ring slots at most
constexpr uint32_t NORM_MAX_SMEM = 226 * 1024;
// The sums of a and b over a warp in one chain: lanes 0 to 15 get a's, the others b's.
VSD float warp_sum2(float a, float b) {
  const bool low = (threadIdx.x & 16u) == 0;
  float v = (low ? a : b) + __shfl_xor_sync(0xffffffffu, low ? b : a, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

}  // namespace vs

// What the forward and the backward take; unused buffers are NULL.
struct NormFwd {
  vs::NormShape s;
  const void *x, *residual;
  uint64_t x_stride, residual_stride;
  vs::Weights w;
  float eps;
  vs::Dropout d;
  void *y, *z;
  float *mean, *rstd;
};
struct NormBwd {
  vs::NormShape s;
  const void *dy, *dz, *z;
  uint64_t dy_stride, dz_stride, z_stride;
  vs::Weights w;
  const float *mean, *rstd;
  vs::Dropout d;
  void *dx, *dresidual;
  int32_t wdtype;
  void *dweight, *dbias;
};

// Of `choices`, the runs of `width` values per lane (on a power of two of lanes) that
// cost a row of `runs` runs the fewest instructions, at about 11 for a value's place,
// used or idle, and 100 for a lane's share of a row; none (k = 0) where a warp cannot
// hold the row.
struct NormFit {
  int k;
  uint32_t cost;
};
inline NormFit norm_fit(uint32_t runs, int width, std::initializer_list<int> choices) {
  NormFit best{0, ~0u};
  for (int k : choices) {
    uint32_t lanes = 1;
    while (lanes * k < runs) lanes *= 2;
    const uint32_t cost = lanes * (uint32_t)(11 * k * width + 100);
    if (lanes <= 32 && cost < best.cost) best = {k, cost};
  }
  return best;
}

// Rows that a thread of the backward adds up one by one, at most (four times as many for
// a tile kernel's lane of more than six values): the error of a chain grows with its
// length, by half a unit a row where the terms are alike (of a mean's gradient, 1055 rows
// 1.6e-5 of the sum, 256 rows 3.8e-6).  Beyond it there are more CTAs than an SM holds at
// once, which add up fewer rows each.
constexpr uint64_t NORM_CHAIN = 256;

// The streaming kernels take contiguous rows on 16-byte aligned buffers: tiles of
// short rows per warp, or a CTA per long row; *taken tells whether the shape is
// one of theirs.
vs_status norm_row_forward(vs_ctx* ctx, int32_t dtype, bool join, const NormFwd& a, bool* taken);
vs_status norm_row_backward(vs_ctx* ctx, int32_t dtype, bool join, const NormBwd& a, bool* taken);
vs_status norm_tile_forward(vs_ctx* ctx, int32_t dtype, bool join, const NormFwd& a, bool* taken);
vs_status norm_tile_backward(vs_ctx* ctx, int32_t dtype, bool join, const NormBwd& a, bool* taken);
// The direct kernels take rows of any stride and alignment, up to a width.
vs_status norm_direct_forward(vs_ctx* ctx, int32_t dtype, bool join, const NormFwd& a, bool* taken);
vs_status norm_direct_backward(vs_ctx* ctx, int32_t dtype, bool join, const NormBwd& a, bool* taken);
// `floats` floats of scratch for one call, 16-byte aligned, on the ctx stream; end
// it after the call's last launch.  The word at `ticket` is zero before the call and
// has to be zero after it.
struct NormScratch {
  float* p = nullptr;
  uint32_t* ticket = nullptr;
  bool pooled = false;
};
vs_status norm_scratch_begin(vs_ctx* ctx, size_t floats, NormScratch* out);
vs_status norm_scratch_end(vs_ctx* ctx, const NormScratch& scratch);
// dw and db from `strips` partial sums [strips][2][cols]
vs_status norm_join_partials(vs_ctx* ctx, uint32_t cols, uint32_t strips, const float* partial, int32_t dtype,
                             void* dweight, void* dbias);
