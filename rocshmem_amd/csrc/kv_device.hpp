// What the key-value cache's kernels share: eight elements of a row at a time
// in the cache's formats, and the checks of the entry points.
#ifndef ROCSHMEM_AMD_KV_DEVICE_HPP_
#define ROCSHMEM_AMD_KV_DEVICE_HPP_

#include "drv_common.hpp"
#include "kv_cache.hpp"

namespace rocshmem {
namespace kv {

typedef unsigned U2 __attribute__((ext_vector_type(2)));
typedef unsigned U4 __attribute__((ext_vector_type(4)));
typedef float F2 __attribute__((ext_vector_type(2)));
typedef float F4 __attribute__((ext_vector_type(4)));
typedef __bf16 B8 __attribute__((ext_vector_type(8)));
typedef _Float16 H8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

// A vector at any address its elements allow: gfx950's global loads and stores
// need no more, and the compiler must not assume more.
template <typename V>
struct __attribute__((packed)) Loose {
  V v;
};
template <typename V>
__device__ __forceinline__ V load_loose(const char *p) {
  return reinterpret_cast<const Loose<V> *>(p)->v;
}
template <typename V>
__device__ __forceinline__ void store_loose(char *p, V v) {
  reinterpret_cast<Loose<V> *>(p)->v = v;
}

// Eight consecutive elements of a format, as they lie in memory (Raw) and as
// 32-bit values; rounding is to nearest even.  E4M3 holds codes: the row's
// scale is the caller's business.
template <int kType>
struct Eight;
template <>
struct Eight<ROCSHMEM_AMD_FLOAT> {
  static constexpr int kBytes = 4;
  struct Raw {
    F4 lo, hi;
  };
  __device__ __forceinline__ static Raw load(const char *p) {
    return Raw{load_loose<F4>(p), load_loose<F4>(p + 16)};
  }
  __device__ __forceinline__ static void widen(const Raw &r, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = r.lo[i];
      x[4 + i] = r.hi[i];
    }
  }
  __device__ __forceinline__ static Raw round(const float (&x)[8]) {
    return Raw{F4{x[0], x[1], x[2], x[3]}, F4{x[4], x[5], x[6], x[7]}};
  }
  __device__ __forceinline__ static void store(char *p, const Raw &r) {
    store_loose(p, r.lo);
    store_loose(p + 16, r.hi);
  }
};
template <typename T, typename T8>
struct EightOf16Bits {
  static constexpr int kBytes = 2;
  using Raw = T8;
  __device__ __forceinline__ static Raw load(const char *p) { return load_loose<T8>(p); }
  __device__ __forceinline__ static void widen(const Raw &r, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(r[i]);
  }
  __device__ __forceinline__ static Raw round(const float (&x)[8]) {
    Raw r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = static_cast<T>(x[i]);
    return r;
  }
  __device__ __forceinline__ static void store(char *p, const Raw &r) { store_loose(p, r); }
};
template <>
struct Eight<ROCSHMEM_AMD_BF16> : EightOf16Bits<__bf16, B8> {};
template <>
struct Eight<ROCSHMEM_AMD_HALF> : EightOf16Bits<_Float16, H8> {};
template <>
struct Eight<ROCSHMEM_AMD_E4M3> {
  static constexpr int kBytes = 1;
  using Raw = U2;
  __device__ __forceinline__ static Raw load(const char *p) { return load_loose<U2>(p); }
  __device__ __forceinline__ static void widen(const Raw &r, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const F2 a = __builtin_amdgcn_cvt_pk_f32_fp8(r[i], false);
      const F2 b = __builtin_amdgcn_cvt_pk_f32_fp8(r[i], true);
      x[4 * i] = a.x;
      x[4 * i + 1] = a.y;
      x[4 * i + 2] = b.x;
      x[4 * i + 3] = b.y;
    }
  }
  __device__ __forceinline__ static Raw round(const float (&x)[8]) {
    Raw r;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
      r[i] = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], w, true);
    }
    return r;
  }
  __device__ __forceinline__ static void store(char *p, const Raw &r) { store_loose(p, r); }
};

// 2^(b - 127) of a scale byte (1..254) as a 32-bit float, and of its negation.
__device__ __forceinline__ float two_to(unsigned byte) { return __uint_as_float(byte << 23); }
// The scale byte of a row whose largest finite magnitude has the bits `top`:
// 448 = 1.75 * 2^8, so a row's exponent less 8 is enough unless its mantissa is
// above 1.75; no less than 2^-126, the smallest scale that is a normal number.
__device__ __forceinline__ unsigned scale_byte(unsigned top) {
  const int b = static_cast<int>(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u);
  return b < 1 ? 1u : static_cast<unsigned>(b);
}

__device__ __forceinline__ void count_refused(unsigned long long *refused, unsigned long long n = 1) {
  __hip_atomic_fetch_add(refused, n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ---- launches and checks of the entry points -------------------------------------------------

// A launch's own status decides: an error that an earlier call of the program has
// left behind for hipGetLastError is not this call's, and stays there.
template <typename Args>
inline bool launch(void (*kernel)(Args), dim3 grid, int lanes, hipStream_t s, const Args &a) {
  void *args[] = {const_cast<Args *>(&a)};
  if (hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, dim3(lanes), args, 0, s) == hipSuccess)
    return true;
  (void)hipGetLastError();
  return false;
}

// The calls launch on the current device, which must be the one the heap is on.
inline bool on_heap_device() {
  int dev = -1;
  return hipGetDevice(&dev) == hipSuccess && dev == runtime::rt().device;
}
inline bool aligned_to(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// n rows of row_elems elements, `stride` elements apart, of es bytes each: false if
// their extent does not fit in 63 bits.
inline bool extent(size_t n, size_t stride, size_t row_elems, size_t es, size_t *bytes) {
  size_t last = 0;
  if (n && __builtin_mul_overflow(n - 1, stride, &last)) return false;
  if (__builtin_add_overflow(last, row_elems, &last) || __builtin_mul_overflow(last, es, &last)) return false;
  *bytes = n ? last : 0;
  return *bytes <= static_cast<size_t>(INT64_MAX);
}

inline bool overlap(const void *a, size_t a_bytes, const void *b, size_t b_bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return a_bytes && b_bytes && x < y + b_bytes && y < x + a_bytes;
}

// The cache a call works on, as its kernels see it.
inline bool take_cache(const rocshmem_amd_kv_cache_t *cache, int my_pe, Layout *out) {
  if (!cache || !drv::valid_actor(my_pe) || !on_heap_device()) return false;
  if (!fill_layout(cache->dtype, cache->page_tokens, cache->kv_heads, cache->head_dim, cache->pages_per_pe,
                   runtime::rt().npes, out))
    return false;
  if (!aligned_to(cache->pages, 16)) return false;
  if (!drv::sym_ok_on(cache->pages, out->page_bytes * out->pages_per_pe, my_pe)) return false;
  out->pages = static_cast<char *>(cache->pages);
  return true;
}

}  // namespace kv
}  // namespace rocshmem

#endif  // ROCSHMEM_AMD_KV_DEVICE_HPP_
