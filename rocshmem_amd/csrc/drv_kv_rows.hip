// Rows of the key-value cache: putting tokens' keys and values into their
// slots (narrowed to e4m3 if the cache is), getting them back, and the join of
// partial attention results that lie on several PEs.
#include "kv_device.hpp"

namespace rocshmem {
namespace kv {

struct RowsArgs {
  Layout cache;
  const detail::Context *ctx;
  unsigned long long *refused;
  char *side[2];         // the caller's keys and values
  uint64_t side_row[2];  // bytes between tokens
  const int64_t *slots;
  uint64_t n_tokens;
};

// The page of a token's slot, as this PE sees it, and the token's place in it.
// Null for a slot that is left out.
__device__ __forceinline__ char *page_of_slot(const RowsArgs &a, int64_t slot, bool counts, uint32_t *at) {
  if (!slot_in_range(a.cache, slot)) {
    if (slot != -1 && counts) count_refused(a.refused);
    return nullptr;
  }
  const Place place = place_of(a.cache, slot);
  const uint32_t pe = owner_of(a.cache, place.page);
  *at = place.at;
  return detail::remote_addr(a.ctx, a.cache.pages, static_cast<int>(pe)) + page_offset(a.cache, place.page, pe);
}

// A lane's share of a row: 16 bytes of the cache, eight elements of 16 bits or
// sixteen of e4m3, as runs of eight.
template <int kCache>
constexpr int kRuns = kCache == ROCSHMEM_AMD_E4M3 ? 2 : 1;

// A group of kLanes lanes moves one row of one token.  Work-group (x, y): row x of
// 2 * kv_heads (all keys, then all values) of 256 / kLanes neighbouring tokens, so that
// the scale bytes of tokens in neighbouring slots leave in one store.  Bound by the
// bytes moved: nothing but the row's largest magnitude is computed, across its
// lanes.  65536 tokens of 8 heads x 128, 16-bit rows to and from e4m3: put 83 us into
// pages filled in order, 96 us into scattered slots (4.9 and 4.2 TB/s) from rows 12 KiB
// apart, 80 and 94 us from rows that follow each other; get 80 and 97 us.  So it is the
// slots that matter: a token's 128-byte pieces of 16 rows lie a page's run of rows apart
// either way, but in order neighbouring tokens' lie together.  20011 tokens into a bf16
// cache 32.6 and 34.2 us (5.0 and 4.8 TB/s).  Two, four or eight tokens a group, all loads
// ahead, took 3 to 12 % longer, and whole tokens a work-group instead of one head the same time.
template <int kSide, int kCache, int kLanes, bool kPut>
__global__ __launch_bounds__(256) void rows_kernel(RowsArgs a) {
  constexpr int kGroups = 256 / kLanes, kEach = 8 * kRuns<kCache>;
  constexpr bool kNarrow = kCache == ROCSHMEM_AMD_E4M3;
  using Side = Eight<kSide>;
  using Cached = Eight<kCache>;
  const bool value = blockIdx.x >= a.cache.kv_heads;
  const uint32_t head = value ? blockIdx.x - a.cache.kv_heads : blockIdx.x;
  const uint32_t lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const bool mine = lane * kEach < a.cache.head_dim;
  const uint32_t element = mine ? lane * kEach : 0;
  char *const rows = a.side[value] + (head * a.cache.head_dim + element) * Side::kBytes;
  for (uint64_t t = static_cast<uint64_t>(blockIdx.y) * kGroups + group; t < a.n_tokens;
       t += static_cast<uint64_t>(gridDim.y) * kGroups) {
    const int64_t slot = a.slots[t];
    char *const row = rows + t * a.side_row[value];
    typename Side::Raw side[kRuns<kCache>];
    if constexpr (kPut) {  // the row is there whatever its slot
#pragma unroll
      for (int r = 0; r < kRuns<kCache>; ++r) side[r] = Side::load(row + 8 * r * Side::kBytes);
    }
    uint32_t at = 0;
    char *const page = page_of_slot(a, slot, blockIdx.x == 0 && lane == 0, &at);
    if (!page) continue;  // the whole group: its lanes agree
    char *const cached = page + row_offset(a.cache, head, at, value) + element * Cached::kBytes;
    char *const scale = page + scale_offset(a.cache, head, at, value);
    float x[kRuns<kCache>][8];
    if constexpr (kPut && kSide == kCache) {
      if (mine) Cached::store(cached, side[0]);
    } else if constexpr (kPut && !kNarrow) {
      Side::widen(side[0], x[0]);
      if (mine) Cached::store(cached, Cached::round(x[0]));
    } else if constexpr (kPut) {
      unsigned top = 0;  // magnitudes of floats order like their bits
#pragma unroll
      for (int r = 0; r < kRuns<kCache>; ++r) {
        Side::widen(side[r], x[r]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const unsigned bits = __float_as_uint(x[r][i]) & 0x7fffffffu;
          top = bits < 0x7f800000u && bits > top ? bits : top;
        }
      }
#pragma unroll
      for (int hop = kLanes / 2; hop; hop /= 2) {
        const unsigned other = __shfl_xor(top, hop, kLanes);
        top = other > top ? other : top;
      }
      const unsigned byte = scale_byte(top);
      const float down = two_to(254 - byte);
      U4 codes;
#pragma unroll
      for (int r = 0; r < kRuns<kCache>; ++r) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          x[r][i] = __builtin_isfinite(x[r][i]) ? x[r][i] * down : __builtin_nanf("");
        const U2 raw = Cached::round(x[r]);
        codes[2 * r] = raw[0];
        codes[2 * r + 1] = raw[1];
      }
      if (mine) store_loose(cached, codes);
      if (lane == 0) *scale = static_cast<char>(byte);
    } else if (mine) {
      typename Cached::Raw raw[kRuns<kCache>];
#pragma unroll
      for (int r = 0; r < kRuns<kCache>; ++r) raw[r] = Cached::load(cached + 8 * r * Cached::kBytes);
      if constexpr (kSide == kCache) {
        Side::store(row, raw[0]);
      } else {
        const float up = kNarrow ? two_to(static_cast<unsigned char>(*scale)) : 1.f;
#pragma unroll
        for (int r = 0; r < kRuns<kCache>; ++r) {
          Cached::widen(raw[r], x[r]);
          if constexpr (kNarrow) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[r][i] *= up;
          }
          Side::store(row + 8 * r * Side::kBytes, Side::round(x[r]));
        }
      }
    }
  }
}

template <int kSide, int kCache, bool kPut>
static bool launch_rows(const RowsArgs &a, hipStream_t s) {
  const auto go = [&](auto lanes) {
    constexpr int kLanes = decltype(lanes)::value;
    const uint64_t chunks = (a.n_tokens + 256 / kLanes - 1) / (256 / kLanes);
    const dim3 grid(2 * a.cache.kv_heads, static_cast<unsigned>(chunks < 65535 ? chunks : 65535));
    return launch(rows_kernel<kSide, kCache, kLanes, kPut>, grid, 256, s, a);
  };
  constexpr int kMost = kMaxHeadDim / (8 * kRuns<kCache>);
  if (a.cache.head_dim <= 64) return go(std::integral_constant<int, kMost / 4>{});
  if (a.cache.head_dim <= 128) return go(std::integral_constant<int, kMost / 2>{});
  return go(std::integral_constant<int, kMost>{});
}

template <bool kPut>
static int move_rows(const rocshmem_amd_kv_cache_t *cache, int dtype, char *k, size_t k_row, char *v,
                     size_t v_row, const int64_t *slots, size_t n_tokens, int my_pe, void *stream) {
  RowsArgs a{};
  if (!take_cache(cache, my_pe, &a.cache)) return -1;
  const size_t es = element_bytes(dtype), row = static_cast<size_t>(a.cache.kv_heads) * a.cache.head_dim;
  if (es < 2) return -1;
  if (!n_tokens) return 0;
  if (!slots || !k || !v || !aligned_to(k, es) || !aligned_to(v, es) || !aligned_to(slots, 8)) return -1;
  if (!kPut && n_tokens > 1 && (k_row < row || v_row < row)) return -1;
  size_t bytes[2], slot_bytes;
  if (!extent(n_tokens, k_row, row, es, &bytes[0]) || !extent(n_tokens, v_row, row, es, &bytes[1]) ||
      !extent(n_tokens, 1, 1, 8, &slot_bytes))
    return -1;
  if (!drv::local_ok(k, bytes[0]) || !drv::local_ok(v, bytes[1]) || !drv::local_ok(slots, slot_bytes)) return -1;
  a.ctx = reinterpret_cast<const detail::Context *>(runtime::rt().driver_ctx_handle(my_pe).ctx_opaque);
  a.refused = runtime::rt().d_kv_refused;
  a.side[0] = k;
  a.side[1] = v;
  a.side_row[0] = k_row * es;
  a.side_row[1] = v_row * es;
  a.slots = slots;
  a.n_tokens = n_tokens;
  hipStream_t s = drv::as_stream(stream);
  const auto for_cache = [&](auto side) {
    constexpr int kSide = decltype(side)::value;
    switch (cache->dtype) {
      case ROCSHMEM_AMD_BF16: return launch_rows<kSide, ROCSHMEM_AMD_BF16, kPut>(a, s);
      case ROCSHMEM_AMD_HALF: return launch_rows<kSide, ROCSHMEM_AMD_HALF, kPut>(a, s);
      default: return launch_rows<kSide, ROCSHMEM_AMD_E4M3, kPut>(a, s);
    }
  };
  bool done;
  switch (dtype) {
    case ROCSHMEM_AMD_BF16: done = for_cache(std::integral_constant<int, ROCSHMEM_AMD_BF16>{}); break;
    case ROCSHMEM_AMD_HALF: done = for_cache(std::integral_constant<int, ROCSHMEM_AMD_HALF>{}); break;
    default: done = for_cache(std::integral_constant<int, ROCSHMEM_AMD_FLOAT>{}); break;
  }
  return done ? 0 : -1;
}

// ---- the join ---------------------------------------------------------------------
struct JoinArgs {
  const detail::Context *ctx;
  const char *partial;
  const float *partial_lse;
  char *out;
  float *lse;
  uint64_t n_pieces;  // 16 bytes of the partial results each
  uint32_t pieces;    // per row
  Divisor by_pieces;
  int first, stride, members;
};

// 16 bytes of a type as 32-bit values, and as many values of another type stored.
template <int kType>
struct Piece {
  static constexpr int kEach = 8;
  __device__ __forceinline__ static void load(const char *p, float (&x)[8]) {
    Eight<kType>::widen(__builtin_nontemporal_load(reinterpret_cast<const typename Eight<kType>::Raw *>(p)), x);
  }
};
template <>
struct Piece<ROCSHMEM_AMD_FLOAT> {
  static constexpr int kEach = 4;
  __device__ __forceinline__ static void load(const char *p, float (&x)[4]) {
    const F4 v = __builtin_nontemporal_load(reinterpret_cast<const F4 *>(p));
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = v[i];
  }
};
template <int kType>
__device__ __forceinline__ void store_values(char *p, const float (&x)[8]) {
  Eight<kType>::store(p, Eight<kType>::round(x));
}
template <int kType>
__device__ __forceinline__ void store_values(char *p, const float (&x)[4]) {
  typedef __bf16 B4 __attribute__((ext_vector_type(4)));
  typedef _Float16 H4 __attribute__((ext_vector_type(4)));
  if constexpr (kType == ROCSHMEM_AMD_FLOAT)
    store_loose(p, F4{x[0], x[1], x[2], x[3]});
  else if constexpr (kType == ROCSHMEM_AMD_BF16)
    store_loose(p, B4{static_cast<__bf16>(x[0]), static_cast<__bf16>(x[1]), static_cast<__bf16>(x[2]),
                      static_cast<__bf16>(x[3])});
  else
    store_loose(p, H4{static_cast<_Float16>(x[0]), static_cast<_Float16>(x[1]), static_cast<_Float16>(x[2]),
                      static_cast<_Float16>(x[3])});
}

// A lane joins 16 bytes of a row.  kAtOnce members' pieces and lse's are on their
// way together; with more members the largest lse is followed from one such batch
// to the next.  Bound by the bytes read: 65536 rows of 128 fp32 from 8 PEs to bf16 in
// 49.7 us, 5.8 TB/s; with work-groups of 256 lanes 51.9, through the caches 54.2, with
// 2048 work-groups that loop 56.0.
template <int kIn, int kOut, int kAtOnce>
__global__ __launch_bounds__(64) void join_kernel(JoinArgs a) {
  constexpr int kEach = Piece<kIn>::kEach;
  const uint64_t step = static_cast<uint64_t>(gridDim.x) * 64;
  for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * 64 + threadIdx.x; i < a.n_pieces; i += step) {
    const uint64_t row = i >> 31 ? i / a.pieces : quotient(static_cast<uint32_t>(i), a.by_pieces);
    float top = -INFINITY, total = 0.f, sum[kEach] = {};
    for (int m0 = 0; m0 < a.members; m0 += kAtOnce) {
      float lse[kAtOnce], x[kAtOnce][kEach];
#pragma unroll
      for (int m = 0; m < kAtOnce; ++m) {
        const int pe = a.first + (m0 + m < a.members ? m0 + m : 0) * a.stride;
        lse[m] = detail::remote_addr(a.ctx, a.partial_lse, pe)[row];
        Piece<kIn>::load(detail::remote_addr(a.ctx, a.partial, pe) + i * 16, x[m]);
      }
      float next = top;
#pragma unroll
      for (int m = 0; m < kAtOnce; ++m) {
        if (m0 + m >= a.members) lse[m] = -INFINITY;
        next = fmaxf(next, lse[m]);
      }
      const float from = next == -INFINITY ? 0.f : next;
      if (m0) {
        const float keep = __builtin_amdgcn_exp2f((top - from) * kLog2e);
        total *= keep;
#pragma unroll
        for (int e = 0; e < kEach; ++e) sum[e] *= keep;
      }
      top = next;
#pragma unroll
      for (int m = 0; m < kAtOnce; ++m) {
        // exactly 0 without tokens, whatever the member's row holds then
        const float w = __builtin_amdgcn_exp2f((lse[m] - from) * kLog2e);
        total += w;
#pragma unroll
        for (int e = 0; e < kEach; ++e) sum[e] += lse[m] == -INFINITY ? 0.f : w * x[m][e];
      }
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
    for (int e = 0; e < kEach; ++e) sum[e] *= inv;
    store_values<kOut>(a.out + i * kEach * Eight<kOut>::kBytes, sum);
    if (a.lse && i == row * a.pieces) a.lse[row] = top + __builtin_amdgcn_logf(total) * kLn2;
  }
}

}  // namespace kv
}  // namespace rocshmem

using namespace rocshmem;
using namespace rocshmem::kv;

extern "C" {

size_t rocshmem_amd_kv_page_bytes(int dtype, int page_tokens, int kv_heads, int head_dim) {
  Layout c;
  return fill_layout(dtype, page_tokens, kv_heads, head_dim, 1, 1, &c) ? c.page_bytes : 0;
}

int rocshmem_amd_kv_row(const rocshmem_amd_kv_cache_t *cache, int npes, int64_t slot, int head, int value,
                        int *pe_out, uint64_t *offset_out, uint64_t *scale_offset_out) {
  Layout c;
  if (!cache || !pe_out || !offset_out || !scale_offset_out) return -1;
  if (!fill_layout(cache->dtype, cache->page_tokens, cache->kv_heads, cache->head_dim, cache->pages_per_pe,
                   npes, &c))
    return -1;
  if (!slot_in_range(c, slot) || head < 0 || head >= cache->kv_heads) return -1;
  const Place at = place_of(c, slot);
  const uint32_t pe = owner_of(c, at.page);
  const uint64_t page = page_offset(c, at.page, pe);
  *pe_out = static_cast<int>(pe);
  *offset_out = page + row_offset(c, static_cast<uint32_t>(head), at.at, value != 0);
  *scale_offset_out = cache->dtype == ROCSHMEM_AMD_E4M3
                          ? page + scale_offset(c, static_cast<uint32_t>(head), at.at, value != 0)
                          : *offset_out;
  return 0;
}

int rocshmem_amd_kv_put(const rocshmem_amd_kv_cache_t *cache, int dtype, const void *k, size_t k_row,
                        const void *v, size_t v_row, const int64_t *slots, size_t n_tokens, int my_pe,
                        rocshmem_amd_stream_t stream) {
  return move_rows<true>(cache, dtype, static_cast<char *>(const_cast<void *>(k)), k_row,
                         static_cast<char *>(const_cast<void *>(v)), v_row, slots, n_tokens, my_pe, stream);
}

int rocshmem_amd_kv_get(const rocshmem_amd_kv_cache_t *cache, int dtype, void *k, size_t k_row, void *v,
                        size_t v_row, const int64_t *slots, size_t n_tokens, int my_pe,
                        rocshmem_amd_stream_t stream) {
  return move_rows<false>(cache, dtype, static_cast<char *>(k), k_row, static_cast<char *>(v), v_row, slots,
                          n_tokens, my_pe, stream);
}

int rocshmem_amd_kv_join(int dtype, const void *partial, const float *partial_lse, size_t n_rows,
                         int head_dim, int out_dtype, void *out, float *lse, int PE_start,
                         int logPE_stride, int PE_size, int my_pe, rocshmem_amd_stream_t stream) {
  if (!drv::valid_actor(my_pe) || !on_heap_device()) return -1;
  const size_t es = element_bytes(dtype), out_es = element_bytes(out_dtype);
  if (es < 2 || out_es < 2 || head_dim < 8 || head_dim % 8) return -1;
  if (logPE_stride < 0 || logPE_stride > 30 || PE_size < 1 || !drv::valid_pe(PE_start)) return -1;
  const int64_t last = PE_start + (static_cast<int64_t>(PE_size - 1) << logPE_stride);
  if (last >= runtime::rt().npes) return -1;
  if (!n_rows) return 0;
  size_t bytes, out_bytes, lse_bytes;
  const size_t d = static_cast<size_t>(head_dim);
  if (!extent(n_rows, d, d, es, &bytes) || !extent(n_rows, d, d, out_es, &out_bytes) ||
      !extent(n_rows, 1, 1, 4, &lse_bytes))
    return -1;
  if (!aligned_to(partial, 16) || !aligned_to(partial_lse, 4) || !drv::sym_ok_on(partial, bytes, my_pe) ||
      !drv::sym_ok_on(partial_lse, lse_bytes, my_pe))
    return -1;
  if (!out || !aligned_to(out, out_es) || !drv::local_ok(out, out_bytes)) return -1;
  if (!aligned_to(lse, 4) || (lse && !drv::local_ok(lse, lse_bytes))) return -1;
  // Nothing that is still to be read may be written over.
  if (overlap(out, out_bytes, partial, bytes) || overlap(out, out_bytes, partial_lse, lse_bytes) ||
      overlap(lse, lse ? lse_bytes : 0, partial, bytes) || overlap(lse, lse ? lse_bytes : 0, partial_lse, lse_bytes))
    return -1;
  JoinArgs a{};
  a.ctx = reinterpret_cast<const detail::Context *>(runtime::rt().driver_ctx_handle(my_pe).ctx_opaque);
  a.partial = static_cast<const char *>(partial);
  a.partial_lse = partial_lse;
  a.out = static_cast<char *>(out);
  a.lse = lse;
  a.pieces = static_cast<uint32_t>(d * es / 16);
  a.by_pieces = make_divisor(a.pieces);
  a.n_pieces = n_rows * a.pieces;
  a.first = PE_start;
  a.stride = 1 << logPE_stride;
  a.members = PE_size;
  const uint64_t wgs = (a.n_pieces + 63) / 64;
  const dim3 grid(static_cast<unsigned>(wgs < (1u << 24) ? wgs : (1u << 24)));
  hipStream_t s = drv::as_stream(stream);
  const auto go = [&](auto in, auto to) {
    constexpr int kIn = decltype(in)::value, kOut = decltype(to)::value;
    if (PE_size <= 2) return launch(join_kernel<kIn, kOut, 2>, grid, 64, s, a);
    if (PE_size <= 4) return launch(join_kernel<kIn, kOut, 4>, grid, 64, s, a);
    return launch(join_kernel<kIn, kOut, 8>, grid, 64, s, a);
  };
  const auto to = [&](auto in) {
    switch (out_dtype) {
      case ROCSHMEM_AMD_BF16: return go(in, std::integral_constant<int, ROCSHMEM_AMD_BF16>{});
      case ROCSHMEM_AMD_HALF: return go(in, std::integral_constant<int, ROCSHMEM_AMD_HALF>{});
      default: return go(in, std::integral_constant<int, ROCSHMEM_AMD_FLOAT>{});
    }
  };
  bool done;
  switch (dtype) {
    case ROCSHMEM_AMD_BF16: done = to(std::integral_constant<int, ROCSHMEM_AMD_BF16>{}); break;
    case ROCSHMEM_AMD_HALF: done = to(std::integral_constant<int, ROCSHMEM_AMD_HALF>{}); break;
    default: done = to(std::integral_constant<int, ROCSHMEM_AMD_FLOAT>{}); break;
  }
  return done ? 0 : -1;
}

}  // extern "C"
