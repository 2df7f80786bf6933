// Rows of the key-value cache: putting tokens' keys and values into their
// slots (narrowed to e4m3 if the cache is), getting them back, and the join of
// partial attention results that lie on several PEs.
#include "kv_device.hpp"

namespace rocshmem {
namespace kv {

constexpr uint64_t kManyRows = 1 << 15;

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

// A group of kLanes lanes moves one row of kAhead tokens, whose loads are all on
// their way before the first is used.  Work-group (x, y): row x of 2 * kv_heads (all
// keys, then all values) of the tokens from y * groups * kAhead on; the groups take
// neighbouring tokens, so that the scale bytes of tokens in neighbouring slots
// leave in one store.  Bound by the bytes moved: nothing but the row's largest
// magnitude is computed, across its lanes.
template <int kSide, int kCache, int kLanes, int kAhead, bool kPut>
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
  for (uint64_t t0 = static_cast<uint64_t>(blockIdx.y) * kGroups * kAhead + group; t0 < a.n_tokens;
       t0 += static_cast<uint64_t>(gridDim.y) * kGroups * kAhead) {
    int64_t slot[kAhead];
    typename Side::Raw side[kAhead][kRuns<kCache>];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const uint64_t t = t0 + k * kGroups;
      slot[k] = t < a.n_tokens ? a.slots[t] : -1;
      if constexpr (kPut) {  // a row is there whatever its slot
        const char *from = rows + (t < a.n_tokens ? t : t0) * a.side_row[value];
#pragma unroll
        for (int r = 0; r < kRuns<kCache>; ++r) side[k][r] = Side::load(from + 8 * r * Side::kBytes);
      }
    }
    char *page[kAhead];
    uint32_t at[kAhead] = {};
    typename Cached::Raw cached[kAhead][kRuns<kCache>] = {};
    unsigned byte[kAhead] = {};
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      page[k] = page_of_slot(a, slot[k], blockIdx.x == 0 && lane == 0, &at[k]);
      if constexpr (!kPut) {
        if (!page[k]) continue;
        const char *from = page[k] + row_offset(a.cache, head, at[k], value) + element * Cached::kBytes;
#pragma unroll
        for (int r = 0; r < kRuns<kCache>; ++r) cached[k][r] = Cached::load(from + 8 * r * Cached::kBytes);
        if constexpr (kNarrow)
          byte[k] = static_cast<unsigned char>(page[k][scale_offset(a.cache, head, at[k], value)]);
      }
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      float x[kRuns<kCache>][8];
      if constexpr (kPut && kNarrow) {
        unsigned top = 0;  // magnitudes of floats order like their bits
#pragma unroll
        for (int r = 0; r < kRuns<kCache>; ++r) {
          Side::widen(side[k][r], x[r]);
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
        byte[k] = scale_byte(top);
        const float down = two_to(254 - byte[k]);
#pragma unroll
        for (int r = 0; r < kRuns<kCache>; ++r)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            x[r][i] = __builtin_isfinite(x[r][i]) ? x[r][i] * down : __builtin_nanf("");
      }
      if (!page[k] || !mine) continue;
      if constexpr (kPut) {
        char *to = page[k] + row_offset(a.cache, head, at[k], value) + element * Cached::kBytes;
        if constexpr (kSide == kCache) {
          Cached::store(to, side[k][0]);
        } else {
          typename Cached::Raw raw[kRuns<kCache>];
#pragma unroll
          for (int r = 0; r < kRuns<kCache>; ++r) {
            if constexpr (!kNarrow) Side::widen(side[k][r], x[r]);
            raw[r] = Cached::round(x[r]);
          }
          if constexpr (kNarrow) {
            store_loose(to, U4{raw[0][0], raw[0][1], raw[1][0], raw[1][1]});
            if (lane == 0) page[k][scale_offset(a.cache, head, at[k], value)] = static_cast<char>(byte[k]);
          } else {
            Cached::store(to, raw[0]);
          }
        }
      } else {
        char *to = rows + (t0 + k * kGroups) * a.side_row[value];
#pragma unroll
        for (int r = 0; r < kRuns<kCache>; ++r) {
          if constexpr (kSide == kCache) {
            Side::store(to, cached[k][r]);
          } else {
            Cached::widen(cached[k][r], x[r]);
            if constexpr (kNarrow) {
              const float up = two_to(byte[k]);
#pragma unroll
              for (int i = 0; i < 8; ++i) x[r][i] *= up;
            }
            Side::store(to + 8 * r * Side::kBytes, Side::round(x[r]));
          }
        }
      }
    }
  }
}

template <int kSide, int kCache, bool kPut>
static void launch_rows(const RowsArgs &a, hipStream_t s) {
  const auto go = [&](auto lanes, auto ahead) {
    constexpr int kLanes = decltype(lanes)::value, kAhead = decltype(ahead)::value;
    constexpr uint64_t kTokens = 256 / kLanes * kAhead;
    const uint64_t chunks = (a.n_tokens + kTokens - 1) / kTokens;
    const dim3 grid(2 * a.cache.kv_heads, static_cast<unsigned>(chunks < 65535 ? chunks : 65535));
    hipLaunchKernelGGL((rows_kernel<kSide, kCache, kLanes, kAhead, kPut>), grid, dim3(256), 0, s, a);
  };
  constexpr int kMost = kMaxHeadDim / (8 * kRuns<kCache>);
  // Several tokens a group once there are enough of them to fill the GPU that way.
  const auto lanes = [&](auto ahead) {
    if (a.cache.head_dim <= 64)
      go(std::integral_constant<int, kMost / 4>{}, ahead);
    else if (a.cache.head_dim <= 128)
      go(std::integral_constant<int, kMost / 2>{}, ahead);
    else
      go(std::integral_constant<int, kMost>{}, ahead);
  };
  if (a.n_tokens * a.cache.kv_heads >= kManyRows)
    lanes(std::integral_constant<int, 4>{});
  else
    lanes(std::integral_constant<int, 1>{});
  DRV_CHECK_HIP(hipGetLastError());
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
      case ROCSHMEM_AMD_BF16: launch_rows<kSide, ROCSHMEM_AMD_BF16, kPut>(a, s); break;
      case ROCSHMEM_AMD_HALF: launch_rows<kSide, ROCSHMEM_AMD_HALF, kPut>(a, s); break;
      default: launch_rows<kSide, ROCSHMEM_AMD_E4M3, kPut>(a, s); break;
    }
  };
  switch (dtype) {
    case ROCSHMEM_AMD_BF16: for_cache(std::integral_constant<int, ROCSHMEM_AMD_BF16>{}); break;
    case ROCSHMEM_AMD_HALF: for_cache(std::integral_constant<int, ROCSHMEM_AMD_HALF>{}); break;
    default: for_cache(std::integral_constant<int, ROCSHMEM_AMD_FLOAT>{}); break;
  }
  return 0;
}

// ---- the join ---------------------------------------------------------------------
struct JoinArgs {
  const detail::Context *ctx;
  const char *partial;
  const float *partial_lse;
  char *out;
  float *lse;
  uint64_t n_pieces;  // rows * pieces per row
  uint32_t pieces;    // of eight elements, per row
  int first, stride, members;
};

// A lane joins eight elements of a row: two walks over the members, for the
// largest lse and for the sums.
template <int kIn, int kOut>
__global__ __launch_bounds__(256) void join_kernel(JoinArgs a) {
  const uint64_t step = static_cast<uint64_t>(gridDim.x) * 256;
  for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x; i < a.n_pieces; i += step) {
    const uint64_t row = i / a.pieces;
    float top = -INFINITY;
    for (int m = 0; m < a.members; ++m)
      top = fmaxf(top, detail::remote_addr(a.ctx, a.partial_lse, a.first + m * a.stride)[row]);
    const float from = top == -INFINITY ? 0.f : top;
    float total = 0.f, sum[8] = {};
    for (int m = 0; m < a.members; ++m) {
      const int pe = a.first + m * a.stride;
      const float lse = detail::remote_addr(a.ctx, a.partial_lse, pe)[row];
      if (lse == -INFINITY) continue;
      const float w = expf(lse - from);
      float x[8];
      Eight<kIn>::widen(Eight<kIn>::load(detail::remote_addr(a.ctx, a.partial, pe) + i * 8 * Eight<kIn>::kBytes), x);
      total += w;
      for (int e = 0; e < 8; ++e) sum[e] += w * x[e];
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    for (int e = 0; e < 8; ++e) sum[e] *= inv;
    Eight<kOut>::store(a.out + i * 8 * Eight<kOut>::kBytes, Eight<kOut>::round(sum));
    if (a.lse && i == row * a.pieces) a.lse[row] = top + logf(total);
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
  JoinArgs a{};
  a.ctx = reinterpret_cast<const detail::Context *>(runtime::rt().driver_ctx_handle(my_pe).ctx_opaque);
  a.partial = static_cast<const char *>(partial);
  a.partial_lse = partial_lse;
  a.out = static_cast<char *>(out);
  a.lse = lse;
  a.pieces = static_cast<uint32_t>(head_dim / 8);
  a.n_pieces = n_rows * a.pieces;
  a.first = PE_start;
  a.stride = 1 << logPE_stride;
  a.members = PE_size;
  const uint64_t wgs = (a.n_pieces + 255) / 256;
  const dim3 grid(static_cast<unsigned>(wgs < (1u << 20) ? wgs : (1u << 20)));
  hipStream_t s = drv::as_stream(stream);
  const auto to = [&](auto in) {
    constexpr int kIn = decltype(in)::value;
    switch (out_dtype) {
      case ROCSHMEM_AMD_BF16:
        hipLaunchKernelGGL((join_kernel<kIn, ROCSHMEM_AMD_BF16>), grid, dim3(256), 0, s, a);
        break;
      case ROCSHMEM_AMD_HALF:
        hipLaunchKernelGGL((join_kernel<kIn, ROCSHMEM_AMD_HALF>), grid, dim3(256), 0, s, a);
        break;
      default:
        hipLaunchKernelGGL((join_kernel<kIn, ROCSHMEM_AMD_FLOAT>), grid, dim3(256), 0, s, a);
        break;
    }
  };
  switch (dtype) {
    case ROCSHMEM_AMD_BF16: to(std::integral_constant<int, ROCSHMEM_AMD_BF16>{}); break;
    case ROCSHMEM_AMD_HALF: to(std::integral_constant<int, ROCSHMEM_AMD_HALF>{}); break;
    default: to(std::integral_constant<int, ROCSHMEM_AMD_FLOAT>{}); break;
  }
  DRV_CHECK_HIP(hipGetLastError());
  return 0;
}

}  // extern "C"
