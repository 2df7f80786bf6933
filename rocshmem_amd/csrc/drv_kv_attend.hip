// Attention of one new token per sequence over the paged key-value cache.
#include "kv_device.hpp"

namespace rocshmem {
namespace kv {

struct AttendArgs {
  Layout cache;
  const detail::Context *ctx;
  unsigned long long *refused;
  const char *q;
  char *out;
  float *lse;
  const int32_t *page_table;
  const int32_t *lengths;
  uint64_t q_row, out_row;  // elements between sequences
  uint64_t table_row;
  int q_heads, group;       // query heads, and how many share a cache head
  int max_len, window, my_pe;
  bool own_pages;
  float scale, softcap;
};

// The tokens of sequence b that take part: [first, end).
struct Span {
  int first, end;
};
__device__ __forceinline__ Span span_of(const AttendArgs &a, int b, bool counts) {
  const int len = a.lengths[b];
  int end = len < 0 ? 0 : len < a.max_len ? len : a.max_len;
  const uint64_t held = a.table_row * a.cache.page_tokens;
  if (static_cast<uint64_t>(end) > held) end = static_cast<int>(held);
  if (end != len && counts) count_refused(a.refused);
  return Span{a.window > 0 && end > a.window ? end - a.window : 0, end};
}

// One wavefront per sequence and query head.  64 tokens at a time, a lane for
// each: the score, the running maximum and sum over the wavefront; then the
// values token by token with the lanes along the row.
template <int kIn, int kCache, int kOut>
__global__ __launch_bounds__(64) void attend_kernel(AttendArgs a) {
  const int b = blockIdx.y, h = blockIdx.x, lane = threadIdx.x;
  const uint32_t head = static_cast<uint32_t>(h / a.group), d = a.cache.head_dim;
  const Span span = span_of(a, b, h == 0 && lane == 0);
  const char *q = a.q + (b * a.q_row + h * d) * Eight<kIn>::kBytes;
  float top = -INFINITY, total = 0.f, acc[8] = {};
  for (int t0 = span.first; t0 < span.end; t0 += 64) {
    const int t = t0 + lane;
    const char *page = nullptr;
    uint32_t at = 0;
    float s = -INFINITY;
    if (t < span.end) {
      const uint32_t index = quotient(static_cast<uint32_t>(t) >> 4, a.cache.by_page_units);
      at = t - index * a.cache.page_tokens;
      const uint32_t number = static_cast<uint32_t>(a.page_table[b * a.table_row + index]);
      if (number >= a.cache.n_pages) {
        if (h == 0 && (at == 0 || t == span.first)) count_refused(a.refused);
      } else {
        const uint32_t pe = owner_of(a.cache, number);
        if (!a.own_pages || static_cast<int>(pe) == a.my_pe)
          page = detail::remote_addr(a.ctx, a.cache.pages, static_cast<int>(pe)) +
                 page_offset(a.cache, number, pe);
      }
    }
    if (page) {
      const char *k = page + row_offset(a.cache, head, at, false);
      float dot = 0.f;
      for (uint32_t e = 0; e < d; e += 8) {
        float x[8], y[8];
        Eight<kIn>::widen(Eight<kIn>::load(q + e * Eight<kIn>::kBytes), x);
        Eight<kCache>::widen(Eight<kCache>::load(k + e * Eight<kCache>::kBytes), y);
        for (int i = 0; i < 8; ++i) dot += x[i] * y[i];
      }
      if (kCache == ROCSHMEM_AMD_E4M3)
        dot *= two_to(static_cast<unsigned char>(page[scale_offset(a.cache, head, at, false)]));
      s = dot * a.scale;
      if (a.softcap > 0.f) s = a.softcap * tanhf(s / a.softcap);
    }
    float tile_top = s;
    for (int hop = 32; hop; hop /= 2) tile_top = fmaxf(tile_top, __shfl_xor(tile_top, hop));
    const float next = fmaxf(top, tile_top), from = next == -INFINITY ? 0.f : next;
    const float p = expf(s - from), keep = expf(top - from);
    float sum = p;
    for (int hop = 32; hop; hop /= 2) sum += __shfl_xor(sum, hop);
    total = total * keep + sum;
    for (int i = 0; i < 8; ++i) acc[i] *= keep;
    top = next;
    const int n = span.end - t0 < 64 ? span.end - t0 : 64;
    for (int j = 0; j < n; ++j) {
      const char *from_page = reinterpret_cast<const char *>(
          __shfl(static_cast<unsigned long long>(reinterpret_cast<uintptr_t>(page)), j));
      const uint32_t from_at = __shfl(at, j);
      float w = __shfl(p, j);
      if (!from_page || lane * 8u >= d) continue;
      float y[8];
      Eight<kCache>::widen(
          Eight<kCache>::load(from_page + row_offset(a.cache, head, from_at, true) + lane * 8 * Eight<kCache>::kBytes), y);
      if (kCache == ROCSHMEM_AMD_E4M3)
        w *= two_to(static_cast<unsigned char>(from_page[scale_offset(a.cache, head, from_at, true)]));
      for (int i = 0; i < 8; ++i) acc[i] += w * y[i];
    }
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  for (int i = 0; i < 8; ++i) acc[i] *= inv;
  if (lane * 8u < d)
    Eight<kOut>::store(a.out + (b * a.out_row + h * d + lane * 8) * Eight<kOut>::kBytes, Eight<kOut>::round(acc));
  if (a.lse && lane == 0) a.lse[static_cast<uint64_t>(b) * a.q_heads + h] = top + logf(total);
}

template <int kIn, int kCache, int kOut>
static void launch_attend(const AttendArgs &a, int n_seqs, hipStream_t s) {
  hipLaunchKernelGGL((attend_kernel<kIn, kCache, kOut>), dim3(a.q_heads, n_seqs), dim3(64), 0, s, a);
  DRV_CHECK_HIP(hipGetLastError());
}

}  // namespace kv
}  // namespace rocshmem

using namespace rocshmem;
using namespace rocshmem::kv;

extern "C" {

size_t rocshmem_amd_kv_attend_bytes(const rocshmem_amd_kv_cache_t *, int, int, int) { return 0; }

int rocshmem_amd_kv_attend(const rocshmem_amd_kv_cache_t *cache, int dtype, const void *q, size_t q_row,
                           int q_heads, int out_dtype, void *out, size_t out_row, float *lse,
                           const int32_t *page_table, size_t table_row, const int32_t *lengths,
                           int n_seqs, int max_len, int window, float scale, float softcap,
                           int pages_from, void *workspace, size_t workspace_bytes, int my_pe,
                           rocshmem_amd_stream_t stream) {
  AttendArgs a{};
  if (!take_cache(cache, my_pe, &a.cache)) return -1;
  if (dtype != ROCSHMEM_AMD_BF16 && dtype != ROCSHMEM_AMD_HALF) return -1;
  if (cache->dtype != ROCSHMEM_AMD_E4M3 && cache->dtype != dtype) return -1;
  if (out_dtype != dtype && out_dtype != ROCSHMEM_AMD_FLOAT) return -1;
  if (pages_from != ROCSHMEM_AMD_KV_ALL_PAGES && pages_from != ROCSHMEM_AMD_KV_OWN_PAGES) return -1;
  if (n_seqs < 0 || n_seqs > 65535 || max_len < 0 || window < 0) return -1;
  if (q_heads < 1 || q_heads % cache->kv_heads || q_heads > 65535) return -1;
  if (!__builtin_isfinite(scale) || !__builtin_isfinite(softcap) || softcap < 0.f) return -1;
  if (!n_seqs) return 0;
  const size_t row = static_cast<size_t>(q_heads) * a.cache.head_dim;
  const size_t es = element_bytes(dtype), out_es = element_bytes(out_dtype);
  if (n_seqs > 1 && out_row < row) return -1;
  size_t q_bytes, out_bytes, table_bytes;
  if (!extent(n_seqs, q_row, row, es, &q_bytes) || !extent(n_seqs, out_row, row, out_es, &out_bytes) ||
      !extent(n_seqs, table_row, table_row, 4, &table_bytes))
    return -1;
  if (!q || !aligned_to(q, es) || !drv::local_ok(q, q_bytes)) return -1;
  if (!out || !aligned_to(out, out_es) || !drv::local_ok(out, out_bytes)) return -1;
  if (!aligned_to(lse, 4) || (lse && !drv::local_ok(lse, 4 * static_cast<size_t>(n_seqs) * q_heads))) return -1;
  if (!lengths || !aligned_to(lengths, 4) || !drv::local_ok(lengths, 4 * static_cast<size_t>(n_seqs))) return -1;
  if (!aligned_to(page_table, 4) || !drv::local_ok(page_table, table_bytes)) return -1;
  if (table_row > static_cast<size_t>(INT32_MAX)) return -1;
  (void)workspace;
  (void)workspace_bytes;
  a.ctx = reinterpret_cast<const detail::Context *>(runtime::rt().driver_ctx_handle(my_pe).ctx_opaque);
  a.refused = runtime::rt().d_kv_refused;
  a.q = static_cast<const char *>(q);
  a.out = static_cast<char *>(out);
  a.lse = lse;
  a.page_table = page_table;
  a.lengths = lengths;
  a.q_row = q_row;
  a.out_row = out_row;
  a.table_row = table_row;
  a.q_heads = q_heads;
  a.group = q_heads / cache->kv_heads;
  a.max_len = max_len;
  a.window = window;
  a.my_pe = my_pe;
  a.own_pages = pages_from == ROCSHMEM_AMD_KV_OWN_PAGES;
  a.scale = scale;
  a.softcap = softcap;
  hipStream_t s = drv::as_stream(stream);
  const auto to = [&](auto in) {
    constexpr int kIn = decltype(in)::value;
    const bool narrow = cache->dtype == ROCSHMEM_AMD_E4M3, wide = out_dtype == ROCSHMEM_AMD_FLOAT;
    if (narrow && wide) launch_attend<kIn, ROCSHMEM_AMD_E4M3, ROCSHMEM_AMD_FLOAT>(a, n_seqs, s);
    if (narrow && !wide) launch_attend<kIn, ROCSHMEM_AMD_E4M3, kIn>(a, n_seqs, s);
    if (!narrow && wide) launch_attend<kIn, kIn, ROCSHMEM_AMD_FLOAT>(a, n_seqs, s);
    if (!narrow && !wide) launch_attend<kIn, kIn, kIn>(a, n_seqs, s);
  };
  if (dtype == ROCSHMEM_AMD_BF16)
    to(std::integral_constant<int, ROCSHMEM_AMD_BF16>{});
  else
    to(std::integral_constant<int, ROCSHMEM_AMD_HALF>{});
  return 0;
}

}  // extern "C"
