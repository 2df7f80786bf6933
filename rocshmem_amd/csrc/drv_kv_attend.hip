// Attention of one new token per sequence over the paged key-value cache.
#include "kv_attend.hpp"

namespace rocshmem {
namespace kv {

constexpr int kMostTokens = 1 << 25;  // of a sequence

// Joins a sequence's splits: out = sum_i 2^(t_i - t) o_i / sum_i 2^(t_i - t) l_i over the
// splits that have tokens, t the largest t_i.  One work-group per sequence and
// query head: kLanes lanes along the row, four elements each, and the splits dealt
// out to the kThreads / kLanes groups, four of a group's on their way at once.  Each
// group keeps its own largest t_i as it goes, and the first four are asked for
// before the length, which only says how many of them count.  A chain of two loads
// and a launch: 4 to 6 us for 512 to 4096 rows.
template <int kLanes, int kThreads>
__global__ __launch_bounds__(kThreads) void attend_join_kernel(AttendArgs a) {
  constexpr int kGroups = kThreads / kLanes, kAhead = 4;
  const int b = blockIdx.y, h = blockIdx.x, lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const uint64_t row = static_cast<uint64_t>(b) * a.q_heads + h;
  const F2 *stat = a.part_stat + row * a.most_splits;
  const uint32_t d = a.cache.head_dim;
  const float *part = a.part + row * a.most_splits * d + (lane * 4u < d ? lane * 4 : 0);
  __shared__ F2 sh_stat[kGroups];
  __shared__ F4 sh_out[kGroups][kLanes];
  F2 s[kAhead];
  F4 o[kAhead];
  const auto load = [&](int i0) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = i0 + k * kGroups, at = i < a.most_splits ? i : 0;
      s[k] = stat[at];
      o[k] = *reinterpret_cast<const F4 *>(part + static_cast<uint64_t>(at) * d);
    }
  };
  load(group);
  const Span span = span_of(a, b, false);
  const int units = span.end_unit() - span.first_unit();
  const int n = splits_here(a, units).count(units);
  if (n <= 1) return;  // its only split has written the result
  float top = -INFINITY, total = 0.f;
  F4 x{0.f, 0.f, 0.f, 0.f};
  for (int i0 = group; i0 < n;) {
    float next = top;
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (i0 + k * kGroups < n) next = fmaxf(next, s[k].x);
    const float from = next == -INFINITY ? 0.f : next, keep = __builtin_amdgcn_exp2f(top - from);
    total *= keep;
    x *= keep;
    top = next;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (i0 + k * kGroups >= n) continue;
      const float w = __builtin_amdgcn_exp2f(s[k].x - from);
      total += w * s[k].y;
      x += w * o[k];
    }
    i0 += kAhead * kGroups;
    if (i0 < n) load(i0);
  }
  sh_out[group][lane] = x;
  if (lane == 0) sh_stat[group] = F2{top, total};
  __syncthreads();
  if (threadIdx.x * 8 >= d) return;
  top = -INFINITY;
  for (int g = 0; g < kGroups; ++g) top = fmaxf(top, sh_stat[g].x);
  const float from = top == -INFINITY ? 0.f : top;
  total = 0.f;
  float y[8] = {};
  for (int g = 0; g < kGroups; ++g) {
    const float w = __builtin_amdgcn_exp2f(sh_stat[g].x - from);
    total += w * sh_stat[g].y;
    for (int e = 0; e < 8; ++e) y[e] += w * sh_out[g][threadIdx.x * 2 + e / 4][e % 4];
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  for (int e = 0; e < 8; ++e) y[e] *= inv;
  store_out(a, b, h, threadIdx.x * 8, y);
  if (a.lse && threadIdx.x == 0) a.lse[row] = (top + __builtin_amdgcn_logf(total)) * kLn2;
}

// How a call is cut.  most_splits 1: sequences are not split.
struct Cut {
  Splits splits;  // of the bound
  int units, wanted, most_splits;
};
static Cut cut_of(const Layout &c, int64_t work_groups_per_split, int64_t max_tokens, bool window) {
  // (a window may start inside a unit)
  const int units = static_cast<int>((max_tokens + 15) / 16) + (window || max_tokens == 0 ? 1 : 0);
  if (left_whole(units, work_groups_per_split, c.row_bytes)) return Cut{Splits{units, 1, 1}, units, 1, 1};
  const int wanted = wanted_splits(work_groups_per_split, static_cast<int>(c.head_dim));
  return Cut{splits_of(units, wanted), units, wanted, static_cast<int>(most_splits(units, wanted))};
}
static int columns_of(int group, int head_dim) {  // tiles of 16 query heads that one work-group takes
  const int tiles = (group + 15) / 16, most = head_dim > 128 ? 1 : 4;
  return tiles < most ? tiles : most;
}
static size_t part_bytes(size_t rows, size_t splits, size_t head_dim) {
  return splits > 1 ? rows * splits * (head_dim + 2) * sizeof(float) : 0;
}

template <int kQ, int kC, int kDim, int kTiles>
static bool launch_one(const AttendArgs &a, int n_seqs, hipStream_t s) {
  const dim3 grid(a.cache.kv_heads * a.tiles, n_seqs, a.most_splits);
  if (a.most_splits == 1) return launch(attend_kernel<kQ, kC, kDim, kTiles, true>, grid, 64 * kWholeWaves, s, a);
  return launch(attend_kernel<kQ, kC, kDim, kTiles, false>, grid, 64 * kSplitWaves, s, a);
}
template <int kQ, int kC, int kDim>
static bool launch_columns(const AttendArgs &a, int n_seqs, int columns, hipStream_t s) {
  if constexpr (kDim <= 128) {
    if (columns == 2) return launch_one<kQ, kC, kDim, 2>(a, n_seqs, s);
    if (columns == 3) return launch_one<kQ, kC, kDim, 3>(a, n_seqs, s);
    if (columns == 4) return launch_one<kQ, kC, kDim, 4>(a, n_seqs, s);
  }
  return launch_one<kQ, kC, kDim, 1>(a, n_seqs, s);
}
// A wavefront for a row where there are few splits, four otherwise.
template <int kLanes>
static bool launch_join(const AttendArgs &a, int n_seqs, hipStream_t s) {
  const dim3 rows(a.q_heads, n_seqs);
  if (a.most_splits <= 4 * 64 / kLanes) return launch(attend_join_kernel<kLanes, 64>, rows, 64, s, a);
  return launch(attend_join_kernel<kLanes, 256>, rows, 256, s, a);
}
template <int kQ, int kC>
static bool launch_attend(const AttendArgs &a, int n_seqs, hipStream_t s) {
  const int columns = columns_of(a.group, static_cast<int>(a.cache.head_dim));
  const bool done = a.cache.head_dim <= 64    ? launch_columns<kQ, kC, 64>(a, n_seqs, columns, s)
                    : a.cache.head_dim <= 128 ? launch_columns<kQ, kC, 128>(a, n_seqs, columns, s)
                                              : launch_columns<kQ, kC, 256>(a, n_seqs, columns, s);
  if (!done || a.most_splits == 1) return done;
  if (a.cache.head_dim <= 64) return launch_join<16>(a, n_seqs, s);
  if (a.cache.head_dim <= 128) return launch_join<32>(a, n_seqs, s);
  return launch_join<64>(a, n_seqs, s);
}

}  // namespace kv
}  // namespace rocshmem

using namespace rocshmem;
using namespace rocshmem::kv;

extern "C" {

size_t rocshmem_amd_kv_attend_bytes(const rocshmem_amd_kv_cache_t *cache, int n_seqs, int q_heads, int max_len) {
  Layout c;
  if (!cache || !fill_layout(cache->dtype, cache->page_tokens, cache->kv_heads, cache->head_dim, 1, 1, &c)) return 0;
  if (n_seqs < 1 || n_seqs > 65535 || max_len < 1 || max_len > kMostTokens || q_heads < 1 || q_heads > 65535 || q_heads % cache->kv_heads) return 0;
  const int group = q_heads / cache->kv_heads, columns = columns_of(group, cache->head_dim);
  const int64_t tiles = (group + 16 * columns - 1) / (16 * columns);
  // Fewer sequences are cut into more splits and may need more, up to as many as make
  // kManyGroups work-groups; from there on they are all cut alike.  (Shorter sequences
  // never have more splits than longer ones.)
  const int64_t per_seq = tiles * cache->kv_heads;
  size_t most = 0;
  for (int64_t n = 1; n <= n_seqs; n = n * per_seq < kManyGroups || n == n_seqs ? n + 1 : n_seqs) {
    const size_t bytes = part_bytes(static_cast<size_t>(n) * q_heads,
                                    cut_of(c, n * per_seq, max_len, true).most_splits, c.head_dim);
    if (bytes > most) most = bytes;
  }
  return most;
}

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
  if (n_seqs < 0 || n_seqs > 65535 || max_len < 0 || max_len > kMostTokens || window < 0) return -1;
  if (q_heads < 1 || q_heads % cache->kv_heads || q_heads > 65535) return -1;
  if (!__builtin_isfinite(scale) || !__builtin_isfinite(softcap) || softcap < 0.f) return -1;
  if (!(__builtin_fabsf(scale) < 0x1p127f)) return -1;  // it is multiplied by log2 e
  if (softcap > 0.f && softcap < 0x1p-100f) return -1;  // scores are divided by it
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
  const size_t rows = static_cast<size_t>(n_seqs) * q_heads;
  a.group = q_heads / cache->kv_heads;
  const int columns = columns_of(a.group, cache->head_dim);
  a.tiles = (a.group + 16 * columns - 1) / (16 * columns);
  const int64_t per_split = static_cast<int64_t>(n_seqs) * cache->kv_heads * a.tiles;
  const size_t needed = part_bytes(rows, cut_of(a.cache, per_split, max_len, true).most_splits, a.cache.head_dim);
  if (needed && (!workspace || !aligned_to(workspace, 16) || workspace_bytes < needed ||
                 !drv::local_ok(workspace, workspace_bytes)))
    return -1;
  // (a window or none, no more splits than that)
  const Cut cut = cut_of(a.cache, per_split, window > 0 && window < max_len ? window : max_len, window > 0);
  a.bound_splits = cut.splits;
  a.bound_units = cut.units;
  a.wanted = cut.wanted;
  a.most_splits = cut.most_splits;
  a.part = static_cast<float *>(workspace);
  a.part_stat = reinterpret_cast<F2 *>(a.part + rows * a.most_splits * a.cache.head_dim);
  a.out_dtype = out_dtype;
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
  a.n_seqs = n_seqs;
  a.q_heads = q_heads;
  a.max_len = max_len;
  a.window = window;
  a.my_pe = my_pe;
  a.own_pages = pages_from == ROCSHMEM_AMD_KV_OWN_PAGES;
  a.scale = scale;
  a.softcap = softcap;
  hipStream_t s = drv::as_stream(stream);
  bool done;
  if (cache->dtype == ROCSHMEM_AMD_BF16)
    done = launch_attend<ROCSHMEM_AMD_BF16, ROCSHMEM_AMD_BF16>(a, n_seqs, s);
  else if (cache->dtype == ROCSHMEM_AMD_HALF)
    done = launch_attend<ROCSHMEM_AMD_HALF, ROCSHMEM_AMD_HALF>(a, n_seqs, s);
  else if (dtype == ROCSHMEM_AMD_BF16)
    done = launch_attend<ROCSHMEM_AMD_BF16, ROCSHMEM_AMD_E4M3>(a, n_seqs, s);
  else
    done = launch_attend<ROCSHMEM_AMD_HALF, ROCSHMEM_AMD_E4M3>(a, n_seqs, s);
  return done ? 0 : -1;
}

}  // extern "C"
