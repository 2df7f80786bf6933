// The paged key-value cache on the symmetric heap: where a token's rows lie,
// and the checks its entry points share.  The arithmetic is plain C++ used by
// host and device code alike.
//
// Pages of a fixed number of tokens are numbered over all PEs: PE p holds pages
// p * pages_per_pe up to (p + 1) * pages_per_pe, one after the other in one
// symmetric object.  A page is one contiguous block, so that moving a page to
// another PE is one putmem:
//
//   keys   [kv_heads][page_tokens][head_dim]
//   values [kv_heads][page_tokens][head_dim]
//   e4m3 only: key scales [kv_heads][page_tokens], value scales, one byte each
//   padding to a multiple of 128 bytes
//
// Head-major within the page: attention reads one head's tokens of a page as
// one run of page_tokens * head_dim elements.
#ifndef ROCSHMEM_AMD_KV_CACHE_HPP_
#define ROCSHMEM_AMD_KV_CACHE_HPP_

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "rocshmem_amd.h"

namespace rocshmem {
namespace kv {

constexpr int kTokenUnit = 16;  // page_tokens and head_dim are multiples of it
constexpr int kMaxHeadDim = 256;

// n / d for 0 <= n < 2^31 as a multiplication: mul = floor(2^(31+l) / d) + 1 with
// l = ceil(log2 d), so that 0 < mul * d - 2^(31+l) <= 2^l and the quotient is
// exact; mul fits in 32 bits because d > 2^(l-1).
struct Divisor {
  uint32_t d, mul, shift;
};
__host__ __device__ inline Divisor make_divisor(uint32_t d) {
  uint32_t l = 0;
  while ((uint64_t{1} << l) < d) ++l;
  return Divisor{d, static_cast<uint32_t>((uint64_t{1} << (31 + l)) / d + 1), 31 + l};
}
__host__ __device__ inline uint32_t quotient(uint32_t n, const Divisor &by) {
  return static_cast<uint32_t>((static_cast<uint64_t>(n) * by.mul) >> by.shift);
}

inline int element_bytes(int dtype) {
  switch (dtype) {
    case ROCSHMEM_AMD_FLOAT: return 4;
    case ROCSHMEM_AMD_BF16:
    case ROCSHMEM_AMD_HALF: return 2;
    case ROCSHMEM_AMD_E4M3: return 1;
    default: return 0;
  }
}

struct Layout {
  char *pages;          // this PE's copy of the symmetric object
  uint64_t page_bytes;
  uint64_t value_offset;                       // from the start of a page
  uint64_t key_scale_offset, value_scale_offset;
  uint32_t row_bytes;                          // one token's row of one head
  uint32_t page_tokens, kv_heads, head_dim;
  uint32_t pages_per_pe, n_pages;              // n_pages: over all PEs
  Divisor by_page_units;                       // page_tokens / 16
  Divisor by_pages_per_pe;
};

struct Place {
  uint32_t page, at;  // page over all PEs, token within it
};
__host__ __device__ inline bool slot_in_range(const Layout &c, int64_t slot) {
  return slot >= 0 && slot < static_cast<int64_t>(c.n_pages) * c.page_tokens;
}
// Slots are divided in units of 16 tokens, so that every quotient is one of
// 31-bit numbers (fill_layout refuses a cache with more units).
__host__ __device__ inline Place place_of(const Layout &c, int64_t slot) {
  Place p;
  p.page = quotient(static_cast<uint32_t>(slot >> 4), c.by_page_units);
  p.at = static_cast<uint32_t>(slot - static_cast<int64_t>(p.page) * c.page_tokens);
  return p;
}
__host__ __device__ inline uint32_t owner_of(const Layout &c, uint32_t page) {
  return quotient(page, c.by_pages_per_pe);
}
// Offset of a page from the start of its owner's copy.
__host__ __device__ inline uint64_t page_offset(const Layout &c, uint32_t page, uint32_t owner) {
  return static_cast<uint64_t>(page - owner * c.pages_per_pe) * c.page_bytes;
}
// Offset within a page of token `at`'s row of head `head`; its scale byte.
__host__ __device__ inline uint64_t row_offset(const Layout &c, uint32_t head, uint32_t at, bool value) {
  return (value ? c.value_offset : 0) +
         static_cast<uint64_t>(head * c.page_tokens + at) * c.row_bytes;
}
__host__ __device__ inline uint64_t scale_offset(const Layout &c, uint32_t head, uint32_t at, bool value) {
  return (value ? c.value_scale_offset : c.key_scale_offset) + head * c.page_tokens + at;
}

// Fills in everything but `pages`; false for a cache that is not supported.
inline bool fill_layout(int dtype, int page_tokens, int kv_heads, int head_dim, int64_t pages_per_pe,
                        int npes, Layout *out) {
  const int es = dtype == ROCSHMEM_AMD_FLOAT ? 0 : element_bytes(dtype);
  if (!es || page_tokens < kTokenUnit || page_tokens % kTokenUnit || page_tokens > 65536) return false;
  if (head_dim < kTokenUnit || head_dim % kTokenUnit || head_dim > kMaxHeadDim) return false;
  if (kv_heads < 1 || kv_heads > 4096 || pages_per_pe < 1 || npes < 1) return false;
  const int64_t units = page_tokens / kTokenUnit;
  if (pages_per_pe > INT32_MAX || pages_per_pe * npes > INT32_MAX / units) return false;
  Layout c{};
  c.row_bytes = static_cast<uint32_t>(head_dim * es);
  c.page_tokens = static_cast<uint32_t>(page_tokens);
  c.kv_heads = static_cast<uint32_t>(kv_heads);
  c.head_dim = static_cast<uint32_t>(head_dim);
  const uint64_t rows = static_cast<uint64_t>(kv_heads) * page_tokens;  // < 2^28
  c.value_offset = rows * c.row_bytes;
  c.key_scale_offset = 2 * c.value_offset;
  c.value_scale_offset = c.key_scale_offset + rows;
  const uint64_t used = c.key_scale_offset + (dtype == ROCSHMEM_AMD_E4M3 ? 2 * rows : 0);
  c.page_bytes = (used + 127) / 128 * 128;
  c.pages_per_pe = static_cast<uint32_t>(pages_per_pe);
  c.n_pages = static_cast<uint32_t>(pages_per_pe * npes);
  c.by_page_units = make_divisor(static_cast<uint32_t>(units));
  c.by_pages_per_pe = make_divisor(c.pages_per_pe);
  *out = c;
  return true;
}

// ---- how attention's work is cut ---------------------------------------------------

// How a sequence's units of 16 tokens are split over work-groups: n_big splits of
// `big`, the rest into ones of `small`.
struct Splits {
  int big, n_big, small;
  __host__ __device__ int begin(int i) const { return i < n_big ? i * big : n_big * big + (i - n_big) * small; }
  __host__ __device__ int size(int i) const { return i < n_big ? big : small; }
  __host__ __device__ int count(int units) const {  // how many have any of so many units
    return units <= n_big * big ? (units + big - 1) / big : n_big + (units - n_big * big + small - 1) / small;
  }
};

// Short sequences take a work-group of eight wavefronts each and no second kernel;
// longer ones are split over work-groups of four.
constexpr int kSplitWaves = 4, kWholeWaves = 8;
// How sequences are split: the first half of the longest as for `wanted` equal
// splits, the second half into splits a third as long (whole steps of the
// wavefronts, no shorter than two), and all sequences alike.  Work-groups start in
// the order of their numbers, so the short splits fill the gaps at the end, where a
// CU with one long split more than the others would be waited for (a CU takes little
// more than its share of the memory's rate, so a split too many on it is not made
// up for).  Measured, us a call, in equal splits / with a half in thirds: 64 sequences to
// 4096 tokens in bf16 99.5 / 95.9, 48 heads on one 56.9 / 50.4, 16 sequences with own
// heads 29.1 / 25.9, 2 to 131072 in e4m3 74.5 / 74.9.
//
// The longest is the longest of the call as a wavefront finds it, not the bound that
// a captured call has to give.  Measured, us, split by a bound of 131072 / by the longest,
// 8 cache heads of 128 in bf16: 1 sequence of 2000 tokens 24.8 / 14.2, 4 of 2000 37.5 /
// 16.1, 4 of 8000 79.4 / 29.7, 16 of 2000 40.0 / 31.4; 64 of 2000, which the bound
// leaves in one piece each, 88.6 / 96.2.  Only where it is near the bound is the bound
// taken, whose splits' places are known beforehand (looking costs such a call about 1 us).
//
// How fine that is goes by the number of sequences, not by how their lengths are spread:
// with 64 or more on 8 cache heads half of the longest is one work-group's.  Where one is
// far longer than all others the call waits for that: 585 us for one sequence of 131072
// tokens among 63 of 300, which take 100 and 23 us in calls of their own.
constexpr int kMostLooked = 256;        // sequences; with more each goes by its own length
constexpr int kStep = 2 * kSplitWaves;  // units of a step of all wavefronts
__host__ __device__ inline Splits splits_of(int units, int wanted) {
  if (units <= 6 * kStep) return Splits{6 * kStep, 1, 2 * kStep};  // one
  int big = (units + wanted - 1) / wanted, small = 2 * kStep;
  big = big > 3 * kStep ? (big + kStep - 1) / kStep * kStep : 3 * kStep;
  if (big / 3 > small) small = (big / 3 + kStep - 1) / kStep * kStep;
  const int n_big = units / 2 / big;
  return Splits{big, n_big > 1 ? n_big : 1, small};
}
// The most splits of a sequence of at most so many units.  With x = units / big <=
// wanted there are floor(x / 2) big ones (one at least) and at most ceil(3 (x - floor(x / 2)))
// small ones, 2 wanted + 2 together (four for wanted = 2, where big is half); and no
// small one is shorter than two steps.
inline int64_t most_splits(int64_t units, int64_t wanted) {
  const int64_t by_number = wanted == 2 ? 4 : 2 * wanted + 2, by_length = units / (2 * kStep) + 2;
  return by_number < by_length ? by_number : by_length;
}
constexpr int64_t kManyGroups = 512;
// How many splits the longest is cut for: 512 work-groups, two for each CU; at least
// two, and three unless work-groups are many already or large (wavefronts of 256
// elements take all registers).  Measured, us, for two / three: 32 sequences to 8000
// and 8 cache heads of 64 in e4m3 46.4 / 39.6, to 4000 in bf16 of 128 56.4 / 52.2, 16
// with 24 heads of 64 28.3 / 26.2; 64 to 4096 with 8 heads of 128 95.9 / 98.6, with 4
// of 256 in e4m3 57.7 / 60.9.
inline int wanted_splits(int64_t work_groups, int head_dim) {
  const int64_t each = (kManyGroups + work_groups - 1) / work_groups;
  const int64_t least = work_groups < kManyGroups && head_dim <= 128 ? 3 : 2;
  return static_cast<int>(each > least ? each : least);
}
// Not split are sequences of at most 48 units, three steps of a wavefront, or 72 where
// that fills half the GPU and rows are short.  Measured, us, whole / split, all sequences
// of 1152 tokens, 72 units: rows of 256 bytes (bf16) on 64 work-groups 17.4 / 15.8, 96
// 17.6 / 18.1, 128 18.4 / 20.4, 192 21.9 / 26.1; (e4m3) 64 20.4 / 17.8, 96 21.1 / 21.4,
// 128 21.4 / 23.6, 192 24.0 / 33.0; of 128 bytes 64 14.3 / 13.4, 128 14.6 / 15.3, 192
// 15.2 / 18.8; of 512 bytes 64 36.9 / 25.5, 128 39.2 / 35.3, and from 160 on 41.1 / 47.0
// (not used).  At 900 tokens, 57 units, the order is the same.
constexpr bool left_whole(int64_t units, int64_t work_groups, int64_t row_bytes) {
  return units <= (work_groups >= 128 && row_bytes <= 256 ? 72 : 48);
}

}  // namespace kv
}  // namespace rocshmem

#endif  // ROCSHMEM_AMD_KV_CACHE_HPP_
