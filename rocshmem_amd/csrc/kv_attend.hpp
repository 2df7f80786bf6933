// Attention of one new token per sequence over the paged key-value cache.
//
//   s_t = scale <q, k_t>,  out = sum_t exp(s_t) v_t / sum_t exp(s_t)
//
// One pass over the tokens with a running maximum and sum.  The query heads that
// share a cache head are the columns of matrix products, so keys and values are
// read once for up to 64 of them (16 where rows are over 128 elements: a wavefront's
// registers hold no more sums; the rest are other work-groups', which read the cache
// again), and nothing but the query, the running sums and two steps of keys (in LDS)
// and values (in registers) is held:
//
//   S^T (tokens x heads) = K Q^T,  O^T (dims x heads) += V^T P^T
//
// with v_mfma_f32_16x16x32.  A lane of the product S^T ends up with four
// consecutive tokens of one head, and the product O^T wants eight tokens of one
// head in a lane as its right operand; the order of a product's inner index is
// free as long as both operands agree, so the eight are the lane's four of each
// of two 16-token units, and P never leaves its lane.  V^T's lane then needs the
// same eight tokens at one column; a lane loads a contiguous piece of each of its
// eight tokens' rows (whole rows side by side across the lanes) and pairs up
// tokens with byte permutes: columns are dealt out so that a lane's piece is one
// element of each of the product's tiles.  No value goes through LDS on the way.
#ifndef ROCSHMEM_AMD_KV_ATTEND_HPP_
#define ROCSHMEM_AMD_KV_ATTEND_HPP_

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
  float *part;        // [sequence][query head][split][head_dim], not yet divided
  F2 *part_stat;      // [sequence][query head][split]: exponent the sums are taken from, and sum
  uint64_t q_row, out_row;  // elements between sequences
  uint64_t table_row;
  int n_seqs;
  int q_heads, group, tiles;  // query heads; how many share a cache head; work-groups that share them out
  int max_len, window, my_pe;
  // else: how the bound would be split, of how many units, and what is asked of
  // splits_of where the sequences are shorter; how many splits one can have at most
  Splits bound_splits;
  int bound_units, wanted, most_splits;
  int out_dtype;
  bool own_pages;
  float scale, softcap;
};

// The tokens of a sequence that take part: [first, end).
struct Span {
  int first, end;
  __device__ __forceinline__ int first_unit() const { return first >> 4; }
  __device__ __forceinline__ int end_unit() const { return (end + 15) >> 4; }
};
__device__ __forceinline__ Span span_of(const AttendArgs &a, int b, bool counts) {
  const int len = a.lengths[b];
  int end = len < 0 ? 0 : len < a.max_len ? len : a.max_len;
  const uint64_t held = a.table_row * a.cache.page_tokens;
  if (static_cast<uint64_t>(end) > held) end = static_cast<int>(held);
  if (end != len && counts) count_refused(a.refused);
  return Span{a.window > 0 && end > a.window ? end - a.window : 0, end};
}

// Eight elements of a result row in the type that was asked for.
__device__ __forceinline__ void store_out(const AttendArgs &a, int b, int h, int e, const float (&x)[8]) {
  const uint64_t at = b * a.out_row + static_cast<uint64_t>(h) * a.cache.head_dim + e;
  if (a.out_dtype == ROCSHMEM_AMD_FLOAT)
    Eight<ROCSHMEM_AMD_FLOAT>::store(a.out + at * 4, Eight<ROCSHMEM_AMD_FLOAT>::round(x));
  else if (a.out_dtype == ROCSHMEM_AMD_BF16)
    Eight<ROCSHMEM_AMD_BF16>::store(a.out + at * 2, Eight<ROCSHMEM_AMD_BF16>::round(x));
  else
    Eight<ROCSHMEM_AMD_HALF>::store(a.out + at * 2, Eight<ROCSHMEM_AMD_HALF>::round(x));
}

// Global memory by its address space: an address put together from lanes would
// otherwise be read as flat memory, whose loads are waited for all at once.
typedef const __attribute__((address_space(1))) char *GlobalBytes;
typedef __attribute__((address_space(3))) char *LdsBytes;
template <typename V>
__device__ __forceinline__ V read_at(GlobalBytes from, uint32_t offset) {
  return *(const __attribute__((address_space(1))) V *)(from + offset);  // NOLINT
}
// What is read once: not kept in the caches at the expense of the rest.
template <typename V>
__device__ __forceinline__ V stream_at(GlobalBytes from, uint32_t offset) {
  return __builtin_nontemporal_load((const __attribute__((address_space(1))) V *)(from + offset));  // NOLINT
}
// 16 bytes a lane straight to LDS, lane l's at `to` + 16 l; counted like a load.
__device__ __forceinline__ void stream_to_lds(GlobalBytes from, uint32_t offset, LdsBytes to) {
  constexpr int kNonTemporal = 2;
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(from + offset),  // NOLINT
                                   (__attribute__((address_space(3))) void *)to, 16, 0, kNonTemporal);
}

// The matrix product of a type, and pairs of values rounded to it.
template <int kType>
struct Mma;
template <>
struct Mma<ROCSHMEM_AMD_BF16> {
  using V = B8;
  using E = __bf16;
  __device__ __forceinline__ static F4 mul(V a, V b, F4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  template <bool kHigh>
  __device__ __forceinline__ static unsigned from_e4m3(unsigned codes) {
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, kHigh));
  }
};
template <>
struct Mma<ROCSHMEM_AMD_HALF> {
  using V = H8;
  using E = _Float16;
  __device__ __forceinline__ static F4 mul(V a, V b, F4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  template <bool kHigh>
  __device__ __forceinline__ static unsigned from_e4m3(unsigned codes) {
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.0f, kHigh));
  }
};

// The larger of the four lanes 16 apart that share a column, in all of them.
__device__ __forceinline__ float max_of_column(float x) {
  unsigned u = __float_as_uint(x);
  auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  u = __float_as_uint(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
  r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_of_column(float x) {
  unsigned u = __float_as_uint(x);
  auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  u = __float_as_uint(__uint_as_float(r[0]) + __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// The splits of a sequence of `own` units: the same for all of a call, up to a number
// of sequences that a wavefront can look at.
__device__ __forceinline__ Splits splits_here(const AttendArgs &a, int own) {
  const int near = a.bound_units - a.bound_units / 4;
  int most = own;
  if (a.n_seqs <= kMostLooked) {
    const auto look = [&](int k) {
      const int i = static_cast<int>(threadIdx.x & 63) + 64 * k;
      const Span s = span_of(a, i < a.n_seqs ? i : a.n_seqs - 1, false);
      const int units = s.end_unit() - s.first_unit();
      most = units > most ? units : most;
    };
    look(0);
    if (a.n_seqs > 64) {
#pragma unroll
      for (int k = 1; k < kMostLooked / 64; ++k) look(k);  // (all on their way at once)
    }
    if (!__any(most >= near))
      for (int hop = 32; hop; hop /= 2) {
        const int other = __shfl_xor(most, hop);
        most = other > most ? other : most;
      }
  }
  if (__any(most >= near)) return a.bound_splits;
  return splits_of(__builtin_amdgcn_readfirstlane(most), a.wanted);
}
__device__ __forceinline__ unsigned uniform(unsigned x) { return __builtin_amdgcn_readfirstlane(x); }

// Wavefronts a SIMD is to hold: as many as the registers allow without spilling in
// the loop (a work-group of eight is two, whose four tiles at 128 spill 84 to 132 bytes).
constexpr int waves_of(int dim, int tiles) {
  if (dim == 64) return tiles < 3 ? 3 : 2;
  if (dim == 128) return tiles == 1 ? 3 : tiles == 4 ? 1 : 2;
  return 2;
}

// One work-group: one split of one sequence's tokens for one cache head and up
// to 16 * kTiles of the query heads that share it.  Its wavefronts share the
// tokens out, take 32 at a step, and join their sums through LDS at the end.
// Bound by the cache's bytes where they are many: 64 sequences to 4096 tokens, 8
// query heads on each of 8 x 128 in bf16, 539 MB in 93.7 us, 5.8 TB/s (medians of 112
// launches); 2 to 131072 in e4m3, 406 MB in 70.1 us, 5.8 TB/s.  Three tiles of heads on
// one cache head, 185 MB in 47.0 us, reach 3.9 TB/s: two wavefronts a SIMD, and their
// products between the loads; four, with one wavefront a SIMD, take 79 us a call.
//
// kQ: the activations' type, kC: the cache's; kDim: head_dim rounded up to 64, 128
// or 256; kWhole: one split.
template <int kQ, int kC, int kDim, int kTiles, bool kWhole>
__global__ __launch_bounds__(64 * (kWhole ? kWholeWaves : kSplitWaves), kWhole ? 2 : waves_of(kDim, kTiles))
void attend_kernel(AttendArgs a) {
  constexpr int kAttendWaves = kWhole ? kWholeWaves : kSplitWaves;
  constexpr bool kNarrow = kC == ROCSHMEM_AMD_E4M3;
  // Scores multiply in the activations' type (e4m3 is exact in either), weights
  // and values in the cache's, or in bf16 where the cache is e4m3: a value's scale
  // is folded into its weight, which may then be as large or small as a scale.
  constexpr int kP = kNarrow ? ROCSHMEM_AMD_BF16 : kC;
  using QM = Mma<kQ>;
  using PM = Mma<kP>;
  constexpr int kBytes = kNarrow ? 1 : 2;
  constexpr int kDots = kDim / 32;                // products along a row of keys
  constexpr int kKeyLoads = kDim * kBytes / 64;   // 16-byte loads for a lane's share of a unit's keys
  constexpr int kCols = kDim / 16;                // elements of a value row in a lane
  constexpr int kWords = kCols * kBytes / 4;      // words they take
  // Weights are kept 2^kLift above exp(s - maximum): the maximum is followed only
  // once a score passes it by 2^kSlack, and fp16's smallest weights keep bits.
  constexpr float kLift = kP == ROCSHMEM_AMD_HALF ? 7.f : 0.f, kSlack = 8.f;

  constexpr int kUnitBytes = kKeyLoads * 1024;    // a unit's keys in LDS
  __shared__ float sh_top[kAttendWaves][16 * kTiles], sh_sum[kAttendWaves][16 * kTiles];
  __shared__ union __attribute__((aligned(16))) {
    char keys[kAttendWaves][2][kUnitBytes];       // each wavefront's next step
    float out[kAttendWaves][16][kDim + 4];        // and at the end its sums
  } sh;
  // Whether the registers hold a step's values as the products take them beside the
  // next step's as they are loaded.
  constexpr bool kEarly = kDim <= 128 || kNarrow;
  // Several tiles' queries would take the registers of another wavefront: they lie
  // in LDS, as the products' lanes hold them.
  constexpr bool kQueryInLds = kTiles > 1;
  __shared__ U4 sh_query[kQueryInLds ? kTiles : 1][kQueryInLds ? kDots : 1][64];

  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int column = lane & 15, quad = lane >> 4;
  // Work-groups go round the XCDs in the order of their numbers.  A sequence's splits
  // move on by one, or an XCD would get all of a long sequence where the cache heads
  // and sequences fill whole rounds.
  const int split = blockIdx.z, b = static_cast<int>((blockIdx.y + split) % gridDim.y);
  const uint32_t head = blockIdx.x / a.tiles, tile = blockIdx.x % a.tiles;
  const int head0 = head * a.group + tile * 16 * kTiles;
  const int heads_here = a.group - static_cast<int>(tile) * 16 * kTiles < 16 * kTiles
                             ? a.group - static_cast<int>(tile) * 16 * kTiles : 16 * kTiles;

  // ---- the tokens: units of 16, a lane for each of this wavefront's ---------------------
  const auto entry_of = [&](int unit) {
    const uint32_t index = quotient(static_cast<uint32_t>(unit), a.cache.by_page_units);
    return index < a.table_row ? static_cast<uint32_t>(a.page_table[b * a.table_row + index]) : ~0u;
  };
  // Where PEs' slices are: asked for now, known when the lengths are.
  const detail::HotWords slices = detail::hot_words(a.ctx);
  // A wavefront's units: runs of at most 64, one after the other, from `from` on.
  struct Runs {
    int from, size, each;  // of all wavefronts over all; of this one in a run
  };
  const auto runs_of = [&](const Splits &splits) {
    const int full = splits.size(split), runs = (full + 64 * kAttendWaves - 1) / (64 * kAttendWaves);
    const int run = runs > 1 ? (full + runs - 1) / runs : full;
    return Runs{splits.begin(split), full, (run + 2 * kAttendWaves - 1) / (2 * kAttendWaves) * 2};
  };
  // Without a window, where the splits are the bound's, a unit's number does not
  // depend on any length, and its entry of the page table is asked for before they
  // are known.
  Runs runs = runs_of(a.bound_splits);
  const uint32_t first_number = a.window > 0 ? 0u : entry_of(runs.from + wave * runs.each + lane);
  bool known = a.window == 0;
  const Span span = span_of(a, b, blockIdx.x == 0 && split == 0 && threadIdx.x == 0);
  const int units = span.end_unit() - span.first_unit();
  asm volatile("" ::"s"(slices.x), "s"(slices.y), "s"(slices.z));  // not asked for later
  bool whole = true;  // no other split has any
  if constexpr (!kWhole) {
    const Splits splits = splits_here(a, units);
    const Runs here = runs_of(splits);
    known = known && here.from == runs.from && here.each == runs.each;
    runs = here;
    if (runs.from >= units && split > 0) return;
    whole = splits.count(units) <= 1;
  }
  const int end = runs.from + runs.size < units ? runs.from + runs.size : units;

  unsigned page_lo, page_hi, unit_row;
  int unit_token, n_units;
  // The pages of the units [first, first + count), at most 64, counted from the
  // sequence's first.
  const auto look_up = [&](int first, int count, bool known) __attribute__((always_inline)) {
    const int unit = span.first_unit() + first + lane;
    bool there = lane < count;
    uint64_t page = 0;
    uint32_t at = 0;
    if (there) {
      const uint32_t index = quotient(static_cast<uint32_t>(unit), a.cache.by_page_units);
      at = static_cast<uint32_t>(unit) * 16 - index * a.cache.page_tokens;
      const uint32_t number = known ? first_number : entry_of(unit);
      if (number >= a.cache.n_pages) {
        there = false;
        if (blockIdx.x == 0 && (at == 0 || unit == span.first_unit())) count_refused(a.refused);
      } else {
        const uint32_t pe = owner_of(a.cache, number);
        there = !a.own_pages || static_cast<int>(pe) == a.my_pe;
        // (detail::remote_addr)
        const int64_t stride = static_cast<int64_t>(slices.x | static_cast<uint64_t>(slices.y) << 32);
        const int64_t hop = stride ? (static_cast<int>(pe) - static_cast<int>(slices.z)) * stride
                                   : detail::peer_hop(a.ctx, static_cast<int>(pe));
        page = reinterpret_cast<uint64_t>(a.cache.pages) + hop + page_offset(a.cache, number, pe);
      }
    }
    page_lo = static_cast<unsigned>(page);
    page_hi = static_cast<unsigned>(page >> 32);
    unit_row = head * a.cache.page_tokens + at;
    unit_token = unit * 16;
    // Close up over what takes no part: another PE's pages where only this one's
    // count, page numbers out of range.
    const uint64_t mask = __ballot(there);
    n_units = __popcll(mask);
    if (mask & (mask + 1)) {
      const int before = __popcll(mask & ((uint64_t{1} << lane) - 1));
      const int to = 4 * (there ? before : n_units + lane - before);
      page_lo = __builtin_amdgcn_ds_permute(to, page_lo);
      page_hi = __builtin_amdgcn_ds_permute(to, page_hi);
      unit_row = __builtin_amdgcn_ds_permute(to, unit_row);
      unit_token = __builtin_amdgcn_ds_permute(to, unit_token);
    }
  };

  // ---- the query, and where the lane's loads are from a unit's first row -----------
  // A unit's keys are one run of 16 rows.  They are fetched as they lie, 1 KiB at a
  // time (fetched by the product's lanes, 64 bytes of 16 rows at a time, the same
  // loop ran at 5.0 TB/s instead of 5.9), into LDS, where a lane finds its piece of
  // one token's row.  Rows would start in the same banks there, so row r's 16-byte
  // pieces lie turned by r: a piece's place comes from turning what is fetched.
  const uint32_t d = a.cache.head_dim, row_bytes = a.cache.row_bytes, pieces = row_bytes / 16;
  const auto turn = [&](uint32_t row) { return pieces < 16 ? row * pieces / 16 : row; };
  constexpr uint32_t kFewest = (kDim == 64 ? 16 : kDim / 2 + 16) * kBytes / 16;  // pieces of a row
  const bool narrow_rows = pieces < 4 * kKeyLoads;
  uint32_t key_from[kKeyLoads], key_at[kKeyLoads];
#pragma unroll
  for (int j = 0; j < kKeyLoads; ++j) {
    const uint32_t place = j * 64 + lane, row = place / pieces, p = place - row * pieces;
    const uint32_t piece = p >= turn(row) ? p - turn(row) : p + pieces - turn(row);
    key_from[j] = row < 16 ? row * row_bytes + piece * 16 : 0;  // beyond the unit: its start again
    uint32_t want = 4 * j + quad;
    if (want >= pieces) want = 0;  // beyond the row: not used
    want += turn(column);
    key_at[j] = column * row_bytes + (want < pieces ? want : want - pieces) * 16;
  }
  const uint32_t piece = column * kCols * kBytes;  // beyond the row: columns that nobody reads
  const uint32_t value_at = 4 * quad * row_bytes + (piece < row_bytes ? piece : 0);
  typename QM::V query[kDots] = {};
  const auto load_query = [&]() __attribute__((always_inline)) {
    for (int n = kQueryInLds ? wave : 0; n < kTiles; n += kAttendWaves) {
      const int h = n * 16 + column;
      const char *row = a.q + (b * a.q_row + static_cast<uint64_t>(head0 + (h < heads_here ? h : 0)) * d) * 2;
#pragma unroll
      for (int j = 0; j < kDots; ++j) {
        const uint32_t e = kNarrow ? (j / 2) * 64 + quad * 16 + (j % 2) * 8 : j * 32 + quad * 8;
        typename QM::V v{};
        if (h < heads_here && e < d) v = load_loose<typename QM::V>(row + e * 2);
        if constexpr (kQueryInLds)
          sh_query[n][j][lane] = __builtin_bit_cast(U4, v);
        else
          query[j] = v;
      }
    }
    if constexpr (kQueryInLds) __syncthreads();
  };

  F4 acc[kTiles][kCols];
  float top[kTiles], sum[kTiles];
#pragma unroll
  for (int n = 0; n < kTiles; ++n) {
    top[n] = -INFINITY;
    sum[n] = 0.f;
#pragma unroll
    for (int c = 0; c < kCols; ++c) acc[n][c] = F4{0.f, 0.f, 0.f, 0.f};
  }

  // ---- one step: two units ---------------------------------------------------------
  unsigned values[8][kWords], key_scales[2], value_scales[2];
  const auto of_lane = [](unsigned x, int i) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(x, i)); };
  // As global memory: an address put together from lanes would be read as flat
  // memory, whose loads are waited for all at once.
  const auto page_of = [&](int i) {
    return (GlobalBytes)(of_lane(page_lo, i) | (static_cast<uint64_t>(of_lane(page_hi, i)) << 32));  // NOLINT
  };
  // An odd number of units: the last step's second one is the first again, left out by its weights.
  const auto unit_of = [&](int step, int u) { return 2 * step + u < n_units ? 2 * step + u : 2 * step; };
  const auto my_keys = [&](int u) { return (LdsBytes)&sh.keys[wave][u][0]; };  // NOLINT
  const auto load_keys = [&](int step) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int i = unit_of(step, u);
      const GlobalBytes page = page_of(i);
      const uint32_t row = of_lane(unit_row, i);
      const GlobalBytes from = page + static_cast<uint64_t>(row) * row_bytes;
#pragma unroll
      for (int j = 0; j < kKeyLoads; ++j) stream_to_lds(from, key_from[j], my_keys(u) + j * 1024);
      if constexpr (kNarrow) key_scales[u] = read_at<unsigned>(page + a.cache.key_scale_offset + row, 4 * quad);
    }
  };
  const auto load_values = [&](int step) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int i = unit_of(step, u);
      const GlobalBytes page = page_of(i);
      const uint32_t row = of_lane(unit_row, i);
      const GlobalBytes from = page + a.cache.value_offset + static_cast<uint64_t>(row) * row_bytes;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint32_t at = value_at + t * row_bytes;
        if constexpr (kWords == 1) {
          values[4 * u + t][0] = stream_at<unsigned>(from, at);
        } else if constexpr (kWords == 2) {
          const U2 v = stream_at<U2>(from, at);
          values[4 * u + t][0] = v[0];
          values[4 * u + t][1] = v[1];
        } else {
#pragma unroll
          for (int w = 0; w < kWords; w += 4) {
            const U4 v = stream_at<U4>(from, at + 4 * w);
#pragma unroll
            for (int x = 0; x < 4; ++x) values[4 * u + t][w + x] = v[x];
          }
        }
      }
      if constexpr (kNarrow) value_scales[u] = read_at<unsigned>(page + a.cache.value_scale_offset + row, 4 * quad);
    }
  };

  constexpr int kOnlyLds = 0xc07f;    // s_waitcnt lgkmcnt(0), leaving loads on their way
  constexpr int kOnlyLoads = 0x0f70;  // s_waitcnt vmcnt(0)
  // A weight as parts of 16 bits whose sum it is, each taking what the one before
  // leaves.  Three bf16 parts cut off (not rounded) hold all 24 bits of it.  Two rounded
  // fp16 parts leave at most 2^-22 of it, and a third would lie below fp16's smallest step
  // for most weights.  With two bf16 parts, 2^-17, one 16-bit result in 430 of 64 sequences
  // to 4096 tokens was the neighbour of what 32-bit arithmetic in another order gives, with
  // three one in 2000; the third costs 0 to 4 % of a call (most with rows of 256).
  constexpr int kParts = kP == ROCSHMEM_AMD_BF16 ? 3 : 2;
  typedef typename PM::V Weights[kParts];
  struct Which {                      // of a step's tokens take part
    bool cut, in[2][4];
  };
  const auto which_of = [&](int step) {
    Which w{};
    int token[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) token[u] = __builtin_amdgcn_readlane(unit_token, unit_of(step, u));
    w.cut = 2 * step + 2 > n_units || token[0] < span.first || token[1] + 16 > span.end;
    if (w.cut) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int t = token[u] + 4 * quad + r;
          w.in[u][r] = t >= span.first && t < span.end && 2 * step + u < n_units;
        }
    }
    return w;
  };
  const auto score = [&](int n, F4 (&s)[2]) {
    s[0] = s[1] = F4{0.f, 0.f, 0.f, 0.f};
    const auto query_of = [&](int j) {
      if constexpr (kQueryInLds)
        return __builtin_bit_cast(typename QM::V, sh_query[n][j][lane]);
      else
        return query[j];
    };
#pragma unroll
    for (int j = 0; j < kKeyLoads; ++j)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        U4 raw = *(const __attribute__((address_space(3))) U4 *)(my_keys(u) + key_at[j]);  // NOLINT
        if (4 * j + 4 > static_cast<int>(kFewest) && narrow_rows && 4u * j + quad >= pieces) raw = U4{0, 0, 0, 0};
        if constexpr (kNarrow) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            U4 k;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              k[2 * w] = QM::template from_e4m3<false>(raw[2 * half + w]);
              k[2 * w + 1] = QM::template from_e4m3<true>(raw[2 * half + w]);
            }
            s[u] = QM::mul(__builtin_bit_cast(typename QM::V, k), query_of(2 * j + half), s[u]);
          }
        } else {
          s[u] = QM::mul(__builtin_bit_cast(typename QM::V, raw), query_of(j), s[u]);
        }
      }
    const float by = a.softcap > 0.f ? a.scale : a.scale * kLog2e;  // to a score, base 2
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float up = by;
        if constexpr (kNarrow) up *= two_to((key_scales[u] >> (8 * r)) & 0xff);
        s[u][r] *= up;
      }
  };
  // What this step multiplies has arrived: keys in LDS, values in registers.
  const auto loads_are_here = [&] {
    __builtin_amdgcn_s_waitcnt(kOnlyLoads);
    __builtin_amdgcn_sched_barrier(0);
  };
  // The keys in LDS have been read, and not only asked for, before the next ones
  // may be fetched over them.
  const auto keys_are_read = [&] {
    __builtin_amdgcn_s_waitcnt(kOnlyLds);
    __builtin_amdgcn_sched_barrier(0);
  };
  const auto weigh = [&](int n, const Which &which, F4 (&s)[2], const unsigned (&scales)[2], Weights &weights) {
    if (a.softcap > 0.f) {
      // cap tanh(x), x = s / cap.  Up to x = 5/8 as s times tanh(x) / x, a polynomial in
      // x^2 (minimax, its own error 2^-27.8), so that small scores keep their bits
      // whatever the cap; beyond, by tanh(x) = 1 - 2 / (e^2x + 1), where that is off by at
      // most six half steps of 2^-24.  (The largest caps times log2 e would be infinite.)
      const float in_scale = 1.f / a.softcap;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float x = s[u][r] * in_scale, y = x * x;
          float t = __builtin_fmaf(y, -0.005704987f, 0.020639088f);
          t = __builtin_fmaf(y, t, -0.053739715f);
          t = __builtin_fmaf(y, t, 0.13331442f);
          t = __builtin_fmaf(y, t, -0.3333328f);
          const float near = s[u][r] * (kLog2e * __builtin_fmaf(y, t, 1.f));
          const float e = __builtin_amdgcn_exp2f(__builtin_fabsf(x) * (2.f * kLog2e));
          t = __builtin_fmaf(-2.f, __builtin_amdgcn_rcpf(e + 1.f), 1.f);
          const float far = __builtin_copysignf(a.softcap * (kLog2e * t), x);
          s[u][r] = y < 0.390625f ? near : far;
        }
    }
    if (which.cut) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[u][r] = which.in[u][r] ? s[u][r] : -INFINITY;
    }
    float most = -INFINITY;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) most = fmaxf(most, s[u][r]);
    if (__any(most > top[n] + kSlack)) {
      const float next = fmaxf(top[n], max_of_column(most));
      const float keep = top[n] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top[n] - next);
      sum[n] *= keep;
#pragma unroll
      for (int c = 0; c < kCols; ++c) acc[n][c] *= keep;
      top[n] = next;
    }
    const float from = top[n] == -INFINITY ? 0.f : top[n] - kLift;
    U4 cut_off[kParts];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        float p[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          p[i] = __builtin_amdgcn_exp2f(s[u][r + i] - from);
          sum[n] += p[i];
          if constexpr (kNarrow) {
            p[i] *= two_to((scales[u] >> (8 * (r + i))) & 0xff);
            if (which.cut) p[i] = which.in[u][r + i] ? p[i] : 0.f;
          }
        }
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
          if constexpr (kP == ROCSHMEM_AMD_BF16) {
            const unsigned bits[2] = {__float_as_uint(p[0]), __float_as_uint(p[1])};
            cut_off[part][2 * u + r / 2] = __builtin_amdgcn_perm(bits[1], bits[0], 0x07060302u);
#pragma unroll
            for (int i = 0; i < 2; ++i) p[i] -= __uint_as_float(bits[i] & 0xffff0000u);
          } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const typename PM::E rounded = static_cast<typename PM::E>(p[i]);
              weights[part][4 * u + r + i] = rounded;
              p[i] -= static_cast<float>(rounded);
            }
          }
        }
      }
    if constexpr (kP == ROCSHMEM_AMD_BF16) {
#pragma unroll
      for (int part = 0; part < kParts; ++part) weights[part] = __builtin_bit_cast(typename PM::V, cut_off[part]);
    }
  };
  const auto clear_values = [&](const Which &which) {  // what lies behind the last token may be anything
    if (which.cut) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int w = 0; w < kWords; ++w) values[4 * u + r][w] = which.in[u][r] ? values[4 * u + r][w] : 0u;
    }
  };
  // Columns c and c + 1 of the lane's eight tokens, as the product takes them.
  const auto pair_up = [&](int c, U4 &even, U4 &odd) {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      if constexpr (kNarrow) {
        const unsigned both = __builtin_amdgcn_perm(values[2 * p + 1][c / 4], values[2 * p][c / 4],
                                                    c % 4 ? 0x07030602u : 0x05010400u);
        even[p] = PM::template from_e4m3<false>(both);
        odd[p] = PM::template from_e4m3<true>(both);
      } else {
        even[p] = __builtin_amdgcn_perm(values[2 * p + 1][c / 2], values[2 * p][c / 2], 0x05040100u);
        odd[p] = __builtin_amdgcn_perm(values[2 * p + 1][c / 2], values[2 * p][c / 2], 0x07060302u);
      }
    }
  };
  const auto add = [&](int n, int c, const U4 &column, const typename PM::V &weights) {
    acc[n][c] = PM::mul(__builtin_bit_cast(typename PM::V, column), weights, acc[n][c]);
  };
  // One step.  All scores first, and the values paired up: then nothing of what was
  // loaded is wanted any more, and the next step's loads are on their way while
  // this one's weights and sums are computed.
  const auto take = [&](int step, bool more) __attribute__((always_inline)) {
    const Which which = which_of(step);
    loads_are_here();
    if constexpr (kEarly) {
      F4 s[kTiles][2];
      U4 columns[kCols];
      unsigned scales[2];
#pragma unroll
      for (int n = 0; n < kTiles; ++n) score(n, s[n]);
      clear_values(which);
#pragma unroll
      for (int c = 0; c < kCols; c += 2) pair_up(c, columns[c], columns[c + 1]);
      if constexpr (kNarrow) {
        scales[0] = value_scales[0];
        scales[1] = value_scales[1];
      }
      if (more) {
        keys_are_read();
        load_keys(step + 1);
        load_values(step + 1);
      }
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        Weights weights;
        weigh(n, which, s[n], scales, weights);
        // Part by part, or two columns after each other where the sums take most
        // registers.  Measured, us, the former / the latter: 64 sequences to 4096 tokens in
        // bf16 96.0 / 99.0, 32 with a window of 1024 and rows of 256 in e4m3 21.7 / 20.8.
        if constexpr (kDim <= 128) {
#pragma unroll
          for (int part = 0; part < kParts; ++part)
#pragma unroll
            for (int c = 0; c < kCols; ++c) add(n, c, columns[c], weights[part]);
        } else {
#pragma unroll
          for (int c = 0; c < kCols; c += 2)
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
              add(n, c, columns[c], weights[part]);
              add(n, c + 1, columns[c + 1], weights[part]);
            }
        }
      }
    } else {
      // Not enough registers for both: tile by tile, keys asked for when the last has
      // scored, values at the end.
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        F4 s[2];
        Weights weights;
        score(n, s);
        if (n == kTiles - 1 && more) {
          keys_are_read();
          load_keys(step + 1);
        }
        weigh(n, which, s, value_scales, weights);
        if (n == 0) clear_values(which);
#pragma unroll
        for (int c = 0; c < kCols; c += 2) {
          U4 even, odd;
          pair_up(c, even, odd);
#pragma unroll
          for (int part = 0; part < kParts; ++part) {
            add(n, c, even, weights[part]);
            add(n, c + 1, odd, weights[part]);
          }
        }
      }
      if (more) load_values(step + 1);
    }
  };

  const auto begin_steps = [&](int first, bool known) __attribute__((always_inline)) {
    const int left = end - first;
    look_up(first, left < runs.each ? left : runs.each, known);
    if (n_units > 0) {
      load_keys(0);
      load_values(0);
    }
  };
  const auto take_steps = [&]() __attribute__((always_inline)) {
    // The last step stands by itself, so that no wait has to allow for loads that
    // were not made.
    const int steps = (n_units + 1) / 2;
    int step = 0;
    for (; step + 1 < steps; ++step) take(step, true);
    if (steps > 0) take(step, false);
  };
  if constexpr (kWhole) {
    begin_steps(wave * runs.each, known);
    load_query();  // behind the first keys and values
    take_steps();
  } else {
    load_query();
    for (int first = runs.from; first < end; first += runs.each * kAttendWaves) {
      begin_steps(first + wave * runs.each, known && first == runs.from);
      take_steps();
      keys_are_read();
    }
  }

  // ---- the wavefronts' sums joined -----------------------------------------------
#pragma unroll
  for (int n = 0; n < kTiles; ++n) {
    sum[n] = sum_of_column(sum[n]);
    if (quad == 0) {
      sh_top[wave][n * 16 + column] = top[n] == -INFINITY ? -INFINITY : top[n] - kLift;
      sh_sum[wave][n * 16 + column] = sum[n];
    }
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < kTiles; ++n) {
    const int mine = n * 16 + column;
    float most = -INFINITY;
#pragma unroll
    for (int w = 0; w < kAttendWaves; ++w) most = fmaxf(most, sh_top[w][mine]);
    const float own_top = sh_top[wave][mine];
    const float keep = own_top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(own_top - most);
    if (n) __syncthreads();  // the tile before has been read
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < kCols; c += 4)
        *reinterpret_cast<F4 *>(&sh.out[wave][column][(4 * quad + r) * kCols + c]) =
            F4{acc[n][c][r] * keep, acc[n][c + 1][r] * keep, acc[n][c + 2][r] * keep, acc[n][c + 3][r] * keep};
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * kDim / 8; i += 64 * kAttendWaves) {
      const int h = i / (kDim / 8), e = i % (kDim / 8) * 8;
      if (n * 16 + h >= heads_here || e >= static_cast<int>(d)) continue;
      float from = -INFINITY, total = 0.f, x[8] = {};
#pragma unroll
      for (int w = 0; w < kAttendWaves; ++w) from = fmaxf(from, sh_top[w][n * 16 + h]);
#pragma unroll
      for (int w = 0; w < kAttendWaves; ++w) {
        const float t = sh_top[w][n * 16 + h];
        // (a sum without a maximum is 0, or NaN from NaN scores alone, which lse has to say)
        total += sh_sum[w][n * 16 + h] * (t == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(t - from));
#pragma unroll
        for (int y = 0; y < 8; ++y) x[y] += sh.out[w][h][e + y];
      }
      const uint64_t row = static_cast<uint64_t>(b) * a.q_heads + head0 + n * 16 + h;
      if (whole) {
        const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
        for (int y = 0; y < 8; ++y) x[y] *= inv;
        store_out(a, b, head0 + n * 16 + h, e, x);
        if (e == 0 && a.lse) a.lse[row] = (from + __builtin_amdgcn_logf(total)) * kLn2;
      } else {
        const uint64_t at = row * a.most_splits + split;
        Eight<ROCSHMEM_AMD_FLOAT>::store(reinterpret_cast<char *>(a.part + at * d + e),
                                         Eight<ROCSHMEM_AMD_FLOAT>::round(x));
        if (e == 0) a.part_stat[at] = F2{from, total};
      }
    }
  }
}

}  // namespace kv
}  // namespace rocshmem

#endif  // ROCSHMEM_AMD_KV_ATTEND_HPP_
