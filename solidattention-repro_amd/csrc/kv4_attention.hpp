// kv4_attention.hpp — what the attention kernels over 4-bit pages share: their
// parameters, the lists of pages, the operands of the matrix cores, and the
// split of a launch's pages into equal shares.
#pragma once

#include "kv4_format.hpp"
#include "sa_internal.hpp"

namespace sa {
namespace kv4 {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kMaxGroups = 4096;   // workgroups, and arrival counters at the front of the workspace
constexpr int kMinUnits = 8;       // pages a workgroup is worth starting for
constexpr float kNegInf = -__builtin_huge_valf();
constexpr float kLowest = -3.0e38f;  // of masked scores: finite, so that a factor of 0 leaves no NaN
constexpr float kLog2e = 1.4426950408889634f;


struct Tile;

struct Params {
  const uint8_t* pool;
  const int32_t* table;
  const int32_t* seq_len;
  const int32_t* sealed;
  const int32_t* selected;
  const int32_t* counts;
  const int32_t* query_start;
  const void* query;
  void* out;
  int32_t* status;
  int32_t* arrive;
  float* records;
  int64_t* tile_info;  // prompt: [0] tiles, [1] units of one KV head, [2] pages of the longest
  Tile* tiles;
  int64_t num_pages;
  int64_t q_stride;
  int32_t tokens;
  int32_t batch;
  int32_t table_stride;
  int32_t sel_stride;
  int32_t select_groups;
  int32_t kv_per_sel;
  int32_t query_heads;
  int32_t kv_heads;
  int32_t group;
  int32_t type;
  float qscale;
};

// ---- lists of pages -----------------------------------------------------------

struct List {
  const int32_t* sel;
  int64_t len;   // tokens that may be read
  int sealed;    // blocks the list's tail starts behind
  int n_sel;
  int total;     // pages
};

// One token a sequence: the selected blocks then the tail, or every page.
// Inconsistent lengths are flagged and clamped to what can be read safely.
__device__ inline List decode_list(const Params& p, int b, int sg) {
  List L{nullptr, p.seq_len[b], 0, 0, 0};
  bool bad = L.len < 0;
  if (p.selected) {
    L.sealed = p.sealed[b];
    L.n_sel = p.counts[static_cast<int64_t>(b) * p.select_groups + sg];
    L.sel = p.selected + (static_cast<int64_t>(b) * p.select_groups + sg) * p.sel_stride;
    bad = bad || L.sealed < 0 || L.len < static_cast<int64_t>(L.sealed) * kPageTokens;
    if (L.n_sel < 0 || L.n_sel > p.sel_stride) {
      L.n_sel = 0;
      flag_status(p.status, kStatusBadLength);
    }
  }
  if (bad) {
    flag_status(p.status, kStatusBadLength);
    if (L.sealed < 0) L.sealed = 0;
    L.len = static_cast<int64_t>(L.sealed) * kPageTokens;
  }
  int64_t tail = (L.len + kPageTokens - 1) / kPageTokens - L.sealed;  // pages
  const int64_t room = p.table_stride - L.sealed;
  if (tail > room) {  // what the table holds of it
    flag_status(p.status, kStatusBadBlock);
    tail = room > 0 ? room : 0;
  }
  L.total = L.n_sel + static_cast<int>(tail);
  return L;
}

struct PageRef {
  int32_t page;   // a readable page in any case
  int32_t valid;  // its tokens (0: skip)
};

__device__ inline PageRef resolve(const Params& p, int b, const List& L, int i) {
  PageRef r{0, 0};
  if (i >= L.total) return r;
  int64_t logical;
  int valid = kPageTokens;
  if (i < L.n_sel) {
    logical = L.sel[i];
    if (logical < 0 || logical >= L.sealed) {
      flag_status(p.status, kStatusBadBlock);
      return r;
    }
  } else {
    logical = static_cast<int64_t>(L.sealed) + (i - L.n_sel);
    const int64_t left = L.len - logical * kPageTokens;
    if (left < kPageTokens) valid = static_cast<int>(left);
  }
  if (logical >= p.table_stride) {
    flag_status(p.status, kStatusBadBlock);
    return r;
  }
  const int32_t page = p.table[static_cast<int64_t>(b) * p.table_stride + logical];
  if (page < 0 || page >= p.num_pages) {
    flag_status(p.status, kStatusBadPage);
    return r;
  }
  r.page = page;
  r.valid = valid;
  return r;
}

// ---- operands of the matrix cores ----------------------------------------------

__device__ inline half8 as_half8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_bit_cast(half8, u32x4{a, b, c, d});
}
__device__ inline half2_t as_half2(uint32_t a) { return __builtin_bit_cast(half2_t, a); }
__device__ inline uint32_t bits_of(half2_t a) { return __builtin_bit_cast(uint32_t, a); }

// x & mask | base in one instruction (the compiler splits it over two literals).
__device__ inline uint32_t and_or(uint32_t x, uint32_t mask, uint32_t base) {
  uint32_t d;
  asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(d) : "v"(x), "s"(mask), "v"(base));
  return d;
}

// Nibbles 0 and 1 of both halves as FP16 integers (less kCentre): moved into
// the mantissa of 1024.0 (bits 0..3) or 64.0 (bits 4..7), which is then taken
// off (exact).
template <int kCentre = 0>
__device__ inline half2_t low_nibbles(uint32_t w) {
  return as_half2(and_or(w, 0x000F000Fu, 0x64006400u)) - half2_t{1024 + kCentre, 1024 + kCentre};
}
template <int kCentre = 0>
__device__ inline half2_t high_nibbles(uint32_t w) {
  return as_half2(and_or(w, 0x00F000F0u, 0x54005400u)) - half2_t{64 + kCentre, 64 + kCentre};
}

// 8 nibbles in the order (0,4), (1,5), (2,6), (3,7).
__device__ inline half8 key_codes(uint32_t w) {
  return as_half8(bits_of(low_nibbles(w)), bits_of(high_nibbles(w)), bits_of(low_nibbles(w >> 8)),
                  bits_of(high_nibbles(w >> 8)));
}

// Nibble n (0..3) of both halves as FP16 integers, less kCentre, times the
// pair of scales (exact: 4 + 7 bits).
template <int N, int kCentre>
__device__ inline uint32_t scaled_codes(uint32_t y, uint32_t scales) {
  const uint32_t w = N < 2 ? y : y >> 8;
  return bits_of((N % 2 == 0 ? low_nibbles<kCentre>(w) : high_nibbles<kCentre>(w)) * as_half2(scales));
}

// a + 8 b = sum + rest, without an error
__device__ inline void add_eight_times(half2_t a, half2_t b, half2_t& sum, half2_t& rest) {
  const half2_t c = b * half2_t{8, 8};
  sum = a + c;
  const half2_t d = sum - a;
  rest = (a - (sum - d)) + (c - d);
}

__device__ inline f32x4 mfma(half8 a, half8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ inline float ldexp2(float x, int e) { return __builtin_ldexpf(x, e); }

// ---- shares of the row of units ---------------------------------------------------
// The pages of all lists form one row of units; workgroup w of `groups` takes
// units [begin(w), begin(w + 1)), whatever lists they belong to.

// One token a sequence: fewer than 2^31 units (refused otherwise), at most 4096
// groups.
struct SmallShare {
  uint32_t units;    // of the whole launch
  uint32_t groups;   // workgroups that take part
  uint32_t each, rest;  // units = each * groups + rest
  __device__ inline void divide() {
    each = units / groups;
    rest = units - each * groups;
  }
  // floor(units * w / groups)
  __device__ inline uint32_t begin(uint32_t w) const { return each * w + rest * w / groups; }
  __device__ inline uint32_t owner(uint32_t u) const {
    uint32_t w = static_cast<uint32_t>(static_cast<float>(u) * (static_cast<float>(groups) / static_cast<float>(units)));
    if (w >= groups) w = groups - 1;
    while (begin(w) > u) --w;
    while (begin(w + 1) <= u) ++w;
    return w;
  }
};

// Tiles of many tokens may pass 2^31 units.  (The 32-bit form for fewer cost
// more than it saved there: 42 against 36 us for 16 sequences of 5 tokens.)
struct Share {
  int64_t units;
  int64_t groups;
  __device__ inline int64_t begin(int64_t w) const { return units * w / groups; }
  __device__ inline int64_t owner(int64_t u) const { return ((u + 1) * groups - 1) / units; }
};

// Lists of few pages, a workgroup for each, are not cut: the shares' sums would
// take longer to meet than the pages to be attended.  With lists for a quarter
// of the launch's workgroups, which then share the memory's rate, that holds
// for longer ones (256 lists at head_dim 64, cut and whole: up to 2 pages 30
// and 7.5 us, 16 pages 17.2 and 10.0, 32 pages 17.3 and 12.9, 63 pages 21.2 and
// 18.4); not for tiles of many rows, whose pages take ten times as long.
constexpr int kWholePages = 16;
constexpr int kWholePagesOfMany = 48;
__device__ inline bool whole_lists(int64_t lists, int64_t longest, int many) {
  return lists <= static_cast<int64_t>(gridDim.x) &&
         longest <= (lists * 4 >= static_cast<int64_t>(gridDim.x) ? many : kWholePages);
}

// `rows` rows (token * group + head) of one sequence, for every KV head.
struct Tile {
  int64_t first;   // unit of its first page, for the first head
  int batch;       // sequence
  int row0;        // its first row of the sequence
  int pages;       // that its last row sees
  int n_tokens;    // query tokens of the sequence
  int token0;      // the first of them
  int len;         // tokens of the sequence
};
static_assert(sizeof(Tile) == 32, "two 16-byte loads");

// The tile of the unit, 0 <= at < tile_info[1]: each lane compares one of 64
// candidates.
__device__ inline int find_tile(const Params& p, int64_t at, int lane) {
  int lo = 0, n = static_cast<int>(p.tile_info[0]);
  while (n > 1) {
    const int step = (n + kWave - 1) / kWave;
    const bool below = lane * step < n && p.tiles[lo + lane * step].first <= at;
    const int k = __popcll(__ballot(below)) - 1;
    lo += k * step;
    n = min(step, n - k * step);
  }
  return lo;
}

// The first list and unit of workgroup w and the end of its share.
struct Start {
  int s;   // tile
  int64_t u, end;
  bool any;
};
__device__ inline Start start_share(const Params& p, Share& sh, int64_t w, int whole_of_many, int lane) {
  const int64_t tiles = p.tile_info[0], per_head = p.tile_info[1], longest = p.tile_info[2];
  sh.units = per_head * p.kv_heads;
  if (sh.units <= 0) return Start{0, 0, 0, false};
  if (whole_lists(tiles * p.kv_heads, longest, whole_of_many)) {
    if (w >= tiles * p.kv_heads) return Start{0, 0, 0, false};
    const int s = static_cast<int>(w) % static_cast<int>(tiles);
    const int64_t u = static_cast<int>(w) / static_cast<int>(tiles) * per_head + p.tiles[s].first;
    return Start{s, u, u + p.tiles[s].pages, true};
  }
  sh.groups = min<int64_t>(gridDim.x, max<int64_t>(1, sh.units / kMinUnits));
  if (w >= sh.groups) return Start{0, 0, 0, false};
  const int64_t u = sh.begin(w);
  return Start{find_tile(p, u % per_head, lane), u, sh.begin(w + 1), true};
}

struct Target {
  int64_t token0;  // first query row of the sequence
  int n_tokens;
  int head0;       // first query head
  int row0;        // first row of the tile (row = token * group + head)
};

// The tiles of `rows` rows each of a batch of query tokens (kv4_attention.hip)
// into p.tiles and p.tile_info.
hipError_t launch_tiles(const Params& p, int rows, hipStream_t stream);
int64_t max_tiles(int64_t batch, int64_t tokens, int group, int rows);

// Tiles of many rows (kv4_prompt.hip; head_dim 64 and 128): rows of a tile,
// workgroups of a launch, floats of one of its two records a workgroup.
int prompt_tile_rows();
int prompt_groups();
size_t prompt_record_floats(int head_dim);
hipError_t launch_prompt_tiles(const Params& p, int head_dim, hipStream_t stream);

}  // namespace kv4
}  // namespace sa
