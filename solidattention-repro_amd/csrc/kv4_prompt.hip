// kv4_prompt.hip — causal attention of many query rows over the pages held in
// 4 bits, for 16-bit queries (gfx950).
//
// The same sums as kv4_attention.hip, arranged for arithmetic: a workgroup's
// tile is 256 rows (row = token * group + head) of one KV head, 32 for each of
// its 8 waves, and all of them attend the same page.  The page's 8 KB of codes
// are turned into FP16 once, scale * code + minimum rounded once (2^-11
// relative, as an FP16 cache's own values), by all waves together, into LDS in
// the order of the operands of v_mfma_f32_32x32x16_f16.  For FP16 queries,
// whose output keeps more bits than BF16's, the keys enter as scale * code
// (exact) and their minima by a product more with the sums of q (the output's
// error falls from 3.3e-4 to 3.0e-4 of it, the time rises by 5%).
//   scores   rows = tokens, columns = query rows: lane (column c = lane % 32,
//            half h = lane / 32) holds tokens 8 (i / 4) + 4 h + i % 4, i < 16.
//   values   rows = channels, columns = query rows; product step s runs over
//            tokens 16 s .. 16 s + 15 in the order in which the lane holds their
//            probabilities, so these never move between lanes.
// While up to four pages are attended out of one set of LDS buffers, the next
// four are turned into the other, each on its way into registers before: one
// barrier every four pages.  Of the two waves of a SIMD one converts a page and
// then attends one, the other attends first, so that one's matrix instructions
// meet the other's vector instructions.
//
// What bounds it: a wave's page costs 16 matrix instructions of 32 cycles at
// head_dim 128, and about as many cycles of vector instructions (16 scores a
// lane: product with the row's factor, exponential, conversion, maximum, sum;
// its part of the page's conversion).  Two waves a SIMD run them against each
// other.  32 rows a wave keep its LDS reads (16 KB a page) under the matrix
// cores' time.  Measured, head_dim 128: 8 chunks of up to 1024 tokens after up
// to 15360, groups of 4, FP16, 1610-1650 us, 770 TFLOP/s; one prompt of 4096 tokens,
// BF16, 163 us, 420 TFLOP/s, of which 40 us are the meeting of cut tiles' sums
// and as much the start of each tile.  (The conversion costs a quarter of the
// time; both pages of a pair from one record: 3% less.)
#include "kv4_attention.hpp"

namespace sa {
namespace kv4 {
namespace {

constexpr int kWaves = 8;
constexpr int kThreads = kWaves * kWave;
constexpr int kWaveRows = 32;
constexpr int kRows = kWaves * kWaveRows;
constexpr float kShift = 6.0f;  // probabilities are held times 2^6, against a maximum that
constexpr float kLag = 9.0f;    // may lag by 2^9: below FP16's largest, 2^16

typedef float float2_t __attribute__((ext_vector_type(2)));

__device__ inline f32x16 mfma32(half8 a, half8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// LDS is handed over; loads from memory stay in flight.
__device__ inline void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int D>
struct Page {
  using F = Format<D>;
  half8 k[D / 16][kWave];     // product step, lane of the operand
  half8 v[D / 32][2][kWave];  // channels' tile, product step, lane
  half8 mins[kPageTokens];    // the keys' minima, the NG groups' over and over
  uint32_t nan[2][F::NG];     // bit t: token 16 T + t of the values' group is NaN
  uint32_t valid;             // tokens (0: no page); right behind the words of `nan`
};

constexpr int kBatch = 4;  // pages of a set: two sets fit the LDS of a compute unit

// A thread's part of a page: waves 0..3 keys, 4..7 values.  Wave (tile T of 16
// tokens = wave % 2, half = wave / 2 % 2), lane (r, j) as in the record:
//   keys    token 16T + r, the words of half the groups of quarter j
//   values  tokens 16T + 4j + i, half the channels of row r
template <int D>
struct Raw {
  using F = Format<D>;
  static constexpr int kKeyWords = F::NG / 2;
  uint32_t codes[D == 64 ? 2 : 4];
  uint32_t s[2];  // keys: a scale a word; values: scales of 4 tokens
  uint32_t m[2];  // minima
};

// Where a thread's part lies in a record, whichever it is, and its first place
// in a Page: 32-bit offsets, so that the records' addresses stay scalar.
template <int D>
struct Place {
  uint32_t codes, s, m, to;
  __device__ inline Place(int wave, int lane) {
    using F = Format<D>;
    const int r = lane % 16, j = lane / 16, T = wave % 2, half = wave / 2 % 2;
    if (wave < 4) {
      const int t = 16 * T + r, d = j * F::NG + half * (F::NG / 2);  // first word of the row
      codes = t * (D / 2) + d * 4;
      s = key_scale<D>(t, half * (F::NG / 2));
      m = key_min<D>(t, half * (F::NG / 2));
      to = (d / 2 * kWave + d % 2 * 32 + t) * 16;
    } else {
      codes = F::kValueCodes + ((T * 4 + j) * 16 + r) * 2 * F::NC;
      s = F::kValueScales + (r * F::NC / 32 * 4 + j) * 16 + T * 8;
      m = s + (F::kValueMins - F::kValueScales);
      const int n = half * (F::NC / 2);
      to = D / 16 * kWave * 16 + ((n / 2 * 2 + T) * kWave + j % 2 * 32 + r) * 16 + j / 2 * 8;
    }
  }
};

template <int D>
__device__ inline void fetch(const uint8_t* rec, const Place<D>& at, int wave, Raw<D>& x) {
  const uint8_t* codes = rec + at.codes;
  const uint8_t* s = rec + at.s;
  const uint8_t* m = rec + at.m;
  if (wave < 4) {
    if constexpr (D == 64) {
      x.codes[0] = *reinterpret_cast<const uint32_t*>(codes);
      x.s[0] = *reinterpret_cast<const uint16_t*>(s);
      x.m[0] = *reinterpret_cast<const uint16_t*>(m);
    } else {
      const uint2 w = *reinterpret_cast<const uint2*>(codes);
      x.codes[0] = w.x, x.codes[1] = w.y;
      x.s[0] = *reinterpret_cast<const uint16_t*>(s);
      x.s[1] = *reinterpret_cast<const uint16_t*>(s + 8);  // the next group's
      x.m[0] = *reinterpret_cast<const uint32_t*>(m);
    }
  } else {
    if constexpr (D == 64) {
      const uint2 w = *reinterpret_cast<const uint2*>(codes);
      x.codes[0] = w.x, x.codes[1] = w.y;
    } else {
      const uint4 w = *reinterpret_cast<const uint4*>(codes);
      x.codes[0] = w.x, x.codes[1] = w.y, x.codes[2] = w.z, x.codes[3] = w.w;
    }
    const uint2 a = *reinterpret_cast<const uint2*>(s), b = *reinterpret_cast<const uint2*>(m);
    x.s[0] = a.x, x.s[1] = a.y;
    x.m[0] = b.x, x.m[1] = b.y;
  }
}

__device__ inline uint32_t scaled(half2_t c, half2_t s, half2_t m) { return bits_of(__builtin_elementwise_fma(c, s, m)); }

// Turns the thread's part into operands.  A NaN minimum of the values goes
// into page.nan instead (0 * NaN would reach the rows that do not see the
// token) and its group enters as 0.
template <int D, bool kExact>
__device__ inline void convert(const Raw<D>& x, Page<D>& page, int valid, const Place<D>& at, int wave, int lane) {
  using F = Format<D>;
  const int r = lane % 16, j = lane / 16, T = wave % 2, half = wave / 2 % 2;
  uint8_t* to = reinterpret_cast<uint8_t*>(&page) + at.to;
  if (wave < 4) {
    if (wave == 0 && lane == 0) page.valid = valid;
    if (kExact && j == 0) {
      if constexpr (D == 64) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          reinterpret_cast<uint16_t*>(&page.mins[16 * T + r])[2 * i + half] = static_cast<uint16_t>(x.m[0]);
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) reinterpret_cast<uint32_t*>(&page.mins[16 * T + r])[2 * i + half] = x.m[0];
      }
    }
#pragma unroll
    for (int i = 0; i < F::NG / 2; ++i) {  // the row's next word is the other half of a product step
      const uint32_t w = x.codes[i];
      const half2_t s = as_half2(x.s[i] * 0x10001u);
      half8& k = *reinterpret_cast<half8*>(to + i * 32 * 16);
      if constexpr (kExact) {
        k = as_half8(bits_of(low_nibbles(w) * s), bits_of(high_nibbles(w) * s), bits_of(low_nibbles(w >> 8) * s),
                     bits_of(high_nibbles(w >> 8) * s));
      } else {
        const half2_t m = as_half2((i % 2 ? x.m[0] >> 16 : x.m[0] & 0xFFFFu) * 0x10001u);
        k = as_half8(scaled(low_nibbles(w), s, m), scaled(high_nibbles(w), s, m), scaled(low_nibbles(w >> 8), s, m),
                     scaled(high_nibbles(w >> 8), s, m));
      }
    }
    return;
  }
  uint32_t s[2] = {x.s[0], x.s[1]}, m[2] = {x.m[0], x.m[1]};
  if (valid < kPageTokens) {  // what lies behind is not the sequence's
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int t = 16 * T + 4 * j + 2 * q;
      const uint32_t mask = (t < valid ? 0x0000FFFFu : 0u) | (t + 1 < valid ? 0xFFFF0000u : 0u);
      s[q] &= mask;
      m[q] &= mask;
    }
  }
  uint32_t nan = 0;  // bit i: token 4j + i of the tile
  const half2_t zero{0, 0};  // a minimum is finite or NaN: its product with 0 is 0 or NaN
  if (__any(((bits_of(as_half2(m[0]) * zero) | bits_of(as_half2(m[1]) * zero)) & 0x7FFF7FFFu) != 0)) {
    asm volatile("");
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const bool lo = (m[q] & 0x7fffu) > 0x7c00u, hi = (m[q] >> 16 & 0x7fffu) > 0x7c00u;
      nan |= (lo ? 1u << 2 * q : 0u) | (hi ? 2u << 2 * q : 0u);
      m[q] &= (lo ? 0xFFFF0000u : ~0u) & (hi ? 0x0000FFFFu : ~0u);
    }
    nan <<= 4 * j;
    nan |= __shfl_xor(nan, 16);
    nan |= __shfl_xor(nan, 32);
  }
  if (half == 0 && j == 0 && r * F::NC % 32 == 0) page.nan[T][r * F::NC / 32] = nan;
  uint32_t p01, p23;  // 4 nibbles of tokens (0,1) and (2,3)
  if constexpr (D == 64) {
    p01 = x.codes[0] >> (half * 8);
    p23 = x.codes[1] >> (half * 8);
  } else {
    const uint32_t sel = half == 0 ? 0x05040100u : 0x07060302u;
    p01 = __builtin_amdgcn_perm(x.codes[1], x.codes[0], sel);
    p23 = __builtin_amdgcn_perm(x.codes[3], x.codes[2], sel);
  }
#pragma unroll
  for (int i = 0; i < F::NC / 2; ++i) {
    const uint32_t a = i < 2 ? p01 : p01 >> 8, b = i < 2 ? p23 : p23 >> 8;
    const half2_t ca = i % 2 ? high_nibbles(a) : low_nibbles(a);
    const half2_t cb = i % 2 ? high_nibbles(b) : low_nibbles(b);
    *reinterpret_cast<uint2*>(to + (i / 2 * 2 * kWave + i % 2 * 16) * 16) =
        make_uint2(scaled(ca, as_half2(s[0]), as_half2(m[0])), scaled(cb, as_half2(s[1]), as_half2(m[1])));
  }
}

template <int D>
struct State {
  half8 q[D / 16];
  half8 sums;        // of the row's groups, in two parts: the minima's operand
  f32x16 acc[D / 32];
  float m, l, factor;
  int limit;        // last position the lane's row sees
  int first, last;  // of the wave's rows
  bool huge;
};

// Attends two pages, the first one's tokens from position pos on.
template <int D, bool kExact>
__device__ inline void attend(const Page<D> (&page)[2], int pos, int lane, State<D>& st) {
  constexpr int kNG = Format<D>::NG, kNC = Format<D>::NC, kOps = D / 16;
  const int h = lane / 32;
  // each page's valid tokens (lane 2 NG) and NaN words (lanes before it)
  const int at = min(lane, 2 * kNG);
  const uint32_t info0 = (&page[0].nan[0][0])[at], info1 = (&page[1].nan[0][0])[at];
  // The operands are read ahead of the products that take them, the values'
  // before the exponentials: read one by one, the LDS's latency took half of
  // the time.
  half8 op[kOps], mins{};
  f32x16 z[2];
#pragma unroll
  for (int i = 0; i < kOps; ++i) op[i] = page[0].k[i][lane];
  if constexpr (kExact) mins = page[0].mins[lane % 32];
  __builtin_amdgcn_sched_barrier(0);
  z[0] = f32x16{};
  if constexpr (kExact) z[0] = mfma32(mins, st.sums, z[0]);
#pragma unroll
  for (int i = 0; i < kOps; ++i) z[0] = mfma32(op[i], st.q[i], z[0]);
#pragma unroll
  for (int i = 0; i < kOps; ++i) op[i] = page[1].k[i][lane];
  if constexpr (kExact) mins = page[1].mins[lane % 32];
  __builtin_amdgcn_sched_barrier(0);
  z[1] = f32x16{};
  if constexpr (kExact) z[1] = mfma32(mins, st.sums, z[1]);
#pragma unroll
  for (int i = 0; i < kOps; ++i) z[1] = mfma32(op[i], st.q[i], z[1]);
#pragma unroll
  for (int i = 0; i < kOps; ++i) op[i] = page[0].v[i / 2][i % 2][lane];
  __builtin_amdgcn_sched_barrier(0);

  const int valid0 = __builtin_amdgcn_readlane(info0, 2 * kNG), valid1 = __builtin_amdgcn_readlane(info1, 2 * kNG);
  // some row does not see all of the two pages
  const bool cut = st.first - pos < 2 * kPageTokens - 1 || valid0 < kPageTokens || valid1 < kPageTokens;
  const int left = max(st.limit - pos + 1, 0);
  const int seen[2] = {min(valid0, left), min(valid1, max(left - kPageTokens, 0))};
  const int sees[2] = {seen[0] - 4 * h, seen[1] - 4 * h};  // of the lane's tokens 8 (i / 4) + i % 4
  if (cut) {
#pragma unroll
    for (int i = 0; i < 32; ++i) z[i / 16][i % 16] = 8 * (i % 16 / 4) + i % 4 < sees[i / 16] ? z[i / 16][i % 16] : kLowest;
  }
  float tops[2] = {z[0][0], z[1][0]};
#pragma unroll
  for (int i = 1; i < 16; ++i) {
    tops[0] = fmaxf(tops[0], z[0][i]);
    tops[1] = fmaxf(tops[1], z[1][i]);
  }
  float top = fmaxf(tops[0], tops[1]) * st.factor;
  if (__any(top > st.m + kLag)) {
    top = fmaxf(xor_max<32>(top), st.m);
    const float f = top > st.m ? __builtin_amdgcn_exp2f(st.m - top) : 1.0f;
    st.m = top;
    st.huge |= __any(!(fabsf(top) < 0x1p20f));
    st.l *= f;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) st.acc[c] *= f;
  }
  const float off = kShift - st.m;
  if (__builtin_expect(st.huge, false)) {
    asm volatile("");  // a branch: as a select it would cost three instructions a score
#pragma unroll
    for (int i = 0; i < 32; ++i) z[i / 16][i % 16] = z[i / 16][i % 16] * st.factor + off;
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) z[i / 16][i % 16] = __builtin_fmaf(z[i / 16][i % 16], st.factor, off);
  }
#pragma unroll
  for (int i = 0; i < 32; ++i) z[i / 16][i % 16] = __builtin_amdgcn_exp2f(z[i / 16][i % 16]);
  if (cut) {
    int again[2] = {sees[0], sees[1]};
    asm volatile("" : "+v"(again[0]), "+v"(again[1]));  // 32 comparisons kept from above would not fit the registers
#pragma unroll
    for (int i = 0; i < 32; ++i) z[i / 16][i % 16] = 8 * (i % 16 / 4) + i % 4 < again[i / 16] ? z[i / 16][i % 16] : 0.0f;
  }
  // the denominator adds what the numerator multiplies: the rounded ones
  uint32_t pairs[16];
  float sum[2] = {st.l, 0.0f};
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const half2_t pair = __builtin_convertvector(float2_t{z[i / 8][2 * i % 16], z[i / 8][2 * i % 16 + 1]}, half2_t);
    sum[i % 2] = __builtin_amdgcn_fdot2(pair, half2_t{1, 1}, sum[i % 2], false);
    pairs[i] = bits_of(pair);
  }
  st.l = sum[0] + sum[1];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const half8 p0 = as_half8(pairs[8 * s], pairs[8 * s + 1], pairs[8 * s + 2], pairs[8 * s + 3]);
    const half8 p1 = as_half8(pairs[8 * s + 4], pairs[8 * s + 5], pairs[8 * s + 6], pairs[8 * s + 7]);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) st.acc[c] = mfma32(op[2 * c], p0, st.acc[c]);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) st.acc[c] = mfma32(op[2 * c + 1], p1, st.acc[c]);
    if (s == 0) {
#pragma unroll
      for (int i = 0; i < kOps; ++i) op[i] = page[1].v[i / 2][i % 2][lane];
    }
  }
  if (__builtin_expect(__any(lane < 2 * kNG && (info0 | info1) != 0), false)) {
    asm volatile("");
#pragma unroll 1
    for (int s = 0; s < 2; ++s) {
      const uint32_t visible = seen[s] >= 32 ? ~0u : (1u << seen[s]) - 1u;
#pragma unroll
      for (int i = 0; i < 16; ++i) {  // channel NC (8 (i / 4) + 4 h + i % 4) + .. of rows 0..15, and again 16..31
        const int g = (8 * (i / 4 % 2) + 4 * h + i % 4) * kNC / 32;
        if ((page[s].nan[0][g] | page[s].nan[1][g] << 16) & visible) {
#pragma unroll
          for (int c = 0; c < D / 32; ++c) st.acc[c][i] = __builtin_nanf("");
        }
      }
    }
  }
}

template <int D>
constexpr int kRecordFloats = kWaves * kWave * (D / 2 + 2);  // a wave's sums, maximum and denominator by lane

template <int D>
__device__ inline void store_row(const Params& p, int64_t token, int head, const State<D>& st, float l, int h) {
  constexpr int NC = Format<D>::NC;
#pragma unroll
  for (int i = 0; i < 8; ++i) {  // row rho = 8 (i / 4) + 4 h + i % 4 of each tile, and rho + 16
    const int ch = NC * (8 * (i / 4) + 4 * h + i % 4);
    float x[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) x[n] = l == 0.0f ? 0.0f : st.acc[n / 2][i + 8 * (n % 2)] / l;
    const int64_t at = (token * p.query_heads + head) * D + ch;
    if constexpr (NC == 4) {
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) =
          make_uint2(pack2(x[0], x[1], p.type), pack2(x[2], x[3], p.type));
    } else {
#pragma unroll
      for (int n = 0; n < NC; n += 8)
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + at + n) =
            make_uint4(pack2(x[n], x[n + 1], p.type), pack2(x[n + 2], x[n + 3], p.type),
                       pack2(x[n + 4], x[n + 5], p.type), pack2(x[n + 6], x[n + 7], p.type));
    }
  }
}

template <int D, bool kExact>
__global__ __launch_bounds__(kThreads, 2) void kv4_prompt_kernel(const Params p) {
  using F = Format<D>;
  __shared__ Page<D> s_page[2][kBatch];
  __shared__ int s_last;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  const int h = lane / 32;
  const Place<D> place(wave, lane);
  const int64_t w = blockIdx.x;
  const int64_t per_head = p.tile_info[1];
  const int tiles = static_cast<int>(p.tile_info[0]);
  Share sh{};
  const Start start = start_share(p, sh, w, kWholePages, lane);
  if (!start.any) return;
  int s = start.s;
  int64_t u = start.u;
  const int64_t end = start.end;

  while (u < end) {
    const int head = static_cast<int>(u / per_head);
    const Tile tile = p.tiles[s];
    const int b = tile.batch, row0 = tile.row0, pages = tile.pages;
    const int64_t list_first = head * per_head + tile.first;
    const int token0 = tile.token0, n_tokens = tile.n_tokens, len = tile.len;
    const List L{nullptr, len, 0, 0, pages};
    const int p0 = static_cast<int>(u - list_first);
    const int p1 = static_cast<int>(min<int64_t>(pages, p0 + (end - u)));
    const int rows = min(kRows, n_tokens * p.group - row0);          // of the tile
    const int mine = min(kWaveRows, rows - wave * kWaveRows);        // of the wave (may be none)
    const int row = row0 + wave * kWaveRows + lane % 32;
    const bool live = lane % 32 < mine;
    const int token = row / p.group, qh = head * p.group + row % p.group;

    const int64_t page_bytes = static_cast<int64_t>(p.kv_heads) * F::kRecord;
    const uint8_t* pool = p.pool + static_cast<int64_t>(head) * F::kRecord;
    PageRef ref{0, 0};
    int looked = p0 - 2 * kWave;  // the lanes hold pages [looked, looked + 64)
    Raw<D> raw[2];
    int raw_valid[2];
    const auto get = [&](int i) {  // pages i and i + 1 into registers (the second may not be there)
      if (i + 1 - looked >= kWave) {
        looked = i;
        ref = PageRef{0, 0};
        if (i + lane < p1) ref = resolve(p, b, L, i + lane);
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int64_t page = __builtin_amdgcn_readlane(ref.page, i + s - looked);
        fetch<D>(pool + page * page_bytes, place, wave, raw[s]);
        raw_valid[s] = __builtin_amdgcn_readlane(ref.valid, i + s - looked);
      }
    };
    get(p0);  // on their way while the rows are read

    State<D> st;
    st.m = kNegInf;
    st.l = 0.0f;
    st.huge = false;
    st.limit = len - n_tokens + (live ? token : n_tokens - 1);
    st.first = __builtin_amdgcn_readfirstlane(st.limit);
    st.last = mine > 0 ? __builtin_amdgcn_readlane(st.limit, mine - 1) : -1;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) st.acc[c] = f32x16{};
    {
      float top = 0.0f, x[D / 16][8];
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const int d = 2 * i + h;
#pragma unroll
        for (int n = 0; n < 8; ++n) x[i][n] = 0.0f;
        if (live)
          load8(p.query,
                static_cast<int64_t>(token0 + token) * p.q_stride + static_cast<int64_t>(qh) * D + 32 * (d % F::NG) +
                    8 * (d / F::NG),
                p.type == kF16 ? kF16 : kBF16, x[i]);
#pragma unroll
        for (int n = 0; n < 8; ++n) top = fmaxf(top, fabsf(x[i][n]));
      }
      top = xor_max<32>(top);
      const int e = top > 0.0f && top < __builtin_huge_valf() ? __builtin_amdgcn_frexp_expf(top) - 1 : 0;
      st.factor = ldexp2(fabsf(p.qscale), e);
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const float v = x[i][n / 2 + (n % 2) * 4];  // operand order (0,4), (1,5), ...
          st.q[i][n] = static_cast<_Float16>(ldexp2(p.qscale < 0.0f ? -v : v, -e));
        }
      if constexpr (kExact) {
        float sum[F::NG / 2] = {};  // of groups h, h + 2, .. (word 2 i + h is of group (2 i + h) % NG)
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int n = 0; n < 8; ++n) sum[i % (F::NG / 2)] += static_cast<float>(st.q[i][n]);
        st.sums = half8{};
#pragma unroll
        for (int g = 0; g < F::NG; ++g) {
          const float other = __shfl_xor(sum[g / 2], 32);
          const float v = h != 0 ? 0.0f : g % 2 == 0 ? sum[g / 2] : other;
          st.sums[g] = static_cast<_Float16>(v);
          st.sums[F::NG + g] = static_cast<_Float16>(v - static_cast<float>(st.sums[g]));
        }
        asm volatile("" : "+v"(st.sums));
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i) asm volatile("" : "+v"(st.q[i]));  // made once, not anew for every page
    }

    const auto put = [&](int i, Page<D>* page) {  // pages i and i + 1, which are in registers; then the next two into them
#pragma unroll
      for (int s = 0; s < 2; ++s) convert<D, kExact>(raw[s], page[s], raw_valid[s], place, wave, lane);
      if (i + 2 < p1) get(i + 2);
    };
    // Pages [a, z) are attended out of one set while [z, y) go into the other,
    // in pairs; sets grow from one pair, so that the first is not waited for
    // longer.  (One place in the code for each: two would copy the sums
    // between them.)
    put(p0, s_page[0]);
    lds_barrier();
    const int late = wave / (kWaves / 2) * 2;
    for (int a = p0, z = p0 + 2, set = 0; a < p1; set ^= 1) {
      const int y = min((p1 - p0 + 1) / 2 * 2 + p0, z + min(kBatch, 2 * (z - a)));
      for (int i = 0; i < max(z - a, y - z) + late; i += 2) {
        if (i >= late && z + i - late < y) put(z + i - late, s_page[set ^ 1] + (i - late));
        if (a + i < z && (a + i) * kPageTokens <= st.last)
          attend<D, kExact>(*reinterpret_cast<const Page<D>(*)[2]>(s_page[set] + i), (a + i) * kPageTokens, lane, st);
      }
      lds_barrier();
      a = z;
      z = y;
    }
    st.l = xor_sum<32>(st.l);

    const bool whole = p0 == 0 && p1 == pages;
    if (whole) {
      if (live) store_row<D>(p, token0 + token, qh, st, st.l, h);
    } else {
      const int64_t w0 = sh.owner(list_first), w1 = sh.owner(list_first + pages - 1);
      const int shares = static_cast<int>(w1 - w0 + 1);
      const auto record = [&](int64_t g, bool first) {
        return p.records + (2 * g + (first ? 1 : 0)) * static_cast<int64_t>(kRecordFloats<D>) +
               wave * kWave * (D / 2 + 2) + lane;
      };
      float* rec = record(w, p0 == 0);
      store_agent(rec, st.m);
      store_agent(rec + kWave, st.l);
#pragma unroll
      for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) store_agent(rec + (2 + c * 16 + i) * kWave, st.acc[c][i]);
      if (last_arrival(p.arrive + w0, shares, &s_last) && mine > 0) {
        float top = kNegInf, sum = 0.0f;
        for (int g = 0; g < shares; ++g) top = fmaxf(top, load_agent(record(w0 + g, g == 0)));
#pragma unroll
        for (int c = 0; c < D / 32; ++c) st.acc[c] = f32x16{};
#pragma unroll 1
        for (int g = 0; g < shares; ++g) {
          const float* y = record(w0 + g, g == 0);
          const float m = load_agent(y), l = load_agent(y + kWave);
          const float f = m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
          sum = __builtin_fmaf(l, f, sum);
#pragma unroll
          for (int c = 0; c < D / 32; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              st.acc[c][i] = __builtin_fmaf(load_agent(y + (2 + c * 16 + i) * kWave), f, st.acc[c][i]);
        }
        if (live) store_row<D>(p, token0 + token, qh, st, sum, h);
      }
    }
    u = list_first + p1;
    if (p1 == pages && ++s == tiles) s = 0;
  }
}

}  // namespace

int prompt_tile_rows() { return kRows; }
int prompt_groups() { return compute_units() < kMaxGroups ? compute_units() : kMaxGroups; }
size_t prompt_record_floats(int head_dim) { return static_cast<size_t>(kWaves) * kWave * (head_dim / 2 + 2); }

hipError_t launch_prompt_tiles(const Params& p, int head_dim, hipStream_t stream) {
  const dim3 grid(prompt_groups());
  const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream, p); };
  if (head_dim == 64) launch(p.type == kF16 ? kv4_prompt_kernel<64, true> : kv4_prompt_kernel<64, false>);
  if (head_dim == 128) launch(p.type == kF16 ? kv4_prompt_kernel<128, true> : kv4_prompt_kernel<128, false>);
  return hipGetLastError();
}

}  // namespace kv4
}  // namespace sa
