// kv4_attention.hip — attention over the pages held in 4 bits, for one token
// a sequence (every page, or selected blocks and the tail) and for several
// (causal, ragged) (gfx950).
//
// out[r] = sum_t p_rt (s_t c_t + m_t) / sum_t p_rt, with p_rt = 2^(z_rt - max)
// and z_rt = log2(e) scale q_r . (s_t c_t + m_t), per group of 32 channels.
//
// Everything runs on v_mfma_f32_16x16x32_f16, whose K is one group:
//   scores   tile T: rows = tokens 16T.., columns = query rows.  The codes
//            enter as FP16 integers and the group's sum takes its token's
//            scale in fp32.  The minima are one more product: m_tg against
//            the groups' sums of q.
//   values   rows = channels, columns = query rows, products over tokens.
//            The operand is c * s, exact in FP16 (7-bit scales); the minima
//            and the denominator are one more product, with rows m_g and 1.
// Both probabilities and maxima live where the score tile leaves them, lane
// (query row, quarter of the tokens), which is the second product's operand.
// fp32 queries and probabilities enter as a high and a low FP16 part (22
// bits); 16-bit queries are exact in one part and the probabilities round to
// FP16 (2^-11 relative).  Queries are scaled by a power of two per row, so that
// none of their parts underflows before 2^-24 of the row's largest.
//
// Work is split by pages, not by lists: the pages of all (sequence, KV head)
// lists form one row of units, and each workgroup takes an equal share of it,
// whatever the lists' lengths.  A list cut by a share's border is merged by the
// last workgroup to finish it.
//
// What bounds it: memory, where the batch is long (8 sequences of up to 131072
// tokens in groups of 4: 184-193 us, 5.2-5.4 TB/s); below that the vector
// instructions of a page (225 at head_dim 64, 325 at 128, 570 for 32 rows, 4
// cycles each: 32 sequences of 5000 to 10000 tokens at head_dim 64 42.7 us, 3.6
// TB/s; 64 of 64 selected blocks in fp32 47 us, 3.6 TB/s); for one sequence of
// 2048 tokens, 11.4 us, the chain length -> table -> record -> sums -> counter
// -> sums of a launch.  The code outside the loop counts there too: fetching it
// for the first time takes longer than running it.
#include "kv4_attention.hpp"

#include <algorithm>
#include <type_traits>

namespace sa {
namespace {

using namespace kv4;

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
// Probabilities are held times 2^shift, against a maximum that may lag the
// true one by `lag` (in exponents of 2): they stay below FP16's largest
// number, and down to 2^-(25 + shift) of the row's largest they are not lost.
// Without a lag every page's maximum would cross lanes and rescale the sums.
template <bool kFine>
constexpr float kShift = kFine ? 14.0f : 6.0f;
template <bool kFine>
constexpr float kLag = kFine ? 1.0f : 9.0f;

// ---- a record in LDS -------------------------------------------------------------
// A wave copies its next record from memory straight into its LDS slot while it
// attends the present one out of registers: no registers are held in flight,
// which leaves room for more waves.

typedef const void __attribute__((address_space(1)))* GlobalPtr;
typedef void __attribute__((address_space(3)))* LdsPtr;
constexpr int kDmaNontemporal = 2;  // a record is read once

template <int D>
__device__ inline void fetch_record(const uint8_t* rec, uint8_t* slot, int lane) {
  constexpr int kBytes = Format<D>::kRecord;
#pragma unroll
  for (int at = 0; at < kBytes; at += kWave * 16)
    if (at + kWave * 16 <= kBytes || lane * 16 < kBytes - at)
      __builtin_amdgcn_global_load_lds((GlobalPtr)(rec + at + lane * 16), (LdsPtr)(slot + at), 16, 0, kDmaNontemporal);
}
__device__ inline void wait_fetch() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// The slot may be fetched into once its reads have returned; another lane's
// word may be read once it has been written.
__device__ inline void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

template <int D>
struct Record {
  using F = Format<D>;
  uint32_t kc[2][F::NG];       // tile T: the lane's word of each group
  uint32_t vc[2][F::NC / 2];   // tile T: 4 tokens x NC nibbles
  uint32_t ks[2][F::NG * 2];   // tile T, group: scales of rows 4j..4j+3
  uint32_t km[2][F::NG / 2];   // minima of token 16T + r
  uint32_t vs[4];              // scales of the lane's channels, 8 slots
  uint32_t vm[4];              // minima of group r % NG, 8 slots
};

template <int N>
__device__ inline void read_words(const uint8_t* p, uint32_t* w) {
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 2) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    w[0] = x.x, w[1] = x.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 x = *reinterpret_cast<const uint4*>(p + 4 * i);
      w[i] = x.x, w[i + 1] = x.y, w[i + 2] = x.z, w[i + 3] = x.w;
    }
  }
}

template <int D>
__device__ inline void read_record(const uint8_t* slot, int lane, Record<D>& x) {
  using F = Format<D>;
  const int r = lane % 16, j = lane / 16;
#pragma unroll
  for (int T = 0; T < 2; ++T) {
    read_words<F::NG / 2>(slot + F::kKeyMins + (16 * T + r) * F::NG * 2, x.km[T]);
    read_words<F::NG>(slot + (16 * T + r) * (D / 2) + j * F::NG * 4, x.kc[T]);
    read_words<F::NG * 2>(slot + F::kKeyScales + (T * 4 + j) * F::NG * 8, x.ks[T]);
    read_words<F::NC / 2>(slot + F::kValueCodes + ((T * 4 + j) * 16 + r) * 2 * F::NC, x.vc[T]);
  }
  read_words<4>(slot + F::kValueMins + (r % F::NG * 4 + j) * 16, x.vm);
  read_words<4>(slot + F::kValueScales + (r * F::NC / 32 * 4 + j) * 16, x.vs);
}

// The value operand of channel n of every row: slots 8j.. of tiles 0 and 1.
template <int D, int N, int kCentre>
__device__ inline half8 value_operand(const Record<D>& x) {
  uint32_t w[4];
#pragma unroll
  for (int T = 0; T < 2; ++T) {
    uint32_t p01, p23;
    if constexpr (D == 64) {  // 16 bits a token: neighbours share a word
      p01 = x.vc[T][0];
      p23 = x.vc[T][1];
    } else {
      constexpr int kStep = D / 128;  // words a token
      constexpr int kWord = N / 8;
      constexpr uint32_t kSel = N % 8 < 4 ? 0x05040100u : 0x07060302u;
      p01 = __builtin_amdgcn_perm(x.vc[T][kStep + kWord], x.vc[T][kWord], kSel);
      p23 = __builtin_amdgcn_perm(x.vc[T][3 * kStep + kWord], x.vc[T][2 * kStep + kWord], kSel);
    }
    w[2 * T] = scaled_codes<N % 4, kCentre>(p01, x.vs[2 * T]);
    w[2 * T + 1] = scaled_codes<N % 4, kCentre>(p23, x.vs[2 * T + 1]);
  }
  return as_half8(w[0], w[1], w[2], w[3]);
}

// ---- the query rows and the state of a wave -------------------------------------

// Row r of tile rt of the list's rows: the lane's operand of the scores, the
// sums of q, and the row's factor from products to exponents of 2.
template <int D, int RT, bool kFine>
struct Rows {
  using F = Format<D>;
  half8 hi[RT][F::NG];
  half8 lo[RT][kFine ? F::NG : 1];
  half8 sums[RT];         // operand of the minima
  float factor[RT];
  int limit[RT];          // last position the row sees
};

// The workgroup's rows, converted once for its waves: a lane takes 8 channels.
// (Unrolled for each wave's own operands the conversion was a third of the
// kernel's code, and fetching instructions took longer than a short list.)
template <int D, int RT, bool kFine>
struct RowStage {
  using F = Format<D>;
  half8 hi[RT * F::NG][kWave];
  half8 lo[kFine ? RT * F::NG : 1][kWave];
  float sum[16 * RT][F::NG];
  float factor[16 * RT];
};

template <int D, int RT, bool kFine>
__device__ inline void load_rows(const Params& p, RowStage<D, RT, kFine>& s, Rows<D, RT, kFine>& q, const Target& tg,
                                 int limit0) {
  using F = Format<D>;
  constexpr int kLanes = D / 8;  // of a row
  const int tid = threadIdx.x, lane = tid % kWave;
#pragma unroll 1
  for (int row = tid / kLanes; row < 16 * RT; row += kThreads / kLanes) {
    const int c = tid % kLanes, g = c / 4, j = c % 4;
    const int token = (tg.row0 + row) / p.group;
    float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (token < tg.n_tokens) {
      const int64_t at = (tg.token0 + token) * p.q_stride +
                         static_cast<int64_t>(tg.head0 + (tg.row0 + row - token * p.group)) * D + 8 * c;
      if constexpr (kFine)
        load8(p.query, at, kF32, x);
      else
        load8(p.query, at, p.type == kF16 ? kF16 : kBF16, x);
    }
    float top = 0.0f;
#pragma unroll
    for (int n = 0; n < 8; ++n) top = fmaxf(top, fabsf(x[n]));
#pragma unroll
    for (int n = 1; n < kLanes; n *= 2) top = fmaxf(top, __shfl_xor(top, n));
    // the row's largest value into [1, 2): a power of two, exact
    const int e = top > 0.0f && top < __builtin_huge_valf() ? __builtin_amdgcn_frexp_expf(top) - 1 : 0;
    half8 hi, lo;
    float sum = 0.0f;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const int i = n / 2 + (n % 2) * 4;  // operand order (0,4), (1,5), ...
      const float v = ldexp2(p.qscale < 0.0f ? -x[i] : x[i], -e);
      hi[n] = static_cast<_Float16>(v);
      lo[n] = static_cast<_Float16>(v - static_cast<float>(hi[n]));
      sum += static_cast<float>(hi[n]);
      if constexpr (kFine) sum += static_cast<float>(lo[n]);
    }
    const int slot = (row / 16) * F::NG + g, of = 16 * j + row % 16;
    s.hi[slot][of] = hi;
    if constexpr (kFine) s.lo[slot][of] = lo;
    sum += __shfl_xor(sum, 1);
    sum += __shfl_xor(sum, 2);
    if (j == 0) s.sum[row][g] = sum;
    if (c == 0) s.factor[row] = ldexp2(fabsf(p.qscale), e);  // not negative: the scale's sign goes to q
  }
  __syncthreads();
  const int r = lane % 16, j = lane / 16;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int row = rt * 16 + r;
    q.limit[rt] = limit0 + min((tg.row0 + row) / p.group, tg.n_tokens - 1);
    q.factor[rt] = s.factor[row];
#pragma unroll
    for (int g = 0; g < F::NG; ++g) {
      q.hi[rt][g] = s.hi[rt * F::NG + g][lane];
      if constexpr (kFine) q.lo[rt][g] = s.lo[rt * F::NG + g][lane];
    }
    // products of the minima: NG slots of high parts, NG of low ones
    half8 op{};
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      float v = 0.0f;
      bool low = false;
      if constexpr (F::NG == 8) {
        v = j < 2 ? s.sum[row][n] : 0.0f;
        low = j == 1;
      } else if (n < 2 * F::NG) {
        v = j == 0 ? s.sum[row][n % F::NG] : 0.0f;
        low = n >= F::NG;
      }
      const _Float16 h = static_cast<_Float16>(v);
      op[n] = low ? static_cast<_Float16>(v - static_cast<float>(h)) : h;
    }
    q.sums[rt] = op;
  }
}

template <int D, int RT>
struct State {
  using F = Format<D>;
  float m[RT];
  f32x4 acc[RT][F::NC];  // channel (4j + i) NC + n of query row r
  f32x4 tail[RT];        // rows 0..NG-1: minima of each group; row NG: the denominator
  bool huge;             // some maximum's rounding is no small change (the same in every lane)
  __device__ inline void reset() {
    huge = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      m[rt] = kNegInf;
      tail[rt] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int n = 0; n < F::NC; ++n) acc[rt][n] = f32x4{0, 0, 0, 0};
    }
  }
};

// Masks the pair of slots (2q, 2q + 1) of the lane beyond `valid` tokens.
__device__ inline uint32_t slot_mask(int q, int j, int valid) {
  const int t = 16 * (q / 2) + 4 * j + 2 * (q % 2);
  return (t < valid ? 0x0000FFFFu : 0u) | (t + 1 < valid ? 0xFFFF0000u : 0u);
}

template <int D, int RT, bool kFine, int N>
__device__ inline void add_values(const Record<D>& x, const half8 (&ph)[RT], const half8 (&pl)[RT],
                                  State<D, RT>& st) {
  const half8 v = value_operand<D, N, kFine ? 8 : 0>(x);
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    st.acc[rt][N] = mfma(v, ph[rt], st.acc[rt][N]);
    if constexpr (kFine) st.acc[rt][N] = mfma(v, pl[rt], st.acc[rt][N]);
  }
  if constexpr (N + 1 < Format<D>::NC) add_values<D, RT, kFine, N + 1>(x, ph, pl, st);
}

// Attends one page: `valid` tokens, the first at position pos; kCausal: a
// row sees the tokens up to its limit.
template <int D, int RT, bool kFine, bool kCausal>
__device__ inline void attend(Record<D>& x, int valid, int pos, int first_limit, const Rows<D, RT, kFine>& q,
                              State<D, RT>& st, int lane) {
  using F = Format<D>;
  const int r = lane % 16, j = lane / 16;
  const bool cut = kCausal && first_limit - pos < kPageTokens - 1;  // some row does not see all of it

  f32x4 z[RT][2];
#pragma unroll
  for (int T = 0; T < 2; ++T) {
    half8 mins;
    {
      const bool on = F::NG == 8 ? j < 2 : j == 0;
      uint32_t w[F::NG / 2];
#pragma unroll
      for (int i = 0; i < F::NG / 2; ++i) w[i] = on ? x.km[T][i] : 0u;
      if constexpr (F::NG == 8)
        mins = as_half8(w[0], w[1], w[2], w[3]);
      else if constexpr (F::NG == 4)
        mins = as_half8(w[0], w[1], w[0], w[1]);
      else
        mins = as_half8(w[0], w[0], 0u, 0u);
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) z[rt][T] = mfma(mins, q.sums[rt], f32x4{0, 0, 0, 0});
#pragma unroll
    for (int g = 0; g < F::NG; ++g) {
      const half8 k = key_codes(x.kc[T][g]);
      const uint32_t s01 = x.ks[T][2 * g], s23 = x.ks[T][2 * g + 1];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        f32x4 d = mfma(k, q.hi[rt][g], f32x4{0, 0, 0, 0});
        if constexpr (kFine) d = mfma(k, q.lo[rt][g], d);
        z[rt][T][0] = __builtin_fmaf(lo_h2f(s01), d[0], z[rt][T][0]);
        z[rt][T][1] = __builtin_fmaf(hi_h2f(s01), d[1], z[rt][T][1]);
        z[rt][T][2] = __builtin_fmaf(lo_h2f(s23), d[2], z[rt][T][2]);
        z[rt][T][3] = __builtin_fmaf(hi_h2f(s23), d[3], z[rt][T][3]);
      }
    }
  }

  half8 ph[RT], pl[RT];
  const bool masked = valid < kPageTokens || cut;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    int seen = valid;
    if (masked) {
      if (kCausal) {
        seen = min(seen, max(q.limit[rt] - pos + 1, 0));
      }
#pragma unroll
      for (int n = 0; n < 8; ++n)
        z[rt][n / 4][n % 4] = 16 * (n / 4) + 4 * j + n % 4 < seen ? z[rt][n / 4][n % 4] : kLowest;
    }
    float top = z[rt][0][0];
#pragma unroll
    for (int n = 1; n < 8; ++n) top = fmaxf(top, z[rt][n / 4][n % 4]);
    top *= q.factor[rt];
    if (__any(top > st.m[rt] + kLag<kFine>)) {
      top = fmaxf(xor_max<32>(xor_max<16>(top)), st.m[rt]);
      const float f = top > st.m[rt] ? __builtin_amdgcn_exp2f(st.m[rt] - top) : 1.0f;
      st.m[rt] = top;
      st.huge |= __any(!(fabsf(top) < 0x1p20f));
      st.tail[rt] *= f;
#pragma unroll
      for (int n = 0; n < F::NC; ++n) st.acc[rt][n] *= f;
    }
    const float off = kShift<kFine> - st.m[rt];
    // one rounding for product and difference: the maximum's own rounding is
    // the row's common factor, unless it passes the whole range of FP16
    float e[8];
    if (__builtin_expect(st.huge, false)) {
      asm volatile("");  // a branch: as a select it would cost three instructions a score
#pragma unroll
      for (int n = 0; n < 8; ++n) e[n] = z[rt][n / 4][n % 4] * q.factor[rt] + off;
    } else {
#pragma unroll
      for (int n = 0; n < 8; ++n) e[n] = __builtin_fmaf(z[rt][n / 4][n % 4], q.factor[rt], off);
    }
#pragma unroll
    for (int n = 0; n < 8; ++n) e[n] = __builtin_amdgcn_exp2f(e[n]);
    if (masked) {
#pragma unroll
      for (int n = 0; n < 8; ++n) e[n] = 16 * (n / 4) + 4 * j + n % 4 < seen ? e[n] : 0.0f;
    }
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      ph[rt][n] = static_cast<_Float16>(e[n]);
      if constexpr (kFine) pl[rt][n] = static_cast<_Float16>(e[n] - static_cast<float>(ph[rt][n]));
    }
  }

  // rows of the last product: the groups' minima, then ones
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (valid < kPageTokens) {
      const uint32_t mask = slot_mask(i, j, valid);  // what lies there is not the sequence's, and may be NaN
      x.vs[i] &= mask;
      x.vm[i] &= mask;
    }
    w[i] = x.vm[i];
  }
  // For fp32 the codes enter less 8, and the minima with 8 scales, in two
  // parts: sums of one sign, whose rounding errors add up, would cancel in the
  // output (64 blocks of 32: 6e-6 of it, against 6e-7; 46 -> 48 us).
  uint32_t low[4];
  if constexpr (kFine) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const half2_t scales = as_half2(__shfl(x.vs[i], 16 * j + r % F::NG * (32 / F::NC)));
      half2_t sum, rest;
      add_eight_times(as_half2(w[i]), scales, sum, rest);
      w[i] = bits_of(sum);
      low[i] = r < F::NG ? bits_of(rest) : 0u;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = r < F::NG ? w[i] : r == F::NG ? 0x3C003C00u : 0u;
  // A NaN minimum in a page that only some rows see wholly: 0 * NaN would
  // reach the others, so it is taken out and added to the rows that see it.
  if constexpr (kCausal) {
    if (cut) {
      bool any = false;
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const bool nan = ((w[n / 2] >> (16 * (n % 2))) & 0x7fffu) > 0x7c00u;
        if (nan) {
          w[n / 2] &= n % 2 ? 0x0000FFFFu : 0xFFFF0000u;
          if constexpr (kFine) low[n / 2] &= n % 2 ? 0x0000FFFFu : 0xFFFF0000u;
        }
        any |= nan;
      }
      if (__any(any)) {
#pragma unroll 1
        for (int t = 0; t < valid; ++t) {  // slot 4T + i of quarter jj of the lane that holds group g's minima
          const int n = 4 * (t / 16) + t % 4;
          uint32_t mine = x.vm[0];
#pragma unroll
          for (int i = 1; i < 4; ++i) mine = n / 2 == i ? x.vm[i] : mine;
          mine = n % 2 ? mine >> 16 : mine & 0xFFFFu;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int g = 4 * j + i;
            const uint32_t h = __shfl(mine, t / 4 % 4 * 16 + g % F::NG);
            if (g < F::NG && (h & 0x7fffu) > 0x7c00u) {
#pragma unroll
              for (int rt = 0; rt < RT; ++rt)
                if (t <= q.limit[rt] - pos) st.tail[rt][i] = __builtin_nanf("");
            }
          }
        }
      }
    }
  }
  const half8 last = as_half8(w[0], w[1], w[2], w[3]);
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    st.tail[rt] = mfma(last, ph[rt], st.tail[rt]);
    if constexpr (kFine) {
      st.tail[rt] = mfma(last, pl[rt], st.tail[rt]);
      st.tail[rt] = mfma(as_half8(low[0], low[1], low[2], low[3]), ph[rt], st.tail[rt]);
    }
  }
  add_values<D, RT, kFine, 0>(x, ph, pl, st);
}

// ---- shares of the row of units ---------------------------------------------------

constexpr int rows_of(int RT) { return 16 * RT; }
constexpr size_t record_floats(int D, int rows) { return static_cast<size_t>(rows) * (D + 2); }

// The waves' sums of 16 rows meet where the records were staged, up to 128
// channels at a time.
template <int D>
struct Meet {
  static constexpr int kChannels = D < 128 ? D : 128;
  static constexpr int kStride = kChannels + 4;  // floats: neighbouring rows in other banks
  static constexpr int kFloats = 16 * kStride;   // of a wave
  static constexpr int kBytes = kWaves * kFloats * 4;
};

__device__ inline void store_out2(const Params& p, int64_t token, int head, int D, int ch, float a, float b) {
  const int64_t at = (token * p.query_heads + head) * D + ch;
  if (p.type == kF32)
    *reinterpret_cast<float2*>(static_cast<float*>(p.out) + at) = make_float2(a, b);
  else
    *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + at) = pack2(a, b, p.type);
}

// Two floats that another workgroup reads in this launch (8-byte aligned).
__device__ inline void store_pair(float* at, float a, float b) {
  store_agent(reinterpret_cast<uint64_t*>(at),
              static_cast<uint64_t>(__float_as_uint(b)) << 32 | __float_as_uint(a));
}
__device__ inline float2 load_pair(const float* at) {
  const uint64_t v = load_agent(reinterpret_cast<const uint64_t*>(at));
  return make_float2(__uint_as_float(static_cast<uint32_t>(v)), __uint_as_float(static_cast<uint32_t>(v >> 32)));
}

// Workgroups a compute unit holds, by their registers.
template <int D, int RT>
constexpr int kPerCu = D == 256 ? 1 : RT == 1 ? 3 : 2;

template <int D, int RT, bool kFine, bool kCausal>
__global__ __launch_bounds__(kThreads, (kPerCu<D, RT>)) void kv4_attention_kernel(const Params p) {
  using F = Format<D>;
  constexpr int kRows = rows_of(RT);
  constexpr int kRecFloats = static_cast<int>(record_floats(D, kRows));
  using M = Meet<D>;
  __shared__ __align__(16) uint8_t s_bytes[std::max<int>(kWaves * F::kRecord, M::kBytes)];
  __shared__ __align__(16) RowStage<D, RT, kFine> s_rows;
  __shared__ float s_m[kWaves][16];
  __shared__ float s_l[kWaves][16];
  __shared__ float s_sum[16];
  __shared__ __align__(16) float s_tail[kWaves][16][20];
  __shared__ int s_last;
  float* s_acc = reinterpret_cast<float*>(s_bytes);
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int lane = tid % kWave;
  const int r = lane % 16, j = lane / 16;
  const uint32_t w = blockIdx.x;
  uint8_t* stage = s_bytes + wave * F::kRecord;

  // ---- the units of the launch, and where this workgroup's share begins ----
  // A list has at least one unit, so that an empty one is written too.
  using unit_t = std::conditional_t<kCausal, int64_t, uint32_t>;
  std::conditional_t<kCausal, Share, SmallShare> sh{};
  unit_t u, end;
  unit_t base = 0;  // units before list (decode: the lists of one selection group's heads) or tile s
  int s = 0;
  if constexpr (kCausal) {
    const Start at = start_share(p, sh, w, kWholePagesOfMany, lane);
    if (!at.any) return;
    s = at.s;
    u = at.u;
    end = at.end;
  } else {
    __shared__ uint32_t s_units[kWaves], s_first[kWaves], s_found[2];
    __shared__ int s_even[kWaves];
    const int lists = p.batch * p.select_groups;
    const int per = (lists + kThreads - 1) / kThreads;
    const int first = min(tid * per, lists), last = min(first + per, lists);
    uint32_t mine = 0, one = 0;  // units of the thread's lists; pages of its first
    uint32_t most = 0;           // and of its longest
    bool even = true;
    for (int i = first; i < last; ++i) {
      const uint32_t n = max(decode_list(p, i / p.select_groups, i % p.select_groups).total, 1);
      if (i == first) one = n;
      even = even && n == one;
      most = max(most, n);
      mine += n * p.kv_per_sel;
    }
    const uint32_t run = wave_prefix_sum(mine);
    const uint32_t head = __builtin_amdgcn_readfirstlane(one);
    even = __all(even && (first == last || one == head));
    const uint32_t all = static_cast<uint32_t>(lists) * p.kv_per_sel;
    const bool whole = __all(whole_lists(all, most, kWholePagesOfMany));
    if (lane == kWave - 1) {
      s_units[wave] = run;
      s_first[wave] = head;
      s_even[wave] = even | whole << 1;
    }
    __syncthreads();
    uint32_t before = 0;
    bool alike = true, all_whole = true;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      if (i < wave) before += s_units[i];
      sh.units += s_units[i];
      all_whole = all_whole && (s_even[i] & 2) != 0;
      alike = alike && (s_even[i] & 1) != 0 && (s_first[i] == s_first[0] || s_units[i] == 0);
    }
    sh.groups = min(gridDim.x, max(1u, sh.units / kMinUnits));
    if (all_whole) {
      if (w >= all) return;
      s = w / p.kv_per_sel;
      const uint32_t pages = max(decode_list(p, s / p.select_groups, s % p.select_groups).total, 1);
      u = w % p.kv_per_sel * pages;  // of the list's own units
      end = u + pages;
    } else {
      // Lists of one length are cut into as many shares each, so that no share
      // crosses from one into the next: one that does writes its sums twice
      // (512 lists of 64 blocks: 57 -> 45 us).
      if (alike && all <= gridDim.x) sh.groups = all * max(1u, sh.groups / all);
      if (w >= sh.groups) return;
      sh.divide();
      u = sh.begin(w);
      end = sh.begin(w + 1);
      before += run - mine;
      if (u - before < mine) {  // (u < before wraps to more than any)
        s_found[0] = first;
        s_found[1] = before;
      }
      __syncthreads();
      s = __builtin_amdgcn_readfirstlane(s_found[0]);
      base = __builtin_amdgcn_readfirstlane(s_found[1]);
    }
  }

  while (u < end) {
    // ---- the list, its rows, and this share's pages [p0, p1) of it ----
    int b, h;
    List L;
    unit_t list_first;   // unit of the list's first page
    int pages;           // units of the list
    Target tg;
    int limit0 = 0;
    if constexpr (kCausal) {
      const int64_t per_head = p.tile_info[1];
      h = static_cast<int>(u / per_head);
      const Tile t = p.tiles[s];
      b = t.batch;
      pages = t.pages;
      list_first = h * per_head + t.first;
      tg.token0 = t.token0;
      tg.n_tokens = t.n_tokens;
      tg.row0 = t.row0;
      limit0 = t.len - t.n_tokens;
      L = List{nullptr, t.len, 0, 0, static_cast<int>((static_cast<uint32_t>(t.len) + kPageTokens - 1) / kPageTokens)};
    } else {
      for (;;) {
        b = s / p.select_groups;
        L = decode_list(p, b, s % p.select_groups);
        pages = max(L.total, 1);
        if (u < base + static_cast<unit_t>(pages) * p.kv_per_sel) break;
        base += static_cast<unit_t>(pages) * p.kv_per_sel;
        ++s;
      }
      const unit_t k = (u - base) / pages;
      h = (s % p.select_groups) * p.kv_per_sel + static_cast<int>(k);
      list_first = base + k * pages;
      tg.token0 = b;
      tg.n_tokens = 1;
      tg.row0 = 0;
    }
    tg.head0 = h * p.group;
    const int p0 = static_cast<int>(u - list_first);
    const int p1 = static_cast<int>(min<int64_t>(pages, p0 + static_cast<int64_t>(end - u)));

    // A lane looks up one of the wave's next 64 pages, so that the chain
    // selected id -> table -> record is walked once for all of them, and the
    // first record is on its way while the rows are read.
    const int64_t head_off = static_cast<int64_t>(h) * F::kRecord;
    const int64_t page_bytes = static_cast<int64_t>(p.kv_heads) * F::kRecord;
    PageRef ref{0, 0};
    const auto fetch = [&](int k) {
      const int64_t page = __builtin_amdgcn_readlane(ref.page, k);
      fetch_record<D>(p.pool + (page * page_bytes + head_off), stage, lane);
    };
    const auto look = [&](int at) {
      ref = PageRef{0, 0};
      if (at + kWaves * lane < p1) ref = resolve(p, b, L, at + kWaves * lane);
      if (at < p1) fetch(0);
    };
    int at = p0 + wave;
    look(at);
    Rows<D, RT, kFine> q;
    load_rows<D, RT, kFine>(p, s_rows, q, tg, limit0);
    State<D, RT> st;
    st.reset();
    const int first_limit = limit0 + tg.row0 / p.group;
    while (at < p1) {
      const int n = min(kWave, (p1 - at + kWaves - 1) / kWaves);
      for (int k = 0; k < n; ++k) {
        wait_fetch();
        Record<D> x;
        read_record<D>(stage, lane, x);
        wait_lds();
        if (k + 1 < n) fetch(k + 1);
        const int valid = __builtin_amdgcn_readlane(ref.valid, k);
        if (valid > 0)
          attend<D, RT, kFine, kCausal>(x, valid, (at + kWaves * k) * kPageTokens, first_limit, q, st, lane);
      }
      at += kWaves * kWave;
      if (at < p1) look(at);
    }

    // ---- the waves' states, then the shares' records ----
    const bool whole = p0 == 0 && p1 == pages;
    float* rec = p.records + (2 * w + (p0 == 0 ? 1 : 0)) * static_cast<int64_t>(kRecFloats);
    const int live_rows = min(kRows, tg.n_tokens * p.group - tg.row0);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      *reinterpret_cast<f32x4*>(&s_tail[wave][r][4 * j]) = st.tail[rt];
      wait_lds();  // the wave's own
      const float l = s_tail[wave][r][F::NG];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float add = s_tail[wave][r][(4 * j + i) * F::NC / 32];
#pragma unroll
        for (int n = 0; n < F::NC; ++n) st.acc[rt][n][i] += add;
      }
      __syncthreads();  // the stages are done with, and the last round's readers
      if (j == 0) {
        s_m[wave][r] = st.m[rt];
        s_l[wave][r] = l;
      }
      __syncthreads();
      float top = kNegInf, sum = 0.0f;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) top = fmaxf(top, s_m[i][r]);
#pragma unroll
      for (int i = 0; i < kWaves; ++i)
        if (s_m[i][r] != kNegInf || s_l[i][r] != 0.0f)
          sum = __builtin_fmaf(s_l[i][r], s_m[i][r] == top ? 1.0f : __builtin_amdgcn_exp2f(s_m[i][r] - top), sum);
      const float f = st.m[rt] == top ? 1.0f : __builtin_amdgcn_exp2f(st.m[rt] - top);
      const int rows = min(16, live_rows - 16 * rt);
      if (wave == 0 && j == 0) {
        s_sum[r] = sum;
        if (!whole && r < rows) store_pair(rec + 2 * (16 * rt + r), top, sum);
      }
      constexpr int kN = M::kChannels / 16;  // of a lane, for each i
#pragma unroll
      for (int c = 0; c < F::NC / kN; ++c) {
        if (c) __syncthreads();
        // channel (4j + i) NC + c kN + n stands at (4j + i) kN + n
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int n = 0; n < kN; n += 4)
            *reinterpret_cast<float4*>(s_acc + wave * M::kFloats + r * M::kStride + (4 * j + i) * kN + n) =
                make_float4(st.acc[rt][c * kN + n][i] * f, st.acc[rt][c * kN + n + 1][i] * f,
                            st.acc[rt][c * kN + n + 2][i] * f, st.acc[rt][c * kN + n + 3][i] * f);
        __syncthreads();
#pragma unroll 1
        for (int e = tid; e < rows * (M::kChannels / 2); e += kThreads) {
          const int of = e / (M::kChannels / 2), at = e % (M::kChannels / 2) * 2;
          const int row = 16 * rt + of, ch = at / kN * F::NC + c * kN + at % kN;
          float a = 0.0f, b = 0.0f;
#pragma unroll
          for (int v = 0; v < kWaves; ++v) {
            const float2 y = *reinterpret_cast<const float2*>(s_acc + v * M::kFloats + of * M::kStride + at);
            a += y.x;
            b += y.y;
          }
          if (whole) {
            const float l = s_sum[of];
            const int token = (tg.row0 + row) / p.group;
            store_out2(p, tg.token0 + token, tg.head0 + (tg.row0 + row - token * p.group), D, ch,
                       l == 0.0f ? 0.0f : a / l, l == 0.0f ? 0.0f : b / l);
          } else {
            store_pair(rec + 2 * kRows + row * D + ch, a, b);
          }
        }
      }
    }
    if (!whole) {
      const int w0 = static_cast<int>(sh.owner(list_first));
      const int w1 = static_cast<int>(sh.owner(list_first + pages - 1));
      const int shares = w1 - w0 + 1;
      if (last_arrival(p.arrive + w0, shares, &s_last)) {
        const auto record = [&](int i) {
          return p.records + (2 * static_cast<int64_t>(w0 + i) + (i == 0 ? 1 : 0)) * kRecFloats;
        };
        // A few channels a thread; with threads to spare each takes every
        // `parts`-th record, and the parts meet in LDS, in order.  One token's
        // lists are cut into many shares, tiles of rows into few.
        constexpr int kWide = kCausal ? 4 : 2, kAtOnce = kCausal ? 4 : 8;  // channels, records on their way
        const int pieces = live_rows * (D / kWide);
        const int parts = min(max(kThreads / pieces, 1), shares);
        const int part = parts > 1 ? tid / pieces : 0;
#pragma unroll 1
        for (int e = tid - part * pieces; e < pieces; e += kThreads) {
          const int row = e / (D / kWide), ch = e % (D / kWide) * kWide;
          // In 64 bits: a share of small weights added to one of a large one
          // loses the same bits every time.
          float top = kNegInf;
          double sum = 0.0, a[kWide] = {};
          const auto add = [&](float m, float l, const float* x) {
            const float to = fmaxf(top, m);
            const double f = m == to ? 1.0f : __builtin_amdgcn_exp2f(m - to);
            const double g = top == to ? 1.0f : __builtin_amdgcn_exp2f(top - to);
            top = to;
            sum = __builtin_fma(l, f, sum * g);
#pragma unroll
            for (int c = 0; c < kWide; ++c) a[c] = __builtin_fma(x[c], f, a[c] * g);
          };
#pragma unroll 1
          for (int i = part; part < parts && i < shares; i += parts * kAtOnce) {
            float2 ml[kAtOnce], x[kAtOnce][kWide / 2];
#pragma unroll
            for (int n = 0; n < kAtOnce; ++n) {
              const float* z = record(min(i + n * parts, shares - 1));
              ml[n] = load_pair(z + 2 * row);
#pragma unroll
              for (int c = 0; c < kWide / 2; ++c) x[n][c] = load_pair(z + 2 * kRows + row * D + ch + 2 * c);
            }
#pragma unroll
            for (int n = 0; n < kAtOnce; ++n)
              if (i + n * parts < shares) add(ml[n].x, ml[n].y, &x[n][0].x);
          }
          if (parts > 1) {  // (one round of the loop)
            float* to = s_acc + (part * pieces + e) * (2 + kWide);
            to[0] = top;
            to[1] = static_cast<float>(sum);
#pragma unroll
            for (int c = 0; c < kWide; ++c) to[2 + c] = static_cast<float>(a[c]);
            __syncthreads();
            if (part > 0) break;
            for (int n = 1; n < parts; ++n) {
              const float* z = s_acc + (n * pieces + e) * (2 + kWide);
              add(z[0], z[1], z + 2);
            }
          }
          const float l = static_cast<float>(sum);
          const int token = (tg.row0 + row) / p.group;
#pragma unroll
          for (int c = 0; c < kWide; c += 2)
            store_out2(p, tg.token0 + token, tg.head0 + (tg.row0 + row - token * p.group), D, ch + c,
                       sum == 0.0 ? 0.0f : static_cast<float>(a[c]) / l,
                       sum == 0.0 ? 0.0f : static_cast<float>(a[c + 1]) / l);
        }
      }
    }

    __syncthreads();  // the next list's records may be fetched over the sums
    u = list_first + p1;
    if constexpr (kCausal) {
      if (p1 == pages && ++s == static_cast<int>(p.tile_info[0])) s = 0;
    }
  }
}

// ---- the tiles of a ragged batch of query tokens ------------------------------------
// A tile's pages end with the last one that its last row sees.  One workgroup.
constexpr int kTileThreads = 1024;

__global__ __launch_bounds__(kTileThreads) void tiles_kernel(const Params p, int rows) {
  __shared__ int32_t before[kTileThreads + 1];
  __shared__ int64_t s_wave[kTileThreads / kWave];
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int per = (p.batch + kTileThreads - 1) / kTileThreads;
  const auto tokens_of = [&](int b) {
    const int64_t a = p.query_start[b], z = p.query_start[b + 1];
    return a >= 0 && z >= a && z <= p.tokens ? static_cast<int>(z - a) : 0;
  };
  const auto tiles_of = [&](int b) {
    return static_cast<int>((static_cast<int64_t>(tokens_of(b)) * p.group + rows - 1) / rows);
  };
  const auto scan = [&](int64_t mine, int64_t& total) {
    int64_t run = mine;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
      const int64_t x = __shfl_up(run, d);
      if (lane >= d) run += x;
    }
    __syncthreads();
    if (lane == kWave - 1) s_wave[wave] = run;
    __syncthreads();
    int64_t pre = 0;
    total = 0;
    for (int i = 0; i < kTileThreads / kWave; ++i) {
      if (i < wave) pre += s_wave[i];
      total += s_wave[i];
    }
    return pre + run - mine;
  };

  // Starts that do not ascend within the rows make sequences share rows:
  // then no tile is attended.
  int64_t mine = 0;
  bool bad = false;
  for (int b = tid * per; b < min((tid + 1) * per, p.batch); ++b) {
    const int64_t a = p.query_start[b], z = p.query_start[b + 1];
    bad |= a < 0 || z < a || z > p.tokens;
    if (tokens_of(b) > p.seq_len[b]) flag_status(p.status, kStatusBadLength);
    mine += tiles_of(b);
  }
  int64_t tiles;
  before[tid] = static_cast<int32_t>(min<int64_t>(scan(mine, tiles), INT32_MAX));
  if (tid == 0) before[kTileThreads] = static_cast<int32_t>(min<int64_t>(tiles, INT32_MAX));
  if (__syncthreads_or(bad)) {
    tiles = 0;
    if (tid == 0) flag_status(p.status, kStatusBadLength);
  }
  int64_t units = 0;
  int longest = 0;
  for (int64_t x0 = 0; x0 < tiles; x0 += kTileThreads) {
    const int64_t x = x0 + tid;
    int b = 0, row0 = 0, pages = 0;
    if (x < tiles) {
      int lo = 0, hi = kTileThreads;
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (before[mid] <= x) lo = mid;
        else hi = mid;
      }
      b = lo * per;
      int64_t at = before[lo];
      for (int n = tiles_of(b); x >= at + n; n = tiles_of(b)) {
        at += n;
        ++b;
      }
      row0 = static_cast<int>(x - at) * rows;
      const int n = tokens_of(b);
      const int last = min((row0 + rows - 1) / p.group, n - 1);
      const int64_t limit = static_cast<int64_t>(p.seq_len[b]) - n + last;
      pages = limit < 0 ? 1 : static_cast<int>(limit / kPageTokens) + 1;
      if (pages > p.table_stride) {  // what the table holds of it
        flag_status(p.status, kStatusBadBlock);
        pages = p.table_stride;
      }
    }
    int64_t sum;
    const int64_t pre = scan(pages, sum);
    if (x < tiles) {
      const int token0 = p.query_start[b];
      p.tiles[x] = Tile{units + pre, b, row0, pages, p.query_start[b + 1] - token0, token0, p.seq_len[b]};
    }
    units += sum;
    longest = max(longest, pages);
  }
  for (int d = 1; d < kWave; d *= 2) longest = max(longest, __shfl_xor(longest, d));
  __syncthreads();
  if (lane == 0) s_wave[wave] = longest;
  __syncthreads();
  int64_t most = 0;
  for (int i = 0; i < kTileThreads / kWave; ++i) most = max(most, s_wave[i]);
  if (tid == 0) {
    p.tile_info[0] = tiles;
    p.tile_info[1] = units;
    p.tile_info[2] = most;
  }
}

// ---- launch ----------------------------------------------------------------------

int grid_groups(int head_dim, int RT) {
  const int per_cu = head_dim == 256 ? kPerCu<256, 1> : RT == 1 ? kPerCu<128, 1> : kPerCu<128, 2>;
  return std::min(kMaxGroups, compute_units() * per_cu);
}

// How a call runs: one token a sequence in a tile of 16 rows; several in this
// file's tiles of 32 rows (16 at head_dim 256, by the registers), or in
// kv4_prompt.hip's of many, from 96 rows a sequence (per KV head) on: 16
// sequences after 8192 tokens, 8 heads of 128, take 86 us in few and 129 in
// many at 48 rows, 150 and 143 at 96, 250 and 161 at 192; after 1024 tokens 27
// and 39, 36 and 43, 50 and 44.
enum class Form { kDecode, kFew, kMany };

struct Plan {
  int rows;         // of a tile
  size_t records;   // bytes
};

Plan plan(Form form, int head_dim) {
  if (form == Form::kMany)
    return {prompt_tile_rows(), 2 * prompt_groups() * prompt_record_floats(head_dim) * sizeof(float)};
  const int RT = form == Form::kFew && head_dim <= 128 ? 2 : 1;
  return {rows_of(RT), 2 * grid_groups(head_dim, RT) * record_floats(head_dim, rows_of(RT)) * sizeof(float)};
}

Form form_of(bool prompt, int64_t tokens, int64_t batch, int group, int head_dim, int type) {
  if (!prompt) return Form::kDecode;
  return type != kF32 && head_dim <= 128 && tokens * group >= 96 * batch ? Form::kMany : Form::kFew;
}

struct Layout {
  size_t records, info, tiles, bytes;
};

Layout layout(const Plan& pl, int64_t batch, int64_t tokens, int group) {
  Layout l{};
  const int64_t tiles = max_tiles(batch, tokens, group, pl.rows);
  l.records = kMaxGroups * sizeof(int32_t);  // behind the arrival counters
  l.info = (l.records + pl.records + 255) / 256 * 256;
  l.tiles = l.info + 256;
  l.bytes = l.tiles + tiles * sizeof(Tile);
  return l;
}

template <int D, int RT, bool kCausal>
void launch_typed(const Params& p, bool fine, hipStream_t stream) {
  const dim3 grid(grid_groups(D, RT));
  if (fine)
    hipLaunchKernelGGL((kv4_attention_kernel<D, RT, true, kCausal>), grid, dim3(kThreads), 0, stream, p);
  else
    hipLaunchKernelGGL((kv4_attention_kernel<D, RT, false, kCausal>), grid, dim3(kThreads), 0, stream, p);
}

template <int D>
void launch_dim(const Params& p, bool fine, hipStream_t stream) {
  if (p.query_start)
    launch_typed<D, D <= 128 ? 2 : 1, true>(p, fine, stream);
  else
    launch_typed<D, 1, false>(p, fine, stream);
}

}  // namespace

namespace kv4 {

int64_t max_tiles(int64_t batch, int64_t tokens, int group, int rows) {
  return tokens * group / rows + std::min(batch, tokens) + 1;
}

hipError_t launch_tiles(const Params& p, int rows, hipStream_t stream) {
  hipLaunchKernelGGL(tiles_kernel, dim3(1), dim3(kTileThreads), 0, stream, p, rows);
  return hipGetLastError();
}

}  // namespace kv4

size_t kv4_attention_workspace_bytes(int32_t batch, int32_t query_heads, int32_t kv_heads, int32_t head_dim,
                                     int64_t tokens) {
  size_t bytes = 0;  // any form's
  for (const Form f : {Form::kDecode, Form::kFew, Form::kMany})
    bytes = std::max(bytes, layout(plan(f, head_dim), batch, tokens, query_heads / kv_heads).bytes);
  return bytes;
}

hipError_t launch_kv4_attention(const Kv4AttnLaunch& a, hipStream_t stream) {
  Params p{};
  p.pool = a.pool;
  p.table = a.table;
  p.seq_len = a.seq_len;
  p.sealed = a.sealed;
  p.selected = a.selected;
  p.counts = a.counts;
  p.query_start = a.query_start;
  p.query = a.query;
  p.out = a.out;
  p.status = a.status;
  p.num_pages = a.num_pages;
  p.q_stride = a.q_stride;
  p.tokens = a.tokens;
  p.batch = a.batch;
  p.table_stride = a.table_stride;
  p.sel_stride = a.sel_stride;
  p.select_groups = a.selected ? a.select_groups : 1;
  p.kv_per_sel = a.kv_heads / p.select_groups;
  p.query_heads = a.query_heads;
  p.kv_heads = a.kv_heads;
  p.group = a.query_heads / a.kv_heads;
  p.type = a.type;
  p.qscale = a.scale * kLog2e;
  const Form form = form_of(a.query_start != nullptr, a.tokens, a.batch, p.group, a.head_dim, a.type);
  const Plan pl = plan(form, a.head_dim);
  const Layout l = layout(pl, a.batch, a.tokens, p.group);
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  p.arrive = reinterpret_cast<int32_t*>(ws);
  p.records = reinterpret_cast<float*>(ws + l.records);
  p.tile_info = reinterpret_cast<int64_t*>(ws + l.info);
  p.tiles = reinterpret_cast<Tile*>(ws + l.tiles);
  if (a.query_start) {
    const hipError_t e = launch_tiles(p, pl.rows, stream);
    if (e != hipSuccess) return e;
  }
  if (form == Form::kMany) return launch_prompt_tiles(p, a.head_dim, stream);
  const bool fine = a.type == kF32;
  if (a.head_dim == 64) launch_dim<64>(p, fine, stream);
  if (a.head_dim == 128) launch_dim<128>(p, fine, stream);
  if (a.head_dim == 256) launch_dim<256>(p, fine, stream);
  return hipGetLastError();
}

}  // namespace sa
