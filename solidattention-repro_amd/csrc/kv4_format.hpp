// kv4_format.hpp — the record of a page held in 4 bits, and the arithmetic of
// its values (device side; the layout is part of the C-ABI, sa_hip.h).
//
// A record is one KV head's 32 tokens of a page: 40 D bytes for head_dim D,
// against 128 D in FP16.  Every row (K or V of a token) is cut into groups of
// 32 channels with an FP16 scale and minimum each: value = scale * code +
// minimum.
//
// Why this layout: a wave reads a record with full-width contiguous loads
// whose lanes receive exactly the operands of v_mfma_f32_16x16x32_f16.  Lane
// (r = lane % 16, j = lane / 16) of that instruction holds row r and 8
// consecutive products k = 8j..8j+7 of each operand.
//   keys    row r is token 16T + r; the lane's 8 products of a group are
//           channels 32g + 8j + n, so its NG groups are NG adjacent words.
//   values  the products run over tokens: slot 8j + 4T + i is token 16T + 4j
//           + i, which is where the lane already holds that token's
//           probability (row 4j + i of score tile T), so the probabilities
//           never move between lanes.  Row r of operand n is channel r NC + n.
// One scale has at most 7 significant bits, so that code * scale (4 + 7 bits)
// is exact in FP16: the value operand of the matrix cores needs no rounding.
#pragma once

#include "sa_device.hpp"

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sa {
namespace kv4 {

constexpr float kLimit = 32000.0f;  // 15 scales of the widest group, 64320, still fit FP16

template <int D>
struct Format {
  static_assert(D == 64 || D == 128 || D == 256, "head_dim");
  static constexpr int NG = D / 32;  // groups of a row
  static constexpr int NC = D / 16;  // channels of a value operand's row
  static constexpr int kValueCodes = 16 * D;
  static constexpr int kKeyScales = 32 * D;
  static constexpr int kKeyMins = 34 * D;
  static constexpr int kValueScales = 36 * D;
  static constexpr int kValueMins = 38 * D;
  static constexpr int kRecord = 40 * D;
};

// ---- one group of 32 channels over 4 adjacent lanes (8 channels each) ---------

struct Group {
  uint32_t codes;  // 8 nibbles of this lane's channels
  uint16_t scale;  // the same in the 4 lanes
  uint16_t minimum;
};

template <int Ctrl>
__device__ inline float quad_min(float a) { return fminf(a, dpp_f<Ctrl>(a)); }
template <int Ctrl>
__device__ inline float quad_max(float a) { return fmaxf(a, dpp_f<Ctrl>(a)); }

// The two fp32 roundings (x - minimum, then the quotient) are part of the
// format's definition: they decide the code of a value next to a border.
__device__ inline Group quantise(const float (&x)[8]) {
  float lo = kLimit, hi = -kLimit;
  bool nan = false;
  float c[8];
#pragma unroll
  for (int n = 0; n < 8; ++n) {
    nan |= x[n] != x[n];
    c[n] = fminf(fmaxf(x[n], -kLimit), kLimit);
    lo = fminf(lo, c[n]);
    hi = fmaxf(hi, c[n]);
  }
  lo = quad_min<kDppQuadXor2>(quad_min<kDppQuadXor1>(lo));
  hi = quad_max<kDppQuadXor2>(quad_max<kDppQuadXor1>(hi));
  float bad = nan ? 1.0f : 0.0f;
  bad = quad_max<kDppQuadXor2>(quad_max<kDppQuadXor1>(bad));
  Group g{0, 0, 0x7e00};
  if (bad != 0.0f) return g;  // a NaN: the whole group reads as NaN
  g.minimum = f2h_rne(lo + 0.0f);
  const float m = h2f(g.minimum);
  const float raw = fmaxf(hi - m, 0.0f) / 15.0f;
  // up to 7 significant bits; below 2^-18 up to a multiple of 2^-24 (FP16 subnormals)
  float s = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, raw) + 0x1FFFFu) & ~0x1FFFFu);
  if (s < 0x1p-18f) s = ceilf(raw * 0x1p24f) * 0x1p-24f;
  g.scale = f2h_rne(s);
  if (s > 0.0f) {
    // The rounded quotient by the scale's reciprocal and one correction: with
    // a scale of 7 bits it equals the division's for every quotient up to 15.5
    // that does not underflow (to code 0 either way), and takes 3 instructions
    // where the division takes 11 (16384 tokens, 8 heads of 128: 33 -> 27 us).
    const float inv = 1.0f / s;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const float d = c[n] - m, q0 = d * inv;
      const float q = fminf(fmaxf(rintf(__builtin_fmaf(__builtin_fmaf(-q0, s, d), inv, q0)), 0.0f), 15.0f);
      g.codes |= static_cast<uint32_t>(q) << (4 * n);
    }
  }
  return g;
}

// ---- rows of a record ---------------------------------------------------------
// `o` is a lane's octet of a row: channels 8o..8o+7.

template <int D>
__device__ inline int key_word(int t, int o) {  // bytes
  using F = Format<D>;
  return t * (D / 2) + ((o % 4) * F::NG + o / 4) * 4;
}
template <int D>
__device__ inline int key_scale(int t, int g) {
  return Format<D>::kKeyScales + 2 * ((t / 4 * Format<D>::NG + g) * 4 + t % 4);
}
template <int D>
__device__ inline int key_min(int t, int g) {
  return Format<D>::kKeyMins + 2 * (t * Format<D>::NG + g);
}
template <int D>
__device__ inline int value_meta(int t, int g) {  // from kValueScales or kValueMins
  return 2 * ((g * 4 + t / 4 % 4) * 8 + 4 * (t / 16) + t % 4);
}

template <int D>
__device__ inline void store_key(uint8_t* rec, int t, int o, const Group& g) {
  *reinterpret_cast<uint32_t*>(rec + key_word<D>(t, o)) = g.codes;
  if (o % 4 == 0) {
    *reinterpret_cast<uint16_t*>(rec + key_scale<D>(t, o / 4)) = g.scale;
    *reinterpret_cast<uint16_t*>(rec + key_min<D>(t, o / 4)) = g.minimum;
  }
}

template <int D>
__device__ inline void store_value(uint8_t* rec, int t, int o, const Group& g) {
  using F = Format<D>;
  uint8_t* base = rec + F::kValueCodes + (t / 4) * 16 * 2 * F::NC + (t % 4) * (F::NC / 2);
  if constexpr (D == 64) {  // a row of 4 channels: 2 bytes
    *reinterpret_cast<uint16_t*>(base + (2 * o) * 8) = static_cast<uint16_t>(g.codes);
    *reinterpret_cast<uint16_t*>(base + (2 * o + 1) * 8) = static_cast<uint16_t>(g.codes >> 16);
  } else if constexpr (D == 128) {
    *reinterpret_cast<uint32_t*>(base + o * 16) = g.codes;
  } else {
    *reinterpret_cast<uint32_t*>(base + (o / 2) * 32 + (o % 2) * 4) = g.codes;
  }
  if (o % 4 == 0) {
    *reinterpret_cast<uint16_t*>(rec + F::kValueScales + value_meta<D>(t, o / 4)) = g.scale;
    *reinterpret_cast<uint16_t*>(rec + F::kValueMins + value_meta<D>(t, o / 4)) = g.minimum;
  }
}

__device__ inline void expand(uint32_t codes, uint16_t scale, uint16_t minimum, float (&x)[8]) {
  const float s = h2f(scale), m = h2f(minimum);
#pragma unroll
  for (int n = 0; n < 8; ++n) x[n] = __builtin_fmaf(static_cast<float>((codes >> (4 * n)) & 15u), s, m);
}

template <int D>
__device__ inline void load_key(const uint8_t* rec, int t, int o, float (&x)[8]) {
  expand(*reinterpret_cast<const uint32_t*>(rec + key_word<D>(t, o)),
         *reinterpret_cast<const uint16_t*>(rec + key_scale<D>(t, o / 4)),
         *reinterpret_cast<const uint16_t*>(rec + key_min<D>(t, o / 4)), x);
}

template <int D>
__device__ inline void load_value(const uint8_t* rec, int t, int o, float (&x)[8]) {
  using F = Format<D>;
  const uint8_t* base = rec + F::kValueCodes + (t / 4) * 16 * 2 * F::NC + (t % 4) * (F::NC / 2);
  uint32_t codes;
  if constexpr (D == 64) {
    codes = *reinterpret_cast<const uint16_t*>(base + (2 * o) * 8) |
            static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(base + (2 * o + 1) * 8)) << 16;
  } else if constexpr (D == 128) {
    codes = *reinterpret_cast<const uint32_t*>(base + o * 16);
  } else {
    codes = *reinterpret_cast<const uint32_t*>(base + (o / 2) * 32 + (o % 2) * 4);
  }
  expand(codes, *reinterpret_cast<const uint16_t*>(rec + F::kValueScales + value_meta<D>(t, o / 4)),
         *reinterpret_cast<const uint16_t*>(rec + F::kValueMins + value_meta<D>(t, o / 4)), x);
}

// ---- rows of 8 values in the caller's type --------------------------------------

enum Type : int32_t { kF32 = 0, kF16 = 1, kBF16 = 2 };

__device__ inline float bf2f(uint16_t bits) { return __builtin_bit_cast(float, static_cast<uint32_t>(bits) << 16); }
// Round to nearest even; a NaN stays one.
__device__ inline uint16_t f2bf_rne(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  if (x != x) return static_cast<uint16_t>((u >> 16) | 0x40u);
  return static_cast<uint16_t>((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}

__device__ inline int type_bytes(int type) { return type == kF32 ? 4 : 2; }

// 8 values from element `at` (16-byte aligned rows)
__device__ inline void load8(const void* p, int64_t at, int type, float (&x)[8]) {
  if (type == kF32) {
    const float4* f = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
    const float4 a = f[0], b = f[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    return;
  }
  const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + at);
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    x[2 * n] = type == kF16 ? lo_h2f(u[n]) : __builtin_bit_cast(float, u[n] << 16);
    x[2 * n + 1] = type == kF16 ? hi_h2f(u[n]) : __builtin_bit_cast(float, u[n] & 0xffff0000u);
  }
}

__device__ inline uint32_t pack2(float a, float b, int type) {
  const uint16_t lo = type == kF16 ? f2h_rne(a) : f2bf_rne(a);
  const uint16_t hi = type == kF16 ? f2h_rne(b) : f2bf_rne(b);
  return static_cast<uint32_t>(lo) | static_cast<uint32_t>(hi) << 16;
}

__device__ inline void store8(void* p, int64_t at, int type, const float (&x)[8]) {
  if (type == kF32) {
    float4* f = reinterpret_cast<float4*>(static_cast<float*>(p) + at);
    f[0] = make_float4(x[0], x[1], x[2], x[3]);
    f[1] = make_float4(x[4], x[5], x[6], x[7]);
    return;
  }
  *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + at) =
      make_uint4(pack2(x[0], x[1], type), pack2(x[2], x[3], type), pack2(x[4], x[5], type), pack2(x[6], x[7], type));
}

}  // namespace kv4
}  // namespace sa
