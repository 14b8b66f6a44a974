// The 8-bit KV cache's format (include/nsd_kv8.h): scales, codes and values,
// shared by its writers, its reader and the attention over it.
#pragma once

#include "nsd_device.h"
#include "nsd_kv8.h"

namespace nsd {
namespace {

typedef f16 f16x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

constexpr int kKv8Tile = kBlockTokens * kHeadDim;  // bytes of a block's K (or V) codes of one layer and head
constexpr int kKv8Units = kKv8Tile / 16;           // its 16-byte units

__device__ inline float kv8_float(uint32_t bits) { return __builtin_bit_cast(float, bits); }

// 2^e of a scale byte (2^-127, which no writer makes, as 0).
__device__ inline float kv8_power(int byte) { return kv8_float((uint32_t)byte << 23); }

// Exponent of the scale for values whose largest finite magnitude has the fp16
// bits m: f 2^p (1 <= f < 2) fits under 448 = 1.75 2^8, or 127 = 1.984375 2^6,
// times 2^(p - 8) or 2^(p - 6), unless f is past that.  0 gives the smallest.
template <int T>
__device__ inline int kv8_exponent(uint32_t m) {
  const uint32_t f = __builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(f16, (uint16_t)m));
  const int p = (int)(f >> 23) - 127;
  const uint32_t frac = f & 0x7fffffu;
  if constexpr (T == NSD_KV8_E4M3) return min(max(p - 8 + (frac > 0x600000u), -15), 8);
  else return min(max(p - 6 + (frac > 0x7e0000u), -24), 9);
}

// |bits| of eight values, and the largest of them.
__device__ inline u16x8 kv8_abs(f16x8 h) { return __builtin_bit_cast(u16x8, h) & (uint16_t)0x7fff; }
__device__ inline uint32_t kv8_most(u16x8 v) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, (uint32_t)v[e]);
  return m;
}
constexpr uint32_t kF16Inf = 0x7c00;  // |bits| from here on are not finite

// Eight values as codes under the scale 2^e.  Division by a power of two is
// exact and the conversion rounds once.  `careful` (one for the wave): values
// may not be finite, or end past the largest code (65504 under 2^8 or 2^9).
template <int T>
__device__ inline u32x2 kv8_codes(f16x8 h, int e, bool careful) {
  u32x2 out;
  if constexpr (T == NSD_KV8_E4M3) {
    const float power = kv8_float((uint32_t)(e + 127) << 23);
    uint32_t nan[2] = {0, 0};
    if (careful) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool off = (__builtin_bit_cast(u16x8, h)[i] & 0x7fffu) >= kF16Inf;
        nan[i / 4] |= off ? 0x7fu << (8 * (i % 4)) : 0u;
        const float x = __builtin_amdgcn_fmed3f((float)h[i], -61440.f, 61440.f);
        h[i] = off ? (f16)0.f : (f16)x;
      }
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      s16x2 c = {0, 0};
      c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(c, f16x2{h[4 * q], h[4 * q + 1]}, power, false);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(c, f16x2{h[4 * q + 2], h[4 * q + 3]}, power, true);
      out[q] = __builtin_bit_cast(uint32_t, c) | nan[q];
    }
  } else {
    // 1.5 2^23 + x has x, to the nearest even, in its low bits
    const float inv = kv8_float((uint32_t)(127 - e) << 23);
    uint32_t t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float x = (float)h[i];
      if (careful) {
        const bool off = (__builtin_bit_cast(u16x8, h)[i] & 0x7fffu) >= kF16Inf;
        x = off ? 0.f : __builtin_amdgcn_fmed3f(x, -65024.f, 65024.f);  // 127 * 2^9
      }
      t[i] = __builtin_bit_cast(uint32_t, __builtin_fmaf(x, inv, 12582912.f));
    }
#pragma unroll
    for (int q = 0; q < 2; ++q)
      out[q] = (__builtin_amdgcn_perm(t[4 * q + 1], t[4 * q], 0x0c0c0400u) |
                __builtin_amdgcn_perm(t[4 * q + 3], t[4 * q + 2], 0x04000c0cu)) ^ 0x80808080u;
  }
  return out;
}

// Four whole numbers held as code + 128: 0x6400 | byte is the fp16 number 1024
// + byte.
__device__ inline void kv8_whole(uint32_t c, f16x2& lo, f16x2& hi) {
  const f16x2 off = {(f16)1152.f, (f16)1152.f};
  lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, c, 0x04010400u)) - off;
  hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, c, 0x04030402u)) - off;
}

// The values of four codes under the scale `power`, exactly.
template <int T>
__device__ inline f16x4 kv8_values4(uint32_t c, float power) {
  f16x2 lo, hi;
  if constexpr (T == NSD_KV8_E4M3) {
    lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, power, false));
    hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, power, true));
  } else {
    kv8_whole(c, lo, hi);
    const f16x2 p = {(f16)power, (f16)power};
    lo *= p;
    hi *= p;
  }
  return f16x4{lo[0], lo[1], hi[0], hi[1]};
}
__device__ inline f16x8 kv8_join(f16x4 a, f16x4 b) { return f16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}; }
template <int T>
__device__ inline f16x8 kv8_values(u32x2 c, float power) {
  return kv8_join(kv8_values4<T>(c[0], power), kv8_values4<T>(c[1], power));
}

// The transpose of a 4 x 4 matrix of bytes, a row a register.
__device__ inline u32x4 kv8_transpose(u32x4 r) {
  const uint32_t a = __builtin_amdgcn_perm(r[1], r[0], 0x05010400u), b = __builtin_amdgcn_perm(r[1], r[0], 0x07030602u);
  const uint32_t c = __builtin_amdgcn_perm(r[3], r[2], 0x05010400u), d = __builtin_amdgcn_perm(r[3], r[2], 0x07030602u);
  return u32x4{__builtin_amdgcn_perm(c, a, 0x05040100u), __builtin_amdgcn_perm(c, a, 0x07060302u),
               __builtin_amdgcn_perm(d, b, 0x05040100u), __builtin_amdgcn_perm(d, b, 0x07060302u)};
}

// Host: whether a cache argument can be used.
inline int check_kv8_cache(const char* who, const nsd_kv8_cache* c, int layer) {
  if (c == nullptr) return fail(NSD_ERR_INVALID, "%s: null cache", who);
  if (!c->k || !c->v || !c->k_scales || !c->v_scales) return fail(NSD_ERR_INVALID, "%s: null cache buffer", who);
  if (!aligned16(c->k) || !aligned16(c->v))
    return fail(NSD_ERR_INVALID, "%s: codes must be 16-byte aligned", who);
  if (c->codes != NSD_KV8_E4M3 && c->codes != NSD_KV8_INT8)
    return fail(NSD_ERR_INVALID, "%s: codes=%d (NSD_KV8_E4M3 or NSD_KV8_INT8)", who, (int)c->codes);
  if (c->num_blocks <= 0 || c->num_layers <= 0 || c->num_kv_heads <= 0)
    return fail(NSD_ERR_INVALID, "%s: bad cache shape (layers=%d, kv_heads=%d, blocks=%lld)", who,
                (int)c->num_layers, (int)c->num_kv_heads, (long long)c->num_blocks);
  if (layer < 0 || layer >= c->num_layers)
    return fail(NSD_ERR_INVALID, "%s: layer=%d outside [0, %d)", who, layer, (int)c->num_layers);
  return NSD_OK;
}

}  // namespace
}  // namespace nsd
