// The layouts of microscaled codes and scales (include/nsd_mx.h), and their
// operand form, shared by the quantisers and the products.
#pragma once

#include "nsd_device.h"
#include "nsd_mx.h"

namespace nsd {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kMxBlock = 32;         // values under one scale
constexpr int kMxTileK = 128;        // k of a tile
constexpr int kMxTile4 = 1024;       // bytes of a tile's 4-bit codes
constexpr int kMxTile8 = 2048;       // and of its 8-bit codes
constexpr int kMxScaleTile = 256;    // scale bytes of 16 rows x 4 tiles of k
constexpr uint8_t kMxNanScale = 255;

inline __host__ __device__ int64_t mx_row_tiles(int64_t rows) { return (rows + 15) / 16; }
inline __host__ __device__ int64_t mx_k_tiles(int64_t n_in) { return (n_in + kMxTileK - 1) / kMxTileK; }

// The 32 fp16 values h as one E4M3 block: its codes, 16 a register quad, and
// its scale byte.  The largest magnitude m = f 2^p (1 <= f < 2) takes 2^(p-8) up
// to f = 1.75 = 448 / 256 and 2^(p-7) above, so no value saturates.
__device__ inline uint32_t mx8_block(const f16x8 (&h)[4], u32x4 (&out)[2]) {
  u16x8 most = __builtin_bit_cast(u16x8, h[0]) & (uint16_t)0x7fff;
#pragma unroll
  for (int q = 1; q < 4; ++q) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x8, h[q]) & (uint16_t)0x7fff);
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, (uint32_t)most[e]);
  uint32_t s = 0;
  float scale = 1.f;  // of a block of zeros, whose scale byte is 0
  if (m != 0) {
    const uint32_t f = __builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(f16, (uint16_t)m));
    s = (f >> 23) - 8 + ((f & 0x7fffffu) > 0x600000u);
    scale = __builtin_bit_cast(float, s << 23);
  }
  if (m >= 0x7c00u) {
    s = kMxNanScale;
    out[0] = out[1] = u32x4{0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu};
    return s;
  }
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const f16x2 a = {h[q / 2][q % 2 * 4], h[q / 2][q % 2 * 4 + 1]};
    const f16x2 b = {h[q / 2][q % 2 * 4 + 2], h[q / 2][q % 2 * 4 + 3]};
    s16x2 c = {0, 0};
    c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(c, a, scale, false);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(c, b, scale, true);
    out[q / 4][q % 4] = __builtin_bit_cast(uint32_t, c);
  }
  return s;
}

// v_mfma_scale_f32_16x16x128_f8f6f4 with A = E2M1, B = E4M3: lane (i = lane %
// 16, g = lane / 16) holds A[i][32g .. 32g+31] in the first four registers,
// and of B the two runs [16g .. 16g+15] and [64+16g .. 64+16g+15] of column i;
// byte BYTE of sa and sb is the scale of block g of row i and of column i.  It
// receives C[4g .. 4g+3][i].
//
// The 32 products of a block are added aligned to the largest of them, whose
// last kept place is 2^-15 of it (measured; a library product in fp16 rounds
// its inputs no finer), blocks to each other and to C in fp32.
template <int BYTE>
__device__ inline f32x4 mx_mfma(i32x4 a, i32x4 b0, i32x4 b1, f32x4 c, int sa, int sb) {
  const i32x8 av = {a[0], a[1], a[2], a[3], 0, 0, 0, 0};
  const i32x8 bv = {b0[0], b0[1], b0[2], b0[3], b1[0], b1[1], b1[2], b1[3]};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 0, BYTE, sa, BYTE, sb);
}

// v_mfma_scale_f32_32x32x64_f8f6f4 likewise: lane (i = lane % 32, g = lane / 32)
// holds A[i][32g .. 32g+31], B's runs [16g .. 16g+15] and [32+16g .. 32+16g+15]
// of column i, the scales (byte BYTE of sa and sb) of block g of row and column
// i, and receives C[8q + 4g .. 8q + 4g + 3][i] in registers 4q .. 4q+3.
template <int BYTE>
__device__ inline f32x16 mx_mfma32(i32x4 a, i32x4 b0, i32x4 b1, f32x16 c, int sa, int sb) {
  const i32x8 av = {a[0], a[1], a[2], a[3], 0, 0, 0, 0};
  const i32x8 bv = {b0[0], b0[1], b0[2], b0[3], b1[0], b1[1], b1[2], b1[3]};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, c, 4, 0, BYTE, sa, BYTE, sb);
}

// Activations to MXFP8 (arguments checked by the caller); in nsd_mx.hip.
int mxfp8_quantize(const void* x, int64_t n_rows, int64_t n_in, void* codes, void* scales, void* stream);

}  // namespace nsd
