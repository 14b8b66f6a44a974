// The layouts of microscaled codes and scales (include/nsd_mx.h), and their
// operand form, shared by the quantisers and the products.
#pragma once

#include <atomic>

#include "nsd_device.h"
#include "nsd_mx.h"
#include "nsd_mx_choose.h"

namespace nsd {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr uint8_t kMxNanScale = 255;

// Whether two buffers share a byte.
inline bool mx_overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  const uintptr_t p = reinterpret_cast<uintptr_t>(a), q = reinterpret_cast<uintptr_t>(b);
  return a && b && a_bytes > 0 && b_bytes > 0 && p < q + b_bytes && q < p + a_bytes;
}

// Scale byte of an E4M3 block whose largest magnitude has the fp16 bits m, and
// its power of two: m = f 2^p (1 <= f < 2) takes 2^(p-8) up to f = 1.75 = 448 /
// 256 and 2^(p-7) above, so no value saturates.  Of a block of zeros the byte
// is 0, of one with an infinity or a NaN 255 (its codes mean nothing).
__device__ inline uint32_t mx8_scale(uint32_t m, float* power) {
  const uint32_t f = __builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(f16, (uint16_t)m));
  const uint32_t s = (f >> 23) - 8 + ((f & 0x7fffffu) > 0x600000u);
  const bool plain = m != 0 && m < 0x7c00u;
  *power = plain ? __builtin_bit_cast(float, s << 23) : 1.f;
  return plain ? s : m ? kMxNanScale : 0;
}
// Eight values over 2^power as codes.
__device__ inline u32x2 mx8_codes(f16x8 h, float power) {
  u32x2 out;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    s16x2 c = {0, 0};
    c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(c, f16x2{h[4 * q], h[4 * q + 1]}, power, false);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(c, f16x2{h[4 * q + 2], h[4 * q + 3]}, power, true);
    out[q] = __builtin_bit_cast(uint32_t, c);
  }
  return out;
}
// |bits| of eight values; the largest of eight.
__device__ inline u16x8 mx_abs_bits(f16x8 h) { return __builtin_bit_cast(u16x8, h) & (uint16_t)0x7fff; }
__device__ inline uint32_t mx_largest(u16x8 v) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, (uint32_t)v[e]);
  return m;
}

// The 32 fp16 values h as one E4M3 block: its codes, 16 a register quad, and
// its scale byte.
__device__ inline uint32_t mx8_block(const f16x8 (&h)[4], u32x4 (&out)[2]) {
  u16x8 most = mx_abs_bits(h[0]);
#pragma unroll
  for (int q = 1; q < 4; ++q) most = __builtin_elementwise_max(most, mx_abs_bits(h[q]));
  float power;
  const uint32_t s = mx8_scale(mx_largest(most), &power);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const u32x2 c = mx8_codes(h[q], power);
    out[q / 2][q % 2 * 2] = s == kMxNanScale ? 0x7f7f7f7fu : c[0];
    out[q / 2][q % 2 * 2 + 1] = s == kMxNanScale ? 0x7f7f7f7fu : c[1];
  }
  return s;
}

// A lane's share of a 16 x 128 tile of fp16 rows as the MFMA's B operand: h[0],
// h[1] the run of 16 k at 16 g, h[2], h[3] the one at 64 + 16 g (g = lane /
// 16).  A block is such a run in each of two neighbouring groups, so its
// largest value needs one exchange (of rows of 16 lanes); the first halves hold
// the blocks 0, 0, 1, 1 and the second 2, 2, 3, 3, and the scale operand wants
// block g from group g: one exchange of half waves.
__device__ inline int mx8_operand(const f16x8 (&h)[4], int lane, i32x4& b0, i32x4& b1) {
  const uint32_t lo = mx_largest(__builtin_elementwise_max(mx_abs_bits(h[0]), mx_abs_bits(h[1])));
  const uint32_t hi = mx_largest(__builtin_elementwise_max(mx_abs_bits(h[2]), mx_abs_bits(h[3])));
  const uint32_t both = lo | hi << 16;
  const auto sw = __builtin_amdgcn_permlane16_swap(both, both, false, false);  // each group and its neighbour
  float p0, p1;
  const uint32_t s0 = mx8_scale(max(sw[0] & 0xffffu, sw[1] & 0xffffu), &p0);
  const uint32_t s1 = mx8_scale(max(sw[0] >> 16, sw[1] >> 16), &p1);
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const u32x2 c = mx8_codes(h[q], p0), d = mx8_codes(h[q + 2], p1);
    b0[2 * q] = (int)c[0];
    b0[2 * q + 1] = (int)c[1];
    b1[2 * q] = (int)d[0];
    b1[2 * q + 1] = (int)d[1];
  }
  const auto ss = __builtin_amdgcn_permlane32_swap(s0, s1, false, false);
  return (int)(lane & 16 ? ss[1] : ss[0]);
}

// v_mfma_scale_f32_16x16x128_f8f6f4 with A = E2M1, B = E4M3: lane (i = lane %
// 16, g = lane / 16) holds A[i][32g .. 32g+31] in the first four registers,
// and of B the two runs [16g .. 16g+15] and [64+16g .. 64+16g+15] of column i;
// byte BYTE of sa and sb is the scale of block g of row i and of column i.  It
// receives C[4g .. 4g+3][i].
//
// Eight products, of neighbours along k, are added at a time: each is cut toward
// zero 13 bits below the largest sum of two operands' exponents among them
// (measured: beside 2^8 2^2 and more, to 448 * 6, 1/8 counts and 1/16 is lost;
// the same in both instructions).  Two eights join, and they C, in fp32, off by
// less than a last place.  Together that is 2e-5 of the sums' norm where a few
// channels are far larger than the rest, of which rounding to fp16 takes 2.1e-4.
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

// g / (1 + exp(-g)) in fp32, by the instructions for 2^x and 1 / x (an ulp
// each): off by (|g| + 6) 2^-23 of the value at most, where fp16 keeps 2^-11.
// The library's expf and division take 40 instructions more, a third of the
// time of a 256 x 256 tile over 4096 k.  At g = -inf the product is NaN, as
// is -inf * 0.
__device__ inline float mx_silu(float g) {
  return g * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.44269504088896341f));
}

// What a product reads and writes.
struct MxArgs {
  const f16* x;        // x [rows][n_in], or null with
  const u32x4* xc;     // x codes [row tiles][T][128] of 16 bytes
  const uint32_t* xs;  // x scales [ceil(T / 4)][row tiles][64]
  const u32x4* wc;     // weight codes [column tiles][T][64]
  const uint32_t* ws;  // weight scales [ceil(T / 4)][column tiles][64]
  f16* y;
  float* part;  // [splits][rows][n], when splits > 1
  int rows, n;  // n: columns of y
  int n_in, T;  // T: tiles of k
  int row_tiles, w_tiles;
  int splits;
};

// Up to 128 rows a workgroup (nsd_mx_stream.h): y = x . W^T, and its gated form.
int mx_stream_linear(const MxArgs& a, const MxConfig& c, hipStream_t st);
int mx_stream_gated(const MxArgs& a, const MxConfig& c, hipStream_t st);

// Raises a kernel's dynamic-LDS limit once per device.
template <auto Kernel, int kLds>
int allow_mx_lds() {
  constexpr int kMaxDevices = 64;
  static std::atomic<bool> done[kMaxDevices];
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  const bool known = e == hipSuccess && dev >= 0 && dev < kMaxDevices;
  if (known && done[dev].load(std::memory_order_relaxed)) return NSD_OK;
  if (e == hipSuccess)
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(Kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
  if (e != hipSuccess) return fail(NSD_ERR_HIP, "mxfp4: LDS attribute: %s", hipGetErrorString(e));
  if (known) done[dev].store(true, std::memory_order_relaxed);
  return NSD_OK;
}

// Activations to MXFP8 (arguments checked by the caller); in nsd_mx.hip.
int mxfp8_quantize(const void* x, int64_t n_rows, int64_t n_in, void* codes, void* scales, void* stream);

}  // namespace nsd
