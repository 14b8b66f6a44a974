// Microscaled (OCP MX) blocks for gfx950: the quantisers of weights (E2M1) and
// activations (E4M3), the packing of a checkpoint's codes, and the way back.
//
// A lane owns one block: row i of a 16-row tile, 32 consecutive k.  It reads
// them as they lie, takes the largest magnitude as an unsigned maximum of bit
// patterns (which puts a NaN above an infinity above every number), and from
// its exponent the scale, so no block needs another lane.  Division by a power
// of two is exact; the one rounding is the conversion's.
//
// All are bound by memory.
#include <algorithm>
#include <initializer_list>

#include "nsd_mx_device.h"

namespace nsd {
namespace {

constexpr int kMxThreads = 256;

__device__ inline float float_of_bits(uint32_t b) { return __builtin_bit_cast(float, b); }
__device__ inline uint32_t bits_of(float f) { return __builtin_bit_cast(uint32_t, f); }

// A block as it lies, and its values in fp32.
template <typename T>
struct MxRaw {
  u32x4 v[sizeof(T) * kMxBlock / 16];
  __device__ void load(const T* p) {
#pragma unroll
    for (unsigned i = 0; i < sizeof(v) / 16; ++i) v[i] = reinterpret_cast<const u32x4*>(p)[i];
  }
};
__device__ inline void values(const MxRaw<f16>& raw, float (&v)[kMxBlock]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f16x8 h = __builtin_bit_cast(f16x8, raw.v[i]);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[8 * i + e] = (float)h[e];
  }
}
__device__ inline void values(const MxRaw<uint16_t>& raw, float (&v)[kMxBlock]) {  // bf16
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t two = raw.v[i][e];
      v[8 * i + 2 * e] = float_of_bits(two << 16);
      v[8 * i + 2 * e + 1] = float_of_bits(two & 0xffff0000u);
    }
}
__device__ inline void values(const MxRaw<float>& raw, float (&v)[kMxBlock]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const f32x4 f = __builtin_bit_cast(f32x4, raw.v[i]);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[4 * i + e] = f[e];
  }
}

__device__ inline int wave_unit() { return blockIdx.x * (kMxThreads / kWave) + (threadIdx.x >> 6); }

__device__ inline uint32_t largest_bits(const float (&v)[kMxBlock]) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < kMxBlock; ++e) m = max(m, bits_of(v[e]) & 0x7fffffffu);
  return m;
}

// One wave per (row tile, four tiles of k): the loads of all four go out before
// the first is worked on, and the lane's four scale bytes leave as one word.
template <typename T>
__global__ void __launch_bounds__(kMxThreads)
mxfp4_quantize_kernel(const T* __restrict__ w, int64_t n_out, int n_in, int row_tiles, int k_tiles,
                      u32x4* __restrict__ codes, uint32_t* __restrict__ scales) {
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int groups = (k_tiles + 3) / 4;
  const int unit = wave_unit();
  if (unit >= row_tiles * groups) return;
  const int64_t tile = unit / groups, row = tile * 16 + i;
  const int kg = unit % groups;
  // a block that does not exist (a row or run of k past the end) is zeros: the
  // first block of the weight is read in its place
  MxRaw<T> raw[4];
  bool live[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int k = (4 * kg + t) * kMxTileK + g * kMxBlock;
    live[t] = row < n_out && k < n_in;
    raw[t].load(w + (live[t] ? row * n_in + k : 0));
  }
  uint32_t word = 0;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    float v[kMxBlock];
    values(raw[t], v);
    uint32_t m = largest_bits(v);
    if (!live[t]) m = 0;
    // floor(log2 m) - 2; below 2^-125 (the field of subnormals is 0) the
    // smallest scale.  v 2^(127 - s): exact, or far below half a code
    const uint32_t s = m >= 0x7f800000u ? kMxNanScale : max((int)(m >> 23) - 2, 0);
    const float inv = live[t] && s != kMxNanScale ? float_of_bits((254u - s) << 23) : 0.f;
    u32x4 out;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t c = 0;
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * q] * inv, v[8 * q + 1] * inv, 1.f, 0);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * q + 2] * inv, v[8 * q + 3] * inv, 1.f, 1);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * q + 4] * inv, v[8 * q + 5] * inv, 1.f, 2);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * q + 6] * inv, v[8 * q + 7] * inv, 1.f, 3);
      out[q] = live[t] && s != kMxNanScale ? c : 0;
    }
    const int kt = 4 * kg + t;
    if (kt < k_tiles) codes[(tile * k_tiles + kt) * 64 + lane] = out;
    word |= s << (8 * t);
  }
  scales[((int64_t)kg * row_tiles + tile) * 64 + lane] = word;
}

// The same cut over codes and scale bytes that exist.
__global__ void __launch_bounds__(kMxThreads)
mxfp4_pack_kernel(const u32x4* __restrict__ row_codes, const uint8_t* __restrict__ row_scales, int64_t n_out,
                  int n_in, int row_tiles, int k_tiles, u32x4* __restrict__ codes,
                  uint32_t* __restrict__ scales) {
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int groups = (k_tiles + 3) / 4, blocks = n_in / kMxBlock;
  const int unit = wave_unit();
  if (unit >= row_tiles * groups) return;
  const int64_t tile = unit / groups, row = tile * 16 + i;
  const int kg = unit % groups;
  uint32_t word = 0;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int kt = 4 * kg + t;
    if (kt >= k_tiles) break;
    const int b = kt * 4 + g;
    u32x4 out = {0, 0, 0, 0};
    uint32_t s = 0;
    if (row < n_out && b < blocks) {
      out = row_codes[row * blocks + b];
      s = row_scales[row * blocks + b];
    }
    codes[(tile * k_tiles + kt) * 64 + lane] = out;
    word |= s << (8 * t);
  }
  scales[((int64_t)kg * row_tiles + tile) * 64 + lane] = word;
}

// One lane per block, one wave per (row tile, tile of k).
__global__ void __launch_bounds__(kMxThreads)
mxfp8_quantize_kernel(const f16* __restrict__ x, int64_t n_rows, int n_in, int row_tiles, int k_tiles,
                      u32x4* __restrict__ codes, uint8_t* __restrict__ scales) {
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int unit = wave_unit();
  if (unit >= row_tiles * k_tiles) return;
  const int64_t tile = unit / k_tiles, row = tile * 16 + i;
  const int kt = unit % k_tiles, k = kt * kMxTileK + g * kMxBlock;
  u32x4 out[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
  uint32_t s = 0;
  if (row < n_rows && k < n_in) {
    const f16x8* src = reinterpret_cast<const f16x8*>(x + row * n_in + k);
    f16x8 h[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) h[q] = src[q];
    s = mx8_block(h, out);
  }
  u32x4* dst = codes + (tile * k_tiles + kt) * 128 + 2 * g * 16 + i;
  dst[0] = out[0];
  dst[16] = out[1];
  scales[((int64_t)(kt >> 2) * row_tiles + tile) * kMxScaleTile + lane * 4 + (kt & 3)] = (uint8_t)s;
}

// ---- the way back ----------------------------------------------------------

// 2^(s - 127), NaN for 255.  2^-127 is subnormal: its bits are not s << 23.
__device__ inline float scale_of(uint32_t s) {
  return float_of_bits(s == kMxNanScale ? 0x7fc00000u : s == 0 ? 0x00400000u : s << 23);
}
__device__ inline float e2m1_value(uint32_t c) {
  const uint32_t e = (c >> 1) & 3, m = c & 1;
  const float a = e ? float_of_bits(((126 + e) << 23) | (m << 22)) : 0.5f * (float)m;
  return c & 8 ? -a : a;
}
__device__ inline float e4m3_value(uint32_t c) {
  const uint32_t e = (c >> 3) & 15, m = c & 7;
  const float a = (c & 127) == 127 ? float_of_bits(0x7fc00000u)
                  : e ? float_of_bits(((120 + e) << 23) | (m << 20)) : (float)m * 0.001953125f;
  return c & 128 ? -a : a;
}

// Stores of eight values.  Non-temporal: left in the caches, the values push out
// what they were made from and are written back later all the same.  The way
// back alone: 8192 x 12288 E4M3 55 -> 47 us, 4096 x 4096 E2M1 10.8 -> 8.7, 24576 x
// 4096 41.7 -> 40.1; there and back 119 -> 92, 19 -> 17 and 99 -> 82.  A kernel
// that reads the values next loses about as much: the way back and a copy take
// 24.4 -> 24.9 us (4096 x 4096), 133 -> 124 (24576 x 4096) and 133 -> 134 (8192 x
// 12288), the way back and a product 33.5 -> 33.8, 76 -> 84 and 100 -> 101.  (The quantisers' loads the
// same way: 92 -> 120 there and back.)
template <typename T>
__device__ inline void store8(T* p, const float (&v)[8]);
template <>
__device__ inline void store8<f16>(f16* p, const float (&v)[8]) {
  f16x8 h;
#pragma unroll
  for (int e = 0; e < 8; ++e) h[e] = (f16)v[e];
  __builtin_nontemporal_store(h, reinterpret_cast<f16x8*>(p));
}
// bf16: exact, but for E4M3 codes below bf16's subnormals.
template <>
__device__ inline void store8<uint16_t>(uint16_t* p, const float (&v)[8]) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  u32x4 h;
#pragma unroll
  for (int e = 0; e < 4; ++e) h[e] = __builtin_bit_cast(uint32_t, bf16x2{(__bf16)v[2 * e], (__bf16)v[2 * e + 1]});
  __builtin_nontemporal_store(h, reinterpret_cast<u32x4*>(p));
}
template <>
__device__ inline void store8<float>(float* p, const float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 2; ++e)
    __builtin_nontemporal_store(f32x4{v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]}, reinterpret_cast<f32x4*>(p) + e);
}

// One wave per (row tile, tile of k), a lane eight values of a row at a time:
// sixteen lanes a row of the tile, so a store is whole runs of four rows.  (A
// lane a block, each store 16 of every 64 bytes: 86 us for 8192 x 12288 E4M3,
// 70 for 24576 x 4096 E2M1; so 60 and 44.)
template <int BITS, typename T>
__global__ void __launch_bounds__(kMxThreads)
mx_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t n_rows, int n_in,
                     int row_tiles, int k_tiles, T* __restrict__ out) {
  const int lane = threadIdx.x & 63, c = lane & 15;
  const int unit = wave_unit();
  if (unit >= row_tiles * k_tiles) return;
  const int64_t tile = unit / k_tiles;
  const int kt = unit % k_tiles, k = kt * kMxTileK + c * 8;
  const uint8_t* src = codes + (tile * k_tiles + kt) * (BITS == 4 ? kMxTile4 : kMxTile8);
  const uint8_t* sc = scales + ((int64_t)(kt >> 2) * row_tiles + tile) * kMxScaleTile + (kt & 3);
  u32x2 code[4];
  uint32_t s[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int i = 4 * q + (lane >> 4);  // row of the tile
    if constexpr (BITS == 4) code[q][0] = *reinterpret_cast<const uint32_t*>(src + c / 4 * 256 + i * 16 + c % 4 * 4);
    else code[q] = *reinterpret_cast<const u32x2*>(src + c / 2 * 256 + i * 16 + c % 2 * 8);
    s[q] = sc[(c / 4 * 16 + i) * 4];
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int64_t row = tile * 16 + 4 * q + (lane >> 4);
    if (row >= n_rows || k >= n_in) continue;
    const float f = scale_of(s[q]);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (BITS == 4) v[e] = e2m1_value(code[q][0] >> (4 * e)) * f;
      else v[e] = e4m3_value(code[q][e / 4] >> (8 * (e % 4))) * f;
    }
    store8(out + row * n_in + k, v);
  }
}

int check_mx(const char* who, int64_t n_rows, int64_t n_in) {
  if (n_rows < 0 || n_rows > INT32_MAX || n_in < kMxBlock || n_in % kMxBlock || n_in > INT32_MAX)
    return fail(NSD_ERR_UNSUPPORTED, "%s: %lld rows of n_in=%lld (a multiple of 32)", who, (long long)n_rows,
                (long long)n_in);
  // a launch has at most one wave per (row tile, tile of k), its lanes counted in 32 bits
  if (mx_row_tiles(n_rows) * mx_k_tiles(n_in) > (UINT32_MAX - kMxThreads) / kWave)
    return fail(NSD_ERR_UNSUPPORTED, "%s: %lld x %lld values are too many", who, (long long)n_rows, (long long)n_in);
  return NSD_OK;
}
int check_dtype(const char* who, int dtype) {
  if (dtype != NSD_DTYPE_F16 && dtype != NSD_DTYPE_BF16 && dtype != NSD_DTYPE_F32)
    return fail(NSD_ERR_UNSUPPORTED, "%s: dtype=%d", who, dtype);
  return NSD_OK;
}
int check_pointers(const char* who, std::initializer_list<const void*> ps) {
  for (const void* p : ps) {
    if (p == nullptr) return fail(NSD_ERR_INVALID, "%s: null pointer", who);
    if (!aligned16(p)) return fail(NSD_ERR_UNSUPPORTED, "%s: pointers must be 16-byte aligned", who);
  }
  return NSD_OK;
}

// Codes and scales of n_rows x n_in values apart from each other and from the
// conversion's other buffers: waves write while others read.
struct MxBuffer {
  const void* p;
  int64_t bytes;
};
int check_apart(const char* who, int bits, int64_t n_rows, int64_t n_in, const void* codes, const void* scales,
                std::initializer_list<MxBuffer> others) {
  int64_t c = 0, s = 0;
  (void)nsd_mx_bytes(bits, n_rows, n_in, &c, &s);
  bool over = mx_overlap(codes, c, scales, s);
  for (const MxBuffer& o : others) over = over || mx_overlap(codes, c, o.p, o.bytes) || mx_overlap(scales, s, o.p, o.bytes);
  return over ? fail(NSD_ERR_INVALID, "%s: the buffers overlap", who) : NSD_OK;
}
int64_t dtype_bytes(int dtype) { return dtype == NSD_DTYPE_F32 ? 4 : 2; }

unsigned wave_grid(int64_t units) { return (unsigned)((units + kMxThreads / kWave - 1) / (kMxThreads / kWave)); }

template <int BITS>
int dequantize(const char* who, const void* codes, const void* scales, int64_t n_rows, int64_t n_in, void* out,
               int dtype, void* stream) {
  if (int rc = check_mx(who, n_rows, n_in)) return rc;
  if (int rc = check_dtype(who, dtype)) return rc;
  if (n_rows == 0) return NSD_OK;
  if (int rc = check_pointers(who, {codes, scales, out})) return rc;
  if (int rc = check_apart(who, BITS, n_rows, n_in, codes, scales, {{out, n_rows * n_in * dtype_bytes(dtype)}})) return rc;
  const int64_t rt = mx_row_tiles(n_rows), kt = mx_k_tiles(n_in);
  auto go = [&](auto* p) {
    hipLaunchKernelGGL((mx_dequantize_kernel<BITS, std::remove_pointer_t<decltype(p)>>), dim3(wave_grid(rt * kt)),
                       dim3(kMxThreads), 0, as_stream(stream), static_cast<const uint8_t*>(codes),
                       static_cast<const uint8_t*>(scales), n_rows, (int)n_in, (int)rt, (int)kt, p);
  };
  if (dtype == NSD_DTYPE_F16) go(static_cast<f16*>(out));
  else if (dtype == NSD_DTYPE_BF16) go(static_cast<uint16_t*>(out));
  else go(static_cast<float*>(out));
  return launch_status(who);
}

}  // namespace

int mxfp8_quantize(const void* x, int64_t n_rows, int64_t n_in, void* codes, void* scales, void* stream) {
  const int64_t rt = mx_row_tiles(n_rows), kt = mx_k_tiles(n_in);
  hipLaunchKernelGGL(mxfp8_quantize_kernel, dim3(wave_grid(rt * kt)), dim3(kMxThreads), 0, as_stream(stream),
                     static_cast<const f16*>(x), n_rows, (int)n_in, (int)rt, (int)kt, static_cast<u32x4*>(codes),
                     static_cast<uint8_t*>(scales));
  return launch_status("mxfp8_quantize");
}

}  // namespace nsd

using namespace nsd;

extern "C" int nsd_mx_bytes(int bits, int64_t n_rows, int64_t n_in, int64_t* codes, int64_t* scales) {
  if (bits != 4 && bits != 8) return fail(NSD_ERR_INVALID, "mx_bytes: bits=%d", bits);
  if (!codes || !scales) return fail(NSD_ERR_INVALID, "mx_bytes: null output");
  if (int rc = check_mx("mx_bytes", n_rows, n_in)) return rc;
  const int64_t rt = mx_row_tiles(n_rows), kt = mx_k_tiles(n_in);
  *codes = rt * kt * (bits == 4 ? kMxTile4 : kMxTile8);
  *scales = rt * ((kt + 3) / 4) * kMxScaleTile;
  return NSD_OK;
}

extern "C" int nsd_mxfp4_quantize(const void* w, int dtype, int64_t n_out, int64_t n_in, void* codes, void* scales,
                                  void* stream) {
  if (int rc = check_mx("mxfp4_quantize", n_out, n_in)) return rc;
  if (int rc = check_dtype("mxfp4_quantize", dtype)) return rc;
  if (n_out == 0) return NSD_OK;
  if (int rc = check_pointers("mxfp4_quantize", {w, codes, scales})) return rc;
  if (int rc = check_apart("mxfp4_quantize", 4, n_out, n_in, codes, scales, {{w, n_out * n_in * dtype_bytes(dtype)}}))
    return rc;
  const int64_t rt = mx_row_tiles(n_out), kt = mx_k_tiles(n_in);
  auto go = [&](const auto* p) {
    hipLaunchKernelGGL((mxfp4_quantize_kernel<std::remove_cv_t<std::remove_pointer_t<decltype(p)>>>),
                       dim3(wave_grid(rt * ((kt + 3) / 4))), dim3(kMxThreads), 0, as_stream(stream), p, n_out, (int)n_in,
                       (int)rt, (int)kt, static_cast<u32x4*>(codes), static_cast<uint32_t*>(scales));
  };
  if (dtype == NSD_DTYPE_F16) go(static_cast<const f16*>(w));
  else if (dtype == NSD_DTYPE_BF16) go(static_cast<const uint16_t*>(w));
  else go(static_cast<const float*>(w));
  return launch_status("mxfp4_quantize");
}

extern "C" int nsd_mxfp4_pack(const void* row_codes, const void* row_scales, int64_t n_out, int64_t n_in, void* codes,
                              void* scales, void* stream) {
  if (int rc = check_mx("mxfp4_pack", n_out, n_in)) return rc;
  if (n_out == 0) return NSD_OK;
  if (!row_scales) return fail(NSD_ERR_INVALID, "mxfp4_pack: null pointer");
  if (int rc = check_pointers("mxfp4_pack", {row_codes, codes, scales})) return rc;
  if (int rc = check_apart("mxfp4_pack", 4, n_out, n_in, codes, scales,
                           {{row_codes, n_out * n_in / 2}, {row_scales, n_out * n_in / kMxBlock}}))
    return rc;
  const int64_t rt = mx_row_tiles(n_out), kt = mx_k_tiles(n_in);
  hipLaunchKernelGGL(mxfp4_pack_kernel, dim3(wave_grid(rt * ((kt + 3) / 4))), dim3(kMxThreads), 0, as_stream(stream),
                     static_cast<const u32x4*>(row_codes), static_cast<const uint8_t*>(row_scales), n_out, (int)n_in,
                     (int)rt, (int)kt, static_cast<u32x4*>(codes), static_cast<uint32_t*>(scales));
  return launch_status("mxfp4_pack");
}

extern "C" int nsd_mxfp4_dequantize(const void* codes, const void* scales, int64_t n_out, int64_t n_in, void* out,
                                    int dtype, void* stream) {
  return dequantize<4>("mxfp4_dequantize", codes, scales, n_out, n_in, out, dtype, stream);
}

extern "C" int nsd_mxfp8_quantize(const void* x, int64_t n_rows, int64_t n_in, void* codes, void* scales,
                                  void* stream) {
  if (int rc = check_mx("mxfp8_quantize", n_rows, n_in)) return rc;
  if (n_rows == 0) return NSD_OK;
  if (int rc = check_pointers("mxfp8_quantize", {x, codes, scales})) return rc;
  if (int rc = check_apart("mxfp8_quantize", 8, n_rows, n_in, codes, scales, {{x, n_rows * n_in * 2}})) return rc;
  return mxfp8_quantize(x, n_rows, n_in, codes, scales, stream);
}

extern "C" int nsd_mxfp8_dequantize(const void* codes, const void* scales, int64_t n_rows, int64_t n_in, void* out,
                                    int dtype, void* stream) {
  return dequantize<8>("mxfp8_dequantize", codes, scales, n_rows, n_in, out, dtype, stream);
}
