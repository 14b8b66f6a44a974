// Products of microscaled weights (MXFP4) and activations (MXFP8) for gfx950:
// y[r][n] = sum_k X[r][k] W[n][k], and the up/gate pair with its SiLU-and-mul.
#include <algorithm>

#include "nsd_mx_device.h"

namespace nsd {
namespace {

// Rows and columns of one call, and values of its output: the kernels count
// tiles and a tile's scale bytes in 32 bits.
constexpr int64_t kMaxMxRows = 1 << 21, kMaxMxColumns = 1 << 27, kMaxMxOut = (int64_t)1 << 40;
constexpr int64_t kMaxMxIn = 1 << 20;  // and a row tile's bytes

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

// ---- decode and verify batches -----------------------------------------------

// A buffer whose loads past `bytes` give zeros: the streams below run ahead of
// their range without a branch, so the loop's waits stay exact.
__device__ inline __amdgpu_buffer_rsrc_t mx_buffer(const void* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00027000);
}
template <bool NT>
__device__ inline i32x4 mx_load16(__amdgpu_buffer_rsrc_t r, int off) {
  return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, NT ? 2 : 0));
}

constexpr int kMxWaves = 4;             // of a workgroup
constexpr int kMxNowhere = 0x40000000;  // an offset past every buffer's end
constexpr int kMxFp16Tiles = 2;         // row tiles of the fp16 form

// MT row tiles by JW column tiles a workgroup (gated: the first half up tiles,
// then their gate tiles).  Its four waves split k: each streams its range's
// weight and x tiles straight into registers, two steps ahead, and multiplies
// all MT x JW pairs, so no wave loads what another one has and no step waits
// for another wave.  The sums meet in LDS at the end, added in wave order.
// FP16: x as it is, cut into blocks between load and product.  NT: the weight
// past the caches.
template <int MT, int JW, bool GATED>
struct MxStream {
  static constexpr int P = GATED ? JW / 2 : JW, PER = GATED ? 2 : 1;  // column tiles of y, sums of one
  static constexpr int YT = P * MT;
  static constexpr int kLds = YT * (kMxWaves - 1) * PER * 1024;
  static_assert(P * PER == JW && kLds <= 160 * 1024);
};

template <int MT, int JW, bool GATED, bool FP16, bool NT>
__global__ void __launch_bounds__(kMxWaves* kWave, 1) mx_stream_kernel(MxArgs a) {
  using S = MxStream<MT, JW, GATED>;
  constexpr int P = S::P, D = 2;
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int out_tiles = (a.n + 15) / 16;
  const int groups = (out_tiles + P - 1) / P;
  const int group = blockIdx.x % groups, split = blockIdx.x / groups;
  const int rt0 = blockIdx.y * MT;
  const int parts = a.splits * kMxWaves, part = split * kMxWaves + wave;
  // a wave's steps [t0, t1), in whole fours (a scale word's tiles of k) where
  // they come out even; ta: the four that t0 lies in, whose other steps are
  // loaded and not multiplied
  const int kgs = (a.T + 3) / 4;
  const bool fours = kgs % parts == 0 || kgs >= 4 * parts;
  const int units = fours ? kgs : a.T, per = fours ? 4 : 1;
  const int t0 = (int)((int64_t)part * units / parts) * per;
  const int t1 = min((int)((int64_t)(part + 1) * units / parts) * per, a.T);
  const int ta = t0 & ~3;
  [[maybe_unused]] const int k_end = min(t1 * kMxTileK, a.n_in);

  __amdgpu_buffer_rsrc_t wb[JW], wsb[JW], xb[MT], xsb[MT];
#pragma unroll
  for (int j = 0; j < JW; ++j) {
    int tile = min(group * P + j % P, out_tiles - 1);
    if (GATED && j >= P) tile += out_tiles;
    wb[j] = mx_buffer(a.wc + ((int64_t)tile * a.T + ta) * 64, (t1 - ta) * kMxTile4);
    wsb[j] = mx_buffer(a.ws + (int64_t)tile * 64, ((kgs - 1) * a.w_tiles + 1) * kMxScaleTile);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int tile = min(rt0 + i, a.row_tiles - 1);
    if constexpr (FP16) {  // rows past the last: zeros
      xb[i] = mx_buffer(a.x + (int64_t)tile * 16 * a.n_in, min(a.rows - tile * 16, 16) * a.n_in * 2);
    } else {
      xb[i] = mx_buffer(a.xc + ((int64_t)tile * a.T + ta) * 128, (t1 - ta) * kMxTile8);
      xsb[i] = mx_buffer(a.xs + (int64_t)tile * 64, ((kgs - 1) * a.row_tiles + 1) * kMxScaleTile);
    }
  }
  f32x4 acc[JW][MT];
#pragma unroll
  for (int j = 0; j < JW; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};

  constexpr int XV = FP16 ? 4 : 2;
  i32x4 w[D][JW], x[D][MT][XV];
  int sw[2][JW], sx[2][MT];  // scales of this four tiles of k, and of the next
  auto load = [&](int u, int t) __attribute__((always_inline)) {
    const int wo = (t - ta) * kMxTile4 + lane * 16, xo = (t - ta) * kMxTile8 + lane * 16;
#pragma unroll
    for (int j = 0; j < JW; ++j) w[u][j] = mx_load16<NT>(wb[j], wo);
    if constexpr (FP16) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // the runs of 16 k at 16 lg and 64 + 16 lg; past the row or the range: zeros
        const int k = t * kMxTileK + h * 64 + lg * 16;
        const int off = k < k_end ? (li * a.n_in + k) * 2 : kMxNowhere;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          x[u][i][2 * h] = mx_load16<false>(xb[i], off);
          x[u][i][2 * h + 1] = mx_load16<false>(xb[i], off + 16);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        x[u][i][0] = mx_load16<false>(xb[i], xo);
        x[u][i][1] = mx_load16<false>(xb[i], xo + 1024);
      }
    }
  };
  auto load_scales = [&](int u, int kg) __attribute__((always_inline)) {
    const int wo = kg * a.w_tiles * kMxScaleTile + lane * 4, xo = kg * a.row_tiles * kMxScaleTile + lane * 4;
#pragma unroll
    for (int j = 0; j < JW; ++j) sw[u][j] = __builtin_amdgcn_raw_buffer_load_b32(wsb[j], wo, 0, 0);
    if constexpr (!FP16) {
#pragma unroll
      for (int i = 0; i < MT; ++i) sx[u][i] = __builtin_amdgcn_raw_buffer_load_b32(xsb[i], xo, 0, 0);
    }
  };
  load_scales(0, ta >> 2);
#pragma unroll
  for (int u = 0; u < D; ++u) load(u, ta + u);
  for (int t = ta; t < t1; t += 4) {
    load_scales(1, (t >> 2) + 1);
    static_for<4>([&](auto uc) __attribute__((always_inline)) {
      constexpr int u = decltype(uc)::value, r = u % D;
      if (t + u >= t0 && t + u < t1) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          i32x4 b0, b1;
          int sb;
          if constexpr (FP16) {
            const f16x8 h[4] = {__builtin_bit_cast(f16x8, x[r][i][0]), __builtin_bit_cast(f16x8, x[r][i][1]),
                                __builtin_bit_cast(f16x8, x[r][i][2]), __builtin_bit_cast(f16x8, x[r][i][3])};
            sb = mx8_operand(h, lane, b0, b1) << 8 * u;
          } else {
            b0 = x[r][i][0];
            b1 = x[r][i][1];
            sb = sx[0][i];
          }
#pragma unroll
          for (int j = 0; j < JW; ++j) acc[j][i] = mx_mfma<u>(w[r][j], b0, b1, acc[j][i], sw[0][j], sb);
        }
      }
      load(r, t + u + D);
    });
#pragma unroll
    for (int j = 0; j < JW; ++j) sw[0][j] = sw[1][j];
    if constexpr (!FP16) {
#pragma unroll
      for (int i = 0; i < MT; ++i) sx[0][i] = sx[1][i];
    }
  }

  // lane (li, lg) holds columns 4 lg .. 4 lg + 3 of a tile for row li
  auto store = [&](int j, int i, f32x4 v, f32x4 gate) __attribute__((always_inline)) {
    const int m = 16 * (rt0 + i) + li, n0 = 16 * (group * P + j) + 4 * lg;
    if (m >= a.rows || n0 >= a.n) return;
    if constexpr (GATED) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] *= gate[e] / (1.f + expf(-gate[e]));
    }
    if (!GATED && a.splits > 1) {  // n a multiple of 8
      *reinterpret_cast<f32x4*>(a.part + ((int64_t)split * a.rows + m) * a.n + n0) = v;
      return;
    }
    f16* y = a.y + (int64_t)m * a.n + n0;
    const f16x4 h = {(f16)v[0], (f16)v[1], (f16)v[2], (f16)v[3]};
    if (a.n % 4 == 0) {
      *reinterpret_cast<f16x4*>(y) = h;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n0 + e < a.n) y[e] = h[e];
    }
  };
  // y tile q is wave q % 4's to finish: it gets the others' sums through LDS
  f32x4* red = reinterpret_cast<f32x4*>(lds_raw) + lane;
  static_for<S::YT>([&](auto qc) __attribute__((always_inline)) {
    constexpr int q = decltype(qc)::value, owner = q % kMxWaves;
    if (wave != owner) {
      f32x4* at = red + (q * (kMxWaves - 1) + wave - (wave > owner)) * S::PER * kWave;
      at[0] = acc[q / MT][q % MT];
      if constexpr (GATED) at[kWave] = acc[q / MT + P][q % MT];
    }
  });
  __syncthreads();
  static_for<S::YT>([&](auto qc) __attribute__((always_inline)) {
    constexpr int q = decltype(qc)::value, owner = q % kMxWaves;
    if (wave == owner) {
      auto sum = [&](int per, f32x4 mine) __attribute__((always_inline)) {
        f32x4 v;
        static_for<kMxWaves>([&](auto oc) __attribute__((always_inline)) {
          constexpr int o = decltype(oc)::value;
          f32x4 part = mine;
          if constexpr (o != owner)
            part = red[((q * (kMxWaves - 1) + o - (o > owner ? 1 : 0)) * S::PER + per) * kWave];
          if constexpr (o == 0) v = part;
          else v += part;
        });
        return v;
      };
      const f32x4 v = sum(0, acc[q / MT][q % MT]);
      f32x4 gate = v;
      if constexpr (GATED) gate = sum(1, acc[q / MT + P][q % MT]);
      store(q / MT, q % MT, v, gate);
    }
  });
}

// ---- prompts ---------------------------------------------------------------

template <int N>
__device__ inline void mx_wait() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// 16 bytes a lane from base + 16 lane to LDS.
__device__ inline void mx_dma(uint32_t lds_addr, const char* base, uint32_t offset) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(lds_addr), "v"(offset), "s"(base)
               : "memory", "m0");
}

template <int WR_, int WC_, int FR_, int FC_, bool GATED_>
struct MxTile {
  static constexpr int WR = WR_, WC = WC_, FR = FR_, FC = FC_;  // waves and 32-wide fragments a wave, over rows and columns
  static constexpr bool GATED = GATED_;
  static constexpr int NW = WR * WC, XT = WR * FR * 2, WT = WC * FC * 2;  // 16-row tiles of x and of the weight
  static constexpr int TM = XT * 16, TN = WT * 16, OUT = GATED ? TN / 2 : TN;
  static constexpr int XI = 2 * XT / NW, WI = WT / NW;  // loads a wave of a step's codes, 1 KB each
  static constexpr int R = 3, kStep = XT * kMxTile8 + WT * kMxTile4, kScales = (XT + WT) * kMxScaleTile;
  static constexpr int kLds = R * kStep + 2 * kScales;
  static_assert(XI * NW == 2 * XT && WI * NW == WT && (XT + WT) / 4 == NW && XT % 4 == 0 && kLds <= 160 * 1024);
};

template <class S>
__global__ void __launch_bounds__(S::NW* kWave) mx_tile_kernel(MxArgs a, int m_tiles, int n_tiles) {
  constexpr int FR = S::FR, FC = S::FC, NW = S::NW, XT = S::XT, WT = S::WT;
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  lds_char* ring = (lds_char*)lds_raw;
  lds_char* scales = ring + S::R * S::kStep;
  const int lane = threadIdx.x & 63, l32 = lane & 31, lg = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wave / S::WC, wc = wave % S::WC;
  // workgroup i runs on XCD i % 8: each XCD a contiguous run of tiles, in bands
  // of eight row tiles
  const int total = m_tiles * n_tiles;
  int id = blockIdx.x;
  {
    const int q = total / kXcds, r = total % kXcds, xcd = id % kXcds, at = id / kXcds;
    id = xcd * q + min(xcd, r) + at;
  }
  constexpr int kBand = 8;
  const int band = id / (kBand * n_tiles), rows_in = min(kBand, m_tiles - band * kBand);
  const int in_band = id - band * kBand * n_tiles;
  const int bm = band * kBand + in_band % rows_in, bn = in_band / rows_in;
  const int T = a.T, out_tiles = (a.n + 15) / 16;

  // this wave's loads of a step: chunks i NW + wave of x (two a tile) and of the weight
  auto w_tile = [&](int j) {
    if constexpr (!S::GATED) return min(bn * WT + j, out_tiles - 1);
    constexpr int H = FC / 2;
    const int c = j / (2 * FC), f = j / 2 % FC;
    const int out = min(bn * (WT / 2) + (c * H + f % H) * 2 + j % 2, out_tiles - 1);
    return f < H ? out : out + out_tiles;
  };
  const char* xsrc[S::XI];
  const char* wsrc[S::WI];
#pragma unroll
  for (int i = 0; i < S::XI; ++i) {
    const int q = i * NW + wave, tile = min(bm * XT + q / 2, a.row_tiles - 1);
    xsrc[i] = reinterpret_cast<const char*>(a.xc) + (int64_t)tile * T * kMxTile8 + q % 2 * 1024;
  }
#pragma unroll
  for (int i = 0; i < S::WI; ++i)
    wsrc[i] = reinterpret_cast<const char*>(a.wc) + (int64_t)w_tile(i * NW + wave) * T * kMxTile4;
  // scales of four steps: this wave's 1 KB is four tiles of x or of the weight
  const bool sx = wave < XT / 4;
  const int s_tile = sx ? min(bm * XT + wave * 4 + (lane >> 4), a.row_tiles - 1)
                        : w_tile((wave - XT / 4) * 4 + (lane >> 4));
  const char* ssrc = reinterpret_cast<const char*>(sx ? a.xs : a.ws);
  const int64_t s_stride = (int64_t)(sx ? a.row_tiles : a.w_tiles) * kMxScaleTile;
  const uint32_t s_off = (uint32_t)s_tile * kMxScaleTile + (lane & 15) * 16;

  auto issue = [&](int t, int slot, auto with_scales) __attribute__((always_inline)) {
    const uint32_t base = (uint32_t)(uintptr_t)(ring + slot * S::kStep);
#pragma unroll
    for (int i = 0; i < S::XI; ++i) mx_dma(base + (i * NW + wave) * 1024, xsrc[i] + (int64_t)t * kMxTile8, lane * 16);
#pragma unroll
    for (int i = 0; i < S::WI; ++i)
      mx_dma(base + XT * kMxTile8 + (i * NW + wave) * 1024, wsrc[i] + (int64_t)t * kMxTile4, lane * 16);
    if constexpr (decltype(with_scales)::value)
      mx_dma((uint32_t)(uintptr_t)(scales + (t >> 2 & 1) * S::kScales + wave * 1024), ssrc + (t >> 2) * s_stride, s_off);
  };

  f32x16 acc[FC][FR];
#pragma unroll
  for (int j = 0; j < FC; ++j)
#pragma unroll
    for (int i = 0; i < FR; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[j][i][e] = 0.f;
  uint32_t sw[FC][2], sxv[FR][2];  // scales of the wave's fragments, blocks lg and 2 + lg, four steps a word
  // lane's place in a fragment: its row's 16-byte run in tile l32 / 16
  const int row16 = (l32 & 15) * 16;
  const int x_at = (l32 >> 4) * kMxTile8 + lg * 256 + row16, w_at = (l32 >> 4) * kMxTile4 + lg * 256 + row16;
  const int s_at = (l32 >> 4) * kMxScaleTile + lg * 64 + (l32 & 15) * 4;

  issue(0, 0, std::true_type{});
  if (T > 1) issue(1, 1, std::false_type{});
  int slot = 0, slot2 = 2;
  for (int t0 = 0; t0 < T; t0 += 4) {
    static_for<4>([&](auto uc) __attribute__((always_inline)) {
      constexpr int u = decltype(uc)::value;
      const int t = t0 + u;
      if (t >= T) return;
      // step t has landed: all but this wave's loads of step t + 1; then
      // everybody's, and everybody is done with step t - 1
      if (t + 1 < T) mx_wait<S::XI + S::WI + (u == 3 ? 1 : 0)>();
      else mx_wait<0>();
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (t + 2 < T) issue(t + 2, slot2, std::bool_constant<u == 2>{});
      const lds_char* xs = ring + slot * S::kStep + wr * FR * 2 * kMxTile8 + x_at;
      const lds_char* wsl = ring + slot * S::kStep + XT * kMxTile8 + wc * FC * 2 * kMxTile4 + w_at;
      slot = slot == 2 ? 0 : slot + 1;
      slot2 = slot2 == 2 ? 0 : slot2 + 1;
      if constexpr (u == 0) {
        const lds_char* sc = scales + (t >> 2 & 1) * S::kScales + s_at;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
          for (int i = 0; i < FR; ++i)
            sxv[i][q] = *(const __attribute__((address_space(3))) uint32_t*)(sc + (wr * FR + i) * 2 * kMxScaleTile + q * 128);
#pragma unroll
          for (int j = 0; j < FC; ++j)
            sw[j][q] = *(const __attribute__((address_space(3))) uint32_t*)(sc + (XT + (wc * FC + j) * 2) * kMxScaleTile + q * 128);
        }
      }
#pragma unroll
      for (int q = 0; q < 2; ++q) {  // 64 k each
        i32x4 x[FR][2], w[FC];
#pragma unroll
        for (int j = 0; j < FC; ++j)
          w[j] = *(const __attribute__((address_space(3))) i32x4*)(wsl + j * 2 * kMxTile4 + q * 512);
#pragma unroll
        for (int i = 0; i < FR; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            x[i][h] = *(const __attribute__((address_space(3))) i32x4*)(xs + i * 2 * kMxTile8 + q * 1024 + h * 512);
#pragma unroll
        for (int i = 0; i < FR; ++i)
#pragma unroll
          for (int j = 0; j < FC; ++j)
            acc[j][i] = mx_mfma32<u>(w[j], x[i][0], x[i][1], acc[j][i], sw[j][q], sxv[i][q]);
      }
    });
  }

  // lane (l32, lg): columns 8 q + 4 lg .. + 3 of a fragment, row l32
  constexpr int H = S::GATED ? FC / 2 : FC;
#pragma unroll
  for (int i = 0; i < FR; ++i) {
    const int m = bm * S::TM + (wr * FR + i) * 32 + l32;
#pragma unroll
    for (int j = 0; j < H; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n0 = bn * S::OUT + (wc * H + j) * 32 + 8 * q + 4 * lg;
        if (m >= a.rows || n0 >= a.n) continue;
        f16x4 h;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = acc[j][i][4 * q + e];
          if constexpr (S::GATED) {
            const float g = acc[j + H][i][4 * q + e];
            v *= g / (1.f + expf(-g));
          }
          h[e] = (f16)v;
        }
        f16* y = a.y + (int64_t)m * a.n + n0;
        if (a.n % 4 == 0) {
          *reinterpret_cast<f16x4*>(y) = h;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n0 + e < a.n) y[e] = h[e];
        }
      }
  }
}

// Raises a kernel's dynamic-LDS limit once per process.
template <auto Kernel, int kLds>
int allow_mx_lds() {
  static const hipError_t attr =
      hipFuncSetAttribute(reinterpret_cast<const void*>(Kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
  return attr == hipSuccess ? NSD_OK : fail(NSD_ERR_HIP, "mxfp4: LDS attribute: %s", hipGetErrorString(attr));
}

struct MxConfig {
  bool tile = false;  // mx_tile_kernel, else mx_stream_kernel with
  int mt = 1, jw = 1, splits = 1;
  bool fp16 = false;  // reads x as it is
  bool nt = false;    // the weight past the caches
};

// Column tiles a workgroup, splits of k over workgroups and the form of x for
// the stream kernel: the cheapest by a model of its time in ns.
//   - A compute unit takes in weight and x together, however they mix, a KB in
//     21 ns where two workgroups share it or it has one to run, in 28 where
//     one's registers leave no room for another; all of them take in 6.1 TB/s
//     of weight at most.
//   - A workgroup's end, its sums through LDS, takes 50 ns a tile.
//   - Splits cost a pass that adds them: 2.5 us and their bytes.
//   - x as fp16 is twice the bytes to every workgroup, and saves the pass that
//     cuts it into blocks, 4 us with its launch.
MxConfig choose_stream(int64_t n_rows, int64_t n, int64_t T, bool gated, bool quantised, int cus) {
  MxConfig best;
  const int64_t row_tiles = mx_row_tiles(n_rows), chunks = (row_tiles + 7) / 8;
  const int mt = (int)((row_tiles + chunks - 1) / chunks);
  const int64_t out_tiles = (n + 15) / 16;
  double least = 1e300;
  for (int fp16 = 0; fp16 <= (!quantised && row_tiles <= kMxFp16Tiles ? 1 : 0); ++fp16)
    for (int jw : {1, 2, 3, 4, 6}) {
      if (gated && jw % 2) continue;
      const int p = gated ? jw / 2 : jw;
      const int64_t groups = (out_tiles + p - 1) / p * chunks;
      const bool two = 4 * jw * mt + (fp16 ? 34 : 18) * mt + 11 * jw + 12 <= 252;
      for (int splits : {1, 2, 3, 4, 6, 8}) {
        // a wave has a step at least; sum_partials takes rows of whole vectors
        if (splits > 1 && (gated || n % 8 || T < kMxWaves * splits)) break;
        const int64_t wgs = groups * splits;
        const double rounds = wgs <= 2 * cus ? (double)((wgs + cus - 1) / cus) : (double)wgs / cus + 0.5;
        const double steps = (double)((T + splits - 1) / splits);
        // rows of x that exist: the others of a tile are not fetched as fp16
        const double x_kb = fp16 ? n_rows * 0.25 : 2.0 * mt;
        double t = std::max(rounds * steps * (jw + x_kb) * (wgs > cus && !two ? 28.0 : 21.0),
                            (double)out_tiles * (gated ? 2 : 1) * T * chunks * kMxTile4 / 6100.0) +
                   rounds * jw * mt * 50.0;
        if (splits > 1) t += 2500.0 + (double)splits * n_rows * n * 8 / 5000.0;
        if (!fp16 && !quantised) t += 4000.0;
        if (t < least) {
          least = t;
          best.mt = mt;
          best.jw = jw;
          best.splits = splits;
          best.fp16 = fp16 != 0;
        }
      }
    }
  // A weight that the 256 MB last-level cache cannot keep from call to call
  // streams faster past it: 330 MB, 16 rows 64.9 -> 59.7 us; one that it keeps
  // (13 to 53 MB, called again and again) slower, 3.7 -> 5.5 and 15.1 -> 16.9,
  // and neither way among other weights.
  best.nt = (double)out_tiles * (gated ? 2 : 1) * T * kMxTile4 > 192e6;
  return best;
}

MxConfig choose_mx(int64_t n_rows, int64_t n, int64_t T, bool gated, bool quantised, int cus) {
  if (n_rows <= 128) return choose_stream(n_rows, n, T, gated, quantised, cus);
  MxConfig c;
  c.tile = true;
  return c;
}

template <class S>
int launch_mx_tile(const MxArgs& a, hipStream_t st) {
  if (int rc = allow_mx_lds<&mx_tile_kernel<S>, S::kLds>()) return rc;
  const int m_tiles = (a.rows + S::TM - 1) / S::TM, n_tiles = (a.n + S::OUT - 1) / S::OUT;
  hipLaunchKernelGGL(mx_tile_kernel<S>, dim3((unsigned)m_tiles * n_tiles), dim3(S::NW * kWave), S::kLds, st, a, m_tiles,
                     n_tiles);
  return launch_status(S::GATED ? "mxfp4_up_gate_silu_and_mul" : "mxfp4_linear");
}

template <int MT, int JW, bool GATED, bool FP16, bool NT>
int launch_mx_stream(const MxArgs& a, hipStream_t st) {
  using S = MxStream<MT, JW, GATED>;
  if (int rc = allow_mx_lds<&mx_stream_kernel<MT, JW, GATED, FP16, NT>, S::kLds>()) return rc;
  const int groups = ((a.n + 15) / 16 + S::P - 1) / S::P;
  hipLaunchKernelGGL((mx_stream_kernel<MT, JW, GATED, FP16, NT>), dim3(groups * a.splits, (a.row_tiles + MT - 1) / MT),
                     dim3(kMxWaves * kWave), S::kLds, st, a);
  return launch_status(GATED ? "mxfp4_up_gate_silu_and_mul" : "mxfp4_linear");
}
template <int MT, int JW, bool GATED>
int launch_mx_stream(const MxArgs& a, const MxConfig& c, hipStream_t st) {
  if constexpr (MT <= kMxFp16Tiles)
    if (c.fp16)
      return c.nt ? launch_mx_stream<MT, JW, GATED, true, true>(a, st) : launch_mx_stream<MT, JW, GATED, true, false>(a, st);
  return c.nt ? launch_mx_stream<MT, JW, GATED, false, true>(a, st) : launch_mx_stream<MT, JW, GATED, false, false>(a, st);
}

template <bool GATED, int... I>
int launch_mx_rows(std::integer_sequence<int, I...>, const MxArgs& a, const MxConfig& c, hipStream_t st) {
  int rc = NSD_ERR_UNSUPPORTED;
  auto with = [&](auto mt) {
    constexpr int MT = decltype(mt)::value;
    if constexpr (!GATED) {
      if (c.jw == 1) return launch_mx_stream<MT, 1, GATED>(a, c, st);
      if (c.jw == 3) return launch_mx_stream<MT, 3, GATED>(a, c, st);
    }
    if (c.jw == 2) return launch_mx_stream<MT, 2, GATED>(a, c, st);
    if (c.jw == 4) return launch_mx_stream<MT, 4, GATED>(a, c, st);
    return launch_mx_stream<MT, 6, GATED>(a, c, st);
  };
  ((c.mt == I + 1 ? (rc = with(std::integral_constant<int, I + 1>{}), 0) : 0), ...);
  return rc;
}

template <bool GATED>
int launch_mx(const MxArgs& a, const MxConfig& c, hipStream_t st) {
  if (!c.tile) return launch_mx_rows<GATED>(std::make_integer_sequence<int, 8>{}, a, c, st);
  const int64_t big = (int64_t)((a.rows + 255) / 256) * ((a.n + (GATED ? 127 : 255)) / (GATED ? 128 : 256));
  if (big >= 200) return launch_mx_tile<MxTile<4, 2, 2, 4, GATED>>(a, st);
  return launch_mx_tile<MxTile<2, 2, 2, 2, GATED>>(a, st);
}

int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

int check_product(const char* who, int64_t n_rows, int64_t n, int64_t n_in) {
  int64_t c, s;
  if (n_rows < 0 || n < 1 || n > kMaxMxColumns || n_rows > kMaxMxRows || n_rows * n > kMaxMxOut)
    return fail(NSD_ERR_UNSUPPORTED, "%s: n_rows=%lld, n_out=%lld", who, (long long)n_rows, (long long)n);
  if (n_in > kMaxMxIn) return fail(NSD_ERR_UNSUPPORTED, "%s: n_in=%lld > %lld", who, (long long)n_in, (long long)kMaxMxIn);
  for (auto [bits, rows] : {std::pair<int, int64_t>{4, n}, {8, n_rows}}) {
    if (int rc = nsd_mx_bytes(bits, rows, n_in, &c, &s)) return rc;
    if (s > INT32_MAX) return fail(NSD_ERR_UNSUPPORTED, "%s: %lld bytes of scales", who, (long long)s);
  }
  return NSD_OK;
}

// The workspace: the rows' codes and scales, when x is fp16, then the partials.
struct MxWorkspace {
  int64_t codes = 0, scales = 0, partials = 0;
  int64_t total() const { return align256(codes) + align256(scales) + partials; }
};
MxWorkspace mx_workspace(int64_t n_rows, int64_t n, int64_t n_in, bool quantised, const MxConfig& c) {
  MxWorkspace w;
  if (!quantised && !c.fp16) (void)nsd_mx_bytes(8, n_rows, n_in, &w.codes, &w.scales);
  if (c.splits > 1) w.partials = c.splits * n_rows * n * (int64_t)sizeof(float);
  return w;
}

template <bool GATED>
int product(const char* who, const void* x, const void* x_codes, const void* x_scales, const void* w_codes,
            const void* w_scales, void* y, int64_t n_rows, int64_t n, int64_t n_in, void* workspace,
            int64_t workspace_bytes, void* stream) {
  if (int rc = check_product(who, n_rows, GATED ? 2 * n : n, n_in)) return rc;
  if (GATED && n % 16) return fail(NSD_ERR_UNSUPPORTED, "%s: inter=%lld (a multiple of 16)", who, (long long)n);
  if (n_rows == 0) return NSD_OK;
  if ((!x && (!x_codes || !x_scales)) || !w_codes || !w_scales || !y)
    return fail(NSD_ERR_INVALID, "%s: null pointer", who);
  for (const void* p : {x, x_codes, x_scales, w_codes, w_scales, (const void*)y, (const void*)workspace})
    if (!aligned16(p)) return fail(NSD_ERR_UNSUPPORTED, "%s: pointers must be 16-byte aligned", who);
  int cus = 0;
  if (int rc = device_cus(&cus)) return rc;
  const int64_t T = mx_k_tiles(n_in);
  const MxConfig c = choose_mx(n_rows, n, T, GATED, x == nullptr, cus);
  const MxWorkspace need = mx_workspace(n_rows, n, n_in, x == nullptr, c);
  if (workspace_bytes < need.total() || (need.total() > 0 && !workspace))
    return fail(NSD_ERR_WORKSPACE, "%s: workspace of %lld bytes, %lld needed", who, (long long)workspace_bytes,
                (long long)need.total());
  char* ws = static_cast<char*>(workspace);
  if (x && !c.fp16) {
    void *codes = ws, *scales = ws + align256(need.codes);
    if (int rc = mxfp8_quantize(x, n_rows, n_in, codes, scales, stream)) return rc;
    x_codes = codes;
    x_scales = scales;
  }
  MxArgs a{};
  a.x = static_cast<const f16*>(x);
  a.n_in = (int)n_in;
  a.xc = static_cast<const u32x4*>(x_codes);
  a.xs = static_cast<const uint32_t*>(x_scales);
  a.wc = static_cast<const u32x4*>(w_codes);
  a.ws = static_cast<const uint32_t*>(w_scales);
  a.y = static_cast<f16*>(y);
  a.part = reinterpret_cast<float*>(ws + align256(need.codes) + align256(need.scales));
  a.rows = (int)n_rows;
  a.n = (int)n;
  a.T = (int)T;
  a.row_tiles = (int)mx_row_tiles(n_rows);
  a.w_tiles = (int)mx_row_tiles(GATED ? 2 * n : n);
  a.splits = c.splits;
  if (int rc = launch_mx<GATED>(a, c, as_stream(stream))) return rc;
  if (c.splits > 1) return nsd_sum_partials(a.part, c.splits, y, n_rows, n, stream);
  return NSD_OK;
}

}  // namespace
}  // namespace nsd

using namespace nsd;

extern "C" int nsd_mx_workspace(int64_t n_rows, int64_t n_out, int64_t n_in, int gated, int quantised,
                                int64_t* bytes) {
  if (!bytes) return fail(NSD_ERR_INVALID, "mx_workspace: null output");
  if (int rc = check_product("mx_workspace", n_rows, n_out, n_in)) return rc;
  int cus = 0;
  if (int rc = device_cus(&cus)) return rc;
  const int64_t n = gated ? n_out / 2 : n_out;
  *bytes = mx_workspace(n_rows, n, n_in, quantised != 0, choose_mx(n_rows, n, mx_k_tiles(n_in), gated != 0, quantised != 0, cus)).total();
  return NSD_OK;
}

extern "C" int nsd_mxfp4_linear(const void* x, const void* x_codes, const void* x_scales, const void* w_codes,
                                const void* w_scales, void* y, int64_t n_rows, int64_t n_out, int64_t n_in,
                                void* workspace, int64_t workspace_bytes, void* stream) {
  return product<false>("mxfp4_linear", x, x_codes, x_scales, w_codes, w_scales, y, n_rows, n_out, n_in, workspace,
                        workspace_bytes, stream);
}

extern "C" int nsd_mxfp4_up_gate_silu_and_mul(const void* x, const void* x_codes, const void* x_scales,
                                              const void* w_codes, const void* w_scales, void* y, int64_t n_rows,
                                              int64_t inter, int64_t n_in, void* workspace, int64_t workspace_bytes,
                                              void* stream) {
  return product<true>("mxfp4_up_gate_silu_and_mul", x, x_codes, x_scales, w_codes, w_scales, y, n_rows, inter, n_in,
                       workspace, workspace_bytes, stream);
}
