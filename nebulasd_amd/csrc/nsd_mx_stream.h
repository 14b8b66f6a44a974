// Products of few rows with an MXFP4 weight, up to 128 of them a workgroup: the
// stream kernel, which nsd_mx_stream_linear.hip and nsd_mx_stream_gated.hip
// compile.
#pragma once

#include "nsd_mx_device.h"

namespace nsd {
namespace {

// A buffer whose loads past `bytes` give zeros: the streams below run ahead of
// their range without a branch, so the loop's waits stay exact.
__device__ inline __amdgpu_buffer_rsrc_t mx_buffer(const void* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00027000);
}
template <bool NT>
__device__ inline i32x4 mx_load16(__amdgpu_buffer_rsrc_t r, int off) {
  return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, NT ? 2 : 0));
}

constexpr int kMxNowhere = 0x40000000;  // an offset past every buffer's end

// MT row tiles by JW column tiles a workgroup (gated: the first half up tiles,
// then their gate tiles).  Its four waves split k: each streams its range's
// weight and x tiles straight into registers, two steps ahead, and multiplies
// all MT x JW pairs, so no wave loads what another one has and no step waits
// for another wave.  The sums meet in LDS at the end, added in wave order.
// FP16: x as it is, cut into blocks between load and product.  NT: the weight
// past the caches.
//
// Bound by a fixed part and the weight's stream.  80 rows x 4096 -> 2 x 12288 (5 x
// 6 tiles, 16 KB into each compute unit a step) takes 7 us and 32 steps of 0.25
// us, 6.3 TB/s of weight out of the last-level cache: 15 us.  Among other weights
// a step is 0.38 us, 4.1 TB/s from memory, and the whole 18; while the weight
// lies in the L2, 0.14 us.  Of the 7 us 3.4 are there with one row tile, too
// (launch, the first loads); the rest are the sums through LDS and the stores,
// 140 to 200 ns a tile.  One row tile's steps take 0.23 us, 6.9 TB/s, and 0.29,
// 5.4 TB/s, among others; past the caches it streams 330 MB at 6.0 TB/s (55 us).
// Branches around the loads instead of bounds made every step wait for all of
// them (17.0 -> 19.0); eight waves, three or four steps ahead, and the x of an XCD
// read by its workgroups beforehand were no faster over the shapes.
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
      for (int e = 0; e < 4; ++e) v[e] *= mx_silu(gate[e]);
    }
    if (!GATED && a.splits > 1) {  // n a multiple of 8
      *reinterpret_cast<f32x4*>(a.part + ((int64_t)split * a.rows + m) * a.n + n0) = v;
      return;
    }
    f16* y = a.y + (int64_t)m * a.n + n0;
    const f16x4 h = {(f16)v[0], (f16)v[1], (f16)v[2], (f16)v[3]};
    typedef f16x4 __attribute__((aligned(2))) f16x4_any;  // rows of any n start where they do
    if (GATED || n0 + 4 <= a.n) {
      *reinterpret_cast<f16x4_any*>(y) = h;
    } else {
#pragma unroll
      for (int e = 0; e < 3; ++e)
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
    if (c.fp16) {
      if constexpr (mx_stream_nt(MT, JW, true))
        if (c.nt) return launch_mx_stream<MT, JW, GATED, true, true>(a, st);
      return launch_mx_stream<MT, JW, GATED, true, false>(a, st);
    }
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

}  // namespace
}  // namespace nsd
