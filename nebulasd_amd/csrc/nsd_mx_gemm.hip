// Products of microscaled weights (MXFP4) and activations (MXFP8) for gfx950:
// y[r][n] = sum_k X[r][k] W[n][k], and the up/gate pair with its SiLU-and-mul.
// Here the tile kernel for many rows and the C entries; the kernel for decode and
// verify batches is in nsd_mx_stream.h, the choice between them in
// nsd_mx_choose.h.
#include <algorithm>

#include "nsd_mx_device.h"

namespace nsd {
namespace {

// Rows and columns of one call, and values of its output: the kernels count
// tiles and a tile's scale bytes in 32 bits.
constexpr int64_t kMaxMxRows = 1 << 21, kMaxMxColumns = 1 << 27, kMaxMxOut = (int64_t)1 << 40;
constexpr int64_t kMaxMxIn = 1 << 20;  // and a row tile's bytes

typedef __attribute__((address_space(3))) i32x4 lds_i32x4;
typedef __attribute__((address_space(3))) int lds_int;

// ---- prompts ---------------------------------------------------------------

template <int N>
__device__ inline void mx_wait() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// 16 bytes a lane from base + offset to LDS.  The wait states are the ones the
// compiler would put between a write of m0, or a VALU's write of the base's
// registers, and the load; it does not look into the asm.
__device__ inline void mx_dma(uint32_t lds_addr, const char* base, uint32_t offset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(lds_addr), "v"(offset), "s"(base)
               : "memory", "m0");
}

// A workgroup computes XT row tiles by WT column tiles over its split of k, in
// steps of 128 k through a ring in LDS.  Tiles lie in memory as the operands
// want them, so a KB of a tile is one load, a fragment two contiguous reads a
// lane, and nothing is swizzled.
//
// Bound by the matrix cores at the clock that power leaves them: up/gate of 8192
// x 4096 -> 12288 takes 583 to 615 us, 2.7 to 2.8 PFLOP/s, busy 71% of the cycles
// at 1.85 GHz; the instruction on random operands in registers, nothing else
// running, does 3.7 to 4.05 (4.97 on zeros).  Tiles of 256 x 256 with one or two
// waves a SIMD, all rows in every wave (it spills) and loads that hit the L2
// alone came out between 5% slower and 5% faster.
template <int WR_, int WC_, int FR_, int FC_, int R_, bool GATED_>
struct MxTile {
  static constexpr int WR = WR_, WC = WC_, FR = FR_, FC = FC_;  // waves and 32-wide fragments a wave, over rows and columns
  static constexpr int R = R_;                                  // steps in the ring
  static constexpr bool GATED = GATED_;
  static constexpr int NW = WR * WC, XT = WR * FR * 2, WT = WC * FC * 2;  // 16-row tiles of x and of the weight
  static constexpr int TM = XT * 16, TN = WT * 16, OUT = GATED ? TN / 2 : TN;
  static constexpr bool kSplits = !GATED && TN == 128;
  static constexpr int SK = (XT + WT) / 4;  // KB of scales of four steps
  // loads a wave, 1 KB each: a step's x and weight, four steps' scales
  static constexpr int XI = 2 * XT / NW, WI = WT / NW, SI = (SK + NW - 1) / NW;
  static constexpr int kStep = XT * kMxTile8 + WT * kMxTile4, kScales = SK * 1024;
  static constexpr int kLds = R * kStep + 2 * kScales;
  static_assert(XI * NW == 2 * XT && WI * NW == WT && XT % 4 == 0 && WT % 4 == 0 && R >= 2 && kLds <= 160 * 1024);
};

template <class S>
__global__ void __launch_bounds__(S::NW* kWave, 2) mx_tile_kernel(MxArgs a, int m_tiles, int n_tiles) {
  constexpr int FR = S::FR, FC = S::FC, NW = S::NW, XT = S::XT, WT = S::WT;
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  lds_char* ring = (lds_char*)lds_raw;
  lds_char* scales = ring + S::R * S::kStep;
  const int lane = threadIdx.x & 63, l32 = lane & 31, lg = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wave / S::WC, wc = wave % S::WC;
  // workgroup i runs on XCD i % 8: each XCD a contiguous run of tiles, in bands
  // of eight row tiles
  const int total = m_tiles * n_tiles, split = blockIdx.x / total;
  int id = blockIdx.x - split * total;
  {
    const int q = total / kXcds, r = total % kXcds, xcd = id % kXcds, at = id / kXcds;
    id = xcd * q + min(xcd, r) + at;
  }
  constexpr int kBand = 8;
  const int band = id / (kBand * n_tiles), rows_in = min(kBand, m_tiles - band * kBand);
  const int in_band = id - band * kBand * n_tiles;
  const int bm = band * kBand + in_band % rows_in, bn = in_band / rows_in;
  const int out_tiles = (a.n + 15) / 16;
  // this split's steps: whole fours, so that a scale word is one split's
  const int fours = (a.T + 3) / 4, four0 = (int)((int64_t)split * fours / a.splits);
  const int T = min(4 * (int)((int64_t)(split + 1) * fours / a.splits), a.T) - 4 * four0;

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
    xsrc[i] = reinterpret_cast<const char*>(a.xc) + ((int64_t)tile * a.T + 4 * four0) * kMxTile8 + q % 2 * 1024;
  }
#pragma unroll
  for (int i = 0; i < S::WI; ++i)
    wsrc[i] = reinterpret_cast<const char*>(a.wc) + ((int64_t)w_tile(i * NW + wave) * a.T + 4 * four0) * kMxTile4;
  // scales of four steps: a KB is four tiles of x or of the weight; where they
  // do not come out even, a wave brings the last one again
  const char* ssrc[S::SI];
  int64_t s_stride[S::SI];
  uint32_t s_off[S::SI];
  int s_kb[S::SI];
#pragma unroll
  for (int i = 0; i < S::SI; ++i) {
    s_kb[i] = min(i * NW + wave, S::SK - 1);
    const bool of_x = s_kb[i] < XT / 4;
    const int tile = of_x ? min(bm * XT + s_kb[i] * 4 + (lane >> 4), a.row_tiles - 1)
                          : w_tile((s_kb[i] - XT / 4) * 4 + (lane >> 4));
    s_stride[i] = (int64_t)(of_x ? a.row_tiles : a.w_tiles) * kMxScaleTile;
    ssrc[i] = reinterpret_cast<const char*>(of_x ? a.xs : a.ws) + four0 * s_stride[i];
    s_off[i] = (uint32_t)tile * kMxScaleTile + (lane & 15) * 16;
  }

  // load i of a step: of x, of the weight, and of the scales with every fourth
  constexpr int N = S::XI + S::WI;
  auto issue = [&](auto ic, int t, int slot) __attribute__((always_inline)) {
    constexpr int i = decltype(ic)::value;
    const uint32_t base = (uint32_t)(uintptr_t)(ring + slot * S::kStep);
    if constexpr (i < S::XI)
      mx_dma(base + (i * NW + wave) * 1024, xsrc[i] + (int64_t)t * kMxTile8, lane * 16);
    else if constexpr (i < N)
      mx_dma(base + XT * kMxTile8 + ((i - S::XI) * NW + wave) * 1024, wsrc[i - S::XI] + (int64_t)t * kMxTile4, lane * 16);
    else
      mx_dma((uint32_t)(uintptr_t)(scales + (t >> 2 & 1) * S::kScales + s_kb[i - N] * 1024),
             ssrc[i - N] + (t >> 2) * s_stride[i - N], s_off[i - N]);
  };

  f32x16 acc[FC][FR];
#pragma unroll
  for (int j = 0; j < FC; ++j)
#pragma unroll
    for (int i = 0; i < FR; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[j][i][e] = 0.f;
  // lane's place in a fragment: its row's 16-byte run in tile l32 / 16
  const int row16 = (l32 & 15) * 16;
  const int x_at = (wr * FR * 2 + (l32 >> 4)) * kMxTile8 + lg * 256 + row16;
  const int w_at = XT * kMxTile8 + (wc * FC * 2 + (l32 >> 4)) * kMxTile4 + lg * 256 + row16;
  const int s_at = (l32 >> 4) * kMxScaleTile + lg * 64 + (l32 & 15) * 4;

  // A step is two halves of 64 k, each a set of fragments in registers: one is
  // multiplied while the other is read.  Scales of the wave's fragments, blocks
  // lg and 2 + lg: a word holds four steps.
  i32x4 x[2][FR][2], w[2][FC];
  int sw[FC][2], sx[FR][2], sw_next[FC][2], sx_next[FR][2];
  constexpr int M = FR * FC, F = 2 * FR + FC;  // products and reads of a half
  auto read = [&](auto qc, auto rc, int slot) __attribute__((always_inline)) {
    constexpr int q = decltype(qc)::value, r = decltype(rc)::value;
    const lds_char* step = ring + slot * S::kStep;
    if constexpr (r < 2 * FR)
      x[q][r / 2][r % 2] = *(const lds_i32x4*)(step + x_at + r / 2 * 2 * kMxTile8 + q * 1024 + r % 2 * 512);
    else
      w[q][r - 2 * FR] = *(const lds_i32x4*)(step + w_at + (r - 2 * FR) * 2 * kMxTile4 + q * 512);
  };
  auto read_scales = [&](int kg) __attribute__((always_inline)) {
    const lds_char* sc = scales + (kg & 1) * S::kScales + s_at;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
#pragma unroll
      for (int i = 0; i < FR; ++i) sx_next[i][q] = *(const lds_int*)(sc + (wr * FR + i) * 2 * kMxScaleTile + q * 128);
#pragma unroll
      for (int j = 0; j < FC; ++j)
        sw_next[j][q] = *(const lds_int*)(sc + (XT + (wc * FC + j) * 2) * kMxScaleTile + q * 128);
    }
  };
  // The products of a half in order, after(i) behind product i.  The matrix
  // pipe takes a product every 64 cycles and a wave issues in order: reads and
  // loads in a bunch, eight waves at once, would fill their queues and hold the
  // products up behind them.  Of the wide tile's waves one with a product ready
  // goes first: 597 -> 583 us for up/gate of 8192 rows (the small one's: 63 -> 64
  // for 1237 x 2080 -> 18993).
  auto multiply = [&](auto qc, auto uc, auto after) __attribute__((always_inline)) {
    constexpr int q = decltype(qc)::value, u = decltype(uc)::value;
    static_for<M>([&](auto mc) __attribute__((always_inline)) {
      constexpr int i = decltype(mc)::value / FC, j = decltype(mc)::value % FC;
      if constexpr (FC > 2) __builtin_amdgcn_s_setprio(1);
      acc[j][i] = mx_mfma32<u>(w[q][j], x[q][i][0], x[q][i][1], acc[j][i], sw[j][q], sx[i][q]);
      if constexpr (FC > 2) __builtin_amdgcn_s_setprio(0);
      after(mc);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  using Q0 = std::integral_constant<int, 0>;
  using Q1 = std::integral_constant<int, 1>;
  // reads 2 m and 2 m + 1 of a half behind product m of the other
  auto read_two = [&](auto qc, auto mc, int slot) __attribute__((always_inline)) {
    constexpr int r = 2 * decltype(mc)::value;
    if constexpr (r < F) read(qc, std::integral_constant<int, r>{}, slot);
    if constexpr (r + 1 < F) read(qc, std::integral_constant<int, r + 1>{}, slot);
  };
  static_assert(2 * M >= F);

  // steps 0 .. R - 1, then step 0 has landed
  constexpr int R = S::R;
  static_for<R>([&](auto tc) __attribute__((always_inline)) {
    constexpr int t = decltype(tc)::value;
    if (t < T) static_for<N + (t % 4 == 0 ? S::SI : 0)>([&](auto i) { issue(i, t, t); });
  });
  if (T >= R) mx_wait<(R - 1) * N>();  // R <= 4: scales with step 0 alone
  else mx_wait<0>();
  asm volatile("s_barrier" ::: "memory");
  read_scales(0);
  static_for<F>([&](auto r) { read(Q0{}, r, 0); });
  int slot = 0;
  for (int t0 = 0; t0 < T; t0 += 4) {
    static_for<4>([&](auto uc) __attribute__((always_inline)) {
      constexpr int u = decltype(uc)::value;
      const int t = t0 + u;
      if (t >= T) return;
      if constexpr (u == 0) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
          for (int i = 0; i < FR; ++i) sx[i][q] = sx_next[i][q];
#pragma unroll
          for (int j = 0; j < FC; ++j) sw[j][q] = sw_next[j][q];
        }
      }
      multiply(Q0{}, uc, [&](auto m) __attribute__((always_inline)) { read_two(Q1{}, m, slot); });
      const int free = slot;
      if (t + 1 < T) {
        // step t is in registers and step t + 1 has landed, all but this wave's
        // loads of the R - 2 steps after it; then the same of everybody
        constexpr int later = (R - 2) * N + (u + 2 <= 4 && 4 < u + R ? S::SI : 0);
        if (t + R - 1 < T) mx_wait<later>();
        else mx_wait<0>();
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        slot = slot == R - 1 ? 0 : slot + 1;
        if constexpr (u == 3) read_scales((t + 1) >> 2);
      }
      const bool more = t + R < T;
      multiply(Q1{}, uc, [&](auto m) __attribute__((always_inline)) {
        read_two(Q0{}, m, slot);  // past the last step: read and not used
        // loads of step t + R
        constexpr int i = decltype(m)::value, n = N + ((u + R) % 4 == 0 ? S::SI : 0), per = (n + M - 1) / M;
        if (more)
          static_for<per>([&](auto e) __attribute__((always_inline)) {
            if constexpr (i * per + decltype(e)::value < n)
              issue(std::integral_constant<int, i * per + decltype(e)::value>{}, t + R, free);
          });
      });
    });
  }

  // The output goes out in whole rows of the wave's columns, by way of LDS (the
  // ring's: every wave is done with it).  Lane (l32, lg) holds columns 8 q + 4 lg
  // .. + 3 of a fragment, row l32.
  if constexpr (S::kSplits) {
    if (a.splits > 1) {  // fp32 sums as they lie; n a multiple of 8
#pragma unroll
      for (int i = 0; i < FR; ++i)
#pragma unroll
        for (int j = 0; j < FC; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int m = bm * S::TM + (wr * FR + i) * 32 + l32, c = bn * S::OUT + (wc * FC + j) * 32 + 8 * q + 4 * lg;
            if (m < a.rows && c < a.n)
              *reinterpret_cast<f32x4*>(a.part + ((int64_t)split * a.rows + m) * a.n + c) =
                  f32x4{acc[j][i][4 * q], acc[j][i][4 * q + 1], acc[j][i][4 * q + 2], acc[j][i][4 * q + 3]};
          }
      return;
    }
  }
  constexpr int H = S::GATED ? FC / 2 : FC, C = H * 32, kPitch = C + 8, ROWS = FR * 32;
  static_assert(NW * ROWS * kPitch * 2 <= S::kLds);
  __syncthreads();
  f16* own = reinterpret_cast<f16*>(lds_raw) + wave * ROWS * kPitch;
#pragma unroll
  for (int i = 0; i < FR; ++i)
#pragma unroll
    for (int j = 0; j < H; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        f16x4 h;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = acc[j][i][4 * q + e];
          if constexpr (S::GATED) v *= mx_silu(acc[j + H][i][4 * q + e]);
          h[e] = (f16)v;
        }
        *reinterpret_cast<f16x4*>(own + (i * 32 + l32) * kPitch + j * 32 + 8 * q + 4 * lg) = h;
      }
  const int m0 = bm * S::TM + wr * ROWS, n0 = bn * S::OUT + wc * C;
  const int rows = min(ROWS, a.rows - m0), cols = min(C, a.n - n0);
  f16* y = a.y + (int64_t)m0 * a.n + n0;
  // Eight values a lane; where rows do not start at whole vectors the stores are
  // of the type's own alignment, and a row's last values may go alone.  1237 x
  // 2080 -> 18993: 55 us, as 18992; value by value 63, in words 80.  (Stores past
  // the caches gain 2 us of 105 at 8192 x 4096 -> 4096, which the next reader loses.)
  typedef f16x8 __attribute__((aligned(2))) f16x8_any;
  for (int r = lane; r < ROWS * (C / 8); r += kWave) {
    const int m = r / (C / 8), c = r % (C / 8) * 8;
    if (m >= rows || c >= cols) continue;
    const f16x8 v = *reinterpret_cast<const f16x8*>(own + m * kPitch + c);
    f16* dst = y + (int64_t)m * a.n + c;
    if (S::GATED || a.n % 8 == 0) {
      *reinterpret_cast<f16x8*>(dst) = v;
    } else if (c + 8 <= cols) {
      *reinterpret_cast<f16x8_any*>(dst) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 7; ++e)
        if (c + e < cols) dst[e] = v[e];
    }
  }
}

template <class S>
int launch_mx_tile(const MxArgs& a, hipStream_t st) {
  if (int rc = allow_mx_lds<&mx_tile_kernel<S>, S::kLds>()) return rc;
  const int m_tiles = (a.rows + S::TM - 1) / S::TM, n_tiles = (a.n + S::OUT - 1) / S::OUT;
  hipLaunchKernelGGL(mx_tile_kernel<S>, dim3((unsigned)m_tiles * n_tiles * a.splits), dim3(S::NW * kWave), S::kLds, st, a, m_tiles,
                     n_tiles);
  return launch_status(S::GATED ? "mxfp4_up_gate_silu_and_mul" : "mxfp4_linear");
}

template <bool GATED>
int launch_mx(const MxArgs& a, const MxConfig& c, hipStream_t st) {
  switch (c.kernel) {
    case kMxTile128x256: return launch_mx_tile<MxTile<2, 2, 2, 4, 2, GATED>>(a, st);
    case kMxTile128: return launch_mx_tile<MxTile<2, 2, 2, 2, 3, GATED>>(a, st);
    default: return GATED ? mx_stream_gated(a, c, st) : mx_stream_linear(a, c, st);
  }
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
  // workgroups that are done write y, and the first launch the workspace, while others still read
  int64_t xc = 0, xs = 0, wc = 0, ws_bytes = 0;
  (void)nsd_mx_bytes(8, n_rows, n_in, &xc, &xs);
  (void)nsd_mx_bytes(4, GATED ? 2 * n : n, n_in, &wc, &ws_bytes);
  auto over = [&](const void* p, int64_t bytes) {
    if (x ? mx_overlap(p, bytes, x, n_rows * n_in * 2) : mx_overlap(p, bytes, x_codes, xc) || mx_overlap(p, bytes, x_scales, xs))
      return "x";
    return mx_overlap(p, bytes, w_codes, wc) || mx_overlap(p, bytes, w_scales, ws_bytes) ? "the weight" : (const char*)nullptr;
  };
  const int64_t y_bytes = n_rows * n * 2;
  if (const char* what = over(y, y_bytes)) return fail(NSD_ERR_INVALID, "%s: y overlaps %s", who, what);
  if (mx_overlap(y, y_bytes, workspace, workspace_bytes))
    return fail(NSD_ERR_INVALID, "%s: y overlaps the workspace", who);
  if (const char* what = over(workspace, workspace_bytes))
    return fail(NSD_ERR_INVALID, "%s: the workspace overlaps %s", who, what);
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
    if (int rc = mxfp8_quantize(x, n_rows, n_in, ws, ws + align256(need.codes), stream)) return rc;
    x_codes = ws;
    x_scales = ws + align256(need.codes);
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
  if (gated && n_out % 32)
    return fail(NSD_ERR_UNSUPPORTED, "mx_workspace: gated n_out=%lld (a multiple of 32)", (long long)n_out);
  if (n_rows == 0) {  // no kernel to choose
    *bytes = 0;
    return NSD_OK;
  }
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
