// Writers and reader of the 8-bit paged KV cache for gfx950 (include/nsd_kv8.h).
//
// A unit is one tile, the K or the V of one block, layer and kv head, and one
// wave owns it: the tile's scale is a maximum over its 16 x 128 values, so it
// needs no other wave.  The values stay in registers between the maximum and
// the conversion.
//
//   K tile: lane 8 t + c (mod 64; t and t + 8) holds dims 8c .. 8c+7 and 64+8c ..
//           64+8c+7 of token t: a RoPE pair in one lane, and its 16 codes the
//           tile's unit 16 c + t.
//   V tile: lane 16 g + i holds dims 8i .. 8i+7 of tokens 4g .. 4g+3, whose codes,
//           transposed by bytes within the lane, are the tile's units 16 g + i and
//           64 + 16 g + i.
//
// Either way fp16 rows are read, and written, in runs of 128 bytes or more, and
// codes in runs of 128 bytes (K) or 1024 (V).
#include <algorithm>

#include "nsd_kv8_device.h"

// fp32 results are rounded to fp32 and then to fp16, as the fp16 prologue does.
#pragma clang fp contract(off)

namespace nsd {
namespace {

constexpr int D = kHeadDim;       // 128
constexpr int BS = kBlockTokens;  // 16
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int64_t kMaxGrid = (1 << 24) - 1;  // a launch's threads stay below 2^32
// Decode/verify rows of a call.  Of 8 kv heads, stored / with the prologue of 32
// heads: 768 in 13 / 18 us, 2048 in 42 / 55, 8192 in 350 / 480, 16384 in 1.2 / 1.5 ms,
// this many in 14 / 19; 2^20 would hold the GPU for seconds.
constexpr int kMaxAppendRows = 1 << 16;

struct Cache {
  u32x4* k;
  u32x4* v;
  uint8_t* ks;
  uint8_t* vs;
  int64_t num_blocks;
  int num_layers, layer, hkv;
};

// Maximum over the wave, in every lane: the 16 lanes of a DPP row by
// neighbours, pairs and two mirrors, then the four rows by gfx950's row swaps.
template <int CTRL>
__device__ inline uint32_t dpp_max(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true));
}
__device__ inline uint32_t wave_max(uint32_t v) {
  v = dpp_max<0xB1>(v);   // quad_perm [1,0,3,2]
  v = dpp_max<0x4E>(v);   // quad_perm [2,3,0,1]
  v = dpp_max<0x141>(v);  // row_half_mirror
  v = dpp_max<0x140>(v);  // row_mirror
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max(b[0], b[1]);
}

// A tile's scale from its values, R runs of eight a lane (zeros where a lane
// has none): the exponent, and whether the conversion has to be careful.
struct Scale {
  int e;
  bool top;  // the largest
  bool careful;
};
template <int T, int R>
__device__ inline Scale tile_scale(const f16x8 (&h)[R], int32_t* status) {
  u16x8 most = kv8_abs(h[0]);
#pragma unroll
  for (int r = 1; r < R; ++r) most = __builtin_elementwise_max(most, kv8_abs(h[r]));
  uint32_t m = wave_max(kv8_most(most));
  bool careful = false;
  if (m >= kF16Inf) {  // the finite ones alone
    careful = true;
    if ((threadIdx.x & 63) == 0) flag_status(status, NSD_STATUS_NONFINITE);
    m = 0;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t b = __builtin_bit_cast(u16x8, h[r])[i] & 0x7fffu;
        m = max(m, b < kF16Inf ? b : 0u);
      }
    m = wave_max(m);
  }
  const int e = kv8_exponent<T>(m);
  const bool top = e == (T == NSD_KV8_E4M3 ? 8 : 9);
  return {e, top, careful || top};
}

// The unit's tile: its codes and its scale byte.
struct Unit {
  u32x4* codes;
  uint8_t* scale;
};
__device__ inline Unit unit_of(const Cache& c, int64_t blk, int head, bool isv) {
  const int64_t tile = (blk * c.num_layers + c.layer) * c.hkv + head;
  return {(isv ? c.v : c.k) + tile * kKv8Units, (isv ? c.vs : c.ks) + tile};
}

__device__ inline u32x4 k_unit(u32x2 lo, u32x2 hi) { return u32x4{lo[0], lo[1], hi[0], hi[1]}; }

// v + v of lane ^ 4, ^ 2 or ^ 1, of eight lanes a row, by DPP: shifts by four
// into the lanes that have a partner there, or permutations of four.  (Through
// LDS, __shfl_xor: 64 rows 4.6 us, 4.4 so.)
template <int M>
__device__ inline float add_lane(float v) {
  const int u = __float_as_int(v);
  int t;
  if constexpr (M == 4) {
    t = __builtin_amdgcn_update_dpp(0, u, 0x104, 0xf, 0x5, false);  // lanes 0 .. 3 of 8: from lane + 4
    t = __builtin_amdgcn_update_dpp(t, u, 0x114, 0xf, 0xa, false);  // lanes 4 .. 7: from lane - 4
  } else {
    t = __builtin_amdgcn_mov_dpp(u, M == 2 ? 0x4E : 0xB1, 0xf, 0xf, true);  // quad_perm [2,3,0,1], [1,0,3,2]
  }
  return v + __int_as_float(t);
}

// What the decode/verify writer reads.  With the prologue (`PRO`) k is
// normalised and rotated before it is stored, and q into q_out.
struct AppendArgs {
  const f16* k;
  const f16* v;
  int64_t k_rs, v_rs;
  const int32_t* bt;
  int64_t bt_rows, bt_stride;
  const int32_t* seq_ids;
  const int32_t* seq_lens;
  int n_rows;
  int kv_groups;  // workgroups of a row's units
  int32_t* status;
  // the prologue's; part: q, k and v are a projection's split partials, fp32
  // [splits, n_rows, (hq + 2 Hkv) 128], and q_rs is its width
  const float* part;
  const f16* q;
  int64_t q_rs;
  f16* q_out;
  const f16* qw;
  const f16* kw;
  float eps;
  const f16* cos_c;
  const f16* sin_c;
  int64_t n_pos;
  int hq;
};

// Eight values of a row: fp16, or the sum of S split partials `per_split`
// elements apart, in their order, as the projection's fp16 output (the rounding
// is the output's).
template <int S>
__device__ inline f16x8 eight_of(const f16* rows, const float* part, int64_t per_split) {
  if constexpr (S == 0) {
    return *reinterpret_cast<const f16x8*>(rows);
  } else {
    f32x4 lo[S], hi[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      lo[s] = *reinterpret_cast<const f32x4*>(part + s * per_split);
      hi[s] = *reinterpret_cast<const f32x4*>(part + s * per_split + 4);
    }
    f16x8 h;
#pragma unroll
    for (int s = 1; s < S; ++s) {
      lo[0] += lo[s];
      hi[0] += hi[s];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = (f16)(e < 4 ? lo[0][e % 4] : hi[0][e % 4]);
    return h;
  }
}

// Where a row goes: its block, or -1 and the flag that says why not.  In parts
// without a branch, so that a caller has several rows' loads in flight: the row's
// numbers, its entry of the block table (any entry, where the numbers are not
// good), and what they say.
struct RowNumbers {
  int sid, len;
};
struct Place {
  int64_t blk, pos;
  int32_t flag;
};
__device__ inline RowNumbers numbers_of(const AppendArgs& a, int64_t r) { return {a.seq_ids[r], a.seq_lens[r]}; }
__device__ inline bool in_table(const AppendArgs& a, const RowNumbers& n) {
  return n.sid >= 0 && n.sid < a.bt_rows && n.len >= 1 && n.len <= a.bt_stride * BS;
}
__device__ inline int entry_of(const AppendArgs& a, const RowNumbers& n) {
  return a.bt[in_table(a, n) ? n.sid * a.bt_stride + (n.len - 1) / BS : 0];
}
template <bool PRO>
__device__ inline Place place_of(const Cache& c, const AppendArgs& a, const RowNumbers& n, int entry) {
  const bool in = in_table(a, n);
  const int64_t pos = (int64_t)n.len - 1;
  const bool turned = !PRO || pos < a.n_pos;
  const bool held = entry >= 0 && entry < c.num_blocks;
  return {in && turned && held ? entry : -1, pos,
          !in ? NSD_STATUS_BAD_SEQ : !turned ? NSD_STATUS_BAD_POSITION : NSD_STATUS_BAD_BLOCK};
}

// The norm's weights of a lane's 16 dims, and the angles of a position.
struct Weights {
  f16x8 lo, hi;
};
__device__ inline Weights weights_of(const f16* w, int c) {
  if (w == nullptr) return {};
  return {*reinterpret_cast<const f16x8*>(w + 8 * c), *reinterpret_cast<const f16x8*>(w + D / 2 + 8 * c)};
}
struct Angles {
  f16x8 cos, sin;
};
__device__ inline Angles angles_of(const AppendArgs& a, int64_t pos, int c) {
  return {*reinterpret_cast<const f16x8*>(a.cos_c + pos * (D / 2) + 8 * c),
          *reinterpret_cast<const f16x8*>(a.sin_c + pos * (D / 2) + 8 * c)};
}

// Dims 8c .. 8c+7 (lo) and 64+8c .. (hi) of a row, eight lanes a row: RMS-
// normalised with w (if `norm`) and rotated by the position's angles, in the
// fp16 prologue's arithmetic bit for bit: it adds x_d^2 + x_{d+64}^2 over a
// butterfly of lanes d ^ 32, ^ 16, ^ 8, ^ 4, ^ 2, ^ 1, which here are the lanes
// c ^ 4, ^ 2, ^ 1 and then the eight of a lane.
__device__ inline void norm_rope(f16x8& lo, f16x8& hi, bool norm, const Weights& w, float eps, const Angles& at) {
  float x0[8], x1[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    x0[j] = (float)lo[j];
    x1[j] = (float)hi[j];
  }
  if (norm) {
    float u[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = sq_pair(x0[j], x1[j]);
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = add_lane<1>(add_lane<2>(add_lane<4>(u[j])));
    const float ss = ((u[0] + u[4]) + (u[2] + u[6])) + ((u[1] + u[5]) + (u[3] + u[7]));
    const float rstd = 1.f / sqrtf(ss / (float)D + eps);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x0[j] = (float)f16_of(x0[j] * rstd * (float)w.lo[j]);
      x1[j] = (float)f16_of(x1[j] * rstd * (float)w.hi[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    lo[j] = f16_of(rope_lo(x0[j], x1[j], (float)at.cos[j], (float)at.sin[j]));
    hi[j] = f16_of(rope_hi(x0[j], x1[j], (float)at.cos[j], (float)at.sin[j]));
  }
}

// Decode/verify rows.  Rows that share a block have to agree on its scale, so
// the block belongs to the first of them: the workgroups of every other row see
// an earlier one in the same block and leave.  A workgroup looks through all
// the rows, 256 at a time, and keeps for each of the block's slots the last row
// that goes there.  So the work grows with the rows' square (kMaxAppendRows).
//
// Bound by latency, one trip to memory after another: row numbers, the block
// table, the tile and then the rows.  64 rows of 16 + 2 x 8 heads with the prologue
// 4.3 us, 16 x 5 of 32 + 2 x 8 5.2 (an empty launch 1.9).  So loads go out together
// (asm that names them keeps them so): one trip less each for the row numbers, the
// norm's weights and a tile's several rows, 4.4 and 5.6 before.
//
// S: 0 for fp16 rows, else the split partials of the projection that makes them
// (a decoder layer's: their sum in a launch of its own costs 3 us more).
template <int T, bool PRO, int S>
__global__ __launch_bounds__(kThreads) void kv8_append_kernel(Cache c, AppendArgs a) {
  static_assert(PRO || S == 0, "only the prologue reads partials");
  const int64_t per_split = a.n_rows * a.q_rs;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kv_wgs = a.n_rows * a.kv_groups;
  if (PRO && (int)blockIdx.x >= kv_wgs) {  // q: eight lanes a head
    const int64_t at = (int64_t)((int)blockIdx.x - kv_wgs) * (kThreads / 8) + (threadIdx.x >> 3);
    const int cc = lane & 7;
    const bool any = at < (int64_t)a.n_rows * a.hq;
    const int64_t r = any ? at / a.hq : 0;
    const int h = any ? (int)(at - r * a.hq) : 0;
    const int64_t from = r * a.q_rs + (int64_t)h * D + 8 * cc;
    f16x8 lo = eight_of<S>(a.q + from, a.part + from, per_split);
    f16x8 hi = eight_of<S>(a.q + from + D / 2, a.part + from + D / 2, per_split);
    const Weights w = weights_of(a.qw, cc);
    const int64_t pos = (int64_t)a.seq_lens[r] - 1;
    const bool in = pos >= 0 && pos < a.n_pos;
    const Angles at_pos = angles_of(a, in ? pos : 0, cc);
    if (any && !in && cc == 0) flag_status(a.status, NSD_STATUS_BAD_POSITION);
    norm_rope(lo, hi, a.qw != nullptr, w, a.eps, at_pos);  // a head's eight lanes agree on any and in
    if (any && in) {
      f16* dst = a.q_out + at * D + 8 * cc;
      *reinterpret_cast<f16x8*>(dst) = lo;
      *reinterpret_cast<f16x8*>(dst + D / 2) = hi;
    }
    return;
  }

  __shared__ unsigned long long s_slot[BS];  // (row + 1) << 32 | position, 0: none
  __shared__ int s_earlier;
  const int r = (int)blockIdx.x / a.kv_groups, group = (int)blockIdx.x - r * a.kv_groups;
  // this row's place and, beside it, the places of the first 256; by a row number
  // in a vector register (+ 0), since a scalar's way there waits for its load
  const RowNumbers own_numbers = numbers_of(a, r + (int)(threadIdx.x >> 16));
  const RowNumbers numbers = numbers_of(a, min((int)threadIdx.x, a.n_rows - 1));
  asm volatile("" ::"v"(own_numbers.sid), "v"(own_numbers.len), "v"(numbers.sid), "v"(numbers.len));  // in one trip
  const int own_entry = entry_of(a, own_numbers), entry = entry_of(a, numbers);
  const Weights kw = PRO ? weights_of(a.kw, lane & 7) : Weights{};
  asm volatile("" ::"v"(own_entry), "v"(entry));
  Place own = place_of<PRO>(c, a, own_numbers, own_entry);
  own.blk = __builtin_amdgcn_readfirstlane((int)own.blk);
  Place p = place_of<PRO>(c, a, numbers, entry);
  if (own.blk < 0) {
    if (group == 0 && threadIdx.x == 0) flag_status(a.status, own.flag);
    return;
  }
  const int unit = group * kWaves + wave;
  const bool live = unit < 2 * c.hkv;
  const bool isv = unit >= c.hkv;
  const Unit u = unit_of(c, own.blk, live ? (isv ? unit - c.hkv : unit) : 0, isv);
  // the tile as it is: two units a lane, in the order of the tile's kind
  u32x4 was[2];
  const int at0 = isv ? lane : (lane & 7) * 16 + (lane >> 3), step = isv ? 64 : 8;
#pragma unroll
  for (int j = 0; j < 2; ++j) was[j] = u.codes[at0 + step * j];
  const int old_byte = *u.scale;

  if (threadIdx.x < BS) s_slot[threadIdx.x] = 0;
  if (threadIdx.x == 0) s_earlier = 0;
  __syncthreads();
  for (int rr = threadIdx.x; rr < a.n_rows; rr += kThreads) {
    if (rr != (int)threadIdx.x) {
      const RowNumbers n = numbers_of(a, rr);
      p = place_of<PRO>(c, a, n, entry_of(a, n));
    }
    if (p.blk != own.blk) continue;
    atomicMax(&s_slot[p.pos % BS], (unsigned long long)(rr + 1) << 32 | (unsigned long long)p.pos);
    if (rr < r) s_earlier = 1;
  }
  __syncthreads();
  if (s_earlier || !live) return;

  const uint32_t fresh = (uint32_t)__builtin_amdgcn_ballot_w64(s_slot[lane & 15] != 0) & 0xffffu;
  const uint32_t below = (1u << (31 - __builtin_clz(fresh))) - 1;
  const uint32_t old = below & ~fresh;  // slots whose tokens stay
  const float power = kv8_power(old_byte);
  const int head = isv ? unit - c.hkv : unit;
  asm volatile("" ::"v"(was[0]), "v"(was[1]));  // the tile is here: what is waited for below are rows
  if (!isv) {
    const int cc = lane & 7, t0 = lane >> 3;
    f16x8 h[4] = {};
    Angles at_pos[2] = {};
    unsigned long long key[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      key[j] = s_slot[t0 + 8 * j];
      // a new row among these eight slots; fp16 rows are read without asking (any
      // row will do), since the loads after a branch begin when those before it end
      if (S == 0 || (fresh >> (8 * j) & 0xff)) {
        const int64_t row = key[j] ? (int64_t)(key[j] >> 32) - 1 : r;
        const f16* src = a.k + row * a.k_rs + (int64_t)head * D + 8 * cc;
        const float* part = a.part + row * a.q_rs + (int64_t)(a.hq + head) * D + 8 * cc;
        h[2 * j] = eight_of<S>(src, part, per_split);
        h[2 * j + 1] = eight_of<S>(src + D / 2, part + D / 2, per_split);
        if constexpr (PRO) at_pos[j] = angles_of(a, key[j] ? (int64_t)(key[j] & 0xffffffffu) : 0, cc);
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int t = t0 + 8 * j;
      if (PRO && (fresh >> (8 * j) & 0xff)) norm_rope(h[2 * j], h[2 * j + 1], a.kw != nullptr, kw, a.eps, at_pos[j]);
      if (!key[j]) h[2 * j] = h[2 * j + 1] = f16x8{};
      if (old >> t & 1) {
        h[2 * j] = kv8_values<T>(u32x2{was[j][0], was[j][1]}, power);
        h[2 * j + 1] = kv8_values<T>(u32x2{was[j][2], was[j][3]}, power);
      }
    }
    const Scale s = tile_scale<T>(h, a.status);
    const bool again = s.e + 127 != old_byte;  // the tokens that stay are rounded again
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int t = t0 + 8 * j;
      if ((fresh | (again ? old : 0u)) >> t & 1)
        u.codes[at0 + 8 * j] =
            k_unit(kv8_codes<T>(h[2 * j], s.e, s.careful), kv8_codes<T>(h[2 * j + 1], s.e, s.careful));
    }
    if (lane == 0) *u.scale = (uint8_t)(s.e + 127);
  } else {
    const int i = lane & 15, t0 = 4 * (lane >> 4);
    const u32x4 a0 = kv8_transpose(was[0]), a1 = kv8_transpose(was[1]);  // a token a register: dims 8i .. +3, +4 .. +7
    f16x8 h[4] = {};
    bool news[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned long long key = s_slot[t0 + j];
      news[j] = key != 0;
      if (S == 0 || (fresh & (0x1111u << j))) {  // a new row among slots j, j + 4, ...
        const int64_t row = key ? (int64_t)(key >> 32) - 1 : r;
        h[j] = eight_of<S>(a.v + row * a.v_rs + (int64_t)head * D + 8 * i,
                           a.part + row * a.q_rs + (int64_t)(a.hq + c.hkv + head) * D + 8 * i, per_split);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f16x8 held = kv8_values<T>(u32x2{a0[j], a1[j]}, power);
      h[j] = news[j] ? h[j] : old >> (t0 + j) & 1 ? held : f16x8{};
    }
    const Scale s = tile_scale<T>(h, a.status);
    // under the largest scale codes that no writer makes there would be
    // infinities, which the attention multiplies by masked tokens' zeros: slots
    // that hold no token become zeros
    const uint32_t put = s.top ? 0xffffu : fresh | (s.e + 127 != old_byte ? old : 0u);
    u32x4 b0 = a0, b1 = a1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const u32x2 w = kv8_codes<T>(h[j], s.e, s.careful);
      b0[j] = put >> (t0 + j) & 1 ? w[0] : b0[j];
      b1[j] = put >> (t0 + j) & 1 ? w[1] : b1[j];
    }
    if (put >> t0 & 0xf) {
      u.codes[lane] = kv8_transpose(b0);
      u.codes[64 + lane] = kv8_transpose(b1);
    }
    if (lane == 0) *u.scale = (uint8_t)(s.e + 127);
  }
}

// Sixteen bytes of a row, and of codes; FAR: past the caches.
template <bool FAR>
__device__ inline f16x8 row16(const f16* p) {
  const f16x8* q = reinterpret_cast<const f16x8*>(p);
  return FAR ? __builtin_nontemporal_load(q) : *q;
}
template <bool FAR>
__device__ inline void put16(u32x4* at, u32x4 v) {
  if (FAR) __builtin_nontemporal_store(v, at);
  else *at = v;
}

// Workgroups run over the units of a block first, so that a block's rows, one
// run in memory, are read or written at one time (units last: prompts of 32k
// tokens x 8 heads stored in 84.2 us with the kernel that makes the rows, 78.5
// so; read back by 92.7 and 86.3 with their reader).

// Whole prompts: grid (block of the prompt x four units of 2 Hkv, prompt).  FAR:
// 1 codes are written past the caches, 2 rows are read past them too.  Bound by
// memory: a prompt of 32749 tokens x 8 heads 38 us, 5.2 TB/s of rows read and
// codes written (a large copy 4.8 to 5.2).
template <int T, int FAR>
__global__ __launch_bounds__(kThreads) void kv8_prefill_kernel(
    Cache c, const f16* __restrict__ k, const f16* __restrict__ v, int64_t n_tokens, const int32_t* __restrict__ bt,
    int64_t bt_rows, int64_t bt_stride, const int32_t* __restrict__ seq_ids, const int32_t* __restrict__ start_locs,
    const int32_t* __restrict__ lens, int64_t max_len, int32_t* status) {
  const int groups = (2 * c.hkv + kWaves - 1) / kWaves;
  const int64_t b = blockIdx.x / groups, s = blockIdx.y;
  const int group = blockIdx.x % groups;
  const int64_t len = lens[s], start = start_locs[s], sid = seq_ids[s];
  if (b * BS >= len) {
    if (len < 0 && blockIdx.x == 0 && threadIdx.x == 0) flag_status(status, NSD_STATUS_BAD_SEQ);
    return;
  }
  const int lane = threadIdx.x & 63;
  const int unit = group * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool first = group == 0 && threadIdx.x == 0;
  if (sid < 0 || sid >= bt_rows || len > bt_stride * BS || len > max_len || start < 0 || start + len > n_tokens) {
    if (first) flag_status(status, NSD_STATUS_BAD_SEQ);
    return;
  }
  const int64_t blk = bt[sid * bt_stride + b];
  if (blk < 0 || blk >= c.num_blocks) {
    if (first) flag_status(status, NSD_STATUS_BAD_BLOCK);
    return;
  }
  if (unit >= 2 * c.hkv) return;
  const bool isv = unit >= c.hkv;
  const int head = isv ? unit - c.hkv : unit;
  const int n = (int)min<int64_t>(BS, len - b * BS);
  const Unit u = unit_of(c, blk, head, isv);
  const int64_t rs = (int64_t)c.hkv * D;
  const f16* rows = (isv ? v : k) + (start + b * BS) * rs + (int64_t)head * D;
  f16x8 h[4];
  if (!isv) {
    const int cc = lane & 7, t0 = lane >> 3;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      h[2 * j] = h[2 * j + 1] = f16x8{};
      if (t0 + 8 * j < n) {
        const f16* src = rows + (t0 + 8 * j) * rs + 8 * cc;
        h[2 * j] = row16<FAR == 2>(src);
        h[2 * j + 1] = row16<FAR == 2>(src + D / 2);
      }
    }
    const Scale sc = tile_scale<T>(h, status);
#pragma unroll
    for (int j = 0; j < 2; ++j)
      put16<FAR != 0>(u.codes + 16 * cc + t0 + 8 * j,
              k_unit(kv8_codes<T>(h[2 * j], sc.e, sc.careful), kv8_codes<T>(h[2 * j + 1], sc.e, sc.careful)));
    if (lane == 0) *u.scale = (uint8_t)(sc.e + 127);
  } else {
    const int i = lane & 15, t0 = 4 * (lane >> 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      h[j] = f16x8{};
      if (t0 + j < n) h[j] = row16<FAR == 2>(rows + (t0 + j) * rs + 8 * i);
    }
    const Scale sc = tile_scale<T>(h, status);
    u32x4 b0, b1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const u32x2 w = kv8_codes<T>(h[j], sc.e, sc.careful);
      b0[j] = w[0];
      b1[j] = w[1];
    }
    put16<FAR != 0>(u.codes + lane, kv8_transpose(b0));
    put16<FAR != 0>(u.codes + 64 + lane, kv8_transpose(b1));
    if (lane == 0) *u.scale = (uint8_t)(sc.e + 127);
  }
}

// Reading back: grid (block from the first token's on x four units, sequence).
// Bound by memory, as a copy is: 32749 tokens x 8 heads 42 us, 4.8 TB/s.  Stores
// that pass the caches make it faster (16 sequences of 256 to 4096 tokens 31 ->
// 24 us) and its reader slower by more (24k tokens, then the prefill attention
// over them: 175.4 -> 182.7).
template <int T>
__global__ __launch_bounds__(kThreads) void kv8_load_kernel(
    Cache c, f16* __restrict__ k, f16* __restrict__ v, int64_t n_tokens, const int32_t* __restrict__ bt,
    int64_t bt_rows, int64_t bt_stride, const int32_t* __restrict__ seq_ids, const int32_t* __restrict__ firsts,
    const int32_t* __restrict__ start_locs, const int32_t* __restrict__ lens, int64_t max_len, int32_t* status) {
  const int groups = (2 * c.hkv + kWaves - 1) / kWaves;
  const int64_t s = blockIdx.y, from = blockIdx.x / groups;
  const int group = blockIdx.x % groups;
  const int64_t first = firsts != nullptr ? firsts[s] : 0, len = lens[s], start = start_locs[s], sid = seq_ids[s];
  const int64_t end = first + len;
  if (len == 0) return;
  const bool says = blockIdx.x == 0 && threadIdx.x == 0;
  if (len < 0 || sid < 0 || sid >= bt_rows || first < 0 || end > bt_stride * BS || len > max_len || start < 0 ||
      start + len > n_tokens) {
    if (says) flag_status(status, NSD_STATUS_BAD_SEQ);
    return;
  }
  const int64_t b = first / BS + from;
  if (b * BS >= end) return;
  const int64_t blk = bt[sid * bt_stride + b];
  if (blk < 0 || blk >= c.num_blocks) {
    if (group == 0 && threadIdx.x == 0) flag_status(status, NSD_STATUS_BAD_BLOCK);
    return;
  }
  const int lane = threadIdx.x & 63;
  const int unit = group * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (unit >= 2 * c.hkv) return;
  const bool isv = unit >= c.hkv;
  const int head = isv ? unit - c.hkv : unit;
  const Unit u = unit_of(c, blk, head, isv);
  const int64_t rs = (int64_t)c.hkv * D;
  // row of the block's token 0, which may lie before the first row
  f16* rows = (isv ? v : k) + (start + b * BS - first) * rs + (int64_t)head * D;
  const int lo = (int)max<int64_t>(0, first - b * BS), hi = (int)min<int64_t>(BS, end - b * BS);
  const float power = kv8_power(*u.scale);
  if (!isv) {
    const int cc = lane & 7, t0 = lane >> 3;
    u32x4 w[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) w[j] = u.codes[16 * cc + t0 + 8 * j];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int t = t0 + 8 * j;
      if (t < lo || t >= hi) continue;
      f16* dst = rows + t * rs + 8 * cc;
      *reinterpret_cast<f16x8*>(dst) = kv8_values<T>(u32x2{w[j][0], w[j][1]}, power);
      *reinterpret_cast<f16x8*>(dst + D / 2) = kv8_values<T>(u32x2{w[j][2], w[j][3]}, power);
    }
  } else {
    const int i = lane & 15, t0 = 4 * (lane >> 4);
    const u32x4 w0 = u.codes[lane], w1 = u.codes[64 + lane];
    const u32x4 a0 = kv8_transpose(w0), a1 = kv8_transpose(w1);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (t0 + j < lo || t0 + j >= hi) continue;
      *reinterpret_cast<f16x8*>(rows + (t0 + j) * rs + 8 * i) = kv8_values<T>(u32x2{a0[j], a1[j]}, power);
    }
  }
}

Cache cache_of(const nsd_kv8_cache* c, int layer) {
  return {static_cast<u32x4*>(c->k),        static_cast<u32x4*>(c->v), static_cast<uint8_t*>(c->k_scales),
          static_cast<uint8_t*>(c->v_scales), c->num_blocks,             c->num_layers,
          layer,                              c->num_kv_heads};
}

// Host: f(integral_constant<int, codes>) for the cache's codes.
template <typename F>
void with_codes(const nsd_kv8_cache* c, F&& f) {
  if (c->codes == NSD_KV8_E4M3) f(std::integral_constant<int, NSD_KV8_E4M3>{});
  else f(std::integral_constant<int, NSD_KV8_INT8>{});
}

int unit_groups(const nsd_kv8_cache* c) { return (2 * c->num_kv_heads + kWaves - 1) / kWaves; }

// The arguments that the decode/verify writers share.
int check_append(const char* who, const AppendArgs& a, const nsd_kv8_cache* cache, int64_t n_rows, int layer) {
  const int rc = check_kv8_cache(who, cache, layer);
  if (rc) return rc;
  if (n_rows < 0 || a.bt_rows <= 0 || a.bt_stride <= 0) return fail(NSD_ERR_INVALID, "%s: bad sizes", who);
  if (n_rows == 0) return NSD_OK;
  if (!a.bt || !a.seq_ids || !a.seq_lens || (!a.part && (!a.k || !a.v)))
    return fail(NSD_ERR_INVALID, "%s: null pointer", who);
  if (!aligned16(a.k) || !aligned16(a.v)) return fail(NSD_ERR_INVALID, "%s: k and v must be 16-byte aligned", who);
  if (n_rows > kMaxAppendRows)
    return fail(NSD_ERR_UNSUPPORTED, "%s: n_rows=%lld (at most %d; a prompt's are nsd_kv8_store_prefill's)", who,
                (long long)n_rows, kMaxAppendRows);
  return NSD_OK;
}

}  // namespace
}  // namespace nsd

using namespace nsd;

extern "C" int nsd_kv8_store(const void* k, const void* v, const nsd_kv8_cache* cache, const int32_t* block_table,
                             int64_t bt_rows, int64_t bt_stride, const int32_t* seq_ids, const int32_t* seq_lens,
                             int64_t n_rows, int layer, int32_t* status, void* stream) {
  AppendArgs a{};
  a.k = static_cast<const f16*>(k);
  a.v = static_cast<const f16*>(v);
  a.bt = block_table;
  a.bt_rows = bt_rows;
  a.bt_stride = bt_stride;
  a.seq_ids = seq_ids;
  a.seq_lens = seq_lens;
  a.status = status;
  const int rc = check_append("kv8_store", a, cache, n_rows, layer);
  if (rc || n_rows == 0) return rc;
  a.k_rs = a.v_rs = (int64_t)cache->num_kv_heads * D;
  a.n_rows = (int)n_rows;
  a.kv_groups = unit_groups(cache);
  const int64_t grid = n_rows * a.kv_groups;
  if (grid > kMaxGrid) return fail(NSD_ERR_UNSUPPORTED, "kv8_store: grid too large");
  with_codes(cache, [&](auto t) {
    hipLaunchKernelGGL((kv8_append_kernel<decltype(t)::value, false, 0>), dim3((unsigned)grid), dim3(kThreads), 0,
                       as_stream(stream), cache_of(cache, layer), a);
  });
  return launch_status("kv8_store");
}

// The prologue over fp16 rows (splits 0) or partials; `a` has what the entries
// differ in: the rows, or `part`, and q_rs.
static int prologue(const char* who, AppendArgs a, int splits, void* q_out, const void* q_norm_w, const void* k_norm_w,
                    float eps, const void* cos_cache, const void* sin_cache, int64_t n_positions,
                    const nsd_kv8_cache* cache, const int32_t* block_table, int64_t bt_rows, int64_t bt_stride,
                    const int32_t* seq_ids, const int32_t* seq_lens, int64_t n_rows, int layer, int num_q_heads,
                    int32_t* status, void* stream) {
  a.bt = block_table;
  a.bt_rows = bt_rows;
  a.bt_stride = bt_stride;
  a.seq_ids = seq_ids;
  a.seq_lens = seq_lens;
  a.status = status;
  a.q_out = static_cast<f16*>(q_out);
  a.qw = static_cast<const f16*>(q_norm_w);
  a.kw = static_cast<const f16*>(k_norm_w);
  a.eps = eps;
  a.cos_c = static_cast<const f16*>(cos_cache);
  a.sin_c = static_cast<const f16*>(sin_cache);
  a.n_pos = n_positions;
  a.hq = num_q_heads;
  const int rc = check_append(who, a, cache, n_rows, layer);
  if (rc) return rc;
  if (num_q_heads <= 0 || n_positions <= 0) return fail(NSD_ERR_INVALID, "%s: bad sizes", who);
  if ((q_norm_w == nullptr) != (k_norm_w == nullptr))
    return fail(NSD_ERR_INVALID, "%s: pass both norm weights or neither", who);
  if (n_rows == 0) return NSD_OK;
  if ((!a.q && !a.part) || !q_out || !cos_cache || !sin_cache) return fail(NSD_ERR_INVALID, "%s: null pointer", who);
  for (const void* p : {(const void*)a.q, (const void*)a.part, (const void*)q_out, cos_cache, sin_cache, q_norm_w,
                        k_norm_w})
    if (!aligned16(p)) return fail(NSD_ERR_INVALID, "%s: rows, tables and norm weights must be 16-byte aligned", who);
  a.n_rows = (int)n_rows;
  a.kv_groups = unit_groups(cache);
  const int64_t grid = n_rows * a.kv_groups + (n_rows * num_q_heads + kThreads / 8 - 1) / (kThreads / 8);
  if (grid > kMaxGrid) return fail(NSD_ERR_UNSUPPORTED, "%s: grid too large", who);
  with_codes(cache, [&](auto t) {
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(kThreads), 0, as_stream(stream), cache_of(cache, layer), a);
    };
    constexpr int T = decltype(t)::value;
    if (splits == 0) go(kv8_append_kernel<T, true, 0>);
    else with_splits(splits, [&](auto count) { go(kv8_append_kernel<T, true, decltype(count)::value>); });
  });
  return launch_status(who);
}

extern "C" int nsd_kv8_qk_norm_rope_store(const void* q, int64_t q_row_stride, void* q_out, const void* k,
                                          int64_t k_row_stride, const void* v, int64_t v_row_stride,
                                          const void* q_norm_w, const void* k_norm_w, float eps,
                                          const void* cos_cache, const void* sin_cache, int64_t n_positions,
                                          const nsd_kv8_cache* cache, const int32_t* block_table, int64_t bt_rows,
                                          int64_t bt_stride, const int32_t* seq_ids, const int32_t* seq_lens,
                                          int64_t n_rows, int layer, int num_q_heads, int32_t* status,
                                          void* stream) {
  const char* who = "kv8_qk_norm_rope_store";
  if (cache != nullptr) {
    const int64_t hkv = cache->num_kv_heads;
    if (q_row_stride < (int64_t)num_q_heads * D || k_row_stride < hkv * D || v_row_stride < hkv * D ||
        (q_row_stride | k_row_stride | v_row_stride) & 7)
      return fail(NSD_ERR_INVALID, "%s: row strides must be multiples of 8 that cover the heads", who);
  }
  if (q != nullptr && q == q_out && q_row_stride != (int64_t)num_q_heads * D)
    return fail(NSD_ERR_INVALID, "%s: q in place has to be contiguous", who);
  AppendArgs a{};
  a.k = static_cast<const f16*>(k);
  a.v = static_cast<const f16*>(v);
  a.k_rs = k_row_stride;
  a.v_rs = v_row_stride;
  a.q = static_cast<const f16*>(q);
  a.q_rs = q_row_stride;
  return prologue(who, a, 0, q_out, q_norm_w, k_norm_w, eps, cos_cache, sin_cache, n_positions, cache, block_table,
                  bt_rows, bt_stride, seq_ids, seq_lens, n_rows, layer, num_q_heads, status, stream);
}

extern "C" int nsd_kv8_qk_norm_rope_store_partials(const float* partials, int splits, void* q_out,
                                                   const void* q_norm_w, const void* k_norm_w, float eps,
                                                   const void* cos_cache, const void* sin_cache, int64_t n_positions,
                                                   const nsd_kv8_cache* cache, const int32_t* block_table,
                                                   int64_t bt_rows, int64_t bt_stride, const int32_t* seq_ids,
                                                   const int32_t* seq_lens, int64_t n_rows, int layer,
                                                   int num_q_heads, int32_t* status, void* stream) {
  const char* who = "kv8_qk_norm_rope_store_partials";
  if (cache == nullptr) return fail(NSD_ERR_INVALID, "%s: null cache", who);
  if (splits < 1 || splits > 8) return fail(NSD_ERR_INVALID, "%s: %d splits (1..8)", who, splits);
  if (n_rows > 0 && partials == nullptr) return fail(NSD_ERR_INVALID, "%s: null pointer", who);
  AppendArgs a{};
  a.part = partials;
  a.q_rs = ((int64_t)num_q_heads + 2 * (int64_t)cache->num_kv_heads) * D;
  return prologue(who, a, splits, q_out, q_norm_w, k_norm_w, eps, cos_cache, sin_cache, n_positions, cache, block_table,
                  bt_rows, bt_stride, seq_ids, seq_lens, n_rows, layer, num_q_heads, status, stream);
}

extern "C" int nsd_kv8_store_prefill(const void* k, const void* v, int64_t n_tokens, const nsd_kv8_cache* cache,
                                     const int32_t* block_table, int64_t bt_rows, int64_t bt_stride,
                                     const int32_t* seq_ids, const int32_t* start_locs, const int32_t* prefill_lens,
                                     int64_t n_seqs, int64_t max_prefill_len, int layer, int32_t* status,
                                     void* stream) {
  const char* who = "kv8_store_prefill";
  const int rc = check_kv8_cache(who, cache, layer);
  if (rc) return rc;
  if (n_seqs < 0 || max_prefill_len < 0 || n_tokens < 0 || bt_rows <= 0 || bt_stride <= 0)
    return fail(NSD_ERR_INVALID, "%s: bad sizes", who);
  if (n_seqs == 0 || max_prefill_len == 0) return NSD_OK;
  if (!k || !v || !block_table || !seq_ids || !start_locs || !prefill_lens)
    return fail(NSD_ERR_INVALID, "%s: null pointer", who);
  if (!aligned16(k) || !aligned16(v)) return fail(NSD_ERR_INVALID, "%s: k and v must be 16-byte aligned", who);
  const int64_t nb = std::min((max_prefill_len + BS - 1) / BS, bt_stride);
  const int64_t grid = nb * unit_groups(cache);
  if (grid > kMaxGrid || n_seqs > 65535) return fail(NSD_ERR_UNSUPPORTED, "%s: grid too large", who);
  // Many rows do not stay in the 256 MB memory-side cache beside what follows.
  // Their codes are read next by a decode step, layers later: written past the
  // caches, 16k tokens x 8 heads (67 MB of rows) with the kernel that makes the
  // rows 42.2 -> 39.5 us, 9k 25.4 -> 25.0, but 9k read back at once 18.4 -> 21.4.
  // The rows themselves, read past them: 32k 38.9 -> 36.6, but 16k, still there
  // when their maker has just ended, 17.7 -> 19.2.
  const int64_t row_bytes = n_tokens * cache->num_kv_heads * (int64_t)(2 * D * sizeof(f16));
  with_codes(cache, [&](auto t) {
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)grid, (unsigned)n_seqs), dim3(kThreads), 0, as_stream(stream),
                         cache_of(cache, layer), static_cast<const f16*>(k), static_cast<const f16*>(v), n_tokens,
                         block_table, bt_rows, bt_stride, seq_ids, start_locs, prefill_lens, max_prefill_len, status);
    };
    constexpr int T = decltype(t)::value;
    if (row_bytes >= 128000000) go(kv8_prefill_kernel<T, 2>);
    else if (row_bytes >= 64000000) go(kv8_prefill_kernel<T, 1>);
    else go(kv8_prefill_kernel<T, 0>);
  });
  return launch_status(who);
}

extern "C" int nsd_kv8_load(void* k, void* v, int64_t n_tokens, const nsd_kv8_cache* cache,
                            const int32_t* block_table, int64_t bt_rows, int64_t bt_stride, const int32_t* seq_ids,
                            const int32_t* first, const int32_t* start_locs, const int32_t* lens, int64_t n_seqs,
                            int64_t max_len, int layer, int32_t* status, void* stream) {
  const char* who = "kv8_load";
  const int rc = check_kv8_cache(who, cache, layer);
  if (rc) return rc;
  if (n_seqs < 0 || max_len < 0 || n_tokens < 0 || bt_rows <= 0 || bt_stride <= 0)
    return fail(NSD_ERR_INVALID, "%s: bad sizes", who);
  if (n_seqs == 0 || max_len == 0 || n_tokens == 0) return NSD_OK;
  if (!k || !v || !block_table || !seq_ids || !start_locs || !lens)
    return fail(NSD_ERR_INVALID, "%s: null pointer", who);
  if (!aligned16(k) || !aligned16(v)) return fail(NSD_ERR_INVALID, "%s: k and v must be 16-byte aligned", who);
  // a range that starts inside a block touches one more
  const int64_t nb = std::min((max_len + BS - 1) / BS + (first != nullptr ? 1 : 0), bt_stride);
  const int64_t grid = nb * unit_groups(cache);
  if (grid > kMaxGrid || n_seqs > 65535) return fail(NSD_ERR_UNSUPPORTED, "%s: grid too large", who);
  with_codes(cache, [&](auto t) {
    hipLaunchKernelGGL(kv8_load_kernel<decltype(t)::value>, dim3((unsigned)grid, (unsigned)n_seqs), dim3(kThreads), 0,
                       as_stream(stream), cache_of(cache, layer), static_cast<f16*>(k), static_cast<f16*>(v),
                       n_tokens, block_table, bt_rows, bt_stride, seq_ids, first, start_locs, lens, max_len, status);
  });
  return launch_status(who);
}
