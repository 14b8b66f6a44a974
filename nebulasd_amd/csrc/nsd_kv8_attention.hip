// Paged verify/decode attention over the 8-bit KV cache for gfx950.
//
// The work is the fp16 attention's (nsd_attention.hip): a workgroup of four
// waves streams one piece, blocks [blk_begin, blk_end) of a (verify group, kv
// head) segment, for all of the segment's query rows, by the same plan; a
// second launch merges the segments cut into pieces.
//
//   S^T[token][row] = K[token][:] . Q[row][:]            (A = K, B = Q^T)
//   O^T[dim][row]  += V^T[dim][token] . P^T[token][row]  (A = V^T, B = P^T)
//
// Both in v_mfma_f32_16x16x32_f16.  A cache's values are fp16 values, so the
// codes become operands without a rounding: E4M3 with the block's scale in the
// one instruction that converts two, whole numbers by a byte permutation and a
// subtraction (K's scale then multiplies the scores, V's the operand).
//
// Wave w takes blocks w, w + 4, ... of the piece by pairs: the 32 tokens of a
// pair are the k of one PV product.  S^T of a block leaves lane (lr, lg) with
// tokens 4lg .. 4lg+3 of row lr, which for the two blocks is P^T's operand as it
// stands, with the pair's tokens in the order that V's operand is put together.
//
// A tile lies in the cache as its operand is held: lane l's 16 bytes of load j
// are unit 64 j + l of the tile.  A wave streams its pairs through a ring of its
// own in LDS, two slots of 8 KB filled by global_load_lds_dwordx4 in runs of 1
// KB; it reads a pair into registers, in runs again (no bank conflict, no
// transpose), and refills the slot before it computes, so a pair and a half is
// in flight at all times.  Lane (i, g) of K holds dims 8c .. 8c+7 and 64+8c ..
// of token i (c = 4 j + g): the query operand has its dims in that order too.
// Of V it holds dims 8i .. 8i+7 of tokens 4g .. 4g+3: tile m of O^T is dims m,
// 8 + m, ..., and a lane ends with 8 dims in a row, one 16-byte store.
//
// Everything that follows the block ids comes through LDS (query rows and
// scales too) and is waited for by count, in the order of issue, so that no
// wait of the compiler's drains the tiles behind it.
//
// Bound by the tiles' intake, us a call with the merge's launch (the bytes at the
// 7.0 TB/s of a contiguous read): 64 rows of 512 to 2048 tokens 26.8 (19.1), 16 x
// 5 of 256 to 4096 18.8 (7.5), 16 x 9 of 1024 to 32768 61.2 (36.8), one row of
// 32768 17.7 (9.6).  The loads and waits alone, without arithmetic, took 24.6,
// 18.0, 52.7 and 18.6 where the kernel (of then) took 27.2, 20.5, 59.7 and 20.0.  A piece
// begins with 3 us of latency (ids, then tiles), or 8 to 9 in a compute unit's
// second workgroup, whose first tiles come behind the burst of everyone's, and
// ends with 1 to 2.6 of merge; the merge launch takes 3 to 4.
//
// Other forms, us in that order unless said, of the kernel with one fp16 number a
// weight:
//   tiles straight into registers, a pair ahead (spills, and a wait for every
//     load at the loop's head): 30.3, 23.3, 85.3 and 22.4 against 28.5, 20.1, 59.4
//     and 19.9
//   four slots a wave (the LDS given at launch: where a kernel's own size leaves
//     one workgroup a compute unit, the compiler moves accumulators between two
//     register files, 16 x 5 16.6 -> 18.9): 32.1, 18.6, 73.0 and 19.6 against 27.2,
//     16.6, 60.6 and 18.1; issuing them all delays the first
//   without nt (a block is read once): 30.9 against 27.7 (64 rows)
//   one workgroup of eight waves a compute unit: 18.7 against 16.9 (16 x 5)
//   the refill behind the products: 16 x 9 -2.7%, 16 x 5 +2%
//   K tiles before V tiles, both in one 4 KB run, scores scaled before the
//     maximum: no difference
#include "nsd_kv8_device.h"
#include "nsd_paged.h"

namespace nsd {
namespace {

struct Kv8Caches {
  const char* k;
  const char* v;
  const uint8_t* ks;
  const uint8_t* vs;
  uint32_t ks_low, vs_low;  // the scales' addresses modulo 4
};

constexpr int kSlot = 4 * kKv8Tile;  // a pair's K tiles, then its V tiles
constexpr int kSlots = 2;
constexpr int kRing = kSlots * kSlot;           // a wave's
constexpr int kScales = 2 * kWave * 4;          // a wave's words with the K and V scales of its blocks
// The waves' rings, the query rows and scales.
constexpr int lds_bytes(int nt) { return kWaves * (kRing + kScales) + nt * 16 * D * 2; }
static_assert(kMergeWave <= kRing, "the merge reuses the rings");
static_assert(2 * lds_bytes(3) <= 160 * 1024, "two workgroups a CU");

// A tile from base + off (a lane's 16 bytes), 1 KB of rows or 64 dwords into LDS;
// the compiler sees neither the loads nor their wait.  Nor does it put the wait
// states that a load to LDS needs behind a write of m0 (one), or of its base by a
// VALU (five).  An offset counts in memory and in LDS: one m0 a tile (one a KB 64 x 1
// 28.1, 27.9 so; 16 x 5 20.0 and 19.85).
__device__ inline void dma_tile(uint32_t lds, const char* base, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2 nt\n\t"
               "global_load_lds_dwordx4 %1, %2 offset:1024 nt"
               : : "s"(lds), "v"(off), "s"(base) : "memory", "m0");
}
__device__ inline void dma16_rows(uint32_t lds, const void* at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               : : "s"(lds), "v"(at) : "memory", "m0");
}
__device__ inline void dma4(uint32_t lds, const void* at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
               : : "s"(lds), "v"(at) : "memory", "m0");
}
template <int N>
__device__ inline void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// A weight goes into the product as two fp16 numbers, itself rounded and what that
// left: off by 2^-22 of itself at most, or by 2^-25 under the smallest normal
// number.  The running maximum's own weight is 2^7, so that the latter is 2^-32 of
// it; the largest, with the lazy maximum, is 2^15.  Outputs then differ from 64 bits
// by their own rounding alone (1.8 to 2.3e-4 of the norm, as fp32 weights'); from
// fp32 weights' outputs by 2e-6 to 4e-5.  One fp16 number: 2.1 to 2.9e-4 and 1.6 to
// 3.2e-4, and the second product's time less, 16 x 5 19.1 for 19.85 us and 16 x 9 59.4
// for 62.7 in a graph, one tile 0.2 for any length.
typedef float f32x2 __attribute__((ext_vector_type(2)));
constexpr float kWeightTop = 7.f;
static_assert(kLazyMax + kWeightTop < 16.f, "fp16 holds 2^15");

// 0x80 in the bytes of four E4M3 codes that are NaN; and fp16 ones for bytes of
// 1 (zeros for 0).
__device__ inline uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
__device__ inline f16x4 ones_of(uint32_t w) {
  w *= 0x3cu;  // the high byte of 1.0
  const u32x2 h = {__builtin_amdgcn_perm(0u, w, 0x010c000cu), __builtin_amdgcn_perm(0u, w, 0x030c020cu)};
  return __builtin_bit_cast(f16x4, h);
}

// A piece table of plans with few pieces.  A launch whose arguments are less than
// 1 KB costs the host less: 2.7 to 3.5 us against 3.9, and a short batch's call is
// the host's.
struct ShortTable {
  uint32_t e[160];
};
static_assert(sizeof(AttnArgs) + sizeof(Kv8Caches) + sizeof(ShortTable) < 1024, "a small launch");

template <int T, int NT, class Table>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2)))
void kv8_attn_kernel(AttnArgs a, Kv8Caches cache, Table pt) {
  __shared__ __align__(16) char smem[lds_bytes(NT)];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  lds_char* lds = (lds_char*)smem;
  lds_char* ring = lds + wave * kRing;
  const lds_char* q_lds = lds + kWaves * kRing;
  const lds_char* scale_lds = q_lds + NT * 16 * D * 2 + wave * kScales;

  // every argument, and the piece's table entry, in one round of scalar loads:
  // left to the compiler they came in four, each a trip to memory
  const uint32_t entry = pt.e[min((int)blockIdx.x, (int)(sizeof(pt.e) / sizeof(uint32_t)) - 1)];
  asm volatile("" ::"s"(a.q), "s"(a.bt), "s"(a.bt_stride), "s"(a.pieces), "s"(a.n_static), "s"(a.n_claimed),
               "s"(a.piece_table), "s"(a.num_blocks), "s"(a.num_layers), "s"(a.layer), "s"(a.hq), "s"(a.hkv),
               "s"(a.gqa), "s"(a.scale_log2), "s"(cache.k), "s"(cache.v), "s"(cache.ks), "s"(cache.vs),
               "s"(cache.ks_low), "s"(cache.vs_low), "s"(entry));

  int rec_idx = blockIdx.x;
  if (rec_idx >= a.n_static) {
    // claim the next record: one device-scope add per workgroup; the last
    // workgroup to claim sets the counter back to zero for the next call
    __shared__ int s_ticket;
    if (threadIdx.x == 0) {
      const int t = __hip_atomic_fetch_add(a.claim, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (t == a.n_claim_wgs - 1) __hip_atomic_store(a.claim, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      s_ticket = t;
    }
    __syncthreads();
    const int t = s_ticket;
    if (t >= a.n_claimed) return;
    rec_idx = a.n_static + t;
  }
  // a static workgroup with the table reads block ids right away (lanes past
  // the piece read a clamped, in-row column and are discarded below)
  const bool tabled = a.piece_table != 0 && (int)blockIdx.x < a.n_static;
  int tab_id = 0;
  if (tabled) {
    int64_t col = (int64_t)(entry >> 16) + wave + kWaves * lane;
    col = col < a.bt_stride ? col : a.bt_stride - 1;
    tab_id = a.bt[(int64_t)(entry & 0xffffu) * a.bt_stride + col];
  }
  // the whole record in one round of scalar loads
  using const_i32p = const __attribute__((address_space(4))) int32_t*;
  const const_i32p rec =
      (const_i32p)(uintptr_t)(a.pieces + (int64_t)__builtin_amdgcn_readfirstlane(rec_idx) * kPieceWords);
  int32_t rv[kPieceWords];
#pragma unroll
  for (int i = 0; i < kPieceWords; ++i) rv[i] = rec[i];
  asm volatile("" ::"s"(rv[0]), "s"(rv[1]), "s"(rv[2]), "s"(rv[3]), "s"(rv[4]), "s"(rv[5]), "s"(rv[6]),
               "s"(rv[7]), "s"(rv[8]), "s"(rv[9]), "s"(rv[10]), "s"(rv[11]));
  const int q_len = rv[kPieceQLen];
  if (q_len == 0) return;  // an empty record
  const int head = rv[kPieceHead], blk0 = rv[kPieceBlkBegin];
  const int nb = rv[kPieceBlkEnd] - blk0;  // 1 .. kMaxPieceBlocks (host-checked)
  const int my_n = nb > wave ? (nb - wave + kWaves - 1) / kWaves : 0;  // this wave's blocks
  const int pairs = (my_n + 1) / 2;
  const int row_start = rv[kPieceRowStart], ctx = rv[kPieceCtx];
  const int lr = lane & 15;
  const int lg = lane >> 4;
  const int n_rows = q_len * a.gqa;

  // Block ids of this wave's blocks (block wave + 4i on lane i).
  int blk_id = tab_id;
  if (!tabled && lane < my_n) blk_id = a.bt[(int64_t)rv[kPieceSeqId] * a.bt_stride + blk0 + wave + kWaves * lane];
  // The query rows of 16-row tiles as the B operand of the score product, shared
  // by the waves: lane (lr, lg) of fragment kk holds dims 64 (kk % 2) + 8 (4 (kk /
  // 2) + lg) .. +7 of row lr; wave w brings fragment w of every tile.  Rows past
  // the group read its row 0 and are never stored.
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int n = 16 * t + lr;
    const int nr = n < n_rows ? n : 0;
    const int qi = nr / a.gqa, gh = nr - qi * a.gqa;
    const f16* qrow = a.q + ((int64_t)(row_start + qi) * a.hq + head * a.gqa + gh) * D;
    dma16_rows((uint32_t)(uintptr_t)q_lds + (4 * t + wave) * 1024, qrow + 64 * (wave & 1) + 8 * (4 * (wave >> 1) + lg));
  }
  const bool bad = lane < my_n && (blk_id < 0 || blk_id >= a.num_blocks);
  const uint64_t bad_mask = __builtin_amdgcn_ballot_w64(bad);
  // the block's tile, of fewer than 2^31 (host-checked); tile 0, masked, for
  // ids outside the pool
  const int tile = lane < my_n && !bad ? (blk_id * a.num_layers + a.layer) * a.hkv + head : 0;
  // the aligned words with its scales
  dma4((uint32_t)(uintptr_t)scale_lds, cache.ks + (((uint32_t)tile + cache.ks_low) & ~3u) - cache.ks_low);
  dma4((uint32_t)(uintptr_t)scale_lds + 256, cache.vs + (((uint32_t)tile + cache.vs_low) & ~3u) - cache.vs_low);

  // pair p's tiles into its slot, 8 loads (4 if it has one block)
  auto issue = [&](int p) __attribute__((always_inline)) {
    const uint32_t slot = (uint32_t)(uintptr_t)ring + (p & 1) * kSlot;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      if (b == 1 && 2 * p + 1 >= my_n) break;
      const uint64_t at = (uint64_t)(uint32_t)__builtin_amdgcn_readlane(tile, 2 * p + b) * kKv8Tile;
      dma_tile(slot + b * kKv8Tile, cache.k + at, lane * 16);
      dma_tile(slot + (2 + b) * kKv8Tile, cache.v + at, lane * 16);
    }
  };
  if (pairs > 0) issue(0);
  if (pairs > 1) issue(1);
  // the query rows and scales have landed; behind them up to 16 loads
  if (my_n >= 4) wait_vm<16>();
  else if (my_n == 3) wait_vm<12>();
  else if (my_n == 2) wait_vm<8>();
  else if (my_n == 1) wait_vm<4>();
  else wait_vm<0>();
  asm volatile("s_barrier" ::: "memory");  // the other waves' query rows
  f16x8 qf[NT][4];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) qf[t][kk] = *(const lds_f16x8*)(q_lds + ((4 * t + kk) * kWave + lane) * 16);
  const uint32_t k_word = *(const lds_u32*)(scale_lds + 4 * lane);
  const uint32_t v_word = *(const lds_u32*)(scale_lds + 256 + 4 * lane);
  const int k_scale = k_word >> (8 * (((uint32_t)tile + cache.ks_low) & 3)) & 0xff;
  // a masked block's bytes may be anything, infinities under its scale too: its values are zeros
  const int v_scale = lane < my_n && !bad ? v_word >> (8 * (((uint32_t)tile + cache.vs_low) & 3)) & 0xff : 0;
  if (bad_mask != 0 && lane == 0) flag_status(a.status, NSD_STATUS_BAD_BLOCK);

  int row_len[NT];  // causal bound of this lane's row in each tile
  float m[NT], l[NT];
  f32x4 acc[NT][8];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int n = 16 * t + lr;
    row_len[t] = n < n_rows ? ctx + n / a.gqa + 1 : ctx + q_len;
    m[t] = -INFINITY;
    l[t] = 0.f;
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) acc[t][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // a weight's exponent, from its score and the row's reference, a score too: their
  // difference loses nothing where it matters, however large they are (scaled
  // scores against a scaled reference, one fused instruction: 16 x 5 19.8 us for 20.1,
  // but both are rounded to whole steps, by which weights pass fp16's largest)
  auto exponent = [&](float score, float reference) __attribute__((always_inline)) {
    return __builtin_fmaf(score - reference, a.scale_log2, kWeightTop);
  };
  float minus = -1.f;
  asm("" : "+s"(minus));  // unknown to the compiler, which has conversions and differences for a known one
  for (int p = 0; p < pairs; ++p) {
    // this pair has landed: behind it are the loads of the next
    if (2 * p + 3 < my_n) wait_vm<8>();
    else if (2 * p + 2 < my_n) wait_vm<4>();
    else wait_vm<0>();
    const lds_char* slot = ring + (p & 1) * kSlot + lane * 16;
    u32x4 kb[2][2], vb[2][2];  // [block][load]
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        kb[b][j] = *(const lds_u32x4*)(slot + b * kKv8Tile + 1024 * j);
        vb[b][j] = *(const lds_u32x4*)(slot + (2 + b) * kKv8Tile + 1024 * j);
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the slot is read
    if (p + 2 < pairs) issue(p + 2);
    // S^T of both blocks
    f32x4 s[2][NT];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const float power = kv8_power(__builtin_amdgcn_readlane(k_scale, 2 * p + b));
#pragma unroll
      for (int t = 0; t < NT; ++t) s[b][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        const u32x4 w = kb[b][kk >> 1];
        f16x8 ka;
        if constexpr (T == NSD_KV8_E4M3) {
          ka = kv8_values<T>(u32x2{w[2 * (kk & 1)], w[2 * (kk & 1) + 1]}, power);
        } else {
          f16x2 x[4];
          kv8_whole(w[2 * (kk & 1)], x[0], x[1]);
          kv8_whole(w[2 * (kk & 1) + 1], x[2], x[3]);
          ka = f16x8{x[0][0], x[0][1], x[1][0], x[1][1], x[2][0], x[2][1], x[3][0], x[3][1]};
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) s[b][t] = mfma_k32(ka, qf[t][kk], s[b][t]);
      }
      if constexpr (T == NSD_KV8_INT8) {
#pragma unroll
        for (int t = 0; t < NT; ++t) s[b][t] *= power;
      }
    }

    const int first[2] = {(blk0 + wave + kWaves * 2 * p) * BS, (blk0 + wave + kWaves * (2 * p + 1)) * BS};
    const bool masked[2] = {((bad_mask >> (2 * p)) & 1) != 0,
                            2 * p + 1 >= my_n || ((bad_mask >> ((2 * p + 1) & 63)) & 1) != 0};
    const bool edge = masked[0] || masked[1] || first[1] + BS > ctx + 1;  // a token may lie past a row's length
    f16x8 pb[NT], pl[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float sv[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) sv[e] = s[e / 4][t][e % 4];
      if (edge) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (masked[e / 4] || first[e / 4] + 4 * lg + e % 4 >= row_len[t]) sv[e] = -INFINITY;
      }
      float mx =
          fmaxf(fmaxf(fmaxf(sv[0], sv[1]), fmaxf(sv[2], sv[3])), fmaxf(fmaxf(sv[4], sv[5]), fmaxf(sv[6], sv[7])));
      mx = rows_max(mx);
      // lazy running max: one decision per wave and tile, on the largest weight's
      // exponent (-inf less itself decides nothing)
      if (__builtin_amdgcn_ballot_w64(exponent(mx, m[t]) > kLazyMax + kWeightTop) != 0) {
        const float m_new = fmaxf(m[t], mx);
        const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m[t] - m_new) * a.scale_log2);
        l[t] *= alpha;
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) acc[t][mt] *= alpha;
        m[t] = m_new;
      }
      const float m_use = m[t] == -INFINITY ? 0.f : m[t];
      float psum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        f32x2 pj;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          pj[i] = __builtin_amdgcn_exp2f(exponent(sv[e + i], m_use));
          psum += pj[i];
        }
        const f16x2 hi = __builtin_convertvector(pj, f16x2);  // a fused product and sum takes it as it is
        const f16x2 lo = {(f16)__builtin_fmaf((float)hi[0], minus, pj[0]),
                          (f16)__builtin_fmaf((float)hi[1], minus, pj[1])};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          pb[t][e + i] = hi[i];
          pl[t][e + i] = lo[i];
        }
      }
      l[t] += psum;
    }

    const float vp0 = kv8_power(__builtin_amdgcn_readlane(v_scale, 2 * p));
    const float vp1 = kv8_power(__builtin_amdgcn_readlane(v_scale, 2 * p + 1));
    if constexpr (T == NSD_KV8_E4M3) {
      // 0 times a NaN is a NaN: where a row masks tokens, NaN codes leave the
      // operand, and the dims that have them end as NaN for the rows that
      // attend them
      if (edge) {
        uint32_t found = 0;
#pragma unroll
        for (int e = 0; e < 16; ++e) found |= nan_bytes(vb[e / 8][e / 4 % 2][e % 4]);
        if (__builtin_amdgcn_ballot_w64(found != 0) != 0) {
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) {
            uint32_t has[2];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              has[b] = nan_bytes(vb[b][mt / 4][mt % 4]) >> 7;
              vb[b][mt / 4][mt % 4] &= ~(has[b] * 0xffu);
            }
            const f16x8 is_nan = kv8_join(ones_of(has[0]), ones_of(has[1]));
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              f16x8 attended = {};
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (!masked[e / 4] && first[e / 4] + 4 * lg + e % 4 < row_len[t]) attended[e] = (f16)1.f;
              const f32x4 hit = mfma_k32(is_nan, attended, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[t][mt][e] = hit[e] > 0.f ? __builtin_nanf("") : acc[t][mt][e];
            }
          }
        }
      }
    }
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) {
      const f16x8 va = kv8_join(kv8_values4<T>(vb[0][mt / 4][mt % 4], vp0), kv8_values4<T>(vb[1][mt / 4][mt % 4], vp1));
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t][mt] = mfma_k32(va, pb[t], acc[t][mt]);
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t][mt] = mfma_k32(va, pl[t], acc[t][mt]);
    }
  }

  // Merge the waves' states, one row tile at a time, in wave order.  Lane (lr, lg)
  // of tile m holds dims 8 (4lg + r) + m of row lr in element r: wave w takes the
  // elements r = w, the dims 32lg + 8w .. +7.  (All tiles in one exchange: no
  // faster.)
  const int slot = rv[kPieceSlot];
  float* mrg = (float*)smem;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const float lt = rows_sum(l[t]);
    __syncthreads();  // the ring, or the previous tile's merge, is read
    float* mine = mrg + wave * (kMergeWave / 4);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<f32x4*>(mine + ((2 * r + h) * kWave + lane) * 4) =
            f32x4{acc[t][4 * h][r], acc[t][4 * h + 1][r], acc[t][4 * h + 2][r], acc[t][4 * h + 3][r]};
    if (lg == 0) {
      mine[kMergeAcc / 4 + lr] = m[t];
      mine[kMergeAcc / 4 + 16 + lr] = lt;
    }
    __syncthreads();
    float mw[kWaves], lw[kWaves];
    float M = -INFINITY;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      mw[v] = mrg[v * (kMergeWave / 4) + kMergeAcc / 4 + lr];
      lw[v] = mrg[v * (kMergeWave / 4) + kMergeAcc / 4 + 16 + lr];
      M = fmaxf(M, mw[v]);
    }
    float L = 0.f, sc[kWaves];
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      sc[v] = mw[v] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mw[v] - M) * a.scale_log2);
      L += lw[v] * sc[v];
    }
    const int n = 16 * t + lr;
    if (n < n_rows) {
      const float inv = L > 0.f ? 1.f / L : L != L ? L : 0.f;
      const int qi = n / a.gqa, gh = n - qi * a.gqa;
      const int64_t orow = (int64_t)(row_start + qi) * a.hq + head * a.gqa + gh;
      f32x4 out[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        out[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int v = 0; v < kWaves; ++v)
          out[h] +=
              *reinterpret_cast<const f32x4*>(mrg + v * (kMergeWave / 4) + ((2 * wave + h) * kWave + lane) * 4) * sc[v];
        out[h] *= inv;
      }
      const int at = 32 * lg + 8 * wave;
      if (slot < 0) {
        f16x8 half;
#pragma unroll
        for (int e = 0; e < 8; ++e) half[e] = (f16)out[e / 4][e % 4];
        *reinterpret_cast<f16x8*>(a.o + orow * D + at) = half;
      } else {  // fp32: a row is rounded once, after the merge
        float* dst = static_cast<float*>(a.part_o) + ((int64_t)slot * a.rows_max + n) * D + at;
        *reinterpret_cast<f32x4*>(dst) = out[0];
        *reinterpret_cast<f32x4*>(dst + 4) = out[1];
      }
      if (wave == 0 && lg == 0) {
        const float log_l = __log2f(L) - kWeightTop;
        const float lse2 = L > 0.f ? __builtin_fmaf(M, a.scale_log2, log_l) : L != L ? L : -INFINITY;
        if (slot >= 0) a.part_lse[(int64_t)slot * a.rows_max + n] = lse2;
        else if (a.lse != nullptr) a.lse[orow] = lse2 * kLn2;
      }
    }
  }
}

template <int T, class Table>
void launch_rows(const AttnCall& c, const Kv8Caches& caches, const Table& table, hipStream_t st) {
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(c.grid), dim3(kThreads), 0, st, c.args, caches, table);
  };
  if (c.row_tiles == 1) go(kv8_attn_kernel<T, 1, Table>);
  else if (c.row_tiles == 2) go(kv8_attn_kernel<T, 2, Table>);
  else go(kv8_attn_kernel<T, 3, Table>);
}
template <int T>
void launch_codes(AttnCall& c, const Kv8Caches& caches, hipStream_t st) {
  ShortTable few;
  constexpr int kFew = sizeof(few.e) / sizeof(few.e[0]);
  const int filled = c.args.piece_table ? c.args.n_static : 0;
  if (c.args.n_static > kFew) {
    end_table(c.pieces.e, filled);
    return launch_rows<T>(c, caches, c.pieces, st);
  }
  short_table(few.e, c.pieces.e, filled);
  launch_rows<T>(c, caches, few, st);
}

}  // namespace
}  // namespace nsd

using namespace nsd;

extern "C" int nsd_kv8_attn_workspace(const int32_t* plan_host, int64_t* bytes) {
  if (plan_host == nullptr || bytes == nullptr) return fail(NSD_ERR_INVALID, "kv8_attn_workspace: null pointer");
  if (plan_host[kPlanMagic] != kPlanMagicValue || plan_host[kPlanVersion] != kPlanVersionValue)
    return fail(NSD_ERR_INVALID, "kv8_attn_workspace: not a plan (bad magic/version)");
  const bool none = plan_host[kPlanCombines] == 0 && plan_host[kPlanClaimed] == 0;
  *bytes = none ? 0 : plan_partial_bytes(plan_host, sizeof(float));
  return NSD_OK;
}

extern "C" int nsd_kv8_paged_attention(const void* q, void* o, float* lse, const nsd_kv8_cache* cache, int layer,
                                       int num_q_heads, const int32_t* block_table, int64_t bt_rows,
                                       int64_t bt_stride, const int32_t* plan_host, const int32_t* plan_dev,
                                       void* workspace, int64_t workspace_bytes, float softmax_scale,
                                       int32_t* status, void* stream) {
  const char* who = "kv8_paged_attention";
  int rc = check_kv8_cache(who, cache, layer);
  if (rc) return rc;
  if (cache->num_blocks > INT32_MAX / cache->num_layers / cache->num_kv_heads)
    return fail(NSD_ERR_UNSUPPORTED, "%s: %lld blocks (at most 2^31 tiles)", who, (long long)cache->num_blocks);
  // masked scores, -inf, have to stay that, and a score less itself 0, in powers of two too
  if (!(softmax_scale > 0.f) || !(softmax_scale * 1.4426950408889634f < INFINITY))
    return fail(NSD_ERR_INVALID, "%s: softmax_scale=%g (a positive number)", who, (double)softmax_scale);
  AttnCall c;
  rc = prepare_attention(who, q, true, o, lse, cache->k, cache->v, cache->num_blocks, cache->num_layers, layer,
                         num_q_heads, cache->num_kv_heads, D, BS, block_table, bt_rows, bt_stride, plan_host,
                         plan_dev, workspace, workspace_bytes, sizeof(float), softmax_scale, status, &c);
  if (rc != NSD_OK || c.grid == 0) return rc;
  const Kv8Caches caches = {static_cast<const char*>(cache->k), static_cast<const char*>(cache->v),
                            static_cast<const uint8_t*>(cache->k_scales), static_cast<const uint8_t*>(cache->v_scales),
                            (uint32_t)(reinterpret_cast<uintptr_t>(cache->k_scales) & 3),
                            (uint32_t)(reinterpret_cast<uintptr_t>(cache->v_scales) & 3)};
  hipStream_t st = as_stream(stream);
  if (cache->codes == NSD_KV8_E4M3) launch_codes<NSD_KV8_E4M3>(c, caches, st);
  else launch_codes<NSD_KV8_INT8>(c, caches, st);
  rc = launch_status(who);
  if (rc != NSD_OK) return rc;
  return launch_merge<float>("kv8_paged_attention: partial merge", c, plan_host, st);
}
