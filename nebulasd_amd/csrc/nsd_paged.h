// Shared by the paged attentions over fp16 and 8-bit caches: the launch's
// arguments (filled from a checked plan), the exchanges of a wave's rows, and
// the second launch that merges the segments cut into pieces.
#pragma once

#include <algorithm>

#include "nsd_device.h"

namespace nsd {
namespace {

constexpr int D = kHeadDim;           // 128
constexpr int BS = kBlockTokens;      // 16
constexpr int kWaves = 4;             // waves per workgroup (per piece)
constexpr int kThreads = kWaves * kWave;
// End-of-piece merge of the waves' softmax states, per 16-row tile: each
// wave's accumulators (8 dim tiles x f32x4 per lane), then its row max and
// row sum (16 floats each).
constexpr int kMergeAcc = 8 * kWave * 16;
constexpr int kMergeWave = kMergeAcc + 2 * 16 * 4;
constexpr float kLn2 = 0.69314718055994531f;
constexpr float kLazyMax = 8.f;       // the running max moves only when exceeded by 2^8
constexpr int kWaitVmcnt0 = (0x7 << 4) | (0xF << 8);  // s_waitcnt vmcnt(0), other counters open
#ifndef NSD_ATTN_COMBINE_TABLE
#define NSD_ATTN_COMBINE_TABLE 1
#endif
constexpr bool kUseCombineTable = NSD_ATTN_COMBINE_TABLE != 0;
#ifndef NSD_ATTN_PIECE_TABLE
#define NSD_ATTN_PIECE_TABLE 1
#endif
constexpr bool kUsePieceTable = NSD_ATTN_PIECE_TABLE != 0;
static_assert(kMaxGroupRows <= 48, "at most three 16-row tiles per wave");
static_assert(kMaxPieceBlocks <= kWaves * kWave, "one block id per lane of its wave");

struct AttnArgs {
  const f16* q;            // [R, Hq, D]
  f16* o;                  // [R, Hq, D]
  float* lse;              // [R, Hq] natural log, optional
  const f16* k_cache;
  const f16* v_cache;
  const int32_t* bt;
  int64_t bt_stride;
  const int32_t* pieces;   // plan: piece records, one per workgroup
  void* part_o;            // [slots, rows_max, D]  normalised O, f16 or float
  float* part_lse;         // [slots, rows_max]  (log2 domain)
  const int32_t* combines; // plan: combine records of the segments cut into pieces
  int32_t* claim;          // claim counter of the claimed records (zero between calls)
  int n_static;            // workgroups below this stream the record of their index
  int n_claimed;           // records after those, claimed in order by the later workgroups
  int n_claim_wgs;         // the later workgroups (each claims once)
  int piece_table;         // 1: the static pieces' block-table positions are in the PieceTable argument
  int32_t* status;
  int64_t num_blocks;
  int64_t blk_stride;      // elements per cache block: L*Hkv*16*128
  int num_layers, layer, hq, hkv, gqa, rows_max;
  float scale_log2;        // softmax_scale * log2(e)
};

// Block-table positions of the static pieces (32 bits each: seq_id 16, first
// block 16), packed into the launch's arguments when there are at most
// kPieceTableMax of them: a workgroup's block ids then load beside its
// record instead of after it.
constexpr int kPieceTableMax = 920;
struct PieceTable {
  uint32_t e[kPieceTableMax];
};

// Max and sum over the four 16-lane rows of a wave (lanes l, l^16, l^32,
// l^48) with gfx950's row-swap moves: v_permlane16_swap pairs rows 0-1 and
// 2-3, v_permlane32_swap pairs rows 0-2 and 1-3; every lane ends with the
// same value.
__device__ inline float rows_max(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const float y = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const uint32_t v = __float_as_uint(y);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ inline float rows_sum(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const float y = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const uint32_t v = __float_as_uint(y);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Second launch: merge the partials of the segments cut into pieces, the
// same exp2-domain combine as phase 2 of the reference
// (paged_attn.py:128-149).  The kernel boundary orders it after every partial
// store of the attention launch.
//
// Threads per (row, 8 dims) of the merge: one while a segment's slots are one
// round of a thread's loads (8), else four (up to 32 slots) or sixteen.  The
// merge is latency-bound, and a round is one more trip to memory: one request
// of 32k tokens, 64 slots a segment, took 8.1 us with one thread in eight
// rounds and takes 3.9 with sixteen threads in one; 9 to 17 slots (ragged
// verify) 4.6 either way.
constexpr int kMergeSlots = 8;

// Eight dims of a partial, f16 or float, as they are loaded and as values; zeros
// if it is a repeated slot's, which may hold an infinity (0 * inf).
struct Part {
  f32x4 lo, hi;
};
__device__ inline f16x8 loaded(const f16* p) { return *reinterpret_cast<const f16x8*>(p); }
__device__ inline Part loaded(const float* p) {
  return {*reinterpret_cast<const f32x4*>(p), *reinterpret_cast<const f32x4*>(p + 4)};
}
// What was loaded is in registers from here on.
__device__ inline void arrived(const f16x8& h) { asm volatile("" ::"v"(h)); }
__device__ inline void arrived(const Part& v) { asm volatile("" ::"v"(v.lo), "v"(v.hi)); }
__device__ inline Part part_of(f16x8 h, bool use) {
  if (!use) h = f16x8{};
  return {f32x4{(float)h[0], (float)h[1], (float)h[2], (float)h[3]},
          f32x4{(float)h[4], (float)h[5], (float)h[6], (float)h[7]}};
}
__device__ inline Part part_of(const Part& v, bool use) {
  return use ? v : Part{f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
}
// A merged row's 1 / W; 0 where no slot attends a token (ids outside the pool).
__device__ inline float merge_inv(float W) { return W == 0.f ? 0.f : 1.f / W; }

// Row n (of the segment's q_len x GQA rows), dims 8 d8 .. 8 d8 + 7, of a
// split segment of kv head `head` whose partials sit in slots [first, first
// + n_slots), at most kMergeSlots: their loads all in flight, the slots
// folded in slot order (log-sum-exp) and the row stored.
template <class P>
__device__ inline void merge_row(const AttnArgs& a, int head, int first, int n_slots, int row_start, int n,
                                 int d8) {
  const P* po = static_cast<const P*>(a.part_o) + ((int64_t)first * a.rows_max + n) * D + 8 * d8;
  const float* pl = a.part_lse + (int64_t)first * a.rows_max + n;
  const int64_t sstride = (int64_t)a.rows_max * D;  // elements between slots
  f32x4 v0[kMergeSlots], v1[kMergeSlots];
  float ls[kMergeSlots];
  decltype(loaded(po)) raw[kMergeSlots];
#pragma unroll
  for (int u = 0; u < kMergeSlots; ++u) {
    const int sidx = u < n_slots ? u : 0;
    ls[u] = pl[(int64_t)sidx * a.rows_max];
    raw[u] = loaded(po + sidx * sstride);
  }
  // all of them, before any is looked at: with a branch around the loads of slots
  // that there are not, the first was waited for before the second
#pragma unroll
  for (int u = 0; u < kMergeSlots; ++u) {
    asm volatile("" ::"v"(ls[u]));
    arrived(raw[u]);
  }
#pragma unroll
  for (int u = 0; u < kMergeSlots; ++u) {
    const Part v = part_of(raw[u], u < n_slots);
    ls[u] = u < n_slots ? ls[u] : -INFINITY;
    v0[u] = v.lo;
    v1[u] = v.hi;
  }
  float M = -INFINITY, W = 0.f;
#pragma unroll
  for (int u = 0; u < kMergeSlots; ++u) M = fmaxf(M, ls[u]);
  // slot 0 holds token 0, which every row attends: -inf only where its block's
  // id is outside the pool, as all the others' are
  const float use = M == -INFINITY ? 0.f : M;
  f32x4 acc0 = {0.f, 0.f, 0.f, 0.f}, acc1 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < kMergeSlots; ++u) {
    const float wgt = exp2f(ls[u] - use);
    acc0 += v0[u] * wgt;
    acc1 += v1[u] * wgt;
    W += wgt;
  }
  const float inv = merge_inv(W);
  const int qi = n / a.gqa, gh = n - qi * a.gqa;
  const int64_t orow = (int64_t)(row_start + qi) * a.hq + head * a.gqa + gh;
  f16x8 hv = {(f16)(acc0[0] * inv), (f16)(acc0[1] * inv), (f16)(acc0[2] * inv),
              (f16)(acc0[3] * inv), (f16)(acc1[0] * inv), (f16)(acc1[1] * inv),
              (f16)(acc1[2] * inv), (f16)(acc1[3] * inv)};
  *reinterpret_cast<f16x8*>(a.o + orow * D + 8 * d8) = hv;
  if (d8 == 0 && a.lse != nullptr) a.lse[orow] = (M + __log2f(W)) * kLn2;
}

// A partly merged row: running max (log2), sum of weights, 8 dims.
struct MergeState {
  float M, W;
  f32x4 lo, hi;
};
__device__ inline void merge_states(MergeState& a, float M2, float W2, f32x4 lo2, f32x4 hi2) {
  const float M = fmaxf(a.M, M2);
  const float use = M == -INFINITY ? 0.f : M;  // neither holds a slot
  const float s1 = exp2f(a.M - use), s2 = exp2f(M2 - use);
  a.lo = a.lo * s1 + lo2 * s2;
  a.hi = a.hi * s1 + hi2 * s2;
  a.W = a.W * s1 + W2 * s2;
  a.M = M;
}

// merge_row for segments of many slots: SL threads take slots sl, sl + SL,
// ... of a (row, 8 dims) each, and their states are merged over the wave's
// 16-lane rows and, past four threads, over the workgroup's waves in LDS, in a
// fixed order.
template <int SL, class P>
__device__ inline void merge_row_wide(const AttnArgs& a, int head, int first, int n_slots, int row_start, int n,
                                      int n_rows, int d8, int sl) {
  const int nr = n < n_rows ? n : 0;  // every thread takes part in the exchanges
  const P* po = static_cast<const P*>(a.part_o) + ((int64_t)first * a.rows_max + nr) * D + 8 * d8;
  const float* pl = a.part_lse + (int64_t)first * a.rows_max + nr;
  MergeState st = {-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
  for (int s0 = sl; s0 < n_slots; s0 += 4 * SL) {
    float ls[4];
    Part h[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int s = s0 + SL * u;
      const int at = s < n_slots ? s : s0;
      ls[u] = s < n_slots ? pl[(int64_t)at * a.rows_max] : -INFINITY;
      h[u] = part_of(loaded(po + (int64_t)at * a.rows_max * D), s < n_slots);
    }
    const float M = fmaxf(fmaxf(fmaxf(ls[0], ls[1]), fmaxf(ls[2], ls[3])), st.M);
    const float use = M == -INFINITY ? 0.f : M;
    const float keep = exp2f(st.M - use);
    st.lo *= keep;
    st.hi *= keep;
    st.W *= keep;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float wgt = exp2f(ls[u] - use);
      st.lo += h[u].lo * wgt;
      st.hi += h[u].hi * wgt;
      st.W += wgt;
    }
    st.M = M;
  }
#pragma unroll
  for (int m = 16; m <= 32; m <<= 1) {  // the wave's four 16-lane rows
    f32x4 lo, hi;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      lo[e] = __shfl_xor(st.lo[e], m, kWave);
      hi[e] = __shfl_xor(st.hi[e], m, kWave);
    }
    const float M2 = __shfl_xor(st.M, m, kWave), W2 = __shfl_xor(st.W, m, kWave);
    merge_states(st, M2, W2, lo, hi);
  }
  if constexpr (SL == 16) {
    __shared__ MergeState s_wave[4][16];
    if ((threadIdx.x & 63) < 16) s_wave[threadIdx.x >> 6][d8] = st;
    __syncthreads();
    if (threadIdx.x >= 16) return;
#pragma unroll
    for (int v = 1; v < 4; ++v) merge_states(st, s_wave[v][d8].M, s_wave[v][d8].W, s_wave[v][d8].lo, s_wave[v][d8].hi);
  }
  if (n >= n_rows || sl != 0) return;
  const float inv = merge_inv(st.W);
  const int qi = n / a.gqa, gh = n - qi * a.gqa;
  const int64_t orow = (int64_t)(row_start + qi) * a.hq + head * a.gqa + gh;
  f16x8 hv;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    hv[e] = (f16)(st.lo[e] * inv);
    hv[e + 4] = (f16)(st.hi[e] * inv);
  }
  *reinterpret_cast<f16x8*>(a.o + orow * D + 8 * d8) = hv;
  if (d8 == 0 && a.lse != nullptr) a.lse[orow] = (st.M + __log2f(st.W)) * kLn2;
}

// Row group `group` of a segment, SL threads per (row, 8 dims): 16 / SL rows
// a workgroup.
template <int SL, class P>
__device__ inline void merge_group(const AttnArgs& a, int head, int first, int n_slots, int row_start, int n_rows,
                                   int group) {
  const int d8 = threadIdx.x & 15, p = threadIdx.x >> 4;
  const int n = group * (16 / SL) + p / SL;
  if constexpr (SL == 1) {
    if (n < n_rows) merge_row<P>(a, head, first, n_slots, row_start, n, d8);
  } else {
    if (group * (16 / SL) < n_rows) merge_row_wide<SL, P>(a, head, first, n_slots, row_start, n, n_rows, d8, p % SL);
  }
}

// Workgroup (c, g) merges row group g of combine record c.
template <int SL, class P>
__global__ __launch_bounds__(256) void combine_kernel(AttnArgs a, int row_groups) {
  const int32_t* c = a.combines + kPieceWords * (blockIdx.x / row_groups);
  merge_group<SL, P>(a, c[kCombHead], c[kCombFirst], c[kCombSlots], c[kCombRowStart], c[kCombQLen] * a.gqa,
                  blockIdx.x % row_groups);
}

// The combine records of plans with at most kCombineTableMax of them, packed
// into the launch's arguments (64 bits each: first slot 20, slots 8, kv head
// 8, first row 20, q_len 8), so that a workgroup reads its record with the
// arguments instead of one more dependent load.  Few of them in a table of their
// own: a launch of less than 1 KB of arguments costs the host 0.4 to 0.8 us less.
constexpr int kCombineTableMax = 448, kCombineTableFew = 96;
template <int N>
struct CombineTable {
  uint64_t e[N];
};
static_assert(sizeof(AttnArgs) + sizeof(CombineTable<kCombineTableFew>) < 1024, "a small launch");

// Workgroup (c, g) = (blockIdx.x, blockIdx.y): the entry's address depends on
// the workgroup index alone, so it loads with the other arguments.
template <int SL, class P, int N>
__global__ __launch_bounds__(256) void combine_table_kernel(AttnArgs a, CombineTable<N> tab) {
  const uint64_t e = tab.e[blockIdx.x];
  // the arguments in one round of loads with it
  asm volatile("" ::"s"(e), "s"(a.gqa), "s"(a.part_o), "s"(a.part_lse), "s"(a.rows_max), "s"(a.o), "s"(a.lse), "s"(a.hq));
  merge_group<SL, P>(a, (int)((e >> 28) & 0xff), (int)(e & 0xfffff), (int)((e >> 20) & 0xff), (int)((e >> 36) & 0xfffff),
                  (int)(e >> 56) * a.gqa, (int)blockIdx.y);
}

// Workspace bytes a plan needs: the claim counter (when it has claimed
// records) and the partials.
inline int64_t plan_partial_bytes(const int32_t* plan_host, int elem = 2) {
  return plan_workspace_bytes(plan_host[kPlanSlots], plan_host[kPlanRowsMax], elem);
}

// A checked call: what its launch is given.
struct AttnCall {
  AttnArgs args;
  PieceTable pieces;
  int grid = 0;      // 0: no rows, nothing to launch
  int row_tiles;     // 16-row tiles of a segment: 1 .. 3
  int n_combine;     // segments cut into pieces
};

// Checks the arguments and the plan of an attention call (`part` holds the
// partials, `part_capacity` bytes, of values of `part_elem` bytes) and fills *c.
inline int prepare_attention(const char* who, const void* q, bool needs_q, void* o, float* lse, const void* k_cache,
                             const void* v_cache, int64_t num_blocks, int num_layers, int layer, int num_q_heads,
                             int num_kv_heads, int head_dim, int block_size, const int32_t* block_table,
                             int64_t bt_rows, int64_t bt_stride, const int32_t* plan_host, const int32_t* plan_dev,
                             void* part, int64_t part_capacity, int part_elem, float softmax_scale, int32_t* status,
                             AttnCall* c) {
  if (head_dim != D) return fail(NSD_ERR_UNSUPPORTED, "%s: head_dim=%d (only 128)", who, head_dim);
  if (block_size != BS)
    return fail(NSD_ERR_UNSUPPORTED, "%s: block_size=%d (only 16)", who, block_size);
  if (!plan_host || !plan_dev) return fail(NSD_ERR_INVALID, "%s: null plan", who);
  if (plan_host[kPlanMagic] != kPlanMagicValue || plan_host[kPlanVersion] != kPlanVersionValue)
    return fail(NSD_ERR_INVALID, "%s: not a plan (bad magic/version)", who);
  if (plan_host[kPlanHq] != num_q_heads || plan_host[kPlanHkv] != num_kv_heads)
    return fail(NSD_ERR_INVALID, "%s: plan built for Hq=%d Hkv=%d, called with %d/%d", who,
                plan_host[kPlanHq], plan_host[kPlanHkv], num_q_heads, num_kv_heads);
  if (num_layers <= 0 || layer < 0 || layer >= num_layers || num_blocks <= 0 || bt_stride <= 0 ||
      bt_rows <= 0)
    return fail(NSD_ERR_INVALID,
                "%s: layer=%d of %d, blocks=%lld, block table %lld x %lld", who, layer,
                num_layers, (long long)num_blocks, (long long)bt_rows, (long long)bt_stride);
  const int grid = plan_host[kPlanWorkers];
  const int n_combine = plan_host[kPlanCombines];
  const int rows_max = plan_host[kPlanRowsMax];
  const int n_rows_plan = plan_host[kPlanRows];
  if (n_rows_plan == 0 || grid == 0) return NSD_OK;  // c->grid 0: nothing to launch
  if ((needs_q && !q) || !o || !k_cache || !v_cache || !block_table)
    return fail(NSD_ERR_INVALID, "%s: null pointer", who);
  if ((needs_q && !aligned16(q)) || !aligned16(o) || !aligned16(k_cache) || !aligned16(v_cache))
    return fail(NSD_ERR_INVALID, "%s: q/o/caches must be 16-byte aligned", who);
  const int nt = (rows_max + 15) / 16;
  const int64_t n_slots = plan_host[kPlanSlots];
  const int n_static = plan_host[kPlanStatic], n_claimed = plan_host[kPlanClaimed];
  const int n_records = plan_host[kPlanPieces];
  if (rows_max < 1 || rows_max > kMaxGroupRows || n_static < 0 || n_static % kXcds != 0 || n_claimed < 0 ||
      n_records != n_static + n_claimed || grid < n_records || (n_claimed == 0 && grid != n_static) ||
      plan_host[kPlanMaxBlocks] < 1 || plan_host[kPlanMaxBlocks] > kMaxPieceBlocks || n_slots < 0 ||
      n_combine < 0)
    return fail(NSD_ERR_INVALID, "%s: corrupt plan header", who);
  if (plan_host[kPlanBtStride] != bt_stride || plan_host[kPlanBtRows] > bt_rows)
    return fail(NSD_ERR_INVALID,
                "%s: plan built for a block table of %d rows x %d, called with "
                "%lld x %lld", who,
                plan_host[kPlanBtRows], plan_host[kPlanBtStride], (long long)bt_rows,
                (long long)bt_stride);
  // the kernel trusts the records it streams blocks from: check every one
  // against the buffers it will touch
  const int gqa = num_q_heads / num_kv_heads;
  const int32_t* pr = plan_host + plan_host[kPlanOffPieces];
  for (int i = 0; i < n_records; ++i) {
    const int32_t* r = pr + kPieceWords * i;
    if (r[kPieceQLen] == 0) continue;  // an empty record: its workgroup exits at once
    const int nb = r[kPieceBlkEnd] - r[kPieceBlkBegin];
    const bool split_ok =
        r[kPieceSlot] < 0 ||
        (r[kPieceComb] >= 0 && r[kPieceComb] < n_combine && r[kPieceCombFirst] >= 0 &&
         r[kPieceCombSlots] >= 2 && r[kPieceCombFirst] + (int64_t)r[kPieceCombSlots] <= n_slots &&
         r[kPieceSlot] >= r[kPieceCombFirst] && r[kPieceSlot] < r[kPieceCombFirst] + r[kPieceCombSlots]);
    if (r[kPieceBlkBegin] < 0 || nb < 1 || nb > kMaxPieceBlocks || r[kPieceBlkEnd] > bt_stride ||
        r[kPieceSeqId] < 0 || r[kPieceSeqId] >= bt_rows || r[kPieceHead] < 0 ||
        r[kPieceHead] >= num_kv_heads || r[kPieceQLen] < 1 || (int64_t)r[kPieceQLen] * gqa > rows_max ||
        r[kPieceRowStart] < 0 || (int64_t)r[kPieceRowStart] + r[kPieceQLen] > n_rows_plan ||
        r[kPieceCtx] < 0 || !split_ok)
      return fail(NSD_ERR_INVALID, "%s: corrupt plan (piece %d)", who, i);
  }
  // ... and every combine record against the partials and the output rows
  const int32_t* cr = plan_host + plan_host[kPlanOffCombines];
  for (int c = 0; c < n_combine; ++c) {
    const int32_t* r = cr + kPieceWords * c;
    if (r[kCombHead] < 0 || r[kCombHead] >= num_kv_heads || r[kCombFirst] < 0 ||
        r[kCombSlots] < 2 || (int64_t)r[kCombFirst] + r[kCombSlots] > n_slots ||
        r[kCombQLen] < 1 || (int64_t)r[kCombQLen] * gqa > rows_max || r[kCombRowStart] < 0 ||
        (int64_t)r[kCombRowStart] + r[kCombQLen] > n_rows_plan)
      return fail(NSD_ERR_INVALID, "%s: corrupt plan (combine %d)", who, c);
  }
  const int64_t part_bytes = plan_partial_bytes(plan_host, part_elem);
  if ((n_combine > 0 || n_claimed > 0) && (part == nullptr || part_capacity < part_bytes || !aligned16(part)))
    return fail(NSD_ERR_WORKSPACE,
                "%s: workspace holds %lld partial bytes, the plan needs %lld", who,
                (long long)part_capacity, (long long)part_bytes);

  AttnArgs& args = c->args;
  args.q = static_cast<const f16*>(q);
  args.o = static_cast<f16*>(o);
  args.lse = lse;
  args.k_cache = static_cast<const f16*>(k_cache);
  args.v_cache = static_cast<const f16*>(v_cache);
  args.bt = block_table;
  args.bt_stride = bt_stride;
  args.pieces = plan_dev + plan_host[kPlanOffPieces];
  char* ws = static_cast<char*>(part);
  args.claim = n_claimed > 0 ? reinterpret_cast<int32_t*>(ws) : nullptr;
  args.n_static = n_static;
  args.n_claimed = n_claimed;
  args.n_claim_wgs = grid - n_static;
  args.part_o = ws + kClaimBytes;
  args.part_lse = reinterpret_cast<float*>(ws + kClaimBytes + n_slots * rows_max * D * part_elem);
  args.combines = plan_dev + plan_host[kPlanOffCombines];
  args.status = status;
  args.num_blocks = num_blocks;
  args.blk_stride = (int64_t)num_layers * num_kv_heads * BS * D;
  args.num_layers = num_layers;
  args.layer = layer;
  args.hq = num_q_heads;
  args.hkv = num_kv_heads;
  args.gqa = gqa;
  args.rows_max = rows_max;
  args.scale_log2 = softmax_scale * 1.4426950408889634f;

  // the static pieces' block-table positions, when they fit the arguments
  PieceTable& pt = c->pieces;
  args.piece_table = kUsePieceTable && n_static <= kPieceTableMax ? 1 : 0;
  for (int i = 0; args.piece_table && i < n_static; ++i) {
    const int32_t* r = pr + kPieceWords * i;
    const bool live = r[kPieceQLen] != 0;
    const int32_t sid = live ? r[kPieceSeqId] : 0, b0 = live ? r[kPieceBlkBegin] : 0;
    if (sid >= (1 << 16) || b0 >= (1 << 16)) {
      args.piece_table = 0;
      break;
    }
    pt.e[i] = (uint32_t)sid | (uint32_t)b0 << 16;
  }
  c->grid = grid;
  c->row_tiles = nt;
  c->n_combine = n_combine;
  return NSD_OK;
}

// The second launch: every segment cut into pieces is merged (none: nothing).
// P: the partials' type.
template <class P>
int launch_merge(const char* who, const AttnCall& call, const int32_t* plan_host, hipStream_t st) {
  const int n_combine = call.n_combine;
  if (n_combine == 0) return NSD_OK;
  const AttnArgs& args = call.args;
  const int32_t* crec = plan_host + plan_host[kPlanOffCombines];
  bool packed = kUseCombineTable && n_combine <= kCombineTableMax;
  int most_slots = 0;
  for (int c = 0; c < n_combine; ++c) most_slots = std::max(most_slots, (int)crec[kPieceWords * c + kCombSlots]);
  CombineTable<kCombineTableMax> tab;
  for (int c = 0; packed && c < n_combine; ++c) {
    const int32_t* r = crec + kPieceWords * c;
    if (r[kCombFirst] >= (1 << 20) || r[kCombSlots] >= 256 || r[kCombHead] >= 256 || r[kCombRowStart] >= (1 << 20) ||
        r[kCombQLen] >= 256) {
      packed = false;
      break;
    }
    tab.e[c] = (uint64_t)r[kCombFirst] | (uint64_t)r[kCombSlots] << 20 | (uint64_t)r[kCombHead] << 28 |
               (uint64_t)r[kCombRowStart] << 36 | (uint64_t)r[kCombQLen] << 56;
  }
  auto merge = [&](auto slc) {
    constexpr int SL = decltype(slc)::value;
    const int groups = (args.rows_max * SL + 15) / 16;
    if (packed && n_combine <= kCombineTableFew) {
      CombineTable<kCombineTableFew> few;
      short_table(few.e, tab.e, n_combine);
      hipLaunchKernelGGL((combine_table_kernel<SL, P, kCombineTableFew>), dim3(n_combine, groups), dim3(256), 0, st,
                         args, few);
    } else if (packed) {
      end_table(tab.e, n_combine);
      hipLaunchKernelGGL((combine_table_kernel<SL, P, kCombineTableMax>), dim3(n_combine, groups), dim3(256), 0, st,
                         args, tab);
    } else {
      hipLaunchKernelGGL((combine_kernel<SL, P>), dim3(n_combine * groups), dim3(256), 0, st, args, groups);
    }
  };
  if (most_slots <= kMergeSlots) merge(std::integral_constant<int, 1>{});
  else if (most_slots <= 4 * kMergeSlots) merge(std::integral_constant<int, 4>{});
  else merge(std::integral_constant<int, 16>{});
  return launch_status(who);
}

}  // namespace
}  // namespace nsd
