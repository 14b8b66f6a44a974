"""GPU parity of the 8-bit KV cache's writers, reader and attention against the oracle.

Codes, scales and values are compared bit for bit; the attention within bounds that the oracle derives from the
inputs (``oracle.kv8_attention``).
"""

from __future__ import annotations

import copy
import ctypes

import numpy as np
import pytest
import torch

import oracle
from nebulasd_amd import _lib
from nebulasd_amd.config import QWEN3_0_6B, QWEN3_8B, EngineConfig, ModelConfig
from nebulasd_amd.hostkv import CopyPlan, CopyRegion, HostKVArena, HostKVCopyBackend, swap_blocks
from nebulasd_amd.infer_state import build_infer_state, rope_cache
from nebulasd_amd.plan import AttnPlan, kv8_plan_for, plan_for
from nebulasd_amd.kernels import (KV8Cache, kv8_load, kv8_paged_attention, kv8_qk_norm_rope_store, kv8_store,
                                  paged_attention, prefill_attention, qk_norm_rope_store)

pytestmark = pytest.mark.gpu

CODES = ["e4m3", "int8"]
DTYPE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def config(hq=4, hkv=2, layers=2, blocks_per_seq=8):
    mc = ModelConfig(dict(QWEN3_8B, num_hidden_layers=layers, num_attention_heads=hq, num_key_value_heads=hkv))
    return mc, EngineConfig(max_blocks_per_seq=blocks_per_seq)


def state(mc, seq_ids, lens, prefill=(), prefill_ids=(), device="cuda"):
    cos, sin = rope_cache(128, mc.rope_theta, max([1, *lens, *prefill]), device)
    return build_infer_state(list(prefill_ids) + list(seq_ids), list(lens), list(prefill), mc, cos, sin, device)


def values_of(cache):
    """What a cache holds: float64 [blocks, layers, heads, 16, 128] of K and of V (numpy)."""
    k, v, ks, vs = cache.codes()
    two = lambda s: np.ldexp(1.0, s.cpu().numpy().astype(int) - 127)[..., None, None]  # noqa: E731
    return k.to(torch.float64).cpu().numpy() * two(ks), v.to(torch.float64).cpu().numpy() * two(vs)


def rows_of(rng, n, hkv, sizes=None):
    """fp16 rows of very different sizes."""
    x = rng.standard_normal((n, hkv, 128))
    return (x * 2.0 ** (rng.uniform(-6, 6, (n, 1, 1)) if sizes is None else sizes)).astype(np.float16)


def gpu_of(x, device="cuda"):
    return torch.from_numpy(np.ascontiguousarray(x)).to(device)


class Mirror:
    """A cache's tiles as the oracle keeps them, for one layer."""

    def __init__(self, cache, layer, codes):
        self.codes, self.layer = codes, layer
        self.held = [x[:, layer].copy() for x in values_of(cache)]
        self.known = np.zeros(self.held[0].shape[:2] + (16,), bool)  # slots whose bytes are pinned
        self.bytes = [np.zeros(self.held[0].shape, np.uint8) for _ in range(2)]
        self.power = [np.zeros(self.held[0].shape[:2], int) for _ in range(2)]

    def append(self, table, seq_ids, lens, k, v):
        where = {}
        for r, (s, n) in enumerate(zip(seq_ids, lens)):
            where.setdefault(int(table[s, (n - 1) // 16]), {})[(n - 1) % 16] = r  # a later row of a position stays
        for blk, slots in where.items():
            for h in range(k.shape[1]):
                for i, x in enumerate((k, v)):
                    self.held[i][blk, h], b, e = oracle.kv8_append(
                        self.held[i][blk, h], {t: x[r, h].astype(np.float64) for t, r in slots.items()}, self.codes)
                    self.power[i][blk, h] = e
                    top = max(slots)
                    self.bytes[i][blk, h, : top + 1] = b[: top + 1]
                self.known[blk, h, : top + 1], self.known[blk, h, top + 1:] = True, False

    def prompt(self, table, seq, k, v):
        for at in range(0, len(k), 16):
            blk = int(table[seq, at // 16])
            for h in range(k.shape[1]):
                for i, x in enumerate((k, v)):
                    part = np.zeros((16, 128))
                    part[: len(x[at:at + 16])] = x[at:at + 16, h]
                    e = oracle.kv8_exponent(part, self.codes)
                    self.held[i][blk, h], self.bytes[i][blk, h] = oracle.kv8_round(part, e, self.codes)
                    self.power[i][blk, h] = e
                self.known[blk, h] = True  # slots behind the prompt as zeros

    def check(self, cache):
        for i, (codes, scales) in enumerate(zip(cache.codes()[:2], cache.codes()[2:])):
            got = codes.view(torch.uint8)[:, self.layer].cpu().numpy()
            want = self.bytes[i]
            assert (got == want)[self.known].all(), f"{'kv'[i]}: {(got != want)[self.known].sum()} codes differ"
            some = self.known.any(-1)
            assert (scales[:, self.layer].cpu().numpy().astype(int) - 127 == self.power[i])[some].all(), "scales"

    def tokens(self, table, seq, n):
        """(k, v) float64 [n, Hkv, 128]."""
        ids = table[seq, : -(-n // 16)]
        return tuple(x[ids].transpose(0, 2, 1, 3).reshape(-1, x.shape[1], 128)[:n] for x in self.held)


def make(codes, gpu, hq=4, hkv=2, layers=2, seqs=3, blocks_per_seq=8, seed=0, pool=None):
    mc, ec = config(hq, hkv, layers, blocks_per_seq)
    rng = np.random.default_rng(seed)
    pool = pool or seqs * blocks_per_seq + 2
    table = rng.permutation(pool)[: seqs * blocks_per_seq].reshape(seqs, blocks_per_seq).astype(np.int32)
    cache = KV8Cache.allocate(pool, mc, DTYPE[codes], gpu)
    return mc, ec, rng, table, gpu_of(table), cache


# ---------------------------------------------------------------- the format


@pytest.mark.parametrize("codes", CODES)
def test_pack_and_layout(gpu, codes):
    rng = np.random.default_rng(0)
    raw = rng.integers(0, 256, (3, 2, 2, 16, 128), dtype=np.uint8)
    k, v = raw, raw[::-1].copy()
    s = gpu_of(rng.integers(100, 140, (3, 2, 2), dtype=np.uint8))
    cache = KV8Cache.pack(gpu_of(k).view(DTYPE[codes]), gpu_of(v).view(DTYPE[codes]), s, s + 1)
    assert (cache.k.cpu().numpy() == oracle.kv8_tiles(k, codes)[0]).all()
    assert (cache.v.cpu().numpy() == oracle.kv8_tiles(v, codes)[1]).all()
    kk, vv, ks, vs = cache.codes()
    assert kk.dtype == DTYPE[codes]
    assert (kk.view(torch.uint8).cpu().numpy() == k).all() and (vv.view(torch.uint8).cpu().numpy() == v).all()
    assert torch.equal(ks, s) and torch.equal(vs, s + 1)
    again = copy.deepcopy(cache)
    assert torch.equal(again.k, cache.k) and again.k.data_ptr() != cache.k.data_ptr()


@pytest.mark.parametrize("codes", CODES)
def test_every_code_under_every_scale_reads_back(gpu, codes):
    top, lo, hi = oracle.KV8_RANGES[codes]
    n = hi - lo + 1
    raw = np.tile(np.arange(256, dtype=np.uint8), (n, 8)).reshape(n, 1, 1, 16, 128)
    if codes == "int8":
        raw[raw == 128] = 0
    s = np.arange(lo, hi + 1).reshape(n, 1, 1) + 127
    raw8 = gpu_of(raw).view(DTYPE[codes])
    cache = KV8Cache.pack(raw8, raw8, gpu_of(s.astype(np.uint8)), gpu_of(s.astype(np.uint8)))
    table = gpu_of(np.arange(n, dtype=np.int32)[None])
    out = [torch.empty(16 * n, 1, 128, dtype=torch.float16, device=gpu) for _ in range(2)]
    one = lambda x: torch.tensor([x], dtype=torch.int32, device=gpu)  # noqa: E731
    kv8_load(*out, cache, table, one(0), one(0), one(16 * n), 16 * n, 0, validate=True)
    want = raw8.double().cpu().numpy()[:, 0, 0] * np.ldexp(1.0, s - 127)
    with np.errstate(over="ignore"):
        want16 = want.astype(np.float16)  # exact but for codes that no writer makes under the largest scale
    for got in out:
        assert np.array_equal(got.cpu().numpy().reshape(want16.shape), want16, equal_nan=True)


@pytest.mark.parametrize("codes", CODES)
def test_every_fp16_value_is_rounded_right(gpu, codes):
    """Blocks whose largest value is each of many fp16 values (every exponent, both sides of every border)."""
    border = [x for p in range(-24, 16) for f in (1.0, 1.5, 1.75, 1.984375) for x in (f * 2.0 ** p,)]
    border = np.array(border + [65504, 65024, 61440, 57344, 0], np.float64).astype(np.float16)
    border = border[np.isfinite(border)].view(np.uint16)
    top = np.unique(np.concatenate((border, border + 1, np.maximum(border, 1) - 1)).clip(0, 0x7bff)).view(np.float16)
    mc, ec, rng, table, bt, cache = make(codes, gpu, hkv=1, hq=1, layers=1, seqs=1, blocks_per_seq=len(top))
    x = rng.uniform(-1, 1, (len(top), 16, 128)) * top.astype(np.float64)[:, None, None]
    x[rng.random(x.shape) < 0.3] *= 2.0 ** -7
    x = x.astype(np.float16)
    x[:, 3, 5] = top
    x[1::2, 3, 5] *= -1
    x = x.reshape(-1, 1, 128)
    st = state(mc, [], [], [len(x)], [0])
    kv8_store(gpu_of(x), gpu_of(x[::-1]), cache, bt, mc, ec, st, 0, validate=True)
    m = Mirror(cache, 0, codes)
    m.prompt(table, 0, x.astype(np.float64), x[::-1].astype(np.float64))
    m.check(cache)


# ---------------------------------------------------------------- writers


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("hkv,lens", [(1, [1]), (2, [16, 33, 0, 5]), (8, [127, 15, 17, 1, 64]), (3, [100, 31])])
def test_store_prompts(gpu, codes, hkv, lens):
    mc, ec, rng, table, bt, cache = make(codes, gpu, hkv=hkv, hq=hkv, seqs=len(lens) + 1)
    cache.k.fill_(0xAB), cache.v.fill_(0xCD), cache.k_scales.fill_(9), cache.v_scales.fill_(7)
    m = Mirror(cache, 1, codes)
    ids = list(range(len(lens)))[::-1]
    k, v = rows_of(rng, sum(lens), hkv), rows_of(rng, sum(lens), hkv)
    kv8_store(gpu_of(k), gpu_of(v), cache, bt, mc, ec, state(mc, [], [], lens, ids), 1, validate=True)
    at = 0
    for s, n in zip(ids, lens):
        m.prompt(table, s, k[at:at + n].astype(np.float64), v[at:at + n].astype(np.float64))
        at += n
    m.check(cache)
    # nothing else is written: the other layer, the blocks of no prompt
    used = {int(b) for s, n in zip(ids, lens) for b in table[s, : -(-n // 16)]}
    rest = [b for b in range(cache.num_blocks) if b not in used]
    assert (cache.k[:, 0] == 0xAB).all() and (cache.v[:, 0] == 0xCD).all() and (cache.k_scales[:, 0] == 9).all()
    assert (cache.k[rest] == 0xAB).all() and (cache.v[rest] == 0xCD).all() and (cache.v_scales[rest] == 7).all()


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("hkv,seqs,q_len", [(1, 1, 1), (2, 3, 1), (8, 5, 5), (3, 4, 9), (2, 3, 17)])
def test_store_rows_step_by_step(gpu, codes, hkv, seqs, q_len):
    """Decode and verify steps over many forwards: rows accepted in part, scales that grow and shrink."""
    mc, ec, rng, table, bt, cache = make(codes, gpu, hkv=hkv, hq=hkv, seqs=seqs, seed=q_len)
    cache.k.fill_(0x7f), cache.v.fill_(0xff), cache.k_scales.fill_(250)  # what an earlier owner left
    m = Mirror(cache, 1, codes)
    have = rng.integers(0, 30, seqs)
    have[0] = 0
    ids = [s for s in range(seqs) for _ in range(int(have[s]))]
    lens = [i + 1 for s in range(seqs) for i in range(int(have[s]))]
    first = rows_of(rng, max(len(ids), 1), hkv), rows_of(rng, max(len(ids), 1), hkv)
    if ids:
        kv8_store(gpu_of(first[0]), gpu_of(first[1]), cache, bt, mc, ec, state(mc, ids, lens), 1, validate=True)
        m.append(table, ids, lens, *first)
        m.check(cache)
    for step in range(6):
        ids = [s for s in range(seqs) for _ in range(q_len)]
        lens = [int(have[s]) + i + 1 for s in range(seqs) for i in range(q_len)]
        k, v = (rows_of(rng, len(ids), hkv, sizes=rng.uniform(-8, 8) if step % 2 else None) for _ in range(2))
        kv8_store(gpu_of(k), gpu_of(v), cache, bt, mc, ec, state(mc, ids, lens), 1, validate=True)
        m.append(table, ids, lens, k, v)
        m.check(cache)
        have += rng.integers(1, q_len + 1, seqs)  # the rest of the rows was rejected


@pytest.mark.parametrize("codes", CODES)
def test_store_rows_in_any_order(gpu, codes):
    """Rows of a block far apart in the batch, out of order, and the same position twice: the last one stays."""
    mc, ec, rng, table, bt, cache = make(codes, gpu, seqs=40, seed=4)
    m = Mirror(cache, 0, codes)
    ids = [s for s in range(40) for _ in range(16)]
    lens = [40 + i for s in range(40) for i in range(16)]
    order = rng.permutation(len(ids))
    ids, lens = ([x[i] for i in order] for x in (ids, lens))
    ids, lens = ids + ids[:50], lens + lens[:50]
    k, v = rows_of(rng, len(ids), 2), rows_of(rng, len(ids), 2)
    kv8_store(gpu_of(k), gpu_of(v), cache, bt, mc, ec, state(mc, ids, lens), 0, validate=True)
    m.append(table, ids, lens, k, v)
    m.check(cache)


@pytest.mark.parametrize("codes", CODES)
def test_prompts_and_rows_in_one_forward(gpu, codes):
    mc, ec, rng, table, bt, cache = make(codes, gpu, seqs=4, seed=5)
    m = Mirror(cache, 1, codes)
    prompts, ids, lens = [20, 33], [2, 2, 3], [1, 2, 1]
    k, v = rows_of(rng, 56, 2), rows_of(rng, 56, 2)
    kv8_store(gpu_of(k), gpu_of(v), cache, bt, mc, ec, state(mc, ids, lens, prompts, [0, 1]), 1, validate=True)
    m.prompt(table, 0, k[:20].astype(np.float64), v[:20].astype(np.float64))
    m.prompt(table, 1, k[20:53].astype(np.float64), v[20:53].astype(np.float64))
    m.append(table, ids, lens, k[53:], v[53:])
    m.check(cache)


@pytest.mark.parametrize("codes", CODES)
def test_values_that_are_not_finite(gpu, codes):
    mc, ec, rng, table, bt, cache = make(codes, gpu, seqs=2, seed=6)
    m = Mirror(cache, 0, codes)
    k, v = rows_of(rng, 20, 2), rows_of(rng, 20, 2)
    k[3, 0, 7], k[3, 1, 9], v[18, 1, 0], v[2, 0, 100] = np.nan, np.inf, -np.inf, np.nan
    st = state(mc, [], [], [20], [0])
    with pytest.raises(RuntimeError, match="not finite"):
        kv8_store(gpu_of(k), gpu_of(v), cache, bt, mc, ec, st, 0, validate=True)
    m.prompt(table, 0, k.astype(np.float64), v.astype(np.float64))
    m.check(cache)
    k1, v1 = rows_of(rng, 3, 2), rows_of(rng, 3, 2)
    k1[1, 1, 64] = np.nan
    with pytest.raises(RuntimeError, match="not finite"):
        kv8_store(gpu_of(k1), gpu_of(v1), cache, bt, mc, ec, state(mc, [0, 0, 0], [21, 22, 23]), 0, validate=True)
    m.append(table, [0, 0, 0], [21, 22, 23], k1, v1)
    m.check(cache)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("fault", ["block", "negative", "seq", "length", "zero"])
def test_bad_metadata_is_flagged_and_skipped(gpu, codes, fault):
    """Of three rows (and two prompts, and two ranges to read) one points outside: it alone is left out."""
    mc, ec, rng, table, bt, cache = make(codes, gpu, seqs=3, seed=7)
    st = state(mc, [0, 1, 2], [5, 6, 7])
    k, v = rows_of(rng, 3, 2), rows_of(rng, 3, 2)
    table = table.copy()
    ids, lens = [0, 1, 2], [5, 6, 7]
    if fault == "block":
        table[1, 0] = cache.num_blocks
    elif fault == "negative":
        table[1, 0] = -1
    elif fault == "seq":
        ids[1] = 3
    else:
        lens[1] = 16 * 8 + 1 if fault == "length" else 0
    st.seq_ids, st.decoding_seq_lens = gpu_of(np.array(ids, np.int32)), gpu_of(np.array(lens, np.int32))
    m = Mirror(cache, 0, codes)
    with pytest.raises(RuntimeError, match="invalid metadata"):
        kv8_store(gpu_of(k), gpu_of(v), cache, gpu_of(table), mc, ec, st, 0, validate=True)
    keep = [0, 2]
    m.append(table, [0, 2], [5, 7], k[keep], v[keep])
    m.check(cache)
    untouched = [b for b in range(cache.num_blocks) if b not in (table[0, 0], table[2, 0])]
    assert (cache.k[untouched] == 0).all() and (cache.v_scales[untouched] == 0).all()
    # the same rows through the prologue
    q = gpu_of(rows_of(rng, 3, 4))
    cos, sin = rope_cache(128, 1e6, 16 * 8 + 1, gpu)
    with pytest.raises(RuntimeError, match="invalid metadata"):
        kv8_qk_norm_rope_store(q, gpu_of(k), gpu_of(v), cache, gpu_of(table), None, None, mc, ec, st, 0, cos, sin,
                               validate=True)
    assert (cache.k[untouched] == 0).all() and (cache.v_scales[untouched] == 0).all()
    # a prompt and a range to read
    if fault != "zero":
        st = state(mc, [], [], [5, 6, 7], [0, 1, 2])
        st.seq_ids, st.prefill_seq_lens = (gpu_of(np.array(x, np.int32)) for x in (ids, lens))
        rows = gpu_of(rows_of(rng, 18, 2))
        before = cache.k[untouched].clone()
        with pytest.raises(RuntimeError, match="invalid metadata"):
            kv8_store(rows, rows, cache, gpu_of(table), mc, ec, st, 0, validate=True)
        assert torch.equal(cache.k[untouched], before)
        out = [torch.full((18, 2, 128), 7.0, dtype=torch.float16, device=gpu) for _ in range(2)]
        with pytest.raises(RuntimeError, match="invalid metadata"):
            kv8_load(*out, cache, gpu_of(table), st.seq_ids, st.prefill_seq_start_locs, st.prefill_seq_lens, 200, 0,
                     validate=True)
        for o in out:
            assert (o[5:11] == 7).all() and not (o[:5] == 7).all() and not (o[11:] == 7).all()


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("norm,strided", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("hq,hkv,q_len", [(4, 2, 5), (16, 8, 1), (5, 1, 17), (40, 8, 3)])
def test_prologue_is_the_fp16_prologue_then_the_store(gpu, codes, norm, strided, hq, hkv, q_len):
    """q, and the rows that are stored, bit for bit ``qk_norm_rope_store``'s."""
    mc, ec, rng, table, bt, cache = make(codes, gpu, hq=hq, hkv=hkv, seqs=4, seed=q_len)
    have = [0, 14, 16, 37]
    ids = [s for s in range(4) for _ in range(q_len)]
    lens = [h + i + 1 for h in have for i in range(q_len)]
    rows = len(ids)
    old = rows_of(rng, sum(have), hkv), rows_of(rng, sum(have), hkv)
    kv8_store(gpu_of(old[0]), gpu_of(old[1]), cache, bt, mc, ec, state(mc, [], [], have, range(4)), 1)
    other = copy.deepcopy(cache)
    qkv = gpu_of(rows_of(rng, rows, hq + 2 * hkv))
    wq, wk = ((1 + 0.5 * torch.randn(128, device=gpu)).half() if norm else None for _ in range(2))
    cos, sin = rope_cache(128, 1e6, 128, gpu)
    st = state(mc, ids, lens)
    q, k, v = qkv.split((hq, hkv, hkv), 1)
    if not strided:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    q_out = torch.empty(rows, hq, 128, dtype=torch.float16, device=gpu)
    kq, kk = q.contiguous().clone(), k.contiguous().clone()
    if strided:
        kv8_qk_norm_rope_store(q, k, v, cache, bt, wq, wk, mc, ec, st, 1, cos, sin, validate=True, q_out=q_out)
        assert torch.equal(q, kq) and torch.equal(k, kk)
    else:
        q_in = q.clone()
        kv8_qk_norm_rope_store(q_in, k, v, cache, bt, wq, wk, mc, ec, st, 1, cos, sin, validate=True)
        q_out = q_in
        assert torch.equal(k, kk)
    fp16 = [torch.zeros(table.size + 2, 2, hkv, 16, 128, dtype=torch.float16, device=gpu) for _ in range(2)]
    qk_norm_rope_store(kq, kk, v.contiguous(), *fp16, bt, wq, wk, mc, ec, st, 1, cos, sin, validate=True)
    assert torch.equal(q_out, kq)
    kv8_store(kk, v.contiguous(), other, bt, mc, ec, st, 1, validate=True)
    for a, b in zip((cache.k, cache.v, cache.k_scales, cache.v_scales), (other.k, other.v, other.k_scales, other.v_scales)):
        assert torch.equal(a, b)
    m = Mirror(cache, 1, codes)
    at = 0
    for s, n in enumerate(have):
        m.prompt(table, s, old[0][at:at + n].astype(np.float64), old[1][at:at + n].astype(np.float64))
        at += n
    m.append(table, ids, lens, kk.cpu().numpy(), v.cpu().numpy())
    m.check(cache)


def test_prologue_position_outside_the_tables(gpu):
    mc, ec, rng, table, bt, cache = make("e4m3", gpu, seqs=2)
    q, k = gpu_of(rows_of(rng, 2, 4)), gpu_of(rows_of(rng, 2, 2))
    cos, sin = rope_cache(128, 1e6, 10, gpu)
    q_out = torch.full_like(q, 7.0)
    with pytest.raises(RuntimeError, match="RoPE"):
        kv8_qk_norm_rope_store(q, k, k, cache, bt, None, None, mc, ec, state(mc, [0, 1], [11, 10]), 0, cos, sin,
                               validate=True, q_out=q_out)
    assert (q_out[0] == 7).all() and not (q_out[1] == 7).any(-1).all()
    assert (cache.v[table[0]] == 0).all() and (cache.v[table[1, 0], 0] != 0).any()


# ---------------------------------------------------------------- reader


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("hkv", [1, 2, 5])
def test_load_ranges(gpu, codes, hkv):
    """Ranges that start and end anywhere in a block; rows of no range stay as they are."""
    mc, ec, rng, table, bt, cache = make(codes, gpu, hkv=hkv, hq=hkv, seqs=3, seed=hkv)
    k, v = rows_of(rng, 3 * 128, hkv), rows_of(rng, 3 * 128, hkv)
    kv8_store(gpu_of(k), gpu_of(v), cache, bt, mc, ec, state(mc, [], [], [128] * 3, range(3)), 1)
    m = Mirror(cache, 1, codes)
    for s in range(3):
        m.prompt(table, s, k[128 * s:128 * s + 128].astype(np.float64), v[128 * s:128 * s + 128].astype(np.float64))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    for ranges in ([(0, 0, 128)], [(1, 15, 2), (1, 15, 1), (2, 16, 16), (0, 0, 0), (0, 127, 1)],
                   [(2, 3, 30), (0, 31, 33), (1, 1, 1), (2, 0, 17)]):
        starts, at = [], 3
        for _, _, n in ranges:
            starts.append(at)
            at += n + 2
        out = [torch.full((at, hkv, 128), 7.0, dtype=torch.float16, device=gpu) for _ in range(2)]
        want = [np.full((at, hkv, 128), 7.0) for _ in range(2)]
        for (s, f, n), st in zip(ranges, starts):
            for w, t in zip(want, m.tokens(table, s, 128)):
                w[st:st + n] = t[f:f + n]
        firsts = i32([f for _, f, _ in ranges]) if any(f for _, f, _ in ranges) else None
        longest = max(n for _, _, n in ranges)
        kv8_load(*out, cache, bt, i32([s for s, _, _ in ranges]), i32(starts), i32([n for _, _, n in ranges]), longest, 1,
                 first=firsts, validate=True)
        for o, w in zip(out, want):
            assert np.array_equal(o.cpu().numpy().astype(np.float64), w)


def test_load_bounds(gpu):
    mc, ec, rng, table, bt, cache = make("int8", gpu, seqs=2)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    for first, start, n, longest in ((0, 0, 129, 200), (120, 0, 9, 9), (-1, 0, 4, 4), (0, 1, 128, 128), (0, -1, 4, 4),
                                     (0, 0, 5, 4)):
        out = [torch.full((128, 2, 128), 7.0, dtype=torch.float16, device=gpu) for _ in range(2)]
        with pytest.raises(RuntimeError, match="invalid metadata"):
            kv8_load(*out, cache, bt, i32(0), i32(start), i32(n), longest, 0, first=i32(first), validate=True)
        assert all((o == 7).all() for o in out)


# ---------------------------------------------------------------- attention


def filled(codes, gpu, hq, hkv, ctxs, q_len, layers=2, seed=0, spread=2.0, dead="stale"):
    """A cache that holds the contexts and new tokens of verify rows, random codes in its other blocks and slots."""
    rng = np.random.default_rng(seed)
    need = [-(-(c + q_len) // 16) for c in ctxs]
    per = max(need)
    mc, ec = config(hq, hkv, layers, per)
    pool = sum(need) + 3
    table = np.full((len(ctxs), per), pool - 1, np.int32)
    ids = rng.permutation(pool - 1)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = ids[at:at + n]
        at += n
    g = torch.Generator(device=gpu).manual_seed(seed)
    x = [torch.randn((pool, layers, hkv, 16, 128), device=gpu, generator=g) for _ in range(2)]
    top, lo, hi = oracle.KV8_RANGES[codes]
    power = [torch.randint(-2, 2, (pool, layers, hkv), device=gpu, generator=g) + (-7 if codes == "e4m3" else -5)
             for _ in range(2)]
    raw = [(t * spread / torch.exp2(p.float())[..., None, None]).round().clamp(-127, 127) for t, p in zip(x, power)]
    raw = [t.to(DTYPE[codes]) for t in raw]
    if codes == "e4m3" and dead == "nan":  # slots that hold no token, and blocks of nobody
        for r, c in enumerate(ctxs):
            last = (c + q_len - 1) % 16 + 1
            for t in raw:
                t.view(torch.uint8)[table[r, need[r] - 1], :, :, last:] = 0x7f
        for t in raw:
            t.view(torch.uint8)[gpu_of(np.append(ids[at:], pool - 1))] = 0xff
    cache = KV8Cache.pack(*raw, *((p + 127).to(torch.uint8) for p in power))
    seq_ids = [s for s in range(len(ctxs)) for _ in range(q_len)]
    lens = [c + i + 1 for c in ctxs for i in range(q_len)]
    q = torch.randn((len(lens), hq, 128), device=gpu, generator=g).half()
    return mc, ec, table, gpu_of(table), cache, seq_ids, lens, q


def check_attention(cache, table, layer, q, seq_ids, lens, o, lse, scale=128 ** -0.5):
    kk, vv = (x[:, layer] for x in values_of(cache))
    q, o, lse = q.cpu().numpy(), o.double().cpu().numpy(), lse.double().cpu().numpy()
    worst = 0.0
    for s in sorted(set(seq_ids)):
        rows = [r for r, i in enumerate(seq_ids) if i == s]
        n = max(lens[r] for r in rows)
        ids = table[s, : -(-n // 16)]
        k, v = (x[ids].transpose(0, 2, 1, 3).reshape(-1, x.shape[1], 128)[:n] for x in (kk, vv))
        wo, wl, oo, lo = oracle.kv8_attention(q[rows], k, v, [lens[r] for r in rows], scale)
        eo, el = np.abs(o[rows] - wo), np.abs(lse[rows] - wl)
        o_in, lse_in = bool((eo <= oo).all()), bool((el <= lo).all())
        assert o_in, f"sequence {s}: o off by {(eo / oo).max():.3g} of the bound"
        assert lse_in, f"sequence {s}: lse off by {(el / lo).max():.3g} of the bound"
        worst = max(worst, (eo / oo).max())
    print(f"worst {worst:.2f} of the bound", flush=True)


def attend(cache, bt, mc, ec, seq_ids, lens, q, layer=1, validate=True, st=None):
    st = st or state(mc, seq_ids, lens)
    o = torch.full_like(q, float("nan"))
    lse = torch.full(q.shape[:2], float("nan"), device=q.device)
    kv8_paged_attention(q, cache, bt, mc, ec, st, layer, o, lse, validate=validate)
    return o, lse, st


EDGES = [0, 1, 14, 15, 16, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 257]


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("hq,hkv,q_len", [(4, 4, 1), (16, 8, 1), (32, 8, 5), (32, 8, 9), (16, 8, 12), (40, 8, 5), (64, 8, 9),
                                          (6, 2, 16), (7, 1, 2), (48, 1, 1)])
def test_attention_block_and_pair_edges(gpu, codes, hq, hkv, q_len):
    mc, ec, table, bt, cache, ids, lens, q = filled(codes, gpu, hq, hkv, EDGES, q_len, dead="nan")
    o, lse, _ = attend(cache, bt, mc, ec, ids, lens, q)
    check_attention(cache, table, 1, q, ids, lens, o, lse)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("hq,hkv,q_len,ctxs", [(16, 8, 1, [4000, 7, 900]), (32, 8, 5, [3000, 250]), (32, 8, 9, [5000]),
                                               (8, 1, 1, [20000]), (4, 2, 3, [9000, 1])])
def test_attention_segments_in_pieces(gpu, codes, hq, hkv, q_len, ctxs):
    mc, ec, table, bt, cache, ids, lens, q = filled(codes, gpu, hq, hkv, ctxs, q_len, seed=1)
    o, lse, st = attend(cache, bt, mc, ec, ids, lens, q)
    assert int(st.kv8_plan.host[_lib.PLAN_COMBINES]) > 0
    check_attention(cache, table, 1, q, ids, lens, o, lse)


@pytest.mark.parametrize("codes", CODES)
def test_attention_of_more_segments_than_slots(gpu, codes):
    """80 sequences of 8 heads: later workgroups claim their pieces."""
    ctxs = [3 * i % 97 for i in range(80)]
    mc, ec, table, bt, cache, ids, lens, q = filled(codes, gpu, 16, 8, ctxs, 1, seed=2)
    o, lse, st = attend(cache, bt, mc, ec, ids, lens, q)
    assert int(st.kv8_plan.host[_lib.PLAN_CLAIMED]) > 0
    check_attention(cache, table, 1, q, ids, lens, o, lse)
    for _ in range(3):
        o2, lse2, _ = attend(cache, bt, mc, ec, ids, lens, q, st=st)
        assert torch.equal(o, o2) and torch.equal(lse, lse2)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("rows", ["fp16 plan", "one by one", "any order"])
def test_attention_by_other_plans(gpu, codes, rows):
    """The fp16 attention's plan, rows each a group of its own, and rows repeated and in any order."""
    q_len = 5
    mc, ec, table, bt, cache, ids, lens, q = filled(codes, gpu, 16, 8, [3000, 250, 31, 90], q_len, seed=16)
    if rows == "any order":
        order = np.random.default_rng(17).permutation(len(ids) * 2) % len(ids)  # every row twice
        ids, lens, q = [ids[r] for r in order], [lens[r] for r in order], q[torch.from_numpy(order).to(gpu)].contiguous()
    st = state(mc, ids, lens)
    if rows == "one by one":
        st.max_group_rows = 1
    if rows == "fp16 plan":
        plan, size = plan_for(st, mc, ec, bt), ctypes.c_int64()
        assert int(plan.host[_lib.PLAN_COMBINES]) > 0
        _lib.call("nsd_kv8_attn_workspace", plan.host_address, ctypes.byref(size))
        st.kv8_plan = AttnPlan(plan.host, plan.dev, None, size.value, 16, 8)
    o, lse, _ = attend(cache, bt, mc, ec, ids, lens, q, st=st)
    check_attention(cache, table, 1, q, ids, lens, o, lse)


@pytest.mark.parametrize("codes", CODES)
def test_attention_over_half_a_million_tokens(gpu, codes):
    """The longest segment that a plan takes, 128 pieces of 256 blocks, of seven blocks again and again."""
    n = 1 << 19
    mc, ec, _, _, cache, _, _, q = filled(codes, gpu, 4, 1, [7 * 16 - 1], 1, layers=1, seed=18)
    ec = EngineConfig(max_blocks_per_seq=n // 16)
    table = np.arange(n // 16, dtype=np.int32)[None] % 7
    o, lse, st = attend(cache, gpu_of(table), mc, ec, [0], [n], q, layer=0)
    assert st.kv8_plan.host[_lib.PLAN_SLOTS] == 128
    with pytest.raises(_lib.NativeLibraryError, match="pieces"):
        attend(cache, gpu_of(np.zeros((1, n // 16 + 1), np.int32)), mc, EngineConfig(max_blocks_per_seq=n // 16 + 1), [0],
               [n + 1], q, layer=0)
    k, v = (x[:7, 0, 0].reshape(-1, 128) for x in values_of(cache))
    times = np.repeat(np.bincount(table[0], minlength=7), 16).astype(np.float64)
    for h in range(4):
        s = k @ q[0, h].double().cpu().numpy() * 128 ** -0.5
        p = times * np.exp(s - s.max())
        want, total = p @ v / p.sum(), p.sum()
        # as oracle.kv8_attention; sums of a lane's 256 weights, four waves and 128 parts in fp32
        ds = 130 * 2.0 ** -24 * (np.abs(k) @ np.abs(q[0, h].double().cpu().numpy())).max() * 128 ** -0.5 + \
            (np.abs(s).max() + np.abs(s - s.max()).max()) * 2.0 ** -22
        off = ((3 * 2.0 ** -11 + 2 * ds + 400 * 2.0 ** -24) * p + times * 2.0 ** -25) @ np.abs(v) / total + 2.0 ** -24
        assert (np.abs(o[0, h].double().cpu().numpy() - want) <= off).all()
        ln = s.max() + np.log(total)
        assert abs(float(lse[0, h]) - ln) <= ds + 400 * 2.0 ** -24 + 2.0 ** -22 * (1 + abs(ln))


@pytest.mark.parametrize("codes", CODES)
def test_attention_is_that_of_the_values(gpu, codes):
    """The fp16 attention over the values read back: the same to the roundings of both."""
    ctxs, q_len = [700, 33, 2000], 5
    mc, ec, table, bt, cache, ids, lens, q = filled(codes, gpu, 32, 8, ctxs, q_len, seed=3)
    o, lse, st = attend(cache, bt, mc, ec, ids, lens, q)
    kc, vc = (gpu_of(x.astype(np.float16)) for x in values_of(cache))
    o16, lse16 = torch.empty_like(q), torch.empty_like(lse)
    paged_attention(q, kc, vc, bt, mc, ec, st, 1, o16, lse16, validate=True)
    check_attention(cache, table, 1, q, ids, lens, o16, lse16)
    check_attention(cache, table, 1, q, ids, lens, o, lse)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("size", [2.0 ** -11, 40.0])
def test_attention_of_small_and_large_values(gpu, codes, size):
    """Values near fp16's smallest, and scores whose weights are all one token's."""
    mc, ec, table, bt, cache, ids, lens, q = filled(codes, gpu, 8, 2, [200, 31], 3, seed=4)
    power = int(np.log2(size))
    cache.k_scales.add_(power), cache.v_scales.add_(min(power, 0))
    o, lse, _ = attend(cache, bt, mc, ec, ids, lens, q)
    check_attention(cache, table, 1, q, ids, lens, o, lse)


def test_attention_nan_reaches_the_rows_that_attend_it(gpu):
    """NaN codes of one token: rows that mask it, and other heads, are as without it."""
    mc, ec, table, bt, cache, ids, lens, q = filled("e4m3", gpu, 8, 2, [60, 45], 5, seed=5)
    clean, _, st = attend(cache, bt, mc, ec, ids, lens, q)
    for which in "kv":
        k, v, ks, vs = cache.codes()
        t = 62  # attended by rows 2, 3, 4 of sequence 0
        (k if which == "k" else v).view(torch.uint8)[table[0, t // 16], 1, 1, t % 16, 3:5] = 0x7f
        o, lse, _ = attend(KV8Cache.pack(k, v, ks, vs), bt, mc, ec, ids, lens, q, st=st)
        hit = torch.zeros(10, 8, 128, dtype=torch.bool, device=gpu)
        hit[2:5, 4:, :] = True
        if which == "v":
            hit[:, :, :3] = hit[:, :, 5:] = False
        assert torch.isnan(o[hit]).all() and torch.equal(o[~hit], clean[~hit])


@pytest.mark.parametrize("codes", CODES)
def test_attention_bad_blocks(gpu, codes):
    """Ids outside the pool are flagged and masked; a row with nothing else left is zero, its lse -inf."""
    mc, ec, table, bt, cache, ids, lens, q = filled(codes, gpu, 4, 2, [100, 20, 3], 2, seed=6)
    bad = table.copy()
    bad[0, 2], bad[1, :], bad[2, 0] = cache.num_blocks, -5, 2 ** 31 - 1
    with pytest.raises(RuntimeError, match="block id"):
        attend(cache, gpu_of(bad), mc, ec, ids, lens, q)
    o, lse, st = attend(cache, gpu_of(bad), mc, ec, ids, lens, q, validate=False)
    assert (o[2:] == 0).all() and (lse[2:] == -np.inf).all()
    kk, vv = (x[:, 1] for x in values_of(cache))
    keep = [b for b in range(-(-102 // 16)) if b != 2]
    tok = np.concatenate([np.arange(16 * b, min(16 * b + 16, 102)) for b in keep])
    k, v = (x[table[0, tok // 16], :, tok % 16] for x in (kk, vv))
    wo, wl, oo, lo = oracle.kv8_attention(q[:2].cpu().numpy(), k, v, [len(tok) - 1, len(tok)], 128 ** -0.5)
    assert (np.abs(o[:2].double().cpu().numpy() - wo) <= oo).all()
    assert (np.abs(lse[:2].double().cpu().numpy() - wl) <= lo).all()


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("n", [1, 3, 17, 40])
def test_slots_without_tokens_hold_any_code(gpu, codes, n):
    """Codes that the largest scale makes infinite, in slots above the rows and in blocks that no piece streams."""
    mc, ec, rng, table, bt, cache = make(codes, gpu, layers=1, seqs=1, blocks_per_seq=4, seed=12)
    cache.k.fill_(0x7E if codes == "e4m3" else 0)  # 448, or -128
    cache.v.fill_(0x7E if codes == "e4m3" else 0)
    cache.k_scales.fill_(255), cache.v_scales.fill_(255)
    m = Mirror(cache, 0, codes)
    q = gpu_of(rows_of(rng, 1, 4, sizes=0.0))
    for t in range(n):
        k, v = rows_of(rng, 1, 2, sizes=0.0), rows_of(rng, 1, 2, sizes=0.0)
        if t % 16 == 0:
            v[0, :, 7] = 65504
        kv8_store(gpu_of(k), gpu_of(v), cache, bt, mc, ec, state(mc, [0], [t + 1]), 0, validate=True)
        m.append(table, [0], [t + 1], k, v)
    m.check(cache)
    o, lse, _ = attend(cache, bt, mc, ec, [0], [n], q, layer=0)
    check_attention(cache, table, 0, q, [0], [n], o, lse)


@pytest.mark.parametrize("codes", CODES)
def test_attention_bad_blocks_among_pieces(gpu, codes):
    """A piece whose blocks are all outside the pool counts for nothing in the merge; a row whose every piece is so is
    zero, its lse -inf."""
    mc, ec, table, bt, cache, ids, lens, q = filled(codes, gpu, 4, 2, [9000, 9000], 2, seed=13)
    bad = table.copy()
    bad[0, 100:], bad[1, :] = cache.num_blocks, -1
    o, lse, st = attend(cache, gpu_of(bad), mc, ec, ids, lens, q, validate=False)
    assert int(st.kv8_plan.host[_lib.PLAN_COMBINES]) > 0
    assert (o[2:] == 0).all() and (lse[2:] == -np.inf).all()
    check_attention(cache, table, 1, q[:2], [0, 0], [1600, 1600], o[:2], lse[:2])


@pytest.mark.parametrize("codes", CODES)
def test_attention_writes_its_rows_alone(gpu, codes):
    mc, ec, table, bt, cache, ids, lens, q = filled(codes, gpu, 8, 2, [33, 700], 2, seed=7)
    room = torch.full((q.numel() + 4096,), 7.0, dtype=torch.float16, device=gpu)
    o = room[2048:2048 + q.numel()]
    before = [t.clone() for t in (cache.k, cache.v, cache.k_scales, cache.v_scales)]
    kv8_paged_attention(q, cache, bt, mc, ec, state(mc, ids, lens), 1, o, validate=True)
    assert (room[:2048] == 7).all() and (room[-2048:] == 7).all()
    want, _, _ = attend(cache, bt, mc, ec, ids, lens, q)
    assert torch.equal(o.view_as(want), want)
    assert all(torch.equal(a, b) for a, b in zip(before, (cache.k, cache.v, cache.k_scales, cache.v_scales)))


def test_tiles_past_32_bits(gpu):
    """A cache of more than 2^32 bytes of K: the last blocks written, read back and attended."""
    mc, ec = config(16, 8, 28, 8)
    blocks = (1 << 32) // (28 * 8 * 2048) + 400
    cache = KV8Cache.allocate(blocks, mc, torch.float8_e4m3fn, gpu)
    table = np.arange(blocks - 16, blocks, dtype=np.int32).reshape(2, 8)
    rng = np.random.default_rng(8)
    k, v = rows_of(rng, 200, 8, sizes=0.0), rows_of(rng, 200, 8, sizes=0.0)
    bt = gpu_of(table)
    kv8_store(gpu_of(k), gpu_of(v), cache, bt, mc, ec, state(mc, [], [], [100, 100], [0, 1]), 27, validate=True)
    k1, v1 = rows_of(rng, 2, 8, sizes=0.0), rows_of(rng, 2, 8, sizes=0.0)
    kv8_store(gpu_of(k1), gpu_of(v1), cache, bt, mc, ec, state(mc, [0, 1], [101, 101]), 27, validate=True)
    small = KV8Cache(*(t[blocks - 16:, 27:].contiguous() for t in (cache.k, cache.v, cache.k_scales, cache.v_scales)),
                     torch.float8_e4m3fn)
    assert (cache.k[: blocks - 16: 97] == 0).all() and (cache.k[-16:, :27] == 0).all()
    m = Mirror(small, 0, "e4m3")
    near = table - (blocks - 16)
    for s in range(2):
        m.prompt(near, s, k[100 * s:100 * s + 100].astype(np.float64), v[100 * s:100 * s + 100].astype(np.float64))
    m.append(near, [0, 1], [101, 101], k1, v1)
    m.check(small)
    out = [torch.empty(202, 8, 128, dtype=torch.float16, device=gpu) for _ in range(2)]
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    kv8_load(*out, cache, bt, i32(0, 1), i32(0, 101), i32(101, 101), 101, 27, validate=True)
    for i, o in enumerate(out):
        assert np.array_equal(o.double().cpu().numpy(), np.concatenate([m.tokens(near, s, 101)[i] for s in range(2)]))
    q = gpu_of(rows_of(rng, 2, 16, sizes=0.0))
    o, lse, _ = attend(cache, bt, mc, ec, [0, 1], [101, 101], q, layer=27)
    check_attention(small, near, 0, q, [0, 1], [101, 101], o, lse)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("seqs,n,hkv", [(4, 3000, 16), (3, 10900, 8)])
def test_large_prompts_are_small_ones(gpu, codes, seqs, n, hkv):
    """Rows enough to be read, and codes to be written, past the caches: the bytes of the same prompts one by one."""
    mc, ec = config(hkv, hkv, 1, -(-n // 16))
    cache, one = (KV8Cache.allocate(seqs * ec.max_blocks_per_seq, mc, DTYPE[codes], gpu) for _ in range(2))
    bt = torch.randperm(cache.num_blocks, device=gpu).to(torch.int32).view(seqs, -1)
    g = torch.Generator(device=gpu).manual_seed(14)
    lens = [n - 7 * s for s in range(seqs)]
    k, v = (torch.randn(sum(lens), hkv, 128, device=gpu, generator=g).half() for _ in range(2))
    assert k.numel() * 4 >= (128000000 if n > 10000 else 64000000)
    kv8_store(k, v, cache, bt, mc, ec, state(mc, [], [], lens, range(seqs)), 0, validate=True)
    at = 0
    for s, m in enumerate(lens):
        for lo in range(0, m, 4000):  # a prompt's blocks from another row of a table on
            part = slice(at + lo, at + min(lo + 4000, m))
            row = torch.zeros_like(bt[:1])
            ids = bt[s, lo // 16:]
            row[0, : len(ids)] = ids
            kv8_store(k[part], v[part], one, row, mc, ec, state(mc, [], [], [part.stop - part.start], [0]), 0, validate=True)
        at += m
    for a, b in zip((cache.k, cache.v, cache.k_scales, cache.v_scales), (one.k, one.v, one.k_scales, one.v_scales)):
        assert torch.equal(a, b)
    out = [torch.empty_like(k) for _ in range(2)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    kv8_load(*out, cache, bt, i32(range(seqs)), i32([sum(lens[:s]) for s in range(seqs)]), i32(lens), n, 0, validate=True)
    for x, y in zip((k, v), out):  # half a step: 2^-4 of the value (below normal codes 2^-9 of the scale), or a scale
        off = x.abs().float() / 16 + 2.0 ** -14 if codes == "e4m3" else x.abs().float().max() / 127
        assert ((x.float() - y.float()).abs() <= off).all()


# ---------------------------------------------------------------- streams, graphs, together


def _step(s, layer=1):
    """One layer's decode step: prologue, attention, and the step's blocks read back."""
    kv8_qk_norm_rope_store(s["q"], s["k"], s["v"], s["cache"], s["bt"], s["w"], s["w"], s["mc"], s["ec"], s["st"], layer,
                           s["cos"], s["sin"], q_out=s["q_out"])
    kv8_paged_attention(s["q_out"], s["cache"], s["bt"], s["mc"], s["ec"], s["st"], layer, s["o"], s["lse"])
    kv8_load(s["k_out"], s["v_out"], s["cache"], s["bt"], s["ids"], s["starts"], s["ends"], 4096, layer)
    return [s[n] for n in ("q_out", "o", "lse", "k_out", "v_out")]


def _step_state(codes, gpu, seed, q_len=5, ctxs=(700, 33, 2000), hq=16, hkv=8):
    mc, ec, table, bt, cache, ids, lens, q = filled(codes, gpu, hq, hkv, list(ctxs), q_len, seed=seed)
    n, total = len(lens), sum(ctxs) + q_len * len(ctxs)
    g = torch.Generator(device=gpu).manual_seed(seed)
    half = lambda *shape: torch.randn(shape, device=gpu, generator=g).half()  # noqa: E731
    ends = [c + q_len for c in ctxs]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    cos, sin = rope_cache(128, 1e6, 4096, gpu)
    st = state(mc, ids, lens)
    kv8_plan_for(st, mc, ec, bt)
    return dict(mc=mc, ec=ec, table=table, bt=bt, cache=cache, st=st, q=half(n, hq, 128), k=half(n, hkv, 128),
                v=half(n, hkv, 128), w=1 + half(128) / 8, cos=cos, sin=sin, q_out=half(n, hq, 128), o=half(n, hq, 128),
                lse=torch.empty(n, hq, device=gpu), k_out=half(total, hkv, 128), v_out=half(total, hkv, 128),
                ids=i32(range(len(ctxs))), ends=i32(ends), starts=i32([sum(ends[:i]) for i in range(len(ends))]),
                seq_ids=ids, lens=lens)


@pytest.mark.parametrize("codes", CODES)
def test_graph_replays(gpu, codes):
    """A captured step, replayed with new inputs and eager work between, gives the eager bits; so do two graphs of one
    plan replayed at once on two streams."""
    a = _step_state(codes, gpu, 1)
    b = dict(a, cache=copy.deepcopy(a["cache"]))
    for n in ("q", "k", "v", "q_out", "o", "lse", "k_out", "v_out"):
        b[n] = a[n].clone()
    eager = dict(b, cache=copy.deepcopy(a["cache"]))
    for n in ("q", "k", "v", "q_out", "o", "lse", "k_out", "v_out"):
        eager[n] = a[n].clone()
    for s in (a, b, eager):  # the tokens of a block remember how often they were rounded: one history for all
        _step(s)
    torch.cuda.synchronize()
    graphs = []
    for s in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            _step(s)
        graphs.append((g, torch.cuda.Stream()))
    for seed in range(4):
        gen = torch.Generator(device=gpu).manual_seed(100 + seed)
        for n in ("q", "k", "v"):
            x = torch.randn(a[n].shape, device=gpu, generator=gen).half() * 2.0 ** seed
            for s in (a, b, eager):
                s[n].copy_(x)
        for s in (a, b):
            for n in ("q_out", "o", "lse", "k_out", "v_out"):
                s[n].zero_()
        want = [t.clone() for t in _step(eager)]
        torch.cuda.synchronize()
        for g, stream in graphs:
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize()
        for s in (a, b):
            for n, w in zip(("q_out", "o", "lse", "k_out", "v_out"), want):
                assert torch.equal(s[n], w), f"replay {seed}: {n}"
            assert torch.equal(s["cache"].k, eager["cache"].k) and torch.equal(s["cache"].v_scales, eager["cache"].v_scales)


def test_a_plan_is_not_made_in_a_capture(gpu):
    """Refused while capturing: the upload's source is host memory that a replay would find changed."""
    a = _step_state("e4m3", gpu, 3, ctxs=(40,))
    a["st"] = state(a["mc"], a["seq_ids"], a["lens"])
    x = torch.zeros(4, device=gpu)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        x.add_(1)
        with pytest.raises(RuntimeError, match="before the capture"):
            kv8_paged_attention(a["q"], a["cache"], a["bt"], a["mc"], a["ec"], a["st"], 1, a["o"])
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    assert (x == 2).all() and a["st"].kv8_plan is None


def test_two_streams_claim_pieces(gpu):
    """More segments than slots, two calls of one plan at once: each claims by a counter of its own."""
    ctxs = [5 * i % 301 for i in range(90)]
    mc, ec, table, bt, cache, ids, lens, q = filled("int8", gpu, 16, 8, ctxs, 1, seed=15)
    q2 = q.flip(0).contiguous()
    want, _, st = attend(cache, bt, mc, ec, ids, lens, q)
    want2, _, _ = attend(cache, bt, mc, ec, ids, lens, q2, st=st)
    assert st.kv8_plan.claims
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(8):
        for s, x in zip(streams, (q, q2)):
            with torch.cuda.stream(s):
                o = torch.empty_like(x)
                kv8_paged_attention(x, cache, bt, mc, ec, st, 1, o)
                outs.append(o)
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert torch.equal(o, (want, want2)[i % 2])


def test_two_streams_share_a_plan(gpu):
    """Two calls with one forward's plan at once, on two streams: scratch is each call's own."""
    mc, ec, table, bt, cache, ids, lens, q = filled("e4m3", gpu, 32, 8, [6000, 5000, 40], 5, seed=9)
    q2 = q.flip(0).contiguous()
    want, _, st = attend(cache, bt, mc, ec, ids, lens, q)
    want2, _, _ = attend(cache, bt, mc, ec, ids, lens, q2, st=st)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        for s, x in zip(streams, (q, q2)):
            with torch.cuda.stream(s):
                o = torch.empty_like(x)
                kv8_paged_attention(x, cache, bt, mc, ec, st, 1, o)
                outs.append(o)
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert torch.equal(o, (want, want2)[i % 2])


@pytest.mark.parametrize("codes", CODES)
def test_another_stream_than_the_default(gpu, codes):
    a, b = _step_state(codes, gpu, 2), _step_state(codes, gpu, 2)
    want = [t.clone() for t in _step(a)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _step(b)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("codes", CODES)
def test_swap_out_and_in(gpu, codes):
    """Block copies of codes and of scales bring a sequence back in other blocks."""
    mc, ec, table, bt, cache, ids, lens, q = filled(codes, gpu, 16, 8, [100], 1, seed=10)
    want, _, _ = attend(cache, bt, mc, ec, ids, lens, q)
    n = table.shape[1]
    host = [torch.empty((n, *t.shape[1:]), dtype=torch.uint8).pin_memory() for t in (cache.k, cache.v, cache.k_scales, cache.v_scales)]
    planes = ((cache.k, cache.v, *host[:2]), (cache.k_scales, cache.v_scales, *host[2:]))
    for p in planes:
        swap_blocks(table[0].tolist(), list(range(n)), False, *p)
    torch.cuda.synchronize()
    back = table[0, ::-1].copy()
    cache.k.fill_(0x55), cache.v.fill_(0x55), cache.k_scales.fill_(1), cache.v_scales.fill_(1)
    for p in planes:
        swap_blocks(list(range(n)), back.tolist(), True, *p)
    got, _, _ = attend(cache, gpu_of(back[None]), mc, ec, ids, lens, q)
    assert torch.equal(got, want)


@pytest.mark.parametrize("engine", ["dma", "kernel"])
def test_host_copies(gpu, engine):
    """A backend for the codes and one for the scales bring blocks to the host and back."""
    rng = np.random.default_rng(19)
    mc, ec = config(16, 8, 4)
    cache = KV8Cache.allocate(20, mc, torch.int8, gpu)
    planes = (cache.k, cache.v), (cache.k_scales, cache.v_scales)
    want = []
    for t in (t for pair in planes for t in pair):
        t.copy_(torch.from_numpy(rng.integers(0, 256, tuple(t.shape), dtype=np.uint8)))
        want.append(t.cpu())
    for k, v in planes:
        arena = HostKVArena.create(total_blocks=9, block_bytes=k[0].numel(), kv_block_shape=tuple(k.shape[1:]))
        backend = HostKVCopyBackend(arena=arena, k_cache=k, v_cache=v, engine=engine)
        extent = arena.make_extent(offset_blocks=1, capacity_blocks=7)
        torch.cuda.synchronize()
        backend.launch(CopyPlan("D2H", (CopyRegion(extent, 5, 0, 7),))).synchronize()
        k.zero_(), v.zero_()
        torch.cuda.synchronize()
        backend.launch(CopyPlan("H2D", (CopyRegion(extent, 11, 0, 7),))).synchronize()
        backend.close()
    for t, w in zip((t for pair in planes for t in pair), want):
        assert torch.equal(t[11:18].cpu(), w[5:12]) and not t[:11].any() and not t[18:].any()


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("model,q_len", [(QWEN3_8B, 5), (QWEN3_0_6B, 1)], ids=["8b-verify", "06b-decode"])
def test_prompt_then_steps(gpu, codes, model, q_len):
    """As a model uses them: prompts attended and stored, then steps whose rows are accepted in part; every step's
    attention against the oracle over what the oracle's cache holds."""
    layers, layer = 2, 1
    mc = ModelConfig(dict(model, num_hidden_layers=layers))
    hq, hkv = mc.num_q_heads, mc.num_kv_heads
    ec = EngineConfig(max_blocks_per_seq=12)
    rng = np.random.default_rng(11)
    prompts = [90, 16, 47]
    table = rng.permutation(40)[:36].reshape(3, 12).astype(np.int32)
    bt = gpu_of(table)
    cache = KV8Cache.allocate(40, mc, DTYPE[codes], gpu)
    m = Mirror(cache, layer, codes)
    cos, sin = rope_cache(128, mc.rope_theta, 192, gpu)
    k, v = rows_of(rng, sum(prompts), hkv, sizes=0.0), rows_of(rng, sum(prompts), hkv, sizes=0.0)
    st = build_infer_state([0, 1, 2], [], prompts, mc, cos, sin, gpu)
    q = gpu_of(rows_of(rng, sum(prompts), hq, sizes=0.0))
    prefill_attention(q, gpu_of(k), gpu_of(v), torch.empty_like(q), mc, ec, st)
    kv8_store(gpu_of(k), gpu_of(v), cache, bt, mc, ec, st, layer, validate=True)
    at = 0
    for s, n in enumerate(prompts):
        m.prompt(table, s, k[at:at + n].astype(np.float64), v[at:at + n].astype(np.float64))
        at += n
    have = np.array(prompts)
    wq, wk = ((1 + 0.2 * torch.randn(128, device=gpu)).half() for _ in range(2))
    for step in range(8):
        ids = [s for s in range(3) for _ in range(q_len)]
        lens = [int(have[s]) + i + 1 for s in range(3) for i in range(q_len)]
        st = build_infer_state(ids, lens, [], mc, cos, sin, gpu)
        qkv = gpu_of(rows_of(rng, len(ids), hq + 2 * hkv, sizes=0.5 * step))
        q, kk, vv = qkv.split((hq, hkv, hkv), 1)
        q_out = torch.empty(len(ids), hq, 128, dtype=torch.float16, device=gpu)
        kv8_qk_norm_rope_store(q, kk, vv, cache, bt, wq, wk, mc, ec, st, layer, cos, sin, validate=True, q_out=q_out)
        o, lse = torch.empty_like(q_out), torch.empty(q_out.shape[:2], device=gpu)
        kv8_paged_attention(q_out, cache, bt, mc, ec, st, layer, o, lse, validate=True)
        rotated = kk.contiguous().clone()
        pool16 = [torch.zeros(40, layers, hkv, 16, 128, dtype=torch.float16, device=gpu) for _ in range(2)]
        qk_norm_rope_store(q.contiguous(), rotated, vv.contiguous(), *pool16, bt, wq, wk, mc, ec, st, layer, cos, sin)
        m.append(table, ids, lens, rotated.cpu().numpy(), vv.cpu().numpy())
        m.check(cache)
        check_attention(cache, table, layer, q_out, ids, lens, o, lse, mc.head_dim ** -0.5)
        have = have + rng.integers(1, q_len + 1, 3)


def test_empty_calls(gpu):
    mc, ec, rng, table, bt, cache = make("e4m3", gpu)
    st = state(mc, [], [])
    none = lambda h: torch.empty(0, h, 128, dtype=torch.float16, device=gpu)  # noqa: E731
    kv8_store(none(2), none(2), cache, bt, mc, ec, st, 0, validate=True)
    cos, sin = rope_cache(128, 1e6, 4, gpu)
    kv8_qk_norm_rope_store(none(4), none(2), none(2), cache, bt, None, None, mc, ec, st, 0, cos, sin, validate=True)
    kv8_paged_attention(none(4), cache, bt, mc, ec, st, 0, none(4), validate=True)
    i0 = torch.empty(0, dtype=torch.int32, device=gpu)
    kv8_load(none(2), none(2), cache, bt, i0, i0, i0, 0, 0, validate=True)
    assert (cache.k == 0).all()


def test_refusals(gpu):
    mc, ec, rng, table, bt, cache = make("e4m3", gpu, seqs=2)
    st = state(mc, [0, 1], [5, 6])
    half = lambda *s: torch.zeros(s, dtype=torch.float16, device=gpu)  # noqa: E731
    q, k, o = half(2, 4, 128), half(2, 2, 128), half(2, 4, 128)
    cos, sin = rope_cache(128, 1e6, 8, gpu)
    i32 = torch.zeros(2, dtype=torch.int32, device=gpu)
    att = dict(q=q, cache=cache, block_table=bt, model_config=mc, engine_config=ec, infer_state=st, cur_layer=0, o=o)
    pro = dict(q=q, k=k, v=k, cache=cache, block_table=bt, q_norm=None, k_norm=None, model_config=mc, engine_config=ec,
               infer_state=st, cur_layer=0, cos_cache=cos, sin_cache=sin)
    sto = dict(k=k, v=k, cache=cache, block_table=bt, model_config=mc, engine_config=ec, infer_state=st, cur_layer=0)
    loa = dict(k=k, v=k, cache=cache, block_table=bt, seq_ids=i32, start_locs=i32, seq_lens=i32, max_len=0, cur_layer=0)
    wide = config(blocks_per_seq=9)[1]
    bad = [
        (kv8_paged_attention, att, dict(q=q.float()), TypeError), (kv8_paged_attention, att, dict(q=q.cpu()), ValueError),
        (kv8_paged_attention, att, dict(q=half(2, 2, 128)), ValueError), (kv8_paged_attention, att, dict(o=half(1, 4, 128)), ValueError),
        (kv8_paged_attention, att, dict(o=o.bfloat16()), TypeError), (kv8_paged_attention, att, dict(lse=half(2, 4)), TypeError),
        (kv8_paged_attention, att, dict(lse=torch.zeros(3, device=gpu)), ValueError),
        (kv8_paged_attention, att, dict(q=q.transpose(0, 1).contiguous().transpose(0, 1)), ValueError),
        (kv8_paged_attention, att, dict(block_table=bt.long()), TypeError), (kv8_paged_attention, att, dict(engine_config=wide), ValueError),
        (kv8_paged_attention, att, dict(cur_layer=2), _lib.NativeLibraryError),
        (kv8_paged_attention, att, dict(model_config=config(hkv=4)[0]), ValueError),
        (kv8_paged_attention, att, dict(infer_state=state(mc, [0], [5])), ValueError),
        (kv8_qk_norm_rope_store, pro, dict(q=q.float()), TypeError), (kv8_qk_norm_rope_store, pro, dict(k=half(2, 3, 128)), ValueError),
        (kv8_qk_norm_rope_store, pro, dict(v=half(3, 2, 128)), ValueError), (kv8_qk_norm_rope_store, pro, dict(q_norm=half(128)), ValueError),
        (kv8_qk_norm_rope_store, pro, dict(q_norm=half(128), k_norm=half(64)), ValueError),
        (kv8_qk_norm_rope_store, pro, dict(sin_cache=sin[:4]), ValueError), (kv8_qk_norm_rope_store, pro, dict(cos_cache=cos.float()), TypeError),
        (kv8_qk_norm_rope_store, pro, dict(q=half(2, 8, 128)[:, :4]), ValueError),
        (kv8_qk_norm_rope_store, pro, dict(k=half(2, 260)[:, :256].view(2, 2, 128)), ValueError),
        (kv8_qk_norm_rope_store, pro, dict(k=half(520)[4:516].view(2, 2, 128)), ValueError),
        (kv8_qk_norm_rope_store, pro, dict(cur_layer=-1), _lib.NativeLibraryError),
        (kv8_store, sto, dict(k=k.float()), TypeError), (kv8_store, sto, dict(k=half(3, 2, 128)), ValueError),
        (kv8_store, sto, dict(v=half(2, 3, 128)), ValueError), (kv8_store, sto, dict(k=k.cpu()), ValueError),
        (kv8_store, sto, dict(block_table=bt[:, :4]), ValueError), (kv8_store, sto, dict(cur_layer=5), _lib.NativeLibraryError),
        (kv8_load, loa, dict(k=k.float()), TypeError), (kv8_load, loa, dict(v=half(1, 2, 128)), ValueError),
        (kv8_load, loa, dict(seq_ids=i32.long()), TypeError), (kv8_load, loa, dict(seq_lens=i32[:1]), ValueError),
        (kv8_load, loa, dict(start_locs=i32.cpu()), ValueError), (kv8_load, loa, dict(first=i32[:1]), ValueError),
        (kv8_load, loa, dict(max_len=-1), _lib.NativeLibraryError),
    ]
    for f, base, change, error in bad:
        with pytest.raises(error):
            f(**{**base, **change})
    with pytest.raises(AttributeError):
        cache.k = cache.v
    for f, base in ((kv8_paged_attention, att), (kv8_qk_norm_rope_store, pro), (kv8_store, sto), (kv8_load, loa)):
        f(**base)
