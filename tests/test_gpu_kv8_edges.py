"""The 8-bit KV cache where a call's answer hangs on more than its kernels' ordinary path: the attention's roundings
counted, lengths below zero, strides of axes of one, and how many rows a call may have."""

from __future__ import annotations

import copy

import numpy as np
import pytest
import torch

from nebulasd_amd.kernels import KV8Cache, kv8_load, kv8_store
from test_gpu_kv8 import (CODES, DTYPE, Mirror, attend, config, filled, gpu_of, make, rows_of, state,
                          values_of)

pytestmark = pytest.mark.gpu


def close_weights(cache, table, layer, q, seq_ids, lens, o, scale):
    """The worst of the outputs' errors over their bounds, for queries of one nonzero dim.

    A score is then one product of an fp16 query and a code's value, 11 x 11 bits: exact in fp32.  What is rounded:
    the scale times log2(e), and its product with the score against the reference (half a step of the largest of them,
    2^-24 each; less where scores are subtracted first); exp2, by a step, 2^-23; a weight
    as a pair of fp16 numbers, 2^-22 of it or 2^-32 of the row's largest; the sums, fp32: a product instruction's by
    2^-22 of what it has added up at most, two a pair of blocks, and ten steps of merging waves and parts; the output,
    half a step of fp16.
    """
    kk, vv = (x[:, layer] for x in values_of(cache))
    q, o = q.double().cpu().numpy(), o.double().cpu().numpy()
    hkv, worst = kk.shape[1], 0.0
    for r, (sid, n) in enumerate(zip(seq_ids, lens)):
        ids = table[sid, : -(-n // 16)]
        k, v = (x[ids].transpose(0, 2, 1, 3).reshape(-1, hkv, 128)[:n] for x in (kk, vv))
        for h in range(q.shape[1]):
            s = k[:, h * hkv // q.shape[1]] @ q[r, h] * scale / np.log(2)
            p = np.exp2(s - s.max())
            w, total = v[:, h * hkv // q.shape[1]], p.sum()
            ds = (2 * np.abs(s).max() + np.abs(s - s.max()).max() + 16) * 2.0 ** -24
            rel = np.log(2) * ds + 2.0 ** -23 + 2.0 ** -22
            off = (2 * rel + (2 * -(-n // 32) + 10) * 2.0 ** -22) * (p @ np.abs(w)) / total
            off += 2.0 ** -32 * np.abs(w).sum(0) / total
            want = p @ w / total
            off += 2.0 ** -11 * (np.abs(want) + off) + 2.0 ** -25
            worst = max(worst, (np.abs(o[r, h] - want) / off).max())
    return worst


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("hq,hkv,q_len,ctxs", [(4, 4, 1, [40, 700]), (16, 8, 1, [300, 5]), (32, 8, 5, [600, 90]),
                                               (32, 8, 9, [500, 33]), (8, 2, 12, [2500]), (4, 1, 1, [6000])],
                         ids=["gqa1", "one-tile", "two-tiles", "three-tiles", "pieces-of-three", "pieces-of-one"])
def test_attention_weights_lose_nothing_that_fp16_outputs_keep(gpu, codes, hq, hkv, q_len, ctxs):
    mc, ec, table, bt, cache, ids, lens, q = filled(codes, gpu, hq, hkv, ctxs, q_len, seed=21)
    g = torch.Generator(device=gpu).manual_seed(22)
    dim = torch.randint(0, 128, (*q.shape[:2], 1), device=gpu, generator=g)
    q = torch.zeros_like(q).scatter_(2, dim, 8 * torch.randn(dim.shape, device=gpu, generator=g).half())
    o, _, _ = attend(cache, bt, mc, ec, ids, lens, q)
    worst = close_weights(cache, table, 1, q, ids, lens, o, mc.head_dim ** -0.5)
    print(f"worst {worst:.2f} of the bound", flush=True)
    assert worst <= 1


@pytest.mark.parametrize("codes", CODES)
def test_a_block_put_back_has_not_seen_rejected_rows(gpu, codes):
    """Verify steps whose rejected rows are far larger than the tokens: written over, they leave the tokens below within a
    step of the largest scale; the block put back and the accepted rows stored again are a cache that never saw them."""
    mc, ec, rng, table, bt, cache = make(codes, gpu, seqs=1, seed=23)
    back, never = copy.deepcopy(cache), copy.deepcopy(cache)
    tensors = lambda c: (c.k, c.v, c.k_scales, c.v_scales)  # noqa: E731
    put = lambda c, x, at: kv8_store(gpu_of(x[0]), gpu_of(x[1]), c, bt, mc, ec, state(  # noqa: E731
        mc, [0] * len(x[0]), list(range(at + 1, at + 1 + len(x[0])))), 1, validate=True)
    m, have, kept, most = Mirror(cache, 1, codes), 0, [], np.full(128, -99)
    rows = lambda n: [rows_of(rng, n, 2, sizes=0.0) for _ in range(2)]  # noqa: E731
    for step in range(20):
        good, bad = rows(1 + step % 3), [x * np.float16(2.0 ** (6 if step % 4 else 11)) for x in rows(2)]
        n, both = len(good[0]), [np.concatenate(x) for x in zip(good, bad)]
        blk = table[0, have // 16]
        saved = [t[blk].clone() for t in tensors(back)]
        for c in (cache, back):
            put(c, both, have)
        m.append(table, [0] * (n + 2), list(range(have + 1, have + n + 3)), *both)
        m.check(cache)
        for b in range(have // 16, (have + n + 1) // 16 + 1):
            part = slice(16 * b, min(16 * b + 16, have + n))
            most[part] = np.maximum(most[part], max(p[table[0, b]].max() for p in m.power))
        for t, s in zip(tensors(back), saved):
            t[blk] = s
        for c in (back, never):
            put(c, good, have)
        kept.append(good)
        have += n
    want = [np.concatenate(x) for x in zip(*kept)]
    live = table[0, : have // 16]  # whole blocks: behind the last token nothing counts
    for a, b in zip(tensors(back), tensors(never)):
        assert torch.equal(a[live.tolist()], b[live.tolist()])
    for w, got in zip(want, m.tokens(table, 0, have)):
        own = 2.0 ** (np.frexp(np.abs(w.astype(np.float64)))[1] - 4)
        step = np.ldexp(1.0, most[:have])[:, None, None]
        off = np.abs(got - w.astype(np.float64))
        assert (off < (step if codes == "int8" else np.maximum(step * 2.0 ** -9, own))).all()


def test_as_many_rows_as_a_call_takes(gpu):
    """65536 rows that fill 4096 blocks, in any order: the bytes of as many prompts of a block."""
    mc, ec = config(1, 1, 1, 1)
    rows, one = (KV8Cache.allocate(4096, mc, torch.int8, gpu) for _ in range(2))
    g = torch.Generator(device=gpu).manual_seed(24)
    bt = torch.randperm(4096, device=gpu, generator=g).to(torch.int32).view(4096, 1)
    k, v = (torch.randn(1 << 16, 1, 128, device=gpu, generator=g).half() for _ in range(2))
    kv8_store(k, v, one, bt, mc, ec, state(mc, [], [], [16] * 4096, range(4096)), 0, validate=True)
    order = torch.randperm(1 << 16, device=gpu, generator=g)
    ids, lens = (order // 16).tolist(), (order % 16 + 1).tolist()
    kv8_store(k[order], v[order], rows, bt, mc, ec, state(mc, ids, lens), 0, validate=True)
    for a, b in zip((rows.k, rows.v, rows.k_scales, rows.v_scales), (one.k, one.v, one.k_scales, one.v_scales)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("n", [-1, -16, -(2 ** 31)])
def test_lengths_below_zero_are_flagged(gpu, codes, n):
    """Of three prompts, and three ranges to read, the one of a negative length is left out and flagged."""
    mc, ec, rng, table, bt, cache = make(codes, gpu, seqs=3, seed=25)
    k, v = gpu_of(rows_of(rng, 40, 2)), gpu_of(rows_of(rng, 40, 2))
    want = copy.deepcopy(cache)
    kv8_store(k, v, want, bt, mc, ec, state(mc, [], [], [17, 0, 23], range(3)), 0, validate=True)
    st = state(mc, [], [], [17, 0, 23], range(3))
    st.prefill_seq_lens = torch.tensor([17, n, 23], dtype=torch.int32, device=gpu)
    with pytest.raises(RuntimeError, match="outside the block table"):
        kv8_store(k, v, cache, bt, mc, ec, st, 0, validate=True)
    assert all(torch.equal(a, b) for a, b in zip((cache.k, cache.v, cache.k_scales), (want.k, want.v, want.k_scales)))
    outs = [[torch.full((40, 2, 128), 7.0, dtype=torch.float16, device=gpu) for _ in range(2)] for _ in range(2)]
    kv8_load(*outs[0], cache, bt, st.seq_ids, st.prefill_seq_start_locs, st.prefill_seq_lens.clamp(min=0), 23, 0, validate=True)
    for first in (None, torch.zeros(3, dtype=torch.int32, device=gpu)):
        with pytest.raises(RuntimeError, match="outside the block table"):
            kv8_load(*outs[1], cache, bt, st.seq_ids, st.prefill_seq_start_locs, st.prefill_seq_lens, 23, 0, first=first,
                     validate=True)
        assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("q_len", [1, 5, 9])
@pytest.mark.parametrize("more", [64.0, 96.0, 160.0])
def test_attention_of_scores_in_the_hundred_millions(gpu, codes, q_len, more):
    """Scores of 269 to 276 million before the scale, those of the later tokens by a few of fp32's steps (32) larger: exact
    sums, whose softmax is that of their differences; no weight leaves fp16's range.

    Twice 2^25 in powers of two, steps of 4: the reference of a row cancels in its weights' exponents (a fused product
    and sum, rounded as the difference is), exp2 and the fp32 sums cost less than 2^-16.
    """
    hq, hkv, n = 8, 2, 512
    mc, ec, table, bt, cache, ids, lens, q = filled(codes, gpu, hq, hkv, [n - q_len], q_len, seed=26)
    k, v, ks, vs = cache.codes()
    power = 4 if codes == "e4m3" else 6
    code = lambda x: torch.tensor(x / 2.0 ** power).to(DTYPE[codes]).view(torch.uint8).item()  # noqa: E731
    raw = torch.zeros_like(k.view(torch.uint8))
    raw[..., 0] = code(4608.0)
    for i in range(32):  # block i, of wave i % 4: larger from one pair of a wave's blocks to the next, and back
        raw[int(table[0, i]), ..., 1 + i // 8 % 3] = code(2.0 ** power)
    cache = KV8Cache.pack(raw.view(k.dtype), v, torch.full_like(ks, 127 + power), vs)
    q = torch.zeros_like(q)
    size = 60000 - 96 * (torch.arange(q_len * hq, device=gpu) % 17).view(q_len, hq)
    q[..., 0] = size.half()
    for i in range(3):
        q[..., 1 + i] = i * more / 2.0 ** power
    o, _, _ = attend(cache, bt, mc, ec, ids, lens, q)
    vv = values_of(cache)[1][table[0], 1].transpose(0, 2, 1, 3).reshape(-1, hkv, 128)
    c = np.float64(np.float32(np.float32(128 ** -0.5) * np.float32(1.4426950408889634)))
    above = np.arange(n) // 128 % 3 * more * c
    for r in range(q_len):
        p = np.exp2(above[: lens[r]] - above[: lens[r]].max())
        for h in range(hq):
            w = vv[: lens[r], h * hkv // hq]
            want = p @ w / p.sum()
            off = 2.0 ** -11 * np.abs(want) + 2.0 ** -16 * (p @ np.abs(w)) / p.sum() + 2.0 ** -25
            assert (np.abs(o[r, h].double().cpu().numpy() - want) <= off).all()


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("q_len", [1, 5, 9])
def test_attention_of_the_largest_scores(gpu, codes, q_len):
    """Every dim of queries and keys near fp16's largest, 5e11 before the scale: finite, and the later tokens' values where
    their scores are larger by a 64th."""
    hq, hkv, n = 8, 2, 600
    mc, ec, table, bt, cache, ids, lens, q = filled(codes, gpu, hq, hkv, [n - q_len], q_len, seed=27)
    k, v, ks, vs = cache.codes()
    top, power = (224.0, 8) if codes == "e4m3" else (126.0, 9)
    code = lambda x: torch.tensor(x).to(DTYPE[codes]).view(torch.uint8).item()  # noqa: E731
    raw = torch.full_like(k.view(torch.uint8), code(top))
    late = torch.from_numpy(table[0, 20:].astype(np.int64)).to(gpu)
    raw[late] = code(240.0 if codes == "e4m3" else 127.0)
    cache = KV8Cache.pack(raw.view(k.dtype), v, torch.full_like(ks, 127 + power), vs)
    for size in (65504.0, -65504.0, 1000.0):
        q = torch.full_like(q, size)
        o, lse, _ = attend(cache, bt, mc, ec, ids, lens, q)
        vv = values_of(cache)[1][table[0], 1].transpose(0, 2, 1, 3).reshape(-1, hkv, 128)
        for r in range(q_len):
            part = slice(320, lens[r]) if size > 0 else slice(0, 320)
            for h in range(hq):
                w = vv[part, h * hkv // hq]  # scores apart by 1e5 and more: no other token has a weight
                off = 2.0 ** -11 * np.abs(w.mean(0)) + 2.0 ** -16 * np.abs(w).mean(0) + 2.0 ** -25
                assert (np.abs(o[r, h].double().cpu().numpy() - w.mean(0)) <= off).all()
        want = size * 128 * 2.0 ** power * ((240.0 if codes == "e4m3" else 127.0) if size > 0 else top) * 128 ** -0.5
        assert (lse.double() / want - 1).abs().max() <= 2.0 ** -21
