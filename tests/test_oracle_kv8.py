"""The 8-bit KV cache's oracle against brute force, torch and closed forms, and the library's refusals (no GPU)."""

from __future__ import annotations

import ctypes
import subprocess
import sys

import numpy as np
import pytest
import torch

import oracle
from nebulasd_amd import _lib
from nebulasd_amd.build import ROOT
from nebulasd_amd.kernels import KV8Cache, kv8_load, kv8_paged_attention, kv8_qk_norm_rope_store, kv8_store
from nebulasd_amd.kernels.kv8 import _Cache
from oracle.kv8 import (KV8_E4M3, KV8_RANGES, kv8_append, kv8_attention, kv8_exponent, kv8_round, kv8_tiles,
                        kv8_untile)

CODES = ["e4m3", "int8"]
FINITE = np.arange(0x7c00, dtype=np.uint16).view(np.float16).astype(np.float64)  # every fp16 magnitude


@pytest.mark.parametrize("codes", CODES)
def test_exponent_is_the_smallest_that_fits(codes):
    top, lo, hi = KV8_RANGES[codes]
    for m in np.concatenate((FINITE[::37], FINITE[-40:], [0.0])):
        e = kv8_exponent([0.0, -m, m / 2, np.nan, np.inf], codes)
        fits = [x for x in range(lo, hi + 1) if m <= top * 2.0 ** x]
        assert e == (min(fits) if fits else hi)
        # only int8's last range is passed, and by less than one of its steps
        assert fits or (codes == "int8" and m - top * 2.0 ** hi < 2.0 ** hi)


@pytest.mark.parametrize("codes", CODES)
def test_round_takes_the_nearest_code(codes):
    rng = np.random.default_rng(1)
    top, lo, hi = KV8_RANGES[codes]
    table = KV8_E4M3 if codes == "e4m3" else np.arange(128.0)
    for e in range(lo, hi + 1):
        v = rng.uniform(-1, 1, 200) * np.minimum(top * 2.0 ** e, 65504.0) * rng.choice([1, 2.0 ** -4, 2.0 ** -9], 200)
        middles = (table[1:] + table[:-1]) / 2 * 2.0 ** e
        v = np.concatenate((v, middles, -middles))
        v = v[np.abs(v) <= (61440.0 if codes == "e4m3" else np.inf)]
        held, byte = kv8_round(v, e, codes)
        all_codes = np.concatenate((table, -table)) * 2.0 ** e
        assert (np.abs(held - v) == np.abs(all_codes - v[:, None]).min(1)).all()
        at = np.searchsorted(table, np.abs(held) / 2.0 ** e)
        tie = np.isin(np.abs(v), middles)
        assert (at[tie] % 2 == 0).all()
        mag = byte & 127 if codes == "e4m3" else np.abs(byte.view(np.int8).astype(int))
        assert (mag == at).all()


def test_round_agrees_with_torch():
    v = np.concatenate((FINITE, -FINITE))
    for e in (-15, -9, -1, 0, 7):
        x = v[np.abs(v) <= 448 * 2.0 ** e]
        want = torch.from_numpy(x / 2.0 ** e).float().to(torch.float8_e4m3fn)
        held, byte = kv8_round(x, e, "e4m3")
        assert (byte == want.view(torch.uint8).numpy()).all()
        assert (held == want.double().numpy() * 2.0 ** e).all()


@pytest.mark.parametrize("codes", CODES)
def test_every_value_of_a_cache_is_an_fp16_value(codes):
    """Every fp16 number under the scale of every block it can be in."""
    top, lo, hi = KV8_RANGES[codes]
    for e in range(lo, hi + 1):
        v = FINITE[FINITE <= (top * 2.0 ** e if e < hi else 65504)]
        held, _ = kv8_round(v, e, codes)
        assert np.isfinite(held.astype(np.float16)).all()
        assert (held.astype(np.float16).astype(np.float64) == held).all()
        # and off by half a step: of the value's own (a tail of the range: 61440, 127 2^9), at least of the block's
        step = 2.0 ** e if codes == "int8" else np.maximum(2.0 ** (e - 9), 2.0 ** (np.frexp(v)[1] - 4))
        cut = v - np.minimum(v, 61440.0 if codes == "e4m3" else 127.0 * 2 ** 9)
        assert (np.abs(held - v) <= step / 2 + cut).all()


@pytest.mark.parametrize("codes", CODES)
def test_values_that_are_not_finite(codes):
    held, byte = kv8_round([np.nan, np.inf, -np.inf, 1.0], 0, codes)
    assert held[3] == 1.0 and (np.isnan(held[:3]).all() if codes == "e4m3" else (held[:3] == 0).all())
    assert (byte[:3] == (127 if codes == "e4m3" else 0)).all()


@pytest.mark.parametrize("codes", CODES)
def test_append_rounds_again_within_a_step(codes):
    """Rows that double in size, one at a time: every token ends less than one step from its value, and the scale is
    that of the values held."""
    rng = np.random.default_rng(2)
    rows = rng.standard_normal((16, 128)) * 2.0 ** (np.arange(16)[:, None] * 0.9 - 6)
    rows = rows.astype(np.float16).astype(np.float64)
    held = np.full((16, 128), np.nan)  # nothing in the block: slots above count for nothing
    for t in range(16):
        held, byte, e = kv8_append(held, {t: rows[t]}, codes)
        assert e == kv8_exponent(held[: t + 1], codes) or e == kv8_exponent(rows[: t + 1], codes)
    step = 2.0 ** e if codes == "int8" else np.maximum(2.0 ** (e - 9), 2.0 ** (np.frexp(np.abs(rows))[1] - 4))
    assert (np.abs(held - rows) < step).all()
    # a planted mistake is seen: the scale one step down
    wrong, _ = kv8_round(rows[15], e - 1, codes)
    right, _ = kv8_round(rows[15], e, codes)
    assert (wrong != right).any() and (right == held[15]).all()


@pytest.mark.parametrize("codes", CODES)
def test_append_at_once_and_one_by_one(codes):
    rng = np.random.default_rng(3)
    rows = rng.uniform(0.5, 1, (16, 128)).astype(np.float16).astype(np.float64)  # one scale throughout
    rows[:, 0] = 1.0
    once, byte, e = kv8_append(np.zeros((16, 128)), dict(enumerate(rows)), codes)
    held = np.zeros((16, 128))
    for t in range(16):
        held, _, e1 = kv8_append(held, {t: rows[t]}, codes)
    assert (held == once).all() and e1 == e
    assert (once == kv8_round(rows, kv8_exponent(rows, codes), codes)[0]).all()
    # rows 3 and 7 alone: 4 to 6 stay, 8 on do not count
    part, _, _ = kv8_append(once * np.where(np.arange(16)[:, None] > 7, 1e4, 1.0), {3: rows[3], 7: rows[7]}, codes)
    assert (part[:8] == once[:8]).all()


def test_attention_oracle():
    rng = np.random.default_rng(4)
    q = rng.standard_normal((3, 4, 128)).astype(np.float16)
    k, v = (rng.standard_normal((40, 2, 128)).astype(np.float16) for _ in range(2))
    lens = [38, 39, 40]
    o, lse, o_off, lse_off = kv8_attention(q, k, v, lens, 128 ** -0.5)
    pad = lambda x: np.concatenate((x, np.zeros((8, 2, 128), np.float16))).reshape(3, 16, 2, 128).transpose(0, 2, 1, 3)  # noqa: E731
    wo, wl = oracle.paged_attention(q, pad(k)[:, None].copy(), pad(v)[:, None].copy(), np.array([[0, 1, 2]]), [0, 0, 0], lens, 0)
    assert np.abs(o - wo).max() < 1e-5 and np.abs(lse - wl).max() < 1e-5
    for r, n in enumerate(lens):
        for h in range(4):
            s = torch.from_numpy(k[:n, h // 2]).double() @ torch.from_numpy(q[r, h]).double() * 128 ** -0.5
            want = torch.softmax(s, 0) @ torch.from_numpy(v[:n, h // 2]).double()
            assert np.abs(o[r, h] - want.numpy()).max() < 1e-12
            assert abs(lse[r, h] - torch.logsumexp(s, 0).item()) < 1e-12
    # the bounds: rounded weights stay within them, a token left out does not
    assert (o_off > 2.0 ** -11 * np.abs(o)).all() and o_off.max() < 0.01 and lse_off.max() < 1e-4
    less, _, _, _ = kv8_attention(q, k, v, [37, 38, 39], 128 ** -0.5)
    assert (np.abs(less - o) > o_off).any()
    empty, none, _, _ = kv8_attention(q, k, v, [0, 0, 0], 1.0)
    assert (empty == 0).all() and (none == -np.inf).all()


@pytest.mark.parametrize("codes", CODES)
def test_tiles(codes):
    rng = np.random.default_rng(5)
    b = rng.integers(0, 256, (2, 16, 128), dtype=np.uint8)
    k, v = kv8_tiles(b, codes)
    assert (kv8_untile(k, codes, 0) == b).all() and (kv8_untile(v, codes, 1) == b).all()
    bias = 128 if codes == "int8" else 0
    # token 5, dim 77 = 64 + 8 + 5: unit 16 * 1 + 5, byte 8 + 5; dim 77 = 8 * 9 + 4 + 1: unit 64 + 16 + 9, byte 4 + 1
    assert (k[:, (16 + 5) * 16 + 13] ^ bias == b[:, 5, 77]).all()
    assert (v[:, (64 + 16 + 9) * 16 + 5] ^ bias == b[:, 5, 77]).all()


# ---------------------------------------------------------------- refusals that need no GPU


def _c(**kw):
    base = dict(k=16, v=16, k_scales=16, v_scales=16, num_blocks=4, num_layers=2, num_kv_heads=2, codes=0)
    return _Cache(**{**base, **kw})


BAD_CACHES = [dict(k=None), dict(v=24), dict(k_scales=None), dict(codes=2), dict(codes=-1), dict(num_blocks=0),
              dict(num_layers=0), dict(num_kv_heads=-1)]


def _refused(name, *args):
    with pytest.raises(_lib.NativeLibraryError, match="status 1|status 2") as e:
        _lib.call(name, *args)
    return str(e.value)


def _store(c, layer=0, rows=1, k=16, v=16, bt=16, bt_rows=1, stride=1):
    return ("nsd_kv8_store", k, v, c and ctypes.byref(c), bt, bt_rows, stride, 16, 16, rows, layer, None, None)


def _prefill(c, layer=0, n=1, longest=1, tokens=1, k=16):
    return ("nsd_kv8_store_prefill", k, 16, tokens, c and ctypes.byref(c), 16, 1, 1, 16, 16, 16, n, longest, layer,
            None, None)


def _load(c, layer=0, n=1, longest=1, tokens=1, k=16, starts=16):
    return ("nsd_kv8_load", k, 16, tokens, c and ctypes.byref(c), 16, 1, 1, 16, None, starts, 16, n, longest, layer,
            None, None)


def _prologue(c, layer=0, rows=1, q=16, q_rs=256, q_out=32, k_rs=256, qn=None, kn=None, pos=1, hq=2, cos=16):
    return ("nsd_kv8_qk_norm_rope_store", q, q_rs, q_out, 16, k_rs, 16, 256, qn, kn, 1e-6, cos, 16, pos,
            c and ctypes.byref(c), 16, 1, 1, 16, 16, rows, layer, hq, None, None)


@pytest.mark.parametrize("call", [_store, _prefill, _load, _prologue], ids=["store", "prefill", "load", "prologue"])
def test_c_refusals_of_a_cache(call):
    assert "null cache" in _refused(*call(None))
    for bad in BAD_CACHES:
        _refused(*call(_c(**bad)))
    for layer in (-1, 2):
        assert "layer" in _refused(*call(_c(), layer=layer))


def test_c_refusals_of_arguments():
    c = _c()
    for kw in (dict(rows=-1), dict(k=None), dict(k=8), dict(v=24), dict(bt=None), dict(bt_rows=0), dict(stride=0),
               dict(rows=(1 << 20) + 1)):
        _refused(*_store(c, **kw))
    for kw in (dict(n=-1), dict(longest=-1), dict(tokens=-1), dict(k=None), dict(k=20), dict(n=65536)):
        _refused(*_prefill(c, **kw))
        _refused(*_load(c, **kw))
    _refused(*_load(c, starts=None))
    for kw in (dict(q=None), dict(q=24), dict(q_out=None), dict(q_rs=128), dict(q_rs=260), dict(k_rs=128), dict(qn=16),
               dict(kn=16), dict(qn=24, kn=16), dict(pos=0), dict(hq=0), dict(cos=24), dict(cos=None), dict(rows=-1),
               dict(q_out=16, q_rs=264)):
        _refused(*_prologue(c, **kw))
    # no rows: nothing to do, and nothing looked at
    for args in (_store(c, rows=0), _prefill(c, n=0), _load(c, n=0), _load(c, longest=0), _prologue(c, rows=0)):
        _lib.call(*args)


def test_c_refusals_of_partials():
    c = _c()

    def args(part=16, splits=2, q_out=16, qn=None, kn=None, cos=16, pos=8, cache=c, bt=16, rows=1, layer=0, hq=4):
        return ("nsd_kv8_qk_norm_rope_store_partials", part, splits, q_out, qn, kn, 1e-6, cos, 16, pos,
                cache and ctypes.byref(cache), bt, 2, 4, 16, 16, rows, layer, hq, None, None)

    for bad in BAD_CACHES:
        _refused(*args(cache=_c(**bad)))
    for kw in (dict(part=None), dict(part=8), dict(splits=0), dict(splits=9), dict(q_out=None), dict(q_out=8), dict(qn=16),
               dict(cos=None), dict(cos=24), dict(pos=0), dict(cache=None), dict(bt=None), dict(rows=-1),
               dict(rows=(1 << 20) + 1), dict(layer=2), dict(hq=0)):
        _refused(*args(**kw))
    _lib.call(*args(rows=0))
    _refused("nsd_decoder_forward_kv8", None, 16, 16, 1, ctypes.byref(c), *[16, 1, 1, 16, 16, 16, 16, 8, None, None, None],
             0, 0.1, -1, None, None, None, None, None)


def test_plans():
    """Every block of every segment in one piece, parts in fp32, and few pieces where they do."""
    from nebulasd_amd.plan import decode_plan, kv8_plan_words
    rng = np.random.default_rng(6)
    for n, hq, hkv, longest, rows in ((1, 32, 8, 60000, 1), (4, 16, 8, 300, 1), (16, 32, 8, 4000, 5), (80, 16, 8, 900, 1),
                                      (40, 8, 1, 3000, 9), (3, 48, 1, 20, 2)):
        ctx = rng.integers(0, longest, n)
        ids = [s for s in range(n) for _ in range(rows)]
        lens = [int(c) + i + 1 for c in ctx for i in range(rows)]
        words, ws = kv8_plan_words(ids, lens, hq, hkv, n, longest // 16 + 2, 256)
        p = decode_plan(words)
        seen = {}
        for rec in p["pieces"]:
            seen.setdefault((int(rec[4]), int(rec[0])), []).append((int(rec[1]), int(rec[2])))
        assert len(seen) == len(p["groups"]) * hkv
        for (row, head), parts in seen.items():
            parts.sort()
            group = next(g for g in p["groups"] if g[0] == row)
            assert parts[0][0] == 0 and parts[-1][1] == -(-int(group[3] + group[1]) // 16)
            assert all(a[1] == b[0] for a, b in zip(parts, parts[1:]))
            assert all(b - a <= 256 for a, b in parts)
            assert len(parts) == 1 or min(b - a for a, b in parts) >= 20  # 24, less the rounding of starts
        fewest = sum(-(-sum(b - a for a, b in parts) // 256) for parts in seen.values())
        assert len(p["pieces"]) <= (256 if fewest <= 256 else max(512, fewest))
        split = p["slots"]
        assert ws == (0 if split == 0 and p["claimed"] == 0 else 256 + -(-split * p["rows_max"] * (4 * 128 + 4) // 256) * 256)
    with pytest.raises(ValueError, match="workers=0"):
        kv8_plan_words([0], [1], 4, 2, 1, 1, 0)
    with pytest.raises(_lib.NativeLibraryError, match="compute units"):
        kv8_plan_words([0], [1], 4, 2, 1, 1, 1 << 17)
    for bad in (dict(seq_ids=[1], seq_lens=[1]), dict(seq_ids=[0], seq_lens=[0]), dict(seq_ids=[0], seq_lens=[17]),
                dict(seq_ids=[-1], seq_lens=[1])):
        with pytest.raises(_lib.NativeLibraryError):
            kv8_plan_words(*bad.values(), 4, 2, 1, 1, 256)
    with pytest.raises(_lib.NativeLibraryError, match="not a plan"):
        _lib.call("nsd_kv8_attn_workspace", np.zeros(64, np.int32).ctypes.data, ctypes.byref(ctypes.c_int64()))


def test_attention_refusals():
    from nebulasd_amd.plan import kv8_plan_words
    words, ws = kv8_plan_words([0, 1], [40, 900], 4, 2, 2, 64, 64)
    buf = words.ctypes.data
    c = _c()

    def args(cache=c, layer=0, q=16, o=16, hq=4, bt=16, bt_rows=2, stride=64, plan=buf, dev=16, work=16, size=ws,
             scale=0.1):
        return ("nsd_kv8_paged_attention", q, o, None, cache and ctypes.byref(cache), layer, hq, bt, bt_rows, stride,
                plan, dev, work, size, scale, None, None)

    assert ws > 0
    for bad in BAD_CACHES:
        _refused(*args(cache=_c(**bad)))
    for kw in (dict(cache=None), dict(layer=2), dict(q=None), dict(q=8), dict(o=None), dict(hq=8), dict(bt=None),
               dict(bt_rows=1), dict(stride=65), dict(dev=None), dict(cache=_c(num_kv_heads=4))):
        _refused(*args(**kw))
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert "softmax_scale" in _refused(*args(scale=scale))
    for kw in (dict(work=None), dict(size=ws - 1), dict(work=8)):
        with pytest.raises(_lib.NativeLibraryError, match="status 4"):
            _lib.call(*args(**kw))


def test_python_refusals():
    u8 = dict(dtype=torch.uint8)
    k = torch.zeros(2, 1, 2, 2048, **u8)
    s = torch.zeros(2, 1, 2, **u8)
    with pytest.raises(ValueError, match="no CPU fallback"):
        KV8Cache(k, k, s, s, torch.int8)
    with pytest.raises(TypeError, match="float8_e4m3fn or torch.int8"):
        KV8Cache(k, k, s, s, torch.float8_e5m2)
    with pytest.raises(TypeError):
        KV8Cache.pack(k, k, s, s)
    with pytest.raises(ValueError, match="16, 128"):
        KV8Cache.pack(k.view(torch.int8), k.view(torch.int8), s, s)
    for f in (kv8_load, kv8_paged_attention, kv8_qk_norm_rope_store, kv8_store):
        assert f.__doc__


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("size", [16.0, 64.0, 1024.0, 4096.0])
def test_rejected_rows_leave_the_grid_of_their_scale(codes, size):
    """A history of steps of two rows, the second rejected and now and then far larger: tokens that stay end less than one
    step of the largest scale since they were written from their values (E4M3: of the value's own steps under it), not
    of the last; a block that never saw those rows keeps them within a step of its own."""
    rng = np.random.default_rng(8)
    rows = rng.standard_normal((16, 128)).astype(np.float16).astype(np.float64)
    held, alone = np.full((16, 128), np.nan), np.full((16, 128), np.nan)
    most = np.full(16, -99)
    for t in range(15):
        draft = (rng.standard_normal(128) * (size if t % 4 == 1 else 0.5)).astype(np.float16).astype(np.float64)
        held, _, e = kv8_append(held, {t: rows[t], t + 1: draft}, codes)
        most[: t + 1] = np.maximum(most[: t + 1], e)
        held, _, e = kv8_append(held, {t: held[t]}, codes)  # the scale without the draft
        alone, _, e1 = kv8_append(alone, {t: rows[t]}, codes)
    own = 2.0 ** (np.frexp(np.abs(rows[:15]))[1] - 4)
    step = lambda e: 2.0 ** e if codes == "int8" else np.maximum(2.0 ** (e - 9), own)  # noqa: E731
    off = np.abs(held[:15] - rows[:15])
    assert (off < step(most[:15, None].astype(float))).all()
    assert (np.abs(alone[:15] - rows[:15]) < step(float(e1))).all()
    if codes == "int8" or size > 1000:
        assert (off >= step(float(e))).any(), "these rows do not tell the two bounds apart"


def test_c_refuses_more_rows_than_an_append_compares():
    """Rows are compared with each other: a count that would hold the GPU for seconds is refused, the one below taken."""
    c = _c()
    for args in (_store, _prologue):
        assert "65536" in _refused(*args(c, rows=(1 << 16) + 1))
    assert "65536" in _refused("nsd_kv8_qk_norm_rope_store_partials", 16, 2, 16, None, None, 1e-6, 16, 16, 8,
                               ctypes.byref(c), 16, 2, 4, 16, 16, (1 << 16) + 1, 0, 4, None, None)


@pytest.mark.parametrize("rows,heads", [(4096, 2 ** 31 - 1), (1, 2 ** 31 - 1), (64, 1 << 24)])
def test_plans_too_large_are_refused(rows, heads):
    """More segments than a plan can hold: an error, where the planner's memory ran out and ended the process (so in a
    process of its own)."""
    code = f"""
import ctypes, numpy as np
from nebulasd_amd import _lib
ids, lens, buf = np.arange({rows}, dtype=np.int32), np.ones({rows}, np.int32), np.zeros(64, np.int32)
at = lambda a: a.ctypes.data_as(ctypes.POINTER(ctypes.c_int32))
lib, words = _lib.load(), ctypes.c_int64()
rc = lib.nsd_kv8_plan_build(at(ids), at(lens), {rows}, {heads}, {heads}, {rows}, 1, 256, 0, at(buf), 64, ctypes.byref(words))
assert rc == 1, rc  # NSD_ERR_INVALID
assert b"too large" in lib.nsd_last_error(), lib.nsd_last_error()
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stderr


def test_attention_refuses_scales_that_are_infinite_in_powers_of_two():
    from nebulasd_amd.plan import kv8_plan_words
    words, ws = kv8_plan_words([0], [40], 4, 2, 1, 64, 64)
    c = _c()
    for scale in (2.4e38, 3.4e38):
        assert "softmax_scale" in _refused("nsd_kv8_paged_attention", 16, 16, None, ctypes.byref(c), 0, 4, 16, 1, 64,
                                           words.ctypes.data, 16, 16, ws, scale, None, None)
