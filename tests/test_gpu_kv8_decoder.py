"""The decoder stack and the speculative loop over an 8-bit KV cache.

The stack's layers are this library's kernels, whose split partials are summed in one order wherever they are read, so
the same kernels called from Python give its bits: caches, outputs and the probed layer are compared for equality, the
probed attention with the oracle too.
"""

from __future__ import annotations

import copy

import numpy as np
import pytest
import torch

import oracle
from nebulasd_amd import _lib
from nebulasd_amd.config import QWEN3_0_6B, QWEN3_8B
from nebulasd_amd.decoder import DecoderStack
from nebulasd_amd.infer_state import build_infer_state
from nebulasd_amd.kernels import (KV8Cache, fused_add_rmsnorm_inplace, kv8_paged_attention, kv8_qk_norm_rope_store,
                                  kv8_qk_norm_rope_store_partials, linear, sum_partials, up_gate_silu_and_mul)
from nebulasd_amd.spec_loop import RandomQwen3, run

pytestmark = pytest.mark.gpu

DTYPE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
CASES = pytest.mark.parametrize("codes,cfg,n_layers,n_req,depth", [
    ("e4m3", QWEN3_0_6B, 4, 64, 0), ("int8", QWEN3_8B, 3, 16, 4), ("e4m3", QWEN3_0_6B, 2, 3, 2),
    ("int8", QWEN3_0_6B, 2, 1, 0)], ids=["0.6b-decode64", "8b-verify16x5", "0.6b-verify3x3", "0.6b-decode1"])


def model_and_rows(codes, cfg, n_layers, n_req, depth, gpu, native=True):
    """A model whose cache holds prompts, and decode/verify rows behind them."""
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(20, 300, (n_req,), generator=g).tolist()
    m = RandomQwen3(dict(cfg, num_hidden_layers=n_layers), [(n + depth + 4) // 16 + 1 for n in lens], gpu, seed=3,
                    native=native, kv_codes=DTYPE[codes])
    prompts = [torch.randint(0, cfg["vocab_size"], (n,), generator=g).tolist() for n in lens]
    m.prefill(list(range(n_req)), prompts)
    sids, slens, toks = [], [], []
    for r, p in enumerate(prompts):
        sids += [r] * (depth + 1)
        slens += list(range(len(p) + 1, len(p) + 2 + depth))
        toks += torch.randint(0, cfg["vocab_size"], (depth + 1,), generator=g).tolist()
    return m, sids, slens, toks


def layers_from_python(m, cache, st, x, res, probe_layer):
    mc = m.mc
    hq, hkv, d = mc.num_q_heads, mc.num_kv_heads, mc.head_dim
    probe = None
    for li, w in enumerate(m.layers):
        fused_add_rmsnorm_inplace(x, res, w["n_in"], mc.rms_norm_eps)
        q, k, v = linear(x, w["wqkv"]).view(-1, hq + 2 * hkv, d).split((hq, hkv, hkv), 1)
        q_out = torch.empty(q.shape, dtype=torch.float16, device=x.device)
        kv8_qk_norm_rope_store(q, k, v, cache, m.block_table, w["q_norm"], w["k_norm"], mc, m.ec, st, li, m.cos, m.sin,
                               q_out=q_out)
        o, lse = torch.empty_like(q_out), torch.empty(q_out.shape[:2], device=x.device)
        kv8_paged_attention(q_out, cache, m.block_table, mc, m.ec, st, li, o, lse)
        if li == probe_layer:
            probe = q_out, o, lse
        o = linear(o.view(x.shape[0], -1), w["wo"])
        fused_add_rmsnorm_inplace(o, res, w["n_post"], mc.rms_norm_eps)
        x = linear(up_gate_silu_and_mul(o, w["wug"]), w["wd"])
    return x, res, probe


def bytes_of(cache):
    return cache.k, cache.v, cache.k_scales, cache.v_scales


def oracle_excess(m, layer, q, o, lse, seq_ids, seq_lens):
    """The largest error of a probed attention, of the oracle's bound."""
    k, v, ks, vs = m.kv8.codes()
    two = lambda s: torch.exp2(s[:, layer].double() - 127)[..., None, None]  # noqa: E731
    kk, vv = ((c[:, layer].double() * two(s)).cpu().numpy() for c, s in ((k, ks), (v, vs)))
    table = m.block_table.cpu().numpy()
    worst = 0.0
    for s in sorted(set(seq_ids)):
        rows = [r for r, i in enumerate(seq_ids) if i == s]
        n = max(seq_lens[r] for r in rows)
        ids = table[s, : -(-n // 16)]
        held = (x[ids].transpose(0, 2, 1, 3).reshape(-1, x.shape[1], 128)[:n] for x in (kk, vv))
        wo, wl, oo, lo = oracle.kv8_attention(q[rows].cpu().numpy(), *held, [seq_lens[r] for r in rows], 128 ** -0.5)
        worst = max(worst, (np.abs(o[rows].double().cpu().numpy() - wo) / oo).max(),
                    (np.abs(lse[rows].double().cpu().numpy() - wl) / lo).max())
    return worst


@CASES
def test_stack_is_its_kernels_from_python(gpu, codes, cfg, n_layers, n_req, depth):
    m, sids, slens, toks = model_and_rows(codes, cfg, n_layers, n_req, depth, gpu)
    room = 128 if depth == 2 else len(sids)
    stack = DecoderStack(m.mc, m.layers, max_rows=room)
    mine = copy.deepcopy(m.kv8)
    st = build_infer_state(sids, slens, [], m.mc, m.cos, m.sin, gpu)
    for probe_layer in (-1, n_layers - 1, 0):  # rows stored again where they are leave the cache as it is
        x = m.embed[torch.tensor(toks, device=gpu)]
        want_x, want_res, want = layers_from_python(m, mine, st, x.clone(), torch.zeros_like(x), probe_layer)
        res = torch.zeros_like(x)
        got = stack.forward_kv8(x, res, m.kv8, m.block_table, m.ec, st, m.cos, m.sin, probe_layer)
        torch.cuda.synchronize()
        assert torch.equal(x, want_x) and torch.equal(res, want_res)
        assert all(torch.equal(a, b) for a, b in zip(bytes_of(m.kv8), bytes_of(mine)))
        if probe_layer < 0:
            assert got is None
        else:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            worst = oracle_excess(m, probe_layer, *got, sids, slens)
            print(f"layer {probe_layer}: worst {worst:.2f} of the bound", flush=True)
            assert worst <= 1


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
@pytest.mark.parametrize("splits", range(1, 9))
def test_prologue_over_partials(gpu, codes, splits):
    """A projection's split partials: the prologue over their sum, bit for bit; a NaN among them ends in its row alone."""
    m, sids, slens, _ = model_and_rows(codes, QWEN3_0_6B, 1, 9, splits - 1, gpu)
    st = build_infer_state(sids, slens, [], m.mc, m.cos, m.sin, gpu)
    mc, n = m.mc, len(sids)
    hq, hkv = mc.num_q_heads, mc.num_kv_heads
    g = torch.Generator(device=gpu).manual_seed(splits)
    part = torch.randn((splits, n, (hq + 2 * hkv) * 128), device=gpu, generator=g)
    if splits == 3:
        part[1, 4, -1] = float("nan")
    mine = copy.deepcopy(m.kv8)
    q, k, v = sum_partials(part).view(n, hq + 2 * hkv, 128).split((hq, hkv, hkv), 1)
    outs = [torch.full((n, hq, 128), 7.0, dtype=torch.float16, device=gpu) for _ in range(2)]
    for w in ((None, None), (m.layers[0]["q_norm"], m.layers[0]["k_norm"])):
        rest = (m.block_table, *w, mc, m.ec, st, 0, m.cos, m.sin)
        kv8_qk_norm_rope_store_partials(part, outs[0], m.kv8, *rest, validate=splits != 3)
        kv8_qk_norm_rope_store(q, k, v, mine, *rest, q_out=outs[1])
        assert torch.equal(*outs)
        assert all(torch.equal(a, b) for a, b in zip(bytes_of(m.kv8), bytes_of(mine)))


def test_prologue_over_partials_refusals(gpu):
    m, sids, slens, _ = model_and_rows("int8", QWEN3_0_6B, 1, 3, 0, gpu)
    st = build_infer_state(sids, slens, [], m.mc, m.cos, m.sin, gpu)
    hq, hkv = m.mc.num_q_heads, m.mc.num_kv_heads
    part = torch.zeros((2, 3, (hq + 2 * hkv) * 128), device=gpu)
    q = torch.zeros((3, hq, 128), dtype=torch.float16, device=gpu)
    call = lambda part=part, q=q, **kw: kv8_qk_norm_rope_store_partials(  # noqa: E731
        part, q, m.kv8, m.block_table, kw.get("w"), None, m.mc, m.ec, st, kw.get("layer", 0), m.cos, m.sin)
    for bad, error in ((dict(part=part.half()), TypeError), (dict(part=part[:, :2].contiguous()), ValueError),
                       (dict(part=part[0]), ValueError), (dict(part=part[:, :, 1:]), ValueError),
                       (dict(part=part.cpu()), ValueError), (dict(q=q[:2]), ValueError),
                       (dict(q=q.float()), TypeError), (dict(w=m.layers[0]["q_norm"]), ValueError),
                       (dict(layer=1), _lib.NativeLibraryError), (dict(part=part[:0]), _lib.NativeLibraryError),
                       (dict(part=torch.cat([part] * 5)), _lib.NativeLibraryError)):
        with pytest.raises(error):
            call(**bad)
    call()


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
def test_stack_in_a_graph(gpu, codes):
    """A captured forward, replayed on new embeddings with eager work between, gives the eager bits."""
    m, sids, slens, toks = model_and_rows(codes, QWEN3_0_6B, 2, 70, 0, gpu)
    st = build_infer_state(sids, slens, [], m.mc, m.cos, m.sin, gpu)
    stack, eager = (DecoderStack(m.mc, m.layers, max_rows=len(sids)) for _ in range(2))
    mine = copy.deepcopy(m.kv8)
    x, res = (torch.zeros((len(sids), m.mc.hidden_size), dtype=torch.float16, device=gpu) for _ in range(2))
    args = (m.block_table, m.ec, st, m.cos, m.sin)
    for s, c in ((stack, m.kv8), (eager, mine)):
        s.forward_kv8(x.clone(), torch.zeros_like(x), c, *args)
    assert st.kv8_plan.claims
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        stack.forward_kv8(x, res, m.kv8, *args)
    for seed in range(3):
        new = m.embed[torch.randint(0, m.mc.vocab_size, (len(sids),), generator=torch.Generator().manual_seed(seed)).to(gpu)]
        x.copy_(new)
        res.zero_()
        g.replay()
        want_res = torch.zeros_like(new)
        eager.forward_kv8(new, want_res, mine, *args)
        torch.cuda.synchronize()
        assert torch.equal(x, new) and torch.equal(res, want_res), f"replay {seed}"
        assert all(torch.equal(a, b) for a, b in zip(bytes_of(m.kv8), bytes_of(mine))), f"replay {seed}"


def test_stack_refusals(gpu):
    m, sids, slens, toks = model_and_rows("e4m3", QWEN3_0_6B, 2, 3, 0, gpu)
    stack = DecoderStack(m.mc, m.layers, max_rows=3)
    st = build_infer_state(sids, slens, [], m.mc, m.cos, m.sin, gpu)
    x = torch.zeros((3, m.mc.hidden_size), dtype=torch.float16, device=gpu)
    call = lambda x=x, res=None, cache=m.kv8, st=st: stack.forward_kv8(  # noqa: E731
        x, torch.zeros_like(x) if res is None else res, cache, m.block_table, m.ec, st, m.cos, m.sin)
    b = bytes_of(m.kv8)
    for cut in (lambda t: t[:, :1].contiguous(), lambda t: t[:, :, :4].contiguous()):
        with pytest.raises(_lib.NativeLibraryError, match="a cache of"):
            call(cache=KV8Cache(*(cut(t) for t in b), torch.float8_e4m3fn))
    with pytest.raises(TypeError):
        call(x=x.float())
    with pytest.raises(ValueError):
        call(x=x[:2])
    with pytest.raises(ValueError, match="only"):
        call(st=build_infer_state([0, 1, 2], [5, 5], [4], m.mc, m.cos, m.sin, gpu))
    with pytest.raises(ValueError, match="1..3"):
        call(st=build_infer_state([0, 1, 2, 2], [5, 5, 5, 6], [], m.mc, m.cos, m.sin, gpu))
    call()
    stack.close()
    with pytest.raises(RuntimeError, match="closed"):
        call()


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
@pytest.mark.parametrize("native", [True, False])
def test_model_forwards(gpu, codes, native):
    """RandomQwen3's two ways through the layers, their sampled attention against the oracle over their caches."""
    m, sids, slens, toks = model_and_rows(codes, QWEN3_0_6B, 3, 16, 2, gpu, native)
    for layer in range(3):
        seen = []
        m.check = layer, lambda *a: seen.append(oracle_excess(*a))
        assert len(m.decode(sids, slens, toks)) == len(sids)
        assert len(seen) == 1 and seen[0] <= 1, seen
    assert bool(m.stacks) == native


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
def test_speculative_loop(gpu, codes):
    """The loop over 8-bit caches: sampled attention calls against the oracle, the same tokens with the forwards side by
    side as one after the other."""
    seen = []

    def make_check():
        def check(model, layer, q, o, lse, seq_ids, seq_lens):
            torch.cuda.synchronize()
            seen.append((model.mc.num_layers, oracle_excess(model, layer, q, o, lse, seq_ids, seq_lens)))
        return check
    how = dict(n_requests=6, prompt_lo=40, prompt_hi=90, new_tokens=10, draft_batch=4, target_batch=2, depth=4, seed=3,
               device=gpu, return_outputs=True, kv_codes=DTYPE[codes])
    res = run(check_every=7, make_check=make_check, **how)
    assert res["generated_tokens"] == 60 and {n for n, _ in seen} == {28, 36}
    assert max(worst for _, worst in seen) <= 1, seen
    assert run(sync_each_forward=True, **how)["outputs"] == res["outputs"]


def test_speculative_loop_accepts(gpu):
    """The draft holds the target's weights: accepted proposals, rows of rejected ones rewritten, two-row steps."""
    small = dict(QWEN3_8B, num_hidden_layers=4)
    how = dict(n_requests=5, prompt_lo=20, prompt_hi=70, new_tokens=24, draft_batch=3, target_batch=2, depth=3, seed=4,
               target_cfg=small, share_weights=True, device=gpu, return_outputs=True, kv_codes=torch.int8)
    res = run(**how)
    assert res["generated_tokens"] == 120 and res["accepted"] > 0 and res["multi_token_appends"] > 0
    assert run(overlap=False, **how)["outputs"] == res["outputs"]
