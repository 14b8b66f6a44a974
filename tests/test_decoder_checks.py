"""What the decoder stack refuses before it calls native code (no GPU: the native calls are stand-ins that record)."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from nebulasd_amd import decoder
from nebulasd_amd.config import QWEN3_8B, EngineConfig, ModelConfig

ROWS, BLOCKS = 3, 4


@pytest.fixture
def stack(monkeypatch):
    """A stack of two layers whose native calls are recorded in ``calls``."""
    s = object.__new__(decoder.DecoderStack)
    s.mc = ModelConfig(dict(QWEN3_8B, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, hidden_size=256))
    s.max_rows, s._handle, s.calls = 128, SimpleNamespace(value=None), []
    s._layers = [{"wqkv": torch.zeros(1)}] * 2
    plan = SimpleNamespace(n_rows=ROWS, workspace_bytes=0, claims=False, host_address=0, host_ptr=lambda: 0,
                           dev=torch.zeros(1, dtype=torch.int32), workspace=torch.zeros(1, dtype=torch.uint8))
    monkeypatch.setattr(decoder, "require_cuda", lambda *t: None)
    monkeypatch.setattr(decoder, "stream_of", lambda t: 0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    monkeypatch.setattr(decoder._lib, "call", lambda name, *a: s.calls.append(name))
    monkeypatch.setattr(decoder, "plan_for", lambda *a: plan)
    monkeypatch.setattr(decoder, "kv8_plan_for", lambda *a: plan)
    return s


def arguments(stack, cos_d=128):
    mc = stack.mc
    half = lambda *shape: torch.zeros(shape, dtype=torch.float16)  # noqa: E731
    state = SimpleNamespace(num_prefill_seqs=0, num_decoding_seqs=ROWS, seq_ids=torch.zeros(ROWS, dtype=torch.int32),
                            decoding_seq_lens=torch.ones(ROWS, dtype=torch.int32), softmax_scale=1.0)
    return dict(x=half(ROWS, mc.hidden_size), residual=half(ROWS, mc.hidden_size),
                block_table=torch.zeros((2, 5), dtype=torch.int32), engine_config=EngineConfig(max_blocks_per_seq=5),
                infer_state=state, cos_cache=half(9, cos_d // 2), sin_cache=half(9, cos_d // 2))


@pytest.mark.parametrize("cache_d,cos_d", [(64, 128), (64, 64), (128, 64), (256, 128)])
def test_forward_refuses_other_head_dims(stack, cache_d, cos_d):
    """Caches, and RoPE tables, of another head_dim than the model's: the stack addresses both by the model's."""
    cache = torch.zeros((BLOCKS, 2, 2, 16, cache_d), dtype=torch.float16)
    with pytest.raises(ValueError):
        stack.forward(k_cache=cache, v_cache=cache, **arguments(stack, cos_d))
    assert not stack.calls


def test_forward_takes_the_models_head_dim(stack):
    cache = torch.zeros((BLOCKS, 2, 2, 16, 128), dtype=torch.float16)
    stack.forward(k_cache=cache, v_cache=cache, **arguments(stack))
    assert stack.calls == ["nsd_decoder_forward"]


def cache8(**change):
    return SimpleNamespace(**{**dict(device=-1, num_layers=2, num_kv_heads=2, _ref=0), **change})


def test_forward_kv8_takes_its_arguments(stack):
    stack.forward_kv8(cache=cache8(), **arguments(stack))
    assert stack.calls == ["nsd_decoder_forward_kv8"]


@pytest.mark.parametrize("block_size", [8, 32])
def test_forward_kv8_refuses_other_block_sizes(stack, block_size):
    """A cache's blocks hold 16 tokens: with another size the table's entries would mean other tokens."""
    args = arguments(stack)
    args["engine_config"] = EngineConfig(block_size=block_size, max_blocks_per_seq=5)
    with pytest.raises(ValueError, match="block_size"):
        stack.forward_kv8(cache=cache8(), **args)
    assert not stack.calls


class Elsewhere(torch.Tensor):
    """A tensor that says it is on another GPU."""

    def get_device(self):
        return 5


def elsewhere(t):
    return t.as_subclass(Elsewhere)


@pytest.mark.parametrize("name,change", [
    *((n, c) for n in ("cos_cache", "sin_cache") for c in (torch.Tensor.float, torch.Tensor.t, elsewhere)),
    *((n, elsewhere) for n in ("x", "residual", "block_table")),
    *((n, c) for n in ("seq_ids", "decoding_seq_lens")
      for c in (torch.Tensor.long, elsewhere, lambda t: t[:-1], lambda t: t.repeat(2)[::2]))])
def test_forward_kv8_refuses_what_its_kernels_cannot_read(stack, name, change):
    args = arguments(stack)
    if name in args:
        args[name] = change(args[name])
        if change is torch.Tensor.t:  # of the right shape, its columns apart
            args[name] = torch.zeros((64, 9), dtype=torch.float16).t()
    else:
        setattr(args["infer_state"], name, change(getattr(args["infer_state"], name)))
    with pytest.raises((TypeError, ValueError)):
        stack.forward_kv8(cache=cache8(), **args)
    assert not stack.calls


def test_forward_kv8_refuses_weights_on_another_gpu(stack):
    stack._layers = [{"wqkv": elsewhere(torch.zeros(1))}] * 2
    with pytest.raises(ValueError, match="weights"):
        stack.forward_kv8(cache=cache8(), **arguments(stack))
    assert not stack.calls


def test_forward_kv8_runs_on_the_caches_device(stack, monkeypatch):
    """A current device that is not the tensors' is changed for the call."""
    on = []

    class Device:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            on.append(self.device)

        def __exit__(self, *e):
            on.append(None)

    def called(name, *a):
        stack.calls.append((name, on[-1] if on else None))

    monkeypatch.setattr(decoder._lib, "call", called)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    monkeypatch.setattr(torch.cuda, "device", Device)
    stack.forward_kv8(cache=cache8(), **arguments(stack))
    assert stack.calls == [("nsd_decoder_forward_kv8", -1)] and on == [-1, None]
