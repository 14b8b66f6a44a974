"""What the 8-bit cache's calls take and refuse before they call native code (no GPU)."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from nebulasd_amd.kernels import kv8

HERE = SimpleNamespace(device=-1)  # as CPU tensors say


def half(*shape):
    return torch.zeros(shape, dtype=torch.float16)


@pytest.mark.parametrize("t,rows,heads,apart", [
    (half(3, 4, 128), 3, 4, 512), (half(3, 9 * 128).view(3, 9, 128)[:, 2:6], 3, 4, 9 * 128),
    # the stride of an axis of one is any number: these are contiguous
    (half(4, 1, 128).transpose(0, 1), 1, 4, 512), (half(1, 3, 128).transpose(0, 1), 3, 1, 128),
    (half(1, 1, 128).transpose(0, 1), 1, 1, 128), (torch.as_strided(half(512), (1, 4, 128), (3, 128, 1)), 1, 4, 512),
    (torch.as_strided(half(1024), (5, 1, 128), (136, 7, 1)), 5, 1, 136)])
def test_rows_of_any_layout_with_contiguous_heads(t, rows, heads, apart):
    assert kv8._rows(HERE, t, "q", rows, heads) == apart


@pytest.mark.parametrize("t,rows,heads", [
    (half(4, 2, 128).transpose(0, 1), 2, 4), (half(1, 4, 128).expand(3, 4, 128), 3, 4), (half(3, 4, 256)[..., ::2], 3, 4),
    (torch.as_strided(half(2048), (3, 4, 128), (516, 128, 1)), 3, 4), (half(3, 4, 128)[:, :, None, 0], 3, 4),
    (torch.as_strided(half(2048), (1, 4, 128), (512, 136, 1)), 1, 4), (half(516)[4:].view(1, 4, 128), 1, 4)])
def test_rows_of_apart_heads_are_refused(t, rows, heads):
    with pytest.raises(ValueError):
        kv8._rows(HERE, t, "q", rows, heads)


class Elsewhere(torch.Tensor):
    """A tensor that says it is on another GPU."""

    def get_device(self):
        return 5


def test_a_plan_on_another_gpu_is_not_used(monkeypatch):
    """An infer state whose plan was made beside another cache's block table: the kernel would read it from that GPU."""
    from nebulasd_amd import plan

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "get_device_properties", lambda d: SimpleNamespace(multi_processor_count=256))
    mc, ec = SimpleNamespace(num_q_heads=4, num_kv_heads=2), SimpleNamespace()
    table = torch.zeros((2, 5), dtype=torch.int32)
    st = SimpleNamespace(seq_ids_list=[0, 1], decoding_seq_lens_list=[7, 80])
    first = plan.kv8_plan_for(st, mc, ec, table)
    assert plan.kv8_plan_for(st, mc, ec, table) is first  # the forward's, for every layer
    other = plan.kv8_plan_for(st, mc, ec, table.as_subclass(Elsewhere))
    assert other is not first and st.kv8_plan is other
