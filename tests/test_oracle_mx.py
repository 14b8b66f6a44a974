"""Pins of the microscaled oracle (no GPU), and the refusals that need none."""

from __future__ import annotations

import ctypes
import subprocess

import numpy as np
import pytest
import torch

import mx_shapes
import oracle
from oracle import E2M1, E4M3, mx_linear, mx_pack_nibbles, mx_quantize, mx_unpack_nibbles, mx_up_gate, mx_values


def test_value_tables():
    assert E2M1.tolist() == [0, .5, 1, 1.5, 2, 3, 4, 6]
    every = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(every, E4M3) and E4M3[-1] == 448


def _blocks(seed, n=64, k=96):
    rng = np.random.default_rng(seed)
    return rng.standard_normal((n, k)) * 2.0 ** rng.integers(-12, 9, (n, 1))


@pytest.mark.parametrize("bits,table", [(4, E2M1), (8, E4M3)])
def test_nearest_code_ties_to_even(bits, table):
    x = _blocks(1).astype(np.float16).astype(np.float64)
    x[:, ::7] = np.round(x[:, ::7] * 64) / 64  # some on middles
    codes, scales = mx_quantize(x, bits)
    s = np.ldexp(1.0, np.repeat(scales.astype(np.int64) - 127, 32, axis=1))
    a, mag = np.abs(x) / s, codes & (2 ** (bits - 1) - 1)
    off = np.abs(a - table[mag])
    every = np.abs(a[..., None] - table)
    assert np.array_equal(off, every.min(-1))  # no code is nearer, saturation included
    ties = (every == off[..., None]).sum(-1) == 2
    assert (mag[ties] % 2 == 0).all()
    assert np.array_equal(codes >> (bits - 1), np.signbit(x))


def test_scale_rules():
    m = np.abs(_blocks(2).reshape(64, 3, 32)).max(-1)
    s4 = mx_quantize(_blocks(2), 4)[1].astype(np.int64) - 127
    s8 = mx_quantize(_blocks(2), 8)[1].astype(np.int64) - 127
    assert (np.ldexp(4.0, s4) <= m).all() and (m < np.ldexp(8.0, s4)).all()
    assert (m <= np.ldexp(448.0, s8)).all() and (m > np.ldexp(448.0, s8 - 1)).all()


def test_codes_match_torch_e4m3():
    x = _blocks(3).astype(np.float16)
    codes, scales = mx_quantize(x, 8)
    s = np.ldexp(1.0, -np.repeat(scales.astype(np.int64) - 127, 32, axis=1))
    want = torch.from_numpy(x.astype(np.float64) * s).float().to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(codes, want)


@pytest.mark.parametrize("bits", [4, 8])
def test_closed_forms(bits):
    x = np.zeros((6, 32))
    x[1, 3] = -1.0
    x[2] = 7.0 if bits == 4 else 448.0   # 7: past 6 at the scale 1
    x[3, 0], x[4, 5] = np.inf, np.nan
    x[5, 0] = 2.0 ** -140
    codes, scales = mx_quantize(x, bits)
    v = mx_values(codes, scales, bits)
    assert scales[0, 0] == 0 and not v[0].any()
    assert v[1, 3] == -1 and np.count_nonzero(v[1]) == 1
    assert int(scales[1, 0]) - 127 == (-2 if bits == 4 else -8)
    assert (v[2] == (6.0 if bits == 4 else 448.0)).all()
    assert (scales[3:5] == 255).all() and np.isnan(v[3:5]).all()
    assert scales[5, 0] == 0 and v[5, 0] == 0
    if bits == 8:
        x = np.full((1, 32), np.nextafter(448.0, 449))  # just past the top: the next scale, no saturation
        assert mx_quantize(x, 8)[1][0, 0] == 128


@pytest.mark.parametrize("bits", [4, 8])
def test_values_quantise_to_themselves(bits):
    codes, scales = mx_quantize(_blocks(4), bits)
    v = mx_values(codes, scales, bits)
    again = mx_values(*mx_quantize(v, bits), bits)
    assert np.array_equal(v, again)


def test_nibbles():
    c = np.arange(64, dtype=np.uint8).reshape(2, 32) % 16
    p = mx_pack_nibbles(c)
    assert p.shape == (2, 16) and p[0, 0] == 0x10 and np.array_equal(mx_unpack_nibbles(p), c)


def test_products():
    w = mx_values(*mx_quantize(_blocks(5, 20, 64), 4), 4)
    one = np.zeros((64, 64), np.float16)
    one[np.arange(64), np.arange(64)] = 1
    assert np.array_equal(mx_linear(one, w), w.T)
    x = _blocks(6, 9, 64).astype(np.float16)
    xv = torch.from_numpy(mx_values(*mx_quantize(x, 8), 8))
    y = torch.nn.functional.linear(xv, torch.from_numpy(w))
    np.testing.assert_allclose(mx_linear(x, w), y.numpy(), rtol=1e-12, atol=1e-12)
    up, gate = y.chunk(2, 1)
    np.testing.assert_allclose(mx_up_gate(x, w), (up * torch.nn.functional.silu(gate)).numpy(), rtol=1e-12, atol=1e-12)
    assert not np.allclose(mx_up_gate(x, np.roll(w, 10, 0)), mx_up_gate(x, w))  # the halves swapped


def test_a_wrong_scale_is_seen():
    x = _blocks(7)
    codes, scales = mx_quantize(x, 4)
    assert not np.allclose(mx_values(codes, scales + 1, 4), mx_values(codes, scales, 4))


def test_bound_covers_every_eight_of_a_block():
    """Four large products a block, one in every eight, each beside seven that just miss its last place."""
    x = np.full((1, 32), 1.875 * 2.0 ** -4, np.float16)
    w = np.ones((1, 32))
    x[0, ::8], w[0, ::8] = 256.0, 4.0
    lost = mx_linear(x, w)[0, 0] - 4 * 1024
    assert lost == 28 * 1.875 * 2.0 ** -4 < oracle.mx_linear_bound(x, w)[0, 0]


@pytest.mark.parametrize("bits", [4, 8])
def test_bound_counts_subnormal_codes_with_their_exponent(bits):
    """Beside a large operand on the other side an eight whose codes are all subnormal is cut as if they were not."""
    x, w = np.full((1, 32), 256.0, np.float16), np.full((1, 32), 6.0)
    if bits == 4:
        w[0, 8:16] = .5   # 2^0 to the instruction
        power = 2.0 ** 8 * 4 * 3 + 2.0 ** 8 * 1
    else:
        x[0, 8:16] = 2.0 ** -9  # 2^-6
        power = 2.0 ** 8 * 4 * 3 + 2.0 ** -6 * 4
    assert oracle.mx_linear_bound(x, w)[0, 0] >= 7 * 2.0 ** -13 * power


def test_cut_products():
    """Beside 2^(8 + 2): 1/8 stays, 1/16 goes, 3/16 becomes 1/8, either sign; another eight is not touched; beside
    448 * 0 nothing is cut; 0.5 in the weight counts as 2^0."""
    x, w = np.zeros((1, 32), np.float16), np.zeros((7, 32))
    x[0, :3], x[0, 8] = (256, 2.0 ** -4, -2.0 ** -3), 2.0 ** -4
    w[0, :2], w[1, :2], w[2, :3] = (4, 2), (4, 1), (4, 3, 0)
    w[3, :3], w[4, 0], w[4, 8], w[5, 1], w[6, :2] = (-4, 0, 1.5), 4, 1, 1, (.5, .5)
    mag = np.searchsorted(E2M1, np.abs(w)).astype(np.uint8) | (np.signbit(w).astype(np.uint8) << 3)
    got = oracle.mx_linear_cut(x, mag, np.full((7, 1), 127, np.uint8))[0]
    assert got.tolist() == [1024 + .125, 1024, 1024 + .125, -1024 - .125, 1024 + 2.0 ** -4, 2.0 ** -4, 128 + 2.0 ** -5]


def test_cut_sums_lie_within_the_bound():
    x = (_blocks(8, 9, 544) * np.where(np.arange(544) % 61 == 0, 24, 1)).astype(np.float16)
    codes, scales = mx_quantize(_blocks(9, 21, 544), 4)
    w = mx_values(codes, scales, 4)
    off = np.abs(oracle.mx_linear_cut(x, codes, scales) - mx_linear(x, w))
    assert off.max() > 0 and (off <= oracle.mx_linear_bound(x, w)).all()


# ---- the C entries, short of a GPU ------------------------------------------------


@pytest.fixture(scope="module")
def lib():
    from nebulasd_amd import _lib
    from nebulasd_amd.build import build

    if not _lib.LIB_PATH.exists():
        build()
    return _lib.load()


def _sizes(lib, bits, rows, n_in):
    c, s = ctypes.c_int64(-1), ctypes.c_int64(-1)
    return lib.nsd_mx_bytes(bits, rows, n_in, ctypes.byref(c), ctypes.byref(s)), c.value, s.value


def test_bytes(lib):
    assert _sizes(lib, 4, 16, 128) == (0, 1024, 256)
    assert _sizes(lib, 8, 16, 128) == (0, 2048, 256)
    assert _sizes(lib, 4, 17, 544) == (0, 2 * 5 * 1024, 2 * 2 * 256)
    assert _sizes(lib, 8, 0, 32) == (0, 0, 0)
    assert _sizes(lib, 4, 151936, 4096) == (0, 151936 * 2048, 9496 * 8 * 256)


@pytest.mark.parametrize("bits,rows,n_in,rc", [(4, 16, 48, 2), (4, 16, 0, 2), (8, -1, 32, 2), (5, 16, 32, 1),
                                               (4, 2 ** 31, 32, 2), (8, 2 ** 31 - 1, 2 ** 31 - 32, 2)])
def test_bytes_refuses(lib, bits, rows, n_in, rc):
    from nebulasd_amd import _lib

    assert _sizes(lib, bits, rows, n_in)[0] == rc and "mx_bytes" in _lib.last_error()


def test_entries_refuse_before_any_launch(lib):
    from nebulasd_amd import _lib

    def refused(rc, got, text):
        assert got == rc and text in _lib.last_error(), (got, _lib.last_error())

    ok, odd = 4096, 4098  # never read: every call below is refused first
    refused(1, lib.nsd_mxfp4_quantize(None, 0, 16, 32, ok, ok, None), "null")
    refused(2, lib.nsd_mxfp4_quantize(ok, 7, 16, 32, ok, ok, None), "dtype=7")
    refused(2, lib.nsd_mxfp4_quantize(ok, 0, 16, 33, ok, ok, None), "n_in=33")
    refused(2, lib.nsd_mxfp4_quantize(odd, 0, 16, 32, ok, ok, None), "aligned")
    refused(1, lib.nsd_mxfp4_pack(ok, None, 16, 32, ok, ok, None), "null")
    refused(2, lib.nsd_mxfp8_quantize(ok, 16, 40, ok, ok, None), "n_in=40")
    refused(2, lib.nsd_mxfp8_dequantize(ok, ok, 16, 32, ok, 3, None), "dtype=3")
    refused(1, lib.nsd_mxfp4_linear(None, None, None, ok, ok, ok, 1, 16, 32, None, 0, None), "null")
    refused(2, lib.nsd_mxfp4_linear(ok, None, None, ok, ok, odd, 1, 16, 32, None, 0, None), "aligned")
    refused(2, lib.nsd_mxfp4_linear(ok, None, None, ok, ok, ok, 1, 0, 32, None, 0, None), "n_out=0")
    refused(2, lib.nsd_mxfp4_linear(ok, None, None, ok, ok, ok, 2 ** 22, 16, 32, None, 0, None), "n_rows")
    refused(2, lib.nsd_mxfp4_up_gate_silu_and_mul(ok, None, None, ok, ok, ok, 1, 24, 32, None, 0, None), "inter=24")
    refused(1, lib.nsd_mxfp4_linear(ok, None, None, ok, ok, ok + 32, 1, 32, 32, None, 0, None), "overlaps")
    refused(1, lib.nsd_mxfp4_linear(None, ok, ok, 1 << 20, 1 << 20, ok, 1, 32, 32, None, 0, None), "overlaps")
    refused(2, lib.nsd_mxfp4_linear(ok, None, None, ok, ok, 1 << 20, 1, 32, 2 ** 20 + 32, None, 0, None), "n_in=1048608")
    # no rows: nothing to launch
    assert lib.nsd_mxfp4_linear(None, None, None, None, None, None, 0, 16, 32, None, 0, None) == 0
    assert lib.nsd_mxfp4_quantize(None, 0, 0, 32, None, None, None) == 0


def _workspace(lib, rows, n_out, n_in, gated=0, quantised=0):
    b = ctypes.c_int64(-1)
    return lib.nsd_mx_workspace(rows, n_out, n_in, gated, quantised, ctypes.byref(b)), b.value


@pytest.mark.parametrize("gated", [0, 1])
@pytest.mark.parametrize("quantised", [0, 1])
def test_no_rows_need_no_workspace(lib, gated, quantised):
    """The shape of an empty batch, which the products take: nothing is chosen for it."""
    assert _workspace(lib, 0, 1024, 1024, gated, quantised) == (0, 0)


@pytest.mark.parametrize("rows", [0, 1, 300])
@pytest.mark.parametrize("n_out", [1, 16, 33, 4080])
def test_workspace_refuses_what_the_gated_product_refuses(lib, rows, n_out):
    """A gated weight has 2 * inter rows, inter a multiple of 16."""
    from nebulasd_amd import _lib

    assert _workspace(lib, rows, n_out, 1024, gated=1)[0] == 2 and f"n_out={n_out} " in _lib.last_error()


def test_blocks_over_their_values_are_refused(lib):
    """No conversion works in place: a wave's blocks are written while others still read."""
    from nebulasd_amd import _lib

    def refused(rc):
        assert rc == 1 and "overlap" in _lib.last_error(), (rc, _lib.last_error())

    # addresses that are never read
    a, far, n, k = 1 << 20, 1 << 24, 32, 256
    codes4, codes8, scales = _sizes(lib, 4, n, k)[1:], _sizes(lib, 8, n, k)[1:], _sizes(lib, 8, n, k)[2]
    assert codes4[0] == 4096 and codes8[0] == 8192 and scales == 512
    for dtype, size in ((0, 2), (1, 2), (2, 4)):
        last = a + n * k * size - 16
        refused(lib.nsd_mxfp4_quantize(a, dtype, n, k, a, far, None))
        refused(lib.nsd_mxfp4_quantize(a, dtype, n, k, last, far, None))
        refused(lib.nsd_mxfp4_quantize(a, dtype, n, k, far, last, None))
        for back in (lib.nsd_mxfp4_dequantize, lib.nsd_mxfp8_dequantize):
            refused(back(a, far, n, k, a, dtype, None))
            refused(back(last, far, n, k, a, dtype, None))
            refused(back(far, last, n, k, a, dtype, None))
    refused(lib.nsd_mxfp8_quantize(a, n, k, a + 2 * n * k - 16, far, None))
    refused(lib.nsd_mxfp8_quantize(a, n, k, far, a, None))
    refused(lib.nsd_mxfp4_pack(a, far, n, k, a, 2 * far, None))
    refused(lib.nsd_mxfp4_pack(far, a, n, k, a, 2 * far, None))
    refused(lib.nsd_mxfp4_pack(a, far, n, k, 2 * far, far + 240, None))
    # codes and scales over each other
    refused(lib.nsd_mxfp4_quantize(a, 0, n, k, far, far + 4080, None))
    refused(lib.nsd_mxfp8_quantize(a, n, k, far, far + 8176, None))
    refused(lib.nsd_mxfp4_pack(a, 2 * a, n, k, far, far + 4080, None))


def test_workspace_over_the_operands_is_refused(lib):
    from nebulasd_amd import _lib

    a, far = 1 << 20, 1 << 24
    for entry, n, w_rows in ((lib.nsd_mxfp4_linear, 64, 64), (lib.nsd_mxfp4_up_gate_silu_and_mul, 32, 64)):
        w_codes, w_scales = _sizes(lib, 4, w_rows, 128)[1:]
        x_codes, x_scales = _sizes(lib, 8, 100, 128)[1:]
        for given, at, size in (((a, None, None), a, 100 * 256), ((None, a, 2 * a), a, x_codes),
                                ((None, a, 2 * a), 2 * a, x_scales), ((a, None, None), 3 * a, w_codes),
                                ((a, None, None), 4 * a, w_scales)):
            for ws in (at, at + size - 16, at - 240):
                rc = entry(*given, 3 * a, 4 * a, far, 100, n, 128, ws, 256, None)
                assert rc == 1 and "workspace overlaps" in _lib.last_error(), (rc, _lib.last_error())


def test_a_workspace_of_no_bytes_overlaps_nothing(lib):
    """It is too small for this shape, which is what the call is refused for (without a GPU: for that)."""
    a, far = 1 << 20, 1 << 24
    for at in (a + 16, 3 * a + 16, far + 16):
        assert lib.nsd_mxfp4_linear(a, None, None, 3 * a, 4 * a, far, 100, 64, 128, at, 0, None) in (3, 4)


# ---- the rule that chooses a product's kernel, compiled for the host -------------

_CHOICE = """
#include "nsd_mx_choose.h"
extern "C" void choice(int64_t rows, int64_t n, int64_t n_in, int gated, int quantised, int cus, int* out) {
  const nsd::MxConfig c = nsd::choose_mx(rows, n, nsd::mx_k_tiles(n_in), gated, quantised, cus);
  const int v[] = {c.kernel, c.mt, c.jw, c.fp16, c.nt, c.splits};
  for (int i = 0; i < 6; ++i) out[i] = v[i];
}
extern "C" int past_caches(int mt, int jw, int fp16) { return nsd::mx_stream_nt(mt, jw, fp16); }
extern "C" int fp16_tiles() { return nsd::kMxFp16Tiles; }
"""
STREAM = 0


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    from nebulasd_amd.build import CSRC

    at = tmp_path_factory.mktemp("mx_choose")
    (at / "choice.cpp").write_text(_CHOICE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", str(at / "choice.cpp"),
                    "-o", str(at / "choice.so")], check=True)
    lib = ctypes.CDLL(str(at / "choice.so"))
    lib.choice.argtypes = [ctypes.c_int64] * 3 + [ctypes.c_int] * 3 + [ctypes.POINTER(ctypes.c_int)]
    return lib


def _choice(rule, rows, n, n_in, gated, quantised, cus=256):
    """(kernel, row tiles, column tiles, x as fp16, past the caches, splits)."""
    out = (ctypes.c_int * 6)()
    rule.choice(rows, n, n_in, gated, quantised, cus, out)
    return tuple(out)


def test_shapes_take_every_kernel(rule):
    """The GPU tests' shapes run every kernel that is compiled, and no kernel is compiled that no shape takes."""
    for gated, shapes in ((0, mx_shapes.LINEAR + mx_shapes.LINEAR_LARGE), (1, mx_shapes.GATED + mx_shapes.GATED_LARGE)):
        taken = {_choice(rule, r, n, k, gated, q)[:5] for r, n, k, q in shapes}
        compiled = {(STREAM, mt, jw, fp16, nt)
                    for mt in range(1, 9) for jw in ((2, 4, 6) if gated else (1, 2, 3, 4, 6))
                    for fp16 in range(2 if mt <= rule.fp16_tiles() else 1)
                    for nt in range(1 + bool(rule.past_caches(mt, jw, fp16)))}
        stream = {c for c in taken if c[0] == STREAM}
        assert stream == compiled, (compiled - stream, stream - compiled)
        assert {c[0] for c in taken} == {0, 1, 2}


def test_large_shapes_go_past_the_caches(rule):
    for gated, shapes in ((0, mx_shapes.LINEAR_LARGE), (1, mx_shapes.GATED_LARGE)):
        assert all(_choice(rule, r, n, k, gated, q)[4] for r, n, k, q in shapes)


def test_wrappers_refuse(lib):
    from nebulasd_amd import kernels as K

    x = torch.zeros(4, 64, dtype=torch.float16)
    for f in (K.mxfp4_quantize, K.mxfp8_quantize):
        with pytest.raises(ValueError, match="GPU tensors"):
            f(x)
    with pytest.raises(ValueError, match="GPU tensors"):
        K.mxfp4_pack(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8))


def test_bound_covers_lost_products():
    """A block whose largest product hides 31 others under 2^-15 of it: the bound allows all of them to be lost."""
    x = np.full((1, 32), 2.0 ** -9, np.float16)
    x[0, 0] = 448.0
    w = np.full((1, 32), 0.5)
    w[0, 0] = 6.0
    lost = mx_linear(x, w)[0, 0] - 448.0 * 6
    assert 0 < lost <= oracle.mx_linear_bound(x, w)[0, 0]
