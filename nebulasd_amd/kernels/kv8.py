"""A paged KV cache in 8 bits: ``KV8Cache``, its writers, its reader and the attention over it.

Decode and verify attention is bound by the cache's stream from memory, and the pool's contexts by its size; an
8-bit cache halves the one and doubles the other.  The functions stand beside ``store_kvcache``,
``qk_norm_rope_store`` and ``paged_attention`` (swiftLLM/swiftllm/worker/kernels/kvcache_mgmt.py:81-122,
worker/layers/transformer_layer.py:114-145, worker/kernels/paged_attn.py:152-222; the reference has only fp16
caches) and take a ``KV8Cache`` in place of ``k_cache, v_cache``; prompts attend their own fp16 rows
(``prefill_attention``) as before.

A block of 16 tokens holds, for every layer and kv head, 16 x 128 codes and one power of two for K, and the same for
V.  Codes are E4M3 (4 significant bits, whatever a value's size) or whole numbers from -127 to 127 (7 bits of the
block's largest).  Every value of a cache is an fp16 value, so reading back is exact.  ``include/nsd_kv8.h`` states
the format, what a row, rejected later or not, does to the tokens that its block holds already, and what becomes of
values that are not finite.
"""

from __future__ import annotations

import ctypes

import torch

from .. import _lib
from ..plan import kv8_plan_for
from ._util import StatusWord, check_block_table, ptr, require, require_cuda, stream_on

HEAD_DIM, BLOCK_TOKENS = 128, 16
TILE = HEAD_DIM * BLOCK_TOKENS  # bytes of a block's K (or V) codes of one layer and kv head
_CODES = {torch.float8_e4m3fn: 0, torch.int8: 1}


class _Cache(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "v", "k_scales", "v_scales")] + \
        [("num_blocks", ctypes.c_int64)] + [(n, ctypes.c_int32) for n in ("num_layers", "num_kv_heads", "codes")]


class KV8Cache:
    """A paged KV cache in 8 bits on one GPU.

    ``k``, ``v``: uint8 [num_blocks, num_layers, num_kv_heads, 2048], codes in the kernels' layout; ``k_scales``,
    ``v_scales``: uint8 [num_blocks, num_layers, num_kv_heads], 2^(byte - 127).  ``dtype``: ``torch.float8_e4m3fn``
    or ``torch.int8``.  Block-granular copies (``swap_blocks``, ``HostKVCopyBackend``) take ``k, v`` as one pair of
    caches and the scales as another.
    """

    __slots__ = ("k", "v", "k_scales", "v_scales", "dtype", "device", "num_blocks", "num_layers", "num_kv_heads", "_c",
                 "_ref")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scales: torch.Tensor, v_scales: torch.Tensor,
                 dtype: torch.dtype):
        if dtype not in _CODES:
            raise TypeError(f"codes are torch.float8_e4m3fn or torch.int8, got {dtype}")
        require_cuda(k, v, k_scales, v_scales)
        for t, n in ((k, "k"), (v, "v"), (k_scales, "k_scales"), (v_scales, "v_scales")):
            require(t, torch.uint8, n)
            if t.get_device() != k.get_device():
                raise ValueError("a cache's tensors must be on one device")
        if k.dim() != 4 or k.shape[3] != TILE or v.shape != k.shape or min(k.shape) < 1:
            raise ValueError(f"k and v must be [num_blocks, num_layers, num_kv_heads, {TILE}]")
        if k_scales.shape != k.shape[:3] or v_scales.shape != k.shape[:3]:
            raise ValueError("scales must be [num_blocks, num_layers, num_kv_heads]")
        if k.data_ptr() % 16 or v.data_ptr() % 16:
            raise ValueError("codes must be 16-byte aligned")
        c = _Cache(k.data_ptr(), v.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(), *k.shape[:3], _CODES[dtype])
        for name, x in zip(self.__slots__, (k, v, k_scales, v_scales, dtype, k.get_device(), *k.shape[:3], c,
                                            ctypes.addressof(c))):
            object.__setattr__(self, name, x)

    def __setattr__(self, name, value):
        raise AttributeError("a KV8Cache is fixed once made: its sizes were checked then")

    def __reduce__(self):  # copy and pickle
        return type(self), (self.k, self.v, self.k_scales, self.v_scales, self.dtype)

    @classmethod
    def allocate(cls, num_blocks: int, model_config, dtype: torch.dtype = torch.float8_e4m3fn,
                 device="cuda") -> "KV8Cache":
        """An empty cache (its bytes mean nothing) for ``model_config``'s layers and kv heads."""
        if int(model_config.head_dim) != HEAD_DIM:
            raise ValueError(f"head_dim {model_config.head_dim}: the kernels serve {HEAD_DIM}")
        shape = (int(num_blocks), int(model_config.num_layers), int(model_config.num_kv_heads))
        codes = [torch.zeros((*shape, TILE), dtype=torch.uint8, device=device) for _ in range(2)]
        scales = [torch.zeros(shape, dtype=torch.uint8, device=device) for _ in range(2)]
        return cls(*codes, *scales, dtype)

    @classmethod
    def pack(cls, k: torch.Tensor, v: torch.Tensor, k_scales: torch.Tensor, v_scales: torch.Tensor) -> "KV8Cache":
        """The cache that holds these codes, [num_blocks, num_layers, num_kv_heads, 16, 128] in the fp16 caches' order
        (``torch.float8_e4m3fn`` or ``torch.int8``; -128 is no code), under these scale bytes."""
        if k.dtype not in _CODES or v.dtype != k.dtype:
            raise TypeError(f"codes are torch.float8_e4m3fn or torch.int8, got {k.dtype} and {v.dtype}")
        if k.dim() != 5 or tuple(k.shape[3:]) != (BLOCK_TOKENS, HEAD_DIM) or v.shape != k.shape:
            raise ValueError(f"codes must be [num_blocks, num_layers, num_kv_heads, {BLOCK_TOKENS}, {HEAD_DIM}]")
        bias = 128 if k.dtype == torch.int8 else 0
        kb, vb = (t.view(torch.uint8) ^ bias for t in (k, v))
        top = k.shape[:3]
        kb = kb.view(*top, 16, 2, 8, 8).permute(0, 1, 2, 5, 3, 4, 6)  # [token, half, c, dim] -> [c, token, half, dim]
        vb = vb.view(*top, 4, 4, 16, 2, 4).permute(0, 1, 2, 6, 3, 5, 7, 4)  # [g, j, i, h, m] -> [h, g, i, m, j]
        return cls(*(t.reshape(*top, TILE) for t in (kb, vb)), k_scales.contiguous(), v_scales.contiguous(), k.dtype)

    def codes(self):
        """``pack``'s inverse: codes and scale bytes ``(k, v, k_scales, v_scales)``."""
        bias = 128 if self.dtype == torch.int8 else 0
        top = self.k.shape[:3]
        kb = self.k.view(*top, 8, 16, 2, 8).permute(0, 1, 2, 4, 5, 3, 6)
        vb = self.v.view(*top, 2, 4, 16, 4, 4).permute(0, 1, 2, 4, 7, 5, 3, 6)
        return (*((t.reshape(*top, BLOCK_TOKENS, HEAD_DIM) ^ bias).view(self.dtype) for t in (kb, vb)),
                self.k_scales.clone(), self.v_scales.clone())


def _call(device: int, name: str, *args) -> None:
    """``name`` on a device and its current stream."""
    f = getattr(_lib.load(), name)
    if device == torch.cuda.current_device():
        rc = f(*args, stream_on(device))
    else:
        with torch.cuda.device(device):
            rc = f(*args, stream_on(device))
    if rc:
        _lib.check(rc, name)


def _on(cache: KV8Cache, *tensors) -> None:
    for t in tensors:
        if t is not None and t.get_device() != cache.device:
            require_cuda(t)
            raise ValueError(f"all tensors must be on the cache's device, cuda:{cache.device}, got {t.device}")


# The checks of a call are a good part of a small one's time, so each begins with
# one test of everything, over as few of a tensor's attributes as tell it (each is
# a tenth of a microsecond), and names the fault only where that fails.
_F16, _I32 = torch.float16, torch.int32


def _packed(cache: KV8Cache, t: torch.Tensor, name: str, heads: int, rows: int) -> None:
    """t: contiguous fp16 [rows, heads, 128] on the cache's device."""
    if t.dtype is _F16 and t.shape == (rows, heads, HEAD_DIM) and t.is_contiguous() and t.get_device() == cache.device:
        return
    _on(cache, t)
    require(t, _F16, name)
    raise ValueError(f"{name} must be [{rows}, {heads}, {HEAD_DIM}], got {tuple(t.shape)}")


def _index(cache: KV8Cache, t: torch.Tensor, name: str, n: int) -> None:
    """t: contiguous int32 of at least n entries on the cache's device."""
    if t.dtype is _I32 and t.ndim == 1 and t.numel() >= n and t.is_contiguous() and t.get_device() == cache.device:
        return
    require(t, _I32, name)
    _on(cache, t)
    raise ValueError(f"{name} must hold {n} entries, got {tuple(t.shape)}")


def _rows(cache: KV8Cache, t: torch.Tensor, name: str, rows: int, heads: int) -> int:
    """t: fp16 [rows, heads, 128] of contiguous heads, aligned, on the cache's device; its row stride."""
    if t.dtype is _F16 and t.shape == (rows, heads, HEAD_DIM) and t.get_device() == cache.device:
        apart, per_head, per_dim = t.stride()
        if per_dim == 1 and per_head == HEAD_DIM and apart % 8 == 0 and apart >= heads * HEAD_DIM and \
                t.data_ptr() % 16 == 0:
            return apart
        # the stride of an axis of one says nothing
        apart = apart if rows > 1 else heads * HEAD_DIM
        if per_dim == 1 and (per_head == HEAD_DIM or heads == 1) and apart % 8 == 0 and apart >= heads * HEAD_DIM and \
                t.data_ptr() % 16 == 0:
            return apart
    _on(cache, t)
    if t.dtype != _F16:
        raise TypeError(f"{name} must be torch.float16, got {t.dtype}")
    raise ValueError(f"{name} must be [{rows}, {heads}, {HEAD_DIM}] with contiguous heads (rows may be strided by a "
                     f"multiple of 8 elements), 16-byte aligned; got {tuple(t.shape)}, strides {t.stride()}")


def _table(cache: KV8Cache, block_table: torch.Tensor, engine_config) -> tuple:
    shape = block_table.shape
    if not (block_table.dtype is _I32 and block_table.is_contiguous() and block_table.get_device() == cache.device and
            len(shape) == 2 and shape[1] == engine_config.max_blocks_per_seq):
        _on(cache, block_table)
        check_block_table(block_table, engine_config)
    if engine_config.block_size != BLOCK_TOKENS:
        raise ValueError(f"engine_config.block_size is {engine_config.block_size}, the cache's blocks hold "
                         f"{BLOCK_TOKENS} tokens")
    return block_table.data_ptr(), shape[0], shape[1]


def _decode_rows(cache: KV8Cache, infer_state) -> tuple:
    """(seq_ids, seq_lens, rows) of the forward's decode/verify rows, as pointers."""
    npf, nd = infer_state.num_prefill_seqs, infer_state.num_decoding_seqs
    _index(cache, infer_state.seq_ids, "infer_state.seq_ids", npf + nd)
    _index(cache, infer_state.decoding_seq_lens, "infer_state.decoding_seq_lens", nd)
    return infer_state.seq_ids.data_ptr() + 4 * npf, infer_state.decoding_seq_lens.data_ptr(), nd


def _prologue_tables(cache: KV8Cache, q_norm, k_norm, cos_cache, sin_cache) -> int:
    """Checks the prologue's norm weights and RoPE tables; the positions that these hold."""
    if (q_norm is None) != (k_norm is None):
        raise ValueError("pass both q_norm and k_norm, or neither")
    if q_norm is not None:
        for t, n in ((q_norm, "q_norm"), (k_norm, "k_norm")):
            if t.dtype is not _F16 or t.shape != (HEAD_DIM,) or not t.is_contiguous() or t.get_device() != cache.device:
                _on(cache, t)
                require(t, _F16, n)
                raise ValueError(f"{n} must be [{HEAD_DIM}], got {tuple(t.shape)}")
    angles = cos_cache.shape
    if len(angles) != 2 or angles[1] != HEAD_DIM // 2 or sin_cache.shape != angles:
        raise ValueError("cos/sin caches must be [max_positions, head_dim/2]")
    for t, n in ((cos_cache, "cos_cache"), (sin_cache, "sin_cache")):
        if t.dtype is not _F16 or not t.is_contiguous() or t.get_device() != cache.device:
            _on(cache, t)
            require(t, _F16, n)
    return angles[0]


def kv8_store(k: torch.Tensor, v: torch.Tensor, cache: KV8Cache, block_table: torch.Tensor, model_config,
              engine_config, infer_state, cur_layer: int, validate: bool = False) -> None:
    """``store_kvcache`` into an 8-bit cache: every token's K/V of the forward at layer ``cur_layer``.

    ``k``/``v``: [num_tokens, Hkv, d] fp16, prompts first, then one row per decode/verify row.  A prompt's blocks are
    written whole; a decode/verify row joins the tokens that its block holds below it.
    """
    table = _table(cache, block_table, engine_config)
    hkv = cache.num_kv_heads
    npf, nd = infer_state.num_prefill_seqs, infer_state.num_decoding_seqs
    npt = infer_state.num_prefill_tokens
    _packed(cache, k, "k", hkv, npt + nd)
    _packed(cache, v, "v", hkv, npt + nd)
    status = StatusWord(k.device) if validate else None
    flags = ptr(status.t) if status else None
    if npf > 0:
        ids, starts, lens = infer_state.seq_ids, infer_state.prefill_seq_start_locs, infer_state.prefill_seq_lens
        _index(cache, ids, "infer_state.seq_ids", npf)
        _index(cache, starts, "infer_state.prefill_seq_start_locs", npf)
        _index(cache, lens, "infer_state.prefill_seq_lens", npf)
        _call(cache.device, "nsd_kv8_store_prefill", k.data_ptr(), v.data_ptr(), npt, cache._ref, *table,
              ids.data_ptr(), starts.data_ptr(), lens.data_ptr(), npf, infer_state.max_prefill_len, int(cur_layer), flags)
    if nd > 0:
        at = 2 * npt * hkv * HEAD_DIM  # bytes of the prompts' rows
        _call(cache.device, "nsd_kv8_store", k.data_ptr() + at, v.data_ptr() + at, cache._ref, *table,
              *_decode_rows(cache, infer_state), int(cur_layer), flags)
    if status is not None:
        status.check("kv8_store")


def kv8_qk_norm_rope_store(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: KV8Cache,
                           block_table: torch.Tensor, q_norm: torch.Tensor | None, k_norm: torch.Tensor | None,
                           model_config, engine_config, infer_state, cur_layer: int, cos_cache: torch.Tensor,
                           sin_cache: torch.Tensor, validate: bool = False,
                           q_out: torch.Tensor | None = None) -> None:
    """``qk_norm_rope_store`` into an 8-bit cache, one launch: the decode/verify rows' QK-norm, RoPE and store.

    ``q`` [rows, Hq, d], ``k``/``v`` [rows, Hkv, d] fp16 may be row-strided slices of one fused q/k/v projection (rows a
    multiple of 8 elements apart); the normalised, rotated q goes to ``q_out``, or, with contiguous q and no ``q_out``,
    into q.  k and v are only read.  ``cos_cache``/``sin_cache``: the full [max_positions, d/2] fp16 tables.
    """
    table = _table(cache, block_table, engine_config)
    rows, hq, hkv = infer_state.num_decoding_seqs, model_config.num_q_heads, cache.num_kv_heads
    q_stride = _rows(cache, q, "q", rows, hq)
    k_stride = _rows(cache, k, "k", rows, hkv)
    v_stride = _rows(cache, v, "v", rows, hkv)
    if q_out is None:
        if not q.is_contiguous():
            raise ValueError("strided q needs q_out (a contiguous [rows, Hq, d] buffer)")
        q_out = q
    else:
        _packed(cache, q_out, "q_out", hq, rows)
    positions = _prologue_tables(cache, q_norm, k_norm, cos_cache, sin_cache)
    if rows == 0:
        return
    if getattr(infer_state, "ignore_kvcache", False):
        raise ValueError("infer_state.ignore_kvcache is set but the forward has decode rows")
    status = StatusWord(q.device) if validate else None
    _call(cache.device, "nsd_kv8_qk_norm_rope_store", q.data_ptr(), q_stride, q_out.data_ptr(), k.data_ptr(), k_stride,
          v.data_ptr(), v_stride, ptr(q_norm), ptr(k_norm), model_config.rms_norm_eps, cos_cache.data_ptr(),
          sin_cache.data_ptr(), positions, cache._ref, *table,
          *_decode_rows(cache, infer_state), int(cur_layer), hq, ptr(status.t) if status else None)
    if status is not None:
        status.check("kv8_qk_norm_rope_store")


def kv8_qk_norm_rope_store_partials(partials: torch.Tensor, q_out: torch.Tensor, cache: KV8Cache,
                                    block_table: torch.Tensor, q_norm: torch.Tensor | None,
                                    k_norm: torch.Tensor | None, model_config, engine_config, infer_state,
                                    cur_layer: int, cos_cache: torch.Tensor, sin_cache: torch.Tensor,
                                    validate: bool = False) -> None:
    """``kv8_qk_norm_rope_store`` over the rows' fused q/k/v projection as split partials, fp32 [splits, rows, (Hq + 2
    Hkv) d] (``linear_partials``); q goes to ``q_out`` [rows, Hq, d]."""
    table = _table(cache, block_table, engine_config)
    rows, hq = infer_state.num_decoding_seqs, model_config.num_q_heads
    width = (hq + 2 * cache.num_kv_heads) * HEAD_DIM
    _on(cache, partials)
    require(partials, torch.float32, "partials")
    if partials.ndim != 3 or partials.shape[1:] != (rows, width):
        raise ValueError(f"partials must be [splits, {rows}, {width}], got {tuple(partials.shape)}")
    _packed(cache, q_out, "q_out", hq, rows)
    positions = _prologue_tables(cache, q_norm, k_norm, cos_cache, sin_cache)
    if rows == 0:
        return
    if getattr(infer_state, "ignore_kvcache", False):
        raise ValueError("infer_state.ignore_kvcache is set but the forward has decode rows")
    status = StatusWord(q_out.device) if validate else None
    _call(cache.device, "nsd_kv8_qk_norm_rope_store_partials", partials.data_ptr(), partials.shape[0],
          q_out.data_ptr(), ptr(q_norm), ptr(k_norm), model_config.rms_norm_eps, cos_cache.data_ptr(),
          sin_cache.data_ptr(), positions, cache._ref, *table, *_decode_rows(cache, infer_state), int(cur_layer), hq,
          ptr(status.t) if status else None)
    if status is not None:
        status.check("kv8_qk_norm_rope_store_partials")


def kv8_load(k: torch.Tensor, v: torch.Tensor, cache: KV8Cache, block_table: torch.Tensor, seq_ids: torch.Tensor,
             start_locs: torch.Tensor, seq_lens: torch.Tensor, max_len: int, cur_layer: int,
             first: torch.Tensor | None = None, validate: bool = False) -> None:
    """The values of cached tokens as packed fp16 rows, exactly.

    Token ``first[s] + i`` (``first`` None: ``i``) of ``block_table[seq_ids[s]]``, ``i < seq_lens[s] <= max_len``, goes
    to row ``start_locs[s] + i`` of ``k`` and ``v`` [rows, Hkv, d]; other rows are left as they are.  The index tensors
    are int32, one entry a sequence.
    """
    if block_table.dtype is not _I32 or block_table.ndim != 2 or not block_table.is_contiguous() or \
            block_table.get_device() != cache.device:
        _on(cache, block_table)
        require(block_table, _I32, "block_table")
        raise ValueError("block_table must be [rows, max_blocks_per_seq]")
    rows = k.shape[0] if k.ndim else 0
    _packed(cache, k, "k", cache.num_kv_heads, rows)
    _packed(cache, v, "v", cache.num_kv_heads, rows)
    n = seq_ids.numel()
    for t, name in ((seq_ids, "seq_ids"), (start_locs, "start_locs"), (seq_lens, "seq_lens"), (first, "first")):
        if t is not None and not (t.dtype is _I32 and t.shape == (n,) and t.is_contiguous() and
                                  t.get_device() == cache.device):
            _index(cache, t, name, n)
            raise ValueError(f"{name} must be [{n}], one entry a sequence")
    if n == 0 or rows == 0:
        return
    status = StatusWord(k.device) if validate else None
    _call(cache.device, "nsd_kv8_load", k.data_ptr(), v.data_ptr(), rows, cache._ref, block_table.data_ptr(),
          *block_table.shape, seq_ids.data_ptr(), ptr(first), start_locs.data_ptr(), seq_lens.data_ptr(), n,
          int(max_len), int(cur_layer), ptr(status.t) if status else None)
    if status is not None:
        status.check("kv8_load")


def kv8_paged_attention(q: torch.Tensor, cache: KV8Cache, block_table: torch.Tensor, model_config, engine_config,
                        infer_state, cur_layer: int, o: torch.Tensor, lse: torch.Tensor | None = None,
                        validate: bool = False) -> None:
    """``paged_attention`` over an 8-bit cache: the attention over the values it holds, with the same plan.

    ``q``: [num_decoding_seqs, Hq, d] fp16; ``o``: as many elements, written in place; ``lse``: fp32 [rows, Hq], the
    natural-log sum of exp(score).  Scratch is the call's own (from the caching allocator), so calls on several
    streams and in several captured graphs share nothing but the forward's plan, which the first call uploads on its
    stream (``infer_state.kv8_plan``; a capture needs it built before).
    """
    table = _table(cache, block_table, engine_config)
    rows, hq = infer_state.num_decoding_seqs, model_config.num_q_heads
    _packed(cache, q, "q", hq, rows)
    if o.dtype is not _F16 or not o.is_contiguous() or o.get_device() != cache.device or o.numel() != rows * hq * HEAD_DIM:
        _on(cache, o)
        require(o, _F16, "o")
        raise ValueError(f"o must hold as many elements as q, {rows} x {hq} x {HEAD_DIM}")
    if lse is not None and (lse.dtype is not torch.float32 or not lse.is_contiguous() or
                            lse.get_device() != cache.device or lse.numel() != rows * hq):
        _on(cache, lse)
        require(lse, torch.float32, "lse")
        raise ValueError("lse must hold num_decoding_seqs * num_q_heads floats")
    if model_config.num_kv_heads != cache.num_kv_heads:
        raise ValueError(f"model_config has {model_config.num_kv_heads} kv heads, the cache {cache.num_kv_heads}")
    if rows == 0:
        return
    plan = kv8_plan_for(infer_state, model_config, engine_config, block_table)
    if plan.n_rows != rows:
        raise ValueError(f"the forward's attention plan covers {plan.n_rows} rows, q has {rows}")
    size, ws = plan.workspace_bytes, None
    if size:
        # the claim counter of plans with more pieces than workgroup slots starts at zero
        ws = (q.new_zeros if plan.claims else q.new_empty)(size, dtype=torch.uint8)
    status = StatusWord(q.device) if validate else None
    _call(cache.device, "nsd_kv8_paged_attention", q.data_ptr(), o.data_ptr(), ptr(lse), cache._ref, int(cur_layer),
          hq, *table, plan.host_address, plan.dev.data_ptr(), ptr(ws), size, infer_state.softmax_scale,
          ptr(status.t) if status else None)
    if status is not None:
        status.check("kv8_paged_attention")
