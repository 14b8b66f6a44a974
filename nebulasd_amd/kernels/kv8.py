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
the format, what a row does to the tokens that its block holds already, and what becomes of values that are not
finite.
"""

from __future__ import annotations

import ctypes

import torch

from .. import _lib
from ..plan import plan_for
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

    __slots__ = ("k", "v", "k_scales", "v_scales", "dtype", "device", "_c", "_ref")

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
        for name, x in zip(self.__slots__, (k, v, k_scales, v_scales, dtype, k.get_device(), c, ctypes.addressof(c))):
            object.__setattr__(self, name, x)

    def __setattr__(self, name, value):
        raise AttributeError("a KV8Cache is fixed once made: its sizes were checked then")

    def __reduce__(self):  # copy and pickle
        return type(self), (self.k, self.v, self.k_scales, self.v_scales, self.dtype)

    @property
    def num_blocks(self) -> int:
        return self.k.shape[0]

    @property
    def num_layers(self) -> int:
        return self.k.shape[1]

    @property
    def num_kv_heads(self) -> int:
        return self.k.shape[2]

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
    if device == torch.cuda.current_device():
        _lib.call(name, *args, stream_on(device))
    else:
        with torch.cuda.device(device):
            _lib.call(name, *args, stream_on(device))


def _on(cache: KV8Cache, *tensors) -> None:
    for t in tensors:
        if t is not None and t.get_device() != cache.device:
            require_cuda(t)
            raise ValueError(f"all tensors must be on the cache's device, cuda:{cache.device}, got {t.device}")


def _index(cache: KV8Cache, t: torch.Tensor, name: str, n: int) -> None:
    require(t, torch.int32, name)
    if t.dim() != 1 or t.shape[0] < n:
        raise ValueError(f"{name} must hold {n} entries, got {tuple(t.shape)}")
    _on(cache, t)


def _rows(t: torch.Tensor, name: str, shape: tuple) -> None:
    if t.dtype != torch.float16:
        raise TypeError(f"{name} must be torch.float16, got {t.dtype}")
    if tuple(t.shape) != shape or t.stride(2) != 1 or t.stride(1) != shape[2] or t.stride(0) % 8 or \
            t.stride(0) < shape[1] * shape[2]:
        raise ValueError(f"{name} must be {list(shape)} with contiguous heads (rows may be strided by a multiple of 8 "
                         f"elements), got {tuple(t.shape)}, strides {t.stride()}")
    if t.data_ptr() % 16:
        raise ValueError(f"{name} must be 16-byte aligned")


def _table(cache: KV8Cache, block_table: torch.Tensor, engine_config) -> tuple:
    _on(cache, block_table)
    check_block_table(block_table, engine_config)
    if int(engine_config.block_size) != BLOCK_TOKENS:
        raise ValueError(f"engine_config.block_size is {engine_config.block_size}, the cache's blocks hold "
                         f"{BLOCK_TOKENS} tokens")
    return block_table.data_ptr(), *block_table.shape


def _decode_rows(cache: KV8Cache, infer_state) -> tuple:
    """(seq_ids, seq_lens, rows) of the forward's decode/verify rows, as pointers."""
    npf, nd = infer_state.num_prefill_seqs, infer_state.num_decoding_seqs
    _index(cache, infer_state.seq_ids, "infer_state.seq_ids", npf + nd)
    _index(cache, infer_state.decoding_seq_lens, "infer_state.decoding_seq_lens", nd)
    return infer_state.seq_ids.data_ptr() + 4 * npf, infer_state.decoding_seq_lens.data_ptr(), nd


def kv8_store(k: torch.Tensor, v: torch.Tensor, cache: KV8Cache, block_table: torch.Tensor, model_config,
              engine_config, infer_state, cur_layer: int, validate: bool = False) -> None:
    """``store_kvcache`` into an 8-bit cache: every token's K/V of the forward at layer ``cur_layer``.

    ``k``/``v``: [num_tokens, Hkv, d] fp16, prompts first, then one row per decode/verify row.  A prompt's blocks are
    written whole; a decode/verify row joins the tokens that its block holds below it.
    """
    _on(cache, k, v)
    table = _table(cache, block_table, engine_config)
    hkv = cache.num_kv_heads
    npf, nd = infer_state.num_prefill_seqs, infer_state.num_decoding_seqs
    npt = infer_state.num_prefill_tokens
    for t, n in ((k, "k"), (v, "v")):
        require(t, torch.float16, n)
        if t.dim() != 3 or tuple(t.shape[1:]) != (hkv, HEAD_DIM) or t.shape[0] != npt + nd:
            raise ValueError(f"{n} must be [{npt + nd}, {hkv}, {HEAD_DIM}], got {tuple(t.shape)}")
    status = StatusWord(k.device) if validate else None
    flags = ptr(status.t) if status else None
    if npf > 0:
        for name in ("prefill_seq_start_locs", "prefill_seq_lens"):
            _index(cache, getattr(infer_state, name), f"infer_state.{name}", npf)
        _index(cache, infer_state.seq_ids, "infer_state.seq_ids", npf)
        _call(cache.device, "nsd_kv8_store_prefill", k.data_ptr(), v.data_ptr(), npt, cache._ref, *table,
              infer_state.seq_ids.data_ptr(), infer_state.prefill_seq_start_locs.data_ptr(),
              infer_state.prefill_seq_lens.data_ptr(), npf, infer_state.max_prefill_len, int(cur_layer), flags)
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
    _on(cache, q, k, v, cos_cache, sin_cache, q_norm, k_norm, q_out)
    table = _table(cache, block_table, engine_config)
    rows, hq, hkv = infer_state.num_decoding_seqs, int(model_config.num_q_heads), cache.num_kv_heads
    for t, n, heads in ((q, "q", hq), (k, "k", hkv), (v, "v", hkv)):
        _rows(t, n, (rows, heads, HEAD_DIM))
    if q_out is None:
        if not q.is_contiguous():
            raise ValueError("strided q needs q_out (a contiguous [rows, Hq, d] buffer)")
        q_out = q
    else:
        require(q_out, torch.float16, "q_out")
        if q_out.shape != q.shape:
            raise ValueError("q_out must have q's shape")
    if (q_norm is None) != (k_norm is None):
        raise ValueError("pass both q_norm and k_norm, or neither")
    for t, n in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        if t is not None:
            require(t, torch.float16, n)
            if tuple(t.shape) != (HEAD_DIM,):
                raise ValueError(f"{n} must be [{HEAD_DIM}]")
    for t, n in ((cos_cache, "cos_cache"), (sin_cache, "sin_cache")):
        require(t, torch.float16, n)
        if t.dim() != 2 or t.shape[1] != HEAD_DIM // 2 or t.shape != cos_cache.shape:
            raise ValueError("cos/sin caches must be [max_positions, head_dim/2]")
    if rows == 0:
        return
    if getattr(infer_state, "ignore_kvcache", False):
        raise ValueError("infer_state.ignore_kvcache is set but the forward has decode rows")
    status = StatusWord(q.device) if validate else None
    _call(cache.device, "nsd_kv8_qk_norm_rope_store", q.data_ptr(), q.stride(0), q_out.data_ptr(), k.data_ptr(),
          k.stride(0), v.data_ptr(), v.stride(0), ptr(q_norm), ptr(k_norm), float(model_config.rms_norm_eps),
          cos_cache.data_ptr(), sin_cache.data_ptr(), cos_cache.shape[0], cache._ref, *table,
          *_decode_rows(cache, infer_state), int(cur_layer), hq, ptr(status.t) if status else None)
    if status is not None:
        status.check("kv8_qk_norm_rope_store")


def kv8_load(k: torch.Tensor, v: torch.Tensor, cache: KV8Cache, block_table: torch.Tensor, seq_ids: torch.Tensor,
             start_locs: torch.Tensor, seq_lens: torch.Tensor, max_len: int, cur_layer: int,
             first: torch.Tensor | None = None, validate: bool = False) -> None:
    """The values of cached tokens as packed fp16 rows, exactly.

    Token ``first[s] + i`` (``first`` None: ``i``) of ``block_table[seq_ids[s]]``, ``i < seq_lens[s] <= max_len``, goes
    to row ``start_locs[s] + i`` of ``k`` and ``v`` [rows, Hkv, d]; other rows are left as they are.  The index tensors
    are int32, one entry a sequence.
    """
    _on(cache, k, v, block_table)
    require(block_table, torch.int32, "block_table")
    if block_table.dim() != 2:
        raise ValueError("block_table must be [rows, max_blocks_per_seq]")
    for t, n in ((k, "k"), (v, "v")):
        require(t, torch.float16, n)
        if t.dim() != 3 or tuple(t.shape[1:]) != (cache.num_kv_heads, HEAD_DIM) or t.shape != k.shape:
            raise ValueError(f"k and v must be [rows, {cache.num_kv_heads}, {HEAD_DIM}], got {tuple(t.shape)}")
    n = seq_ids.shape[0] if seq_ids.dim() == 1 else -1
    for t, name in ((seq_ids, "seq_ids"), (start_locs, "start_locs"), (seq_lens, "seq_lens"), (first, "first")):
        if t is not None:
            _index(cache, t, name, max(n, 0))
            if t.shape[0] != n:
                raise ValueError(f"{name} must be [{n}], one entry a sequence")
    if n == 0 or k.shape[0] == 0:
        return
    status = StatusWord(k.device) if validate else None
    _call(cache.device, "nsd_kv8_load", k.data_ptr(), v.data_ptr(), k.shape[0], cache._ref, block_table.data_ptr(),
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
    streams and in several captured graphs share nothing.
    """
    _on(cache, q, o, lse)
    table = _table(cache, block_table, engine_config)
    rows, hq = infer_state.num_decoding_seqs, int(model_config.num_q_heads)
    require(q, torch.float16, "q")
    require(o, torch.float16, "o")
    if tuple(q.shape) != (rows, hq, HEAD_DIM) or o.numel() != q.numel():
        raise ValueError(f"q must be [{rows}, {hq}, {HEAD_DIM}] and o hold as many elements")
    if lse is not None:
        require(lse, torch.float32, "lse")
        if lse.numel() != rows * hq:
            raise ValueError("lse must hold num_decoding_seqs * num_q_heads floats")
    if int(model_config.num_kv_heads) != cache.num_kv_heads:
        raise ValueError(f"model_config has {model_config.num_kv_heads} kv heads, the cache {cache.num_kv_heads}")
    if rows == 0:
        return
    plan = plan_for(infer_state, model_config, engine_config, block_table)
    if plan.n_rows != rows:
        raise ValueError(f"the forward's attention plan covers {plan.n_rows} rows, q has {rows}")
    size, ws = plan.workspace_bytes, None
    if size:
        # the claim counter of plans with more pieces than workgroup slots starts at zero
        claims = int(plan.host[_lib.PLAN_CLAIMED]) > 0
        ws = (torch.zeros if claims else torch.empty)(size, dtype=torch.uint8, device=q.device)
    status = StatusWord(q.device) if validate else None
    _call(cache.device, "nsd_kv8_paged_attention", q.data_ptr(), o.data_ptr(), ptr(lse), cache._ref, int(cur_layer),
          hq, *table, plan.host_ptr(), plan.dev.data_ptr(), ptr(ws), size, float(infer_state.softmax_scale),
          ptr(status.t) if status else None)
    if status is not None:
        status.check("kv8_paged_attention")
