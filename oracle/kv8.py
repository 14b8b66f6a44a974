"""numpy restatement of the 8-bit paged KV cache, in 64 bits (the oracle for ``nebulasd_amd.kernels.kv8``).

TEST INFRASTRUCTURE ONLY: imported by ``tests/``; never by the product package.  The reference has no counterpart (its
caches are fp16).

How each function is pinned (``tests/test_oracle_kv8.py``):

* ``kv8_exponent``  -- brute force over every power of the range.
* ``kv8_round``     -- brute force over every code (no code is nearer, ties to the even one); torch's own
  ``float8_e4m3fn`` conversion; every result is an fp16 value; a planted mistake (the scale one step down).
* ``kv8_append``    -- one call equals whole blocks rounded at once where no scale changes; re-rounding bounds; slots
  above are ignored.
* ``kv8_attention`` -- ``oracle.paged_attention`` on the values; torch in float64.
* ``kv8_tiles``     -- its inverse, and positions counted by hand.
"""

from __future__ import annotations

import numpy as np

__all__ = ["KV8_RANGES", "KV8_E4M3", "kv8_exponent", "kv8_round", "kv8_append", "kv8_attention", "kv8_tiles",
           "kv8_untile"]

# codes: (largest code, smallest and largest exponent of a scale)
KV8_RANGES = {"e4m3": (448.0, -15, 8), "int8": (127.0, -24, 9)}
# The non-negative E4M3 values, in code order.
KV8_E4M3 = np.array([m * 2.0 ** -9 for m in range(8)]
                    + [(8 + m) * 2.0 ** (p - 3) for p in range(-6, 9) for m in range(8)][:-1])


def kv8_exponent(values, codes):
    """Exponent of the scale for a set of values: the smallest 2^e of the range with m <= top 2^e (the largest e if
    there is none), m the largest finite magnitude."""
    top, lo, hi = KV8_RANGES[codes]
    v = np.asarray(values, np.float64)
    m = np.abs(v[np.isfinite(v)]).max(initial=0.0)
    for e in range(lo, hi):
        if m <= top * 2.0 ** e:
            return e
    return hi


def kv8_round(values, e, codes):
    """(values they are held as, codes as bytes) under the scale 2^e: nearest, ties to the even code; E4M3 values end at
    61440, whole numbers at 127; not finite: NaN (127) in E4M3, 0 in whole numbers.  Bytes are E4M3's or int8's."""
    v = np.asarray(values, np.float64)
    off = ~np.isfinite(v)
    a = np.where(off, 0.0, v) / 2.0 ** e  # exact: a power of two
    if codes == "int8":
        c = np.clip(np.rint(a), -127, 127)
        return c * 2.0 ** e, c.astype(np.int8).view(np.uint8)
    mag = np.minimum(np.abs(a), 61440.0 / 2.0 ** e)
    hi = np.clip(np.searchsorted(KV8_E4M3, mag), 1, len(KV8_E4M3) - 1)
    d_lo, d_hi = mag - KV8_E4M3[hi - 1], KV8_E4M3[hi] - mag
    c = np.where((d_hi < d_lo) | ((d_hi == d_lo) & (hi % 2 == 0)), hi, hi - 1)
    held = np.copysign(KV8_E4M3[c], v) * 2.0 ** e
    byte = (c | np.signbit(v) << 7).astype(np.uint8)
    return np.where(off, np.nan, held), np.where(off, 127, byte).astype(np.uint8)


def kv8_append(held, rows, codes):
    """One tile of a block: ``held`` [16, 128] the values it holds, ``rows`` {slot: row of 128}.  Returns its new values
    (slots above the highest one written, and unwritten, as they were: they hold no token), bytes and exponent; bytes
    of slots that hold no token mean nothing."""
    held = np.array(held, np.float64)
    top = max(rows)
    live = [t for t in range(top) if t not in rows]
    e = kv8_exponent(np.concatenate([held[live].ravel()] + [np.ravel(r) for r in rows.values()]), codes)
    out, byte = held.copy(), np.zeros(held.shape, np.uint8)
    for t in range(top + 1):
        out[t], byte[t] = kv8_round(rows.get(t, held[t]), e, codes)
    return out, byte, e


def kv8_attention(q, k, v, lens, scale):
    """q [rows, Hq, 128], one sequence's k, v [tokens, Hkv, 128] (float64), row r attending lens[r] tokens: (o, lse), and
    bounds of a kernel's errors that rounds weights to fp16 (by half a step: 2^-11, or 2^-25 below fp16's normal
    numbers, of weights whose largest is one at least), a part's and the whole output to fp16, and sums in fp32."""
    rows, hq, d = q.shape
    hkv = k.shape[1]
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    o, lse = np.zeros(q.shape), np.full((rows, hq), -np.inf)
    o_off, lse_off = np.zeros(q.shape), np.zeros((rows, hq))
    for r in range(rows):
        n = lens[r]
        if n < 1:
            continue
        for h in range(hq):
            kk, vv = k[:n, h * hkv // hq], v[:n, h * hkv // hq]
            s = kk @ q[r, h] * scale
            m = s.max()
            p = np.exp(s - m)
            total = p.sum()
            o[r, h], lse[r, h] = p @ vv / total, m + np.log(total)
            # fp32: 128 products summed in any order, times the scale, and exp2 of up to |s - m| / ln 2 (its argument
            # rounded twice, and itself by two steps)
            ds = (130 * 2.0 ** -24 * (np.abs(kk) @ np.abs(q[r, h])) * abs(scale)).max() + (np.abs(s).max() + np.abs(s - m).max()) * 2.0 ** -22
            with np.errstate(invalid="ignore"):
                o_off[r, h] = ((2.0 ** -11 + 2 * ds) * p + 2.0 ** -25) @ np.abs(vv) / total
                o_off[r, h] += 2 * (2.0 ** -11 * (p @ np.abs(vv) / total) + 2.0 ** -25)
            lse_off[r, h] = ds + n * 2.0 ** -24 + 2.0 ** -22 * (1 + abs(lse[r, h]))
    return o, lse, o_off, lse_off


def kv8_tiles(codes_bytes, codes):
    """Bytes [..., 16, 128] of K tiles and of V tiles as the cache holds them: ([..., 2048], [..., 2048])."""
    b = np.asarray(codes_bytes, np.uint8)
    b = b ^ np.uint8(128 if codes == "int8" else 0)  # whole numbers are held as code + 128
    k, v = (np.empty(b.shape[:-2] + (2048,), np.uint8) for _ in range(2))
    for t in range(16):
        for dim in range(128):
            c, half = dim % 64 // 8, dim // 64
            k[..., (16 * c + t) * 16 + 8 * half + dim % 8] = b[..., t, dim]
            i, h, m = dim // 8, dim // 4 % 2, dim % 4
            v[..., (64 * h + 16 * (t // 4) + i) * 16 + 4 * m + t % 4] = b[..., t, dim]
    return k, v


def kv8_untile(tiles, codes, is_v):
    """``kv8_tiles``'s inverse."""
    place = kv8_tiles(np.arange(2048).reshape(16, 128) % 256, "e4m3")[is_v], kv8_tiles(
        np.arange(2048).reshape(16, 128) // 256, "e4m3")[is_v]
    at = place[0].astype(int) + 256 * place[1].astype(int)  # at[byte of the tile] = 128 token + dim
    out = np.empty(np.shape(tiles), np.uint8)
    out[..., at] = tiles
    return out.reshape(np.shape(tiles)[:-1] + (16, 128)) ^ np.uint8(128 if codes == "int8" else 0)
