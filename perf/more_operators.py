"""A paged KV cache held in 8 bits: written, read back and attended, as timed cases.

A block of 16 tokens of one layer and kv head holds, for K and for V, 16 x 128 codes of 8 bits and one power
of two 2^e; a value is code * 2^e.  The codes are E4M3 (e in [-15, 8]) or whole numbers (-127 .. 127, e in
[-24, 9]).  ``kind`` says what a case calls:

* ``write``      the K and V rows of whole prompts into the cache, and the values read back;
* ``prologue``   decode or verify rows: QK-norm, RoPE, the new K and V into blocks that hold earlier tokens;
                 the rotated q, and the values of every block written;
* ``read``       the values of cached sequences, as packed fp16 rows;
* ``attention``  decode or verify rows over the cache.

Scale of a block: the smallest 2^e of the range that leaves its largest magnitude no more than 448 (E4M3) or
127 (whole numbers).  A value rounds to the nearest code, ties to the even one; E4M3 values end at 61440, so
that every value of a cache is an fp16 value.  A row at position p goes to slot p % 16 of its block: the
tokens below it stay, and are cut again where the block's scale changes; slots above it hold no token.
"""

import math
import random

import torch

own = False

DEV = "cuda"
D = 128
BS = 16
EPS = 1e-6
THETA = 1000000.0
LAYERS, LAYER = 2, 1  # the caches' layers, and the one that a call works on
MOST_CODES = 160000 * 8  # tokens x kv heads of a case


def listed():
    return [
        # A chunk of the speculative loop's prompts, as they enter the target's cache.
        dict(name="write_16_prompts_e4m3", kind="write", codes="e4m3",
             batch=16, lo=128, hi=1024, hq=16, hkv=8, lengths=1),
        # One long prompt.
        dict(name="write_1_prompt_32k_int8", kind="write", codes="int8",
             batch=1, lo=32749, hi=32749, hq=32, hkv=8, lengths=2),
        # One request's next token: latency alone.
        dict(name="prologue_1x1_int8", kind="prologue", codes="int8",
             batch=1, q_len=1, lo=900, hi=900, hq=16, hkv=8, lengths=3),
        # The draft's decode batch.
        dict(name="prologue_64x1_e4m3", kind="prologue", codes="e4m3",
             batch=64, q_len=1, lo=512, hi=2048, hq=16, hkv=8, lengths=4),
        # The target's verify batch: rows of a request share a block, or lie on both sides of its end.
        dict(name="prologue_16x5_int8", kind="prologue", codes="int8",
             batch=16, q_len=5, lo=256, hi=4096, hq=32, hkv=8, lengths=5),
        # Cached sequences handed to code that wants fp16 rows.
        dict(name="read_16_e4m3", kind="read", codes="e4m3", batch=16, lo=256, hi=4096, hq=32, hkv=8, lengths=6),
        # One short sequence of odd length.
        dict(name="read_1_int8", kind="read", codes="int8", batch=1, lo=333, hi=333, hq=40, hkv=8, lengths=7),
        # Four short requests: a decode call that is latency alone.
        dict(name="attention_4x1_e4m3", kind="attention", codes="e4m3",
             batch=4, q_len=1, lo=64, hi=256, hq=16, hkv=8, lengths=8),
        # The draft's decode batch.
        dict(name="attention_64x1_int8", kind="attention", codes="int8",
             batch=64, q_len=1, lo=512, hi=2048, hq=16, hkv=8, lengths=9),
        # The target's verify batch.
        dict(name="attention_16x5_e4m3", kind="attention", codes="e4m3",
             batch=16, q_len=5, lo=256, hi=4096, hq=32, hkv=8, lengths=10),
        # Verify rows over contexts of very different lengths.
        dict(name="attention_16x9_e4m3", kind="attention", codes="e4m3",
             batch=16, q_len=9, lo=1024, hi=32768, hq=32, hkv=8, lengths=11),
        # One request with a long context.
        dict(name="attention_1x1_32k_int8", kind="attention", codes="int8",
             batch=1, q_len=1, lo=32768, hi=32768, hq=32, hkv=8, lengths=12),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["write", "prologue", "prologue", "read", "attention", "attention", "attention"])
    hq, hkv = rng.choice([(16, 8), (32, 8), (40, 8), (64, 8), (32, 4), (8, 8)])
    batch = _spread(rng, 1, 64)
    hi = _spread(rng, 1, max(1, min(32768, MOST_CODES // (batch * hkv) - 16)))
    case = dict(kind=kind, codes=rng.choice(["e4m3", "int8"]), batch=batch, lo=_spread(rng, 1, hi), hi=hi, hq=hq,
                hkv=hkv, lengths=rng.randrange(1 << 30))
    if kind in ("prologue", "attention"):
        case["q_len"] = rng.choice([1, 1, 2, 3, 5, 7, 9, 12])
    return case


def _lengths(case):
    """Tokens of each sequence: of a write or a read all of them, else those before the new rows."""
    rng = random.Random(case["lengths"])
    return [_spread(rng, case["lo"], case["hi"]) for _ in range(case["batch"])]


def _written(case):
    """(first token, tokens) of the blocks that a prologue's rows lie in, for each sequence."""
    n = case["q_len"]
    return [(c // BS * BS, c + n - c // BS * BS) for c in _lengths(case)]


# ---------------------------------------------------------------- the format, plain


def _two_to(e):
    """2^e for whole e in fp32, exactly (exp2 and pow may be off by a last place, which moves a tie)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _power(most, codes):
    """Exponent of the block's scale for its largest magnitude (fp32)."""
    top, lo, hi = (448.0, -15, 8) if codes == "e4m3" else (127.0, -24, 9)
    m, p = torch.frexp(most / top)  # rounding of the quotient cannot cross a power of two: top has 3 or 7 bits
    return torch.where(most > 0, p - (m == 0.5).to(p.dtype), lo).clamp(lo, hi)


def _round(v, e, codes):
    """fp32 values to what they are held as, scale 2^e."""
    step = _two_to(e)
    if codes == "int8":
        return torch.round(v / step).clamp(-127, 127) * step
    a = v.clamp(-61440, 61440) / step
    ulp = _two_to(torch.frexp(a).exponent.clamp(min=-5) - 4)  # 3 bits after the leading one, 2^-9 at least
    return torch.round(a / ulp) * ulp * step


def _held(v, codes):
    """fp32 [..., 16, 128]: whole blocks as the values they are held as, and their exponents [...]."""
    e = _power(v.abs().amax((-2, -1)), codes)
    return _round(v, e[..., None, None], codes), e


# ---------------------------------------------------------------- inputs


def _rows(g, *shape):
    """K or V rows of a trained model: channels of different size, a few far larger."""
    x = torch.randn(*shape, device=DEV, generator=g)
    size = 0.25 + torch.rand(shape[-2:], device=DEV, generator=g)
    return x.mul_(size * torch.where(torch.rand(shape[-2:], device=DEV, generator=g) < 1 / 64, 12.0, 1.0))


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    hq, hkv = case["hq"], case["hkv"]
    lens, batch, codes = _lengths(case), case["batch"], case["codes"]
    n = case.get("q_len", 0)
    per_row = (max(lens) + n + BS - 1) // BS
    need = batch * per_row + 1
    order = torch.randperm(need, device=DEV, generator=g).to(torch.int32)
    s = {"case": case, "table": order[: batch * per_row].view(batch, per_row).contiguous()}
    s["lens"] = torch.tensor(lens, device=DEV, dtype=torch.int32)
    if case["kind"] == "write":
        # nothing in the cache yet
        s["k"], s["v"] = _rows(g, sum(lens), hkv, D).half(), _rows(g, sum(lens), hkv, D).half()
        s["k_held"] = s["v_held"] = torch.zeros(need, LAYERS, hkv, BS, D, device=DEV, dtype=torch.float16)
        s["k_power"] = s["v_power"] = torch.zeros(need, LAYERS, hkv, device=DEV, dtype=torch.int32)
    else:
        for x in "kv":
            held, e = [], []
            for part in range(0, need, 1024):
                rows = _rows(g, min(1024, need - part), LAYERS, hkv, BS, 1, D).squeeze(-2).half().float()
                h, p = _held(rows, codes)
                held.append(h.half())
                e.append(p.int())
            s[x + "_held"], s[x + "_power"] = torch.cat(held), torch.cat(e)
    if case["kind"] == "attention":
        s["q"] = torch.randn(batch * n, hq, D, device=DEV, generator=g).half()
        s["scale"] = D ** -0.5
        s["o"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(batch * n, hq, device=DEV)
    if case["kind"] == "prologue":
        # the fused q/k/v projection's rows
        qkv = torch.randn(batch * n, hq + 2 * hkv, D, device=DEV, generator=g)
        s["qkv"] = qkv.mul_(0.5 + 2 * torch.rand(hq + 2 * hkv, D, device=DEV, generator=g)).half()
        s["q_norm"], s["k_norm"] = ((1 + 0.3 * torch.randn(D, device=DEV, generator=g)).half() for _ in range(2))
        angle = torch.arange(per_row * BS, device=DEV).double()[:, None] * THETA ** (
            -torch.arange(0, D, 2, device=DEV).double() / D)
        s["cos"], s["sin"] = angle.cos().half(), angle.sin().half()
        s["q_out"] = torch.empty(batch * n, hq, D, device=DEV, dtype=torch.float16)
    if case["kind"] != "attention":
        parts = _written(case) if case["kind"] == "prologue" else [(0, m) for m in lens]
        starts = [sum(m for _, m in parts[:i]) for i in range(batch + 1)]
        s["first"], s["count"] = (torch.tensor(c, device=DEV, dtype=torch.int32) for c in zip(*parts))
        s["starts"] = torch.tensor(starts[:-1], device=DEV, dtype=torch.int32)
        s["longest"] = max(m for _, m in parts)
        s["k_out"], s["v_out"] = (torch.empty(starts[-1], hkv, D, device=DEV, dtype=torch.float16) for _ in range(2))
    if own:
        _own_state(s, lens)
    return s


def _own_state(s, lens):
    """The cache, and the forward's metadata (its plan among it), which all layers of a forward share."""
    from nebulasd_amd.config import EngineConfig, ModelConfig
    from nebulasd_amd.infer_state import build_infer_state
    from nebulasd_amd.kernels import KV8Cache
    case = s["case"]
    hq, hkv = case["hq"], case["hkv"]
    n = case.get("q_len", 0)
    s["mc"] = ModelConfig(dict(model_type="qwen3", num_hidden_layers=LAYERS, num_attention_heads=hq,
                               num_key_value_heads=hkv, hidden_size=hq * D, head_dim=D, vocab_size=151936,
                               max_position_embeddings=40960, intermediate_size=4 * hq * D, rope_theta=THETA,
                               rms_norm_eps=EPS))
    s["ec"] = EngineConfig(block_size=BS, max_blocks_per_seq=s["table"].shape[1])
    s["seq_ids"] = torch.arange(case["batch"], device=DEV, dtype=torch.int32)
    codes = [(s[x + "_held"].float() * _two_to(-s[x + "_power"])[..., None, None]).to(
        torch.float8_e4m3fn if case["codes"] == "e4m3" else torch.int8) for x in "kv"]
    powers = [(s[x + "_power"] + 127).to(torch.uint8) for x in "kv"]
    s["cache"] = KV8Cache.pack(*codes, *powers)
    tables = s.get("cos", s["table"].new_zeros(s["table"].shape[1] * BS, D // 2).half())
    if case["kind"] in ("write", "read"):
        s["state"] = build_infer_state(list(range(case["batch"])), [], lens, s["mc"], tables, tables, DEV)
    else:
        ids = [r for r in range(case["batch"]) for _ in range(n)]
        ends = [c + i + 1 for c in lens for i in range(n)]
        s["state"] = build_infer_state(ids, ends, [], s["mc"], tables, tables, DEV)


# ---------------------------------------------------------------- one pass


def run(s):
    kind = s["case"]["kind"]
    if own:
        from nebulasd_amd import kernels
        where = (s["cache"], s["table"])
        if kind == "attention":
            kernels.kv8_paged_attention(s["q"], *where, s["mc"], s["ec"], s["state"], LAYER, s["o"], s["lse"])
            return s["o"], s["lse"]
        out = {}
        if kind == "write":
            kernels.kv8_store(s["k"], s["v"], *where, s["mc"], s["ec"], s["state"], LAYER)
        if kind == "prologue":
            hq, hkv = s["case"]["hq"], s["case"]["hkv"]
            q, k, v = s["qkv"].split((hq, hkv, hkv), 1)
            kernels.kv8_qk_norm_rope_store(q, k, v, *where, s["q_norm"], s["k_norm"], s["mc"], s["ec"], s["state"],
                                           LAYER, s["cos"], s["sin"], q_out=s["q_out"])
            out["q"] = s["q_out"]
        kernels.kv8_load(s["k_out"], s["v_out"], *where, s["seq_ids"], s["starts"], s["count"], s["longest"], LAYER,
                         first=s["first"] if kind == "prologue" else None)
        return {**out, "k": s["k_out"], "v": s["v_out"]}
    return {"write": _write, "prologue": _prologue, "read": _read, "attention": _attention}[kind](s)


def _pages(s, x):
    """The values of every sequence's blocks: fp32 [batch, blocks, heads, 16, 128]."""
    return s[x + "_held"][s["table"].long(), LAYER].float()


def _tokens(pages):
    """[batch, blocks, heads, 16, 128] -> [batch, tokens, heads, 128]."""
    return pages.transpose(2, 3).flatten(1, 2)


def _packed(s, values, first=None):
    """Rows of values [batch, tokens, heads, 128]: s["count"] of each sequence from `first` (fp16)."""
    at = torch.arange(s["longest"], device=DEV)
    use = at < s["count"][:, None]
    seq = torch.arange(len(use), device=DEV)[:, None].expand_as(use)[use]
    tok = (at + first[:, None] if first is not None else at.expand_as(use))[use]
    return values[seq, tok].half()


def _write(s):
    out, codes = {}, s["case"]["codes"]
    batch, blocks = s["table"].shape
    at = torch.arange(blocks * BS, device=DEV)
    use = at < s["count"][:, None]
    row = (s["starts"][:, None] + at).clamp(max=len(s["k"]) - 1)
    for x in "kv":
        rows = s[x].float()[row] * use[..., None, None]  # past the prompt's end: no token
        pages = rows.view(batch, blocks, BS, -1, D).transpose(2, 3)
        out[x] = _packed(s, _tokens(_held(pages, codes)[0]))
    return out


def _read(s):
    return {x: _packed(s, _tokens(_pages(s, x))) for x in "kv"}


def _prologue(s):
    case = s["case"]
    hq, hkv = case["hq"], case["hkv"]
    n, batch = case["q_len"], case["batch"]
    x, v = s["qkv"].float().split((hq + hkv, hkv), 1)
    # the normalised and the rotated row are fp16 rows, as each of the two operators by itself leaves them
    w = torch.cat((s["q_norm"].float().expand(hq, D), s["k_norm"].float().expand(hkv, D)))
    x = (x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w).half().float()
    ends = s["lens"][:, None] + torch.arange(n, device=DEV)  # positions of the new rows
    c, sn = (t[ends.flatten().long()].float()[:, None] for t in (s["cos"], s["sin"]))
    a, b = x.chunk(2, -1)
    x = torch.cat((a * c - b * sn, a * sn + b * c), -1).half()
    out = {"q": x[:, :hq]}
    # the blocks that are written: at most (14 + n) / 16 + 1 of each sequence
    span = (BS - 2 + n) // BS + 1
    first = s["first"].long()
    at = torch.arange(span * BS, device=DEV)
    place = first[:, None] + at  # positions
    block = (first[:, None] // BS + torch.arange(span, device=DEV)).clamp(max=s["table"].shape[1] - 1)
    new = place - s["lens"][:, None]  # which of the new rows a position is
    is_new, is_old = (new >= 0) & (new < n), new < 0
    row = new.clamp(0, n - 1) + n * torch.arange(batch, device=DEV)[:, None]
    for name, rows in (("k", x[:, hq:].float()), ("v", v)):
        old = _tokens(s[name + "_held"][s["table"].gather(1, block).long(), LAYER].float())
        values = torch.where(is_new[..., None, None], rows[row], old * is_old[..., None, None])
        pages = values.view(batch, span, BS, hkv, D).transpose(2, 3)
        out[name] = _packed(s, _tokens(_held(pages, case["codes"])[0]))
    return out


def _attention(s):
    case = s["case"]
    hq, hkv = case["hq"], case["hkv"]
    n, batch = case["q_len"], case["batch"]
    k, v = (_pages(s, x).transpose(1, 2).flatten(2, 3) for x in "kv")  # [batch, heads, tokens, 128]
    q = s["q"].float().view(batch, n, hkv, hq // hkv, D).permute(0, 2, 4, 1, 3).reshape(batch, hkv, D, -1)
    score = (k @ q) * s["scale"]  # [batch, heads, tokens, rows x group]
    end = s["lens"][:, None] + torch.arange(n, device=DEV) + 1
    off = torch.arange(k.shape[2], device=DEV)[:, None] >= end.repeat_interleave(hq // hkv, 1)[:, None]
    score.masked_fill_(off[:, None], -math.inf)
    most = score.amax(2, keepdim=True)
    p = torch.exp(score - most)
    total = p.sum(2, keepdim=True)
    o = (p / total).transpose(2, 3).contiguous() @ v
    o = o.view(batch, hkv, n, hq // hkv, D).transpose(1, 2).reshape(batch * n, hq, D)
    lse = (most + torch.log(total)).view(batch, hkv, n, hq // hkv).transpose(1, 2).reshape(batch * n, hq)
    return o.half(), lse


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    hq, hkv = case["hq"], case["hkv"]
    lens, kind = _lengths(case), case["kind"]
    token = 2 * hkv * D  # codes of a token's K and V
    scales = 2 * hkv
    if kind == "write":
        t, blocks = sum(lens), sum(-(-m // BS) for m in lens)
        # rows in, codes and scales out; codes and scales in, rows out
        return {"bytes": t * token * 2 + 2 * (t * token + blocks * scales) + t * token * 2, "flops": 5 * t * token}
    if kind == "read":
        t, blocks = sum(lens), sum(-(-m // BS) for m in lens)
        return {"bytes": t * token + blocks * scales + t * token * 2, "flops": t * token}
    n = case["q_len"]
    rows = n * len(lens)
    if kind == "prologue":
        out = sum(m for _, m in _written(case))
        blocks = sum((c + n - 1) // BS - c // BS + 1 for c in lens)
        # rows in, q out; the earlier tokens in, the new ones out; the blocks in and their values out
        old = out - rows
        return {"bytes": rows * (hq + 2 * hkv) * D * 2 + rows * hq * D * 2 + (old + rows) * token + 2 * blocks * scales
                + out * token + blocks * scales + out * token * 2, "flops": 10 * rows * (hq + 2 * hkv) * D}
    tokens = sum(c + n for c in lens)
    blocks = sum(-(-(c + n) // BS) for c in lens)
    # codes and scales, q, o, lse
    return {"bytes": tokens * token + blocks * (scales + 4) + 2 * rows * hq * D * 2 + rows * hq * 4,
            "flops": sum(4 * hq * D * (c + i + 1) for c in lens for i in range(n))}


# ---------------------------------------------------------------- the same in 64 bits


_E4M3 = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (p - 3) for p in range(-6, 9) for m in range(8)][:-1]


def _nearest(v, codes):
    """float64 [blocks, values]: each block over its scale, to the nearest code, ties to the even place."""
    lo, hi, values = (-15, 8, _E4M3) if codes == "e4m3" else (-24, 9, range(128))
    values = torch.tensor(list(values), device=DEV, dtype=torch.float64)
    powers = torch.tensor([2.0 ** e for e in range(lo, hi + 1)], device=DEV, dtype=torch.float64)
    most = v.abs().amax(1)
    # the first power with most <= top * power
    power = powers[torch.searchsorted(powers * values[-1], most).clamp(max=hi - lo)][:, None]
    a = (v.abs() / power).contiguous()
    middle = (values[1:] + values[:-1]) / 2
    below, above = torch.searchsorted(middle, a), torch.searchsorted(middle, a, right=True)
    place = torch.where((below != above) & (below % 2 == 1), above, below)  # on a middle: the even one of the two
    return torch.sign(v) * torch.clamp(values[place] * power, max=61440.0 if codes == "e4m3" else math.inf)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    hq, hkv = case["hq"], case["hkv"]
    lens, codes, kind, n = _lengths(case), case["codes"], case["kind"], case.get("q_len", 0)
    out = {}

    def cached(x, seq, tokens):  # [tokens, heads, 128]
        pages = s[x + "_held"][s["table"][seq, : -(-tokens // BS)].long(), LAYER].double()
        return pages.permute(0, 2, 1, 3).reshape(-1, hkv, D)[:tokens]

    def blocks(rows):  # rows of one sequence from a block's start: each block and head by itself
        got = []
        for part in rows.split(BS):
            got.append(_nearest(part.transpose(0, 1).reshape(hkv, -1), codes).view(hkv, -1, D).transpose(0, 1))
        return torch.cat(got)

    if kind == "read":
        return {x: torch.cat([cached(x, i, m) for i, m in enumerate(lens)]) for x in "kv"}
    if kind == "write":
        return {x: torch.cat([blocks(p) for p in s[x].double().split(lens)]) for x in "kv"}
    if kind == "prologue":
        rows = s["qkv"].double()
        place = torch.tensor([c + i for c in lens for i in range(n)], device=DEV)
        turn = torch.complex(s["cos"].double(), s["sin"].double())[place][:, None]
        done = []
        for part, w in ((rows[:, :hq], s["q_norm"]), (rows[:, hq:hq + hkv], s["k_norm"])):
            part = part / torch.sqrt(part.pow(2).sum(-1, keepdim=True) / D + EPS) * w.double()
            part = part.half().double()  # part of the definition: both steps leave fp16 rows
            z = torch.complex(part[..., :D // 2], part[..., D // 2:]) * turn
            done.append(torch.cat((z.real, z.imag), -1).half().double())
        out["q"] = done[0]
        for x, new in (("k", done[1]), ("v", rows[:, hq + hkv:])):
            got = []
            for i, (c, fresh) in enumerate(zip(lens, new.split(n))):
                got.append(blocks(torch.cat((cached(x, i, c)[c // BS * BS:], fresh))))
            out[x] = torch.cat(got)
        return out
    o, lse = [], []
    for i, c in enumerate(lens):
        k, v = (cached(x, i, c + n).transpose(0, 1).contiguous() for x in "kv")  # [heads, tokens, 128]
        q = s["q"][i * n:(i + 1) * n].double().view(n, hkv, hq // hkv, D)
        late = torch.arange(c + n, device=DEV) > c + torch.arange(n, device=DEV)[:, None]  # [n, tokens]
        for j in range(n):
            score = q[j] @ k.transpose(1, 2).contiguous() * s["scale"]  # [heads, group, tokens]
            score = score.masked_fill(late[j], -math.inf)
            lse.append(torch.logsumexp(score, -1).view(hq))
            o.append((torch.softmax(score, -1) @ v).view(hq, D))
    return torch.stack(o), torch.stack(lse)
