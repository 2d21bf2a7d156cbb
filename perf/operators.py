"""Cases of the decoder operators: rotary positions, per-head query/key norms with
the rotation, appending to and reading from a paged key/value cache, and attention
over that cache.

Every operator has a plain form in elementary torch operations (``own`` false) and
the framework's call (``own`` true); both take what ``prepare`` gives.

Conventions shared by the cases
  * Rotary table ``[positions, rot/2, 2]`` float32: (cos, sin) of each position and
    frequency, times the amplitude of the scaling; rotated pairs are (i, i + rot/2)
    in the "half" layout and (2i, 2i + 1) in the "interleaved" one.
  * Cache pages ``[pages, kv_heads, page_size, dim]``; a 4-bit cache holds e2m1
    codes, two to a byte (even element in the low nibble), and an e4m3 scale for
    each 16 elements, ``[pages, kv_heads, page_size, dim/16]``.
  * New tokens of all sequences stand one behind the other, ``[tokens, heads, dim]``;
    ``seq_starts`` [batch + 1] says where each sequence's begin and ``seq_lens``
    [batch] how long each sequence is with them. Token i of n new ones has the
    position ``seq_len - n + i``.
"""
import math
import random

import torch

own = False

GAIN = 0.5  # per-cache float32 factor of the 4-bit values


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # The encoder block's own shape (8 x 512 tokens, 12 heads of 64), every position rotated.
        dict(name="rotary_block", op="rotary", dtype="float16", form="bhsd", batch=8, heads=12, seq=512, dim=64, rot=64,
             layout="half", scaling="none", factor=1.0, positions=512),
        # A packed prefill far out in a context stretched 32-fold; half of each head rotated, in pairs.
        dict(name="rotary_long_partial", op="rotary", dtype="bfloat16", form="tokens", batch=1, heads=24, seq=4111, dim=128,
             rot=64, layout="interleaved", scaling="yarn", factor=32.0, positions=131072),
        # Queries and keys of the encoder block's fused projection, normalised and rotated.
        dict(name="qk_norm_block", op="qk_norm", dtype="float16", batch=8, q_heads=12, kv_heads=12, seq=512, dim=64, rot=64,
             layout="half", scaling="none", factor=1.0, positions=512),
        # One new token of each of 48 sequences: a launch with little to do, where latency counts.
        dict(name="qk_norm_decode", op="qk_norm", dtype="bfloat16", batch=1, q_heads=32, kv_heads=8, seq=48, dim=128, rot=128,
             layout="half", scaling="linear", factor=4.0, positions=8192),
        # A decode step of 33 sequences: rotate q and k, write k and v to their pages.
        dict(name="append_decode", op="append", dtype="bfloat16", bits=16, lens=11, batch=33, q_len=1, max_len=4096, q_heads=32,
             kv_heads=8, dim=128, page=16, rot=128, layout="half", scaling="none", factor=1.0),
        # Ragged prompts written to a 4-bit cache and read back as the values they became.
        dict(name="append_prompts_4bit", op="append", dtype="bfloat16", bits=4, lens=12, batch=8, q_len=1024, max_len=2048,
             q_heads=0, kv_heads=8, dim=128, page=64, rot=128, layout="half", scaling="none", factor=1.0),
        # A cached prefix of a few sequences read back as dense keys and values.
        dict(name="read_prefix", op="read", dtype="float16", bits=16, lens=13, batch=5, q_len=300, max_len=700, kv_heads=12,
             dim=64, page=16),
        # Long 4-bit contexts read back whole.
        dict(name="read_long_4bit", op="read", dtype="bfloat16", bits=4, lens=14, batch=2, q_len=65536, max_len=65536,
             kv_heads=8, dim=128, page=32),
        # One sequence, one token, a short context: the smallest decode step.
        dict(name="attn_one", op="attn", dtype="float16", bits=16, lens=15, batch=1, q_len=1, max_len=517, q_heads=12,
             kv_heads=12, dim=64, page=16, window=0),
        # A serving batch of 64 sequences of very different lengths, 4 query heads to a key head.
        dict(name="attn_decode_ragged", op="attn", dtype="bfloat16", bits=16, lens=16, batch=64, q_len=1, max_len=8191,
             q_heads=32, kv_heads=8, dim=128, page=16, window=0),
        # Four very long contexts held in 4 bits.
        dict(name="attn_long_4bit", op="attn", dtype="bfloat16", bits=4, lens=17, batch=4, q_len=1, max_len=131072,
             q_heads=32, kv_heads=8, dim=128, page=64, window=0),
        # Chunks of 1024 prompt tokens that join contexts of up to 16384: the work of products.
        dict(name="attn_chunk", op="attn", dtype="bfloat16", bits=16, lens=18, batch=3, q_len=1024, max_len=16384,
             q_heads=32, kv_heads=8, dim=128, page=32, window=0),
    ]


def _log(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("rotary", "qk_norm", "append", "read", "attn", "attn", "attn"))
    dim = rng.choice((64, 96, 128))
    c = dict(op=op, dtype=rng.choice(("float16", "bfloat16")))
    if op in ("rotary", "qk_norm", "append"):
        c.update(layout=rng.choice(("half", "interleaved")), scaling=rng.choice(("none", "linear", "ntk", "yarn")))
        c.update(factor=1.0 if c["scaling"] == "none" else float(rng.choice((2, 4, 8, 32))))
        c.update(rot=rng.choice((dim, dim, dim // 2)))
    if op == "rotary":
        c.update(form=rng.choice(("bhsd", "tokens")), batch=1, heads=rng.randint(1, 32), dim=dim, positions=_log(rng, 4500, 131072))
        c.update(seq=_log(rng, 1, 4500))
        if c["form"] == "bhsd":
            c.update(batch=rng.randint(1, 8), seq=max(1, c["seq"] // 8))
        return c
    kv = rng.choice((1, 2, 4, 8, 12))
    group = rng.choice((1, 2, 4, 8))
    if op == "qk_norm":
        c.update(batch=rng.randint(1, 4), q_heads=kv * group, kv_heads=kv, dim=dim, positions=_log(rng, 4500, 131072))
        c.update(seq=_log(rng, 1, max(1, min(4500, 100000 // (c["batch"] * kv * (group + 1))))))
        return c
    c.update(bits=rng.choice((16, 16, 4)), lens=rng.randint(1, 1 << 20), kv_heads=kv, dim=dim, page=rng.choice((8, 16, 32, 64, 128)))
    if op == "append":
        c.update(batch=_log(rng, 1, 64), q_heads=kv * group if c["bits"] == 16 else 0)
        c.update(q_len=_log(rng, 1, max(1, 4096 // c["batch"])), max_len=4096)
        return c
    if op == "read":
        c.update(batch=_log(rng, 1, 32))
        c.update(q_len=_log(rng, 1, 131072 // c["batch"]))
        c.update(max_len=c["q_len"] + rng.randint(0, 1000))
        return c
    c.update(q_heads=kv * group, window=rng.choice((0, 0, 0, 1024)))
    step = rng.choice(("one", "one", "few", "chunk"))
    if step == "chunk":
        c.update(batch=rng.randint(1, 3), q_len=_log(rng, 32, 1024))
        c.update(max_len=_log(rng, c["q_len"], max(c["q_len"], 384000 // max(32, c["q_heads"]))))
    else:
        c.update(batch=_log(rng, 1, 64), q_len=1 if step == "one" else rng.randint(2, 8))
        c.update(max_len=_log(rng, 8, 393216 // c["batch"] // max(1, kv * c["q_len"] // 8)))
    return c


def _lens(c):
    """(new tokens, whole length) of each sequence: ragged, fixed by the case."""
    r = random.Random(c["lens"])
    got = []
    for _ in range(c["batch"]):
        n = c["q_len"] if c["q_len"] == 1 or c["op"] == "attn" and c["q_len"] >= 32 else r.randint(max(1, c["q_len"] // 2), c["q_len"])
        got.append((n, r.randint(max(n, c["max_len"] // 8), max(n, c["max_len"]))))
    n, _ = got[0]
    got[0] = (n, max(n, c["max_len"]))
    return got


def work(c):
    size = 2
    d = c["dim"]
    if c["op"] == "rotary":
        n = c["batch"] * c["seq"]
        return {"bytes": 2 * n * c["heads"] * d * size + min(n, c["positions"]) * c["rot"] * 4, "flops": 3 * n * c["heads"] * c["rot"]}
    if c["op"] == "qk_norm":
        n, h = c["batch"] * c["seq"], c["q_heads"] + c["kv_heads"]
        return {"bytes": 2 * n * h * d * size + min(n, c["positions"]) * c["rot"] * 4, "flops": n * h * (3 * c["rot"] + 4 * d)}
    lens = _lens(c)
    t = sum(n for n, _ in lens)
    row = d * size if c["bits"] == 16 else d // 2 + d // 16  # a cached key or value of one head
    if c["op"] == "append":
        moved = t * c["kv_heads"] * 2 * (d * size + row) + 2 * t * c["q_heads"] * d * size + t * c["rot"] * 4
        if c["bits"] == 4:  # read back
            moved += t * c["kv_heads"] * 2 * (d * size + row)
        return {"bytes": moved, "flops": 3 * t * (c["q_heads"] + c["kv_heads"]) * c["rot"]}
    if c["op"] == "read":
        return {"bytes": t * c["kv_heads"] * 2 * (d * size + row), "flops": 0}
    keys = flops = 0
    for n, whole in lens:
        keys += min(whole, c["window"] + n - 1) if c["window"] else whole
        for p in range(whole - n, whole):
            flops += 4 * c["q_heads"] * d * (min(p + 1, c["window"]) if c["window"] else p + 1)
    return {"bytes": keys * c["kv_heads"] * 2 * row + 2 * t * c["q_heads"] * d * size, "flops": flops}


# ---------------------------------------------------------------- the inputs

def _frequencies(rot, scaling, factor):
    """Angles per position, and the amplitude, in 64 bits."""
    i = torch.arange(rot // 2, dtype=torch.float64)
    base = 10000.0
    if scaling == "ntk":  # a larger base, so that the slowest frequency is stretched by the factor
        base *= factor ** (rot / max(rot - 2, 1))
    freq = base ** (-2.0 * i / rot)
    amplitude = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":  # frequencies by parts: fast ones kept, slow ones stretched, a ramp between
        original = 4096.0
        turn = lambda n: rot * math.log(original / (n * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(math.floor(turn(32.0)), 0), min(math.ceil(turn(1.0)), rot - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        freq = freq / factor * ramp + freq * (1 - ramp)
        amplitude = 0.1 * math.log(factor) + 1.0
    return freq, amplitude


def _table(c, positions):
    freq, amplitude = _frequencies(c["rot"], c["scaling"], c["factor"])
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * freq.cuda()
    return torch.stack((angle.cos() * amplitude, angle.sin() * amplitude), -1).float().contiguous()


def _e2m1_codes(x):
    """Codes (0..15) of the nearest e2m1 values, ties to the even one, saturating."""
    a = x.abs().clamp(max=6.0)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = torch.round(a / step) * step
    low = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4))  # 0 .5 1 1.5 2 3 4 6 -> 0..7
    return low.to(torch.uint8) | (torch.signbit(x).to(torch.uint8) << 3)


def _quantise(x, gain):
    """float32 [..., dim] -> (codes [..., dim], e4m3 scales [..., dim/16])."""
    y = (x / gain).unflatten(-1, (-1, 16))
    s = (y.abs().amax(-1) / 6.0).clamp(max=448.0).to(torch.float8_e4m3fn)
    s32 = s.float()[..., None]
    return _e2m1_codes(torch.where(s32 > 0, y / s32, torch.zeros_like(y))).flatten(-2), s


def _values(codes, scales, gain):
    """What codes [..., dim] and e4m3 scales [..., dim/16] stand for, in float32."""
    mags = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    return (mags[codes.long()].unflatten(-1, (-1, 16)) * scales.float()[..., None]).flatten(-2) * gain


def _pack(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _unpack(packed):
    return torch.stack((packed & 15, packed >> 4), -1).flatten(-2)


def prepare(c, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dtype = getattr(torch, c["dtype"])
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=dtype)  # noqa: E731
    s = dict(c=c, gain=GAIN if c.get("bits") == 4 else 1.0)
    if c["op"] in ("rotary", "qk_norm"):
        n = c["seq"]
        s["table"] = _table(c, c["positions"])
        first = torch.randint(0, max(1, c["positions"] - n + 1), (c["batch"], 1), generator=g, device="cuda")
        s["pos"] = (first + torch.arange(n, device="cuda")).contiguous()
        if c["op"] == "rotary":
            if c["form"] == "tokens":
                s["x"], s["pos"] = randn(n, c["heads"], c["dim"]), s["pos"][0]
            else:
                s["x"] = randn(c["batch"], c["heads"], n, c["dim"])
            return s
        # Views of a fused projection [batch, seq, (q + 2 kv) heads, dim], as the attention takes them.
        qkv = randn(c["batch"], n, c["q_heads"] + 2 * c["kv_heads"], c["dim"])
        s["q"] = qkv[:, :, :c["q_heads"]].transpose(1, 2)
        s["k"] = qkv[:, :, c["q_heads"]:c["q_heads"] + c["kv_heads"]].transpose(1, 2)
        s["q_weight"] = (1 + 0.2 * randn(c["dim"])).to(dtype)
        s["k_weight"] = (1 + 0.2 * randn(c["dim"])).to(dtype)
        return s
    lens = _lens(c)
    heads, d, page = c["kv_heads"], c["dim"], c["page"]
    need = [-(-whole // page) for _, whole in lens]
    pages, wide = sum(need) + 3, max(need)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    at, rows = 0, []
    for n in need:  # entries behind a sequence's last page are never looked at; they hold a page that is none
        rows.append(torch.nn.functional.pad(order[at:at + n], (0, wide - n), value=-1))
        at += n
    s["page_table"] = torch.stack(rows).contiguous()
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    s["tokens"] = starts[-1]
    s["seq_starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["seq_lens"] = torch.tensor([whole for _, whole in lens], dtype=torch.int32, device="cuda")
    s["max_q"], s["max_len"] = max(n for n, _ in lens), max(whole for _, whole in lens)
    for name in ("k", "v"):
        if c["bits"] == 16:
            s[name + "_pages"], s[name + "_scales"] = randn(pages, heads, page, d), None
        else:
            codes = torch.empty(pages, heads, page, d // 2, dtype=torch.uint8, device="cuda")
            scales = torch.empty(pages, heads, page, d // 16, dtype=torch.float8_e4m3fn, device="cuda")
            for a in range(0, pages, 4096):
                q, e = _quantise(randn(min(4096, pages - a), heads, page, d).float(), GAIN)
                codes[a:a + 4096], scales[a:a + 4096] = _pack(q), e
            s[name + "_pages"], s[name + "_scales"] = codes, scales
    if c["op"] == "append":
        qkv = randn(s["tokens"], c["q_heads"] + 2 * heads, d)
        s["q"] = qkv[:, :c["q_heads"]] if c["q_heads"] else None
        s["k"], s["v"] = qkv[:, c["q_heads"]:c["q_heads"] + heads], qkv[:, c["q_heads"] + heads:]
        s["table"] = _table(c, c["max_len"])
    elif c["op"] == "attn":
        s["q"] = randn(s["tokens"], c["q_heads"], d)
    if own:  # the handle that a program keeps beside its cache
        from lunara_b200.runtime import ops
        s["cache"] = ops.PagedKVCache(s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"], k_gain=s["gain"], v_gain=s["gain"])
    return s


# ------------------------------------------------------------ the plain forms

def _rotate(x, table, pos, layout):
    """x [..., heads, tokens or 1, dim] in float32 times the rotation at `pos`, whose shape x's leading ones broadcast with."""
    cs = table[pos]
    cos, sin = cs[..., 0], cs[..., 1]
    rot = 2 * cos.shape[-1]
    if layout == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., rot:]), -1)
    a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    return torch.cat((torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2), x[..., rot:]), -1)


def _norm(x, weight, eps):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight.float()


def _slots(s):
    """(sequence, position) of each new token."""
    starts, lens = s["seq_starts"].long(), s["seq_lens"].long()
    token = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(starts, token, right=True) - 1
    return seq, lens[seq] - (starts[seq + 1] - token)


def _picked(scales, *index):
    return scales.view(torch.uint8)[index].view(torch.float8_e4m3fn)


def _cached(s, name, index):
    """Pages picked by `index` as float32 values [..., heads, page, dim]."""
    p = s[name + "_pages"][index]
    return p.float() if s["c"]["bits"] == 16 else _values(_unpack(p), _picked(s[name + "_scales"], index), s["gain"])


def _plain_append(s):
    c = s["c"]
    seq, pos = _slots(s)
    page = s["page_table"][seq, pos // c["page"]].long()
    slot = pos % c["page"]
    k = _rotate(s["k"].float(), s["table"], pos[:, None], c["layout"])
    if c["bits"] == 16:
        s["k_pages"][page, :, slot] = k.to(s["k"].dtype)
        s["v_pages"][page, :, slot] = s["v"]
        out = {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        if s["q"] is not None:
            out["q"] = _rotate(s["q"].float(), s["table"], pos[:, None], c["layout"]).to(s["q"].dtype)
        return out
    out = {}
    for name, x in (("k", k), ("v", s["v"].float())):
        codes, scales = _quantise(x, s["gain"])
        s[name + "_pages"][page, :, slot] = _pack(codes)
        s[name + "_scales"].view(torch.uint8)[page, :, slot] = scales.view(torch.uint8)
        out[name] = _values(codes, scales, s["gain"]).to(s["k"].dtype)
    return out


def _plain_read(s):
    c = s["c"]
    seq, pos = _slots(s)
    page = s["page_table"][seq, pos // c["page"]].long()
    out = {}
    for name in ("k", "v"):
        p = s[name + "_pages"][page, :, pos % c["page"]]
        if c["bits"] == 4:
            e = _picked(s[name + "_scales"], page, slice(None), pos % c["page"])
            p = _values(_unpack(p), e, s["gain"]).to(getattr(torch, c["dtype"]))
        out[name] = p
    return out


def _plain_attention(s):
    c = s["c"]
    b, hk, d = c["batch"], c["kv_heads"], c["dim"]
    starts, lens = s["seq_starts"].long(), s["seq_lens"].long()
    count = starts[1:] - starts[:-1]
    index = s["page_table"].clamp(min=0).long()
    k, v = (_cached(s, n, index).transpose(1, 2).flatten(2, 3)[:, :, :s["max_len"]] for n in ("k", "v"))  # [b, hk, len, d]
    i = torch.arange(s["max_q"], device="cuda")
    row = (starts[:-1, None] + i).clamp(max=s["tokens"] - 1)  # [b, max_q]
    q = s["q"][row].float().unflatten(2, (hk, -1)).permute(0, 2, 3, 1, 4)  # [b, hk, group, max_q, d]
    score = (q.flatten(2, 3) @ k.transpose(2, 3)).unflatten(2, (-1, s["max_q"])) / math.sqrt(d)
    pos = (lens - count)[:, None] + i  # [b, max_q]
    key = torch.arange(s["max_len"], device="cuda")
    keep = (key <= pos[..., None]) & (key < lens[:, None, None])
    if c["window"]:
        keep &= key > pos[..., None] - c["window"]
    keep = keep[:, None, None]
    score.masked_fill_(~keep, float("-inf"))
    top = score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ v).unflatten(2, (-1, s["max_q"])) / total.clamp(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)  # [b, max_q, heads, d]
    seq, at = _slots(s)
    return o[seq, at - (lens - count)[seq]].to(s["q"].dtype)


def run(s):
    c = s["c"]
    op = c["op"]
    if own:
        from lunara_b200.runtime import ops
        if op == "rotary":
            return ops.rotary(s["x"], s["pos"], s["table"], layout=c["layout"])
        if op == "qk_norm":
            return ops.qk_norm_rotary(s["q"], s["k"], s["pos"], s["table"], q_weight=s["q_weight"], k_weight=s["k_weight"],
                                      eps=1e-6, layout=c["layout"])
        where = (s["cache"], s["page_table"], s["seq_starts"], s["seq_lens"])
        if op == "append":
            q = ops.kv_append(s["k"], s["v"], *where, table=s["table"], layout=c["layout"], Q=s["q"])
            if c["bits"] == 4:
                k, v = ops.kv_read(*where, tokens=s["tokens"], dtype=s["k"].dtype)
                return {"k": k, "v": v}
            out = {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}
            return out if q is None else {**out, "q": q}
        if op == "read":
            k, v = ops.kv_read(*where, tokens=s["tokens"], dtype=getattr(torch, c["dtype"]))
            return {"k": k, "v": v}
        return ops.paged_attention(s["q"], *where, window=c["window"], max_q_len=s["max_q"])
    if op == "rotary":
        pos = s["pos"][:, None] if c["form"] == "tokens" else s["pos"][:, None, :]
        return _rotate(s["x"].float(), s["table"], pos, c["layout"]).to(s["x"].dtype)
    if op == "qk_norm":
        pos = s["pos"][:, None, :]
        return tuple(_rotate(_norm(s[n].float(), s[n + "_weight"], 1e-6), s["table"], pos, c["layout"]).to(s[n].dtype) for n in ("q", "k"))
    return {"append": _plain_append, "read": _plain_read, "attn": _plain_attention}[op](s)


# ------------------------------------------------------- the definition in 64 bits

def _turned(x, pos, c):
    """Each pair as a complex number times the unit vector of its angle, in 64 bits; pos [tokens], x [tokens, heads, dim]."""
    freq, amplitude = _frequencies(c["rot"], c["scaling"], c["factor"])
    angle = pos.double()[:, None] * freq.to(pos.device)
    unit = torch.polar(torch.full_like(angle, amplitude), angle)[:, None]
    out, half = x.clone(), c["rot"] // 2
    first, second = (slice(0, half), slice(half, 2 * half)) if c["layout"] == "half" else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * unit
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _sequence(s, name, b, length):
    """Keys or values of one sequence's first `length` positions in 64 bits, [length, heads, dim]."""
    page = s["c"]["page"]
    ids = s["page_table"][b, :-(-length // page)].long()
    x = s[name + "_pages"][ids]
    if s["c"]["bits"] == 4:
        mags = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
        nib = torch.stack((x % 16, x // 16), -1).flatten(-2).long()
        x = mags[nib % 8] * (1 - 2 * (nib // 8)) * _picked(s[name + "_scales"], ids).double().repeat_interleave(16, -1) * s["gain"]
    return x.double().transpose(1, 2).reshape(-1, x.shape[1], x.shape[-1])[:length]


def exact(c, seed):
    if c["op"] == "append" and c["bits"] == 4:
        return None  # what a 4-bit code stands for has no value in 64 bits
    s = prepare(c, seed)
    if c["op"] == "rotary":
        if c["form"] == "tokens":
            return _turned(s["x"].double(), s["pos"], c)
        return torch.stack([_turned(x.double().transpose(0, 1), p, c).transpose(0, 1) for x, p in zip(s["x"], s["pos"])])
    if c["op"] == "qk_norm":
        out = []
        for n in ("q", "k"):
            x = s[n].double()
            x = x / (x.pow(2).sum(-1, keepdim=True) / c["dim"] + 1e-6).sqrt() * s[n + "_weight"].double()
            out.append(torch.stack([_turned(y.transpose(0, 1), p, c).transpose(0, 1) for y, p in zip(x, s["pos"])]))
        return tuple(out)
    lens = _lens(c)
    if c["op"] == "append":
        out = {n + "_pages": s[n + "_pages"].double() for n in ("k", "v")}
        qs, at = [], 0
        for b, (n, whole) in enumerate(lens):
            pos = torch.arange(whole - n, whole, device="cuda")
            ids = s["page_table"][b].long()[pos // c["page"]]
            out["k_pages"][ids, :, pos % c["page"]] = _turned(s["k"][at:at + n].double(), pos, c)
            out["v_pages"][ids, :, pos % c["page"]] = s["v"][at:at + n].double()
            if s["q"] is not None:
                qs.append(_turned(s["q"][at:at + n].double(), pos, c))
            at += n
        return {**out, "q": torch.cat(qs)} if qs else out
    if c["op"] == "read":
        return {n: torch.cat([_sequence(s, n, b, whole)[whole - m:] for b, (m, whole) in enumerate(lens)]) for n in ("k", "v")}
    outs, at = [], 0
    for b, (n, whole) in enumerate(lens):
        k, v = _sequence(s, "k", b, whole), _sequence(s, "v", b, whole)
        back = torch.arange(whole - n, whole, device="cuda")[:, None] - torch.arange(whole, device="cuda")  # how far back each key lies
        hidden = (back < 0) | (back >= c["window"]) if c["window"] else back < 0
        q = s["q"][at:at + n].double()
        o = torch.empty_like(q)
        for h in range(c["q_heads"]):
            kh = h // (c["q_heads"] // c["kv_heads"])
            w = torch.softmax((q[:, h] @ k[:, kh].T * c["dim"] ** -0.5).masked_fill(hidden, float("-inf")), -1)
            o[:, h] = w @ v[:, kh]
        outs.append(o)
        at += n
    return torch.cat(outs)
