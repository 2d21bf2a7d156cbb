"""GPU parity of the decoder operators (rotary positions, query/key norms, paged cache,
paged attention) against their definitions in 64 bits.

Tolerances are sums of what the arithmetic can be off by. h = finfo.eps / 2 is half a step
of the output's type, relative to the value.
  rotary    h |y| for the output and 2^-21 (|a| + |b|) for the fp32 table entries (2^-24),
            products (2^-24) and sum (2^-24) of a pair, with room for amplitudes up to 2.
  norms     h |y| and 2^-19 (|a| + |b|): the sum of squares of a lane's 16 terms and the
            shuffles (<= 21 roundings, halved by the root), rsqrtf (2 ulp), the division,
            two products and the rotation stay below 32 roundings of 2^-24.
  attention h |o| for the output; (hp + 2 d + (n + 8) 2^-24 + 2^-13) sum p |v| for the
            probabilities: hp their 16-bit rounding (0 for fp32 caches), d the score's
            error (dim + 2) 2^-24 scale sum |q||k| (which enters p and the sum), n the
            number of keys summed, 2^-13 the exponential (cubic: 7.5e-5; 2^-18 in fp32,
            which has no cubic).
fp16 results below its normal range are off by half its smallest step, 2^-25. So are fp16
probabilities (fp16 queries, and every product with a 4-bit cache): one below 2^-14 of its
row's largest is off by up to 2^-25 of that, whatever its own size, and the largest is at
least 1 in the sum that divides it; that moves the output by up to 2^-25 sum |v| over the
keys. It shows where the values of the keys that matter are zeros, as 4-bit codes can be.
The rounding of the output is half a step of the computed value, which is off by the other
terms already: they count (1 + h) times.
"""
import pytest
import torch

from oracle import decoder as ref

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
TINY = 2.0 ** -25


def _ops():
    from lunara_b200.runtime import ops
    return ops


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def within(out, want, tol, what):
    out = out.detach().cpu().to(torch.float64)
    assert out.shape == want.shape, what
    assert torch.isfinite(out).all(), f"{what}: not finite"
    over = (out - want).abs() - tol
    assert (over <= 0).all(), f"{what}: off by {(out - want).abs().max():.3e}, {over.max():.3e} over the tolerance"


def cos_sin(table, pos):
    t = table.cpu().to(torch.float64)[pos.cpu().long()]
    return t[..., 0], t[..., 1]


def partner_sum(x, rot, layout):
    """|a| + |b| of each element's pair, |x| behind rot."""
    a = x.abs()
    out = a.clone()
    if layout == "half":
        s = a[..., :rot // 2] + a[..., rot // 2:rot]
        out[..., :rot // 2] = out[..., rot // 2:rot] = s
    else:
        s = a[..., 0:rot:2] + a[..., 1:rot:2]
        out[..., 0:rot:2] = out[..., 1:rot:2] = s
    return out


# ──────────────────────────────────────────────────────────── rotary ──

ROTARY = [  # batch, heads, seq, dim, rot
    (2, 3, 5, 64, 64), (1, 12, 512, 64, 64), (3, 5, 17, 128, 128), (2, 4, 33, 128, 64), (1, 7, 9, 96, 96), (1, 2, 9, 96, 48),
    (1, 1, 1, 64, 32), (2, 2, 7, 80, 80), (2, 3, 4, 72, 18), (1, 3, 5, 10, 2), (1, 2, 3, 256, 256), (1, 2, 2, 576, 64),
    (1, 40, 300, 64, 16),
]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("shape", ROTARY)
def test_rotary(shape, layout, dtype):
    batch, heads, seq, dim, rot = shape
    ops = _ops()
    g = torch.Generator().manual_seed(dim + rot + seq)
    x = torch.randn(batch, heads, seq, dim, generator=g).to(dtype)
    table = ops.rotary_table(2000, rot)
    pos = torch.randint(0, 2000, (batch, seq), generator=g)
    want_cs = [t[:, None] for t in cos_sin(table, pos)]
    want = ref.rotate(x.double(), *want_cs, layout)
    tol = half_step(dtype) * want.abs() + 2.0 ** -21 * partner_sum(x.double(), rot, layout) + TINY
    out = ops.rotary(x.cuda(), pos.cuda(), table, layout=layout)
    within(out, want, tol, "rotary")
    assert torch.equal(ops.rotary(x.cuda(), pos.cuda().int(), table, layout=layout), out)
    y = x.cuda()
    assert ops.rotary(y, pos.cuda(), table, layout=layout, out=y) is y and torch.equal(y, out)
    # A strided view of a fused projection, and shared positions.
    fused = torch.randn(batch, seq, heads + 2, dim, generator=g).to(dtype)
    view = fused.cuda()[:, :, 1:1 + heads].transpose(1, 2)
    shared = torch.arange(100, 100 + seq)
    want = ref.rotate(fused[:, :, 1:1 + heads].transpose(1, 2).double(), *cos_sin(table, shared), layout)
    tol = half_step(dtype) * want.abs() + 2.0 ** -21 * partner_sum(want, rot, layout) * 2 + TINY
    within(ops.rotary(view, shared.cuda(), table, layout=layout), want, tol, "rotary of a view")
    # Packed tokens, from an odd offset (no 16-byte alignment).
    flat = torch.randn(seq * heads * dim + 1, generator=g).to(dtype)
    odd = flat.cuda()[1:].view(seq, heads, dim)
    want = ref.rotate(flat[1:].view(seq, heads, dim).double(), *(t[:, None] for t in cos_sin(table, shared)), layout)
    tol = half_step(dtype) * want.abs() + 2.0 ** -21 * partner_sum(want, rot, layout) * 2 + TINY
    within(ops.rotary(odd, shared.cuda(), table, layout=layout), want, tol, "rotary of tokens")
    assert ops.device_error() == 0


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_inverse_is_its_gradient(layout):
    """Against the formula's transpose, and against differences: <g, R x'> - <g, R x> = <R^T g, x' - x>."""
    ops = _ops()
    g = torch.Generator().manual_seed(5)
    x, dx, up = (torch.randn(2, 3, 11, 64, generator=g) for _ in range(3))
    table = ops.rotary_table(500, 32, scaling={"type": "yarn", "factor": 4.0, "original_positions": 100})
    pos = torch.randint(0, 500, (2, 11), generator=g)
    c, s = (t[:, None] for t in cos_sin(table, pos))
    want = ref.rotate(up.double(), c, -s, layout)
    back = ops.rotary(up.cuda(), pos.cuda(), table, layout=layout, inverse=True)
    within(back, want, half_step(F32) * want.abs() + 2.0 ** -21 * partner_sum(up.double(), 32, layout), "gradient")
    turn = lambda t: ops.rotary(t.cuda(), pos.cuda(), table, layout=layout).cpu().double()  # noqa: E731
    moved = ((turn(x + dx) - turn(x)) * up).sum()
    along = (back.cpu().double() * ((x + dx).double() - x.double())).sum()
    # 4224 terms, each off by at most 2^-20 times its two factors' size.
    assert abs(moved - along) <= 2.0 ** -20 * 4 * (up.abs() * (x.abs() + dx.abs() + 1)).sum()


def test_rotary_position_outside_the_table():
    ops = _ops()
    table = ops.rotary_table(16, 64)
    for dim in (64, 66):   # the vector and the general kernel
        x = torch.randn(1, 2, 4, dim, device="cuda")
        pos = torch.tensor([3, 16, -1, 15], device="cuda")
        out = ops.rotary(x, pos, table)
        assert ops.device_error() == 0x501 and ops.device_error() == 0
        assert (out[:, :, 1:3] == 0).all() and (out[:, :, 0] != 0).any() and (out[:, :, 3] != 0).any()


def test_rotary_empty():
    ops = _ops()
    table = ops.rotary_table(16, 64)
    pos = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert ops.rotary(torch.empty(2, 3, 0, 64, device="cuda"), pos, table).shape == (2, 3, 0, 64)
    assert ops.rotary(torch.empty(0, 3, 64, device="cuda"), pos, table).shape == (0, 3, 64)


# ─────────────────────────────────────────────────────── query/key norms ──

@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("shape", [(2, 12, 12, 40, 64, 64), (1, 8, 2, 33, 128, 128), (1, 3, 1, 5, 96, 48), (2, 2, 2, 3, 72, 24),
                                   (1, 1, 1, 1, 64, 64), (1, 4, 1, 6, 512, 64), (3, 32, 8, 1, 128, 64), (1, 33, 7, 500, 64, 64)])
def test_qk_norm_rotary(shape, layout, dtype):
    batch, hq, hk, seq, dim, rot = shape
    ops = _ops()
    g = torch.Generator().manual_seed(dim * seq)
    qkv = torch.randn(batch, seq, hq + 2 * hk, dim, generator=g).to(dtype)
    w = [(1 + 0.3 * torch.randn(dim, generator=g)).to(dtype) for _ in range(2)]
    table = ops.rotary_table(1000, rot)
    pos = torch.randint(0, 1000, (batch, seq), generator=g)
    c, s = (t[:, None] for t in cos_sin(table, pos))
    dev = qkv.cuda()
    views = [(0, hq), (hq, hk)]
    qv, kv = (dev[:, :, a:a + n].transpose(1, 2) for a, n in views)
    for weights, tab in ((w, table), ([None, None], table), (w, None)):
        got = ops.qk_norm_rotary(qv, kv, pos.cuda(), tab, *(None if x is None else x.cuda() for x in weights), eps=1e-5, layout=layout)
        for out, (a, n), weight in zip(got, views, weights):
            y = ref.rms_norm(qkv[:, :, a:a + n].transpose(1, 2), weight, 1e-5)
            want = y if tab is None else ref.rotate(y, c, s, layout)
            size = y.abs() if tab is None else partner_sum(y, rot, layout)
            within(out, want, half_step(dtype) * want.abs() + 2.0 ** -19 * size + TINY, "qk_norm_rotary")
    same = ops.qk_norm_rotary(qv, kv, pos.cuda(), table, w[0].cuda(), w[1].cuda(), eps=1e-5, layout=layout, out_q=qv, out_k=kv)
    fresh = qkv.cuda()
    again = ops.qk_norm_rotary(*(fresh[:, :, a:a + n].transpose(1, 2) for a, n in views), pos.cuda(), table, w[0].cuda(),
                               w[1].cuda(), eps=1e-5, layout=layout)
    assert all(torch.equal(a, b) for a, b in zip(same, again))
    assert torch.equal(dev[:, :, hq + hk:].cpu(), qkv[:, :, hq + hk:])   # the values beside them are untouched
    assert ops.device_error() == 0


def test_qk_norm_of_zero_rows():
    ops = _ops()
    q = torch.zeros(1, 2, 3, 64, device="cuda", dtype=F16)
    a, b = ops.qk_norm_rotary(q, q.clone(), torch.arange(3, device="cuda"), ops.rotary_table(8, 64))
    assert (a == 0).all() and (b == 0).all()


# ───────────────────────────────────────────────────────── paged cache ──

def cache_of(p, device="cuda", on=None):
    ops = _ops()
    t = {k: v.to(device) for k, v in (on or p.tensors).items()}
    return ops.PagedKVCache(t["k"], t["v"], t.get("k_scales"), t.get("v_scales"), k_gain=p.gain, v_gain=p.gain), t


def where(p):
    return p.page_table.cuda(), p.seq_starts.cuda(), p.seq_lens.cuda()


# Sequences of (new tokens, length): decode steps, prompts, an empty one, padding (shorter than its tokens).
RAGGED = {
    "decode": [(1, 1), (1, 17), (1, 300), (1, 64)],
    "mixed": [(5, 5), (0, 40), (1, 33), (37, 100), (2, 1), (1, 0), (64, 64)],
    "one": [(1, 1)],
}


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("lens,heads,q_heads,dim,rot,page", [
    ("decode", 2, 8, 128, 128, 16), ("mixed", 3, 0, 64, 64, 8), ("mixed", 2, 4, 96, 48, 24), ("mixed", 1, 2, 64, 32, 1),
    ("one", 8, 32, 128, 64, 64), ("mixed", 2, 2, 112, 20, 16), ("mixed", 12, 12, 64, 0, 16),
])
def test_kv_append(lens, heads, q_heads, dim, rot, page, layout, bits, dtype):
    ops = _ops()
    p = ref.Paged(RAGGED[lens], heads, dim, page, dtype, seed=dim + page, bits=bits, gain=0.75 if bits == 4 else 1.0, extra_tokens=3)
    g = torch.Generator().manual_seed(9)
    qkv = torch.randn(p.tokens, q_heads + 2 * heads, dim, generator=g).to(dtype)
    q, k, v = qkv[:, :q_heads], qkv[:, q_heads:q_heads + heads], qkv[:, q_heads + heads:]
    table = ops.rotary_table(512, rot) if rot else None
    cache, t = cache_of(p)
    dev = qkv.cuda()
    out_q = torch.full((p.tokens, q_heads, dim), 7.0, dtype=dtype, device="cuda") if q_heads else None
    got = ops.kv_append(dev[:, q_heads:q_heads + heads], dev[:, q_heads + heads:], cache, *where(p), table=table, layout=layout,
                        Q=dev[:, :q_heads] if q_heads else None, out_q=out_q)
    assert got is out_q
    f32 = table.cpu() if rot else None

    def turned(x, pos, dt):
        if not rot:
            return x.to(dt)
        cs = f32[pos].to(dt)[:, None]
        return ref.rotate(x.to(dt), cs[..., 0], cs[..., 1], layout)

    spread = lambda x: partner_sum(x.double(), rot, layout) if rot else torch.zeros_like(x, dtype=torch.float64)  # noqa: E731
    want_q = torch.full((p.tokens, q_heads, dim), 7.0, dtype=torch.float64)
    tol_q = torch.zeros_like(want_q)
    touched = {n: x.clone() for n, x in p.tensors.items()}
    at = 0
    for b, (n, whole) in enumerate(p.lens):
        pos = torch.arange(whole - n, whole)
        real = pos >= 0
        rows = slice(at, at + n)
        if q_heads:
            want_q[rows] = 0
            want_q[rows][real] = turned(q[rows][real], pos[real], torch.float64)
            tol_q[rows] = half_step(dtype) * want_q[rows].abs() + 2.0 ** -21 * spread(q[rows]) + TINY
        pos = pos[real]
        if len(pos):
            ids, slot = p.page_table[b].long()[pos // page], pos % page
            if bits == 16:
                want = turned(k[rows][real], pos, torch.float64)
                within(t["k"].cpu()[ids, :, slot], want, half_step(dtype) * want.abs() + 2.0 ** -21 * spread(k[rows][real]) + TINY, "keys")
                touched["k"][ids, :, slot] = t["k"].cpu()[ids, :, slot]
                touched["v"][ids, :, slot] = v[rows][real]
            else:
                p.tensors = touched
                p.put("k", b, pos, turned(k[rows][real], pos, torch.float32))
                p.put("v", b, pos, v[rows][real].float())
        at += n
    for name, x in touched.items():   # slots that no token owns keep their bytes
        now = t[name].cpu()
        assert torch.equal(now.view(torch.uint8), x.contiguous().view(torch.uint8)), name
    if q_heads:
        within(out_q, want_q, tol_q, "queries")
        # In place: the same rows, those behind the last sequence untouched.
        here = dev[:, :q_heads]
        before = here[p.owned:].clone()
        ops.kv_append(dev[:, q_heads:q_heads + heads], dev[:, q_heads + heads:], cache, *where(p), table=table, layout=layout, Q=here, out_q=here)
        assert torch.equal(here[:p.owned], out_q[:p.owned]) and torch.equal(here[p.owned:], before)
    assert ops.device_error() == 0


def test_kv_append_4bit_extremes():
    """Scales that saturate, vanish or are not numbers; ties; infinities."""
    ops = _ops()
    rows = torch.zeros(8, 16)
    rows[0] = torch.tensor([6, 5, 3.5, 2.5, 1.75, 1.25, .75, .25, -.25, -.75, -1.25, -1.75, -2.5, -3.5, -5, -6.0])   # every tie
    rows[1, 3] = 60000.0          # beyond 448 * 6
    rows[2] = 1e-4                # a scale that rounds to zero
    rows[3, 5] = float("nan")
    rows[4, 2], rows[4, 9] = float("inf"), -float("inf")
    rows[5] = torch.linspace(-3, 3, 16)
    rows[6, 0] = 0.011            # a subnormal scale
    x = rows.reshape(1, 1, 128).expand(2, 1, 128).contiguous()
    for dtype in (F32, F16, BF16):
        cache = ops.PagedKVCache.allocate(2, 1, 4, 128, dtype="e2m1")
        tab, starts, lens = (torch.tensor(a, dtype=torch.int32, device="cuda") for a in ([[1]], [0, 2], [3]))
        xd = x.to(dtype).cuda()
        ops.kv_append(xd, xd, cache, tab, starts, lens)
        codes, scales = ref.quantise(x.to(dtype).float(), 1.0)
        for pages, sc in ((cache.k_pages, cache.k_scales), (cache.v_pages, cache.v_scales)):
            assert torch.equal(pages[1, 0, 1:3].cpu(), ref.pack(codes)[:, 0])
            assert torch.equal(sc.view(torch.uint8)[1, 0, 1:3].cpu(), scales[:, 0])
            assert (pages[0] == 0).all() and (pages[1, 0, 0] == 0).all()
        k, v = ops.kv_read(cache, tab, starts, lens, tokens=2, dtype=dtype)
        want = ref.values(codes, scales, 1.0)
        assert torch.equal(k.cpu().double().nan_to_num(-1), want.to(dtype).double().nan_to_num(-1)) and torch.equal(k.isnan(), v.isnan())
        assert k[0, 0, 48:64].isnan().all() and not k[0, 0, 64:].isnan().any()


def test_kv_append_4bit_every_scale():
    """Blocks of every e4m3 scale and of the largest magnitudes around its rounding, elements around every code's ties."""
    ops = _ops()
    g = torch.Generator().manual_seed(17)
    scales = torch.arange(1, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    amax = torch.cat([scales * 6 * (1 + k * 2.0 ** -23) for k in (-1, 0, 1)] + [(scales[1:] + scales[:-1]) * 3 * (1 + k * 2.0 ** -23) for k in (-1, 0, 1)])
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]).repeat(2) * torch.tensor([1.0] * 7 + [-1.0] * 7)
    x = torch.zeros(len(amax), 16)
    x[:, 0] = amax
    s = ref.quantise(x, 1.0)[1].view(torch.float8_e4m3fn).float()
    x[:, 1:15] = ties * s * (1 + torch.randint(-2, 3, (len(amax), 14), generator=g) * 2.0 ** -23)
    x[:, 15] = torch.randn(len(amax), generator=g) * amax / 3
    x = torch.nn.functional.pad(x, (0, 0, 0, (-len(x)) % 4)).view(-1, 1, 64)
    n = len(x)
    cache = ops.PagedKVCache.allocate((n + 7) // 8, 1, 8, 64, dtype="e2m1")
    tab = torch.arange((n + 7) // 8, dtype=torch.int32, device="cuda")[None]
    starts, lens = torch.tensor([0, n], dtype=torch.int32, device="cuda"), torch.tensor([n], dtype=torch.int32, device="cuda")
    ops.kv_append(x.cuda(), x.cuda(), cache, tab, starts, lens)
    codes, scale_bytes = ref.quantise(x, 1.0)
    assert torch.equal(cache.k_pages.view(-1, 32)[:n].cpu(), ref.pack(codes)[:, 0])
    assert torch.equal(cache.v_scales.view(torch.uint8).view(-1, 4)[:n].cpu(), scale_bytes[:, 0])


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("heads,dim,page", [(2, 128, 16), (3, 64, 1), (1, 96, 24), (2, 48, 7), (2, 1024, 4)])
def test_kv_read(heads, dim, page, bits, dtype):
    ops = _ops()
    p = ref.Paged(RAGGED["mixed"], heads, dim, page, dtype, seed=3, bits=bits, gain=1.5 if bits == 4 else 1.0)
    cache, _ = cache_of(p)
    got = ops.kv_read(cache, *where(p), tokens=p.tokens, dtype=dtype)
    for i, out in enumerate(got):
        want = torch.zeros(p.tokens, heads, dim, dtype=torch.float64)
        at = 0
        for b, (n, whole) in enumerate(p.lens):
            real = min(n, whole)
            want[at + n - real:at + n] = p.seqs[b][i][whole - real:whole]
            at += n
        # fp32(scale * gain) and the product round once each, then the output.
        within(out, want, (half_step(dtype) + (2.0 ** -22 if bits == 4 else 0)) * want.abs(), "read")
        if bits == 16:
            assert torch.equal(out.cpu(), want.to(dtype))
    assert ops.device_error() == 0


def test_bad_pages_and_lengths_are_recorded():
    ops = _ops()
    for bits in (16, 4):
        p = ref.Paged([(2, 20), (1, 9), (1, 40)], 2, 64, 8, F16, seed=4, bits=bits)
        cache, t = cache_of(p)
        before = {n: x.clone() for n, x in t.items()}
        k = torch.randn(4, 2, 64, device="cuda", dtype=F16)
        tab, starts, lens = where(p)
        tab[0, 2], tab[1, 1] = 10 ** 6, -5             # the pages of positions 18, 19 and 8
        assert ops.kv_append(k, k, cache, tab, starts, lens) is None
        assert ops.device_error() == 0x502
        lens[2] = 41                                    # position 40 is behind the page table
        ops.kv_append(k[3:], k[3:], cache, tab[2:], torch.tensor([0, 1], dtype=torch.int32, device="cuda"), lens[2:])
        assert ops.device_error() == 0x503
        changed = {n: (x.view(torch.uint8) != before[n].view(torch.uint8)).flatten(1).any(1).cpu() for n, x in t.items()}
        page = int(p.page_table[2, 4])                  # only position 39 was written
        assert all(int(c.sum()) == 1 and c[page] for c in changed.values())
        out, _ = ops.kv_read(cache, tab, starts, torch.tensor([20, 9, 41], dtype=torch.int32, device="cuda"), tokens=4, dtype=F16)
        assert ops.device_error() in (0x502, 0x503)
        assert (out == 0).all()


# ──────────────────────────────────────────────────── paged attention ──

def check_attention(p, q_heads, window=0, scale=None, max_q_len=None, q=None, what=""):
    ops = _ops()
    q = p.queries(q_heads) if q is None else q
    cache, _ = cache_of(p)
    out = torch.full(q.shape, 7.0, dtype=p.dtype, device="cuda")
    got = ops.paged_attention(q.cuda(), cache, *where(p), scale=scale, window=window, max_q_len=max_q_len, out=out)
    assert got is out
    scale = p.dim ** -0.5 if scale is None else scale
    want = torch.full(q.shape, 7.0, dtype=torch.float64)
    tol = torch.zeros_like(want)
    at = 0
    hp = 0.0 if p.dtype == F32 else half_step(p.dtype)
    ex = 2.0 ** -18 if p.dtype == F32 else 2.0 ** -13
    for b, (n, whole) in enumerate(p.lens):
        k, v = p.seqs[b]
        o, spread, reach = ref.attend(q[at:at + n], k, v, whole - n, scale, window)
        want[at:at + n] = o
        d = (p.dim + 2) * 2.0 ** -24 * reach[..., None]
        inner = (hp + 2 * d + (whole + 8) * 2.0 ** -24 + ex) * spread
        if p.bits == 4 or p.dtype == F16:
            inner = inner + TINY * v.abs().sum(0).repeat_interleave(q_heads // p.heads, 0)
        tol[at:at + n] = half_step(p.dtype) * o.abs() + (1 + half_step(p.dtype)) * inner + TINY
        at += n
    within(out, want, tol, what or "paged attention")
    assert ops.device_error() == 0
    return out


SEQS = {
    "decode": [(1, 1), (1, 2), (1, 17), (1, 300), (1, 64), (1, 129), (1, 1000)],
    "mixed": [(5, 5), (0, 40), (1, 333), (37, 100), (2, 1), (1, 0), (64, 64), (3, 700), (130, 260)],
    "long": [(1, 5000), (1, 4999), (2, 3000)],
    "one": [(1, 1)],
    "chunks": [(128, 128), (200, 513), (1, 1), (257, 900)],
}


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("lens,kv_heads,group,dim,page", [
    ("decode", 2, 1, 64, 16), ("decode", 2, 4, 128, 16), ("decode", 1, 8, 128, 64), ("decode", 1, 16, 64, 8),
    ("decode", 2, 3, 96, 24), ("mixed", 2, 4, 128, 16), ("mixed", 2, 2, 64, 1), ("mixed", 1, 7, 96, 32),
    ("mixed", 2, 1, 256, 16), ("mixed", 1, 20, 64, 16), ("mixed", 1, 2, 48, 16), ("long", 4, 8, 128, 128), ("long", 12, 1, 64, 16),
    ("one", 1, 1, 64, 16), ("chunks", 2, 4, 128, 32), ("chunks", 3, 1, 64, 16), ("chunks", 1, 5, 128, 7), ("chunks", 2, 4, 96, 16),
    ("chunks", 1, 3, 32, 256), ("chunks", 2, 2, 64, 128), ("chunks", 2, 2, 128, 8),
])
def test_paged_attention(lens, kv_heads, group, dim, page, bits, dtype):
    p = ref.Paged(SEQS[lens], kv_heads, dim, page, dtype, seed=dim + page + group, bits=bits, gain=0.5 if bits == 4 else 1.0,
                  extra_tokens=2)
    q = p.queries(kv_heads * group)
    first = check_attention(p, kv_heads * group, q=q)
    hinted = check_attention(p, kv_heads * group, q=q, max_q_len=max(n for n, _ in p.lens))
    assert first.shape == hinted.shape


@pytest.mark.parametrize("lens", ["mixed", "chunks"])
@pytest.mark.parametrize("dim,dtype", [(64, F32), (20, F32), (128, F32), (40, F16), (200, BF16), (6, F16)])
def test_paged_attention_other_dims(dim, dtype, lens):
    p = ref.Paged(SEQS[lens], 2, dim, 8, dtype, seed=dim)
    check_attention(p, 4)


@pytest.mark.parametrize("window", [1, 7, 64, 100, 5000])
@pytest.mark.parametrize("lens", ["mixed", "long", "chunks"])
@pytest.mark.parametrize("bits,dim", [(16, 64), (16, 128), (4, 128), (16, 80)])
def test_paged_attention_window(window, lens, bits, dim):
    p = ref.Paged(SEQS[lens], 2, dim, 16, BF16, seed=window, bits=bits)
    check_attention(p, 8, window=window)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("lens", ["decode", "chunks"])
def test_paged_attention_strides_and_shared_pages(lens, bits):
    """Queries out of a fused projection, keys and values in one tensor, sequences that share pages."""
    ops = _ops()
    p = ref.Paged(SEQS[lens], 2, 128, 16, F16, seed=12, bits=bits)
    cache, t = cache_of(p)
    q = torch.randn(p.tokens, 12, 128).half().cuda()
    plain = ops.paged_attention(q[:, :8].contiguous(), cache, *where(p))
    both = torch.stack((t["k"], t["v"]), 1)
    scales = [t.get(n) for n in ("k_scales", "v_scales")]
    view = ops.PagedKVCache(both[:, 0], both[:, 1], *scales)
    assert torch.equal(ops.paged_attention(q[:, :8], view, *where(p)), plain)
    twice = [x.repeat_interleave(2, 0) if i != 1 else x for i, x in enumerate(where(p))]
    n = (p.seq_starts[1:] - p.seq_starts[:-1]).repeat_interleave(2)
    twice[1] = torch.cat((torch.zeros(1), n.cumsum(0))).int().cuda()
    rows = torch.cat([torch.arange(a, b).repeat(2) for a, b in zip(p.seq_starts[:-1].tolist(), p.seq_starts[1:].tolist())])
    doubled = ops.paged_attention(q[:, :8][rows.cuda()], cache, *twice)
    wide = torch.empty(p.tokens, 3, 8, 128, dtype=F16, device="cuda")
    assert torch.equal(ops.paged_attention(q[:, :8], cache, *where(p), out=wide[:, 1]), plain)
    # The work may be split at other places: equal up to the rounding of 16-bit outputs and probabilities.
    assert (doubled.float() - plain[rows.cuda()].float()).abs().max() <= 2.0 ** -9 * 4


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dim", [64, 128, 40])
def test_paged_attention_masked_places_do_not_leak(bits, dim):
    """Slots behind a sequence's end hold NaN (the pool's filling); keys outside the window too."""
    if bits == 4 and dim == 40:
        dim = 48
    p = ref.Paged([(1, 37), (3, 50), (1, 0), (2, 3)], 2, dim, 16, F16, seed=8, bits=bits)
    pos = torch.arange(0, 20)
    for name in ("k", "v"):   # the first 20 positions of sequence 1 are not numbers; its queries see the last 16 keys
        p.put(name, 1, pos, torch.full((20, 2, dim), float("nan"), dtype=F16))
    out = check_attention(p, 4, window=16)
    assert (out[4] == 0).all()   # the row of the empty sequence


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dim", [64, 128, 24])
def test_paged_attention_nan_key_poisons_its_rows_only(bits, dim):
    ops = _ops()
    if bits == 4 and dim == 24:
        dim = 32
    p = ref.Paged([(1, 40), (6, 150), (1, 90)], 2, dim, 16, BF16, seed=9, bits=bits)
    bad = torch.randn(1, 2, dim).bfloat16()
    bad[0, 1, 3] = float("nan")
    p.put("k", 1, torch.tensor([147]), bad)   # queries of sequence 1 stand at 144..149
    cache, _ = cache_of(p)
    out = ops.paged_attention(p.queries(6).cuda(), cache, *where(p))
    nan = out.isnan().all(-1).cpu()
    want = torch.zeros(8, 6, dtype=torch.bool)
    want[4:7, 3:] = True
    assert torch.equal(nan, want) and torch.equal(out.isnan().any(-1).cpu(), want)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("lens", ["decode", "chunks"])
def test_paged_attention_bad_pages(lens, bits):
    """Keys of a page outside the cache are left out; a length behind the page table is cut."""
    ops = _ops()
    p = ref.Paged(SEQS[lens], 2, 128, 16, BF16, seed=10, bits=bits)
    q = p.queries(4)
    cache, _ = cache_of(p)
    tab, starts, lens_ = where(p)
    b = len(p.lens) - 1
    tab[b, 3] = cache.num_pages
    out = ops.paged_attention(q.cuda(), cache, tab, starts, lens_)
    assert ops.device_error() == 0x502
    n, whole = p.lens[b]
    k, v = p.seqs[b]
    want = []
    for i in range(n):   # the definition over the keys that are left
        pos = whole - n + i
        keep = [j for j in range(pos + 1) if j // 16 != 3]
        o = ref.attend(q[p.owned - n + i][None], k[keep], v[keep], len(keep) - 1, 128 ** -0.5)[0]
        want.append(o)
    want = torch.cat(want)
    assert ((out[-n:].cpu().double() - want).abs() <= 2.0 ** -6 * (want.abs() + 1)).all()
    lens_[0] = 16 * tab.shape[1] + 5
    tab[0] = 0
    ops.paged_attention(q.cuda(), cache, tab, starts, lens_)
    assert ops.device_error() in (0x502, 0x503)


@pytest.mark.parametrize("size", [600.0, 2.0 ** 100, 2.0 ** -80, 0.0])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("lens", [[(1, 200), (4, 77)], [(64, 200), (150, 300)]])
def test_paged_attention_extreme_scores(lens, bits, size):
    """Scores far beyond the 16-bit ranges, and queries far below them, neither overflow nor lose the softmax."""
    p = ref.Paged(lens, 2, 128, 16, BF16, seed=13, bits=bits)
    q = p.queries(4) * size
    if size == 2.0 ** 100:   # one-hot rows: a rounding of the score cannot change which key is the largest
        ops = _ops()
        cache, _ = cache_of(p)
        out = ops.paged_attention(q.cuda(), cache, *where(p)).cpu().double()
        at = 0
        for b, (n, whole) in enumerate(p.lens):
            k, v = p.seqs[b]
            want = ref.attend(q[at:at + n], k, v, whole - n, 128 ** -0.5)[0]
            assert ((out[at:at + n] - want).abs() <= half_step(BF16) * want.abs() + TINY).all()
            at += n
        return
    check_attention(p, 4, q=q, what="extreme scores")


@pytest.mark.parametrize("bits,dim", [(16, 64), (16, 128), (4, 128), (16, 20)])
@pytest.mark.parametrize("lens", ["mixed", "chunks"])
@pytest.mark.parametrize("scale", [0.0, -0.1, 1.0])
def test_paged_attention_scales(scale, lens, bits, dim):
    p = ref.Paged(SEQS[lens], 2, dim, 16, BF16, seed=15, bits=bits)
    check_attention(p, 4, scale=scale)


@pytest.mark.parametrize("bits", [16, 4])
def test_paged_attention_many_sequences(bits):
    """More sequences than one launch plans for."""
    g = torch.Generator().manual_seed(16)
    lens = [(n, n + w) for n, w in zip(torch.randint(0, 3, (2100,), generator=g).tolist(), torch.randint(0, 40, (2100,), generator=g).tolist())]
    p = ref.Paged(lens, 1, 64, 8, F16, seed=16, bits=bits, extra_tokens=2)
    check_attention(p, 2)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("lens", ["decode", "chunks", "long"])
def test_paged_attention_deterministic_and_captured(lens, bits):
    """The same call twice, on two streams at once, and in two captured graphs whose lengths change between replays."""
    ops = _ops()
    p = ref.Paged(SEQS[lens], 2, 128, 16, BF16, seed=14, bits=bits)
    q = p.queries(8).cuda()
    cache, _ = cache_of(p)
    tab, starts, lens_ = where(p)
    call = lambda: ops.paged_attention(q, cache, tab, starts, lens_)  # noqa: E731
    want = call()
    assert torch.equal(call(), want)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams * 3:
        with torch.cuda.stream(s):
            outs.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graphs, held = [], []
    for s in streams:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            held.append(call())
        graphs.append(g)
    for shorter in (0, 1):
        lens_.copy_((p.seq_lens - shorter).clamp(min=0))
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        now = call()
        assert all(torch.equal(o, now) for o in held)
    assert ops.device_error() == 0


# ───────────────────────────────────────────────── the operators together ──

@pytest.mark.parametrize("dtype,bits", [(F16, 16), (BF16, 16), (BF16, 4), (F32, 16)])
def test_decoding_step_by_step(dtype, bits):
    """Two prompts prefilled in chunks, then decoded token by token: at every step the norm, the
    rotation, the append and the attention equal dense attention over everything so far."""
    ops = _ops()
    heads, group, dim, page = 2, 4, 64, 16
    table = ops.rotary_table(300, dim, scaling={"type": "ntk", "factor": 2.0})
    cache = ops.PagedKVCache.allocate(40, heads, page, dim, dtype="e2m1" if bits == 4 else dtype)
    order = torch.randperm(40, generator=torch.Generator().manual_seed(1)).int()
    tab = order[:40].view(2, 20).cuda()
    g = torch.Generator().manual_seed(2)
    w = (1 + 0.2 * torch.randn(dim, generator=g)).to(dtype).cuda()
    have = [0, 0]
    past = [[[], []], [[], []]]   # per sequence: keys, values, as the cache was given them
    for step in ([70, 33], [60, 1], [1, 1], [1, 0], [0, 1], [2, 3], [1, 1]):
        n = sum(step)
        qkv = torch.randn(n, heads * (group + 2), dim, generator=g).to(dtype).cuda()
        q, k, v = qkv[:, :heads * group], qkv[:, heads * group:heads * (group + 1)], qkv[:, heads * (group + 1):]
        starts = torch.tensor([0, step[0], n], dtype=torch.int32, device="cuda")
        have = [a + b for a, b in zip(have, step)]
        lens = torch.tensor(have, dtype=torch.int32, device="cuda")
        pos = torch.cat([torch.arange(h - s, h) for h, s in zip(have, step)]).cuda()
        nq, nk = ops.qk_norm_rotary(q, k, pos, None, w, w)          # norm alone, the rotation on the way to the cache
        rq = ops.kv_append(nk, v, cache, tab, starts, lens, table=table, Q=nq)
        out = ops.paged_attention(rq, cache, tab, starts, lens)
        rk = ops.rotary(nk, pos, table)                             # the same by the single operators
        assert torch.equal(ops.rotary(nq, pos, table), rq)
        one_q, one_k = ops.qk_norm_rotary(q, k, pos, table, w, w)
        # One rounding fewer than norm and rotation apart: two half steps of a pair's size (below 8 here).
        assert (one_q.float() - rq.float()).abs().max() <= 2 * half_step(dtype) * 16
        at = 0
        for b, s in enumerate(step):
            if bits == 4:
                kk, vv = ops.kv_read(cache, tab, starts, lens, tokens=n, dtype=dtype)
            else:
                kk, vv = rk, v
            past[b][0].append(kk[at:at + s].cpu())
            past[b][1].append(vv[at:at + s].cpu())
            if s:
                pk, pv = (torch.cat(x) for x in past[b])
                o, spread, reach = ref.attend(rq[at:at + s].cpu(), pk, pv, have[b] - s, dim ** -0.5)
                hp = 0.0 if dtype == F32 else half_step(dtype)
                d = (dim + 2) * 2.0 ** -24 * reach[..., None]
                ex = 2.0 ** -18 if dtype == F32 else 2.0 ** -13
                inner = (hp + 2 * d + (have[b] + 8) * 2.0 ** -24 + ex) * spread
                if bits == 4 or dtype == F16:
                    inner = inner + TINY * pv.double().abs().sum(0).repeat_interleave(group, 0)
                tol = half_step(dtype) * o.abs() + (1 + half_step(dtype)) * inner + TINY
                within(out[at:at + s], o, tol, f"sequence {b} at {have[b]}")
            at += s
    assert ops.device_error() == 0


def test_prefill_equals_the_dense_attention():
    """One prompt per sequence, all of it new: the paged attention and the framework's dense causal attention."""
    ops = _ops()
    B, S, H, D = 2, 320, 3, 64
    g = torch.Generator().manual_seed(6)
    q, k, v = (torch.randn(B, S, H, D, generator=g).half().cuda() for _ in range(3))
    cache = ops.PagedKVCache.allocate(B * 20, H, 16, D)
    tab = torch.randperm(B * 20, generator=g).int().view(B, 20).cuda()
    starts = torch.tensor([0, S, 2 * S], dtype=torch.int32, device="cuda")
    lens = torch.full((B,), S, dtype=torch.int32, device="cuda")
    flat = lambda t: t.reshape(B * S, H, D)  # noqa: E731
    ops.kv_append(flat(k), flat(v), cache, tab, starts, lens)
    out = ops.paged_attention(flat(q), cache, tab, starts, lens, max_q_len=S)
    dense = ops.attention(*(t.transpose(1, 2) for t in (q, k, v)), causal=True).transpose(1, 2).reshape(B * S, H, D)
    # Each is off by a half step of the output and of its probabilities: values below 4, weights summing to 1.
    assert (out.float() - dense.float()).abs().max() <= 4 * 4 * half_step(F16)
    k2, v2 = ops.kv_read(cache, tab, starts, lens, tokens=B * S)
    assert torch.equal(k2, flat(k)) and torch.equal(v2, flat(v))
