"""GPU tests of the decoder operators at the edges of their ranges: scales of partly filled
tiles, signs of zero, finite values of any size at masked places, scores far from zero in rows
that are cut, factors near fp32's ends, rows that no sequence owns, and large batches.

Tolerances as in test_gpu_decoder, whose helpers these use; where a test derives its own, the
terms stand beside it.
"""
import numpy as np
import pytest
import torch

from oracle import decoder as ref
from test_gpu_decoder import BF16, F16, F32, TINY, _ops, cache_of, check_attention, half_step, where, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,page,heads", [(32, 8, 1), (32, 64, 2), (96, 16, 2), (96, 128, 1), (64, 16, 2), (128, 16, 2)])
def test_4bit_scales_of_every_group(dim, page, heads, dtype):
    """Keys and values whose 16-element blocks differ in size by up to 2^8 from one key to the next."""
    p = ref.Paged([(1, 300), (5, 77), (1, 31), (2, 1000)], heads, dim, page, dtype, seed=dim + page, bits=4)
    for b, (_, whole) in enumerate(p.lens):
        for i, name in enumerate(("k", "v")):
            size = 2.0 ** torch.randint(-4, 1 if name == "k" else 5, (whole, heads, dim // 16, 1), generator=p.g)
            x = (torch.randn(whole, heads, dim // 16, 16, generator=p.g) * size).flatten(2).to(dtype)
            p.seqs[b][i] = p.put(name, b, torch.arange(whole), x)
    check_attention(p, 4 * heads)


def test_kv_append_4bit_signs_of_zero():
    """A negative zero keeps its sign in the code, as its quotient by the scale does; in a block of zeros there is no quotient."""
    ops = _ops()
    x = torch.randn(8, 2, 64, generator=torch.Generator().manual_seed(21))
    x[:, :, ::3] = -0.0
    x[:, :, 1::6] = 0.0
    x[3] = -0.0
    for dtype in (F32, F16, BF16):
        for skip in (0, 1):   # 16-byte aligned rows, and others
            flat = torch.zeros(x.numel() + 1, dtype=dtype, device="cuda")
            rows = flat[skip:skip + x.numel()].view(8, 2, 64)
            rows.copy_(x)
            cache = ops.PagedKVCache.allocate(1, 2, 8, 64, dtype="e2m1")
            tab, starts, lens = (torch.tensor(a, dtype=torch.int32, device="cuda") for a in ([[0]], [0, 8], [8]))
            ops.kv_append(rows, rows, cache, tab, starts, lens)
            codes, scales = ref.quantise(x.to(dtype).float(), 1.0)
            assert (codes == 8).any()
            assert torch.equal(cache.k_pages[0].cpu(), ref.pack(codes).transpose(0, 1)), (dtype, skip)
            assert torch.equal(cache.v_scales.view(torch.uint8)[0].cpu(), scales.transpose(0, 1))


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (80, 7)])
@pytest.mark.parametrize("lens", [[(100, 100), (128, 128), (64, 128)], [(4, 100), (2, 128), (1, 100)]])
def test_huge_values_behind_a_row_do_not_reach_it(lens, dim, page):
    """Values of the order of 2^121 at the last ten positions, which only the last tokens see. (All keys stand in one block of
    128, so probabilities before the division are at most 1, and ten such values stay below fp32's largest number.)"""
    p = ref.Paged(lens, 2, dim, page, BF16, seed=dim + page)
    for b, (_, whole) in enumerate(p.lens):
        pos = torch.arange(whole - 10, whole)
        x = (2.0 ** 121 * (1 + torch.rand(10, 2, dim, generator=p.g))).to(BF16)
        p.seqs[b][1][pos] = p.put("v", b, pos, x)
    check_attention(p, 4)


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (80, 7)])
@pytest.mark.parametrize("lens,size", [([(100, 228), (40, 200)], 2.0 ** 126), ([(3, 228)], 2.0 ** 121)])
def test_huge_values_of_far_lower_scores_do_not_count(lens, size, dim, page):
    """Huge values whose keys' scores lie 200 below the others': weights of e^-200 leave nothing of them. (Where a part of the
    work has no other keys, their weights in it are 1, and 32 of them have to sum to an fp32 number.)"""
    p = ref.Paged(lens, 2, dim, page, BF16, seed=dim + page)
    scale = 0.125
    for b, (_, whole) in enumerate(p.lens):
        k, v = (x.clone() for x in p.seqs[b])
        k[:, :, 0] = 0
        k[:40, :, 0] = -100
        v[:40] = size
        p.seqs[b] = [p.put(name, b, torch.arange(whole), x.to(BF16)) for name, x in (("k", k), ("v", v))]
    q = p.queries(4)
    q[:, :, 0] = 16
    check_attention(p, 4, q=q, scale=scale)


# Scores of the order of 2^17 that are exact in fp32 (2^17 and sixteenths), so that what an output can be off by
# has no score term: half a step of it and of the probabilities, 2^-13 for the exponential (1.2e-4), and a 2^-24 for
# each key's sum and for the factors.

def _far_pair(factor=1.4426950408889634):
    """Two offsets whose products with the factor are rounded farthest apart in fp32."""
    x = np.arange(0, 8, 1 / 16)
    off = ((131072 + x).astype(np.float32) * np.float32(factor)).astype(np.float64) - (131072 + x) * float(np.float32(factor))
    best = max(((abs(off[i] - off[j]), i, j) for i in range(len(x)) for j in range(len(x)) if abs(x[i] - x[j]) <= 1), key=lambda t: t[0])
    assert best[0] > 0.01
    return float(x[best[1]]), float(x[best[2]])


def _far_scores(lens, tall, split):
    """One key head of 64: keys (256, x, 0 ..) with x of two values, `split` keys of the first; queries (512, 1 or `tall`, 0 ..)."""
    p = ref.Paged(lens, 1, 64, 16, F16, seed=31)
    a, b = _far_pair()
    for s, (_, whole) in enumerate(p.lens):
        k = torch.zeros(whole, 1, 64)
        k[:, 0, 0] = 256
        k[:, 0, 1] = torch.where(torch.arange(whole) < split, min(a, b), max(a, b))
        v = torch.zeros(whole, 1, 64)
        v[:split] = 1
        v[:, 0, 5] = torch.randn(whole, generator=p.g)
        p.seqs[s] = [p.put("k", s, torch.arange(whole), k.half()), p.put("v", s, torch.arange(whole), v.half())]
    q = torch.zeros(p.tokens, 1, 64)
    q[:, 0, 0], q[:, 0, 1] = 512, 1
    q[1::2, 0, 1] = tall
    return p, q.half()


def _check_far(p, q):
    ops = _ops()
    cache, _ = cache_of(p)
    out = ops.paged_attention(q.cuda(), cache, *where(p), scale=1.0)
    at, h = 0, half_step(F16)
    for b, (n, whole) in enumerate(p.lens):
        k, v = p.seqs[b]
        want, spread, _ = ref.attend(q[at:at + n], k, v, whole - n, 1.0)
        tol = h * want.abs() + (1 + h) * (h + 2.0 ** -13 + (whole + 16) * 2.0 ** -24) * spread + (1 + whole) * TINY
        within(out[at:at + n], want, tol, f"sequence {b}")
        at += n


@pytest.mark.parametrize("n", [1, 4, 12, 64, 300])
def test_far_scores_of_cut_rows(n):
    """One sequence, cut into many parts that have one of two maxima."""
    _check_far(*_far_scores([(n, 4096 + n)], 1.0, 2048))


def test_far_scores_of_whole_rows():
    """Prompts of two key blocks, many of them to a run; every second row's maximum grows far, so that all rows are rescaled."""
    _check_far(*_far_scores([(40, 256)] * 300, 60.0, 128))


@pytest.mark.parametrize("dim", [32, 20])
def test_fp32_weights_are_fp32(dim):
    """Two keys with scores 0 and -x, values 0 and 1: the output is e^-x / (1 + e^-x), every product exact. Off by the
    exponential (2 ulp), the sum, the rescaling product, the division and its product: below 8 roundings of 2^-24."""
    ops = _ops()
    n = 60
    p = ref.Paged([(1, 2)] * n, 1, dim, 8, F32, seed=4)
    q = torch.zeros(n, 1, dim)
    q[:, 0, 0] = 1
    want = torch.empty(n, dtype=torch.float64)
    for b in range(n):
        x = b / 2 + 0.25
        k, v = torch.zeros(2, 1, dim), torch.zeros(2, 1, dim)
        far = b % 2   # which of the two keys comes first
        k[far, 0, 0] = -x
        v[far] = 1
        p.put("k", b, torch.arange(2), k)
        p.put("v", b, torch.arange(2), v)
        want[b] = np.exp(-x) / (1 + np.exp(-x))
    cache, _ = cache_of(p)
    out = ops.paged_attention(q.cuda(), cache, *where(p), scale=1.0)
    want = want[:, None, None].expand(n, 1, dim)
    within(out, want, 2.0 ** -21 * want, "weights")


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("lens", [[(1, 200), (4, 77), (1, 3000)], [(64, 200), (150, 300)]])
@pytest.mark.parametrize("scale,size", [(0.0, 2.0 ** -110), (0.0, 2.0 ** 110), (2.0 ** -110, 2.0 ** 100), (2.0 ** -100, 2.0 ** -60),
                                        (2.0 ** -110, 2.0 ** 110), (-2.0 ** -105, 2.0 ** 105), (2.0 ** 100, 2.0 ** -100)])
def test_scales_near_the_ends(scale, size, lens, bits):
    """The scale takes its part at any size, zero included; queries make up for it, or do not."""
    p = ref.Paged(lens, 2, 128, 16, BF16, seed=16, bits=bits)
    check_attention(p, 4, scale=scale, q=p.queries(4) * size)


@pytest.mark.parametrize("dim", [64, 128])
def test_4bit_queries_at_the_upper_end(dim):
    """Rows with an element of 2^127 and more, the others far below."""
    p = ref.Paged([(1, 200), (3, 50), (40, 90)], 2, dim, 16, BF16, seed=17, bits=4)
    q = torch.randn(p.tokens, 4, dim, generator=p.g) * 2.0 ** 124
    q = q.clamp(-2.0 ** 126, 2.0 ** 126)
    q[:, :, 3] = 1.5 * 2.0 ** 127 * (1 - 2 * torch.randint(0, 2, q.shape[:2], generator=p.g))
    check_attention(p, 4, scale=2.0 ** -126, q=q.to(BF16))


@pytest.mark.parametrize("bits,dim,dtype", [(16, 64, BF16), (4, 128, F16), (16, 20, F16), (16, 64, F32), (4, 48, BF16)])
@pytest.mark.parametrize("lens", [[(1, 17), (0, 3), (1, 300)], [(100, 130), (0, 0)], [(0, 5), (0, 0)], []])
def test_rows_of_no_sequence_are_zero_in_new_outputs(lens, bits, dim, dtype):
    """Padded batches: memory that the call allocates holds nothing of what stood there before."""
    ops = _ops()
    p = ref.Paged(lens, 2, dim, 16, dtype, seed=18, bits=bits, extra_tokens=5)
    cache, _ = cache_of(p)
    k = torch.randn(p.tokens, 2, dim, generator=p.g).to(dtype).cuda()
    q = p.queries(4).cuda()

    def fresh(call, shape):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        dirt = [torch.full(shape, float("nan"), dtype=dtype, device="cuda") for _ in range(4)]
        del dirt
        got = call()
        for out in got if isinstance(got, tuple) else (got,):
            assert out.shape == shape and (out[p.owned:] == 0).all()
            assert torch.isfinite(out).all()

    fresh(lambda: ops.kv_append(k, k, cache, *where(p), Q=q, table=ops.rotary_table(400, 16)), tuple(q.shape))
    fresh(lambda: ops.kv_read(cache, *where(p), tokens=p.tokens, dtype=dtype), (p.tokens, 2, dim))
    fresh(lambda: ops.paged_attention(q, cache, *where(p)), tuple(q.shape))
    assert ops.device_error() == 0


@pytest.mark.parametrize("dim", [64, 128])
def test_many_sequences_with_prompts_among_them(dim):
    """More sequences than one launch plans for, with prompts (tcgen05) among single tokens in each share of them."""
    g = torch.Generator().manual_seed(19)
    lens = [(int(n), int(n) + int(w)) for n, w in zip(torch.randint(0, 3, (2100,), generator=g), torch.randint(0, 40, (2100,), generator=g))]
    for b, pair in {3: (40, 300), 1023: (70, 70), 1024: (33, 500), 1500: (17, 400), 1501: (200, 1000), 2047: (16, 90), 2048: (130, 130),
                    2099: (64, 700)}.items():
        lens[b] = pair
    p = ref.Paged(lens, 1, dim, 8, F16, seed=20, extra_tokens=2)
    check_attention(p, 2)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("n,group", [(1, 1), (1, 8), (2, 8)])
def test_one_long_sequence_of_one_key_head(n, group, bits):
    """All of the GPU's warps share one row tile, whose join has over a thousand parts."""
    ops = _ops()
    p = ref.Paged([(n, 50000)], 1, 128, 32, BF16, seed=n + group, bits=bits)
    q = p.queries(group)
    out = check_attention(p, group, q=q)
    cache, _ = cache_of(p)
    assert torch.equal(ops.paged_attention(q.cuda(), cache, *where(p)), out)


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, F16), (64, F16), (20, BF16), (64, F32)])
@pytest.mark.parametrize("lens", [[(100, 300), (40, 128)], [(2, 300), (1, 128)]])
def test_infinite_scores(lens, dim, dtype):
    """A row with a score of +inf, or 0 * inf, has no softmax and is NaN, in whichever column of a block that key stands;
    a score of -inf weighs nothing; a row whose scores are all -inf is zero."""
    ops = _ops()
    p = ref.Paged(lens, 1, dim, 16, dtype, seed=22)
    keys = [0, 1, 7, 8, 9, 16, 33, 64, 70, 101, 127]
    for at in keys:   # one at a time; the queries' first elements are +1, -1 and 0 in turn
        q = p.queries(3)
        q[:, :, 0] = torch.tensor([1.0, -1.0, 0.0])
        for b, (_, whole) in enumerate(p.lens):
            k = p.seqs[b][0].clone().to(dtype)
            k[at, 0, 0] = float("inf")
            p.put("k", b, torch.arange(whole), k)
        cache, _ = cache_of(p)
        out = ops.paged_attention(q.cuda(), cache, *where(p)).cpu()
        row = 0
        for b, (n, whole) in enumerate(p.lens):
            k, v = p.seqs[b]
            for i in range(n):
                pos = whole - n + i
                if pos < at:
                    assert torch.isfinite(out[row]).all(), (at, b, i)
                else:
                    assert out[row, 0].isnan().all() and out[row, 2].isnan().all(), (at, b, i)
                    keep = [j for j in range(pos + 1) if j != at]
                    want = ref.attend(q[row:row + 1, 1:2], k[keep], v[keep], len(keep) - 1, dim ** -0.5)[0] if keep else torch.zeros(1, 1, dim)
                    assert ((out[row, 1].double() - want[0, 0]).abs() <= 2.0 ** -6 * (want[0, 0].abs() + 1)).all(), (at, b, i)
                row += 1
    for b, (_, whole) in enumerate(p.lens):
        k = p.seqs[b][0].clone().to(dtype)
        k[:, 0, 0] = float("inf")
        p.put("k", b, torch.arange(whole), k)
    q = p.queries(3)
    q[:, :, 0] = -1
    cache, _ = cache_of(p)
    assert (ops.paged_attention(q.cuda(), cache, *where(p)) == 0).all()


@pytest.mark.parametrize("bits,dtype", [(16, BF16), (4, BF16), (16, F32)])
def test_caches_beyond_4_gib(bits, dtype):
    """Pages whose bytes stand beyond 2^32: the operators do there what they do in a small cache."""
    ops = _ops()
    heads, dim, page = 2, 128, 16
    row = {(16, BF16): 256, (4, BF16): 64, (16, F32): 512}[bits, dtype]
    far = (5 << 30) // (heads * page * row)
    small = ops.PagedKVCache.allocate(64, heads, page, dim, dtype="e2m1" if bits == 4 else dtype)
    tensors = [t for t in (small.k_pages, small.v_pages, small.k_scales, small.v_scales) if t is not None]
    big = ops.PagedKVCache(*(torch.empty(far + 64, *t.shape[1:], dtype=t.dtype, device="cuda") for t in tensors))
    g = torch.Generator().manual_seed(23)
    order = torch.randperm(64, generator=g).int()
    tab = torch.full((3, 20), -1, dtype=torch.int32)
    lens, new = [300, 17, 260], [200, 17, 1]
    at = 0
    for b, n in enumerate(lens):
        need = -(-n // page)
        tab[b, :need] = order[at:at + need]
        at += need
    starts = torch.tensor([0] + lens).cumsum(0).int().cuda()
    whole = torch.tensor(lens, dtype=torch.int32, device="cuda")
    k, v = (torch.randn(sum(lens), heads, dim, generator=g).to(dtype).cuda() for _ in range(2))
    tabs = tab.cuda(), torch.where(tab >= 0, tab + far, tab).cuda()
    out = []
    for cache, t in zip((small, big), tabs):
        ops.kv_append(k, v, cache, t, starts, whole)
        got = list(ops.kv_read(cache, t, starts, whole, tokens=sum(lens), dtype=dtype))
        for count in (new, [1, 1, 1]):
            s = torch.tensor([0] + count).cumsum(0).int().cuda()
            q = torch.randn(sum(count), 4, dim, generator=torch.Generator().manual_seed(24)).to(dtype).cuda()
            got.append(ops.paged_attention(q, cache, t, s, whole))
        out.append(got)
    assert all(torch.equal(a, b) for a, b in zip(*out)) and out[0][2].abs().sum() > 0
    if bits == 16:
        assert torch.equal(out[1][0], k) and torch.equal(out[1][1], v)
    assert ops.device_error() == 0


@pytest.mark.parametrize("bits", [16, 4])
def test_a_cache_without_pages(bits):
    """Every key's page is outside the cache: recorded, and all rows are zero."""
    ops = _ops()
    cache = ops.PagedKVCache.allocate(0, 2, 16, 64, dtype="e2m1" if bits == 4 else F16)
    tab, starts, lens = (torch.tensor(a, dtype=torch.int32, device="cuda") for a in ([[0] * 8], [0, 60], [100]))
    q = torch.randn(60, 4, 64, device="cuda", dtype=F16)
    out = ops.paged_attention(q, cache, tab, starts, lens)
    assert ops.device_error() == 0x502 and (out == 0).all()
    assert ops.kv_append(q[:, :2], q[:, 2:], cache, tab, starts, lens) is None
    assert ops.device_error() == 0x502
    k, v = ops.kv_read(cache, tab, starts, lens, tokens=60, dtype=F16)
    assert ops.device_error() == 0x502 and (k == 0).all() and (v == 0).all()


@pytest.mark.parametrize("bits,dim,dtype", [(16, 64, BF16), (4, 128, F16), (16, 20, F16)])
@pytest.mark.parametrize("lens", [[(1, 17), (1, 300)], [(100, 130), (3, 50)]])
def test_tokens_before_the_first_sequence(lens, bits, dim, dtype):
    """Sequences that begin behind the call's first tokens: those rows are left, or zero in a new output, the others as ever."""
    ops = _ops()
    p = ref.Paged(lens, 2, dim, 16, dtype, seed=25, bits=bits, extra_tokens=4)
    q = p.queries(4).cuda()
    k = torch.randn(p.tokens, 2, dim, generator=p.g).to(dtype).cuda()
    table = ops.rotary_table(400, 16)
    tab, starts, seq_lens = where(p)
    n = p.owned
    moved = lambda x: torch.cat((x[n:], x[:n]))  # noqa: E731  (the four tokens of no sequence to the front)
    plain, late = cache_of(p)[0], cache_of(p)[0]
    want = [ops.kv_append(k, k, plain, tab, starts, seq_lens, table=table, Q=q), *ops.kv_read(plain, tab, starts, seq_lens, p.tokens, dtype),
            ops.paged_attention(q, plain, tab, starts, seq_lens)]
    at = starts + 4
    got = [ops.kv_append(moved(k), moved(k), late, tab, at, seq_lens, table=table, Q=moved(q)), *ops.kv_read(late, tab, at, seq_lens, p.tokens, dtype),
           ops.paged_attention(moved(q), late, tab, at, seq_lens)]
    for a, b in zip(want, got):
        assert torch.equal(a[:n], b[4:]) and (b[:4] == 0).all() and (a[n:] == 0).all()
    out = torch.full_like(q, 7.0)
    assert torch.equal(ops.paged_attention(moved(q), late, tab, at, seq_lens, out=out)[4:], got[3][4:]) and (out[:4] == 7).all()
    assert torch.equal(late.k_pages.view(torch.uint8), plain.k_pages.view(torch.uint8))
    assert ops.device_error() == 0


@pytest.mark.parametrize("bits,dim,dtype", [(16, 128, BF16), (4, 64, F16), (16, 20, F16), (16, 64, F32)])
def test_the_output_may_be_the_queries(bits, dim, dtype):
    """In place, where rows are cut between many warps, whole, without keys, and on both kernels."""
    ops = _ops()
    p = ref.Paged([(1, 3000), (200, 900), (3, 40), (2, 0), (128, 128)], 2, dim, 16, dtype, seed=26, bits=bits, extra_tokens=2)
    cache, _ = cache_of(p)
    q = p.queries(6).cuda()
    want = ops.paged_attention(q, cache, *where(p))
    here = q.clone()
    assert ops.paged_attention(here, cache, *where(p), out=here) is here
    assert torch.equal(here[:p.owned], want[:p.owned]) and torch.equal(here[p.owned:], q[p.owned:])


@pytest.mark.parametrize("bits", [16, 4])
def test_a_captured_decode_step_replayed(bits):
    """Norm, rotation, append and attention of a padded batch as one graph, whose lengths grow on the device, against the same
    calls outside of it; two graphs over two caches are replayed on two streams at once."""
    ops = _ops()
    heads, group, dim, page, batch = 2, 4, 128, 16, 5
    g = torch.Generator().manual_seed(27)
    table = ops.rotary_table(200, dim)
    w = torch.rand(dim, generator=g).bfloat16().cuda() + 0.5
    first = torch.tensor([0, 15, 16, 90, 47], dtype=torch.int32)
    starts = torch.arange(batch + 1, dtype=torch.int32, device="cuda")
    rows = heads * (group + 2)

    class Side:
        def __init__(self):
            self.cache = ops.PagedKVCache.allocate(40, heads, page, dim, dtype="e2m1" if bits == 4 else BF16)
            self.tab = torch.randperm(40, generator=g).int().view(batch, 8).cuda()
            self.lens = first.clone().cuda()
            self.qkv = torch.zeros(batch + 2, rows, dim, dtype=BF16, device="cuda")   # two rows of no sequence

        def step(self):
            self.lens.add_(1)
            q, k, v = self.qkv.split([heads * group, heads, heads], 1)
            pos = torch.cat((self.lens - 1, self.lens.new_zeros(2)))
            nq, nk = ops.qk_norm_rotary(q, k, pos, None, w, w)
            rq = ops.kv_append(nk, v, self.cache, self.tab, starts, self.lens, table=table, Q=nq)
            return ops.paged_attention(rq, self.cache, self.tab, starts, self.lens)

    graphed, plain, streams, graphs, outs = [], [], [], [], []
    for _ in range(2):
        a, b = Side(), Side()
        b.tab.copy_(a.tab)
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            a.step()   # (once before the capture)
        torch.cuda.synchronize()
        for t in (a.cache.k_pages, a.cache.v_pages) + ((a.cache.k_scales.view(torch.uint8), a.cache.v_scales.view(torch.uint8)) if bits == 4 else ()):
            t.zero_()
        a.lens.copy_(first)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = a.step()
        graphed.append(a), plain.append(b), streams.append(s), graphs.append(graph), outs.append(out)
    for _ in range(30):
        for a, b in zip(graphed, plain):
            b.qkv.copy_(torch.randn(b.qkv.shape, generator=g).bfloat16())
            a.qkv.copy_(b.qkv)
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for out, b, a in zip(outs, plain, graphed):
            want = b.step()
            assert torch.equal(out, want) and torch.isfinite(out).all() and (out[batch:] == 0).all()
            assert torch.equal(a.lens, b.lens)
    for a, b in zip(graphed, plain):
        assert torch.equal(a.cache.k_pages.view(torch.uint8), b.cache.k_pages.view(torch.uint8))
    assert ops.device_error() == 0
