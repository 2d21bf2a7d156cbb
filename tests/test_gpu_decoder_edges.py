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
