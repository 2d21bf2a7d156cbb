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
