"""CPU restatements of the decoder operators -- TEST INFRASTRUCTURE ONLY.

Rotary positions, per-head norms and attention are computed in 64 bits from their
definitions; the 4-bit quantisation, whose result is a code, follows its definition in
fp32 operations rounded one by one (torch's CPU arithmetic), so codes compare exactly.
The product path (``lunara_b200``) never calls this module.
"""
from __future__ import annotations

from typing import List, Optional, Tuple

import torch

F64 = torch.float64
E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, layout: str) -> torch.Tensor:
    """x [..., dim]; cos, sin [..., rot / 2] broadcast against x's leading dimensions. In x's dtype."""
    half = cos.shape[-1]
    out = x.clone()
    if layout == "half":
        a, b = x[..., :half], x[..., half:2 * half]
        out[..., :half], out[..., half:2 * half] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        out[..., 0:2 * half:2], out[..., 1:2 * half:2] = a * cos - b * sin, b * cos + a * sin
    return out


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor], eps: float) -> torch.Tensor:
    x = x.to(F64)
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return y if weight is None else y * weight.to(F64)


def quantise(x: torch.Tensor, gain: float) -> Tuple[torch.Tensor, torch.Tensor]:
    """fp32 [..., dim] -> (codes 0..15 [..., dim], e4m3 scale bytes [..., dim / 16])."""
    inv = torch.tensor(1.0) / torch.tensor(gain, dtype=torch.float32)
    y = (x.float() * inv).unflatten(-1, (-1, 16))
    amax = y.abs().amax(-1)
    s = torch.where(torch.isnan(amax), amax, (amax / 6.0).clamp(max=448.0)).to(torch.float8_e4m3fn)
    s32 = s.float()[..., None]
    z = torch.where(s32 > 0, y / s32, torch.zeros_like(y))
    a = z.abs()
    # Index of the nearest e2m1 magnitude; a tie goes to the even code.
    mids = (E2M1[1:] + E2M1[:-1]) / 2
    low = torch.zeros_like(a, dtype=torch.int64)
    for i, m in enumerate(mids):
        low += (a > m) | ((a == m) & (i % 2 == 1))
    return (low + 8 * torch.signbit(z)).to(torch.uint8).flatten(-2), s.view(torch.uint8)


def values(codes: torch.Tensor, scale_bytes: torch.Tensor, gain: float) -> torch.Tensor:
    """What codes and scales stand for, in 64 bits."""
    sign = 1.0 - 2.0 * (codes >= 8)
    mag = E2M1.to(F64)[(codes & 7).long()] * sign
    s = scale_bytes.view(torch.float8_e4m3fn).to(F64) * float(torch.tensor(gain, dtype=torch.float32))
    return (mag.unflatten(-1, (-1, 16)) * s[..., None]).flatten(-2)


def pack(codes: torch.Tensor) -> torch.Tensor:
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def unpack(packed: torch.Tensor) -> torch.Tensor:
    return torch.stack((packed & 15, packed >> 4), -1).flatten(-2)


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, first: int, scale: float, window: int = 0):
    """One sequence in 64 bits: q [n, heads, dim] at positions first.., k and v [length, kv_heads, dim].

    Returns (o, spread, reach): the output, sum_j p_j |v_j| (what a relative error of the
    probabilities can move it by), and the largest |scale| sum |q||k| over visible keys
    (what rounding moves a score by, times its relative error). A row that sees no key is 0."""
    n, heads, dim = q.shape
    group = heads // k.shape[1]
    k, v = (t.to(F64).repeat_interleave(group, 1).transpose(0, 1) for t in (k, v))
    q = q.to(F64).transpose(0, 1)
    pos = first + torch.arange(n)[:, None]
    key = torch.arange(k.shape[1])[None, :]
    seen = (key <= pos) & (pos >= 0)
    if window:
        seen &= key > pos - window
    s = (q @ k.transpose(1, 2) * scale).masked_fill(~seen, float("-inf"))
    top = s.amax(-1, keepdim=True) if s.shape[-1] else torch.full((heads, n, 1), float("-inf"), dtype=F64)
    p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    p = p * seen
    reach = (q.abs() @ k.abs().transpose(1, 2) * abs(scale) * seen).amax(-1) if s.shape[-1] else torch.zeros(heads, n, dtype=F64)
    # Unseen values take no part even where they are not finite.
    return ((p @ torch.nan_to_num(v)).transpose(0, 1), (p @ torch.nan_to_num(v).abs()).transpose(0, 1), reach.transpose(0, 1))


class Paged:
    """A ragged batch with its page table and a pool whose unused slots hold NaN."""

    def __init__(self, lens: List[Tuple[int, int]], heads: int, dim: int, page: int, dtype, seed: int, bits: int = 16,
                 gain: float = 1.0, extra_pages: int = 2, extra_tokens: int = 0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.heads, self.dim, self.page, self.dtype, self.bits, self.gain = lens, heads, dim, page, dtype, bits, gain
        self.g = g
        need = [-(-max(whole, 0) // page) for _, whole in lens]
        pages = sum(need) + extra_pages
        order = torch.randperm(pages, generator=g)
        table = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n].to(torch.int32)
            at += n
        self.page_table = table
        starts = [0]
        for n, _ in lens:
            starts.append(starts[-1] + n)
        self.seq_starts = torch.tensor(starts, dtype=torch.int32)
        self.seq_lens = torch.tensor([whole for _, whole in lens], dtype=torch.int32)
        self.tokens = starts[-1] + extra_tokens
        self.owned = starts[-1]
        self.seqs = []   # (k, v) of each sequence [length, heads, dim], what the cache stands for, float64
        shape = (pages, heads, page)
        self.tensors = {}
        for name in ("k", "v"):
            if bits == 4:
                self.tensors[name] = torch.full((*shape, dim // 2), 0x77, dtype=torch.uint8)
                self.tensors[name + "_scales"] = torch.full((*shape, dim // 16), 0x7F, dtype=torch.uint8)   # NaN
            else:
                self.tensors[name] = torch.full((*shape, dim), float("nan"), dtype=dtype)
        for b, (_, whole) in enumerate(lens):
            pair = []
            for name in ("k", "v"):
                x = torch.randn(max(whole, 0), heads, dim, generator=g).to(dtype)
                pair.append(self.put(name, b, torch.arange(max(whole, 0)), x))
            self.seqs.append(pair)

    def put(self, name: str, b: int, pos: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
        """Store rows x [n, heads, dim] at positions of sequence b; returns what they stand for."""
        page, slot = self.page_table[b].long()[pos // self.page], pos % self.page
        if self.bits == 4:
            codes, scales = quantise(x, self.gain)
            self.tensors[name][page, :, slot] = pack(codes)
            self.tensors[name + "_scales"][page, :, slot] = scales
            return values(codes, scales, self.gain)
        self.tensors[name][page, :, slot] = x
        return x.to(F64)

    def queries(self, q_heads: int) -> torch.Tensor:
        return torch.randn(self.tokens, q_heads, self.dim, generator=self.g).to(self.dtype)
