"""Paged key/value cache: the tensors of a cache and the handle the kernels take.

Pages are ``[num_pages, kv_heads, page_size, head_dim]``, keys and values apart, in
fp16, bf16 or fp32, or in 4 bits: e2m1 codes as bytes ``[..., head_dim / 2]`` (the even
element in the low nibble) and e4m3 scales ``[..., head_dim / 16]``, one per 16
elements; a stored value is ``code * (scale * gain)``. Which pages belong to which
sequence is the caller's page table; the handle knows nothing of it.
"""
from __future__ import annotations

import math
import struct
from typing import Optional

import torch

from lunara_b200.runtime import _lib

_DTYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}
_CACHE = struct.Struct("17q2d")   # lunarad_cache


class PagedKVCache:
    """Keys and values of one layer. The tensors stay the caller's and may be views
    (for instance ``all_layers[i]`` or ``kv[:, 0]``) as long as each page's head holds
    its ``[page_size, head_dim]`` contiguously. What the kernels take (addresses, strides,
    sizes, gains) is packed once, so a handle's attributes cannot be assigned to: a pool
    that has grown gets a new handle."""

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, k_scales: Optional[torch.Tensor] = None,
                 v_scales: Optional[torch.Tensor] = None, k_gain: float = 1.0, v_gain: float = 1.0):
        assert k_pages.dim() == 4 and v_pages.shape == k_pages.shape, \
            "k_pages and v_pages must be [num_pages, kv_heads, page_size, head_dim] alike"
        assert k_pages.dtype == v_pages.dtype and k_pages.device == v_pages.device, \
            "k_pages and v_pages must share a dtype and a device"
        self.bits = 4 if k_pages.dtype == torch.uint8 else 8 * k_pages.element_size()
        self.num_pages, self.kv_heads, self.page_size, width = k_pages.shape
        self.k_pages, self.v_pages, self.k_scales, self.v_scales = k_pages, v_pages, k_scales, v_scales
        self.k_gain, self.v_gain = float(k_gain), float(v_gain)
        self.device = k_pages.device
        if self.bits == 4:
            self.head_dim, self.dtype = 2 * width, None
            assert width % 8 == 0, "a 4-bit cache needs a head_dim that is a multiple of 16"
            assert k_scales is not None and v_scales is not None, "a 4-bit cache needs k_scales and v_scales"
            for s in (k_scales, v_scales):
                assert s.dtype in (torch.uint8, torch.float8_e4m3fn) and s.device == self.device, \
                    "scales must be e4m3 (float8_e4m3fn or its bytes) on the pages' device"
                assert s.shape == (*k_pages.shape[:3], width // 8), "scales must be [num_pages, kv_heads, page_size, head_dim / 16]"
                self._check_inner(s)
            for gain in (self.k_gain, self.v_gain):
                if not (gain > 0 and math.isfinite(gain)):
                    raise ValueError(f"gains must be positive numbers, got {gain}")
            kind = _lib.KIND_E2M1
            ks, vs = k_scales, v_scales
        else:
            self.head_dim, self.dtype = width, k_pages.dtype
            if k_pages.dtype not in _DTYPES:
                raise TypeError(f"unsupported cache dtype {k_pages.dtype}; expected float16, bfloat16, float32 or uint8 codes")
            assert k_scales is None and v_scales is None, "only a 4-bit cache has scales"
            if self.k_gain != 1.0 or self.v_gain != 1.0:
                raise ValueError("only a 4-bit cache has gains")
            kind = _DTYPES[k_pages.dtype]
            ks = vs = None
        for p in (k_pages, v_pages):
            self._check_inner(p)
        stride = lambda t, i: 0 if t is None else t.stride(i)  # noqa: E731
        ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
        self._args = _CACHE.pack(
            ptr(k_pages), ptr(v_pages), ptr(ks), ptr(vs), k_pages.stride(0), k_pages.stride(1), v_pages.stride(0),
            v_pages.stride(1), stride(ks, 0), stride(ks, 1), stride(vs, 0), stride(vs, 1), self.num_pages, self.kv_heads,
            self.page_size, self.head_dim, kind, self.k_gain, self.v_gain)
        self._address = _lib.address_of(self._args)
        self._packed = True

    def __setattr__(self, name: str, value) -> None:
        if "_packed" in self.__dict__:
            raise AttributeError(f"a PagedKVCache keeps its tensors' addresses: make a new one instead of assigning {name}")
        super().__setattr__(name, value)

    def __delattr__(self, name: str) -> None:
        raise AttributeError(f"a PagedKVCache keeps its tensors' addresses: {name} cannot be deleted")

    def __reduce__(self):
        """Copies and unpickled handles are made anew, from their own tensors' addresses."""
        return type(self), (self.k_pages, self.v_pages, self.k_scales, self.v_scales, self.k_gain, self.v_gain)

    @staticmethod
    def _check_inner(t: torch.Tensor) -> None:
        _, _, slots, width = t.shape
        assert (width == 1 or t.stride(3) == 1) and (slots == 1 or t.stride(2) == width), \
            "a page's head must hold its [page_size, head_dim] contiguously"

    @classmethod
    def allocate(cls, num_pages: int, kv_heads: int, page_size: int, head_dim: int, dtype=torch.float16,
                 device="cuda", k_gain: float = 1.0, v_gain: float = 1.0) -> "PagedKVCache":
        """A zeroed cache; ``dtype`` is float16, bfloat16, float32 or ``"e2m1"`` (4 bits)."""
        shape = (num_pages, kv_heads, page_size)
        if dtype == "e2m1":
            assert head_dim % 16 == 0, "a 4-bit cache needs a head_dim that is a multiple of 16"
            codes = [torch.zeros(*shape, head_dim // 2, dtype=torch.uint8, device=device) for _ in range(2)]
            scales = [torch.zeros(*shape, head_dim // 16, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
                      for _ in range(2)]
            return cls(*codes, *scales, k_gain=k_gain, v_gain=v_gain)
        return cls(*(torch.zeros(*shape, head_dim, dtype=dtype, device=device) for _ in range(2)), k_gain=k_gain, v_gain=v_gain)
