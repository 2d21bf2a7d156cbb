"""Torch-facing decoder operators over the C ABI of ``include/lunara_b200_decoder.h``:
rotary positions, per-head query/key norms with the rotation, the paged key/value cache
and attention over it.

As in ``lunara_b200.runtime.ops`` (which re-exports these), torch owns every buffer and
the work is enqueued on torch's current stream, of the tensors' device. Shape errors raise
``AssertionError``, library errors ``ValueError`` or ``LunaraError``. The operators are
inference operators: they record no autograd graph (``rotary(..., inverse=True)`` is the
gradient of ``rotary``).

Ragged batches: the tokens of all sequences stand one behind the other;
``seq_starts`` int32 [batch + 1] says where each sequence's begin, ``seq_lens`` int32
[batch] how long each sequence is with them, ``page_table`` int32 [batch, max_pages] which
page holds its positions ``page_size * i`` onwards. Token ``i`` of ``n`` has position
``seq_len - n + i``; a negative one marks padding (written nowhere, zero in outputs).
Tokens before ``seq_starts[0]`` and behind ``seq_starts[batch]`` belong to no sequence; their
rows are left as they were in an output that is given, and zero in one that the call
allocates. All three live on the device, so a captured graph follows their contents. What is
wrong in them (a page outside the cache, a position outside the tables) is kept as a device
error (``ops.device_error()``) and treated as padding, never as an access out of bounds.
"""
from __future__ import annotations

import math
import struct
from typing import Dict, Optional, Tuple

import torch

from lunara_b200.runtime import _lib
from lunara_b200.runtime.kv_cache import PagedKVCache

_DTYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}
_LAYOUTS = {"half": _lib.ROTARY_HALF, "interleaved": _lib.ROTARY_INTERLEAVED}

# The argument structs of the header: 8-byte fields, packed in one go (a ctypes.Structure
# filled field by field costs several microseconds more per call).
_ROTARY = struct.Struct("21q")
_QK_NORM = struct.Struct("31qd")
_APPEND = struct.Struct("30q")
_READ = struct.Struct("11q")
_ATTENTION = struct.Struct("20qd")


def _dtype_code(t: torch.Tensor) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {t.dtype}; expected float16, bfloat16 or float32") from None


def _layout_code(layout: str) -> int:
    try:
        return _LAYOUTS[layout]
    except KeyError:
        raise ValueError(f"layout must be 'half' or 'interleaved', got {layout!r}") from None


# These run on every call of a decode step, whose kernels take a few microseconds: each
# tensor property is read once, and the messages are only made when they are needed.

def _check_device(like: torch.Tensor, *ts: Optional[torch.Tensor]) -> int:
    """Index of the device that all the tensors are on."""
    assert like.is_cuda, "lunara kernels take CUDA tensors"
    index = like.get_device()
    for t in ts:
        assert t is None or t.get_device() == index, f"all tensors must be on {like.device}, got {t.device}"
    return index


_current_device, _current_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _call(name: str, args: bytes, index: int, *more) -> None:
    """Run an entry point on the current stream of device `index`."""
    if _current_device() != index:
        with torch.cuda.device(index):
            return _call(name, args, index, *more)
    rc = getattr(_lib.load(), name)(args, *more, _current_stream(index))
    if rc:
        _lib.check(rc)


def _rows(t: torch.Tensor, name: str):
    """(lunarad_view, (batch, heads, seq, dim)) of [B, H, S, D] or [tokens, H, D]."""
    shape, st = t.shape, t.stride()
    if len(shape) == 4:
        batch, heads, seq, dim = shape
        view = (t.data_ptr(), st[0], st[1], st[2])
    else:
        assert len(shape) == 3, f"{name} must be [B, H, S, D] or [tokens, H, D]"
        batch, (seq, heads, dim) = 1, shape
        view = (t.data_ptr(), 0, st[1], st[0])
    assert st[-1] == 1 or dim <= 1, f"{name} needs a unit inner stride"
    return view, (batch, heads, seq, dim)


def _output(out: Optional[torch.Tensor], like: torch.Tensor, name: str):
    """(output, its lunarad_view); a new one is dense, in the order of like's strides."""
    if out is None:
        out = torch.empty_like(like)
        st = out.stride()
        if st[-1] != 1:
            out = torch.empty_like(like, memory_format=torch.contiguous_format)
            st = out.stride()
    else:
        assert out.shape == like.shape and out.dtype == like.dtype, f"{name} must be {tuple(like.shape)} {like.dtype}"
        st = out.stride()
        assert st[-1] == 1 or out.shape[-1] <= 1, f"{name} needs a unit inner stride"
        assert 0 not in st or all(s != 0 or n <= 1 for n, s in zip(out.shape, st)), \
            f"{name} is an expanded view; it cannot be written"
    return out, (out.data_ptr(), st[0], st[1], st[2]) if len(st) == 4 else (out.data_ptr(), 0, st[1], st[0])


def _zero_rest(out: torch.Tensor, batch: int) -> int:
    """For an output in fresh memory: the flag that zeroes the rows of no sequence. Where there is no
    sequence at all no kernel runs, and the rows are cleared here."""
    if batch == 0:
        out.zero_()
        return 0
    return _lib.ZERO_REST


# ───────────────────────────────────────────────────────────── rotary ──

def rotary_table(positions: int, rot_dim: int, base: float = 10000.0, scaling: Optional[Dict[str, float]] = None,
                 device="cuda") -> torch.Tensor:
    """The (cos, sin) table ``[positions, rot_dim / 2, 2]`` float32 that the rotary operators
    read, computed in 64 bits (angles of far positions lose their digits in 32).

    Frequency i is ``base ** (-2 i / rot_dim)``. ``scaling`` stretches a context:

    * ``{"type": "linear", "factor": f}``: every frequency divided by f;
    * ``{"type": "ntk", "factor": f}``: the base times ``f ** (rot_dim / (rot_dim - 2))``, which
      keeps the fastest frequency and divides the slowest by f;
    * ``{"type": "yarn", "factor": f, "original_positions": n, "beta_fast": 32, "beta_slow": 1,
      "amplitude": a}``: frequencies that turn more than beta_fast times over the n original
      positions are kept, those below beta_slow turns divided by f, with a linear ramp between;
      cos and sin times a (default ``0.1 ln f + 1``).
    """
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError(f"rot_dim must be even and positive, got {rot_dim}")
    if positions < 1:
        raise ValueError(f"positions must be positive, got {positions}")
    if not base > 1.0:
        raise ValueError(f"base must be above 1, got {base}")
    i = torch.arange(rot_dim // 2, dtype=torch.float64, device=device)
    amplitude = 1.0
    kind = "none" if scaling is None else scaling.get("type")
    if kind not in ("none", "linear", "ntk", "yarn"):
        raise ValueError(f"unknown scaling type {kind!r}")
    factor = 1.0 if kind == "none" else float(scaling["factor"])
    if not (factor >= 1.0 and math.isfinite(factor)):
        raise ValueError(f"scaling factor must be at least 1, got {factor}")
    if kind == "ntk":
        if rot_dim == 2:
            raise ValueError("ntk scaling needs a rot_dim above 2")
        base = base * factor ** (rot_dim / (rot_dim - 2))
    freq = base ** (-2.0 * i / rot_dim)
    if kind == "linear":
        freq = freq / factor
    elif kind == "yarn":
        original = float(scaling["original_positions"])
        if not original > 0:
            raise ValueError(f"original_positions must be positive, got {original}")
        fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))
        # The index whose frequency turns `turns` times over the original positions.
        index = lambda turns: rot_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(math.floor(index(fast)), 0), min(math.ceil(index(slow)), rot_dim - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        freq = freq / factor * ramp + freq * (1 - ramp)
        amplitude = float(scaling.get("amplitude", 0.1 * math.log(factor) + 1.0))
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq
    return torch.stack((angle.cos() * amplitude, angle.sin() * amplitude), dim=-1).to(torch.float32).contiguous()


def _table(table: Optional[torch.Tensor], dim: int, layout: str) -> Tuple[int, int, int, int]:
    code = _layout_code(layout)
    if table is None:
        return 0, 0, 0, code
    shape = table.shape
    assert len(shape) == 3 and shape[2] == 2 and table.dtype is torch.float32 and table.is_contiguous(), \
        "table must be a contiguous float32 [positions, rot_dim / 2, 2] (rotary_table)"
    rot = 2 * shape[1]
    assert rot <= dim, f"the table rotates {rot} elements of a head of {dim}"
    return table.data_ptr(), shape[0], rot, code


def _positions(positions: torch.Tensor, batch: int, seq: int, rank: int) -> Tuple[int, int, int]:
    dtype, shape, st = positions.dtype, positions.shape, positions.stride()
    assert dtype is torch.int64 or dtype is torch.int32, "positions must be int32 or int64"
    if len(shape) == 1:
        assert shape[0] == seq, f"positions must be [{seq}], got {tuple(shape)}"
        stride = 0
    else:
        assert rank == 4 and shape == (batch, seq), f"positions must be [{seq}] or [{batch}, {seq}], got {tuple(shape)}"
        stride = st[0]
    assert st[-1] == 1 or seq <= 1, "positions need a unit inner stride"
    return positions.data_ptr(), 8 if dtype is torch.int64 else 4, stride


def rotary(X: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, layout: str = "half",
           inverse: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotate the heads of X, [B, H, S, D] or [tokens, H, D] (any strides, unit inner one).

    The pair (a, b) of frequency i becomes ``(a cos - b sin, b cos + a sin)`` with (cos, sin)
    = ``table[position, i]``: elements (i, i + rot/2) in the "half" layout, (2i, 2i + 1) in the
    "interleaved" one; elements from rot on pass through. fp32 arithmetic, one rounding.
    ``positions`` int32 or int64, [S] or [B, S] ([tokens] for a 3-D X). ``out`` may be X.
    ``inverse`` turns back (the gradient). A position outside the table records a device
    error and its row is zero-filled."""
    x, sizes = _rows(X, "X")
    rot = _table(table, sizes[3], layout)
    assert table is not None, "rotary needs a table"
    pos = _positions(positions, sizes[0], sizes[2], X.dim())
    code = _dtype_code(X)
    device = _check_device(X, positions, table, out)
    out, y = _output(out, X, "out")
    _call("lunarad_rotary", _ROTARY.pack(*x, *y, *pos, *rot, *sizes, 1 if inverse else 0, code), device)
    return out


def _weight(w: Optional[torch.Tensor], like: torch.Tensor, dim: int, name: str) -> int:
    if w is None:
        return 0
    assert w.dim() == 1 and w.numel() == dim and w.dtype is like.dtype and w.is_contiguous(), f"{name} must be [{dim}] {like.dtype}, contiguous"
    return w.data_ptr()


def qk_norm_rotary(Q: torch.Tensor, K: torch.Tensor, positions: torch.Tensor, table: Optional[torch.Tensor],
                   q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                   layout: str = "half", out_q: Optional[torch.Tensor] = None,
                   out_k: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Normalise every head of Q and K, ``x / sqrt(mean(x^2) + eps) * weight``, and rotate it, in
    one launch. Q [B, Hq, S, D] and K [B, Hk, S, D], or [tokens, H, D], any strides (views of a
    fused projection); weights [D] or None; ``table=None`` normalises only. Statistics and
    rotation in fp32, one rounding. Outputs may be the inputs."""
    q, (batch, q_heads, seq, dim) = _rows(Q, "Q")
    k, (kb, k_heads, ks, kd) = _rows(K, "K")
    rank = Q.dim()
    assert kb == batch and ks == seq and kd == dim and K.dim() == rank, "Q and K must agree in batch, positions and head dim"
    assert Q.dtype is K.dtype, "Q and K must share a dtype"
    rot = _table(table, dim, layout)
    pos = _positions(positions, batch, seq, rank)
    code = _dtype_code(Q)
    device = _check_device(Q, K, positions, table, q_weight, k_weight, out_q, out_k)
    wq, wk = _weight(q_weight, Q, dim, "q_weight"), _weight(k_weight, Q, dim, "k_weight")
    out_q, oq = _output(out_q, Q, "out_q")
    out_k, ok = _output(out_k, K, "out_k")
    _call("lunarad_qk_norm_rotary", _QK_NORM.pack(*q, *k, *oq, *ok, wq, wk, *pos, *rot, batch, q_heads, k_heads, seq, dim, code,
                                                  eps), device)
    return out_q, out_k


# ─────────────────────────────────────────────────── paged cache ──

def _sequences(page_table: torch.Tensor, seq_starts: torch.Tensor, seq_lens: torch.Tensor, tokens: int) -> Tuple[int, ...]:
    shape, stride = page_table.shape, page_table.stride()
    batch = seq_lens.numel()
    assert len(shape) == 2 and shape[0] == batch and seq_lens.dim() == 1, "page_table must be [batch, max_pages] and seq_lens [batch]"
    assert seq_starts.dim() == 1 and seq_starts.numel() == batch + 1, f"seq_starts must be [{batch + 1}], got {tuple(seq_starts.shape)}"
    i32 = torch.int32
    assert page_table.dtype is i32 and seq_starts.dtype is i32 and seq_lens.dtype is i32, "page_table, seq_starts and seq_lens must be int32"
    assert (stride[1] == 1 or shape[1] <= 1) and seq_lens.is_contiguous() and seq_starts.is_contiguous(), \
        "page_table, seq_starts and seq_lens need a unit inner stride"
    return page_table.data_ptr(), seq_starts.data_ptr(), seq_lens.data_ptr(), stride[0], shape[1], batch, tokens


def kv_append(K: torch.Tensor, V: torch.Tensor, cache: PagedKVCache, page_table: torch.Tensor, seq_starts: torch.Tensor,
              seq_lens: torch.Tensor, table: Optional[torch.Tensor] = None, layout: str = "half",
              Q: Optional[torch.Tensor] = None, out_q: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Write the new tokens' K and V, [tokens, kv_heads, D] (any strides), to their pages, K
    rotated at its position when a ``table`` is given. With Q [tokens, q_heads, D] the queries
    are rotated in the same launch into ``out_q`` (which may be Q) and returned. ``seq_lens``
    count the new tokens. A 4-bit cache gets the e2m1 codes and e4m3 scales of the values times
    ``1 / gain``. Two tokens of one call must not share a slot (sequences may share pages that
    nobody writes to)."""
    k, (_, heads, tokens, dim) = _rows(K, "K")
    v, v_sizes = _rows(V, "V")
    assert K.dim() == 3 and V.dim() == 3 and heads == cache.kv_heads and dim == cache.head_dim and v_sizes == (1, heads, tokens, dim), \
        f"K and V must be [tokens, {cache.kv_heads}, {cache.head_dim}], got {tuple(K.shape)} and {tuple(V.shape)}"
    dtype = K.dtype
    assert V.dtype is dtype and (cache.dtype is None or dtype is cache.dtype), "K, V and the cache must share a dtype"
    rot = _table(table, dim, layout)
    code = _dtype_code(K)
    q_heads, q, o = 0, (0, 0, 0, 0), (0, 0, 0, 0)
    if Q is not None:
        q, (_, q_heads, q_tokens, q_dim) = _rows(Q, "Q")
        assert Q.dim() == 3 and q_tokens == tokens and q_dim == dim and Q.dtype is dtype, f"Q must be [{tokens}, q_heads, {dim}] {dtype}"
    else:
        assert out_q is None, "out_q without Q"
    seqs = _sequences(page_table, seq_starts, seq_lens, tokens)
    device = _check_device(cache.k_pages, K, V, table, Q, out_q, page_table, seq_starts, seq_lens)
    rest = 0
    if Q is not None:
        fresh = out_q is None
        out_q, o = _output(out_q, Q, "out_q")
        if fresh:
            rest = _zero_rest(out_q, seqs[5])
    _call("lunarad_kv_append", _APPEND.pack(*k, *v, *q, *o, cache._address, *seqs, *rot, q_heads, code | rest), device)
    return out_q


def kv_read(cache: PagedKVCache, page_table: torch.Tensor, seq_starts: torch.Tensor, seq_lens: torch.Tensor, tokens: int,
            dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of the last ``seq_starts[b + 1] - seq_starts[b]`` positions of each
    sequence as dense [tokens, kv_heads, D] tensors, in the cache's dtype (``dtype``, float16 by
    default, for a 4-bit one); zeros where a token is padding or no sequence's."""
    if dtype is None:
        dtype = torch.float16 if cache.dtype is None else cache.dtype
    assert cache.dtype is None or dtype == cache.dtype, f"a {cache.dtype} cache is read as such, not as {dtype}"
    assert tokens >= 0, "tokens must not be negative"
    seqs = _sequences(page_table, seq_starts, seq_lens, tokens)
    device = _check_device(cache.k_pages, page_table, seq_starts, seq_lens)
    k = cache.k_pages.new_empty((tokens, cache.kv_heads, cache.head_dim), dtype=dtype)
    v = torch.empty_like(k)
    code = _dtype_code(k) | _zero_rest(k, seqs[5]) | _zero_rest(v, seqs[5])
    _call("lunarad_kv_read", _READ.pack(k.data_ptr(), v.data_ptr(), cache._address, *seqs, code), device)
    return k, v


def paged_attention(Q: torch.Tensor, cache: PagedKVCache, page_table: torch.Tensor, seq_starts: torch.Tensor,
                    seq_lens: torch.Tensor, scale: Optional[float] = None, window: int = 0,
                    max_q_len: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(Q K^T * scale) V over the cached keys, for Q [tokens, q_heads, D] (any strides).

    A token at position p sees the keys 0..p of its sequence, with ``window`` > 0 the last
    ``window`` of them; its own key and value must be in the cache (``kv_append`` first). Query
    head h reads key head ``h // (q_heads // kv_heads)``. ``scale`` defaults to ``1 / sqrt(D)``.
    fp32 softmax; a row that sees no key is zero, one with a score of +inf or NaN is NaN. Slots
    that no token sees may hold anything; a value that is not finite may reach the other tokens
    of its sequence in the call. ``max_q_len``, the most tokens any sequence has here, is a hint
    that steers the choice of kernels (default: any number). ``out`` may be Q."""
    q, (_, q_heads, tokens, dim) = _rows(Q, "Q")
    assert Q.dim() == 3 and dim == cache.head_dim, f"Q must be [tokens, q_heads, {cache.head_dim}], got {tuple(Q.shape)}"
    assert cache.dtype is None or Q.dtype is cache.dtype, "Q and the cache must share a dtype"
    assert q_heads > 0 and q_heads % cache.kv_heads == 0, f"{q_heads} query heads are no multiple of {cache.kv_heads} key heads"
    code = _dtype_code(Q)
    seqs = _sequences(page_table, seq_starts, seq_lens, tokens)
    device = _check_device(cache.k_pages, Q, out, page_table, seq_starts, seq_lens)
    fresh = out is None
    out, o = _output(out, Q, "out")
    rest = _zero_rest(out, seqs[5]) if fresh else 0
    if scale is None:
        scale = dim ** -0.5
    args = _ATTENTION.pack(*q, *o, cache._address, *seqs, q_heads, window, max_q_len or 0, code | rest, scale)
    need = _lib.load().lunarad_paged_attention_workspace(args, device)
    if need < 0:
        _lib.check(-need)
    workspace = Q.new_empty((need + 1) // 2 if code != _lib.F32 else (need + 3) // 4) if need else None
    _call("lunarad_paged_attention", args, device, workspace.data_ptr() if need else None, need)
    return out
