"""More of the decoder operators on CPU: flags and refusals of the C ABI, the cache handle, the oracle's
bounds."""
import copy
import ctypes
import math
import pickle

import pytest
import torch

from lunara_b200.runtime import _lib, decoder, kv_cache, ops
from oracle import decoder as ref
from test_decoder_cpu import SEQS, VIEW, append, attention, cache, err, qk_norm, read, rotary


def test_zero_rest_is_a_flag_of_the_ragged_calls():
    flag = _lib.ZERO_REST
    for call in (append, read, attention):
        assert call(seqs=(16, 16, 16, 8, 8, 2, 0), dtype=flag) == _lib.OK
        assert call(seqs=(0, 0, 0, 8, 8, 0, 5), dtype=flag) == _lib.ERR_INVALID_ARG and "no sequence" in err()
        assert call(dtype=flag | 7) == _lib.ERR_INVALID_ARG and "dtype" in err()
        assert call(dtype=flag << 1) == _lib.ERR_INVALID_ARG and "dtype" in err()
        assert call(dtype=flag | _lib.BF16) == _lib.ERR_INVALID_ARG and "differ" in err()
    for call in (rotary, qk_norm):
        assert call(dtype=flag) == _lib.ERR_INVALID_ARG and "dtype" in err()
    c = cache()
    packed = [decoder._ATTENTION.pack(*VIEW, *VIEW, c, *SEQS, 4, 0, 0, f, 0.1) for f in (0, flag)]
    lib = _lib.load()
    assert lib.lunarad_paged_attention_workspace(packed[0], 0) == lib.lunarad_paged_attention_workspace(packed[1], 0) > 0


def test_null_arguments_refused():
    lib = _lib.load()
    for call in (lib.lunarad_rotary, lib.lunarad_qk_norm_rotary, lib.lunarad_kv_append, lib.lunarad_kv_read):
        assert call(None, None) == _lib.ERR_INVALID_ARG and "NULL" in err()
    assert lib.lunarad_paged_attention(None, None, 0, None) == _lib.ERR_INVALID_ARG and "NULL" in err()
    assert lib.lunarad_paged_attention_workspace(None, 0) == -_lib.ERR_INVALID_ARG and "NULL" in err()


def test_cache_handles_cannot_be_changed():
    """The kernels get packed addresses: another tensor in an attribute would be ignored, and the old one's memory freed."""
    for kind in (torch.float16, "e2m1"):
        c = ops.PagedKVCache.allocate(4, 2, 8, 64, dtype=kind, device="cpu")
        pages = c.k_pages
        for name in ("k_pages", "v_pages", "k_scales", "v_scales", "k_gain", "num_pages", "page_size", "head_dim", "dtype", "other"):
            with pytest.raises(AttributeError, match="new one"):
                setattr(c, name, torch.zeros(8, 2, 8, 64))
        with pytest.raises(AttributeError):
            del c.k_pages
        assert c.k_pages is pages and c.num_pages == 4


@pytest.mark.parametrize("kind", [torch.float32, "e2m1"])
def test_copies_of_cache_handles_have_their_own_addresses(kind):
    """A deep copy, and a handle that was pickled, point at their own tensors; a shallow one shares them."""
    c = ops.PagedKVCache.allocate(4, 2, 8, 64, dtype=kind, device="cpu")
    if kind == "e2m1":   # scales as bytes: torch does not load float8 tensors from a plain pickle
        c = ops.PagedKVCache(c.k_pages, c.v_pages, c.k_scales.view(torch.uint8), c.v_scales.view(torch.uint8), k_gain=0.5, v_gain=3.0)
    c.k_pages.random_(0, 200)
    shallow = copy.copy(c)
    assert shallow.k_pages is c.k_pages and shallow._args == c._args
    for other in (copy.deepcopy(c), pickle.loads(pickle.dumps(c))):
        assert torch.equal(other.k_pages, c.k_pages) and other.k_pages.data_ptr() != c.k_pages.data_ptr()
        fields = kv_cache._CACHE.unpack(other._args)
        tensors = (other.k_pages, other.v_pages) + ((other.k_scales, other.v_scales) if kind == "e2m1" else ())
        assert fields[:len(tensors)] == tuple(t.data_ptr() for t in tensors)
        assert fields[4:] == kv_cache._CACHE.unpack(c._args)[4:]
        assert ctypes.string_at(other._address, len(other._args)) == other._args


@pytest.mark.parametrize("scale", [0.3, -0.3])
def test_the_oracles_reach_bounds_every_score(scale):
    """`reach`, from which the attention's tolerance takes the scores' rounding, is scale's magnitude times sum |q||k|, whatever its sign."""
    g = torch.Generator().manual_seed(1)
    q, k = torch.randn(3, 2, 16, generator=g), torch.randn(7, 1, 16, generator=g)
    reach = ref.attend(q, k, k, 4, scale)[2]
    for i in range(3):
        for h in range(2):
            sums = [float((q[i, h].double().abs() * k[j, 0].double().abs()).sum()) for j in range(4 + i + 1)]
            assert float(reach[i, h]) == pytest.approx(0.3 * max(sums), rel=1e-12)


@pytest.mark.parametrize("scale,gain,ok", [(1e39, 1.0, False), (-1e300, 1.0, False), (3e38, 1.0, False), (1e30, 1e10, False), (2e38, 1.0, True),
                                           (1e39, 0.1, True), (1e-300, 1.0, True), (0.0, 1.0, True)])
def test_scales_beyond_fp32_refused(scale, gain, ok):
    """Accepted ones get as far as the workspace that these calls lack."""
    for kind in (_lib.KIND_E2M1, _lib.F16) if gain == 1.0 else (_lib.KIND_E2M1,):
        assert attention(c=cache(kind=kind, gain=gain), scale=scale) == _lib.ERR_INVALID_ARG and ("workspace" if ok else "fp32") in err(), err()


@pytest.mark.parametrize("rot,base,original,factor,fast,slow", [(128, 10000.0, 4096, 16.0, 32.0, 1.0), (64, 500000.0, 8192, 8.0, 32.0, 1.0),
                                                                 (80, 10000.0, 2048, 4.0, 24.0, 2.0)])
def test_yarn_ramp(rot, base, original, factor, fast, slow):
    """Every frequency against the definition, by bisection instead of logarithms: frequency i turns
    original / (2 pi) * base^(-2 i / rot) times. Indices up to the last whole one with at least `fast` turns are kept, those from
    the first whole one with at most `slow` turns on are divided by the factor, a straight line lies between."""
    turns = lambda i: original / (2 * math.pi) * base ** (-2 * i / rot)  # noqa: E731
    low = max(i for i in range(rot) if turns(i) >= fast)
    high = min(i for i in range(rot) if turns(i) <= slow)
    assert 0 < low < high < rot // 2 + 8
    scaling = {"type": "yarn", "factor": factor, "original_positions": original, "beta_fast": fast, "beta_slow": slow, "amplitude": 1.0}
    t = ops.rotary_table(2, rot, base=base, scaling=scaling, device="cpu")
    got = torch.atan2(t[1, :, 1].double(), t[1, :, 0].double())
    seen = set()
    for i in range(rot // 2):
        f = base ** (-2 * i / rot)
        share = 0.0 if i <= low else 1.0 if i >= high else (i - low) / (high - low)
        seen.add(0 < share < 1)
        want = f * (1 - share) + f / factor * share
        # An entry is off by half a step: 2^-24 of it, 2^-25 at most (below 1); the angle by no more than both together.
        assert abs(float(got[i]) - want) <= 2.0 ** -24, i
        assert abs(float(t[1, i, 1]) - math.sin(want)) <= 2.0 ** -24 * abs(math.sin(want)) + 1e-15, i
    assert seen == {True, False}


def test_a_hint_beyond_the_tokens_counts_as_them():
    """The kernels that a hint chooses show in the workspace; the hint times the heads of a group passes 64 bits here."""
    c, lib = cache(), _lib.load()
    need = [lib.lunarad_paged_attention_workspace(decoder._ATTENTION.pack(*VIEW, *VIEW, c, 16, 16, 16, 8, 8, 2, 64, 8, 0, hint, 0, 0.1), 0)
            for hint in (64, 65, 1 << 62, (1 << 63) - 1, 1)]
    assert need[0] == need[1] == need[2] == need[3] > need[4] > 0
