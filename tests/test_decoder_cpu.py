"""The decoder operators on CPU: the argument structs' layout, refusals by the C ABI and by the
torch layer (before any device is touched), and the rotary table's formulas."""
import math
import shutil
import struct
import subprocess
from pathlib import Path

import pytest
import torch

from lunara_b200.runtime import _lib, decoder, kv_cache, ops
from oracle import decoder as ref

HEADER = Path(__file__).resolve().parents[1] / "include" / "lunara_b200_decoder.h"

STRUCTS = {"lunarad_rotary_args": decoder._ROTARY, "lunarad_qk_norm_rotary_args": decoder._QK_NORM,
           "lunarad_kv_append_args": decoder._APPEND, "lunarad_kv_read_args": decoder._READ,
           "lunarad_paged_attention_args": decoder._ATTENTION, "lunarad_cache": kv_cache._CACHE}


def test_library_exports_the_header():
    import re
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(lunarad_\w+)\s*\(", text)))
    assert declared == sorted(_lib.DECODER_SIGNATURES)
    lib = _lib.load()
    for name in declared:
        assert hasattr(lib, name), name


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_struct_layout(tmp_path):
    src = tmp_path / "sizes.c"
    src.write_text(f'#include <stdio.h>\n#include "{HEADER}"\nint main(void) {{\n' +
                   "".join(f'printf("%zu\\n", sizeof({n}));\n' for n in STRUCTS) + "return 0; }\n")
    subprocess.run(["gcc", str(src), "-o", str(tmp_path / "sizes")], check=True)
    out = subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(x) for x in out] == [s.size for s in STRUCTS.values()]


def err():
    return _lib.load().lunara_last_error_string().decode()


def cache(kind=_lib.F16, dim=64, page=16, heads=2, pages=4, scales=16, gain=1.0, ptr=16, page_stride=1 << 14):
    packed = kv_cache._CACHE.pack(ptr, ptr, scales, scales, page_stride, 1 << 10, page_stride, 1 << 10, 256, 128, 256, 128, pages,
                                  heads, page, dim, kind, gain, 1.0)
    cache.keep = packed
    return _lib.address_of(packed)


VIEW = (16, 4096, 64, 256)
SEQS = (16, 16, 16, 8, 8, 2, 5)
TABLE = (16, 100, 64, 0)


def rotary(x=VIEW, y=VIEW, pos=(16, 8, 0), table=TABLE, shape=(2, 3, 4, 64), inverse=0, dtype=0):
    return _lib.load().lunarad_rotary(decoder._ROTARY.pack(*x, *y, *pos, *table, *shape, inverse, dtype), None)


def qk_norm(table=TABLE, shape=(2, 4, 2, 4, 64), dtype=0, eps=1e-6, weights=(0, 0), k=VIEW):
    return _lib.load().lunarad_qk_norm_rotary(
        decoder._QK_NORM.pack(*VIEW, *k, *VIEW, *k, *weights, 16, 8, 0, *table, *shape, dtype, eps), None)


def append(c=None, seqs=SEQS, table=TABLE, q_heads=0, dtype=0, k=VIEW, q=VIEW):
    return _lib.load().lunarad_kv_append(
        decoder._APPEND.pack(*k, *VIEW, *q, *q, cache() if c is None else c, *seqs, *table, q_heads, dtype), None)


def read(c=None, seqs=SEQS, dtype=0, out=16):
    return _lib.load().lunarad_kv_read(decoder._READ.pack(out, out, cache() if c is None else c, *seqs, dtype), None)


def attention(c=None, seqs=SEQS, q_heads=4, window=0, max_q=0, dtype=0, scale=0.1, q=VIEW):
    return _lib.load().lunarad_paged_attention(
        decoder._ATTENTION.pack(*q, *VIEW, cache() if c is None else c, *seqs, q_heads, window, max_q, dtype, scale), None, 0, None)


@pytest.mark.parametrize("call,needle", [
    (lambda: rotary(dtype=7), "dtype"), (lambda: rotary(shape=(-1, 3, 4, 64)), "negative"),
    (lambda: rotary(shape=(1 << 20, 3, 1 << 20, 64)), "2^30"), (lambda: rotary(shape=(2, 70000, 4, 64)), "65535"),
    (lambda: rotary(table=(16, 100, 66, 0)), "rot 66"), (lambda: rotary(table=(16, 100, 3, 0)), "rot 3"),
    (lambda: rotary(table=(16, 100, 64, 2)), "layout"), (lambda: rotary(table=(0, 100, 64, 0)), "empty"),
    (lambda: rotary(table=(16, 0, 64, 0)), "empty"), (lambda: rotary(table=(8, 100, 64, 0)), "aligned"),
    (lambda: rotary(pos=(0, 8, 0)), "positions"), (lambda: rotary(pos=(16, 2, 0)), "position_bytes"),
    (lambda: rotary(pos=(20, 8, 0)), "aligned"), (lambda: rotary(x=(0, 1, 1, 1)), "X is NULL"),
    (lambda: rotary(y=(17, 1, 1, 1)), "Y is not aligned"),
    (lambda: qk_norm(eps=-1.0), "eps"), (lambda: qk_norm(eps=math.nan), "eps"), (lambda: qk_norm(k=(0, 1, 1, 1)), "K is NULL"),
    (lambda: qk_norm(shape=(2, 40000, 40000, 4, 64)), "65535"), (lambda: qk_norm(weights=(17, 0)), "weights"),
    (lambda: append(c=0), "cache is NULL"), (lambda: append(c=cache(kind=9)), "kind"), (lambda: append(c=cache(kind=1)), "differ"),
    (lambda: append(c=cache(page=0)), "shape"), (lambda: append(c=cache(page=1 << 21)), "too large"),
    (lambda: append(c=cache(ptr=0)), "NULL"), (lambda: append(c=cache(kind=16, dim=72)), "multiple of 16"),
    (lambda: append(c=cache(kind=16, scales=0)), "scales"), (lambda: append(c=cache(kind=16, ptr=20)), "8-byte"),
    (lambda: append(c=cache(kind=16, page_stride=12)), "8-byte"), (lambda: append(c=cache(kind=16, gain=0.0)), "gains"),
    (lambda: append(c=cache(kind=16, gain=math.inf)), "gains"), (lambda: append(c=cache(kind=16, gain=1e-40)), "gains"),
    (lambda: append(c=cache(kind=16, dim=1024)), "512"), (lambda: append(c=cache(ptr=17)), "aligned"),
    (lambda: append(seqs=(16, 0, 16, 8, 8, 2, 5)), "NULL"), (lambda: append(seqs=(16, 18, 16, 8, 8, 2, 5)), "aligned"),
    (lambda: append(seqs=(16, 16, 16, 4, 8, 2, 5)), "overlap"), (lambda: append(seqs=(16, 16, 16, 8, 8, -2, 5)), "negative"),
    (lambda: append(seqs=(16, 16, 16, 8, 8, 2, 1 << 31)), "2^30"), (lambda: append(q_heads=-1), "q_heads"),
    (lambda: append(q_heads=4, q=(0, 1, 1, 1)), "Q is NULL"), (lambda: append(k=(0, 1, 1, 1)), "K is NULL"),
    (lambda: read(dtype=1), "differ"), (lambda: read(out=0), "NULL"), (lambda: read(out=17), "aligned"),
    (lambda: attention(q_heads=3), "multiple"), (lambda: attention(q_heads=0), "multiple"), (lambda: attention(dtype=1), "differ"),
    (lambda: attention(seqs=(16, 16, 16, 8, 8, 2, 1 << 30)), "2^31"), (lambda: attention(c=cache(dim=512)), "256"), (lambda: attention(window=-1), "window"),
    (lambda: attention(max_q=-1), "max_q_len"), (lambda: attention(scale=math.inf), "finite"),
    (lambda: attention(seqs=(16, 16, 16, 1 << 29, 1 << 29, 2, 5)), "2^31"), (lambda: attention(q=(0, 1, 1, 1)), "Q is NULL"),
])
def test_refused_by_the_library(call, needle):
    assert call() in (_lib.ERR_INVALID_ARG, _lib.ERR_UNSUPPORTED)
    assert needle in err(), err()


def test_empty_work_is_ok_without_device():
    assert rotary(shape=(0, 3, 4, 64), x=(0, 0, 0, 0)) == _lib.OK
    assert qk_norm(shape=(2, 4, 2, 0, 64)) == _lib.OK
    empty = (0, 0, 0, 8, 8, 0, 5)
    assert append(seqs=empty) == read(seqs=empty) == attention(seqs=empty) == _lib.OK
    assert attention(seqs=(16, 16, 16, 8, 8, 2, 0)) == _lib.OK


def test_workspace_refuses_like_the_call():
    lib = _lib.load()
    bad = decoder._ATTENTION.pack(*VIEW, *VIEW, cache(), *SEQS, 3, 0, 0, 0, 0.1)
    assert lib.lunarad_paged_attention_workspace(bad, 0) == -_lib.ERR_INVALID_ARG
    good = decoder._ATTENTION.pack(*VIEW, *VIEW, cache(), *SEQS, 4, 0, 0, 0, 0.1)
    assert lib.lunarad_paged_attention_workspace(good, 0) > 0
    assert lib.lunarad_paged_attention(good, None, 0, None) == _lib.ERR_INVALID_ARG and "workspace" in err()


# ── the torch layer ──────────────────────────────────────────────────────────

I32 = torch.int32


def pages(**kw):
    return ops.PagedKVCache.allocate(4, 2, 8, 64, device="cpu", **kw)


def seqs(batch=2, tokens=3):
    return torch.zeros(batch, 2, dtype=I32), torch.zeros(batch + 1, dtype=I32), torch.zeros(batch, dtype=I32)


def test_cpu_tensors_refused():
    t = ops.rotary_table(8, 64, device="cpu")
    x, pos = torch.zeros(1, 2, 3, 64), torch.zeros(3, dtype=torch.int64)
    q = torch.zeros(3, 4, 64, dtype=torch.float16)
    kv = q[:, :2]
    for call in (lambda: ops.rotary(x, pos, t), lambda: ops.qk_norm_rotary(x, x, pos, t),
                 lambda: ops.kv_append(kv, kv, pages(), *seqs()), lambda: ops.kv_read(pages(), *seqs(), tokens=3),
                 lambda: ops.paged_attention(q, pages(), *seqs())):
        with pytest.raises(AssertionError, match="CUDA"):
            call()


@pytest.mark.parametrize("call,needle", [
    (lambda x, pos, t: ops.rotary(x[0, 0], pos, t), "must be"),
    (lambda x, pos, t: ops.rotary(x.transpose(2, 3), pos, t), "unit"),
    (lambda x, pos, t: ops.rotary(x, pos.float(), t), "int32 or int64"),
    (lambda x, pos, t: ops.rotary(x, pos[:2], t), "positions must be"),
    (lambda x, pos, t: ops.rotary(x[..., :32], pos, t), "head of 32"),
    (lambda x, pos, t: ops.rotary(x, pos, t.double()), "float32"),
    (lambda x, pos, t: ops.rotary(x, pos, None), "table"),
    (lambda x, pos, t: ops.qk_norm_rotary(x, x[:, :, :2], pos, t), "agree"),
    (lambda x, pos, t: ops.qk_norm_rotary(x, x.half(), pos, t), "dtype"),
])
def test_shapes_refused(call, needle):
    with pytest.raises(AssertionError, match=needle):
        call(torch.zeros(1, 2, 3, 64), torch.zeros(3, dtype=torch.int64), ops.rotary_table(8, 64, device="cpu"))


def test_values_refused():
    x, pos, t = torch.zeros(1, 2, 3, 64), torch.zeros(3, dtype=torch.int64), ops.rotary_table(8, 64, device="cpu")
    with pytest.raises(ValueError, match="layout"):
        ops.rotary(x, pos, t, layout="pairs")
    with pytest.raises(TypeError, match="dtype"):
        ops.rotary(x.double(), pos, t)
    for bad in (dict(rot_dim=3), dict(rot_dim=0), dict(positions=0), dict(base=1.0), dict(scaling={"type": "other", "factor": 2}),
                dict(scaling={"type": "linear", "factor": 0.5}), dict(scaling={"type": "ntk", "factor": 2.0}, rot_dim=2),
                dict(scaling={"type": "yarn", "factor": 2.0, "original_positions": 0})):
        with pytest.raises(ValueError):
            ops.rotary_table(**{"positions": 8, "rot_dim": 64, "device": "cpu", **bad})


def test_caches_refused():
    z = lambda *s, dtype=torch.float16: torch.zeros(*s, dtype=dtype)  # noqa: E731
    u8 = torch.uint8
    for bad in (lambda: ops.PagedKVCache(z(4, 2, 8, 64), z(4, 2, 8, 32)), lambda: ops.PagedKVCache(z(4, 2, 64), z(4, 2, 64)),
                lambda: ops.PagedKVCache(z(4, 8, 2, 64).transpose(1, 2), z(4, 8, 2, 64).transpose(1, 2)),
                lambda: ops.PagedKVCache(z(4, 2, 8, 32, dtype=u8), z(4, 2, 8, 32, dtype=u8)),
                lambda: ops.PagedKVCache(z(4, 2, 8, 20, dtype=u8), z(4, 2, 8, 20, dtype=u8), z(4, 2, 8, 2, dtype=u8), z(4, 2, 8, 2, dtype=u8)),
                lambda: ops.PagedKVCache(*(z(4, 2, 8, 32, dtype=u8),) * 2, *(z(4, 2, 8, 4),) * 2),
                lambda: ops.PagedKVCache(*(z(4, 2, 8, 32, dtype=u8),) * 2, *(z(4, 2, 8, 3, dtype=u8),) * 2),
                lambda: ops.PagedKVCache(z(4, 2, 8, 64), z(4, 2, 8, 64), z(4, 2, 8, 4, dtype=u8), z(4, 2, 8, 4, dtype=u8)),
                lambda: ops.PagedKVCache.allocate(4, 2, 8, 40, dtype="e2m1", device="cpu")):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(TypeError):
        ops.PagedKVCache(z(4, 2, 8, 64, dtype=torch.float64), z(4, 2, 8, 64, dtype=torch.float64))
    for gain in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="gain"):
            ops.PagedKVCache.allocate(4, 2, 8, 64, dtype="e2m1", device="cpu", k_gain=gain)
    with pytest.raises(ValueError, match="gain"):
        pages(k_gain=2.0)


@pytest.mark.parametrize("change,needle", [
    (lambda a: a[0].long(), "int32"), (lambda a: a[0][0], "page_table"), (lambda a: a[0].repeat(1, 2)[:, ::2], "unit"),
    (lambda a: a[0][:1], "page_table"),
])
def test_page_tables_refused(change, needle):
    tab, starts, lens = seqs()
    q = torch.zeros(3, 4, 64, dtype=torch.float16)
    with pytest.raises(AssertionError, match=needle):
        decoder._sequences(change((tab,)), starts, lens, 3)
    with pytest.raises(AssertionError, match="seq_starts"):
        decoder._sequences(tab, starts[:-1], lens, 3)
    with pytest.raises(AssertionError, match="multiple"):
        ops.paged_attention(q[:, :3], pages(), tab, starts, lens)
    with pytest.raises(AssertionError, match="must be"):
        ops.paged_attention(q[..., :32], pages(), tab, starts, lens)
    with pytest.raises(AssertionError, match="dtype"):
        ops.kv_append(q[:, :2].float(), q[:, :2].float(), pages(), tab, starts, lens)
    with pytest.raises(AssertionError, match="read as such"):
        ops.kv_read(pages(), tab, starts, lens, tokens=3, dtype=torch.float32)


def test_expanded_outputs_refused():
    with pytest.raises(AssertionError, match="expanded"):
        decoder._output(torch.zeros(1, 1, 64).expand(3, 2, 64), torch.zeros(3, 2, 64), "out")


# ── the rotary table ─────────────────────────────────────────────────────────

def frequencies(table):
    """Angle of position 1 of each frequency."""
    return torch.atan2(table[1, :, 1].double(), table[1, :, 0].double())


def test_table_far_positions():
    t = ops.rotary_table(200001, 64, device="cpu")
    for pos in (0, 1, 777, 200000):
        for i in (0, 5, 31):
            a = pos * 10000.0 ** (-2 * i / 64)
            assert abs(float(t[pos, i, 0]) - math.cos(a)) <= 2.0 ** -24 + 1e-10
            assert abs(float(t[pos, i, 1]) - math.sin(a)) <= 2.0 ** -24 + 1e-10


def test_table_scalings():
    plain = frequencies(ops.rotary_table(2, 64, device="cpu"))
    close = lambda a, b: torch.allclose(a, b, rtol=2e-7, atol=1e-12)  # noqa: E731  (float32 entries)
    linear = frequencies(ops.rotary_table(2, 64, device="cpu", scaling={"type": "linear", "factor": 4.0}))
    assert close(linear, plain / 4)
    ntk = frequencies(ops.rotary_table(2, 64, device="cpu", scaling={"type": "ntk", "factor": 4.0}))
    assert close(ntk[0], plain[0]) and close(ntk[-1], plain[-1] / 4)
    scaling = {"type": "yarn", "factor": 8.0, "original_positions": 2048}
    table = ops.rotary_table(2, 64, device="cpu", scaling=scaling)
    yarn = frequencies(table)
    turns = 2048 * plain / (2 * math.pi)
    assert close(yarn[turns > 40], plain[turns > 40]) and close(yarn[turns < 0.7], plain[turns < 0.7] / 8)
    mid = (turns < 20) & (turns > 2)
    assert ((yarn[mid] < plain[mid]) & (yarn[mid] > plain[mid] / 8)).all()
    assert float(table[0, 0, 0]) == pytest.approx(0.1 * math.log(8.0) + 1, rel=1e-7)
    assert float(ops.rotary_table(2, 64, device="cpu", scaling={**scaling, "amplitude": 1.0})[0, 0, 0]) == 1.0


# ── the 4-bit definition itself ──────────────────────────────────────────────

def test_quantise_definition():
    """Nearest e2m1 value with ties to the even code, by search over all sixteen values."""
    z = torch.cat((torch.linspace(-7, 7, 2801), torch.tensor([.25, .75, 1.25, 1.75, 2.5, 3.5, 5.0])))
    z = torch.nn.functional.pad(z, (0, (-len(z)) % 15)).view(-1, 15)
    x = torch.cat((torch.full((len(z), 1), 6.0), z.clamp(-6, 6)), 1)   # amax 6: the scale is 1
    codes, scales = ref.quantise(x, 1.0)
    assert (scales == 0x38).all()
    got = ref.values(codes, scales, 1.0)
    dist = (x.double()[..., None] - torch.cat((ref.E2M1, -ref.E2M1)).double()).abs()
    assert torch.equal((got - x).abs(), dist.amin(-1))
    tie = (dist == dist.amin(-1, keepdim=True)).sum(-1) == 2
    tie &= x != 0
    assert tie.any() and (codes[tie] % 2 == 0).all()


def test_pack_order():
    assert ref.pack(torch.tensor([1, 2, 3, 4], dtype=torch.uint8)).tolist() == [0x21, 0x43]
    assert ref.unpack(torch.tensor([0x21, 0x43], dtype=torch.uint8)).tolist() == [1, 2, 3, 4]
    assert struct.calcsize("q") == 8
