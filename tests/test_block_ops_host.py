"""CPU checks of residual_norm, the 8-bit checkpoints, silu_mul, rotary and the 8-bit cache: what the C entry
points refuse before any launch (given made-up device addresses), scratch sizes, and what the Python
layer refuses.  No kernel runs."""
import ctypes
import os

import pytest
import torch

from vibetensor_b200 import _lib

P = 0x10000  # a made-up device address: never dereferenced, the calls below end before a launch
F32, I64, F16, BF16, I32 = _lib.F32, _lib.I64, _lib.F16, _lib.BF16, _lib.I32


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(_lib.LIB_PATH):
        from vibetensor_b200 import build
        build.build()
    return _lib.lib()


def refused(L, status, text):
    assert status == 1, status
    assert text in L.vbt_b200_last_error().decode(), L.vbt_b200_last_error()


def norm(L, r=P, n=P, x=P, y=P, gate=None, dtype=BF16, rows=4, cols=64, strides=(64, 64, 0), per=4, flags=3):
    return L.vbt_b200_residual_norm(r, n, P, P, x, y, P, gate, P, dtype, rows, cols, *strides, per, 1.0, 1.0, 1e-6, flags, None)


def test_residual_norm_refusals(L):
    refused(L, norm(L, rows=-1), "negative size")
    refused(L, norm(L, rows=1 << 36), "too many rows")
    refused(L, norm(L, dtype=I64), "floating dtype")
    for kw in (dict(x=None), dict(y=None), dict(r=None), dict(n=None)):
        refused(L, norm(L, **kw), "null pointer")
    refused(L, norm(L, strides=(-64, 64, 0)), "negative row stride")
    for per in (0, 3, -4):
        refused(L, norm(L, gate=P, per=per), "rows_per_gate")
    assert norm(L, rows=0, x=None) == 0 and norm(L, cols=0, x=None) == 0


def back(L, dx=P, dy=P, dgp=P, dgate=None, dgn=P, dr=P, dn=P, y=P, r=P, i1=P, i2=P, gate=None, dtype=BF16, rows=4, cols=64,
         stride=64, per=4, flags=3, ws=P, nbytes=1 << 40):
    return L.vbt_b200_residual_norm_backward(dx, dy, dgp, dgate, dgn, dr, dn, y, r, i1, i2, P, gate, P, dtype, rows, cols,
                                             stride, stride, stride, stride, 0, per, 1.0, 1.0, flags, ws, nbytes, None)


def test_residual_norm_backward_refusals(L):
    refused(L, back(L, cols=-1), "negative size")
    refused(L, back(L, dtype=I32), "floating dtype")
    refused(L, back(L, dgate=P), "dgate without a gate")
    refused(L, back(L, flags=2), "dgamma_post without")
    refused(L, back(L, flags=1), "dgamma_pre without")
    refused(L, back(L, gate=P, per=3), "rows_per_gate")
    refused(L, back(L, dx=None), "null pointer")
    refused(L, back(L, dn=None, dr=None, flags=0, dgp=None, dgn=None), "null pointer")
    for kw in (dict(dn=None), dict(r=None), dict(i2=None)):
        refused(L, back(L, **kw), "needs dn, r and inv_pre")
    for kw in (dict(y=None), dict(i1=None)):
        refused(L, back(L, **kw), "needs y and inv_post")
    refused(L, back(L, y=None, flags=2, dgp=None, gate=P, dgate=P), "dgate needs y")
    refused(L, back(L, stride=-1), "negative row stride")
    refused(L, back(L, nbytes=16), "workspace too small")
    refused(L, back(L, ws=None), "workspace too small")
    assert back(L, cols=0) == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scratch_covers_every_form(L, dtype):
    need = ctypes.c_size_t()
    f = L.vbt_b200_residual_norm_backward_workspace_bytes
    for rows, per, cols in ((1, 1, 1), (16, 16, 4096), (32768, 4096, 4096), (6151, 6151, 1365), (100000, 4, 128), (64, 1, 64),
                            (8192, 8192, 16384), (50, 25, 70001)):
        assert f(rows, cols, dtype, per, 0, ctypes.byref(need)) == 0
        # two rows of column sums at least, and a bound: no more partial rows than rows and card
        assert 8 * cols <= need.value <= 4 * cols * (2 * 148 * 4 * 8 + min(rows, 148 * 4 * 8 * 9) + 148 * 4 * 8)
    assert f(0, 64, dtype, 1, 0, ctypes.byref(need)) == 0 and need.value == 0
    refused(L, f(10, 64, dtype, 3, 0, ctypes.byref(need)), "rows_per_gate")
    refused(L, f(10, 64, dtype, 5, 0, None), "null output")
    g = L.vbt_b200_rmsnorm_backward8_workspace_bytes
    for rows, cols in ((1, 1), (32768, 4096), (5, 20001), (262144, 128)):
        assert g(rows, cols, dtype, 0, ctypes.byref(need)) == 0
        assert 4 * cols <= need.value <= 4 * cols * 148 * 8 * 8
    refused(L, g(1, 1, I64, 0, ctypes.byref(need)), "floating dtype")


def test_checkpoint_refusals(L):
    refused(L, L.vbt_b200_checkpoint8(P, P, P, BF16, 2, 4, 64, 64, None), "unknown 8-bit format")
    refused(L, L.vbt_b200_checkpoint8(P, P, P, I64, 0, 4, 64, 64, None), "floating dtype")
    refused(L, L.vbt_b200_checkpoint8(P, None, P, F32, 0, 4, 64, 64, None), "null pointer")
    refused(L, L.vbt_b200_checkpoint8(P, P, P, F32, 0, 4, 64, -64, None), "negative row stride")
    refused(L, L.vbt_b200_checkpoint8(P, P, P, F32, 0, 1 << 35, 64, 64, None), "too many groups")
    refused(L, L.vbt_b200_checkpoint8_restore(P, P, None, F32, 0, 4, 64, None), "null pointer")
    refused(L, L.vbt_b200_rmsnorm_checkpoint8(P, P, P, P, None, P, F32, 0, 4, 64, 64, 1e-6, None), "null pointer")
    refused(L, L.vbt_b200_rmsnorm_backward8(P, P, P, P, P, P, P, F32, 0, 4, 64, 64, P, 4, None), "workspace too small")
    refused(L, L.vbt_b200_rmsnorm_backward8(P, None, P, P, P, None, P, F32, 0, 4, 64, 64, None, 0, None), "null pointer")
    refused(L, L.vbt_b200_silu_mul(P, P, None, P, P, P, P, F32, 0, 4, 64, 64, 64, None), "all four outputs")
    refused(L, L.vbt_b200_silu_mul(P, None, None, None, None, P, None, F32, 0, 4, 64, 64, 64, None), "null pointer")
    refused(L, L.vbt_b200_silu_mul_backward(P, P, P, P, P, P, None, F32, 0, 4, 64, 64, 64, 64, None), "both factors or neither")
    for rows, cols in ((0, 64), (4, 0)):
        assert L.vbt_b200_checkpoint8(None, None, None, F32, 0, rows, cols, cols, None) == 0
        assert L.vbt_b200_silu_mul(None, None, None, None, None, None, None, F32, 0, rows, cols, cols, cols, None) == 0


def rot(L, q=P, qo=P, hq=2, k=P, ko=P, hk=1, dtype=BF16, batch=1, tokens=3, dim=64, pos=P, pdt=I64, freq=P, half=32,
        sections=(32,)):
    st = (ctypes.c_int64 * 15)(*([64] * 15))
    return L.vbt_b200_rotary(qo, q, hq, ko, k, hk, st, dtype, batch, tokens, dim, pos, pdt, freq, half,
                             (ctypes.c_int64 * 5)(*sections), len(sections), 0, 0, None)


def test_rotary_refusals(L):
    refused(L, rot(L, dtype=I64), "floating dtype")
    refused(L, rot(L, tokens=-1), "negative size")
    refused(L, rot(L, half=33, sections=(33,)), "more pairs")
    refused(L, rot(L, sections=(16, 15)), "do not sum")
    refused(L, rot(L, sections=(40, -8)), "negative section")
    refused(L, rot(L, sections=(8, 8, 8, 4, 4)), "1 to 4 sections")
    refused(L, rot(L, pdt=F16), "positions must be")
    for kw in (dict(q=None), dict(qo=None), dict(ko=None), dict(pos=None), dict(freq=None)):
        refused(L, rot(L, **kw), "null pointer")
    refused(L, rot(L, hq=20000), "too many heads")
    refused(L, rot(L, batch=1 << 20, tokens=1 << 20), "too many tokens")
    assert rot(L, tokens=0) == 0 and rot(L, hq=0, k=None) == 0


def write(L, slots=100, heads=2, dim=64, fmt=0, k=P, v=P, dtype=BF16, sl=P, sdt=I64, tokens=3, owner=P, cache=P, st=(128, 64)):
    s2 = (ctypes.c_int64 * 2)(*st)
    return L.vbt_b200_kv_cache_write(cache, P, P, P, slots, heads, dim, fmt, k, s2, v, s2, dtype, sl, sdt, tokens, owner, None,
                                     None)


def read(L, rows=3, slots=96, page=16, heads=2, dim=64, fmt=0, ko=P, dtype=BF16, table=P, tdt=I64, tstride=4, pages=4, starts=P,
         seqs=2):
    return L.vbt_b200_kv_cache_read(ko, P, dtype, rows, P, P, P, P, slots, page, heads, dim, fmt, table, tdt, tstride, pages,
                                    starts, seqs, 0, None, None)


def test_cache_refusals(L):
    for f in (write, read):
        refused(L, f(L, fmt=5), "unknown 8-bit format")
        refused(L, f(L, dtype=I64), "floating dtype")
        refused(L, f(L, heads=-1), "negative size")
        refused(L, f(L, heads=1 << 14, dim=1 << 14), "rows too wide")
    refused(L, write(L, sdt=F32), "slots must be")
    refused(L, write(L, tokens=-1), "number of tokens")
    for kw in (dict(owner=None), dict(cache=None), dict(k=None), dict(sl=None)):
        refused(L, write(L, **kw), "null pointer")
    refused(L, write(L, st=(-1, 64)), "negative stride")
    assert write(L, tokens=0, k=None) == 0
    refused(L, read(L, page=0), "page_size")
    refused(L, read(L, slots=95), "page_size")
    refused(L, read(L, rows=1 << 31), "too many rows")
    refused(L, read(L, tdt=BF16), "page_table must be")
    refused(L, read(L, tstride=-1), "negative size")
    for kw in (dict(ko=None), dict(starts=None), dict(table=None)):
        refused(L, read(L, **kw), "null pointer")
    assert read(L, rows=0, ko=None) == 0


def test_python_layer_takes_no_cpu_tensors():
    from vibetensor_b200 import cache, kernels
    x = torch.ones(4, 64)
    i = torch.ones(4)
    q, pos, f = torch.ones(3, 2, 64), torch.zeros(3, dtype=torch.int64), torch.ones(32)
    held = kernels.Checkpoint8(torch.zeros(4, 64, dtype=torch.int8), torch.ones(4, 1), "int8", torch.float32)
    for call in (lambda: kernels.residual_norm(x, x), lambda: kernels.residual_norm_backward(x, x, x, x, i, i),
                 lambda: kernels.checkpoint8(x), lambda: kernels.checkpoint8_restore(held),
                 lambda: kernels.rmsnorm_checkpoint8(x), lambda: kernels.rmsnorm_backward(x, held, i),
                 lambda: kernels.silu_mul(x, x), lambda: kernels.silu_mul_checkpoint8(x, x),
                 lambda: kernels.silu_mul_backward(x, x, x), lambda: kernels.rotary(q, None, pos, f),
                 lambda: kernels.rotary_backward(q, None, pos, f), lambda: cache.QuantCache(2, 4, 2, 64, device="cpu")):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_overlap_of_views():
    """Which outputs ``rotary`` takes beside its inputs: itself, or memory that shares nothing with them."""
    from vibetensor_b200.kernels import _overlap
    qkv = torch.zeros(2, 5, 12 * 8)
    q, k = qkv[..., :64].unflatten(-1, (8, 8)), qkv[..., 64:80].unflatten(-1, (2, 8))
    assert not _overlap(q, k) and not _overlap(k, q)
    assert _overlap(q, qkv[..., 8:72].unflatten(-1, (8, 8)))
    assert _overlap(q, q) and not _overlap(q, q.clone())
    assert not _overlap(q[:1], q[1:]) and _overlap(q[:, :3], q[:, 2:])
    assert not _overlap(q[:, :0], q)


class OnCard(torch.Tensor):
    """A CPU tensor that passes for a CUDA one where only its shape and strides are looked at."""
    is_cuda = property(lambda self: True)


@pytest.mark.parametrize("x", [
    pytest.param(torch.arange(4 * 48).reshape(4, 1, 48).chunk(6, -1)[1], id="one part of a projection, one row per sample"),
    pytest.param(torch.arange(4 * 48).reshape(4, 1, 1, 48)[..., 8:16], id="the same, two axes of one"),
    pytest.param(torch.arange(6 * 48).reshape(2, 3, 1, 48)[..., 8:16], id="one row per sample and step"),
    pytest.param(torch.arange(6 * 48).reshape(1, 6, 48)[..., 8:16], id="a leading axis of one"),
    pytest.param(torch.arange(6 * 48).reshape(2, 1, 3, 48)[..., 8:16], id="an axis of one in the middle"),
    pytest.param(torch.arange(4 * 5 * 8).reshape(4, 5, 8)[:, -1:], id="the last token of each sample"),
    pytest.param(torch.arange(4 * 6 * 8).reshape(4, 6, 8)[:, ::2], id="every other token"),
    pytest.param(torch.arange(4 * 6 * 8).reshape(4, 6, 8)[:, 1:4], id="some tokens of each sample"),
    pytest.param(torch.arange(4 * 6 * 8).reshape(4, 6, 8).transpose(0, 1), id="samples behind tokens"),
    pytest.param(torch.arange(8).expand(5, 8), id="one row for all"),
    pytest.param(torch.arange(4 * 8).reshape(4, 1, 8).expand(4, 3, 8), id="one row per sample for all tokens"),
    pytest.param(torch.arange(999).as_strided((4, 1, 8), (48, 7, 1)), id="an axis of one with a stride of its own"),
    pytest.param(torch.arange(96).reshape(1, 1, 96)[..., 8:16], id="one row"),
    pytest.param(torch.arange(4 * 6).reshape(4, 6)[:, 2:3], id="single values"),
    pytest.param(torch.arange(48)[::3], id="a strided row"),
    pytest.param(torch.arange(48).reshape(6, 8).t(), id="columns"),
])
def test_rows_of_a_view(monkeypatch, x):
    """What the row ops hand to a kernel -- a first value, a number of rows and one stride -- reaches the
    view's own values, whatever axes of one lie between."""
    from vibetensor_b200 import kernels
    monkeypatch.setattr(kernels._ops, "contiguous", lambda t: t.contiguous())
    monkeypatch.setattr(kernels, "_FLOATS", (torch.int64,))
    view, rows, cols, stride = kernels._rows_view(x.as_subclass(OnCard), "rows")
    got = view.as_subclass(torch.Tensor).as_strided((rows, cols), (stride, 1))
    assert torch.equal(got, x.reshape(-1, x.shape[-1]))


class FakeLib:
    """Stands in for the library: takes note of the calls and launches nothing."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *args: self.calls.append(name) or 0


@pytest.fixture
def host_only(monkeypatch):
    from vibetensor_b200 import kernels
    fake = FakeLib()
    monkeypatch.setattr(kernels, "lib", lambda: fake)
    monkeypatch.setattr(kernels, "stream_ptr", lambda t=None: 0)
    return fake


def test_rotary_output_replaces_its_own_operand_only(host_only):
    """An output may be the operand in its place.  Queries that are also the keys are read by the other
    half of the launch: an output there would be turned while it is still read."""
    from vibetensor_b200 import kernels
    q, other = (torch.zeros(2, 5, 3, 64).as_subclass(OnCard) for _ in range(2))
    pos, f = torch.zeros(2, 5, dtype=torch.int64), torch.ones(32)
    for call in (kernels.rotary, kernels.rotary_backward):
        for out in ((q, other), (other, q)):
            with pytest.raises(ValueError, match="overlaps an input"):
                call(q, q, pos, f, out=out)
        with pytest.raises(ValueError, match="overlaps an input"):
            call(q, other, pos, f, out=(other, q))     # each in the other's place
    assert not host_only.calls
    kernels.rotary(q, other, pos, f, out=(q, other))
    kernels.rotary(q, q, pos, f)
    kernels.rotary(q, None, pos, f, out=(q, None))
    assert host_only.calls == ["vbt_b200_rotary"] * 3


def test_rotary_output_values_are_apart(host_only):
    """Outputs whose own values share memory are refused, whichever way they come to."""
    from vibetensor_b200 import kernels
    q = torch.zeros(2, 5, 3, 64).as_subclass(OnCard)
    pos, f = torch.zeros(2, 5, dtype=torch.int64), torch.ones(32)
    base = torch.zeros(4000)
    for strides in ((0, 192, 64, 1), (960, 0, 64, 1), (960, 192, 0, 1), (960, 192, 63, 1), (960, 128, 64, 1), (64, 192, 64, 1),
                    (191, 192, 960, 1)):
        with pytest.raises(ValueError, match="share memory"):
            kernels.rotary(q, None, pos, f, out=(base.as_strided(q.shape, strides).as_subclass(OnCard), None))
    assert not host_only.calls
    for strides in ((960, 192, 64, 1), (192, 384, 64, 1), (64, 512, 128, 1), (1500, 240, 80, 1)):
        kernels.rotary(q, None, pos, f, out=(base.as_strided(q.shape, strides).as_subclass(OnCard), None))
    one = q[:1, :1]
    kernels.rotary(one, None, pos[:1, :1], f, out=(base.as_strided(one.shape, (0, 0, 64, 1)).as_subclass(OnCard), None))
    assert len(host_only.calls) == 5


def test_scratch_of_as_many_rows_as_there_may_be(L):
    need = ctypes.c_size_t()
    f = L.vbt_b200_residual_norm_backward_workspace_bytes
    most = (1 << 31) - 1
    for per in (1, most):
        for cols in (64, 4096, 4095, 16384, 70001):
            assert f(most, cols, BF16, per, 0, ctypes.byref(need)) == 0
            assert 8 * cols <= need.value < 1 << 40
    refused(L, f(1 << 31, 64, BF16, 1 << 31, 0, ctypes.byref(need)), "too many rows")
    refused(L, back(L, rows=1 << 31), "too many rows")
