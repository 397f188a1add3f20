"""residual_norm, 8-bit activation checkpoints, silu_mul, rotary and the 8-bit key/value cache against
plain 64-bit forms of their formulas.

Tolerances are derived, not fitted.  u = 2^-24 is half a step of fp32.  A value computed in fp32 from
terms of total magnitude M is off by at most K * u * M, where K counts the roundings on the longest
path: a row sum is sequential over at most 137 values per thread (70001 / 512 and 20001 / 256 in the
kernels for rows of any length, 16 in the others) plus a tree of at most 15 levels, a sum over rows
over at most rows / 296 rows per block plus the fold (at most 8 rows per thread and step, 15 levels), square roots, exponentials and sines add at most 4 each, the products
around them at most 10.  K = 192 covers every size below (137 + 15 + 14 < 192).  Storing to t
adds half a step, eps(t) / 2 relative, and half the smallest subnormal.  8-bit levels and scales are a
fixed sequence of correctly rounded fp32 operations: they are compared bit for bit."""
import ctypes

import numpy as np
import pytest
import torch

from tests.util import note_worst

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U, K = 2.0 ** -24, 192
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -24, BF16: 2.0 ** -133}


@pytest.fixture(scope="module")
def kernels():
    from vibetensor_b200 import kernels as k
    return k


@pytest.fixture(scope="module")
def cache():
    from vibetensor_b200 import cache as c
    return c


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, shape, dtype=F32, scale=1.0):
    return (scale * torch.randn(shape, generator=g, device="cuda")).to(dtype)


def close(label, got, want, mass, k=K):
    """|got - want| <= k u mass + half a step of got's type (and of its smallest value)."""
    got64 = got.double().reshape(want.shape)
    bound = k * U * mass + (torch.finfo(got.dtype).eps / 2) * want.abs() + TINY[got.dtype]
    err = (got64 - want).abs()
    assert torch.isfinite(got64).all(), f"{label}: not finite"
    worst = (err / bound).max().item() if err.numel() else 0.0
    note_worst(f"{label} {str(got.dtype)[6:]} (of its bound)", worst, 1.0)
    assert worst <= 1.0, f"{label}: {worst:.3f} times its bound at {int((err / bound).argmax())}"


# ------------------------------------------------------------------------------- residual_norm
def expand_gate(gate, shape):
    return torch.ones((), dtype=torch.float64, device="cuda") if gate is None else gate.double().expand(shape)


def join_ref(x, y, gp, gate, gn, eps, post, pre, a, b):
    x, y = x.double(), y.double()
    g = expand_gate(gate, x.shape)
    i1 = (y.pow(2).mean(-1, keepdim=True) + eps).rsqrt() if post else torch.ones_like(y[..., :1])
    gp = gp.double() if gp is not None else 1.0
    gn = gn.double() if gn is not None else 1.0
    v = y * i1 * gp if post else y
    r = a * x + b * g * v
    mass = (a * x).abs() + (b * g * v).abs()
    i2 = (r.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    rho = (mass.pow(2).sum(-1, keepdim=True) / r.pow(2).sum(-1, keepdim=True).clamp_min(1e-300)).sqrt()
    n = r * i2 * gn
    return dict(r=r, n=n, i1=i1[..., 0].reshape(-1), i2=i2[..., 0].reshape(-1), mass=mass,
                n_mass=i2 * mass * (gn if isinstance(gn, float) else gn.abs()) + n.abs() * (1 + 2 * rho), rho=rho.reshape(-1))


def join_bwd_ref(dr, dn, y, r, i1, i2, gp, gate, gn, a, b):
    shape = (dn if dn is not None else dr).shape
    d = shape[-1]
    z = torch.zeros(shape, dtype=torch.float64, device="cuda")
    dr = z if dr is None else dr.double()
    g = expand_gate(gate, shape)
    G, mG = dr.clone(), dr.abs()
    out = {}
    if i2 is not None:
        j = i2.double().reshape(shape[:-1] + (1,))
        dn, r = dn.double(), r.double()
        gn = gn.double() if gn is not None else torch.ones(d, dtype=torch.float64, device="cuda")
        t = dn * gn
        G = G + j * t - r * j ** 3 * (t * r).mean(-1, keepdim=True)
        mG = mG + (j * t).abs() + (r * j ** 3).abs() * (t * r).abs().mean(-1, keepdim=True)
        out["dgn"] = ((dn * r * j).reshape(-1, d).sum(0), (dn * r * j).abs().reshape(-1, d).sum(0))
    out["dx"] = (a * G, abs(a) * mG)
    lead = tuple(range(len(shape) - 1))
    if y is not None:
        y = y.double()
    if i1 is not None:
        i = i1.double().reshape(shape[:-1] + (1,))
        gp = gp.double() if gp is not None else torch.ones(d, dtype=torch.float64, device="cuda")
        v = y * i * gp
    else:
        v = y
    if gate is not None:
        full, mfull = b * G * v, (b * v).abs() * mG
        over = tuple(k for k in lead if gate.dim() == 1 or gate.shape[k] == 1)
        out["dgate"] = tuple(t.sum(over, keepdim=True).reshape(gate.shape) if over else t for t in (full, mfull))
    dv, mdv = b * G * g, (b * g).abs() * mG
    if i1 is not None:
        out["dgp"] = tuple(t.reshape(-1, d).sum(0) for t in (dv * y * i, mdv * (y * i).abs()))
        w = gp
        out["dy"] = (i * dv * w - y * i ** 3 * (dv * w * y).mean(-1, keepdim=True),
                     (i * w).abs() * mdv + (y * i ** 3).abs() * (mdv * (w * y).abs()).mean(-1, keepdim=True))
    else:
        out["dy"] = (dv, mdv)
    return out


def gate_for(g, kind, shape, dtype):
    if kind == "none":
        return None
    if kind == "channel":
        return randn(g, shape[-1:], dtype)
    if kind == "sample":
        return randn(g, shape[:1] + (1,) * (len(shape) - 2) + shape[-1:], dtype)
    return randn(g, shape, dtype)


# one width per kernel variant, with the odd ones that take single values
COLS = [1, 7, 64, 128, 200, 333, 512, 1000, 1365, 2048, 4096, 5000, 8192, 12345, 16384, 16400, 20001,
        33000, 70001]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("cols", COLS)
def test_residual_norm(kernels, dtype, cols):
    g = gen(cols)
    for shape, kind in (((3, 5, cols), "sample"), ((1, 1, cols), "none"), ((2, 37, cols), "channel"), ((2, 3, cols), "full")):
        x, y = randn(g, shape, dtype, 2.0), randn(g, shape, dtype)
        gp, gn = 1 + 0.1 * randn(g, (cols,)), 1 + 0.1 * randn(g, (cols,))
        gate = gate_for(g, kind, shape, dtype)
        a, b = (1.0, 1.0) if kind != "channel" else (0.7, -1.3)
        r, n, i1, i2 = kernels.residual_norm(x, y, gp, gate, gn, 1e-6, residual_scale=a, branch_scale=b)
        w = join_ref(x, y, gp, gate, gn, 1e-6, True, True, a, b)
        close("residual_norm r", r, w["r"], w["mass"])
        close("residual_norm n", n, w["n"], w["n_mass"])
        close("residual_norm inv_post", i1, w["i1"], w["i1"])
        close("residual_norm inv_pre", i2, w["i2"], w["i2"] * (1 + 2 * w["rho"]))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("cols", COLS)
def test_residual_norm_backward(kernels, dtype, cols):
    g = gen(1000 + cols)
    for shape, kind in (((3, 5, cols), "sample"), ((1, 1, cols), "none"), ((2, 37, cols), "channel"), ((2, 3, cols), "full"),
                        ((40, 2, cols), "sample")):
        if cols > 8192 and shape[0] == 40:
            continue
        y, r = randn(g, shape, dtype), randn(g, shape, dtype, 2.0)
        dr, dn = randn(g, shape, dtype), randn(g, shape, dtype)
        gp, gn = 1 + 0.1 * randn(g, (cols,)), 1 + 0.1 * randn(g, (cols,))
        gate = gate_for(g, kind, shape, dtype)
        i1 = (y.double().pow(2).mean(-1) + 1e-6).rsqrt().float().reshape(-1)
        i2 = (r.double().pow(2).mean(-1) + 1e-6).rsqrt().float().reshape(-1)
        a, b = (1.0, 1.0) if kind != "channel" else (0.7, -1.3)
        got = dict(zip(("dx", "dy", "dgp", "dgate", "dgn"), kernels.residual_norm_backward(
            dr, dn, y, r, i1, i2, gp, gate, gn, residual_scale=a, branch_scale=b)))
        want = join_bwd_ref(dr, dn, y, r, i1, i2, gp, gate, gn, a, b)
        assert (got["dgate"] is None) == (gate is None)
        for name, (t, mass) in want.items():
            close(f"residual_norm_backward {name}", got[name], t, mass)


@pytest.mark.parametrize("cols", [64, 1365, 4096, 20001])
def test_residual_norm_parts_switched_off(kernels, cols):
    g = gen(7)
    shape = (6, 11, cols)
    x, y = randn(g, shape, BF16, 2.0), randn(g, shape, BF16)
    for post, pre, kind in ((False, True, "none"), (True, False, "sample"), (False, False, "channel"), (False, True, "full")):
        gate = gate_for(g, kind, shape, BF16)
        r, n, i1, i2 = kernels.residual_norm(x, y, gate=gate, post_norm=post, pre_norm=pre)
        w = join_ref(x, y, None, gate, None, 1e-6, post, pre, 1.0, 1.0)
        assert (n is None) == (i2 is None) == (not pre) and (i1 is None) == (not post)
        close("residual_norm r, a norm off", r, w["r"], w["mass"])
        if pre:
            close("residual_norm n, a norm off", n, w["n"], w["n_mass"])
        dr, dn = randn(g, shape, BF16), randn(g, shape, BF16) if pre else None
        got = dict(zip(("dx", "dy", "dgp", "dgate", "dgn"),
                       kernels.residual_norm_backward(dr, dn, y, r, i1, i2, gate=gate)))
        assert got["dgp"] is None and got["dgn"] is None
        want = join_bwd_ref(dr, dn, y, r, i1, i2, None, gate, None, 1.0, 1.0)
        for name in ("dx", "dy", "dgate"):
            if name in want:
                close(f"residual_norm_backward {name}, a norm off", got[name], *want[name])
        if pre:  # the stream's gradient may be missing
            got = kernels.residual_norm_backward(None, dn, y, r, i1, i2, gate=gate)
            want = join_bwd_ref(None, dn, y, r, i1, i2, None, gate, None, 1.0, 1.0)
            close("residual_norm_backward dx, no stream gradient", got[0], *want["dx"])
        if not post and gate is None:  # then y is not read, and what is in it does not matter
            ref = kernels.residual_norm_backward(dr, dn, None, r, None, i2)
            bad = kernels.residual_norm_backward(dr, dn, torch.full_like(y, float("nan")), r, None, i2)
            assert all(torch.equal(p, q) for p, q in zip(ref[:2], bad[:2]))


def test_residual_norm_gradients_match_differences(kernels):
    """Central differences of the 64-bit forward, against the kernels' gradients in fp32.  The
    difference of two forwards a step h apart is off by h^2 times a third derivative of order one
    and by 2^-53 / h; with h = 1e-5 both are below 1e-9 of the directional derivative's mass."""
    g = gen(3)
    shape, eps = (4, 3, 40), 1e-6
    x, y = randn(g, shape, F32, 2.0), randn(g, shape)
    gp, gn, gate = 1 + 0.1 * randn(g, (40,)), 1 + 0.1 * randn(g, (40,)), randn(g, (4, 1, 40))
    dr, dn = randn(g, shape), randn(g, shape)
    r, n, i1, i2 = kernels.residual_norm(x, y, gp, gate, gn, eps, residual_scale=0.9, branch_scale=1.1)
    dx, dy, dgp, dgate, dgn = kernels.residual_norm_backward(dr, dn, y, r, i1, i2, gp, gate, gn, residual_scale=0.9,
                                                             branch_scale=1.1)

    def loss(x, y, gp, gate, gn):
        w = join_ref(x, y, gp, gate, gn, eps, True, True, 0.9, 1.1)
        return ((w["r"] * dr.double()).sum() + (w["n"] * dn.double()).sum()).item()
    args = [x, y, gp, gate, gn]
    for i, grad in enumerate((dx, dy, dgp, dgate, dgn)):
        v = torch.randn(args[i].shape, generator=g, device="cuda", dtype=torch.float64)
        h = 1e-5
        up, dn_ = list(args), list(args)
        up[i], dn_[i] = args[i].double() + h * v, args[i].double() - h * v
        diff = (loss(*up) - loss(*dn_)) / (2 * h)
        prod = grad.double() * v
        # fp32 gradient entries are off by K u of a mass of at most ten times their rows' scale
        assert abs(prod.sum().item() - diff) <= 10 * K * U * prod.abs().sum().item() + 1e-8 * prod.abs().sum().item()


def test_residual_norm_strided_rows_and_empty(kernels):
    g = gen(11)
    base = randn(g, (50, 3 * 256), BF16)
    x, y = base[:, :256], base[:, 300:556]            # row stride 768, y starts off a 16-byte boundary
    gp = torch.ones(256, device="cuda")
    r, n, i1, i2 = kernels.residual_norm(x, y, gp, None, gp)
    r2, n2, j1, j2 = kernels.residual_norm(x.contiguous(), y.contiguous(), gp, None, gp)
    w = join_ref(x, y, gp, None, gp, 1e-6, True, True, 1.0, 1.0)
    for t in (r, r2):
        close("residual_norm strided", t, w["r"], w["mass"])
    xt = randn(g, (256, 40)).t()                       # the last stride is not 1
    r, *_ = kernels.residual_norm(xt, xt)
    w = join_ref(xt, xt, None, None, None, 1e-6, True, True, 1.0, 1.0)
    close("residual_norm transposed", r, w["r"], w["mass"])
    e = torch.empty((0, 64), device="cuda")
    r, n, i1, i2 = kernels.residual_norm(e, e)
    assert r.shape == (0, 64) and i1.shape == (0,)
    g64 = torch.ones(64, device="cuda")
    dx, dy, dgp, dgate, dgn = kernels.residual_norm_backward(e, e, e, e, i1, i2, g64, None, g64)
    assert dgp.abs().sum() == 0 and dgn.abs().sum() == 0 and dx.shape == (0, 64)


def test_residual_norm_sums_are_reproducible(kernels):
    g = gen(12)
    shape = (8, 700, 1024)
    t = [randn(g, shape, BF16) for _ in range(4)]
    i = torch.ones(5600, device="cuda")
    gam, gate = torch.ones(1024, device="cuda"), randn(g, (8, 1, 1024), BF16)
    a = kernels.residual_norm_backward(*t, i, i, gam, gate, gam)
    for _ in range(3):
        b = kernels.residual_norm_backward(*t, i, i, gam, gate, gam)
        assert all(torch.equal(p, q) for p, q in zip(a, b))


# ------------------------------------------------------------------------------ 8-bit checkpoints
TOP = {"int8": np.float32(127), "e4m3": np.float32(448)}


def held_ref(x, fmt):
    """numpy fp32: (levels as float64, scale as float32) of rows x [n, d] in groups of 128."""
    n, d = x.shape
    groups = -(-d // 128)
    z = np.zeros((n, groups * 128), np.float32)
    z[:, :d] = x
    z = z.reshape(n, groups, 128)
    amax = np.abs(z).max(-1)                        # numpy's max keeps a NaN
    with np.errstate(all="ignore"):
        dead = amax < np.float32(2.0 ** -119)
        up = np.where(dead, np.float32(0), TOP[fmt] / np.where(dead, np.float32(1), amax)).astype(np.float32)
        scale = np.where(dead, np.float32(0), amax * np.float32(np.float32(1) / TOP[fmt])).astype(np.float32)
        p = (z * up[..., None]).astype(np.float32)
        if fmt == "int8":
            q = np.nan_to_num(np.rint(p), nan=0.0).astype(np.float64)
        else:
            q = torch.from_numpy(p).to(torch.float8_e4m3fn).double().numpy()
    return q.reshape(n, -1)[:, :d], scale


def check_held(c, x, fmt):
    q, scale = held_ref(x.float().cpu().numpy().reshape(-1, x.shape[-1]), fmt)
    got = c.q.cpu().double().numpy().reshape(q.shape) if fmt == "e4m3" else c.q.cpu().numpy().astype(np.float64).reshape(q.shape)
    assert np.array_equal(got, q, equal_nan=True)
    assert np.array_equal(c.scale.cpu().numpy(), scale, equal_nan=True)


def acts(g, shape, dtype):
    x = randn(g, shape, dtype)
    return x * torch.where(torch.rand(shape[-1], generator=g, device="cuda") < 0.02, 20.0, 1.0).to(dtype)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("cols", [1, 8, 127, 128, 129, 136, 1000, 1024, 5000])
def test_checkpoint8_bit_for_bit(kernels, fmt, dtype, cols):
    g = gen(cols)
    for rows in (1, 3, 70):
        x = acts(g, (rows, cols), dtype)
        c = kernels.checkpoint8(x, fmt)
        check_held(c, x, fmt)
        want = (c.q.float().reshape(rows, cols) * c.scale.repeat_interleave(128, 1)[:, :cols])
        for dt in (dtype, F32, BF16):
            assert torch.equal(kernels.checkpoint8_restore(c, dt), want.to(dt))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_checkpoint8_special_values(kernels, fmt):
    x = torch.zeros((8, 256), device="cuda")
    x[1, 5] = float("nan")
    x[2, 6] = float("inf")
    x[3, 7] = float("-inf")
    x[4] = 1e-40                       # below 2^-119: held as zeros
    x[5, :128] = 2.0 ** -119
    x[6, 3] = 3.0e38
    x[7] = torch.arange(256, device="cuda") / 128 - 1
    x[1:4, 130:] = 1.0
    r = kernels.checkpoint8_restore(kernels.checkpoint8(x, fmt))
    assert torch.equal(r[0], x[0]) and torch.equal(r[4], torch.zeros(256, device="cuda"))
    assert torch.isnan(r[1:4, :128]).all() and not torch.isnan(r[1:4, 128:]).any()   # the whole group, no other
    check_held(kernels.checkpoint8(x[4:], fmt), x[4:], fmt)
    assert r[5, 0].item() > 0 and torch.isfinite(r[6]).all()
    # half a step: scale / 2 for int8, 2^-4 of a value (or of the smallest level) for e4m3
    amax = x[7].abs().reshape(2, 128).amax(-1).repeat_interleave(128)
    bound = amax / 254 if fmt == "int8" else torch.maximum(x[7].abs() * 2.0 ** -4, amax * 2.0 ** -10 / 448)
    assert ((r[7] - x[7]).abs() <= bound * (1 + 8 * U)).all()


def test_checkpoint8_strides_and_ranks(kernels):
    g = gen(5)
    base = acts(g, (2, 9, 700), BF16)
    x = base[..., 3:603]                              # unaligned rows of a wider tensor
    check_held(kernels.checkpoint8(x), x.reshape(-1, 600), "int8")
    v = acts(g, (300,), F32)
    c = kernels.checkpoint8(v)
    assert c.q.shape == (300,) and c.scale.shape == (1, 3) and c.nbytes() == 312
    e = kernels.checkpoint8(torch.empty((0, 64), device="cuda"))
    assert kernels.checkpoint8_restore(e).shape == (0, 64)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("cols", [1, 64, 120, 128, 200, 512, 1000, 1365, 2048, 4096, 5000, 8192, 16384, 20001])
def test_rmsnorm_kept_in_8_bits(kernels, fmt, dtype, cols):
    g = gen(cols)
    rows = 41 if cols < 8192 else 5
    x, dy, gamma = acts(g, (rows, cols), dtype), randn(g, (rows, cols), dtype), 1 + 0.1 * randn(g, (cols,))
    out, inv, c = kernels.rmsnorm_checkpoint8(x, gamma, 1e-6, fmt)
    check_held(c, x, fmt)
    w = join_ref(x, x, None, None, gamma, 1e-6, False, True, 1.0, 0.0)
    close("rmsnorm_checkpoint8 out", out, w["n"], w["n"].abs())
    close("rmsnorm_checkpoint8 inv_rms", inv, w["i2"], w["i2"])
    dx, dgamma = kernels.rmsnorm_backward(dy, c, inv, gamma)
    kept = kernels.checkpoint8_restore(c, F32)
    want = join_bwd_ref(None, dy, None, kept, None, inv, None, None, gamma, 1.0, 1.0)
    close("rmsnorm_backward of a checkpoint, dx", dx, *want["dx"])
    close("rmsnorm_backward of a checkpoint, dgamma", dgamma, *want["dgn"])
    dx2, none = kernels.rmsnorm_backward(dy, c, inv)
    want = join_bwd_ref(None, dy, None, kept, None, inv, None, None, None, 1.0, 1.0)
    assert none is None
    close("rmsnorm_backward of a checkpoint, no gamma", dx2, *want["dx"])


def silu_ref(d, a, b):
    d, a, b = d.double(), a.double(), b.double()
    s = torch.sigmoid(a)
    h = a * s * b
    da, db = d * b * s * (1 + a * torch.sigmoid(-a)), d * a * s
    return (h, h.abs()), (da, (d * b * s).abs() * (1 + a.abs())), (db, db.abs())


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("cols", [1, 8, 120, 128, 333, 1000, 4096])
def test_silu_mul(kernels, fmt, dtype, cols):
    g = gen(cols)
    both = acts(g, (37, 2 * cols), dtype)
    a, b, d = both[:, :cols], both[:, cols:], randn(g, (37, cols), dtype)
    h, ca, cb = kernels.silu_mul_checkpoint8(a, b, fmt)
    check_held(ca, a, fmt)
    check_held(cb, b, fmt)
    (hw, hm), (daw, dam), (dbw, dbm) = silu_ref(d, a, b)
    close("silu_mul", h, hw, hm)
    assert torch.equal(h, kernels.silu_mul(a, b))
    da, db = kernels.silu_mul_backward(d, a, b)
    close("silu_mul_backward gate", da, daw, dam)
    close("silu_mul_backward up", db, dbw, dbm)
    da, db = kernels.silu_mul_backward(d, ca, cb)
    _, (daw, dam), (dbw, dbm) = silu_ref(d, kernels.checkpoint8_restore(ca, F32), kernels.checkpoint8_restore(cb, F32))
    close("silu_mul_backward of checkpoints, gate", da, daw, dam)
    close("silu_mul_backward of checkpoints, up", db, dbw, dbm)


def test_silu_mul_far_values_and_differences(kernels):
    a = torch.tensor([-1e4, -200.0, -89.0, -20.0, 0.0, 20.0, 89.0, 1e4], device="cuda")
    b, d = torch.full_like(a, 2.0), torch.full_like(a, 3.0)
    (hw, hm), (daw, dam), (dbw, dbm) = silu_ref(d, a, b)
    tiny = 1e-30                                       # e^-89 and below may vanish in fp32
    close("silu_mul far", kernels.silu_mul(a, b), hw, hm + tiny / (K * U))
    da, db = kernels.silu_mul_backward(d, a, b)
    close("silu_mul_backward far", da, daw, dam + tiny / (K * U))
    x = torch.linspace(-6, 6, 101, device="cuda")
    one = torch.ones_like(x)
    da, db = kernels.silu_mul_backward(one, x, one)
    x64, h = x.double(), 1e-5
    f = lambda t: t * torch.sigmoid(t)  # noqa: E731
    diff = (f(x64 + h) - f(x64 - h)) / (2 * h)
    assert ((da.double() - diff).abs() <= 16 * U * (1 + x64.abs()) + 1e-9).all()


# ------------------------------------------------------------------------------------- rotary
def rotary_ref(x, pos, freq, sections, interleaved, inverse):
    """x [b, t, h, d], pos [axes, b, t]; returns (want, mass)."""
    half = freq.shape[0]
    ang, i = [], 0
    for a, n in enumerate(sections):
        ang.append(pos[a].double()[..., None] * freq[i:i + n].double())
        i += n
    ang = torch.cat(ang, -1)[:, :, None]
    c, s = ang.cos(), ang.sin() * (-1 if inverse else 1)
    x = x.double()
    want, mass = x.clone(), torch.zeros_like(x)
    p, q = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = x[..., p], x[..., q]
    want[..., p], want[..., q] = a * c - b * s, b * c + a * s
    mass[..., p] = mass[..., q] = a.abs() + b.abs()
    return want, mass


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,half,sections", [(128, 64, (16, 24, 24)), (128, 64, (64,)), (80, 32, (16, 16)), (80, 40, (0, 40)),
                                               (72, 18, (5, 6, 7)), (40, 10, (3, 3, 2, 2)), (7, 3, (1, 2)), (6, 0, (0,)),
                                               (64, 4, (4,)), (256, 128, (128,)), (66, 33, (33,))])
def test_rotary(kernels, dtype, interleaved, dim, half, sections):
    g = gen(dim)
    freq = torch.exp(-torch.arange(half, device="cuda") * 0.13)
    for b, t, hq, hk in ((2, 5, 4, 2), (1, 1, 3, 1), (3, 130, 5, 5), (1, 400, 1, 1), (64, 1, 8, 2)):
        q, k = randn(g, (b, t, hq, dim), dtype), randn(g, (b, t, hk, dim), dtype)
        pos = torch.randint(-10, 2000000, (len(sections), b, t), generator=g, device="cuda")
        for inverse, call in ((False, kernels.rotary), (True, kernels.rotary_backward)):
            got = call(q, k, pos, freq, sections, interleaved)
            for x, o in zip((q, k), got):
                want, mass = rotary_ref(x, pos, freq, sections, interleaved, inverse)
                # sine, cosine and the reduced angle are off by at most 4 u, the products by 3
                close("rotary", o, want, mass, 8)
                assert torch.equal(o[..., 2 * half:], x[..., 2 * half:])


def test_rotary_views_positions_and_in_place(kernels):
    g = gen(9)
    half, sections = 32, (8, 12, 12)
    freq = torch.exp(-torch.arange(half, device="cuda") * 0.2)
    qkv = randn(g, (2, 6, 12 * 64), BF16)
    q, k = qkv[..., :8 * 64].unflatten(-1, (8, 64)), qkv[..., 8 * 64:10 * 64].unflatten(-1, (2, 64))
    pos = torch.randint(0, 5000, (3, 2, 6), generator=g, device="cuda")
    want = [rotary_ref(x, pos, freq, sections, False, False) for x in (q, k)]
    a = kernels.rotary(q, k, pos, freq, sections)
    b = kernels.rotary(q.contiguous(), None, pos.int(), freq, sections)
    assert b[1] is None and torch.equal(a[0], b[0])
    assert torch.equal(kernels.rotary(q, k, pos.float(), freq, sections)[1], a[1])
    for o, (w, m) in zip(a, want):
        close("rotary views", o, w, m, 8)
    # heads before tokens, rank 3, and one row of positions for the whole batch
    qt = randn(g, (2, 8, 6, 64), BF16).transpose(1, 2)
    o, _ = kernels.rotary(qt, None, pos[:, :1], freq, sections)
    w, m = rotary_ref(qt, pos[:, :1].expand(3, 2, 6), freq, sections, False, False)
    close("rotary transposed heads", o, w, m, 8)
    o3, _ = kernels.rotary(q[0], None, pos[:, 0], freq, sections)
    assert torch.equal(o3, a[0][0])
    odd = randn(g, (2, 6, 3, 130), BF16)[..., 1:65]    # rows off every vector boundary
    o, _ = kernels.rotary(odd, None, pos, freq, sections, interleaved=True)
    w, m = rotary_ref(odd, pos, freq, sections, True, False)
    close("rotary unaligned", o, w, m, 8)
    for il in (False, True):                           # in place, and back again
        x, y = q.clone(), k.clone()
        ret = kernels.rotary(x, y, pos, freq, sections, il, out=(x, y))
        assert ret[0] is x and torch.equal(x, kernels.rotary(q, k, pos, freq, sections, il)[0])
        view = qkv.clone()
        vq = view[..., :8 * 64].unflatten(-1, (8, 64))
        kernels.rotary(vq, None, pos, freq, sections, il, out=(vq, None))
        assert torch.equal(vq, x) and torch.equal(view[..., 8 * 64:], qkv[..., 8 * 64:])
    e = torch.empty((2, 0, 8, 64), device="cuda")
    assert kernels.rotary(e, None, torch.empty((3, 2, 0), device="cuda", dtype=torch.int64), freq, sections)[0].shape == e.shape


def test_rotary_gradient_matches_differences(kernels):
    """The turn is linear: <w, rotary(q + h v) - rotary(q - h v)> / 2h = <rotary_backward(w), v>
    exactly; the kernels' sides are off by 8 u of |w| and |v| per product."""
    g = gen(21)
    freq = torch.exp(-torch.arange(16, device="cuda") * 0.3)
    pos = torch.randint(0, 100000, (1, 2, 9), generator=g, device="cuda")
    q, w, v = (randn(g, (2, 9, 3, 40)) for _ in range(3))
    grad, _ = kernels.rotary_backward(w, None, pos[0], freq)
    up, _ = rotary_ref(q.double() + v.double(), pos, freq, (16,), False, False)
    dn, _ = rotary_ref(q.double() - v.double(), pos, freq, (16,), False, False)
    diff = ((up - dn) / 2 * w.double()).sum().item()
    mass = (w.abs().double().sum() * v.abs().max()).item()
    assert abs((grad.double() * v.double()).sum().item() - diff) <= 16 * U * mass


# -------------------------------------------------------------------------------------- cache
def read_ref(c, table, starts, rows):
    """(k, v) as float64 and a mask of the rows that a sequence owns."""
    out = []
    for q, s in ((c.k, c.k_scale), (c.v, c.v_scale)):
        full = (q.float() * s[..., None]).reshape(c.num_slots, c.num_heads, c.head_dim)
        o = torch.zeros((rows, c.num_heads, c.head_dim), device="cuda")
        own = torch.zeros(rows, dtype=torch.bool, device="cuda")
        for i in range(table.shape[0]):
            a, b = int(starts[i]), int(starts[i + 1])
            for p in range(b - a):
                pg = p // c.page_size
                page = int(table[i, pg]) if pg < table.shape[1] else -1
                if a + p < rows:
                    own[a + p] = True
                    if 0 <= page < c.num_pages:
                        o[a + p] = full[page * c.page_size + p % c.page_size]
        out.append(o)
    return out[0], out[1], own


def check_slots(c, k, v, slots):
    """Every named slot holds the last token that names it, bit for bit."""
    last = {int(s): i for i, s in enumerate(slots.tolist()) if 0 <= int(s) < c.num_slots}
    for x, q, s in ((k, c.k, c.k_scale), (v, c.v, c.v_scale)):
        idx = torch.tensor(list(last.values()))
        at = torch.tensor(list(last.keys()))
        rows = x.float().cpu()[idx].reshape(len(last) * c.num_heads, c.head_dim).numpy()
        big = np.abs(rows).max(-1)
        with np.errstate(all="ignore"):
            dead = big < np.float32(2.0 ** -119)
            up = np.where(dead, np.float32(0), TOP[c.fmt] / np.where(dead, np.float32(1), big)).astype(np.float32)
            scale = np.where(dead, np.float32(0), big * np.float32(np.float32(1) / TOP[c.fmt])).astype(np.float32)
            p = rows * up[:, None]
        want = np.rint(p) if c.fmt == "int8" else torch.from_numpy(p).to(torch.float8_e4m3fn).float().numpy()
        got = q.reshape(c.num_slots, c.num_heads, c.head_dim).cpu().float()[at].reshape(want.shape).numpy()
        assert np.array_equal(got, want)
        assert np.array_equal(s.reshape(c.num_slots, c.num_heads).cpu()[at].reshape(-1).numpy(), scale)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,dim,page", [(8, 128, 16), (1, 64, 1), (3, 80, 48), (2, 7, 5), (2, 256, 16), (1, 32, 32),
                                            (2, 1024, 4), (1, 1, 3), (5, 72, 16)])
def test_cache_write_and_read(cache, fmt, dtype, heads, dim, page):
    g = gen(dim)
    c = cache.QuantCache(23, page, heads, dim, fmt=fmt)
    lens = [1, page, 0, 2 * page + 1, min(3, page)]
    need = [-(-n // page) for n in lens]
    perm = torch.randperm(23, generator=g, device="cuda")
    table = torch.full((5, max(need)), -1, dtype=torch.int64, device="cuda")
    starts, slots, used = [0], [], 0
    for i, n in enumerate(lens):
        mine = perm[used:used + need[i]]
        used += need[i]
        table[i, :need[i]] = mine
        starts.append(starts[-1] + n)
        at = torch.arange(n, device="cuda")
        slots.append(mine[at // page] * page + at % page if n else at)
    slots = torch.cat(slots)
    order = torch.randperm(slots.numel(), generator=g, device="cuda")
    slots = slots[order]
    k, v = acts(g, (slots.numel(), heads, dim), dtype), acts(g, (slots.numel(), heads, dim), dtype)
    c.write(k, v, slots)
    check_slots(c, k, v, slots)
    total = starts[-1]
    starts = torch.tensor(starts, device="cuda")
    for dt in (F32, F16, BF16):
        wk, wv, own = read_ref(c, table, starts, total + 4)
        rk, rv = c.read(table, starts, total + 4, dtype=dt)
        assert own.sum() == total and torch.equal(rk, wk.to(dt)) and torch.equal(rv, wv.to(dt))
        # rows behind the last sequence are left as they were
        out = (torch.full((total + 4, heads, dim), 7.0, dtype=dt, device="cuda"), torch.full((total + 4, heads, dim), 7.0, dtype=dt, device="cuda"))
        c.read(table.int(), starts, out=out)
        assert torch.equal(out[0][:total], rk[:total]) and (out[0][total:] == 7).all() and (out[1][total:] == 7).all()
    # an int32 slot list, strided keys and values out of a fused projection
    both = acts(g, (slots.numel(), 2 * heads, dim), dtype)
    c.write(both[:, :heads], both[:, heads:], slots.int())
    check_slots(c, both[:, :heads], both[:, heads:], slots)


@pytest.mark.parametrize("tokens", [2, 40, 512, 513, 3000])
def test_cache_equal_slots_keep_the_last_token_whole(cache, tokens):
    g = gen(tokens)
    c = cache.QuantCache(40, 16, 4, 64)
    for trial in range(3):
        slots = torch.randint(0, max(2, tokens // 7), (tokens,), generator=g, device="cuda")
        slots[torch.rand(tokens, generator=g, device="cuda") < 0.1] = -1
        k, v = acts(g, (tokens, 4, 64), BF16), acts(g, (tokens, 4, 64), BF16)
        c.write(k, v, slots)
        check_slots(c, k, v, slots)
        assert c._owner.abs().sum() == 0


@pytest.mark.parametrize("seqs", [1, 31, 32, 33, 1025, 3000])
def test_cache_read_finds_its_sequence(cache, seqs):
    """Many short and empty sequences, their number around the search's 32-way steps."""
    g = gen(seqs)
    heads, dim, page = 1, 8, 2
    lens = torch.randint(0, 4, (seqs,), generator=g, device="cuda")
    lens[0] = 0
    starts = torch.zeros(seqs + 1, dtype=torch.int64, device="cuda")
    starts[1:] = lens.cumsum(0)
    total = int(starts[-1])
    table = torch.arange(2 * seqs, device="cuda").reshape(seqs, 2)[torch.randperm(seqs, generator=g, device="cuda")]
    c = cache.QuantCache(2 * seqs, page, heads, dim)
    k = acts(g, (c.num_slots, heads, dim), F32)
    c.write(k, -k, torch.arange(c.num_slots, device="cuda"))
    rk, rv = c.read(table, starts, total + 3, dtype=F32)
    row = torch.arange(total, device="cuda")
    s = torch.searchsorted(starts, row, right=True) - 1
    at = row - starts[s]
    slot = table[s, at // page] * page + at % page
    full = (c.k.float() * c.k_scale[..., None]).reshape(c.num_slots, heads, dim)
    assert torch.equal(rk[:total], full[slot]) and torch.equal(rv[:total], -full[slot]) and (rk[total:] == 0).all()
    # sequences that begin behind row 0: the rows in front belong to nobody
    rk2, _ = c.read(table, starts + 2, total + 2, dtype=F32)
    assert (rk2[:2] == 0).all() and torch.equal(rk2[2:], rk[:total])


def test_cache_bad_slots_and_pages(cache):
    from vibetensor_b200 import ops
    g = gen(2)
    c = cache.QuantCache(4, 8, 2, 32)
    st = ops.IndexStatus("cuda")
    k, v = acts(g, (6, 2, 32), F32), acts(g, (6, 2, 32), F32)
    for slots in ([0, 5, -1, 32, 1 << 40, 31],):
        t = torch.tensor(slots, device="cuda")
        c.write(k, v, t, status=st)
        check_slots(c, k, v, t)
        with pytest.raises(IndexError, match="out of range"):
            st.check("QuantCache.write", c.num_slots)
        st.check("QuantCache.write", c.num_slots)      # cleared
        c.write(k, v, t)                               # nothing to record into
    table = torch.tensor([[0, 9], [3, -2]], device="cuda")
    starts = torch.tensor([0, 20, 36], device="cuda")  # sequence 0 runs past its table, both name a bad page
    rk, rv = c.read(table, starts, 36, dtype=F32, status=st)
    wk, wv, _ = read_ref(c, table, starts, 36)
    assert torch.equal(rk, wk) and torch.equal(rv, wv)
    with pytest.raises(IndexError, match="20 bad indices"):
        st.check("QuantCache.read", c.num_pages)
    e = c.read(torch.empty((0, 3), dtype=torch.int64, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda"), 5)
    assert (e[0] == 0).all() and e[0].shape == (5, 2, 32)
    c.write(k[:0], v[:0], torch.empty(0, dtype=torch.int64, device="cuda"))


def test_cache_starts_that_do_not_ascend(cache):
    # the search for row 0's sequence ends at sequence 0, which starts at 100: no position of it
    from vibetensor_b200 import ops
    c = cache.QuantCache(4, 16, 2, 32)
    k = torch.ones(64, 2, 32, device="cuda")
    c.write(k, k, torch.arange(64, device="cuda"))
    table = torch.zeros((32, 4), dtype=torch.int64, device="cuda")
    starts = torch.full((33,), 100, device="cuda")
    starts[20] = 0
    st = ops.IndexStatus("cuda")
    rk, rv = c.read(table, starts, 64, dtype=F32, status=st)
    assert (rk == 0).all() and (rv == 0).all()
    with pytest.raises(IndexError, match="64 bad indices"):
        st.check("QuantCache.read", c.num_pages)


def test_cache_status_on_the_cache_device(cache):
    from vibetensor_b200 import ops
    c = cache.QuantCache(1, 4, 2, 32)
    k, st = torch.ones(1, 2, 32, device="cuda"), ops.IndexStatus("cpu")
    slots = torch.zeros(1, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError, match="requires CUDA tensors"):
        c.write(k, k, slots, status=st)
    with pytest.raises(RuntimeError, match="requires CUDA tensors"):
        c.read(slots[None], torch.arange(2, device="cuda"), 1, status=st)


def test_cache_special_rows(cache):
    c = cache.QuantCache(2, 4, 2, 16)
    k = torch.ones((3, 2, 16), device="cuda")
    k[0, 0, 3] = float("nan")
    k[1, 1, 2] = float("inf")
    k[2] = 0
    c.write(k, k, torch.arange(3, device="cuda"))
    rk, _ = c.read(torch.zeros((1, 1), dtype=torch.int64, device="cuda"), torch.tensor([0, 3], device="cuda"), 3, dtype=F32)
    assert torch.isnan(rk[0, 0]).all() and torch.equal(rk[0, 1], k[0, 1]) and torch.isnan(rk[1, 1]).all()
    assert torch.equal(rk[1, 0], k[1, 0]) and torch.equal(rk[2], k[2])


def test_cache_offsets_past_32_bits(cache):
    """A cache of more than 2^32 bytes of keys: slots near its end."""
    heads, dim, page = 8, 128, 64
    pages = (1 << 32) // (heads * dim * page) + 64
    c = cache.QuantCache(pages, page, heads, dim)
    g = gen(4)
    slots = torch.tensor([0, c.num_slots - 1, (1 << 32) // (heads * dim) + 3, 5], device="cuda")
    k, v = acts(g, (4, heads, dim), BF16), acts(g, (4, heads, dim), BF16)
    c.write(k, v, slots)
    table = (slots // page).reshape(4, 1)
    one = cache.QuantCache(1, 4, heads, dim)
    one.write(k, v, torch.arange(4, device="cuda"))
    rk, rv = one.read(torch.zeros((1, 1), dtype=torch.int64, device="cuda"), torch.tensor([0, 4], device="cuda"), 4)
    for i in range(4):
        off = int(slots[i]) % page
        ck, cv = c.read(table[i:i + 1], torch.tensor([0, off + 1], device="cuda"), off + 1)
        assert torch.equal(ck[off], rk[i]) and torch.equal(cv[off], rv[i])
    del c
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------ as they are used
def block_step(kernels, c, w, x, pos, slots, table, starts, freq, sections, hq, hk, dim, total):
    """One block's bandwidth-bound work around torch's products: join, projections, rotary, cache,
    gated activation, join."""
    n, _ = kernels.rmsnorm(x, w["g0"])
    qkv = n @ w["qkv"]
    q = qkv[..., :hq * dim].unflatten(-1, (hq, dim))
    k = qkv[..., hq * dim:(hq + hk) * dim].unflatten(-1, (hk, dim))
    v = qkv[..., (hq + hk) * dim:].unflatten(-1, (hk, dim))
    q, k = kernels.rotary(q, k, pos, freq, sections)
    c.write(k, v, slots)
    ck, cv = c.read(table, starts, total, dtype=x.dtype)
    att = torch.einsum("thd,shd->hts", q.float(), ck.repeat_interleave(hq // hk, 1).float())
    o = torch.einsum("hts,shd->thd", kernels.softmax(att * dim ** -0.5), cv.repeat_interleave(hq // hk, 1).float())
    y = o.to(x.dtype).reshape(x.shape[0], -1) @ w["o"]
    r, n, _, _ = kernels.residual_norm(x, y, w["g1"], w["gate"], w["g2"])
    gu = n @ w["gu"]
    f = gu.shape[-1] // 2
    h, _, _ = kernels.silu_mul_checkpoint8(gu[:, :f], gu[:, f:])
    return kernels.residual_norm(r, h @ w["down"], w["g1"], w["gate"], w["g2"])[:2], (q, ck, cv)


def test_a_block_with_all_of_them_eager_and_captured(kernels, cache):
    g = gen(31)
    T, d, hq, hk, dim, f, page = 24, 256, 4, 2, 64, 512, 16
    w = {n: randn(g, s, BF16, s[0] ** -0.5) for n, s in dict(qkv=(d, (hq + 2 * hk) * dim), o=(hq * dim, d), gu=(d, 2 * f),
                                                            down=(f, d)).items()}
    w.update(g0=torch.ones(d, device="cuda"), g1=1 + 0.1 * randn(g, (d,)), g2=1 + 0.1 * randn(g, (d,)), gate=randn(g, (d,), BF16))
    freq, sections = torch.exp(-torch.arange(32, device="cuda") * 0.2), (8, 12, 12)
    pos = torch.randint(0, 900, (3, T), generator=g, device="cuda")
    table = torch.tensor([[3, 1]], device="cuda")
    at = torch.arange(T, device="cuda")
    slots, starts = table[0][at // page] * page + at % page, torch.tensor([0, T], device="cuda")
    c = cache.QuantCache(4, page, hk, dim)
    x = randn(g, (T, d), BF16)
    args = (kernels, c, w, x, pos, slots, table, starts, freq, sections, hq, hk, dim, T)
    (r, n), (q, ck, cv) = block_step(*args)
    # the cache holds the turned keys to half a level of each head's largest value
    nn, _ = kernels.rmsnorm(x, w["g0"])
    k = (nn @ w["qkv"])[..., hq * dim:(hq + hk) * dim].unflatten(-1, (hk, dim))
    kt, m = rotary_ref(k[None], pos[:, None], freq, sections, False, False)
    amax = kt[0].abs().amax(-1, keepdim=True)
    # half a level, a bf16 rounding of the turned key before and of the read value after it
    assert ((ck.double() - kt[0]).abs() <= amax * (1 / 254 + 2.0 ** -8 + 2.0 ** -8)).all()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        block_step(*args)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (gr, gn), _ = block_step(*args)
    x2 = randn(g, (T, d), BF16)
    x.copy_(x2)
    c.k_scale.zero_()
    graph.replay()
    torch.cuda.synchronize()
    (r2, n2), _ = block_step(*args)
    assert torch.equal(gr, r2) and torch.equal(gn, n2) and not torch.equal(r2, r)


def test_backward_calls_captured_twice_and_replayed_side_by_side(kernels):
    """Two graphs of the backward pass replayed on two streams at once: each owns its scratch."""
    g = gen(32)
    shape = (4, 500, 1024)
    gam, gate = torch.ones(1024, device="cuda"), randn(g, (4, 1, 1024), BF16)
    inv = torch.ones(2000, device="cuda")
    sets, graphs, outs = [], [], []
    for i in range(2):
        t = [randn(g, shape, BF16) for _ in range(4)]
        kept = kernels.checkpoint8(t[3])
        sets.append((t, kept))
        kernels.residual_norm_backward(*t, inv, inv, gam, gate, gam)
    torch.cuda.synchronize()
    for t, kept in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = kernels.residual_norm_backward(*t, inv, inv, gam, gate, gam) + kernels.rmsnorm_backward(t[0], kept, inv, gam)
        graphs.append(graph)
        outs.append(o)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for (t, kept), o in zip(sets, outs):
        want = kernels.residual_norm_backward(*t, inv, inv, gam, gate, gam) + kernels.rmsnorm_backward(t[0], kept, inv, gam)
        assert all(torch.equal(p, q) for p, q in zip(o, want))


def test_launches_go_to_the_current_stream(kernels, cache):
    """A chain on a side stream, ordered by that stream alone."""
    g = gen(33)
    x = randn(g, (4096, 2048), BF16)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = x * 2
        c = kernels.checkpoint8(y)
        r, n, i1, i2 = kernels.residual_norm(y, kernels.checkpoint8_restore(c))
        from vibetensor_b200 import _lib
        assert _lib.last_launch_info().stream == s.cuda_stream
    s.synchronize()
    y2 = x * 2
    r2, *_ = kernels.residual_norm(y2, kernels.checkpoint8_restore(kernels.checkpoint8(y2)))
    assert torch.equal(r, r2)


# ------------------------------------------------------------------------------- guard bands
def guarded(n, dtype, offset):
    buf = torch.full((n + 64,), 3, dtype=torch.int8 if dtype == torch.int8 else dtype, device="cuda")
    return buf, buf[offset:offset + n]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,cols,off", [(5, 136, 16), (5, 137, 16), (3, 4096, 16), (3, 136, 3), (2, 20001, 16), (1, 1, 1)])
def test_nothing_is_written_outside_the_outputs(dtype, rows, cols, off):
    """The C entry points on outputs in the middle of sentinel-filled buffers, at ragged widths and
    unaligned bases."""
    from vibetensor_b200 import _lib
    L = _lib.lib()
    g = gen(cols)
    code, stream = _lib.dtype_code(dtype), _lib.stream_ptr(torch.empty(1, device="cuda"))
    x, y, d = (randn(g, (rows, cols), dtype) for _ in range(3))
    groups = -(-cols // 128)
    gam = torch.ones(cols, device="cuda")
    inv = torch.ones(rows, device="cuda")
    bufs = []

    def out(n, dt):
        buf, view = guarded(n, dt, off)
        bufs.append((buf, n))
        return view
    r, n = out(rows * cols, dtype), out(rows * cols, dtype)
    i1, i2 = out(rows, F32), out(rows, F32)
    _lib.check(L.vbt_b200_residual_norm(r.data_ptr(), n.data_ptr(), i1.data_ptr(), i2.data_ptr(), x.data_ptr(), y.data_ptr(),
                                        gam.data_ptr(), gam.to(dtype).data_ptr(), gam.data_ptr(), code, rows, cols, cols,
                                        cols, 0, rows, 1.0, 1.0, 1e-6, 3, stream))
    need = ctypes.c_size_t()
    _lib.check(L.vbt_b200_residual_norm_backward_workspace_bytes(rows, cols, code, rows, 0, ctypes.byref(need)))
    ws = out(need.value, torch.int8)
    if ws.data_ptr() % 4:                              # scratch is taken at float alignment
        bufs.pop()
        ws = torch.empty(need.value + 16, dtype=torch.int8, device="cuda")
    dx, dy = out(rows * cols, dtype), out(rows * cols, dtype)
    dg1, dg2, dgate = out(cols, F32), out(cols, F32), out(cols, dtype)
    gate = gam.to(dtype)
    _lib.check(L.vbt_b200_residual_norm_backward(
        dx.data_ptr(), dy.data_ptr(), dg1.data_ptr(), dgate.data_ptr(), dg2.data_ptr(), x.data_ptr(), d.data_ptr(), y.data_ptr(),
        x.data_ptr(), inv.data_ptr(), inv.data_ptr(), gam.data_ptr(), gate.data_ptr(), gam.data_ptr(), code, rows, cols, cols,
        cols, cols, cols, 0, rows, 1.0, 1.0, 3, ws.data_ptr(), need.value, stream))
    q, sc = out(rows * cols, torch.int8), out(rows * groups, F32)
    _lib.check(L.vbt_b200_checkpoint8(q.data_ptr(), sc.data_ptr(), x.data_ptr(), code, 0, rows, cols, cols, stream))
    o = out(rows * cols, dtype)
    _lib.check(L.vbt_b200_checkpoint8_restore(o.data_ptr(), q.data_ptr(), sc.data_ptr(), code, 0, rows, cols, stream))
    o2, i3, q2, s2 = out(rows * cols, dtype), out(rows, F32), out(rows * cols, torch.int8), out(rows * groups, F32)
    _lib.check(L.vbt_b200_rmsnorm_checkpoint8(o2.data_ptr(), i3.data_ptr(), q2.data_ptr(), s2.data_ptr(), x.data_ptr(),
                                              gam.data_ptr(), code, 0, rows, cols, cols, 1e-6, stream))
    assert torch.equal(q, q2) and torch.equal(sc, s2)
    _lib.check(L.vbt_b200_rmsnorm_backward8_workspace_bytes(rows, cols, code, 0, ctypes.byref(need)))
    ws2 = torch.empty(need.value, dtype=torch.int8, device="cuda")
    dx2, dg3 = out(rows * cols, dtype), out(cols, F32)
    _lib.check(L.vbt_b200_rmsnorm_backward8(dx2.data_ptr(), dg3.data_ptr(), d.data_ptr(), q.data_ptr(), sc.data_ptr(),
                                            inv.data_ptr(), gam.data_ptr(), code, 0, rows, cols, cols, ws2.data_ptr(), need.value,
                                            stream))
    h, qa, sa, qb, sb = out(rows * cols, dtype), out(rows * cols, torch.int8), out(rows * groups, F32), \
        out(rows * cols, torch.int8), out(rows * groups, F32)
    _lib.check(L.vbt_b200_silu_mul(h.data_ptr(), qa.data_ptr(), sa.data_ptr(), qb.data_ptr(), sb.data_ptr(), x.data_ptr(),
                                   y.data_ptr(), code, 1, rows, cols, cols, cols, stream))
    da, db = out(rows * cols, dtype), out(rows * cols, dtype)
    _lib.check(L.vbt_b200_silu_mul_backward(da.data_ptr(), db.data_ptr(), d.data_ptr(), qa.data_ptr(), sa.data_ptr(),
                                            qb.data_ptr(), sb.data_ptr(), code, 1, rows, cols, cols, cols, cols, stream))
    torch.cuda.synchronize()
    for buf, n in bufs:
        assert (buf[:off] == 3).all() and (buf[off + n:] == 3).all()


# ---------------------------------------------------------------------------------- refusals
def test_refusals(kernels, cache):
    g = gen(1)
    x = randn(g, (4, 8, 64))
    cpu = torch.ones(4, 8, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.residual_norm(cpu, cpu)
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.residual_norm(x, cpu)
    with pytest.raises(TypeError):
        kernels.residual_norm(x, x.bfloat16())
    with pytest.raises(TypeError):
        kernels.residual_norm(x.long(), x.long())
    with pytest.raises(ValueError, match="shape"):
        kernels.residual_norm(x, x[:3])
    with pytest.raises(TypeError, match="gamma_post"):
        kernels.residual_norm(x, x, torch.ones(63, device="cuda"))
    with pytest.raises(ValueError, match="switched off"):
        kernels.residual_norm(x, x, torch.ones(64, device="cuda"), post_norm=False)
    for shape in ((63,), (8, 64), (1, 8, 64), (4, 8, 1), (4, 1, 63), (2, 1, 64)):
        with pytest.raises(ValueError, match="broadcast"):
            kernels.residual_norm(x, x, gate=torch.ones(shape, device="cuda"))
    with pytest.raises(TypeError, match="gate"):
        kernels.residual_norm(x, x, gate=torch.ones(64, device="cuda", dtype=BF16))
    i = torch.ones(32, device="cuda")
    with pytest.raises(ValueError, match="no gradient"):
        kernels.residual_norm_backward(None, None, x, x, i, i)
    with pytest.raises(ValueError, match="grad_n and r"):
        kernels.residual_norm_backward(x, None, x, x, i, i)
    with pytest.raises(ValueError, match="without inv_pre"):
        kernels.residual_norm_backward(x, x, x, x, i, None)
    with pytest.raises(ValueError, match="y is needed"):
        kernels.residual_norm_backward(x, x, None, x, i, i)
    with pytest.raises(TypeError, match="inv_pre"):
        kernels.residual_norm_backward(x, x, x, x, i, i[:5])
    with pytest.raises(ValueError, match="fmt"):
        kernels.checkpoint8(x, "int4")
    with pytest.raises(TypeError):
        kernels.checkpoint8(x.double())
    c = kernels.checkpoint8(x)
    with pytest.raises(TypeError):
        kernels.checkpoint8_restore(c, torch.float64)
    with pytest.raises(TypeError, match="same dtype"):
        kernels.rmsnorm_backward(x.bfloat16(), c, i)
    with pytest.raises(ValueError, match="same shape"):
        kernels.rmsnorm_backward(x[:2], c, i)
    with pytest.raises(TypeError, match="both"):
        kernels.silu_mul_backward(x, c, x)
    with pytest.raises(ValueError, match="two formats"):
        kernels.silu_mul_backward(x, c, kernels.checkpoint8(x, "e4m3"))
    bad = kernels.Checkpoint8(c.q, c.scale[:3], "int8", F32)
    with pytest.raises(ValueError, match="do not match"):
        kernels.checkpoint8_restore(bad)
    q, f = randn(g, (2, 5, 3, 64)), torch.ones(32, device="cuda")
    pos = torch.zeros((2, 5), dtype=torch.int64, device="cuda")
    for call, exc in ((lambda: kernels.rotary(q[0, 0], None, pos, f), ValueError), (lambda: kernels.rotary(q, q[:1], pos, f), ValueError),
                      (lambda: kernels.rotary(q, q.bfloat16(), pos, f), TypeError), (lambda: kernels.rotary(q, None, pos, f.double()), TypeError),
                      (lambda: kernels.rotary(q, None, pos.bool(), f), TypeError),
                      (lambda: kernels.rotary(q, None, pos, torch.ones(33, device="cuda")), ValueError),
                      (lambda: kernels.rotary(q, None, pos, f, (16, 16)), ValueError),
                      (lambda: kernels.rotary(q, None, pos[None], f, (31,)), ValueError),
                      (lambda: kernels.rotary(q, None, pos[:, :4], f), ValueError),
                      (lambda: kernels.rotary(q, None, pos, f, out=(q[:1], None)), ValueError),
                      (lambda: kernels.rotary(q[:, 1:], None, pos[:, 1:], f, out=(q[:, :-1], None)), ValueError),
                      (lambda: kernels.rotary(q, q, pos, f, out=(q, q)), ValueError),
                      (lambda: kernels.rotary(q, None, pos, f, out=(q[:, :1].expand(2, 5, 3, 64), None)), ValueError),
                      (lambda: kernels.rotary(q, None, pos.cpu(), f), RuntimeError)):
        with pytest.raises(exc):
            call()
    kv = cache.QuantCache(2, 4, 3, 16)
    k, s = randn(g, (5, 3, 16)), torch.arange(5, device="cuda")
    for call, exc in ((lambda: kv.write(k, k[:4], s), ValueError), (lambda: kv.write(k, k.half(), s), TypeError),
                      (lambda: kv.write(k, k, s.float()), TypeError), (lambda: kv.write(k, k, s[None]), ValueError),
                      (lambda: kv.write(k.cpu(), k, s), RuntimeError), (lambda: kv.read(s[None], s[:3], 4), ValueError),
                      (lambda: kv.read(s[None], s[:2].int(), 4), TypeError), (lambda: kv.read(s[None], s[:2]), ValueError),
                      (lambda: kv.read(s[None], s[:2], 4, dtype=torch.float64), TypeError),
                      (lambda: kv.read(s[None], s[:2], out=(k, k[:4])), ValueError),
                      (lambda: kv.read(s[None], s[:2], out=(k, k)), ValueError),
                      (lambda: cache.QuantCache(2, 4, 3, 16, fmt="int4"), ValueError), (lambda: cache.QuantCache(0, 4, 3, 16), ValueError),
                      (lambda: cache.QuantCache(2, 4, 3, 16, device="cpu"), RuntimeError)):
        with pytest.raises(exc):
            call()


# ------------------------------------------------------------------------ views with an axis of one
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols", [64, 129, 1024])
def test_parts_of_a_projection_with_one_token_or_row_per_sample(kernels, dtype, cols):
    """[batch, 1, k * cols] cut along its last axis: a modulation row per sample, or the one new token of
    each request.  Every sample's own row counts, as in the dense copy of the part."""
    g = gen(cols + 1)
    batch, tokens = 5, 7
    gam = 1 + 0.1 * randn(g, (cols,))
    mod = randn(g, (batch, 1, 6 * cols), dtype)
    x, y, dr, dn = (randn(g, (batch, tokens, cols), dtype) for _ in range(4))

    def same(call, *views):
        # the reads of an unaligned part go another way, the arithmetic per value does not
        got, want = call(*views), call(*(v.contiguous() for v in views))
        for a, b in zip(got, want):
            if a is not None:
                close("a part of a projection", a, b.double(), b.double().abs() + 1.0)
    for i in (1, 5):
        gate = mod.chunk(6, -1)[i]
        assert not gate.is_contiguous()
        r, n, i1, i2 = kernels.residual_norm(x, y, gam, gate, gam)
        w = join_ref(x, y, gam, gate, gam, 1e-6, True, True, 1.0, 1.0)
        close("residual_norm r, a part as the gate", r, w["r"], w["mass"])
        got = dict(zip(("dx", "dy", "dgp", "dgate", "dgn"),
                       kernels.residual_norm_backward(dr, dn, y, r, i1, i2, gam, gate, gam)))
        for name, (t, mass) in join_bwd_ref(dr, dn, y, r, i1, i2, gam, gate, gam, 1.0, 1.0).items():
            close(f"residual_norm_backward {name}, a part as the gate", got[name], t, mass)
    new = mod[..., cols:2 * cols], mod[..., 3 * cols:4 * cols]     # [batch, 1, cols]
    inv = torch.rand(batch, generator=g, device="cuda") + 0.5
    same(lambda a, b: kernels.residual_norm(a, b, gam, None, gam), *new)
    same(lambda a, b: kernels.residual_norm_backward(a, b, b, a, inv, inv, gam, a, gam), *new)
    same(lambda a, b: (kernels.silu_mul(a, b),), *new)
    same(lambda a, b: kernels.silu_mul_backward(b, a, b), *new)
    same(lambda a: (kernels.checkpoint8_restore(kernels.checkpoint8(a)),), new[0])
    same(lambda a, b: kernels.silu_mul_backward(b, kernels.checkpoint8(a), kernels.checkpoint8(b)), *new)
    same(lambda a: kernels.rmsnorm_checkpoint8(a, gam)[:2], new[0])
    same(lambda a, b: kernels.rmsnorm_backward(b, kernels.checkpoint8(a), inv, gam), *new)
    same(lambda a: kernels.rmsnorm(a, gam), new[0])
    same(lambda a, b: kernels.rmsnorm_backward(b, a, inv, gam), *new)
    same(lambda a: (kernels.softmax(a), kernels.log_softmax(a)), new[0])
    same(lambda a, b: (kernels.softmax_backward(a, b), kernels.log_softmax_backward(a, b)), *new)


# ---------------------------------------------------------------------------- rows of any magnitude
def row_steps(cols):
    """Roundings on the longest path of a gradient of one row, K of ``close``: a thread adds up at most
    16 values (one of every 512 in the kernels for rows of any length), a warp has 5 levels, a row at
    most one warp per 256 values and no more than 128; the products around the sums are at most 14."""
    return max(16, -(-cols // 512)) + 5 + min(128, -(-cols // 256)) + 14


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols", [64, 333, 512, 1365, 4096, 16400, 70001])
def test_gradients_of_rows_of_any_magnitude(kernels, dtype, cols):
    """A norm's gradient is that of its row's direction over the row's size: it keeps its relative
    accuracy for rows as large as the forward pass takes and, with a small eps, as small."""
    g = gen(cols + 2)
    shape, k = (2, 3, cols), row_steps(cols) + 6    # six rows for a column sum
    gp, gn = 1 + 0.1 * randn(g, (cols,)), 1 + 0.1 * randn(g, (cols,))
    for rms_y, rms_r, top in ((1e17, 1.0, 1.0), (1.0, 1e17, 1.0), (3e16, 1e17, 1e-3), (1e15, 3e13, 1e-6), (1e-15, 1e-12, 1.0),
                              (1e-17, 1e-17, 10.0), (1e-16, 1e16, 1.0)):
        y, r = randn(g, shape, dtype, rms_y), randn(g, shape, dtype, rms_r)
        # what arrives at r and at n moves the stream by about the same
        dr, dn = randn(g, shape, dtype, top / rms_r), randn(g, shape, dtype, top)
        i1 = y.double().pow(2).mean(-1).rsqrt().float().reshape(-1)
        i2 = r.double().pow(2).mean(-1).rsqrt().float().reshape(-1)
        for kind in ("none", "sample", "full"):
            gate = gate_for(g, kind, shape, dtype)
            got = dict(zip(("dx", "dy", "dgp", "dgate", "dgn"), kernels.residual_norm_backward(dr, dn, y, r, i1, i2, gp, gate, gn)))
            for name, (t, mass) in join_bwd_ref(dr, dn, y, r, i1, i2, gp, gate, gn, 1.0, 1.0).items():
                close(f"residual_norm_backward {name}, any magnitude", got[name], t, mass, k)
    z, d = torch.zeros(shape, dtype=dtype, device="cuda"), randn(g, shape, dtype, 1e-6)
    i = torch.full((6,), 1e15, device="cuda")      # zero rows and an eps of 1e-30
    dx, dy, dgp, _, dgn = kernels.residual_norm_backward(None, d, z, z, i, i, gp, None, gn)
    want = d.double() * gn.double() * 1e15
    close("residual_norm_backward dx, zero rows", dx, want, want.abs(), k)
    want = want * gp.double() * 1e15
    close("residual_norm_backward dy, zero rows", dy, want, want.abs(), k)
    assert (dgp == 0).all() and (dgn == 0).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols", [64, 333, 512, 1365, 4096, 16384, 20001])
def test_rmsnorm_gradients_from_8_bits_of_rows_of_any_magnitude(kernels, fmt, dtype, cols):
    g = gen(cols + 3)
    gamma = 1 + 0.1 * randn(g, (cols,))
    k = row_steps(cols) + -(-cols // 256) - min(128, -(-cols // 256)) + 7   # seven rows for a column sum
    for rms, top in ((1e17, 1.0), (1e15, 1e-6), (3e13, 1.0), (1e-12, 1.0), (1e-17, 10.0)):
        x, dy = randn(g, (7, cols), dtype, rms), randn(g, (7, cols), dtype, top)
        inv = x.double().pow(2).mean(-1).rsqrt().float()
        c = kernels.checkpoint8(x, fmt)
        kept = c.q.double() * c.scale.double().repeat_interleave(128, 1)[:, :cols]
        for gam in (gamma, None):
            dx, dgamma = kernels.rmsnorm_backward(dy, c, inv, gam)
            want = join_bwd_ref(None, dy, None, kept, None, inv, None, None, gam, 1.0, 1.0)
            close("rmsnorm_backward of a checkpoint, dx, any magnitude", dx, *want["dx"], k)
            if gam is not None:
                close("rmsnorm_backward of a checkpoint, dgamma, any magnitude", dgamma, *want["dgn"], k)
    z, d = kernels.checkpoint8(torch.zeros((7, cols), dtype=dtype, device="cuda"), fmt), randn(g, (7, cols), dtype, 1e-6)
    dx, dgamma = kernels.rmsnorm_backward(d, z, torch.full((7,), 1e15, device="cuda"), gamma)   # an eps of 1e-30
    want = d.double() * gamma.double() * 1e15
    close("rmsnorm_backward of a checkpoint, zero rows", dx, want, want.abs(), k)
    assert (dgamma == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_silu_mul_keeps_what_exp_leaves(kernels, dtype):
    """Down to where exp(-gate) overflows (gate = -88.72) the activation is a number of 1e-37, and a
    large factor brings it back.  The sigmoid is below the normal numbers there: up to 2^-23 of it
    (u = 2^-24 is 2 of these at most four times over), besides the usual eight roundings."""
    a = torch.linspace(-88.7, -80, 301, device="cuda").to(dtype)
    a = a[a >= -88.72]
    b, d = torch.full_like(a, 1e30), torch.full_like(a, 3.0)
    (hw, hm), (daw, dam), (dbw, dbm) = silu_ref(d, a, b)
    # the exponent's argument is rounded: |gate| u, and exp by 2 u beside it
    k = 88.72 * 2 + 16
    close("silu_mul near exp's end", kernels.silu_mul(a, b), hw, hm, k)
    da, db = kernels.silu_mul_backward(d, a, b)
    close("silu_mul_backward gate near exp's end", da, daw, dam, k)
    close("silu_mul_backward up near exp's end", db, dbw, dbm, k)


# ---------------------------------------------------------------------- more rows than fit the card
def column_steps(rows, cols, per):
    """Roundings on the longest path of a sum over rows: a worker -- one of at least 148, or 16 clusters
    where blocks share a row -- takes at most twice its share one after the other, the rows of one gate row
    at most all, and a fold adds at most 64 partial rows per thread and 15 levels."""
    return 2 * -(-rows // (16 if cols > 8192 else 148)) + per + 80


# rows well above the workers of a launch and no multiple of them, gate rows in numbers around them, rows
# per gate row that a warp's rows at once do not divide
MANY = [((1819, 11), 64), ((6670, 3), 120), ((20011, 1), 130), ((1297, 7), 200), ((9007,), 333), ((811, 7), 512), ((8, 769), 1365),
        ((3001,), 1000), ((43, 70), 4096), ((37, 41), 4095), ((29, 53), 5000), ((601, 2), 8192), ((3, 117), 12345), ((4, 90), 16384),
        ((2, 151), 20001), ((2, 307), 66000)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lead,cols", MANY)
def test_residual_norm_and_backward_of_many_rows(kernels, dtype, lead, cols):
    g = gen(cols + 4)
    shape, rows = lead + (cols,), int(np.prod(lead))
    k = row_steps(cols)
    x, y, dr, dn = (randn(g, shape, dtype) for _ in range(4))
    gp, gn = 1 + 0.1 * randn(g, (cols,)), 1 + 0.1 * randn(g, (cols,))
    for kind in ("none", "sample", "channel", "full"):
        if kind == "sample" and len(lead) == 1 or kind == "full" and rows * cols > 1 << 24:
            continue
        gate = gate_for(g, kind, shape, dtype)
        r, n, i1, i2 = kernels.residual_norm(x, y, gp, gate, gn, 1e-6, residual_scale=0.7, branch_scale=1.3)
        w = join_ref(x, y, gp, gate, gn, 1e-6, True, True, 0.7, 1.3)
        close("residual_norm r, many rows", r, w["r"], w["mass"], k)
        close("residual_norm n, many rows", n, w["n"], w["n_mass"], k)
        close("residual_norm inv_post, many rows", i1, w["i1"], w["i1"], k)
        close("residual_norm inv_pre, many rows", i2, w["i2"], w["i2"] * (1 + 2 * w["rho"]), k)
        del w, n
        got = dict(zip(("dx", "dy", "dgp", "dgate", "dgn"), kernels.residual_norm_backward(
            dr, dn, y, r, i1, i2, gp, gate, gn, residual_scale=0.7, branch_scale=1.3)))
        want = join_bwd_ref(dr, dn, y, r, i1, i2, gp, gate, gn, 0.7, 1.3)
        per = rows // lead[0] if kind == "sample" else 0
        for name, (t, mass) in want.items():
            over = 0 if name in ("dx", "dy") else column_steps(rows, cols, per)
            close(f"residual_norm_backward {name}, many rows", got[name], t, mass, k + over)
        del want, got


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,cols", [(20011, 64), (20011, 130), (9007, 200), (9007, 333), (6151, 512), (6151, 1365), (3001, 4096),
                                       (1507, 4095), (1507, 8192), (613, 16384), (1811, 20001)])
def test_rmsnorm_kept_in_8_bits_of_many_rows(kernels, fmt, dtype, rows, cols):
    g = gen(cols + 5)
    k = row_steps(cols) + max(0, -(-cols // 256) - 128)
    x, dy, gamma = acts(g, (rows, cols), dtype), randn(g, (rows, cols), dtype), 1 + 0.1 * randn(g, (cols,))
    out, inv, c = kernels.rmsnorm_checkpoint8(x, gamma, 1e-6, fmt)
    flat = kernels.checkpoint8(x, fmt)                 # compared bit for bit with the host's elsewhere
    assert torch.equal(c.q.view(torch.int8), flat.q.view(torch.int8)) and torch.equal(c.scale, flat.scale)
    some = torch.randint(0, rows, (64,), generator=g, device="cuda")
    check_held(kernels.Checkpoint8(c.q[some], c.scale[some], fmt, dtype), x[some], fmt)
    w = join_ref(x, x, None, None, gamma, 1e-6, False, True, 1.0, 0.0)
    close("rmsnorm_checkpoint8 out, many rows", out, w["n"], w["n"].abs(), k)
    close("rmsnorm_checkpoint8 inv_rms, many rows", inv, w["i2"], w["i2"], k)
    del w
    dx, dgamma = kernels.rmsnorm_backward(dy, c, inv, gamma)
    kept = kernels.checkpoint8_restore(c, F32)
    want = join_bwd_ref(None, dy, None, kept, None, inv, None, None, gamma, 1.0, 1.0)
    close("rmsnorm_backward of a checkpoint, dx, many rows", dx, *want["dx"], k)
    close("rmsnorm_backward of a checkpoint, dgamma, many rows", dgamma, *want["dgn"], k + column_steps(rows, cols, 0))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,t,hq,hk,dim,half,sections", [(7, 2857, 2, 1, 64, 32, (8, 12, 12)), (1, 20011, 1, 1, 32, 16, (16,)),
                                                         (3, 4001, 3, 2, 80, 20, (5, 15)), (1201, 5, 4, 1, 40, 20, (7, 6, 7)),
                                                         (2, 3989, 2, 2, 7, 3, (1, 2)), (64, 300, 1, 1, 8, 4, (1, 1, 1, 1)),
                                                         (5, 1201, 8, 2, 128, 64, (16, 24, 24))])
def test_rotary_several_tokens_per_block(kernels, dtype, interleaved, b, t, hq, hk, dim, half, sections):
    """Enough tokens that a block takes several of them, across the samples' ends and with a ragged last
    block; queries and keys are parts of one projection."""
    g = gen(t)
    freq = torch.exp(-torch.arange(half, device="cuda") * 0.13)
    qkv = randn(g, (b, t, (hq + 2 * hk) * dim), dtype)
    q, k = qkv[..., :hq * dim].unflatten(-1, (hq, dim)), qkv[..., hq * dim:(hq + hk) * dim].unflatten(-1, (hk, dim))
    pos = torch.randint(-10, 2000000, (len(sections), b, t), generator=g, device="cuda")
    for inverse, call in ((False, kernels.rotary), (True, kernels.rotary_backward)):
        for x, o in zip((q, k), call(q, k, pos, freq, sections, interleaved)):
            want, mass = rotary_ref(x, pos, freq, sections, interleaved, inverse)
            close("rotary, several tokens per block", o, want, mass, 8)
            assert torch.equal(o[..., 2 * half:], x[..., 2 * half:])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lead,cols", [((400, 9), 4096), ((100, 40), 4096), ((1200, 23), 1365), ((70, 90), 1365), ((9000, 50), 64),
                                       ((40, 333), 200), ((97, 40), 16384), ((300, 7), 20001), ((2, 1), 4096), ((3, 2), 64),
                                       ((700, 5), 33000), ((90, 8), 70001)])
def test_gate_rows_that_are_cut(kernels, dtype, lead, cols):
    """Gate rows fewer and more than the workers of a launch, of more and fewer rows than a worker takes:
    whole ones, ones that two workers share and ones that many do."""
    g = gen(lead[0])
    shape, rows = lead + (cols,), lead[0] * lead[1]
    if rows * cols > 1 << 26:
        shape, rows = (lead[0] // 5,) + shape[1:], lead[0] // 5 * lead[1]
    y, r, dr, dn = (randn(g, shape, dtype) for _ in range(4))
    gp, gn, gate = 1 + 0.1 * randn(g, (cols,)), 1 + 0.1 * randn(g, (cols,)), gate_for(g, "sample", shape, dtype)
    i1, i2 = (t.float().pow(2).mean(-1).add(1e-6).rsqrt().reshape(-1) for t in (y, r))
    got = dict(zip(("dx", "dy", "dgp", "dgate", "dgn"), kernels.residual_norm_backward(dr, dn, y, r, i1, i2, gp, gate, gn)))
    k = row_steps(cols)
    for name, (t, mass) in join_bwd_ref(dr, dn, y, r, i1, i2, gp, gate, gn, 1.0, 1.0).items():
        over = 0 if name in ("dx", "dy") else column_steps(rows, cols, shape[1])
        close(f"residual_norm_backward {name}, gate rows cut", got[name], t, mass, k + over)
