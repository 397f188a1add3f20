"""The bandwidth-bound work around a transformer block's matrix products, as measurable cases.

Four operators: the join of a branch with the residual stream between two RMS norms (``join``),
activations kept in 8 bits for the backward pass (``keep``), rotary positions with several axes
(``rotary``) and a paged key/value cache in 8 bits (``cache``).  Each case is one pass a user's
program makes.  With ``own`` false ``run`` computes the plain form in elementary torch operations;
with ``own`` true it calls this package.  ``exact`` is the definition in 64 bits, written apart.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}
GROUP = 128           # values that share a scale in an 8-bit activation
TINY = 2.0 ** -119    # a group whose largest magnitude is below this is held as zeros
TOP = {"int8": 127.0, "e4m3": 448.0}
EPS = 1e-6


# ------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one decoding step of 16 requests between two blocks: launch latency is what counts
        dict(name="join decode", op="join", way="forward", dtype="bfloat16", rows=16, cols=4096, gate="none",
             per=16, post=True, pre=True),
        # training, eight samples of 4096 tokens, one modulation row per sample
        dict(name="join training forward", op="join", way="forward", dtype="bfloat16", rows=32768, cols=4096,
             gate="group", per=4096, post=True, pre=True),
        dict(name="join training backward", op="join", way="backward", dtype="bfloat16", rows=32768, cols=4096,
             gate="group", per=4096, post=True, pre=True),
        # a width that no vector divides, 32-bit, one learned gate per channel
        dict(name="join odd backward", op="join", way="backward", dtype="float32", rows=6151, cols=1365,
             gate="channel", per=6151, post=True, pre=True),
        # a short sequence's activations into 8 bits and back, a width with a ragged last group
        dict(name="keep short", op="keep", what="round", fmt="int8", dtype="float16", rows=77, cols=5000),
        # a norm's forward and backward pass with its input kept in 8 bits between them
        dict(name="keep norm", op="keep", what="norm", fmt="e4m3", dtype="bfloat16", rows=32768, cols=4096),
        # a gated activation's forward and backward pass, both factors kept in 8 bits
        dict(name="keep gated", op="keep", what="gated", fmt="int8", dtype="bfloat16", rows=16384, cols=8192),
        # one new token of 64 requests at far positions
        dict(name="rotary decode", op="rotary", way="forward", dtype="bfloat16", batch=64, tokens=1, hq=32, hk=8, dim=128,
             sections="16,24,24", paired=False),
        # a clip of 8 frames of 48 x 48 patches, the axes are time, height and width
        dict(name="rotary video", op="rotary", way="forward", dtype="bfloat16", batch=1, tokens=18432, hq=32, hk=8, dim=128,
             sections="16,24,24", paired=False),
        # gradients of images' queries and keys, neighbouring pairs, part of a head left unrotated
        dict(name="rotary image backward", op="rotary", way="backward", dtype="float32", batch=3, tokens=1531, hq=6, hk=2,
             dim=80, sections="16,16", paired=True),
        # one decoding step: 64 requests add a token each and their whole contexts are read
        dict(name="cache decode", op="cache", fmt="int8", dtype="bfloat16", seqs=64, least=200, most=8000, fresh=1,
             page=16, heads=8, dim=128),
        # short prompts written whole, odd lengths, pages that end inside a tile
        dict(name="cache prompts", op="cache", fmt="e4m3", dtype="float16", seqs=5, least=90, most=700, fresh=700,
             page=48, heads=3, dim=80),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.4 else max(lo, n // 64 * 64)


def draw(rng):
    op = rng.choice(["join", "keep", "rotary", "cache"])
    dtype = rng.choice(["float32", "float16", "bfloat16", "bfloat16"])
    fmt = rng.choice(["int8", "e4m3"])
    scale = SIZE[dtype] // 2
    if op == "join":
        cols = _width(rng, 64, 16384)
        rows = _log(rng, 1, max(2, min(32768, (1 << 27) // (cols * scale))))
        gate = rng.choice(["none", "channel", "group", "full"])
        per = rows
        if gate == "group":
            per = max(1, _log(rng, 1, rows))
            rows = rows // per * per
        post = rng.random() < 0.8
        pre = rng.random() < 0.8 or not post
        return dict(op=op, way=rng.choice(["forward", "backward"]), dtype=dtype, rows=rows, cols=cols, gate=gate,
                    per=per, post=post, pre=pre)
    if op == "keep":
        cols = _width(rng, 64, 16384)
        rows = _log(rng, 1, max(2, min(32768, (1 << 27) // (cols * scale))))
        return dict(op=op, what=rng.choice(["round", "norm", "gated"]), fmt=fmt, dtype=dtype, rows=rows, cols=cols)
    if op == "rotary":
        dim = rng.choice([32, 40, 64, 72, 80, 96, 128, 128, 160, 256])
        hk = rng.choice([1, 2, 3, 4, 8])
        hq = hk * rng.choice([1, 2, 4, 5])
        batch = rng.choice([1, 2, 3, 16, 64])
        most = (1 << 26) // (batch * (hq + hk) * dim * scale)
        tokens = 1 if rng.random() < 0.3 else _log(rng, 2, max(3, min(20000, most)))
        half = dim // 2 if rng.random() < 0.6 else dim // 4
        axes = rng.choice([1, 2, 3])
        cut = sorted(rng.randint(0, half) for _ in range(axes - 1))
        ends = cut + [half]
        sections = ",".join(str(e - b) for b, e in zip([0] + cut, ends))
        return dict(op=op, way=rng.choice(["forward", "backward"]), dtype=dtype, batch=batch, tokens=tokens, hq=hq, hk=hk,
                    dim=dim, sections=sections, paired=rng.random() < 0.5)
    heads = rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([32, 64, 72, 80, 96, 128, 128, 160, 256])
    seqs = _log(rng, 1, 64)
    most = max(8, min(8000, (1 << 27) // (seqs * heads * dim * scale)))
    most = _log(rng, 8, most)
    least = max(1, _log(rng, 1, most))
    fresh = 1 if rng.random() < 0.5 else _log(rng, 1, most)
    return dict(op=op, fmt=fmt, dtype=dtype, seqs=seqs, least=least, most=most, fresh=fresh,
                page=rng.choice([1, 16, 16, 32, 48, 64, 128]), heads=heads, dim=dim)


def _sections(case):
    """Pairs of a head that turn with each axis' position."""
    return [int(n) for n in case["sections"].split(",")]


def _lengths(case):
    """The requests' context lengths, spread over the logarithm of their range; fixed by the case."""
    n, lo, hi = case["seqs"], case["least"], case["most"]
    return [int(round(lo * (hi / lo) ** (((7 * i + 3) % n + 0.5) / n))) for i in range(n)]


def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "join":
        n, d = case["rows"], case["cols"]
        g = {"none": 0, "channel": d, "group": n // case["per"] * d, "full": n * d}[case["gate"]]
        norms = 4 * (d + n) * (case["post"] + case["pre"])
        if case["way"] == "forward":   # x and y are read, the stream and the next norm are written
            return dict(bytes=e * (n * d * (3 + case["pre"]) + g) + norms, flops=n * d * (3 + 4 * case["post"] + 4 * case["pre"]))
        reads_y = case["post"] or case["gate"] != "none"
        return dict(bytes=e * (n * d * (3 + reads_y + 2 * case["pre"]) + 2 * g) + norms + 4 * d * (case["post"] + case["pre"]),
                    flops=n * d * (4 + 9 * case["post"] + 9 * case["pre"]))
    if case["op"] == "keep":
        n, d = case["rows"], case["cols"]
        q = n * d + 4 * n * (-(-d // GROUP))   # one kept tensor, written in one call and read in the other
        if case["what"] == "round":
            return dict(bytes=2 * e * n * d + 2 * q, flops=6 * n * d)
        if case["what"] == "norm":             # x, out, dy, dx and the kept x
            return dict(bytes=4 * e * n * d + 2 * q + 12 * n + 12 * d, flops=18 * n * d)
        return dict(bytes=6 * e * n * d + 4 * q, flops=40 * n * d)   # gate, up, out, dout, dgate, dup and two kept
    if case["op"] == "rotary":
        t = case["batch"] * case["tokens"]
        width = case["dim"] * (case["hq"] + case["hk"])
        half = sum(_sections(case))
        return dict(bytes=2 * e * t * width + 8 * t * len(_sections(case)) + 4 * half,
                    flops=t * (case["hq"] + case["hk"]) * half * 6)
    h, d = case["heads"], case["dim"]
    lens = _lengths(case)
    total, new = sum(lens), sum(min(case["fresh"], n) for n in lens)
    pages = sum(-(-n // case["page"]) for n in lens)
    return dict(bytes=2 * new * h * (d * (e + 1) + 4) + 8 * new + 2 * total * h * (d * (e + 1) + 4) + 8 * pages + 8 * case["seqs"],
                flops=2 * h * d * (new * 6 + total))


# ------------------------------------------------------------------------------ the inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(1000003 * seed + 17)


def _acts(g, shape, dtype, spread=1.0):
    """Activations: normal values, a few channels an order of magnitude louder than the others."""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(spread)
    loud = torch.rand(shape[-1], generator=g, device="cuda") < 0.01
    return x.mul_(torch.where(loud, 12.0, 1.0)).to(dtype)


def _gamma(g, cols):
    return 1.0 + 0.1 * torch.randn(cols, generator=g, device="cuda")


def prepare(case, seed):
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    return dict(case=case, **globals()["_prepare_" + case["op"]](case, g, dt))


def _prepare_join(case, g, dt):
    n, d = case["rows"], case["cols"]
    s = dict(gp=_gamma(g, d) if case["post"] else None, gn=_gamma(g, d) if case["pre"] else None, gate=None,
             alpha=1.0, beta=1.0 if case["gate"] != "none" else 0.25)
    if case["gate"] != "none":
        s["gate"] = (0.3 * torch.randn({"channel": (d,), "group": (n // case["per"], 1, d), "full": (n, d)}[case["gate"]],
                                       generator=g, device="cuda")).to(dt)
    shape = (n // case["per"], case["per"], d) if case["gate"] == "group" else (n, d)
    y = _acts(g, shape, dt, 0.8)
    if case["way"] == "forward":
        return dict(s, x=_acts(g, shape, dt, 2.0), y=y)
    # the forward pass left the stream and the two reciprocal norms; gradients come from the stream and the next block
    s["r"] = _acts(g, shape, dt, 2.0)
    s["y"] = y
    rows = lambda t: t.float().pow(2).mean(-1).add(EPS).rsqrt().reshape(-1)  # noqa: E731
    s["inv_post"] = rows(y) if case["post"] else None
    s["inv_pre"] = rows(s["r"]) if case["pre"] else None
    s["dr"] = torch.randn(shape, generator=g, device="cuda").mul_(0.01).to(dt)
    s["dn"] = torch.randn(shape, generator=g, device="cuda").mul_(0.01).to(dt) if case["pre"] else None
    return s


def _prepare_keep(case, g, dt):
    n, d = case["rows"], case["cols"]
    if case["what"] == "round":
        return dict(x=_acts(g, (n, d), dt))
    if case["what"] == "norm":
        return dict(x=_acts(g, (n, d), dt, 2.0), gamma=_gamma(g, d),
                    dy=torch.randn((n, d), generator=g, device="cuda").mul_(0.01).to(dt))
    both = _acts(g, (n, 2 * d), dt, 1.5)   # the two factors come out of one projection
    return dict(gate=both[:, :d], up=both[:, d:], dy=torch.randn((n, d), generator=g, device="cuda").mul_(0.01).to(dt))


def _prepare_rotary(case, g, dt):
    b, t, d = case["batch"], case["tokens"], case["dim"]
    sections = _sections(case)
    half, axes = sum(sections), len(sections)
    qkv = torch.randn((b, t, (case["hq"] + 2 * case["hk"]) * d), generator=g, device="cuda").to(dt)  # a fused projection
    q = qkv[..., :case["hq"] * d].unflatten(-1, (case["hq"], d))
    k = qkv[..., case["hq"] * d:(case["hq"] + case["hk"]) * d].unflatten(-1, (case["hk"], d))
    start = torch.randint(0, 1000000, (axes, b, 1), generator=g, device="cuda")
    step = torch.arange(t, device="cuda")
    across = max(1, int(math.sqrt(t / 2)))
    grid = [step // (across * across), step // across % across, step % across][-axes:] if axes > 1 else [step]
    pos = start + torch.stack(grid)[:, None, :]
    freq = torch.exp(torch.arange(half, device="cuda", dtype=torch.float64) * (-math.log(1e4) / max(half, 1))).float()
    which = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], device="cuda")
    return dict(q=q, k=k, pos=pos, freq=freq, sections=sections, which=which)


def _quantise(x, fmt):
    """x [..., n] in 32 bits -> (held values in 8 bits, scale [...]): one scale for the last dimension."""
    top = torch.full((), TOP[fmt], device=x.device)
    amax = x.abs().amax(-1)
    dead = amax < TINY
    inv = torch.where(dead, torch.zeros_like(amax), top / amax)
    scale = torch.where(dead, torch.zeros_like(amax), amax * (1.0 / top))
    z = x * inv.unsqueeze(-1)
    return (z.round().to(torch.int8) if fmt == "int8" else z.to(torch.float8_e4m3fn)), scale


def _prepare_cache(case, g, dt):
    h, d, page = case["heads"], case["dim"], case["page"]
    lens = _lengths(case)
    total = sum(lens)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda")
    table = torch.zeros((case["seqs"], max(need)), dtype=torch.int64, device="cuda")
    starts = torch.zeros(case["seqs"] + 1, dtype=torch.int64)
    slots, used = [], 0
    for i, n in enumerate(lens):
        mine = order[used:used + need[i]]
        table[i, :need[i]] = mine
        used += need[i]
        starts[i + 1] = starts[i] + n
        at = torch.arange(n - min(case["fresh"], n), n, device="cuda")
        slots.append(mine[at // page] * page + at % page)
    slots = torch.cat(slots)
    held = []
    for _ in range(2):
        held += list(_quantise(_acts(g, (pages * page, h, d), torch.float32), case["fmt"]))
    fresh = slots.numel()
    s = dict(k=_acts(g, (fresh, h, d), dt), v=_acts(g, (fresh, h, d), dt), slots=slots, table=table, starts=starts.cuda(),
             total=total, out=None)
    if own:
        from vibetensor_b200 import cache
        c = cache.QuantCache(pages, page, h, d, fmt=case["fmt"], device="cuda")
        for name, t in zip(("k", "k_scale", "v", "v_scale"), held):
            getattr(c, name).copy_(t.view(getattr(c, name).shape))
        return dict(s, cache=c)
    return dict(s, held=held)


# ------------------------------------------------------------------------------- one pass
def run(state):
    return globals()[("_own_" if own else "_plain_") + state["case"]["op"]](state)


def _own_join(s):
    from vibetensor_b200 import kernels
    c = s["case"]
    if c["way"] == "forward":
        r, n, inv_post, inv_pre = kernels.residual_norm(
            s["x"], s["y"], s["gp"], s["gate"], s["gn"], EPS, post_norm=c["post"], pre_norm=c["pre"],
            residual_scale=s["alpha"], branch_scale=s["beta"])
        return [t for t in (r, n, inv_post, inv_pre) if t is not None]
    out = kernels.residual_norm_backward(
        s["dr"], s["dn"], s["y"], s["r"], s["inv_post"], s["inv_pre"], s["gp"], s["gate"], s["gn"],
        residual_scale=s["alpha"], branch_scale=s["beta"])
    return [t for t in out if t is not None]


def _own_keep(s):
    from vibetensor_b200 import kernels
    c = s["case"]
    if c["what"] == "round":
        return kernels.checkpoint8_restore(kernels.checkpoint8(s["x"], c["fmt"]))
    if c["what"] == "norm":
        out, inv, kept = kernels.rmsnorm_checkpoint8(s["x"], s["gamma"], EPS, c["fmt"])
        dx, dgamma = kernels.rmsnorm_backward(s["dy"], kept, inv, s["gamma"])
        return [out, inv, dx, dgamma]
    out, kept_gate, kept_up = kernels.silu_mul_checkpoint8(s["gate"], s["up"], c["fmt"])
    return [out, *kernels.silu_mul_backward(s["dy"], kept_gate, kept_up)]


def _own_rotary(s):
    from vibetensor_b200 import kernels
    c = s["case"]
    call = kernels.rotary if c["way"] == "forward" else kernels.rotary_backward
    return list(call(s["q"], s["k"], s["pos"], s["freq"], s["sections"], interleaved=c["paired"]))


def _own_cache(s):
    dt = DTYPES[s["case"]["dtype"]]
    s["cache"].write(s["k"], s["v"], s["slots"])
    return list(s["cache"].read(s["table"], s["starts"], s["total"], dtype=dt))


def _plain_join(s):
    c = s["case"]
    dt = s["y"].dtype
    gp = s["gp"] if s["gp"] is not None else 1.0
    gn = s["gn"] if s["gn"] is not None else 1.0
    gate = 1.0 if s["gate"] is None else s["gate"].float()
    y = s["y"].float()
    if c["way"] == "forward":
        out = []
        inv_post = None
        if c["post"]:
            inv_post = torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS)
            y = y * inv_post * gp
        r = s["alpha"] * s["x"].float() + s["beta"] * (y * gate)
        out.append(r.to(dt))
        inv_pre = None
        if c["pre"]:
            inv_pre = torch.rsqrt((r * r).mean(-1, keepdim=True) + EPS)
            out.append((r * inv_pre * gn).to(dt))
        return out + [t.reshape(-1) for t in (inv_post, inv_pre) if t is not None]
    lead = tuple(range(y.dim() - 1))
    up = s["dr"].float()
    dgn = dgp = dgate = None
    if c["pre"]:
        inv = s["inv_pre"].view(y.shape[:-1] + (1,))
        dn, hat = s["dn"].float(), s["r"].float() * inv
        dgn = (dn * hat).sum(lead)
        dn = dn * gn
        up = up + inv * (dn - hat * (dn * hat).mean(-1, keepdim=True))
    dx = s["alpha"] * up
    up = s["beta"] * up
    hat = y * s["inv_post"].view(y.shape[:-1] + (1,)) if c["post"] else y
    if s["gate"] is not None:
        full = up * (hat * gp)
        dgate = {"channel": lambda: full.sum(lead), "group": lambda: full.sum(-2, keepdim=True), "full": lambda: full}[c["gate"]]().to(dt)
        up = up * gate
    dy = up
    if c["post"]:
        dgp = (up * hat).sum(lead)
        dv = up * gp
        dy = s["inv_post"].view(y.shape[:-1] + (1,)) * (dv - hat * (dv * hat).mean(-1, keepdim=True))
    return [t for t in (dx.to(dt), dy.to(dt), dgp, dgate, dgn) if t is not None]


def _groups(x):
    """[n, d] -> [n, groups, GROUP] in 32 bits, the last group filled up with zeros."""
    n, d = x.shape
    out = torch.zeros((n, -(-d // GROUP) * GROUP), device=x.device)
    out[:, :d] = x
    return out.view(n, -1, GROUP)


def _keep_and_restore(x, fmt):
    q, scale = _quantise(_groups(x), fmt)
    return (q.float() * scale.unsqueeze(-1)).view(x.shape[0], -1)[:, :x.shape[1]]


def _plain_keep(s):
    c = s["case"]
    if c["what"] == "round":
        return _keep_and_restore(s["x"], c["fmt"]).to(s["x"].dtype)
    dt = s["dy"].dtype
    dy = s["dy"].float()
    if c["what"] == "norm":
        x = s["x"].float()
        inv = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        out = (x * inv * s["gamma"]).to(dt)
        hat = _keep_and_restore(s["x"], c["fmt"]) * inv
        dgamma = (dy * hat).sum(0)
        dy = dy * s["gamma"]
        return [out, inv.reshape(-1), (inv * (dy - hat * (dy * hat).mean(-1, keepdim=True))).to(dt), dgamma]
    gate, up = s["gate"].float(), s["up"].float()
    out = (gate / (1.0 + torch.exp(-gate)) * up).to(dt)
    gate, up = _keep_and_restore(s["gate"], c["fmt"]), _keep_and_restore(s["up"], c["fmt"])
    sig = 1.0 / (1.0 + torch.exp(-gate))
    return [out, (dy * up * sig * (1.0 + gate * (1.0 - sig))).to(dt), (dy * gate * sig).to(dt)]


def _plain_rotary(s):
    c = s["case"]
    half = sum(s["sections"])
    ang = s["pos"][s["which"]].permute(1, 2, 0).double() * s["freq"].double()
    if c["way"] == "backward":
        ang = -ang
    cos, sin = ang.cos().float()[:, :, None], ang.sin().float()[:, :, None]
    res = []
    for x in (s["q"], s["k"]):
        f = x.float()
        o = f.clone()
        a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if c["paired"] else (slice(0, half), slice(half, 2 * half))
        o[..., a] = f[..., a] * cos - f[..., b] * sin
        o[..., b] = f[..., b] * cos + f[..., a] * sin
        res.append(o.to(x.dtype))
    return res


def _plain_cache(s):
    c = s["case"]
    dt = DTYPES[c["dtype"]]
    row = torch.arange(s["total"], device="cuda")
    seq = (row[:, None] >= s["starts"][None, 1:]).sum(1)
    at = row - s["starts"][seq]
    slot = s["table"][seq, at // c["page"]] * c["page"] + at % c["page"]
    out = []
    for x, q, scale in ((s["k"], s["held"][0], s["held"][1]), (s["v"], s["held"][2], s["held"][3])):
        nq, ns = _quantise(x.float(), c["fmt"])
        q.view(torch.int8)[s["slots"]] = nq.view(torch.int8)
        scale[s["slots"]] = ns
        out.append((q.view(torch.int8)[slot].view(q.dtype).float() * scale[slot].unsqueeze(-1)).to(dt))
    return out


# --------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return globals()["_exact_" + case["op"]](s, case)


def _wide(t, like=None):
    return None if t is None else t.to(torch.float64)


def _exact_join(s, case):
    d = case["cols"]
    n = case["rows"]
    flat = lambda t: None if t is None else _wide(t).reshape(-1, d)  # noqa: E731
    y = flat(s["y"])
    one = torch.ones(1, dtype=torch.float64, device="cuda")
    gate = flat(s["gate"])
    if gate is not None and gate.shape[0] not in (1, n):
        gate = gate.repeat_interleave(n // gate.shape[0], 0)
    g = one if gate is None else gate
    gp = _wide(s["gp"]) if case["post"] else one
    gn = _wide(s["gn"]) if case["pre"] else one
    mean_square = lambda t: torch.einsum("nd,nd->n", t, t)[:, None] / d  # noqa: E731
    if case["way"] == "forward":
        inv_post = 1.0 / torch.sqrt(mean_square(y) + EPS) if case["post"] else None
        v = y * inv_post * gp if case["post"] else y
        r = flat(s["x"]) * s["alpha"] + v * g * s["beta"]
        inv_pre = 1.0 / torch.sqrt(mean_square(r) + EPS) if case["pre"] else None
        out = [r.view(s["y"].shape)]
        if case["pre"]:
            out.append((r * inv_pre * gn).view(s["y"].shape))
        return out + [i[:, 0] for i in (inv_post, inv_pre) if i is not None]
    total = flat(s["dr"])
    dgn = dgp = dgate = None
    if case["pre"]:
        i, dn, r = _wide(s["inv_pre"])[:, None], flat(s["dn"]), flat(s["r"])
        dgn = torch.einsum("nd,nd->d", dn, r * i)
        total = total + i * dn * gn - r * i ** 3 * torch.einsum("nd,nd->n", dn * gn, r)[:, None] / d
    dx = total * s["alpha"]
    dbranch = total * s["beta"]
    i = _wide(s["inv_post"])[:, None] if case["post"] else one
    if gate is not None:
        full = dbranch * y * i * gp
        dgate = full if case["gate"] == "full" else full.reshape(s["gate"].numel() // d, -1, d).sum(1)
        dgate = dgate.reshape(s["gate"].shape)
    dv = dbranch * g
    dy = dv
    if case["post"]:
        dgp = torch.einsum("nd,nd->d", dv, y * i)
        dy = i * dv * gp - y * i ** 3 * torch.einsum("nd,nd->n", dv * gp, y)[:, None] / d
    return [t for t in (dx.view(s["y"].shape), dy.view(s["y"].shape), dgp, dgate, dgn) if t is not None]


def _held(x, fmt):
    """The values that x [m, n] stands for after it was held in 8 bits, row by row.

    Which of two neighbouring levels a value takes is part of the definition and is decided in 32
    bits: the product of the value with the correctly rounded quotient of the top level and the
    row's largest magnitude, to the nearest level, ties to the even one."""
    x = x.to(torch.float32)
    big = x.abs().max(-1, keepdim=True).values
    live = big >= TINY
    up = torch.where(live, torch.full_like(big, TOP[fmt]) / torch.where(live, big, 1.0), 0.0)
    step = torch.where(live, big * torch.full_like(big, 1.0 / TOP[fmt]), 0.0).double()
    z = (x * up).double()
    if fmt == "int8":
        lower = z.floor()
        part = z - lower
        level = torch.where((part > 0.5) | ((part == 0.5) & (lower.remainder(2) == 1)), lower + 1, lower)
    else:
        power = torch.floor(torch.log2(z.abs().clamp_min(2.0 ** -6)))
        power = torch.where(torch.exp2(power) > z.abs().clamp_min(2.0 ** -6), power - 1, power)
        grain = torch.exp2(power.clamp_min(-6.0) - 3.0)   # three fraction bits, the least exponent is -6
        part = z / grain
        lower = part.floor()
        rest = part - lower
        level = torch.where((rest > 0.5) | ((rest == 0.5) & (lower.remainder(2) == 1)), lower + 1, lower) * grain
    return level * step


def _held_wide(x, fmt):
    n, d = x.shape
    parts = [_held(x[:, a:a + GROUP], fmt) for a in range(0, d, GROUP)]
    return torch.cat(parts, 1)


def _exact_keep(s, case):
    if case["what"] == "round":
        return _held_wide(s["x"], case["fmt"])
    dy = _wide(s["dy"])
    d = case["cols"]
    if case["what"] == "norm":
        x, gamma = _wide(s["x"]), _wide(s["gamma"])
        i = 1.0 / torch.sqrt(torch.einsum("nd,nd->n", x, x) / d + EPS)
        out = x * i[:, None] * gamma
        kept = _held_wide(s["x"], case["fmt"])
        dx = dy * gamma * i[:, None] - kept * (i ** 3 * torch.einsum("nd,nd->n", dy * gamma, kept) / d)[:, None]
        return [out, i, dx, torch.einsum("nd,nd,n->d", dy, kept, i)]
    act = lambda t: t * torch.sigmoid(t)  # noqa: E731
    out = act(_wide(s["gate"])) * _wide(s["up"])
    gate, up = _held_wide(s["gate"], case["fmt"]), _held_wide(s["up"], case["fmt"])
    sig = torch.sigmoid(gate)
    return [out, dy * up * (sig + gate * sig * torch.sigmoid(-gate)), dy * act(gate)]


def _exact_rotary(s, case):
    half = sum(s["sections"])
    sign = 1.0 if case["way"] == "forward" else -1.0
    turns, first = [], 0
    for axis, n in enumerate(s["sections"]):
        turns.append(s["pos"][axis].double()[..., None] * s["freq"][first:first + n].double())
        first += n
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), sign * torch.cat(turns, -1))[:, :, None]
    out = []
    for x in (s["q"], s["k"]):
        w = _wide(x)
        rot, rest = w[..., :2 * half], w[..., 2 * half:]
        if case["paired"]:
            z = torch.complex(rot[..., 0::2].contiguous(), rot[..., 1::2].contiguous()) * turn
            rot = torch.stack((z.real, z.imag), -1).flatten(-2)
        else:
            z = torch.complex(rot[..., :half].contiguous(), rot[..., half:].contiguous()) * turn
            rot = torch.cat((z.real, z.imag), -1)
        out.append(torch.cat((rot, rest), -1))
    return out


def _exact_cache(s, case):
    h, d, page = case["heads"], case["dim"], case["page"]
    if "held" in s:
        parts = s["held"]
    else:
        c = s["cache"]
        parts = [c.k, c.k_scale, c.v, c.v_scale]
    out = []
    table, starts = s["table"].tolist(), s["starts"].tolist()
    where = torch.cat([torch.tensor(table[i], device="cuda")[:, None].mul(page).add(torch.arange(page, device="cuda"))
                       .flatten()[:starts[i + 1] - starts[i]] for i in range(case["seqs"])])
    for new, q, scale in ((s["k"], parts[0], parts[1]), (s["v"], parts[2], parts[3])):
        full = q.reshape(-1, h, d).float().double() * scale.reshape(-1, h, 1).double()
        full[s["slots"]] = _held(new.reshape(-1, d), case["fmt"]).reshape(new.shape)
        out.append(full[where])
    return out
