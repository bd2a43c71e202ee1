"""The feed-forward block's operators (causaldiffae_amd.ops_block) against their definitions in 64 bits.

Bounds are elementwise and follow the arithmetic: `u` = 2^-24 is half a step of fp32, `half(t)` half a step of the result's type; a sum of n products
is off by at most (n + 8) u times the sum of the magnitudes whatever the order of its terms."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

u = 2.0 ** -24
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
DEV = "cuda"


def half(t):
    return torch.finfo(t).eps / 2


def least(t):
    """half the distance of the smallest numbers of a type (fp16 and bf16 results below the normal range)"""
    return {BF16: 2.0 ** -134, F16: 2.0 ** -25, F32: 2.0 ** -150}[t]


def blk():
    from causaldiffae_amd import ops_block
    return ops_block


def rnd(seed, *shape, dtype=F32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(*shape, generator=g)).to(dtype).to(DEV)


def within(name, got, ref, bound):
    err = (got.double() - ref).abs()
    bound = bound + half(got.dtype) * ref.abs() + least(got.dtype)
    bad = ~(err <= bound)
    assert not bad.any(), (name, int(bad.sum()), float((err / bound)[bad].max()), bad.nonzero()[0].tolist())


# ----------------------------------------------------------------------------- linear_act
ACT = {
    "none": lambda z: z, "silu": lambda z: z * torch.sigmoid(z), "relu": torch.relu, "gelu": lambda z: 0.5 * z * (1 + torch.erf(z / math.sqrt(2))),
    "gelu_tanh": lambda z: 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))),
}


def linear_reference(x, w, b, res, act, dy):
    """values and bounds (without the final rounding) in 64 bits"""
    t = x.dtype
    x, w, dy = x.double(), w.double(), dy.double()
    K, N, M = x.shape[1], w.shape[0], x.shape[0]
    z = x @ w.t() + (0 if b is None else b.double())
    S = x.abs() @ w.abs().t() + (0 if b is None else b.double().abs())
    zerr = (K + 8) * u * S
    zg = z.clone().requires_grad_(True)
    with torch.enable_grad():
        a = ACT[act](zg)
        (slope,) = torch.autograd.grad(a.sum(), zg)
    y = a.detach() + (0 if res is None else res.double())
    # every slope is below 1.13; sigmoid, erf and exp are good to a few steps
    out = {"y": (y, 1.13 * zerr + 16 * u * (z.abs() + y.abs() + 1e-3))}
    dz = dy * slope
    if act == "none":
        dzerr = torch.zeros_like(dz)
    elif act == "relu":
        dzerr = dy.abs() * (z.abs() <= zerr + 2.0 ** -24)
    else:                                          # the second derivatives are below 0.8; z is kept in 11 bits
        dzerr = dy.abs() * (0.8 * (zerr + 2.0 ** -11 * z.abs() + 2.0 ** -25) + 32 * u)
    op = dzerr + (0 if act == "none" else half(t) * dz.abs() + least(t))           # as an operand dz is rounded
    out["dx"] = (dz @ w, op @ w.abs() + (N + 8) * u * ((dz.abs() + op) @ w.abs()))
    out["dw"] = (dz.t() @ x, op.t() @ x.abs() + (M + 8) * u * ((dz.abs() + op).t() @ x.abs()))
    out["db"] = (dz.sum(0), dzerr.sum(0) + (M + 8) * u * (dz.abs() + dzerr).sum(0))
    return out


def check_linear(x, w, b, res, act, dy):
    for t in (x, w, b, res):
        if t is not None:
            t.requires_grad_(True)
    y = blk().linear_act(x, w, b, res=res, act=act)
    leaves = [t for t in (x, w, b, res) if t is not None]
    grads = dict(zip(map(id, leaves), torch.autograd.grad(y, leaves, dy)))
    K, N = w.shape[1], w.shape[0]
    x2, dy2 = x.detach().reshape(-1, K), dy.reshape(-1, N)
    ref = linear_reference(x2, w.detach(), None if b is None else b.detach(), None if res is None else res.detach().reshape(-1, N), act, dy2)
    assert y.dtype == x.dtype and y.shape == x.shape[:-1] + (N,)
    within("y", y.detach().reshape(-1, N), *ref["y"])
    within("dx", grads[id(x)].reshape(-1, K), *ref["dx"])
    within("dw", grads[id(w)], *ref["dw"])
    if b is not None:
        within("db", grads[id(b)], *ref["db"])
    if res is not None:
        assert torch.equal(grads[id(res)], dy)


SIZES = [(1, 1, 1), (1, 512, 2048), (3, 8, 16), (16, 64, 40), (17, 100, 33), (31, 2048, 24), (64, 392, 130), (128, 128, 128), (129, 136, 264), (200, 27, 7),
         (257, 513, 255), (1000, 384, 1536), (1021, 393, 771), (4100, 72, 200), (300, 1600, 1024)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_linear_act_sizes(M, K, N, dtype):
    act = list(ACT)[(M + K + N) % 5]
    print(M, K, N, dtype, act, flush=True)
    res = rnd(4, M, N, dtype=dtype) if (M + N) % 2 else None
    check_linear(rnd(1, M, K, dtype=dtype), rnd(2, N, K, dtype=dtype, scale=K ** -0.5), rnd(3, N, dtype=dtype), res, act, rnd(5, M, N, dtype=dtype))


@pytest.mark.parametrize("splits", [1, 2, 5])
@pytest.mark.parametrize("tile", [1, 2, 3, 4])
@pytest.mark.parametrize("M,K,N", [(300, 136, 520), (129, 1000, 65), (77, 393, 260), (513, 64, 8)])
def test_linear_act_tiles(M, K, N, tile, splits):
    """every tile and split at sizes inside one tile, on its edges and past them (by themselves such sizes take the small ones)"""
    from causaldiffae_amd._lib import tune_scope
    with tune_scope(lin16_tile=tile, lin16_splits=splits):
        dtype = (BF16, F16)[tile % 2]
        check_linear(rnd(1, M, K, dtype=dtype), rnd(2, N, K, dtype=dtype, scale=K ** -0.5), rnd(3, N, dtype=dtype), rnd(4, M, N, dtype=dtype), "gelu", rnd(5, M, N, dtype=dtype))


def test_linear_act_large():
    """sizes that take the large tiles by themselves, several rounds of them, against 64 bits"""
    M, K, N = 4352, 1032, 4104
    x, w, dy = rnd(1, M, K, dtype=BF16), rnd(2, N, K, dtype=BF16, scale=K ** -0.5), rnd(3, M, N, dtype=BF16)
    check_linear(x, w, rnd(4, N, dtype=BF16), None, "none", dy)


@pytest.mark.parametrize("act", list(ACT))
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear_act_activations(act, dtype):
    """pre-activations from far below to far above the range where an activation bends"""
    x = rnd(1, 96, 64, dtype=dtype)
    x = (x.float() * torch.logspace(-3, 1.5, 96, device=DEV)[:, None]).to(dtype)
    check_linear(x, rnd(2, 72, 64, dtype=dtype, scale=0.3), None, rnd(3, 96, 72, dtype=dtype), act, rnd(4, 96, 72, dtype=dtype))


@pytest.mark.parametrize("K,N,pad,off", [(64, 48, 8, 0), (64, 48, 3, 1), (50, 36, 5, 3), (128, 136, 0, 4)])
def test_linear_act_strides(K, N, pad, off):
    """rows inside wider rows, at any alignment; a weight whose storage is transposed; three leading dimensions; an expanded gradient"""
    big = rnd(1, 6 * 11, K + pad + off, dtype=BF16)
    x = big[:, off:off + K].unflatten(0, (6, 11))
    w = rnd(2, K, N, dtype=BF16, scale=K ** -0.5).t()
    b = rnd(3, 2 * N, dtype=BF16)[::2]
    res = rnd(4, 6, 11, N + pad, dtype=BF16)[..., :N]
    dy = rnd(5, N, dtype=BF16).expand(6, 11, N)
    check_linear(x.detach(), w.detach(), b.detach(), res.detach(), "gelu", dy)


def test_linear_act_no_rows():
    x, w, b = rnd(1, 0, 24, dtype=BF16).requires_grad_(True), rnd(2, 16, 24, dtype=BF16).requires_grad_(True), rnd(3, 16, dtype=BF16).requires_grad_(True)
    y = blk().linear_act(x, w, b, act="silu")
    assert y.shape == (0, 16)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert dx.shape == (0, 24) and not dw.any() and not db.any()


def test_linear_act_partial_gradients():
    """each input alone"""
    x, w, b, res, dy = rnd(1, 50, 40, dtype=BF16), rnd(2, 24, 40, dtype=BF16, scale=0.2), rnd(3, 24, dtype=BF16), rnd(4, 50, 24, dtype=BF16), rnd(5, 50, 24, dtype=BF16)
    ref = linear_reference(x, w, b, res, "silu", dy)
    for name, t in (("dx", x), ("dw", w), ("db", b)):
        t = t.clone().requires_grad_(True)
        args = [t if k == name else v for k, v in (("dx", x), ("dw", w), ("db", b))]
        (g,) = torch.autograd.grad(blk().linear_act(*args, res=res, act="silu"), t, dy)
        within(name, g, *ref[name])
    r = res.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(blk().linear_act(x, w, b, res=r, act="silu"), r, dy)
    assert torch.equal(g, dy)


def test_linear_act_without_bias():
    x, w, res, dy = rnd(1, 2, 25, 40, dtype=F16), rnd(2, 24, 40, dtype=F16, scale=0.2), rnd(3, 2, 25, 24, dtype=F16), rnd(4, 2, 25, 24, dtype=F16)
    check_linear(x, w, None, res, "gelu_tanh", dy)
    x, w, res = (t.detach() for t in (x, w, res))
    with torch.no_grad():
        y = blk().linear_act(x.requires_grad_(True), w, None, res, "gelu_tanh")
    assert not y.requires_grad and torch.equal(y, blk().linear_act(x, w, None, res, "gelu_tanh").detach())


def test_first_derivatives_only():
    """a gradient of a gradient raises instead of being zero"""
    x, w = rnd(1, 6, 16, dtype=BF16).requires_grad_(True), rnd(2, 16, 16, dtype=BF16).requires_grad_(True)
    for y in (blk().linear_act(x, w, act="silu"), blk().residual_norm(x, x, pre=w[0])[1]):
        (g,) = torch.autograd.grad(y.float().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="first derivatives"):
            g.float().sum().backward()


def test_accumulating_backward():
    """.backward() twice into the leaves' .grad, an input that occurs twice, and outputs of which one is not used"""
    x, w = rnd(1, 12, 16, dtype=F32).requires_grad_(True), (1 + rnd(2, 16)).requires_grad_(True)
    r, uu = blk().residual_norm(x, x, alpha=2.0, pre=w, kind="rms")
    (3 * r).sum().backward()
    assert torch.equal(x.grad, torch.full_like(x, 9.0)) and w.grad is not None and not w.grad.any()
    blk().residual_norm(x, x, alpha=2.0, pre=w, kind="rms")[0].sum().backward()
    assert torch.equal(x.grad, torch.full_like(x, 12.0))


def test_linear_act_rows_do_not_mix():
    """a row that is not finite stays alone, at a size with rows, columns and k outside full tiles"""
    x, w = rnd(1, 131, 72, dtype=BF16), rnd(2, 133, 72, dtype=BF16, scale=0.1)
    clean = blk().linear_act(x, w, act="gelu")
    x[130] = float("nan")
    x[7, 3] = float("inf")
    y = blk().linear_act(x, w, act="gelu")
    keep = [i for i in range(131) if i not in (7, 130)]
    assert torch.equal(y[keep], clean[keep]) and y[130].isnan().all()


def test_linear_act_writes_nothing_else():
    """rows and columns beside the result stay as they were"""
    from causaldiffae_amd._lib import check, lib, stream
    for M, K, N, ldy in ((5, 24, 16, 24), (131, 40, 67, 80), (130, 512, 136, 144)):
        x, w = rnd(1, M, K, dtype=BF16), rnd(2, N, K, dtype=BF16)
        y, z = torch.full((M + 3, ldy), 7.0, dtype=BF16, device=DEV), torch.full((M + 3, ldy), 7.0, dtype=F16, device=DEV)
        need = lib.cdae_lin16_workspace_bytes(0, M, N, K)
        ws = torch.empty(need, dtype=torch.uint8, device=DEV)
        check(lib.cdae_lin16_fwd(x.data_ptr(), K, w.data_ptr(), K, None, None, 0, y.data_ptr(), ldy, z.data_ptr(), ldy, M, N, K, 1, 0, ws.data_ptr(), need, stream()))
        for t in (y, z):
            assert (t[M:] == 7).all() and (t[:, N:] == 7).all()
        assert torch.equal(y[:M, :N], blk().linear_act(x, w, act="silu"))


# ----------------------------------------------------------------------------- residual_norm
def norm_reference(x, f, v, alpha, post, pre, kind, eps, dr, du):
    """values and bounds in 64 bits for rows x [B, T, C]; v: gate, scale, shift, w1, b1, w2, b2 (None where absent)"""
    t = {k: (None if a is None else a.double()) for k, a in v.items()}
    x, f, dr, du = (None if a is None else a.double() for a in (x, f, dr, du))
    B, T, C = x.shape
    each = lambda a: a[:, None, :] if a.dim() == 2 else a
    one = torch.ones(C, dtype=torch.float64, device=x.device)

    def stats(a):
        m = a.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(a[..., :1])
        i = 1 / torch.sqrt((a - m).pow(2).mean(-1, keepdim=True) + eps)
        n = (a - m) * i
        # sums of a row are at most 30 additions deep: the mean is off by 30 u rms, which the centred values and the variance inherit
        return n, i, 64 * u * (1 + a.pow(2).mean(-1, keepdim=True).sqrt() * i) * (1 + n.abs())

    w1, b1 = (one if t["w1"] is None else t["w1"]), (0 * one if t["b1"] is None else t["b1"])
    w2, b2 = (one if t["w2"] is None else t["w2"]), (0 * one if t["b2"] is None else t["b2"])
    g = alpha * (one if t["gate"] is None else each(t["gate"]))
    s = 1 + (0 * one if t["scale"] is None else each(t["scale"]))
    out = {}
    if f is None:
        r, rerr, n1, n1err, i1, p = x, torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x), None, torch.zeros_like(x)
    else:
        n1, i1, n1err = stats(f) if post else (f, None, torch.zeros_like(f))
        p = n1 * w1 + b1
        perr = w1.abs() * n1err + 4 * u * (n1.abs() * w1.abs() + b1.abs())
        r = x + g * p
        rerr = g.abs() * perr + 4 * u * (x.abs() + (g * p).abs())
        out["r"] = (r, rerr)
    D = torch.zeros_like(x) if dr is None else dr
    Derr = torch.zeros_like(x)
    mean = lambda a: a.mean(-1, keepdim=True)
    if pre:
        n2, i2, n2err = stats(r)
        n2err = n2err + i2 * (rerr + mean(rerr ** 2).sqrt() * (1 + n2.abs()))
        q = n2 * w2 + b2
        qerr = w2.abs() * n2err + 4 * u * (n2.abs() * w2.abs() + b2.abs())
        uu = q * s + (0 if t["shift"] is None else each(t["shift"]))
        out["u"] = (uu, s.abs() * qerr + 8 * u * ((q * s).abs() + uu.abs()))
        if du is not None:
            h = du * s * w2
            irel = 64 * u * (1 + mean(r ** 2).sqrt() * i2) + i2 * mean(rerr ** 2).sqrt()
            back = h - mean(h * n2) * n2 - (mean(h) if kind == "layer" else 0)
            size = h.abs() + mean(h.abs()) + n2.abs() * mean((h * n2).abs())
            D = D + i2 * back
            Derr = Derr + i2 * (64 * u + irel) * size + i2 * (n2err * mean((h * n2).abs()) + n2.abs() * mean(h.abs() * n2err)) + 4 * u * D.abs()
    out["dx"] = (D, Derr)
    total = lambda a, like: a.sum((0, 1)) if like is None or like.dim() == 1 else a.sum(1)
    deep = lambda a, err, like: (total(a, like), total(err, like) + 1e3 * u * total(a.abs(), like))      # column sums: far below 1000 additions deep
    if f is not None:
        dp = D * g
        dperr = Derr * g.abs() + 4 * u * dp.abs()
        h, herr = dp * w1, dperr * w1.abs()
        if post:
            irel = 64 * u * (1 + mean(f ** 2).sqrt() * i1)
            size = h.abs() + mean(h.abs()) + n1.abs() * mean((h * n1).abs())
            df = i1 * (h - mean(h * n1) * n1 - (mean(h) if kind == "layer" else 0))
            out["df"] = (df, i1 * (64 * u + irel) * size + i1 * (herr + mean(herr) + n1.abs() * mean(herr * n1.abs()) + n1err * mean((h * n1).abs()) + n1.abs() * mean(h.abs() * n1err)))
        else:
            out["df"] = (dp, dperr)
        out["dgate"] = deep(alpha * D * p, abs(alpha) * (Derr * p.abs() + D.abs() * perr), t["gate"])
        out["dw1"] = deep(dp * n1, dperr * n1.abs() + dp.abs() * n1err, None)
        out["db1"] = deep(dp, dperr, None)
    if pre and du is not None:
        out["dscale"] = deep(du * q, du.abs() * qerr, t["scale"])
        out["dshift"] = deep(du, 0 * du, t["shift"])
        out["dw2"] = deep(du * s * n2, (du * s).abs() * n2err, None)
        out["db2"] = deep(du * s, 4 * u * (du * s).abs(), None)
    return out


def check_norm(x, f, v, alpha=1.0, post=False, pre=True, kind="layer", eps=1e-5, dr=None, du=None, shape=None):
    B, T, C = shape or x.shape
    leaves = {"x": x, "f": f, **v}
    leaves = {k: t.requires_grad_(True) for k, t in leaves.items() if t is not None}
    r, uu = blk().residual_norm(x, f, gate=v["gate"], alpha=alpha, post=(v["w1"], v["b1"]) if post else None, pre=(v["w2"], v["b2"]) if pre else None,
                                scale=v["scale"], shift=v["shift"], kind=kind, eps=eps)
    outs = [(o, d) for o, d in ((r, dr), (uu, du)) if d is not None]
    if f is None:
        assert r is x
    got = dict(zip(["d" + k for k in leaves], torch.autograd.grad([o for o, _ in outs], list(leaves.values()), [d for _, d in outs], allow_unused=True)))
    rows = lambda a: None if a is None else a.detach().reshape(B, T, C)
    ref = norm_reference(rows(x), rows(f), {k: None if a is None else a.detach() for k, a in v.items()}, alpha, post, pre, kind, eps, rows(dr), rows(du))
    got["r"], got["u"] = (r if f is not None else None), uu
    for k, (a, e) in ref.items():
        if got.get(k) is not None:
            shape_of = got[k].reshape(a.shape).detach()
            within(k, shape_of, a, e)
    want = {"dx"} | ({"df"} if f is not None else set())
    assert want <= {k for k, g in got.items() if g is not None}
    return got


def vectors(B, C, dtype, gate, mod, post, bias, vec=None, w=None):
    """gate and mod: None, "channel" or "sample"; vec, w: their types"""
    vec, w = vec or dtype, w or dtype
    of = lambda mode, seed, s, off=0.0: None if mode is None else (off + rnd(seed, *((C,) if mode == "channel" else (B, C)), scale=s)).to(vec)
    return {"gate": of(gate, 11, 0.4, 0.5), "scale": of(mod, 12, 0.3), "shift": of(mod, 13, 0.3),
            "w1": (1 + rnd(14, C, scale=0.1)).to(w) if post else None, "b1": rnd(15, C, scale=0.2).to(w) if post and bias else None,
            "w2": (1 + rnd(16, C, scale=0.1)).to(w), "b2": rnd(17, C, scale=0.2).to(w) if bias else None}


NORM_SIZES = [(1, 1, 1), (2, 3, 7), (4, 1, 512), (3, 5, 8), (2, 77, 64), (5, 33, 100), (2, 130, 384), (3, 41, 1001), (2, 9, 2048), (1, 3, 4100), (1, 2, 8192), (1, 3000, 24),
              (64, 1, 72)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("B,T,C", NORM_SIZES)
def test_residual_norm_sizes(B, T, C, dtype):
    i = B + T + C
    kind, post, gate, mod = ("layer", "rms")[i % 2], bool(i % 3), (None, "channel", "sample")[i % 3], (None, "sample", "channel")[(i // 2) % 3]
    print(B, T, C, dtype, kind, post, gate, mod, flush=True)
    v = vectors(B, C, dtype, gate, mod, post, kind == "layer")
    r = lambda s: rnd(s, B, T, C, dtype=dtype)
    check_norm(r(1), r(2), v, 0.7, post, True, kind, dr=r(3), du=r(4))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("B,T,C,kind,post", [(2, 300, 4100, "layer", True), (1, 600, 8192, "rms", True), (3, 400, 5001, "layer", False), (1, 5000, 600, "rms", True)])
def test_residual_norm_walks(B, T, C, kind, post, dtype):
    """several rows for every block, forward and backward"""
    v = vectors(B, C, dtype, "sample", "sample", post, True)
    r = lambda s: rnd(s, B, T, C, dtype=dtype)
    check_norm(r(1), r(2), v, 0.7, post, True, kind, dr=r(3), du=r(4))


@pytest.mark.parametrize("gate", [None, "channel", "sample"])
@pytest.mark.parametrize("mod", [None, "channel", "sample"])
@pytest.mark.parametrize("vec,w", [(BF16, F32), (F32, BF16)])
def test_residual_norm_vectors(gate, mod, vec, w):
    """every mixture of vectors for a sample and for all, in the rows' type or fp32"""
    v = vectors(3, 136, BF16, gate, mod, True, True, vec, w)
    r = lambda s: rnd(s, 3, 29, 136, dtype=BF16)
    got = check_norm(r(1), r(2), v, -0.5, True, True, "layer", dr=r(3), du=r(4))
    assert all(got["d" + k].dtype == a.dtype and got["d" + k].shape == a.shape for k, a in v.items() if a is not None)


@pytest.mark.parametrize("case", ["pre only", "post only", "residual only", "dr only", "du only"])
def test_residual_norm_parts(case):
    B, T, C = 2, 37, 200
    r = lambda s: rnd(s, B, T, C, dtype=BF16)
    v = vectors(B, C, BF16, None if case == "pre only" else "sample", "sample", case != "residual only" and case != "pre only", True)
    if case in ("post only", "residual only"):
        for k in ("scale", "shift", "w2", "b2"):
            v[k] = None
    pre = case not in ("post only", "residual only")
    check_norm(r(1), None if case == "pre only" else r(2), v, 1.0, v["w1"] is not None, pre, "layer",
               dr=r(3) if case in ("post only", "residual only", "dr only") else None, du=r(4) if pre and case != "dr only" else None)


def test_residual_norm_without_weights():
    r = lambda s: rnd(s, 2, 5, 96, dtype=F32)
    check_norm(r(1), r(2), dict.fromkeys(("gate", "scale", "shift", "w1", "b1", "w2", "b2")), 1.0, True, True, "rms", dr=r(3), du=r(4))


def test_residual_norm_strides():
    """rows inside wider rows at odd alignments, gate / scale / shift as slices of one projection, an NHWC activation, expanded gradients"""
    N, C, H, W = 2, 52, 4, 6
    x = rnd(1, N, H, W, C + 3, dtype=BF16)[..., 1:1 + C]
    f = rnd(2, N, C, H, W, dtype=BF16).contiguous(memory_format=torch.channels_last).permute(0, 2, 3, 1)
    ada = rnd(3, N, 3 * C, dtype=BF16)
    v = {**dict.fromkeys(("w1", "b1", "b2")), "gate": ada[:, :C], "scale": ada[:, C:2 * C], "shift": ada[:, 2 * C:], "w2": rnd(4, C, dtype=BF16)}
    v = {k: None if a is None else a.detach() for k, a in v.items()}
    dr, du = rnd(5, C, dtype=BF16).expand(N, H, W, C), rnd(6, N, H, W, 2 * C, dtype=BF16)[..., ::2]
    check_norm(x.detach(), f.detach(), v, 1.0, False, True, "layer", dr=dr, du=du, shape=(N, H * W, C))


def test_residual_norm_two_dimensional_rows():
    """[M, C] with vectors for M / 5 samples"""
    r = lambda s: rnd(s, 35, 40, dtype=F16)
    v = vectors(7, 40, F16, "sample", "sample", True, False)
    check_norm(r(1), r(2), v, 1.0, True, True, "rms", dr=r(3), du=r(4), shape=(7, 5, 40))


def test_residual_norm_constant_and_huge_rows():
    """rows without variance, rows far from zero, rows of the type's largest values beside ordinary ones"""
    C = 264
    x = rnd(1, 1, 6, C, dtype=F32)
    x[0, 0], x[0, 1], x[0, 2] = 0.0, 3.0, 1e4 + x[0, 2]
    x[0, 3] *= 1e18
    f = rnd(2, 1, 6, C, dtype=F32)
    f[0, :3] = 0.0
    v = vectors(1, C, F32, None, None, False, True)
    check_norm(x, f, v, 1.0, False, True, "layer", dr=rnd(3, 1, 6, C), du=rnd(4, 1, 6, C))


def test_residual_norm_many_samples():
    """a vector for every row, more samples than one pass of the folding blocks' lanes"""
    v = vectors(5000, 24, BF16, "sample", "sample", False, True)
    r = lambda s: rnd(s, 5000, 24, dtype=BF16)
    check_norm(r(1), r(2), v, 1.0, False, True, "layer", dr=r(3), du=r(4), shape=(5000, 1, 24))


def test_residual_norm_no_rows():
    x = torch.empty(0, 5, 16, dtype=BF16, device=DEV).requires_grad_(True)
    w = rnd(1, 16, dtype=BF16).requires_grad_(True)
    r, uu = blk().residual_norm(x, x, pre=w)
    assert r.shape == uu.shape == (0, 5, 16)
    dx, dw = torch.autograd.grad([r, uu], [x, w], [torch.empty_like(r), torch.empty_like(uu)])
    assert dx.shape == x.shape and not dw.any()


def test_residual_norm_differences():
    """gradients against central differences of the kernel's own forward: fp32 rows, steps of 2^-7, so truncation (h^2 / 6 times the third derivative,
    below 1 here) is under 1e-4 and the differences' rounding under 64 u / h of the sums"""
    x, f = rnd(1, 1, 2, 12), rnd(2, 1, 2, 12)
    gate, w1, w2 = 0.5 + rnd(3, 12, scale=0.1), 1 + rnd(4, 12, scale=0.1), 1 + rnd(5, 12, scale=0.1)
    c1, c2 = rnd(6, 1, 2, 12), rnd(7, 1, 2, 12)
    args = [t.requires_grad_(True) for t in (x, f, gate, w1, w2)]

    def loss():
        r, uu = blk().residual_norm(x, f, gate=gate, post=w1, pre=w2, kind="rms", eps=1e-2)
        return (r.double() * c1.double()).sum() + (uu.double() * c2.double()).sum()

    grads = torch.autograd.grad(loss(), args)
    h = 2.0 ** -7
    for t, g in zip(args, grads):
        flat = t.detach().reshape(-1)
        for i in range(0, flat.numel(), 5):
            with torch.no_grad():
                keep = flat[i].clone()
                flat[i] = keep + h
                up = loss()
                flat[i] = keep - h
                down = loss()
                flat[i] = keep
            assert abs(float((up - down) / (2 * h)) - float(g.reshape(-1)[i])) < 1e-2


# ----------------------------------------------------------------------------- gradient norm and clipping
def grads_of(sizes, types, seed=0, scale=0.1):
    return [rnd(seed + i, n, dtype=types[i % len(types)], scale=scale) for i, n in enumerate(sizes)]


def exact_norm(grads, scale=1.0):
    return abs(scale) * math.sqrt(math.fsum(float(g.double().pow(2).sum()) for g in grads))


LISTS = [[1], [0], [5, 0, 3], [16384, 16385, 16383, 1], [100003] + [7] * 200 + [64] * 200, [1] * 700, [300001, 12, 1 << 20]]


@pytest.mark.parametrize("types", [(F32,), (BF16,), (F16, F32, BF16)])
@pytest.mark.parametrize("sizes", LISTS, ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("over", [0.5, 4.0])
def test_clip_sizes(sizes, types, over):
    grads = grads_of(sizes, types)
    n = exact_norm(grads, 0.25)
    max_norm = n / over if n else 1.0
    ref = [g.double() * (0.25 * min(1.0, max_norm / (n + 1e-6))) for g in grads]
    # the squares and their sum are exact to fp64: one rounding to fp32 is left
    assert abs(float(blk().grad_norm(grads, 0.25)) - n) <= 2 * u * n
    out = [torch.empty(g.shape, dtype=F32, device=DEV) for g in grads]
    got = blk().clip_grad_norm_(grads, max_norm, scale=0.25, out=out)
    assert got.dtype == F32 and got.dim() == 0 and abs(float(got) - n) <= 2 * u * n
    for o, r in zip(out, ref):
        within("out", o, r, 2 * u * r.abs())                    # the factor is rounded, the product is rounded
    before = [g._version for g in grads]
    blk().clip_grad_norm_(grads, max_norm, scale=0.25)
    assert all(g._version > b for g, b in zip(grads, before))
    for g, r in zip(grads, ref):
        within("in place", g, r, 2 * u * r.abs())


def test_clip_leaves_small_gradients_alone():
    grads = grads_of([1000, 33], (BF16, F32))
    keep = [g.clone() for g in grads]
    n = blk().clip_grad_norm_(grads, 1e3)
    assert abs(float(n) - exact_norm(keep)) <= 2 * u * float(n) and all(torch.equal(a, b) for a, b in zip(grads, keep))
    blk().clip_grad_norm_(grads, 0.0)
    assert all(not g.any() for g in grads)
    g = rnd(1, 70)
    g[3] = float("inf")
    k = g.clone()
    blk().clip_grad_norm_([g], math.inf)                        # nothing is clipped, whatever the norm
    assert torch.equal(g, k)


def test_clip_strides():
    """transposed, channels-last, sliced and 16-bit tensors at odd addresses; views of one buffer"""
    base = rnd(1, 40, 30)
    flat = rnd(2, 1001, dtype=BF16)
    grads = [base.t(), rnd(3, 2, 8, 3, 3).contiguous(memory_format=torch.channels_last), rnd(4, 20, 50)[:, 3:41], rnd(5, 9, dtype=F16)[1:], flat[1:400], flat[400:], rnd(6, 3, 0, 2)]
    keep = [g.clone() for g in grads]
    n = exact_norm(keep)
    got = blk().clip_grad_norm_(grads, n / 8)
    assert abs(float(got) - n) <= 2 * u * n
    for g, k in zip(grads, keep):
        within("g", g, k.double() * (n / 8 / (n + 1e-6)), 2 * u * k.double().abs())
    assert float(blk().grad_norm([base.expand(3, 40, 30)])) == pytest.approx(exact_norm([base]) * math.sqrt(3), rel=4 * u)
    out = [torch.empty(30, 40, device=DEV)]
    blk().clip_grad_norm_([base.t()], 1e9, out=out)
    assert torch.equal(out[0], base.t())


def test_clip_range_and_nonfinite():
    """magnitudes whose squares leave fp32; a norm that is not finite is returned, and nothing is written when the caller asks for an error"""
    from causaldiffae_amd import CdaeError
    big, small = torch.full((1000,), 1e30, device=DEV), torch.full((77,), 1e-30, device=DEV)
    assert float(blk().grad_norm([big])) == pytest.approx(1e30 * math.sqrt(1000), rel=1e-6)
    assert float(blk().grad_norm([small])) == pytest.approx(1e-30 * math.sqrt(77), rel=1e-6)
    for bad in (float("inf"), float("nan")):
        g = rnd(1, 100)
        g[50] = bad
        k = g.clone()
        with pytest.raises(CdaeError, match="not finite"):
            blk().clip_grad_norm_([g], 1.0, error_if_nonfinite=True)
        assert torch.equal(g.nan_to_num(), k.nan_to_num())
        n = float(blk().clip_grad_norm_([g], 1.0))
        assert n == bad or (math.isnan(n) and math.isnan(bad))
        assert g.isnan().all() if math.isnan(bad) else (g[50].isnan() and not g[:50].any())


def test_clip_empty_list():
    assert float(blk().grad_norm([])) == 0.0 and float(blk().clip_grad_norm_([], 1.0)) == 0.0


# ----------------------------------------------------------------------------- refusals
def test_refusals():
    from causaldiffae_amd import CdaeError
    b = blk()
    x, w = rnd(1, 4, 16, dtype=BF16), rnd(2, 8, 16, dtype=BF16)
    f32 = rnd(1, 4, 16)
    bad = [
        lambda: b.linear_act(x, w, act="tanh"), lambda: b.linear_act(f32, w.float()), lambda: b.linear_act(x, w.half()), lambda: b.linear_act(x, w[:, :15]),
        lambda: b.linear_act(x, w, rnd(1, 7, dtype=BF16)), lambda: b.linear_act(x, w, rnd(1, 8)), lambda: b.linear_act(x, w, res=rnd(1, 8, dtype=BF16)),
        lambda: b.linear_act(x, w.cpu()), lambda: b.linear_act(x.cpu(), w.cpu()),
        lambda: b.residual_norm(x), lambda: b.residual_norm(x, gate=w[0, :16], pre=(None, None)), lambda: b.residual_norm(x, x.float()), lambda: b.residual_norm(x, x[:3]),
        lambda: b.residual_norm(x, x, kind="batch"), lambda: b.residual_norm(x, x, eps=-1.0), lambda: b.residual_norm(x, x, alpha=float("nan")),
        lambda: b.residual_norm(x, x, pre=w[0, :15]), lambda: b.residual_norm(x, x, scale=w[0]), lambda: b.residual_norm(x, x, gate=rnd(1, 3, 16, dtype=BF16)),
        lambda: b.residual_norm(x, x, gate=rnd(1, 1, 16, dtype=BF16), pre=(None, None), scale=rnd(1, 2, 16, dtype=BF16)),
        lambda: b.residual_norm(x, x, gate=rnd(1, 16, dtype=F16)), lambda: b.residual_norm(x, x, gate=rnd(1, 16), pre=(None, None), scale=rnd(1, 16, dtype=BF16)),
        lambda: b.residual_norm(x[None], x[None], gate=rnd(1, 4, 16, dtype=BF16)),
        lambda: b.residual_norm(rnd(1, 1, 8193), None, pre=(None, None)), lambda: b.residual_norm(x.long(), None, pre=(None, None)),
        lambda: b.clip_grad_norm_([x], -1.0), lambda: b.clip_grad_norm_([x], float("nan")), lambda: b.clip_grad_norm_([x.cpu()], 1.0), lambda: b.clip_grad_norm_([x.double()], 1.0),
        lambda: b.clip_grad_norm_([x, x], 1.0), lambda: b.clip_grad_norm_([f32, f32[1:]], 1.0), lambda: b.clip_grad_norm_([f32[:1].expand(4, 16)], 1.0),
        lambda: b.clip_grad_norm_([x], 1.0, out=[]), lambda: b.clip_grad_norm_([x], 1.0, out=[f32[:3]]), lambda: b.clip_grad_norm_([x, x], 1.0, out=[f32, f32]),
        lambda: b.clip_grad_norm_([f32[:2], f32[2:]], 1.0, out=[f32[2:], f32[:2]]), lambda: b.grad_norm([x], scale=float("nan")), lambda: b.grad_norm(["x"]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(CdaeError):
            call()
            print("not refused:", i, flush=True)


# ----------------------------------------------------------------------------- together, on streams and in graphs
class Block:
    """two feed-forward blocks on rows [B, T, C], conditioned by one projection of an embedding, in the operators' own types"""

    def __init__(self, C=64, H=160, E=32, dtype=BF16):
        self.p = {}
        for i in range(2):
            self.p[f"w1.{i}"], self.p[f"b1.{i}"] = rnd(10 + i, H, C, dtype=dtype, scale=C ** -0.5), rnd(20 + i, H, dtype=dtype, scale=0.1)
            self.p[f"w2.{i}"], self.p[f"b2.{i}"] = rnd(30 + i, C, H, dtype=dtype, scale=H ** -0.5), rnd(40 + i, C, dtype=dtype, scale=0.1)
            self.p[f"ada.{i}"] = rnd(50 + i, 3 * C, E, dtype=dtype, scale=0.2 * E ** -0.5)
            self.p[f"norm.{i}"] = (1 + rnd(60 + i, C, scale=0.1)).to(dtype)
        for t in self.p.values():
            t.requires_grad_(True)

    def __call__(self, x, emb, ops):
        C = x.shape[-1]
        linear, norm = ops
        r, f, gate = x, None, None
        for i in range(2):
            a = linear(emb, self.p[f"ada.{i}"], act="silu")
            r, h = norm(r, f, gate=gate, alpha=0.7, pre=self.p[f"norm.{i}"], scale=a[:, :C], shift=a[:, C:2 * C], kind="rms")
            gate = a[:, 2 * C:]
            f = linear(linear(h, self.p[f"w1.{i}"], self.p[f"b1.{i}"], act="gelu"), self.p[f"w2.{i}"], self.p[f"b2.{i}"])
        return norm(r, f, gate=gate, alpha=0.7)[0]

    def step(self, x, emb, dy, max_norm=1.0):
        y = self(x, emb, (blk().linear_act, blk().residual_norm))
        grads = list(torch.autograd.grad(y, list(self.p.values()), dy))
        n = blk().clip_grad_norm_(grads, max_norm)
        return [y.detach(), n, *grads]


def plain_ops():
    def linear(x, w, b=None, act="none"):
        z = x.double() @ w.double().t()
        return ACT[act](z if b is None else z + b.double())

    def norm(x, f, gate=None, alpha=1.0, pre=None, scale=None, shift=None, kind="rms"):
        r = x.double()
        if f is not None:
            r = r + alpha * gate.double()[:, None] * f.double()
        if pre is None:
            return r, None
        n = r / torch.sqrt(r.pow(2).mean(-1, keepdim=True) + 1e-5) * pre.double()
        return r, n * (1 + scale.double()[:, None]) + shift.double()[:, None]

    return linear, norm


def test_block_training_step():
    """two blocks forward and backward and the clipping of their gradients against the same in 64 bits: every activation between the operators is
    rounded to bf16 (2^-8 of its size at most), and a result lies behind at most twelve of them"""
    b = Block()
    x, emb, dy = rnd(1, 4, 25, 64, dtype=BF16), rnd(2, 4, 32, dtype=BF16), rnd(3, 4, 25, 64, dtype=BF16)
    y, n, *grads = b.step(x, emb, dy, max_norm=2.0)
    ref = b(x, emb, plain_ops())
    want = torch.autograd.grad(ref, list(b.p.values()), dy.double())
    total = math.sqrt(math.fsum(float(g.double().pow(2).sum()) for g in want))
    far = lambda a, r: float((a.double() - r).norm() / r.norm())
    assert far(y, ref.detach()) < 12 * 2.0 ** -8 and abs(float(n) - total) < 12 * 2.0 ** -8 * total
    for name, g, r in zip(b.p, grads, want):
        assert far(g, r.double() * (2.0 / total)) < 24 * 2.0 ** -8, name


def test_block_repeats_to_the_bit():
    b = Block(C=136, H=200)
    args = rnd(1, 3, 70, 136, dtype=BF16), rnd(2, 3, 32, dtype=BF16), rnd(3, 3, 70, 136, dtype=BF16)
    first = b.step(*args)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, b.step(*args)))


def test_block_on_other_streams():
    """two streams at once, each with its own step: nothing is shared between calls"""
    blocks = [Block(), Block(C=72, H=96)]
    args = [(rnd(1, 4, 25, C, dtype=BF16), rnd(2, 4, 32, dtype=BF16), rnd(3, 4, 25, C, dtype=BF16)) for C in (64, 72)]
    want = [b.step(*a) for b, a in zip(blocks, args)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in blocks]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(blocks[i].step(*args[i]))
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        assert all(torch.equal(p, q) for r in runs for p, q in zip(w, r))


def test_block_in_two_graphs():
    """two captured steps, replayed several times in turn and on two streams at once, with eager work between; new inputs through the captured buffers"""
    blocks = [Block(), Block(C=72, H=96)]
    args = [[rnd(1, 4, 25, C, dtype=BF16), rnd(2, 4, 32, dtype=BF16), rnd(3, 4, 25, C, dtype=BF16)] for C in (64, 72)]
    graphs, outs = [], []
    for b, a in zip(blocks, args):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            b.step(*a)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(b.step(*a))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in blocks]
    for k in range(4):
        for i, a in enumerate(args):
            a[0].copy_(rnd(100 + 10 * k + i, *a[0].shape, dtype=BF16))
        want = [b.step(*a) for b, a in zip(blocks, args)]
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for w, o in zip(want, outs):
            assert all(torch.equal(p, q) for p, q in zip(w, o)), k


def test_capture_beside_an_eager_graph():
    """a leaf whose live eager graph was made on the default stream: the captured forward is refused before it launches anything, and the capture ends
    as any other; once that graph is gone the same step is captured"""
    from causaldiffae_amd import CdaeError
    x, w = rnd(1, 6, 64, dtype=BF16).requires_grad_(), rnd(2, 48, 64, dtype=BF16).requires_grad_()
    v = rnd(3, 64).requires_grad_()
    eager = [blk().linear_act(x, w, act="gelu"), blk().residual_norm(x.detach(), pre=v)[1]]
    calls = [lambda: blk().linear_act(x.detach(), w, act="gelu"), lambda: blk().residual_norm(x.detach(), pre=v)[1]]
    for call in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            other = w.detach() * 2
            with pytest.raises(CdaeError, match="alive"):
                call()
            with pytest.raises(CdaeError, match="captured"):
                blk().clip_grad_norm_([other], 1.0, error_if_nonfinite=True)
            with torch.no_grad():
                call()
        g.replay()
        assert torch.equal(other, w.detach() * 2)
    dy = [rnd(4 + i, *e.shape, dtype=BF16) for i, e in enumerate(eager)]
    want = [torch.autograd.grad(e, leaf, d)[0] for e, leaf, d in zip(eager, (w, v), dy)]
    del eager
    torch.cuda.synchronize()
    for call, leaf, d, one in zip(calls, (w, v), dy, want):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got, = torch.autograd.grad(call(), leaf, d)
        for _ in range(3):
            got.zero_()
            g.replay()
            assert torch.equal(got, one)


def test_linear_act_far_rows():
    """rows more than 2^22 values apart, forward and backward"""
    far = (1 << 23) + 8
    big = torch.zeros(5 * far, dtype=BF16, device=DEV)
    away = lambda r, C: big.as_strided((5, C), (far, 1), 4096 * r)
    x, w, dy = rnd(1, 5, 64, dtype=BF16), rnd(2, 48, 64, dtype=BF16), rnd(3, 5, 48, dtype=BF16)
    xs, ws, ds = away(0, 64).copy_(x).requires_grad_(), w.clone().requires_grad_(), away(1, 48).copy_(dy)
    for act in ("none", "silu"):
        a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
        ya, yb = blk().linear_act(a, b, act=act), blk().linear_act(xs, ws, act=act)
        assert torch.equal(ya, yb)
        for p, q in zip(torch.autograd.grad(ya, (a, b), dy), torch.autograd.grad(yb, (xs, ws), ds)):
            assert torch.equal(p, q)


# ----------------------------------------------------------------------------- clipping inside the optimizer step
def test_optimizer_step_clips():
    """FusedAdamWEMA.step(max_norm) is the step whose grad_scale is the factor of the definition, and leaves the gradients as they are"""
    from causaldiffae_amd.nn import Linear
    from causaldiffae_amd.train_util import FusedAdamWEMA

    def build():
        torch.manual_seed(3)
        m = torch.nn.Sequential(Linear(33, 50), Linear(50, 7)).to(DEV)
        opt = FusedAdamWEMA(m, lr=1e-2, weight_decay=0.1, ema_rates=(0.9, 0.99))
        opt.zero_grad()
        for i, p in enumerate(m.parameters()):
            p.grad.copy_(rnd(i, *p.shape))
        return m, opt

    (m1, a), (m2, b) = build(), build()
    n = exact_norm([p.grad for p in m1.parameters()], 0.5)
    for max_norm in (n / 3, n * 3, math.inf):
        keep = a.flat.grad.clone()
        a.step(grad_scale=0.5, max_norm=max_norm)
        factor = blk().grad_factor([b.flat.grad], max_norm, 0.5)
        assert abs(float(factor[1]) - 0.5 * min(1.0, max_norm / (n + 1e-6))) <= 2 * u
        b.step(grad_scale=float(factor[1]))
        assert torch.equal(keep, a.flat.grad)
        for p, q in ((a.flat.flat, b.flat.flat), (a.m, b.m), (a.v, b.v), *zip(a.ema, b.ema)):
            assert torch.equal(p, q)


def test_train_loop_clips():
    """TrainLoop(grad_clip): with a bound far above the norm a step is bit for bit the step without one; with a small bound the first moments are the
    clipped gradient's (beta1 = 0.9: m = 0.1 factor g), whose norm is the bound"""
    from improved_diffusion import script_util as su
    from improved_diffusion.train_util import TrainLoop
    data = iter([(torch.rand(2, 1, 32, 32) * 2 - 1, {"y": torch.tensor([1, 7])})] * 3)
    batch, cond = next(data)

    def loop(clip):
        torch.manual_seed(0)
        cfg = dict(image_size=32, in_channels=1, num_channels=32, num_res_blocks=1, class_cond=True, timestep_respacing="")
        model, diff = su.create_model_and_diffusion(**{**su.model_and_diffusion_defaults(), **cfg})
        model.to(DEV)
        with torch.no_grad():                       # (the zero-initialised output convs would leave most gradients at zero)
            for p in model.parameters():
                p.add_(0.02 * torch.randn(p.shape, device=DEV))
        lp = TrainLoop(model=model, diffusion=diff, data=data, batch_size=2, microbatch=-1, lr=1e-3, ema_rate="0.99", log_interval=10 ** 9, save_interval=10 ** 9,
                       resume_checkpoint="", grad_clip=clip)
        torch.manual_seed(5)
        lp.forward_backward(batch, cond)
        return lp

    a, b, c = loop(0.0), loop(1e6), loop(0.125)
    b.opt.flat.grad.copy_(a.opt.flat.grad)          # (two backward passes need not agree to the bit)
    n = exact_norm([a.opt.flat.grad])
    assert 0.125 < n < 1e6
    for lp in (a, b, c):
        lp.optimize_normal()
    assert torch.equal(a.opt.flat.flat, b.opt.flat.flat) and torch.equal(a.opt.m, b.opt.m)
    g = c.opt.flat.grad.double()
    nc = float(g.norm())
    within("m", c.opt.m, 0.1 * g * (0.125 / (nc + 1e-6)), 8 * u * g.abs() * (0.125 / nc))
    assert exact_norm([c.opt.m]) == pytest.approx(0.0125, rel=1e-4)
    with pytest.raises(ValueError):
        TrainLoop(model=None, diffusion=None, data=None, batch_size=1, microbatch=1, lr=0.0, ema_rate="0", log_interval=1, save_interval=1, resume_checkpoint="", grad_clip=-1.0)


# ----------------------------------------------------------------------------- offsets beyond 32 bits
def tail_of(rows, C, seed, dtype=BF16, last=300):
    """[rows, C] zeros whose last rows are not"""
    t = torch.zeros(rows, C, dtype=dtype, device=DEV)
    t[-last:] = rnd(seed, last, C, dtype=dtype)
    return t


def test_linear_act_long():
    """2.3 billion values in and out: the last rows are those of a call on them alone, and so are the sums when only they have a gradient"""
    M, C = (1 << 24) + 3, 136
    x, w, b = tail_of(M, C, 1), rnd(2, C, C, dtype=BF16, scale=0.1), rnd(3, C, dtype=BF16)
    xs = x[-300:].clone().requires_grad_(True)
    x, w, b = (t.requires_grad_(True) for t in (x, w, b))
    y, ys = blk().linear_act(x, w, b, act="silu"), blk().linear_act(xs, w, b, act="silu")
    assert torch.equal(y[-300:], ys) and torch.equal(y[0], blk().linear_act(torch.zeros_like(xs[:1]), w, b, act="silu")[0])
    dy = tail_of(M, C, 4)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    ref = linear_reference(xs.detach(), w.detach(), b.detach(), None, "silu", dy[-300:])
    within("dx", dx[-300:], *ref["dx"])
    assert not dx[:-300].any()
    within("dw", dw, *ref["dw"])
    within("db", db, *ref["db"])


def test_residual_norm_long():
    M, C = (1 << 22) + 1, 520
    x, f, dr, du = (tail_of(M, C, i) for i in range(4))
    v = vectors(1, C, BF16, "channel", "channel", True, True)
    leaves = [t.requires_grad_(True) for t in (x, f, *v.values())]
    call = lambda x, f: blk().residual_norm(x, f, gate=v["gate"], post=(v["w1"], v["b1"]), pre=(v["w2"], v["b2"]), scale=v["scale"], shift=v["shift"])
    r, uu = call(x, f)
    rs, us = call(x[-300:].detach(), f[-300:].detach())
    assert torch.equal(r[-300:], rs) and torch.equal(uu[-300:], us)
    got = torch.autograd.grad([r, uu], leaves, [dr, du])
    t = {k: a.detach() for k, a in v.items()}
    ref = norm_reference(x[-300:][None].detach(), f[-300:][None].detach(), t, 1.0, True, True, "layer", 1e-5, dr[-300:][None], du[-300:][None])
    for k, g in zip(["x", "f", *v], got):
        within("d" + k, g[-300:][None] if k in "xf" else g, *ref["d" + k])
    assert not got[0][:-300].any() and not got[1][:-300].any()


def test_clip_long():
    g = torch.zeros((1 << 31) + 20001, dtype=BF16, device=DEV)
    g[-1], g[5] = 3.0, 4.0
    assert float(blk().grad_norm([g])) == 5.0
    assert float(blk().clip_grad_norm_([g], 2.5)) == 5.0
    assert float(g[-1]) == 1.5 and float(g[5]) == 2.0


# ----------------------------------------------------------------------------- recomputed forwards
class Recomputed(torch.autograd.Function):
    """a checkpoint that recomputes its function and differentiates it inside its own backward"""

    @staticmethod
    def forward(ctx, fn, *inputs):
        ctx.fn = fn
        ctx.save_for_backward(*inputs)
        with torch.no_grad():
            return fn(*inputs)

    @staticmethod
    def backward(ctx, dy):
        with torch.enable_grad():
            leaves = [t.detach().requires_grad_() for t in ctx.saved_tensors]
            y = ctx.fn(*leaves)
        return (None, *torch.autograd.grad(y, leaves, dy))


def two_layers(act):
    args = [rnd(1, 30, 24, dtype=BF16), rnd(2, 40, 24, dtype=BF16, scale=0.2), rnd(3, 40, dtype=BF16), rnd(4, 16, 40, dtype=BF16, scale=0.2)]
    fn = lambda x, w1, b1, w2: blk().linear_act(blk().linear_act(x, w1, b1, act=act), w2, act=act)
    return fn, [t.requires_grad_() for t in args], rnd(5, 30, 16, dtype=BF16)


@pytest.mark.parametrize("act", ["gelu", "none"])
def test_linear_act_in_a_checkpoint(act):
    """the package's checkpoint recomputes the forward inside a backward that was asked for some inputs only"""
    from causaldiffae_amd.nn import checkpoint
    fn, leaves, dy = two_layers(act)
    want = torch.autograd.grad(fn(*leaves), leaves, dy)
    for pick in ([0], [1], [3], [0, 1, 2, 3]):
        got = torch.autograd.grad(checkpoint(fn, leaves, (), True), [leaves[i] for i in pick], dy)
        assert all(torch.equal(g, want[i]) for g, i in zip(got, pick))


@pytest.mark.parametrize("act", ["gelu", "none"])
def test_linear_act_recomputed_with_a_backward_of_its_own(act):
    fn, leaves, dy = two_layers(act)
    want = torch.autograd.grad(fn(*leaves), leaves, dy)
    for pick in ([0], [3], [0, 1, 2, 3]):
        got = torch.autograd.grad(Recomputed.apply(fn, *leaves), [leaves[i] for i in pick], dy)
        assert all(torch.equal(g, want[i]) for g, i in zip(got, pick))


def test_residual_norm_in_a_checkpoint():
    from causaldiffae_amd.nn import checkpoint
    fn = lambda x, w: blk().residual_norm(x, x, pre=w)[1]
    leaves, dy = [rnd(1, 9, 40).requires_grad_(), rnd(2, 40).requires_grad_()], rnd(3, 9, 40)
    want = torch.autograd.grad(fn(*leaves), leaves, dy)
    for i in range(2):
        for run in (lambda: checkpoint(fn, leaves, (), True), lambda: Recomputed.apply(fn, *leaves)):
            assert torch.equal(torch.autograd.grad(run(), leaves[i], dy)[0], want[i])


# ----------------------------------------------------------------------------- more samples than a launch has blocks
@pytest.mark.parametrize("kind,T", [("layer", 1), ("rms", 1), ("layer", 3)])
def test_residual_norm_more_samples_than_blocks(kind, T):
    """blocks that walk several chunks of an odd number of sums (one norm, one or three rows a sample), against the same samples in calls of one chunk a block"""
    B, C, part = (1 << 20) + 5, 520, 1 << 18
    g = torch.Generator(device=DEV).manual_seed(7)
    x = torch.randn(B, T, C, generator=g, device=DEV, dtype=BF16)
    scale = torch.randn(B, C, generator=g, device=DEV, dtype=BF16)
    w = 1 + rnd(1, C, dtype=BF16, scale=0.1)
    got = blk().residual_norm(x, pre=w, scale=scale, kind=kind)[1]
    for b in range(0, B, part):
        assert torch.equal(got[b:b + part], blk().residual_norm(x[b:b + part], pre=w, scale=scale[b:b + part], kind=kind)[1]), b


# ----------------------------------------------------------------------------- activations far below one
@pytest.mark.parametrize("M,K,N", [(5, 16, 24), (40, 24, 67), (64, 4096, 72), (3, 1, 1)])
@pytest.mark.parametrize("dtype,xs,ws", [(BF16, 1e-9, 1.0), (BF16, 1e-15, 1e-15), (F16, 1e-4, 1e-5)])
def test_linear_act_relu_small(M, K, N, dtype, xs, ws):
    """rows of one sign each with a positive weight, so that every sum has its sign: the slope is 1 on the positive rows however small z is"""
    sign = 1.0 - 2.0 * (torch.arange(M, device=DEV) % 2)[:, None]
    x = (sign * xs * (0.5 + rnd(1, M, K).abs()) / K).to(dtype) if dtype == BF16 else (sign * xs * (0.5 + rnd(1, M, K).abs())).to(dtype)
    w, dy = (ws * (0.5 + rnd(2, N, K).abs())).to(dtype), rnd(3, M, N, dtype=dtype)
    b = torch.zeros(N, dtype=dtype, device=DEV)
    x, w, b = (t.requires_grad_() for t in (x, w, b))
    dx, dw, db = torch.autograd.grad(blk().linear_act(x, w, b, act="relu"), (x, w, b), dy)
    dz = dy.double() * (sign > 0)
    for name, g, a, c in (("dx", dx, dz, w.detach().double()), ("dw", dw, dz.t(), x.detach().double()), ("db", db[None], torch.ones(1, M, dtype=torch.float64, device=DEV), dz)):
        within(name, g, a @ c, (a.shape[1] + 8) * u * (a.abs() @ c.abs()))


# ----------------------------------------------------------------------------- tensors that are more than their values
def test_forward_mode_is_refused():
    """a tangent would be lost without a word"""
    import torch.autograd.forward_ad as fwad
    from causaldiffae_amd import CdaeError
    x, w, v = rnd(1, 6, 16, dtype=BF16), rnd(2, 8, 16, dtype=BF16), rnd(3, 6, 8, dtype=BF16)
    with fwad.dual_level():
        dual = lambda t: fwad.make_dual(t, torch.ones_like(t))
        calls = [lambda: blk().linear_act(dual(x), w), lambda: blk().linear_act(x, dual(w)), lambda: blk().linear_act(x, w, dual(w[:, 0])), lambda: blk().linear_act(x, w, res=dual(v)),
                 lambda: blk().residual_norm(dual(x), x), lambda: blk().residual_norm(x, dual(x)), lambda: blk().residual_norm(x, x, gate=dual(x[0])),
                 lambda: blk().residual_norm(x, pre=dual(x[0])), lambda: blk().grad_norm([x, dual(x)]), lambda: blk().clip_grad_norm_([dual(x)], 1.0),
                 lambda: blk().clip_grad_norm_([x], 1.0, out=[dual(x.clone())])]
        for call in calls:
            with pytest.raises(CdaeError, match="forward"):
                call()
        assert torch.equal(blk().linear_act(x, w), blk().linear_act(x.clone(), w))
        a = x.clone().requires_grad_()
        for y in (blk().linear_act(a, w), *blk().residual_norm(a, x, pre=x[0])):
            with pytest.raises(RuntimeError, match="forward"):
                torch.autograd.grad(y, a, dual(torch.ones_like(y)))


def test_tensors_negated_lazily():
    """a tensor whose values lie negated in memory counts with its values"""
    neg = torch._neg_view
    x, f, w = rnd(1, 6, 16, dtype=BF16), rnd(2, 6, 16, dtype=BF16), rnd(3, 8, 16, dtype=BF16)
    b, res = rnd(4, 8, dtype=BF16), rnd(5, 6, 8, dtype=BF16)
    for i in range(4):
        args = [x, w, b, res]
        args[i] = -args[i]
        want = blk().linear_act(*args, act="silu")
        args[i] = neg([x, w, b, res][i])
        assert args[i].is_neg() and torch.equal(blk().linear_act(*args, act="silu"), want)
    for k in ("x", "f", "gate", "scale", "pre"):
        args = {"x": x, "f": f, "gate": x[0], "scale": f[:2], "pre": w[0]}
        want = blk().residual_norm(**{**args, k: -args[k]})
        got = blk().residual_norm(**{**args, k: neg(args[k])})
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    leaf = w.clone().requires_grad_()
    g, = torch.autograd.grad(blk().linear_act(x, leaf), leaf, neg(res))
    assert torch.equal(g, torch.autograd.grad(blk().linear_act(x, leaf), leaf, -res)[0])
    leaf = x.clone().requires_grad_()
    g, = torch.autograd.grad(blk().residual_norm(leaf, pre=w[0])[1], leaf, neg(f))
    assert torch.equal(g, torch.autograd.grad(blk().residual_norm(leaf, pre=w[0])[1], leaf, -f)[0])
    n = exact_norm([x])
    out = torch.empty(6, 16, device=DEV)
    blk().clip_grad_norm_([neg(x)], n / 2, out=[out])
    within("out", out, -x.double() * (n / 2 / (n + 1e-6)), 2 * u * x.double().abs())
    a = x.clone()
    blk().clip_grad_norm_([neg(a)], n / 2)
    within("in place", a, x.double() * (n / 2 / (n + 1e-6)), 2 * u * x.double().abs())


def test_layouts_are_refused():
    from causaldiffae_amd import CdaeError
    x, w = rnd(1, 6, 16), rnd(2, 8, 16, dtype=BF16)
    sparse = x.relu().to_sparse()
    for call in (lambda: blk().linear_act(sparse.to(BF16), w), lambda: blk().linear_act(x.to(BF16), w.relu().to_sparse()), lambda: blk().residual_norm(sparse, x), lambda: blk().residual_norm(x, sparse),
                 lambda: blk().residual_norm(x, pre=x[0].relu().to_sparse()), lambda: blk().grad_norm([sparse]),
                 lambda: blk().clip_grad_norm_([x], 1.0, out=[torch._neg_view(torch.empty_like(x))])):
        with pytest.raises(CdaeError):
            call()


@pytest.mark.parametrize("B,T,C,dtype,gate,mod", [(9000, 1, 1000, BF16, "sample", "sample"), (20000, 2, 264, F32, "channel", "sample"), (70000, 1, 72, F16, "sample", "channel"),
                                                  (600, 1, 8192, BF16, "channel", "channel"), (40, 1, 520, F32, "sample", "sample"), (33, 3, 5, BF16, "sample", None)])
def test_residual_norm_sample_folds(B, T, C, dtype, gate, mod):
    """few rows a sample: samples folded in groups, and (the first three) in several slabs that share one place for their column sums"""
    v = vectors(B, C, dtype, gate, mod, True, True)
    r = lambda s: rnd(s, B, T, C, dtype=dtype)
    check_norm(r(1), r(2), v, 0.7, True, True, "layer", dr=r(3), du=r(4))


def test_residual_norm_without_vector_gradients():
    """vectors that need no gradient: the gradients of the rows are the same, without the column sums' scratch"""
    B, T, C = 2000, 1, 4000
    v = vectors(B, C, BF16, "sample", "sample", True, True)
    x, f, dr, du = (rnd(s, B, T, C, dtype=BF16) for s in (1, 2, 3, 4))
    call = lambda: blk().residual_norm(x, f, gate=v["gate"], post=(v["w1"], v["b1"]), pre=(v["w2"], v["b2"]), scale=v["scale"], shift=v["shift"])
    x.requires_grad_(), f.requires_grad_()
    outs = call()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    alone = torch.autograd.grad(outs, (x, f), (dr, du))
    assert torch.cuda.max_memory_allocated() - before < 3 * x.numel() * 2
    for t in v.values():
        t.requires_grad_()
    both = torch.autograd.grad(call(), (x, f, *v.values()), (dr, du))
    assert all(torch.equal(p, q) for p, q in zip(alone, both))


def test_residual_norm_gradients_own_their_memory():
    """a gradient that is kept or saved keeps nothing else"""
    v = vectors(3, 40, BF16, "sample", "sample", True, True)
    got = check_norm(rnd(1, 3, 7, 40, dtype=BF16), rnd(2, 3, 7, 40, dtype=BF16), v, 1.0, True, True, "layer", dr=rnd(3, 3, 7, 40, dtype=BF16), du=rnd(4, 3, 7, 40, dtype=BF16))
    for k, g in got.items():
        if k.startswith("d"):
            assert g.untyped_storage().nbytes() == g.numel() * g.element_size(), k


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("act,low", [("gelu", -12.5), ("gelu_tanh", -9.0), ("silu", -80.0)])
def test_linear_act_tails(act, low, dtype):
    """the activation's and the slope's own accuracy where they fall towards zero: one-value rows, so z is the input, exact in fp16 too.  Relative bounds:
    an exponential 2^t is off by (t + 2) u relative per rounding of t, of which there are at most four, everything else by a few u"""
    z = torch.linspace(low, 9.0, 1 << 14, device=DEV).to(BF16).to(dtype).unique()[:, None]
    x, w = z.clone().requires_grad_(), torch.ones(1, 1, dtype=dtype, device=DEV)
    y = blk().linear_act(x, w, act=act)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    z = z.double()
    if act == "gelu":
        s, t = 0.5 * torch.special.erfc(-z / math.sqrt(2)), 0.7213475204444817 * z * z
        slope, size = s + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), s + z.abs() * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    else:
        a, da = (z, torch.ones_like(z)) if act == "silu" else (1.5957691216057308 * (z + 0.044715 * z ** 3), 1.5957691216057308 * (1 + 0.134145 * z * z))
        s, t = torch.sigmoid(a), 1.4426950408889634 * a.abs()
        slope, size = s * (1 + z * torch.sigmoid(-a) * da), s * (1 + z.abs() * torch.sigmoid(-a) * da)
    rel = (4 * t + 32) * u
    within("y", y.detach(), z * s, rel * (z * s).abs())
    # (as an operand dz is rounded, and the product by one rounds no further)
    within("dx", dx, slope, rel * size)


def test_saved_tensors_that_come_back_in_another_layout():
    """hooks on saved tensors (offloading, compression) may hand back the same values in any layout"""
    def other_layout(t):
        return t.mT.contiguous().mT if t.dim() > 1 else torch.stack([t, t], -1)[:, 0]

    x, w, b = rnd(1, 3, 10, 40, dtype=BF16), rnd(2, 24, 40, dtype=BF16, scale=0.2), rnd(3, 24, dtype=BF16)
    f, dr, du, v = rnd(4, 3, 10, 40, dtype=BF16), rnd(5, 3, 10, 40, dtype=BF16), rnd(6, 3, 10, 40, dtype=BF16), vectors(3, 40, BF16, "sample", "sample", True, True)
    leaves = [t.requires_grad_() for t in (x, f, *v.values())]
    linear = lambda: torch.autograd.grad(blk().linear_act(x, w, b, act="gelu"), (x, w, b), rnd(7, 3, 10, 24, dtype=BF16))
    norm = lambda: torch.autograd.grad(blk().residual_norm(x, f, gate=v["gate"], post=(v["w1"], v["b1"]), pre=(v["w2"], v["b2"]), scale=v["scale"], shift=v["shift"]), leaves, (dr, du))
    w.requires_grad_(), b.requires_grad_()
    for run in (linear, norm):
        want = run()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, other_layout):
            got = run()
        assert all(torch.equal(p, q) for p, q in zip(got, want)), run
