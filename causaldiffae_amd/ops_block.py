"""Operators of an embedding-conditioned feed-forward block on rows, and of the step that trains it (kernels: lin16.hip, resnorm.hip, gradclip.hip):

    linear_act       y = act(x W^T + b) + res                              bf16 / fp16 rows
    residual_norm    r = x + alpha gate o post(f),  u = pre(r) o (1 + scale) + shift          bf16 / fp16 / fp32 rows
    grad_norm        the global norm of many gradients
    clip_grad_norm_  gradients times min(1, max_norm / norm), in place or into other buffers

A block is residual_norm -> linear_act (activation) -> linear_act -> residual_norm: the second residual_norm closes this block and opens the next.
Rows are the last dimension: an activation [N, C, H, W] in this package's NHWC storage is passed as x.permute(0, 2, 3, 1).

Sums, statistics and products accumulate in fp32 (the norm of the gradients in fp64) and every result is rounded once.  Calls run on the current
stream of their tensors' device, allocate their scratch themselves for the one call, neither synchronise nor copy to the host, keep nothing between
calls and can be captured into a graph.  Wrong arguments raise CdaeError; there is no CPU form.
"""
import array
import contextlib
import ctypes
import math

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from ._lib import CdaeError, ResNorm, check, lib, stream

TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
ACTS = {"none": 0, "silu": 1, "relu": 3, "gelu": 5, "gelu_tanh": 6}
MAX_FEATURES = 8192          # widest row of residual_norm

_NOTHING = contextlib.nullcontext()
_LIN_FWD, _LIN_BWD = 0, 1


def _refuse(ok, what):
    if not ok:
        raise CdaeError(what)


def _on(dev):
    """Makes `dev` the current device for a launch (its current stream is then the one the launch goes to)."""
    return _NOTHING if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _device_of(who, x, others):
    _refuse(isinstance(x, torch.Tensor) and x.is_cuda, f"{who}: tensors on an MI355X device required; there is no CPU form")
    for t in others:
        _refuse(t is None or (isinstance(t, torch.Tensor) and t.device == x.device), f"{who}: all tensors on one device ({x.device})")


def _rows(t, C):
    """[..., C] as rows [M, C] whose values lie side by side, at any pitch of at least a row (a copy where they do not)."""
    t = t.reshape(-1, C)
    if (C == 1 or t.stride(1) == 1) and (t.shape[0] <= 1 or t.stride(0) >= C):
        return t
    return t.contiguous()


def _pitch(t, C):
    return C if t.shape[0] <= 1 else t.stride(0)


def _scratch(nbytes, dev):
    return torch.empty(max(1, nbytes), dtype=torch.uint8, device=dev)


# ----------------------------------------------------------------------------- linear layer with activation and residual
class _LinearAct(Function):
    @staticmethod
    def forward(ctx, x, w, b, res, act):
        M, K = x.shape
        N = w.shape[0]
        dev = x.device
        dt = TYPES[x.dtype]
        grad = any(ctx.needs_input_grad[:3])
        y = torch.empty((M, N), dtype=x.dtype, device=dev)
        z = torch.empty((M, N), dtype=torch.float16, device=dev) if grad and act else None
        if M:
            need = lib.cdae_lin16_workspace_bytes(_LIN_FWD, M, N, K)
            with _on(dev):
                ws = _scratch(need, dev)
                check(lib.cdae_lin16_fwd(x.data_ptr(), _pitch(x, K), w.data_ptr(), _pitch(w, K), _ptr(b), _ptr(res), 0 if res is None else _pitch(res, N),
                                         y.data_ptr(), N, _ptr(z), N, M, N, K, act, dt, ws.data_ptr(), need, stream()))
        if grad:
            ctx.save_for_backward(x, w, z)
            ctx.act = act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        dres = dy if ctx.needs_input_grad[3] else None
        if not any(ctx.needs_input_grad[:3]):
            return None, None, None, dres, None
        x, w, z = ctx.saved_tensors
        M, K = x.shape
        N = w.shape[0]
        dev = x.device
        new = torch.empty if M else torch.zeros                  # (no rows: the sums over them are zero)
        dx = torch.empty((M, K), dtype=x.dtype, device=dev) if ctx.needs_input_grad[0] else None
        dw = new((N, K), dtype=x.dtype, device=dev) if ctx.needs_input_grad[1] else None
        db = new((N,), dtype=x.dtype, device=dev) if ctx.needs_input_grad[2] else None
        if M:
            dyr = _rows(dy, N)
            need = lib.cdae_lin16_workspace_bytes(_LIN_BWD, M, N, K)
            with _on(dev):
                ws = _scratch(need, dev)
                check(lib.cdae_lin16_bwd(dyr.data_ptr(), _pitch(dyr, N), x.data_ptr(), _pitch(x, K), w.data_ptr(), _pitch(w, K), _ptr(z), N, _ptr(dx), K,
                                         _ptr(dw), K, _ptr(db), M, N, K, ctx.act, TYPES[x.dtype], ws.data_ptr(), need, stream()))
        return dx, dw, db, dres, None


def linear_act(x, w, b=None, res=None, act="none"):
    """y = act(x @ w^T + b) + res for rows x [..., K], a weight [N, K], a bias [N] and a residual [..., N], all bf16 or all fp16; y has their type.
    act: "none", "silu", "relu", "gelu" or "gelu_tanh".  Where a gradient is wanted the pre-activation is kept in fp16 beside x and w.  Rows at any
    pitch and alignment are taken as they are; fp32 rows belong to ops.linear."""
    _device_of("linear_act", x, (w, b, res))
    _refuse(act in ACTS, f"linear_act: act is one of {', '.join(ACTS)}")
    _refuse(x.dtype in (torch.bfloat16, torch.float16), f"linear_act: bf16 or fp16 rows (got {x.dtype}; ops.linear takes fp32)")
    _refuse(x.dim() >= 1 and w.dim() == 2 and w.shape[0] >= 1 and w.shape[1] >= 1 and x.shape[-1] == w.shape[1],
            f"linear_act: rows [..., K] and a weight [N, K] (got {tuple(x.shape)} and {tuple(w.shape)})")
    N, K = w.shape
    shape = x.shape[:-1] + (N,)
    _refuse(w.dtype == x.dtype and (b is None or b.dtype == x.dtype) and (res is None or res.dtype == x.dtype), "linear_act: x, w, b and res of one type")
    _refuse(b is None or tuple(b.shape) == (N,), f"linear_act: a bias [{N}]")
    _refuse(res is None or res.shape == shape, f"linear_act: a residual {tuple(shape)} (nothing is broadcast)")
    _refuse(x.numel() // K < 2 ** 31, "linear_act: fewer than 2^31 rows")
    y = _LinearAct.apply(_rows(x, K), _rows(w, K), None if b is None else b.contiguous(), None if res is None else _rows(res, N), ACTS[act])
    return y.view(shape)


# ----------------------------------------------------------------------------- the norms around a block
class _ResidualNorm(Function):
    @staticmethod
    def forward(ctx, x, f, gate, scale, shift, w1, b1, w2, b2, cfg):
        B, T, C, alpha, eps, layer, post, pre = cfg
        M = B * T
        dev = x.device
        ctx.set_materialize_grads(False)
        r = torch.empty((M, C), dtype=x.dtype, device=dev) if f is not None else None
        u = torch.empty((M, C), dtype=x.dtype, device=dev) if pre else None
        if M:
            p = _fill(x, f, gate, scale, shift, w1, b1, w2, b2, cfg)
            p.r, p.u = _ptr(r), _ptr(u)
            with _on(dev):
                check(lib.cdae_resnorm_fwd(ctypes.byref(p), stream()))
        ctx.save_for_backward(x, f, gate, scale, shift, w1, b1, w2, b2)
        ctx.cfg = cfg
        return r, u

    @staticmethod
    @once_differentiable
    def backward(ctx, dr, du):
        tensors = ctx.saved_tensors
        if dr is None and du is None:
            return (None,) * 10
        B, T, C = ctx.cfg[:3]
        M = B * T
        x = tensors[0]
        dev = x.device
        rows = lambda t, i: torch.empty((M, C), dtype=t.dtype, device=dev) if ctx.needs_input_grad[i] else None
        vec = lambda t, i: (torch.empty if M else torch.zeros)(t.shape, dtype=t.dtype, device=dev) if ctx.needs_input_grad[i] else None
        grads = [rows(t, i) if i < 2 else vec(t, i) for i, t in enumerate(tensors)]
        if M:
            p = _fill(*tensors, ctx.cfg)
            dr, du = (None if d is None else _rows(d, C) for d in (dr, du))
            p.dr, p.ld_dr = _ptr(dr), 0 if dr is None else _pitch(dr, C)
            p.du, p.ld_du = _ptr(du), 0 if du is None else _pitch(du, C)
            p.dx, p.df, p.dgate, p.dscale, p.dshift, p.dw1, p.db1, p.dw2, p.db2 = (_ptr(g) for g in grads)
            need = lib.cdae_resnorm_workspace_bytes(B, T, C)
            with _on(dev):
                ws = _scratch(need, dev)
                p.ws, p.ws_bytes = ws.data_ptr(), need
                check(lib.cdae_resnorm_bwd(ctypes.byref(p), stream()))
        return (*grads, None)


def _fill(x, f, gate, scale, shift, w1, b1, w2, b2, cfg):
    B, T, C, alpha, eps, layer, post, pre = cfg
    p = ResNorm()
    p.B, p.T, p.C, p.dt, p.layer, p.post, p.pre, p.alpha, p.eps = B, T, C, TYPES[x.dtype], layer, post, pre, alpha, eps
    f32 = torch.float32
    p.vec32 = int(any(v is not None and v.dtype == f32 for v in (gate, scale, shift)))
    p.w32 = int(any(v is not None and v.dtype == f32 for v in (w1, b1, w2, b2)))
    p.x, p.ld_x = x.data_ptr(), _pitch(x, C)
    if f is not None:
        p.f, p.ld_f = f.data_ptr(), _pitch(f, C)
    if gate is not None:
        p.gate, p.shared_gate, p.ld_gate = gate.data_ptr(), int(gate.dim() == 1), gate.stride(0)
    if scale is not None:
        p.scale, p.shared_scale, p.ld_scale = scale.data_ptr(), int(scale.dim() == 1), scale.stride(0)
    if shift is not None:
        p.shift, p.shared_shift, p.ld_shift = shift.data_ptr(), int(shift.dim() == 1), shift.stride(0)
    p.w1, p.b1, p.w2, p.b2 = _ptr(w1), _ptr(b1), _ptr(w2), _ptr(b2)
    return p


def _norm_arg(who, n):
    """None -> (absent, None, None); a weight, or a (weight, bias) pair whose members may be None -> (present, weight, bias)"""
    if n is None:
        return 0, None, None
    if isinstance(n, torch.Tensor):
        return 1, n, None
    _refuse(isinstance(n, (tuple, list)) and len(n) == 2, f"residual_norm: {who} is None, a weight or a (weight, bias) pair")
    return 1, n[0], n[1]


def residual_norm(x, f=None, *, gate=None, alpha=1.0, post=None, pre=None, scale=None, shift=None, kind="layer", eps=1e-5):
    """The norms before and after a block, its gate and the residual scale in one pass; returns (r, u):

        r = x + alpha * gate o post(f)            u = pre(r) o (1 + scale) + shift

    x, f: rows [..., C] of one type (bf16, fp16 or fp32), C <= 8192.  f None: r is x itself (the first norm of a network).  pre None: u is None (the
    last block).  post and pre: None (no norm), a weight [C], or a pair (weight, bias) of which either may be None; both are layer norms or, with
    kind="rms", rms norms.  gate, scale, shift: None, one vector [C] for all rows, or one for each sample [B, C], where B is x.shape[0] (rows [M, C]:
    any B that divides M, a sample's rows following each other).  gate, scale and shift are in the rows' type or all in fp32, and so are the weights."""
    w = {}
    has_post, w["w1"], w["b1"] = _norm_arg("post", post)
    has_pre, w["w2"], w["b2"] = _norm_arg("pre", pre)
    vec = {"gate": gate, "scale": scale, "shift": shift}
    _device_of("residual_norm", x, (f, *vec.values(), *w.values()))
    _refuse(kind in ("layer", "rms"), 'residual_norm: kind is "layer" or "rms"')
    _refuse(x.dtype in TYPES, f"residual_norm: bf16, fp16 or fp32 rows (got {x.dtype})")
    _refuse(x.dim() >= 1 and 1 <= x.shape[-1] <= MAX_FEATURES, f"residual_norm: rows of 1 to {MAX_FEATURES} features")
    C = x.shape[-1]
    M = x.numel() // C
    _refuse(M < 2 ** 31, "residual_norm: fewer than 2^31 rows")
    _refuse(math.isfinite(alpha) and math.isfinite(eps) and eps >= 0, "residual_norm: alpha finite, eps finite and not negative")
    _refuse(f is None or (f.shape == x.shape and f.dtype == x.dtype), "residual_norm: f of x's shape and type")
    _refuse(f is not None or has_pre, "residual_norm: without f there is only the pre norm to compute")
    _refuse(f is not None or (gate is None and not has_post), "residual_norm: a gate and a post norm belong to f")
    _refuse(has_pre or (scale is None and shift is None), "residual_norm: scale and shift belong to the pre norm")
    for name, v in w.items():
        _refuse(v is None or (tuple(v.shape) == (C,) and v.dtype in (x.dtype, torch.float32)), f"residual_norm: {name[0] == 'w' and 'a weight' or 'a bias'} [{C}] in the rows' type or fp32")
    _refuse(len({v.dtype for v in w.values() if v is not None}) <= 1, "residual_norm: weights and biases of one type")
    B = None
    for name, v in vec.items():
        if v is None:
            continue
        _refuse(v.dtype in (x.dtype, torch.float32) and v.dim() in (1, 2) and v.shape[-1] == C, f"residual_norm: {name} [{C}] or [B, {C}] in the rows' type or fp32")
        if v.dim() == 2:
            _refuse(v.shape[0] == x.shape[0] if x.dim() > 2 else v.shape[0] >= 1 and M % v.shape[0] == 0 or v.shape[0] == M,
                    f"residual_norm: {name} has a row for each sample of x (got {tuple(v.shape)} beside {tuple(x.shape)})")
            _refuse(B in (None, v.shape[0]), "residual_norm: gate, scale and shift for the same samples")
            B = v.shape[0]
    _refuse(len({v.dtype for v in vec.values() if v is not None}) <= 1, "residual_norm: gate, scale and shift of one type")
    side = lambda v: v if v is None or v.stride(-1) == 1 or C == 1 else v.contiguous()
    B = 1 if B is None else B
    T = M // B if B else 0
    cfg = (B, T, C, float(alpha), float(eps), int(kind == "layer"), has_post, has_pre)
    r, u = _ResidualNorm.apply(_rows(x, C), None if f is None else _rows(f, C), *(side(v) for v in vec.values()), *(side(v) for v in w.values()), cfg)
    return x if f is None else r.view(x.shape), None if u is None else u.view(x.shape)


# ----------------------------------------------------------------------------- the global norm of many gradients
def _dense(t):
    """values without gaps or overlap, in whatever order of the dimensions"""
    if t.is_contiguous():
        return True
    at = 1
    for st, n in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1):
        if st != at:
            return False
        at *= n
    return True


class _List:
    """Gradients as the arrays the library takes."""

    def __init__(self, who, tensors):
        self.t = list(tensors)
        for t in self.t:
            _refuse(isinstance(t, torch.Tensor) and t.is_cuda and t.layout == torch.strided and t.dtype in TYPES,
                    f"{who}: dense bf16, fp16 or fp32 tensors on an MI355X device; there is no CPU form")
        devs = {t.device for t in self.t}
        _refuse(len(devs) <= 1, f"{who}: tensors of one device")
        self.dev = devs.pop() if devs else torch.device("cuda", torch.cuda.current_device())

    def arrays(self):
        self._keep = (array.array("Q", [t.data_ptr() for t in self.t]), array.array("q", [t.numel() for t in self.t]), array.array("i", [TYPES[t.dtype] for t in self.t]))
        return tuple(a.buffer_info()[0] for a in self._keep)


def _number(who, name, v, least=None):
    v = float(v)
    _refuse(not math.isnan(v) and (least is None or v >= least), f"{who}: {name} must be a number" + ("" if least is None else f" >= {least:g}"))
    return v


def _norm_into(who, lst, scale, max_norm):
    """fp32 [norm, factor] on the device"""
    out = torch.empty(2, dtype=torch.float32, device=lst.dev)
    need = lib.cdae_grad_workspace_bytes()
    with _on(lst.dev):
        ws = _scratch(need, lst.dev)
        p, n, ty = lst.arrays()
        check(lib.cdae_grad_norm(p, n, ty, len(lst.t), scale, max_norm, out.data_ptr(), ws.data_ptr(), need, stream()))
    return out


def grad_norm(grads, scale=1.0):
    """|scale| * sqrt(sum of all squares) over a list of gradients (any sizes, bf16 / fp16 / fp32 mixed) as a fp32 scalar on their device.  Squares
    and sums are fp64, in a fixed order: the result is finite wherever it fits fp32, and the same in every run."""
    scale = _number("grad_norm", "scale", scale)
    lst = _List("grad_norm", [t if not isinstance(t, torch.Tensor) or _dense(t) else t.contiguous() for t in grads])
    return _norm_into("grad_norm", lst, scale, math.inf)[0]


def grad_factor(grads, max_norm, scale=1.0):
    """fp32 [2] on the device: the norm, and the factor scale * min(1, max_norm / (norm + 1e-6)) that clips by it (FusedAdamWEMA.step reads it there)."""
    scale, max_norm = _number("grad_factor", "scale", scale), _number("grad_factor", "max_norm", max_norm, 0.0)
    lst = _List("grad_factor", [t if not isinstance(t, torch.Tensor) or _dense(t) else t.contiguous() for t in grads])
    return _norm_into("grad_factor", lst, scale, max_norm)


def clip_grad_norm_(grads, max_norm, scale=1.0, out=None, error_if_nonfinite=False):
    """out_i = g_i * scale * min(1, max_norm / (norm + 1e-6)) with norm = grad_norm(grads, scale), which is returned (fp32 scalar on the device).

    grads: the gradients themselves ([p.grad for p in model.parameters() if p.grad is not None]), any sizes and strides, bf16 / fp16 / fp32 mixed.
    scale: what the gradients have to be multiplied by first (1 / loss scale, 1 / ranks of a sum).  out: None (in place), or tensors of the same shapes
    and any of the types, e.g. fp32 master gradients; outputs may not share memory with each other or with another gradient.  A norm that is not finite
    leaves zeros or NaN: error_if_nonfinite=True raises instead, before anything is written, at the cost of waiting for the device."""
    who = "clip_grad_norm_"
    scale, max_norm = _number(who, "scale", scale), _number(who, "max_norm", max_norm, 0.0)
    src = _List(who, grads)
    later = []                                           # (tensor with gaps, dense copy): written back at the end
    if out is None:
        dst = src
        for i, t in enumerate(src.t):
            if not _dense(t):
                _refuse(all(st for st, n in zip(t.stride(), t.shape) if n > 1), f"{who}: an expanded tensor cannot be written in place")
                src.t[i] = t.contiguous()
                later.append((t, src.t[i]))
    else:
        dst = _List(who, out)
        _refuse(len(dst.t) == len(src.t) and all(a.shape == b.shape for a, b in zip(src.t, dst.t)) and (dst.dev == src.dev or not src.t),
                f"{who}: out is a tensor of the same shape for every gradient, on the same device")
        for i, (a, b) in enumerate(zip(src.t, dst.t)):
            _refuse(_dense(b), f"{who}: outputs without gaps")
            if not _dense(a) or (a.stride() != b.stride() and not (a.is_contiguous() and b.is_contiguous())):
                src.t[i] = torch.empty_strided(b.shape, b.stride(), dtype=a.dtype, device=a.device).copy_(a)
    if error_if_nonfinite:
        n = _norm_into(who, src, scale, max_norm)[0]
        _refuse(math.isfinite(n.item()), f"{who}: the norm of the gradients is not finite ({n.item()})")
    norm = torch.empty(2, dtype=torch.float32, device=src.dev)
    need = lib.cdae_grad_workspace_bytes()
    with _on(src.dev):
        ws = _scratch(need, src.dev)
        p, n, ty = src.arrays()
        po, _, to = dst.arrays() if dst is not src else (p, n, ty)
        check(lib.cdae_grad_clip(p, n, ty, po, to, len(src.t), scale, max_norm, norm.data_ptr(), ws.data_ptr(), need, stream()))
        for t, c in later:
            t.copy_(c)
    torch.autograd.graph.increment_version(dst.t)        # (the kernel wrote them behind autograd's back)
    return norm[0]
