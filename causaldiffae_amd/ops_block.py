"""Operators of an embedding-conditioned feed-forward block on rows, and of the step that trains it (kernels: lin16.hip, resnorm.hip, gradclip.hip):

    linear_act       y = act(x W^T + b) + res                              bf16 / fp16 rows
    residual_norm    r = x + alpha gate o post(f),  u = pre(r) o (1 + scale) + shift          bf16 / fp16 / fp32 rows
    grad_norm        the global norm of many gradients
    clip_grad_norm_  gradients times min(1, max_norm / norm), in place or into other buffers

A block is residual_norm -> linear_act (activation) -> linear_act -> residual_norm: the second residual_norm closes this block and opens the next.
Rows are the last dimension: an activation [N, C, H, W] in this package's NHWC storage is passed as x.permute(0, 2, 3, 1).

Sums, statistics and products accumulate in fp32 (the norm of the gradients in fp64) and every result is rounded once.  linear_act's backward rounds twice
more in between, both named there: with an activation, its gradients of x and w are 1.4 times as far from the exact ones as one rounding would leave them.

Calls run on the current stream of their tensors' device, allocate their scratch themselves for the one call, neither synchronise nor copy to the host,
keep nothing between calls and can be captured into a graph.  (A backward pass is captured together with its forward, and only while no eager graph over the
same leaves, made on the default stream, is alive: the captured forward raises then.)  Gradients are first derivatives; a second one raises, and so does an
input that carries a forward-mode tangent.  Wrong tensors and values raise CdaeError; there is no CPU form.  The checks and the autograd nodes are native
(csrc/block_ext.cpp): the kernels of a call are shorter than the same dispatch from Python.
"""
import torch

from . import _lib  # (libcdae.so, which the extension calls, and its errors)

try:
    from . import _block_ext as _ext
except ImportError as e:
    raise ImportError(f"causaldiffae_amd/_block_ext.so does not load ({e}): build it first (causaldiffae_amd/csrc/build.sh)") from e

_ext.set_errors(_lib.CdaeError, torch.OutOfMemoryError)

MAX_FEATURES = 8192          # widest row of residual_norm


def linear_act(x, w, b=None, res=None, act="none"):
    """y = act(x @ w^T + b) + res for rows x [..., K], a weight [N, K], a bias [N] and a residual [..., N], all bf16 or all fp16; y has their type.
    act: "none", "silu", "relu", "gelu" or "gelu_tanh".  With an activation, where a gradient is wanted, the pre-activation is kept in fp16 beside x and w, and
    the gradient dz that it leads to is rounded to the rows' type as an operand of the products that give dx and dw (the bias gradient adds it unrounded).
    Rows at any pitch and alignment are taken; fp32 rows belong to ops.linear."""
    return _ext.linear_act(x, w, b, res, act)


def _norm_arg(who, n):
    """None -> (absent, None, None); a weight, or a (weight, bias) pair whose members may be None -> (present, weight, bias)"""
    if n is None:
        return False, None, None
    if not isinstance(n, (tuple, list)):
        return True, n, None
    if len(n) != 2:
        raise _lib.CdaeError(f"residual_norm: {who} is None, a weight or a (weight, bias) pair")
    return True, n[0], n[1]


def residual_norm(x, f=None, *, gate=None, alpha=1.0, post=None, pre=None, scale=None, shift=None, kind="layer", eps=1e-5):
    """The norms before and after a block, its gate and the residual scale in one pass; returns (r, u):

        r = x + alpha * gate o post(f)            u = pre(r) o (1 + scale) + shift

    x, f: rows [..., C] of one type (bf16, fp16 or fp32), C <= 8192.  f None: r is x itself (the first norm of a network).  pre None: u is None (the
    last block).  post and pre: None (no norm), a weight [C], or a pair (weight, bias) of which either may be None; both are layer norms or, with
    kind="rms", rms norms.  gate, scale, shift: None, one vector [C] for all rows, or one for each sample [B, C], where B is x.shape[0] (rows [M, C]:
    any B that divides M, a sample's rows following each other).  gate, scale and shift are in the rows' type or all in fp32, and so are the weights."""
    return _ext.residual_norm(x, f, gate, scale, shift, *_norm_arg("post", post), *_norm_arg("pre", pre), alpha, kind, eps)


def grad_norm(grads, scale=1.0):
    """|scale| * sqrt(sum of all squares) over a list of gradients (any sizes, bf16 / fp16 / fp32 mixed) as a fp32 scalar on their device.  Squares
    and sums are fp64, in a fixed order: the result is finite wherever it fits fp32, and the same in every run."""
    return _ext.grad_norm(grads, scale)


def grad_factor(grads, max_norm, scale=1.0):
    """fp32 [2] on the device: the norm, and the factor scale * min(1, max_norm / (norm + 1e-6)) that clips by it (FusedAdamWEMA.step reads it there)."""
    return _ext.grad_factor(grads, max_norm, scale)


def clip_grad_norm_(grads, max_norm, scale=1.0, out=None, error_if_nonfinite=False):
    """out_i = g_i * scale * min(1, max_norm / (norm + 1e-6)) with norm = grad_norm(grads, scale), which is returned (fp32 scalar on the device).

    grads: the gradients themselves ([p.grad for p in model.parameters() if p.grad is not None]), any sizes and strides, bf16 / fp16 / fp32 mixed.
    scale: what the gradients have to be multiplied by first (1 / loss scale, 1 / ranks of a sum).  out: None (in place), or tensors of the same shapes
    and any of the types, e.g. fp32 master gradients; outputs may not share memory with each other or with another gradient.  A norm that is not finite
    leaves zeros or NaN: error_if_nonfinite=True raises instead, before anything is written, at the cost of waiting for the device
    (and so not inside a captured graph)."""
    return _ext.clip_grad_norm_(grads, max_norm, scale, out, error_if_nonfinite)
