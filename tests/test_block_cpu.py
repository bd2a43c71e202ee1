"""Refusals and sizes of the feed-forward block's entry points that are decided on the host, before any launch (no GPU)."""
import array
import ctypes
import os
import subprocess
import sys

import pytest
import torch

from causaldiffae_amd import CdaeError, ops_block
from causaldiffae_amd._lib import ResNorm, lib

PTR = 0x10000          # never followed: every call below is refused first


def refused(rc, word):
    assert rc == -1 and word in lib.cdae_last_error().decode(), (rc, lib.cdae_last_error())


def test_workspace_sizes():
    assert lib.cdae_lin16_workspace_bytes(0, 0, 8, 8) == 0 and lib.cdae_lin16_workspace_bytes(7, 8, 8, 8) == 0
    for op in (0, 1):
        assert lib.cdae_lin16_workspace_bytes(op, 1, 1, 1) > 0
        assert lib.cdae_lin16_workspace_bytes(op, 1 << 20, 4096, 4096) >= (1 << 20) * 4096 * 2         # (sizes beyond 32 bits)
        copies = ((1 << 20) + 4096) * 4096 * 2                                                         # (of operands that the kernel cannot read as they lie)
        spared = lib.cdae_lin16_workspace_bytes(op, 1 << 20, 4096, 4096) - lib.cdae_lin16_workspace_bytes(op | 8, 1 << 20, 4096, 4096)
        assert copies - (1 << 24) <= spared <= copies                                                  # (the backward's partial sums share their place)
    assert lib.cdae_resnorm_workspace_bytes(1, 1, 8193) == 0 and lib.cdae_resnorm_workspace_bytes(0, 1, 8) == 0
    assert lib.cdae_resnorm_workspace_bytes(1, 1, 8192) >= 4 * 4 * 8192
    assert lib.cdae_grad_workspace_bytes() >= 8 * 1024


def test_linear_refusals():
    def fwd(M=4, N=8, K=8, act=0, dt=0, ldx=8, ldw=8, ldy=8, x=PTR, y=PTR, ws=PTR, ws_bytes=1 << 30):
        return lib.cdae_lin16_fwd(x, ldx, PTR, ldw, None, None, 0, y, ldy, None, 0, M, N, K, act, dt, ws, ws_bytes, None)

    def bwd(M=4, N=8, K=8, act=0, dt=0, dy=PTR, x=PTR, w=PTR, z=None, dx=PTR, dw=PTR, ws_bytes=1 << 30):
        return lib.cdae_lin16_bwd(dy, 8, x, 8, w, 8, z, 8, dx, 8, dw, 8, None, M, N, K, act, dt, PTR, ws_bytes, None)

    for kw in (dict(M=-1), dict(N=0), dict(K=0)):
        refused(fwd(**kw), "required")
        refused(bwd(**kw), "required")
    for kw in (dict(M=(1 << 30) + 1), dict(N=(1 << 22) + 1), dict(K=(1 << 22) + 1)):
        refused(fwd(**kw), "at most")
        refused(bwd(**kw), "at most")
    refused(fwd(dt=2), "type")
    refused(bwd(dt=3), "type")
    for a in (2, 4, 7, -1):
        refused(fwd(act=a), "activation")
        refused(bwd(act=a), "activation")
    for kw in (dict(ldx=7), dict(ldw=7), dict(ldy=7), dict(x=None), dict(y=None)):
        refused(fwd(**kw), "pitches")
    refused(fwd(ws_bytes=16), "workspace")
    refused(fwd(ws=None), "workspace")
    refused(fwd(ws=PTR + 8), "workspace")
    refused(fwd(x=PTR + 2, ws_bytes=lib.cdae_lin16_workspace_bytes(8, 4, 8, 8)), "workspace")
    refused(bwd(ws_bytes=16), "workspace")
    refused(bwd(M=0), "no rows")
    refused(bwd(dy=None), "dy")
    refused(bwd(act=1), "z with an activation")
    refused(bwd(w=None), "w for dx")
    refused(bwd(x=None), "x for dw")
    assert fwd(M=0) == 0


def test_norm_refusals():
    def args(**kw):
        p = ResNorm()
        d = dict(B=2, T=3, C=8, dt=0, layer=1, pre=1, alpha=1.0, eps=1e-5, x=PTR, ld_x=8, u=PTR, du=PTR, ld_du=8, ws=PTR, ws_bytes=1 << 20)
        for k, v in {**d, **kw}.items():
            setattr(p, k, v)
        return ctypes.byref(p)

    both = (lib.cdae_resnorm_fwd, lib.cdae_resnorm_bwd)
    for f in both:
        for kw in (dict(B=0), dict(T=0), dict(C=0), dict(C=8193)):
            refused(f(args(**kw), None), "required")
        refused(f(args(B=1 << 20, T=1 << 20), None), "rows")
        refused(f(args(dt=3), None), "type")
        refused(f(args(x=None), None), "required")
        refused(f(args(gate=PTR), None), "block output")
        refused(f(args(pre=0, f=PTR, r=PTR, scale=PTR), None), "pre norm")
        refused(f(args(f=PTR, r=PTR, w1=PTR), None), "post norm")
        refused(f(args(eps=-1.0), None), "eps")
        refused(f(args(eps=float("nan")), None), "eps")
    refused(lib.cdae_resnorm_fwd(args(u=None), None), "u with a pre norm")
    refused(lib.cdae_resnorm_fwd(args(f=PTR), None), "r with a block output")
    refused(lib.cdae_resnorm_bwd(args(du=None), None), "gradient of r or of u")
    refused(lib.cdae_resnorm_bwd(args(df=PTR), None), "not there")
    refused(lib.cdae_resnorm_bwd(args(dscale=PTR), None), "not there")
    refused(lib.cdae_resnorm_bwd(args(ws_bytes=16), None), "workspace")
    refused(lib.cdae_resnorm_bwd(args(B=1 << 22, C=1, T=1), None), "samples")


def test_grad_refusals():
    def call(ptrs=(PTR,), sizes=(16,), types=(2,), outs=None, out_types=None, max_norm=1.0, norm=PTR, ws_bytes=1 << 20):
        keep = [array.array("Q", ptrs), array.array("q", sizes), array.array("i", types), array.array("Q", outs or ptrs), array.array("i", out_types or types)]
        p, n, t, o, ot = (k.buffer_info()[0] for k in keep)
        return (lib.cdae_grad_norm(p, n, t, len(ptrs), 1.0, max_norm, norm, PTR, ws_bytes, None),
                lib.cdae_grad_clip(p, n, t, o, ot, len(ptrs), 1.0, max_norm, norm, PTR, ws_bytes, None))

    for kw in (dict(sizes=(-1,)), dict(ptrs=(0,)), dict(types=(3,)), dict(types=(-1,)), dict(norm=None), dict(ws_bytes=8), dict(max_norm=-1.0), dict(max_norm=float("nan"))):
        assert call(**kw) == (-1, -1), kw

    def clip(**kw):
        keep = {k: array.array(c, kw[k]) for k, c in (("ptrs", "Q"), ("sizes", "q"), ("types", "i"), ("outs", "Q"), ("out_types", "i"))}
        a = {k: v.buffer_info()[0] for k, v in keep.items()}
        return lib.cdae_grad_clip(a["ptrs"], a["sizes"], a["types"], a["outs"], a["out_types"], len(kw["ptrs"]), 1.0, 1.0, PTR, PTR, 1 << 20, None)

    far = 0x900000
    # the same tensor twice, an overlapping pair, outputs that overlap, an output over another gradient, an output of another size over its own gradient
    for ptrs, sizes, types, outs, out_types in (
            ((PTR, PTR), (16, 16), (2, 2), (PTR, PTR), (2, 2)), ((PTR, PTR + 32), (16, 16), (2, 2), (PTR, PTR + 32), (2, 2)),
            ((PTR, far), (16, 16), (2, 2), (PTR, PTR + 60), (2, 2)), ((PTR, far), (16, 16), (2, 2), (far, PTR), (2, 2)), ((PTR,), (16,), (0,), (PTR,), (2,)),
            ((PTR,), (16,), (2,), (PTR + 4,), (2,))):
        refused(clip(ptrs=ptrs, sizes=sizes, types=types, outs=outs, out_types=out_types), "shares memory" if len(set(outs)) == len(outs) else "share memory")


def test_host_tensors_are_refused():
    x = torch.zeros(4, 8, dtype=torch.bfloat16)
    for call in (lambda: ops_block.linear_act(x, x), lambda: ops_block.residual_norm(x, x), lambda: ops_block.grad_norm([x]), lambda: ops_block.clip_grad_norm_([x], 1.0)):
        with pytest.raises(CdaeError):
            call()


@pytest.mark.parametrize("B,T,C", [(1 << 20, 1, 520), (65536, 1, 1024), (1 << 17, 1, 8192), (9000, 1, 1000), (600, 1, 8192), (1 << 21, 3, 64), (32, 256, 384), (8, 4096, 2048)])
def test_norm_scratch_stays_beside_the_rows(B, T, C):
    """with a vector for every row the column sums of all samples would be many times the rows: the backward keeps 64 MB, or less than one tensor of 16-bit rows"""
    assert 16 * C <= lib.cdae_resnorm_workspace_bytes(B, T, C) <= (64 << 20) + 2 * B * T * C


def test_training_without_clipping_needs_no_extension():
    """where the extension does not load, the trainer does, and only a bound on the gradients asks for it"""
    code = """
import sys
sys.modules["causaldiffae_amd._block_ext"] = None
from causaldiffae_amd import train_util
import improved_diffusion.train_util
kw = dict(model=None, diffusion=None, data=None, batch_size=1, microbatch=1, lr=0.0, ema_rate="0", log_interval=1, save_interval=1, resume_checkpoint="")
try:
    train_util.TrainLoop(**kw, grad_clip=1.0)
except ImportError as e:
    print("refused:", e)
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "refused: causaldiffae_amd/_block_ext.so does not load" in done.stdout, (done.stdout, done.stderr[-2000:])


def test_extension_is_built_for_this_torch():
    """the build records which torch the extension was compiled against, and builds it again for another"""
    with open(os.path.join(os.path.dirname(ops_block.__file__), "csrc", "build", ".ext")) as f:
        assert f.read().split()[:2] == ["torch", torch.__version__]
