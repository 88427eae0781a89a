"""What the entry points of group norm, linear layers and distillation have to refuse in the tensor layer, without a GPU."""
import ctypes as C

import pytest
import torch

from test_rowops_refusals import FAKE, bad, gn, lin, refused

BIG = 2 ** 32 + 5                                        # whose low 32 bits are a small positive number


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_sizes_that_do_not_fit_a_descriptor():
    """Descriptors hold 32-bit sizes: a larger one must not be cut down to its low half (which a kernel would then take for
    the size of a small, successful call)."""
    from cvae_gan_amd import ops
    f32, i32, need = torch.float32, torch.int32, "32 bits"
    x, w, y = meta(BIG, 1), meta(8, 1), meta(BIG, 8)
    bad(lambda: ops.linear_act_fwd(x, w, y), need)
    bad(lambda: ops.linear_act_bwd(y, x, w, dw=meta(8, 1)), need)
    bad(lambda: ops.linear_act_workspace(x, w, backward=True), need)
    bad(lambda: ops.linear_act_fwd(meta(65537, 65537, 8), meta(8, 8), meta(65537, 65537, 8)), need)      # a product of sizes
    bad(lambda: ops.linear_act_fwd(meta(2, BIG), meta(8, BIG), meta(2, 8)), need)
    bad(lambda: ops.linear_act_fwd(meta(2, 8), meta(BIG, 8), meta(2, BIG)), need)
    one = meta(8, dtype=f32)
    for shape in ((BIG, 8), (1, BIG, 8), (3, 65537, 65537, 8), (1, BIG * 8)):
        x = meta(*shape)
        v, st = meta(shape[-1], dtype=f32), meta(2, shape[0], 1, dtype=f32)
        bad(lambda: ops.gn_act_fwd(x, None, x, 1, None, v, v), need)
        bad(lambda: ops.gn_act_bwd(x, x, None, meta(*shape), None, 1, st, v, v, v, v), need)
        bad(lambda: ops.gn_act_workspace(x, 1), need)
    x = meta(2, 16, 8)
    bad(lambda: ops.gn_act_fwd(x, None, x, 2 ** 32 + 2, meta(2, 2, 2, dtype=f32), one, one), need)
    bad(lambda: ops.gn_act_fwd(x, None, x, -2, None, one, one), need)
    bad(lambda: ops.gn_act_fwd(x, None, x, 2.5, None, one, one), "groups")
    for rows, v, top in (((BIG,), 4, 2), ((65537, 65537), 4, 2), ((2,), BIG, 2), ((2,), 4, BIG)):
        bad(lambda: ops.distill_topk(meta(*rows, v), meta(*rows, top, dtype=f32), meta(*rows, top, dtype=i32), meta(1, dtype=f32),
                                     meta(*rows, dtype=f32)), need)


@pytest.mark.parametrize("n", [2 ** 31 - 1, 2 ** 31])
def test_the_largest_size(n):
    from cvae_gan_amd import ops
    if n < 2 ** 31:
        assert ops._sizes(0, n) == (0, n)
    else:
        bad(lambda: ops._sizes(n), "32 bits")


@pytest.mark.parametrize("T", [1.1e20, 1e30, 1e38, 3e38])
def test_distillation_temperatures_beyond_its_exponents(T):
    """e^(d / T) is taken with log2(e) / T in two f32 parts, which have to be normal numbers.  The low one was 1e-30 where nothing
    was left for it, more than the high one from T = 1.4e30 on (a logit at f32's lowest value at T = 1e38: 0 in the place of 0.03)."""
    from cvae_gan_amd._lib import lib, DistillDesc
    d = DistillDesc()
    d.dtype, d.R, d.V, d.top, d.temperature, d.grad_scale = 0, 4, 100, 5, T, 1.0
    assert "temperature" in refused(lib.cvg_distill_topk, C.byref(d), FAKE, FAKE, FAKE, None, FAKE, FAKE, FAKE, None)


def test_workspaces_of_the_more_exact_weight_gradient():
    """dw in f32 behind an activation needs more than dw in bf16; what Python allocates serves every activation and type."""
    from cvae_gan_amd import ops
    from cvae_gan_amd._lib import lib
    M, N, K = 512, 256, 128
    need = {(act, dt): lib.cvg_linear_act_workspace(C.byref(lin(M=M, N=N, K=K, act=act, dw_dtype=dt)), 1) for act in (0, 2) for dt in (0, 1)}
    assert need[2, 0] > need[2, 1] == need[0, 0] == need[0, 1]
    d = C.byref(lin(M=M, N=N, K=K, act=2, dw_dtype=0))
    P = [FAKE + (i << 24) for i in range(8)]
    assert "workspace" in refused(lib.cvg_linear_act_bwd, d, *P[:7], P[7], need[2, 1], None)
    x, w = torch.zeros(M, K, dtype=torch.bfloat16), torch.zeros(N, K, dtype=torch.bfloat16)
    assert ops.linear_act_workspace(x, w, backward=True).numel() == need[2, 0]


def test_small_outputs_over_other_tensors():
    """Parameter gradients, statistics, losses: an output that is an input, or another output, is written while workgroups still
    read the other.  (One sample of 2^20 pixels, so that group norm takes its two kernels.)"""
    from cvae_gan_amd._lib import lib, DistillDesc
    P = [FAKE + (i << 24) for i in range(12)]
    d, size = C.byref(gn(B=1, HW=1 << 20)), 1 << 40
    fwd = dict(x=P[0], res=P[1], y=P[2], stats=P[3], gamma=P[4], beta=P[5])
    for out, other in (("stats", "gamma"), ("stats", "beta"), ("y", "gamma"), ("y", "beta"), ("stats", "x"), ("stats", "y"), ("stats", "res")):
        assert "another tensor" in refused(lib.cvg_gn_act_fwd, d, *{**fwd, out: fwd[other]}.values(), P[9], size, None), (out, other)
    bwd = dict(dy=P[0], x=P[1], res=P[2], dx=P[3], dres=P[4], stats=P[5], gamma=P[6], beta=P[7], dgamma=P[8], dbeta=P[9])
    for out, others in (("dgamma", set(bwd) - {"dgamma"}), ("dbeta", set(bwd) - {"dbeta"}), ("dx", ("stats", "gamma", "beta")),
                        ("dres", ("stats", "gamma", "beta"))):
        for other in others:
            assert "another tensor" in refused(lib.cvg_gn_act_bwd, d, *{**bwd, out: bwd[other]}.values(), P[10], size, None), (out, other)
    d = C.byref(lin(M=64))
    fwd = dict(x=P[0], w=P[1], bias=P[2], res=P[3], y=P[4], pre=P[5])
    for out in ("y", "pre"):
        assert "another tensor" in refused(lib.cvg_linear_act_fwd, d, *{**fwd, out: fwd["bias"]}.values(), P[9], size, None), out
    bwd = dict(dy=P[0], x=P[1], w=P[2], pre=P[3], dx=P[4], dw=P[5], dbias=P[6])
    for out, other in (("dx", "dw"), ("dw", "dbias"), ("dbias", "dx"), ("dbias", "pre"), ("dbias", "x")):
        assert "another tensor" in refused(lib.cvg_linear_act_bwd, d, *{**bwd, out: bwd[other]}.values(), P[9], size, None), (out, other)
    dd = DistillDesc()
    dd.dtype, dd.R, dd.V, dd.top, dd.temperature = 1, 4, 100, 5, 1.0
    call = dict(logits=P[0], top_val=P[1], top_idx=P[2], row_weight=P[3], loss=P[4], row_loss=P[5], dlogits=P[6])
    for out, others in (("loss", set(call) - {"loss"}), ("row_loss", set(call) - {"row_loss"}), ("dlogits", ("top_val", "top_idx", "row_weight"))):
        for other in others:
            assert "another tensor" in refused(lib.cvg_distill_topk, C.byref(dd), *{**call, out: call[other]}.values(), None), (out, other)


def test_torch_operators_keep_to_their_schemas():
    """torch.ops.cvaegan.* declare their inputs as read only: what ops.py does in place they refuse.  (Called behind the
    dispatcher, which has no CPU kernel; everything else about the call is right, so that the next refusal is the device's.)"""
    from cvae_gan_amd import ops, torch_ops as t
    x, y, z, one, st = torch.zeros(2, 3, 8), torch.zeros(2, 3, 8), torch.zeros(2, 3, 8), torch.ones(8), torch.zeros(2, 2, 1)

    def gn_fwd(y, res=None):
        t._gn_act_fwd(x, res, y, 1, st, one, one, 1e-5, ops.ACT_SILU, None)
    bad(lambda: gn_fwd(y), "device tensors")
    bad(lambda: gn_fwd(x), "y is an input")
    bad(lambda: gn_fwd(y, res=y), "y is an input")

    def gn_bwd(dx, dres):
        t._gn_act_bwd(y, x, z, dx, dres, 1, st, one, one, one.clone(), one.clone(), ops.ACT_SILU, None)
    bad(lambda: gn_bwd(x.clone(), None), "device tensors")
    bad(lambda: gn_bwd(y, None), "dx is an input")
    bad(lambda: gn_bwd(x.clone(), y), "dres is an input")
    w = torch.zeros(8, 8)
    bad(lambda: t._linear_act_fwd(x, w, y, None, z, None, ops.ACT_NONE, None), "device tensors")
    bad(lambda: t._linear_act_fwd(x, w, z, None, z, None, ops.ACT_NONE, None), "y is an input")
    lg, tv, ti = torch.zeros(4, 50), torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int32)

    def distill(dl):
        t._distill_topk(lg, tv, ti, torch.zeros(()), torch.zeros(4), dl, None, 1.0, 1.0)
    bad(lambda: distill(torch.zeros(4, 50)), "device tensors")
    bad(lambda: distill(lg), "dlogits is an input")
