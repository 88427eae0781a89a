"""What the group-norm, linear and distillation entry points refuse, without a GPU: every call here must fail in
validation, before anything is launched (pointers are made-up aligned addresses that are never read)."""
import ctypes as C

import pytest
import torch

FAKE = 1 << 20


def refused(fn, *args):
    from cvae_gan_amd import _lib
    rc = fn(*args)
    assert rc != 0
    return _lib.lib.cvg_last_error().decode()


def gn(**kw):
    from cvae_gan_amd._lib import GnDesc
    d = GnDesc()
    base = dict(dtype=1, B=2, HW=16, C=64, G=8, act=2, eps=1e-5)
    base.update(kw)
    for k, v in base.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw, needle", [
    (dict(dtype=2), "dtype"), (dict(C=12, G=4), "multiple of 8"), (dict(G=7), "divide"), (dict(HW=0), "HW"), (dict(B=-1), "B -1"),
    (dict(act=4), "activation"), (dict(act=-1), "activation"), (dict(C=8192, G=1), "too wide"), (dict(C=8 * 1027, G=8), "too wide"),
    (dict(x_ld=56), "pitch"), (dict(y_ld=68), "pitch"), (dict(dres_ld=-64), "pitch"), (dict(eps=-1.0), "eps"),
    (dict(B=1 << 20, HW=1 << 12), "pixel rows"), (dict(G=0), "G 0"),
])
def test_group_norm_descriptors(kw, needle):
    from cvae_gan_amd._lib import lib
    d = C.byref(gn(**kw))
    assert needle in refused(lib.cvg_gn_act_fwd, d, FAKE, None, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 30, None)
    assert needle in refused(lib.cvg_gn_act_bwd, d, FAKE, FAKE, None, FAKE, None, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 30, None)
    assert lib.cvg_gn_act_workspace(d, 1) == 0


def test_group_norm_pointers_and_workspaces():
    from cvae_gan_amd._lib import lib
    d = C.byref(gn(HW=1 << 20))
    fwd, bwd = lib.cvg_gn_act_fwd, lib.cvg_gn_act_bwd
    assert "null" in refused(fwd, d, None, None, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 40, None)
    assert "null" in refused(fwd, d, FAKE, None, FAKE, FAKE, None, FAKE, FAKE, 1 << 40, None)
    assert "16-byte" in refused(fwd, d, FAKE + 2, None, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 40, None)
    assert "16-byte" in refused(fwd, d, FAKE, FAKE + 8, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 40, None)
    assert lib.cvg_gn_act_workspace(d, 0) > 0
    assert "workspace" in refused(fwd, d, FAKE, None, FAKE, FAKE, FAKE, FAKE, FAKE, lib.cvg_gn_act_workspace(d, 0) - 1, None)
    assert "workspace" in refused(fwd, d, FAKE, None, FAKE, FAKE, FAKE, FAKE, None, 1 << 40, None)
    assert "null" in refused(bwd, d, FAKE, FAKE, None, FAKE, None, None, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 40, None)
    assert "null" in refused(bwd, d, FAKE, FAKE, None, FAKE, None, FAKE, FAKE, FAKE, None, FAKE, FAKE, 1 << 40, None)
    assert "workspace" in refused(bwd, d, FAKE, FAKE, None, FAKE, None, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 16, None)


def lin(**kw):
    from cvae_gan_amd._lib import LinearDesc
    d = LinearDesc()
    base = dict(dtype=1, M=4, N=32, K=16, act=2, dw_dtype=0)
    base.update(kw)
    for k, v in base.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw, needle", [
    (dict(dtype=3), "dtype"), (dict(dtype=0, dw_dtype=1), "dw_dtype"), (dict(M=-1), "M -1"), (dict(N=0), "N 0"), (dict(K=0), "K 0"),
    (dict(act=9), "activation"), (dict(x_ld=15), "pitch"), (dict(w_ld=8), "pitch"), (dict(y_ld=31), "pitch"), (dict(dy_ld=-1), "pitch"),
])
def test_linear_descriptors(kw, needle):
    from cvae_gan_amd._lib import lib
    d = C.byref(lin(**kw))
    assert needle in refused(lib.cvg_linear_act_fwd, d, FAKE, FAKE, None, None, FAKE, None, FAKE, 1 << 40, None)
    assert needle in refused(lib.cvg_linear_act_bwd, d, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 40, None)


def test_linear_workspace_sizes():
    """Plans over ordinary and degenerate sizes: no division by an empty range, sizes bounded by the operands'."""
    from cvae_gan_amd._lib import lib
    for dtype in (0, 1):
        for M in (0, 1, 7, 64, 1000, 100000):
            for N in (1, 64, 1003, 2000000):
                for K in (1, 8, 515, 8192):
                    d = C.byref(lin(dtype=dtype, M=M, N=N, K=K))
                    f, b = lib.cvg_linear_act_workspace(d, 0), lib.cvg_linear_act_workspace(d, 1)
                    if lib.cvg_linear_act_fwd(d, None, None, None, None, None, None, None, 0, None) != 0 and b"too many" in lib.cvg_last_error():
                        assert f == 0 and b == 0
                        continue
                    assert 0 <= f <= b < 1 << 50 and (f > 0 or M <= 16) and (b > 0) == (M > 0)


def test_linear_pointers_and_workspaces():
    from cvae_gan_amd._lib import lib
    d = C.byref(lin())
    fwd, bwd = lib.cvg_linear_act_fwd, lib.cvg_linear_act_bwd
    assert "null" in refused(fwd, d, FAKE, None, None, None, FAKE, None, FAKE, 1 << 40, None)
    assert "misaligned" in refused(fwd, d, FAKE + 1, FAKE, None, None, FAKE, None, FAKE, 1 << 40, None)
    assert "pre" in refused(bwd, d, FAKE, FAKE, FAKE, None, FAKE, None, None, FAKE, 1 << 40, None)
    assert "needs w" in refused(bwd, d, FAKE, FAKE, None, FAKE, FAKE, None, None, FAKE, 1 << 40, None)
    assert "needs x" in refused(bwd, d, FAKE, None, FAKE, FAKE, None, FAKE, None, FAKE, 1 << 40, None)
    assert "misaligned dw" in refused(bwd, d, FAKE, FAKE, FAKE, FAKE, None, FAKE + 2, None, FAKE, 1 << 40, None)
    assert "workspace" in refused(bwd, d, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, lib.cvg_linear_act_workspace(d, 1) - 1, None)
    assert "workspace" in refused(bwd, d, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE + 4, 1 << 40, None)


@pytest.mark.parametrize("kw, needle", [
    (dict(dtype=5), "dtype"), (dict(V=0), "V 0"), (dict(R=-2), "R -2"), (dict(top=0), "teacher entries"), (dict(top=1025), "teacher entries"),
    (dict(temperature=0.0), "temperature"), (dict(temperature=-1.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
    (dict(temperature=float("inf")), "temperature"), (dict(temperature=1e-39), "temperature"), (dict(logits_ld=99), "pitches"), (dict(dlogits_ld=1), "pitches"),
    (dict(top_ld=3), "pitches"),
])
def test_distill_descriptors(kw, needle):
    from cvae_gan_amd._lib import lib, DistillDesc
    d = DistillDesc()
    base = dict(dtype=1, R=4, V=100, top=5, temperature=1.0, grad_scale=1.0)
    base.update(kw)
    for k, v in base.items():
        setattr(d, k, v)
    assert needle in refused(lib.cvg_distill_topk, C.byref(d), FAKE, FAKE, FAKE, None, FAKE, FAKE, FAKE, None)


def test_distill_pointers():
    from cvae_gan_amd._lib import lib, DistillDesc
    d = DistillDesc()
    d.dtype, d.R, d.V, d.top, d.temperature = 1, 4, 100, 5, 1.0
    f = lib.cvg_distill_topk
    assert "null loss" in refused(f, C.byref(d), FAKE, FAKE, FAKE, None, None, FAKE, FAKE, None)
    assert "null tensor" in refused(f, C.byref(d), FAKE, None, FAKE, None, FAKE, FAKE, FAKE, None)
    assert "misaligned" in refused(f, C.byref(d), FAKE + 1, FAKE, FAKE, None, FAKE, FAKE, None, None)
    d.logits_ld = 128
    assert "in place" in refused(f, C.byref(d), FAKE, FAKE, FAKE, None, FAKE, FAKE, FAKE, None)


def test_sizes_beyond_a_launch():
    """Row counters step past the end of the rows and a launch holds fewer than 2^32 threads: what would not fit is refused."""
    from cvae_gan_amd._lib import lib, DistillDesc
    d = C.byref(gn(B=1, HW=0x7fffffff))
    assert "pixel rows" in refused(lib.cvg_gn_act_fwd, d, FAKE, None, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 62, None)
    d = C.byref(gn(B=1, HW=1, C=1 << 30, G=1 << 27))
    assert "C 1073741824" in refused(lib.cvg_gn_act_fwd, d, FAKE, None, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 62, None)
    d = C.byref(gn(B=0x7fff0000, HW=1))
    assert "too many" in refused(lib.cvg_gn_act_fwd, d, FAKE, None, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 62, None)
    assert "too many" in refused(lib.cvg_gn_act_bwd, d, FAKE, FAKE, None, FAKE, None, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 62, None)
    for kw in (dict(M=64 << 12, N=64 << 10), dict(M=64 << 12, K=64 << 10, N=8), dict(M=1, N=64 << 11, K=64 << 11)):
        d = C.byref(lin(**kw))
        assert "too many" in refused(lib.cvg_linear_act_fwd, d, FAKE, FAKE, None, None, FAKE, None, FAKE, 1 << 62, None)
        assert "too many" in refused(lib.cvg_linear_act_bwd, d, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 62, None)
    dd = DistillDesc()
    dd.dtype, dd.R, dd.V, dd.top, dd.temperature = 1, 0x7fffffff, 1, 1, 1.0
    assert "R 2147483647" in refused(lib.cvg_distill_topk, C.byref(dd), FAKE, FAKE, FAKE, None, FAKE, FAKE, FAKE, None)


def test_outputs_over_inputs():
    """An output may be the tensor the declaration names, at its pitch, and no other."""
    from cvae_gan_amd._lib import lib
    A, B_, D_, E = (FAKE + (i << 24) for i in range(4))
    d = C.byref(gn(y_ld=128))
    assert "in place" in refused(lib.cvg_gn_act_fwd, d, A, None, A, B_, B_, B_, E, 1 << 40, None)
    assert "in place" in refused(lib.cvg_gn_act_fwd, d, A, D_, D_, B_, B_, B_, E, 1 << 40, None)
    assert "in place" in refused(lib.cvg_gn_act_bwd, d, A, B_, None, A, None, E, E, E, E, E, E, 1 << 40, None)
    assert "in place" in refused(lib.cvg_gn_act_bwd, d, A, B_, None, D_, A, E, E, E, E, E, E, 1 << 40, None)
    for dx, dres in ((B_, None), (D_, None), (A, A), (A, B_), (A, D_)):
        assert "another tensor" in refused(lib.cvg_gn_act_bwd, C.byref(gn()), A, B_, D_, dx, dres, E, E, E, E, E, E, 1 << 40, None)
    d = C.byref(lin(M=64, y_ld=64))
    fwd, bwd, F = lib.cvg_linear_act_fwd, lib.cvg_linear_act_bwd, FAKE + (9 << 24)
    assert "in place" in refused(fwd, d, A, B_, None, D_, D_, None, E, 1 << 40, None)
    for y, pre in ((A, None), (B_, None), (F, F), (F, A), (F, B_), (F, D_)):
        assert "another tensor" in refused(fwd, d, A, B_, None, D_, y, pre, E, 1 << 40, None)
    for dx, dw in ((A, None), (B_, None), (None, D_), (None, F)):
        assert "another tensor" in refused(bwd, d, A, B_, D_, F, dx, dw, None, E, 1 << 40, None)


def bad(call, needle):
    from cvae_gan_amd.ops import CvgError
    with pytest.raises(CvgError, match=needle):
        call()


def test_tensor_checks():
    """Shapes, types and strides are refused by the tensor layer; a CPU tensor is refused last."""
    from cvae_gan_amd import ops
    x, one = torch.zeros(2, 4, 4, 16), torch.ones(16)
    st = torch.zeros(2, 2, 4)
    y = torch.zeros_like(x)
    bad(lambda: ops.gn_act_fwd(x, None, y, 4, st, one, one), "device tensors")
    bad(lambda: ops.gn_act_fwd(x, None, y[:1], 4, st, one, one), "y has shape")
    bad(lambda: ops.gn_act_fwd(x, None, y.bfloat16(), 4, st, one, one), "y is torch.bfloat16")
    bad(lambda: ops.gn_act_fwd(x, None, y, 4, st, one[:8], one), "gamma has shape")
    bad(lambda: ops.gn_act_fwd(x, None, y, 4, st.double(), one, one), "stats is")
    bad(lambda: ops.gn_act_fwd(x, None, y, 2, st, one, one), "stats has shape")
    bad(lambda: ops.gn_act_fwd(x.half(), None, y, 4, st, one, one), "bfloat16")
    bad(lambda: ops.gn_act_fwd(x, None, y, 4, st, one, one, act=7), "activation")
    bad(lambda: ops.gn_act_fwd(x.permute(0, 3, 1, 2), None, y.permute(0, 3, 1, 2), 4, st, torch.ones(4), torch.ones(4)), "consecutive")
    bad(lambda: ops.gn_act_fwd(torch.zeros(2, 8, 4, 16)[:, ::2], None, y, 4, st, one, one), "one pitch")
    bad(lambda: ops.gn_act_fwd(torch.zeros(1, 1, 1, 16).expand(2, 4, 4, 16), None, y, 4, st, one, one), "overlap")
    bad(lambda: ops.gn_act_bwd(y, x, None, y, None, 4, st, one, one, one, one[:3]), "dbeta has shape")
    xl, w, yl = torch.zeros(3, 5, 16), torch.zeros(8, 16), torch.zeros(3, 5, 8)
    bad(lambda: ops.linear_act_fwd(xl, w, yl), "device tensors")
    bad(lambda: ops.linear_act_fwd(xl, w[:, :8], yl), "w has shape")
    bad(lambda: ops.linear_act_fwd(xl, w.bfloat16(), yl), "w is")
    bad(lambda: ops.linear_act_fwd(xl, w, yl[..., :4]), "y has shape")
    bad(lambda: ops.linear_act_fwd(xl, w.t().contiguous().t(), yl), "consecutive")
    bad(lambda: ops.linear_act_fwd(xl, w, yl, bias=torch.zeros(8, dtype=torch.bfloat16)), "bias is")
    bad(lambda: ops.linear_act_fwd(xl, w, yl, res=torch.zeros(3, 5, 1).expand(3, 5, 8)), "consecutive")
    bad(lambda: ops.linear_act_bwd(yl, xl, w, dw=w.bfloat16()), "dw is")
    bad(lambda: ops.linear_act_bwd(yl, xl, w, dx=xl[:2]), "dx has shape")
    lg, tv, ti = torch.zeros(4, 50), torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int32)
    loss, rl = torch.zeros(()), torch.zeros(4)
    bad(lambda: ops.distill_topk(lg, tv, ti, loss, rl), "device tensors")
    bad(lambda: ops.distill_topk(lg, tv, ti.long(), loss, rl), "top_idx is")
    bad(lambda: ops.distill_topk(lg, tv, ti[:, :2], loss, rl), "top_idx has shape")
    bad(lambda: ops.distill_topk(lg, tv, ti, torch.zeros(2), rl), "loss has to be")
    bad(lambda: ops.distill_topk(lg, tv, ti, loss, rl[:3]), "row_loss has shape")
    bad(lambda: ops.distill_topk(lg, tv.bfloat16(), ti, loss, rl), "top_val is")
    bad(lambda: ops.distill_topk(lg, tv, torch.zeros(4, 5, dtype=torch.int32)[:, :3], loss, rl), "share their strides")
    bad(lambda: ops.distill_topk(lg, tv, ti, loss, rl, dlogits=lg[:, :49]), "dlogits has shape")
