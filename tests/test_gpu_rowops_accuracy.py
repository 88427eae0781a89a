"""Accuracy of the row operators in the 2-norm, where element-wise bounds that grow with the length of a sum see little."""
import math

import pytest
import torch

from test_gpu_rowops import BF, F32, act64, ops, rnd  # noqa: F401

pytestmark = pytest.mark.gpu


def off(got, ref):
    return float((got.double() - ref).norm() / ref.norm())


# M, N, K: small tiles, tiles of 128 and 256, rows of no whole 16 bytes, one row, split and whole ranges of rows
@pytest.mark.parametrize("size", [(1, 8, 8), (16, 40, 72), (777, 303, 115), (2048, 264, 520), (2048, 1032, 1032), (4096, 2048, 64),
                                  (2056, 4104, 4104)], ids=lambda c: "x".join(map(str, c)))
def test_f32_weight_gradient_behind_an_activation(ops, size):  # noqa: F811
    """bf16 data, dw in f32: 2e-5 of its norm.  dz in two bf16 parts is off by at most 2^-16 of itself, 2^-16 / sqrt(3) = 8.8e-6
    in the mean square; its own f32 arithmetic by 16 u = 1e-6; sums of M <= 4096 products, 16 at a time, by u sqrt(M / 16) = 1e-6.
    (Rounded to bf16 once it is off by 1.7e-3.)"""
    M, N, K = size
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    x, w = rnd(g, M, K, dtype=BF), rnd(g, N, K, dtype=BF, scale=1 / math.sqrt(K))
    dy = rnd(g, M, N, dtype=BF, scale=0.1)
    for act, pre_dtype in (("gelu", F32), ("silu", BF), ("lrelu", F32)):
        a = ops.ACTS[act]
        pre = rnd(g, M, N, dtype=pre_dtype)
        gd = dy.double() * act64(pre.double(), act)[1]
        ref = gd.t() @ x.double()
        runs = []
        for with_dx in (True, False):
            dx = torch.full_like(x, float("nan")) if with_dx else None
            dw, db = torch.full((N, K), float("nan"), device="cuda"), torch.full((N,), float("nan"), device="cuda")
            ws = ops.linear_act_workspace(x, w, backward=True)
            ops.linear_act_bwd(dy, x, w, pre=pre, dx=dx, dw=dw, dbias=db, act=a, ws=ws)
            assert off(dw, ref) < 2e-5, (act, off(dw, ref))
            # (a sum of M terms of both signs; 2-norms: u sqrt(M) and 16 u of the terms' norm)
            assert float((db.double() - gd.sum(0)).norm()) < 2e-6 * float(gd.norm()) * math.sqrt(M)
            runs.append(dw)
            if with_dx and x.numel() > 1000:              # (enough elements for a mean square)
                # once rounded operand, once rounded result: 2^-8 / sqrt(3) = 2.26e-3 each at the worst
                assert off(dx, gd @ w.double()) < math.sqrt(2) * 2.0 ** -8 / math.sqrt(3) + 1e-5
        assert torch.equal(*runs)


def test_f32_weight_gradient_of_infinite_gradients(ops):  # noqa: F811
    """An infinite or undefined element of dy makes its own row of dw infinite or undefined, and no other."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = rnd(g, 40, 24, dtype=BF).abs() + 1
    w, pre, dy = rnd(g, 16, 24, dtype=BF), rnd(g, 40, 16).abs(), rnd(g, 40, 16, dtype=BF)
    dy[3, 5], dy[7, 9] = float("inf"), float("nan")
    dw = torch.empty(16, 24, device="cuda")
    ops.linear_act_bwd(dy, x, w, pre=pre, dw=dw, act=ops.ACT_LRELU)
    rest = [i for i in range(16) if i not in (5, 9)]
    assert bool((dw[5] == float("inf")).all()) and bool(torch.isnan(dw[9]).all()) and bool(torch.isfinite(dw[rest]).all())


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_f32_sums_of_bf16_data(ops, act):  # noqa: F811
    """Parameter gradients are f32 sums of unrounded terms.  Their activations' derivatives come from v_exp_f32 and v_rcp_f32 as
    they are: off by some 4 u (1 + |v|) each, against terms of about half of |dy|, 2e-6 of the terms' norm at |v| <= 3; the
    sums' own roundings and those of xhat add less."""
    from test_gpu_rowops import gn_ref
    g = torch.Generator(device="cuda").manual_seed(3)
    for B, HW, C, G in ((64, 1024, 128, 32), (2, 16384, 64, 32)):
        x, dy, gamma, beta = rnd(g, B, HW, C, dtype=BF, scale=1.5, mean=0.3), rnd(g, B, HW, C, dtype=BF), rnd(g, C, mean=1.0, scale=0.2), rnd(g, C, scale=0.2)
        ref = gn_ref(x, None, gamma, beta, G, 1e-5, act, dy)
        y, dx, stats, dg, db = torch.empty_like(x), torch.empty_like(x), torch.empty(2, B, G, device="cuda"), torch.empty_like(gamma), torch.empty_like(gamma)
        ops.gn_act_fwd(x, None, y, G, stats, gamma, beta, act=ops.ACTS[act])
        ops.gn_act_bwd(dy, x, None, dx, None, G, stats, gamma, beta, dg, db, act=ops.ACTS[act])
        assert off(dg, ref["dgamma"]) < 5e-6 and off(db, ref["dbeta"]) < 5e-6
    M, N, K = 4096, 512, 64
    x, w, dy, pre = rnd(g, M, K, dtype=BF), rnd(g, N, K, dtype=BF), rnd(g, M, N, dtype=BF), rnd(g, M, N)
    db = torch.empty(N, device="cuda")
    ops.linear_act_bwd(dy, x, w, pre=pre, dbias=db, act=ops.ACTS[act])
    ref = (dy.double() * act64(pre.double(), act)[1]).sum(0)
    assert off(db, ref) < 5e-6
