"""The kernel forms that large calls take: the widest group norm, many tiles a sample, workgroups that walk over rows of
distillation, long sums.  Inputs put weight on single elements (last ones, first ones, ones at many places), so that an
element left out of a sum is an error of order one, and bounds count the additions that a form really chains."""
import math

import pytest
import torch

from test_gpu_rowops import BF, F32, HALF, U, distill_ref, gn_ref, lin_check, ops, rnd, within  # noqa: F401

pytestmark = pytest.mark.gpu


def off(got, ref):
    return float((got.double() - ref).norm() / ref.norm())


def signs(g, *shape):
    return torch.where(torch.rand(*shape, generator=g, device="cuda") < 0.5, -1.0, 1.0)


# ---- group norm ----------------------------------------------------------------------------------------------
def gn_inputs(g, B, HW, C, G, dtype, with_res, away_from_zero):
    if away_from_zero:
        # x = +-(0.5 .. 2.5), every value with its negative in the same group: mean 0, |xhat| >= 0.3, and with gamma >= 0.7,
        # |beta| + |res| < 0.08 no argument of the activation comes near zero
        half = 0.5 + 2 * torch.rand(B, HW // 2, C, generator=g, device="cuda")
        half *= signs(g, *half.shape)
        x = torch.cat([half, -half.flip(1)], 1)
        if HW % 2:
            sign = 1 - 2 * (torch.arange(C, device="cuda") % 2)
            x = torch.cat([x, sign.expand(B, 1, C).float()], 1)
        x = x.to(dtype)
        gamma = 0.7 + 0.6 * torch.rand(C, generator=g, device="cuda")
        beta = 0.1 * torch.rand(C, generator=g, device="cuda") - 0.05
        res = (0.05 * torch.rand(B, HW, C, generator=g, device="cuda") - 0.025).to(dtype) if with_res else None
    else:
        x = rnd(g, B, HW, C, dtype=dtype, scale=1.5, mean=0.5)
        for i, row in enumerate((0, HW - 1, HW - 2, HW // 2, 7 * HW // 8)):      # one heavy element per group and row
            x[:, row, (i % (C // G))::(C // G)] = 30.0 if i % 2 else -30.0
        gamma, beta = rnd(g, C, mean=1.0, scale=0.3), rnd(g, C, scale=0.3)
        res = rnd(g, B, HW, C, dtype=dtype) if with_res else None
    return x, gamma, beta, res, rnd(g, B, HW, C, dtype=dtype)


def gn_check(ops, B, HW, C, G, dtype, act, with_res, forward=True, backward=True, ws=None, tiles=1):  # noqa: F811
    """Chains: 128 as in the module of the small cases; merging the tiles of a sample adds one term per 64 of them (forward)
    or per tile (backward), the parameters' gradients one per 16 partial rows."""
    g = torch.Generator(device="cuda").manual_seed(B + HW + C + G)
    x, gamma, beta, res, dy = gn_inputs(g, B, HW, C, G, dtype, with_res, act == "lrelu")
    ref = gn_ref(x, res, gamma, beta, G, 1e-5, act, dy if backward else None)
    if act == "lrelu":
        nearest = float(ref["y"].abs().min())
        assert nearest > 0.2 * 0.05
    a, nan = ops.ACTS[act], float("nan")
    y, stats = torch.full_like(x, nan), torch.full((2, B, G), nan, device="cuda")
    if forward:
        ops.gn_act_fwd(x, res, y, G, stats, gamma, beta, act=a, ws=ws)
        D = 128 + tiles / 64
        within(y, ref["y"], D * U * ref["S"], "y " + act)
        within(stats[0], ref["mean"], D * U * ref["big"], "mean")
    else:
        stats[0], stats[1] = ref["mean"], ref["rstd"]
    if not backward:
        return
    dx, dres = torch.full_like(x, nan), torch.full_like(x, nan) if with_res else None
    dgamma, dbeta = torch.full_like(gamma, nan), torch.full_like(gamma, nan)
    ops.gn_act_bwd(dy, x, res, dx, dres, G, stats, gamma, beta, dgamma, dbeta, act=a, ws=ws)
    within(dx, ref["dx"], (128 + tiles) * U * ref["Sdx"], "dx " + act)
    if with_res:
        within(dres, ref["dres"], 128 * U * ref["Sdres"], "dres " + act)
    Dp = 128 + B * tiles / 16
    within(dgamma, ref["dgamma"], Dp * U * ref["Sdgamma"], "dgamma " + act)
    within(dbeta, ref["dbeta"], Dp * U * ref["Sdbeta"], "dbeta " + act)


# A workgroup has at most 512 threads and holds its tile in registers: one tile of HW rows takes HW / 512 chunks of 8
# channels a thread at least.  That there is one tile follows from the workspace, which holds one set of sums per tile.
@pytest.mark.parametrize("dtype, with_res, HW", [(BF, False, 4097), (BF, False, 5000), (BF, False, 8192), (BF, True, 3000), (BF, True, 4096),
                                                 (F32, False, 2049), (F32, False, 4096), (F32, True, 1025), (F32, True, 2048)],
                     ids=lambda v: {BF: "bf16", F32: "f32"}.get(v, str(v)))
def test_group_norm_backward_with_full_registers(ops, dtype, with_res, HW):  # noqa: F811
    B, C, G = 33, 64, 32
    one_tile = torch.empty(B * 2 * C * 4, dtype=torch.uint8, device="cuda")
    for act in ("lrelu", "silu", "gelu", "none"):
        gn_check(ops, B, HW, C, G, dtype, act, with_res, forward=False, ws=one_tile)


@pytest.mark.parametrize("dtype, with_res, HW", [(BF, False, 4097), (BF, True, 5000), (BF, False, 8192), (F32, False, 2049), (F32, True, 4096)],
                     ids=lambda v: {BF: "bf16", F32: "f32"}.get(v, str(v)))
def test_group_norm_forward_with_full_registers(ops, dtype, with_res, HW):  # noqa: F811
    B, C, G = 33, 64, 32
    nothing = torch.empty(0, dtype=torch.uint8, device="cuda")       # (one tile per sample and slab needs none)
    for act in ("lrelu", "silu", "gelu", "none"):
        gn_check(ops, B, HW, C, G, dtype, act, with_res, backward=False, ws=nothing)


# the trunk's stages at a large batch, and slabs wider than one chunk
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("case", [(256, 1024, 128, 32), (256, 4096, 64, 32), (96, 1000, 96, 12), (260, 63, 64, 8)],
                         ids=lambda c: "x".join(map(str, c)))
def test_group_norm_large_batches(ops, case, dtype):  # noqa: F811
    for act, with_res in (("lrelu", True), ("silu", False)):
        gn_check(ops, *case, dtype, act, with_res, tiles=64)


# more tiles a sample than a wave has lanes, and more than 8 MB of x in all
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("case", [(1, 360001, 64, 32), (2, 90001, 64, 8), (1, 70000, 8, 1), (1, 40000, 136, 17), (3, 30011, 128, 4)],
                         ids=lambda c: "x".join(map(str, c)))
def test_group_norm_many_tiles(ops, case, dtype):  # noqa: F811
    B, HW, C, G = case
    from cvae_gan_amd.ops import lib, _gn_desc
    import ctypes
    x = torch.empty(B, HW, C, dtype=dtype, device="meta")
    tiles = int(lib.cvg_gn_act_workspace(ctypes.byref(_gn_desc(x, G, 0)), 1)) // (B * 2 * C * 4)
    assert tiles > 16
    for act, with_res in (("lrelu", False), ("gelu", True)):
        gn_check(ops, B, HW, C, G, dtype, act, with_res, tiles=tiles)


def test_group_norm_in_the_two_norm(ops):  # noqa: F811
    """f32: y is off by a handful of u |x - mean| rstd and u |mean| rstd each, dx by the same: 2e-6 of their norms."""
    for B, HW, C, G in ((1, 360001, 64, 32), (33, 4096, 64, 32), (2, 1000, 72, 9)):
        g = torch.Generator(device="cuda").manual_seed(HW)
        x, dy, gamma, beta = rnd(g, B, HW, C, mean=1.0), rnd(g, B, HW, C), rnd(g, C, mean=1.0, scale=0.3), rnd(g, C)
        ref = gn_ref(x, None, gamma, beta, G, 1e-5, "silu", dy)
        y, dx, stats = torch.empty_like(x), torch.empty_like(x), torch.empty(2, B, G, device="cuda")
        dg, db = torch.empty_like(gamma), torch.empty_like(gamma)
        ops.gn_act_fwd(x, None, y, G, stats, gamma, beta, act=ops.ACT_SILU)
        ops.gn_act_bwd(dy, x, None, dx, None, G, stats, gamma, beta, dg, db, act=ops.ACT_SILU)
        assert off(y, ref["y"]) < 2e-6 and off(dx, ref["dx"]) < 2e-6


# ---- linear --------------------------------------------------------------------------------------------------
# Every contraction's last nine terms, and its first, carry most of the result.
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("size", [(1, 64, 8200), (3, 264, 8200), (16, 40, 4104), (64, 512, 8192), (256, 128, 8192), (17, 100, 4105), (130, 264, 520),
                                  (8200, 72, 136), (777, 303, 115), (70, 8200, 64), (1030, 776, 200), (2048, 2048, 72)],
                         ids=lambda c: "x".join(map(str, c)))
def test_linear_ends_of_long_sums(ops, size, dtype):  # noqa: F811
    M, N, K = size
    g = torch.Generator(device="cuda").manual_seed(M + 3 * N + 5 * K)
    x, w = rnd(g, M, K, dtype=dtype), rnd(g, N, K, dtype=dtype, scale=1 / math.sqrt(K))
    dy = rnd(g, M, N, dtype=dtype)

    def sign(*shape):
        return signs(g, *shape)
    places = (0,) + tuple(range(-9, 0))
    for i, p in enumerate(places):
        if -p <= K:
            x[i::10, p] = 30.0                     # of y: row m has its weight at place m mod 10 ...
            w[:, p] = sign(N).to(dtype)            # ... of dx too, with dy's
        if -p <= N:
            dy[i::10, p] = 30.0
            w[p, :] = sign(K).to(dtype)
        if -p <= M:
            dy[p, i::10] = 30.0                    # of dw: every column of dy has its weight in one row
            x[p, :] = sign(K).to(dtype)
    lin_check(ops, x, w, rnd(g, N), None, dy, "none", F32, "none")
    lin_check(ops, x, w, None, None, dy, "silu", dtype, "silu")


@pytest.mark.parametrize("size", [(2048, 1024, 8192), (256, 128, 8192), (3, 264, 8200), (1, 4096, 8192), (8192, 264, 136)],
                         ids=lambda c: "x".join(map(str, c)))
def test_linear_f32_in_the_two_norm(ops, size):  # noqa: F811
    """f32 sums of length L in chains of n additions are off by u sqrt(n / 6) of their norm: chains of at most 512 additions
    (256 of two products behind each other, then the 16 sums of 512 products, slabs or waves) leave 5.5e-7.  One chain of
    4096 would be off by 1.6e-6."""
    M, N, K = size
    g = torch.Generator(device="cuda").manual_seed(K)
    x, w, dy = rnd(g, M, K), rnd(g, N, K), rnd(g, M, N)
    y, dx, dw = torch.empty(M, N, device="cuda"), torch.empty_like(x), torch.empty_like(w)
    ops.linear_act_fwd(x, w, y)
    ops.linear_act_bwd(dy, x, w, dx=dx, dw=dw)
    for got, ref in ((y, x.double() @ w.double().t()), (dx, dy.double() @ w.double()), (dw, dy.double().t() @ x.double())):
        assert off(got, ref) < 1e-6, off(got, ref)


# ---- distillation --------------------------------------------------------------------------------------------
# Rows, classes: more rows than the launch has workgroups (2048 waves' rows times 4, 1024, 512 or 256), for every number of
# registers a row may take; each form with rows of whole vectors and with rows that start anywhere.
WALKS = {BF: [(8300, 496), (8300, 500), (4200, 2000), (4200, 2003), (1100, 8000), (1100, 7999), (1100, 8200), (1030, 20000), (1030, 20001),
              (1030, 32000), (1030, 32003), (600, 45000), (600, 45001), (600, 60000), (600, 60001), (300, 90008), (300, 90001), (300, 131072),
              (300, 131001), (530, 140000), (530, 140001)],
         F32: [(8300, 496), (8300, 500), (4200, 2000), (4200, 2001), (1100, 8000), (1100, 8001), (1030, 10000), (1030, 10001), (1030, 16000),
               (1030, 16001), (600, 20000), (600, 20003), (600, 32000), (600, 32003), (300, 45000), (300, 45001), (300, 60000), (300, 60001),
               (530, 70000), (530, 70001)]}


@pytest.mark.parametrize("dtype, R, V", [(t, *c) for t in WALKS for c in WALKS[t]], ids=lambda v: {BF: "bf16", F32: "f32"}.get(v, str(v)))
def test_distill_more_rows_than_workgroups(ops, dtype, R, V):  # noqa: F811
    """A thread adds 8 exponentials per vector and rescales once: chains of 8 + 3 (V / 8 / threads) + 3 (6 + threads / 64)
    roundings and a few of the exponentials themselves, at most 160 while a row stays in registers (16 vectors a thread), and 3
    more per 8192 classes beyond that."""
    g = torch.Generator(device="cuda").manual_seed(R + V)
    k, T, scale = 11, 1.5, 0.5
    logits = rnd(g, R, V, dtype=dtype, scale=2.0)
    r = torch.arange(R, device="cuda")
    at = torch.randint(0, V, (R,), generator=g, device="cuda")
    for i, place in enumerate((0, V - 1, V - 2, V - 8, V - 9, 7, 8)):
        at[i::16] = place
    logits[r, at] = 20.0                           # most of the row's sum sits in one place
    ti = torch.randint(0, V, (R, k), generator=g, device="cuda", dtype=torch.int32)
    ti[:, 1] = ti[:, 0]                            # the same class twice
    ti[::2, 2] = at[::2].int()
    ti[1::3, 3] = V - 1
    ti[::5, 4:] = -1                               # fewer entries than other rows
    tv = rnd(g, R, k, scale=2.0)
    w = torch.rand(R, generator=g, device="cuda")
    w[r % 7 == 3] = 0                              # rows without weight, without entries, and others, behind each other
    ti[r % 11 == 5] = -1
    logits[r % 14 == 3] = float("nan")             # (weight 0: anything)
    nan = float("nan")
    loss, rl, dl = torch.full((), nan, device="cuda"), torch.full((R,), nan, device="cuda"), torch.full_like(logits, nan)
    ops.distill_topk(logits, tv, ti, loss, rl, dlogits=dl, row_weight=w, temperature=T, grad_scale=scale)
    # the same rows, few enough to have a workgroup each
    part = 128
    l1, r1, d1 = torch.empty_like(loss), torch.empty_like(rl), torch.empty_like(dl)
    for a in range(0, R, part):
        s = slice(a, a + part)
        ops.distill_topk(logits[s], tv[s], ti[s], l1, r1[s], dlogits=d1[s], row_weight=w[s], temperature=T, grad_scale=scale)
    assert torch.equal(rl, r1) and torch.equal(dl, d1)
    # without a gradient (another order of the sums where a row does not fit 256 threads), in place
    ops.distill_topk(logits, tv, ti, l1, r1, row_weight=w, temperature=T, grad_scale=scale)
    D = 160 + 3 * V / 8192
    own = logits.clone()
    ops.distill_topk(own, tv, ti, loss, rl, dlogits=own, row_weight=w, temperature=T, grad_scale=scale)
    assert torch.equal(own, dl)
    for a in range(0, R, 600):                     # (64-bit copies of the logits, a few rows at a time)
        s = slice(a, a + 600)
        rows, Srow, grad, Sgrad = distill_ref(logits[s], tv[s], ti[s], w[s], T, scale)
        within(rl[s], rows, D * U * Srow, "row_loss")
        within(r1[s], rows, D * U * Srow, "row_loss without a gradient")
        within(dl[s], grad, D * U * Sgrad, "dlogits")
    # (the total: f32 sums over 1024 threads, then 6 + 16 more)
    assert abs(float(loss) - float(rl.double().sum())) <= (R / 1024 + 24) * U * float(rl.abs().double().sum())


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("V", [50, 3000, 70000])
def test_distill_infinite_entries_of_the_teacher(ops, dtype, V):  # noqa: F811
    """+inf among a row's entries has no softmax: NaN in its own row.  Where the class is outside it is absent, and -inf alone
    is a row without entries."""
    g = torch.Generator(device="cuda").manual_seed(V)
    inf = float("inf")
    logits, tv = rnd(g, 7, V, dtype=dtype), rnd(g, 7, 3)
    ti = torch.stack([torch.randperm(V, generator=g, device="cuda")[:3] for _ in range(7)]).int()
    tv[0, 1] = inf                                 # beside finite ones
    tv[1, :] = inf                                 # alone
    tv[2, 0], tv[2, 1], tv[2, 2] = -inf, inf, -inf
    tv[3, 0], ti[3, 0] = inf, V                    # absent
    tv[4, :] = -inf
    tv[5, 0], w = inf, torch.ones(7, device="cuda")
    w[5] = 0
    loss, rl, dl = torch.empty((), device="cuda"), torch.empty(7, device="cuda"), torch.empty_like(logits)
    ops.distill_topk(logits, tv, ti, loss, rl, dlogits=dl, row_weight=w)
    assert bool(torch.isnan(rl[:3]).all()) and bool(torch.isfinite(rl[3:]).all())
    assert float(rl[4]) == 0 and float(rl[5]) == 0 and float(dl[4:6].float().abs().max()) == 0
    assert bool(torch.isfinite(dl[3:].float()).all()) and bool(torch.isnan(dl[:3].float()).any(1).all())


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("V", [600, 1500, 5000, 40000, 70001])
def test_distill_many_entries_over_many_rows(ops, dtype, V):  # noqa: F811
    """More teacher entries than threads, in rows that follow each other in one workgroup."""
    g = torch.Generator(device="cuda").manual_seed(V)
    R, k = {600: 8300, 1500: 4200}.get(V, 1100), min(V, 600)
    logits, tv, w = rnd(g, R, V, dtype=dtype), rnd(g, R, k), torch.ones(R, device="cuda")
    ti = torch.rand(R, V, generator=g, device="cuda").argsort(1)[:, :k].int() if V < 2000 else \
        torch.randint(0, V, (R, k), generator=g, device="cuda", dtype=torch.int32)
    loss, rl, dl = torch.empty((), device="cuda"), torch.empty(R, device="cuda"), logits.clone()
    ops.distill_topk(dl, tv, ti, loss, rl, dlogits=dl)
    # chains as above, and k / 64 + 6 additions for the teacher's sum, at most k for a class that all entries name
    D = 160 + 3 * V / 8192 + k / 64 + 8
    for a in list(range(0, R, 1024)) + [R - 200]:
        s = slice(a, a + 200)
        rows, Srow, grad, Sgrad = distill_ref(logits[s], tv[s], ti[s], w[s], 1.0, 1.0)
        within(rl[s], rows, D * U * Srow, "row_loss")
        within(dl[s], grad, D * U * Sgrad, "dlogits")
