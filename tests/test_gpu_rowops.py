"""Group normalisation + activation, the linear layer with its epilogue and the top-logit distillation loss against
plain 64-bit statements of their definitions.

Tolerances.  u = 2^-24 is half a step of f32 relative to the value, HALF[t] the same of the output's type.  Every
comparison allows HALF[t] |ref| for the one rounding of the output plus D u S, where S is the sum of the magnitudes
that enter the result in 64 bits (not the result, which may have cancelled) and D counts the f32 roundings on the
longest chain behind it:
  group norm     a sum passes at most 16 register adds, 6 shuffles, 64 LDS or tile entries, and a handful of operations
                 after it: D = 128 covers it and the few ulps of exp and rsqrt; parameter gradients add one row of
                 partial sums per sample or tile in eight lanes: D = 128 + rows / 8 + 8
  linear         a product sum of length K in any order: D = K + 8; a column sum of M rows: D = M + 8
  distillation   row sums of at most V / 64 + 6 + 16 adds; exp and log: D = 64 + V / 64, times (1 + |argument|)
The activations' second derivatives are below 1.2 in magnitude, their first below 1.2."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from cvae_gan_amd import ops as o
    return o


def within(got, ref, slack, what):
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    g = got.double()
    # a value beyond the largest finite one of the output's type rounds to infinity
    ref = torch.where(ref.abs() > torch.finfo(got.dtype).max, ref.sign() * float("inf"), ref)
    assert torch.equal(torch.isfinite(g), torch.isfinite(ref)), what + ": non-finite values differ"
    fin = torch.isfinite(ref)
    tol = HALF[got.dtype] * ref.abs() + slack + 1e-37
    bad = ((g - ref).abs() > tol) & fin
    assert not bool(bad.any()), "%s: %d of %d beyond tolerance, worst ratio %.3g at %s" % (
        what, int(bad.sum()), bad.numel(), float(((g - ref).abs() / tol)[fin].max()), bad.nonzero()[0].tolist())


def act64(v, act):
    if act == "lrelu":
        return torch.where(v > 0, v, 0.2 * v), torch.where(v > 0, 1.0, 0.2).to(v)
    if act == "silu":
        p = torch.sigmoid(v)
        return v * p, p + v * p * (1 - p)
    if act == "gelu":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (v + 0.044715 * v ** 3))
        return 0.5 * v * (1 + t), 0.5 * (1 + t) + 0.5 * v * (1 - t * t) * c * (1 + 3 * 0.044715 * v * v)
    return v, torch.ones_like(v)


def rnd(g, *shape, dtype=F32, scale=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale + mean).to(dtype)


# ---- group norm ----------------------------------------------------------------------------------------------
def gn_ref(x, res, gamma, beta, G, eps, act, dy=None):
    B, C = x.shape[0], x.shape[-1]
    xd = x.double().reshape(B, -1, G, C // G)
    n = xd.shape[1] * xd.shape[3]
    mean = xd.mean((1, 3), keepdim=True)
    var = ((xd - mean) ** 2).mean((1, 3), keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    xh = (xd - mean) * r
    ga, be = gamma.double().reshape(G, -1), beta.double().reshape(G, -1)
    rd = res.double().reshape(xd.shape) if res is not None else torch.zeros_like(xd)
    pre = xh * ga + be + rd
    big = xd.abs().amax((1, 3), keepdim=True)
    y, k = act64(pre, act)
    S = (r * ga.abs() * big + (xh * ga).abs() + be.abs() + rd.abs())
    out = {"y": y, "S": S * 1.2 + pre.abs(), "mean": mean[:, 0, :, 0], "rstd": r[:, 0, :, 0], "big": big[:, 0, :, 0]}
    if dy is not None:
        dyd = dy.double().reshape(xd.shape)
        g = dyd * k
        gg = g * ga
        m1, m2 = gg.mean((1, 3), keepdim=True), (gg * xh).mean((1, 3), keepdim=True)
        out["dx"] = r * (gg - m1 - xh * m2)
        out["dres"] = g
        out["dgamma"], out["dbeta"] = (g * xh).sum((0, 1)).reshape(C), g.sum((0, 1)).reshape(C)
        # what an error of pre (D u S) and of xhat (D u r big) does to g and to the sums
        dg = dyd.abs() * S * 1.2 + g.abs()
        e = r * big + xh.abs()
        a1 = (dg * ga.abs()).mean((1, 3), keepdim=True)
        a2 = (dg * ga.abs() * xh.abs() + gg.abs() * e).mean((1, 3), keepdim=True)
        out["Sdx"] = r * (dg * ga.abs() + a1 + xh.abs() * a2 + e * m2.abs())
        out["Sdres"] = dg
        out["Sdgamma"] = (dg * xh.abs() + g.abs() * e).sum((0, 1)).reshape(C)
        out["Sdbeta"] = dg.sum((0, 1)).reshape(C)
    for q in ("y", "S", "dx", "dres", "Sdx", "Sdres"):
        if q in out:
            out[q] = out[q].reshape(x.shape)
    return out


GN_CASES = [
    # B, spatial, C, G
    (1, (1,), 8, 1), (2, (1, 1), 16, 16), (3, (5, 7), 24, 3), (2, (4, 4), 512, 32), (5, (13,), 72, 9),
    (2, (33, 31), 64, 32), (1, (64, 64), 64, 32), (2, (17, 19), 40, 8), (1, (9, 9), 2048, 1), (3, (3, 3), 88, 8),
    (2, (40, 41), 96, 2), (1, (1500,), 8, 8), (1, (6, 6), 4096, 2), (2, (50, 3), 136, 17), (1, (200, 100), 32, 4),
    (4, (1000,), 56, 7), (3, (9, 5), 4096, 1), (2, (70,), 8192, 2), (1, (4, 3), 3000, 1),
]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("case", GN_CASES, ids=lambda c: "x".join(map(str, (c[0],) + c[1] + c[2:])))
def test_group_norm(ops, case, dtype):
    B, sp, C, G = case
    g = torch.Generator(device="cuda").manual_seed(B * 1000 + C + G)
    for act, with_res in (("silu", False), ("gelu", True), ("none", False), ("lrelu", True)):
        x = rnd(g, B, *sp, C, dtype=dtype, scale=1.5, mean=3.0)
        gamma, beta = rnd(g, C, mean=1.0, scale=0.3), rnd(g, C, scale=0.3)
        res = rnd(g, B, *sp, C, dtype=dtype) if with_res else None
        dy = rnd(g, B, *sp, C, dtype=dtype)
        y, dx = torch.full_like(x, float("nan")), torch.full_like(x, float("nan"))
        dres = torch.full_like(x, float("nan")) if with_res else None
        stats = torch.full((2, B, G), float("nan"), device="cuda")
        dgamma, dbeta = torch.full_like(gamma, float("nan")), torch.full_like(gamma, float("nan"))
        a = ops.ACTS[act]
        ops.gn_act_fwd(x, res, y, G, stats, gamma, beta, act=a)
        ref = gn_ref(x, res, gamma, beta, G, 1e-5, act, dy)
        n = x[0].numel() // G
        within(y, ref["y"], 128 * U * ref["S"], "y")
        within(stats[0], ref["mean"], 128 * U * ref["big"], "mean")
        # var + eps carries the error of the mean squared away and 128 u of itself
        within(stats[1], ref["rstd"], 128 * U * ref["rstd"] * (1 + (ref["rstd"] * ref["big"]) ** 2 * 128 * U), "rstd")
        ops.gn_act_bwd(dy, x, res, dx, dres, G, stats, gamma, beta, dgamma, dbeta, act=a)
        D = 128 * 1.0
        if act == "lrelu":
            # an argument within its own rounding error of zero may take either slope, and every sum it enters has two
            # right values: gradients are compared where the draw has no such element (the smaller cases)
            if not bool((ref["y"].abs() > 128 * U * ref["S"]).all()):
                continue
        within(dx, ref["dx"], D * U * ref["Sdx"], "dx " + act)
        if with_res:
            within(dres, ref["dres"], D * U * ref["Sdres"], "dres " + act)
        rows = B * (x[0].numel() // C)
        Dp = D + rows / 8 + 8
        within(dgamma, ref["dgamma"], Dp * U * ref["Sdgamma"], "dgamma " + act)
        within(dbeta, ref["dbeta"], Dp * U * ref["Sdbeta"], "dbeta " + act)
        assert n >= 1


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_group_norm_pitches_in_place_and_neighbours(ops, dtype):
    """Channel slices of wider tensors, in and out; the channels beside the slice keep their values; y over res."""
    g = torch.Generator(device="cuda").manual_seed(4)
    B, H, W, C, G = 2, 9, 11, 48, 6
    wide = [rnd(g, B, H, W, 80, dtype=dtype) for _ in range(6)]
    x, res, y, dy, dx, dres = [t[..., 16:64] for t in wide]
    before = [t.clone() for t in wide]
    gamma, beta = rnd(g, C, mean=1.0), rnd(g, C)
    stats = torch.empty(2, B, G, device="cuda")
    ops.gn_act_fwd(x, res, y, G, stats, gamma, beta, act=ops.ACT_SILU)
    dgamma, dbeta = torch.empty_like(gamma), torch.empty_like(gamma)
    ops.gn_act_bwd(dy, x, res, dx, dres, G, stats, gamma, beta, dgamma, dbeta, act=ops.ACT_SILU)
    ref = gn_ref(x, res, gamma, beta, G, 1e-5, "silu", dy)
    within(y, ref["y"], 128 * U * ref["S"], "y")
    within(dx, ref["dx"], 128 * U * ref["Sdx"], "dx")
    within(dres, ref["dres"], 128 * U * ref["Sdres"], "dres")
    for t, b in zip(wide, before):
        assert torch.equal(t[..., :16], b[..., :16]) and torch.equal(t[..., 64:], b[..., 64:])
    res2, dy2 = res.contiguous(), dy.contiguous()
    ops.gn_act_fwd(x, res2, res2, G, stats, gamma, beta, act=ops.ACT_SILU)
    assert torch.equal(res2, y)
    ops.gn_act_bwd(dy2, x, res, dy2, dres, G, stats, gamma, beta, dgamma, dbeta, act=ops.ACT_SILU)
    assert torch.equal(dy2, dx)


def test_group_norm_offsets_and_constant_groups(ops):
    """|mean| >> std keeps its digits (the sums of squares are taken about the mean); a constant group is beta."""
    g = torch.Generator(device="cuda").manual_seed(9)
    for HW in (64, 40000):
        x = rnd(g, 2, HW, 16, mean=1000.0)
        x[1, :, :8] = 7.0
        gamma, beta = torch.ones(16, device="cuda"), rnd(g, 16)
        y, stats = torch.empty_like(x), torch.empty(2, 2, 2, device="cuda")
        ops.gn_act_fwd(x, None, y, 2, stats, gamma, beta, act=ops.ACT_NONE)
        ref = gn_ref(x, None, gamma, beta, 2, 1e-5, "none")
        within(y, ref["y"], 128 * U * ref["S"], "y")
        # x - mean is off by the mean's rounding, 1000 u, about 1e-4 of the tolerance an uncentred variance would need
        assert float((stats[1] - ref["rstd"]).abs()[0].max()) < 1e-4


def test_group_norm_nonfinite_values_stay_in_their_group(ops):
    x = torch.randn(2, 50, 32, device="cuda").to(BF)
    x[0, 3, 0], x[1, 7, 9] = float("inf"), float("nan")
    y = torch.empty_like(x)
    ops.gn_act_fwd(x, None, y, 4, None, torch.ones(32, device="cuda"), torch.zeros(32, device="cuda"), act=ops.ACT_SILU)
    fin = torch.isfinite(y)
    assert bool(fin[0, :, 8:].all()) and bool(fin[1, :, :8].all()) and bool(fin[1, :, 16:].all())
    assert not bool(fin[0, :, :8].any()) and not bool(fin[1, :, 8:16].any())


def test_group_norm_empty_batch(ops):
    x = torch.empty(0, 4, 4, 16, device="cuda")
    one, z = torch.ones(16, device="cuda"), torch.full((16,), 5.0, device="cuda")
    stats = torch.empty(2, 0, 4, device="cuda")
    ops.gn_act_fwd(x, None, torch.empty_like(x), 4, stats, one, one)
    z2 = z.clone()
    ops.gn_act_bwd(x, x, None, torch.empty_like(x), None, 4, stats, one, one, z, z2)
    assert float(z.abs().max()) == 0 and float(z2.abs().max()) == 0


# ---- linear --------------------------------------------------------------------------------------------------
LIN_CASES = [
    # M, N, K
    (1, 1, 1), (1, 64, 64), (1, 1000, 515), (2, 24, 8), (3, 136, 72), (16, 256, 512), (17, 100, 33), (33, 48, 200),
    (64, 512, 128), (100, 77, 129), (130, 264, 264), (256, 128, 1096), (300, 520, 96), (515, 9, 17), (777, 303, 115), (513, 512, 320),
    (1, 4096, 1032), (3, 264, 8200), (16, 40, 4104), (1, 2056, 4104), (5, 2056, 24), (48, 640, 1024), (2048, 40, 8), (1030, 776, 200),
]


def lin_check(ops, x, w, bias, res, dy, act, dw_dtype, what, ws=None, pre_dtype=None):
    M, N, K = x.shape[0], w.shape[0], w.shape[1]
    dtype = x.dtype
    nan = float("nan")
    y = torch.full((M, N), nan, dtype=dtype, device="cuda")
    pre = torch.full((M, N), nan, dtype=pre_dtype or dtype, device="cuda")
    a = ops.ACTS[act]
    ops.linear_act_fwd(x, w, y, bias=bias, res=res, pre=pre, act=a, ws=ws)
    xd, wd = x.double(), w.double()
    b = bias.double() if bias is not None else torch.zeros(N, device="cuda", dtype=torch.float64)
    rp = xd @ wd.t() + b
    S = (xd.abs() @ wd.abs().t() + b.abs()) * (K + 8) * U
    within(pre, rp, S, what + " pre")
    rd = res.double() if res is not None else torch.zeros_like(rp)
    # 1.2 S through the activation, 16 u (1 + |pre|) |pre| for its own exp and division, one rounding of the sum with res
    yr = act64(rp, act)[0] + rd
    within(y, yr, 1.2 * S + 16 * U * (1 + rp.abs()) * rp.abs() + 4 * U * rd.abs(), what + " y")
    dx = torch.full_like(x, nan)
    dw = torch.full((N, K), nan, dtype=dw_dtype, device="cuda")
    db = torch.full((N,), nan, device="cuda")
    ops.linear_act_bwd(dy, x, w, pre=pre, dx=dx, dw=dw, dbias=db, act=a, ws=ws)
    g = dy.double() * act64(pre.double(), act)[1]             # from the argument the forward call kept
    # g: its own arithmetic (16 u), and for an activation its one rounding to the data's type
    eg = g.abs() * 16 * U + dy.double().abs() * 16 * U + (HALF[dtype] * g.abs() if act != "none" else 0)
    within(dx, g @ wd, (g.abs() @ wd.abs()) * (N + 8) * U + eg @ wd.abs(), what + " dx")
    within(dw, g.t() @ xd, (g.abs().t() @ xd.abs()) * (M + 8) * U + eg.t() @ xd.abs(), what + " dw")
    within(db, g.sum(0), g.abs().sum(0) * (M + 8) * U + (g.abs() + dy.double().abs()).sum(0) * 16 * U, what + " dbias")
    return y, dx, dw, db


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("case", LIN_CASES, ids=lambda c: "x".join(map(str, c)))
def test_linear(ops, case, dtype):
    M, N, K = case
    g = torch.Generator(device="cuda").manual_seed(M + 7 * N + 31 * K)
    x, w = rnd(g, M, K, dtype=dtype), rnd(g, N, K, dtype=dtype, scale=1 / math.sqrt(K))
    bias, dy, res = rnd(g, N), rnd(g, M, N, dtype=dtype), rnd(g, M, N, dtype=dtype)
    lin_check(ops, x, w, bias, None, dy, "none", F32, "none")
    lin_check(ops, x, w, bias, res, dy, "gelu", dtype, "gelu")
    lin_check(ops, x, w, None, None, dy, "silu", F32, "silu", pre_dtype=F32)
    lin_check(ops, x, w, None, res, dy, "lrelu", dtype, "lrelu")


# The sizes at which the wider tiles are taken, with one to many stages of k, ends inside a tile, and rows that take copies
# and single elements.
@pytest.mark.parametrize("case", [(4096, 4096, 64), (4100, 4104, 136), (4096, 4099, 130), (4096, 4096, 328), (2056, 4104, 4100),
                                  (1000, 1000, 2056), (2048, 2048, 72)], ids=lambda c: "x".join(map(str, c)))
def test_linear_wide(ops, case):
    M, N, K = case
    g = torch.Generator(device="cuda").manual_seed(M + 7 * N + 31 * K)
    x, w = rnd(g, M, K, dtype=BF), rnd(g, N, K, dtype=BF, scale=1 / math.sqrt(K))
    bias, dy, res = rnd(g, N), rnd(g, M, N, dtype=BF), rnd(g, M, N, dtype=BF)
    lin_check(ops, x, w, bias, res, dy, "gelu", F32, "gelu", pre_dtype=F32)
    lin_check(ops, x, w, bias, None, dy, "none", BF, "none")


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("size", [(70, 144, 136), (4, 272, 264), (300, 264, 520)])
@pytest.mark.parametrize("off", [0, 1, 8])
def test_linear_pitches_and_neighbours(ops, dtype, size, off):
    """Column slices of wider tensors at aligned and unaligned offsets; what lies beside the outputs stays; the
    elements of the wider rows beside the operands are NaN and must not be multiplied in."""
    M, N, K = size
    g = torch.Generator(device="cuda").manual_seed(off + M)
    nan = float("nan")

    def sliced(r, c, dt=dtype, scale=1.0):
        big = torch.full((r + 2, c + 24), nan, dtype=dt, device="cuda")
        s = big[1:r + 1, off:off + c]
        s.copy_(rnd(g, r, c, dtype=dt, scale=scale))
        return big, s

    (_, x), (_, w), (_, dy), (_, res) = sliced(M, K), sliced(N, K, scale=1 / math.sqrt(K)), sliced(M, N), sliced(M, N)
    bias = rnd(g, N)
    y0, dx0, dw0, _ = lin_check(ops, x, w, bias, res, dy, "silu", F32, "sliced")
    outs = [sliced(M, N), sliced(M, N), sliced(M, K), sliced(N, K, F32)]
    (yb, y), (pb, pre), (dxb, dx), (dwb, dw) = outs
    ops.linear_act_fwd(x, w, y, bias=bias, res=res, pre=pre, act=ops.ACT_SILU)
    ops.linear_act_bwd(dy, x, w, pre=pre, dx=dx, dw=dw, act=ops.ACT_SILU)
    for big, s, ref in ((yb, y, y0), (dxb, dx, dx0), (dwb, dw, dw0)):
        # the output's pitch may choose another order of the sum, never another value beyond rounding
        assert float((s.double() - ref.double()).abs().max()) <= 2 * (HALF[s.dtype] + 600 * U) * float(ref.abs().max())
        mask = torch.ones_like(big, dtype=torch.bool)
        mask[1:s.shape[0] + 1, off:off + s.shape[1]] = False
        assert bool(torch.isnan(big[mask]).all()), "a neighbour of the output was written"
        assert bool(torch.isfinite(s).all())


def test_linear_gradients_match_differences(ops):
    """d(sum(y * c))/dx, dw, dbias against central differences of the 64-bit definition."""
    g = torch.Generator(device="cuda").manual_seed(2)
    x, w, b, c = rnd(g, 5, 12), rnd(g, 7, 12, scale=0.4), rnd(g, 7), rnd(g, 5, 7)
    for act in ("silu", "gelu"):
        a = ops.ACTS[act]
        y, pre = torch.empty(5, 7, device="cuda"), torch.empty(5, 7, device="cuda")
        ops.linear_act_fwd(x, w, y, bias=b, pre=pre, act=a)
        dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
        ops.linear_act_bwd(c, x, w, pre=pre, dx=dx, dw=dw, dbias=db, act=a)

        def f(x_, w_, b_):
            return float((act64(x_ @ w_.t() + b_, act)[0] * c.double()).sum())
        h = 1e-5
        args = [x.double(), w.double(), b.double()]
        for i, got in enumerate((dx, dw, db)):
            for pos in ((0, 0), (1, 3), (4, 6)):
                if i == 2:
                    pos = pos[1:]
                hi, lo = [t.clone() for t in args], [t.clone() for t in args]
                hi[i][pos] += h
                lo[i][pos] -= h
                num = (f(*hi) - f(*lo)) / (2 * h)
                # central differences: h^2 times a third derivative of order 10, and 1e-16 * 50 / h
                assert abs(num - float(got[pos])) < 1e-8 + 1e-9 + 200 * U * 20


def test_linear_no_rows(ops):
    x, w = torch.empty(0, 16, device="cuda"), torch.randn(8, 16, device="cuda")
    ops.linear_act_fwd(x, w, torch.empty(0, 8, device="cuda"))
    dw, db = torch.full((8, 16), 3.0, device="cuda"), torch.full((8,), 3.0, device="cuda")
    ops.linear_act_bwd(torch.empty(0, 8, device="cuda"), x, w, dx=torch.empty_like(x), dw=dw, dbias=db)
    assert float(dw.abs().max()) == 0 and float(db.abs().max()) == 0


def test_linear_nonfinite_rows_stay_in_their_rows(ops):
    """A padded row may hold anything: it reaches its own output row only (sums over other rows never see it)."""
    for M, N, K in ((5, 72, 80), (200, 264, 512)):
        for dtype in (BF, F32):
            x, w = torch.randn(M, K, device="cuda").to(dtype), torch.randn(N, K, device="cuda").to(dtype)
            x[2] = float("nan")
            x[3] = float("inf")
            y = torch.empty(M, N, dtype=dtype, device="cuda")
            ops.linear_act_fwd(x, w, y, act=ops.ACT_GELU)
            fin = torch.isfinite(y).all(1)
            keep = torch.ones(M, dtype=torch.bool, device="cuda")
            keep[2] = keep[3] = False
            assert bool(fin[keep].all()) and not bool(fin[2])


# ---- distillation --------------------------------------------------------------------------------------------
def distill_ref(logits, tv, ti, w, T, scale):
    R, V = logits.shape
    z = logits.double() / T
    logq = torch.log_softmax(z, 1)
    inside = (ti >= 0) & (ti < V) & (tv != float("-inf"))
    t = torch.where(inside, tv.double() / T, torch.full_like(tv, float("-inf"), dtype=torch.float64))
    live = inside.any(1) & (w != 0)
    t = torch.where(live[:, None], t, torch.zeros_like(t))
    logp = torch.log_softmax(t, 1)
    p = torch.where(inside | ~live[:, None], logp.exp(), torch.zeros_like(t))
    idx = torch.where(inside, ti, torch.zeros_like(ti)).long()
    lq = logq.gather(1, idx)
    terms = torch.where(inside & (p > 0), p * (logp - lq), torch.zeros_like(p))
    mags = torch.where(inside & (p > 0), p * (logp.abs() + lq.abs() + 1), torch.zeros_like(p))
    zero = torch.zeros(R, dtype=torch.float64, device=logits.device)
    rows = torch.where(live, w.double() * T * T * terms.sum(1), zero)
    Srow = torch.where(live, w.double().abs() * T * T * mags.sum(1), zero)
    q = logq.exp()
    top = torch.zeros_like(q)
    top.scatter_add_(1, idx, torch.where(inside, p, torch.zeros_like(p)))
    targ = torch.zeros_like(q)
    targ.scatter_add_(1, idx, torch.where(inside, p * (1 + logp.abs()), torch.zeros_like(p)))
    c = (w.double() * T * scale)[:, None]
    grad = torch.where(live[:, None], c * (q - top), torch.zeros_like(q))
    qarg = torch.where(q > 0, q * (2 + logq.abs()), torch.zeros_like(q))
    Sgrad = torch.where(live[:, None], c.abs() * (qarg + 2 * targ), torch.zeros_like(q))
    return rows, Srow, grad, Sgrad


def distill_check(ops, logits, tv, ti, w, T, scale, what, in_place=False):
    R, V = logits.shape
    loss = torch.full((), float("nan"), device="cuda")
    rl = torch.full((R,), float("nan"), device="cuda")
    wr = torch.ones(R, device="cuda") if w is None else w
    rows, Srow, grad, Sgrad = distill_ref(logits, tv, ti, wr, T, scale)
    dl = logits if in_place else torch.full_like(logits, float("nan"))
    ops.distill_topk(logits, tv, ti, loss, rl, dlogits=dl, row_weight=w, temperature=T, grad_scale=scale)
    D = 64 + V / 64 + tv.shape[1] / 64
    within(rl, rows, D * U * Srow, what + " row_loss")
    within(loss, rows.sum(), (D + R / 64 + 32) * U * Srow.sum(), what + " loss")
    within(dl, grad, D * U * Sgrad, what + " dlogits")
    return loss, rl, dl


DIST_CASES = [(1, 1, 1), (3, 7, 7), (5, 100, 10), (64, 16, 3), (9, 1000, 64), (4, 1003, 130), (2, 8192, 128), (3, 32768, 64),
              (2, 33333, 100), (2, 70001, 1024), (9, 1500, 1024), (1, 131072, 128), (1, 140000, 33), (1, 300007, 5)]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("case", DIST_CASES, ids=lambda c: "x".join(map(str, c)))
def test_distill(ops, case, dtype):
    R, V, k = case
    g = torch.Generator(device="cuda").manual_seed(V + k)
    for T in (1.0, 2.5):
        logits = rnd(g, R, V, dtype=dtype, scale=2.0)
        ti = torch.stack([torch.randperm(V, generator=g, device="cuda")[:k] for _ in range(R)]).int()
        tv = rnd(g, R, k, scale=2.0)
        w = torch.rand(R, generator=g, device="cuda")
        distill_check(ops, logits, tv, ti, w, T, 0.25, "plain")
        distill_check(ops, logits, tv, ti, None, T, 1.0, "no weight")
        distill_check(ops, logits.clone(), tv, ti, w, T, -0.5, "in place", in_place=True)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("V", [50, 3000, 70000])
def test_distill_absent_entries_masks_and_duplicates(ops, dtype, V):
    g = torch.Generator(device="cuda").manual_seed(V)
    R, k = 8, 20
    logits = rnd(g, R, V, dtype=dtype, scale=2.0)
    ti = torch.stack([torch.randperm(V, generator=g, device="cuda")[:k] for _ in range(R)]).int()
    tv = rnd(g, R, k, scale=2.0)
    w = torch.ones(R, device="cuda")
    ti[0, 5:] = -1                         # fewer entries than the others
    ti[1, 3], ti[1, 4] = V, 2 ** 31 - 1    # outside
    ti[2, :] = -1                          # none at all
    ti[3, 7] = ti[3, 2]                    # the same class twice, and thrice
    ti[3, 11] = ti[3, 2]
    tv[4, ::2] = float("-inf")             # teacher probability zero
    tv[5, :] = float("-inf")               # nothing left
    w[6] = 0
    logits[6] = float("nan")               # a padding row holds anything
    logits[2] = float("inf")
    lowest = torch.finfo(dtype).min
    other = ti[7].long().tolist()
    keep = [i for i in range(V) if i not in other]
    logits[7, keep[: len(keep) // 2]] = lowest          # masked classes of the student
    logits[7, keep[len(keep) // 2: -1]] = float("-inf")
    distill_check(ops, logits, tv, ti, w, 2.0, 1.0, "mixed")
    masked = torch.full_like(logits, lowest)            # masked throughout: uniform
    masked[1::2, V // 2] = 1.0                          # ... or but for one class
    distill_check(ops, masked, tv, ti, w, 0.5, 1.0, "masked")
    # a masked class that the teacher wants: the loss is infinite, the gradient is not
    l2 = logits.clone()
    l2[7, other[0]] = float("-inf")
    loss, rl, dl = torch.empty((), device="cuda"), torch.empty(R, device="cuda"), torch.empty_like(l2)
    ops.distill_topk(l2, tv, ti, loss, rl, dlogits=dl, row_weight=w)
    assert float(rl[7]) == float("inf") and bool(torch.isfinite(dl).all())
    assert float(rl[2]) == 0 and float(rl[5]) == 0 and float(rl[6]) == 0
    assert float(dl[[2, 5, 6]].float().abs().max()) == 0
    tv2 = tv.clone()
    tv2[0, 0] = float("nan")               # a NaN of the teacher spoils its own row only
    ops.distill_topk(logits, tv2, ti, loss, rl, dlogits=dl, row_weight=w)
    assert bool(torch.isnan(rl[0])) and bool(torch.isfinite(rl[1:]).all()) and bool(torch.isfinite(dl[1:].float()).all())


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("V", [37, 2501, 40003])
def test_distill_unaligned_rows_and_neighbours(ops, dtype, V):
    g = torch.Generator(device="cuda").manual_seed(V)
    R, k = 5, 9
    for off_in, off_out in ((1, 1), (3, 3), (0, 5), (2, 0)):
        big = torch.full((R + 1, V + 13), float("nan"), dtype=dtype, device="cuda")
        logits = big[:R, off_in:off_in + V]
        logits.copy_(rnd(g, R, V, dtype=dtype, scale=2.0))
        bo = torch.full((R + 1, V + 9), 77.0, dtype=dtype, device="cuda")
        dl = bo[:R, off_out:off_out + V]
        tk = torch.zeros(R, k + 3, device="cuda")
        tv = tk[:, 1:k + 1]
        tv.copy_(rnd(g, R, k))
        tik = torch.full((R, k + 3), -5, dtype=torch.int32, device="cuda")
        ti = tik[:, 2:k + 2]
        ti.copy_(torch.stack([torch.randperm(V, generator=g, device="cuda")[:k] for _ in range(R)]).int())
        loss, rl = torch.empty((), device="cuda"), torch.empty(R, device="cuda")
        ops.distill_topk(logits, tv, ti, loss, rl, dlogits=dl, temperature=1.5)
        rows, Srow, grad, Sgrad = distill_ref(logits, tv, ti, torch.ones(R, device="cuda"), 1.5, 1.0)
        D = 64 + V / 64
        within(rl, rows, D * U * Srow, "row_loss")
        within(dl, grad, D * U * Sgrad, "dlogits")
        mask = torch.ones_like(bo, dtype=torch.bool)
        mask[:R, off_out:off_out + V] = False
        assert bool((bo[mask] == 77.0).all())


def test_distill_loss_only_and_no_rows(ops):
    g = torch.Generator(device="cuda").manual_seed(1)
    logits, tv = rnd(g, 6, 500, dtype=BF), rnd(g, 6, 4)
    ti = torch.randint(0, 500, (6, 4), generator=g, device="cuda").int()
    la, ra, lb, rb = torch.empty((), device="cuda"), torch.empty(6, device="cuda"), torch.empty(1, device="cuda"), torch.empty(6, device="cuda")
    ops.distill_topk(logits, tv, ti, la, ra)
    ops.distill_topk(logits, tv, ti, lb, rb, dlogits=torch.empty_like(logits))
    assert torch.equal(ra, rb) and float(la) == float(lb)
    ops.distill_topk(logits[:0], tv[:0], ti[:0], la, ra[:0], dlogits=logits[:0])
    assert float(la) == 0


def test_distill_gradient_matches_differences(ops):
    g = torch.Generator(device="cuda").manual_seed(5)
    logits, tv = rnd(g, 3, 12), rnd(g, 3, 4)
    ti = torch.stack([torch.randperm(12, generator=g, device="cuda")[:4] for _ in range(3)]).int()
    w = torch.tensor([1.0, 0.5, 2.0], device="cuda")
    loss, rl, dl = torch.empty((), device="cuda"), torch.empty(3, device="cuda"), torch.empty_like(logits)
    ops.distill_topk(logits, tv, ti, loss, rl, dlogits=dl, row_weight=w, temperature=2.0, grad_scale=3.0)

    def f(l):
        z = torch.log_softmax(l / 2.0, 1).gather(1, ti.long())
        lp = torch.log_softmax(tv.double() / 2.0, 1)
        return float((w.double() * 4.0 * (lp.exp() * (lp - z)).sum(1)).sum()) * 3.0
    h = 1e-5
    for pos in [(0, 0), (1, int(ti[1, 0])), (2, 11), (2, int(ti[2, 3]))]:
        hi, lo = logits.double(), logits.double()
        hi[pos] += h
        lo[pos] -= h
        assert abs((f(hi) - f(lo)) / (2 * h) - float(dl[pos])) < 1e-8 + 100 * U * 6


# ---- as they are used ----------------------------------------------------------------------------------------
def chain(ops, t, bufs):
    """One training pass of a student head: norm + activation -> hidden layer -> logits -> distillation, and back."""
    b = bufs
    ops.gn_act_fwd(t["x"], t["res"], b["h"], 4, b["stats"], t["gamma"], t["beta"], act=ops.ACT_SILU, ws=b["ws_gn"])
    feat = b["h"].view(t["x"].shape[0], -1)
    ops.linear_act_fwd(feat, t["w1"], b["a"], bias=t["b1"], pre=b["pre"], act=ops.ACT_GELU, ws=b["ws1"])
    ops.linear_act_fwd(b["a"], t["w2"], b["logits"], bias=t["b2"], ws=b["ws2"])
    ops.distill_topk(b["logits"], t["tv"], t["ti"], b["loss"], b["rl"], dlogits=b["dl"], temperature=2.0, grad_scale=0.1)
    ops.linear_act_bwd(b["dl"], b["a"], t["w2"], dx=b["da"], dw=b["dw2"], dbias=b["db2"], ws=b["ws2"])
    ops.linear_act_bwd(b["da"], feat, t["w1"], pre=b["pre"], dx=b["dh"].view_as(feat), dw=b["dw1"], dbias=b["db1"], act=ops.ACT_GELU,
                       ws=b["ws1"])
    ops.gn_act_bwd(b["dh"], t["x"], t["res"], b["dx"], b["dres"], 4, b["stats"], t["gamma"], t["beta"], b["dg"], b["dbt"],
                   act=ops.ACT_SILU, ws=b["ws_gn"])
    return [b[k] for k in ("loss", "rl", "dl", "dw2", "db2", "dw1", "db1", "dx", "dres", "dg", "dbt")]


def chain_setup(ops, dtype, B=24, side=5, C=32, H=72, V=210, k=12, seed=3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    F = side * side * C
    t = dict(x=rnd(g, B, side, side, C, dtype=dtype), res=rnd(g, B, side, side, C, dtype=dtype), gamma=rnd(g, C, mean=1.0, scale=0.2),
             beta=rnd(g, C, scale=0.2), w1=rnd(g, H, F, dtype=dtype, scale=F ** -0.5), b1=rnd(g, H, scale=0.1),
             w2=rnd(g, V, H, dtype=dtype, scale=H ** -0.5), b2=rnd(g, V, scale=0.1), tv=rnd(g, B, k, scale=2.0),
             ti=torch.stack([torch.randperm(V, generator=g, device="cuda")[:k] for _ in range(B)]).int())
    e = lambda *s, dt=dtype: torch.zeros(*s, dtype=dt, device="cuda")   # noqa: E731
    b = dict(h=e(B, side, side, C), stats=e(2, B, 4, dt=F32), a=e(B, H), pre=e(B, H), logits=e(B, V), loss=e(1, dt=F32), rl=e(B, dt=F32),
             dl=e(B, V), da=e(B, H), dw2=e(V, H, dt=F32), db2=e(V, dt=F32), dh=e(B, side, side, C), dw1=e(H, F, dt=F32), db1=e(H, dt=F32),
             dx=e(B, side, side, C), dres=e(B, side, side, C), dg=e(C, dt=F32), dbt=e(C, dt=F32))
    b["ws_gn"] = ops.gn_act_workspace(t["x"], 4, backward=True)
    b["ws1"] = ops.linear_act_workspace(b["h"].view(B, -1), t["w1"], act=ops.ACT_GELU, backward=True)
    b["ws2"] = ops.linear_act_workspace(b["a"], t["w2"], backward=True)
    return t, b


def chain_ref(t):
    """The same in float64 autograd."""
    v = {k: t[k].double().requires_grad_() for k in ("x", "res", "gamma", "beta", "w1", "b1", "w2", "b2")}
    B, C = t["x"].shape[0], t["x"].shape[-1]
    xn = torch.nn.functional.group_norm(v["x"].permute(0, 3, 1, 2), 4, v["gamma"], v["beta"], 1e-5).permute(0, 2, 3, 1) + v["res"]
    h = (xn * torch.sigmoid(xn)).reshape(B, -1)
    a = torch.nn.functional.gelu(h @ v["w1"].t() + v["b1"], approximate="tanh")
    logits = a @ v["w2"].t() + v["b2"]
    lp = torch.log_softmax(t["tv"].double() / 2.0, 1)
    rl = 4.0 * (lp.exp() * (lp - torch.log_softmax(logits / 2.0, 1).gather(1, t["ti"].long()))).sum(1)
    (0.1 * rl.sum()).backward()
    return rl.detach(), v


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
def test_chain_forward_and_backward(ops, dtype):
    t, b = chain_setup(ops, dtype)
    out = chain(ops, t, b)
    rl, v = chain_ref(t)
    # f32: every stage adds errors of order 1e3 u of its operands' norms; bf16: each of the eight rounded tensors on the
    # way adds at most 2^-8 of its own norm, amplified by at most the Lipschitz constants of the stages (about 2 together)
    tol = 4e-4 if dtype == F32 else 16 * 2.0 ** -8
    assert float((out[1].double() - rl).norm() / rl.norm()) < tol
    for got, name in zip(out[3:], ("w2", "b2", "w1", "b1", "x", "res", "gamma", "beta")):
        ref = v[name].grad
        assert float((got.double().view_as(ref) - ref).norm() / ref.norm()) < tol, name


@pytest.mark.parametrize("big", [False, True], ids=["small", "large"])
def test_chain_in_a_graph_on_streams_and_repeated(ops, big):
    """Captured and replayed with new inputs between the replays and eager work around them; two captured chains that
    run side by side with their own workspaces; a side stream: bit-identical to the eager run each time."""
    kw = dict(B=96, side=24, C=64, H=520, V=4100, k=40) if big else {}
    t, b = chain_setup(ops, BF, **kw)
    t2, b2 = chain_setup(ops, BF, seed=8, **kw)
    eager = [o.clone() for o in chain(ops, t, b)]
    eager2 = [o.clone() for o in chain(ops, t2, b2)]
    again = chain(ops, t, b)
    assert all(torch.equal(p, q) for p, q in zip(eager, again))
    torch.cuda.synchronize()
    graphs = []
    for tt, bb in ((t, b), (t2, b2)):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            chain(ops, tt, bb)
        graphs.append(gr)
    swap = {k: t[k].clone() for k in ("x", "w1", "tv")}
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for rep in range(4):
        for o in chain_outputs(b) + chain_outputs(b2):
            o.fill_(float("nan"))
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            graphs[0].replay()
        with torch.cuda.stream(s2):
            graphs[1].replay()
        torch.cuda.synchronize()
        want = eager if rep != 2 else other
        assert all(torch.equal(p, q) for p, q in zip(want, chain_outputs(b))), rep
        assert all(torch.equal(p, q) for p, q in zip(eager2, chain_outputs(b2))), rep
        if rep == 1:                       # new inputs in the same buffers
            t["x"].mul_(0.5).add_(0.25)
            t["w1"].neg_()
            t["tv"].mul_(1.5)
            other = [o.clone() for o in chain(ops, t, b)]
            assert not torch.equal(other[0], eager[0])
        if rep == 2:
            for k in swap:
                t[k].copy_(swap[k])
    with torch.cuda.stream(s1):
        side = chain(ops, t, b)
    s1.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(eager, side))


def chain_outputs(b):
    return [b[k] for k in ("loss", "rl", "dl", "dw2", "db2", "dw1", "db1", "dx", "dres", "dg", "dbt")]


def test_torch_operators(ops):
    """The same kernels as torch.ops.cvaegan.*."""
    import cvae_gan_amd.torch_ops  # noqa: F401
    t, b = chain_setup(ops, BF)
    ref = [o.clone() for o in chain(ops, t, b)]
    ns = torch.ops.cvaegan
    t, b = chain_setup(ops, BF)
    ns.gn_act_fwd(t["x"], t["res"], b["h"], 4, b["stats"], t["gamma"], t["beta"], 1e-5, ops.ACT_SILU, b["ws_gn"])
    feat = b["h"].view(t["x"].shape[0], -1)
    ns.linear_act_fwd(feat, t["w1"], b["a"], t["b1"], None, b["pre"], ops.ACT_GELU, None)
    ns.linear_act_fwd(b["a"], t["w2"], b["logits"], t["b2"], None, None, ops.ACT_NONE, b["ws2"])
    ns.distill_topk(b["logits"], t["tv"], t["ti"], b["loss"], b["rl"], b["dl"], None, 2.0, 0.1)
    ns.linear_act_bwd(b["dl"], b["a"], t["w2"], None, b["da"], b["dw2"], b["db2"], ops.ACT_NONE, b["ws2"])
    ns.linear_act_bwd(b["da"], feat, t["w1"], b["pre"], b["dh"].view_as(feat), b["dw1"], b["db1"], ops.ACT_GELU, None)
    ns.gn_act_bwd(b["dh"], t["x"], t["res"], b["dx"], b["dres"], 4, b["stats"], t["gamma"], t["beta"], b["dg"], b["dbt"], ops.ACT_SILU,
                  b["ws_gn"])
    assert all(torch.equal(p, q) for p, q in zip(ref, chain_outputs(b)))


def pitched(rows, width, pitch, dtype):
    """[rows, width] at a pitch that puts the last rows beyond 2^31 elements; the memory between the rows stays as it is."""
    return torch.empty(rows * pitch, dtype=dtype, device="cuda").as_strided((rows, width), (pitch, 1))


# 4000000 elements is a pitch that the tile kernel addresses directly, 6000000 one whose operands are copied and whose
# outputs go element by element
@pytest.mark.parametrize("pitch", [4000000, 6000000])
def test_offsets_beyond_32_bits(ops, pitch):
    """The same numbers at a pitch of megabytes and dense: the same results."""
    g = torch.Generator(device="cuda").manual_seed(pitch)
    M, N, K = 560, 72, 136

    def far(t):
        p = pitched(t.shape[0], t.shape[1], pitch, t.dtype)
        p.copy_(t)
        return p
    x, w, dy, res = rnd(g, M, K, dtype=BF), rnd(g, N, K, dtype=BF), rnd(g, M, N, dtype=BF), rnd(g, M, N, dtype=BF)
    got = []
    for f in (lambda t: t.clone(), far):
        xx, dd, rr = f(x), f(dy), f(res)
        y, pre, dx = f(torch.zeros_like(res)), f(torch.zeros_like(res)), f(torch.zeros_like(x))
        dw, db = torch.empty(N, K, device="cuda"), torch.empty(N, device="cuda")
        ops.linear_act_fwd(xx, w, y, res=rr, pre=pre, act=ops.ACT_SILU)
        ops.linear_act_bwd(dd, xx, w, pre=pre, dx=dx, dw=dw, dbias=db, act=ops.ACT_SILU)
        one = f(torch.zeros_like(res))
        ops.linear_act_fwd(xx[-20:], w, one[-20:], res=rr[-20:])
        got.append([t.clone() for t in (y, pre, dx, dw, db, one[-20:])])
        del xx, dd, rr, y, pre, dx, one
    assert all(torch.equal(p, q) for p, q in zip(*got))
    B, C, G = 2, 64, 8
    x, dy = rnd(g, M, C, dtype=BF), rnd(g, M, C, dtype=BF)
    gamma, beta = rnd(g, C, mean=1.0), rnd(g, C)
    got = []
    for f in (lambda t: t.clone(), far):
        xx, dd, y, dx = [f(t).view(B, M // B, C) if f is not far else f(t).unflatten(0, (B, M // B)) for t in (x, dy, x, x)]
        stats, dg, dbt = torch.empty(2, B, G, device="cuda"), torch.empty(C, device="cuda"), torch.empty(C, device="cuda")
        ops.gn_act_fwd(xx, None, y, G, stats, gamma, beta, act=ops.ACT_SILU)
        ops.gn_act_bwd(dd, xx, None, dx, None, G, stats, gamma, beta, dg, dbt, act=ops.ACT_SILU)
        got.append([t.clone() for t in (y, dx, stats, dg, dbt)])
        del xx, dd, y, dx
    assert all(torch.equal(p, q) for p, q in zip(*got))
    V = 3000
    logits, tv = rnd(g, M, V, dtype=BF), rnd(g, M, 5)
    ti = torch.randint(0, V, (M, 5), generator=g, device="cuda", dtype=torch.int32)
    got = []
    for f in (lambda t: t.clone(), far):
        ll, dl = f(logits), f(torch.zeros_like(logits))
        loss, rl = torch.empty((), device="cuda"), torch.empty(M, device="cuda")
        ops.distill_topk(ll, tv, ti, loss, rl, dlogits=dl, temperature=2.0)
        got.append([t.clone() for t in (loss, rl, dl)])
        del ll, dl
    assert all(torch.equal(p, q) for p, q in zip(*got))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("size", [(5, 48, 72), (130, 264, 264), (300, 77, 129)])
def test_linear_gradients_one_at_a_time(ops, dtype, size):
    """Every subset of the gradients is what the call for all of them gives."""
    M, N, K = size
    g = torch.Generator(device="cuda").manual_seed(M)
    x, w, dy, pre = rnd(g, M, K, dtype=dtype), rnd(g, N, K, dtype=dtype), rnd(g, M, N, dtype=dtype), rnd(g, M, N)
    for act in (ops.ACT_NONE, ops.ACT_GELU):
        def run(which):
            out = [torch.full(s, float("nan"), dtype=t, device="cuda") if i in which else None
                   for i, (s, t) in enumerate((((M, K), dtype), ((N, K), F32), ((N,), F32)))]
            ops.linear_act_bwd(dy, x, w, pre=pre, dx=out[0], dw=out[1], dbias=out[2], act=act)
            return out
        full = run((0, 1, 2))
        for which in ((0,), (1,), (2,), (0, 1), (0, 2), (1, 2)):
            for i, t in enumerate(run(which)):
                assert (t is None) == (i not in which) and (t is None or torch.equal(t, full[i])), which


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_vectors_at_any_element(ops, dtype):
    """Parameter vectors, statistics and teacher entries that start on no 16-byte border; stats left out."""
    g = torch.Generator(device="cuda").manual_seed(11)

    def odd(t):
        p = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape)
        return p.copy_(t)
    for B, HW, C, G in ((3, 35, 40, 5), (1, 4096, 64, 8)):
        x, dy, gamma, beta = rnd(g, B, HW, C, dtype=dtype), rnd(g, B, HW, C, dtype=dtype), rnd(g, C, mean=1.0), rnd(g, C)
        got = []
        for f in (torch.clone, odd):
            y, dx, y2 = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
            st, dg, db = f(torch.zeros(2, B, G, device="cuda")), f(torch.zeros_like(gamma)), f(torch.zeros_like(gamma))
            ops.gn_act_fwd(x, None, y, G, st, f(gamma), f(beta), act=ops.ACT_GELU)
            ops.gn_act_fwd(x, None, y2, G, None, f(gamma), f(beta), act=ops.ACT_GELU)
            ops.gn_act_bwd(dy, x, None, dx, None, G, st, f(gamma), f(beta), dg, db, act=ops.ACT_GELU)
            assert torch.equal(y, y2)
            got.append((y, dx, st, dg, db))
        assert all(torch.equal(p, q) for p, q in zip(*got))
    for M, N, K in ((7, 40, 32), (200, 136, 72)):
        x, w, bias, dy = rnd(g, M, K, dtype=dtype), rnd(g, N, K, dtype=dtype), rnd(g, N), rnd(g, M, N, dtype=dtype)
        got = []
        for f in (torch.clone, odd):
            y, db = torch.empty(M, N, dtype=dtype, device="cuda"), f(torch.zeros_like(bias))
            ops.linear_act_fwd(x, w, y, bias=f(bias), act=ops.ACT_SILU)
            ops.linear_act_bwd(dy, x, w, dbias=db)
            got.append((y, db))
        assert all(torch.equal(p, q) for p, q in zip(*got))
    logits, tv, wt = rnd(g, 9, 1000, dtype=dtype), rnd(g, 9, 6), rnd(g, 9).abs()
    ti = torch.randint(0, 1000, (9, 6), generator=g, device="cuda", dtype=torch.int32)
    got = []
    for f in (torch.clone, odd):
        loss, rl, dl = f(torch.zeros(1, device="cuda")), f(torch.zeros(9, device="cuda")), torch.empty_like(logits)
        ops.distill_topk(logits, f(tv), f(ti), loss, rl, dlogits=dl, row_weight=f(wt))
        got.append((loss, rl, dl))
    assert all(torch.equal(p, q) for p, q in zip(*got))
