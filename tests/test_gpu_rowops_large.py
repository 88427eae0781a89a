"""Group norm, linear layers and distillation at the largest sizes their limits allow, or past 2^31 elements."""
import math

import pytest
import torch

from test_gpu_rowops import BF, F32, U, act64, distill_ref, gn_ref, lin_check, ops, rnd, within  # noqa: F401

pytestmark = pytest.mark.gpu


def off(got, ref):
    return float((got.double() - ref).norm() / ref.norm())


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def test_group_norm_of_more_than_2_31_elements(ops):  # noqa: F811
    """2100 samples of 16384 pixels and 64 channels, in 16 tiles each; parameter gradients: partial rows of 2100 x 16 tiles in at
    most 16 chains, zero-mean terms: 2e-5 of the norm."""
    B, HW, C, G, g = 2100, 16384, 64, 32, gen(1)
    x, dy = (torch.randn(B, HW, C, generator=g, device="cuda", dtype=BF) for _ in range(2))
    gamma, beta = rnd(g, C, mean=1.0, scale=0.2), rnd(g, C, scale=0.2)
    y, dx, stats = torch.empty_like(x), torch.empty_like(x), torch.empty(2, B, G, device="cuda")
    dg, db = torch.empty_like(gamma), torch.empty_like(gamma)
    ops.gn_act_fwd(x, None, y, G, stats, gamma, beta, act=ops.ACT_SILU)
    ops.gn_act_bwd(dy, x, None, dx, None, G, stats, gamma, beta, dg, db, act=ops.ACT_SILU)
    sums = [torch.zeros(C, dtype=torch.float64, device="cuda") for _ in range(2)]
    for b in range(0, B, 100):
        s = slice(b, b + 100)
        ref = gn_ref(x[s], None, gamma, beta, G, 1e-5, "silu", dy[s])
        sums[0] += ref["dgamma"]
        sums[1] += ref["dbeta"]
        if b in (0, 1000, 2000):
            within(y[s], ref["y"], 128 * U * ref["S"], "y")
            within(dx[s], ref["dx"], 144 * U * ref["Sdx"], "dx")
        del ref
    assert off(dg, sums[0]) < 2e-5 and off(db, sums[1]) < 2e-5


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_group_norm_of_the_most_channels(ops, dtype):  # noqa: F811
    B, HW, C, G, g = 2, 3, 1 << 24, 1 << 21, gen(2)
    x, dy = rnd(g, B, HW, C, dtype=dtype), rnd(g, B, HW, C, dtype=dtype)
    gamma, beta = rnd(g, C, mean=1.0, scale=0.2), rnd(g, C, scale=0.2)
    y, dx, stats = torch.empty_like(x), torch.empty_like(x), torch.empty(2, B, G, device="cuda")
    dg, db = torch.empty_like(gamma), torch.empty_like(gamma)
    ops.gn_act_fwd(x, None, y, G, stats, gamma, beta, act=ops.ACT_GELU)
    ops.gn_act_bwd(dy, x, None, dx, None, G, stats, gamma, beta, dg, db, act=ops.ACT_GELU)
    ref = gn_ref(x, None, gamma, beta, G, 1e-5, "gelu", dy)
    within(y, ref["y"], 128 * U * ref["S"], "y")
    within(dx, ref["dx"], 128 * U * ref["Sdx"], "dx")
    within(dg, ref["dgamma"], 136 * U * ref["Sdgamma"], "dgamma")
    within(db, ref["dbeta"], 136 * U * ref["Sdbeta"], "dbeta")


def test_linear_of_the_most_rows(ops):  # noqa: F811
    """268435392 rows of 8 to 8: x, y and their gradients hold 2^31 elements each.  Sums over rows run in 64 slabs (or 128 blocks
    of 8 lanes) of 262144 additions each: u sqrt(262144 / 6) = 1.3e-5 of the norm, and 9e-6 for dz in two bf16 parts."""
    M, N, K, g = 64 * 0x3fffff, 8, 8, gen(3)
    x, dy = (torch.randn(M, 8, generator=g, device="cuda", dtype=BF) for _ in range(2))
    w, bias = rnd(g, N, K, dtype=BF, scale=1 / math.sqrt(K)), rnd(g, N)
    y, pre, dx = (torch.empty(M, 8, device="cuda", dtype=BF) for _ in range(3))
    dw, db = torch.empty(N, K, device="cuda"), torch.empty(N, device="cuda")
    ops.linear_act_fwd(x, w, y, bias=bias, pre=pre, act=ops.ACT_SILU)
    ops.linear_act_bwd(dy, x, w, pre=pre, dx=dx, dw=dw, dbias=db, act=ops.ACT_SILU)
    rdw, rdb = torch.zeros(N, K, dtype=torch.float64, device="cuda"), torch.zeros(N, dtype=torch.float64, device="cuda")
    step = 1 << 22
    for a in range(0, M, step):
        s = slice(a, a + step)
        xd, gd = x[s].double(), dy[s].double() * act64(pre[s].double(), "silu")[1]
        rdw += gd.t().contiguous() @ xd
        rdb += gd.sum(0)
        if a in (0, 32 * step) or a + step >= M:
            v = xd @ w.double().t().contiguous() + bias.double()
            for got, ref, most in ((pre[s], v, 2.3e-3), (y[s], act64(v, "silu")[0], 2.3e-3), (dx[s], gd @ w.double(), 3.2e-3)):
                assert off(got, ref) < most
                assert off(got[-64:], ref[-64:]) < 2 * most          # (the last rows)
    assert off(dw, rdw) < 3e-5 and off(db, rdb) < 3e-5


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("size", [(5, 8, 2000000), (20, 24, 2000000), (3, 2000000, 8), (33, 2000000, 16)], ids=lambda c: "x".join(map(str, c)))
def test_linear_of_the_widest_rows(ops, dtype, size):  # noqa: F811
    """Rows of two million: element-wise bounds at the ends (places that carry most of a sum), 2-norms for the whole."""
    M, N, K = size
    g = gen(4)
    x, w, dy = rnd(g, M, K, dtype=dtype), rnd(g, N, K, dtype=dtype, scale=1 / math.sqrt(K)), rnd(g, M, N, dtype=dtype)
    x[:, -1], w[:, -1] = 1000.0, 1.0
    dy[:, -1], w[-1, :] = 1000.0, 1.0
    y, dx, dw, db = lin_check(ops, x, w, rnd(g, N), None, dy, "none", F32, "none")
    assert off(dx, dy.double() @ w.double()) < (2.3e-3 if dtype == BF else 2e-6)
    # f32 chains of 2000000 / 64 splits / 2 products an instruction, folded every 256
    assert off(dw, dy.double().t().contiguous() @ x.double()) < 2e-6


@pytest.mark.parametrize("V", [0x7ffffff0, 0x7fffffe9])
def test_distill_of_the_most_classes(ops, V):  # noqa: F811
    """One row of 2^31 - 16 bf16 logits in place, zero but for its ends.  A thread's 262144 vectors are added 64 at a time:
    within 64 of them e^-20 each gets lost beside a spike (64 x 8 x 2e-9), then 4096 + 22 roundings of u / sqrt(3) in the mean
    square, 2.2e-6 together: 1e-5 allowed."""
    logits = torch.zeros(1, V, dtype=BF, device="cuda")
    for i in (0, V - 1):
        logits[0, i] = 20.0
    ti = torch.tensor([[0, V - 1, 5, 1 << 30, V - 9]], dtype=torch.int32, device="cuda")
    tv = torch.tensor([[1.0, 2.0, 0.5, 0.25, 0.125]], device="cuda")
    loss, rl = torch.empty((), device="cuda"), torch.empty(1, device="cuda")
    ops.distill_topk(logits, tv, ti, loss, rl, dlogits=logits, grad_scale=1e6)
    z = V - 2 + 2 * math.exp(20.0)
    p = torch.softmax(tv[0].double(), 0).tolist()
    lq = [20.0 - math.log(z)] * 2 + [-math.log(z)] * 3
    want = sum(q * (math.log(q) - l) for q, l in zip(p, lq))
    assert abs(float(rl) - want) < 1e-5 * want and float(loss) == float(rl)
    rest = 1e6 / z
    for c, q, l in zip(ti[0].tolist(), p, lq):
        g = 1e6 * (math.exp(l) - q)
        assert abs(float(logits[0, c]) - g) < 2.0 ** -8 * abs(g) + 1e-4
        logits[0, c] = rest
    least, most = torch.aminmax(logits)
    assert abs(float(least) - rest) < 2.0 ** -8 * rest and float(most) == float(least)


def test_distill_of_more_than_2_31_logits(ops):  # noqa: F811
    R, V, k, g = 2200000, 1000, 5, gen(5)
    logits = torch.randn(R, V, generator=g, device="cuda", dtype=BF)
    tv, w = rnd(g, R, k), torch.rand(R, generator=g, device="cuda")
    ti = torch.randint(0, V, (R, k), generator=g, device="cuda", dtype=torch.int32)
    loss, rl, dl = torch.empty((), device="cuda"), torch.empty(R, device="cuda"), torch.empty_like(logits)
    ops.distill_topk(logits, tv, ti, loss, rl, dlogits=dl, row_weight=w)
    for s in (slice(0, 500), slice(1100000, 1100500), slice(R - 500, R)):
        rows, Srow, grad, Sgrad = distill_ref(logits[s], tv[s], ti[s], w[s], 1.0, 1.0)
        within(rl[s], rows, 160 * U * Srow, "row_loss")
        within(dl[s], grad, 160 * U * Sgrad, "dlogits")
    # (1024 chains of 2149 sums of one sign, then 6 + 16)
    assert abs(float(loss) - float(rl.double().sum())) < (R / 1024 + 24) * U * float(loss)
    assert bool(torch.isfinite(rl).all())


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("T, scale", [(1e-37, 1e30), (1e-10, 1e8), (50.0, 1.0), (1e4, 1.0), (1e20, 1.0)])
def test_distill_temperatures(ops, dtype, T, scale):  # noqa: F811
    """From one-hot to uniform.  (The loss, T^2 times a difference of logarithms, is compared at the scale of its terms.)"""
    g = gen(6)
    for V in (300, 9001):
        logits, tv, w = rnd(g, 6, V, dtype=dtype, scale=3.0), rnd(g, 6, 7, scale=3.0), torch.ones(6, device="cuda")
        ti = torch.stack([torch.randperm(V, generator=g, device="cuda")[:7] for _ in range(6)]).int()
        logits[2, ::3] = torch.finfo(dtype).min
        logits[3, 1::2] = float("-inf")
        ti[3] = ti[3] // 2 * 2
        loss, rl, dl = torch.empty((), device="cuda"), torch.empty(6, device="cuda"), torch.empty_like(logits)
        ops.distill_topk(logits, tv, ti, loss, rl, dlogits=dl, row_weight=w, temperature=T, grad_scale=scale)
        rows, Srow, grad, Sgrad = distill_ref(logits, tv, ti, w, T, scale)
        within(dl, grad, 160 * U * Sgrad, "dlogits")
        if 1e-15 < T < 1e15:                       # (T^2 of the others leaves the range of f32)
            within(rl, rows, 160 * U * Srow, "row_loss")


def test_workspaces_of_the_call_in_a_graph(ops):  # noqa: F811
    """ws=None inside a capture: the graph's own memory, and the same results at every replay."""
    g = gen(7)
    x, w, dy, pre = rnd(g, 500, 515, dtype=BF), rnd(g, 303, 515, dtype=BF), rnd(g, 500, 303, dtype=BF), rnd(g, 500, 303)
    xg, dyg, gamma, beta = rnd(g, 1, 5000, 64, dtype=BF), rnd(g, 1, 5000, 64, dtype=BF), rnd(g, 64), rnd(g, 64)
    out = [torch.empty_like(dy), torch.empty_like(x), torch.empty(303, 515, device="cuda"), torch.empty(303, device="cuda"),
           torch.empty_like(xg), torch.empty_like(xg), torch.empty(64, device="cuda"), torch.empty(64, device="cuda")]
    stats = torch.empty(2, 1, 8, device="cuda")

    def run():
        ops.linear_act_fwd(x, w, out[0], act=ops.ACT_SILU)
        ops.linear_act_bwd(dy, x, w, pre=pre, dx=out[1], dw=out[2], dbias=out[3], act=ops.ACT_SILU)
        ops.gn_act_fwd(xg, None, out[4], 8, stats, gamma, beta, act=ops.ACT_GELU)
        ops.gn_act_bwd(dyg, xg, None, out[5], None, 8, stats, gamma, beta, out[6], out[7], act=ops.ACT_GELU)
    run()
    want = [t.clone() for t in out]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for rep in range(4):
        for t in out:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, out)), rep
        run()
        assert all(torch.equal(p, q) for p, q in zip(want, out)), rep
