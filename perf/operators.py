"""Workloads of the row operators: group normalisation with an activation, the linear layer with a fused
epilogue, and the distillation loss over a teacher's top logits.

Every case is one call sequence as a training step or a serving call makes it.  With `own` false `run` computes
it from elementary torch operations in 32 bits; with `own` true it calls cvae_gan_amd.ops.  `exact` restates the
definitions in 64 bits."""
import math

import numpy as np
import torch

own = False

GN_EPS = 1e-5
SLOPE = 0.2
BF16, F32 = "bf16", "f32"
DTYPES = {BF16: torch.bfloat16, F32: torch.float32}


# ---- cases ------------------------------------------------------------------------------------------------
def listed():
    return [
        # one 64 x 64 picture in the trunk's first stage at serving time: latency
        gn("gn_one_picture", BF16, 1, 64, 64, 64, 32, "silu", False, False),
        # the second stage of the benchmark's trunk with its skip tensor, forward only
        gn("gn_stage_res", BF16, 256, 32, 32, 128, 32, "lrelu", True, False),
        # the first stage of the benchmark's trunk at the benchmark's batch, forward and backward
        gn("gn_stage_train", BF16, 256, 64, 64, 64, 32, "silu", False, True),
        # a ragged crop in exact f32 with a skip tensor, forward and backward
        gn("gn_crop_train_f32", F32, 3, 37, 53, 72, 9, "silu", True, True),
        # one token through a square projection with its residual stream: the weights are all there is to read
        linear("linear_token", BF16, 1, 4096, 4096, "none", True, False),
        # the generator's second fully connected layer (528 -> 8192) at the reference's training batch
        linear("linear_fc", BF16, 550, 8192, 528, "lrelu", False, False),
        # the encoder's head (8192 -> 128) at the benchmark's batch, in exact f32, forward and backward
        linear("linear_head_train_f32", F32, 256, 128, 8192, "silu", False, True),
        # sizes that fit no tile and rows that start on no 16-byte border; weight gradients in f32
        linear("linear_odd_train", BF16, 777, 1003, 515, "none", True, True),
        # a wide layer of a large network, forward and backward
        linear("linear_wide_train", BF16, 8192, 4096, 4096, "gelu", True, True),
        # the classifier's own size: 100 classes
        distill("distill_classes", F32, 256, 100, 10, 2.0),
        # a student over a mid-sized vocabulary
        distill("distill_mid", BF16, 2048, 32768, 64, 1.0),
        # a long batch of positions over a large vocabulary
        distill("distill_large", BF16, 4096, 131072, 100, 2.0),
    ]


def gn(name, dtype, batch, height, width, channels, groups, act, res, train):
    return {"name": name, "op": "gn", "dtype": dtype, "batch": batch, "height": height, "width": width,
            "channels": channels, "groups": groups, "act": act, "res": res, "train": train}


def linear(name, dtype, rows, n, k, act, res, train):
    return {"name": name, "op": "linear", "dtype": dtype, "rows": rows, "n": n, "k": k, "act": act, "res": res, "train": train}


def distill(name, dtype, rows, classes, top, temperature):
    return {"name": name, "op": "distill", "dtype": dtype, "rows": rows, "classes": classes, "top": top,
            "temperature": temperature}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gn", "linear", "distill"])
    dtype = rng.choice([BF16, BF16, F32])
    if op == "gn":
        per = 8 * rng.randint(1, 4)
        channels = per * _log(rng, 1, 64)
        height, width = _log(rng, 1, 64), _log(rng, 1, 64)
        # any divisor of the channel count is a valid number of groups; a group of a handful of values is normalised
        # almost to signs, whose gradient is what cancellation leaves of it
        groups = rng.choice([g for g in range(1, channels + 1)
                             if channels % g == 0 and channels // g <= 256 and channels // g * height * width >= 16] or [1])
        batch = max(1, min(_log(rng, 1, 256), (1 << 25) // (channels * height * width)))
        train = rng.random() < 0.5
        # the slope of LeakyReLU jumps at zero: a sum that lands a rounding error away from zero takes the other
        # slope, so its backward pass has no value to compare there; forward it is continuous
        act = rng.choice(["silu", "gelu", "none"] if train else ["silu", "gelu", "none", "lrelu"])
        return _unnamed(gn("", dtype, batch, height, width, channels, groups, act, rng.random() < 0.4, train))
    if op == "linear":
        rows, n, k = _log(rng, 1, 8192), _log(rng, 16, 8192), _log(rng, 16, 8192)
        if rng.random() < 0.6:
            n, k = (n + 7) // 8 * 8, (k + 7) // 8 * 8
        if dtype == F32:
            rows = min(rows, 1024)
        rows = max(1, min(rows, (1 << 36) // (n * k)))
        train = rng.random() < 0.5
        act = rng.choice(["silu", "gelu", "none"] if train else ["silu", "gelu", "none", "lrelu"])
        return _unnamed(linear("", dtype, rows, n, k, act, rng.random() < 0.5, train))
    classes = _log(rng, 16, 131072)
    rows = max(1, min(_log(rng, 1, 4096), 260000000 // classes))
    return _unnamed(distill("", dtype, rows, classes, rng.randint(1, min(classes, 128)), rng.choice([1.0, 2.0, 4.0])))


def _unnamed(case):
    del case["name"]
    return case


# ---- inputs -----------------------------------------------------------------------------------------------
def prepare(case, seed):
    return _prepare(case, seed, "cuda")


def _prepare(case, seed, device):
    g = torch.Generator(device=device).manual_seed(int(seed))
    t = DTYPES[case["dtype"]]

    def normal(*shape, mean=0.0, std=1.0, to=t):
        return torch.randn(*shape, generator=g, device=device).mul_(std).add_(mean).to(to)

    s = {"case": case}
    if case["op"] == "gn":
        B, H, W, C = case["batch"], case["height"], case["width"], case["channels"]
        s["x"] = (normal(B, H, W, C, mean=0.3, std=1.5, to=torch.float32) + normal(C, to=torch.float32)).to(t)
        s["gamma"] = normal(C, mean=1.0, std=0.2, to=torch.float32)
        s["beta"] = normal(C, std=0.2, to=torch.float32)
        s["res"] = normal(B, H, W, C) if case["res"] else None
        s["dy"] = normal(B, H, W, C, std=0.1) if case["train"] else None
    elif case["op"] == "linear":
        M, N, K = case["rows"], case["n"], case["k"]
        s["x"] = normal(M, K)
        s["w"] = normal(N, K, std=1.0 / math.sqrt(K))
        s["bias"] = normal(N, std=0.1, to=torch.float32)
        s["res"] = normal(M, N) if case["res"] else None
        s["dy"] = normal(M, N, std=0.1) if case["train"] else None
    else:
        R, V, k = case["rows"], case["classes"], case["top"]
        step = V // k
        j = torch.arange(k, device=device)
        first = torch.randint(0, V, (R, 1), generator=g, device=device)
        s["top_idx"] = ((first + j * step) % V).to(torch.int32)
        top = 8.0 - 6.0 * j / k + normal(R, k, std=0.3, to=torch.float32)
        s["top_val"] = top
        logits = normal(R, V, std=1.5)
        near = (top + normal(R, k, to=torch.float32)).to(t)      # a student that has begun to follow its teacher
        s["logits"] = logits.scatter_(1, s["top_idx"].long(), near)
        # one position in eight is padding
        s["row_weight"] = (torch.rand(R, generator=g, device=device) > 0.125).float()
        s["grad_scale"] = 1.0 / R
    if own:
        _buffers(s)
    return s


def _buffers(s):
    """What a program of this package allocates once: outputs, saved tensors and workspaces."""
    from cvae_gan_amd import ops
    c = s["case"]
    if c["op"] == "gn":
        x = s["x"]
        s["act"] = ops.ACTS[c["act"]]
        s["y"] = torch.empty_like(x)
        s["stats"] = torch.empty(2, c["batch"], c["groups"], device=x.device)
        s["ws"] = ops.gn_act_workspace(x, c["groups"], backward=c["train"])
        if c["train"]:
            s["dx"] = torch.empty_like(x)
            s["dres"] = torch.empty_like(x) if c["res"] else None
            s["dgamma"], s["dbeta"] = torch.empty_like(s["gamma"]), torch.empty_like(s["beta"])
    elif c["op"] == "linear":
        x, w = s["x"], s["w"]
        s["act"] = ops.ACTS[c["act"]]
        s["y"] = torch.empty(c["rows"], c["n"], dtype=x.dtype, device=x.device)
        # f32: the bias gradient, an f32 sum, keeps the digits of the activation's derivative
        s["pre"] = torch.empty_like(s["y"], dtype=torch.float32) if c["train"] and c["act"] != "none" else None
        s["ws"] = ops.linear_act_workspace(x, w, act=s["act"], backward=c["train"])
        if c["train"]:
            s["dx"] = torch.empty_like(x)
            s["dw"] = torch.empty(w.shape, dtype=_dw_dtype(c), device=x.device)
            s["dbias"] = torch.empty_like(s["bias"])
    else:
        s["dlogits"] = torch.empty_like(s["logits"])
        s["row_loss"] = torch.empty(c["rows"], device=s["logits"].device)
        s["loss"] = torch.empty((), device=s["logits"].device)


def _dw_dtype(case):
    # behind an activation the products are taken with the rounded slope-scaled gradient, so the weight gradient
    # has no more digits than the type of the activations; without one it is an f32 sum of exact products
    return torch.float32 if case["act"] == "none" else DTYPES[case["dtype"]]


# ---- one pass ---------------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if own:
        return {"gn": _gn_own, "linear": _linear_own, "distill": _distill_own}[op](s)
    return {"gn": _gn_plain, "linear": _linear_plain, "distill": _distill_plain}[op](s)


def _gn_own(s):
    from cvae_gan_amd import ops
    c = s["case"]
    ops.gn_act_fwd(s["x"], s["res"], s["y"], c["groups"], s["stats"], s["gamma"], s["beta"], eps=GN_EPS, act=s["act"],
                   ws=s["ws"])
    if not c["train"]:
        return {"y": s["y"]}
    ops.gn_act_bwd(s["dy"], s["x"], s["res"], s["dx"], s["dres"], c["groups"], s["stats"], s["gamma"], s["beta"],
                   s["dgamma"], s["dbeta"], act=s["act"], ws=s["ws"])
    out = {"y": s["y"], "dx": s["dx"], "dgamma": s["dgamma"], "dbeta": s["dbeta"]}
    if c["res"]:
        out["dres"] = s["dres"]
    return out


def _linear_own(s):
    from cvae_gan_amd import ops
    ops.linear_act_fwd(s["x"], s["w"], s["y"], bias=s["bias"], res=s["res"], pre=s["pre"], act=s["act"], ws=s["ws"])
    if not s["case"]["train"]:
        return {"y": s["y"]}
    ops.linear_act_bwd(s["dy"], s["x"], s["w"], pre=s["pre"], dx=s["dx"], dw=s["dw"], dbias=s["dbias"], act=s["act"],
                       ws=s["ws"])
    return {"y": s["y"], "dx": s["dx"], "dw": s["dw"], "dbias": s["dbias"]}


def _distill_own(s):
    from cvae_gan_amd import ops
    ops.distill_topk(s["logits"], s["top_val"], s["top_idx"], s["loss"], s["row_loss"], dlogits=s["dlogits"],
                     row_weight=s["row_weight"], temperature=s["case"]["temperature"], grad_scale=s["grad_scale"])
    return {"loss": s["loss"], "row_loss": s["row_loss"], "dlogits": s["dlogits"]}


def _gelu_arg(v):
    # GELU's tanh form, 0.5 v (1 + tanh u), written as v * sigmoid(2 u)
    return 2.0 * 0.7978845608028654 * (v + 0.044715 * v * v * v)


def _sigmoid(v):
    return 1.0 / (1.0 + torch.exp(-v))


def _act(v, act):
    if act == "lrelu":
        return torch.where(v > 0, v, SLOPE * v)
    if act == "silu":
        return v * _sigmoid(v)
    if act == "gelu":
        return v * _sigmoid(_gelu_arg(v))
    return v


def _slope(v, act):
    if act == "lrelu":
        return torch.where(v > 0, torch.ones_like(v), torch.full_like(v, SLOPE))
    if act == "silu":
        p = _sigmoid(v)
        return p * (1.0 + v * (1.0 - p))
    if act == "gelu":
        p = _sigmoid(_gelu_arg(v))
        return p * (1.0 + v * (1.0 - p) * 2.0 * 0.7978845608028654 * (1.0 + 3.0 * 0.044715 * v * v))
    return torch.ones_like(v)


def _gn_plain(s):
    c = s["case"]
    B, C, G = c["batch"], c["channels"], c["groups"]
    n = c["height"] * c["width"]
    t = s["x"].dtype
    x = s["x"].float().reshape(B, n, G, C // G)
    cnt = float(n * (C // G))
    mean = x.sum((1, 3), keepdim=True) / cnt
    d = x - mean
    rstd = 1.0 / torch.sqrt((d * d).sum((1, 3), keepdim=True) / cnt + GN_EPS)
    xhat = d * rstd
    gamma, beta = s["gamma"].reshape(G, -1), s["beta"].reshape(G, -1)
    pre = xhat * gamma + beta
    if c["res"]:
        pre = pre + s["res"].float().reshape(pre.shape)
    out = {"y": _act(pre, c["act"]).reshape(s["x"].shape).to(t)}
    if not c["train"]:
        return out
    g = s["dy"].float().reshape(pre.shape) * _slope(pre, c["act"])
    gg = g * gamma
    a = gg.sum((1, 3), keepdim=True) / cnt
    b = (gg * xhat).sum((1, 3), keepdim=True) / cnt
    out["dx"] = (rstd * (gg - a - xhat * b)).reshape(s["x"].shape).to(t)
    out["dgamma"] = (g * xhat).sum((0, 1)).reshape(C)
    out["dbeta"] = g.sum((0, 1)).reshape(C)
    if c["res"]:
        out["dres"] = g.reshape(s["x"].shape).to(t)
    return out


def _linear_plain(s):
    c = s["case"]
    t = s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    pre = x @ w.t() + s["bias"]
    y = _act(pre, c["act"])
    if c["res"]:
        y = y + s["res"].float()
    out = {"y": y.to(t)}
    if not c["train"]:
        return out
    g = s["dy"].float() * _slope(pre, c["act"])
    out["dx"] = (g @ w).to(t)
    out["dw"] = (g.t() @ x).to(_dw_dtype(c))
    out["dbias"] = g.sum(0)
    return out


def _distill_plain(s):
    c = s["case"]
    T = c["temperature"]
    idx = s["top_idx"].long()
    z = s["logits"].float() / T
    z = z - z.max(1, keepdim=True).values
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    t = s["top_val"] / T
    t = t - t.max(1, keepdim=True).values
    pe = torch.exp(t)
    psum = pe.sum(1, keepdim=True)
    p = pe / psum
    diff = (t - torch.log(psum)) - (z.gather(1, idx) - torch.log(total))
    w = s["row_weight"]
    rows = w * T * T * (p * diff).sum(1)
    grad = e / total
    grad.scatter_add_(1, idx, -p)
    grad *= (w * (T * s["grad_scale"])).unsqueeze(1)
    return {"loss": rows.sum(), "row_loss": rows, "dlogits": grad.to(s["logits"].dtype)}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------
def exact(case, seed):
    s = _prepare(case, seed, "cuda")
    return {"gn": _gn_exact, "linear": _linear_exact, "distill": _distill_exact}[case["op"]](case, s)


def _act_exact(v, act):
    """The activation and its derivative."""
    if act == "none":
        return v, torch.ones_like(v)
    if act == "lrelu":
        up = (v > 0).double()
        k = up + SLOPE * (1 - up)
        return v * k, k
    if act == "silu":
        p = torch.sigmoid(v)
        return v * p, p + v * p * (1 - p)
    c = math.sqrt(2.0 / math.pi)
    th = torch.tanh(c * (v + 0.044715 * v ** 3))
    return 0.5 * v * (1 + th), 0.5 * (1 + th) + 0.5 * v * (1 - th * th) * c * (1 + 3 * 0.044715 * v * v)


def _gn_exact(case, s):
    B, C, G = case["batch"], case["channels"], case["groups"]
    parts = {k: [] for k in ("y", "dx", "dres")}
    dgamma = torch.zeros(C, dtype=torch.float64, device=s["x"].device)
    dbeta = torch.zeros_like(dgamma)
    gamma, beta = s["gamma"].double(), s["beta"].double()
    per = max(1, (1 << 24) // (s["x"].numel() // B))
    for b in range(0, B, per):                       # a few samples at a time
        x = s["x"][b:b + per].double().flatten(1, 2)
        nb, n = x.shape[:2]
        by_group = x.view(nb, n, G, C // G).permute(0, 2, 1, 3).flatten(2)
        mean = by_group.mean(2)
        var = by_group.var(2, unbiased=False)
        widen = lambda v: v.repeat_interleave(C // G, dim=1).unsqueeze(1)   # noqa: E731
        r = widen(1.0 / torch.sqrt(var + GN_EPS))
        xhat = (x - widen(mean)) * r
        pre = xhat * gamma + beta
        if case["res"]:
            pre = pre + s["res"][b:b + per].double().flatten(1, 2)
        y, k = _act_exact(pre, case["act"])
        parts["y"].append(y.view(s["x"][b:b + per].shape))
        if case["train"]:
            g = s["dy"][b:b + per].double().flatten(1, 2) * k
            dgamma += (g * xhat).sum((0, 1))
            dbeta += g.sum((0, 1))
            gg = g * gamma
            mean_of = lambda v: widen(v.view(nb, n, G, C // G).mean((1, 3)))   # noqa: E731
            dx = r * (gg - mean_of(gg) - xhat * mean_of(gg * xhat))
            parts["dx"].append(dx.view(s["x"][b:b + per].shape))
            if case["res"]:
                parts["dres"].append(g.view(s["x"][b:b + per].shape))
    out = {"y": torch.cat(parts["y"])}
    if case["train"]:
        out.update(dx=torch.cat(parts["dx"]), dgamma=dgamma, dbeta=dbeta)
        if case["res"]:
            out["dres"] = torch.cat(parts["dres"])
    return out


def _linear_exact(case, s):
    x, w = s["x"].double(), s["w"].double()
    v, k = _act_exact(torch.addmm(s["bias"].double(), x, w.t()), case["act"])
    out = {"y": v + s["res"].double() if case["res"] else v}
    if case["train"]:
        g = s["dy"].double() * k
        out.update(dx=torch.mm(g, w), dw=torch.mm(g.t(), x), dbias=g.sum(0))
    return out


def _distill_exact(case, s):
    T = float(case["temperature"])
    R = case["rows"]
    loss_rows = []
    grads = []
    per = max(1, (1 << 26) // case["classes"])
    for r in range(0, R, per):
        z = s["logits"][r:r + per].double() / T
        logq = z - torch.logsumexp(z, 1, keepdim=True)
        logp = torch.log_softmax(s["top_val"][r:r + per].double() / T, 1)
        p = logp.exp()
        idx = s["top_idx"][r:r + per].long()
        w = s["row_weight"][r:r + per].double()
        loss_rows.append(w * T * T * (p * (logp - logq.gather(1, idx))).sum(1))
        q = logq.exp()
        q.scatter_add_(1, idx, -p)
        grads.append(q * (w * T * s["grad_scale"]).unsqueeze(1))
    rows = torch.cat(loss_rows)
    return {"loss": rows.sum(), "row_loss": rows, "dlogits": torch.cat(grads)}


# ---- what a pass cannot do without ------------------------------------------------------------------------
def work(case):
    es = 2 if case["dtype"] == BF16 else 4
    if case["op"] == "gn":
        n = case["batch"] * case["height"] * case["width"] * case["channels"]
        tensors = 2 + (1 if case["res"] else 0)                                  # x, y, res
        flops = 10 * n
        if case["train"]:
            tensors += 2 + (1 if case["res"] else 0)                             # dy, dx, dres
            flops += 25 * n
        return {"bytes": n * tensors * es + 16 * case["channels"], "flops": flops}
    if case["op"] == "linear":
        M, N, K = case["rows"], case["n"], case["k"]
        size = (M * K + N * K + M * N * (2 if case["res"] else 1)) * es + 4 * N
        flops = 2 * M * N * K
        if case["train"]:
            size += (M * N + M * K) * es + N * K * (4 if case["act"] == "none" else es) + 4 * N
            flops *= 3
        return {"bytes": size, "flops": flops}
    R, V, k = case["rows"], case["classes"], case["top"]
    return {"bytes": 2 * R * V * es + R * k * 8 + 8 * R, "flops": 8 * R * V}


if __name__ == "__main__":
    for case in listed():
        w = work(case)
        print("%-24s %9.3f MB %12.4f GFLOP" % (case["name"], w["bytes"] / 1e6, w["flops"] / 1e9))
    print("%.2f GB in all" % np.sum([work(c)["bytes"] / 1e9 for c in listed()]))
