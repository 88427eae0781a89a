"""Thin torch-tensor wrappers over the C ABI (include/cvaegan.h).

torch supplies device memory and the current HIP stream; every function here
enqueues exactly the kernels of one C entry point on that stream."""
import ctypes as C

import torch

from ._lib import lib, check, ConvDesc, WMap, PackJob, CvgError, F32, BF16, PAD_ZERO, PAD_REFLECT  # noqa: F401
from ._lib import GnDesc, LinearDesc, DistillDesc, ACT_NONE, ACT_LRELU, ACT_SILU, ACT_GELU  # noqa: F401

_DT = {torch.float32: F32, torch.bfloat16: BF16}
ACTS = {"none": ACT_NONE, "lrelu": ACT_LRELU, "silu": ACT_SILU, "gelu": ACT_GELU}


def dt(t_or_dtype):
    d = t_or_dtype.dtype if isinstance(t_or_dtype, torch.Tensor) else t_or_dtype
    return _DT[d]


def ptr(t):
    if t is None:
        return None
    assert t.is_cuda, "cvae_gan_amd ops need device tensors"
    return t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


def elt(dtype):
    return 2 if dtype == torch.bfloat16 else 4


def conv_fwd(desc, x, w, y, bias=None, cbias=None, labels=None, res=None, gate=None, ws=None):
    check(lib.cvg_conv_fwd(C.byref(desc), ptr(x), ptr(w), ptr(y), ptr(bias), ptr(cbias), ptr(labels),
                           ptr(res), ptr(gate), ptr(ws), ws.numel() * ws.element_size() if ws is not None else 0,
                           stream()))


def conv_fwd_workspace(desc):
    return int(lib.cvg_conv_fwd_workspace(C.byref(desc)))


def conv_wgrad(desc, x, dy, dy_ld, wmap, grad, ws, accumulate=False):
    check(lib.cvg_conv_wgrad(C.byref(desc), ptr(x), ptr(dy), dy_ld, C.byref(wmap), ptr(grad), int(accumulate),
                             ptr(ws), ws.numel() * ws.element_size(), stream()))


class ConvGroup:
    """Up to four convolutions of one input over one output grid, launched together."""

    def __init__(self, descs, weights):
        assert 1 <= len(descs) <= 4 and len(descs) == len(weights)
        self.n = len(descs)
        self.descs = (ConvDesc * self.n)(*descs)
        self.w = (C.c_void_p * self.n)(*[ptr(w) for w in weights])
        self._keep = weights

    def run(self, x, y, gate=None):
        """gate (laid out as y): y = conv * LeakyReLU'(gate)."""
        check(lib.cvg_conv_fwd_group(self.n, self.descs, ptr(x), self.w, ptr(y), ptr(gate), stream()))


def conv_wgrad_workspace(desc):
    return int(lib.cvg_conv_wgrad_workspace(C.byref(desc)))


def conv_fwd_kernel(desc):
    """Name of the kernel family the library picks for this descriptor."""
    return lib.cvg_conv_fwd_kernel(C.byref(desc)).decode()


def conv_wgrad_kernel(desc):
    return lib.cvg_conv_wgrad_kernel(C.byref(desc)).decode()


def conv_wgrad_strided(desc, x, dy, wmap, grad, ws, accumulate=False):
    """dy addressed through desc.y_*_pitch (see include/cvaegan.h)."""
    check(lib.cvg_conv_wgrad_strided(C.byref(desc), ptr(x), ptr(dy), C.byref(wmap), ptr(grad), int(accumulate),
                                     ptr(ws), ws.numel() * ws.element_size(), stream()))


def weight_pack(desc, wmap, canonical, packed):
    assert packed.numel() >= desc.w_rows * desc.w_ld and dt(packed) == desc.dtype
    check(lib.cvg_weight_pack(C.byref(desc), C.byref(wmap), ptr(canonical), ptr(packed), stream()))


class PackBatch:
    """Every packed-weight layout of a network, repacked by one launch.
    items: (desc, wmap, canonical f32 tensor, packed tensor); the tensors must stay alive and in place."""

    def __init__(self, items, device):
        jobs = (PackJob * len(items))()
        blocks = 0
        for i, (desc, wmap, canonical, packed) in enumerate(items):
            assert packed.numel() >= desc.w_rows * desc.w_ld and dt(packed) == desc.dtype
            nb = lib.cvg_weight_pack_job(C.byref(desc), C.byref(wmap), ptr(canonical), ptr(packed), blocks,
                                         C.byref(jobs[i]))
            if nb < 0:
                raise CvgError(lib.cvg_last_error().decode())
            blocks += nb
        self.n_jobs, self.blocks = len(items), blocks
        raw = torch.frombuffer(bytearray(bytes(jobs)), dtype=torch.uint8)
        self.table = raw.to(device)
        self._keep = items

    def run(self):
        check(lib.cvg_weight_pack_batch(ptr(self.table), self.n_jobs, self.blocks, stream()))


def label_bias(w_stem, cbias, cout, y_dim):
    check(lib.cvg_label_bias(ptr(w_stem), ptr(cbias), cout, y_dim, stream()))


def label_bias_bwd(dy, labels, B, pixels, cout, y_dim, dw, dbias, ws):
    check(lib.cvg_label_bias_bwd(ptr(dy), dt(dy), ptr(labels), B, pixels, cout, y_dim, ptr(dw), ptr(dbias),
                                 ptr(ws), stream()))


def pack_image(x, xpad, B, P):
    check(lib.cvg_pack_image(ptr(x), ptr(xpad), B, P, dt(xpad), stream()))


def bn_stats_blocks(M, C_):
    return int(lib.cvg_bn_stats_blocks(M, C_))


def bn_stats(x, M, C_, stats, running_mean, running_var, nbt, ws):
    check(lib.cvg_bn_stats(ptr(x), dt(x), M, C_, ptr(stats), ptr(running_mean), ptr(running_var), ptr(nbt),
                           ptr(ws), stream()))


def conv_stats_partials(desc):
    """Partial rows cvg_conv_fwd_stats writes for this layer (0: the layer runs on the gather kernel)."""
    return int(lib.cvg_conv_stats_partials(C.byref(desc)))


def conv_fwd_stats(desc, x, w, y, partials, bias=None, cbias=None, labels=None):
    check(lib.cvg_conv_fwd_stats(C.byref(desc), ptr(x), ptr(w), ptr(y), ptr(bias), ptr(cbias), ptr(labels),
                                 ptr(partials), stream()))


def bn_stats_finalize(partials, nblk, M, C_, stats, running_mean, running_var, nbt):
    check(lib.cvg_bn_stats_finalize(ptr(partials), nblk, M, C_, ptr(stats), ptr(running_mean), ptr(running_var),
                                    ptr(nbt), stream()))


def bn_stats_static(x, M, C_, stats, running_mean, running_var, nbt):
    """bn_stats without a workspace: the partials go to a static array inside the library (C <= 1024)."""
    check(lib.cvg_bn_stats_static(ptr(x), dt(x), M, C_, ptr(stats), ptr(running_mean), ptr(running_var), ptr(nbt), stream()))


def bn_eval_stats(rm, rv, C_, stats):
    check(lib.cvg_bn_eval_stats(ptr(rm), ptr(rv), C_, ptr(stats), stream()))


def bn_act_fwd(x, res, y, M, C_, stats, gamma, beta):
    check(lib.cvg_bn_act_fwd(ptr(x), ptr(res), ptr(y), dt(x), M, C_, ptr(stats), ptr(gamma), ptr(beta), stream()))


def bn_act_bwd(dy, y, x, dx, M, C_, stats, gamma, dgamma, dbeta, ws, beta=None):
    """y=None with beta: the activation's sign is recomputed from x instead of read from y;
    y=None without beta: dy already carries the activation's derivative."""
    check(lib.cvg_bn_act_bwd(ptr(dy), ptr(y), ptr(x), ptr(dx), dt(x), M, C_, ptr(stats), ptr(gamma), ptr(beta),
                             ptr(dgamma), ptr(dbeta), ptr(ws), stream()))


def colsum(x, M, C_, ld, out, ws, map_d=1, map_a=1, map_b=0):
    check(lib.cvg_colsum(ptr(x), dt(x), M, C_, ld, ptr(out), map_d, map_a, map_b, ptr(ws), stream()))


def permute_f32(src, out, n, d=1, a=1, b=0):
    check(lib.cvg_permute_f32(ptr(src), ptr(out), n, d, a, b, stream()))


def reparam_kl_fwd(h, eps, labels, B, z, y_dim, zin_ld, zin, z_mean, z_sigma, kl, batch_size, h_ld=None):
    """h_ld: row pitch of h (default: its second dimension)."""
    h_ld = h.shape[-1] if h_ld is None else h_ld
    check(lib.cvg_reparam_kl_fwd(ptr(h), dt(h), h_ld, ptr(eps), ptr(labels), B, z, y_dim, zin_ld, ptr(zin),
                                 ptr(z_mean), ptr(z_sigma), ptr(kl), float(batch_size), stream()))


def reparam_kl_bwd(dzin, zin_ld, eps, z_mean, z_sigma, g_mean, g_sigma, kl_scale, batch_size, B, z, dh, h_ld=None):
    h_ld = dh.shape[-1] if h_ld is None else h_ld
    check(lib.cvg_reparam_kl_bwd(ptr(dzin), dt(dzin), zin_ld, ptr(eps), ptr(z_mean), ptr(z_sigma), ptr(g_mean),
                                 ptr(g_sigma), float(kl_scale), float(batch_size), B, z, ptr(dh), h_ld, stream()))


def labels_prepare(labels, out, n, n_class, bad):
    check(lib.cvg_labels_prepare(ptr(labels), ptr(out), n, n_class, ptr(bad), stream()))


def lrelu_dropout_fwd(x, mask, y, n):
    check(lib.cvg_lrelu_dropout_fwd(ptr(x), ptr(mask), ptr(y), dt(x), n, stream()))


def lrelu_dropout_bwd(dy, y, mask, dx, n):
    check(lib.cvg_lrelu_dropout_bwd(ptr(dy), ptr(y), ptr(mask), ptr(dx), dt(y), n, stream()))


def dropout_mask(mask, n, seed):
    check(lib.cvg_dropout_mask(ptr(mask), n, seed, stream()))


def upsample_pad_fwd(x, u, B, h, w, C_):
    check(lib.cvg_upsample_pad_fwd(ptr(x), ptr(u), dt(x), B, h, w, C_, stream()))


def upsample_pad_bwd(du, dx, B, h, w, C_):
    check(lib.cvg_upsample_pad_bwd(ptr(du), ptr(dx), dt(du), B, h, w, C_, stream()))


def upsample_taps_fwd(v, bias, y, B, h, w, N):
    """y [B][2h][2w][N] = bias + the up-sampling / padding / tap-shift operator applied to v [B][h][w][9][N]."""
    check(lib.cvg_upsample_taps_fwd(ptr(v), ptr(bias), ptr(y), dt(v), B, h, w, N, stream()))


def upsample_taps_bwd(dy, z, B, h, w, N):
    """z [B][h][w][9][N] = the nine tap-shifted transposed up-samplings of dy [B][2h][2w][N]."""
    check(lib.cvg_upsample_taps_bwd(ptr(dy), ptr(z), dt(dy), B, h, w, N, stream()))


def reflect_fold(dxp, dx, B, H, W, C_, pad):
    check(lib.cvg_reflect_fold(ptr(dxp), ptr(dx), dt(dxp), B, H, W, C_, pad, stream()))


def tanh_fwd(pre, dec, B, P):
    check(lib.cvg_tanh_fwd(ptr(pre), ptr(dec), dt(pre), B, P, stream()))


def image_u8_to_f32(hwc_u8, nchw_f32, B, P):
    assert hwc_u8.dtype == torch.uint8 and nchw_f32.dtype == torch.float32
    check(lib.cvg_image_u8_to_f32(ptr(hwc_u8), ptr(nchw_f32), B, P, stream()))


def mfma_rate_probe(out, workgroups, iters):
    """Measurement aid: a pure MFMA loop (see cvg_mfma_rate_probe); returns the FLOPs it executes."""
    assert out.dtype == torch.float32 and out.numel() >= workgroups * 256
    check(lib.cvg_mfma_rate_probe(ptr(out), workgroups, iters, stream()))
    return workgroups * 4 * iters * 32 * 32768


def window_col_sum(v, out, B, rows, P):
    check(lib.cvg_window_col_sum(ptr(v), ptr(out), dt(v), B, rows, P, stream()))


def tail_sum_tanh(v, bias, pre, dec, B, P):
    check(lib.cvg_tail_sum_tanh(ptr(v), ptr(bias), ptr(pre), ptr(dec), dt(v), B, P, stream()))


def tanh_bwd(d_dec, dec, dpre, B, P, dpre_win=None):
    check(lib.cvg_tanh_bwd(ptr(d_dec), ptr(dec), ptr(dpre), ptr(dpre_win),
                           dt(dpre), B, P, stream()))


def mse_fwd_bwd(dec, x, d_dec, ll, numel, batch_size, scale, ws):
    check(lib.cvg_mse_fwd_bwd(ptr(dec), ptr(x), ptr(d_dec), ptr(ll), numel, float(batch_size), float(scale),
                              ptr(ws), stream()))


def adamw(p, g, m, v, n, lr, beta1, beta2, eps, wd, step):
    check(lib.cvg_adamw(ptr(p), ptr(g), ptr(m), ptr(v), n, lr, beta1, beta2, eps, wd, step, stream()))


def adamw_dev(p, g, m, v, n, lr, beta1, beta2, eps, wd, step_counter, bc):
    check(lib.cvg_adamw_dev(ptr(p), ptr(g), ptr(m), ptr(v), n, lr, beta1, beta2, eps, wd, ptr(step_counter),
                            ptr(bc), stream()))


def dropout_mask_dev(mask, n, seed_counter):
    check(lib.cvg_dropout_mask_dev(ptr(mask), n, ptr(seed_counter), stream()))


def cast(src, out, n):
    check(lib.cvg_cast(ptr(src), dt(src), ptr(out), dt(out), n, stream()))


def nhwc_to_nchw(src, out, B, HW, C_, ld):
    check(lib.cvg_nhwc_to_nchw(ptr(src), dt(src), ptr(out), B, HW, C_, ld, stream()))


def nchw_to_nhwc(src, out, B, HW, C_, ld):
    check(lib.cvg_nchw_to_nhwc(ptr(src), ptr(out), dt(out), B, HW, C_, ld, stream()))


# ---- adversarial extension (discriminator / classifier heads and losses) -------------------
def gan_d_head(h, ld, w, b, M, F, n_real, grad_scale, dw, db, loss, dh, ws):
    check(lib.cvg_gan_d_head(ptr(h), dt(h), ld, ptr(w), ptr(b), M, F, n_real, grad_scale, ptr(dw), ptr(db), ptr(loss),
                             ptr(dh), ptr(ws), stream()))


def gan_c_head(h, ld, W, b, labels, M, F, y, n_real, grad_scale, dW, db, loss, dh, ws):
    check(lib.cvg_gan_c_head(ptr(h), dt(h), ld, ptr(W), ptr(b), ptr(labels), M, F, y, n_real, grad_scale, ptr(dW),
                             ptr(db), ptr(loss), ptr(dh), ptr(ws), stream()))


def gan_feature_match(h, ld, M, F, r0, r1, f0, f1, grad_scale, loss, dh):
    check(lib.cvg_gan_feature_match(ptr(h), dt(h), ld, M, F, r0, r1, f0, f1, grad_scale, ptr(loss), ptr(dh), stream()))


def gan_class_feature_match(h, ld, F, labels_real, labels_fake, r0, r1, f0, f1, n_class, centres, seen, momentum,
                            grad_scale, loss, dh, ws):
    check(lib.cvg_gan_class_feature_match(ptr(h), dt(h), ld, F, ptr(labels_real), ptr(labels_fake), r0, r1, f0, f1, n_class,
                                          ptr(centres), ptr(seen), momentum, grad_scale, ptr(loss), ptr(dh), ptr(ws),
                                          stream()))


def gan_pair_feature_match(h, ld, F, r0, f0, n, grad_scale, loss, dh, ws):
    check(lib.cvg_gan_pair_feature_match(ptr(h), dt(h), ld, F, r0, f0, n, grad_scale, ptr(loss), ptr(dh), ptr(ws), stream()))


def axpy(y, x, alpha, n=None):
    """y += alpha * x (f32)."""
    assert y.dtype == torch.float32 and x.dtype == torch.float32
    check(lib.cvg_axpy_f32(ptr(y), ptr(x), alpha, y.numel() if n is None else n, stream()))


# ---- inference: eval-mode BatchNorm + LeakyReLU in the convolution's epilogue ----------------
def bn_eval_scale_shift(rm, rv, gamma, beta, C_, scale, shift):
    check(lib.cvg_bn_eval_scale_shift(ptr(rm), ptr(rv), ptr(gamma), ptr(beta), C_, ptr(scale), ptr(shift), stream()))


def conv_bn_act_fwd(desc, x, w, y, scale, shift, bias=None, cbias=None, labels=None, res=None):
    check(lib.cvg_conv_bn_act_fwd(C.byref(desc), ptr(x), ptr(w), ptr(y), ptr(bias), ptr(cbias), ptr(labels),
                                  ptr(scale), ptr(shift), ptr(res), stream()))


# ---- group normalisation, fused linear layers, distillation ---------------------------------
# Sizes and pitches come from the tensors; shapes, types, strides and devices are checked before anything is
# launched (CvgError).  Kernels run on the current stream of the tensors' device.  A workspace is scratch for one call:
# it may be reused by the next call on the same stream, calls that may overlap need their own; ws=None allocates one.
def _need(ok, fmt, *args):
    if not ok:
        raise CvgError(fmt % args)


def _sizes(*sizes):
    """Sizes on their way into a descriptor's 32-bit fields, which would keep the low half of a larger number."""
    for n in sizes:
        if not 0 <= n < 2 ** 31:
            raise CvgError("size %d does not fit the kernels' 32 bits" % n)
    return sizes


def _is(name, t, shape, dtype, device):
    """t (when given) has this shape, type and device."""
    if t is None or (t.shape == shape and t.dtype == dtype and t.device == device):
        return
    _need(tuple(t.shape) == tuple(shape), "%s has shape %s, expected %s", name, tuple(t.shape), tuple(shape))
    _need(t.dtype == dtype, "%s is %s, expected %s", name, t.dtype, dtype)
    _need(False, "%s is on %s, the other operands on %s", name, t.device, device)


def _vec(name, t, shape, device):
    """A dense f32 tensor."""
    _is(name, t, shape, torch.float32, device)
    if t is not None and not t.is_contiguous():
        raise CvgError("%s has to be contiguous" % name)


def _pitch(name, t):
    """Distance in elements between consecutive rows of the last dimension; all leading dimensions have to
    enumerate rows at that one distance."""
    if t is None or t.is_contiguous():
        return 0
    if t.numel() == 0:
        return 0
    width = t.shape[-1]
    _need(width == 1 or t.stride(-1) == 1, "%s: the elements of a row have to be consecutive", name)
    pitch, span = None, 1
    for n, st in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if n == 1:
            continue
        if pitch is None:
            pitch = st
        _need(st == pitch * span, "%s: strides %s do not put the rows at one pitch", name, t.stride())
        span *= n
    if pitch is None:
        return 0
    _need(pitch >= width, "%s: rows of %d elements overlap at pitch %d", name, width, pitch)
    _need(pitch < 2 ** 31, "%s: pitch %d", name, pitch)
    return pitch


def _launch(fn, dev, *args):
    if dev.type != "cuda":
        raise CvgError("cvae_gan_amd ops need device tensors")
    if dev.index == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    if rc != 0:
        check(rc)


def _p(t):
    return None if t is None else t.data_ptr()


def _bytes(n, device):
    return torch.empty(n, dtype=torch.uint8, device=device)


def _nbytes(t):
    return 0 if t is None else t.numel() * t.element_size()


def _scratch(ws, query, d, backward, device):
    if ws is None:
        n = int(query(C.byref(d), backward))
        return _bytes(n, device) if n else None
    if ws.device != device or not ws.is_contiguous():
        raise CvgError("the workspace has to be contiguous on %s" % device)
    return ws


_ACT_VALUES = frozenset(ACTS.values())


def _gn_desc(x, G, act, eps=0.0):
    shape = x.shape
    _need(len(shape) >= 2 and x.dtype in _DT, "x has to be [B, ..., C] in float32 or bfloat16")
    hw = 1
    for n in shape[1:-1]:
        hw *= n
    _need(act in _ACT_VALUES, "activation %r", act)
    _need(G == int(G), "%r groups", G)
    return GnDesc(_DT[x.dtype], *_sizes(shape[0], hw, shape[-1], int(G)), act, 0, 0, 0, 0, 0, eps)


def gn_act_workspace(x, G, backward=False):
    """Workspace (a uint8 tensor) for gn_act_fwd on tensors like x, with backward also for gn_act_bwd."""
    return _bytes(int(lib.cvg_gn_act_workspace(C.byref(_gn_desc(x, G, ACT_NONE)), int(backward))), x.device)


def gn_act_fwd(x, res, y, G, stats, gamma, beta, eps=1e-5, act=ACT_LRELU, ws=None):
    """y = act(groupnorm(x) * gamma + beta [+ res]); x, res, y [B, ..., C] channels last, stats f32 [2, B, G] (mean,
    1 / std; None: not kept), gamma / beta f32 [C]."""
    d = _gn_desc(x, G, act, eps)
    dev, c = x.device, (d.C,)
    _is("res", res, x.shape, x.dtype, dev)
    _is("y", y, x.shape, x.dtype, dev)
    _vec("gamma", gamma, c, dev)
    _vec("beta", beta, c, dev)
    _vec("stats", stats, (2, d.B, d.G), dev)
    d.x_ld, d.res_ld, d.y_ld = _pitch("x", x), _pitch("res", res), _pitch("y", y)
    ws = _scratch(ws, lib.cvg_gn_act_workspace, d, 0, dev)
    _launch(lib.cvg_gn_act_fwd, dev, C.byref(d), _p(x), _p(res), _p(y), _p(stats), _p(gamma), _p(beta), _p(ws), _nbytes(ws))


def gn_act_bwd(dy, x, res, dx, dres, G, stats, gamma, beta, dgamma, dbeta, act=ACT_LRELU, ws=None):
    """Gradients of gn_act_fwd: res as in the forward call, stats from it; dres may be None."""
    d = _gn_desc(x, G, act)
    dev, c = x.device, (d.C,)
    for n, t in (("dy", dy), ("res", res), ("dx", dx), ("dres", dres)):
        _is(n, t, x.shape, x.dtype, dev)
    for n, t in (("gamma", gamma), ("beta", beta), ("dgamma", dgamma), ("dbeta", dbeta)):
        _vec(n, t, c, dev)
    _vec("stats", stats, (2, d.B, d.G), dev)
    d.x_ld, d.res_ld, d.y_ld = _pitch("x", x), _pitch("res", res), _pitch("dy", dy)
    d.dx_ld, d.dres_ld = _pitch("dx", dx), _pitch("dres", dres)
    ws = _scratch(ws, lib.cvg_gn_act_workspace, d, 1, dev)
    _launch(lib.cvg_gn_act_bwd, dev, C.byref(d), _p(dy), _p(x), _p(res), _p(dx), _p(dres), _p(stats), _p(gamma), _p(beta),
            _p(dgamma), _p(dbeta), _p(ws), _nbytes(ws))


def _linear_desc(x, w, act):
    _need(x.dim() >= 1 and w.dim() == 2 and x.dtype in _DT, "x has to be [..., K] and w [N, K], in float32 or bfloat16")
    N, K = w.shape
    _is("w", w, (N, x.shape[-1]), x.dtype, x.device)
    _need(act in _ACT_VALUES, "activation %r", act)
    m = 1
    for n in x.shape[:-1]:
        m *= n
    return LinearDesc(_DT[x.dtype], *_sizes(m, N, K), act, F32, F32, _pitch("x", x), _pitch("w", w))


def _pre(d, pre, x, shape):
    if pre is not None:
        _need(pre.dtype == torch.float32 or pre.dtype == x.dtype, "pre is %s", pre.dtype)
        _is("pre", pre, shape, pre.dtype, x.device)
        d.pre_dtype = _DT[pre.dtype]
        d.pre_ld = _pitch("pre", pre)


def linear_act_workspace(x, w, act=ACT_NONE, backward=False):
    """Workspace (a uint8 tensor) for linear_act_fwd on these operands, with backward also for linear_act_bwd (whatever
    the activation and the type of dw)."""
    d = _linear_desc(x, w, ACT_SILU if backward else act)
    return _bytes(int(lib.cvg_linear_act_workspace(C.byref(d), int(backward))), x.device)


def linear_act_fwd(x, w, y, bias=None, res=None, pre=None, act=ACT_NONE, ws=None):
    """y = act(x @ w.T + bias) + res; x [..., K], w [N, K], y / res / pre [..., N], bias f32 [N].  pre (float32
    or x's type) receives the activation's argument for linear_act_bwd."""
    d = _linear_desc(x, w, act)
    dev, out = x.device, x.shape[:-1] + (d.N,)
    _is("y", y, out, x.dtype, dev)
    _is("res", res, out, x.dtype, dev)
    _pre(d, pre, x, out)
    _vec("bias", bias, (d.N,), dev)
    d.y_ld, d.res_ld = _pitch("y", y), _pitch("res", res)
    ws = _scratch(ws, lib.cvg_linear_act_workspace, d, 0, dev)
    _launch(lib.cvg_linear_act_fwd, dev, C.byref(d), _p(x), _p(w), _p(bias), _p(res), _p(y), _p(pre), _p(ws), _nbytes(ws))


def linear_act_bwd(dy, x, w, pre=None, dx=None, dw=None, dbias=None, act=ACT_NONE, ws=None):
    """Gradients of linear_act_fwd, each optional: dx like x, dw [N, K] (float32 or x's type), dbias f32 [N].  An
    activation needs the pre of the forward call; the gradient of res is dy itself.  dx and a bfloat16 dw are taken with
    dy act'(pre) rounded to bfloat16, a float32 dw with 16 bits of it (at twice the time of that product)."""
    d = _linear_desc(x, w, act)
    dev, out = x.device, x.shape[:-1] + (d.N,)
    _is("dy", dy, out, x.dtype, dev)
    _pre(d, pre, x, out)
    _is("dx", dx, x.shape, x.dtype, dev)
    if dw is not None:
        _need(dw.dtype == torch.float32 or dw.dtype == x.dtype, "dw is %s", dw.dtype)
        _is("dw", dw, w.shape, dw.dtype, dev)
        d.dw_dtype = _DT[dw.dtype]
    _vec("dbias", dbias, (d.N,), dev)
    d.dy_ld, d.dx_ld, d.dw_ld = _pitch("dy", dy), _pitch("dx", dx), _pitch("dw", dw)
    ws = _scratch(ws, lib.cvg_linear_act_workspace, d, 1, dev)
    _launch(lib.cvg_linear_act_bwd, dev, C.byref(d), _p(dy), _p(x), _p(w), _p(pre), _p(dx), _p(dw), _p(dbias), _p(ws),
            _nbytes(ws))


def distill_topk(logits, top_val, top_idx, loss, row_loss, dlogits=None, row_weight=None, temperature=1.0, grad_scale=1.0):
    """Distillation loss against a teacher's top logits, and its gradient: logits [..., V], top_val f32 / top_idx int32
    [..., top], row_loss / row_weight f32 [...], loss f32 scalar (one element); dlogits like logits (or logits itself)."""
    _need(logits.dim() >= 1 and logits.dtype in _DT, "logits have to be [..., V] in float32 or bfloat16")
    _need(top_val.dim() >= 1, "top_val has to be [..., top]")
    rows, dev, top = logits.shape[:-1], logits.device, top_val.shape[-1]
    r = 1
    for n in rows:
        r *= n
    _is("top_val", top_val, rows + (top,), torch.float32, dev)
    _is("top_idx", top_idx, rows + (top,), torch.int32, dev)
    _vec("row_loss", row_loss, rows, dev)
    _vec("row_weight", row_weight, rows, dev)
    _is("dlogits", dlogits, logits.shape, logits.dtype, dev)
    _need(loss.numel() == 1 and loss.dtype == torch.float32 and loss.device == dev, "loss has to be one float32 on %s", dev)
    top_ld = _pitch("top_val", top_val)
    _need((top_ld or top) == (_pitch("top_idx", top_idx) or top), "top_val and top_idx have to share their strides")
    d = DistillDesc(_DT[logits.dtype], *_sizes(r, logits.shape[-1], top), _pitch("logits", logits), _pitch("dlogits", dlogits), top_ld,
                    float(temperature), float(grad_scale))
    _launch(lib.cvg_distill_topk, dev, C.byref(d), _p(logits), _p(top_val), _p(top_idx), _p(row_weight), _p(loss),
            _p(row_loss), _p(dlogits))
