"""Tensor-level wrappers over include/nfe_dense.h (mapping network, modulated convs, resize, layouts).
Activations are NHWC fp32 between layers."""
import ctypes

import torch

from . import _lib
from .ops import _dev, _on, _ptr, _stream

MATH = {None: _lib.NFE_CONV_BF16X3, "bf16x3": _lib.NFE_CONV_BF16X3, "bf16": _lib.NFE_CONV_BF16, "fp16": _lib.NFE_CONV_F16,
        _lib.NFE_CONV_BF16X3: _lib.NFE_CONV_BF16X3, _lib.NFE_CONV_BF16: _lib.NFE_CONV_BF16, _lib.NFE_CONV_F16: _lib.NFE_CONV_F16}


def _call(dev, rc_fn, what):
    with _on(dev.index):
        _lib.check(rc_fn(), what)


def nchw_to_nhwc(x):
    lib = _lib.load()
    x = _dev(x, "x", (None, None, None, None))
    N, C, H, W = x.shape
    out = torch.empty(N, H, W, C, dtype=torch.float32, device=x.device)
    _call(x.device, lambda: lib.nfe_nchw_to_nhwc(_ptr(x), N, C, H, W, _ptr(out), _stream()), "nfe_nchw_to_nhwc")
    return out


def nhwc_to_nchw(x):
    if x.requires_grad and torch.is_grad_enabled():      # part of an autograd graph (plane editing): a view keeps it differentiable
        return x.permute(0, 3, 1, 2).contiguous()
    lib = _lib.load()
    x = _dev(x, "x", (None, None, None, None))
    N, H, W, C = x.shape
    out = torch.empty(N, C, H, W, dtype=torch.float32, device=x.device)
    _call(x.device, lambda: lib.nfe_nhwc_to_nchw(_ptr(x), N, C, H, W, _ptr(out), _stream()), "nfe_nhwc_to_nchw")
    return out


def nhwc_to_planes(x):
    """[N,H,W,96] -> tri-plane gather layout [N,3,H,W,32]."""
    lib = _lib.load()
    x = _dev(x, "planes", (None, None, None, 96))
    N, H, W, _ = x.shape
    out = torch.empty(N, 3, H, W, 32, dtype=torch.float32, device=x.device)
    _call(x.device, lambda: lib.nfe_nhwc_to_planes(_ptr(x), N, H, W, _ptr(out), _stream()), "nfe_nhwc_to_planes")
    return out


def plane_stats_nhwc(x):
    """compute_mean_var on NHWC [N,H,W,C] -> mean, std [N,C,1,1]."""
    lib = _lib.load()
    x = _dev(x, "planes", (None, None, None, None))
    N, H, W, C = x.shape
    mean = torch.empty(N, C, 1, 1, dtype=torch.float32, device=x.device)
    std = torch.empty_like(mean)
    scratch = torch.empty(N * C * 2, dtype=torch.float64, device=x.device)
    _call(x.device, lambda: lib.nfe_plane_stats_nhwc(_ptr(x), N, H * W, C, _ptr(mean), _ptr(std), _ptr(scratch), _stream()),
          "nfe_plane_stats_nhwc")
    return mean, std


def _wide_rows(what, out, out_offset, rows, cols, dev):
    """(view, row stride) of columns out_offset .. of the caller's buffer, which has to hold rows x cols there."""
    if out.dtype != torch.float32 or out.dim() != 2 or not out.is_contiguous() or out.device != dev or out.shape[0] != rows or \
            out_offset < 0 or out.shape[1] < out_offset + cols:
        raise ValueError(f"{what}: out must be float32 [{rows}, S] on {dev}, contiguous, with {cols} columns from out_offset {out_offset}; got {out.dtype} "
                         f"{list(out.shape)} on {out.device}")
    return out[:, out_offset:], out.shape[1]


def fully_connected(x, weight, bias, weight_gain, bias_gain=1.0, lrelu=False, out=None, out_offset=0):
    """FullyConnectedLayer.forward; `out` (a [N,S] buffer) + out_offset write into a wider row (concat)."""
    lib = _lib.load()
    x = _dev(x, "x", (None, None))
    N, fin = x.shape
    weight = _dev(weight, "weight", (None, fin))
    fout = weight.shape[0]
    if bias is not None:
        bias = _dev(bias, "bias", (fout,))
    if out is None:
        out = torch.empty(N, fout, dtype=torch.float32, device=x.device)
        view, stride = out, fout
    else:
        view, stride = _wide_rows("fully_connected", out, out_offset, N, fout, x.device)
    _call(x.device, lambda: lib.nfe_fully_connected(_ptr(x), _ptr(weight), _ptr(bias), N, fin, fout, float(weight_gain),
                                                    float(bias_gain), int(bool(lrelu)),
                                                    ctypes.c_void_p(view.data_ptr()), stride, _stream()), "nfe_fully_connected")
    return out


def fully_connected_grouped(groups):
    """nfe_fully_connected_grouped: groups = [(x [N,in] (rows may be strided: a column block of ws), weight, bias, weight_gain,
    bias_gain)] -> list of [N,out] tensors, one launch for all of them."""
    lib = _lib.load()
    outs, keep = [], []
    arr = (_lib.FcGroup * len(groups))()
    N, dev = groups[0][0].shape[0], groups[0][0].device
    for i, (x, w, b, wg, bg) in enumerate(groups):
        assert x.is_cuda and x.dtype == torch.float32 and x.dim() == 2 and x.shape[0] == N and x.stride(1) == 1
        w = _dev(w, "weight", (None, x.shape[1]))
        y = torch.empty(N, w.shape[0], dtype=torch.float32, device=dev)
        g = arr[i]
        g.x, g.x_stride, g.w, g.b, g.y = x.data_ptr(), x.stride(0) if N > 1 else x.shape[1], w.data_ptr(), (b.data_ptr() if b is not None else None), y.data_ptr()
        g.in_features, g.out_features, g.weight_gain, g.bias_gain = x.shape[1], w.shape[0], float(wg), float(bg)
        outs.append(y); keep += [x, w, b]
    _call(dev, lambda: lib.nfe_fully_connected_grouped(arr, len(groups), N, _stream()), "nfe_fully_connected_grouped")
    return outs


def conv_demod_grouped(pairs, prenormalize=False):
    """nfe_conv_demod_grouped: pairs = [(styles [N,cin], wsq [cout,cin])] -> list of dcoef [N,cout], one launch.
    prenormalize (fp16 operand mode) -> (list of dcoef, list of pre-normalised styles): see conv_demod."""
    lib = _lib.load()
    arr = (_lib.DemodGroup * len(pairs))()
    N, dev = pairs[0][0].shape[0], pairs[0][0].device
    outs, norms = [], []
    for i, (s, wsq) in enumerate(pairs):
        d = torch.empty(N, wsq.shape[0], dtype=torch.float32, device=dev)
        g = arr[i]
        g.styles, g.wsq, g.dcoef, g.cin, g.cout = s.data_ptr(), wsq.data_ptr(), d.data_ptr(), s.shape[1], wsq.shape[0]
        if prenormalize:
            norms.append(torch.empty_like(s))
            g.styles_norm = norms[-1].data_ptr()
        outs.append(d)
    _call(dev, lambda: lib.nfe_conv_demod_grouped(arr, len(pairs), N, _stream()), "nfe_conv_demod_grouped")
    return (outs, norms) if prenormalize else outs


def normalize_2nd_moment(x, out=None, out_offset=0):
    lib = _lib.load()
    x = _dev(x, "x", (None, None))
    N, f = x.shape
    if out is None:
        out = torch.empty_like(x)
        view, stride = out, f
    else:
        view, stride = _wide_rows("normalize_2nd_moment", out, out_offset, N, f, x.device)
    _call(x.device, lambda: lib.nfe_normalize_2nd_moment(_ptr(x), N, f, ctypes.c_void_p(view.data_ptr()), stride, _stream()),
          "nfe_normalize_2nd_moment")
    return out


def broadcast_truncate(w, w_avg, num_ws, psi=1.0, cutoff=None):
    lib = _lib.load()
    w = _dev(w, "w", (None, None))
    N, D = w.shape
    if w_avg is not None:
        w_avg = _dev(w_avg, "w_avg", (D,))
    cutoff = num_ws if cutoff is None else int(cutoff)
    ws = torch.empty(N, num_ws, D, dtype=torch.float32, device=w.device)
    _call(w.device, lambda: lib.nfe_broadcast_truncate(_ptr(w), _ptr(w_avg), N, D, num_ws, float(psi), cutoff, _ptr(ws), _stream()),
          "nfe_broadcast_truncate")
    return ws


def conv_pack(weight, math=None, prenormalize=False):
    """[Cout,Cin,k,k] -> (packed MFMA fragment image, wsq [Cout,Cin]).  math='fp16' packs fp16 operand words (for layers run with
    math='fp16' only); every other mode shares the bf16 hi + lo image.  prenormalize (fp16, demodulated layers): the reference's
    weight pre-normalisation (networks_stylegan2.py:55); pair it with conv_demod(.., prenormalize=True)."""
    lib = _lib.load()
    weight = _dev(weight, "weight", (None, None, None, None))
    cout, cin, k, _ = weight.shape
    words = lib.nfe_conv_packed_words(cout, cin, k)
    if words == 0:
        raise RuntimeError(f"conv_pack: unsupported weight shape {list(weight.shape)}")
    f16 = MATH[math] == _lib.NFE_CONV_F16
    assert f16 or not prenormalize, "prenormalize belongs to the fp16 operand mode"
    packed = torch.empty(words + (cout if f16 else 0), dtype=torch.float32, device=weight.device)
    wsq = torch.empty(cout, cin, dtype=torch.float32, device=weight.device)
    if f16:
        _call(weight.device, lambda: lib.nfe_conv_pack_f16(_ptr(weight), cout, cin, k, int(bool(prenormalize)), _ptr(packed), _ptr(wsq), _stream()),
              "nfe_conv_pack_f16")
    else:
        _call(weight.device, lambda: lib.nfe_conv_pack(_ptr(weight), cout, cin, k, _ptr(packed), _ptr(wsq), _stream()), "nfe_conv_pack")
    return packed, wsq


def conv_demod(styles, wsq, prenormalize=False):
    """dcoef [N,Cout].  prenormalize (fp16 operand mode): -> (dcoef, styles / max|styles| per sample), the reference's style
    pre-normalisation (networks_stylegan2.py:56); wsq must come from conv_pack(.., 'fp16', prenormalize=True)."""
    lib = _lib.load()
    styles = _dev(styles, "styles", (None, None))
    N, cin = styles.shape
    wsq = _dev(wsq, "wsq", (None, cin))
    cout = wsq.shape[0]
    d = torch.empty(N, cout, dtype=torch.float32, device=styles.device)
    sn = torch.empty_like(styles) if prenormalize else None
    _call(styles.device, lambda: lib.nfe_conv_demod(_ptr(styles), _ptr(wsq), N, cin, cout, _ptr(d), _ptr(sn), _stream()), "nfe_conv_demod")
    return (d, sn) if prenormalize else d


FAST_PATH = True      # tests flip this to compare the LDS-DMA 3x3 path with the generic kernel


class SplitImage:
    """bf16 hi(+lo) image of a modulated NHWC activation, produced by one layer for the 3x3 layer that consumes it."""

    def __init__(self, data, shape, math):
        self.data, self.shape, self.math = data, tuple(shape), math


def can_chain(mode, math, n, h, w, cin, cout):
    """True if a layer of these sizes runs the fast path and can therefore take a SplitImage input."""
    if not FAST_PATH:
        return False
    return bool(_lib.load().nfe_conv_accepts_split(int(mode), h, w, cin, cout))


def fuses_rgb(mode, math, n, h, w, cin, cout, rgb_channels):
    """True if a 3x3 layer of these sizes can evaluate the block's ToRGB in its epilogue (nfe_conv_fuses_rgb)."""
    if not FAST_PATH:
        return False
    return bool(_lib.load().nfe_conv_fuses_rgb(int(mode), MATH[math], n, h, w, cin, cout, rgb_channels))


def splits_in_epilogue(mode, n, h, w, cin, cout):
    """True if a plain 3x3 layer of these sizes writes the consuming layer's SplitImage from its own epilogue
    (nfe_conv_splits_in_epilogue): the fp32 output may then be skipped (want_out=False) when nobody else reads it."""
    if not FAST_PATH:
        return False
    return bool(_lib.load().nfe_conv_splits_in_epilogue(int(mode), n, h, w, cin, cout))


def describe(mode, math, n, h, w, cin, cout, rgb_channels=0):
    """nfe_conv_describe: which kernels a layer of these sizes runs at batch n (diagnostic text)."""
    buf = ctypes.create_string_buffer(256)
    _lib.check(_lib.load().nfe_conv_describe(int(mode), MATH[math], n, h, w, cin, cout, int(rgb_channels), buf, 256), "nfe_conv_describe")
    return buf.value.decode()


def modulated_conv(x, styles, packed, cout, mode, bias, dcoef=None, noise=None, noise_strength=0.0, lrelu=True,
                   act_gain=1.0, clamp=None, skip=None, out_planes=False, math=None, next_styles=None, want_out=True, rgb=None):
    """nfe_modulated_conv.  x [N,H,W,Cin] NHWC (or a SplitImage of the modulated input) -> [N,Ho,Wo,Cout]
    (or [N,3,Ho,Wo,32] if out_planes).  With next_styles [N,Cout] also returns the SplitImage for the consuming
    3x3 layer: (out, split); out is None if want_out is False (up-sampling layers, and plain ones where splits_in_epilogue()).
    rgb = (weight [C,Cout], styles [N,Cout], bias [C], skip [N,H/2,W/2,C] or None, clamp): the block's ToRGB evaluated in
    this layer's epilogue (only where fuses_rgb() is true) -> returns (out or None, rgb_image [N,H,W,C]) (+ split with next_styles)."""
    lib = _lib.load()
    a = _lib.ConvArgs()
    a.struct_size = ctypes.sizeof(_lib.ConvArgs)
    a.mode, a.math = int(mode), MATH[math]
    if isinstance(x, SplitImage):
        assert x.math == MATH[math], "SplitImage was produced for another math mode"
        N, H, W, cin = x.shape
        a.x_split = x.data.data_ptr()
        dev = x.data.device
    else:
        x = _dev(x, "x", (None, None, None, None))
        N, H, W, cin = x.shape
        a.x = x.data_ptr()
        dev = x.device
    styles = _dev(styles, "styles", (N, cin))
    a.styles, a.packed = styles.data_ptr(), _dev(packed, "packed").data_ptr()
    keep = [x, styles, packed]
    if dcoef is not None:
        dcoef = _dev(dcoef, "dcoef", (N, cout)); a.dcoef = dcoef.data_ptr()
    up = 2 if mode == _lib.NFE_CONV_3X3_UP2 else 1
    Ho, Wo = H * up, W * up
    if noise is not None:
        noise = _dev(noise, "noise")
        assert tuple(noise.shape[-2:]) == (Ho, Wo) and noise.numel() in (Ho * Wo, N * Ho * Wo), "noise must be [Ho,Wo] or [N,1,Ho,Wo]"
        a.noise, a.noise_strength = noise.data_ptr(), float(noise_strength)
        a.noise_n_stride = Ho * Wo if noise.numel() == N * Ho * Wo and N > 1 else 0
    bias = _dev(bias, "bias", (cout,)); a.bias = bias.data_ptr()
    a.n, a.h, a.w, a.cin, a.cout = N, H, W, cin, cout
    a.lrelu, a.act_gain = int(bool(lrelu)), float(act_gain)
    a.clamp = -1.0 if clamp is None else float(clamp)
    if skip is not None:
        skip = _dev(skip, "skip", (N, H // 2, W // 2, cout)); a.skip = skip.data_ptr()
    a.out_planes = int(bool(out_planes))
    out = None
    rgb_out = None
    if rgb is not None:
        rw, rs, rb, rskip, rclamp = rgb
        C = rw.shape[0]
        rw = _dev(rw.reshape(C, cout), "rgb_weight", (C, cout)); rs = _dev(rs, "rgb_styles", (N, cout)); rb = _dev(rb, "rgb_bias", (C,))
        rgb_out = torch.empty(N, Ho, Wo, C, dtype=torch.float32, device=dev)
        a.rgb_weight, a.rgb_styles, a.rgb_bias, a.rgb_out, a.rgb_channels = rw.data_ptr(), rs.data_ptr(), rb.data_ptr(), rgb_out.data_ptr(), C
        a.rgb_clamp = -1.0 if rclamp is None else float(rclamp)
        if rskip is not None:
            rskip = _dev(rskip, "rgb_skip", (N, H // 2, W // 2, C)); a.rgb_skip = rskip.data_ptr()
        keep += [rw, rs, rb, rskip, rgb_out]
    if want_out or (next_styles is None and rgb is None):
        out = torch.empty((N, 3, Ho, Wo, 32) if out_planes else (N, Ho, Wo, cout), dtype=torch.float32, device=dev)
        a.out = out.data_ptr()
    split = None
    if next_styles is not None:
        next_styles = _dev(next_styles, "next_styles", (N, cout))
        split = SplitImage(torch.empty(int(lib.nfe_conv_split_floats(a.math, N, Ho, Wo, cout)), dtype=torch.float32, device=dev), (N, Ho, Wo, cout), a.math)
        a.next_styles, a.next_split = next_styles.data_ptr(), split.data.data_ptr()
    scratch = None
    n_scratch = int(lib.nfe_conv_scratch_floats(a.mode, a.math, N, H, W, cin, cout)) if FAST_PATH else (N * (2 * H + 1) * (2 * W + 1) * cout if up == 2 else 0)
    if n_scratch:                    # up-conv intermediate, or the pre-split input image of the 3x3 fast path
        scratch = torch.empty(n_scratch, dtype=torch.float32, device=dev)
        a.scratch, a.scratch_floats = scratch.data_ptr(), n_scratch
    keep += [dcoef, noise, bias, skip, scratch, next_styles, split]
    _call(dev, lambda: lib.nfe_modulated_conv(ctypes.byref(a), _stream()), "nfe_modulated_conv")
    if rgb is not None:
        return (out, rgb_out) if next_styles is None else (out, rgb_out, split)
    return out if next_styles is None else (out, split)


def upfirdn2d(x, up=1, down=1, padding=(0, 0), gain=1.0):
    """upfirdn2d (torch_utils/ops/upfirdn2d.py:120) with the path's [1,3,3,1] filter on NHWC: x [N,H,W,C] -> [N,OH,OW,C]."""
    lib = _lib.load()
    x = _dev(x, "x", (None, None, None, None))
    N, H, W, C = x.shape
    p0, p1 = int(padding[0]), int(padding[1])
    oh, ow = (H * up + p0 + p1 - 4) // down + 1, (W * up + p0 + p1 - 4) // down + 1
    out = torch.empty(N, oh, ow, C, dtype=torch.float32, device=x.device)
    _call(x.device, lambda: lib.nfe_upfirdn2d(_ptr(x), N, H, W, C, int(up), int(down), p0, p1, float(gain), _ptr(out), _stream()), "nfe_upfirdn2d")
    return out


def upsample2d(x):
    """upfirdn2d.upsample2d(x, f, up=2) (upfirdn2d.py:315-350): the skip path of SynthesisBlock (networks_stylegan2.py:453)."""
    return upfirdn2d(x, up=2, padding=(2, 1), gain=4.0)


def resize_bilinear_backward(g, h, w, antialias=True):
    """Adjoint of resize_bilinear: g [N,OH,OW,C] (gradient of the resized image) -> [N,h,w,C] (gradient of its input)."""
    lib = _lib.load()
    g = _dev(g, "g", (None, None, None, None))
    N, OH, OW, C = g.shape
    out = torch.empty(N, int(h), int(w), C, dtype=torch.float32, device=g.device)
    _call(g.device, lambda: lib.nfe_resize_bilinear_backward(_ptr(g), N, int(h), int(w), C, OH, OW, int(bool(antialias)), _ptr(out), _stream()),
          "nfe_resize_bilinear_backward")
    return out


def upfirdn2d_polyphase(x, padding=(2, 2), gain=1.0):
    """upfirdn2d(x, up=1, down=1, padding, gain) [N,OH,OW,C] delivered as its four polyphase images stacked along the channels:
    [N, ceil(OH/2), ceil(OW/2), 4C], zeros beyond OH / OW (include/nfe_dense.h: nfe_upfirdn2d_polyphase)."""
    lib = _lib.load()
    x = _dev(x, "x", (None, None, None, None))
    N, H, W, C = x.shape
    OH, OW = H + padding[0] + padding[1] - 3, W + padding[0] + padding[1] - 3
    out = torch.empty(N, (OH + 1) // 2, (OW + 1) // 2, 4 * C, dtype=torch.float32, device=x.device)
    _call(x.device, lambda: lib.nfe_upfirdn2d_polyphase(_ptr(x), N, H, W, C, int(padding[0]), int(padding[1]), float(gain), _ptr(out), _stream()),
          "nfe_upfirdn2d_polyphase")
    return out


def bias_act_backward(out, grad=None, grad_rgb=None, rgb_w=None, rgb_s=None, scale=None, gain=1.0, clamp=None):
    """Backward of bias_act('lrelu', gain, clamp) (bias_act.py:93-125) at a layer's saved output `out` [N,H,W,C], in ONE pass, with the
    block's transposed ToRGB folded in (include/nfe_dense.h: nfe_bias_act_backward):
    ((grad or 0) + (grad_rgb @ rgb_w) * rgb_s) * gain * (0.2 if out < 0 else 1) * (|out| < clamp) * (scale or 1).
    grad [N,H,W,C] or None; grad_rgb [N,H,W,K] with rgb_w [K,C], rgb_s [N,C] or None; scale [N,C] or None."""
    lib = _lib.load()
    out = _dev(out, "out", (None, None, None, None))
    N, H, W, C = out.shape
    if grad is not None:
        grad = _dev(grad.contiguous(), "grad", (N, H, W, C))
    K = 0
    if grad_rgb is not None:
        K = int(grad_rgb.shape[-1])
        grad_rgb = _dev(grad_rgb.contiguous(), "grad_rgb", (N, H, W, K))
        rgb_w = _dev(rgb_w.contiguous(), "rgb_w", (K, C))
        rgb_s = _dev(rgb_s.contiguous(), "rgb_s", (N, C))
    if scale is not None:
        scale = _dev(scale.contiguous(), "scale", (N, C))
    dst = torch.empty_like(out)
    _call(out.device, lambda: lib.nfe_bias_act_backward(_ptr(out), _ptr(grad), _ptr(grad_rgb), _ptr(rgb_w), _ptr(rgb_s), K, _ptr(scale), float(gain),
                                                        float(clamp) if clamp is not None else 0.0, N, H * W, C, _ptr(dst), _stream()),
          "nfe_bias_act_backward")
    return dst


def resize_bilinear(x, oh, ow, antialias=True):
    """F.interpolate(mode='bilinear', align_corners=False, antialias=...) on NHWC."""
    lib = _lib.load()
    x = _dev(x, "x", (None, None, None, None))
    N, H, W, C = x.shape
    out = torch.empty(N, oh, ow, C, dtype=torch.float32, device=x.device)
    _call(x.device, lambda: lib.nfe_resize_bilinear(_ptr(x), N, H, W, C, int(oh), int(ow), int(bool(antialias)), _ptr(out), _stream()),
          "nfe_resize_bilinear")
    return out


# ---- 8-bit rows and weights (include/nfe_dense.h: e4m3 values, one fp32 scale for every block of 128) -------------------------
FP8_BLOCK = 128
_FP8_MATMUL_ARGS = ctypes.sizeof(_lib.Fp8MatmulArgs)
_FP8_TYPES = {torch.float32: _lib.NFE_F32, torch.bfloat16: _lib.NFE_BF16, torch.float16: _lib.NFE_F16}


def _fp8_blocks(n):
    return -(-n // FP8_BLOCK)


# what the library takes; a larger number must not reach it, as its 32-bit arguments would hold the low bits alone
_FP8_ROWS, _FP8_COLS, _FP8_OUT, _FP8_MATMUL_ROWS = (1 << 31) - 1, 1 << 30, 65535 * FP8_BLOCK, 1 << 30


def _fp8_size(name, t, rows, cols):
    if t.shape[0] > rows or t.shape[1] > cols:
        raise ValueError(f"{name}: {list(t.shape)} is too large, at most [{rows}, {cols}]")


def _fp8_rows(t, name, like=None):
    """_dev for the types the 8-bit operators read: a contiguous GPU matrix (of like's shape and type)."""
    if isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in _FP8_TYPES and t.dim() == 2 and (like is None or (t.shape == like.shape and t.dtype == like.dtype)):
        _fp8_size(name, t, _FP8_ROWS, _FP8_COLS)
        return t.contiguous()
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor, got {type(t)}")
    if not t.is_cuda:
        raise RuntimeError(f"{name}: tensor is on {t.device}; this path runs only on the GPU (no CPU fallback)")
    if t.dtype not in _FP8_TYPES:
        raise RuntimeError(f"{name}: expected float32, bfloat16 or float16, got {t.dtype}")
    expected = [None, None] if like is None else list(like.shape)
    assert t.dim() == 2 and (like is None or t.shape == like.shape), f"{name}: wrong shape {list(t.shape)}, expected {expected}"
    raise RuntimeError(f"{name}: expected {like.dtype}, got {t.dtype}")


def _fp8_check(what, *ts):
    """One device (its index is returned), and no gradient asked for."""
    index = ts[0].get_device()
    for t in ts:
        if t is not None:
            if t.get_device() != index:
                raise RuntimeError(f"{what}: the tensors are on several devices")
            if t.requires_grad and torch.is_grad_enabled():
                raise RuntimeError(f"{what}: 8-bit operands carry no gradient; detach the inputs or call it under torch.no_grad()")
    return index


def _address(t):
    return t.data_ptr() if t is not None else None


def _fp8_out(what, out, out_offset, rows, cols, dev):
    """(q, scale) buffers for rows of `cols` columns: new ones (scale block-major), or the columns from out_offset of the caller's."""
    width, blocks = _fp8_blocks(cols) * FP8_BLOCK, _fp8_blocks(cols)
    if out is None:
        if out_offset:
            raise ValueError(f"{what}: out_offset needs out")
        return torch.empty(rows, width, dtype=torch.float8_e4m3fn, device=dev), torch.empty_strided((rows, blocks), (1, rows), dtype=torch.float32, device=dev)
    q, scale = out
    b = out_offset // FP8_BLOCK
    if out_offset % FP8_BLOCK or out_offset < 0 or q.dtype != torch.float8_e4m3fn or q.dim() != 2 or not q.is_contiguous() or q.shape[0] != rows or \
            q.shape[1] % FP8_BLOCK or q.shape[1] < out_offset + width or scale.dtype != torch.float32 or \
            tuple(scale.shape) != (rows, q.shape[1] // FP8_BLOCK) or 0 in scale.stride():
        raise ValueError(f"{what}: out must be (q float8_e4m3fn [{rows}, W] contiguous, scale float32 [{rows}, W / {FP8_BLOCK}]) with W a multiple of "
                         f"{FP8_BLOCK} that holds {width} columns from out_offset, itself a multiple of {FP8_BLOCK}")
    if q.device != dev or scale.device != dev:
        raise RuntimeError(f"{what}: the tensors are on several devices")
    return q[:, out_offset:out_offset + width], scale[:, b:b + blocks]


def rms_norm_fp8(x, weight=None, residual=None, eps=1e-8, out=None, out_offset=0):
    """nfe_rms_norm_fp8: h = x + residual; y = h * rsqrt(mean(h^2) + eps) * weight, rounded to e4m3 with one fp32 scale for every 128 columns.
    x [N,K] fp32 / bf16 / fp16, residual like x, weight [K] fp32.  Returns (q [N, Kp] float8_e4m3fn, scale [N, Kp / 128] fp32) - Kp is K
    rounded up to 128, the columns from K on are zero - and with a residual also h [N,K] in x's type.  y ~ q * scale per block.
    A NaN in a row makes the row NaN; an infinity makes its own block NaN and the row's other blocks zero.
    out = (q, scale) buffers and out_offset (columns, a multiple of 128) write into wider rows.  Inference only."""
    x = _fp8_rows(x, "x")
    N, K = x.shape
    residual = _fp8_rows(residual, "residual", x) if residual is not None else None
    weight = _dev(weight, "weight", (K,)) if weight is not None else None
    index = _fp8_check("rms_norm_fp8", x, residual, weight)
    if K == 0 or not eps >= 2.0 ** -126:
        raise ValueError("rms_norm_fp8: rows need at least one column and eps must be a positive normal number (2^-126 at least)")
    q, scale = _fp8_out("rms_norm_fp8", out, out_offset, N, K, x.device)
    h = torch.empty_like(x) if residual is not None else None
    if N:
        with _on(index):
            _lib.check(_lib.load().nfe_rms_norm_fp8(x.data_ptr(), _address(residual), _address(weight), _FP8_TYPES[x.dtype], N, K, eps, _address(h),
                                                    q.data_ptr(), q.stride(0), scale.data_ptr(), scale.stride(0), scale.stride(1), _stream()), "nfe_rms_norm_fp8")
    return (q, scale) if residual is None else (q, scale, h)


def quantize_fp8(x, out=None, out_offset=0):
    """nfe_quantize_fp8: rms_norm_fp8 without the norm (the operand of the next layer's fp8_matmul) -> (q, scale).  A NaN or an
    infinity makes its block of 128 columns NaN."""
    x = _fp8_rows(x, "x")
    N, K = x.shape
    index = _fp8_check("quantize_fp8", x)
    if K == 0:
        raise ValueError("quantize_fp8: rows need at least one column")
    q, scale = _fp8_out("quantize_fp8", out, out_offset, N, K, x.device)
    if N:
        with _on(index):
            _lib.check(_lib.load().nfe_quantize_fp8(x.data_ptr(), _FP8_TYPES[x.dtype], N, K, q.data_ptr(), q.stride(0), scale.data_ptr(), scale.stride(0),
                                                    scale.stride(1), _stream()), "nfe_quantize_fp8")
    return q, scale


class Fp8Weight:
    """e4m3 weights [out_features, in_features] in fp8_matmul's operand order, with their scales [ceil(out / 128), ceil(in / 128)]."""

    def __init__(self, packed, scale, out_features, in_features):
        n, k = int(out_features), int(in_features)
        if not isinstance(packed, torch.Tensor) or not isinstance(scale, torch.Tensor):
            raise TypeError(f"Fp8Weight: expected torch.Tensors, got {type(packed)} and {type(scale)}")
        size = -(-n // 16) * _fp8_blocks(k) * 16 * FP8_BLOCK                 # nfe_fp8_weight_bytes
        if n <= 0 or k <= 0 or packed.dtype != torch.uint8 or packed.numel() != size or not packed.is_contiguous() or \
                scale.dtype != torch.float32 or tuple(scale.shape) != (_fp8_blocks(n), _fp8_blocks(k)) or not scale.is_contiguous() or \
                scale.device != packed.device:
            raise ValueError(f"Fp8Weight: [{n}, {k}] needs packed uint8 [{size}] and scale float32 [{_fp8_blocks(n)}, {_fp8_blocks(k)}], both contiguous "
                             "and on one device")
        self.packed, self.scale, self.out_features, self.in_features = packed, scale, n, k
        self._stream = self._current_stream()

    def _current_stream(self):
        return torch._C._cuda_getCurrentRawStream(self.packed.get_device()) if self.packed.is_cuda else None

    def used(self):
        """For a holder that may drop the weights while a product on the current stream has still to read them: on a stream other than the one
        they were made on, their memory is handed out again only after what that stream has been given so far."""
        if self._stream != self._current_stream():
            for t in (self.packed, self.scale):
                t.record_stream(torch.cuda.current_stream(t.device))


def _fp8_weight_buffer(lib, n, k, dev):
    if n == 0 or k == 0:
        raise ValueError(f"fp8_weight: empty weight [{n}, {k}]")
    return torch.empty(int(lib.nfe_fp8_weight_bytes(n, k)), dtype=torch.uint8, device=dev)


def fp8_weight(weight, gain=1.0):
    """nfe_fp8_weight_quantize: weight [out, in] (fp32 / bf16 / fp16), rounded to e4m3 with one scale for every 128 x 128 block; gain
    multiplies the scales (FullyConnectedLayer's weight_gain).  A NaN or an infinity makes its whole block NaN."""
    lib = _lib.load()
    if isinstance(weight, torch.Tensor) and weight.dim() == 2:
        _fp8_size("weight", weight, _FP8_OUT, _FP8_COLS)
    weight = _fp8_rows(weight, "weight").detach()
    n, k = weight.shape
    packed = _fp8_weight_buffer(lib, n, k, weight.device)
    scale = torch.empty(_fp8_blocks(n), _fp8_blocks(k), dtype=torch.float32, device=weight.device)
    _call(weight.device, lambda: lib.nfe_fp8_weight_quantize(_ptr(weight), _FP8_TYPES[weight.dtype], n, k, float(gain), _ptr(packed), _ptr(scale), _stream()),
          "nfe_fp8_weight_quantize")
    return Fp8Weight(packed, scale, n, k)


def fp8_weight_from(q, scale):
    """Weights that are e4m3 already: q [out, in] float8_e4m3fn, scale [ceil(out / 128), ceil(in / 128)] fp32 (copied)."""
    lib = _lib.load()
    if not isinstance(q, torch.Tensor) or q.dtype != torch.float8_e4m3fn or q.dim() != 2:
        raise RuntimeError("fp8_weight_from: q must be a float8_e4m3fn tensor [out, in]")
    if q.device.type != "cuda":
        raise RuntimeError(f"fp8_weight_from: q is on {q.device}; this path runs only on the GPU (no CPU fallback)")
    _fp8_size("q", q, _FP8_OUT, _FP8_COLS)
    q = q.contiguous()
    n, k = q.shape
    scale = _dev(scale, "scale", (_fp8_blocks(n), _fp8_blocks(k)))
    if scale.device != q.device:
        raise RuntimeError("fp8_weight_from: the tensors are on several devices")
    packed = _fp8_weight_buffer(lib, n, k, q.device)
    _call(q.device, lambda: lib.nfe_fp8_weight_pack(_ptr(q), n, k, _ptr(packed), _stream()), "nfe_fp8_weight_pack")
    return Fp8Weight(packed, scale.detach().clone(), n, k)


def fp8_matmul(q, scale, weight, bias=None, bias_gain=1.0, lrelu=False, out_dtype=torch.float32):
    """nfe_fp8_matmul: FullyConnectedLayer.forward on the 8-bit rows of rms_norm_fp8 / quantize_fp8 and an Fp8Weight:
    act( (q * scale) @ (w * w_scale).T + bias * bias_gain ), act = linear or lrelu(0.2) * sqrt(2), rounded once to out_dtype -> [N, out].
    out_dtype fp32 sums exact products in fp32; bf16 and fp16 use the 8-bit matrix instructions at twice the rate, whose sums over a block
    are off by less than 7 2^-13 sum|products|: typically 1.5e-5 of the result, below the output's own rounding, but above it where the
    products cancel.  A 16-bit result of exact sums is out_dtype=torch.float32 and a cast.
    q [N, Kp] float8_e4m3fn with Kp = in_features rounded up to 128 (zeros, or any finite values, from in_features on), scale [N, Kp / 128]
    fp32 of any strides (block-major, as rms_norm_fp8 returns it, is read fastest).  Inference only."""
    if not isinstance(weight, Fp8Weight):
        raise TypeError(f"fp8_matmul: weight must be an Fp8Weight (fp8_weight, fp8_weight_from), got {type(weight)}")
    if not isinstance(q, torch.Tensor) or q.dtype != torch.float8_e4m3fn:
        raise RuntimeError(f"fp8_matmul: q must be a float8_e4m3fn tensor, got {getattr(q, 'dtype', type(q))}")
    if not q.is_cuda:
        raise RuntimeError(f"fp8_matmul: q is on {q.device}; this path runs only on the GPU (no CPU fallback)")
    if out_dtype not in _FP8_TYPES:
        raise RuntimeError(f"fp8_matmul: out_dtype must be float32, bfloat16 or float16, got {out_dtype}")
    n, k = weight.out_features, weight.in_features
    kb = _fp8_blocks(k)
    width = kb * FP8_BLOCK
    assert q.dim() == 2 and q.shape[1] == width, \
        f"q: wrong shape {list(q.shape)}, expected [N, {width}] ({k} input features in blocks of {FP8_BLOCK})"
    _fp8_size("q", q, _FP8_MATMUL_ROWS, width)
    N = q.shape[0]
    if not isinstance(scale, torch.Tensor) or scale.dtype != torch.float32 or scale.shape != (N, kb):
        raise RuntimeError(f"fp8_matmul: scale must be a float32 tensor [{N}, {kb}]")
    bias = _dev(bias, "bias", (n,)) if bias is not None else None
    index = _fp8_check("fp8_matmul", q, scale, weight.packed, bias)
    out = torch.empty(N, n, dtype=out_dtype, device=q.device)
    if N == 0:
        return out
    stride, inner = q.stride()
    if inner != 1 or q.data_ptr() % 16 or (N > 1 and (stride % 16 or stride < width)):
        q = q.clone(memory_format=torch.contiguous_format)      # contiguous() would return a contiguous q at an odd address as it is
        stride = width
    a = _lib.Fp8MatmulArgs(_FP8_MATMUL_ARGS, N, n, k, q.data_ptr(), stride if N > 1 else width, scale.data_ptr(), scale.stride(0), scale.stride(1),
                           weight.packed.data_ptr(), weight.scale.data_ptr(), _address(bias), bias_gain, 1 if lrelu else 0, _FP8_TYPES[out_dtype],
                           out.data_ptr())
    with _on(index):
        _lib.check(_lib.load().nfe_fp8_matmul(ctypes.byref(a), _stream()), "nfe_fp8_matmul")
    return out


def describe_fp8_matmul(m, n, out_dtype=torch.float32, q_stride=FP8_BLOCK, scale_row_stride=1):
    """nfe_fp8_matmul_describe: which kernel fp8_matmul runs for m rows and n outputs (diagnostic text)."""
    buf = ctypes.create_string_buffer(64)
    _lib.check(_lib.load().nfe_fp8_matmul_describe(int(m), int(n), int(q_stride), int(scale_row_stride), _FP8_TYPES[out_dtype], buf, 64), "nfe_fp8_matmul_describe")
    return buf.value.decode()
