"""Operators of a differential-attention block on torch tensors: rotary positions, differential attention, and the norms either side of a
block with its gate and residual scale (rz_rotary, rz_diff_attention, rz_residual_norm of include/radzero_hip.h).

They work on GPU tensors alone, on the current stream of the tensors' device, never wait for it and may be captured into a graph.  They are
forward only, like everything here: an input that asks for a gradient, or carries a forward-mode one, is refused.  Types are float32, bfloat16 and float16 for tokens;
weights, gates and lambda vectors are float32.  Strides are free except that columns are contiguous; what a kernel cannot take raises ValueError.

    freqs, amplitude = rotary_frequencies(64, axes=2, device="cuda")
    q, k = rotary(q, k, positions=patch_rows_and_columns, freqs=freqs, amplitude=amplitude)
    ctx = diff_attention(q, k, v, lambda_qk, lambda_init=0.2, norm_weight=w, out_scale=0.8)
    h, xn = residual_norm(h, out_projection, scale=layer_scale, pre_norm=Norm(weight, bias))
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _lib

_DTYPES = {torch.float32: _lib.RZ_F32, torch.bfloat16: _lib.RZ_BF16, torch.float16: _lib.RZ_F16}
_CAUSAL = {None: 0, "start": 1, "end": 2}
_LAYOUT = {"half": 0, "interleaved": 1}
_NORM = {"layer": 1, "rms": 2}


class Norm(NamedTuple):
    """A norm of rows: kind "layer" ((x - mean) / sqrt(var + eps) * weight + bias) or "rms" (x / sqrt(mean x^2 + eps) * weight + bias)."""
    weight: Optional[torch.Tensor] = None
    bias: Optional[torch.Tensor] = None
    eps: float = 1e-6
    kind: str = "layer"


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _tokens(x, name, dim, like=None):
    """Says what is wrong with a tensor of tokens."""
    _need(isinstance(x, torch.Tensor) and x.dim() == dim, f"{name} must be a tensor of {dim} dimensions")
    _need(x.is_cuda, f"{name} must be on the GPU (there is no CPU fallback)")
    _need(x.dtype in _DTYPES, f"{name} must be float32, bfloat16 or float16")
    _need(x.stride(-1) == 1 or x.shape[-1] == 1, f"{name}: columns must be contiguous")
    _need(not (x.requires_grad and torch.is_grad_enabled()), f"{name} asks for a gradient: these operators are forward only (torch.no_grad())")
    if like is not None:
        _need(x.dtype == like.dtype, f"{name} must be {like.dtype}")
        _need(x.device == like.device, f"{name} must be on {like.device}")


def _vector(x, name, shape, device):
    """Address of a contiguous float32 tensor, 0 for None."""
    if x is None:
        return 0
    if not (isinstance(x, torch.Tensor) and x.dtype is torch.float32 and x.shape == shape and x.device == device and x.is_contiguous() and not x.requires_grad):
        _need(isinstance(x, torch.Tensor) and x.dtype == torch.float32 and x.shape == shape, f"{name} must be float32 {tuple(shape)}")
        _need(x.device == device and x.is_contiguous(), f"{name} must be contiguous on {device}")
        _need(not torch.is_grad_enabled(), f"{name} asks for a gradient: these operators are forward only (torch.no_grad())")
    return x.data_ptr()


def _no_tangents(*inputs):
    """Tensors that carry a forward-mode derivative do not say so in requires_grad."""
    for x in inputs:
        _need(not isinstance(x, torch.Tensor) or forward_ad.unpack_dual(x).tangent is None, "an input carries a forward-mode derivative: these operators have none")


def _differentiating():
    """Inside a level of forward-mode differentiation (then inputs are looked at one by one)?"""
    return getattr(forward_ad, "_current_level", 0) >= 0


_empty_like = torch.empty_like


def _new(like):
    """A contiguous tensor of this one's shape, type and device, the cheapest way (empty_like would keep other strides too)."""
    return _empty_like(like) if like.is_contiguous() else like.new_empty(tuple(like.shape))


def _output(out, like_shape, dtype, device, name):
    _need(isinstance(out, torch.Tensor) and out.shape == like_shape and out.dtype == dtype and out.device == device,
          f"{name} must be {dtype} {tuple(like_shape)} on {device}")
    _need(all(s for s, n in zip(out.stride(), out.shape) if n > 1) and (out.stride(-1) == 1 or out.shape[-1] == 1), f"{name}: columns must be contiguous, rows apart")
    _need(not (out.requires_grad and torch.is_grad_enabled()), f"{name} asks for a gradient: these operators are forward only (torch.no_grad())")
    if _differentiating():
        _no_tangents(out)
    return out


def _written(*outs):
    """Tensors of the caller's were written: a backward pass that saved one of them before has to notice, as after any in-place operation."""
    for x in outs:
        if x is not None:
            increment_version(x)


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_entry = {}


def _fn(name, *argtypes):
    """An entry point that takes its struct as bytes (the prototypes in _lib.SYMBOLS take the ctypes mirrors)."""
    fn = _entry.get(name)
    if fn is None:
        fn = _entry[name] = ctypes.CFUNCTYPE(_lib.SYMBOLS[name][0], ctypes.c_char_p, *argtypes)((name, _lib.load()))
    return fn


def _call(name, argtypes, device, *args):
    index = device.index
    if index == torch.cuda.current_device():
        rc = _fn(name, *argtypes)(*args, _raw_stream(index))
    else:                                                # kernels go to the tensors' device, on its current stream
        with torch.cuda.device(device):
            rc = _fn(name, *argtypes)(*args, _raw_stream(index))
    if rc:
        _lib.check(rc, name)


_NOT_PACKED = (struct.error, OverflowError)


def _not_packed(args, e):
    """What a struct does not take is a bad argument like any other."""
    return ValueError(f"{args.__name__}: a size beyond 32 bits or an argument that is no number ({e})")


_STREAM = (ctypes.c_void_p,)
_WORKSPACE_STREAM = (ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p)


def rotary_frequencies(rotary_dim: int, *, base: float = 10000.0, axes: int = 1, scaling: Optional[dict] = None, device=None) -> Tuple[torch.Tensor, float]:
    """(frequencies in float64, amplitude) for `rotary`: f_p = base^(-p / P), p = 0 .. P - 1, with P = rotary_dim / (2 axes) pairs per axis;
    shape (P,) for one axis, (axes, P) for several (an image's rows and columns).

    scaling stretches a table made for `original_length` positions to `factor` times as many:
      {"kind": "linear", "factor": s}   every frequency divided by s
      {"kind": "ntk", "factor": s}      base s^(P / (P - 1)): the fastest pair stays, the slowest is divided by s
      {"kind": "yarn", "factor": s, "original_length": L, "beta_fast": 32, "beta_slow": 1}
            f (g + (1 - g) / s) with g = 1 for pairs that turn at least beta_fast times over L, 0 below beta_slow, linear between; amplitude 0.1 ln s + 1
    """
    _need(axes >= 1 and rotary_dim >= 2 * axes and rotary_dim % (2 * axes) == 0, "rotary_dim must be a multiple of 2 * axes")
    pairs = rotary_dim // (2 * axes)
    p = torch.arange(pairs, dtype=torch.float64)
    amplitude = 1.0
    freqs = base ** (-p / pairs)
    if scaling is not None:
        kind, s = scaling.get("kind"), float(scaling.get("factor", 0.0))
        _need(s >= 1.0, "scaling: factor must be at least 1")
        if kind == "linear":
            freqs = freqs / s
        elif kind == "ntk":
            _need(pairs > 1, "scaling: ntk needs more than one pair per axis")
            freqs = (base * s ** (pairs / (pairs - 1))) ** (-p / pairs)
        elif kind == "yarn":
            length = float(scaling.get("original_length", 0.0))
            fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))
            _need(length > 0 and fast > slow, "scaling: yarn needs original_length > 0 and beta_fast > beta_slow")
            g = ((freqs * length / (2 * math.pi) - slow) / (fast - slow)).clamp(0.0, 1.0)
            freqs = freqs * (g + (1 - g) / s)
            amplitude = 0.1 * math.log(s) + 1.0
        else:
            raise ValueError("scaling: kind must be linear, ntk or yarn")
    if axes > 1:
        freqs = freqs.expand(axes, pairs).contiguous()
    return freqs.to(device), amplitude


def rotary(q: torch.Tensor, k: Optional[torch.Tensor] = None, *, positions: torch.Tensor, freqs: torch.Tensor, layout: str = "half",
           amplitude: float = 1.0, out=None):
    """Rotary positions on q (batch, tokens, heads, head_dim) and, in the same launch, k (batch, tokens, k_heads, head_dim).

    freqs: float64, (P,) or (axes, P) as `rotary_frequencies` makes them; the first 2 * freqs.numel() columns turn, the others pass through.
    positions: int64, (tokens,) or (batch, tokens), with a last dimension of `axes` if freqs has two dimensions; |position| < 2^31.
    layout: "half" pairs column p with p + rotary_dim / 2, "interleaved" 2 p with 2 p + 1.
    out: tensors to write (q_out, or (q_out, k_out)); q_out may be q itself, k_out k; no other overlap.  Returns q_out, or (q_out, k_out) with k."""
    if _differentiating():
        _no_tangents(q, k, freqs)
    if not (isinstance(q, torch.Tensor) and q.is_cuda and q.dtype in _DTYPES and q.dim() == 4 and q.stride(3) == 1 and not q.requires_grad):
        _tokens(q, "q", 4)
    b, n, hq, d = q.shape
    dev, dt = q.device, q.dtype
    hk, ks = 0, (0, 0, 0)
    if k is not None:
        if not (isinstance(k, torch.Tensor) and k.dtype is dt and k.device == dev and k.dim() == 4 and k.stride(3) == 1 and not k.requires_grad):
            _tokens(k, "k", 4, q)
        kb, kn, hk, kd = k.shape
        _need(kb == b and kn == n and kd == d, "q and k must agree in batch, tokens and head_dim")
    _need(layout in _LAYOUT, "layout must be half or interleaved")
    _need(isinstance(freqs, torch.Tensor) and freqs.dtype is torch.float64 and freqs.dim() in (1, 2) and freqs.device == dev and freqs.is_contiguous(),
          "freqs must be contiguous float64 (pairs,) or (axes, pairs) on q's device")
    _need(not (freqs.requires_grad and torch.is_grad_enabled()), "freqs asks for a gradient: these operators are forward only (torch.no_grad())")
    pos = positions
    _need(isinstance(pos, torch.Tensor) and pos.dtype is torch.int64 and pos.device == dev, "positions must be int64 on q's device")
    shape, strides, axes = tuple(pos.shape), pos.stride(), 1
    if freqs.dim() == 2:
        axes = freqs.shape[0]
        _need(len(shape) in (2, 3) and shape[-1] == axes and (strides[-1] == 1 or axes == 1), "positions need a contiguous last dimension of one value per axis")
        shape, strides = shape[:-1], strides[:-1]
    _need(shape == (b, n) or shape == (n,), "positions must be (tokens,) or (batch, tokens)")
    if out is None:
        qo, ko = _new(q), None if k is None else _new(k)
    else:
        qo, ko = (out, None) if k is None else out
        qo = _new(q) if qo is None else _output(qo, q.shape, dt, dev, "out")
        ko = None if k is None else _new(k) if ko is None else _output(ko, k.shape, dt, dev, "out")
    kos, kp, kop = ks, 0, 0
    if hk:
        ks, kos, kp, kop = k.stride(), ko.stride(), k.data_ptr(), ko.data_ptr()
    qs, qos = q.stride(), qo.stride()
    try:
        args = _lib.RzRotaryArgs.pack(
            _DTYPES[dt], _LAYOUT[layout], b, n, hq, hk, d, 2 * freqs.numel(), axes, amplitude, q.data_ptr(), qs[0], qs[1], qs[2], kp, ks[0], ks[1], ks[2],
            qo.data_ptr(), qos[0], qos[1], qos[2], kop, kos[0], kos[1], kos[2], pos.data_ptr(), strides[0] if len(shape) == 2 else 0, strides[-1], freqs.data_ptr())
    except _NOT_PACKED as e:
        raise _not_packed(_lib.RzRotaryArgs, e) from None
    _call("rz_rotary", _STREAM, dev, args)
    if out is not None:
        _written(qo, ko)
    return qo if k is None else (qo, ko)


def diff_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lambda_qk: torch.Tensor, *, lambda_init: float, scale: Optional[float] = None,
                   causal: Optional[str] = None, kv_lens: Optional[torch.Tensor] = None, attention_mask: Optional[torch.Tensor] = None,
                   norm_weight: Optional[torch.Tensor] = None, norm_eps: float = 1e-5, out_scale: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out_scale * norm((softmax(scale q1 k1^T) - lambda softmax(scale q2 k2^T)) v), lambda = exp(lq1 . lk1) - exp(lq2 . lk2) + lambda_init.

    q (batch, n_q, heads, 2 d), k and v (batch, n_k, kv_heads, 2 d), d = 32, 64 or 128; a row of q and k is [first map | second map]; heads a multiple
    of kv_heads.  lambda_qk float32 (4, d) = lq1, lk1, lq2, lk2, or (heads, 4, d).  scale: 1 / sqrt(d) by default.
    causal: "start" = query i is token i and sees keys 0 .. i; "end" = the queries are the last n_q tokens of their sequence.
    kv_lens int32 or int64 (batch,): only the first kv_lens[b] keys count.  attention_mask integer or bool (batch, n_k): 0 = hidden, as a tokenizer gives it (int64 as it
    is, other types through a copy).  A query that sees
    no key gets zeros; what hidden keys hold changes nothing.  norm_weight float32 (2 d): root-mean-square norm of every head's output.
    Sums and statistics are float32; the 16-bit types round each weight for the product with v (float16: weights too small for it lose at most 2^-13 of
    a row's sum together, over up to 2^22 keys); float32 products may be taken from three bf16 parts of each
    operand (2^-22 of |a||b| off, and 2^-126 of the other for values so small that a part of theirs ends there; an infinity that a query sees then gives NaN).
    bfloat16 and float32 results are finite while |v| * 2^15 * keys is.
    16-byte alignment of q, k, v and out and of their strides is required.  Returns (batch, n_q, heads, 2 d), in `out` (no input's memory) if given."""
    if _differentiating():
        _no_tangents(q, k, v, lambda_qk, norm_weight)
    if not (isinstance(q, torch.Tensor) and q.is_cuda and q.dtype in _DTYPES and q.dim() == 4 and not q.requires_grad):
        _tokens(q, "q", 4)
    dev, dt = q.device, q.dtype
    for x, name in ((k, "k"), (v, "v")):
        if not (isinstance(x, torch.Tensor) and x.dtype is dt and x.device == dev and x.dim() == 4 and not x.requires_grad):
            _tokens(x, name, 4, q)
    (b, n_q, h, w), (kb, n_k, hk, kw) = q.shape, k.shape
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    d = w // 2
    _need(w in (64, 128, 256), "the last dimension must be 64, 128 or 256 (two maps of 32, 64 or 128)")
    _need(kb == b and kw == w and v.shape == k.shape, "k and v must be (batch, n_k, kv_heads, 2 d), like q in batch and 2 d")
    _need(qs[3] == 1 and ks[3] == 1 and vs[3] == 1, "q, k, v: columns must be contiguous")
    _need(h >= 1 and hk >= 1, "there must be a head of q and of k")
    _need(causal in _CAUSAL, "causal must be None, start or end")
    per_head = isinstance(lambda_qk, torch.Tensor) and lambda_qk.dim() == 3
    lam = _vector(lambda_qk, "lambda_qk", (h, 4, d) if per_head else (4, d), dev)
    _need(lam, "lambda_qk must be a tensor")
    lens = 0
    if kv_lens is not None:
        _need(isinstance(kv_lens, torch.Tensor) and kv_lens.shape == (b,) and kv_lens.device == dev and kv_lens.dtype in (torch.int32, torch.int64),
              "kv_lens must be int32 or int64 (batch,) on q's device")
        if kv_lens.dtype is torch.int64:
            kv_lens = kv_lens.clamp(0, n_k).to(torch.int32)
        kv_lens = kv_lens.contiguous()
        lens = kv_lens.data_ptr()
    mask, mask_stride = 0, 0
    if attention_mask is not None:
        x = attention_mask
        _need(isinstance(x, torch.Tensor) and x.shape == (b, n_k) and x.device == dev and not x.dtype.is_floating_point and not x.dtype.is_complex,
              "attention_mask must be integer or bool (batch, n_k) on q's device")
        x = x.to(torch.int64)
        if n_k > 1 and x.stride(1) != 1:
            x = x.contiguous()
        attention_mask, mask, mask_stride = x, x.data_ptr(), x.stride(0)
    given, out = out, _new(q) if out is None else _output(out, q.shape, dt, dev, "out")
    os = out.stride()
    w_ptr = _vector(norm_weight, "norm_weight", (w,), dev)
    try:
        args = _lib.RzDiffAttentionArgs.pack(
            _DTYPES[dt], b, h, hk, n_q, n_k, d, _CAUSAL[causal], d ** -0.5 if scale is None else scale, lambda_init, norm_eps, out_scale,
            q.data_ptr(), qs[0], qs[1], qs[2], k.data_ptr(), ks[0], ks[1], ks[2], v.data_ptr(), vs[0], vs[1], vs[2], out.data_ptr(), os[0], os[1], os[2],
            lam, 4 * d if per_head else 0, w_ptr, lens, mask, mask_stride)
    except _NOT_PACKED as e:
        raise _not_packed(_lib.RzDiffAttentionArgs, e) from None
    need = _fn("rz_diff_attention_workspace")(args)
    ws = q.new_empty(need, dtype=torch.uint8) if need else None
    _call("rz_diff_attention", _WORKSPACE_STREAM, dev, args, ws.data_ptr() if need else 0, need)
    _written(given)
    return out


def residual_norm(residual: torch.Tensor, y: Optional[torch.Tensor] = None, *, pre_norm: Optional[Norm], post_norm: Optional[Norm] = None,
                  scale: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, alpha: float = 1.0, dtype: Optional[torch.dtype] = None, out=None):
    """(r, x) with r = alpha * residual + scale * gate * post_norm(y) and x = pre_norm(r): a block's output joins the residual stream and the next block's
    operand leaves with it.

    residual (rows, dim) or (batch, rows, dim), float32 or y's type; y of the same shape (None: r = alpha * residual).  scale float32 (dim,).
    gate float32: (dim,), (batch, dim), (batch, rows, dim) or, for a residual of two dimensions, (dim,) or (rows, dim).
    x has y's type (without y: `dtype`, else the residual's).  pre_norm None: x is None.  out: (r, x) to write; either may be `residual` or `y` itself,
    no other overlap.
    Without y and alpha, and no place given for it, r is `residual` itself (a copy if x is written over that).
    pre_norm's statistics are those of r in float32, before it is rounded to the residual's type."""
    if _differentiating():
        _no_tangents(residual, y, scale, gate, *(pre_norm or ()), *(post_norm or ()))
    nd = residual.dim() if isinstance(residual, torch.Tensor) else 0
    _need(nd == 2 or nd == 3, "residual must be (rows, dim) or (batch, rows, dim)")
    hs = residual.stride()
    if not (residual.is_cuda and residual.dtype in _DTYPES and hs[-1] == 1 and not residual.requires_grad):
        _tokens(residual, "residual", nd)
    dev, rt, shape = residual.device, residual.dtype, residual.shape
    dim = shape[-1]
    t = rt if dtype is None else dtype
    yp, ys = 0, (0, 0, 0)
    if y is not None:
        if not (isinstance(y, torch.Tensor) and y.dtype in _DTYPES and y.device == dev and y.dim() == nd and y.stride(-1) == 1 and not y.requires_grad):
            _tokens(y, "y", nd)
        _need(y.shape == shape and y.device == dev, "y must have the residual's shape and device")
        _need(dtype is None or dtype is y.dtype, "x has y's type")
        t, yp, ys = y.dtype, y.data_ptr(), y.stride()
    else:
        _need(post_norm is None and scale is None and gate is None, "post_norm, scale and gate need y")
    _need(t in _DTYPES and (rt is torch.float32 or rt is t), "the residual must be float32 or of x's type")
    gp, gb, gr = 0, 0, 0
    if gate is not None:
        _need(isinstance(gate, torch.Tensor) and gate.dtype is torch.float32 and gate.device == dev and 1 <= gate.dim() <= nd, "gate must be float32 on the residual's device")
        full = (dim,) if gate.dim() == 1 else shape if gate.dim() == nd else (shape[0], dim)
        _need(tuple(gate.shape) == tuple(full) and (gate.stride(-1) == 1 or dim == 1), "gate must be (dim,), (batch, dim) or the residual's shape, columns contiguous")
        _need(not (gate.requires_grad and torch.is_grad_enabled()), "gate asks for a gradient: these operators are forward only (torch.no_grad())")
        st = gate.stride()
        gp = gate.data_ptr()
        gb, gr = (0, 0) if gate.dim() == 1 else (st[0], st[1]) if gate.dim() == 3 else (st[0], 0) if nd == 3 else (0, st[0])
    ro, xo = (None, None) if out is None else out
    rp, rs, xp, xs = 0, (0, 0, 0), 0, (0, 0, 0)
    if y is not None or alpha != 1.0 or ro is not None or pre_norm is None or (isinstance(xo, torch.Tensor) and xo.data_ptr() == residual.data_ptr()):
        # the last: x over the residual, r is a copy
        ro = _new(residual) if ro is None else _output(ro, shape, rt, dev, "out[0]")
        rp, rs = ro.data_ptr(), ro.stride()
    else:
        ro = residual
    post_kind, post_eps, post_w, post_b, pre_kind, pre_eps, pre_w, pre_b = 0, 0.0, 0, 0, 0, 0.0, 0, 0
    if post_norm is not None:
        post_w, post_b, post_eps, post_kind = post_norm
        _need(post_kind in _NORM, "post_norm.kind must be layer or rms")
        post_kind, post_w, post_b = _NORM[post_kind], _vector(post_w, "post_norm.weight", (dim,), dev), _vector(post_b, "post_norm.bias", (dim,), dev)
    if pre_norm is not None:
        pre_w, pre_b, pre_eps, pre_kind = pre_norm
        _need(pre_kind in _NORM, "pre_norm.kind must be layer or rms")
        pre_kind, pre_w, pre_b = _NORM[pre_kind], _vector(pre_w, "pre_norm.weight", (dim,), dev), _vector(pre_b, "pre_norm.bias", (dim,), dev)
        xo = _output(xo, shape, t, dev, "out[1]") if xo is not None else _new(residual) if rt is t else _new(y) if y is not None else residual.new_empty(tuple(shape), dtype=t)
        xp, xs = xo.data_ptr(), xo.stride()
    else:
        _need(xo is None, "out[1] needs pre_norm")
    if nd == 2:
        batch, rows, hs, ys, rs, xs = 1, shape[0], (0, *hs), (0, *ys), (0, *rs), (0, *xs)
    else:
        batch, rows = shape[0], shape[1]
    scale_ptr = _vector(scale, "scale", (dim,), dev)
    try:
        args = _lib.RzResidualNormArgs.pack(
            _DTYPES[t], _DTYPES[rt], batch, rows, dim, post_kind, pre_kind, alpha, post_eps, pre_eps, yp, ys[0], ys[1], residual.data_ptr(), hs[0], hs[1], rp, rs[0], rs[1],
            xp, xs[0], xs[1], post_w, post_b, scale_ptr, gp, gb, gr, pre_w, pre_b)
    except _NOT_PACKED as e:
        raise _not_packed(_lib.RzResidualNormArgs, e) from None
    _call("rz_residual_norm", _STREAM, dev, args)
    if out is not None:
        _written(*out)
    return ro, xo
