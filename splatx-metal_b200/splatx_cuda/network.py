"""Operators for training a network beside the splats: attention, the norm and rotation of its queries
and keys, linear layers, layer norm, AdamW.

The reference has no counterpart: its trainer updates the Gaussians themselves. A network that
predicts, refines or conditions them (tokens of splats or of image patches) trains with these.
Inputs are CUDA tensors and stay where they are; every call enqueues on the current stream of the
tensors' device, allocates its results (and a workspace, where it needs one) from torch and does
not synchronise. Contract violations raise ``ValueError``, device failures ``RuntimeError``.

    out, lse = attention_fwd(q, k, v, causal=True)           # [batch, tokens, heads, head_dim]
    v_q, v_k, v_v = attention_bwd(v_out, q, k, v, out, lse, causal=True)
    y, mean, rstd = layer_norm_fwd(x, weight, bias)
    v_x, v_weight, v_bias = layer_norm_bwd(v_y, x, weight, mean, rstd)
    y, pre = linear_fwd(x, weight, bias, activation="gelu", keep=True)
    v_x, v_weight, v_bias = linear_bwd(v_y, x, weight, bias, pre, activation="gelu")
    q, k = qk_norm_rotary_fwd(q, k, positions, axes=(32, 48, 48))  # [batch, tokens, axes]
    AdamW(params, lr=1e-3, state_bits=8).step()              # params with .grad, or step(grads)

``attention``, ``linear``, ``qk_norm_rotary`` and ``layer_norm`` are the same with torch's autograd
(first derivatives; a second one raises ``RuntimeError``).
"""
from __future__ import annotations

import ctypes as C
import functools
import math

import numpy as np
import torch
from torch.autograd.function import once_differentiable

from . import _native as _nat
from ._native import check

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
RUN = 256  # consecutive values of an 8-bit moment that share a scale


def _dtype(t: torch.Tensor, what: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{what}: float32, float16 or bfloat16 needed, got {t.dtype}")
    return code


def _on(device: torch.device, what: str, *others) -> None:
    """Refuses tensors (or None) that are not on the CUDA device of the call's first one."""
    if device.type != "cuda":
        raise ValueError(f"{what}: CUDA tensors needed (there is no CPU path)")
    for t in others:
        if t is not None and t.device != device:
            raise ValueError(f"{what}: a tensor is on {t.device}, not on {device}")


# the current stream's handle without a torch.cuda.Stream made for it, which takes a short call 3 of its 20 us
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


class _at:
    """The device made current for one call (left alone where it is already) and its stream."""

    __slots__ = ("index", "was")

    def __init__(self, device):
        self.index, self.was = device.index, torch.cuda.current_device()

    def __enter__(self):
        if self.was != self.index:
            torch.cuda.set_device(self.index)
        return _raw_stream(self.index)

    def __exit__(self, *exc):
        if self.was != self.index:
            torch.cuda.set_device(self.was)
        return False


def attention_status() -> int:
    """Status bits the attention kernels of the current device have set since the last call (0: all
    is well; 1: a bounded wait inside a kernel ran out and its outputs are invalid). Synchronises."""
    st = C.c_uint32(0)
    check(_nat.lib().sxcuda_attention_status(C.byref(st)))
    return int(st.value)


# ---------------------------------------------------------------- attention

def _view(t: torch.Tensor) -> tuple:
    s = t.stride()
    return t.data_ptr(), s[0], s[1], s[2]


def _heads_last(t: torch.Tensor, what: str) -> torch.Tensor:
    """t with a contiguous last axis. A 16-bit t whose rows the tensor-core kernels' copies do not
    reach (an odd offset or stride, a broadcast axis such as the gradient of a sum) is copied: that
    costs a pass over it, the kernel without tensor cores many times the whole call."""
    if t.dim() != 4:
        raise ValueError(f"{what}: [batch, tokens, heads, head_dim] needed, got {tuple(t.shape)}")
    n, s = t.shape, t.stride()
    if s[3] != 1 and n[3] != 1:
        return t.contiguous()
    if n[3] % 8 or t.dtype == torch.float32:
        return t
    reached = not ((s[0] | s[1] | s[2] | t.data_ptr() >> 1) & 7) and s[0] and s[1] and s[2]
    if reached or not (t.data_ptr() % 16 or any(n[i] > 1 and (s[i] % 8 or not s[i]) for i in range(3))):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _attention_inputs(what, q, k, v, scale, causal, q_lens, kv_lens):
    q, k, v = _heads_last(q, what), _heads_last(k, what), _heads_last(v, what)
    code = _dtype(q, what)
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"{what}: q, k and v must have one dtype")
    b, n, h, d = q.shape
    kb, kn, kh, kd = k.shape
    if k.shape != v.shape or kb != b or kd != d:
        raise ValueError(f"{what}: k and v must both be [{b}, tokens, heads, {d}], got "
                         f"{tuple(k.shape)} and {tuple(v.shape)}")
    device = q.device
    _on(device, what, k, v, q_lens, kv_lens)
    for name, lens in (("q_lens", q_lens), ("kv_lens", kv_lens)):
        if lens is not None and (lens.dtype != torch.int32 or lens.shape != (b,) or
                                 not lens.is_contiguous()):
            raise ValueError(f"{what}: {name} must be a contiguous int32 tensor of [{b}]")
    ins = _nat.SxAttentionInputs(
        _view(q), _view(k), _view(v), None if q_lens is None else q_lens.data_ptr(),
        None if kv_lens is None else kv_lens.data_ptr(), b, n, kn, h, kh, d, code,
        (1.0 / math.sqrt(d) if d else 1.0) if scale is None else scale, causal)
    return q, k, v, ins, device


def _workspace(entry, device, ins):
    """(tensor, its pointer, its size) of the workspace that the entry point asks for; where it needs
    none, a pointer that it does not read."""
    nbytes = C.c_size_t(0)
    check(entry(C.byref(ins), None, None, None, C.byref(nbytes), None))
    if not nbytes.value:
        return None, 16, nbytes
    ws = torch.empty(nbytes.value, dtype=torch.uint8, device=device)
    return ws, ws.data_ptr(), nbytes


def attention_fwd(q, k, v, *, scale=None, causal=False, q_lens=None, kv_lens=None):
    """softmax(scale q k^T) v per head: (out like q, lse [batch, heads, tokens] in float32).

    q: [batch, q_len, heads, head_dim]; k, v: [batch, kv_len, kv_heads, head_dim] with heads a
    multiple of kv_heads; float32, float16 or bfloat16, head_dim 1..128, any strides with the last
    axis contiguous. scale defaults to 1 / sqrt(head_dim). q_lens, kv_lens: int32 [batch] token
    counts of a padded batch; what lies beyond them is not used. causal: query i sees key j where
    j <= i + kv_len - q_len (the lengths of its batch entry). A query that sees no key gets output 0
    and log-sum -inf; one that sees a score of NaN or +inf, or only -inf, is NaN. A k or v that is
    not finite may also reach queries whose causal mask hides it (0 * NaN is NaN)."""
    q, k, v, ins, device = _attention_inputs("attention_fwd", q, k, v, scale, causal, q_lens, kv_lens)
    b, n, h, _ = q.shape
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = q.new_empty((b, h, n), dtype=torch.float32)
    ov, entry = _nat.SxAttentionView(*_view(out)), _nat.lib().sxcuda_attention_fwd
    with _at(device) as stream:
        ws, at, nbytes = _workspace(entry, device, ins)
        check(entry(C.byref(ins), C.byref(ov), lse.data_ptr(), at, C.byref(nbytes), stream))
    return out, lse


def attention_bwd(v_out, q, k, v, out, lse, *, scale=None, causal=False, q_lens=None, kv_lens=None):
    """Gradients (v_q, v_k, v_v) of attention_fwd for the gradient v_out of its output; out and lse
    are the forward's. Deterministic."""
    what = "attention_bwd"
    q, k, v, ins, device = _attention_inputs(what, q, k, v, scale, causal, q_lens, kv_lens)
    for name, t in (("v_out", v_out), ("out", out)):
        if t.shape != q.shape or t.dtype != q.dtype:
            raise ValueError(f"{what}: {name} must be like q")
    if lse.shape != (q.shape[0], q.shape[2], q.shape[1]) or lse.dtype != torch.float32 or \
            not lse.is_contiguous():
        raise ValueError(f"{what}: lse must be a contiguous float32 tensor of [batch, heads, tokens]")
    _on(device, what, v_out, out, lse)
    v_out, out = _heads_last(v_out, what), _heads_last(out, what)
    gin = _nat.SxAttentionGradsIn(_view(out), lse.data_ptr(), _view(v_out))
    grads = tuple(torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k, v))
    gout = _nat.SxAttentionGrads(*(_view(t) for t in grads))
    entry = _nat.lib().sxcuda_attention_bwd
    with _at(device) as stream:
        ws, at, nbytes = _workspace(entry, device, ins)
        check(entry(C.byref(ins), C.byref(gin), C.byref(gout), at, C.byref(nbytes), stream))
    return grads


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, causal, q_lens, kv_lens):
        out, lse = attention_fwd(q, k, v, scale=scale, causal=causal, q_lens=q_lens, kv_lens=kv_lens)
        ctx.save_for_backward(q, k, v, out, lse, q_lens, kv_lens)
        ctx.how = {"scale": scale, "causal": causal}
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, v_out):
        q, k, v, out, lse, q_lens, kv_lens = ctx.saved_tensors
        grads = attention_bwd(v_out, q, k, v, out, lse, q_lens=q_lens, kv_lens=kv_lens, **ctx.how)
        return (*grads, None, None, None, None)


def attention(q, k, v, *, scale=None, causal=False, q_lens=None, kv_lens=None):
    """attention_fwd's output, differentiable in q, k and v."""
    return _Attention.apply(q, k, v, scale, causal, q_lens, kv_lens)


# ---------------------------------------------------------------- layer norm

def _rows(t: torch.Tensor, cols: int):
    """t as (tensor, rows, distance of rows): as it is where its rows are, else a copy."""
    if t.is_contiguous():
        return t, t.numel() // cols, cols
    if t.dim() != 2:
        t = t.reshape(-1, cols)
    if (cols > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < cols):
        t = t.contiguous()
    return t, t.shape[0], t.stride(0)


def _norm_inputs(what, x, weight, bias, eps):
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"{what}: x needs a last axis of at least 1, got {tuple(x.shape)}")
    cols, device, code = x.shape[-1], x.device, _dtype(x, what)
    _on(device, what, weight, bias)
    first = bias if weight is None else weight
    for p in (weight, bias):
        if p is not None and (p.shape != (cols,) or not p.is_contiguous() or p.dtype != first.dtype):
            raise ValueError(f"{what}: weight and bias must be contiguous tensors of [{cols}] with "
                             "one dtype")
    flat, rows, stride = _rows(x, cols)
    ins = _nat.SxLayerNormInputs(
        flat.data_ptr(), None if weight is None else weight.data_ptr(),
        None if bias is None else bias.data_ptr(), rows, cols, stride, code,
        _DTYPES[torch.float32] if first is None else _dtype(first, what), eps)
    return flat, ins, device, cols


def layer_norm_fwd(x, weight=None, bias=None, *, eps=1e-5):
    """Layer norm over the last axis: (y like x, mean, rstd of x.shape[:-1] in float32). weight and
    bias (each may be None: ones, zeros) have one dtype, which need not be x's."""
    flat, ins, device, cols = _norm_inputs("layer_norm_fwd", x, weight, bias, eps)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    mean = x.new_empty(x.shape[:-1], dtype=torch.float32)
    rstd = torch.empty_like(mean)
    with _at(device) as stream:
        check(_nat.lib().sxcuda_layer_norm_fwd(C.byref(ins), y.data_ptr(), cols, mean.data_ptr(),
                                               rstd.data_ptr(), stream))
    return y, mean, rstd


def layer_norm_bwd(v_y, x, weight, mean, rstd):
    """Gradients (v_x, v_weight, v_bias) of layer_norm_fwd; the weights' have the weight's dtype
    (float32 where weight is None). mean and rstd are the forward's. Deterministic."""
    what = "layer_norm_bwd"
    flat, ins, device, cols = _norm_inputs(what, x, weight, None, 0.0)
    if v_y.shape != x.shape or v_y.dtype != x.dtype:
        raise ValueError(f"{what}: v_y must be like x")
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.shape != x.shape[:-1] or t.dtype != torch.float32 or not t.is_contiguous():
            raise ValueError(f"{what}: {name} must be a contiguous float32 tensor of "
                             f"{tuple(x.shape[:-1])}")
    _on(device, what, v_y, mean, rstd)
    g, _, g_stride = _rows(v_y, cols)
    v_x = torch.empty_like(x, memory_format=torch.contiguous_format)
    v_w = torch.empty(cols, dtype=torch.float32, device=device) if weight is None else torch.empty_like(weight)
    v_b = torch.empty_like(v_w)
    gin = _nat.SxLayerNormGradsIn(mean.data_ptr(), rstd.data_ptr(), g.data_ptr(), g_stride)
    out = _nat.SxLayerNormGrads(v_x.data_ptr(), cols, v_w.data_ptr(), v_b.data_ptr())
    entry = _nat.lib().sxcuda_layer_norm_bwd
    with _at(device) as stream:
        ws, at, nbytes = _workspace(entry, device, ins)
        check(entry(C.byref(ins), C.byref(gin), C.byref(out), at, C.byref(nbytes), stream))
    return v_x, v_w, v_b


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_fwd(x, weight, bias, eps=eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.bias = bias is not None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, v_y):
        x, weight, mean, rstd = ctx.saved_tensors
        v_x, v_w, v_b = layer_norm_bwd(v_y, x, weight, mean, rstd)
        return v_x, None if weight is None else v_w, v_b if ctx.bias else None, None


def layer_norm(x, weight=None, bias=None, *, eps=1e-5):
    """layer_norm_fwd's y, differentiable in x, weight and bias."""
    return _LayerNorm.apply(x, weight, bias, float(eps))


# ---------------------------------------------------------------- linear layers

_ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}


def linear_status() -> int:
    """Status bits the linear and qk_norm_rotary kernels of the current device have set since the last
    call (0: all is well; 1: a bounded wait inside a kernel ran out and its outputs are invalid).
    Synchronises."""
    st = C.c_uint32(0)
    check(_nat.lib().sxcuda_linear_status(C.byref(st)))
    return int(st.value)


def _linear_inputs(what, x, weight, bias, activation):
    if activation not in _ACTIVATIONS:
        raise ValueError(f"{what}: activation must be one of {list(_ACTIVATIONS)}, got {activation!r}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError(f"{what}: x [..., in] and weight [out, in] needed, got {tuple(x.shape)} and "
                         f"{tuple(weight.shape)}")
    if weight.dtype != x.dtype:
        raise ValueError(f"{what}: x and weight must have one dtype, got {x.dtype} and {weight.dtype}")
    device, code = x.device, _dtype(x, what)
    n, cols = weight.shape
    _on(device, what, weight, bias)
    if bias is not None and (bias.shape != (n,) or not bias.is_contiguous()):
        raise ValueError(f"{what}: bias must be a contiguous tensor of [{n}]")
    flat, rows, x_stride = _rows(x, cols)
    w, _, w_stride = _rows(weight, cols)
    ins = _nat.SxLinearInputs(
        flat.data_ptr(), w.data_ptr(), None if bias is None else bias.data_ptr(), rows, cols, n, x_stride,
        w_stride, code, 0 if bias is None else _dtype(bias, what), _ACTIVATIONS[activation])
    return flat, w, ins, device


def linear_fwd(x, weight, bias=None, *, activation=None, residual=None, keep=False):
    """act(x weight^T + bias) + residual: (y [..., out], pre).

    x: [..., in]; weight: [out, in] of x's dtype (float32, float16 or bfloat16); bias: [out] of any of
    them; residual: like y. activation: None, "relu", "silu", "gelu" (with the normal distribution
    function) or "gelu_tanh" (its tanh form). Sums, bias, activation and residual are taken in 32 bits
    and rounded once. pre is x weight^T + bias rounded to x's dtype, which linear_bwd needs where there
    is an activation; None unless keep. 16-bit types run on the tensor cores."""
    what = "linear_fwd"
    flat, w, ins, device = _linear_inputs(what, x, weight, bias, activation)
    n = weight.shape[0]
    y = x.new_empty((*x.shape[:-1], n))
    pre = torch.empty_like(y) if keep else None
    out = _nat.SxLinearOutputs(None, 0, y.data_ptr(), n, pre.data_ptr() if keep else None, n)
    if residual is not None:
        if residual.shape != y.shape or residual.dtype != y.dtype:
            raise ValueError(f"{what}: residual must be like y, {y.dtype} of {tuple(y.shape)}")
        _on(device, what, residual)
        r, _, out.residual_stride = _rows(residual, n)
        out.residual = r.data_ptr()
    entry = _nat.lib().sxcuda_linear_fwd
    with _at(device) as stream:
        ws, at, nbytes = _space(device, entry, C.byref(ins), C.byref(out))
        check(entry(C.byref(ins), C.byref(out), at, C.byref(nbytes), stream))
    return y, pre


def _space(device, entry, *args):
    nbytes = C.c_size_t(0)
    check(entry(*args, None, C.byref(nbytes), None))
    if not nbytes.value:
        return None, 16, nbytes
    ws = torch.empty(nbytes.value, dtype=torch.uint8, device=device)
    return ws, ws.data_ptr(), nbytes


def linear_bwd(v_y, x, weight, bias=None, pre=None, *, activation=None, needs_x=True, needs_weight=True):
    """Gradients (v_x, v_weight, v_bias) of linear_fwd for the gradient v_y of its y (which is also the
    residual's). pre is the forward's, needed with an activation and only then. v_bias is like bias, None
    without one; v_x and v_weight are None where they are not needed. v_y act'(pre) is rounded to x's dtype
    before the products with x and weight, not before its sum. Deterministic."""
    what = "linear_bwd"
    flat, w, ins, device = _linear_inputs(what, x, weight, bias, activation)
    n = weight.shape[0]
    if v_y.shape != (*x.shape[:-1], n) or v_y.dtype != x.dtype:
        raise ValueError(f"{what}: v_y must be {x.dtype} of {(*x.shape[:-1], n)}")
    if (pre is None) != (activation is None):
        raise ValueError(f"{what}: pre is needed with an activation, and only then")
    _on(device, what, v_y, pre)
    g, _, g_stride = _rows(v_y, n)
    gin = _nat.SxLinearGradsIn(g.data_ptr(), g_stride, None, n)
    if pre is not None:
        if pre.shape != v_y.shape or pre.dtype != v_y.dtype:
            raise ValueError(f"{what}: pre must be like v_y")
        z, _, gin.pre_stride = _rows(pre, n)
        gin.pre = z.data_ptr()
    v_x = torch.empty_like(x, memory_format=torch.contiguous_format) if needs_x else None
    v_w = torch.empty_like(weight, memory_format=torch.contiguous_format) if needs_weight else None
    v_b = None if bias is None else torch.empty_like(bias)
    cols = weight.shape[1]
    out = _nat.SxLinearGrads(v_x.data_ptr() if needs_x else None, cols,
                             v_w.data_ptr() if needs_weight else None, cols,
                             None if v_b is None else v_b.data_ptr())
    entry = _nat.lib().sxcuda_linear_bwd
    with _at(device) as stream:
        ws, at, nbytes = _space(device, entry, C.byref(ins), C.byref(gin), C.byref(out))
        check(entry(C.byref(ins), C.byref(gin), C.byref(out), at, C.byref(nbytes), stream))
    return v_x, v_w, v_b


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        keep = activation is not None and any(ctx.needs_input_grad[:3])
        y, pre = linear_fwd(x, weight, bias, activation=activation, residual=residual, keep=keep)
        ctx.save_for_backward(x, weight, bias, pre)
        ctx.activation = activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, v_y):
        x, weight, bias, pre = ctx.saved_tensors
        needs = ctx.needs_input_grad
        v_x = v_w = v_b = None
        if any(needs[:3]):
            v_x, v_w, v_b = linear_bwd(v_y, x, weight, bias if needs[2] else None, pre,
                                       activation=ctx.activation, needs_x=needs[0], needs_weight=needs[1])
        return v_x, v_w, v_b, v_y if needs[3] else None, None


def linear(x, weight, bias=None, *, activation=None, residual=None):
    """linear_fwd's y, differentiable in x, weight, bias and residual. Without gradients to come (no_grad, inference
    mode, inputs that need none) nothing is kept for them."""
    if not torch.is_grad_enabled():  # needs_input_grad does not say: it goes by the inputs alone
        return linear_fwd(x, weight, bias, activation=activation, residual=residual)[0]
    return _Linear.apply(x, weight, bias, residual, activation)


# ---------------------------------------------------------------- norm and rotation of queries and keys

_PAIRS = {"axis": 0, "whole": 1, "neighbours": 2}
_POSITIONS = {torch.float32: 0, torch.int32: 1, torch.int64: 2}


_Four = C.c_int32 * 4


@functools.lru_cache(maxsize=64)
def _ladder(axes, base):
    """The pairs' frequencies base^(-2 j / dim), pair j of each axis, as a C array that is only read."""
    freqs = [base ** (-2.0 * j / d) for d in axes for j in range(d // 2)]
    return (C.c_double * max(len(freqs), 1))(*freqs)


@functools.lru_cache(maxsize=64)
def _axes_for(axes, d):
    """The axes as C has them; None where they do not fit heads of d values."""
    if not 1 <= len(axes) <= 4 or any(a < 0 or a % 2 for a in axes) or sum(axes) > d:
        return None
    return _Four(*axes)


@functools.lru_cache(maxsize=256)
def _rotary_space(index, d, norm):
    """Bytes of the backward's workspace, which the device, the head's size and norm decide."""
    ins = _nat.SxRotaryInputs(batch=0, tokens=0, q_heads=1, head_dim=d, axes=1, norm=norm)
    nbytes = C.c_size_t(0)
    check(_nat.lib().sxcuda_qk_norm_rotary_bwd(C.byref(ins), None, None, C.byref(nbytes), None))
    return nbytes.value


def _freqs(what, axes, base, freqs):
    if freqs is not None:
        if len(freqs) != sum(axes) // 2:
            raise ValueError(f"{what}: {sum(axes) // 2} freqs needed, got {len(freqs)}")
        return (C.c_double * max(len(freqs), 1))(*[float(f) for f in freqs])
    if not (isinstance(base, (int, float)) and base > 0 and math.isfinite(base)):
        raise ValueError(f"{what}: base must be a number above zero")
    return _ladder(axes, float(base))


def _head_rows(t, what):
    if t.dim() != 4:
        raise ValueError(f"{what}: [batch, tokens, heads, head_dim] needed, got {tuple(t.shape)}")
    return t.contiguous() if t.stride(3) != 1 and t.shape[3] != 1 else t


def _rotary_inputs(what, q, k, positions, axes, base, freqs, pairs, norm, q_weight, k_weight, eps):
    q = _head_rows(q, what)
    b, n, h, d = q.shape
    code, device = _dtype(q, what), q.device
    if k is not None:
        k = _head_rows(k, what)
        if k.dtype != q.dtype or k.shape[:2] != q.shape[:2] or k.shape[3] != d:
            raise ValueError(f"{what}: k must be {q.dtype} of [{b}, {n}, heads, {d}], got {k.dtype} of "
                             f"{tuple(k.shape)}")
    elif k_weight is not None:
        raise ValueError(f"{what}: k_weight needs k")
    if pairs not in _PAIRS:
        raise ValueError(f"{what}: pairs must be one of {list(_PAIRS)}")
    axes = tuple(map(int, axes))
    c_axes = _axes_for(axes, d)
    if c_axes is None:
        raise ValueError(f"{what}: axes must be 1 to 4 even numbers of values, at most {d} together, got {axes}")
    code_at = _POSITIONS.get(positions.dtype)
    if code_at is None:
        raise ValueError(f"{what}: positions must be float32, int32 or int64, got {positions.dtype}")
    if positions.requires_grad:
        raise ValueError(f"{what}: positions get no gradient: detach() them")
    if positions.shape not in ((b, n, len(axes)), (n, len(axes))):
        raise ValueError(f"{what}: positions must be [{b}, {n}, {len(axes)}] or [{n}, {len(axes)}], got "
                         f"{tuple(positions.shape)}")
    first = k_weight if q_weight is None else q_weight
    for w in (q_weight, k_weight):
        if w is not None and (not norm or w.shape != (d,) or not w.is_contiguous() or w.dtype != first.dtype):
            raise ValueError(f"{what}: q_weight and k_weight need norm and must be contiguous tensors of "
                             f"[{d}] with one dtype")
    _on(device, what, k, positions, q_weight, k_weight)
    at = positions.stride()
    table = _freqs(what, axes, base, freqs)
    ins = _nat.SxRotaryInputs(
        _view(q), _view(q) if k is None else _view(k), positions.data_ptr(), at[0] if len(at) == 3 else 0,
        at[-2], at[-1], C.addressof(table), None if q_weight is None else q_weight.data_ptr(),
        None if k_weight is None else k_weight.data_ptr(), b, n, h, 0 if k is None else k.shape[2], d,
        len(axes), c_axes, _PAIRS[pairs], code, 0 if first is None else _dtype(first, what),
        code_at, bool(norm), eps)
    return q, k, ins, device, table


def qk_norm_rotary_fwd(q, k, positions, *, axes, base=10000.0, freqs=None, pairs="axis", norm=True,
                       q_weight=None, k_weight=None, eps=1e-6):
    """Queries and keys normalised per head, x / sqrt(mean x^2 + eps) * weight, and rotated by the
    positions of their tokens: (q, k) as new tensors.

    q: [batch, tokens, heads, head_dim]; k: the same with heads of its own, or None; float32, float16 or
    bfloat16, head_dim up to 256, any strides with the last axis contiguous (views of a joint projection).
    positions: [batch, tokens, axes] or [tokens, axes] in float32, int32 or int64: places in an image
    (row, column), a video (time, row, column), a scene (x, y, z), or one number; they get no gradient.
    axes: how many values of a head each axis rotates, in pairs; those behind the sum are not rotated.
    Pair j of an axis with d values turns by position * base^(-2 j / d), or by position * freqs[i], i
    counting the pairs of all axes. pairs: which values are one: "axis": j and j + d / 2 of the axis' own
    run of values; "whole": i and i + sum(axes) / 2; "neighbours": 2 i and 2 i + 1. norm=False only
    rotates. q_weight, k_weight: [head_dim], None for ones. Positions are taken as float64, angles to 2^-28
    of a turn up to 2^76 turns (from 2^80 on as 0)."""
    what = "qk_norm_rotary_fwd"
    q, k, ins, device, table = _rotary_inputs(what, q, k, positions, axes, base, freqs, pairs, norm,
                                              q_weight, k_weight, eps)
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_out = None if k is None else torch.empty_like(k, memory_format=torch.contiguous_format)
    qv = _nat.SxAttentionView(*_view(q_out))
    kv = None if k is None else C.byref(_nat.SxAttentionView(*_view(k_out)))
    with _at(device) as stream:
        check(_nat.lib().sxcuda_qk_norm_rotary_fwd(C.byref(ins), C.byref(qv), kv, stream))
    return q_out, k_out


def qk_norm_rotary_bwd(v_q_out, v_k_out, q, k, positions, *, axes, base=10000.0, freqs=None, pairs="axis",
                       norm=True, q_weight=None, k_weight=None, eps=1e-6):
    """Gradients (v_q, v_k, v_q_weight, v_k_weight) of qk_norm_rotary_fwd for the gradients of its
    outputs; None for what was not given. Deterministic."""
    what = "qk_norm_rotary_bwd"
    q, k, ins, device, table = _rotary_inputs(what, q, k, positions, axes, base, freqs, pairs, norm,
                                              q_weight, k_weight, eps)
    if (v_k_out is None) != (k is None):
        raise ValueError(f"{what}: v_k_out is needed with k, and only then")
    grads = []
    for name, g, t in (("v_q_out", v_q_out, q), ("v_k_out", v_k_out, k)):
        if t is not None and (g.shape != t.shape or g.dtype != t.dtype):
            raise ValueError(f"{what}: {name} must be {t.dtype} of {tuple(t.shape)}")
        grads.append(None if t is None else _head_rows(g, what))
    _on(device, what, *grads)
    outs = [None if t is None else torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k)]
    d = q.shape[3]
    v_w = [None if w is None else torch.empty_like(w) for w in (q_weight, k_weight)]
    none = (None, 0, 0, 0)
    g = _nat.SxRotaryGrads(*(none if t is None else _view(t) for t in (*grads, *outs)),
                           *(None if w is None else w.data_ptr() for w in v_w))
    with _at(device) as stream:
        nbytes = C.c_size_t(_rotary_space(device.index, d, bool(norm)))
        ws = torch.empty(nbytes.value, dtype=torch.uint8, device=device) if nbytes.value else None
        check(_nat.lib().sxcuda_qk_norm_rotary_bwd(C.byref(ins), C.byref(g), 16 if ws is None else ws.data_ptr(),
                                                   C.byref(nbytes), stream))
    return (*outs, *v_w)


class _QkNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, q_weight, k_weight, how):
        ctx.save_for_backward(q, k, positions, q_weight, k_weight)
        ctx.how = how
        return qk_norm_rotary_fwd(q, k, positions, q_weight=q_weight, k_weight=k_weight, **how)

    @staticmethod
    @once_differentiable
    def backward(ctx, v_q_out, v_k_out):
        q, k, positions, q_weight, k_weight = ctx.saved_tensors
        v_q, v_k, v_qw, v_kw = qk_norm_rotary_bwd(v_q_out, None if k is None else v_k_out, q, k, positions,
                                                  q_weight=q_weight, k_weight=k_weight, **ctx.how)
        return v_q, v_k, None, v_qw, v_kw, None


def qk_norm_rotary(q, k, positions, *, axes, base=10000.0, freqs=None, pairs="axis", norm=True,
                   q_weight=None, k_weight=None, eps=1e-6):
    """qk_norm_rotary_fwd's (q, k), differentiable in q, k and the weights."""
    # as they are now: the backward must not see what a caller makes of its lists meanwhile
    freqs = None if freqs is None else tuple(map(float, freqs))
    how = {"axes": tuple(axes), "base": base, "freqs": freqs, "pairs": pairs, "norm": norm, "eps": eps}
    return _QkNormRotary.apply(q, k, positions, q_weight, k_weight, how)


# ---------------------------------------------------------------- AdamW

_TENSOR = np.dtype(_nat.SxAdamwTensor)


class AdamW:
    """AdamW (decoupled weight decay, bias correction) over all parameters in one launch. Each parameter
    counts its own steps, which its bias correction goes by: one without a gradient is skipped and does
    not count. (Parameters with different counts take a launch for each count.)

    params: tensors, or dicts {"params": [...], "lr": ..., "weight_decay": ...} for groups with a
    rate or decay of their own (other keys are refused). They must be contiguous CUDA tensors of
    one device. Moments are held in 32 bits, or with state_bits=8 as e4m3 codes of m and of sqrt(v)
    with a float32 scale for every 256 values (2.03 bytes for a value's two moments in place of 8).

    state: moments to go on from, {"exp_avg": [...], "exp_avg_sq": [...], "step": n} and, with 8
    bits, "exp_avg_scale" and "exp_avg_sq_scale", one tensor per parameter in order; the tensors are
    used and updated in place. n: the steps taken, one number or one per parameter. ``state()`` returns
    them."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *,
                 state_bits=32, state=None):
        what = "AdamW"
        if state_bits not in (8, 32):
            raise ValueError(f"{what}: state_bits must be 8 or 32")
        groups = [] if isinstance(params, (torch.Tensor, dict)) else list(params)
        if groups and not any(isinstance(g, dict) for g in groups):
            groups = [{"params": groups}]
        self.params, rates, decays = [], [], []
        for g in groups:
            if not isinstance(g, dict) or "params" not in g:
                raise ValueError(f"{what}: params are tensors, or dicts that each have 'params'")
            if unknown := set(g) - {"params", "lr", "weight_decay"}:
                raise ValueError(f"{what}: a group has an lr and a weight_decay of its own, no "
                                 f"{', '.join(map(str, unknown))}")
            mine = [None] if isinstance(g["params"], torch.Tensor) else list(g["params"])
            if not all(isinstance(p, torch.Tensor) for p in mine):
                raise ValueError(f"{what}: params must be a sequence of tensors")
            self.params += mine
            rates += [float(g.get("lr", lr))] * len(mine)
            decays += [float(g.get("weight_decay", weight_decay))] * len(mine)
        if not self.params:
            raise ValueError(f"{what}: no parameters")
        self.device = self.params[0].device
        _on(self.device, what, *self.params)
        for p in self.params:
            _dtype(p, what)
            if not p.is_contiguous():
                raise ValueError(f"{what}: parameters must be contiguous")
        self._kept = self._facts()
        self.bits = state_bits
        self._cfg = _nat.SxAdamwConfig(float(betas[0]), float(betas[1]), float(eps), 1.0, 0,
                                       state_bits)
        self._state = self._bind(what, state)
        self._at = [p.data_ptr() for p in self.params]
        self._apart(what)
        n = len(self.params)
        self._table = np.zeros(n, dtype=_TENSOR)
        self._table["n"] = [p.numel() for p in self.params]
        self._table["param_dtype"] = [_DTYPES[p.dtype] for p in self.params]
        self._table["lr"], self._table["weight_decay"] = rates, decays
        for key, tensors in self._state.items():
            self._table[key] = [t.data_ptr() for t in tensors]

    def _bind(self, what, state):
        eight = self.bits == 8
        kinds = {"exp_avg": torch.float8_e4m3fn if eight else torch.float32}
        kinds["exp_avg_sq"] = kinds["exp_avg"]
        if eight:
            kinds["exp_avg_scale"] = kinds["exp_avg_sq_scale"] = torch.float32
        if state is not None and set(state) != {*kinds, "step"}:
            raise ValueError(f"{what}: state needs {sorted({*kinds, 'step'})}")
        taken = 0 if state is None else state["step"]
        taken = list(taken) if isinstance(taken, (list, tuple)) else [taken] * len(self.params)
        if len(taken) != len(self.params) or any(int(t) < 0 for t in taken):
            raise ValueError(f"{what}: step must be a number of at least 0, or one per parameter")
        self._steps = np.array([int(t) for t in taken], dtype=np.int64)
        self._even = bool((self._steps == self._steps[0]).all())  # one count, which a step need not sort
        mine = {}
        for key, dtype in kinds.items():
            sizes = [-(-p.numel() // RUN) if key.endswith("scale") else p.numel()
                     for p in self.params]
            if state is None:
                mine[key] = [torch.zeros(n, dtype=dtype, device=self.device) for n in sizes]
                continue
            mine[key] = list(state[key])
            if len(mine[key]) != len(sizes):
                raise ValueError(f"{what}: {key} needs {len(sizes)} tensors")
            for t, n in zip(mine[key], sizes):
                if t.dtype != dtype or t.numel() != n or not t.is_contiguous() or \
                        t.device != self.device:
                    raise ValueError(f"{what}: {key} needs contiguous {dtype} tensors of the "
                                     "parameters' sizes and device")
            # the kernel has their addresses: tensors of the optimiser's own hold that memory, whatever
            # the caller gives its own tensors or lists later
            mine[key] = [t.detach() for t in mine[key]]
        return mine

    def _apart(self, what):
        """Refuses parameters and moments that share memory: CTAs would update it without order."""
        spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size())
                       for ts in (self.params, *self._state.values()) for t in ts if t.numel())
        if any(start < end for (_, end), (start, _) in zip(spans, spans[1:])):
            raise ValueError(f"{what}: parameters or moments overlap in memory, or one is given more "
                             "than once")

    def _facts(self) -> list:
        """What a step relies on of the parameters, which may have been given other memory since."""
        return [[p.numel() for p in self.params], [p.dtype for p in self.params]]

    def state(self) -> dict:
        """The moments (views of what the next step updates) and the number of steps taken, as the
        constructor takes them: one number where it is the same for every parameter, else one per
        parameter."""
        taken = self._steps.tolist()
        return {**{key: [t.detach() for t in ts] for key, ts in self._state.items()},
                "step": taken[0] if len(set(taken)) == 1 else taken}

    def set_lr(self, lr):
        """The learning rate of the next steps: a number, or one per parameter."""
        self._table["lr"] = lr

    def step(self, grads=None, *, grad_scale=1.0):
        """One step on `grads` (one per parameter) or on the parameters' .grad; parameters whose
        gradient is None stay as they are. grad_scale multiplies every gradient. Not to be captured in
        a graph (RuntimeError): a step's number and bias corrections are arguments of its launch."""
        what = "AdamW.step"
        grads = [p.grad for p in self.params] if grads is None else list(grads)
        if len(grads) != len(self.params):
            raise ValueError(f"{what}: {len(self.params)} gradients needed, got {len(grads)}")
        params = self.params
        if self._facts() != self._kept or not all([p.is_contiguous() for p in params]):
            raise ValueError(f"{what}: a parameter's size, dtype, device or layout has changed")
        table, at = self._table, [p.data_ptr() for p in params]
        if at != self._at:  # an address says which device it is on, too
            _on(self.device, what, *params)
            self._apart(what)
            self._at = at
        table["param"] = at
        there = [i for i, g in enumerate(grads) if g is not None]
        if len(there) < len(grads):
            params, grads = [params[i] for i in there], [grads[i] for i in there]
            table = np.ascontiguousarray(table[there])
        kinds, index = [_DTYPES.get(g.dtype) for g in grads], self.device.index
        if None in kinds or [g.shape for g in grads] != [p.shape for p in params] or \
                not all([g.is_contiguous() and g.get_device() == index for g in grads]):
            raise ValueError(f"{what}: a gradient must be a contiguous float32, float16 or bfloat16 "
                             "tensor of its parameter's shape and device")
        table["grad"], table["grad_dtype"] = [g.data_ptr() for g in grads], kinds
        self._cfg.grad_scale = float(grad_scale)
        if self._even and len(there) == len(self.params):
            launches = {int(self._steps[0]) + 1: slice(None)}
        else:
            numbers, there = self._steps[there] + 1, np.array(there, dtype=np.intp)
            launches = {n: np.flatnonzero(numbers == n) for n in sorted(set(numbers.tolist()))}
            if len(launches) > 1 and not np.isfinite([table["lr"], table["weight_decay"]]).all():
                raise ValueError(f"{what}: lr and weight_decay must be finite")  # before the first
            self._even = False
        with _at(self.device) as stream:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"{what}: a step cannot be captured in a graph: every replay would "
                                   "be the same step, with its bias corrections")
            for number, mine in launches.items():
                some = len(launches) > 1
                rows = np.ascontiguousarray(table[mine]) if some else table
                self._cfg.step = number
                check(_nat.lib().sxcuda_adamw_step(rows.ctypes.data, len(rows), C.byref(self._cfg),
                                                   stream))
                self._steps[slice(None) if self._even else there[mine]] = number
                # autograd's check of saved tensors sees that the parameters are not what they were
                torch.autograd.graph.increment_version([params[i] for i in mine] if some else params)
        self._even = self._even or bool((self._steps == self._steps[0]).all())
