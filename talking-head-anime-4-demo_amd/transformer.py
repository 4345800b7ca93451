"""Operators of a transformer block over token sequences, at inference, on the GPU: what the posers' networks have inside (attention, normalisation +
FiLM + residual, reduced-precision matrix products), for sequences of any length, prompts and single tokens over a cache.

``quantize_tokens``         tokens (or weight rows) to int8 with one scale each
``int8_linear``             int8 x int8 matrix product with scales for each token and channel
``residual_norm``           the norms behind and in front of a block, with its gate and the residual sum
``differential_attention``  the difference of two softmax maps with learned weights

All of them enqueue on ``torch.cuda.current_stream()`` of their tensors' device, never synchronise, and can be captured into a graph.  Wrong arguments raise
AssertionError here or ``_capi.Tha4Error`` from the C ABI (include/tha4_hip.h); nothing falls back to another implementation.  They are forward
operators: tensors that require gradients are refused while gradients are enabled.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Tuple, Union

import torch
from torch import Tensor

from . import _capi

_DTYPES = {torch.float32: _capi.F32, torch.float16: _capi.F16, torch.bfloat16: _capi.BF16}
_ONE_ROW = 2 ** 63 - 1


def _stream(t: Tensor):
    return torch.cuda.current_stream(t.device).cuda_stream


def _check(condition: bool, message: str) -> None:
    if not condition:
        raise AssertionError(message)


def _check_tensors(device: torch.device, **tensors: Optional[Tensor]) -> None:
    for name, t in tensors.items():
        if t is None:
            continue
        if not t.is_cuda:
            raise AssertionError(f"{name} must be on the GPU")
        if t.device != device:
            raise AssertionError(f"{name} is on {t.device}, the first argument on {device}")
        if t.requires_grad and torch.is_grad_enabled():
            raise AssertionError(f"{name} requires a gradient: this is a forward operator (use torch.no_grad())")


def _rows(t: Tensor) -> Tensor:
    """[..., c] -> [rows, c] with contiguous rows; a copy only where the strides leave no other way."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.shape[1] <= 1 or t.stride(1) == 1 else t.contiguous()


def _stride(t: Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _pointer(t: Optional[Tensor]):
    return None if t is None else t.data_ptr()


def quantize_tokens(x: Tensor) -> Tuple[Tensor, Tensor]:
    """x [..., c] fp32 / fp16 / bf16 -> (int8 [..., c], fp32 scales [...]): ``q = x / scale`` rounded to the nearest integer (ties to even), ``scale = max |x| / 127``.
    A row of zeros gets scale 0; a row that holds an infinity or a NaN gets scale NaN (products with it are NaN) and zeros.
    Weights [n, c] are quantised for each channel by the same call."""
    lib = _capi.load_library()
    _check(x.dim() >= 1 and x.shape[-1] >= 1 and x.dtype in _DTYPES, "x must be a float32, float16 or bfloat16 tensor [..., c] with c >= 1")
    _check_tensors(x.device, x=x)
    rows = _rows(x)
    q = torch.empty(rows.shape, dtype=torch.int8, device=x.device)
    scale = torch.empty(rows.shape[0], dtype=torch.float32, device=x.device)
    _capi.check(lib, lib.tha4_quantize_tokens_i8(rows.data_ptr(), _DTYPES[x.dtype], rows.shape[0], rows.shape[1], _stride(rows), q.data_ptr(), rows.shape[1],
                                                 scale.data_ptr(), _stream(x)), "tha4_quantize_tokens_i8")
    return q.view(x.shape), scale.view(x.shape[:-1])


def int8_linear(x: Tensor, weight: Tensor, weight_scale: Tensor, *, x_scale: Optional[Tensor] = None, bias: Optional[Tensor] = None,
                out_dtype: Optional[torch.dtype] = None) -> Tensor:
    """x [..., k] times int8 weight [n, k] with fp32 weight_scale [n] -> [..., n]: ``y = x_scale weight_scale (x_q . weight) + bias``.

    x is float (quantised for each token on the way, as by ``quantize_tokens``; the result has its type unless ``out_dtype`` says otherwise) or int8 with
    fp32 ``x_scale`` [...] (then ``out_dtype`` is needed).  The sums are exact 32-bit integers (k <= 131071), scaled in fp32 and rounded once."""
    lib = _capi.load_library()
    _check(weight.dim() == 2 and weight.dtype == torch.int8 and weight.shape[1] >= 1, "weight must be an int8 tensor [n, k] with k >= 1")
    n, k = weight.shape
    _check(x.dim() >= 1 and x.shape[-1] == k, f"x must be [..., {k}]")
    _check(weight_scale.dtype == torch.float32 and weight_scale.shape == (n,), f"weight_scale must be a float32 tensor [{n}]")
    _check(bias is None or (bias.dtype == torch.float32 and bias.shape == (n,)), f"bias must be a float32 tensor [{n}]")
    _check_tensors(x.device, x=x, weight=weight, weight_scale=weight_scale, x_scale=x_scale, bias=bias)
    if x.dtype == torch.int8:
        _check(x_scale is not None and x_scale.dtype == torch.float32 and x_scale.shape == x.shape[:-1], "int8 x needs a float32 x_scale [...]")
        _check(out_dtype in _DTYPES, "int8 x needs an out_dtype of float32, float16 or bfloat16")
        q, scale = _rows(x), x_scale.reshape(-1).contiguous()
    else:
        _check(x_scale is None, "x_scale belongs to an int8 x")
        out_dtype = out_dtype or x.dtype
        _check(x.dtype in _DTYPES and out_dtype in _DTYPES, "x and out_dtype must be float32, float16 or bfloat16 (or x int8)")
        q, scale = quantize_tokens(_rows(x))
    w = weight if weight.stride(1) == 1 or k == 1 else weight.contiguous()
    weight_scale = weight_scale.contiguous()
    bias = None if bias is None else bias.contiguous()
    m = q.shape[0]
    y = torch.empty((m, n), dtype=out_dtype, device=x.device)
    args = _capi.Tha4LinearI8Args(q.data_ptr(), scale.data_ptr(), w.data_ptr(), weight_scale.data_ptr(), _pointer(bias), y.data_ptr(),
                                  m, n, k, _stride(q), _stride(w), n, _DTYPES[out_dtype])
    _capi.check(lib, lib.tha4_linear_i8(C.byref(args), _stream(x)), "tha4_linear_i8")
    return y.view(x.shape[:-1] + (n,))


def _per_row(t: Optional[Tensor], name: str, shape, cols: int) -> Tuple[Optional[Tensor], int, int]:
    """A vector [c], a tensor [samples, c] / [samples, 1, .., c] or a full [..., c] -> (rows, their stride, rows of the input for each)."""
    if t is None:
        return None, 0, 1
    _check(t.dim() >= 1 and t.shape[-1] == cols, f"{name} must be [..., {cols}]")
    rows = math.prod(shape[:-1])
    if t.dim() > 2 and math.prod(t.shape[1:-1]) == 1:
        t = t.reshape(t.shape[0], cols)
    t = _rows(t)
    have = t.shape[0]
    if have == 1:
        return t, cols, _ONE_ROW
    _check(have > 0 and rows % have == 0 and (have == rows or (len(shape) > 1 and have == shape[0]) or len(shape) == 2),
           f"{name} must have one row, one for each sample or one for each token")
    return t, _stride(t), max(rows // have, 1)


def residual_norm(residual: Tensor, branch: Optional[Tensor] = None, *, gate: Optional[Tensor] = None, gate_activation: str = "none",
                  residual_scale: Union[float, Tensor] = 1.0, post_norm: str = "rms", post_weight: Optional[Tensor] = None, post_bias: Optional[Tensor] = None,
                  pre_norm: str = "rms", pre_weight: Optional[Tensor] = None, pre_bias: Optional[Tensor] = None,
                  film: Optional[Tuple[Tensor, Tensor]] = None, eps: float = 1e-5) -> Tuple[Tensor, Tensor]:
    """What lies between two blocks of a transformer, in one pass:

        h = residual_scale * residual + act(gate) * (post_norm(branch) * post_weight + post_bias)
        y = (pre_norm(h) * pre_weight + pre_bias) * (1 + film[0]) + film[1]

    residual, branch [..., c]; returns (h, y): the residual stream, in residual's type, and the next block's input, in branch's.  ``branch`` None: in front of the first
    block.  Norms are "rms", "layer" or "none", with their statistics (and y) in fp32 from the unrounded h.  residual_scale: a number or a vector [c].
    gate: [c], one row for each sample ([samples, c]; the first dimension of residual, or consecutive equal shares of its rows) or for each token; activation "none" or
    "sigmoid".  film: (scale, shift), shaped like a gate.  Types: branch fp32 / fp16 / bf16; residual and gate that or fp32; vectors and film all that or all fp32."""
    lib = _capi.load_library()
    _check(residual.dim() >= 1 and residual.shape[-1] >= 1, "residual must be [..., c] with c >= 1")
    shape, cols = residual.shape, residual.shape[-1]
    dtype = residual.dtype if branch is None else branch.dtype
    _check(dtype in _DTYPES and residual.dtype in (dtype, torch.float32), "branch must be float32, float16 or bfloat16, and residual that type or float32")
    _check(branch is None or branch.shape == shape, f"branch must have residual's shape {tuple(shape)}")
    _check(post_norm in _capi.NORM_KINDS and pre_norm in _capi.NORM_KINDS, f"post_norm / pre_norm must be one of {sorted(_capi.NORM_KINDS)}")
    _check(gate_activation in _capi.GATE_ACTIVATIONS, f"gate_activation must be one of {sorted(_capi.GATE_ACTIVATIONS)}")
    _check(gate is None or gate.dtype in (dtype, torch.float32), "gate must have branch's type or float32")
    _check(film is None or (len(film) == 2 and film[0].shape == film[1].shape), "film must be (scale, shift) of one shape")
    vector = residual_scale if isinstance(residual_scale, Tensor) else None
    film_s, film_t = film if film is not None else (None, None)
    vectors = {"residual_scale": vector, "post_weight": post_weight, "post_bias": post_bias, "pre_weight": pre_weight, "pre_bias": pre_bias}
    for name, v in vectors.items():
        _check(v is None or v.shape == (cols,), f"{name} must be a vector [{cols}]")
    types = {v.dtype for v in list(vectors.values()) + [film_s, film_t] if v is not None}
    _check(len(types) <= 1 and types <= {dtype, torch.float32}, "vectors and film must all be float32 or all of branch's type")
    _check_tensors(residual.device, residual=residual, branch=branch, gate=gate, film_scale=film_s, film_shift=film_t, **vectors)
    vector, post_weight, post_bias, pre_weight, pre_bias = (None if v is None else v.contiguous() for v in vectors.values())
    gate, gate_stride, gate_rows = _per_row(gate, "gate", shape, cols)
    if film is not None:
        if film_s.stride() != film_t.stride():
            film_s, film_t = film_s.contiguous(), film_t.contiguous()
    film_s, film_stride, film_rows = _per_row(film_s, "film", shape, cols)
    film_t = _per_row(film_t, "film", shape, cols)[0]
    r = _rows(residual)
    b = None if branch is None else _rows(branch)
    rows = r.shape[0]
    h = torch.empty((rows, cols), dtype=residual.dtype, device=residual.device)
    y = torch.empty((rows, cols), dtype=dtype, device=residual.device)
    args = _capi.Tha4ResidualNormArgs(
        r.data_ptr(), _pointer(b), _pointer(gate), _pointer(vector), _pointer(post_weight), _pointer(post_bias), _pointer(pre_weight), _pointer(pre_bias),
        _pointer(film_s), _pointer(film_t), h.data_ptr(), y.data_ptr(), rows, cols, _stride(r), 0 if b is None else _stride(b), gate_stride, film_stride, cols, cols,
        gate_rows, film_rows, _DTYPES[dtype], _DTYPES[residual.dtype], _DTYPES[dtype if gate is None else gate.dtype], _DTYPES[types.pop() if types else torch.float32],
        _capi.NORM_KINDS[post_norm], _capi.NORM_KINDS[pre_norm], _capi.GATE_ACTIVATIONS[gate_activation], 1.0 if vector is not None else float(residual_scale), eps)
    _capi.check(lib, lib.tha4_residual_norm(C.byref(args), _stream(residual)), "tha4_residual_norm")
    return h.view(shape), y.view(shape)


def _heads(t: Tensor, name: str) -> Tensor:
    """A 16-byte-aligned view (or, where the strides do not allow one, copy) with contiguous rows."""
    if t.stride(3) != 1 or any(s % 8 for s, n in zip(t.stride()[:3], t.shape) if n > 1) or t.data_ptr() % 16:
        return t.contiguous()
    return t


def _strides(t: Tensor):
    return tuple(s if n > 1 else 0 for s, n in zip(t.stride()[:3], t.shape))


def differential_attention(q: Tensor, k: Tensor, v: Tensor, lambda_vectors: Tensor, lambda_init: float, *, causal: bool = False,
                           q_lengths: Optional[Tensor] = None, kv_lengths: Optional[Tensor] = None, mask: Optional[Tensor] = None, scale: Optional[float] = None,
                           norm: bool = True, norm_weight: Optional[Tensor] = None, eps: float = 1e-5, out: Optional[Tensor] = None) -> Tensor:
    """``softmax(scale q1 k1^T) v - lambda softmax(scale q2 k2^T) v`` with ``lambda = exp(l0 . l1) - exp(l2 . l3) + lambda_init``, then (``norm``)
    ``(1 - lambda_init) * o / sqrt(mean(o^2) + eps) * norm_weight`` over the value columns of each head.

    q [batch, q_len, 2 heads, d], k [batch, k_len, 2 kv_heads, d] (maps 1 and 2 of head h at 2h and 2h + 1), v [batch, k_len, kv_heads, 2d] fp16 or bf16, d 32, 64
    or 128, heads a multiple of kv_heads -> [batch, q_len, heads, 2d].  Any strides with contiguous rows of d (views of a fused projection or of a longer
    cache).  lambda_vectors fp32 [4, d] or [4, heads, d].  scale: 1 / sqrt(d).

    kv_lengths int32 [batch]: the valid keys of each sequence (what lies behind them is never read into a result); q_lengths int32 [batch]: its valid queries - rows
    behind them are zero, or left as they are in a given ``out``.  causal: the last valid query sees the last valid key.  mask: bool, broadcastable to
    [batch, heads, q_len, k_len], True = visible.  A query that sees no key answers zero.  k_len may be 0."""
    lib = _capi.load_library()
    _check(q.dim() == 4 and k.dim() == 4 and v.dim() == 4, "q, k and v must be [batch, tokens, heads, d]")
    _check(q.dtype in (torch.float16, torch.bfloat16) and k.dtype == q.dtype and v.dtype == q.dtype, "q, k and v must all be float16 or all bfloat16")
    batch, q_len, heads2, d = q.shape
    k_len, kv2 = k.shape[1], k.shape[2]
    _check(d in (32, 64, 128), "the head dimension must be 32, 64 or 128")
    _check(heads2 > 0 and kv2 > 0 and heads2 % 2 == 0 and kv2 % 2 == 0 and heads2 % kv2 == 0, "q and k must hold pairs of heads, q a multiple of k's")
    _check(k.shape == (batch, k_len, kv2, d) and v.shape == (batch, k_len, kv2 // 2, 2 * d), "k must be [batch, k_len, 2 kv_heads, d] and v [batch, k_len, kv_heads, 2 d]")
    heads = heads2 // 2
    _check(lambda_vectors.dtype == torch.float32 and lambda_vectors.shape in ((4, d), (4, heads, d)), f"lambda_vectors must be float32 [4, {d}] or [4, {heads}, {d}]")
    _check(norm_weight is None or (norm and norm_weight.dtype == torch.float32 and norm_weight.shape == (2 * d,)), f"norm_weight must be float32 [{2 * d}] (with norm)")
    for name, t in (("q_lengths", q_lengths), ("kv_lengths", kv_lengths)):
        _check(t is None or (t.dtype == torch.int32 and t.shape == (batch,)), f"{name} must be an int32 tensor [{batch}]")
    _check_tensors(q.device, q=q, k=k, v=v, lambda_vectors=lambda_vectors, norm_weight=norm_weight, q_lengths=q_lengths, kv_lengths=kv_lengths, mask=mask, out=out)
    mask_stride = (0, 0, 0, 0)
    if mask is not None:
        _check(mask.dtype == torch.bool, "mask must be a bool tensor")
        try:
            mask = mask.expand(batch, heads, q_len, k_len)
        except RuntimeError:
            raise AssertionError(f"mask must be broadcastable to {(batch, heads, q_len, k_len)}") from None
        mask_stride = mask.stride()
    shape = (batch, q_len, heads, 2 * d)
    if out is None:
        out = (torch.empty if q_lengths is None else torch.zeros)(shape, dtype=q.dtype, device=q.device)
    else:
        _check(out.shape == shape and out.dtype == q.dtype and out.stride(3) == 1 and out.data_ptr() % 8 == 0 and
               not any(s % 4 for s, n in zip(out.stride()[:3], shape) if n > 1), f"out must be {shape} of q's type, with contiguous rows aligned to 8 bytes")
    q, k, v = _heads(q, "q"), _heads(k, "k"), _heads(v, "v")
    lambda_vectors = lambda_vectors if lambda_vectors.stride(-1) == 1 else lambda_vectors.contiguous()
    norm_weight, q_lengths, kv_lengths = (None if t is None else t.contiguous() for t in (norm_weight, q_lengths, kv_lengths))
    args = _capi.Tha4DiffAttentionArgs(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lambda_vectors.data_ptr(), _pointer(norm_weight), _pointer(q_lengths), _pointer(kv_lengths),
        _pointer(mask), None, 0, _strides(q), _strides(k), _strides(v), _strides(out), mask_stride,
        lambda_vectors.stride(0), lambda_vectors.stride(1) if lambda_vectors.dim() == 3 else 0,
        _DTYPES[q.dtype], batch, q_len, k_len, heads, kv2 // 2, d, causal, norm, 1.0 / math.sqrt(d) if scale is None else scale, lambda_init, eps)
    need = lib.tha4_diff_attention_workspace(C.byref(args))
    if need < 0:
        _capi.check(lib, need, "tha4_diff_attention_workspace")
    if need:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        args.workspace_dev, args.workspace_bytes = workspace.data_ptr(), need
    _capi.check(lib, lib.tha4_diff_attention(C.byref(args), _stream(q)), "tha4_diff_attention")
    return out
