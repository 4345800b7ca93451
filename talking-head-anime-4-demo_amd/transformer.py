"""Operators of a transformer block over token sequences, at inference, on the GPU: relatives of what the posers' networks have inside (attention, normalisation +
FiLM + residual, reduced-precision matrix products), for sequences of any length, prompts and single tokens over a cache.  The posers do not call them.

``quantize_tokens``         tokens (or weight rows) to int8 with one scale each
``int8_linear``             int8 x int8 matrix product with scales for each token and channel
``residual_norm``           the norms behind and in front of a block, with its gate and the residual sum
``differential_attention``  the difference of two softmax maps with learned weights

All of them enqueue on ``torch.cuda.current_stream()`` of their tensors' device, never synchronise, and can be captured into a graph.  Wrong arguments raise
AssertionError here or ``_capi.Tha4Error`` from the C ABI (include/tha4_hip.h); nothing falls back to another implementation.  They are forward
operators: tensors that require gradients are refused while gradients are enabled, tensors with a forward-mode tangent always, and so are views whose memory holds
the negated values (``Tensor.is_neg``).
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _capi

_DTYPES = {torch.float32: _capi.F32, torch.float16: _capi.F16, torch.bfloat16: _capi.BF16}
_ONE_ROW = 2 ** 63 - 1
_stream = torch._C._cuda_getCurrentRawStream        # what torch.cuda.current_stream(device).cuda_stream returns, for a twentieth of its time


def _library():
    return _capi._lib or _capi.load_library()


def _check_tensors(first: Tensor, *others: Optional[Tensor]) -> int:
    """The device all of them live on.  (A single-token call costs the host more than the GPU: the checks below are written for speed.)"""
    if not first.is_cuda:
        raise AssertionError("tensors must be on the GPU")
    device = first.get_device()
    gradient, negated = first.requires_grad, first.is_neg()
    for t in others:
        if t is not None:
            if t.get_device() != device:
                raise AssertionError(f"tensors must be on one GPU: {t.device} and {first.device}")
            gradient = gradient or t.requires_grad
            negated = negated or t.is_neg()
    if negated:
        raise AssertionError("a tensor's memory holds its values negated (a view of a complex conjugate): pass tensor.resolve_neg()")
    if gradient and torch.is_grad_enabled():
        raise AssertionError("an input requires a gradient: this is a forward operator (use torch.no_grad())")
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in (first,) + others):
        raise AssertionError("an input carries a forward-mode tangent: this operator has no derivative (use unpack_dual(tensor).primal)")
    return device


def _rows(t: Tensor, cols: int) -> Tuple[Tensor, int]:
    """[..., cols] as rows of contiguous elements: (tensor at the first row, elements from row to row).  A copy only where the strides leave no other way."""
    if t.is_contiguous():
        return t, cols
    if t.dim() != 2:
        t = t.reshape(-1, cols)
    if cols > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, t.stride(0) if t.shape[0] > 1 else cols


def quantize_tokens(x: Tensor) -> Tuple[Tensor, Tensor]:
    """x [..., c] fp32 / fp16 / bf16 -> (int8 [..., c], fp32 scales [...]): ``q = x / scale`` rounded to the nearest integer (ties to even), ``scale = max |x| / 127``.
    A row of zeros gets scale 0; a row that holds an infinity or a NaN gets scale NaN (products with it are NaN) and zeros.
    Weights [n, c] are quantised for each channel by the same call."""
    lib = _library()
    code = _DTYPES.get(x.dtype)
    if code is None or x.dim() < 1 or x.shape[-1] < 1:
        raise AssertionError("x must be a float32, float16 or bfloat16 tensor [..., c] with c >= 1")
    device = _check_tensors(x)
    shape = x.shape
    cols = shape[-1]
    q = torch.empty(shape, dtype=torch.int8, device=x.device)
    scale = torch.empty(shape[:-1], dtype=torch.float32, device=x.device)
    r, stride = _rows(x, cols)
    status = lib.tha4_quantize_tokens_i8(r.data_ptr(), code, scale.numel(), cols, stride, q.data_ptr(), cols, scale.data_ptr(), _stream(device))
    if status:
        _capi.check(lib, status, "tha4_quantize_tokens_i8")
    return q, scale


def int8_linear(x: Tensor, weight: Tensor, weight_scale: Tensor, *, x_scale: Optional[Tensor] = None, bias: Optional[Tensor] = None,
                out_dtype: Optional[torch.dtype] = None) -> Tensor:
    """x [..., k] times int8 weight [n, k] with fp32 weight_scale [n] -> [..., n]: ``y = x_scale weight_scale (x_q . weight) + bias``.

    x is float (quantised for each token on the way, as by ``quantize_tokens``; the result has its type unless ``out_dtype`` says otherwise) or int8 with
    fp32 ``x_scale`` [...] (then ``out_dtype`` is needed).  The sums are exact 32-bit integers (k <= 131071), scaled in fp32 and rounded once."""
    lib = _library()
    if weight.dim() != 2 or weight.dtype != torch.int8 or weight.shape[1] < 1:
        raise AssertionError("weight must be an int8 tensor [n, k] with k >= 1")
    n, k = weight.shape
    shape = x.shape
    if not shape or shape[-1] != k:
        raise AssertionError(f"x must be [..., {k}]")
    if weight_scale.dtype != torch.float32 or weight_scale.shape != (n,):
        raise AssertionError(f"weight_scale must be a float32 tensor [{n}]")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (n,)):
        raise AssertionError(f"bias must be a float32 tensor [{n}]")
    if x.dtype == torch.int8:
        code = _capi.I8
        if x_scale is None or x_scale.dtype != torch.float32 or x_scale.shape != shape[:-1]:
            raise AssertionError("int8 x needs a float32 x_scale [...]")
        x_scale = x_scale.contiguous()
    else:
        code = _DTYPES.get(x.dtype)
        out_dtype = out_dtype or x.dtype
        if x_scale is not None:
            raise AssertionError("x_scale belongs to an int8 x")
    out_code = _DTYPES.get(out_dtype)
    if code is None or out_code is None:
        raise AssertionError("x must be float32, float16, bfloat16 or int8, and out_dtype (needed for int8) one of the first three")
    device = _check_tensors(x, weight, weight_scale, x_scale, bias)
    w, w_stride = _rows(weight, k)
    if not weight_scale.is_contiguous():
        weight_scale = weight_scale.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    y = torch.empty(shape[:-1] + (n,), dtype=out_dtype, device=x.device)
    r, stride = _rows(x, k)
    m = x.numel() // k
    args = _capi.Tha4LinearI8Args(r.data_ptr(), None if x_scale is None else x_scale.data_ptr(), w.data_ptr(), weight_scale.data_ptr(),
                                  None if bias is None else bias.data_ptr(), y.data_ptr(), None, 0, m, n, k, stride, w_stride, n, code, out_code)
    need = lib.tha4_linear_i8_workspace(args)
    if need > 0:
        workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
        args.workspace_dev, args.workspace_bytes = workspace.data_ptr(), need
    status = lib.tha4_linear_i8(args, _stream(device))
    if status:
        _capi.check(lib, status, "tha4_linear_i8")
    return y


def _per_row(t: Tensor, name: str, shape, cols: int, rows: int) -> Tuple[Tensor, int, int]:
    """A gate or FiLM tensor -> (its rows, their stride, rows of the input for each): one row ([c], [1, .., c]), a row for each sample ([samples, c],
    [samples, 1, .., c]; for a two-dimensional input any number of consecutive equal shares) or for each token (the input's shape, or [rows, c])."""
    if t.shape == shape:
        return _rows(t, cols) + (1,)
    if t.dim() < 1 or t.shape[-1] != cols:
        raise AssertionError(f"{name} must be [..., {cols}]")
    have = t.numel() // cols
    lead = t.shape[0] if t.dim() > 1 else 1
    if have != lead or (have not in (1, rows, shape[0]) and (len(shape) != 2 or have < 1 or rows % have)):
        raise AssertionError(f"{name} must have one row, one for each sample or one for each token")
    t, stride = _rows(t.reshape(have, cols), cols)
    return t, stride, _ONE_ROW if have == 1 else max(rows // have, 1)


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
    lib = _library()
    shape = residual.shape
    if not shape or shape[-1] < 1:
        raise AssertionError("residual must be [..., c] with c >= 1")
    cols = shape[-1]
    rows = residual.numel() // cols
    residual_type = residual.dtype
    dtype = residual_type if branch is None else branch.dtype
    code = _DTYPES.get(dtype)
    if code is None or residual_type not in (dtype, torch.float32):
        raise AssertionError("branch must be float32, float16 or bfloat16, and residual that type or float32")
    if branch is not None and branch.shape != shape:
        raise AssertionError(f"branch must have residual's shape {tuple(shape)}")
    post, pre, activation = _capi.NORM_KINDS.get(post_norm), _capi.NORM_KINDS.get(pre_norm), _capi.GATE_ACTIVATIONS.get(gate_activation)
    if post is None or pre is None or activation is None:
        raise AssertionError(f"post_norm / pre_norm must be one of {sorted(_capi.NORM_KINDS)}, gate_activation one of {sorted(_capi.GATE_ACTIVATIONS)}")
    vector = residual_scale if isinstance(residual_scale, Tensor) else None
    film_s, film_t = (None, None) if film is None else film
    device = _check_tensors(residual, branch, gate, film_s, film_t, vector, post_weight, post_bias, pre_weight, pre_bias)
    params = None
    pointers = []
    keep = []                                       # what a pointer below points into lives until the call has been enqueued
    for v in (vector, post_weight, post_bias, pre_weight, pre_bias):
        if v is None:
            pointers.append(None)
            continue
        if v.shape != (cols,):
            raise AssertionError(f"residual_scale and the norms' weights and biases must be vectors [{cols}]")
        if params is not None and v.dtype != params:
            raise AssertionError("vectors and film must all be float32 or all of branch's type")
        params = v.dtype
        if not v.is_contiguous():
            v = v.contiguous()
            keep.append(v)
        pointers.append(v.data_ptr())
    gate_at, gate_stride, gate_rows, gate_code = None, 0, 1, code
    if gate is not None:
        if gate.dtype not in (dtype, torch.float32):
            raise AssertionError("gate must have branch's type or float32")
        gate_code = _DTYPES[gate.dtype]
        gate, gate_stride, gate_rows = _per_row(gate, "gate", shape, cols, rows)
        gate_at = gate.data_ptr()
    film_at, shift_at, film_stride, film_rows = None, None, 0, 1
    if film is not None:
        if film_s.shape != film_t.shape or film_s.dtype != film_t.dtype or (params is not None and film_s.dtype != params):
            raise AssertionError("film must be (scale, shift) of one shape and type; vectors and film must all be float32 or all of branch's type")
        params = film_s.dtype
        if film_s.stride() != film_t.stride():
            film_s, film_t = film_s.contiguous(), film_t.contiguous()
        film_s, film_stride, film_rows = _per_row(film_s, "film", shape, cols, rows)
        film_t = _per_row(film_t, "film", shape, cols, rows)[0]
        film_at, shift_at = film_s.data_ptr(), film_t.data_ptr()
    if params is not None and params not in (dtype, torch.float32):
        raise AssertionError("vectors and film must all be float32 or all of branch's type")
    dense = residual.is_contiguous()
    h = torch.empty_like(residual) if dense else torch.empty(shape, dtype=residual_type, device=residual.device)
    y = torch.empty_like(residual) if dense and dtype is residual_type else torch.empty(shape, dtype=dtype, device=residual.device)
    r, r_stride = _rows(residual, cols)
    b, b_stride = (None, 0) if branch is None else _rows(branch, cols)
    args = _capi.Tha4ResidualNormArgs(
        r.data_ptr(), None if b is None else b.data_ptr(), gate_at, *pointers, film_at, shift_at, h.data_ptr(), y.data_ptr(), rows, cols,
        r_stride, b_stride, gate_stride, film_stride, cols, cols, gate_rows, film_rows, code, _DTYPES[residual_type], gate_code, _DTYPES[params or torch.float32],
        post, pre, activation, 1.0 if vector is not None else residual_scale, eps)
    status = lib.tha4_residual_norm(args, _stream(device))
    if status:
        _capi.check(lib, status, "tha4_residual_norm")
    return h, y


def _heads(t: Tensor) -> Tuple[Tensor, Tuple[int, int, int]]:
    """(tensor, strides over batch, token and head): 16-byte aligned with contiguous rows, copied where the strides do not allow that."""
    if t.is_contiguous():
        if t.data_ptr() % 16:
            t = t.clone()
        _, n, h, d = t.shape
        return t, (n * h * d, h * d, d)             # (its own strides say nothing where a dimension has one entry)
    if t.stride(3) != 1 or t.data_ptr() % 16 or any(s % 8 for s, n in zip(t.stride()[:3], t.shape) if n > 1):
        t = t.contiguous()
    return t, tuple(s if n > 1 else 0 for s, n in zip(t.stride()[:3], t.shape))


def differential_attention(q: Tensor, k: Tensor, v: Tensor, lambda_vectors: Tensor, lambda_init: float, *, causal: bool = False,
                           q_lengths: Optional[Tensor] = None, kv_lengths: Optional[Tensor] = None, mask: Optional[Tensor] = None, scale: Optional[float] = None,
                           norm: bool = True, norm_weight: Optional[Tensor] = None, eps: float = 1e-5, out: Optional[Tensor] = None) -> Tensor:
    """``softmax(scale q1 k1^T) v - lambda softmax(scale q2 k2^T) v`` with ``lambda = exp(l0 . l1) - exp(l2 . l3) + lambda_init``, then (``norm``)
    ``(1 - lambda_init) * o / sqrt(mean(o^2) + eps) * norm_weight`` over the value columns of each head.

    q [batch, q_len, 2 heads, d], k [batch, k_len, 2 kv_heads, d] (maps 1 and 2 of head h at 2h and 2h + 1), v [batch, k_len, kv_heads, 2d] fp16 or bf16, d 32, 64
    or 128, heads a multiple of kv_heads -> [batch, q_len, heads, 2d].  Any strides with contiguous rows of d (views of a fused projection or of a longer
    cache).  lambda_vectors fp32 [4, d] or [4, heads, d].  scale: 1 / sqrt(d).

    kv_lengths int32 [batch]: the valid keys of each sequence (what lies behind them is never read into a result); q_lengths int32 [batch]: its valid queries - rows
    behind them are zero, or left as they are in a given ``out`` (which shares no memory with q, k or v).  causal: the last valid query sees the last valid key.  mask: bool, broadcastable to
    [batch, heads, q_len, k_len], True = visible.  A query that sees no key answers zero.  k_len may be 0."""
    lib = _library()
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise AssertionError("q, k and v must be [batch, tokens, heads, d]")
    dtype = q.dtype
    if dtype not in (torch.float16, torch.bfloat16) or k.dtype != dtype or v.dtype != dtype:
        raise AssertionError("q, k and v must all be float16 or all bfloat16")
    batch, q_len, heads2, d = q.shape
    _, k_len, kv2, _ = k.shape
    if d not in (32, 64, 128):
        raise AssertionError("the head dimension must be 32, 64 or 128")
    if heads2 < 2 or kv2 < 2 or heads2 % 2 or kv2 % 2 or heads2 % kv2:
        raise AssertionError("q and k must hold pairs of heads, q a multiple of k's")
    heads, kv_heads = heads2 // 2, kv2 // 2
    if k.shape != (batch, k_len, kv2, d) or v.shape != (batch, k_len, kv_heads, 2 * d):
        raise AssertionError("k must be [batch, k_len, 2 kv_heads, d] and v [batch, k_len, kv_heads, 2 d]")
    if lambda_vectors.dtype != torch.float32 or lambda_vectors.shape not in ((4, d), (4, heads, d)):
        raise AssertionError(f"lambda_vectors must be float32 [4, {d}] or [4, {heads}, {d}]")
    if norm_weight is not None and (not norm or norm_weight.dtype != torch.float32 or norm_weight.shape != (2 * d,)):
        raise AssertionError(f"norm_weight must be float32 [{2 * d}] (with norm)")
    for t in (q_lengths, kv_lengths):
        if t is not None and (t.dtype != torch.int32 or t.shape != (batch,)):
            raise AssertionError(f"q_lengths and kv_lengths must be int32 tensors [{batch}]")
    device = _check_tensors(q, k, v, lambda_vectors, norm_weight, q_lengths, kv_lengths, mask, out)
    mask_at, mask_stride = None, (0, 0, 0, 0)
    if mask is not None:
        if mask.dtype != torch.bool:
            raise AssertionError("mask must be a bool tensor")
        try:
            mask = mask.expand(batch, heads, q_len, k_len)
        except RuntimeError:
            raise AssertionError(f"mask must be broadcastable to {(batch, heads, q_len, k_len)}") from None
        mask_at, mask_stride = mask.data_ptr(), mask.stride()
    shape = (batch, q_len, heads, 2 * d)
    if out is None:
        out = (torch.empty if q_lengths is None else torch.zeros)(shape, dtype=dtype, device=q.device)
        out_stride = (q_len * heads * 2 * d, heads * 2 * d, 2 * d)
    else:
        if out.shape != shape or out.dtype != dtype or out.stride(3) != 1 or out.data_ptr() % 8 or any(s % 4 for s, n in zip(out.stride()[:3], shape) if n > 1):
            raise AssertionError(f"out must be {shape} of q's type, with contiguous rows aligned to 8 bytes")
        out_stride = tuple(s if n > 1 else 0 for s, n in zip(out.stride()[:3], shape))
    (q, q_stride), (k, k_stride), (v, v_stride) = _heads(q), _heads(k), _heads(v)
    if lambda_vectors.stride(-1) != 1:
        lambda_vectors = lambda_vectors.contiguous()
    norm_weight, q_lengths, kv_lengths = (t if t is None or t.is_contiguous() else t.contiguous() for t in (norm_weight, q_lengths, kv_lengths))
    args = _capi.Tha4DiffAttentionArgs(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lambda_vectors.data_ptr(), None if norm_weight is None else norm_weight.data_ptr(),
        None if q_lengths is None else q_lengths.data_ptr(), None if kv_lengths is None else kv_lengths.data_ptr(), mask_at, None, 0,
        *q_stride, *k_stride, *v_stride, *out_stride, *mask_stride, lambda_vectors.stride(0), lambda_vectors.stride(1) if lambda_vectors.dim() == 3 else 0,
        _DTYPES[dtype], batch, q_len, k_len, heads, kv_heads, d, causal, norm, d ** -0.5 if scale is None else scale, lambda_init, eps)
    need = lib.tha4_diff_attention_workspace(args)
    if need > 0:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        args.workspace_dev, args.workspace_bytes = workspace.data_ptr(), need
    status = lib.tha4_diff_attention(args, _stream(device))
    if status:
        _capi.check(lib, status, "tha4_diff_attention")
    return out
