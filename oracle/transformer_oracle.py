"""64-bit definitions of the transformer block operators (include/tha4_hip.h, tha4_amd/transformer.py), and how far an implementation that sums in fp32 may be off.

Each function takes the operator's inputs as they are (any type) and returns float64 tensors; the `*_bound` values next to them come from counting roundings:
u = 2^-24 for every fp32 operation, `half` = torch.finfo(type).eps / 2 for a rounding to that type."""
import math

import torch

U = 2.0 ** -24


def half(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def quantize(x):
    """(q, scale): scale in fp32, q = the integer nearest to the exact quotient.  In 64 bits the quotient of two 24-bit numbers rounds to k + 1/2 only if it is
    k + 1/2 (it differs from it by at least 2^-25 of it otherwise), so round() decides as the exact quotient would."""
    d = x.double()
    amax = d.abs().amax(-1)
    bad = ~torch.isfinite(d).all(-1)
    scale = (amax / 127).float()
    safe = torch.where(bad | (scale == 0), torch.ones_like(scale), scale).double()
    q = torch.round(torch.where(bad[..., None], torch.zeros_like(d), d) / safe[..., None]).clamp(-127, 127)
    q = torch.where((bad | (scale == 0))[..., None], torch.zeros_like(q), q)
    return q.to(torch.int8), torch.where(bad, torch.full_like(scale, math.nan), scale)


def int8_linear(q, q_scale, w, w_scale, bias, dtype):
    """(y, bound): exact sums; fp32: the sum to fp32, two products, the bias, then one rounding to `dtype` (half the smallest subnormal where it underflows)."""
    p = (q.double() @ w.double().t()) * q_scale.double()[..., None] * w_scale.double()
    y = p if bias is None else p + bias.double()
    return y, 4 * U * p.abs() + (U + half(dtype) * (1 + 8 * U)) * y.abs() + torch.finfo(dtype).smallest_normal * half(dtype) * 2


def _norm(x, dx, kind, weight, bias, eps, terms):
    """A norm of x (known to dx) and its bound: `terms` roundings in a sum, the subtraction of the mean, the root, the products."""
    n = x.shape[-1]
    if kind == "none":
        v, dv, k = x, dx, torch.ones_like(x[..., :1])
        dk = 0.0
    else:
        v, dv = x, dx
        if kind == "layer":
            mean = x.sum(-1, keepdim=True) / n
            dmean = dx.sum(-1, keepdim=True) / n + (terms + 2) * U * x.abs().sum(-1, keepdim=True) / n
            v = x - mean
            dv = dx + dmean + U * v.abs()
        ms = (v * v).sum(-1, keepdim=True) / n
        dms = 2 * (v.abs() * dv).sum(-1, keepdim=True) / n + (dv * dv).sum(-1, keepdim=True) / n + (terms + 4) * U * (ms + eps)
        k = 1 / torch.sqrt(ms + eps)
        dk = 0.5 * dms / (ms + eps) + 4 * U                       # relative
    w = torch.ones_like(x) if weight is None else weight.double().expand_as(x)
    b = torch.zeros_like(x) if bias is None else bias.double().expand_as(x)
    y = v * k * w + b
    return y, (dv * k + v.abs() * k * (dk + 3 * U)) * w.abs() * 1.01 + U * y.abs()


def _spread(t, rows):
    return t.double().reshape(-1, t.shape[-1]).repeat_interleave(rows // t.reshape(-1, t.shape[-1]).shape[0], 0)


def residual_norm(residual, branch=None, gate=None, gate_activation="none", residual_scale=1.0, post_norm="rms", post_weight=None, post_bias=None,
                  pre_norm="rms", pre_weight=None, pre_bias=None, film=None, eps=1e-5, terms=None):
    """((h, bound), (y, bound)); `terms`: the longest chain of additions in a sum (rows of c over 256 threads, then 14 levels of tree)."""
    shape, c = residual.shape, residual.shape[-1]
    r = residual.double().reshape(-1, c)
    rows = r.shape[0]
    terms = terms or c // 256 + 8 + 24
    rs = residual_scale.double() if isinstance(residual_scale, torch.Tensor) else float(torch.tensor(residual_scale, dtype=torch.float32))
    h = r * rs
    dh = 2 * U * h.abs()
    if branch is not None:
        x = branch.double().reshape(-1, c)
        n, dn = _norm(x, torch.zeros_like(x), post_norm, post_weight, post_bias, eps, terms)
        if gate is not None:
            g = _spread(gate, rows)
            dg = torch.zeros_like(g)
            if gate_activation == "sigmoid":
                dg = (g.abs() * 2 + 8) * U                        # the argument of the power of two is rounded (|g| log2(e) u), the power, the sum, the quotient
                g = 1 / (1 + torch.exp(-g))
                dg = dg * g
            dn = dn * g.abs() + n.abs() * dg + U * (n * g).abs()
            n = n * g
        h = h + n
        dh = dh + dn + U * h.abs()
    y, dy = _norm(h, dh, pre_norm, pre_weight, pre_bias, eps, terms)
    if film is not None:
        s, t = _spread(film[0], rows), _spread(film[1], rows)
        dy = dy * (1 + s).abs() + 3 * U * (y.abs() * (1 + s.abs()) + t.abs())
        y = y * (1 + s) + t
    out = residual.dtype
    ydt = residual.dtype if branch is None else branch.dtype
    # (below the smallest normal number a rounding is off by half a step there, however small the value: smallest_normal * half)
    return ((h.reshape(shape), (dh + half(out) * (h.abs() + dh) + torch.finfo(out).smallest_normal * half(out)).reshape(shape)),
            (y.reshape(shape), (dy + half(ydt) * (y.abs() + dy) + torch.finfo(ydt).smallest_normal * half(ydt)).reshape(shape)))


def visible(batch, q_len, k_len, causal, q_lengths, kv_lengths, mask, device):
    """bool [batch, 1 or heads, q_len, k_len]"""
    nq = torch.full((batch,), q_len, device=device) if q_lengths is None else q_lengths.long().clamp(0, q_len)
    nk = torch.full((batch,), k_len, device=device) if kv_lengths is None else kv_lengths.long().clamp(0, k_len)
    i = torch.arange(q_len, device=device)[None, None, :, None]
    j = torch.arange(k_len, device=device)[None, None, None, :]
    nq, nk = nq[:, None, None, None], nk[:, None, None, None]
    seen = (j < nk) & (i < nq)
    if causal:
        seen = seen & (j <= i + nk - nq)
    return seen if mask is None else seen & mask


def differential_attention(q, k, v, lambda_vectors, lambda_init, causal=False, q_lengths=None, kv_lengths=None, mask=None, scale=None, norm=True,
                           norm_weight=None, eps=1e-5):
    """(out, bound).  A weight p is the sum of two numbers of the inputs' type (half(type)^2; the fp16 weights are held 2^12 times as large at least, so one that is
    subnormal there is off by 2^-25 2^-12 of a sum of weights of at least 1); scores carry (d + 4) u of sum |q k|; the sums over the keys, both parts' and the weights' own, 3 k_len u."""
    batch, q_len, heads2, d = q.shape
    k_len, heads, group = k.shape[1], heads2 // 2, heads2 // k.shape[2]
    scale = 1 / math.sqrt(d) if scale is None else scale
    seen = visible(batch, q_len, k_len, causal, q_lengths, kv_lengths, mask, q.device)
    qd = q.double().view(batch, q_len, heads, 2, d)
    kd = k.double().view(batch, k_len, heads // group, 2, d).repeat_interleave(group, 2)
    vd = v.double().repeat_interleave(group, 2).permute(0, 2, 1, 3).contiguous()                  # [b, h, k, 2d]
    valid = seen.any(2).any(1) if k_len else None                                               # keys that nobody sees count for nothing, whatever they hold
    if valid is not None:
        kd = torch.where(valid[:, :, None, None, None], kd, torch.zeros_like(kd))
        vd = torch.where(valid[:, None, :, None], vd, torch.zeros_like(vd))
    lam = lambda_vectors.double() if lambda_vectors.dim() == 3 else lambda_vectors.double()[:, None, :]
    e0, e1 = torch.exp((lam[0] * lam[1]).sum(-1)), torch.exp((lam[2] * lam[3]).sum(-1))
    dot = ((lam[0] * lam[1]).abs().sum(-1) + (lam[2] * lam[3]).abs().sum(-1))
    dlam = ((e0 + e1) * ((d + 2) * dot * U + 4 * U) + 4 * U * abs(lambda_init))[None, :, None, None]
    lam = (e0 - e1 + lambda_init)[None, :, None, None]
    maps, errs = [], []
    for i in (0, 1):
        qi, ki = qd[:, :, :, i].permute(0, 2, 1, 3).contiguous(), kd[:, :, :, i].permute(0, 2, 3, 1).contiguous()
        s = torch.matmul(qi, ki) * scale
        top = torch.matmul(qi.abs(), ki.abs()) * scale
        s = torch.where(seen, s, torch.full_like(s, -math.inf))
        m = s.amax(-1, keepdim=True) if k_len else s.new_full(s.shape[:-1] + (1,), -math.inf)
        p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
        l = p.sum(-1, keepdim=True)
        a = torch.where(l > 0, p / l, torch.zeros_like(p))
        ds = torch.where(seen, (d + 6) * U * top, torch.zeros_like(top))
        ds = (ds.amax(-1, keepdim=True) if k_len else torch.zeros_like(m)) + 4 * U * torch.where(m.isfinite(), m.abs(), torch.zeros_like(m))
        rel = half(q.dtype) ** 2 + 2.02 * ds + (3 * k_len + 60) * U
        small = 2.0 ** -37 if q.dtype == torch.float16 else 0.0
        err = torch.matmul(a, vd.abs()) * rel + small * torch.where(l > 0, 1 / l.clamp_min(1e-300), torch.zeros_like(l)) * torch.matmul(seen.double().expand_as(p), vd.abs())
        maps.append(torch.matmul(a, vd))
        errs.append(err)
    o = maps[0] - lam * maps[1]
    do = errs[0] + lam.abs() * errs[1] + dlam * maps[1].abs() + 3 * U * (maps[0].abs() + (lam * maps[1]).abs())
    if norm:
        ms = (o * o).mean(-1, keepdim=True)
        ms = torch.where(ms + eps > 0, ms, torch.ones_like(ms))                  # a row of zeros stays one, also with eps = 0
        g = (1 - lambda_init) / torch.sqrt(ms + eps)
        w = torch.ones(2 * d, dtype=torch.float64, device=q.device) if norm_weight is None else norm_weight.double()
        dms = 2 * (o.abs() * do).mean(-1, keepdim=True) + (do * do).mean(-1, keepdim=True) + (2 * d + 8) * U * ms
        rel = 0.5 * dms / (ms + eps) * 1.05 + 8 * U
        do = abs(1 - lambda_init) / torch.sqrt(ms + eps) * w.abs() * (do + o.abs() * rel)
        o = o * g * w
    out, bound = o.permute(0, 2, 1, 3), do.permute(0, 2, 1, 3)
    return out, bound + half(q.dtype) * (out.abs() + bound) + torch.finfo(q.dtype).smallest_normal * half(q.dtype) * 2
