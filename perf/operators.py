"""What the operators of a transformer block (``tha4_amd.transformer``) are measured on.

Three operators: the 8-bit matrix product with its quantisation of the tokens, the pair of norms around a block fused with gate and
residual, and differential attention (prompts, padded batches, single tokens over a cache).  ``run`` with ``own = False`` states each one in
elementary torch operations; with ``own = True`` it calls the framework.
"""
import math
import random

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_DEVICE = "cuda:0"


def listed():
    return [
        # one token through a square projection of a 4096-wide block: the latency of a decode step
        {"name": "linear 1 token", "op": "linear", "m": 1, "n": 4096, "k": 4096, "type": "bf16", "bias": False},
        # 16 streams decoded together through a widening projection: the weights are the traffic
        {"name": "linear 16 tokens", "op": "linear", "m": 16, "n": 16384, "k": 8192, "type": "f16", "bias": True},
        # nothing divides anything: a pruned layer, fp32 activations
        {"name": "linear ragged", "op": "linear", "m": 777, "n": 1001, "k": 1111, "type": "f32", "bias": True},
        # a long prompt through a large projection: the matrix pipe
        {"name": "linear prompt", "op": "linear", "m": 8192, "n": 8192, "k": 8192, "type": "bf16", "bias": False},
        # one token between two blocks
        {"name": "norm 1 token", "op": "norm", "rows": 1, "c": 4096, "samples": 1, "type": "bf16", "kind": "rms", "gate": "channel", "film": False},
        # the token maps of eight frames (16 x 16 x 256 channels), conditioned for each frame
        {"name": "norm frames", "op": "norm", "rows": 2048, "c": 256, "samples": 8, "type": "f32", "kind": "layer", "gate": "sample", "film": True},
        # a long prompt, every element gated
        {"name": "norm prompt", "op": "norm", "rows": 16384, "c": 8192, "samples": 1, "type": "bf16", "kind": "rms", "gate": "full", "film": False},
        # the token maps of eight frames: 256 tokens, 8 heads, 32 channels
        {"name": "attention frames", "op": "attention", "batch": 8, "q": 256, "k": 256, "heads": 8, "kv_heads": 8, "d": 32, "type": "f16", "causal": False, "ragged": False},
        # a padded batch of prompts, one of them empty and one a single token
        {"name": "attention padded", "op": "attention", "batch": 5, "q": 1777, "k": 1777, "heads": 16, "kv_heads": 4, "d": 64, "type": "bf16", "causal": True, "ragged": True},
        # one long prompt
        {"name": "attention prompt", "op": "attention", "batch": 1, "q": 8192, "k": 8192, "heads": 8, "kv_heads": 8, "d": 128, "type": "bf16", "causal": True, "ragged": False},
        # 32 streams decoded together, each with a cache of its own length
        {"name": "attention decode", "op": "attention", "batch": 32, "q": 1, "k": 16384, "heads": 16, "kv_heads": 4, "d": 64, "type": "bf16", "causal": True, "ragged": True},
        # one stream over a very long cache
        {"name": "attention long cache", "op": "attention", "batch": 1, "q": 1, "k": 131072, "heads": 8, "kv_heads": 2, "d": 128, "type": "f16", "causal": True, "ragged": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "norm", "attention"])
    kind = rng.choice(["f32", "f16", "bf16"])
    if op == "linear":
        while True:
            m, n, k = _log(rng, 1, 8192), _log(rng, 64, 16384), _log(rng, 64, 8192)
            if rng.random() < 0.5:
                n, k = -(-n // 64) * 64, -(-k // 64) * 64
            if m * n * k <= 8192 ** 3:
                return {"op": op, "m": m, "n": n, "k": k, "type": kind, "bias": rng.random() < 0.5}
    if op == "norm":
        while True:
            samples, c = rng.randint(1, 8), _log(rng, 32, 8192)
            rows = samples * _log(rng, 1, 4096)
            if rng.random() < 0.7:
                c = -(-c // 16) * 16
            if rows * c <= 8192 * 8192:
                return {"op": op, "rows": rows, "c": c, "samples": samples, "type": kind, "kind": rng.choice(["rms", "layer"]),
                        "gate": rng.choice(["none", "channel", "sample", "full"]), "film": rng.random() < 0.4}
    kind = rng.choice(["f16", "bf16"])
    kv = rng.choice([1, 2, 4, 8])
    heads, d, batch = kv * rng.choice([1, 2, 4]), rng.choice([32, 64, 128]), _log(rng, 1, 32)
    ragged = rng.random() < 0.5
    if rng.random() < 0.5:
        while True:
            k = _log(rng, 1, 65536)
            if batch * k * kv * d <= 32 * 16384 * 4 * 64:
                return {"op": op, "batch": batch, "q": rng.choice([1, 1, 2, 4]), "k": k, "heads": heads, "kv_heads": kv, "d": d, "type": kind, "causal": True, "ragged": ragged}
            batch = _log(rng, 1, 32)
    while True:
        q = _log(rng, 16, 4096)
        k = q if ragged or rng.random() < 0.7 else _log(rng, 16, 4096)
        if batch * heads * q * k <= 8 * 4096 * 4096:
            return {"op": op, "batch": batch, "q": q, "k": k, "heads": heads, "kv_heads": kv, "d": d, "type": kind, "causal": rng.random() < 0.6, "ragged": ragged}
        batch = _log(rng, 1, 32)


def _lengths(case):
    """Valid keys of each sequence: the last full, with an empty and a single-token one where the batch has room."""
    if not case["ragged"]:
        return [case["k"]] * case["batch"]
    r = random.Random(case["batch"] * 65537 + case["k"])
    got = [r.randint(1, case["k"]) for _ in range(case["batch"])]
    if case["batch"] > 2:
        got[0], got[1] = 0, 1
    got[-1] = case["k"]
    return got


def _prompt(case):
    """A padded batch of prompts (its queries are padded like its keys) rather than new tokens over a cache."""
    return case["ragged"] and case["q"] == case["k"]


def prepare(case, seed):
    g = torch.Generator(device=_DEVICE).manual_seed(int(seed))
    t = _TYPES[case["type"]]

    def normal(*shape, dtype=torch.float32, std=1.0, mean=0.0):
        return torch.empty(shape, dtype=dtype, device=_DEVICE).normal_(mean, std, generator=g)

    s = {"case": case}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        x = normal(m, k) * normal(k, std=0.6).exp()           # channels of unlike size, as behind a norm
        s["x"] = x.to(t)
        s["w"] = torch.randint(-127, 128, (n, k), dtype=torch.int8, device=_DEVICE, generator=g)
        s["w_scale"] = normal(n, std=0.3).exp() / (127.0 * math.sqrt(k))
        s["bias"] = normal(n, std=0.5) if case["bias"] else None
    elif case["op"] == "norm":
        rows, c, b = case["rows"], case["c"], case["samples"]
        s["residual"] = normal(rows, c, dtype=t, std=2.0, mean=0.1)
        s["branch"] = normal(rows, c, dtype=t, std=0.7, mean=0.2)
        gate = {"none": None, "channel": (1, c), "sample": (b, c), "full": (rows, c)}[case["gate"]]
        s["gate"] = None if gate is None else normal(*gate, dtype=t, mean=0.3)
        s["post_weight"], s["pre_weight"] = normal(c, std=0.2, mean=1.0), normal(c, std=0.2, mean=1.0)
        layer = case["kind"] == "layer"
        s["post_bias"], s["pre_bias"] = (normal(c, std=0.1), normal(c, std=0.1)) if layer else (None, None)
        s["film"] = (normal(b, c, std=0.3), normal(b, c, std=0.3)) if case["film"] else None
    else:
        b, h, kv, d = case["batch"], case["heads"], case["kv_heads"], case["d"]
        s["q"] = normal(b, case["q"], 2 * h, d, dtype=t)
        s["k"] = normal(b, case["k"], 2 * kv, d, dtype=t)
        s["v"] = normal(b, case["k"], kv, 2 * d, dtype=t, mean=0.1)
        s["lambdas"] = normal(4, d, std=0.1)
        s["norm_weight"] = normal(2 * d, std=0.2, mean=1.0)
        s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=_DEVICE) if case["ragged"] else None
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------------------------
def _plain_linear(s):
    x = s["x"].float()
    scale = (x.abs().amax(1).double() / 127).float()
    # in 64 bits: whether a quotient of two 32-bit numbers is above or below a half decides the whole step
    q = torch.round(x.double() / scale.double().clamp_min(1e-300)[:, None]).clamp_(-127, 127).float()
    y = (q @ s["w"].float().t()) * scale[:, None] * s["w_scale"]
    return (y if s["bias"] is None else y + s["bias"]).to(s["x"].dtype)


def _plain_norm(s):
    case = s["case"]

    def norm(v, weight, bias):
        if bias is not None:
            v = v - v.mean(1, keepdim=True)
        v = v * torch.rsqrt(v.square().mean(1, keepdim=True) + 1e-5) * weight
        return v if bias is None else v + bias

    def wide(v):       # [samples, c] -> [rows, c]
        return v.float().repeat_interleave(case["rows"] // v.shape[0], 0)

    r = norm(s["branch"].float(), s["post_weight"], s["post_bias"])
    if s["gate"] is not None:
        gate = wide(s["gate"])
        r = r * (torch.sigmoid(gate) if case["gate"] == "full" else gate)
    h = s["residual"].float() * 0.9 + r
    y = norm(h, s["pre_weight"], s["pre_bias"])
    if s["film"] is not None:
        y = y * (1 + wide(s["film"][0])) + wide(s["film"][1])
    return {"h": h.to(s["residual"].dtype), "y": y.to(s["branch"].dtype)}


def _visible(case, lengths, device):
    """[batch, q, k]: which keys a query sees; query rows behind the last see none."""
    b, nq, nk = case["batch"], case["q"], case["k"]
    n = torch.full((b,), nk, device=device) if lengths is None else lengths.long()
    i, j = torch.arange(nq, device=device)[None, :, None], torch.arange(nk, device=device)[None, None, :]
    seen = (j < n[:, None, None]).expand(b, nq, nk)
    first = torch.zeros_like(n) if _prompt(case) else n - nq
    if case["causal"]:
        seen = seen & (j <= i + first[:, None, None])
    return seen & (i < n[:, None, None]) if _prompt(case) else seen


def _plain_attention(s):
    case = s["case"]
    b, h, kv, d, nq, nk = case["batch"], case["heads"], case["kv_heads"], case["d"], case["q"], case["k"]
    g = h // kv
    # [b, kv, g, 2, q, d] x [b, kv, 1, 2, d, k]
    q = s["q"].float().view(b, nq, kv, g, 2, d).permute(0, 2, 4, 3, 1, 5).reshape(b * kv * 2, g * nq, d)
    k = s["k"].float().view(b, nk, kv, 2, d).permute(0, 2, 3, 4, 1).reshape(b * kv * 2, d, nk)
    v = s["v"].float().permute(0, 2, 1, 3).reshape(b * kv, nk, 2 * d)
    seen = _visible(case, s["lengths"], q.device)
    score = torch.bmm(q, k).view(b, kv, 2, g, nq, nk) * (1 / math.sqrt(d))
    score = score.masked_fill(~seen[:, None, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - top.masked_fill(top == -math.inf, 0))
    p = e / e.sum(-1, keepdim=True).clamp_min(1e-30)
    lam = torch.exp((s["lambdas"][0] * s["lambdas"][1]).sum()) - torch.exp((s["lambdas"][2] * s["lambdas"][3]).sum()) + 0.5
    a = (p[:, :, 0] - lam * p[:, :, 1]).reshape(b * kv, g * nq, nk)
    o = torch.bmm(a, v).view(b, kv, g, nq, 2 * d).permute(0, 3, 1, 2, 4).reshape(b, nq, h, 2 * d)
    o = o * torch.rsqrt(o.square().mean(-1, keepdim=True) + 1e-5) * s["norm_weight"] * (1 - 0.5)
    return o.to(s["q"].dtype)


# ---- one pass ----------------------------------------------------------------------------------------------------------------------------
def _own(s):
    from tha4_amd import transformer
    case = s["case"]
    if case["op"] == "linear":
        return transformer.int8_linear(s["x"], s["w"], s["w_scale"], bias=s["bias"])
    if case["op"] == "norm":
        h, y = transformer.residual_norm(s["residual"], s["branch"], gate=s["gate"], gate_activation="sigmoid" if case["gate"] == "full" else "none",
                                         residual_scale=0.9, post_norm=case["kind"], post_weight=s["post_weight"], post_bias=s["post_bias"],
                                         pre_norm=case["kind"], pre_weight=s["pre_weight"], pre_bias=s["pre_bias"], film=s["film"], eps=1e-5)
        return {"h": h, "y": y}
    return transformer.differential_attention(s["q"], s["k"], s["v"], s["lambdas"], 0.5, causal=case["causal"], kv_lengths=s["lengths"],
                                              q_lengths=s["lengths"] if _prompt(case) else None, norm_weight=s["norm_weight"], eps=1e-5)


def run(state):
    if own:
        return _own(state)
    return {"linear": _plain_linear, "norm": _plain_norm, "attention": _plain_attention}[state["case"]["op"]](state)


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": size * m * (k + n) + n * k + 4 * n * (2 if case["bias"] else 1), "flops": 2 * m * n * k}
    if case["op"] == "norm":
        rows, c = case["rows"], case["c"]
        gate = {"none": 0, "channel": 1, "sample": case["samples"], "full": rows}[case["gate"]]
        params = (4 if case["kind"] == "layer" else 2) + (2 * case["samples"] if case["film"] else 0)
        return {"bytes": size * c * (4 * rows + gate) + 4 * c * params, "flops": 20 * rows * c}
    b, h, kv, d, nq = case["batch"], case["heads"], case["kv_heads"], case["d"], case["q"]
    keys = queries = pairs = 0
    for n in _lengths(case):
        rows = n if _prompt(case) else nq
        first = 0 if _prompt(case) else n - nq
        keys, queries = keys + n, queries + rows
        if not case["causal"]:
            pairs += rows * n
            continue
        lo, hi = max(0, -first), min(rows, n - first)      # rows lo .. hi - 1 see i + first + 1 keys, the ones behind see all n
        pairs += max(0, hi - lo) * (2 * first + lo + hi + 1) // 2 + max(0, rows - max(hi, 0)) * n
    return {"bytes": 2 * d * (size * kv * 2 * keys + size * h * (queries + b * nq)), "flops": 12 * d * h * pairs}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        x = s["x"].to(torch.float64)
        scale = (x.abs().max(dim=1).values / 127).to(torch.float32).to(torch.float64)       # the scale is kept in 32 bits
        steps = torch.where(scale[:, None] > 0, x / scale[:, None], torch.zeros_like(x)).round().clamp(-127, 127)
        y = torch.mm(steps * scale[:, None], (s["w"].to(torch.float64) * s["w_scale"].to(torch.float64)[:, None]).t())
        return y if s["bias"] is None else y + s["bias"].to(torch.float64)
    if case["op"] == "norm":
        sample = torch.arange(case["rows"], device=_DEVICE) // (case["rows"] // case["samples"])

        def normed(v, weight, bias):
            if case["kind"] == "layer":
                v = v - v.sum(-1, keepdim=True) / v.shape[-1]
            v = weight.to(torch.float64) * v / torch.sqrt((v * v).sum(-1, keepdim=True) / v.shape[-1] + 1e-5)
            return v + bias.to(torch.float64) if case["kind"] == "layer" else v

        h = normed(s["branch"].to(torch.float64), s["post_weight"], s["post_bias"])
        if case["gate"] == "full":
            h = h / (1 + torch.exp(-s["gate"].to(torch.float64)))
        elif case["gate"] != "none":
            h = h * s["gate"].to(torch.float64)[sample if case["gate"] == "sample" else torch.zeros_like(sample)]
        h = h + 0.9 * s["residual"].to(torch.float64)
        y = normed(h, s["pre_weight"], s["pre_bias"])
        if s["film"] is not None:
            y = y + y * s["film"][0].to(torch.float64)[sample] + s["film"][1].to(torch.float64)[sample]
        return {"h": h, "y": y}
    b, h, kv, d, nq = case["batch"], case["heads"], case["kv_heads"], case["d"], case["q"]
    lam = s["lambdas"].to(torch.float64)
    lam = math.exp(float(lam[0] @ lam[1])) - math.exp(float(lam[2] @ lam[3])) + 0.5
    out = torch.zeros(b, nq, h, 2 * d, dtype=torch.float64, device=_DEVICE)
    for i, n in enumerate(_lengths(case)):
        rows = n if _prompt(case) else nq
        if not n or not rows:
            continue
        seen = None
        if case["causal"]:
            seen = torch.arange(n, device=_DEVICE)[None, :] <= torch.arange(rows, device=_DEVICE)[:, None] + (0 if _prompt(case) else n - nq)
        for j in range(h):
            o = 0
            for m in (0, 1):
                score = s["q"][i, :rows, 2 * j + m].to(torch.float64) @ s["k"][i, :n, 2 * (j // (h // kv)) + m].to(torch.float64).t() / math.sqrt(d)
                if seen is not None:
                    score = torch.where(seen, score, torch.full_like(score, -math.inf))
                p = torch.nan_to_num(torch.softmax(score, -1), nan=0.0)     # a query that sees nothing answers zero
                o = o + (1.0 if m == 0 else -lam) * (p @ s["v"][i, :n, j // (h // kv)].to(torch.float64))
            out[i, :rows, j] = 0.5 * o / torch.sqrt((o * o).mean(-1, keepdim=True) + 1e-5) * s["norm_weight"].to(torch.float64)
    return out
