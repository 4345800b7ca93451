"""Transformer block operators on the device against their 64-bit definitions (oracle/transformer_oracle.py, whose bounds count roundings)."""
import math

import pytest
import torch

import tha4_amd  # noqa: F401
from oracle import transformer_oracle as oracle
from tha4_amd import _capi, transformer

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def dev():
    _capi.load_library()
    assert any("libtha4_" in l and ".so" in l for l in open("/proc/self/maps").read().splitlines())
    return torch.device("cuda:0")


def rng(seed):
    return torch.Generator(device="cuda:0").manual_seed(seed)


def randn(g, *shape, dtype=F32, std=1.0, mean=0.0):
    return torch.empty(shape, device="cuda:0", dtype=F32).normal_(mean, std, generator=g).to(dtype)


def within(got, ref):
    want, bound = ref
    assert got.shape == want.shape
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside; worst {float((off / bound).max()):.3g} of the bound at {torch.nonzero(bad)[0].tolist()}"


# ---- quantisation ----------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (1, 512), (5, 520), (2, 2048), (3, 2056), (4, 4096), (2, 8192), (2, 8200), (1, 16384), (2, 16392), (1, 20000), (7, 1111), (0, 64), (257, 64)])
def test_quantize(dtype, rows, cols):
    g = rng(rows * 1000 + cols)
    x = randn(g, rows, cols, dtype=dtype) * randn(g, rows, 1).exp().to(dtype)
    if cols > 8 and rows > 1:
        top = x[0].abs().max()
        x[0, 1], x[0, 2] = top / 2, -top / 2          # beside a tie: 63.5 steps, but for the rounding of the scale
    q, s = transformer.quantize_tokens(x)
    wq, ws = oracle.quantize(x)
    assert torch.equal(s, ws) and torch.equal(q, wq)


def test_quantize_extremes():
    x = torch.randn(9, 96, generator=torch.Generator().manual_seed(3)).to("cuda:0")
    x[0] = 0
    x[1, 5] = math.inf
    x[2, 7] = math.nan
    x[3] *= 1e38 / x[3].abs().max()
    x[4] *= 2.0 ** -130                               # a subnormal scale
    x[5] = 0
    x[5, 3] = 2.0 ** -149                             # 1 / 127 of it is 0
    x[6] = 0
    x[6, 0] = 190 * 2.0 ** -149                       # the scale rounds to one step of the subnormals: 190 of them, kept at 127
    x[7] = torch.arange(96) - 47.5
    x[7, 0] = 127.0                                   # scale 1: halves are ties
    for t in (x, x[:, :95]):                          # and with rows that are not 16-byte aligned
        q, s = transformer.quantize_tokens(t)
        wq, ws = oracle.quantize(t)
        assert torch.equal(q, wq) and torch.equal(torch.nan_to_num(s, nan=-1.0), torch.nan_to_num(ws, nan=-1.0))
        assert s[1].isnan() and s[2].isnan() and not q[1].any() and s[0] == 0 and s[5] == 0 and q[6, 0] == 127


# ---- 8-bit product ---------------------------------------------------------------------------------------------------------------------------
LINEAR = [(1, 1, 1), (1, 16, 64), (1, 4096, 4096), (2, 48, 16), (3, 130, 1111), (16, 1024, 512), (17, 33, 272), (33, 200, 4080), (64, 512, 2048), (65, 129, 144), (100, 257, 1000),
          (128, 128, 128), (129, 385, 320), (256, 256, 4096), (300, 511, 777), (511, 1024, 48), (1024, 1280, 640), (1000, 96, 8192), (1, 7, 131071), (70, 9, 131056), (512, 2048, 1024), (0, 8, 16), (2, 0, 16)]


@pytest.mark.parametrize("m,n,k", LINEAR)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_int8_linear(m, n, k, dtype):
    g = rng(m + 10 * n + 100 * k)
    q = torch.randint(-128, 128, (m, k), device="cuda:0", generator=g).to(torch.int8)
    w = torch.randint(-128, 128, (n, k), device="cuda:0", generator=g).to(torch.int8)
    qs, ws, b = randn(g, m).exp() / 100, randn(g, n).exp() / (100 * math.sqrt(k)), randn(g, n)
    for bias in (None, b):
        within(transformer.int8_linear(q, w, ws, x_scale=qs, bias=bias, out_dtype=dtype), oracle.int8_linear(q, qs, w, ws, bias, dtype))


def test_int8_linear_is_exact_at_the_largest_sums():
    for m in (1, 40, 200):
        q = torch.full((m, 131071), -128, dtype=torch.int8, device="cuda:0")
        w = torch.full((20, 131071), -128, dtype=torch.int8, device="cuda:0")
        one = torch.ones(200, device="cuda:0")
        y = transformer.int8_linear(q, w, one[:20], x_scale=one[:m], out_dtype=F32)
        assert torch.equal(y, torch.full_like(y, 131071 * 16384.0))           # 2147467264: below 2^31, a multiple of 2^14


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("m,n,k", [(1, 256, 256), (7, 65, 100), (130, 260, 512)])
def test_int8_linear_from_float_tokens(m, n, k, dtype):
    g = rng(5)
    x = randn(g, 2, m, k, dtype=dtype)
    wq, ws = transformer.quantize_tokens(randn(g, n, k))
    y = transformer.int8_linear(x, wq, ws)
    assert y.shape == (2, m, n) and y.dtype == dtype
    q, s = oracle.quantize(x)
    within(y, oracle.int8_linear(q, s, wq, ws, None, dtype))
    x[0, 0, 3] = math.nan
    y = transformer.int8_linear(x, wq, ws)
    assert y[0, 0].isnan().all() and not y[1].isnan().any() and not y[0, 1:].isnan().any()


@pytest.mark.parametrize("m", [1, 20, 150, 300])
def test_int8_linear_strided_and_unaligned(m):
    g = rng(m)
    big = torch.randint(-127, 128, (m, 700), device="cuda:0", generator=g).to(torch.int8)
    wbig = torch.randint(-127, 128, (96, 800), device="cuda:0", generator=g).to(torch.int8)
    qs, ws = torch.ones(m, device="cuda:0"), torch.ones(96, device="cuda:0") / 64
    for q, w in ((big[:, :512], wbig[:, 32:544]), (big[:, 3:515], wbig[:, :512]), (big[:, 16:517], wbig[:, 5:506]), (big[:, :512], wbig.t().contiguous().t()[:, :512])):
        within(transformer.int8_linear(q, w, ws, x_scale=qs, out_dtype=BF16), oracle.int8_linear(q, qs, w, ws, None, BF16))


# ---- norms -----------------------------------------------------------------------------------------------------------------------------------
def norm_inputs(g, shape, dtype, residual_dtype, params, gate, film):
    c = shape[-1]
    kw = dict(residual=randn(g, *shape, dtype=residual_dtype, std=2.0, mean=0.3), branch=randn(g, *shape, dtype=dtype, mean=0.5))
    for n in ("post_weight", "pre_weight"):
        kw[n] = randn(g, c, dtype=params, std=0.3, mean=1.0)
    for n in ("post_bias", "pre_bias"):
        kw[n] = randn(g, c, dtype=params, std=0.3)
    per = {"vector": (c,), "sample": (shape[0], c), "full": shape}
    kw["gate"] = None if gate is None else randn(g, *per[gate], dtype=dtype)
    kw["film"] = None if film is None else (randn(g, *per[film], dtype=params, std=0.3), randn(g, *per[film], dtype=params))
    return kw


@pytest.mark.parametrize("dtype,residual_dtype", [(F32, F32), (F16, F16), (BF16, BF16), (BF16, F32), (F16, F32)])
@pytest.mark.parametrize("shape", [(1, 1, 8), (2, 3, 64), (1, 1, 512), (3, 5, 520), (1, 2, 2048), (2, 2, 4096), (1, 3, 8192), (1, 2, 16384), (2, 3, 7), (1, 2, 1111), (1, 1, 16392), (1, 1, 40000)])
def test_residual_norm(shape, dtype, residual_dtype):
    g = rng(sum(shape))
    for i, (post, pre, gate, act, film, params) in enumerate([("rms", "rms", "full", "sigmoid", None, F32), ("layer", "layer", "sample", "none", "sample", dtype),
                                                              ("none", "rms", "vector", "none", "vector", F32), ("rms", "none", None, "none", "full", dtype)]):
        kw = norm_inputs(g, shape, dtype, residual_dtype, params, gate, film)
        kw.update(post_norm=post, pre_norm=pre, gate_activation=act, residual_scale=0.7, eps=1e-5)
        h, y = transformer.residual_norm(**kw)
        assert h.dtype == residual_dtype and y.dtype == dtype
        want_h, want_y = oracle.residual_norm(**kw)
        within(h, want_h)
        within(y, want_y)


def test_residual_norm_options():
    g = rng(9)
    x, c = randn(g, 6, 40, 256, dtype=BF16), 256
    h, y = transformer.residual_norm(x)                                        # in front of the first block
    assert torch.equal(h, x)
    within(y, oracle.residual_norm(x)[1])
    scale = randn(g, c)
    h, y = transformer.residual_norm(x, x * 2, residual_scale=scale, pre_norm="none")
    want = oracle.residual_norm(x, x * 2, residual_scale=scale, pre_norm="none")
    within(h, want[0])
    within(y, want[1])
    # a gate of one row for each sample, given with a token dimension; strided rows; an unaligned view
    gate = randn(g, 6, 1, c, dtype=BF16)
    wide = randn(g, 6, 40, 3 * c, dtype=BF16)
    h, y = transformer.residual_norm(wide[..., :c], wide[..., c:2 * c], gate=gate)
    want = oracle.residual_norm(wide[..., :c], wide[..., c:2 * c], gate=gate[:, 0])
    within(h, want[0])
    within(y, want[1])
    h, y = transformer.residual_norm(wide[..., 1:c + 1], wide[..., 2:c + 2], gate=gate)
    want = oracle.residual_norm(wide[..., 1:c + 1], wide[..., 2:c + 2], gate=gate[:, 0])
    within(h, want[0])
    within(y, want[1])
    h, y = transformer.residual_norm(x[:0], x[:0])
    assert h.shape == (0, 40, 256)
    # what would mean a row for each token of every sample is not taken for a row for each sample
    two = randn(g, 2, 2, c)
    with pytest.raises(AssertionError, match="one row"):
        transformer.residual_norm(two, two, gate=randn(g, 1, 2, c))
    with pytest.raises(AssertionError, match="one row"):
        transformer.residual_norm(two, two, film=(randn(g, 1, 2, c), randn(g, 1, 2, c)))
    for gate in (randn(g, 2, c), randn(g, 1, 1, c), randn(g, 4, c)):
        h, y = transformer.residual_norm(two, two, gate=gate)
        within(h, oracle.residual_norm(two, two, gate=gate)[0])
    # rows do not touch each other: an infinity or a NaN stays in its row; a row of zeros has no variance
    x = randn(g, 12, 512)
    b = randn(g, 12, 512)
    clean = transformer.residual_norm(x, b)
    b[3, 100], b[7, 0] = math.inf, math.nan
    b[5] = 0
    x[5] = 0
    h, y = transformer.residual_norm(x, b)
    keep = [r for r in range(12) if r not in (3, 5, 7)]
    assert torch.equal(h[keep], clean[0][keep]) and torch.equal(y[keep], clean[1][keep])
    assert not h[5].any() and not y[5].any() and y[3].isnan().any() and y[7].isnan().all()


def test_residual_norm_many_rows():
    g = rng(10)
    x, b, gate = (randn(g, 70001, 72, dtype=BF16) for _ in range(3))
    h, y = transformer.residual_norm(x, b, gate=gate, gate_activation="sigmoid")
    want = oracle.residual_norm(x, b, gate=gate, gate_activation="sigmoid")
    within(h, want[0])
    within(y, want[1])


# ---- differential attention ------------------------------------------------------------------------------------------------------------------
def attention_inputs(g, batch, q_len, k_len, heads, kv_heads, d, dtype, per_head=False):
    q, k = randn(g, batch, q_len, 2 * heads, d, dtype=dtype), randn(g, batch, k_len, 2 * kv_heads, d, dtype=dtype)
    v = randn(g, batch, k_len, kv_heads, 2 * d, dtype=dtype, mean=0.2)
    lam = randn(g, 4, heads, d, std=0.15) if per_head else randn(g, 4, d, std=0.15)
    return q, k, v, lam, randn(g, 2 * d, std=0.2, mean=1.0)


ATTENTION = [  # batch, q_len, k_len, heads, kv_heads
    (1, 1, 1, 1, 1), (2, 1, 33, 4, 1), (3, 1, 700, 8, 2), (1, 1, 5000, 4, 4), (2, 4, 1300, 4, 1), (1, 16, 16, 2, 2), (1, 17, 40, 1, 1), (2, 5, 64, 8, 2),
    (1, 128, 128, 2, 1), (2, 129, 257, 2, 2), (1, 300, 300, 4, 2), (1, 64, 1000, 2, 1), (1, 100, 9000, 3, 1), (2, 33, 5000, 4, 1), (1, 257, 31, 2, 2), (8, 256, 256, 8, 8), (1, 40, 9000, 1, 1), (3, 70, 0, 2, 1), (2, 3, 0, 2, 1)]


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: "x".join(map(str, c)))
def test_attention(case, dtype, d):
    g = rng(sum(case) + d)
    q, k, v, lam, w = attention_inputs(g, *case, d, dtype, per_head=case[0] > 1)
    for causal in (False, True):
        for norm in (True, False):
            kw = dict(causal=causal, norm=norm, norm_weight=w if norm else None)
            within(transformer.differential_attention(q, k, v, lam, 0.6, **kw), oracle.differential_attention(q, k, v, lam, 0.6, **kw))


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("q_len", [1, 3, 150, 1000])
def test_attention_lengths(q_len, d):
    """Caches of their own lengths: empty, one key, inside and at the end of a tile, full; what lies behind is NaN."""
    g = rng(q_len + d)
    lengths = torch.tensor([0, 1, 63, 64, 65, 500, 1500, 1501, -7, 99999], dtype=torch.int32, device="cuda:0")
    q, k, v, lam, w = attention_inputs(g, 10, q_len, 1501, 4, 2, d, BF16)
    for b, n in enumerate(lengths.tolist()):
        k[b, max(n, 0):], v[b, max(n, 0):] = math.nan, math.inf
    for causal in (True, False):
        got = transformer.differential_attention(q, k, v, lam, 0.5, causal=causal, kv_lengths=lengths, norm_weight=w)
        within(got, oracle.differential_attention(q, k, v, lam, 0.5, causal=causal, kv_lengths=lengths, norm_weight=w))
        assert not got[0].any() and not got[8].any()


@pytest.mark.parametrize("d", [32, 64, 128])
def test_attention_padded_batch(d):
    g = rng(d)
    lengths = torch.tensor([0, 1, 333, 200, 128], dtype=torch.int32, device="cuda:0")
    q, k, v, lam, w = attention_inputs(g, 5, 333, 333, 4, 2, d, F16)
    for b, n in enumerate(lengths.tolist()):
        q[b, n:], k[b, n:], v[b, n:] = math.nan, math.nan, math.nan
    kw = dict(causal=True, q_lengths=lengths, kv_lengths=lengths, norm_weight=w)
    want = oracle.differential_attention(torch.nan_to_num(q), k, v, lam, 0.5, **kw)
    got = transformer.differential_attention(q, k, v, lam, 0.5, **kw)
    within(got, want)
    out = torch.full_like(got, 7.0)
    assert transformer.differential_attention(q, k, v, lam, 0.5, out=out, **kw) is out
    for b, n in enumerate(lengths.tolist()):
        assert torch.equal(out[b, :n], got[b, :n]) and (out[b, n:] == 7.0).all() and not got[b, n:].any()
    few = torch.tensor([0, 1, 3, 2, 3], dtype=torch.int32, device="cuda:0")               # and on the path for few queries
    kw = dict(causal=True, q_lengths=few, kv_lengths=lengths, norm_weight=w)
    q3 = torch.nan_to_num(q[:, :3])
    out = torch.full((5, 3, 4, 2 * d), 7.0, dtype=F16, device="cuda:0")
    transformer.differential_attention(q3, k, v, lam, 0.5, out=out, **kw)
    want, bound = oracle.differential_attention(q3, k, v, lam, 0.5, **kw)
    for b, n in enumerate(few.tolist()):
        within(out[b, :n], (want[b, :n], bound[b, :n]))
        assert (out[b, n:] == 7.0).all()


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("q_len,k_len", [(1, 300), (4, 1200), (200, 130), (50, 6000)])
def test_attention_mask(q_len, k_len, d):
    g = rng(q_len + k_len + d)
    q, k, v, lam, w = attention_inputs(g, 2, q_len, k_len, 4, 2, d, BF16)
    full = torch.rand(2, 4, q_len, k_len, device="cuda:0", generator=g) > 0.6
    full[1, 2] = False                                                          # a head that sees nothing
    full[0, 1, q_len // 2] = False                                              # a row that sees nothing
    for mask in (full, full[:, :1], full[:1, :, :1], full[0, 0], full.transpose(2, 3).contiguous().transpose(2, 3)):
        for causal in (False, True):
            got = transformer.differential_attention(q, k, v, lam, 0.5, causal=causal, mask=mask, norm_weight=w)
            within(got, oracle.differential_attention(q, k, v, lam, 0.5, causal=causal, mask=mask, norm_weight=w))
    got = transformer.differential_attention(q, k, v, lam, 0.5, mask=full)
    assert not got[1, :, 2].any() and not got[0, q_len // 2, 1].any()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("q_len,k_len,bad", [(200, 200, 150), (3, 90, 88), (4, 1030, 1027), (40, 9000, 8980)])
def test_values_that_a_query_does_not_see_do_not_reach_it(q_len, k_len, bad, dtype, d):
    g = rng(bad + d)
    q, k, v, lam, w = attention_inputs(g, 2, q_len, k_len, 4, 2, d, dtype)
    clean = transformer.differential_attention(q, k, v, lam, 0.5, causal=True, norm=False)
    first = bad - (k_len - q_len)                                                # the first query that sees key `bad`
    for what in (math.nan, math.inf, -math.inf):
        k2, v2 = k.clone(), v.clone()
        v2[0, bad, 1, 5] = what
        got = transformer.differential_attention(q, k2, v2, lam, 0.5, causal=True, norm=False)
        assert torch.equal(got[1], clean[1]) and torch.equal(got[0, :first], clean[0, :first])
        hit = got[0, first:, 2:, 5]
        assert not hit.isfinite().any()
        rest = torch.ones_like(got[0, first:], dtype=torch.bool)
        rest[:, 2:, 5] = False
        assert torch.equal(got[0, first:][rest], clean[0, first:][rest])
        k2[0, bad, 2, 0] = what
        got = transformer.differential_attention(q, k2, v, lam, 0.5, causal=True, norm=False)
        assert torch.equal(got[0, :first], clean[0, :first])
    mask = torch.ones(k_len, dtype=torch.bool, device="cuda:0")
    mask[bad] = False
    want = transformer.differential_attention(q, k, v, lam, 0.5, mask=mask)
    k[:, bad], v[:, bad] = math.inf, math.nan
    assert torch.equal(transformer.differential_attention(q, k, v, lam, 0.5, mask=mask), want)


@pytest.mark.parametrize("q_len", [2, 140])
def test_attention_strided_views(q_len):
    g = rng(q_len)
    heads, kv, d, n = 4, 2, 64, 140
    fused = randn(g, 2, n, 2 * heads * d + 4 * kv * d, dtype=BF16)                # one projection, cut into q, k and v
    q = fused[:, :q_len, :2 * heads * d].unflatten(2, (2 * heads, d))
    k = fused[..., 2 * heads * d:2 * heads * d + 2 * kv * d].unflatten(2, (2 * kv, d))
    v = fused[..., 2 * heads * d + 2 * kv * d:].unflatten(2, (kv, 2 * d))
    lam, w = randn(g, 4, heads, d, std=0.1), randn(g, 2 * d)
    want = oracle.differential_attention(q, k, v, lam, 0.5, causal=True, norm_weight=w)
    within(transformer.differential_attention(q, k, v, lam, 0.5, causal=True, norm_weight=w), want)
    hq, hk, hv = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v))      # heads in front of tokens
    within(transformer.differential_attention(hq, hk, hv, lam, 0.5, causal=True, norm_weight=w), want)
    pad = [torch.cat([t, t[:, :1]], 1)[:, 1:] if t.shape[1] == n else t for t in (q, k, v)]  # another order of keys: rows that start later in memory
    assert pad[1].storage_offset() > 0
    within(transformer.differential_attention(q, pad[1], pad[2] if q_len == n else pad[2], lam, 0.5, norm_weight=w),
           oracle.differential_attention(q, pad[1], pad[2], lam, 0.5, norm_weight=w))
    odd = torch.empty(fused.numel() + 1, dtype=BF16, device="cuda:0")[1:].view_as(fused).copy_(fused)      # 2-byte aligned: copied first
    qo = odd[:, :q_len, :2 * heads * d].unflatten(2, (2 * heads, d))
    within(transformer.differential_attention(qo, k, v, lam, 0.5, causal=True, norm_weight=w), want)
    odd = torch.empty(1, 1, 2 * heads * d + 3, dtype=BF16, device="cuda:0").expand(1, 1, -1)[..., :2 * heads * d]       # one token of a row of odd length
    one = odd.unflatten(2, (2 * heads, d)).copy_(q[:1, :1])
    within(transformer.differential_attention(one, k[:1], v[:1], lam, 0.5, norm_weight=w), oracle.differential_attention(one, k[:1], v[:1], lam, 0.5, norm_weight=w))
    out = torch.empty(2, heads, q_len, 2 * d, dtype=BF16, device="cuda:0").transpose(1, 2)
    within(transformer.differential_attention(q, k, v, lam, 0.5, causal=True, norm_weight=w, out=out), want)


@pytest.mark.parametrize("q_len", [1, 200])
def test_attention_large_scores(q_len):
    """One key takes all the weight, scores in the hundreds and growing along the keys (every tile raises the maximum)."""
    g = rng(q_len)
    q, k, v, lam, w = attention_inputs(g, 1, q_len, 400, 2, 2, 64, BF16)
    k = (k * torch.linspace(0.1, 40, 400, device="cuda:0")[None, :, None, None]).to(BF16)
    within(transformer.differential_attention(q, k, v, lam, 0.5, norm_weight=w), oracle.differential_attention(q, k, v, lam, 0.5, norm_weight=w))
    within(transformer.differential_attention(q, k, v, lam, 0.5, scale=3.0), oracle.differential_attention(q, k, v, lam, 0.5, scale=3.0))


def test_cache_behind_four_gigabytes():
    """Offsets of keys beyond 2^32 bytes: all keys but the last three are zero vectors with zero values, so the answer has a closed form."""
    n, d = 2 ** 23 + 7, 128
    k = torch.zeros(1, n, 2, d, dtype=F16, device="cuda:0")
    v = torch.zeros(1, n, 1, 2 * d, dtype=F16, device="cuda:0")
    assert k.numel() * 2 > 2 ** 32 and v.numel() * 2 > 2 ** 32
    g = rng(4)
    v[0, -3:] = randn(g, 3, 1, 2 * d, dtype=F16)
    q = randn(g, 1, 1, 2, d, dtype=F16)
    k[0, -3:, 0] = q[0, 0, 0] * 4                                                # map 1 sees the last three, map 2 everything alike
    lam = torch.zeros(4, d, device="cuda:0")                                     # lambda = lambda_init
    got = transformer.differential_attention(q, k, v, lam, 0.5, norm=False)
    s = float((q[0, 0, 0].double() * k[0, -1, 0].double()).sum()) / math.sqrt(d)
    a = math.exp(s) / (3 * math.exp(s) + n - 3)
    want = (a - 0.5 / n) * v[0, -3:, 0].double().sum(0)
    assert s > 30 and (got[0, 0, 0].double() - want).abs().max() < 4e-3


# ---- as they are used ------------------------------------------------------------------------------------------------------------------------
class Block:
    """One transformer block out of the operators, and the same in 64 bits from the same int8 weights."""

    def __init__(self, g, c, heads, kv, d, dtype):
        self.heads, self.kv, self.d, self.dtype = heads, kv, d, dtype
        self.qkv = transformer.quantize_tokens(randn(g, (2 * heads + 4 * kv) * d, c, std=c ** -0.5))
        self.out = transformer.quantize_tokens(randn(g, c, heads * 2 * d, std=(2 * heads * d) ** -0.5))
        self.lam, self.sub = randn(g, 4, heads, d, std=0.1), randn(g, 2 * d, std=0.1, mean=1.0)
        self.pre, self.post, self.gate = randn(g, c, std=0.1, mean=1.0), randn(g, c, std=0.1, mean=1.0), randn(g, c, std=0.3, mean=1.0)

    def run(self, x, cache_k=None, cache_v=None, at=0, lengths=None):
        h, y = transformer.residual_norm(x, pre_weight=self.pre)
        z = transformer.int8_linear(y, *self.qkv)
        a, b = 2 * self.heads * self.d, 2 * self.kv * self.d
        q, k, v = z[..., :a].unflatten(2, (2 * self.heads, self.d)), z[..., a:a + b].unflatten(2, (2 * self.kv, self.d)), z[..., a + b:].unflatten(2, (self.kv, 2 * self.d))
        if cache_k is not None:
            cache_k[:, at:at + x.shape[1]], cache_v[:, at:at + x.shape[1]] = k, v
            k, v = cache_k, cache_v
        o = transformer.differential_attention(q, k, v, self.lam, 0.5, causal=True, kv_lengths=lengths, norm_weight=self.sub)
        return transformer.residual_norm(h, transformer.int8_linear(o.flatten(2), *self.out), gate=self.gate, post_weight=self.post, pre_weight=self.pre)

    def oracle(self, x):
        """Roundings to the type happen where the operators hand over tensors of that type; each operator is within its own bound of this."""
        t = self.dtype
        h, y = (r[0] for r in oracle.residual_norm(x, pre_weight=self.pre))
        q8, s8 = oracle.quantize(y.to(t))
        z = oracle.int8_linear(q8, s8, *self.qkv, None, t)[0].to(t)
        a, b = 2 * self.heads * self.d, 2 * self.kv * self.d
        q, k, v = z[..., :a].unflatten(2, (2 * self.heads, self.d)), z[..., a:a + b].unflatten(2, (2 * self.kv, self.d)), z[..., a + b:].unflatten(2, (self.kv, 2 * self.d))
        o = oracle.differential_attention(q, k, v, self.lam, 0.5, causal=True, norm_weight=self.sub)[0].to(t)
        q8, s8 = oracle.quantize(o.flatten(2))
        return [r[0] for r in oracle.residual_norm(x, oracle.int8_linear(q8, s8, *self.out, None, t)[0].to(t), gate=self.gate, post_weight=self.post, pre_weight=self.pre)]


def near(a, b):
    """Two runs whose roundings to bf16 and int8 fall differently here and there: each changes one element by one step, 2^-8 or 1/127 of the largest; of a row of c
    elements' sums that stays below the sum of a few such steps: 2 % of the row's norm."""
    a, b = a.double(), b.double()
    assert ((a - b).norm(dim=-1) <= 0.02 * b.norm(dim=-1)).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_block_on_a_prompt_then_token_by_token(dtype):
    g = rng(12)
    block = Block(g, 256, 4, 2, 32, dtype)
    x = randn(g, 2, 150, 256, dtype=dtype)
    h, y = block.run(x)
    want = block.oracle(x)
    near(h, want[0])
    near(y, want[1])
    ck = torch.full((2, 192, 4, 32), math.nan, dtype=dtype, device="cuda:0")      # a cache longer than what is in it
    cv = torch.full((2, 192, 2, 64), math.nan, dtype=dtype, device="cuda:0")
    n = torch.full((2,), 140, dtype=torch.int32, device="cuda:0")
    h0, y0 = block.run(x[:, :140], ck, cv, 0, n)
    near(h0, want[0][:, :140])
    for i in range(140, 150):
        n += 1
        hi, yi = block.run(x[:, i:i + 1], ck, cv, i, n)
        near(hi[:, 0], want[0][:, i])
        near(yi[:, 0], want[1][:, i])


def test_captured_blocks_replay_like_eager_calls():
    """Two graphs of the same operators with workspaces of their own, replayed in turn with eager work between."""
    g = rng(13)
    block = Block(g, 256, 4, 2, 64, BF16)
    xs = [randn(g, 1, 1, 256, dtype=BF16) for _ in range(2)]
    ck, cv = randn(g, 1, 4096, 4, 64, dtype=BF16), randn(g, 1, 4096, 2, 128, dtype=BF16)
    n = torch.full((1,), 4000, dtype=torch.int32, device="cuda:0")

    def step(x):
        h, y = block.run(x)
        q = y.expand(1, 2, 256).reshape(1, 1, 8, 64)
        return transformer.differential_attention(q, ck, cv, block.lam, 0.5, causal=True, kv_lengths=n, norm_weight=block.sub), h

    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x in xs:
            step(x)
    torch.cuda.current_stream().wait_stream(side)
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(x))
        graphs.append(graph)
    for r in range(4):
        for x in xs:
            x.normal_(generator=g)
        n.fill_(1000 * r + 3)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for x, out in zip(xs, outs):
            want = step(x)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_streams_and_repeats():
    """The same bits on another stream, called again, and beside another call in flight."""
    g = rng(14)
    q, k, v, lam, w = attention_inputs(g, 2, 1, 9000, 8, 2, 64, BF16)
    x, wq, ws = randn(g, 40, 1024, dtype=BF16), torch.randint(-127, 128, (512, 1024), device="cuda:0", generator=g).to(torch.int8), randn(g, 512).exp()
    torch.cuda.synchronize()
    want = [transformer.differential_attention(q, k, v, lam, 0.5), transformer.int8_linear(x, wq, ws), transformer.residual_norm(x, x)[1]]
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(3):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append([transformer.differential_attention(q, k, v, lam, 0.5), transformer.int8_linear(x, wq, ws), transformer.residual_norm(x, x)[1]])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for one in got for a, b in zip(one, want))


def test_refusals_on_the_device():
    x = torch.zeros(2, 64, device="cuda:0")
    with pytest.raises(AssertionError, match="gradient"):
        transformer.residual_norm(x.clone().requires_grad_())
    with torch.no_grad():
        transformer.residual_norm(x.clone().requires_grad_())
    with pytest.raises(AssertionError, match="on one GPU"):
        transformer.residual_norm(x, x, post_weight=torch.ones(64))
    one = torch.ones(64, device="cuda:0")
    with pytest.raises(AssertionError, match="all be float32"):
        transformer.residual_norm(x, x, pre_weight=one, post_weight=one.to(BF16))
    with pytest.raises(AssertionError, match="all be float32"):
        transformer.residual_norm(x, x, pre_weight=one, film=(one.half(), one.half()))
    with pytest.raises(AssertionError, match="vectors"):
        transformer.residual_norm(x, x, pre_weight=one[:1])
    with pytest.raises(AssertionError, match="one row"):
        transformer.residual_norm(torch.zeros(4, 6, 64, device="cuda:0"), torch.zeros(4, 6, 64, device="cuda:0"), gate=torch.zeros(3, 64, device="cuda:0"))
    with pytest.raises(AssertionError, match="x_scale"):
        transformer.int8_linear(x.to(torch.int8), torch.zeros(4, 64, dtype=torch.int8, device="cuda:0"), torch.ones(4, device="cuda:0"))
    with pytest.raises(_capi.Tha4Error, match="131071"):
        transformer.int8_linear(torch.zeros(1, 131072, device="cuda:0"), torch.zeros(1, 131072, dtype=torch.int8, device="cuda:0"), torch.ones(1, device="cuda:0"))
    q = torch.zeros(1, 1, 2, 64, dtype=F16, device="cuda:0")
    v = torch.zeros(1, 1, 1, 128, dtype=F16, device="cuda:0")
    with pytest.raises(_capi.Tha4Error, match="scale"):
        transformer.differential_attention(q, q, v, torch.zeros(4, 64, device="cuda:0"), 0.5, scale=-1.0)


TWIN_CODE = r'''
import sys, torch
sys.path.insert(0, sys.argv[1])
import tha4_amd
from tha4_amd import transformer as T
g = torch.Generator(device="cuda:0").manual_seed(21)
r = lambda *s, dtype=torch.bfloat16: torch.empty(s, device="cuda:0").normal_(generator=g).to(dtype)
i8 = lambda *s: torch.randint(-127, 128, s, device="cuda:0", generator=g).to(torch.int8)
out = []
for m, n, k in ((1, 512, 4096), (16, 16384, 1024), (30, 8192, 1024), (100, 300, 2048), (1024, 1280, 512), (1000, 4096, 1024), (3000, 5000, 640), (200, 257, 333)):
    out.append(T.int8_linear(r(m, k), i8(n, k), r(n, dtype=torch.float32)))
for rows, c in ((3, 256), (5, 1024), (9, 4096), (3, 8192), (2, 16384), (4, 77)):
    out += T.residual_norm(r(rows, c), r(rows, c), gate=r(rows, c), gate_activation="sigmoid", post_norm="layer")
for d in (32, 64, 128):
    lam = r(4, d, dtype=torch.float32) * 0.1
    for b, q, kl, h, kv in ((1, 700, 700, 2, 1), (16, 300, 300, 8, 8), (2, 1, 3000, 4, 1), (1, 1, 70000, 8, 2), (3, 40, 1000, 2, 2)):
        n = torch.randint(0, kl + 1, (b,), device="cuda:0", generator=g).to(torch.int32)
        Q, K, V = r(b, q, 2 * h, d), r(b, kl, 2 * kv, d), r(b, kl, kv, 2 * d)
        out += [T.differential_attention(Q, K, V, lam, 0.5, causal=True), T.differential_attention(Q, K, V, lam, 0.5, kv_lengths=n)]
torch.cuda.synchronize()
torch.save([o.cpu() for o in out], sys.argv[2])
'''


def test_same_bits_as_the_forced_wait_twin(tmp_path):
    """The library whose every wait waits for everything (csrc/libtha4_hip_wait0.so) computes the same bits: no copy, LDS read or matrix result is used before it is there."""
    import os
    import subprocess
    import sys
    from tha4_amd import _build
    if not os.path.exists(_build.TWIN) or os.path.getmtime(_build.TWIN) < os.path.getmtime(_build.LIB):
        pytest.skip("forced-wait twin not built, or older than the library")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    got = []
    for lib in (_build.LIB, _build.TWIN):
        to = str(tmp_path / os.path.basename(lib)) + ".pt"
        done = subprocess.run([sys.executable, "-c", TWIN_CODE, root, to], env=dict(os.environ, THA4_HIP_LIB=lib), capture_output=True, text=True, timeout=110)
        assert done.returncode == 0, done.stderr[-2000:]
        got.append(torch.load(to, weights_only=True))
    assert len(got[0]) == len(got[1]) and all(torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)) for a, b in zip(*got))
