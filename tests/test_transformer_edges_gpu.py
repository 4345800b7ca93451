"""Transformer block operators on the device where their promises are hardest to keep: small differences of large maps, weights far below the largest, single kernels of
the dispatch, the ends of the ranges.  Against the same 64-bit definitions and bounds as test_transformer_gpu.py."""
import math

import pytest
import torch

import tha4_amd  # noqa: F401
from oracle import transformer_oracle as oracle
from test_transformer_gpu import attention_inputs, randn, rng, within
from tha4_amd import _capi, transformer

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def dev():
    _capi.load_library()
    assert any("libtha4_" in l and ".so" in l for l in open("/proc/self/maps").read().splitlines())


# ---- attention: the weights' precision -------------------------------------------------------------------------------------------------------
# One case for each form: prompts with 64 and with 128 queries a workgroup, few queries in one range, in several, and in several row tiles
FORMS = [(2, 200, 500, 2, 1), (8, 256, 256, 8, 8), (48, 256, 256, 4, 4), (2, 1, 200, 4, 2), (1, 4, 5000, 4, 1), (1, 40, 9000, 1, 1)]


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", FORMS, ids=lambda c: "x".join(map(str, c)))
def test_a_small_difference_of_the_maps_keeps_its_bits(case, dtype, d):
    """Maps that see nearly the same, lambda 1: what remains is a tenth of a map and less, where weights of 8 or 11 bits would cost several times the rounding of the result."""
    g = rng(sum(case) + d)
    q, k, v, _, _ = attention_inputs(g, *case, d, dtype)
    for t in (q, k):
        t[:, :, 1::2] = (0.99 * t[:, :, 0::2].float() + 0.14 * t[:, :, 1::2].float()).to(dtype)
    lam = torch.zeros(4, d, device="cuda:0")                                     # lambda = lambda_init
    for causal in (False, True):
        got = transformer.differential_attention(q, k, v, lam, 1.0, causal=causal, norm=False)
        want, bound = oracle.differential_attention(q, k, v, lam, 1.0, causal=causal, norm=False)
        within(got, (want, bound))
        rounding = (want.to(dtype).double() - want).norm() / want.norm()         # the least an answer of this type can be off
        assert (got.double() - want).norm() / want.norm() <= 1.05 * rounding


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("gap", [16.0, 18.0, 22.0])
@pytest.mark.parametrize("q_len,k_len,d", [(1, 256, 64), (1, 131072, 128), (4, 20000, 64), (300, 4096, 64), (300, 4096, 128), (256, 512, 32)])
def test_a_key_that_takes_all_the_weight_and_gives_nothing(q_len, k_len, d, gap, dtype):
    """A first key with weight e^gap times the others' and values of zero: the answer is what all the others together contribute."""
    g = rng(q_len + k_len)
    q, k, v, _, w = attention_inputs(g, 1, q_len, k_len, 2, 1, d, dtype)
    v += 0.8
    q[..., 0] = 8.0
    k *= 0.7
    k[..., 0] = 0
    k[0, 0] = 0
    k[0, 0, :, 0] = gap * math.sqrt(d) / 8.0
    v[0, 0] = 0
    lam = torch.zeros(4, d, device="cuda:0")
    kw = dict(norm_weight=w, eps=1e-14)
    want, bound = oracle.differential_attention(q, k, v, lam, 0.25, **kw)
    got = transformer.differential_attention(q, k, v, lam, 0.25, **kw)
    within(got, (want, bound))
    assert float(want.abs().mean()) > 0.1


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("q_len,k_len", [(1, 300), (200, 300), (2, 4000)])
def test_scores_beyond_the_exponents_of_a_weight(q_len, k_len, dtype):
    """Scores of 1e6 and more, where a step of the 32-bit score is a factor of the weight: still one key takes everything, and no weight leaves the type's range."""
    d = 64
    g = rng(q_len + k_len)
    q, k, v, lam, _ = attention_inputs(g, 1, q_len, k_len, 2, 1, d, dtype)
    q[...] = 0
    k[...] = 0
    q[..., 0] = 30000.0
    order = torch.randperm(k_len, device="cuda:0", generator=g)
    k[0, :, :, 0] = (order.float() * 16)[:, None].to(dtype)                      # products up to 30000 * 16 * 4000; all different, many of them within a rounding of each other's weight
    k[0, order.argmax(), :, 0] = 65504.0 if dtype == F16 else 2.0 ** 17
    got = transformer.differential_attention(q, k, v, torch.zeros(4, d, device="cuda:0"), 0.25, norm=False)
    want = v[0, order.argmax(), 0].double() * 0.75
    assert (got.double() - want).abs().max() <= 2 * oracle.half(dtype) * want.abs().max()


# ---- attention: queries that see nothing -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("q_len,k_len", [(1, 200), (3, 6000), (40, 9000), (150, 150), (300, 700), (2, 0), (70, 0)])
def test_a_query_that_sees_no_key_answers_zero_without_eps(q_len, k_len, d, dtype):
    """eps = 0: the norm of a row of zeros.  An empty sequence, a head and a row that are masked wholly, no keys at all; one range of keys, several, prompts."""
    g = rng(q_len + k_len + d)
    q, k, v, lam, w = attention_inputs(g, 2, q_len, k_len, 4, 2, d, dtype)
    lengths = torch.tensor([0, k_len], dtype=torch.int32, device="cuda:0")
    mask = torch.ones(2, 4, q_len, k_len, dtype=torch.bool, device="cuda:0")
    mask[1, 1], mask[1, 2, q_len // 2] = False, False
    for causal in (False, True):
        for kw in (dict(kv_lengths=lengths), dict(mask=mask)):
            kw.update(causal=causal, norm_weight=w, eps=0.0)
            got = transformer.differential_attention(q, k, v, lam, 0.5, **kw)
            within(got, oracle.differential_attention(q, k, v, lam, 0.5, **kw))
            assert not (got[0] if "mask" not in kw else got[1, :, 1]).any() and not (got[1, q_len // 2, 2].any() and "mask" in kw)


# ---- tensors whose memory is not all they are ------------------------------------------------------------------------------------------------
def calls(dtype=BF16):
    """(name, function, its tensor arguments by name): one call of each operator with everything that it can be given."""
    g = rng(11)
    x, c = randn(g, 6, 64, dtype=dtype), randn(g, 64)
    w = transformer.quantize_tokens(randn(g, 32, 64))
    q, k, v, lam, nw = attention_inputs(g, 2, 3, 40, 2, 1, 32, dtype)
    return [("quantize", transformer.quantize_tokens, dict(x=x)),
            ("linear", transformer.int8_linear, dict(x=x, weight=w[0], weight_scale=w[1], bias=randn(g, 32))),
            ("linear int8", lambda **a: transformer.int8_linear(w[0], out_dtype=F32, **a), dict(weight=w[0], weight_scale=w[1], x_scale=w[1], bias=randn(g, 32))),
            ("norm", lambda film_scale, film_shift, **a: transformer.residual_norm(film=(film_scale, film_shift), post_norm="layer", pre_norm="layer", **a),
             dict(residual=x, branch=x + 1, gate=x * 2, residual_scale=c, post_weight=c + 1, post_bias=c + 2, pre_weight=c + 3, pre_bias=c + 4, film_scale=randn(g, 2, 64), film_shift=randn(g, 2, 64))),
            ("attention", lambda **a: transformer.differential_attention(lambda_init=0.5, **a),
             dict(q=q, k=k, v=v, lambda_vectors=lam, norm_weight=nw, out=torch.empty(2, 3, 2, 64, dtype=dtype, device="cuda:0")))]


def negated_view(t):
    """A view that holds t's values as the negative of what lies in memory."""
    v = torch._neg_view(-t)
    assert v.is_neg() and torch.equal(v, t)
    return v


@pytest.mark.parametrize("at", range(5))
def test_negated_views_and_forward_mode_tangents_are_refused(at):
    from torch.autograd import forward_ad
    name, f, tensors = calls()[at]
    f(**tensors)
    for which, t in tensors.items():
        if not t.is_floating_point():
            continue
        with pytest.raises(AssertionError, match="negated"):
            f(**{**tensors, which: negated_view(t)})
        f(**{**tensors, which: negated_view(t).resolve_neg()})
        with forward_ad.dual_level():
            f(**tensors)                                                         # (a level without tangents changes nothing)
            with pytest.raises(AssertionError, match="tangent"):
                f(**{**tensors, which: forward_ad.make_dual(t, torch.ones_like(t))})
    z = torch.randn(6, 64, dtype=torch.complex64, device="cuda:0").conj()
    with pytest.raises(AssertionError, match="negated"):
        transformer.quantize_tokens(z.imag)


# ---- the int8 product: every kernel that its rule can choose ---------------------------------------------------------------------------------
PRODUCTS = [  # m, n, k; rows of w and x 16-byte aligned where k is a multiple of 16
    (16, 16400, 1024), (5, 16384, 80), (16, 16385, 1040),                        # few tokens, tiles of 64 channels
    (30, 16400, 512), (17, 16450, 2064),                                         # ... and 32 tokens
    (30, 8200, 1024), (32, 8193, 48),                                            # tiles of 32 channels x 32 tokens
    (32, 16401, 1001), (16, 16400, 333),                                         # the same sizes, unaligned
    (3000, 5000, 640), (3100, 4097, 2064), (3000, 5000, 333),                    # 256 x 256 tiles, aligned and not
    (1000, 4096, 1024), (1025, 3585, 144), (1000, 4096, 1001),                   # 128 x 128
    (1024, 1281, 336), (1000, 1300, 1488), (1024, 1281, 333),                    # 64 x 64, one group
    (33, 65, 16), (257, 1000, 4112), (257, 1000, 4001)]                          # 64 x 64, four groups


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_every_product_kernel_against_the_definition(m, n, k, dtype):
    g = rng(m + n + k)
    w, ws = transformer.quantize_tokens(randn(g, n, k))
    ws = ws * (randn(g, n) * 0.2).exp() / math.sqrt(k)
    bias = randn(g, n)
    x = randn(g, m, k, dtype=dtype) * randn(g, m, 1).exp().to(dtype)
    xq, xs = oracle.quantize(x)
    got = transformer.int8_linear(x, w, ws, bias=bias)
    within(got, oracle.int8_linear(xq, xs, w, ws, bias, dtype))
    assert torch.equal(transformer.int8_linear(xq, w, ws, x_scale=xs, bias=bias, out_dtype=dtype), got)
    within(transformer.int8_linear(xq, w, ws, x_scale=xs, out_dtype=dtype), oracle.int8_linear(xq, xs, w, ws, None, dtype))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("m,n,k", [(3, 130, 1111), (1, 65, 20001), (1, 300, 32768), (1, 33, 32769), (4, 70, 8192), (4, 70, 8193), (2, 100, 4100), (3, 64, 4104), (4, 50, 1), (2, 17, 15)])
def test_tokens_quantised_inside_the_product(m, n, k, dtype):
    g = rng(m * n + k)
    w, ws = transformer.quantize_tokens(randn(g, n, k))
    bias = randn(g, n)
    wide = randn(g, m, k + 5, dtype=dtype)
    for x in (wide[:, :k].contiguous(), wide[:, :k], wide[:, 5:]):               # rows of another stride, at another alignment
        xq, xs = oracle.quantize(x)
        within(transformer.int8_linear(x, w, ws / math.sqrt(k), bias=bias), oracle.int8_linear(xq, xs, w, ws / math.sqrt(k), bias, dtype))


@pytest.mark.parametrize("m,n", [(1, 64), (20, 130), (33, 65), (600, 520)])
@pytest.mark.parametrize("k", [131071, 131056])
def test_the_longest_sums_are_exact(m, n, k):
    """k = 131071 of the largest products: 2^31 - 16384, and the same negative; scales of one, so the answer is the integer rounded to fp32."""
    x = torch.full((m, k), -128, dtype=torch.int8, device="cuda:0")
    w = torch.full((n, k), -128, dtype=torch.int8, device="cuda:0")
    x[0::2, 77], w[1::2] = 127, 127
    x[m // 2] = torch.randint(-128, 128, (k,), device="cuda:0", generator=rng(k + m)).to(torch.int8)
    one = lambda c: torch.ones(c, device="cuda:0")
    got = transformer.int8_linear(x, w, one(n), x_scale=one(m), out_dtype=F32)
    assert torch.equal(got, (x.double() @ w.double().t()).float())


# ---- more rows, channels or sequences than one launch has workgroups -------------------------------------------------------------------------
def places(n, *borders):
    """Slices around 0, the borders between launches, and the end."""
    return [slice(max(at - 40, 0), min(at + 40, n)) for at in (0, *borders, n)]


@pytest.mark.parametrize("rows,cols", [(2 ** 24 + 333, 7), (2 ** 26 + 111, 8)])      # a workgroup a row, four rows a workgroup
def test_more_rows_than_one_launch_holds(rows, cols):
    g = rng(cols)
    border = (2 ** 32 - 1) // 256 * (1 if cols == 7 else 4)
    assert rows > border
    x = torch.empty(rows, cols, dtype=BF16, device="cuda:0").normal_(generator=g)
    q, s = transformer.quantize_tokens(x)
    h, y = transformer.residual_norm(x, x, gate=x, pre_norm="layer")
    for p in places(rows, border):
        wq, ws = oracle.quantize(x[p])
        assert torch.equal(q[p], wq) and torch.equal(s[p], ws)
        (wh, bh), (wy, by) = oracle.residual_norm(x[p], x[p], x[p], pre_norm="layer")
        within(h[p], (wh, bh))
        within(y[p], (wy, by))
    gate = randn(g, 1, cols, dtype=BF16)
    film = randn(g, 1, cols), randn(g, 1, cols)
    h, y = transformer.residual_norm(x, x, gate=gate, film=film)
    for p in places(rows, border):
        (wh, bh), (wy, by) = oracle.residual_norm(x[p], x[p], gate, film=film)
        within(h[p], (wh, bh))
        within(y[p], (wy, by))


def test_more_channels_than_one_launch_holds():
    n, k = 2 ** 27 + 1000, 3
    g = rng(5)
    border = (2 ** 32 - 1) // 512 * 16
    w = torch.randint(-127, 128, (n, k), dtype=torch.int8, device="cuda:0", generator=g)
    ws = torch.empty(n, device="cuda:0").uniform_(0.5, 2.0, generator=g)
    bias = torch.empty(n, device="cuda:0").normal_(generator=g)
    x = randn(g, 2, k, dtype=F16)
    y = transformer.int8_linear(x, w, ws, bias=bias)
    xq, xs = oracle.quantize(x)
    y8 = transformer.int8_linear(xq[:1], w, ws, x_scale=xs[:1], bias=bias, out_dtype=BF16)
    for p in places(n, border):
        within(y[:, p], oracle.int8_linear(xq, xs, w[p], ws[p], bias[p], F16))
        within(y8[:, p], oracle.int8_linear(xq[:1], xs[:1], w[p], ws[p], bias[p], BF16))


def test_more_tiles_than_one_launch_holds():
    m, k = 2 ** 31 - 1, 1
    border = (2 ** 32 - 1) // 512 * 256
    x = torch.arange(97, device="cuda:0", dtype=torch.int16).sub_(48).to(torch.int8).repeat(m // 97 + 1)[:m, None]
    w = torch.tensor([[3]], dtype=torch.int8, device="cuda:0")
    xs = torch.full((1,), 0.5, device="cuda:0").expand(m).contiguous()
    y = transformer.int8_linear(x, w, torch.ones(1, device="cuda:0"), x_scale=xs, out_dtype=F16)
    for p in places(m, border):
        assert torch.equal(y[p], (x[p].float() * 1.5).half())


@pytest.mark.parametrize("q_len,heads,batch", [(1, 1, 2 ** 24 + 100), (16, 1, 2 ** 24 + 100), (17, 2, 2 ** 22 + 100)])     # few queries in one range, prompts
def test_more_sequences_than_one_launch_holds(q_len, heads, batch):
    d = 32
    g = rng(q_len)
    border = (2 ** 32 - 1) // 256 if q_len <= 16 else (2 ** 32 - 1) // 512 // heads
    q1, k1, v1, _, _ = attention_inputs(g, 7, q_len, 2, heads, 1, d, BF16)
    lam = torch.zeros(4, d, device="cuda:0")
    index = torch.arange(batch, device="cuda:0") % 7
    q = q1[:1].expand(batch, -1, -1, -1)
    v = v1[index]
    k = k1[:1].expand(batch, -1, -1, -1)
    lengths = (index % 3).to(torch.int32)
    mask = (torch.arange(batch, device="cuda:0") % 5 != 3)[:, None, None, None]
    got = transformer.differential_attention(q, k, v, lam, 0.5, kv_lengths=lengths, mask=mask, norm=False)
    for p in places(batch, border):
        kw = dict(kv_lengths=lengths[p], mask=mask[p], norm=False)
        within(got[p], oracle.differential_attention(q[p], k[p], v[p], lam, 0.5, **kw))
    del got
    q_lengths = (torch.arange(batch, device="cuda:0") % (q_len + 1)).to(torch.int32)
    out = torch.empty(batch, q_len, heads, 2 * d, dtype=BF16, device="cuda:0").fill_(7.0)
    transformer.differential_attention(q, k, v, lam, 0.5, q_lengths=q_lengths, causal=True, norm=False, out=out)
    for p in places(batch, border):
        want, bound = oracle.differential_attention(q[p], k[p], v[p], lam, 0.5, q_lengths=q_lengths[p], causal=True, norm=False)
        valid = torch.arange(q_len, device="cuda:0")[None] < q_lengths[p][:, None]
        assert (out[p][~valid] == 7.0).all()
        within(out[p][valid], (want[valid], bound[valid]))


# ---- graphs whose lengths and masks change between replays -----------------------------------------------------------------------------------
@pytest.mark.parametrize("q_len,k_len", [(300, 300), (3, 5000)])
def test_a_captured_padded_batch_replays_with_other_lengths(q_len, k_len):
    """Lengths, mask and inputs are read when the graph runs; rows behind the last query are zero again in every replay.  q has to be copied first (2-byte aligned)."""
    g = rng(q_len)
    q, k, v, lam, w = attention_inputs(g, 4, q_len, k_len, 4, 2, 64, F16)
    q = torch.empty(q.numel() + 1, dtype=F16, device="cuda:0")[1:].view_as(q).copy_(q)
    nq, nk = torch.zeros(4, dtype=torch.int32, device="cuda:0"), torch.zeros(4, dtype=torch.int32, device="cuda:0")
    mask = torch.ones(4, 1, q_len, k_len, dtype=torch.bool, device="cuda:0")

    def step():
        return transformer.differential_attention(q, k, v, lam, 0.5, causal=True, q_lengths=nq, kv_lengths=nk, mask=mask, norm_weight=w)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for r in range(5):
        nq.copy_(torch.randint(0, q_len + 1, (4,), device="cuda:0", generator=g))
        nk.copy_(torch.randint(0, k_len + 1, (4,), device="cuda:0", generator=g))
        mask.copy_(torch.rand(mask.shape, device="cuda:0", generator=g) > 0.3)
        q.normal_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        within(out, oracle.differential_attention(q, k, v, lam, 0.5, causal=True, q_lengths=nq, kv_lengths=nk, mask=mask, norm_weight=w))


def test_two_host_threads_call_at_once():
    """Each on a stream of its own, with refused calls between: the bits of a call made alone, and every thread its own error text."""
    import threading
    g = rng(21)
    q, k, v, lam, w = attention_inputs(g, 2, 2, 3000, 8, 2, 64, BF16)
    x, wq, ws = randn(g, 7, 1024, dtype=F16), torch.randint(-127, 128, (512, 1024), device="cuda:0", generator=g).to(torch.int8), randn(g, 512).exp()

    def calls():
        return [transformer.differential_attention(q, k, v, lam, 0.5), transformer.int8_linear(x, wq, ws), *transformer.residual_norm(x, x)]

    want = calls()
    torch.cuda.synchronize()
    failed = []

    def work(refused, word):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(30):
                    got = calls()
                    with pytest.raises(_capi.Tha4Error, match=word):
                        refused()
                    s.synchronize()
                    assert all(torch.equal(a, b) for a, b in zip(got, want))
        except BaseException as e:
            failed.append(e)

    threads = [threading.Thread(target=work, args=a) for a in ((lambda: transformer.residual_norm(x, x, eps=-1.0), "eps"),
                                                               (lambda: transformer.differential_attention(q, k, v, lam, 0.5, scale=-1.0), "scale"))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
