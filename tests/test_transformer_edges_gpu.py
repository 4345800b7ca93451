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
