"""Transformer block operators, without a GPU: what the entry points refuse, and the 64-bit oracle against direct statements of the definitions."""
import ctypes as C
import math

import pytest
import torch

import tha4_amd  # noqa: F401
from oracle import transformer_oracle as oracle
from tha4_amd import _capi, transformer


@pytest.fixture(scope="module")
def lib(built):
    return _capi.load_library()


def host(n=64):
    """Host memory that no entry point may take for device memory."""
    b = (C.c_char * n)()
    return C.cast(b, C.c_void_p), b


def refused(lib, status, *words):
    assert status == -1
    text = lib.tha4_last_error().decode()
    for w in words:
        assert w in text, text


def test_quantize_refuses(lib):
    p, keep = host()
    q = lib.tha4_quantize_tokens_i8
    refused(lib, q(p, 3, 1, 8, 8, p, 8, p, None), "x_dtype")
    refused(lib, q(p, 0, -1, 8, 8, p, 8, p, None), "rows")
    refused(lib, q(p, 0, 1, 0, 8, p, 8, p, None), "cols")
    refused(lib, q(None, 0, 1, 8, 8, p, 8, p, None), "NULL")
    refused(lib, q(p, 0, 1, 8, 8, p, 4, p, None), "q_row_stride")
    refused(lib, q(p, 0, 1, 8, 8, p, 8, p, None), "device pointers")
    assert q(None, 0, 0, 8, 8, None, 8, None, None) == 0                     # no rows: nothing to do


def linear_args(p, **more):
    a = dict(x_dev=p, x_scale_dev=p, w_dev=p, w_scale_dev=p, bias_dev=None, y_dev=p, m=1, n=1, k=1, x_row_stride=1, w_row_stride=1, y_row_stride=1, x_dtype=3, y_dtype=0)
    a.update(more)
    return C.byref(_capi.Tha4LinearI8Args(**{n: v.value if isinstance(v, C.c_void_p) else v for n, v in a.items()}))


def test_linear_refuses(lib):
    p, keep = host()
    f = lib.tha4_linear_i8
    refused(lib, f(None, None), "NULL")
    assert lib.tha4_linear_i8_workspace(None) == -1
    refused(lib, f(linear_args(p, y_dtype=7), None), "y_dtype")
    refused(lib, f(linear_args(p, x_dtype=4), None), "x_dtype")
    refused(lib, lib.tha4_linear_i8_workspace(linear_args(p, x_dtype=4)), "x_dtype")
    refused(lib, f(linear_args(p, x_scale_dev=None), None), "x_scale")
    refused(lib, f(linear_args(p, x_dtype=2), None), "x_scale")
    refused(lib, f(linear_args(p, x_dtype=2, x_scale_dev=None, m=100, k=64, x_row_stride=64), None), "workspace")
    refused(lib, f(linear_args(p, k=0), None), "k must be positive")
    refused(lib, f(linear_args(p, m=-1), None), "negative")
    refused(lib, f(linear_args(p, k=131072), None), "131071")
    refused(lib, f(linear_args(p, w_scale_dev=None), None), "NULL")
    refused(lib, f(linear_args(p, n=2), None), "y_row_stride")
    refused(lib, f(linear_args(p), None), "device pointers")
    assert f(linear_args(None, m=0), None) == 0


def norm_args(p, **more):
    a = dict(residual_dev=p, branch_dev=p, h_dev=p, y_dev=p, rows=1, cols=8, residual_row_stride=8, branch_row_stride=8, h_row_stride=8, y_row_stride=8, gate_rows=1, film_rows=1,
             residual_scale=1.0, eps=1e-5)
    a.update(more)
    return C.byref(_capi.Tha4ResidualNormArgs(**{n: v.value if isinstance(v, C.c_void_p) else v for n, v in a.items()}))


def test_norm_refuses(lib):
    p, keep = host()
    f = lib.tha4_residual_norm
    refused(lib, f(None, None), "NULL")
    refused(lib, f(norm_args(p, dtype=9), None), "dtype")
    refused(lib, f(norm_args(p, residual_dtype=1), None), "residual_dtype")
    refused(lib, f(norm_args(p, post_norm=3), None), "norm")
    refused(lib, f(norm_args(p, gate_activation=2), None), "gate")
    refused(lib, f(norm_args(p, cols=0), None), "cols")
    refused(lib, f(norm_args(p, eps=-1.0), None), "eps")
    refused(lib, f(norm_args(p, eps=math.nan), None), "eps")
    refused(lib, f(norm_args(p, residual_scale=math.inf), None), "residual_scale")
    refused(lib, f(norm_args(p, residual_dev=None), None), "residual")
    refused(lib, f(norm_args(p, branch_dev=None, gate_dev=p), None), "branch")
    refused(lib, f(norm_args(p, film_scale_dev=p), None), "together")
    refused(lib, f(norm_args(p, y_dev=None, pre_weight_dev=p), None), "need y")
    refused(lib, f(norm_args(p, h_dev=None, y_dev=None), None), "one of h and y")
    refused(lib, f(norm_args(p, gate_dev=p, gate_rows=0), None), "gate_rows")
    refused(lib, f(norm_args(p, y_row_stride=4), None), "strides")
    refused(lib, f(norm_args(p, residual_row_stride=-8), None), "negative")
    refused(lib, f(norm_args(p), None), "device pointers")
    assert f(norm_args(None, rows=0), None) == 0


def attention_args(p, **more):
    a = dict(q_dev=p, k_dev=p, v_dev=p, out_dev=p, lambda_vectors_dev=p, dtype=2, batch=1, q_len=1, k_len=1, heads=1, kv_heads=1, head_dim=32, scale=1.0, lambda_init=0.5, eps=1e-5)
    a.update(more)
    return C.byref(_capi.Tha4DiffAttentionArgs(**{n: v.value if isinstance(v, C.c_void_p) else v for n, v in a.items()}))


def test_attention_refuses(lib):
    p, keep = host(256)
    p = C.c_void_p((p.value + 15) // 16 * 16)
    f = lib.tha4_diff_attention
    refused(lib, f(None, None), "NULL")
    assert lib.tha4_diff_attention_workspace(None) == -1
    for call in (lambda a: f(a, None), lib.tha4_diff_attention_workspace):
        refused(lib, call(attention_args(p, dtype=0)), "f16 or bf16")
        refused(lib, call(attention_args(p, head_dim=48)), "head_dim")
        refused(lib, call(attention_args(p, heads=3, kv_heads=2)), "multiple")
        refused(lib, call(attention_args(p, kv_heads=0)), "kv_heads")
        refused(lib, call(attention_args(p, q_len=-1)), "negative")
    refused(lib, f(attention_args(p, scale=0.0), None), "scale")
    refused(lib, f(attention_args(p, scale=math.nan), None), "scale")
    refused(lib, f(attention_args(p, eps=-1.0), None), "eps")
    refused(lib, f(attention_args(p, lambda_init=math.inf), None), "lambda_init")
    refused(lib, f(attention_args(p, q_dev=None), None), "NULL")
    refused(lib, f(attention_args(p, k_dev=None), None), "k / v")
    refused(lib, f(attention_args(C.c_void_p(p.value + 2)), None), "aligned")
    refused(lib, f(attention_args(p, k_stride_1=4), None), "multiples of 8")
    refused(lib, f(attention_args(p, k_stride_1=1 << 24), None), "2^24")
    refused(lib, f(attention_args(p, k_stride_0=-8), None), "negative")
    refused(lib, f(attention_args(p, k_len=1 << 20), None), "workspace")     # few queries over a long cache: its ranges meet in a workspace
    refused(lib, f(attention_args(p), None), "device pointers")
    assert f(attention_args(p, batch=0), None) == 0
    assert f(attention_args(p, q_len=0), None) == 0


def test_argument_blocks_have_the_header_s_layout(tmp_path):
    """Sizes and a late field's offset of the ctypes mirrors against the compiler's."""
    import os
    import subprocess
    from tha4_amd import _build
    names = {"tha4_linear_i8_args": (_capi.Tha4LinearI8Args, "y_dtype"), "tha4_residual_norm_args": (_capi.Tha4ResidualNormArgs, "eps"),
             "tha4_diff_attention_args": (_capi.Tha4DiffAttentionArgs, "lambda_init")}
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "tha4_hip.h"\nint main(void) {' +
                   "".join(f'printf("%zu %zu\\n", sizeof({n}), offsetof({n}, {f}));' for n, (_, f) in names.items()) + "return 0;}\n")
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-I", _build.INCLUDE, str(src), "-o", exe], check=True)
    lines = subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split("\n")
    for (cls, field), line in zip(names.values(), lines):
        assert line.split() == [str(C.sizeof(cls)), str(getattr(cls, field).offset)]


def test_workspace_is_a_function_of_the_sizes(lib):
    a = attention_args(None, k_len=131072, batch=2, heads=8, kv_heads=2, head_dim=128)
    n = lib.tha4_diff_attention_workspace(a)
    assert n > 0 and n == lib.tha4_diff_attention_workspace(a)
    assert lib.tha4_diff_attention_workspace(attention_args(None, q_len=512, k_len=512)) == 0
    assert lib.tha4_diff_attention_workspace(attention_args(None, q_len=64, k_len=32768, head_dim=128)) > 0      # few prompts' workgroups over many keys: divided, too
    assert lib.tha4_diff_attention_workspace(attention_args(None, q_len=8192, k_len=8192, heads=64, kv_heads=64)) == 0


def test_python_refuses_cpu_tensors_and_wrong_shapes(lib):
    x = torch.zeros(2, 32)
    w, ws = torch.zeros(4, 32, dtype=torch.int8), torch.ones(4)
    with pytest.raises(AssertionError, match="GPU"):
        transformer.quantize_tokens(x)
    with pytest.raises(AssertionError, match="float32, float16 or bfloat16"):
        transformer.quantize_tokens(x.double())
    with pytest.raises(AssertionError, match="GPU"):
        transformer.int8_linear(x, w, ws)
    with pytest.raises(AssertionError, match=r"\[\.\.\., 32\]"):
        transformer.int8_linear(torch.zeros(2, 31), w, ws)
    with pytest.raises(AssertionError, match="weight_scale"):
        transformer.int8_linear(x, w, torch.ones(5))
    with pytest.raises(AssertionError, match="GPU"):
        transformer.residual_norm(x)
    with pytest.raises(AssertionError, match="shape"):
        transformer.residual_norm(x, torch.zeros(3, 32))
    with pytest.raises(AssertionError, match="post_norm"):
        transformer.residual_norm(x, x, post_norm="batch")
    q = torch.zeros(1, 3, 4, 32, dtype=torch.bfloat16)
    v = torch.zeros(1, 3, 2, 64, dtype=torch.bfloat16)
    lam = torch.zeros(4, 32)
    with pytest.raises(AssertionError, match="GPU"):
        transformer.differential_attention(q, q, v, lam, 0.5)
    with pytest.raises(AssertionError, match="float16"):
        transformer.differential_attention(q.float(), q.float(), v.float(), lam, 0.5)
    with pytest.raises(AssertionError, match="v \\[batch"):
        transformer.differential_attention(q, q, v[..., :32], lam, 0.5)
    with pytest.raises(AssertionError, match="pairs"):
        transformer.differential_attention(q[:, :, :3], q, v, lam, 0.5)
    with pytest.raises(AssertionError, match="lambda_vectors"):
        transformer.differential_attention(q, q, v, lam[:2], 0.5)
    with pytest.raises(AssertionError, match="int32"):
        transformer.differential_attention(q, q, v, lam, 0.5, kv_lengths=torch.ones(1))


def test_oracle_quantize_rounds_the_exact_quotient():
    from fractions import Fraction
    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, 40, generator=g)
    x[1] = x[1].to(torch.bfloat16).float()
    x[2, 3], x[2, 4] = x[2].abs().max(), x[2].abs().max() / 2            # half of the largest: next to a tie
    x[3] *= 2.0 ** -140                                                    # a scale among the subnormals
    x[4] = 0
    q, s = oracle.quantize(x)
    for r in range(6):
        for c in range(40):
            if float(s[r]) == 0:
                assert q[r, c] == 0
                continue
            t = Fraction(float(x[r, c])) / Fraction(float(s[r]))
            assert int(q[r, c]) == max(-127, min(127, round(t)))           # Fraction rounds ties to even


def test_oracle_attention_against_a_direct_statement():
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(2, 5, n, d, generator=g).double() for n, d in ((4, 32), (2, 32), (1, 64)))
    k, v = torch.cat([k, k], 1)[:, :7], torch.cat([v, v], 1)[:, :7]
    lam, w = torch.randn(4, 2, 32, generator=g) * 0.1, torch.rand(64, generator=g)
    mask = torch.rand(2, 1, 5, 7, generator=g) > 0.3
    q, k, v = q.half(), k.half(), v.half()
    out, bound = oracle.differential_attention(q, k, v, lam, 0.4, causal=True, kv_lengths=torch.tensor([7, 3]), mask=mask, norm_weight=w)
    for b in range(2):
        n = (7, 3)[b]
        for h in range(2):
            la = math.exp(float(lam[0, h].double() @ lam[1, h].double())) - math.exp(float(lam[2, h].double() @ lam[3, h].double())) + 0.4
            for i in range(5):
                see = [j for j in range(n) if j <= i + n - 5 and mask[b, 0, i, j]]
                o = torch.zeros(64, dtype=torch.float64)
                for m, sign in ((0, 1.0), (1, -la)):
                    if see:
                        p = torch.softmax((k[b, see, m].double() @ q[b, i, 2 * h + m].double()) / math.sqrt(32), 0)
                        o += sign * (p @ v[b, see, 0].double())
                o = 0.6 * o / torch.sqrt((o * o).mean() + 1e-5) * w
                assert torch.allclose(out[b, i, h], o, atol=1e-12)
    assert (bound >= 0).all() and float(bound.max()) < 0.02


def test_oracle_attention_of_nothing_is_zero_without_eps():
    g = torch.Generator().manual_seed(3)
    q, k, v = torch.randn(2, 4, 2, 32, generator=g).half(), torch.randn(2, 6, 2, 32, generator=g).half(), torch.randn(2, 6, 1, 64, generator=g).half()
    out, bound = oracle.differential_attention(q, k, v, torch.zeros(4, 32), 0.5, kv_lengths=torch.tensor([0, 6]), eps=0.0)
    assert not out[0].any() and out[1].abs().min(-1)[0].isfinite().all() and bound.isfinite().all()
    assert torch.allclose((out[1] ** 2).mean(-1), torch.full((4, 1), 0.25, dtype=torch.float64))


def test_attention_refuses_a_scale_that_overflows_with_its_factor(lib):
    """The softmax is taken in powers of two: scale * log2(e) has to be a number, or every difference of scores is 0 * inf."""
    p, keep = host(256)
    p = C.c_void_p((p.value + 15) // 16 * 16)
    refused(lib, lib.tha4_diff_attention(attention_args(p, scale=2.5e38), None), "scale")
    refused(lib, lib.tha4_diff_attention(attention_args(p, scale=2.3e38), None), "device pointers")


def test_nothing_in_the_operators_object_can_throw(built):
    """Host code of the operators allocates nothing and throws nothing (a C entry point has no one to catch it): its object needs no symbol for either."""
    import os
    import subprocess
    from tha4_amd import _build
    obj = os.path.join(_build.OBJECTS, "tha4_transformer.product.o")
    if not os.path.exists(obj):
        pytest.skip("the library was built elsewhere: its objects are not here")
    names = subprocess.run(["nm", "-u", "-C", obj], capture_output=True, text=True, check=True).stdout
    for word in ("std::__throw", "__cxa_throw", "operator new", "basic_string", "vector"):
        assert word not in names, [l for l in names.splitlines() if word in l]


def test_attention_refuses_an_output_whose_rows_overlap(lib):
    p, keep = host(256)
    p = C.c_void_p((p.value + 15) // 16 * 16)
    shape = dict(batch=2, q_len=3, heads=4, kv_heads=2, k_len=5, head_dim=32)
    for batch, token, head in ((0, 256, 64), (768, 0, 64), (768, 256, 0), (768, 256, 60), (768, 128, 64), (512, 256, 64), (64, 512, 64)):
        refused(lib, lib.tha4_diff_attention(attention_args(p, out_stride_0=batch, out_stride_1=token, out_stride_2=head, **shape), None), "overlap")
    for batch, token, head in ((768, 256, 64), (256, 512, 64), (64 * 12, 64, 64 * 3), (64, 512, 128), (64 * 3, 64, 64 * 6), (0, 256, 64)):
        many = dict(shape, batch=1) if batch == 0 else shape                      # (64, 512, 128): rows b + 8 t + 2 h, all different
        refused(lib, lib.tha4_diff_attention(attention_args(p, out_stride_0=batch, out_stride_1=token, out_stride_2=head, **many), None), "device pointers")


def test_oracle_norm_bound_holds_for_a_perfect_answer_among_the_subnormals():
    """The least that an fp16 answer can be off, for values down to the subnormals, is inside the bound."""
    x = (torch.randn(4, 64, generator=torch.Generator().manual_seed(4)) * torch.logspace(-7, 0, 64)).half()
    for want, bound in oracle.residual_norm(x, x, post_norm="none", pre_norm="rms", eps=1.0):
        assert ((want.half().double() - want).abs() <= bound).all()
        assert (want.abs() < 2.0 ** -14).any()
