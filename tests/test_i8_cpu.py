"""Refusals of the 8-bit operators, at the C ABI and from Python: nothing here
launches a kernel or needs a GPU."""

import ctypes as C

import pytest

import ridge_b200 as rb
from ridge_b200._native import RIDGE_BF16, RIDGE_EINVAL, RIDGE_F16, RIDGE_F32, RIDGE_OK, lib

torch = pytest.importorskip("torch")

P = 1 << 20          # a pointer-like value on every alignment used here; never read
Q, S, X, R, W, H = (P * i for i in range(1, 7))


def quantize(x=X, type=RIDGE_F16, q=Q, scale=S, M=4, D=64, ldx=64, ldq=64):
    return lib.ridge_quantize_i8(x, type, q, scale, M, D, ldx, ldq, None)


def norm(x=X, residual=R, weight=W, type=RIDGE_BF16, residual_out=H, q=Q, scale=S, M=4, D=64,
         ldx=64, ldr=64, ldro=64, ldq=64, eps=1e-6):
    return lib.ridge_rms_norm_i8(x, residual, weight, type, residual_out, q, scale, M, D, ldx, ldr,
                                 ldro, ldq, eps, None)


def silu(gate=X, up=R, type=RIDGE_F32, q=Q, scale=S, M=4, D=64, ldg=64, ldu=64, ldq=64):
    return lib.ridge_silu_mul_i8(gate, up, type, q, scale, M, D, ldg, ldu, ldq, None)


def dequantize(q=Q, scale=S, type=RIDGE_F16, out=X, M=4, D=64, ldq=64, ldo=64):
    return lib.ridge_dequantize_i8(q, scale, type, out, M, D, ldq, ldo, None)


def gemm(A=X, sa=S, B=R, sb=W, bias=None, type=RIDGE_F16, Cp=H, M=4, N=8, K=64, lda=64, ldb=64,
         ldc=8):
    return lib.ridge_gemm_i8(A, sa, B, sb, bias, type, Cp, M, N, K, lda, ldb, ldc, None)


ROWS = [quantize, norm, silu, dequantize]


@pytest.mark.parametrize("call", ROWS + [gemm], ids=lambda f: f.__name__)
@pytest.mark.parametrize("bad", [dict(type=3), dict(type=-1), dict(M=-1), dict(M=1 << 31)], ids=str)
def test_types_and_extents(call, bad):
    assert call(**bad) == RIDGE_EINVAL


@pytest.mark.parametrize("call", ROWS, ids=lambda f: f.__name__)
@pytest.mark.parametrize("bad", [dict(D=-1), dict(D=1 << 31), dict(ldq=63), dict(q=None),
                                 dict(scale=None), dict(scale=S + 2), dict(ldq=1 << 57)], ids=str)
def test_rows(call, bad):
    assert call(**bad) == RIDGE_EINVAL


@pytest.mark.parametrize("call,bad", [
    (quantize, dict(x=None)), (quantize, dict(x=X + 1)), (quantize, dict(ldx=63)),
    (norm, dict(x=None)), (norm, dict(weight=None)), (norm, dict(weight=W + 1)),
    (norm, dict(residual=None)), (norm, dict(residual_out=None)), (norm, dict(ldr=10)),
    (norm, dict(ldro=10)), (norm, dict(eps=0.0)), (norm, dict(eps=-1.0)),
    (norm, dict(eps=float("nan"))), (norm, dict(eps=float("inf"))),
    (silu, dict(gate=None)), (silu, dict(up=None)), (silu, dict(up=R + 2)), (silu, dict(ldu=1)),
    (dequantize, dict(out=None)), (dequantize, dict(out=X + 1)), (dequantize, dict(ldo=63)),
], ids=lambda v: v.__name__ if callable(v) else str(v))
def test_operands(call, bad):
    assert call(**bad) == RIDGE_EINVAL


@pytest.mark.parametrize("call,bad", [
    (quantize, dict(q=X)), (quantize, dict(q=X + 3 * 128 + 100)), (quantize, dict(scale=X)),
    (quantize, dict(scale=Q + 100)),
    (norm, dict(q=X)), (norm, dict(q=R)), (norm, dict(q=W)), (norm, dict(q=H)),
    (norm, dict(scale=H + 64)), (norm, dict(residual_out=W - 128)),
    (norm, dict(residual_out=X + 2)),                   # neither x nor apart from it
    (norm, dict(residual_out=X, ldro=72)),              # x, at another pitch
    (silu, dict(q=R + 64)), (dequantize, dict(out=Q)), (dequantize, dict(out=S)),
    (gemm, dict(Cp=X)), (gemm, dict(Cp=R)), (gemm, dict(Cp=S)), (gemm, dict(Cp=W)),
    (gemm, dict(bias=H)),
], ids=lambda v: v.__name__ if callable(v) else str(v))
def test_outputs_do_not_share_bytes(call, bad):
    assert call(**bad) == RIDGE_EINVAL


@pytest.mark.parametrize("bad", [
    dict(N=-1), dict(K=-1), dict(N=1 << 31), dict(K=1 << 17, lda=1 << 17, ldb=1 << 17),
    dict(lda=48), dict(lda=72), dict(ldb=72), dict(ldb=32), dict(ldc=7), dict(A=X + 8),
    dict(B=R + 8), dict(A=None), dict(B=None), dict(sa=None), dict(sb=None), dict(Cp=None),
    dict(sa=S + 1), dict(sb=W + 2), dict(Cp=H + 1), dict(bias=Q + 1), dict(lda=1 << 40),
    dict(ldc=1 << 57),
], ids=str)
def test_gemm_operands(bad):
    assert gemm(**bad) == RIDGE_EINVAL


def test_nothing_to_do_is_ok():
    for call in ROWS + [gemm]:
        assert call(M=0) == RIDGE_OK
    assert gemm(N=0) == RIDGE_OK
    assert dequantize(D=0) == RIDGE_OK


def test_python_refuses_what_is_not_on_a_gpu_or_not_rows():
    x = torch.zeros(4, 64, dtype=torch.float16)
    q = torch.zeros(4, 64, dtype=torch.int8)
    s = torch.zeros(4)
    with pytest.raises(ValueError):
        rb.quantize_i8(x)
    with pytest.raises(TypeError):
        rb.quantize_i8(x.double())
    with pytest.raises(ValueError):
        rb.rms_norm_i8(x, x[0])
    with pytest.raises(ValueError):
        rb.silu_mul_i8(x, x)
    with pytest.raises(TypeError):
        rb.dequantize_i8(x, s)
    with pytest.raises(ValueError):
        rb.dequantize_i8(q, s)
    with pytest.raises(TypeError):
        rb.gemm_i8(x, s, q, s)
    with pytest.raises(ValueError):
        rb.gemm_i8(q, s, q, s)
    with pytest.raises(ValueError):
        rb.quantize_i8(x[0])


def test_type_codes_match_the_header():
    assert (RIDGE_F16, RIDGE_BF16, RIDGE_F32) == (0, 1, 2)
    assert lib.ridge_gemm_i8.restype is C.c_int
