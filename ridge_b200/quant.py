"""Linear layers with 8-bit operands: quantising rows (plain, behind an RMS norm,
behind a gated activation), the way back, and the int8 GEMM that reads them.

An 8-bit array is a pair (q, scale): q (M, D) int8 in -127..127 and scale (M,)
float32, standing for scale[i] * q[i, j]. Activations are quantised by token and
weights by output channel, both with the rows contiguous, so

    q, s, h = rms_norm_i8(x, gain, residual=h)          # h += x; q ~ gain * h / rms(h)
    y = gemm_i8(q, s, w_q, w_scale)                     # w_q, w_scale = quantize_i8(w)

is a linear layer with w (N, K) behind a norm. The C ABI is in
include/ridge_b200.h; like `gemm`, the calls launch on `stream` (default: torch's
current stream of the tensors' device) and never synchronise. They check what can
be checked on the host and raise TypeError, ValueError or RidgeError before
anything is launched.

Outputs that a call allocates come from the pool of the stream it launches on.
q is allocated with its row pitch rounded up to 16 bytes, which is what gemm_i8
needs; pass `out` to write into an array of your own.
"""

from __future__ import annotations

import math

from ._native import RIDGE_BF16, RIDGE_F16, RIDGE_F32, check, lib

torch = None    # imported by the first call: the package itself does not need it
_TYPES = {}


def _need_torch():
    global torch
    import torch as module
    _TYPES.update({module.float16: RIDGE_F16, module.bfloat16: RIDGE_BF16,
                   module.float32: RIDGE_F32})
    torch = module


def _type_code(dtype, what):
    if torch is None:
        _need_torch()
    code = _TYPES.get(dtype)
    if code is None:
        raise TypeError("%s is float16, bfloat16 or float32, not %s" % (what, dtype))
    return code


def _rows(t, what):
    """(M, D, pitch) of a 2-D CUDA tensor with contiguous rows."""
    shape = t.shape
    if len(shape) != 2:
        raise ValueError("%s is a matrix of rows, got shape %s" % (what, tuple(shape)))
    if not t.is_cuda:
        raise ValueError("%s is not a CUDA tensor" % what)
    M, D = shape
    pitch, step = t.stride()
    if step != 1 and D > 1:
        raise ValueError("%s: rows must be contiguous (inner stride 1)" % what)
    if pitch < D:
        if M > 1:
            raise ValueError("%s: rows overlap (pitch %d, length %d)" % (what, pitch, D))
        pitch = D
    return M, D, pitch


def _like(t, what, device, dtype, shape):
    """Checks a tensor that has to match another in device, type and shape."""
    if t.dtype is dtype and t.shape == shape and t.device == device:
        return
    if t.device != device:
        raise ValueError("%s is on %s, expected %s" % (what, t.device, device))
    if t.dtype != dtype:
        raise TypeError("%s is %s, expected %s" % (what, t.dtype, dtype))
    if t.shape != shape:
        raise ValueError("%s has shape %s, expected %s" % (what, tuple(t.shape), tuple(shape)))


def _like_rows(t, what, device, dtype, shape):
    """The pitch of rows that have to match others in device, type and shape."""
    if t.dtype is not dtype or t.shape != shape or t.device != device:
        _like(t, what, device, dtype, shape)
    pitch, step = t.stride()
    if step == 1 and pitch >= shape[1]:
        return pitch
    return _rows(t, what)[2]


def _vector(t, what, device, dtype, n):
    if t.dtype is not dtype or t.shape != (n,) or t.device != device:
        _like(t, what, device, dtype, (n,))
    if n > 1 and t.stride(0) != 1:
        raise ValueError("%s must be contiguous" % what)


def _run(device, stream, call):
    """call(handle) with the tensors' device current; on a stream other than torch's
    current one, inside that stream's context, so that outputs come from its pool."""
    index = device.index
    if stream is None and torch._C._cuda_getDevice() == index:
        return call(torch._C._cuda_getCurrentRawStream(index))
    with torch.cuda.device(index):
        if stream is None:
            return call(torch._C._cuda_getCurrentRawStream(index))
        handle = stream if isinstance(stream, int) else stream.cuda_stream
        if handle == 0:
            stream = torch.cuda.default_stream(index)
        elif isinstance(stream, int):
            stream = torch.cuda.ExternalStream(stream, device=index)
        with torch.cuda.stream(stream):
            return call(handle)


def _new(shape, strides, dtype, device):
    return torch.empty_strided(shape, strides, dtype=dtype, device=device)


def _given(M, D, device, out, scale):
    """Checks the arrays that a caller passed for (q, scale); q's pitch."""
    pitch = (D + 15) // 16 * 16
    if out is not None:
        pitch = _like_rows(out, "out", device, torch.int8, (M, D))
    if scale is not None:
        _vector(scale, "scale", device, torch.float32, M)
    return pitch


def _outputs(M, D, pitch, device, out, scale):
    """(q, scale): the given arrays or new ones."""
    if out is None:
        out = _new((M, D), (pitch, 1), torch.int8, device)
    if scale is None:
        scale = _new((M,), (1,), torch.float32, device)
    return out, scale


def quantize_i8(x, out=None, scale=None, stream=None):
    """(q, scale) of the rows of x (M, D), float16, bfloat16 or float32:
    scale = max |row| / 127, q = row / scale to the nearest whole number. A row of
    zeros has scale 0; a row with an infinity or NaN has a scale that is not
    finite, and q = 0."""
    code = _type_code(x.dtype, "x")
    M, D, ldx = _rows(x, "x")
    device = x.device
    ldq = _given(M, D, device, out, scale)

    def call(handle):
        q, s = _outputs(M, D, ldq, device, out, scale)
        st = lib.ridge_quantize_i8(x.data_ptr(), code, q.data_ptr(), s.data_ptr(), M, D, ldx, ldq,
                                   handle)
        if st:
            check(st, "ridge_quantize_i8 %dx%d" % (M, D))
        return q, s
    return _run(device, stream, call)


def rms_norm_i8(x, weight, residual=None, eps=1e-6, out=None, scale=None, residual_out=None,
                stream=None):
    """(q, scale, h) of y = weight * h / sqrt(mean(h^2) + eps) with h = x + residual,
    or h = x without one (h is then returned as None).

    x, residual (M, D) and weight (D,) have one type. h is rounded once to that type;
    the norm reads the unrounded sum. residual_out receives h and may be residual
    or x itself; by default it is a new tensor."""
    code = _type_code(x.dtype, "x")
    M, D, ldx = _rows(x, "x")
    device, dtype = x.device, x.dtype
    _vector(weight, "weight", device, dtype, D)
    eps = float(eps)
    if not 0 < eps < math.inf:
        raise ValueError("eps is finite and above 0, got %r" % eps)
    ldr = ldh = D
    if residual is not None:
        ldr = _like_rows(residual, "residual", device, dtype, (M, D))
        if residual_out is not None:
            ldh = _like_rows(residual_out, "residual_out", device, dtype, (M, D))
    elif residual_out is not None:
        raise ValueError("residual_out needs a residual")
    ldq = _given(M, D, device, out, scale)
    # An empty tensor's address is null, which at the C ABI means "not given".
    add = residual is not None and M > 0 and D > 0

    def call(handle):
        q, s = _outputs(M, D, ldq, device, out, scale)
        h = residual_out
        if h is None and residual is not None:
            h = _new((M, D), (D, 1), dtype, device)
        st = lib.ridge_rms_norm_i8(x.data_ptr(), residual.data_ptr() if add else None,
                                   weight.data_ptr(), code, h.data_ptr() if add else None,
                                   q.data_ptr(), s.data_ptr(), M, D, ldx, ldr, ldh, ldq, eps,
                                   handle)
        if st:
            check(st, "ridge_rms_norm_i8 %dx%d" % (M, D))
        return q, s, h
    return _run(device, stream, call)


def silu_mul_i8(gate, up, out=None, scale=None, stream=None):
    """(q, scale) of y = up * gate / (1 + exp(-gate)). gate and up (M, D) have one
    type and may be the two halves of one (M, 2 D) tensor."""
    code = _type_code(gate.dtype, "gate")
    M, D, ldg = _rows(gate, "gate")
    device = gate.device
    ldu = _like_rows(up, "up", device, gate.dtype, (M, D))
    ldq = _given(M, D, device, out, scale)

    def call(handle):
        q, s = _outputs(M, D, ldq, device, out, scale)
        st = lib.ridge_silu_mul_i8(gate.data_ptr(), up.data_ptr(), code, q.data_ptr(),
                                   s.data_ptr(), M, D, ldg, ldu, ldq, handle)
        if st:
            check(st, "ridge_silu_mul_i8 %dx%d" % (M, D))
        return q, s
    return _run(device, stream, call)


def dequantize_i8(q, scale, out=None, dtype=None, stream=None):
    """The values scale[i] * q[i, j], rounded once to dtype (float16 by default,
    or that of `out`)."""
    if torch is None:
        _need_torch()
    if q.dtype != torch.int8:
        raise TypeError("q is int8, got %s" % q.dtype)
    M, D, ldq = _rows(q, "q")
    _vector(scale, "scale", q.device, torch.float32, M)
    if dtype is None:
        dtype = torch.float16 if out is None else out.dtype
    code = _type_code(dtype, "dtype")
    device = q.device
    ldo = D
    if out is not None:
        ldo = _like_rows(out, "out", device, dtype, (M, D))

    def call(handle):
        o = _new((M, D), (D, 1), dtype, device) if out is None else out
        st = lib.ridge_dequantize_i8(q.data_ptr(), scale.data_ptr(), code, o.data_ptr(), M, D,
                                     ldq, ldo, handle)
        if st:
            check(st, "ridge_dequantize_i8 %dx%d" % (M, D))
        return o
    return _run(device, stream, call)


def gemm_i8(a, a_scale, b, b_scale, bias=None, out=None, dtype=None, stream=None):
    """out[i, j] = a_scale[i] * b_scale[j] * sum_k a[i, k] * b[j, k] (+ bias[j]).

    a (M, K) and b (N, K) int8 with float32 scales (M,) and (N,), as the quantising
    calls return them; out (M, N) float16 (default), bfloat16 or float32, bias (N,)
    of that type. The integer sum is exact (K < 131072). a and b start on 16 bytes
    and their row pitches are multiples of 16 (RidgeError otherwise)."""
    if torch is None:
        _need_torch()
    if a.dtype != torch.int8 or b.dtype != torch.int8:
        raise TypeError("ridge_b200.gemm_i8 takes int8 operands")
    M, K, lda = _rows(a, "a")
    N, Kb, ldb = _rows(b, "b")
    if K != Kb:
        raise ValueError("expected a (M, K) and b (N, K), got %s and %s" % (tuple(a.shape),
                                                                         tuple(b.shape)))
    device = a.device
    if b.device != device:
        raise ValueError("b is on %s, expected %s" % (b.device, device))
    _vector(a_scale, "a_scale", device, torch.float32, M)
    _vector(b_scale, "b_scale", device, torch.float32, N)
    if dtype is None:
        dtype = torch.float16 if out is None else out.dtype
    code = _type_code(dtype, "dtype")
    if bias is not None:
        _vector(bias, "bias", device, dtype, N)
    ldc = N
    if out is not None:
        ldc = _like_rows(out, "out", device, dtype, (M, N))

    def call(handle):
        o = _new((M, N), (N, 1), dtype, device) if out is None else out
        st = lib.ridge_gemm_i8(a.data_ptr(), a_scale.data_ptr(), b.data_ptr(), b_scale.data_ptr(),
                               None if bias is None else bias.data_ptr(), code, o.data_ptr(), M, N,
                               K, lda, ldb, ldc, handle)
        if st:
            check(st, "ridge_gemm_i8 %dx%dx%d" % (M, N, K))
        return o
    return _run(device, stream, call)
