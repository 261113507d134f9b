"""GPU parity of the 8-bit operators against their definitions in 64 bits.

Bounds. u = 2^-24 is the relative error of one FP32 rounding; eps/2 that of one
rounding to the output's type (torch.finfo).

quantising: scale is one division away from max|y|, q is the whole number nearest
  to v * inv with inv = 127 / max|v| rounded once, so against the unrounded y / scale
  it is off by half a step plus 127 times the relative errors of v, of max|v| and of
  inv. With e the relative error of v itself (0 for quantize_i8; 2u for the norm, an
  addition and a product; SILU for the activation): step error 0.5 + 127 (2 e + 2 u).
norm: rstd = 1 / sqrt(sumsq / D + eps); a thread adds up to T squares one after the other,
  then at most 10 + 5 levels of pairs, all positive: relative error (T + 15 + 3) u, halved by
  the square root, plus 4 u for its own steps; scale adds 2 e + 2 u.
activation: e^-x within 2 + 1.173 |x| units of 2^-23 (an exponent rounded in FP32, then the
  hardware's ex2), a reciprocal within 2 units, then an addition and two products.
gemm: the integer is exact; FP32 rounds it, its product with sb and the final fused
  multiply-add: 2 u of the product and u of the result, plus one rounding to the type.
"""

import pytest

torch = pytest.importorskip("torch")
pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]

if torch.cuda.is_available():
    import ridge_b200 as rb

U = 2.0 ** -24
TYPES = [torch.float16, torch.bfloat16, torch.float32]
# Rows of one warp, of one CTA at each chunk count, at the edges between them, and longer
# than registers hold; whole 16-byte rows and odd ones; one element.
LENGTHS = [1, 2, 7, 8, 31, 128, 129, 256, 264, 1000, 1024, 1032, 2600, 4096, 4097, 8192, 11008,
           16384, 16385, 16392, 32768, 32776, 40001]


def _rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)


def _check_rows(q, scale, y, e, scale_tol):
    """q, scale against 64-bit rows y whose FP32 form is off by a relative e."""
    torch.cuda.synchronize()
    assert rb.device_error() == 0
    want = y.abs().amax(1) / 127
    s = scale.double()
    assert ((s - want).abs() <= want * scale_tol + 2.0 ** -149).all()
    assert (q[want == 0] == 0).all()
    live = want > 0
    off = (q[live].double() - y[live] / want[live][:, None]).abs().max().item() if live.any() else 0
    assert off <= 0.5 + 127 * (2 * e + 2 * U), off
    assert q.abs().max() <= 127
    if live.any():
        assert (q[live].abs().amax(1) == 127).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("D", LENGTHS)
def test_quantize_lengths(D, dtype):
    for M in (1, 5, 200):
        x = _rand((M, D), dtype, D + M)
        if M > 1:
            x[2] = 0
        q, s = rb.quantize_i8(x)
        assert q.shape == (M, D) and q.stride(0) % 16 == 0
        _check_rows(q, s, x.double(), 0.0, U * 1.01)


def _norm64(x, r, w, eps):
    h = x.double() + (r.double() if r is not None else 0)
    return h, h / torch.sqrt((h * h).mean(1, keepdim=True) + eps) * w.double()


def _norm_tol(D):
    terms = max(32, D // 1024 + 8)
    return ((terms + 18) / 2 + 4 + 6) * U


@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("D", LENGTHS)
def test_norm_lengths(D, dtype, add):
    for M in (1, 4, 190):
        x = _rand((M, D), dtype, D + M)
        r = _rand((M, D), dtype, D + M + 1, 2.0) if add else None
        w = _rand((D,), dtype, D, 0.3) + 1
        if M > 1:
            x[1] = 0
            if add:
                r[1] = 0
        q, s, h = rb.rms_norm_i8(x, w, residual=r, eps=1e-5)
        h64, y = _norm64(x, r, w, 1e-5)
        _check_rows(q, s, y, 2 * U, _norm_tol(D))
        if add:
            half = torch.finfo(dtype).eps / 2
            assert ((h.double() - h64).abs() <= h64.abs() * (half * 1.01 + U) + 2.0 ** -25).all()
        else:
            assert h is None


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("D", LENGTHS)
def test_silu_lengths(D, dtype):
    for M in (1, 6, 180):
        both = _rand((M, 2 * D), dtype, D + M, 2.0)
        gate, up = both[:, :D], both[:, D:]     # the two halves of one product
        q, s = rb.silu_mul_i8(gate, up)
        g = gate.double()
        y = g / (1 + torch.exp(-g)) * up.double()
        e = (2 + 1.173 * g.abs().max().item() + 2) * 2 * U + 3 * U
        _check_rows(q, s, y, e, e + 2 * U)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (1, 16384), (3, 5), (7, 48), (300, 64), (129, 1000),
                                   (64, 16400), (2000, 16)], ids=str)
def test_dequantize(shape, dtype):
    g = torch.Generator("cuda").manual_seed(3)
    q = torch.randint(-128, 128, shape, dtype=torch.int8, device="cuda", generator=g)
    s = torch.rand(shape[0], device="cuda", generator=g)
    out = rb.dequantize_i8(q, s, dtype=dtype)
    want = q.double() * s.double()[:, None]
    tol = want.abs() * (torch.finfo(dtype).eps / 2 * 1.01 + U) + 2.0 ** -25
    assert ((out.double() - want).abs() <= tol).all()


def test_dequantize_gives_back_what_quantize_took():
    x = _rand((50, 777), torch.float32, 1)
    q, s = rb.quantize_i8(x)
    back = rb.dequantize_i8(q, s, dtype=torch.float32)
    assert ((back - x).abs() <= s[:, None] * (0.5 + 1e-4)).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("D", [40, 1000, 1024, 5003, 40000])
def test_rows_that_are_not_finite_poison_themselves_alone(D, dtype):
    x = _rand((6, D), dtype, 5)
    x[1, D // 2] = float("nan")
    x[2, 0] = float("inf")
    x[3, D - 1] = -float("inf")
    x[4, 1], x[4, D - 1] = float("inf"), float("nan")
    w = torch.ones(D, dtype=dtype, device="cuda")
    up = torch.ones_like(x)
    clean = x[[0, 5]].double()
    for name, (q, s) in {"quantize": rb.quantize_i8(x), "norm": rb.rms_norm_i8(x, w)[:2],
                         "silu": rb.silu_mul_i8(x, up)}.items():
        assert not torch.isfinite(s[1:5]).any(), name
        assert (q[1:5] == 0).all(), name
        assert torch.isfinite(s[[0, 5]]).all(), name
    q, s = rb.quantize_i8(x)
    _check_rows(q[[0, 5]], s[[0, 5]], clean, 0.0, U * 1.01)
    out = rb.gemm_i8(*rb.quantize_i8(x), *rb.quantize_i8(up))
    assert torch.isnan(out[1:5]).all() and not torch.isnan(out[[0, 5]]).any()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_extreme_magnitudes(dtype):
    """The largest values, and rows below the threshold under which the reciprocal would
    overflow, are quantised like others. (The scale of a row near the smallest FP32 number is
    itself subnormal, so it is held to an absolute half step of 2^-149 only.)"""
    info = torch.finfo(dtype)
    base = _rand((1, 520), torch.float32, 9).clamp(-3, 3) / 3
    base[0, 17] = 1.0
    tops = [info.max, info.max / 7, 1.0, info.tiny * 500, 2.0 ** -14]
    if dtype != torch.float16:
        tops += [2.0 ** -99, 2.0 ** -101, 2.0 ** -118]
    x = torch.cat([base * t for t in tops]).to(dtype)
    q, s = rb.quantize_i8(x)
    _check_rows(q, s, x.double(), 0.0, U * 1.01)


def test_outputs_of_the_callers_own():
    """Row pitches, starts off the 16-byte grid, and nothing written outside the rows."""
    for dtype in TYPES:
        wide = _rand((9, 400), dtype, 2)
        for first in (0, 1, 8):
            x = wide[:, first:first + 320]
            buf = torch.full((9, 352), 77, dtype=torch.int8, device="cuda")
            q = buf[:, 5 * (first % 2):][:, :320]
            s = torch.empty(11, device="cuda")[1:10]
            got = rb.quantize_i8(x, out=q, scale=s)
            assert got[0] is q and got[1] is s
            _check_rows(q, s, x.double(), 0.0, U * 1.01)
            rest = torch.ones_like(buf, dtype=torch.bool)
            rest[:, 5 * (first % 2):][:, :320] = False
            assert (buf[rest] == 77).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("D", [1, 7, 9, 16, 250, 1001, 2048, 4099, 9000, 16390, 40003])
def test_rows_that_start_anywhere(D, dtype):
    """Every offset of a row's start in 16 bytes, on every operand, each its own; what lies
    around the rows is not written."""
    M = 5
    pitch = D + 11
    for k in range(0, 9):
        def place(t, first):
            buf = torch.full((M * pitch + 64,), 3.0, dtype=t.dtype, device="cuda")
            view = buf[first:].as_strided((M, D), (pitch, 1), first)
            view.copy_(t)
            return buf, view
        x0, r0 = _rand((M, D), dtype, k), _rand((M, D), dtype, k + 50)
        xb, x = place(x0, k)
        rb_, r = place(r0, (3 * k + 1) % 9)
        hb, h = place(torch.zeros_like(x0), (5 * k + 2) % 9)
        wb = torch.full((D + 20,), 3.0, dtype=dtype, device="cuda")
        w = wb[(7 * k) % 9:][:D]
        w.copy_(_rand((D,), dtype, 7, 0.2) + 1)
        q, s, got = rb.rms_norm_i8(x, w, residual=r, residual_out=h)
        h64, y = _norm64(x0, r0, w, 1e-6)
        _check_rows(q, s, y, 2 * U, _norm_tol(D))
        half = torch.finfo(dtype).eps / 2
        assert ((h.double() - h64).abs() <= h64.abs() * (half * 1.01 + U) + 2.0 ** -25).all()
        h.fill_(3.0)
        assert (hb == 3.0).all()
        q, s = rb.quantize_i8(x)
        _check_rows(q, s, x0.double(), 0.0, U * 1.01)
        q, s = rb.silu_mul_i8(x, r)
        g = x0.double()
        e = (2 + 1.173 * g.abs().max().item() + 2) * 2 * U + 3 * U
        _check_rows(q, s, g / (1 + torch.exp(-g)) * r0.double(), e, e + 2 * U)
        ob, o = place(torch.zeros_like(x0), (2 * k + 3) % 9)
        rb.dequantize_i8(q, s, out=o)
        want = q.double() * s.double()[:, None]
        assert ((o.double() - want).abs() <= want.abs() * (half * 1.01 + U) + 2.0 ** -25).all()
        o.fill_(3.0)
        assert (ob == 3.0).all()


@pytest.mark.parametrize("D", [512, 4096, 5001, 16001, 40000, 40007])
@pytest.mark.parametrize("into", ["residual", "x"])
def test_norm_adds_in_place(D, into):
    x, r = _rand((33, D), torch.bfloat16, 1), _rand((33, D), torch.bfloat16, 2)
    if D % 8:
        x = _rand((33, D + 3), torch.bfloat16, 1)[:, 1:D + 1].clone(
            memory_format=torch.preserve_format)
    w = _rand((D,), torch.bfloat16, 3)
    q, s, h = rb.rms_norm_i8(x, w, residual=r)
    x2, r2 = x.clone(), r.clone()
    target = r2 if into == "residual" else x2
    q2, s2, h2 = rb.rms_norm_i8(x2, w, residual=r2, residual_out=target)
    assert h2 is target
    assert torch.equal(q, q2) and torch.equal(s, s2) and torch.equal(h, target)
    assert torch.equal(x2 if into == "residual" else r2, x if into == "residual" else r)


# ------------------------------------------------------------------ the product

def _operands(M, N, K, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    pitch = (K + 15) // 16 * 16

    def side(rows):
        # what lies behind a row's end is not part of it
        q = torch.randint(-128, 128, (rows, max(pitch, 16)), dtype=torch.int8, device="cuda",
                          generator=g)[:, :K]
        return q, torch.rand(rows, device="cuda", generator=g) * 0.01 + 1e-4
    return (*side(M), *side(N))


def _check_gemm(out, a, sa, b, sb, bias):
    torch.cuda.synchronize()
    assert rb.device_error() == 0
    product = (a.double() @ b.double().T) * sa.double()[:, None] * sb.double()
    want = product + (bias.double() if bias is not None else 0)
    half = torch.finfo(out.dtype).eps / 2
    tol = 2.1 * U * product.abs() + (half + 2 * U) * want.abs() + 2.0 ** -25
    off = (out.double() - want).abs() - tol
    assert (off <= 0).all(), "worst excess %.3g at %s" % (
        off.max().item(), divmod(off.argmax().item(), out.shape[1]))


# One token to many; around every token tile, channel tile and K block; below one of each.
SHAPES = [(1, 1, 1), (1, 16, 16), (1, 9000, 8191), (2, 4095, 2049), (3, 129, 4100), (4, 4096, 2047),
          (2, 33, 8), (4, 7, 40000), (1, 128, 128), (1, 8192, 1024), (2, 130, 96), (7, 1000, 129),
          (15, 127, 31), (16, 256, 4096), (17, 300, 640), (33, 4096, 512), (64, 129, 1000),
          (100, 640, 2048), (128, 8192, 256), (129, 1003, 385), (255, 257, 130), (256, 512, 1024),
          (257, 256, 128), (300, 1000, 2600), (517, 1003, 260), (512, 512, 4096),
          (1000, 4100, 192), (2049, 513, 384), (4096, 1024, 64), (700, 16, 1000),
          (3000, 1, 17), (513, 70, 16384)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%dx%d" % s)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_gemm_shapes(shape, dtype):
    M, N, K = shape
    a, sa, b, sb = _operands(M, N, K)
    bias = _rand((N,), dtype, 4) if (M + N) % 2 else None
    out = rb.gemm_i8(a, sa, b, sb, bias=bias, dtype=dtype)
    _check_gemm(out, a, sa, b, sb, bias)
    again = rb.gemm_i8(a, sa, b, sb, bias=bias, dtype=dtype)
    assert torch.equal(out.view(torch.uint8), again.view(torch.uint8))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(3840, 1280, 256), (3840, 1270, 2100), (2304, 2400, 700),
                                   (19000, 300, 96), (5000, 5000, 128)],
                         ids=lambda s: "%dx%dx%d" % s)
def test_gemm_more_tiles_than_pairs(shape, dtype):
    """Several rounds of tiles, the last of them few (75 or 90 tiles of 256 x 256) or many."""
    a, sa, b, sb = _operands(*shape, seed=8)
    bias = _rand((shape[1],), dtype, 9)
    _check_gemm(rb.gemm_i8(a, sa, b, sb, bias=bias, dtype=dtype), a, sa, b, sb, bias)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("N,K", [(4096, 4096), (1003, 1000), (5000, 333), (16, 16384), (3, 15)])
def test_gemm_rows_do_not_depend_on_the_batch(N, K, dtype):
    """A token's row is the same bits whichever kernel and tile the batch around it takes."""
    a, sa, b, sb = _operands(700, N, K, 11)
    bias = _rand((N,), dtype, 12)
    whole = rb.gemm_i8(a, sa, b, sb, bias=bias, dtype=dtype)
    for M in (1, 2, 3, 4, 5, 64, 130, 256, 257):
        part = rb.gemm_i8(a[:M], sa[:M], b, sb, bias=bias, dtype=dtype)
        assert torch.equal(part, whole[:M]), M


@pytest.mark.parametrize("M", [3, 200, 600])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_gemm_output_pitch_and_alignment(M, dtype):
    """Rows of C that start anywhere; nothing outside C is written."""
    N, K = 333, 272
    a, sa, b, sb = _operands(M, N, K, 1)
    bias = _rand((N + 1,), dtype, 6)[1:]
    for first, pitch in [(0, 336), (1, 336), (3, 337), (8, 400)]:
        buf = torch.full((M + 2, pitch + 16), 7.0, dtype=dtype, device="cuda")
        flat = buf.view(-1)[first:]
        out = flat.as_strided((M, N), (pitch, 1), flat.storage_offset() + pitch)
        rb.gemm_i8(a, sa, b, sb, bias=bias, out=out)
        _check_gemm(out, a, sa, b, sb, bias)
        out.fill_(7.0)
        assert (buf == 7.0).all()


@pytest.mark.parametrize("M", [1, 20, 256, 1000])
def test_gemm_without_k_is_the_bias(M):
    a = torch.empty((M, 0), dtype=torch.int8, device="cuda")
    b = torch.empty((70, 0), dtype=torch.int8, device="cuda")
    sa, sb = torch.ones(M, device="cuda"), torch.ones(70, device="cuda")
    bias = _rand((70,), torch.float16, 1)
    assert torch.equal(rb.gemm_i8(a, sa, b, sb, bias=bias), bias.expand(M, 70))
    assert (rb.gemm_i8(a, sa, b, sb) == 0).all()


def test_empty_arrays():
    e8 = torch.empty((0, 32), dtype=torch.int8, device="cuda")
    b = torch.ones((5, 32), dtype=torch.int8, device="cuda")
    none, five = torch.empty(0, device="cuda"), torch.ones(5, device="cuda")
    assert rb.gemm_i8(e8, none, b, five).shape == (0, 5)
    assert rb.gemm_i8(b, five, e8, none).shape == (5, 0)
    x = torch.empty((0, 64), dtype=torch.float16, device="cuda")
    w = torch.ones(64, dtype=torch.float16, device="cuda")
    q, s, h = rb.rms_norm_i8(x, w, residual=x.clone())
    assert q.shape == (0, 64) and s.shape == (0,) and h.shape == (0, 64)
    x = torch.empty((4, 0), dtype=torch.float16, device="cuda")
    s = torch.full((4,), 9.0, device="cuda")
    rb.quantize_i8(x, scale=s)
    assert (s == 0).all()
    assert rb.dequantize_i8(torch.empty((4, 0), dtype=torch.int8, device="cuda"), s).shape == (4, 0)


@pytest.mark.parametrize("M", [1, 130, 300])
def test_gemm_longest_sum(M):
    """K = 2^17 - 1 of the largest products: the sum ends just below 2^31."""
    K = (1 << 17) - 1
    a = torch.full((M, K + 1), -128, dtype=torch.int8, device="cuda")[:, :K]
    b = torch.full((130, K + 1), -128, dtype=torch.int8, device="cuda")[:, :K]
    out = rb.gemm_i8(a, torch.ones(M, device="cuda"), b, torch.ones(130, device="cuda"),
                     dtype=torch.float32)
    assert (out == torch.tensor(K * 16384, dtype=torch.float64).float().cuda()).all()


def test_offsets_past_32_bits():
    """Rows of C, and of a quantised input, more than 2^31 elements from their start."""
    M, N, K, pitch = 66000, 40, 32, 33000
    assert (M - 1) * pitch > 2 ** 31
    a, sa, b, sb = _operands(M, N, K, 2)
    buf = torch.zeros(M * pitch, dtype=torch.float16, device="cuda")
    out = buf.as_strided((M, N), (pitch, 1))
    rb.gemm_i8(a, sa, b, sb, out=out)
    _check_gemm(out, a, sa, b, sb, None)
    few = torch.empty((3, 16), dtype=torch.int8, device="cuda")
    far = buf.as_strided((3, 16), (M // 3 * pitch, 1), pitch * (M // 3) - 16)
    far.copy_(_rand((3, 16), torch.float16, 3))
    q, s = rb.quantize_i8(far, out=few)
    _check_rows(q, s, far.double(), 0.0, U * 1.01)


def test_other_streams_and_graphs():
    """A call on a stream of its own, and captured calls replayed on new data."""
    M, N, K = 24, 520, 384
    x, w = _rand((M, K), torch.bfloat16, 1), _rand((N, K), torch.bfloat16, 2)
    gain, res = torch.ones(K, dtype=torch.bfloat16, device="cuda"), _rand((M, K), torch.bfloat16, 3)
    wq, ws = rb.quantize_i8(w)

    def layer():
        q, s, h = rb.rms_norm_i8(x, gain, residual=res)
        return rb.gemm_i8(q, s, wq, ws, dtype=torch.bfloat16), h
    want = [t.clone() for t in layer()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    q, s, h = rb.rms_norm_i8(x, gain, residual=res, stream=side)
    y = rb.gemm_i8(q, s, wq, ws, dtype=torch.bfloat16, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(y, want[0]) and torch.equal(h, want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, h = layer()
    for seed in (1, 9):
        x.copy_(_rand((M, K), torch.bfloat16, seed))
        graph.replay()
        torch.cuda.synchronize()
        if seed == 1:
            assert torch.equal(y, want[0]) and torch.equal(h, want[1])
        now = [t.clone() for t in (y, h)]
        assert all(torch.equal(p, q) for p, q in zip(now, layer()))


def test_two_products_at_once():
    """Launches on two streams share nothing."""
    cases = [_operands(40, 3000, 2048, 5), _operands(700, 900, 1024, 6)]
    want = [rb.gemm_i8(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            got[i].append(rb.gemm_i8(*cases[i], stream=st))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_beside_the_fp16_family():
    """Products of both families on two streams: they share SMs and Tensor Memory."""
    c = _operands(20, 4096, 2048, 7)
    want = rb.gemm_i8(*c)
    a, b = _rand((700, 1024), torch.float16, 1), _rand((900, 1024), torch.float16, 2)
    pair = rb.TileConfig(256, 256, 32, 2, 4, 8, 2)
    want16 = rb.gemm(a, b, config=pair)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got, got16 = [], []
    for _ in range(8):
        got.append(rb.gemm_i8(*c, stream=streams[0]))
        with torch.cuda.stream(streams[1]):
            got16.append(rb.gemm(a, b, config=pair))
    torch.cuda.synchronize()
    assert rb.device_error() == 0
    assert all(torch.equal(g, want) for g in got)
    assert all(torch.equal(g, want16) for g in got16)


def test_the_same_tensor_twice():
    """One tensor as both inputs of the addition, and as both operands of a product."""
    x = _rand((12, 640), torch.bfloat16, 3)
    w = torch.ones(640, dtype=torch.bfloat16, device="cuda")
    q, s, h = rb.rms_norm_i8(x, w, residual=x.clone())
    q2, s2, _ = rb.rms_norm_i8(x, w, residual=x, residual_out=x)
    assert torch.equal(q, q2) and torch.equal(s, s2) and torch.equal(h, x)
    _check_gemm(rb.gemm_i8(q, s, q, s, dtype=torch.float32), q, s, q, s, None)


@pytest.mark.parametrize("M", [1, 9, 300])
def test_mlp_block(M):
    """The operators as a gated MLP runs them, against the same block in 64 bits with the
    same 8-bit rounding of its operands."""
    D, F = 512, 1408
    dt = torch.bfloat16
    x, res = _rand((M, D), dt, 1), _rand((M, D), dt, 2)
    gain = _rand((D,), dt, 3, 0.1) + 1
    w1, w2 = _rand((2 * F, D), dt, 4, D ** -0.5), _rand((D, F), dt, 5, F ** -0.5)
    w1q, w1s = rb.quantize_i8(w1)
    w2q, w2s = rb.quantize_i8(w2)
    q, s, h = rb.rms_norm_i8(x, gain, residual=res)
    both = rb.gemm_i8(q, s, w1q, w1s, dtype=torch.float32)
    q2, s2 = rb.silu_mul_i8(both[:, :F], both[:, F:])
    y = rb.gemm_i8(q2, s2, w2q, w2s, dtype=dt)
    assert rb.device_error() == 0

    def grid(t):
        s = t.abs().amax(1, keepdim=True) / 127
        return torch.round(t / s) * s
    _, n = _norm64(x, res, gain, 1e-6)
    b64 = grid(n) @ grid(w1.double()).T
    g64, u64 = b64[:, :F], b64[:, F:]
    act = g64 * torch.sigmoid(g64) * u64
    want = grid(act) @ grid(w2.double()).T
    # Elements at a rounding border may fall a step to the other side: in the first operand of
    # either product with probability about 127 * 2^-20 each, which moves an output by less than
    # one step of one operand element; bf16 rounds the rest.
    step = act.abs().amax(1, keepdim=True) / 127 * w2.double().abs().max()
    assert ((y.double() - want).abs() <= want.abs() * 2.0 ** -8 + 6 * step).all()
    # Without the 8-bit grids the block differs by their noise: 2 operands of about
    # 1/sqrt(12) step of max/127 each, a few per cent of the output's size.
    f64 = _norm64(x, res, gain, 1e-6)[1] @ w1.double().T
    free = f64[:, :F] * torch.sigmoid(f64[:, :F]) * f64[:, F:] @ w2.double().T
    assert (y.double() - free).norm() <= 0.06 * free.norm()
