"""The 8-bit integer operators (include/hcrag.h hcr_*_rows_device / hcr_int8_linear_device, bound
by hcrag_amd.int8) against their definitions in 64 bits.

Tolerances are bounds, from u = 2^-24 (half a step of fp32) and h = half a step of the output type:
  linear   float(acc), * sx, and the final fma round once each: 2.01 u |acc sx sw| + u |y| + h |y|
  quantise without an activation: q and scale are single IEEE fp32 operations, so bits are equal
  gelu     Phi from a fitted logistic form (within 3.6e-8) plus the rcp / exp2 approximations and
           four roundings, derived in test_int8_rows_gpu.py: |dv| <= 1.6e-7 |x| + 4 u |v|
  norm     _norm_bound below
  q of any v with error dv: |q - 127 v / a| <= 1/2 + 127 (dv + da) / a + 127 * 4 u, a = max |v|
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

gpu = pytest.mark.gpu
U = 2.0 ** -24
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: U}
LEAST = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}   # half a subnormal step
D = torch.float64


def _ops():
    import hcrag_amd
    return hcrag_amd


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _int8(g, rows, cols, stride=None, lo=-127, hi=127):
    """int8 rows whose padding holds other values."""
    stride = stride or (cols + 15) // 16 * 16
    return torch.randint(lo, hi + 1, (rows, stride), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)[:, :cols]


def _scales(g, n):
    return (0.5 + torch.rand(n, generator=g, device="cuda")) * 2.0 ** -6


def _linear_check(y, x, sx, w, sw, bias):
    p = (x.to(D) @ w.to(D).T) * sx.to(D)[:, None] * sw.to(D)
    ref = p if bias is None else p + bias.to(D)
    h = HALF[y.dtype]
    tol = 2.01 * U * p.abs() + (U + h) * 1.001 * ref.abs() + LEAST[y.dtype]
    over = (y.to(D) - ref).abs() - tol
    assert bool((over <= 0).all()), float(over.max())


# ---- linear -------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("K", [1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 192, 255, 257, 384, 640, 999, 1024, 2049, 4096])
@pytest.mark.parametrize("T,N", [(1, 1), (1, 257), (5, 33), (16, 64), (17, 130)])
def test_linear_depths(T, N, K):
    m, g = _ops(), _gen(K * 1000 + T)
    x, w, sx, sw = _int8(g, T, K), _int8(g, N, K), _scales(g, T), _scales(g, N)
    bias = torch.randn(N, generator=g, device="cuda")
    y = m.int8_linear(m.Int8Rows(x, sx), m.Int8Rows(w, sw), bias=bias, dtype=torch.float32)
    _linear_check(y, x, sx, w, sw, bias)


@gpu
@pytest.mark.parametrize("out", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("T", [1, 2, 3, 15, 31, 32, 33, 47, 48, 49, 63, 64, 65, 95, 127, 128, 129, 191, 255, 256, 257, 511, 513, 1000, 2049, 5000])
def test_linear_tokens(T, out):
    m, g = _ops(), _gen(T)
    for N, K in ((1, 64), (3, 100), (66, 33), (127, 256), (384, 384), (769, 200), (1030, 768)):
        x, w, sx, sw = _int8(g, T, K), _int8(g, N, K), _scales(g, T), _scales(g, N)
        y = m.int8_linear(m.Int8Rows(x, sx), m.Int8Rows(w, sw), dtype=DT[out])
        _linear_check(y, x, sx, w, sw, None)


@gpu
@pytest.mark.parametrize("T,N", [(1, 5), (40, 40), (300, 300), (1500, 1300)])
def test_linear_extreme_sums(T, N):
    """Every product 2^14 at the largest depth: sums just below 2^31."""
    m, K = _ops(), 131071
    x = torch.full((T, K + 1), -128, dtype=torch.int8, device="cuda")[:, :K]
    w = torch.full((N, K + 1), -128, dtype=torch.int8, device="cuda")[:, :K]
    one_t, one_n = torch.ones(T, device="cuda"), torch.ones(N, device="cuda")
    y = m.int8_linear(m.Int8Rows(x, one_t), m.Int8Rows(w, one_n), dtype=torch.float32)
    assert bool((y == float(np.float32(2 ** 14 * K))).all())
    x.fill_(127)
    y = m.int8_linear(m.Int8Rows(x, one_t), m.Int8Rows(w, one_n), dtype=torch.float32)
    assert bool((y == float(np.float32(-127 * 128 * K))).all())


@gpu
@pytest.mark.parametrize("out", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("T,N,K", [(1, 70, 100), (37, 61, 130), (260, 259, 300), (1027, 515, 400), (4099, 777, 384)])
def test_linear_strides_and_what_lies_around(T, N, K, out):
    """Wide strides of every operand, an output that starts off alignment; nothing outside the
    output's columns and rows is written."""
    m, g = _ops(), _gen(7)
    x, w = _int8(g, T, K, 1024), _int8(g, N, K, 2048)
    sx, sw = _scales(g, T + 1)[1:], _scales(g, N + 1)[1:]
    bias = torch.randn(N + 1, generator=g, device="cuda")[1:]
    for first in (0, 1, 4, 8):
        buf = torch.full((T + 3, N + 19), 7.0, dtype=DT[out], device="cuda")
        m.int8_linear(m.Int8Rows(x, sx), m.Int8Rows(w, sw), bias=bias, out=buf[1:T + 1, first:first + N])
        _linear_check(buf[1:T + 1, first:first + N], x, sx, w, sw, bias)
        buf[1:T + 1, first:first + N] = 7.0
        assert bool((buf == 7.0).all())


@gpu
@pytest.mark.parametrize("T", [3, 100, 1000, 9000, 66000])
def test_linear_f16_subnormal_results(T):
    """Results below f16's normal range keep its subnormal steps (bound: half of one)."""
    m, g = _ops(), _gen(T)
    for N, K in ((257, 96), (1024, 1024)):
        x, w = _int8(g, T, K), _int8(g, N, K)
        sx, sw = _scales(g, T) * 2.0 ** -10, _scales(g, N) * 2.0 ** -14
        y = m.int8_linear(m.Int8Rows(x, sx), m.Int8Rows(w, sw), dtype=torch.float16)
        assert bool((y[:, :64].abs() < 6e-5).any()) and bool((y != 0).any())
        _linear_check(y, x, sx, w, sw, None)


@gpu
@pytest.mark.parametrize("out", ["f16", "bf16", "f32"])
def test_linear_rows_do_not_depend_on_the_batch(out):
    """The same row through every kernel and chunk: the same bits."""
    m, g = _ops(), _gen(17)
    for N, K in ((384, 384), (1155, 1100), (4096, 1024)):
        T = 20000
        x, w, sx, sw = _int8(g, T, K), _int8(g, N, K), _scales(g, T), _scales(g, N)
        bias = torch.randn(N, generator=g, device="cuda")
        W = m.Int8Rows(w, sw)
        y = m.int8_linear(m.Int8Rows(x, sx), W, bias=bias, dtype=DT[out])
        for n in (1, 16, 40, 200, 700, 3000, 9000):
            assert torch.equal(m.int8_linear(m.Int8Rows(x[:n], sx[:n]), W, bias=bias, dtype=DT[out]), y[:n])


@gpu
def test_linear_offsets_past_32_bits():
    m, g = _ops(), _gen(3)
    T, N, K = (1 << 17) + 3, 16400, 17
    x, w, sx, sw = _int8(g, T, K), _int8(g, N, K), _scales(g, T), _scales(g, N)
    y = m.int8_linear(m.Int8Rows(x, sx), m.Int8Rows(w, sw), dtype=torch.float16)
    assert y.numel() > 2 ** 31
    _linear_check(y[-300:], x[-300:], sx[-300:], w, sw, None)
    _linear_check(y[:300], x[:300], sx[:300], w, sw, None)


@gpu
def test_linear_more_features_than_one_launch():
    """Features are cut like tokens: 2^22 of them a launch."""
    m, g = _ops(), _gen(9)
    T, N, K = 3, 2 ** 22 + 301, 16
    x, w = _int8(g, T, K), _int8(g, N, K)
    sx, sw, b = _scales(g, T), _scales(g, N), torch.randn(N, generator=g, device="cuda")
    y = m.int8_linear(m.Int8Rows(x, sx), m.Int8Rows(w, sw), bias=b, dtype=torch.float32)
    _linear_check(y, x, sx, w, sw, b)


@gpu
def test_linear_far_rows():
    """Rows 8 MiB apart, whose tiles 31-bit offsets do not reach, and more outputs than one launch."""
    m, g = _ops(), _gen(10)
    T, N, K, ld = 700, 2 ** 22 - 5, 16, 2 ** 23 + 16
    xs = torch.empty(T * ld, device="cuda", dtype=torch.int8)
    x = xs.as_strided((T, K), (ld, 1))
    x.copy_(_int8(g, T, K))
    w = _int8(g, N, K)
    sx, sw = _scales(g, T), _scales(g, N)
    y = m.int8_linear(m.Int8Rows(x, sx), m.Int8Rows(w, sw))
    for f in (slice(0, 200), slice(N // 2, N // 2 + 200), slice(N - 200, N)):
        _linear_check(y[:, f], x, sx, w[f], sw[f], None)


@gpu
@pytest.mark.parametrize("T", [1, 40, 700, 3000])
def test_linear_nan_scales_stay_in_their_row(T):
    m, g = _ops(), _gen(11)
    N, K = 200, 320
    x, w, sx, sw = _int8(g, T, K), _int8(g, N, K), _scales(g, T), _scales(g, N)
    sx[T // 2] = float("nan")
    x[T // 2] = 0
    y = m.int8_linear(m.Int8Rows(x, sx), m.Int8Rows(w, sw), dtype=torch.float16)
    assert bool(y[T // 2].isnan().all())
    keep = [t for t in range(T) if t != T // 2]
    _linear_check(y[keep], x[keep], sx[keep], w, sw, None)


@gpu
def test_empty_calls():
    m = _ops()
    x0 = m.quantize_rows(torch.empty(0, 40, dtype=torch.float16, device="cuda"))
    assert x0.shape == (0, 40) and x0.dequantize().shape == (0, 40)
    w = m.quantize_rows(torch.randn(8, 40, device="cuda"))
    assert m.int8_linear(x0, w).shape == (0, 8)
    assert m.int8_linear(w, x0).shape == (8, 0)
    n = m.norm_quantize(torch.empty(0, 40, device="cuda"), torch.ones(40, device="cuda"))
    assert n.shape == (0, 40)


# ---- quantise -----------------------------------------------------------------------------
COLS = [1, 3, 7, 8, 9, 17, 64, 255, 384, 511, 512, 513, 768, 1000, 1023, 1024, 1025, 2047, 2048, 2049, 2999, 4095, 4096,
        4097, 6143, 6145, 8191, 8192, 8193, 16384, 20001, 32767, 32768]


def _quant_definition(v32):
    """q and scale of fp32 rows, in single IEEE fp32 operations (numpy).  A row that is not finite:
    q 0 and scale NaN."""
    v = v32.float().cpu().numpy()
    bad = ~np.isfinite(v).all(1)
    if bad.any():
        q, s = _quant_definition(torch.from_numpy(np.where(bad[:, None], np.float32(0), v)))
        return q, np.where(bad, np.float32("nan"), s)
    a = np.abs(v).max(1)
    zero = a < np.float32(2.0 ** -100)
    inv = np.where(zero, np.float32(0), np.float32(127) / np.where(zero, np.float32(1), a))
    return (np.rint(v * inv[:, None]).astype(np.int8), np.where(zero, np.float32(0), a / np.float32(127)))


@gpu
@pytest.mark.parametrize("xt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("cols", COLS)
def test_quantize_bits(cols, xt):
    m, g = _ops(), _gen(cols)
    for rows in (1, 2, 5, 33):
        x = (torch.randn(rows, cols, generator=g, device="cuda") * 3).to(DT[xt])
        r = m.quantize_rows(x)
        q, s = _quant_definition(x)
        assert np.array_equal(r.q.cpu().numpy(), q)
        assert np.array_equal(r.scale.cpu().numpy(), s)
        for o in DT.values():
            want = (torch.from_numpy(q.astype(np.float32)) * torch.from_numpy(s)[:, None]).to(o)
            assert torch.equal(r.dequantize(o).cpu(), want)


@gpu
@pytest.mark.parametrize("cols", [5, 200, 700, 1500, 3000, 5000, 9000])
def test_quantize_edges(cols):
    """Rows of zeros, of one value, below and at the least magnitude, at the type's ends; NaN and
    infinities make their own row NaN and no other."""
    m, g = _ops(), _gen(cols)
    x = torch.randn(16, cols, generator=g, device="cuda")
    x[0] = 0.0
    x[1] = -2.5
    x[2] = 2.0 ** -101
    x[3] = 0.0
    x[3, cols // 2] = -(2.0 ** -100)
    x[4] *= 3e38 / x[4].abs().max()
    x[5] = -0.0
    x[6] = 1e-44                                  # subnormal
    x[7] = torch.arange(cols, device="cuda") % 255 - 127.0
    x[7, 0] = 127.0                               # a whole number of steps, ends included
    x[8] = (torch.arange(cols, device="cuda") % 253 - 126.0) + 0.5
    x[8, 0] = 127.0                               # every element half way between two steps
    x[9, 0] = float("nan")
    x[10, cols - 1] = float("inf")
    x[11, cols // 2] = -float("inf")
    x[12] = float("nan")
    x[13, cols - 1] = float("nan")
    x[14] = float("inf")
    r = m.quantize_rows(x)
    q, s = _quant_definition(x)     # (row 4's factor is past fp32 at some widths: the row is then infinite)
    assert np.array_equal(r.q.cpu().numpy(), q)
    assert np.array_equal(r.scale.cpu().numpy(), s, equal_nan=True)
    assert bool(r.scale[9:15].isnan().all()) and bool((r.q[9:15] == 0).all())
    assert bool(r.dequantize()[9:15].isnan().all())


@gpu
@pytest.mark.parametrize("xt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("cols", [7, 384, 1000, 4096, 10000])
def test_quantize_strided(cols, xt):
    """Rows of a wider buffer, aligned and not; the output's padding and neighbours stay."""
    m, g = _ops(), _gen(cols)
    for first in (0, 1, 8):
        x = torch.randn(9, cols + 24, generator=g, device="cuda").to(DT[xt])[:, first:first + cols]
        ldq = (cols + 15) // 16 * 16 + 32
        buf = torch.full((11, ldq), 77, dtype=torch.int8, device="cuda")
        sc = torch.full((11,), 5.0, device="cuda")
        m.quantize_rows(x, out=m.Int8Rows(buf[1:10, :cols], sc[1:10]))
        q, s = _quant_definition(x)
        assert np.array_equal(buf[1:10, :cols].cpu().numpy(), q)
        assert np.array_equal(sc[1:10].cpu().numpy(), s)
        buf[1:10, :cols] = 77
        assert bool((buf == 77).all()) and sc[0] == 5.0 and sc[10] == 5.0


def _rows_check(r, v, dv):
    """int8 rows of v [rows, cols] (64 bits) that the kernel computed within dv."""
    a = v.abs().amax(1, keepdim=True)
    da = dv.amax(1, keepdim=True)
    q = r.q.to(D)
    over = (q - 127 * v / a).abs() - (0.5 + 127 * (dv + da) / a + 127 * 4 * U)
    assert bool((over <= 0).all()), float(over.max())
    over = (r.scale.to(D)[:, None] - a / 127).abs() - (da / 127 + 2 * U * a / 127)
    assert bool((over <= 0).all()), float(over.max())


@gpu
@pytest.mark.parametrize("xt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("cols", [1, 9, 384, 1536, 2049, 2999, 4096, 4097, 6143, 6145, 8200])
def test_quantize_gelu(cols, xt):
    m, g = _ops(), _gen(cols)
    x = (torch.randn(21, cols, generator=g, device="cuda") * 4).to(DT[xt])
    x[:, 0] = 2.0                      # (an all-negative row would be all cancellation: still bounded, but
    r = m.quantize_rows(x, act="gelu") # a = max |v| would be tiny)
    v = x.to(D) * torch.special.ndtr(x.to(D))
    _rows_check(r, v, 1.6e-7 * x.to(D).abs() + 4 * U * v.abs())


@gpu
def test_quantize_more_rows_than_one_launch():
    """A wave per row: 2^26 rows are 2^32 threads, which no grid holds."""
    m = _ops()
    rows = 2 ** 26 + 77
    x = (torch.arange(rows, device="cuda", dtype=torch.int32) % 4001 - 2000).to(torch.float16)[:, None]
    r = m.quantize_rows(x)
    a = x[:, 0].float()
    assert torch.equal(r.q[:, 0].to(torch.int32), torch.sign(a).to(torch.int32) * 127)
    assert torch.equal(r.scale, (a.to(D).abs() / 127).float())   # (no quotient is near a tie: 127 is odd)
    v = r.dequantize(torch.float32)
    assert torch.equal(v[:, 0], r.q[:, 0].float() * r.scale)


@gpu
def test_quantize_offsets_past_32_bits():
    m = _ops()
    rows, cols = 70001, 32768
    x = torch.zeros(rows, cols, dtype=torch.float16, device="cuda")
    g = _gen(2)
    x[-40:] = torch.randn(40, cols, generator=g, device="cuda").to(torch.float16)
    r = m.quantize_rows(x)
    assert r.q.numel() > 2 ** 31
    q, s = _quant_definition(x[-40:])
    assert np.array_equal(r.q[-40:].cpu().numpy(), q) and np.array_equal(r.scale[-40:].cpu().numpy(), s)
    assert bool((r.scale[:-40] == 0).all())
    y = r.dequantize(torch.float16)
    want = (torch.from_numpy(q.astype(np.float32)) * torch.from_numpy(s)[:, None]).to(torch.float16)
    assert torch.equal(y[-40:].cpu(), want)


# ---- norm ---------------------------------------------------------------------------------
def _norm_reference(x, r, weight, bias, norm, eps):
    """(h, v, dv) in 64 bits.  dv bounds the fp32 kernel: h rounds once (u |h|); a sum of a row is
    at most 60 additions deep (32 in a thread, 6 over a wave, 16 over waves), so the mean is within
    61 u mean|h| of its value and the centred element within e = 3 u |h| + 62 u mean|h|; the second
    moment then within 62 u + 2 rms(e) / sd relative, of which rsqrt takes half and adds 4 u; three
    roundings remain."""
    h = x.to(D) if r is None else x.to(D) + r.to(D)
    mean = h.mean(1, keepdim=True) if norm == "layer" else torch.zeros_like(h[:, :1])
    d = h - mean
    sd = (d * d).mean(1, keepdim=True).add(eps).sqrt()
    n = d / sd * weight.to(D)
    v = n if bias is None else n + bias.to(D)
    e = 3 * U * h.abs()
    if norm == "layer":
        e = e + 62 * U * h.abs().mean(1, keepdim=True)
    rel = 31 * U + (e * e).mean(1, keepdim=True).sqrt() / sd + 4 * U
    dv = e / sd * weight.to(D).abs() + n.abs() * (rel + 3 * U) + U * v.abs()
    return h, v, 1.01 * dv


def _norm_check(m, x, r, weight, bias, norm, eps, yt, with_sum):
    sum_out = torch.empty_like(r) if with_sum else None
    y = torch.empty(x.shape, dtype=yt, device="cuda") if yt is not None else None
    out = m.norm_quantize(x, weight, bias=bias, residual=r, norm=norm, eps=eps, sum_out=sum_out, norm_out=y)
    h, v, dv = _norm_reference(x, r, weight, bias, norm, eps)
    _rows_check(out, v, dv)
    if with_sum:
        assert torch.equal(sum_out, (x.float() + r.float()).to(r.dtype))
    if y is not None:
        over = (y.to(D) - v).abs() - (dv + HALF[yt] * (v.abs() + dv) + LEAST[yt])
        assert bool((over <= 0).all()), float(over.max())


@gpu
@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("cols", [2, *COLS[1:]])
def test_norm_widths(cols, norm):
    m, g = _ops(), _gen(cols)
    weight = 1 + 0.2 * torch.randn(cols, generator=g, device="cuda")
    bias = 0.3 * torch.randn(cols, generator=g, device="cuda")
    for rows in (1, 3, 6):
        x = torch.randn(rows, cols, generator=g, device="cuda").to(torch.float16)
        r = torch.randn(rows, cols, generator=g, device="cuda") * 2 + 0.5
        _norm_check(m, x, r, weight, bias, norm, 1e-6, torch.float32, True)


@gpu
@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("rt", [None, "f16", "bf16", "f32"])
@pytest.mark.parametrize("xt", ["f16", "bf16", "f32"])
def test_norm_types(xt, rt, norm):
    m, g = _ops(), _gen(5)
    for rows, cols in ((7, 77), (5, 384), (3, 1024), (2, 3000)):
        weight = 1 + 0.2 * torch.randn(cols, generator=g, device="cuda")
        bias = 0.3 * torch.randn(cols, generator=g, device="cuda")
        x = (torch.randn(rows, cols, generator=g, device="cuda") * 5).to(DT[xt])
        r = None if rt is None else torch.randn(rows, cols, generator=g, device="cuda").to(DT[rt])
        for yt in (None, torch.float16, torch.bfloat16, torch.float32):
            for b in (None, bias):
                _norm_check(m, x, r, weight, b, norm, 1e-5, yt, rt is not None)


@gpu
@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("cols", [40, 768, 1001, 2500, 5000, 7000])
def test_norm_in_place_and_strided(cols, norm):
    """sum_out over the residual, norm_out over the residual or x; rows of wider buffers, aligned
    and not; what lies around the outputs stays."""
    m, g = _ops(), _gen(cols)
    weight = 1 + 0.2 * torch.randn(cols + 1, generator=g, device="cuda")
    for first in (0, 1, 16):
        w = weight[first & 1:][:cols]
        xb = torch.randn(9, cols + 40, generator=g, device="cuda").to(torch.bfloat16)
        rb = torch.randn(9, cols + 40, generator=g, device="cuda")
        x, r = xb[1:8, first:first + cols], rb[1:8, first:first + cols]
        want_sum = torch.empty(7, cols, device="cuda")
        want_y = torch.empty(7, cols, device="cuda")
        want = m.norm_quantize(x, w, residual=r, norm=norm, sum_out=want_sum, norm_out=want_y)
        _rows_check(want, *_norm_reference(x, r, w, None, norm, 1e-12)[1:])
        rb1 = rb.clone()
        got = m.norm_quantize(x, w, residual=rb1[1:8, first:first + cols], norm=norm, sum_out=rb1[1:8, first:first + cols])
        assert torch.equal(got.q, want.q) and torch.equal(got.scale, want.scale)
        assert torch.equal(rb1[1:8, first:first + cols], want_sum)
        rb1[1:8, first:first + cols] = r
        assert torch.equal(rb1, rb)
        rb2 = rb.clone()
        got = m.norm_quantize(x, w, residual=rb2[1:8, first:first + cols], norm=norm, norm_out=rb2[1:8, first:first + cols])
        assert torch.equal(got.q, want.q) and torch.equal(rb2[1:8, first:first + cols], want_y)
        xb3 = xb.clone()
        got = m.norm_quantize(xb3[1:8, first:first + cols], w, residual=r, norm=norm, norm_out=xb3[1:8, first:first + cols])
        assert torch.equal(got.q, want.q) and torch.equal(xb3[1:8, first:first + cols], want_y.to(torch.bfloat16))
        xb3[1:8, first:first + cols] = x
        assert torch.equal(xb3, xb)


@gpu
@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("cols", [33, 900, 6000])
def test_norm_edges(cols, norm):
    m, g = _ops(), _gen(cols)
    weight = 1 + 0.2 * torch.randn(cols, generator=g, device="cuda")
    bias = 0.3 * torch.randn(cols, generator=g, device="cuda")
    x = torch.randn(8, cols, generator=g, device="cuda")
    x[1] = 0.0                                    # zeros: v = bias
    x[2] = 1000.0 + 0.01 * x[2]                   # a mean far above the deviations
    x[3, cols // 2] = float("nan")
    x[4, 0] = float("inf")
    x[5] *= 1e25                                  # squares past fp32
    x[6] *= 1e-25                                 # eps decides
    out = m.norm_quantize(x, weight, bias=bias, norm=norm, eps=1e-6)
    fine = [0, 1, 2, 6, 7]
    _, v, dv = _norm_reference(x[fine], None, weight, bias, norm, 1e-6)
    _rows_check(_Rows(out.q[fine], out.scale[fine]), v, dv)
    assert bool(out.scale[3:6].isnan().all()) and bool((out.q[3:6] == 0).all())
    zero = m.norm_quantize(torch.zeros(2, cols, device="cuda"), weight, norm=norm, eps=1e-6)
    assert bool((zero.scale == 0).all()) and bool((zero.q == 0).all())


class _Rows:
    def __init__(self, q, scale):
        self.q, self.scale = q, scale


# ---- together -----------------------------------------------------------------------------
def _half_layer(m, x, r, p):
    """What a layer of the encoder does between its attention and its end."""
    rows = m.norm_quantize(x, p["g"], p["b"], residual=r, norm_out=r)
    y = m.int8_linear(rows, p["w1"], bias=p["b1"], dtype=torch.float16)
    rows = m.quantize_rows(y, act="gelu")
    y = m.int8_linear(rows, p["w2"], bias=p["b2"], dtype=torch.float16)
    return m.norm_quantize(y, p["g"], p["b"], residual=r, norm_out=r)


def _half_layer_inputs(m, T, H, F, seed):
    g = _gen(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")   # noqa: E731
    p = dict(g=1 + 0.1 * n(H), b=0.1 * n(H), b1=0.1 * n(F), b2=0.1 * n(H),
             w1=m.quantize_rows(n(F, H) / H ** 0.5), w2=m.quantize_rows(n(H, F) / F ** 0.5))
    return n(T, H).to(torch.float16), n(T, H), p


@gpu
@pytest.mark.parametrize("T,H,F", [(1, 384, 1536), (14, 384, 1536), (613, 384, 1536), (2500, 128, 512)])
def test_together_against_64_bits(T, H, F):
    """The run in 64 bits with the same int8 grids.  An element that differs by rounding (f16
    products: 2^-11 of its value, under 1/16 of a step of max|v| / 127) lands on another step in at
    most 1 of 8 cases, so a quantisation's disagreement has a 2-norm under sqrt(1/8) of a step per
    element, which is 1.23 times what the rounding to steps itself costs (1/sqrt(12)).  The products
    and norms of the run have unit gain, and two quantisations lie before the result: a relative
    2-norm of at most 2 * step / sqrt(8)."""
    m = _ops()
    x, r, p = _half_layer_inputs(m, T, H, F, T)
    r0 = r.clone()
    out = _half_layer(m, x, r, p)

    def rows64(v):
        s = v.abs().amax(1, keepdim=True) / 127
        return torch.round(v / s) * s

    def norm64(h):
        d = h - h.mean(1, keepdim=True)
        return d / ((d * d).mean(1, keepdim=True) + 1e-12).sqrt() * p["g"].to(D) + p["b"].to(D)

    w = lambda k: p[k].q.to(D) * p[k].scale.to(D)[:, None]      # noqa: E731
    n = norm64(x.to(D) + r0.to(D))
    y = rows64(n) @ w("w1").T + p["b1"].to(D)
    y = rows64(y * torch.special.ndtr(y)) @ w("w2").T + p["b2"].to(D)
    want = norm64(y + n)
    step = want.abs().amax(1) / 127 / want.pow(2).mean(1).sqrt()
    bound = 2 * float(step.max()) / 8 ** 0.5
    rel = float((r.to(D) - want).norm() / want.norm())
    assert rel <= bound, (rel, bound)
    assert torch.equal(out.q, m.quantize_rows(r).q)             # the int8 rows are those of norm_out


@gpu
def test_captured_and_replayed():
    """A graph of the whole run, replayed among eager work: every replay equals the eager result."""
    m = _ops()
    for T in (1, 14, 300, 2100):
        x, r, p = _half_layer_inputs(m, T, 384, 1536, T)
        r0 = r.clone()
        want = _half_layer(m, x, r, p)
        want_q, want_s, want_r = want.q.clone(), want.scale.clone(), r.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            r.copy_(r0)
            _half_layer(m, x, r, p)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r.copy_(r0)
            got = _half_layer(m, x, r, p)
        for i in range(4):
            graph.replay()
            if i % 2:
                other = _half_layer(m, x, r0.clone(), p)        # eager work between the replays
                assert torch.equal(other.q, want_q)
            torch.cuda.synchronize()
            assert torch.equal(got.q, want_q) and torch.equal(got.scale, want_s) and torch.equal(r, want_r)


@gpu
def test_two_streams_and_threads_at_once():
    import threading
    m = _ops()
    sets = [_half_layer_inputs(m, 800 + 100 * i, 384, 1536, i) for i in range(3)]
    want = [_half_layer(m, x, r.clone(), p).q.clone() for x, r, p in sets]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            x, r, p = sets[i]
            for _ in range(5):
                got = _half_layer(m, x, r.clone(), p)
                s.synchronize()
                if not torch.equal(got.q, want[i]):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


# ---- results larger than any cache (256 MiB and more: non-temporal loads and stores) ----------
PARTS = (slice(0, 300), slice(35000, 35300), slice(-301, None))


@gpu
@pytest.mark.parametrize("out", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("K", [384, 1024])
def test_linear_past_the_caches(K, out):
    """The same bits as parts of the batch, which the caches hold."""
    m, g = _ops(), _gen(K)
    T, N = 70001, 2048
    x, w = _int8(g, T, K), _int8(g, N, K)
    sx, sw, b = _scales(g, T), _scales(g, N), torch.randn(N, generator=g, device="cuda")
    rows = m.Int8Rows(w, sw)
    y = m.int8_linear(m.Int8Rows(x, sx), rows, bias=b, dtype=DT[out])
    for p in PARTS:
        want = m.int8_linear(m.Int8Rows(x[p], sx[p]), rows, bias=b, dtype=DT[out])
        assert torch.equal(y[p], want)
        _linear_check(want, x[p], sx[p], w, sw, b)


@gpu
@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("xt,rt,yt", [("bf16", "bf16", "bf16"), ("f16", "f32", "f16"), ("f32", "f16", "f32")])
@pytest.mark.parametrize("cols", [1001, 2304])
def test_rows_past_the_caches(cols, xt, rt, yt, norm):
    m, g = _ops(), _gen(cols)
    T = 70001
    x = torch.randn(T, cols, generator=g, device="cuda").to(DT[xt])
    r = torch.randn(T, cols, generator=g, device="cuda").to(DT[rt])
    w, b = torch.randn(cols, generator=g, device="cuda"), torch.randn(cols, generator=g, device="cuda")
    total, y = torch.empty_like(r), torch.empty(T, cols, device="cuda", dtype=DT[yt])
    q = m.norm_quantize(x, w, b, residual=r, norm=norm, sum_out=total, norm_out=y)
    gelu, v = m.quantize_rows(x, act="gelu"), q.dequantize(DT[yt])
    for p in PARTS:
        n = len(x[p])
        part_total, part_y = torch.empty(n, cols, device="cuda", dtype=DT[rt]), torch.empty(n, cols, device="cuda", dtype=DT[yt])
        part = m.norm_quantize(x[p], w, b, residual=r[p], norm=norm, sum_out=part_total, norm_out=part_y)
        assert torch.equal(q.q[p], part.q) and torch.equal(q.scale[p], part.scale)
        assert torch.equal(total[p], part_total) and torch.equal(y[p], part_y)
        assert torch.equal(v[p], part.dequantize(DT[yt]))
        part = m.quantize_rows(x[p], act="gelu")
        assert torch.equal(gelu.q[p], part.q) and torch.equal(gelu.scale[p], part.scale)


@gpu
def test_rows_keep_their_checked_buffers():
    m = _ops()
    r = m.quantize_rows(torch.ones(3, 5, device="cuda"))
    for name in ("q", "scale"):
        with pytest.raises(AttributeError):
            setattr(r, name, torch.ones(3))


@gpu
def test_refusals_of_device_tensors():
    m = _ops()
    x = torch.randn(4, 32, device="cuda")
    g = torch.ones(32, device="cuda")
    rows = m.quantize_rows(x)
    with pytest.raises(ValueError, match="dtype"):
        m.quantize_rows(x.double())
    with pytest.raises(ValueError, match="dimension"):
        m.quantize_rows(x[0])
    with pytest.raises(ValueError, match="contiguous"):
        m.quantize_rows(x.T)
    with pytest.raises(ValueError, match="stride"):
        m.quantize_rows(x[:1].expand(4, 32))
    with pytest.raises(ValueError, match="activation"):
        m.quantize_rows(x, act="relu")
    with pytest.raises(ValueError, match="cols"):
        m.quantize_rows(torch.zeros(1, 32769, device="cuda"))
    with pytest.raises(ValueError, match="cols"):
        m.quantize_rows(torch.zeros(1, 0, device="cuda"))
    with pytest.raises(ValueError, match="gradient"):
        m.quantize_rows(x.clone().requires_grad_())
    with torch.no_grad():
        m.quantize_rows(x.clone().requires_grad_())
    with pytest.raises(ValueError, match="out"):
        m.quantize_rows(x, out=m.Int8Rows.empty(3, 32, x.device))
    with pytest.raises(ValueError, match="norm"):
        m.norm_quantize(x, g, norm="batch")
    with pytest.raises(ValueError, match="weight"):
        m.norm_quantize(x, g[:31])
    with pytest.raises(ValueError, match="weight"):
        m.norm_quantize(x, g.half())
    with pytest.raises(ValueError, match="residual"):
        m.norm_quantize(x, g, residual=x[:3])
    with pytest.raises(ValueError, match="sum_out"):
        m.norm_quantize(x, g, sum_out=torch.empty_like(x))
    with pytest.raises(ValueError, match="sum_out"):
        m.norm_quantize(x, g, residual=x, sum_out=torch.empty_like(x).half())
    with pytest.raises(ValueError, match="eps"):
        m.norm_quantize(x, g, eps=-1.0)
    with pytest.raises(ValueError, match="device tensor"):
        m.norm_quantize(x, g, residual=x.cpu())
    with pytest.raises(ValueError, match="16 bytes"):
        m.Int8Rows(torch.zeros(4, 40, dtype=torch.int8, device="cuda")[:, :33], torch.ones(4, device="cuda"))
    with pytest.raises(ValueError, match="16 bytes"):
        m.Int8Rows(torch.zeros(4, 48, dtype=torch.int8, device="cuda")[:, 1:33], torch.ones(4, device="cuda"))
    with pytest.raises(ValueError, match="scales"):
        m.Int8Rows(rows.q, rows.scale[:3])
    with pytest.raises(ValueError, match="depth"):
        m.int8_linear(rows, m.quantize_rows(x[:, :16].contiguous()))
    with pytest.raises(ValueError, match="bias"):
        m.int8_linear(rows, rows, bias=g)
    with pytest.raises(ValueError, match="dtype"):
        m.int8_linear(rows, rows, dtype=torch.float64)
    with pytest.raises(ValueError, match="out"):
        m.int8_linear(rows, rows, out=torch.empty(4, 5, device="cuda"))
    with pytest.raises(ValueError, match="Int8Rows"):
        m.int8_linear(x, rows)
