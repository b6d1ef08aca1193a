"""What the 8-bit integer operators refuse, or have to say, beyond their arguments' shapes: rows on the
host, gradients and tensors that others have saved, buffers in each other's place."""
import os
import pickle
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")


def _ops():
    import hcrag_amd
    return hcrag_amd


def _host_rows(rows, cols):
    """Rows in host memory, as a loader leaves them (it fills the slots without the constructor)."""
    m = _ops()
    r = object.__new__(m.Int8Rows)
    r._q, r._scale = torch.zeros(rows, cols, dtype=torch.int8), torch.ones(rows)
    return pickle.loads(pickle.dumps(r))


# ---- rows in host memory: no host address may reach a kernel (all refused before any HIP call) ----
def test_empty_rows_on_the_host_are_refused():
    for device in ("cpu", torch.device("cpu"), "meta"):
        with pytest.raises(ValueError, match="device tensor"):
            _ops().Int8Rows.empty(4, 32, device)


def test_restored_host_rows_are_refused():
    m = _ops()
    x, w = _host_rows(4, 32), _host_rows(8, 32)
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        with pytest.raises(ValueError, match="device tensor"):
            x.dequantize(dtype)
        with pytest.raises(ValueError, match="device tensor"):
            m.int8_linear(x, w, dtype=dtype)
    with pytest.raises(ValueError, match="device tensor"):
        m.int8_linear(x, w, bias=torch.zeros(8))
    with pytest.raises(ValueError, match="device tensor"):
        m.int8_linear(x, w, out=torch.zeros(4, 8))
    with pytest.raises(ValueError, match="device tensor"):
        _host_rows(0, 32).dequantize()
    with pytest.raises(ValueError, match="device tensor"):
        m.quantize_rows(torch.zeros(4, 32), out=x)


# ---- outputs in the place of vectors, scales in the place of anything: refused before any HIP call ----
def _distinct():
    """Arguments of the four C entry points, every buffer in a place of its own (never read: what is
    called here is refused)."""
    from hcrag_amd import _lib
    lib = _lib.lib()
    places = {n: (i + 1) << 24 for i, n in enumerate("x r w b s y q scale out sx sw".split())}

    def quant(x, q, scale, **_):
        return lib.hcr_quant_rows_device(x, _lib.HCR_F32, 64, 4, 64, 0, q, 64, scale, None)

    def norm(x, r, w, b, s, y, q, scale, **_):
        return lib.hcr_norm_quant_rows_device(_lib.NORM_QUANT_ARGS.pack(
            x, 64, r, 64, w, b, s, 64, y, 64, q, 64, scale, 4, 64, _lib.HCR_F32, _lib.HCR_F32, _lib.HCR_F32, 0, 1e-6), None)

    def dequant(q, scale, out, **_):
        return lib.hcr_dequant_rows_device(q, 64, scale, 4, 64, out, _lib.HCR_F32, 64, None)

    def linear(x, sx, w, sw, b, out, **_):
        return lib.hcr_int8_linear_device(x, 64, sx, 4, w, 64, sw, 64, 64, b, out, _lib.HCR_F32, 64, None)

    return places, dict(quant=quant, norm=norm, dequant=dequant, linear=linear)


@pytest.mark.parametrize("call,output,operands", [
    ("quant", "q", "x"), ("quant", "scale", "x q"),
    ("norm", "scale", "x r w b s y q"), ("norm", "q", "x r w b s y"), ("norm", "s", "x w b y"), ("norm", "y", "w b"),
    ("dequant", "out", "q scale"), ("linear", "out", "x sx w sw b")])
def test_outputs_that_start_where_an_operand_does(call, output, operands):
    from hcrag_amd import _lib
    places, calls = _distinct()
    for other in operands.split():
        assert calls[call](**{**places, output: places[other]}) == _lib.HCR_EINVAL, other
        assert b"overlap" in _lib.lib().hcr_last_error(), other


# ---- the package without torch ----------------------------------------------------------------
def test_star_import_does_not_need_torch():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hc-rag_amd")
    code = (f"import sys; sys.path.insert(0, {path!r}); sys.modules['torch'] = None\n"
            "from hcrag_amd import *\n"
            "import hcrag_amd; assert VectorIndex is hcrag_amd.VectorIndex and 'int8_linear' in dir(hcrag_amd)")
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    from hcrag_amd import Int8Rows, int8, int8_linear, norm_quantize, quantize_rows  # noqa: F401


# ---- gradients: refused, never dropped in silence ---------------------------------------------
def _norm_buffers():
    x, r = torch.randn(5, 96, device="cuda"), torch.randn(5, 96, device="cuda")
    return x, r, torch.ones(96, device="cuda")


def _written(m):
    """(name, the buffer, a call that writes it) for every buffer that a caller may hand out."""
    x, r, g = _norm_buffers()
    rows, w = m.quantize_rows(x), m.quantize_rows(torch.randn(7, 96, device="cuda"))
    out, y = m.Int8Rows.empty(5, 96, x.device), torch.empty(5, 7, device="cuda")
    total, normed = torch.empty_like(r), torch.empty_like(r)
    yield "sum_out", total, lambda: m.norm_quantize(x, g, residual=r, sum_out=total)
    yield "norm_out", normed, lambda: m.norm_quantize(x, g, residual=r, norm_out=normed)
    yield "residual", r, lambda: m.norm_quantize(x, g, residual=r, norm_out=r)
    yield "norm scale", out.scale, lambda: m.norm_quantize(x, g, out=out)
    yield "norm q", out.q, lambda: m.norm_quantize(x, g, out=out)
    yield "scale", out.scale, lambda: m.quantize_rows(x, out=out)
    yield "q", out.q, lambda: m.quantize_rows(x, out=out)
    yield "out", y, lambda: m.int8_linear(rows, w, out=y)


@pytest.mark.gpu
def test_writes_are_seen_by_autograd():
    """A buffer that a backward pass has saved and an operator overwrites: the backward raises."""
    for name, buf, call in _written(_ops()):
        buf.zero_()
        before = buf._version
        call()
        assert buf._version > before, name
        if buf.is_floating_point():
            a = torch.ones_like(buf, requires_grad=True)
            (a * buf).sum().backward()                      # nothing written in between: fine
            saved = (a * buf).sum()
            call()
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                saved.backward()


@pytest.mark.gpu
def test_writes_to_inference_tensors():
    """They keep no version: written all the same, in the mode and (the call has no gradient) outside."""
    m = _ops()
    with torch.inference_mode():
        x, r, g = _norm_buffers()
        m.norm_quantize(x, g, residual=r, norm_out=r)
    with torch.no_grad():
        m.norm_quantize(x, g, residual=r, norm_out=r)


@pytest.mark.gpu
def test_scales_that_ask_for_a_gradient_are_refused():
    m = _ops()
    q = torch.ones(4, 32, dtype=torch.int8, device="cuda")
    with torch.no_grad():
        wrapped = m.Int8Rows(q, torch.ones(4, device="cuda", requires_grad=True))
    later = m.Int8Rows(q, torch.ones(4, device="cuda"))
    later.scale.requires_grad_()
    plain = m.Int8Rows(q, torch.ones(4, device="cuda"))
    for rows in (wrapped, later):
        for call in (lambda: m.int8_linear(rows, plain), lambda: m.int8_linear(plain, rows), lambda: rows.dequantize(),
                     lambda: m.quantize_rows(torch.ones(4, 32, device="cuda"), out=rows),
                     lambda: m.norm_quantize(torch.ones(4, 32, device="cuda"), torch.ones(32, device="cuda"), out=rows)):
            with pytest.raises(ValueError, match="gradient"):
                call()
        with torch.no_grad():
            assert torch.equal(m.int8_linear(rows, plain), m.int8_linear(plain, plain))
            assert bool((rows.dequantize() == 1).all())


@pytest.mark.gpu
def test_forward_mode_tangents_are_refused():
    import torch.autograd.forward_ad as fw
    m = _ops()
    x, r, g = _norm_buffers()
    rows = m.quantize_rows(x)
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))                  # noqa: E731
        wrapped = object.__new__(m.Int8Rows)                                  # (past the constructor's own check)
        wrapped._q, wrapped._scale = rows.q, dual(rows.scale)
        for call in (lambda: m.quantize_rows(dual(x)), lambda: m.norm_quantize(dual(x), g),
                     lambda: m.norm_quantize(x, dual(g)), lambda: m.norm_quantize(x, g, bias=dual(g)),
                     lambda: m.norm_quantize(x, g, residual=dual(r)), lambda: m.Int8Rows(rows.q, dual(rows.scale)),
                     lambda: m.int8_linear(rows, rows, bias=dual(g[:5].contiguous())), lambda: m.int8_linear(wrapped, rows),
                     lambda: m.int8_linear(rows, wrapped), lambda: wrapped.dequantize(),
                     lambda: m.quantize_rows(x, out=wrapped)):
            with pytest.raises(ValueError, match="gradient"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="gradient"):
                call()
        assert torch.equal(m.quantize_rows(x).q, rows.q)                      # no tangent: as ever


# ---- launches ---------------------------------------------------------------------------------
@pytest.mark.gpu
def test_linear_far_rows_few_features():
    """Weight rows 8 MiB apart and so many tokens that a launch over all of them would have 2^32 threads
    (a workgroup takes 32 features, however few there are)."""
    m = _ops()
    T, N, K, ld = 2 ** 29, 2, 16, 2 ** 23 + 16
    w = torch.zeros(N * ld, device="cuda", dtype=torch.int8).as_strided((N, K), (ld, 1))
    w[0, 0], w[1, 1] = 2, -3
    x = torch.zeros(T, K, device="cuda", dtype=torch.int8)
    step = 2 ** 26
    for t in range(0, T, step):
        at = torch.arange(t, t + step, device="cuda")
        x[t:t + step, 0], x[t:t + step, 1] = (at % 251 - 125).to(torch.int8), (at % 113 - 56).to(torch.int8)
    y = m.int8_linear(m.Int8Rows(x, torch.ones(T, device="cuda")), m.Int8Rows(w, torch.ones(N, device="cuda")))
    for t in range(0, T, step):
        at = torch.arange(t, t + step, device="cuda")
        assert torch.equal(y[t:t + step, 0], ((at % 251 - 125) * 2).to(y.dtype))       # (whole numbers that f16 holds)
        assert torch.equal(y[t:t + step, 1], ((at % 113 - 56) * -3).to(y.dtype))
