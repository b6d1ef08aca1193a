"""What the 8-bit integer operators refuse, or have to say, beyond their arguments' shapes: rows on the
host, gradients and tensors that others have saved, buffers in each other's place."""
import pickle

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
