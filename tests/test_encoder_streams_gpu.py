"""The encoder's calls on different streams after one that failed when part of it was under way."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_int8_wiring import _batch, _weights  # noqa: E402

pytestmark = pytest.mark.gpu
CFG = dict(vocab_size=211, hidden=128, layers=2, heads=2, intermediate=256, max_position=9000, type_vocab=2)


@pytest.mark.parametrize("dtype", ["i8", "f16", "f32"])
@pytest.mark.parametrize("n_failing", [40, 200])            # (one sub-batch, and two on two streams)
@pytest.mark.parametrize("n", [20, 300])
def test_after_a_call_that_failed_on_another_stream(n, n_failing, dtype):
    """8500 tokens do not fit the attention's LDS, which shows when the embeddings and the first product
    are under way: the next call, on another stream, waits for those."""
    from hcrag_amd import BertEncoder
    enc = BertEncoder(dict(CFG, layer_norm_eps=1e-12, pooling=0, normalize=1), _weights(CFG, 5), dtype=dtype)
    ids, mask = (torch.from_numpy(a).cuda() for a in _batch(CFG, [24, 30, 7, 64] * (n // 4), 6))
    want = torch.empty(n, 128, device="cuda")
    enc.encode_device(ids, mask, want)
    long = torch.randint(0, CFG["vocab_size"], (n_failing, 8500), dtype=torch.int32, device="cuda")
    ones, none = torch.ones_like(long), torch.empty(n_failing, 128, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        got = torch.full_like(want, -1.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[0]), pytest.raises(ValueError, match="too long"):
            enc.encode_device(long, ones, none)
        with torch.cuda.stream(streams[1]):
            enc.encode_device(ids, mask, got)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    assert np.isfinite(want.cpu().numpy()).all()
