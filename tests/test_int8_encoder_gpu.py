"""The encoder's 8-bit integer mode (``BertEncoder(dtype="i8")``, hcr_encoder_create(HCR_I8)).

Against a 64-bit computation of the same quantised model: an element that differs by rounding (f16
products: 2^-11 of its value, under 1/16 of a step of max|v| / 127) lands on another step in at most
1 of 8 cases, so one quantisation's disagreement has a 2-norm under sqrt(1/8) of a step per element.
Products, attention and norms have at most unit gain on the residual stream, so L layers (4
quantisations each, 1 before them) stay within (4 L + 1) * step / sqrt(8), relative, step the largest
max|v| / (127 rms) met.

Against fp32 BertModel: an operand rounded to steps of max|v| / 127 with max|v| <= 5 rms is off by
5 / 127 / sqrt(12) = 1.1 % of its norm, a product of two such by 1.6 %, a layer's two branches (two
products each) by 2.3 % each of a stream that is at least as large; 6 layers: sqrt(12) * 2.3 % = 8 %,
cosine >= 0.9968.  The bar is 0.99.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
transformers = pytest.importorskip("transformers")

from test_encoder_gpu import MINILM, TINY, _batch, _encoder, _hf_model, _ref_embed  # noqa: E402

pytestmark = pytest.mark.gpu
D = torch.float64


def _rows64(v, seen):
    a = v.abs().amax(1, keepdim=True)
    seen.append(float((a / 127 / v.pow(2).mean(1, keepdim=True).sqrt()).max()))
    return torch.round(v * 127 / a) * a / 127


def _emulate(conf, m, ids, mask, pooling):
    """The quantised model in 64 bits; returns (embeddings, largest step / rms)."""
    sd = {k: v.detach().to("cuda", D) for k, v in m.state_dict().items()}
    heads, dh = conf.num_attention_heads, conf.hidden_size // conf.num_attention_heads
    seen = []

    def norm(h, p):
        d = h - h.mean(1, keepdim=True)
        return d / ((d * d).mean(1, keepdim=True) + 1e-12).sqrt() * sd[p + ".weight"] + sd[p + ".bias"]

    def linear(x, p):
        return _rows64(x, seen) @ _rows64(sd[p + ".weight"], []).T + sd[p + ".bias"]

    out = []
    for row, keep in zip(ids, mask):
        S = int(keep.sum())
        t = torch.from_numpy(row[:S].astype(np.int64)).cuda()
        e = "embeddings."
        x = norm(sd[e + "word_embeddings.weight"][t] + sd[e + "token_type_embeddings.weight"][0]
                 + sd[e + "position_embeddings.weight"][:S], e + "LayerNorm")
        for i in range(conf.num_hidden_layers):
            p = f"encoder.layer.{i}."
            q, k, v = (linear(x, p + "attention.self." + n) for n in ("query", "key", "value"))
            ctx = torch.empty_like(x)
            for h in range(heads):
                s = slice(h * dh, (h + 1) * dh)
                ctx[:, s] = torch.softmax(q[:, s] @ k[:, s].T / dh ** 0.5, 1) @ v[:, s]
            x = norm(linear(ctx, p + "attention.output.dense") + x, p + "attention.output.LayerNorm")
            y = linear(x, p + "intermediate.dense")
            y = linear(y * torch.special.ndtr(y), p + "output.dense")
            x = norm(y + x, p + "output.LayerNorm")
        v = x.mean(0) if pooling == "mean" else x[0]
        out.append(v / v.norm())
    return torch.stack(out).cpu().numpy(), max(seen)


@pytest.mark.parametrize("pooling", ["mean", "cls"])
@pytest.mark.parametrize("lens", [[1], [1, 1, 1, 1, 1], [37], [1, 2, 37, 36, 5, 17, 33, 3, 9, 10, 11, 12, 37]])
def test_against_the_quantised_model_in_64_bits(lens, pooling):
    conf, m = _hf_model(TINY, 1)
    ids, mask = _batch(np.random.default_rng(0), len(lens), 37, TINY["vocab_size"], lens=lens)
    got = _encoder(conf, m, "i8", pooling).encode_ids(ids, mask)
    want, step = _emulate(conf, m, ids, mask, pooling)
    bound = (4 * TINY["num_hidden_layers"] + 1) * step / 8 ** 0.5
    rel = np.linalg.norm(got - want, axis=1)
    print("relative", rel.max(), "bound", bound)
    assert rel.max() <= bound


@pytest.mark.parametrize("n,S", [(1, 14), (24, 128), (300, 40)])
def test_against_fp32_bert(n, S):
    conf, m = _hf_model(MINILM, 2)
    ids, mask = _batch(np.random.default_rng(1), n, S, MINILM["vocab_size"])
    got = _encoder(conf, m, "i8").encode_ids(ids, mask)
    ref = _ref_embed(m, ids, mask)
    cos = np.sum(got * ref, 1)
    print("least cosine", cos.min())
    assert cos.min() >= 0.99
    assert np.allclose(np.linalg.norm(got, axis=1), 1.0, atol=1e-5)


def test_a_sequence_does_not_depend_on_its_batch():
    """Alone (few-token kernels, one stream) and among 299 others (tiles, two streams): the same
    bits, since the integer sums are exact and everything else is per row."""
    conf, m = _hf_model(MINILM, 3)
    ids, mask = _batch(np.random.default_rng(5), 300, 40, MINILM["vocab_size"])
    enc = _encoder(conf, m, "i8")
    every = enc.encode_ids(ids, mask)
    assert np.array_equal(every, enc.encode_ids(ids, mask))
    for i in (0, 7, 150, 299):
        assert np.array_equal(every[i], enc.encode_ids(ids[i:i + 1], mask[i:i + 1])[0])


def test_device_call_empty_masks_and_names():
    from hcrag_amd import BertEncoder, config_from_hf
    conf, m = _hf_model(TINY, 4)
    enc = BertEncoder(config_from_hf(conf.to_dict(), "mean", True), m.state_dict(), dtype="int8")
    ids, mask = _batch(np.random.default_rng(2), 5, 20, TINY["vocab_size"])
    mask[2] = 0                                   # a sequence without tokens
    want = enc.encode_ids(ids, mask)
    assert np.array_equal(want[2], np.zeros_like(want[2])) and np.isfinite(want).all()
    out = torch.full((5, enc.hidden), 3.0, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        enc.encode_device(torch.from_numpy(ids).cuda(), torch.from_numpy(mask).cuda(), out)
    s.synchronize()
    assert np.array_equal(out.cpu().numpy(), want)
    mask[:] = 0
    assert np.array_equal(enc.encode_ids(ids, mask), np.zeros_like(want))
    assert enc.encode_ids(ids[:0], mask[:0]).shape == (0, enc.hidden)


@pytest.mark.parametrize("dtype", ["i8", "f16", "f32"])
@pytest.mark.parametrize("sizes", [(300,) * 4, (100,) * 4, (300, 90, 290, 100)])
def test_calls_on_two_streams_one_after_the_other(sizes, dtype):
    """Small batches run on the caller's stream, large ones on it and one more: the next call may come
    on another stream without a wait in between."""
    conf, m = _hf_model(MINILM, 6)
    enc = _encoder(conf, m, dtype)
    rng = np.random.default_rng(8)
    host = [_batch(rng, n, 64, MINILM["vocab_size"]) for n in sizes]
    batches = [tuple(torch.from_numpy(a).cuda() for a in b) for b in host]
    want = []
    for ids, mask in batches:
        out = torch.empty(len(ids), enc.hidden, device="cuda")
        enc.encode_device(ids, mask, out)
        torch.cuda.synchronize()
        want.append(out)
    if dtype == "i8":                             # (one sequence: one stream, kernels for few tokens)
        assert np.array_equal(want[1][80].cpu().numpy(), enc.encode_ids(*(a[80:81] for a in host[1]))[0])
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.full_like(w, -1.0) for w in want]
    torch.cuda.synchronize()
    for i, (ids, mask) in enumerate(batches):
        with torch.cuda.stream(streams[i % 2]):
            enc.encode_device(ids, mask, outs[i])
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)
