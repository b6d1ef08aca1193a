"""That every part of the encoder's 8-bit integer mode does its work: models whose branches are as large as
their residual streams (weights of deviation 1 / sqrt(fan in), biases of 1/2, peaked attention), against the
same quantised model in 64 bits.

The bar is what the mode's own roundings can do, from the 64-bit model itself: the kernels round to f16 where a
product, the softmax's weights or the attention's result leave fp32, by at most 2^-11 of the value, and a value
moved by that much may land on the next step of the int8 grid after it.  The 64-bit model is run several times
with every such value moved by the full 2^-11, up or down at random, and the bar is 3 times the largest change
of an embedding (real roundings are smaller; a changed step is one like those that the noise changes).

On the CPU, with no kernel involved: each fault below changes the embeddings by more than the bar, so the
comparison on the GPU would show it."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

D = torch.float64
CONFIGS = {
    "heads of 64": dict(vocab_size=211, hidden=128, layers=2, heads=2, intermediate=256, max_position=160, type_vocab=2),
    "heads of 32": dict(vocab_size=97, hidden=192, layers=1, heads=6, intermediate=320, max_position=64, type_vocab=2),
    "heads of 16": dict(vocab_size=97, hidden=64, layers=2, heads=4, intermediate=192, max_position=64, type_vocab=1),
    "1088 wide": dict(vocab_size=97, hidden=1088, layers=1, heads=17, intermediate=2176, max_position=64, type_vocab=2),
}
LENS = [1, 2, 37, 36, 5, 17, 33, 3, 9, 10, 11, 12, 37]


def _weights(cfg, seed):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)                               # noqa: E731
    H, F = cfg["hidden"], cfg["intermediate"]
    sd = {"embeddings.word_embeddings.weight": n(cfg["vocab_size"], H),
          "embeddings.position_embeddings.weight": n(cfg["max_position"], H),
          "embeddings.token_type_embeddings.weight": n(cfg["type_vocab"], H)}

    def norm(p):
        sd[p + ".weight"], sd[p + ".bias"] = 1 + 0.3 * n(H), 0.3 * n(H)

    def linear(p, rows, cols, gain=1.0):
        sd[p + ".weight"], sd[p + ".bias"] = gain * n(rows, cols) / cols ** 0.5, 0.5 * n(rows)

    norm("embeddings.LayerNorm")
    for i in range(cfg["layers"]):
        p = f"encoder.layer.{i}."
        linear(p + "attention.self.query", H, H, 1.5)
        linear(p + "attention.self.key", H, H, 1.5)
        linear(p + "attention.self.value", H, H)
        linear(p + "attention.output.dense", H, H)
        norm(p + "attention.output.LayerNorm")
        linear(p + "intermediate.dense", F, H)
        linear(p + "output.dense", H, F, 1.5)
        norm(p + "output.LayerNorm")
    return sd


def _batch(cfg, lens, seed):
    rng = np.random.default_rng(seed)
    S = max(lens)
    ids, mask = np.zeros((len(lens), S), np.int32), np.zeros((len(lens), S), np.int32)
    for i, L in enumerate(lens):
        ids[i, :L] = rng.integers(0, cfg["vocab_size"], size=L)
        mask[i, :L] = 1
    return ids, mask


def _rows(v):
    a = v.abs().amax(1, keepdim=True)
    return torch.round(v * 127 / a) * a / 127


def _embed64(cfg, weights, ids, mask, pooling, noise=None, fault=None):
    """Unit embeddings of the quantised model in 64 bits; ``noise``: a generator that moves what the kernels
    round to f16; ``fault``: a part done wrong."""
    sd = {k: v.to(D) for k, v in weights.items()}
    H, heads = cfg["hidden"], cfg["heads"]
    dh = H // heads

    def moved(v):
        return v if noise is None else v * (1 + 2.0 ** -11 * (2 * torch.randint(0, 2, v.shape, generator=noise) - 1))

    def norm(h, p):
        if fault == "norms swapped" and "layer" in p:
            p = p.replace("attention.output", "X") if "attention.output" in p else p.replace("output", "attention.output")
            p = p.replace("X", "output")
        d = h - h.mean(1, keepdim=True)
        return d / ((d * d).mean(1, keepdim=True) + 1e-12).sqrt() * sd[p + ".weight"] + sd[p + ".bias"]

    def linear(x, p):
        w, b = sd[p + ".weight"], sd[p + ".bias"]
        a = w.abs().amax(1, keepdim=True) / 127
        q = torch.round(w / a)
        if fault == "channel scales shifted":
            a = a.roll(1, 0)
        if fault == p.split(".", 3)[-1] + " without bias":
            b = torch.zeros_like(b)
        x = _rows(x)
        if fault == "token scales shifted":
            s = x.abs().amax(1, keepdim=True)
            x = x / s * s.roll(1, 0)
        return moved(x @ (q * a).T + b)

    S = ids.shape[1]
    pos = [torch.from_numpy(np.nonzero(m)[0]) for m in mask]
    where = torch.cat([torch.full((len(p),), i) for i, p in enumerate(pos)])
    tok = torch.cat([torch.from_numpy(ids[i].astype(np.int64))[p] for i, p in enumerate(pos)])
    place = torch.cat(pos)
    e = "embeddings."
    x = (sd[e + "word_embeddings.weight"][tok] + sd[e + "token_type_embeddings.weight"][0]
         + (0 if fault == "no positions" else sd[e + "position_embeddings.weight"][:S][place]))
    x = norm(x, e + "LayerNorm")
    for i in range(cfg["layers"]):
        p = f"encoder.layer.{i}."
        q, k, v = (linear(x, p + "attention.self." + n) for n in ("query", "key", "value"))
        if fault == "q and k swapped":
            q, k = k, q
        if fault == "k and v swapped":
            k, v = v, k
        ctx = torch.zeros_like(x)
        for j in range(heads):
            s = slice(j * dh, (j + 1) * dh)
            score = q[:, s] @ k[:, s].T / (1 if fault == "no attention scale" else dh ** 0.5)
            if fault == "uniform attention":
                score = torch.zeros_like(score)
            if fault != "sequences see each other":
                score = score.masked_fill(where[:, None] != where[None, :], -torch.inf)
            at = slice(((j + 1) % heads) * dh, ((j + 1) % heads + 1) * dh) if fault == "heads rotated" else s
            ctx[:, at] = moved(torch.softmax(score, 1)) @ v[:, s]
        y = linear(moved(ctx), p + "attention.output.dense")
        if fault == "no attention":
            y = torch.zeros_like(y)
        x = norm(y + (0 if fault == "no residual at attention" else x), p + "attention.output.LayerNorm")
        y = linear(x, p + "intermediate.dense")
        act = {"relu": torch.relu, "no activation": lambda t: t}.get(fault, lambda t: t * torch.special.ndtr(t))
        y = linear(act(y), p + "output.dense")
        if fault == "no FFN":
            y = torch.zeros_like(y)
        x = norm(y + (0 if fault == "no residual at FFN" else x), p + "output.LayerNorm")
    out = []
    for i in range(len(pos)):
        t = x[where == i]
        v = t.mean(0) if pooling == "mean" else t[0]
        out.append(v / v.norm())
    return torch.stack(out).numpy()


def _bar(cfg, weights, ids, mask, pooling):
    """(the 64-bit embeddings, the bar)"""
    want = _embed64(cfg, weights, ids, mask, pooling)
    worst = 0.0
    for seed in range(8):
        other = _embed64(cfg, weights, ids, mask, pooling, noise=torch.Generator().manual_seed(seed))
        worst = max(worst, np.linalg.norm(other - want, axis=1).max())
    return want, 3 * worst


FAULTS = ["no FFN", "no attention", "uniform attention", "no attention scale", "q and k swapped", "k and v swapped",
          "heads rotated", "sequences see each other", "norms swapped", "no residual at attention", "no residual at FFN",
          "relu", "no activation", "no positions", "channel scales shifted", "token scales shifted",
          *(n + " without bias" for n in ("attention.self.query", "attention.self.value", "attention.output.dense",
                                          "intermediate.dense", "output.dense"))]


@pytest.mark.parametrize("pooling", ["mean", "cls"])
@pytest.mark.parametrize("name", CONFIGS)
def test_every_fault_is_past_the_bar(name, pooling):
    """(key biases are left out: they move a row's scores by one constant, which the softmax takes out)"""
    cfg = CONFIGS[name]
    weights, (ids, mask) = _weights(cfg, 11), _batch(cfg, LENS, 12)
    want, bar = _bar(cfg, weights, ids, mask, pooling)
    for fault in FAULTS:
        err = np.linalg.norm(_embed64(cfg, weights, ids, mask, pooling, fault=fault) - want, axis=1).max()
        print(f"{fault:40s} {err:.4f}  bar {bar:.4f}")
        assert err > 1.5 * bar, (fault, err, bar)


@pytest.mark.gpu
@pytest.mark.parametrize("pooling", ["mean", "cls"])
@pytest.mark.parametrize("name", CONFIGS)
def test_encoder_against_the_quantised_model(name, pooling):
    from hcrag_amd import BertEncoder
    cfg = CONFIGS[name]
    weights = _weights(cfg, 11)
    enc = BertEncoder(dict(cfg, layer_norm_eps=1e-12, pooling=0 if pooling == "mean" else 1, normalize=1), weights, dtype="i8")
    many = 40 if cfg["hidden"] < 512 else 2                   # (40: two streams; the 64-bit model takes its time)
    for lens, seed in ((LENS, 12), ([37], 13), ([20, 20, 20], 14), ([1, 1, 1, 1, 1], 15), ([2, 31, 64, 1] * many, 16)):
        ids, mask = _batch(cfg, lens, seed)
        want, bar = _bar(cfg, weights, ids, mask, pooling)
        err = np.linalg.norm(enc.encode_ids(ids, mask) - want, axis=1).max()
        print(f"{len(lens)} sequences: {err:.4f}  bar {bar:.4f}")
        assert err <= bar


@pytest.mark.gpu
@pytest.mark.parametrize("n,S", [(1, 14), (24, 128), (300, 40)])
def test_cosine_to_fp32_on_seeded_weights(n, S):
    """What the header states for seeded weights: at least 0.9999."""
    pytest.importorskip("transformers")
    import test_encoder_gpu as T
    for cfg, seed in ((T.MINILM, 2), (T.MINILM, 21)):
        conf, m = T._hf_model(cfg, seed)
        ids, mask = T._batch(np.random.default_rng(seed), n, S, cfg["vocab_size"])
        cos = np.sum(T._encoder(conf, m, "i8").encode_ids(ids, mask) * T._ref_embed(m, ids, mask), 1)
        print("least cosine", cos.min())
        assert cos.min() >= 0.9999
