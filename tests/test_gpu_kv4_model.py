"""Llama models whose keys and values are held in 4 bits, and log probabilities of texts: append, attention and scores as a model runs them."""
import numpy as np
import pytest

import kv4_ref as ref
import zamitar_models
from alice_llm_b200 import _lib, synth
from softmodel import SMOOTH_MIX, soft_model

pytestmark = pytest.mark.gpu

CFG = dict(num_layers=2, hidden_dim=512, intermediate_dim=1024, num_heads=4, num_kv_heads=2, head_dim=128,
           vocab_size=1000, max_seq_len=640, rope_theta=500000.0, eps=1e-5, neox_rope=0)


@pytest.fixture(scope="module")
def eng():
    from alice_llm_b200.gpu import GpuEngine
    e = GpuEngine(0)
    yield e
    e.close()


def dense(entry, rows, cols):
    pos, neg, scale = entry[1]
    bits = lambda a: np.unpackbits(np.asarray(a, np.uint8).reshape(rows, -1), axis=1, bitorder="little")[:, :cols].astype(np.float64)  # noqa: E731
    return (bits(pos) - bits(neg)) * np.asarray(scale, np.float64)[:, None]


class Plain:
    """The ternary model in 64 bits, over the keys and values that the device holds."""

    def __init__(self, model):
        c = model["config"]
        self.c, self.model = c, model
        H, F, Q, K = c["hidden_dim"], c["intermediate_dim"], c["num_heads"] * 128, c["num_kv_heads"] * 128
        shapes = dict(q=(Q, H), k=(K, H), v=(K, H), o=(H, Q), gate=(F, H), up=(F, H), down=(H, F))
        self.layers = [{n: dense(L[n], *s) for n, s in shapes.items()} for L in model["layers"]]
        self.head = dense(model["output"], c["vocab_size"], H)
        raw = np.asarray(model["embedding"][1], np.uint8).reshape(c["vocab_size"], H // 32, 34)
        self.embed = (raw[..., :2].copy().view(np.float16).astype(np.float64) * raw[..., 2:].view(np.int8).astype(np.float64)).reshape(c["vocab_size"], H)

    def norm(self, x, w):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.c["eps"]) * np.asarray(w, np.float64)

    def run(self, gm, tokens, start):
        """Logits of consecutive tokens from position start, with the cache as gm holds it; checks what is held of them on the way."""
        c, n = self.c, len(tokens)
        kh, heads = c["num_kv_heads"], c["num_heads"]
        table = ref.rope(start + n, 128, c["rope_theta"])
        pos = start + np.arange(n)
        x = self.embed[np.asarray(tokens)]
        for l, (W, L) in enumerate(zip(self.layers, self.model["layers"])):
            h = self.norm(x, L["attn_norm"])
            q, k, v = (h @ W[i].T for i in "qkv")
            turn = lambda a, m: ref.rotate(a.reshape(n, m, 128), table, pos, 128, c["neox_rope"])  # noqa: E731
            q, k = turn(q, heads), turn(k, kh)
            kd, vd = (a.astype(np.float64).reshape(start + n, kh, 128) for a in gm.kv_read(l, 0, start + n))
            for held, own in ((kd[start:], k), (vd[start:], v.reshape(n, kh, 128))):
                _, d, m = ref.quantize(own)
                # half a step, what the formats of step and minimum round, and what f32 products before them are off (1e-4 of a row)
                room = np.repeat(0.5 * d + (np.abs(m) + 15 * d) * 2.0 ** -10, 32, -1) + 1e-4 * np.abs(own).max()
                assert (np.abs(held - own) <= room).all()
            out, _ = ref.attention(q, kd, vd, start, 128 ** -0.5)
            x = x + out.reshape(n, -1) @ W["o"].T
            h = self.norm(x, L["ffn_norm"])
            g = h @ W["gate"].T
            x = x + (g / (1 + np.exp(-g)) * (h @ W["up"].T)) @ W["down"].T
        return self.norm(x, self.model["output_norm"]) @ self.head.T


def near(got, want):
    """The models' gate everywhere in this suite: 1e-3 of the larger of 1 and the value, and of the row's norm."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    return (np.abs(got - want) <= 1e-3 * np.maximum(np.abs(want), 1)).all() and np.linalg.norm(got - want) <= 1e-3 * np.linalg.norm(want)


@pytest.mark.parametrize("heads,kv_heads,neox", [(4, 2, 0), (8, 8, 1), (5, 1, 0), (8, 1, 1)])
def test_logits_over_the_held_cache(eng, heads, kv_heads, neox):
    from alice_llm_b200.gpu import GpuModel
    rng = np.random.default_rng(heads)
    model = soft_model(rng, dict(CFG, num_heads=heads, num_kv_heads=kv_heads, neox_rope=neox), SMOOTH_MIX)
    gm, plain = GpuModel.load(eng, model, kv_cache="q4"), Plain(model)
    kv = kv_heads * 128
    for l in range(2):
        gm.kv_write(l, 0, rng.normal(size=(37, kv)), rng.normal(size=(37, kv)))
    gm.set_position(37)
    for i, tok in enumerate([1, 17, 999, 3]):                      # single tokens
        assert near(gm.forward_and_read(tok), plain.run(gm, [tok], 37 + i)[0])
    got = gm.forward_batch_and_read([5, 6, 7]).reshape(3, -1)      # a draft
    assert near(got, plain.run(gm, [5, 6, 7], 41))
    gm.rollback_to(42)
    prompt = rng.integers(0, 1000, 300)                            # more than a piece
    rows = [0, 15, 255, 256, 299]
    got = gm.forward_rows(prompt, rows)
    assert gm.position() == 342
    assert near(got, plain.run(gm, prompt, 42)[rows])
    gm.free()


def test_written_rows_are_held_to_the_bit(eng):
    from alice_llm_b200.gpu import GpuModel
    rng = np.random.default_rng(1)
    gm = GpuModel.load(eng, synth.make_llama(rng, CFG), kv_cache="q4")
    k, v = (rng.normal(size=(600, 2, 128)).astype(np.float32) for _ in range(2))
    gm.kv_write(1, 3, k, v)
    for lo, n in ((3, 600), (200, 70), (3, 1)):
        gk, gv = gm.kv_read(1, lo, n)
        assert np.array_equal(gk.reshape(n, 2, 128), ref.held(k.astype(np.float64))[lo - 3:lo - 3 + n].astype(np.float32))
        assert np.array_equal(gv.reshape(n, 2, 128), ref.held(v.astype(np.float64))[lo - 3:lo - 3 + n].astype(np.float32))
    assert not np.any(gm.kv_read(0, 0, 640)[0]) and not np.any(gm.kv_read(1, 603, 37)[1])
    gm.reset()
    assert not np.any(gm.kv_read(1, 0, 640)[0])
    with pytest.raises(_lib.AliceError):
        gm.kv_write(0, 600, k[:41], v[:41])
    gm.free()


@pytest.mark.parametrize("mix", [None, SMOOTH_MIX])
def test_greedy_decoding_is_stepping(eng, mix):
    """The captured step, replayed, against steps whose logits are read; again after a reset, and beside a model with an f32 cache."""
    from alice_llm_b200.gpu import GpuModel
    rng = np.random.default_rng(2)
    model = soft_model(rng, CFG, mix)
    gm, other = GpuModel.load(eng, model, kv_cache="q4"), GpuModel.load(eng, model)
    first = gm.decode_greedy(7, 20)
    other.decode_greedy(7, 5)
    gm.reset()
    assert np.array_equal(gm.decode_greedy(7, 20), first)
    gm.reset()
    tok = 7
    for want in first:
        tok = int(np.argmax(gm.forward_and_read(tok)))
        assert tok == want
    assert gm.position() == 20
    gm.rollback_to(4)
    assert np.array_equal(gm.decode_greedy(int(first[3]), 16), first[4:])
    gm.free(), other.free()


def scores(logits, targets, top):
    z = logits.astype(np.float64)
    z = z - z.max(1, keepdims=True)
    lp = z - np.log(np.exp(z).sum(1, keepdims=True))
    order = np.argsort(-logits.astype(np.float64), axis=1, kind="stable")[:, :top]
    at = np.arange(len(z))
    return (lp[at, targets], -(np.exp(lp) * lp).sum(1), (logits > logits[at, targets][:, None]).sum(1) + 1, order, np.take_along_axis(lp, order, 1))


def check_scores(gm, tokens, targets, top):
    """Against the same logits brought to the host. Sums of 1000 exponentials lose less than 400 * 2^-24 (the kernel's own test derives it)."""
    gm.reset()
    lg = gm.forward_rows(tokens, np.arange(len(tokens)))
    gm.reset()
    got = gm.log_probs(tokens, targets, top=top)
    assert gm.position() == len(tokens)
    want = scores(lg, np.asarray(targets), top)
    for name, w in zip(("log_probs", "entropy", "rank", "top_ids", "top_log_probs"), want):
        if name not in got:
            assert top == 0 and name.startswith("top")
        elif name in ("rank", "top_ids"):
            assert np.array_equal(got[name], w), name
        else:
            assert (np.abs(got[name] - w) <= 400 * 2.0 ** -24 * (1 + np.abs(w))).all(), name


@pytest.mark.parametrize("kv_cache", ["f32", "q4"])
@pytest.mark.parametrize("n", [1, 2, 8, 9, 257, 300])
def test_log_probs_of_llama_models(eng, kv_cache, n):
    from alice_llm_b200.gpu import GpuModel
    rng = np.random.default_rng(n)
    gm = GpuModel.load(eng, soft_model(rng, CFG), kv_cache=kv_cache)
    tokens, targets = rng.integers(0, 1000, (2, n))
    for top in (0, 5, 32):
        check_scores(gm, tokens, targets, top)
    gm.free()


def test_log_probs_of_layer_stacks(eng):
    from alice_llm_b200.gpu import GpuModel
    rng = np.random.default_rng(5)
    cfg = zamitar_models.config([zamitar_models.latent(), zamitar_models.delta()])
    gm = GpuModel.load_stack(eng, (cfg, zamitar_models.weights(cfg)), dtype="float32", max_seq_len=64)
    vocab = gm.vocab_size()
    tokens, targets = rng.integers(0, vocab, (2, 40))
    check_scores(gm, tokens, targets, 4)
    gm.free()


def test_a_text_scored(eng):
    """Without targets: every token but the first, behind those before it; the sum is the text's."""
    from alice_llm_b200.gpu import GpuModel
    rng = np.random.default_rng(6)
    gm = GpuModel.load(eng, soft_model(rng, CFG), kv_cache="q4")
    text = rng.integers(0, 1000, 50)
    got = gm.log_probs(text)
    gm.reset()
    want = gm.log_probs(text[:-1], text[1:])
    assert all(np.array_equal(got[k], want[k]) for k in ("log_probs", "entropy", "rank")) and set(got) == {"log_probs", "entropy", "rank"}
    assert (got["log_probs"] < 0).all() and (got["rank"] >= 1).all()
    gm.reset()
    assert gm.log_probs(text[:1])["log_probs"].size == 0 and gm.position() == 0
    gm.free()


def test_refusals(eng):
    from alice_llm_b200.gpu import AliceError, GpuModel
    model = synth.make_llama(np.random.default_rng(7), CFG)
    with pytest.raises(AliceError) as ei:
        GpuModel.load(eng, model, kv_cache="q8")
    assert ei.value.code == _lib.E_INVALID
    gm = GpuModel.load(eng, model, kv_cache="q4")
    for args, kw, code in ((([1, 2], [3]), {}, _lib.E_SHAPE), (([1], [1000]), {}, _lib.E_INVALID), (([1000], [1]), {}, _lib.E_INVALID), (([1], [1]), {"top": 33}, _lib.E_SHAPE),
                           (([1], [1]), {"top": -1}, _lib.E_SHAPE), (([1] * 641, [1] * 641), {}, _lib.E_SHAPE)):
        with pytest.raises(AliceError) as ei:
            gm.log_probs(*args, **kw)
        assert ei.value.code == code
    assert gm.position() == 0 and np.isfinite(gm.forward_and_read(1)).all()
    gm.free()


def test_a_refused_text_moves_nothing(eng):
    """A token that is none in the last piece of a text: no piece before it has been taken either."""
    from alice_llm_b200.gpu import GpuModel
    gm = GpuModel.load(eng, synth.make_llama(np.random.default_rng(8), CFG), kv_cache="q4")
    text = np.arange(600) % CFG["vocab_size"]
    gm.forward(5)
    before = [x.copy() for x in gm.kv_read(1, 0, 1)]
    for bad in (599, 300, 0):
        wrong = text.copy()
        wrong[bad] = CFG["vocab_size"]
        with pytest.raises(_lib.AliceError) as ei:
            gm.log_probs(wrong, text)
        assert ei.value.code == _lib.E_INVALID and gm.position() == 1
    assert all(np.array_equal(a, b) for a, b in zip(before, gm.kv_read(1, 0, 1)))
    gm.free()
