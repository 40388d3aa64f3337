"""Attention over the 4-bit cache at six standard deviations of its roundings: what a lost remainder, sums that run on too long or a power of two for things that
lie far apart would exceed (tests/test_kv4_tolerance_cpu.py)."""
import numpy as np
import pytest

import kv4_ref as ref
from test_gpu_kv4 import Step

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def engine():
    from alice_llm_b200.gpu import GpuEngine
    e = GpuEngine()
    yield e
    e.close()


def check(s, scale=None):
    got, scale, at = s.attend(scale=scale), scale or s.dim ** -0.5, 0
    for i, (p, t) in enumerate(zip(s.past, s.tokens)):
        kc, vc, raw = ref.quantize(s.turn(s.k[i], i)), ref.quantize(s.v[i].astype(np.float64)), s.q[at:at + t]
        rows = ref.rotate(raw, s.table, p + np.arange(t), s.rot, s.neox)
        want, w = ref.attention(rows, ref.values(*kc), ref.values(*vc), p, scale)
        tol = ref.rms_tolerance(rows, raw, ref.partners(raw, s.rot, s.neox), kc, vc, w, p, scale)
        off = np.abs(got[at:at + t] - want)
        assert (off <= tol).all(), f"sequence {i}: worst {np.max(off / tol):.3g} of the tolerance"
        at += t


@pytest.mark.parametrize("group", [1, 3, 4, 5, 8, 16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_single_tokens(engine, group, dim):
    s = Step(engine, 2 * group, 2, dim, 32, [0, 1, 15, 16, 130, 700, 2500], [1] * 7, dim, True, seed=group)
    s.fill()
    check(s)


@pytest.mark.parametrize("past", [5000, 20000])
def test_long_contexts(engine, past):
    s = Step(engine, 8, 2, 128, 64, [past, 3, past // 3], [1, 1, 1], 128, False, seed=past)
    s.fill()
    check(s)


@pytest.mark.parametrize("heads,kv_heads,dim,tokens", [(4, 4, 64, [2, 5]), (8, 2, 128, [3, 4, 1]), (6, 2, 256, [5, 17]),          # jobs of 4 to 16 rows
                                                       (8, 2, 128, [40, 9]), (14, 2, 64, [33, 70]), (5, 1, 128, [130])])         # jobs of 128 rows
def test_several_tokens(engine, heads, kv_heads, dim, tokens):
    s = Step(engine, heads, kv_heads, dim, 16, [(307 * i + 211) % 900 for i in range(len(tokens))], tokens, 32, False, seed=len(tokens) + dim)
    s.fill()
    check(s)


# One token with 1 and 7 query heads a key head (jobs of 4 and 8 rows), three with 4 (16 rows); of 256 dims 8 rows at most.
SHAPES = [(1, 1, 64), (7, 1, 64), (4, 3, 64), (1, 1, 128), (7, 1, 128), (4, 3, 128), (1, 1, 256), (7, 1, 256)]


def plain(rng, past, tokens, dim):
    return [rng.normal(size=(past + tokens, 2, dim)).astype(np.float32) for _ in range(2)]


@pytest.mark.parametrize("group,tokens,dim", SHAPES)
@pytest.mark.parametrize("far", [8, 16, 20, 30])
def test_blocks_of_a_head_far_apart(engine, group, tokens, dim, far):
    """Steps of blocks 2^far apart, from head to head in another order."""
    rng = np.random.default_rng(far)
    k, v = plain(rng, 700, tokens, dim)
    apart = np.array([0, far, far // 2, 2] * 2)[:dim // 32]
    v *= np.repeat(np.stack([2.0 ** (8 - apart), 2.0 ** (8 - apart[::-1])]), 32, 1).astype(np.float32)
    s = Step(engine, 2 * group, 2, dim, 16, [700], [tokens], seed=far, k=[k], v=[v])
    s.fill()
    check(s)


def scored(rng, past, tokens, dim, at, lead, group):
    """Keys and queries whose scores are near 0 but for those of positions `at`, which are near `lead`."""
    k, _ = plain(rng, past, tokens, dim)
    k *= 0.05
    q = rng.normal(size=(tokens, 2 * group, dim)).astype(np.float32) * 0.1
    q[..., :32] += 2.0
    k[..., :32] *= 0.1
    k[at] = 0
    k[at, :, :32] = lead / (2.0 * 32) * dim ** 0.5
    return q, k


@pytest.mark.parametrize("group,tokens,dim", SHAPES)
@pytest.mark.parametrize("far", [16, 18, 20, 30])
@pytest.mark.parametrize("at", [[0], [5], [350], [690], [0, 100, 101, 500], list(range(32, 64)), list(range(64, 400, 3))])
def test_large_values_that_hardly_count(engine, group, tokens, dim, far, at):
    """Values 2^far times as large as the others whose keys are e^-23 as probable: alone in a tile, side by side, in many tiles."""
    rng = np.random.default_rng(far)
    q, k = scored(rng, 700, tokens, dim, at, -23.0, group)
    _, v = plain(rng, 700, tokens, dim)
    v *= 2.0 ** -14
    v[at] *= np.float32(2.0 ** far)
    s = Step(engine, 2 * group, 2, dim, 32, [700], [tokens], seed=far, k=[k], v=[v])
    s.q = q
    s.fill()
    check(s)


@pytest.mark.parametrize("group,tokens,dim", SHAPES)
@pytest.mark.parametrize("value", [0.0, 2.0 ** -30, 2.0 ** -20, 2.0 ** -9])
@pytest.mark.parametrize("at", [0, 17, 690])
def test_a_key_with_nearly_all_the_weight_and_little_value(engine, group, tokens, dim, value, at):
    """What the others have is small beside it in weight alone. Once in all dims, once in one block of them."""
    rng = np.random.default_rng(at)
    q, k = scored(rng, 700, tokens, dim, [at], 16.0, group)
    _, v = plain(rng, 700, tokens, dim)
    v[at, 0] *= np.float32(value)
    v[at, 1, 32:64] *= np.float32(value)
    s = Step(engine, 2 * group, 2, dim, 32, [700], [tokens], seed=at, k=[k], v=[v])
    s.q = q
    s.fill()
    check(s)


@pytest.mark.parametrize("group,tokens,dim", SHAPES)
@pytest.mark.parametrize("value,noise", [(2.0 ** -5, 2.0 ** -18), (1.0, 2.0 ** -11), (2.0 ** -16, 0.0), (1.0, 0.0)])
def test_a_key_with_nearly_all_the_weight_and_a_value_that_hardly_varies(engine, group, tokens, dim, value, noise):
    """Steps far below those of the others beside a minimum that is not, and steps of 0."""
    rng = np.random.default_rng(9)
    q, k = scored(rng, 300, tokens, dim, [130], 16.0, group)
    _, v = plain(rng, 300, tokens, dim)
    v[130] = (value + noise * v[130]).astype(np.float32)
    s = Step(engine, 2 * group, 2, dim, 32, [300], [tokens], seed=9, k=[k], v=[v])
    s.q = q
    s.fill()
    check(s)


@pytest.mark.parametrize("group,tokens,dim", SHAPES)
@pytest.mark.parametrize("lift", [2.0 ** -20, 2.0 ** -16, 2.0 ** -13, 2.0 ** -11, 2.0 ** -9, 2.0 ** -7, 2.0 ** 15])
def test_steps_of_every_magnitude(engine, group, tokens, dim, lift):
    """Values 2^6 apart around a magnitude: the least and the largest steps half precision has, and those between."""
    rng = np.random.default_rng(4)
    k, v = plain(rng, 300, tokens, dim)
    v *= (lift * 2.0 ** rng.integers(-3, 4, (300 + tokens, 2, 1))).astype(np.float32)
    s = Step(engine, 2 * group, 2, dim, 32, [300], [tokens], seed=4, k=[k], v=[v])
    s.fill()
    check(s)


def test_values_that_are_all_zero_or_constant(engine):
    for value in (0.0, -3.5):
        rng = np.random.default_rng(2)
        k, v = plain(rng, 300, 1, 128)
        v[:] = value
        v[150:, 1, 64:] = rng.normal(size=(151, 64))
        s = Step(engine, 4, 2, 128, 16, [300], [1], k=[k], v=[v])
        s.fill()
        check(s)


def test_steps_at_the_ends_of_half_precision(engine):
    """Steps from the least subnormal number to the largest there is, within a block, from token to token and all at once."""
    rng = np.random.default_rng(3)
    for lift in (2.0 ** -22, 2.0 ** -15, 1.0, 2.0 ** 17):
        for wild in (0, 3, 12):
            k, v = plain(rng, 500, 1, 128)
            v *= (lift * 2.0 ** rng.integers(-wild, wild + 1, (501, 2, 1))).astype(np.float32)
            s = Step(engine, 4, 2, 128, 16, [500], [1], k=[k], v=[v])
            s.fill()
            check(s)


# ---- the same with many tiles a warp ---------------------------------------------------------------------------------------------------


def check_many(e, group, k, v, q, tokens, copies=300):
    """`copies` sequences over the same pages but for their last one (their new tokens), which all have the rows and queries of one: every warp goes through a
    dozen tiles and more, through the ends of sequences and their beginnings."""
    past, dim = len(k) - tokens, k.shape[-1]
    assert past % 16 == 0 and tokens <= 16
    shared = past // 16
    cache = e.kv4_cache(shared + copies, 16, 2, dim)
    batch = e.kv4_batch(cache, 2 * group, copies, max(past, copies * tokens), shared + 1)
    order = np.random.default_rng(0).permutation(shared + copies)
    tables = np.concatenate([np.tile(order[:shared], (copies, 1)), order[shared:, None]], 1)
    batch.set([0], [past], tables[:1])
    e.kv4_append(cache, batch, e.upload_f32(k[:past]), e.upload_f32(v[:past]))
    batch.set([past] * copies, [tokens] * copies, tables)
    e.kv4_append(cache, batch, *(e.upload_f32(np.tile(x[past:], (copies, 1, 1))) for x in (k, v)))
    out = e.alloc_f32(copies * q.size)
    e.kv4_attention(cache, batch, e.upload_f32(np.tile(q, (copies, 1, 1))), out, dim ** -0.5)
    got = e.read_f32(out).reshape(copies, *q.shape)
    kc, vc = ref.quantize(k.astype(np.float64)), ref.quantize(v.astype(np.float64))
    want, w = ref.attention(q.astype(np.float64), ref.values(*kc), ref.values(*vc), past, dim ** -0.5)
    tol = ref.rms_tolerance(q, q, np.zeros_like(q), kc, vc, w, past, dim ** -0.5)
    off = np.abs(got - want)
    assert (off <= tol).all(), f"worst {np.max(off / tol):.3g} of the tolerance, in {np.mean((off > tol).any((1, 2, 3))):.3g} of the sequences"
    batch.free()
    cache.free()


def ordinary(rng, tokens, group, dim):
    return rng.normal(size=(tokens, 2 * group, dim)).astype(np.float32)


MANY = [(1, 1, 64), (7, 1, 64), (4, 3, 64), (1, 1, 128), (4, 1, 128), (7, 1, 128), (4, 3, 128), (1, 1, 256), (7, 1, 256)]


@pytest.mark.parametrize("group,tokens,dim", MANY)
def test_many_ordinary(engine, group, tokens, dim):
    rng = np.random.default_rng(1)
    k, v = plain(rng, 704, tokens, dim)
    check_many(engine, group, k * np.float32(2), v, ordinary(rng, tokens, group, dim), tokens)


@pytest.mark.parametrize("group,tokens,dim", MANY)
def test_many_scores_that_rise_and_fall(engine, group, tokens, dim):
    """References that move up and down: by waves, by steps, at single keys."""
    n = 704 + tokens
    for shape in (np.linspace(0, 60, n), np.linspace(60, 0, n), 30 * np.sin(np.arange(n) / 40), np.where(np.arange(n) % 100 == 7, 25, 0), np.where(np.arange(n) // 150 % 2, 20, 0)):
        rng = np.random.default_rng(2)
        q, k = scored(rng, 704, tokens, dim, np.arange(n), shape[:, None, None].astype(np.float32), group)
        _, v = plain(rng, 704, tokens, dim)
        check_many(engine, group, k, v, q, tokens)


@pytest.mark.parametrize("group,tokens,dim", MANY)
@pytest.mark.parametrize("far", [8, 16, 30])
def test_many_blocks_of_a_head_far_apart(engine, group, tokens, dim, far):
    rng = np.random.default_rng(far)
    k, v = plain(rng, 704, tokens, dim)
    apart = np.array([0, far, far // 2, 2] * 2)[:dim // 32]
    v *= np.repeat(np.stack([2.0 ** (8 - apart), 2.0 ** (8 - apart[::-1])]), 32, 1).astype(np.float32)
    check_many(engine, group, k, v, ordinary(rng, tokens, group, dim), tokens)


@pytest.mark.parametrize("group,tokens,dim", MANY)
@pytest.mark.parametrize("far", [16, 20, 30])
@pytest.mark.parametrize("at", [[0], [350], [0, 100, 101, 500], list(range(32, 64)), list(range(64, 400, 3)), list(range(0, 704, 50))])
def test_many_large_values_that_hardly_count(engine, group, tokens, dim, far, at):
    rng = np.random.default_rng(far)
    q, k = scored(rng, 704, tokens, dim, at, -23.0, group)
    _, v = plain(rng, 704, tokens, dim)
    v *= 2.0 ** -14
    v[at] *= np.float32(2.0 ** far)
    check_many(engine, group, k, v, q, tokens)


@pytest.mark.parametrize("group,tokens,dim", MANY)
@pytest.mark.parametrize("value", [0.0, 2.0 ** -20, 2.0 ** -9, 2.0 ** -5])
@pytest.mark.parametrize("at", [[0], [17], [350], [0, 40, 300, 301]])
def test_many_keys_with_nearly_all_the_weight_and_little_value(engine, group, tokens, dim, value, at):
    rng = np.random.default_rng(5)
    q, k = scored(rng, 704, tokens, dim, at, 16.0, group)
    _, v = plain(rng, 704, tokens, dim)
    v[at, 0] *= np.float32(value)
    v[at, 1, 32:64] *= np.float32(value)
    check_many(engine, group, k, v, q, tokens)


@pytest.mark.parametrize("group,tokens,dim", MANY)
def test_many_tiles_of_every_magnitude(engine, group, tokens, dim):
    """Steps that grow, shrink and jump from tile to tile, over all that half precision has; zeros among them."""
    n = 704 + tokens
    tile = np.arange(n) // 16
    for e in (tile / 2 - 20, 2 - tile / 2, (tile * 7) % 29 - 18, np.where(tile % 5 == 0, 3, -12), np.where(np.arange(n) % 24 == 0, -np.inf, tile % 9)):
        rng = np.random.default_rng(6)
        k, v = plain(rng, 704, tokens, dim)
        v *= (2.0 ** e)[:, None, None].astype(np.float32)
        check_many(engine, group, k, v, ordinary(rng, tokens, group, dim), tokens)


@pytest.mark.parametrize("group,tokens,dim", MANY)
def test_many_least_steps_behind_steps_far_apart(engine, group, tokens, dim):
    """Odd blocks of 32 dims have steps of 2^-24 throughout; the others are zero but for the first two tiles of one, where they lie far apart."""
    rng = np.random.default_rng(7)
    k, v = plain(rng, 704, tokens, dim)
    k *= 0.1
    blocks = v.reshape(len(v), 2, dim // 32, 32)
    blocks[:, :, 1::2] = rng.integers(0, 16, blocks[:, :, 1::2].shape) * 2.0 ** -24
    blocks[:, :, 1::2, 0], blocks[:, :, 1::2, 1] = 0, 15 * 2.0 ** -24
    blocks[:, :, 0::2] = 0
    blocks[:32, :, 0 if dim == 64 else 2] = rng.normal(size=(32, 2, 32)) * np.where(np.arange(32) % 3 == 0, 2.0 ** -20, 1.0)[:, None, None]
    check_many(engine, group, k, v, ordinary(rng, tokens, group, dim), tokens)


# ---- jobs of 128 rows -------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("shape", ["flat", "up", "down", "waves", "peaks", "steps"])
def test_prompts_behind_long_contexts(engine, dim, shape):
    """Numbers of one magnitude, references that move up and stay: dozens of blocks of keys, several to a part of the keys."""
    group, tokens, past = 2, 24, 3000
    n = np.arange(past + tokens)
    rng = np.random.default_rng(8)
    if shape == "flat":
        k, v = plain(rng, past, tokens, dim)
        q = ordinary(rng, tokens, group, dim)
    else:
        lead = {"up": n / 60, "down": 50 - n / 60, "waves": 12 * np.sin(n / 90), "peaks": np.where(n % 400 == 7, 12, 0), "steps": np.where(n // 500 % 2, 8, 0)}[shape]
        q, k = scored(rng, past, tokens, dim, n, lead[:, None, None].astype(np.float32), group)
        _, v = plain(rng, past, tokens, dim)
    s = Step(engine, 2 * group, 2, dim, 64, [past], [tokens], seed=8, k=[k], v=[v])
    s.q = q
    s.fill()
    check(s)


@pytest.mark.parametrize("dim", [64, 128])
def test_prompts_with_blocks_of_a_head_far_apart(engine, dim):
    """Within what one power of two for 256 positions holds: steps 2^16 apart keep 22 bits less two."""
    group, tokens = 2, 24
    rng = np.random.default_rng(16)
    k, v = plain(rng, 700, tokens, dim)
    v *= np.repeat(2.0 ** -np.array([0, 16, 8, 2])[:dim // 32], 32)[None, None].astype(np.float32)
    s = Step(engine, 2 * group, 2, dim, 16, [700], [tokens], seed=16, k=[k], v=[v])
    s.fill()
    check(s)
