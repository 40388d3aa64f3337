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
