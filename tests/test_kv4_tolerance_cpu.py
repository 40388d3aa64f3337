"""What the tolerances of the attention over the 4-bit cache can tell apart: operands as pairs of half-precision numbers pass, single ones do not."""
import numpy as np
import pytest

import kv4_ref as ref


def rows(past, group, dim, blocks=None, seed=0):
    """(q, cache of keys, of values) of one token with `group` heads over one key head; blocks: a factor for each 32 dims of the values."""
    rng = np.random.default_rng(seed)
    k = rng.normal(size=(past + 1, 1, dim)) * (1 + 5 * (rng.random(dim) < 0.05))
    v = rng.normal(size=(past + 1, 1, dim))
    if blocks is not None:
        v *= np.repeat(blocks, 32)
    return rng.normal(size=(1, group, dim)), ref.quantize(k), ref.quantize(v)


def worst(q, kc, vc, past, **how):
    scale = q.shape[-1] ** -0.5
    want, w = ref.attention(q, ref.values(*kc), ref.values(*vc), past, scale)
    tol = ref.rms_tolerance(q, q, np.zeros_like(q), kc, vc, w, past, scale)
    return np.max(np.abs(ref.attention_in_halves(q, kc, vc, past, scale, **how) - want) / tol), np.median(tol / np.abs(want))


@pytest.mark.parametrize("past", [76, 700, 5000, 20000])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_pairs_pass_and_halves_do_not(past, dim):
    q, kc, vc = rows(past, 4, dim, seed=past + dim)
    got, share = worst(q, kc, vc, past)
    assert got < 0.25                                  # the rest of the room is for f32 and the sums, which this has in 64 bits
    assert share < 1e-3
    assert worst(q, kc, vc, past, q_parts=1)[0] > 2
    assert worst(q, kc, vc, past, w_parts=1)[0] > 2


@pytest.mark.parametrize("far", [16, 18, 20])
def test_one_power_of_two_for_all_blocks_does_not_pass_where_blocks_are_apart(far):
    q, kc, vc = rows(700, 4, 128, blocks=2.0 ** -np.array([0, far, far / 2, 4]), seed=far)
    assert worst(q, kc, vc, 700)[0] < 0.25
    assert worst(q, kc, vc, 700, by_block=False)[0] > 4
