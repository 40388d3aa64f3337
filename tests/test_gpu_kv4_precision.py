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
