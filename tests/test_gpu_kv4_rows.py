"""Rows into and out of the 4-bit cache where a warp takes many heads one after the other, blocks of every kind among them, to the bit."""
import numpy as np
import pytest

import kv4_ref as ref
from test_gpu_kv4 import Step, odd_rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def engine():
    from alice_llm_b200.gpu import GpuEngine
    e = GpuEngine()
    yield e
    e.close()


@pytest.mark.parametrize("dim,kv_heads,tokens,rot,neox", [(64, 8, 2500, 64, True), (128, 8, 2500, 128, False), (128, 5, 3100, 32, True), (256, 3, 2000, 256, True), (256, 8, 700, 128, False),
                                                          (64, 13, 1900, 16, False)])
def test_many_tokens_of_many_heads(engine, dim, kv_heads, tokens, rot, neox):
    """One in three rows is one on which a quantizer can go wrong: ties, constants, infinities, NaN, the ends of half precision and of f32; the others are ordinary, of
    every magnitude."""
    rng = np.random.default_rng(dim + kv_heads)
    odd = odd_rows(dim)
    x = [(rng.normal(size=(tokens, kv_heads, dim)) * 10.0 ** rng.integers(-6, 5, (tokens, kv_heads, 1))).astype(np.float32) for _ in range(2)]
    for y in x:
        at = rng.random((tokens, kv_heads)) < 1 / 3
        y[at] = odd[rng.integers(0, len(odd), at.sum())]
    s = Step(engine, kv_heads, kv_heads, dim, 64, [0], [tokens], rot, neox, k=[x[0]], v=[x[1]])
    s.append([(x[0], x[1])], [0], [tokens])
    k, v = s.read([0], [tokens])
    with np.errstate(invalid="ignore", over="ignore"):
        for got, want in ((k, ref.held(s.turn(x[0], 0))), (v, ref.held(x[1].astype(np.float64)))):
            assert np.array_equal(got, want.astype(np.float32), equal_nan=True)
