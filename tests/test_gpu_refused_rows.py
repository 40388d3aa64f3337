"""Calls whose rows would leave their buffers or meet one another there are refused before anything runs."""
import pytest

from alice_llm_b200 import _lib

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def engine():
    from alice_llm_b200.gpu import GpuEngine
    e = GpuEngine()
    yield e
    e.close()


def refused(code, f, *a, **k):
    with pytest.raises(_lib.AliceError) as ei:
        f(*a, **k)
    assert ei.value.code == code


@pytest.mark.parametrize("rows,stride", [(2 ** 24 + 1, 2 ** 40), (2 ** 25 + 1, 2 ** 40), (2 ** 24 + 1, 2 ** 40 - 1), (2, 2 ** 40), (2, 101)])
def test_logits_that_need_more_words_than_64_bits_count(engine, rows, stride):
    """(rows - 1) * stride is a multiple of 2^64 for the first two: a buffer of one row is not enough for them."""
    e = engine
    x, ent = e.alloc_f32(100), e.alloc_f32(2 ** 25 + 1)
    refused(_lib.E_SHAPE, e.log_probs, x, rows, 100, None, None, entropy=ent, stride=stride)
