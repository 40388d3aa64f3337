"""What can be said of the 4-bit cache without a device: the format's error, and the batches that are refused."""
import numpy as np
import pytest

import kv4_ref as ref
from alice_llm_b200 import _lib
from alice_llm_b200.gpu import AliceError, kv4_batch_check

SIZES = dict(pages=10, page_tokens=16, max_seqs=4, max_tokens=64, max_pages=5)


def test_values_are_within_half_a_step():
    x = np.random.default_rng(0).normal(size=(50, 2, 64)) * 3
    c, d, m = ref.quantize(x)
    assert c.min() == 0 and c.max() == 15
    # half a step, and what rounding the minimum (up to 2^-12 of it) and the step (15 times 2^-12 of it, or half the least step of 2^-24) can add
    room = np.repeat(d / 2 + np.abs(m) * 2.0 ** -11 + 15 * d * 2.0 ** -11 + 15 * 2.0 ** -24, 32, -1)
    assert (np.abs(ref.values(c, d, m) - x) <= room).all()


@pytest.mark.parametrize("past,tokens,tables", [
    ([], [], np.zeros((0, 1))),
    ([0], [1], [[3]]),
    ([15], [1], [[9]]),
    ([15, 40], [2, 8], [[1, 2, 0], [4, 5, 6]]),
    ([0, 0], [0, 5], [[77, 77], [3, 99]]),              # nothing of a sequence without new tokens is looked at, nor entries past the need
    ([32, 32], [1, 1], [[7, 8, 1], [7, 8, 2]]),         # a shared prefix
    ([64], [16], [[0, 1, 2, 3, 4]]),
])
def test_batches_that_are_taken(past, tokens, tables):
    kv4_batch_check(**SIZES, past=past, tokens=tokens, tables=tables)


@pytest.mark.parametrize("past,tokens,tables,code", [
    ([0] * 5, [1] * 5, [[p] for p in range(5)], _lib.E_SHAPE),               # more sequences than the batch has room for
    ([0, 0], [33, 32], [[0, 1, 2], [3, 4, 5]], _lib.E_SHAPE),                # more tokens
    ([80], [1], [[0, 1, 2, 3, 4, 5]], _lib.E_SHAPE),                         # more pages
    ([16], [1], [[0]], _lib.E_SHAPE),                                        # a table that is too short
    ([0], [1], [[10]], _lib.E_INVALID),                                      # no such page
    ([20], [1], [[11, 3]], _lib.E_INVALID),                                  # among those that are read
    ([3, 5], [1, 1], [[4], [4]], _lib.E_INVALID),                            # written by two sequences
    ([16], [20], [[0, 4, 4]], _lib.E_INVALID),                               # twice by one
    ([2 ** 31 - 1], [1], [[0, 1, 2, 3, 4]], _lib.E_SHAPE),
    ([2 ** 32 - 1], [2 ** 32 - 1], [[0, 1, 2, 3, 4]], _lib.E_SHAPE),
    ([0], [1], [[2 ** 32 - 1]], _lib.E_INVALID),
    ([0, 1], [1], [[1]], _lib.E_SHAPE),                                      # arrays of different batches
    ([0], [1], [1], _lib.E_SHAPE),
])
def test_batches_that_are_refused(past, tokens, tables, code):
    with pytest.raises(AliceError) as ei:
        kv4_batch_check(**SIZES, past=past, tokens=tokens, tables=tables)
    assert ei.value.code == code


def test_null_handles_are_refused():
    lib = _lib.load()
    assert lib.alice_kv4_create(None, 1, 16, 1, 64, None) == _lib.E_INVALID
    assert lib.alice_kv4_batch_create(None, None, 1, 1, 1, 1, None) == _lib.E_INVALID
    assert lib.alice_kv4_batch_set(None, 0, None, None, None, 0) == _lib.E_INVALID
    assert lib.alice_kv4_append(None, None, None, None, 0, None, 0, None, 0, 0) == _lib.E_INVALID
    assert lib.alice_kv4_read(None, None, None, None, 0, None, 0) == _lib.E_INVALID
    assert lib.alice_kv4_attention(None, None, None, None, 0, None, 0, None, 0, 0, 1.0) == _lib.E_INVALID
    assert lib.alice_log_probs(None, None, 1, 1, 0, None, None, None, None, 0, None, None) == _lib.E_INVALID
    assert lib.alice_kv4_free(None) == 0 and lib.alice_kv4_batch_free(None) == 0
    assert lib.alice_kv4_batch_check(1, 16, 1, 1, 1, 1, None, None, None, 1) == _lib.E_INVALID
    assert lib.alice_kv4_batch_check(1, 0, 1, 1, 1, 0, None, None, None, 1) == _lib.E_SHAPE
