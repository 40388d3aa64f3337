"""Calls whose rows would leave their buffers or meet one another there are refused before anything runs."""
import numpy as np
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


def cache(e, tokens=8, heads=4, kv_heads=2, dim=64):
    c = e.kv4_cache(2, 16, kv_heads, dim)
    return c, e.kv4_batch(c, heads, 1, tokens, 2)


def test_reads_into_rows_that_meet(engine):
    """Keys and values of two wider rows each that lie partly over one another; side by side in one buffer of rows they do not."""
    import torch
    e, w = engine, 128
    c, b = cache(e)
    b.set([0], [2], [[0, 1]])
    x = torch.zeros(8 * w, device="cuda")
    torch.cuda.synchronize()
    at = lambda o: e.buf_from_device(x[o:].data_ptr(), 8 * w - o)
    for off in (4, w // 2, w - 4, 3 * w - 4, 2 * w + 4):
        refused(_lib.E_INVALID, e.kv4_read, c, b, at(0), at(off), k_stride=2 * w, v_stride=2 * w)
        refused(_lib.E_INVALID, e.kv4_read, c, b, at(off), at(0), k_stride=2 * w, v_stride=2 * w)
    refused(_lib.E_INVALID, e.kv4_read, c, b, at(0), at(2 * w), k_stride=2 * w, v_stride=w)
    for off in (w, 3 * w):
        e.kv4_read(c, b, at(0), at(off), k_stride=2 * w, v_stride=2 * w)
        e.kv4_read(c, b, at(off), at(0), k_stride=2 * w, v_stride=2 * w)
    e.kv4_read(c, b, at(0), at(3 * w), k_stride=2 * w, v_stride=w)
    e.sync()


def test_queries_and_outputs_in_one_buffer(engine):
    """Side by side in wider rows they are taken, and give what buffers of their own give; partly over one another they are not."""
    import torch
    e, w, n = engine, 256, 3
    c, b = cache(e)
    b.set([0], [8], [[0, 1]])
    rng = np.random.default_rng(0)
    e.kv4_append(c, b, *(e.upload_f32(rng.normal(size=8 * 128)) for _ in range(2)))
    b.set([5], [n], [[0, 1]])
    q = rng.normal(size=(n, w)).astype(np.float32)
    out = e.alloc_f32(n * w)
    e.kv4_attention(c, b, e.upload_f32(q), out, 0.125)
    want = e.read_f32(out).reshape(n, w)
    x = torch.full((3 * n, 2 * w + 4), 7.0, device="cuda")      # room for outputs that begin rows behind the queries
    x[:n, :w] = torch.from_numpy(q).cuda()
    torch.cuda.synchronize()
    flat = x.view(-1)
    at = lambda o: e.buf_from_device(flat[o:].data_ptr(), flat.numel() - o)
    ld = 2 * w + 4
    for off in (0, 4, w - 4, w + 8, ld, 2 * ld):
        refused(_lib.E_INVALID, e.kv4_attention, c, b, at(0), at(off), 0.125, q_stride=ld, out_stride=ld)
    e.kv4_attention(c, b, at(0), at(w + 4), 0.125, q_stride=ld, out_stride=ld)
    e.sync()
    got = x.cpu().numpy()
    assert np.array_equal(got[:n, w + 4:], want) and np.array_equal(got[:n, :w], q) and (got[:n, w:w + 4] == 7).all() and (got[n:] == 7).all()


@pytest.mark.parametrize("first", [0, 1])
def test_a_replay_with_more_tokens_than_lie_apart_does_nothing(first):
    """Captured with no or one new token; outputs begin a row behind the queries, where a second query would lie."""
    import torch
    from alice_llm_b200.gpu import GpuEngine
    e, w = GpuEngine(), 256
    stream = torch.cuda.Stream()
    e.set_stream(stream.cuda_stream)
    c, b = cache(e)
    rng = np.random.default_rng(1)
    b.set([0], [8], [[0, 1]])
    e.kv4_append(c, b, *(e.upload_f32(rng.normal(size=8 * 128)) for _ in range(2)))
    x = torch.full((6 * w,), 7.0, device="cuda")
    x[:w] = torch.from_numpy(rng.normal(size=w).astype(np.float32)).cuda()
    torch.cuda.synchronize()
    before = x.cpu().numpy()
    kv = torch.full((6 * 128,), 5.0, device="cuda")
    torch.cuda.synchronize()
    at = lambda t, o: e.buf_from_device(t[o:].data_ptr(), t.numel() - o)
    q, out, k, v = at(x, 0), at(x, w), at(kv, 0), at(kv, 128)
    b.set([7], [first], [[0, 1]])
    e.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        e.kv4_attention(c, b, q, out, 0.125)
    read = torch.cuda.CUDAGraph()
    with torch.cuda.graph(read, stream=stream):
        e.kv4_read(c, b, k, v)
    for g, t, start in ((graph, x, before), (read, kv, np.full(6 * 128, 5, np.float32))):
        b.set([6], [2], [[0, 1]])
        with torch.cuda.stream(stream):
            g.replay()
        with pytest.raises(_lib.AliceError) as ei:
            e.sync()
        assert ei.value.code == _lib.E_KERNEL and np.array_equal(t.cpu().numpy(), start)
        b.set([7], [1], [[0, 1]])
        with torch.cuda.stream(stream):
            g.replay()
        e.sync()
        now = t.cpu().numpy()
        n = w if t is x else 128
        assert (now[n:2 * n] != start[n:2 * n]).all() and (now[2 * n:] == start[2 * n:]).all()
    del graph, read
    e.close()
