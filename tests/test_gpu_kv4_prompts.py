"""Attention of many new tokens over the 4-bit cache (jobs of 128 rows) against 64-bit numpy, at the bound of its roundings."""
import subprocess
import sys

import numpy as np
import pytest

import kv4_ref as ref
from alice_llm_b200 import _lib
from test_gpu_kv4 import Step

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def engine():
    from alice_llm_b200.gpu import GpuEngine
    e = GpuEngine()
    yield e
    e.close()


@pytest.mark.parametrize("heads,kv_heads,tokens", [(1, 1, 35), (2, 1, 64), (6, 2, 43), (5, 1, 26), (14, 2, 19), (8, 1, 16), (16, 1, 9), (40, 1, 4), (150, 1, 1), (9, 3, 100)])
@pytest.mark.parametrize("dim,rot,neox,page", [(64, 64, True, 16), (128, 128, False, 64), (128, 128, True, 48), (128, 32, True, 4096), (64, 16, False, 32), (128, 0, False, 16)])
def test_groups_and_rotations(engine, heads, kv_heads, tokens, dim, rot, neox, page):
    s = Step(engine, heads, kv_heads, dim, page, [37], [tokens], rot, neox, seed=heads + dim)
    s.fill()
    s.check()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("past", [0, 1, 15, 16, 47, 48, 63, 64, 191, 192, 215, 216, 217, 255, 256, 257, 1000, 3000])
def test_lengths(engine, dim, past):
    s = Step(engine, 4, 2, dim, 32, [past], [41], dim, True, seed=past)
    s.fill()
    s.check()


@pytest.mark.parametrize("tokens,past", [([40, 1, 0, 2, 70, 9], [10, 300, 5, 64, 500, 0]), ([1] * 20 + [33] * 3, list(range(0, 460, 20))), ([64, 64], [0, 1]), ([5, 4, 3], [700, 700, 700])])
def test_prompts_beside_single_tokens(engine, tokens, past):
    for dim in (64, 128):
        s = Step(engine, 8, 2, dim, 16, past, tokens, dim, False, seed=len(tokens))
        s.fill()
        s.check()


def test_scores_that_rise_and_fall(engine):
    """The reference of the weights moves at every block of keys, at the last one only, at some rows only, and not at all."""
    n = 700
    for shape in (np.linspace(0, 60, n), np.linspace(60, 0, n), np.where(np.arange(n) == 655, 50, 0), 30 * np.sin(np.arange(n) / 9)):
        s = Step(engine, 4, 2, 128, 64, [n - 40], [40], seed=3)
        s.k[0][:] *= 0.02
        s.k[0][:, 0, :] += (shape / 128 ** 0.5)[:, None].astype(np.float32)      # the other key head's scores stay where they are
        s.q[:, :2] = 1 + 0.01 * s.q[:, :2]
        s.fill()
        s.check()


def test_wide_ranges(engine):
    """Values and keys that differ by 2^16 from token to token and head to head, queries far from 1, scores far from 0."""
    rng = np.random.default_rng(1)
    past, t = 500, 40
    for scale, lift in ((0.1, 1.0), (2.0, 1e-4), (1e-3, 1e3)):
        v = [(rng.normal(size=(past + t, 2, 128)) * 2.0 ** rng.integers(-8, 8, (past + t, 2, 1)) * lift).astype(np.float32)]
        k = [(rng.normal(size=(past + t, 2, 128)) * 3).astype(np.float32)]
        s = Step(engine, 4, 2, 128, 16, [past], [t], k=k, v=v)
        s.fill()
        s.check(scale=scale)
        s.check(scale=scale / 1e3, q=s.q * np.float32(1e3))
        s.check(scale=scale * 1e6, q=s.q * np.float32(1e-6))
    k = [(rng.normal(size=(past + t, 2, 128)) * 2.0 ** rng.integers(-8, 8, (past + t, 2, 1))).astype(np.float32)]
    s = Step(engine, 4, 2, 128, 16, [past], [t], k=k)
    s.fill()
    s.check(scale=1e-3)


@pytest.mark.parametrize("dim", [64, 128])
def test_what_is_not_seen_has_no_part(engine, dim):
    """Infinities and NaN behind the positions that rows see change no bit of theirs where they lie behind the end, and make NaN what sees them."""
    n = 40
    s = Step(engine, 4, 2, dim, 32, [35, 20], [n, 1], dim, True, seed=2)
    s.fill()
    clean, (want, tol) = s.attend(), s.expect()
    bad = np.full((40, 2, dim), np.nan, np.float32)
    bad[::2] = np.inf
    s.append([(bad[:20], bad[:20]), (bad[:11], bad[:11])], [35 + n, 21], [20, 11])
    s.batch.set(s.past, s.tokens, s.tables)
    assert np.array_equal(s.attend(), clean)
    # a key of the 31st new token and a block of a value of the 11th position: seen by those from there on
    part = s.v[0][10:11].copy()
    part[0, 1, 40] = np.inf
    s.append([(bad[:1], s.v[0][65:66]), (bad[:0], bad[:0])], [65, 0], [1, 0])
    s.append([(s.k[0][10:11], part), (bad[:0], bad[:0])], [10, 0], [1, 0])
    s.batch.set(s.past, s.tokens, s.tables)
    got = s.attend()
    assert np.isnan(got[30:n]).all() and np.isnan(got[:n, 2:, 32:64]).all()
    rest = np.ones(got.shape, bool)
    rest[30:n] = rest[:n, 2:, 32:64] = False
    assert (np.abs(got - want) <= tol)[rest].all()
    s.append([(s.k[0][65:66], s.v[0][65:66]), (bad[:0], bad[:0])], [65, 0], [1, 0])
    s.append([(s.k[0][10:11], s.v[0][10:11]), (bad[:0], bad[:0])], [10, 0], [1, 0])
    s.batch.set(s.past, s.tokens, s.tables)
    q = s.q.copy()
    q[0, 1, 5], q[17, 2, 0] = np.nan, np.inf
    got = s.attend(q=q)
    assert np.isnan(got[0, 1]).all() and np.isnan(got[17, 2]).all()
    keep = np.ones(got.shape[:2], bool)
    keep[0, 1] = keep[17, 2] = False
    assert np.array_equal(got[keep], clean[keep])


def test_queries_of_zero_strides_and_rows_behind_the_last(engine):
    import torch
    s = Step(engine, 4, 2, 128, 16, [40], [33], seed=4)
    s.q[3] = 0
    s.fill()
    s.check()
    first = s.attend()
    assert all(np.array_equal(s.attend(), first) for _ in range(3))
    q = torch.full((33, 4 * 128 + 4), 9.0, device="cuda")
    q[:, :512] = torch.from_numpy(s.q.reshape(33, 512)).cuda()
    out = torch.full((36, 4 * 128 + 8), 7.0, device="cuda")
    torch.cuda.synchronize()
    engine.kv4_attention(s.cache, s.batch, engine.buf_from_device(q.data_ptr(), q.numel()), engine.buf_from_device(out.data_ptr(), out.numel()), 128 ** -0.5, q_stride=516, out_stride=520)
    engine.sync()
    got = out.cpu().numpy()
    assert np.array_equal(got[:33, :512].reshape(33, 4, 128), first) and (got[33:] == 7).all() and (got[:, 512:] == 7).all()


def test_a_part_of_the_keys_each(engine):
    """One job or few over long contexts (clusters share the keys), and more than the chip has room for at once."""
    for past, tokens, heads, kv_heads in (([9000], [20], 2, 1), ([4000, 90], [17, 30], 3, 1), ([130] * 100, [20] * 100, 6, 3)):
        s = Step(engine, heads, kv_heads, 128, 64, past, tokens, seed=len(past))
        s.fill()
        s.check()


def test_captured_prompts_follow_the_batch(engine):
    import torch
    from alice_llm_b200.gpu import GpuEngine
    e = GpuEngine()
    stream = torch.cuda.Stream()
    e.set_stream(stream.cuda_stream)
    s = Step(e, 8, 2, 64, 16, [30, 45], [40, 40], 64, True, seed=11)
    s.fill()
    want, tol = s.expect()
    qb, ob = e.upload_f32(s.q), e.alloc_f32(s.q.size)
    call = lambda: e.kv4_attention(s.cache, s.batch, qb, ob, 0.125, rope=s.rope, rot_dims=64, neox=True)
    call()
    e.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call()

    def replay():
        with torch.cuda.stream(stream):
            graph.replay()
        return e.read_f32(ob).reshape(s.q.shape)

    assert (np.abs(replay() - want) <= tol).all()
    s.batch.set([30, 45], [33, 0], s.tables)      # fewer jobs
    assert (np.abs(replay()[:33] - want[:33]) <= tol[:33]).all()
    s.batch.set([30, 45], [0, 0], s.tables)
    replay()
    e.sync()
    s.batch.set([0, 0], [70, 10], s.tables)       # as many (3 and 1), cut otherwise
    replay()
    e.sync()
    s.batch.set([30, 45], [33, 1], s.tables)      # a single token as well: another kernel
    replay()
    with pytest.raises(_lib.AliceError) as ei:
        e.sync()
    assert ei.value.code == _lib.E_KERNEL
    s.batch.set([30, 45], [33, 0], s.tables)
    small = torch.cuda.CUDAGraph()
    e.sync()
    with torch.cuda.graph(small, stream=stream):
        call()
    s.batch.set(s.past, s.tokens, s.tables)       # more jobs
    with torch.cuda.stream(stream):
        small.replay()
    with pytest.raises(_lib.AliceError) as ei:
        e.sync()
    assert ei.value.code == _lib.E_KERNEL
    del small
    s.batch.set(s.past, s.tokens, s.tables)
    assert (np.abs(replay() - want) <= tol).all()
    e.sync()
    del graph
    e.close()


def test_a_capture_of_an_empty_batch_follows_it_too(engine):
    import torch
    from alice_llm_b200.gpu import GpuEngine
    e = GpuEngine()
    stream = torch.cuda.Stream()
    e.set_stream(stream.cuda_stream)
    s = Step(e, 2, 1, 64, 16, [30], [1], seed=5)
    s.append([(s.k[0][:30], s.v[0][:30])], [0], [30])
    kb, vb, qb, ob = e.upload_f32(s.k[0][30:]), e.upload_f32(s.v[0][30:]), e.upload_f32(s.q), e.alloc_f32(s.q.size)
    s.batch.set([30], [0], s.tables)
    e.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        e.kv4_append(s.cache, s.batch, kb, vb)
        e.kv4_attention(s.cache, s.batch, qb, ob, 0.125)
    s.batch.set([30], [1], s.tables)
    with torch.cuda.stream(stream):
        graph.replay()
    got = e.read_f32(ob).reshape(s.q.shape)
    want, tol = s.expect()
    assert (np.abs(got - want) <= tol).all()
    e.sync()
    del graph
    e.close()


FIRST = """
import sys
sys.path[:0] = %r
import numpy as np, torch
from test_gpu_kv4 import Step
from alice_llm_b200.gpu import GpuEngine
e = GpuEngine()
stream = torch.cuda.Stream()
e.set_stream(stream.cuda_stream)
s = Step(e, 4, 1, 128, 16, [50], [12], seed=1)
s.fill()
q, o = e.upload_f32(s.q), e.alloc_f32(s.q.size)
e.sync()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=stream):
    e.kv4_attention(s.cache, s.batch, q, o, 128 ** -0.5)
with torch.cuda.stream(stream):
    graph.replay()
want, tol = s.expect()
assert (np.abs(e.read_f32(o).reshape(s.q.shape) - want) <= tol).all()
"""


def test_first_call_in_a_capture():
    done = subprocess.run([sys.executable, "-c", FIRST % [p for p in sys.path if p]], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stderr[-2000:]


def test_two_engines_at_once(engine):
    from alice_llm_b200.gpu import GpuEngine
    other = GpuEngine()
    a, b = (Step(e, 8, 2, 128, 64, [1000, 10], [50, 20], seed=i) for i, e in ((1, engine), (2, other)))
    a.fill(); b.fill()
    want = a.attend(), b.attend()
    outs = [(s, s.e.upload_f32(s.q), [s.e.alloc_f32(s.q.size) for _ in range(8)]) for s in (a, b)]
    for i in range(8):
        for s, q, o in outs:
            s.e.kv4_attention(s.cache, s.batch, q, o[i], 128 ** -0.5)
    for (s, _, o), w in zip(outs, want):
        for x in o:
            assert np.array_equal(s.e.read_f32(x).reshape(s.q.shape), w)
    other.close()


def test_a_capture_behind_few_positions_replayed_behind_many(engine):
    import torch
    from alice_llm_b200.gpu import GpuEngine
    e = GpuEngine()
    stream = torch.cuda.Stream()
    e.set_stream(stream.cuda_stream)
    s = Step(e, 20, 1, 128, 64, [3000], [2], seed=1)
    s.fill()
    want, tol = s.expect()
    q, o = e.upload_f32(s.q), e.alloc_f32(s.q.size)
    s.batch.set([3], [2], s.tables)
    e.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        e.kv4_attention(s.cache, s.batch, q, o, 128 ** -0.5)
    s.batch.set(s.past, s.tokens, s.tables)
    with torch.cuda.stream(stream):
        graph.replay()
    got = e.read_f32(o).reshape(s.q.shape)
    assert (np.abs(got - want) <= tol).all()
    e.sync()
    del graph
    e.close()
