"""The paged 4-bit key / value cache on the device against 64-bit numpy: codes to the bit, attention to the bound of its roundings."""
import numpy as np
import pytest

import kv4_ref as ref
from alice_llm_b200 import _lib

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def engine():
    from alice_llm_b200.gpu import GpuEngine
    e = GpuEngine()
    yield e
    e.close()


class Step:
    """A batch of sequences over one cache whose past has been filled in, with scattered pages."""

    def __init__(self, e, heads, kv_heads, dim, page, past, tokens, rot=0, neox=False, seed=0, k=None, v=None, spare=2):
        rng = np.random.default_rng(seed)
        self.e, self.heads, self.kv_heads, self.dim, self.past, self.tokens, self.rot, self.neox = e, heads, kv_heads, dim, past, tokens, rot, neox
        need = [-(-(p + t) // page) for p, t in zip(past, tokens)]
        pages = sum(need) + spare
        order = rng.permutation(pages).astype(np.uint32)
        self.tables = np.full((len(past), max(need + [1])), 2 ** 32 - 1, np.uint32)      # entries that are not needed name no page
        at = 0
        for s, n in enumerate(need):
            self.tables[s, :n] = order[at:at + n]
            at += n
        self.k = [rng.normal(size=(p + t, kv_heads, dim)).astype(np.float32) * (1 + 5 * (rng.random((kv_heads, dim)) < 0.05)).astype(np.float32) for p, t in zip(past, tokens)] if k is None else k
        self.v = [rng.normal(size=(p + t, kv_heads, dim)).astype(np.float32) for p, t in zip(past, tokens)] if v is None else v
        self.table = ref.rope(max([p + t for p, t in zip(past, tokens)]) + 64, rot) if rot else None
        self.rope = e.upload_f32(self.table) if rot else None
        self.cache = e.kv4_cache(max(pages, 1), page, kv_heads, dim)
        self.batch = e.kv4_batch(self.cache, heads, len(past), max(1, sum(p + t for p, t in zip(past, tokens))), self.tables.shape[1])
        self.q = rng.normal(size=(sum(tokens), heads, dim)).astype(np.float32)

    def turn(self, x, s):
        return ref.rotate(x, self.table, np.arange(len(x)), self.rot, self.neox)

    def append(self, rows, past, tokens):
        """rows: (k, v) of every sequence's new tokens."""
        self.batch.set(past, tokens, self.tables)
        k, v = (np.concatenate([np.asarray(r[i], np.float32).reshape(-1) for r in rows] + [np.zeros(0, np.float32)]) for i in (0, 1))
        self.e.kv4_append(self.cache, self.batch, self.e.upload_f32(k), self.e.upload_f32(v), rope=self.rope, rot_dims=self.rot, neox=self.neox)

    def fill(self):
        """The past in one step, the new tokens in another; leaves the batch at the new tokens."""
        self.append([(k[:p], v[:p]) for k, v, p in zip(self.k, self.v, self.past)], [0] * len(self.past), self.past)
        self.append([(k[p:], v[p:]) for k, v, p in zip(self.k, self.v, self.past)], self.past, self.tokens)

    def read(self, past, tokens):
        self.batch.set(past, tokens, self.tables)
        n = sum(tokens) * self.kv_heads * self.dim
        k, v = self.e.alloc_f32(n), self.e.alloc_f32(n)
        self.e.kv4_read(self.cache, self.batch, k, v)
        return [self.e.read_f32(x).reshape(-1, self.kv_heads, self.dim) for x in (k, v)]

    def attend(self, scale=None, q=None):
        out = self.e.alloc_f32(self.q.size)
        self.e.kv4_attention(self.cache, self.batch, self.e.upload_f32(self.q if q is None else q), out, scale or self.dim ** -0.5, rope=self.rope, rot_dims=self.rot, neox=self.neox)
        return self.e.read_f32(out).reshape(self.q.shape)

    def expect(self, scale=None, q=None):
        """(attention in 64 bits, how far f32 may be from it)."""
        scale, q = scale or self.dim ** -0.5, self.q if q is None else q
        outs, tols, at = [], [], 0
        for s, (p, t) in enumerate(zip(self.past, self.tokens)):
            kc, vc = ref.quantize(self.turn(self.k[s], s)), ref.quantize(self.v[s].astype(np.float64))
            raw = q[at:at + t]
            rows = ref.rotate(raw, self.table, p + np.arange(t), self.rot, self.neox)
            o, w = ref.attention(rows, ref.values(*kc), ref.values(*vc), p, scale)
            outs.append(o)
            tols.append(ref.tolerance(raw, ref.partners(raw, self.rot, self.neox), kc, vc, w, p, scale))
            at += t
        return np.concatenate(outs), np.concatenate(tols)

    def check(self, **kw):
        got, (want, tol) = self.attend(**kw), self.expect(**kw)
        off = np.abs(got - want)
        assert (off <= tol).all(), f"worst {np.max(off / tol):.3g} of the tolerance"


# ---- the cache ----------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dim,rot,neox", [(64, 0, False), (64, 64, True), (64, 32, False), (128, 128, False), (128, 128, True), (128, 64, True), (128, 16, True),
                                          (256, 256, True), (256, 128, False)])
@pytest.mark.parametrize("page", [16, 64])
def test_appended_rows_are_the_formulas_to_the_bit(engine, dim, rot, neox, page):
    s = Step(engine, 3, 3, dim, page, [0, 37, 100, 15], [1, 30, 5, 2], rot, neox, seed=dim + rot)
    s.fill()
    for past, tokens in ((s.past, s.tokens), ([0] * 4, s.past)):
        k, v = s.read(past, tokens)
        want_k = np.concatenate([ref.held(s.turn(x, i))[p:p + t] for i, (x, p, t) in enumerate(zip(s.k, past, tokens))])
        want_v = np.concatenate([ref.held(x.astype(np.float64))[p:p + t] for x, p, t in zip(s.v, past, tokens)])
        assert np.array_equal(k, want_k.astype(np.float32)) and np.array_equal(v, want_v.astype(np.float32))


def odd_rows(dim):
    """Rows on which a quantizer can go wrong: ties, constants, infinities, NaN, numbers at the ends of half precision and of f32."""
    rng = np.random.default_rng(5)
    rows = [np.arange(dim) % 31 / 2.0, np.zeros(dim), np.full(dim, -3.7), np.full(dim, 1e-9), rng.normal(size=dim) * 1e-6, rng.normal(size=dim) * 1e5,
            rng.normal(size=dim) * 1e38, np.where(np.arange(dim) == 40, np.inf, 1.0), np.where(np.arange(dim) == 1, -np.inf, rng.normal(size=dim)),
            np.where(np.arange(dim) == 33, np.nan, rng.normal(size=dim)), np.where(np.arange(dim) % 32 == 0, 65504.0, 65503.0), -np.arange(dim) * 1e3,
            np.where(np.arange(dim) % 2 == 0, 3.4e38, -3.4e38), rng.integers(-8, 8, dim) * 0.25, np.linspace(0, 2.0 ** -14, dim), np.full(dim, -0.0)]
    return np.array(rows, np.float32)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rot", [0, 32])
def test_odd_rows(engine, dim, rot):
    rows = odd_rows(dim)
    x = rows.reshape(len(rows), 1, dim)
    s = Step(engine, 1, 1, dim, 16, [0], [len(rows)], rot, True, k=[x], v=[x])
    s.append([(x, x)], [0], [len(rows)])
    k, v = s.read([0], [len(rows)])
    with np.errstate(invalid="ignore"):
        for got, want in ((k, ref.held(s.turn(x, 0))), (v, ref.held(x.astype(np.float64)))):
            assert np.array_equal(got, want.astype(np.float32), equal_nan=True)


def test_rows_with_strides_and_the_rest_left_alone(engine):
    """k and v as parts of one buffer of wider rows; pages and outputs that are not the batch's keep what they held."""
    e, kh, dim = engine, 2, 64
    s = Step(e, 2, kh, dim, 16, [3, 0], [4, 2], 64, False, seed=3)
    ones = np.ones((s.cache.pages * 16, kh, dim), np.float32)
    whole = e.kv4_batch(s.cache, 2, 1, len(ones), s.cache.pages)
    whole.set([0], [len(ones)], np.arange(s.cache.pages)[None])
    e.kv4_append(s.cache, whole, e.upload_f32(ones), e.upload_f32(ones))
    import torch
    ld = 3 * kh * dim
    rows = torch.randn(6, ld, device="cuda")
    k, v = (e.buf_from_device(rows[:, i * kh * dim:].data_ptr(), 5 * ld + kh * dim) for i in (1, 2))
    torch.cuda.synchronize()
    s.batch.set(s.past, s.tokens, s.tables)
    e.kv4_append(s.cache, s.batch, k, v, rope=s.rope, rot_dims=64, k_stride=ld, v_stride=ld)
    host = rows.cpu().numpy()
    raw_k, raw_v = host[:, kh * dim:2 * kh * dim].reshape(6, kh, dim), host[:, 2 * kh * dim:].reshape(6, kh, dim)
    pos = np.array([3, 4, 5, 6, 0, 1])
    want_k = ref.held(ref.rotate(raw_k, s.table, pos, 64, False)).astype(np.float32)
    want_v = ref.held(raw_v.astype(np.float64)).astype(np.float32)
    out = torch.full((7, ld), 5.0, device="cuda")
    torch.cuda.synchronize()
    ko, vo = (e.buf_from_device(out[:, i * kh * dim:].data_ptr(), 5 * ld + kh * dim) for i in (0, 2))
    e.kv4_read(s.cache, s.batch, ko, vo, k_stride=ld, v_stride=ld)
    e.sync()
    got = out.cpu().numpy()
    assert np.array_equal(got[:6, :kh * dim].reshape(6, kh, dim), want_k) and np.array_equal(got[:6, 2 * kh * dim:].reshape(6, kh, dim), want_v)
    assert (got[6] == 5).all() and (got[:, kh * dim:2 * kh * dim] == 5).all()
    n = ones.size
    ko, vo = e.alloc_f32(n), e.alloc_f32(n)
    e.kv4_read(s.cache, whole, ko, vo)
    flat = e.read_f32(ko).reshape(ones.shape), e.read_f32(vo).reshape(ones.shape)
    touched = [s.tables[0, 0] * 16 + p for p in (3, 4, 5, 6)] + [s.tables[1, 0] * 16 + p for p in (0, 1)]
    left = np.setdiff1d(np.arange(len(ones)), touched)
    assert all((f[left] == 1).all() for f in flat)
    assert np.array_equal(flat[0][touched], want_k) and np.array_equal(flat[1][touched], want_v)


# ---- attention ------------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 7, 8, 12, 16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_single_tokens(engine, group, dim):
    s = Step(engine, 2 * group, 2, dim, 32, [0, 1, 15, 16, 31, 200, 77], [1] * 7, dim, True, seed=group)
    s.fill()
    s.check()


@pytest.mark.parametrize("tokens", [[2], [5, 1, 3], [8] * 3, [17, 0, 33, 1], [0, 0], [130]])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 64), (8, 2, 128), (5, 1, 128), (6, 2, 256)])
def test_several_tokens(engine, tokens, heads, kv_heads, dim):
    past = [(37 * i + 11) % 90 for i in range(len(tokens))]
    s = Step(engine, heads, kv_heads, dim, 16, past, tokens, 32, False, seed=len(tokens))
    s.fill()
    s.check()


@pytest.mark.parametrize("dim,rot", [(64, 16), (64, 48), (128, 96), (128, 112), (256, 16), (256, 144), (256, 192), (256, 240), (256, 256)])
@pytest.mark.parametrize("neox", [False, True])
def test_parts_of_a_head_rotated(engine, dim, rot, neox):
    """Pairs whose halves lie with other lanes, and dims that are not rotated."""
    s = Step(engine, 6, 2, dim, 32, [37, 0, 5], [1, 1, 3], rot, neox, seed=rot)
    s.fill()
    s.check()


@pytest.mark.parametrize("page", [16, 48, 64, 4096])
@pytest.mark.parametrize("past", [2047, 5000])
def test_long_contexts(engine, past, page):
    s = Step(engine, 8, 2, 128, page, [past, 3, past // 3], [1, 1, 1], 128, False, seed=past)
    s.fill()
    s.check()


def test_one_sequence_over_many_ctas_and_many_over_one(engine):
    for past in ([20000], [5] * 300, [9000, 2, 2, 2]):
        s = Step(engine, 4, 1, 64, 64, past, [1] * len(past), seed=len(past))
        s.fill()
        s.check()


def test_a_key_that_stands_out(engine):
    """One key far above the rest, at the borders of tiles and pages: its value is the result."""
    past = 700
    for at in (0, 15, 16, 31, 32, 63, 64, 350, 688, 699, 700):
        s = Step(engine, 4, 2, 128, 32, [past], [1], seed=at)
        s.q[:] = 1.0
        s.k[0][:] *= 0.01
        s.k[0][at] = 9.0
        s.fill()
        got, held = s.attend(), ref.held(s.v[0].astype(np.float64))[at]
        # exp of the score's lead, 128 * 9 / sqrt(128) less what the others have, leaves nothing of the others in f32
        assert np.abs(got.reshape(2, 2, 128) - held[:, None]).max() <= 64 * 2.0 ** -22 * np.abs(s.v[0]).max()
        s.check()


def test_wide_ranges(engine):
    """Steps of values that differ by 2^20 from token to token and head to head, queries far from 1, scores far from 0."""
    for scale, lift in ((0.1, 1.0), (2.0, 1e-4), (1e-3, 3e4)):
        rng = np.random.default_rng(1)
        past = 400
        v = [(rng.normal(size=(past + 1, 2, 128)) * 2.0 ** rng.integers(-10, 10, (past + 1, 2, 1)) * lift).astype(np.float32)]
        k = [(rng.normal(size=(past + 1, 2, 128)) * 3).astype(np.float32)]
        s = Step(engine, 4, 2, 128, 16, [past], [1], k=k, v=v)
        s.fill()
        s.check(scale=scale)
        s.check(scale=scale / 1e3, q=s.q * np.float32(1e3))
        s.check(scale=scale * 1e6, q=s.q * np.float32(1e-6))


def test_what_is_not_seen_has_no_part(engine):
    """Infinities and NaN behind the positions a token sees, in its last tile and in pages it does not have, change no bit; what it sees
    of them makes it NaN."""
    s = Step(engine, 4, 2, 64, 32, [35, 20], [3, 1], 64, True, seed=2)
    s.fill()
    clean = s.attend()
    bad = np.full((40, 2, 64), np.nan, np.float32)
    bad[::2] = np.inf
    # positions behind the end, in the last page of each sequence
    s.append([(bad[:20], bad[:20]), (bad[:11], bad[:11])], [38, 21], [20, 11])
    s.batch.set(s.past, s.tokens, s.tables)
    assert np.array_equal(s.attend(), clean)
    # the last new token of the first sequence: seen by itself alone
    s.append([(bad[:1], s.v[0][37:38]), (bad[:0], bad[:0])], [37, 0], [1, 0])
    s.batch.set(s.past, s.tokens, s.tables)
    got = s.attend()
    assert np.array_equal(got[[0, 1, 3]], clean[[0, 1, 3]]) and np.isnan(got[2]).all()
    # a value's block: NaN in the dims of that block
    part = s.v[0][37:38].copy()
    part[0, 1, 40] = np.inf
    s.append([(s.k[0][37:38], part), (bad[:0], bad[:0])], [37, 0], [1, 0])
    s.batch.set(s.past, s.tokens, s.tables)
    got = s.attend()
    assert np.isnan(got[2, 2:, 32:]).all() and np.isfinite(got[2, :2]).all() and np.isfinite(got[2, 2:, :32]).all()
    q = s.q.copy()
    q[0, 1, 5], q[3, 2, 0] = np.nan, np.inf
    s.fill()
    got = s.attend(q=q)
    assert np.isnan(got[0, 1]).all() and np.isnan(got[3, 2]).all()
    keep = np.ones((4, 4), bool)
    keep[0, 1] = keep[3, 2] = False
    assert np.array_equal(got[keep], clean[keep])


def test_queries_of_zero_and_rows_behind_the_last(engine):
    s = Step(engine, 4, 2, 128, 16, [40, 7], [1, 1], seed=4)
    s.q[0] = 0
    s.fill()
    s.check()
    import torch
    out = torch.full((4, 4 * 128 + 8), 7.0, device="cuda")
    torch.cuda.synchronize()
    buf = engine.buf_from_device(out.data_ptr(), out.numel())
    engine.kv4_attention(s.cache, s.batch, engine.upload_f32(s.q), buf, 128 ** -0.5, out_stride=4 * 128 + 8)
    engine.sync()
    got = out.cpu().numpy()
    assert np.array_equal(got[:2, :512].reshape(2, 4, 128), s.attend()) and (got[2:] == 7).all() and (got[:, 512:] == 7).all()


def test_shared_prefix_pages(engine):
    """Two sequences over the same pages of a prefix answer as two with pages of their own."""
    s = Step(engine, 4, 2, 64, 16, [32, 32], [1, 1], 64, False, seed=6)
    s.k[1][:32], s.v[1][:32] = s.k[0][:32], s.v[0][:32]
    s.fill()
    want = s.attend()
    s.tables[1, :2] = s.tables[0, :2]
    s.batch.set(s.past, s.tokens, s.tables)
    assert np.array_equal(s.attend(), want)


def test_the_same_call_twice_gives_the_same_bits(engine):
    s = Step(engine, 8, 2, 128, 64, [3000, 70, 1500], [1, 1, 1], seed=7)
    s.fill()
    first = s.attend()
    for _ in range(5):
        assert np.array_equal(s.attend(), first)


def test_one_batch_for_several_layers(engine):
    """Caches of several layers in turn through one batch, as a model does, and a step behind the first."""
    e, heads, kh, dim = engine, 4, 2, 64
    steps = [Step(e, heads, kh, dim, 16, [50, 9], [1, 1], 64, True, seed=i) for i in range(3)]
    for s in steps:
        s.tables = steps[0].tables
        s.batch = steps[0].batch
        s.fill()
    outs = [s.attend() for s in steps]
    for s, o in zip(steps, outs):
        want, tol = s.expect()
        assert (np.abs(o - want) <= tol).all()


# ---- capture, streams ------------------------------------------------------------------------------------------------------------------


def test_captured_step_follows_the_batch(engine):
    """Append and attention captured once and replayed for further tokens of the sequences."""
    import torch
    from alice_llm_b200.gpu import GpuEngine
    e = GpuEngine()
    stream = torch.cuda.Stream()
    e.set_stream(stream.cuda_stream)
    s = Step(e, 4, 2, 64, 16, [30, 45], [12, 12], 64, True, seed=11)
    s.append([(k[:p], v[:p]) for k, v, p in zip(s.k, s.v, s.past)], [0, 0], s.past)
    kb, vb, qb, ob = (e.alloc_f32(n) for n in (2 * 2 * 64, 2 * 2 * 64, 2 * 4 * 64, 2 * 4 * 64))
    graph = None
    got = []
    for i in range(12):
        s.batch.set([p + i for p in s.past], [1, 1], s.tables)
        e.write_f32(kb, np.stack([k[p + i] for k, p in zip(s.k, s.past)]))
        e.write_f32(vb, np.stack([v[p + i] for v, p in zip(s.v, s.past)]))
        e.write_f32(qb, s.q[[i, 12 + i]])

        def calls():
            e.kv4_append(s.cache, s.batch, kb, vb, rope=s.rope, rot_dims=64, neox=True)
            e.kv4_attention(s.cache, s.batch, qb, ob, 0.125, rope=s.rope, rot_dims=64, neox=True)

        if i == 0:
            calls()
        elif graph is None:
            graph = torch.cuda.CUDAGraph()
            e.sync()
            with torch.cuda.graph(graph, stream=stream):
                calls()
                with pytest.raises(_lib.AliceError):
                    s.batch.set(s.past, [1, 1], s.tables)
        if i:
            with torch.cuda.stream(stream):
                graph.replay()
        got.append(e.read_f32(ob).reshape(2, 4, 64))
    e.sync()
    s.batch.set(s.past, s.tokens, s.tables)
    want, tol = s.expect()
    got = np.concatenate([np.stack([g[0] for g in got]), np.stack([g[1] for g in got])])
    assert (np.abs(got - want) <= tol).all()
    # a batch that wants other jobs than the captured kernel's is reported, not run
    s.batch.set(s.past, [4, 4], s.tables)
    with torch.cuda.stream(stream):
        graph.replay()
    with pytest.raises(_lib.AliceError) as ei:
        e.sync()
    assert ei.value.code == _lib.E_KERNEL
    e.sync()
    del graph
    e.close()


def test_two_engines_at_once(engine):
    """Two engines, each with a cache and a batch of its own, on streams of their own."""
    from alice_llm_b200.gpu import GpuEngine
    other = GpuEngine()
    a, b = (Step(e, 8, 2, 128, 64, [4000, 10], [1, 1], seed=i) for i, e in ((1, engine), (2, other)))
    a.fill(); b.fill()
    want = a.attend(), b.attend()
    outs = []
    for s in (a, b):
        outs.append((s, s.e.upload_f32(s.q), [s.e.alloc_f32(s.q.size) for _ in range(8)]))
    for i in range(8):
        for s, q, o in outs:
            s.e.kv4_attention(s.cache, s.batch, q, o[i], 128 ** -0.5)
    for (s, _, o), w in zip(outs, want):
        for x in o:
            assert np.array_equal(s.e.read_f32(x).reshape(s.q.shape), w)
    other.close()


# ---- refusals ----------------------------------------------------------------------------------------------------------------------------


def test_refusals(engine):
    e = engine
    E = _lib.AliceError

    def refused(code, f, *a, **k):
        with pytest.raises(E) as ei:
            f(*a, **k)
        assert ei.value.code == code

    for args in ((0, 16, 1, 64), (1, 0, 1, 64), (1, 8, 1, 64), (1, 20, 1, 64), (1, 8192, 1, 64), (1, 16, 0, 64), (1, 16, 1, 32), (1, 16, 1, 96), (1, 16, 1, 100),
                 (2 ** 31, 16, 1, 64)):
        refused(_lib.E_SHAPE, e.kv4_cache, *args)
    c = e.kv4_cache(4, 16, 2, 64)
    for args in ((3, 1, 1, 1), (0, 1, 1, 1), (2, 0, 1, 1), (2, 1, 0, 1), (2, 1, 1, 0), (2, 1, 2 ** 31, 1), (2, 2 ** 20, 1, 2 ** 20)):
        refused(_lib.E_SHAPE, e.kv4_batch, c, *args)
    b = e.kv4_batch(c, 4, 2, 8, 3)
    refused(_lib.E_INVALID, b.set, [0], [1], [[4]])
    refused(_lib.E_INVALID, b.set, [0, 0], [1, 1], [[1], [1]])
    refused(_lib.E_SHAPE, b.set, [0], [9], [[1]])
    b.set([5, 0], [2, 1], [[1], [2]])
    kv, q, out, rope = e.alloc_f32(3 * 128), e.alloc_f32(3 * 256), e.alloc_f32(3 * 256), e.alloc_f32(7 * 64)
    v2 = e.alloc_f32(3 * 128)
    small = e.alloc_f32(3 * 128 - 1)
    refused(_lib.E_SHAPE, e.kv4_append, c, b, small, kv)
    refused(_lib.E_SHAPE, e.kv4_append, c, b, kv, small)
    refused(_lib.E_SHAPE, e.kv4_append, c, b, kv, kv, k_stride=127)
    refused(_lib.E_SHAPE, e.kv4_append, c, b, kv, kv, k_stride=130)
    refused(_lib.E_SHAPE, e.kv4_append, c, b, kv, kv, k_stride=132)
    refused(_lib.E_SHAPE, e.kv4_append, c, b, kv, kv, rope=rope, rot_dims=24)
    refused(_lib.E_SHAPE, e.kv4_append, c, b, kv, kv, rope=rope, rot_dims=80)
    refused(_lib.E_SHAPE, e.kv4_append, c, b, kv, kv, rope=rope)
    refused(_lib.E_INVALID, e.kv4_append, c, b, kv, kv, rot_dims=64)
    refused(_lib.E_SHAPE, e.kv4_append, c, b, kv, kv, rope=e.alloc_f32(7 * 64 - 1), rot_dims=64)
    refused(_lib.E_INVALID, e.kv4_read, c, b, kv, kv)
    refused(_lib.E_SHAPE, e.kv4_attention, c, b, small, out, 1.0)
    refused(_lib.E_SHAPE, e.kv4_attention, c, b, q, small, 1.0)
    refused(_lib.E_INVALID, e.kv4_attention, c, b, q, q, 1.0)
    refused(_lib.E_INVALID, e.kv4_attention, c, b, q, out, float("nan"))
    refused(_lib.E_INVALID, e.kv4_attention, c, b, q, out, float("inf"))
    other = e.kv4_cache(4, 32, 2, 64)
    refused(_lib.E_SHAPE, e.kv4_attention, other, b, q, out, 1.0)
    fewer = e.kv4_cache(2, 16, 2, 64)
    refused(_lib.E_SHAPE, e.kv4_append, fewer, b, kv, v2)
    from alice_llm_b200.gpu import GpuEngine
    e2 = GpuEngine()
    refused(_lib.E_INVALID, e2.kv4_append, c, b, kv, v2)
    refused(_lib.E_INVALID, e.kv4_append, c, b, e2.alloc_f32(3 * 128), v2)
    refused(_lib.E_INVALID, e2.kv4_batch, c, 4, 1, 1, 1)
    e2.close()
    # what was refused has left the batch as it was
    e.kv4_append(c, b, kv, v2, rope=rope, rot_dims=64)
    e.kv4_attention(c, b, q, out, 1.0, rope=rope, rot_dims=64)
    e.sync()


def test_nothing_to_do(engine):
    """No sequences, or none with new tokens: calls that write nothing."""
    e = engine
    c = e.kv4_cache(2, 16, 1, 64)
    b = e.kv4_batch(c, 2, 2, 4, 1)
    x, y = e.upload_f32(np.full(64, 3.0)), e.upload_f32(np.full(128, 4.0))
    for args in ((), ([0, 5], [0, 0], [[0], [1]])):
        if args:
            b.set(*args)
        e.kv4_append(c, b, x, x)
        e.kv4_attention(c, b, x, y, 1.0)
    e.sync()
    assert (e.read_f32(y) == 4).all()


def test_handles_outlive_their_engine():
    from alice_llm_b200.gpu import GpuEngine
    e = GpuEngine()
    c = e.kv4_cache(2, 16, 1, 64)
    b = e.kv4_batch(c, 1, 1, 1, 1)
    e._children.clear()
    e.close()
    b.free()
    c.free()
