"""Log probabilities, entropy, rank and alternatives of rows of logits against 64-bit numpy."""
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


def run(e, x, target, top, stride=0, words=None):
    n, v = x.shape
    buf = e.upload_f32(x) if words is None else words
    lp, ent, rank = e.alloc_f32(n), e.alloc_f32(n), e.alloc_f32(n)
    ids, tlp = (e.alloc_f32(n * top), e.alloc_f32(n * top)) if top else (None, None)
    e.log_probs(buf, n, v, e.upload_u32(target), lp, entropy=ent, rank=rank, top=top, top_ids=ids, top_log_probs=tlp, stride=stride)
    return (e.read_f32(lp), e.read_f32(ent), e.read_u32(rank).astype(np.int64), e.read_u32(ids).reshape(n, top).astype(np.int64) if top else None,
            e.read_f32(tlp).reshape(n, top) if top else None)


def check(e, x, target, top, **kw):
    """Against 64 bits. A difference x - m is rounded once (2^-24 of it) and its exponential is off by that and by less than 2^-22; sums of
    them lose 2^-24 a step, and a thread, warp and CTA adds up fewer than vocab / 256 + 300 in a chain. f32 has no numbers
    below 2^-149 and whole ones from 2^-126 on: each exponential may be off by that much besides (and its product with z by |z| times as much)."""
    lp, ent, rank, ids, tlp = run(e, x, target, top, **kw)
    n, v = x.shape
    xd = x.astype(np.float64)
    m = xd.max(1, keepdims=True)
    z = xd - m
    at = xd.argmax(1)
    w = np.exp(z)
    w[np.arange(n), at] = 0
    s = w.sum(1)
    zs = np.where(z > -np.inf, z, 0.0)
    with np.errstate(invalid="ignore"):
        tilt = (w * zs).sum(1)
    unit = 2.0 ** -24
    chain = (v / 256 + 300) * unit
    off_s = (chain * s + unit * (w * np.abs(zs)).sum(1)) / (1 + s) + v * 2.0 ** -126
    tol_l = off_s + 4 * unit * np.log1p(s)
    want = z[np.arange(n), target] - np.log1p(s)
    tol = tol_l + 4 * unit * np.abs(np.where(np.isfinite(want), want, 0)) + 4 * unit * np.abs(zs[np.arange(n), target])
    ok = np.isfinite(want)
    assert np.array_equal(lp[~ok], want[~ok])
    assert (np.abs(lp - want)[ok] <= tol[ok]).all(), np.max((np.abs(lp - want) / tol)[ok])
    h = np.log1p(s) - tilt / (1 + s)
    off_t = (chain * np.abs(tilt) + unit * (w * zs * zs).sum(1)) / (1 + s) + np.abs(tilt) / (1 + s) * (off_s + 4 * unit) + 200 * v * 2.0 ** -126
    assert (np.abs(ent - h) <= tol_l + off_t + 4 * unit * h).all(), np.max(np.abs(ent - h) / (tol_l + off_t + 4 * unit * h))
    assert np.array_equal(rank, (x > x[np.arange(n), target][:, None]).sum(1) + 1)
    if top:
        order = np.argsort(-xd, axis=1, kind="stable")[:, :top]
        assert np.array_equal(ids, order)
        want = np.take_along_axis(z, order, 1) - np.log1p(s)[:, None]
        ok = np.isfinite(want)
        tol = tol_l[:, None] + 8 * unit * np.abs(np.where(ok, want, 0)) + 8 * unit * np.log1p(s)[:, None]
        assert np.array_equal(tlp[~ok], want[~ok]) and (np.abs(tlp - want)[ok] <= tol[ok]).all()


@pytest.mark.parametrize("vocab", [1, 2, 3, 31, 32, 255, 1000, 4095, 4096, 8191, 8193, 16385, 50257])
@pytest.mark.parametrize("rows", [1, 3, 40])
def test_rows(engine, vocab, rows):
    rng = np.random.default_rng(vocab + rows)
    x = (rng.normal(size=(rows, vocab)) * 3).astype(np.float32)
    for top in sorted({0, min(1, vocab), min(5, vocab), min(32, vocab)}):
        check(engine, x, rng.integers(0, vocab, rows), top)


@pytest.mark.parametrize("rows,vocab,top", [(1, 128256, 20), (8, 128256, 5), (500, 32000, 3), (2, 400003, 32)])
def test_large(engine, rows, vocab, top):
    rng = np.random.default_rng(rows)
    x = (rng.normal(size=(rows, vocab)) * 2).astype(np.float32)
    x[:, 77] += 14
    check(engine, x, np.where(rng.random(rows) < 0.5, 77, rng.integers(0, vocab, rows)), top)


def test_one_token_has_nearly_everything(engine):
    """What the others have is small beside 1 and still there."""
    x = np.full((6, 3000), -20.0, np.float32)
    for r, lead in enumerate((5.0, 12.0, 25.0, 60.0, 90.0, 130.0)):
        x[r, 100 + r] += lead
    check(engine, x, 100 + np.arange(6), 4)
    lp = run(engine, x, 100 + np.arange(6), 0)[0]
    assert lp[2] < 0 and lp[3] < 0          # -2999 exp(-25), exp(-60): not rounded away


def test_ties_go_to_the_lowest_index(engine):
    rng = np.random.default_rng(3)
    x = rng.integers(-2, 3, (7, 9001)).astype(np.float32)
    x[1] = 0.5
    x[2] = -0.0
    x[2, ::2] = 0.0
    x[3, :] = -1e30
    check(engine, x, rng.integers(0, 9001, 7), 32)
    x = np.sort(x, 1)
    check(engine, x, rng.integers(0, 9001, 7), 32)
    check(engine, np.ascontiguousarray(x[:, ::-1]), rng.integers(0, 9001, 7), 32)


@pytest.mark.parametrize("top", [1, 7, 32])
def test_logits_that_keep_rising(engine, top):
    """Every logit is above all before it: a list of what exceeds an earlier bound would not end. Rows enough that a CTA has many rounds of one."""
    x = np.arange(60001, dtype=np.float32)[None] * np.linspace(1e-4, 1e-3, 200, dtype=np.float32)[:, None]
    x[1::3] = np.floor(x[1::3] * 4) / 4
    x[2::3] = x[2::3, ::-1]
    check(engine, x, np.arange(200) * 300, top)


def test_tokens_that_are_ruled_out(engine):
    rng = np.random.default_rng(4)
    x = (rng.normal(size=(5, 6000)) * 4).astype(np.float32)
    x[0, 1:] = -np.inf                       # one token is left
    x[1, rng.random(6000) < 0.99] = -np.inf
    x[2, 40:] = -np.inf
    x[3, :5990] = -np.inf
    x[4, 7] = np.finfo(np.float32).min
    target = np.array([0, int(np.argmax(x[1])), 5000, 5999, 7])
    check(engine, x, target, 32)
    lp, ent, rank, ids, tlp = run(engine, x, target, 32)
    assert lp[0] == 0 and ent[0] == 0 and rank[2] == 41 and lp[2] == -np.inf
    assert list(ids[0][:3]) == [0, 1, 2] and (tlp[0, 1:] == -np.inf).all()


def test_far_logits(engine):
    rng = np.random.default_rng(5)
    for k in (1e4, 1e30, 3e38):
        check(engine, ((rng.random((3, 5000)) - 0.5) * k).astype(np.float32), rng.integers(0, 5000, 3), 8)
    check(engine, (rng.normal(size=(3, 5000)) * 1e-30).astype(np.float32), rng.integers(0, 5000, 3), 8)


def test_rows_that_say_nothing(engine):
    rng = np.random.default_rng(6)
    x = rng.normal(size=(6, 10000)).astype(np.float32)
    x[0, 9999], x[1, 0], x[2, 5000] = np.nan, np.inf, -np.nan
    x[3] = -np.inf
    lp, ent, rank, ids, tlp = run(engine, x, np.array([1, 0, 3, 4, 10000, 2 ** 32 - 1]), 3)
    assert np.isnan(lp).all() and np.isnan(ent[:4]).all() and (rank == 0).all()
    assert (ids[:4] == 2 ** 32 - 1).all() and np.isnan(tlp[:4]).all()
    # a target that is no token leaves the rest of its row
    assert np.isfinite(ent[4:]).all() and np.isfinite(tlp[4:]).all()
    order = np.argsort(-x[4:].astype(np.float64), axis=1, kind="stable")[:, :3]
    assert np.array_equal(ids[4:], order)


def test_strides_offsets_and_outputs_left_out(engine):
    import torch
    e = engine
    rng = np.random.default_rng(7)
    wide = (rng.normal(size=(9, 1003)) * 2).astype(np.float32)
    wide[:, 900:] = 1e9                     # past the rows: not looked at
    dev = torch.from_numpy(wide).cuda()
    torch.cuda.synchronize()
    x = np.ascontiguousarray(wide[:, :900])
    words = e.buf_from_device(dev.data_ptr(), 8 * 1003 + 900)
    check(e, x, rng.integers(0, 900, 9), 6, stride=1003, words=words)
    t, lp, ent = rng.integers(0, 900, 9), e.alloc_f32(9), e.alloc_f32(9)
    full = run(e, x, t, 4)
    buf = e.upload_f32(x)
    e.log_probs(buf, 9, 900, e.upload_u32(t), lp)
    assert np.array_equal(e.read_f32(lp), full[0])
    e.log_probs(buf, 9, 900, None, None, entropy=ent)
    assert np.array_equal(e.read_f32(ent), full[1])
    ids, tlp = e.alloc_f32(36), e.alloc_f32(36)
    e.log_probs(buf, 9, 900, None, None, top=4, top_ids=ids, top_log_probs=tlp)
    assert np.array_equal(e.read_u32(ids).reshape(9, 4), full[3]) and np.array_equal(e.read_f32(tlp).reshape(9, 4), full[4])
    # rows behind the last keep what they held
    more = e.upload_f32(np.full(12, 3.0))
    e.log_probs(buf, 9, 900, e.upload_u32(t), more)
    assert (e.read_f32(more)[9:] == 3).all()
    e.log_probs(buf, 0, 900, e.upload_u32(t), more)
    assert np.array_equal(e.read_f32(more)[:9], full[0])


def test_the_same_rows_give_the_same_bits_alone_and_replayed(engine):
    import torch
    from alice_llm_b200.gpu import GpuEngine
    e = GpuEngine()
    stream = torch.cuda.Stream()
    e.set_stream(stream.cuda_stream)
    rng = np.random.default_rng(8)
    x = (rng.normal(size=(4, 20001)) * 3).astype(np.float32)
    t = rng.integers(0, 20001, 4)
    first = run(e, x, t, 7)
    xb, tb, lp, ent, rank, ids, tlp = e.upload_f32(x), e.upload_u32(t), *(e.alloc_f32(n) for n in (4, 4, 4, 28, 28))
    e.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        e.log_probs(xb, 4, 20001, tb, lp, entropy=ent, rank=rank, top=7, top_ids=ids, top_log_probs=tlp)
    for _ in range(3):
        with torch.cuda.stream(stream):
            graph.replay()
        assert np.array_equal(e.read_f32(lp), first[0]) and np.array_equal(e.read_f32(ent), first[1])
        assert np.array_equal(e.read_u32(ids).reshape(4, 7), first[3]) and np.array_equal(e.read_f32(tlp).reshape(4, 7), first[4])
    y = x[::-1].copy()
    e.write_f32(xb, y)
    e.write_f32(tb, np.ascontiguousarray(t[::-1], np.uint32).view(np.float32))
    with torch.cuda.stream(stream):
        graph.replay()
    assert np.array_equal(e.read_f32(lp), first[0][::-1])
    del graph
    e.close()


def test_refusals(engine):
    e = engine
    x, t, lp = e.alloc_f32(300), e.upload_u32([1, 2, 3]), e.alloc_f32(3)
    ids, tlp = e.alloc_f32(15), e.alloc_f32(15)

    def refused(code, *a, **k):
        with pytest.raises(_lib.AliceError) as ei:
            e.log_probs(*a, **k)
        assert ei.value.code == code

    refused(_lib.E_SHAPE, x, 3, 0, t, lp)
    refused(_lib.E_SHAPE, x, 3, 101, t, lp)
    refused(_lib.E_SHAPE, x, 3, 100, t, lp, stride=99)
    refused(_lib.E_SHAPE, x, 3, 100, t, lp, stride=101)
    refused(_lib.E_SHAPE, x, 3, 100, t, e.alloc_f32(2))
    refused(_lib.E_SHAPE, x, 3, 100, e.upload_u32([1]), lp)
    refused(_lib.E_INVALID, x, 3, 100, None, lp)
    refused(_lib.E_INVALID, x, 3, 100, None, None, rank=lp)
    refused(_lib.E_SHAPE, x, 3, 100, t, lp, top=33, top_ids=ids, top_log_probs=tlp)
    refused(_lib.E_SHAPE, x, 30, 4, t, lp, top=5, top_ids=ids, top_log_probs=tlp)
    refused(_lib.E_SHAPE, x, 3, 100, t, lp, top=6, top_ids=ids, top_log_probs=tlp)
    refused(_lib.E_INVALID, x, 3, 100, t, lp, top=2, top_ids=ids)
    refused(_lib.E_INVALID, x, 3, 100, t, lp, entropy=lp)
    refused(_lib.E_INVALID, x, 3, 100, t, x)
    refused(_lib.E_INVALID, x, 3, 100, t, t)
    refused(_lib.E_SHAPE, x, 2 ** 31, 100, t, lp)
