"""Operators beside the matrix products, as cases that can be timed and compared.

  append     keys and values of new tokens into a paged cache that holds them in 4 bits, the keys rotated to their positions on the way
  attend     attention of one or several new tokens of several sequences over such a cache, the queries rotated on the way
  log_probs  log probability of a given token, its rank, the entropy and the most probable alternatives of rows of logits

The cache's format: blocks of 32 values along a head have a minimum m and a step d in half precision and a code of 4 bits a value; a value is
m + d * code with m = half(min), d = half(max(max - m, 0) / 15), code = the nearest whole number to (x - m) / d, ties to the even one.
"""
import math
import random

import numpy as np
import torch

own = False   # false: the plain forms below; true: this framework's calls

DEV = "cuda"
BLOCK = 32
HALF_MAX = 65504.0


def case_append(kv_heads, dim, rot, neox, page, seqs, past, tokens, mix):
    return dict(kind="append", kv_heads=kv_heads, dim=dim, rot=rot, neox=neox, page=page, seqs=seqs, past=past, tokens=tokens, mix=mix)


def case_attend(heads, kv_heads, dim, rot, neox, page, seqs, past, tokens, mix):
    return dict(kind="attend", heads=heads, kv_heads=kv_heads, dim=dim, rot=rot, neox=neox, page=page, seqs=seqs, past=past, tokens=tokens, mix=mix)


def case_log_probs(rows, vocab, top):
    return dict(kind="log_probs", rows=rows, vocab=vocab, top=top)


def listed():
    """past and tokens are the largest of the batch; mix 0 gives every sequence that much, another number ragged lengths up to it."""
    named = {
        # a decoding step of eight users of an 8B model, one layer: the smallest call
        "append_step_8": case_append(8, 128, 128, False, 64, 8, 3900, 1, 5),
        # drafts of up to five tokens of 37 users, heads of 64, half of each head rotated, small pages
        "append_drafts_d64": case_append(2, 64, 32, True, 16, 37, 1500, 5, 9),
        # three prompts of different lengths taken in together
        "append_prompts": case_append(8, 128, 128, True, 64, 3, 700, 2741, 4),
        # one user of an 8B model at the start of a conversation: latency
        "attend_one_short": case_attend(32, 8, 128, 128, False, 64, 1, 199, 1, 0),
        # a serving step of 64 users with contexts of all lengths
        "attend_batch_ragged": case_attend(32, 8, 128, 128, False, 64, 64, 4095, 1, 3),
        # one user of a 70B model behind a long document
        "attend_long": case_attend(64, 8, 128, 128, True, 64, 1, 131007, 1, 0),
        # drafts of eight tokens being verified, five query heads a key head
        "attend_drafts": case_attend(40, 8, 128, 128, False, 32, 8, 2999, 8, 6),
        # a prompt behind a context that is there already
        "attend_prompt": case_attend(32, 8, 128, 128, True, 64, 1, 1021, 2048, 0),
        # heads of 64, seven a key head, pages of 16, some sequences with several tokens
        "attend_d64": case_attend(14, 2, 64, 64, True, 16, 24, 1777, 3, 8),
        # the token just decoded with five alternatives, as a chat interface shows them
        "log_probs_one": case_log_probs(1, 128256, 5),
        # every token of a text scored, no alternatives
        "log_probs_text": case_log_probs(777, 32000, 0),
        # a serving step's worth of rows with twenty alternatives each, a vocabulary that is no multiple of four
        "log_probs_batch": case_log_probs(256, 151643, 20),
    }
    return [dict(c, name=n) for n, c in named.items()]


def _between(rng, lo, hi):
    """A whole number spread over the logarithm of the range."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("append", "attend", "attend", "log_probs"))
    if kind == "log_probs":
        vocab = _between(rng, 2000, 160000)
        rows = _between(rng, 1, max(1, min(2000, 38_000_000 // vocab)))
        return case_log_probs(rows, vocab, rng.choice((0, 1, 5, 20, 32)))
    dim = rng.choice((64, 128, 128))
    kv_heads, group = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 3, 4, 5, 7, 8))
    rot = rng.choice((dim, dim // 2, 0))
    neox, page, mix = rng.random() < 0.5, rng.choice((16, 32, 64, 128)), rng.choice((0, 1, 2, 3))
    seqs = _between(rng, 1, 64)
    if kind == "append":
        tokens = _between(rng, 1, max(1, 4000 // seqs))
        return case_append(kv_heads, dim, rot, neox, page, seqs, _between(rng, 1, 4000), tokens, mix)
    if rng.random() < 0.6:
        tokens, past = 1, _between(rng, 1, 131072 // seqs)
    elif rng.random() < 0.5:
        tokens, past = rng.randint(2, 9), _between(rng, 1, 131072 // seqs)
    else:
        seqs = rng.randint(1, 3)
        tokens, past = _between(rng, 10, 65536 // (seqs * max(32, kv_heads * group))), _between(rng, 1, 1000)
    return case_attend(kv_heads * group, kv_heads, dim, rot, neox, page, seqs, past, tokens, mix)


def lengths(case):
    """(past, new tokens) of every sequence, by the case alone."""
    n = case["seqs"]
    if not case["mix"]:
        return [case["past"]] * n, [case["tokens"]] * n
    r = random.Random(case["mix"] * 1000 + n)
    past = [r.randint(0, case["past"]) for _ in range(n)]
    tokens = [r.randint(max(1, case["tokens"] // 2), case["tokens"]) for _ in range(n)]
    past[r.randrange(n)], tokens[r.randrange(n)] = case["past"], case["tokens"]
    return past, tokens


def work(case):
    if case["kind"] == "log_probs":
        n, v, k = case["rows"], case["vocab"], case["top"]
        return {"bytes": 4.0 * n * v + n * (16 + 8 * k), "flops": 4.0 * n * v}
    past, tokens = lengths(case)
    total, kh, d = sum(tokens), case["kv_heads"], case["dim"]
    held = kh * d * 1.25                      # bytes of a token: codes of keys and values, a step and a minimum for every 32
    rows = total * case["rot"] * 4
    if case["kind"] == "append":              # keys and values read, their codes written, the values they stand for handed back
        return {"bytes": float(total * (kh * d * 16 + held) + rows), "flops": 30.0 * total * kh * d}
    seen = sum(p + t for p, t in zip(past, tokens))
    pairs = sum(t * p + t * (t + 1) // 2 for p, t in zip(past, tokens))
    return {"bytes": float(seen * held + 8 * total * case["heads"] * d + rows), "flops": 4.0 * pairs * case["heads"] * d}


# ---- inputs ----------------------------------------------------------------------------------------------


def rope_table(positions, rot):
    """(sin, cos) of every rotated pair at every position, rounded once from 64 bits."""
    freq = 500000.0 ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
    angle = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * freq
    return torch.stack((torch.sin(angle), torch.cos(angle)), -1).float().contiguous()


def keys_and_values(gen, tokens, kv_heads, dim):
    """Rows with the spread of a trained model's: some channels of the keys stand out, values are near normal."""
    loud = 1.0 + 4.0 * (torch.rand(kv_heads, dim, generator=gen, device=DEV) < 0.06)
    k = torch.randn(tokens, kv_heads, dim, generator=gen, device=DEV) * loud
    v = torch.randn(tokens, kv_heads, dim, generator=gen, device=DEV) * 0.6
    return k, v


def _engine():
    """The one engine of a program, on the stream of its tensors."""
    from alice_llm_b200.gpu import GpuEngine
    if not hasattr(_engine, "one"):
        _engine.one = GpuEngine()
    _engine.one.set_stream(torch.cuda.current_stream().cuda_stream)
    return _engine.one


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    if case["kind"] == "log_probs":
        return _prepare_log_probs(case, gen)
    past, tokens = lengths(case)
    kh, dim, page, rot = case["kv_heads"], case["dim"], case["page"], case["rot"]
    need = [-(-(p + t) // page) for p, t in zip(past, tokens)]
    wide = max(need)
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=gen, device=DEV)
    table, at = torch.zeros(len(past), wide, dtype=torch.int64, device=DEV), 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    seq = torch.repeat_interleave(torch.arange(len(past), device=DEV), torch.tensor(tokens, device=DEV))
    first = torch.tensor([sum(tokens[:s]) for s in range(len(past))], device=DEV)
    start = torch.tensor(past, device=DEV)
    pos = start[seq] + torch.arange(sum(tokens), device=DEV) - first[seq]
    st = dict(case=case, seq=seq, pos=pos, start=start, first=first, count=torch.tensor(tokens, device=DEV), table=table, rope=rope_table(max(p + t for p, t in zip(past, tokens)), rot) if rot else None)
    if case["kind"] == "append":
        st["k"], st["v"] = keys_and_values(gen, sum(tokens), kh, dim)
    else:
        st["q"] = torch.randn(sum(tokens), case["heads"], dim, generator=gen, device=DEV) * 1.5
        k, v = keys_and_values(gen, pages * page, kh, dim)
        st["kc"], st["vc"] = _in_codes(k), _in_codes(v)           # what the pages hold: [pages * page, kv heads, ...]
    if own:
        e = _engine()
        wrap = lambda t: e.buf_from_device(t.data_ptr(), t.numel())  # noqa: E731
        cache = e.kv4_cache(pages, page, kh, dim)
        batch = e.kv4_batch(cache, case.get("heads", kh), len(past), sum(tokens), wide)
        # a server keeps lengths and page tables on the host; each step hands them over
        st.update(engine=e, cache=cache, batch=batch, step=(past, tokens, table.cpu().numpy().astype(np.uint32)), rope_buf=wrap(st["rope"]) if rot else None)
        if case["kind"] == "append":
            st["k_out"], st["v_out"] = torch.empty_like(st["k"]), torch.empty_like(st["v"])
            st.update({n + "_buf": wrap(st[n]) for n in ("k", "v", "k_out", "v_out")})
        else:
            st["out"] = torch.empty_like(st["q"])
            st.update({n + "_buf": wrap(st[n]) for n in ("q", "out")})
            whole = e.kv4_batch(cache, kh, 1, pages * page, pages)
            whole.set([0], [pages * page], np.arange(pages)[None])
            e.kv4_append(cache, whole, wrap(k), wrap(v))
            e.sync()
            whole.free()
    return st


def _prepare_log_probs(case, gen):
    n, v, k = case["rows"], case["vocab"], case["top"]
    # logits of a language model: a normal spread, a few tokens far above the rest in most rows, some tokens ruled out
    x = torch.randn(n, v, generator=gen, device=DEV) * 2.2
    peaks = torch.randint(0, v, (n, 8), generator=gen, device=DEV)
    lift = torch.rand(n, 8, generator=gen, device=DEV) * 16.0 * torch.rand(n, 1, generator=gen, device=DEV)
    x.scatter_add_(1, peaks, lift)
    x[:, torch.randint(0, v, (max(1, v // 500),), generator=gen, device=DEV)] = -math.inf
    likely = torch.rand(n, generator=gen, device=DEV) < 0.7
    target = torch.where(likely, x.argmax(1), torch.randint(0, v, (n,), generator=gen, device=DEV)).to(torch.int32)
    st = dict(case=case, x=x, target=target)
    if own:
        e = _engine()
        wrap = lambda t: e.buf_from_device(t.data_ptr(), t.numel())  # noqa: E731
        st["lp"], st["entropy"] = torch.empty(n, device=DEV), torch.empty(n, device=DEV)
        st["rank"] = torch.empty(n, dtype=torch.int32, device=DEV)
        st["top_ids"], st["top_lp"] = torch.empty(n, k, dtype=torch.int32, device=DEV), torch.empty(n, k, device=DEV)
        st.update(engine=e, **{m + "_buf": wrap(st[m]) for m in ("x", "target", "lp", "entropy", "rank")})
        st.update({m + "_buf": wrap(st[m]) if k else None for m in ("top_ids", "top_lp")})
    return st


# ---- plain forms -----------------------------------------------------------------------------------------


def _half(x):
    """The half-precision number nearest to each 64-bit one, as a 64-bit one."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), torch.clamp(e, min=-13) - 11)
    return (torch.round(x / step) * step).clamp(-HALF_MAX, HALF_MAX)


def _in_codes(x):
    """-> (codes [..., dim] uint8, step and minimum [..., dim / 32] in half precision). In 64 bits: values next to a border."""
    x = x.double().unflatten(-1, (-1, BLOCK))
    m = _half(x.amin(-1))
    d = _half((x.amax(-1) - m).clamp(min=0) / 15)
    code = torch.round((x - m[..., None]) / torch.where(d > 0, d, 1.0)[..., None]).clamp(0, 15)
    code = torch.where((d > 0)[..., None], code, 0.0)
    return code.to(torch.uint8).flatten(-2), d.half(), m.half()


def _values(codes, d, m):
    c = codes.unflatten(-1, (-1, BLOCK)).float()
    return torch.addcmul(m.float()[..., None], c, d.float()[..., None]).flatten(-2)


def _rotated(x, table, pos, rot, neox):
    """x [tokens, heads, dim] in 64 bits, its first rot entries turned by the angles of its position."""
    x = x.double()
    if not rot:
        return x
    sin, cos = table.double()[pos].unbind(-1)
    sin, cos = sin[:, None], cos[:, None]
    part, rest = x[..., :rot], x[..., rot:]
    a, b = part.chunk(2, -1) if neox else (part[..., 0::2], part[..., 1::2])
    turned = (a * cos - b * sin, a * sin + b * cos)
    part = torch.cat(turned, -1) if neox else torch.stack(turned, -1).flatten(-2)
    return torch.cat((part, rest), -1)


def _plain_append(st):
    c = st["case"]
    k = _rotated(st["k"], st["rope"], st["pos"], c["rot"], c["neox"])
    return {"k": _values(*_in_codes(k)), "v": _values(*_in_codes(st["v"]))}


def _plain_attend(st):
    c = st["case"]
    heads, kh, dim, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    group = heads // kh
    q = _rotated(st["q"], st["rope"], st["pos"], c["rot"], c["neox"]).float()
    seqs, most = len(st["start"]), int(c["tokens"])
    of = st["first"][:, None] + torch.arange(most, device=DEV)                      # padded: token t of sequence s is row of[s, t]
    there = torch.arange(most, device=DEV) < st["count"][:, None]
    q = q[torch.where(there, of, 0)].view(seqs, most, kh, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs, kh, most * group, dim)
    slots = (st["table"][:, :, None] * page + torch.arange(page, device=DEV)).flatten(1)
    keys = _values(*(t[slots] for t in st["kc"])).permute(0, 2, 3, 1)               # [seqs, kv heads, dim, positions]
    s = torch.matmul(q, keys).mul_(1.0 / math.sqrt(dim)).view(seqs, kh, most, group, -1)
    del keys
    seen = torch.arange(slots.shape[1], device=DEV) <= (st["start"][:, None] + torch.arange(most, device=DEV))[..., None]
    s.masked_fill_(~seen[:, None, :, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(seqs, kh, most * group, -1), _values(*(t[slots] for t in st["vc"])).permute(0, 2, 1, 3))
    o = (o.view(seqs, kh, most, group, dim) / total).permute(0, 2, 1, 3, 4).reshape(seqs, most, heads, dim)
    return {"out": o[there]}


def _plain_log_probs(st):
    x, k = st["x"], st["case"]["top"]
    top, at = x.max(1, keepdim=True)
    z = x - top
    e = z.exp().scatter_(1, at, 0.0)                       # without the largest, whose term is 1: what is small beside it is kept
    rest = e.sum(1)
    log_sum = torch.log1p(rest)
    chosen = x.gather(1, st["target"].long()[:, None])
    got = {"lp": (chosen - top)[:, 0] - log_sum, "entropy": log_sum - torch.where(z > -math.inf, e * z, 0.0).sum(1) / (1 + rest),
           "rank": ((x > chosen).sum(1) + 1).to(torch.int32)}
    if k:
        ids = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :k]
        got["top_ids"], got["top_lp"] = ids.to(torch.int32), x.gather(1, ids) - top - log_sum[:, None]
    return got


# ---- one pass --------------------------------------------------------------------------------------------


def run(st):
    c = st["case"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "log_probs": _plain_log_probs}[c["kind"]](st)
    elif "step" in st:
        st["batch"].set(*st["step"])      # the places of its tokens and its jobs are worked out within the step
    e = st["engine"]
    if c["kind"] == "append":
        e.kv4_append(st["cache"], st["batch"], st["k_buf"], st["v_buf"], rope=st["rope_buf"], rot_dims=c["rot"], neox=c["neox"])
        e.kv4_read(st["cache"], st["batch"], st["k_out_buf"], st["v_out_buf"])
        return {"k": st["k_out"], "v": st["v_out"]}
    if c["kind"] == "attend":
        e.kv4_attention(st["cache"], st["batch"], st["q_buf"], st["out_buf"], 1.0 / math.sqrt(c["dim"]), rope=st["rope_buf"], rot_dims=c["rot"], neox=c["neox"])
        return {"out": st["out"]}
    e.log_probs(st["x_buf"], c["rows"], c["vocab"], st["target_buf"], st["lp_buf"], entropy=st["entropy_buf"], rank=st["rank_buf"], top=c["top"],
                top_ids=st["top_ids_buf"], top_log_probs=st["top_lp_buf"])
    got = {"lp": st["lp"], "entropy": st["entropy"], "rank": st["rank"]}
    return dict(got, top_ids=st["top_ids"], top_lp=st["top_lp"]) if c["top"] else got


# ---- from the definitions, in 64 bits --------------------------------------------------------------------


def _exact_codes(rows):
    """numpy: the values that rows [n, 32] of 64-bit numbers become."""
    low = rows.min(1).astype(np.float16).astype(np.float64)
    step = (np.maximum(rows.max(1) - low, 0.0) / 15.0).astype(np.float16).astype(np.float64)
    with np.errstate(divide="ignore", invalid="ignore"):
        code = np.where(step[:, None] > 0, np.minimum(np.maximum(np.rint((rows - low[:, None]) / step[:, None]), 0.0), 15.0), 0.0)
    return low[:, None] + step[:, None] * code


def _exact_turn(x, st):
    """numpy: pairs as complex numbers times cos + i sin."""
    c = st["case"]
    rot = c["rot"]
    if not rot:
        return x
    w = st["rope"].cpu().numpy().astype(np.float64)[st["pos"].cpu().numpy()]
    turn = (w[..., 1] + 1j * w[..., 0])[:, None, :]
    x = x.copy()
    if c["neox"]:
        z = (x[..., :rot // 2] + 1j * x[..., rot // 2:rot]) * turn
        x[..., :rot // 2], x[..., rot // 2:rot] = z.real, z.imag
    else:
        z = (x[..., 0:rot:2] + 1j * x[..., 1:rot:2]) * turn
        x[..., 0:rot:2], x[..., 1:rot:2] = z.real, z.imag
    return x


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "append":
        k = _exact_turn(st["k"].cpu().numpy().astype(np.float64), st)
        v = st["v"].cpu().numpy().astype(np.float64)
        return {n: _exact_codes(x.reshape(-1, BLOCK)).reshape(x.shape) for n, x in (("k", k), ("v", v))}
    if case["kind"] == "attend":
        return {"out": _exact_attend(st)}
    x = st["x"].double()
    k = case["top"]
    p = torch.softmax(x, 1)
    log_p = torch.log_softmax(x, 1)
    at = st["target"].long()
    got = {"lp": log_p.gather(1, at[:, None])[:, 0], "entropy": -torch.xlogy(p, p).sum(1), "rank": None}
    if k:
        got["top_ids"], got["top_lp"] = None, torch.topk(log_p, k, dim=1)[0]
    return got


def _exact_attend(st):
    c = st["case"]
    kh, dim = c["kv_heads"], c["dim"]
    group = c["heads"] // kh
    q = torch.from_numpy(_exact_turn(st["q"].cpu().numpy().astype(np.float64), st)).to(DEV) / math.sqrt(dim)
    out = torch.empty_like(q)
    wide = lambda t, i: (t[0][i].double().view(-1, kh, dim // BLOCK, BLOCK) * t[1][i].double()[..., None] + t[2][i].double()[..., None]).view(-1, kh, dim)  # noqa: E731
    for s, (first, n, past) in enumerate(zip(st["first"].tolist(), st["count"].tolist(), st["start"].tolist())):
        j = torch.arange(past + n, device=DEV)
        slots = st["table"][s][j // c["page"]] * c["page"] + j % c["page"]
        k, v = wide(st["kc"], slots), wide(st["vc"], slots)
        hidden = j[None] > past + torch.arange(n, device=DEV)[:, None]
        for h in range(c["heads"]):
            a = (q[first:first + n, h] @ k[:, h // group].T).masked_fill(hidden, -math.inf)
            out[first:first + n, h] = torch.softmax(a, 1) @ v[:, h // group]
    return out
