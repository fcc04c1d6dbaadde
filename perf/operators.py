"""The operators of a paged key-value cache, and the log probabilities a step answers with, as
cases that can be timed and compared.

  append    b2w4_paged_prepare: Q/K norm and rotary embedding of merged qkv rows, keys and values
            into the pages of their sequences
  decode    b2w4_paged_attention, one new token per sequence
  run       b2w4_paged_attention, ragged runs of new tokens (prompts, chunks of prompts)
  fork      b2w4_pages_fork and b2w4_pages_free
  compact   b2w4_pages_compact
  copy      b2w4_pages_copy
  logprobs  b2w4_logprobs

Head layouts are those of the benchmark's decoders (32 / 8, 32 / 4 and 64 / 4 heads of 128) and
a generic one of 64 / 8 heads of 64; the vocabulary is theirs too.  `own` chooses between the
operators written out in elementary tensor operations and the library's calls.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
VOCAB = 151936


# --------------------------------------------------------------------------------- cases

def listed():
    return [
        # a decode step of sixty-four sequences: the launch and a few dependent loads are all of it
        dict(name="append_step", kind="append", type="bf16", heads=32, kv_heads=4, dim=128,
             page=16, sequences=64, longest=4000, new=1, lens=1),
        # three prompts at once into a cache of 32-bit numbers
        dict(name="append_prompts", kind="append", type="f32", heads=32, kv_heads=8, dim=128,
             page=32, sequences=3, longest=2600, new=2600, lens=2),
        # one sequence behind a short context: latency
        dict(name="decode_one", kind="decode", type="f32", heads=32, kv_heads=8, dim=128, page=16,
             sequences=1, longest=300, window=0, sinks=0, lens=3),
        # a full batch of ragged sequences, a window with a few first tokens kept
        dict(name="decode_window", kind="decode", type="f16", heads=64, kv_heads=8, dim=64,
             page=32, sequences=64, longest=8000, window=1024, sinks=4, lens=4),
        # two long documents: few rows, work only along the cache
        dict(name="decode_long", kind="decode", type="bf16", heads=64, kv_heads=4, dim=128,
             page=64, sequences=2, longest=120001, window=0, sinks=0, lens=5),
        # the next chunk of a prompt, the cache in 32 bits as the decoder keeps it by default
        dict(name="run_chunk", kind="run", type="f32", heads=32, kv_heads=8, dim=128, page=16,
             sequences=1, longest=1233, new=333, window=0, sinks=0, lens=6),
        # chunks of several prompts in one call, none of them of a tile's length
        dict(name="run_ragged", kind="run", type="f16", heads=64, kv_heads=8, dim=64, page=16,
             sequences=6, longest=3500, new=700, window=512, sinks=8, lens=7),
        # a long prompt under a window
        dict(name="run_window", kind="run", type="bf16", heads=32, kv_heads=8, dim=128, page=64,
             sequences=1, longest=6000, new=6000, window=2048, sinks=4, lens=8),
        # eight samples of one prompt: shared pages, a copied last one in every layer; given back
        dict(name="fork_eight", kind="fork", pages=256, page=16, row_bytes=2048, planes=72,
             parents=1, children=8, longest=1001, lens=9),
        # a pool after many requests: a quarter of the pages has to move
        dict(name="compact_pool", kind="compact", pages=2048, page=32, row_bytes=2048, planes=16,
             used=0.6, lens=10),
        # one sampled token
        dict(name="logprobs_step", kind="logprobs", rows=1, vocab=VOCAB, top=5),
        # a prompt's tokens scored
        dict(name="logprobs_prompt", kind="logprobs", rows=600, vocab=VOCAB, top=20),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "decode", "run", "run", "run", "fork",
                       "compact", "copy", "logprobs", "logprobs"])
    lens = rng.randrange(1 << 20)
    if kind == "logprobs":
        vocab = _log_int(rng, 1000, VOCAB)
        return dict(kind=kind, rows=_log_int(rng, 1, min(2000, 90_000_000 // vocab)), vocab=vocab,
                    top=rng.randint(1, 32))
    if kind in ("fork", "compact", "copy"):
        page = rng.choice([8, 16, 24, 32, 64])
        base = dict(kind=kind, page=page, row_bytes=rng.choice([512, 1024, 2048]), lens=lens)
        if kind == "fork":
            longest = _log_int(rng, 1, 2000)
            children = rng.randint(1, 16)
            return dict(base, pages=2 * (longest // page + 2) + 4 * children,
                        planes=rng.randint(2, 40), parents=rng.randint(1, 2), children=children,
                        longest=longest)
        pages = _log_int(rng, 16, 1500)
        planes = max(1, min(rng.randint(2, 80), (1 << 30) // (pages * page * base["row_bytes"])))
        if kind == "copy":
            return dict(base, pages=pages, planes=planes, pairs=_log_int(rng, 1, pages // 3))
        return dict(base, pages=pages, planes=planes, used=round(rng.uniform(0.2, 0.9), 3))
    dim = rng.choice([64, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 7, 8, 16] if kv_heads < 8 else [1, 2, 4, 8])
    case = dict(kind=kind, type=rng.choice(["f32", "f16", "bf16"]), heads=heads, kv_heads=kv_heads,
                dim=dim, page=rng.choice([8, 16, 24, 32, 64, 128]), lens=lens)
    windowed = rng.random() < 0.5
    window = _log_int(rng, 16, 4096) if windowed else 0
    sinks = rng.randint(0, 64) if windowed else 0
    if kind == "append":
        new = rng.choice([1, _log_int(rng, 2, 2000)])
        return dict(case, sequences=rng.randint(1, 64) if new == 1 else rng.randint(1, 3), new=new,
                    longest=new + _log_int(rng, 1, 4000))
    if kind == "decode":
        sequences = _log_int(rng, 1, 96)
        most = 60_000_000 // (sequences * kv_heads * dim)
        return dict(case, sequences=sequences, longest=_log_int(rng, 1, min(100_000, most)),
                    window=window, sinks=sinks)
    sequences, new = rng.randint(1, 6), _log_int(rng, 2, 1500)
    most = max(new, min(6000, 100_000_000 // (sequences * heads * new)))
    return dict(case, sequences=sequences, new=new, longest=rng.randint(new, most), window=window,
                sinks=sinks)


def _shape(case):
    """Tokens of each sequence, and how many of them are new: the first sequence has the most."""
    rng = random.Random(case["lens"])
    long, new, n = case["longest"], case.get("new", 1), case["sequences"]
    news = [new] + [rng.randint(1, new) for _ in range(n - 1)]
    lengths = [long] + [_log_int(rng, max(m, long // 16), long) for m in news[1:]]
    return lengths, news


# -------------------------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 71)
    return g


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prepare_paged(case, g):
    """A cache whose sequences own pages all over the pool, and this call's rows."""
    lengths, news = _shape(case)
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    need = [-(-n // page) for n in lengths]
    table_len = max(need)
    pages = sum(need) + 3
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    tables = torch.zeros((len(lengths), table_len), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = order[at:at + n]
        at += n
    kind, type_ = case["kind"], TYPES[case["type"]]
    shape = (pages, kv, page, dim)
    # normalised, rotated keys; values of the projection's size
    k = torch.randn(shape, device="cuda", generator=g).to(type_)
    v = torch.randn(shape, device="cuda", generator=g).mul_(2.0).to(type_)
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    rows = starts[-1]
    state = dict(case=case, k=k, v=v, tables=tables, lengths=_ints(lengths), starts=_ints(starts),
                 rows=rows, max_new=max(news), max_length=max(lengths))
    if kind == "append":
        width = (heads + 2 * kv) * dim
        state["qkv"] = torch.randn((rows, width), device="cuda", generator=g).mul_(3.0)
        state["q_weight"] = torch.randn(dim, device="cuda", generator=g).mul_(0.05).add_(1.0)
        state["k_weight"] = torch.randn(dim, device="cuda", generator=g).mul_(0.05).add_(1.0)
        angle = (torch.arange(max(lengths), device="cuda", dtype=torch.float64)[:, None] *
                 1e6 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim))
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    else:
        state["q"] = torch.randn((rows, heads * dim), device="cuda", generator=g)
    state["out"] = torch.empty((rows, heads * dim), device="cuda")
    return state


def _prepare_pages(case, g):
    """A pool's planes (one per layer for keys, one for values) and its bookkeeping."""
    pages, page, planes = case["pages"], case["page"], case["planes"]
    data = torch.randint(-30000, 30000, (planes, pages, page * case["row_bytes"] // 2),
                         dtype=torch.int16, device="cuda", generator=g)
    state = dict(case=case, data=data, planes=[data[i] for i in range(planes)])
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    if case["kind"] == "copy":
        state["src"], state["dst"] = order[:case["pairs"]], order[case["pairs"]:2 * case["pairs"]]
        return state
    rng = random.Random(case["lens"])
    if case["kind"] == "fork":
        slots = case["parents"] + case["children"]
        lengths = [case["longest"]] + [rng.randint(1, case["longest"])
                                       for _ in range(case["parents"] - 1)]
        lengths += [0] * case["children"]
    else:  # sequences of many lengths until the share of the pool is used
        lengths, want = [], max(1, int(case["used"] * pages))
        while want > 0:
            n = min(want, rng.randint(1, max(1, pages // 8)))
            lengths.append(n * page - rng.randrange(page))
            want -= n
        slots = len(lengths)
    need = [-(-n // page) for n in lengths]
    tables = torch.zeros((slots, max(need)), dtype=torch.int32, device="cuda")
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = order[at:at + n]
        refs[order[at:at + n].long()] = 1
        at += n
    state.update(tables=tables, refs=refs, lengths=_ints(lengths))
    if case["kind"] == "fork":
        state["parents"] = _ints([rng.randrange(case["parents"]) for _ in range(case["children"])])
        state["children"] = _ints(list(range(case["parents"], slots)))
    else:
        state.update(tables0=tables.clone(), refs0=refs.clone(),
                     used=torch.zeros(1, dtype=torch.int32, device="cuda"))
    return state


def _prepare_logprobs(case, g):
    rows, vocab, top = case["rows"], case["vocab"], case["top"]
    x = torch.randn((rows, vocab), device="cuda", generator=g).mul_(2.5)
    # tokens that a sampler has ruled out
    x[:, torch.randint(0, vocab, (vocab // 50,), device="cuda", generator=g)] = -math.inf
    target = torch.randint(0, vocab, (rows,), device="cuda", generator=g).to(torch.int32)
    return dict(case=case, x=x, target=target, logprob=torch.empty(rows, device="cuda"),
                entropy=torch.empty(rows, device="cuda"),
                values=torch.empty((rows, top), device="cuda"),
                indices=torch.empty((rows, top), dtype=torch.int32, device="cuda"))


def prepare(case, seed):
    g = _gen(seed)
    if case["kind"] == "logprobs":
        return _prepare_logprobs(case, g)
    if case["kind"] in ("fork", "compact", "copy"):
        return _prepare_pages(case, g)
    return _prepare_paged(case, g)


# ------------------------------------------------------------------------- the plain forms

def _rows_of(s):
    """Sequence and position of every row."""
    starts = s["starts"].long()
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    return seq, s["lengths"].long()[seq] - starts[seq + 1] + row


def _plain_append(s):
    case = s["case"]
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    seq, pos = _rows_of(s)
    x = s["qkv"].view(s["rows"], heads + 2 * kv, dim)

    def norm_rotate(x, w):
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
        c, n = s["cos"][pos][:, None], s["sin"][pos][:, None]
        a, b = x[..., :dim // 2], x[..., dim // 2:]
        return torch.cat([a * c - b * n, a * n + b * c], dim=-1)

    s["out"].copy_(norm_rotate(x[:, :heads], s["q_weight"]).view(s["rows"], -1))
    ids = s["tables"][seq, pos // page].long()
    s["k"][ids, :, pos % page] = norm_rotate(x[:, heads:heads + kv], s["k_weight"]).to(s["k"].dtype)
    s["v"][ids, :, pos % page] = x[:, heads + kv:].to(s["v"].dtype)
    return s["out"], s["k"], s["v"]


def _plain_attention(s):
    case = s["case"]
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    n, group, most = case["sequences"], heads // kv, s["max_new"]
    key = torch.arange(s["max_length"], device="cuda")
    lengths, starts = s["lengths"].long(), s["starts"].long()
    ids = s["tables"][:, key // page].long()
    there = key < lengths[:, None]

    def gather(cache):  # [n, kv, keys, dim]
        rows = cache.permute(0, 2, 1, 3)[ids, key % page].float()
        return rows.masked_fill(~there[:, :, None, None], 0.0).transpose(1, 2)

    seq, pos = _rows_of(s)
    at = torch.arange(s["rows"], device="cuda") - starts[seq]
    q = torch.zeros((n, most, kv, group, dim), device="cuda")
    q[seq, at] = s["q"].view(-1, kv, group, dim)
    q = q.permute(0, 2, 1, 3, 4).reshape(n, kv, most * group, dim)
    score = torch.matmul(q, gather(s["k"]).transpose(2, 3)).mul_(dim ** -0.5)
    p = lengths - (starts[1:] - starts[:-1])
    p = p[:, None] + torch.arange(most, device="cuda")          # position of each query
    seen = (key <= p[..., None]) & there[:, None]
    if case["window"] > 0:
        seen &= (key > p[..., None] - case["window"]) | (key < case["sinks"])
    score = score.view(n, kv, most, group, -1).masked_fill_(~seen[:, None, :, None], -math.inf)
    score = score.view(n, kv, most * group, -1)
    top = score.amax(-1, keepdim=True)
    score.sub_(top.masked_fill_(top == -math.inf, 0.0)).exp_()
    total = score.sum(-1, keepdim=True)
    o = torch.matmul(score, gather(s["v"])).div_(total.clamp_min_(1e-38))
    o = o.view(n, kv, most, group, dim).permute(0, 2, 1, 3, 4)
    s["out"].copy_(o[seq, at].reshape(s["rows"], -1))
    return s["out"]


def _plain_fork(s):
    page, tables, refs, lengths = s["case"]["page"], s["tables"], s["refs"], s["lengths"]
    parents, children = s["parents"].long(), s["children"].long()
    length = lengths[parents].long()
    full, part = length // page, length % page > 0
    column = torch.arange(tables.shape[1], device="cuda")
    rows = tables[parents]
    shared = column < full[:, None]
    free = torch.sort((refs > 0).to(torch.int32), stable=True).indices  # ascending, free ones first
    new = free[torch.cumsum(part, 0) - 1]
    last = torch.gather(rows, 1, full.clamp_max(tables.shape[1] - 1)[:, None])[:, 0].long()
    s["data"][:, new[part]] = s["data"][:, last[part]]
    refs[new[part]] = 1
    refs.index_add_(0, rows[shared].long(), torch.ones_like(rows[shared]))
    own_page = (column == full[:, None]) & part[:, None]
    rows = torch.where(own_page, new[:, None].to(torch.int32), rows)
    tables[children] = torch.where(shared | own_page, rows, tables[children])
    lengths[children] = length.to(torch.int32)


def _plain_free(s, slots):
    page, tables, refs, lengths = s["case"]["page"], s["tables"], s["refs"], s["lengths"]
    column = torch.arange(tables.shape[1], device="cuda")
    held = tables[slots][column < (lengths[slots].long()[:, None] + page - 1) // page].long()
    refs.index_add_(0, held, torch.full_like(held, -1, dtype=torch.int32))
    lengths[slots] = 0


def _plain_compact(s):
    page, tables, refs = s["case"]["page"], s["tables"], s["refs"]
    at = torch.arange(refs.shape[0], device="cuda")
    count = (refs > 0).sum()
    holes = at[(refs == 0) & (at < count)]
    movers = at[(refs > 0) & (at >= count)]
    s["data"][:, holes] = s["data"][:, movers]
    new = at.to(torch.int32)
    new[movers] = holes.to(torch.int32)
    held = (torch.arange(tables.shape[1], device="cuda") <
            (s["lengths"].long()[:, None] + page - 1) // page)
    tables.copy_(torch.where(held, new[tables.long()], tables))
    refs[holes] = refs[movers]
    refs[movers] = 0
    s["used"].copy_(count)


def _plain_logprobs(s):
    x, top = s["x"], s["case"]["top"]
    shifted = x - x.amax(-1, keepdim=True)
    e = shifted.exp()
    total = e.sum(-1, keepdim=True)
    logp = shifted - total.log()
    p = e / total
    entropy = -(p * logp.masked_fill(p == 0, 0.0)).sum(-1)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    return (torch.gather(logp, 1, s["target"].long()[:, None])[:, 0], entropy,
            torch.gather(logp, 1, order), order.to(torch.int32))


# --------------------------------------------------------------------- the library's calls

_context = None


def _library(s):
    """The context of the GPU, and what a program keeps beside its tensors: descriptors of the
    cache, the batch and the pool, and a work area."""
    global _context
    from __graft_entry__ import load_package
    capi = load_package().capi
    if _context is None:
        _context = capi.Context(0)
    _context.set_stream(torch.cuda.current_stream().cuda_stream)
    if "kept" not in s:
        case, kept = s["case"], {}
        if case["kind"] in ("append", "decode", "run"):
            kept["cache"] = capi.PagedCache(s["k"], s["v"])
            kept["batch"] = capi.PagedBatch(
                s["tables"], s["lengths"], s["max_length"], rows=s["rows"], max_new=s["max_new"],
                starts=None if case.get("new", 1) == 1 else s["starts"])
            if case["kind"] != "append":
                kept["work"] = torch.empty(_context.paged_attention_work(case["heads"],
                                                                         case["dim"]),
                                           dtype=torch.uint8, device="cuda")
        elif case["kind"] != "logprobs":
            kept["planes"] = capi.PagePlanes(s["planes"])
            if case["kind"] != "copy":
                kept["pool"] = capi.PagePool(s["refs"], s["tables"], s["lengths"], case["page"])
            if case["kind"] == "compact":
                kept["work"] = torch.empty(case["pages"], dtype=torch.int32, device="cuda")
        s["kept"] = kept
    return _context, s["kept"]


def run(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "append":
        if not own:
            return _plain_append(s)
        c, kept = _library(s)
        c.paged_prepare(kept["cache"], kept["batch"], s["qkv"], case["heads"], s["q_weight"],
                        s["k_weight"], 1e-6, s["cos"], s["sin"], s["out"])
        return s["out"], s["k"], s["v"]
    if kind in ("decode", "run"):
        if not own:
            return _plain_attention(s)
        c, kept = _library(s)
        c.paged_attention(kept["cache"], kept["batch"], s["q"], case["heads"], s["out"],
                          case["dim"] ** -0.5, kept["work"], window=case["window"],
                          sinks=case["sinks"])
        return s["out"]
    if kind == "fork":  # samples of a sequence begin, and end
        if not own:
            _plain_fork(s)
        else:
            c, kept = _library(s)
            c.pages_fork(kept["pool"], kept["planes"], s["parents"], s["children"])
        between = s["tables"].clone(), s["refs"].clone(), s["lengths"].clone()
        if not own:
            _plain_free(s, s["children"].long())
        else:
            c.pages_free(kept["pool"], s["children"])
        return between + (s["refs"], s["lengths"], s["data"])
    if kind == "compact":  # the same pool again: what was moved still lies where it was
        s["tables"].copy_(s["tables0"])
        s["refs"].copy_(s["refs0"])
        if not own:
            _plain_compact(s)
        else:
            c, kept = _library(s)
            c.pages_compact(kept["pool"], kept["planes"], kept["work"], used=s["used"])
        return s["tables"], s["refs"], s["used"], s["data"]
    if kind == "copy":
        if not own:
            s["data"][:, s["dst"].long()] = s["data"][:, s["src"].long()]
        else:
            c, kept = _library(s)
            c.pages_copy(kept["planes"], s["src"], s["dst"])
        return s["data"]
    if not own:
        return _plain_logprobs(s)
    c, kept = _library(s)
    c.logprobs(s["x"], s["target"], s["logprob"], s["entropy"], s["values"], s["indices"])
    return s["logprob"], s["entropy"], s["values"], s["indices"]


# ------------------------------------------------------------------------------ work, exact

def _pairs(length, new, window, sinks):
    """(query, key) pairs that see each other, and keys that any query sees."""
    first = length - new
    pairs = 0
    for p in range(first, length):
        pairs += p + 1 if window <= 0 else min(p + 1, window + min(sinks, max(0, p + 1 - window)))
    from_ = 0 if window <= 0 else max(0, first - window + 1)
    return pairs, length - from_ + min(sinks, from_)


def work(case):
    kind = case["kind"]
    if kind == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + case["rows"] * (12 + 8 * case["top"]), "flops": 5 * n}
    if kind in ("fork", "compact", "copy"):
        plane_page = case["page"] * case["row_bytes"] * case["planes"]
        if kind == "copy":
            return {"bytes": 2 * case["pairs"] * plane_page, "flops": 0}
        if kind == "fork":
            rng = random.Random(case["lens"])
            lengths = [case["longest"]] + [rng.randint(1, case["longest"])
                                           for _ in range(case["parents"] - 1)]
            picked = [lengths[rng.randrange(case["parents"])] for _ in range(case["children"])]
            return {"bytes": sum(2 * plane_page * (n % case["page"] > 0) + 12 * (n // case["page"])
                                 for n in picked) + 4 * case["pages"], "flops": 0}
        moved = case["pages"] * case["used"] * (1 - case["used"])
        return {"bytes": int(2 * moved * plane_page) + 16 * case["pages"], "flops": 0}
    lengths, news = _shape(case)
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    size = 4 if case["type"] == "f32" else 2
    rows = sum(news)
    if kind == "append":
        return {"bytes": rows * ((2 * heads + 2 * kv) * dim * 4 + 2 * kv * dim * size + dim * 4),
                "flops": rows * (heads + kv) * dim * 8}
    seen = [_pairs(n, m, case["window"], case["sinks"]) for n, m in zip(lengths, news)]
    return {"bytes": 8 * rows * heads * dim + sum(k for _, k in seen) * kv * dim * 2 * size,
            "flops": 4 * heads * dim * sum(p for p, _ in seen)}


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("fork", "compact", "copy"):
        return None
    if kind == "logprobs":
        logp, entropy, values = [], [], []
        for i in range(case["rows"]):
            x = s["x"][i].double()
            lp = x - torch.logsumexp(x, 0)
            logp.append(lp[s["target"][i].long()])
            kept = lp[lp > -math.inf]
            entropy.append(-(kept.exp() * kept).sum())
            values.append(torch.topk(lp, case["top"]).values)
        return torch.stack(logp), torch.stack(entropy), torch.stack(values), None
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    group = heads // kv
    lengths, news = _shape(case)
    out = torch.zeros((s["rows"], heads, dim), dtype=torch.float64, device="cuda")
    if kind == "append":
        k, v = s["k"].double(), s["v"].double()
    first = 0
    for i, (length, new) in enumerate(zip(lengths, news)):
        ids = s["tables"][i, :-(-length // page)].long()
        if kind == "append":
            rows = s["qkv"][first:first + new].double().view(new, -1, dim)
            p = torch.arange(length - new, length, device="cuda")
            turn = torch.complex(s["cos"][p].double(), s["sin"][p].double())[:, None]

            def rotated(x, w):
                x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / dim + 1e-6) * w.double()
                z = torch.complex(x[..., :dim // 2].contiguous(), x[..., dim // 2:].contiguous())
                z = z * turn
                return torch.cat([z.real, z.imag], -1)
            out[first:first + new] = rotated(rows[:, :heads], s["q_weight"])
            k[ids[p // page], :, p % page] = rotated(rows[:, heads:heads + kv], s["k_weight"])
            v[ids[p // page], :, p % page] = rows[:, heads + kv:]
        else:
            q = s["q"][first:first + new].double().view(new, heads, dim)
            p = torch.arange(length - new, length, device="cuda")[:, None]
            j = torch.arange(length, device="cuda")[None]
            hidden = j > p
            if case["window"] > 0:
                hidden |= (p - j >= case["window"]) & (j >= case["sinks"])
            for h in range(kv):
                keys = s["k"][ids, h].double().reshape(-1, dim)[:length]
                values = s["v"][ids, h].double().reshape(-1, dim)[:length]
                for f in range(h * group, (h + 1) * group):
                    score = (q[:, f] @ keys.T) / math.sqrt(dim)
                    score[hidden] = -math.inf
                    out[first:first + new, f] = torch.softmax(score, -1) @ values
        first += new
    out = out.view(s["rows"], -1)
    return (out, k, v) if kind == "append" else out
