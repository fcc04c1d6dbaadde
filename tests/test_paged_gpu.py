"""The paged cache on the GPU against 64 bits: the step that fills the pages, attention of single
tokens and of runs, windows and sinks, every type and head size, ragged batches, pages of any
size, what is masked holding NaN, strides, slots, replays, and device data that are wrong."""
import math

import pytest
import torch

import paged_reference as ref
from __graft_entry__ import load_package

pkg = load_package()
capi = pkg.capi
pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ctx():
    c = capi.Context(0)
    yield c
    c.close()


def gen(seed):
    return torch.Generator().manual_seed(seed)


def starts_of(news):
    s = [0]
    for n in news:
        s.append(s[-1] + n)
    return s


def run(ctx, case, seed, q=None, change=None, window=0, sinks=0, pad=0, fill=math.nan,
        check=True, norm=True):
    """case: lengths, news (None: one row each, no starts), page, heads, kv, dim, dtype, slots."""
    g = gen(seed)
    lengths, news = case["lengths"], case.get("news")
    heads, kv, dim, dtype = case["heads"], case["kv"], case["dim"], case["dtype"]
    slots = case.get("slots")
    k, v, tables, held = ref.make_pool(lengths, case["page"], kv, dim, dtype, g, slots, fill=fill)
    used = list(range(len(lengths))) if slots is None else slots
    starts = starts_of(news or [1] * len(lengths))
    rows = starts[-1] + pad
    q = torch.randn(rows, heads * dim, generator=g) if q is None else q
    if change:
        change(q, k, v, tables, held)
    scale = dim ** -0.5
    want, bound = ref.attention(q[:starts[-1]], k, v, tables, held, case["page"], starts, used,
                                heads, scale, window, sinks)
    cache = capi.PagedCache(k.cuda(), v.cuda())
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    if slots is None and not news:  # idle slots behind the sequences
        tables, held = tables[:len(lengths)], held[:len(lengths)]
    batch = capi.PagedBatch(tables.cuda(), held.cuda(), case.get("max_length", max(lengths) or 1),
                            slots=None if slots is None and not news else ints(used),
                            starts=ints(starts) if news else None, rows=rows if news else None,
                            max_new=max(news) if news else 1)
    width = heads * dim
    qd = torch.full((rows, width + 8), 7.0, device="cuda")[:, :width]
    qd.copy_(q)
    out = torch.full((rows, width + 4), -3.0, device="cuda")
    work = torch.empty(ctx.paged_attention_work(heads, dim), dtype=torch.uint8, device="cuda")
    work.fill_(0xff)
    torch.cuda.synchronize()
    ctx.paged_attention(cache, batch, qd, heads, out[:, :width], scale, work, window=window,
                        sinks=sinks)
    ctx.sync()
    got = out.cpu()
    assert (got[:, width:] == -3.0).all(), "wrote beside its rows"
    assert (got[starts[-1]:] == -3.0).all(), "wrote behind the last sequence"
    got = got[:starts[-1], :width]
    if check:
        off = (got.double() - want).abs()
        assert torch.isfinite(got).all()
        assert (off <= bound).all(), float((off / bound).max())
        assert not norm or ref.norm_error(got, want) <= 2e-6
    return got, want, bound, (cache, batch, qd, out, work, width)


TYPES = [F32, F16, BF16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (4, 4, 64), (16, 1, 128), (40, 2, 64),
                                          (7, 1, 192), (6, 2, 256)])
@pytest.mark.parametrize("page,lengths", [(16, [1, 0, 16, 17, 129, 300]), (5, [64, 63, 0, 65]),
                                          (1, [40]), (400, [333, 399])])
def test_single_tokens(ctx, dtype, heads, kv, dim, page, lengths):
    run(ctx, dict(lengths=lengths, page=page, heads=heads, kv=kv, dim=dim, dtype=dtype), 1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (64, 0), (100, 4), (33, 70), (5000, 3), (0, 9),
                                          (200, 199)])
def test_single_tokens_under_a_window(ctx, dtype, window, sinks):
    run(ctx, dict(lengths=[1, 64, 0, 130, 777, 301], page=24, heads=8, kv=2, dim=128, dtype=dtype),
        2, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (16, 2, 64), (5, 1, 128), (3, 3, 64),
                                          (4, 2, 192), (4, 2, 256), (66, 1, 64)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
def test_runs(ctx, dtype, heads, kv, dim, window, sinks):
    run(ctx, dict(lengths=[150, 33, 0, 64, 201], news=[150, 1, 0, 31, 70], page=16, heads=heads,
                  kv=kv, dim=dim, dtype=dtype), 3, window=window, sinks=sinks, pad=3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 200), (64, 0), (128, 64), (129, 1),
                                          (100000, 0)])
@pytest.mark.parametrize("page", [7, 64, 128])
def test_runs_under_a_window(ctx, dtype, window, sinks, page):
    run(ctx, dict(lengths=[400, 257], news=[130, 257], page=page, heads=4, kv=1, dim=128,
                  dtype=dtype), 4, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", TYPES)
def test_long_single_token_in_an_order_of_pages(ctx, dtype):
    run(ctx, dict(lengths=[20011, 5, 9000], page=32, heads=8, kv=2, dim=64, dtype=dtype), 5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (32, 2, 64), (5, 1, 192), (20, 2, 256),
                                          (130, 1, 64)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (700, 5)])
def test_a_few_rows_behind_a_long_cache(ctx, dtype, heads, kv, dim, window, sinks):
    run(ctx, dict(lengths=[5000, 5, 1, 1200], news=[3, 0, 1, 2], slots=[3, 0, 1, 4], page=24,
                  heads=heads, kv=kv, dim=dim, dtype=dtype), 15, window=window, sinks=sinks, pad=2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("news", [[5, 7], [140, 90]])
def test_more_rows_than_tokens(ctx, dtype, news):
    """Rows ahead of a sequence's first token have none: zeros."""
    got, _, _, _ = run(ctx, dict(lengths=[2, 60], news=news, page=16, heads=8, kv=2, dim=128,
                                 dtype=dtype), 16)
    assert (got[:news[0] - 2] == 0).all() and (got[news[0] - 2:news[0]] != 0).any()


@pytest.mark.parametrize("news", [None, [9, 1, 30]])
def test_slots_of_a_larger_table(ctx, news):
    run(ctx, dict(lengths=[100, 7, 55], news=news, slots=[5, 0, 3], page=16, heads=8, kv=2,
                  dim=128, dtype=BF16), 6)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("news", [None, [90, 41]])
def test_extreme_scores_and_values(ctx, dtype, news):
    """Scores of hundreds (in 32 bits off by some 1e-5, so their probabilities too: the bound takes
    that in), values of one sign, a key that all others vanish beside."""
    def change(q, k, v, tables, held):
        q.mul_(40.0)
        v.abs_()
        k[tables[0, 0], :, 3] *= 8
    run(ctx, dict(lengths=[90, 300], news=news, page=16, heads=8, kv=2, dim=128, dtype=dtype), 7,
        change=change, norm=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("news", [None, [64, 130]])
def test_a_later_token_that_holds_nan_changes_no_earlier_row(ctx, dtype, news):
    """The last token's key and value are NaN and infinite: only its own row may know."""
    case = dict(lengths=[64, 200], news=news, page=16, heads=8, kv=2, dim=128, dtype=dtype)

    def spoil(q, k, v, tables, held):
        for s, n in enumerate((64, 200)):
            row = tables[s, (n - 1) // 16]
            k[row, :, (n - 1) % 16, ::2] = math.nan
            v[row, :, (n - 1) % 16] = math.inf
    got, want, bound, _ = run(ctx, case, 8, change=spoil, check=False)
    last = [0, 1] if not news else [63, 193]
    mine = torch.ones(got.shape[0], dtype=torch.bool)
    mine[last] = False
    assert torch.isnan(got[last]).all()
    assert ((got.double() - want).abs() <= bound)[mine].all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("news", [None, [70]])
def test_keys_of_minus_infinity_take_no_part(ctx, dtype, news):
    """A key whose score is -inf (or the type's lowest value) has probability zero, and its value
    row, infinite here, contributes nothing."""
    case = dict(lengths=[100], news=news, page=16, heads=4, kv=1, dim=128, dtype=dtype)
    low = torch.finfo(dtype).min
    q = torch.rand(70 if news else 1, 4 * 128, generator=gen(3)) + 0.5

    def change(q, k, v, tables, held):
        for j, x in ((5, -math.inf), (17, low / 2)):
            page = tables[0, j // 16]
            k[page, :, j % 16] = x
            v[page, :, j % 16] = math.inf
    got, _, _, _ = run(ctx, case, 9, q=q, change=change, check=False)

    def drop(q, k, v, tables, held):  # what is left: value zero with probability zero
        for j in (5, 17):
            page = tables[0, j // 16]
            k[page, :, j % 16] = -1e4
            v[page, :, j % 16] = 0.0
    _, want, bound, _ = run(ctx, case, 9, q=q, change=drop, check=False)
    assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("news", [None, [130, 20, 77]])
def test_the_same_bits_again_and_replayed(ctx, dtype, news):
    case = dict(lengths=[2000, 20, 800], news=news, page=16, heads=8, kv=2, dim=128, dtype=dtype)
    got, _, _, (cache, batch, q, out, work, width) = run(ctx, case, 10, window=500, sinks=4)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    call = lambda: ctx.paged_attention(cache, batch, q, 8, out[:, :width], 128 ** -0.5, work,  # noqa: E731
                                       window=500, sinks=4)
    with torch.cuda.stream(side):
        ctx.set_stream(side.cuda_stream)
        with torch.cuda.graph(graph, stream=side):
            call()
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[:got.shape[0], :width].cpu(), got)
    # shorter sequences through the same graph: lengths are read when it runs
    batch.keep[1].copy_(torch.tensor([130, 0, 77] + [0] * (batch.slots - 3), dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    short = out[:, :width].clone()
    call()
    ctx.sync()
    assert torch.equal(out[:, :width], short)
    assert (short[130:150] if news else short[1]).abs().max() == 0  # no token, no key
    ctx.set_stream(0)


@pytest.mark.parametrize("news", [None, [40, 30]])
def test_wrong_device_data_are_reported_and_left_out(ctx, news):
    """Pages that the pool has not: their keys are left out; the context stays usable."""
    case = dict(lengths=[64, 30], news=news, page=16, heads=4, kv=2, dim=128, dtype=BF16)
    got, _, _, (cache, batch, q, out, work, width) = run(ctx, case, 11)
    batch.keep[0][0, 1] = 1 << 20
    torch.cuda.synchronize()
    ctx.paged_attention(cache, batch, q, 4, out[:, :width], 128 ** -0.5, work)
    with pytest.raises(capi.B200W4Error, match="outside of what the call has"):
        ctx.sync()
    again = out[:got.shape[0], :width].cpu()
    first = 1 if news is None else 40
    assert torch.equal(again[first:], got[first:])  # the other sequence
    assert torch.isfinite(again).all() and not torch.equal(again, got)
    run(ctx, case, 11)


def test_refusals(ctx):
    case = dict(lengths=[64, 30], page=16, heads=4, kv=2, dim=128, dtype=BF16)
    _, _, _, (cache, batch, q, out, work, width) = run(ctx, case, 12)
    o = out[:, :width]
    call = lambda **kw: ctx.paged_attention(**{**dict(cache=cache, batch=batch, q=q, heads=4,  # noqa: E731
                                                      out=o, scale=1.0, work=work), **kw})
    launches = ctx.launches
    for bad in (dict(heads=3), dict(window=-1), dict(sinks=-1), dict(work=work[:16]),
                dict(work=work[8:]), dict(q=o), dict(q=q[:, 1:]), dict(out=out[:, 1:]),
                dict(out=q), dict(q=q[:, :8].contiguous())):
        with pytest.raises(capi.B200W4Error):
            call(**bad)
    qkv = torch.zeros(2, 8 * 128, device="cuda")
    table = torch.zeros(64, 64, device="cuda")
    for bad in (dict(qkv=qkv[:, :-1].contiguous()), dict(q_out=qkv[:, :512]), dict(heads=5)):
        with pytest.raises(capi.B200W4Error):
            ctx.paged_prepare(**{**dict(cache=cache, batch=batch, qkv=qkv, heads=4, q_weight=None,
                                        k_weight=None, eps=1e-6, cos=table, sin=table, q_out=o),
                                 **bad})
    assert ctx.launches == launches


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (4, 4, 64), (2, 1, 192), (5, 1, 256)])
@pytest.mark.parametrize("news,slots", [(None, None), ([5, 0, 33, 1], None), ([5, 3, 33, 1],
                                                                             [4, 0, 2, 1])])
@pytest.mark.parametrize("weights", [True, False])
def test_prepare(ctx, dtype, heads, kv, dim, news, slots, weights):
    """Norm (dim products, a mean, a root, a quotient: dim / 2 + 8 roundings at most matter) and
    rotation (three roundings) in 32 bits, then half a step of the cache's type."""
    g = gen(13)
    lengths, page = [40, 0, 33, 17] if not slots else [40, 3, 33, 17], 8
    k, v, tables, held = ref.make_pool(lengths, page, kv, dim, dtype, g, slots)
    used = list(range(4)) if slots is None else slots
    starts = starts_of(news or [1] * 4)
    rows = starts[-1]
    qkv = torch.randn(rows, (heads + 2 * kv) * dim, generator=g) * 3
    qw = torch.randn(dim, generator=g) * 0.1 + 1 if weights else None
    kw = torch.randn(dim, generator=g) * 0.1 + 1 if weights else None
    angle = torch.rand(40, dim // 2, generator=g) * 6.28
    cos, sin = angle.cos(), angle.sin()
    q, new = ref.prepare(qkv, held, starts, used, heads, kv, dim, qw, kw, 1e-6, cos, sin)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    cache = capi.PagedCache(k.cuda(), v.cuda())
    if news is None:
        tables, held = tables[:4], held[:4]
    batch = capi.PagedBatch(tables.cuda(), held.cuda(), 40,
                            slots=None if news is None else ints(used),
                            starts=ints(starts) if news else None, rows=rows if news else None,
                            max_new=max(news) if news else 1)
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    wide = torch.zeros(rows, qkv.shape[1] + 3, device="cuda")
    wide[:, :-3] = qkv.cuda()
    q_out = torch.full((rows, heads * dim), 5.0, device="cuda")
    ctx.paged_prepare(cache, batch, wide[:, :-3], heads, dev(qw), dev(kw), 1e-6, cos.cuda(),
                      sin.cuda(), q_out)
    ctx.sync()
    eps = 2.0 ** -24
    pair = lambda x: torch.cat([x[..., dim // 2:], x[..., :dim // 2]], -1)  # noqa: E731
    size = lambda x: (x.abs() + pair(x).abs()) * 2  # noqa: E731
    slack = (dim / 2 + 11) * eps
    assert ((q_out.cpu().double().view(q.shape) - q).abs() <= size(q) * slack).all()
    for want_k, want_v in [(k.clone(), v.clone())]:
        for s, (p, nk, nv) in zip(used, new):
            ids = tables[s][p // page].long()
            got = cache.keep[0].cpu()[ids, :, p % page].double()
            tiny = 2.0 ** -24 if dtype == F16 else 0.0  # below fp16's normal numbers
            limit = size(nk) * slack * 2 + nk.abs() * (ref.EPS[dtype] if dtype != F32 else 0) + tiny
            assert ((got - nk).abs() <= limit).all()
            want_k[ids, :, p % page] = cache.keep[0].cpu()[ids, :, p % page]
            want_v[ids, :, p % page] = nv.float().to(dtype)
        assert torch.equal(cache.keep[0].cpu(), want_k)  # nothing else was written
        assert torch.equal(cache.keep[1].cpu(), want_v)


def test_prepare_takes_the_bits_of_the_contiguous_form(ctx):
    """One sequence in one page that is the whole cache: b2w4_qkv_prepare's bits."""
    g = gen(14)
    qkv = torch.randn(9, 12 * 128, generator=g).cuda()
    w = (torch.randn(128, generator=g) * 0.1 + 1).cuda()
    cos, sin = (torch.from_numpy(t).cuda() for t in capi.rope_tables(64, 0, 128, 1e6))
    q0, k0, v0 = (torch.zeros(n, 128, device="cuda") for n in (9 * 8, 2 * 64, 2 * 64))
    ctx.qkv_prepare(qkv, 9, 8, 2, 128, w, w, 1e-6, cos, sin, 20, q0, k0, v0, 64)
    cache = capi.PagedCache(torch.zeros(1, 2, 64, 128, device="cuda"),
                            torch.zeros(1, 2, 64, 128, device="cuda"))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = capi.PagedBatch(ints([[0]]), ints([29]), 64, starts=ints([0, 9]), rows=9, max_new=9)
    q1 = torch.zeros(9, 8 * 128, device="cuda")
    ctx.paged_prepare(cache, batch, qkv, 8, w, w, 1e-6, cos, sin, q1)
    ctx.sync()
    assert torch.equal(q0.view(9, -1), q1)
    assert torch.equal(k0.view(1, 2, 64, 128), cache.keep[0])
    assert torch.equal(v0.view(1, 2, 64, 128), cache.keep[1])


def test_a_slot_named_twice_is_reported(ctx):
    cache = capi.PagedCache(torch.zeros(2, 1, 8, 64, device="cuda"),
                            torch.zeros(2, 1, 8, 64, device="cuda"))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = capi.PagedBatch(ints([[0], [1]]), ints([3, 3]), 8, slots=ints([1, 1]))
    qkv = torch.ones(2, 3 * 64, device="cuda")
    qkv[1] = 2.0
    table = torch.zeros(8, 32, device="cuda")
    ctx.paged_prepare(cache, batch, qkv, 1, None, None, 1e-6, table, table,
                      torch.zeros(2, 64, device="cuda"))
    with pytest.raises(capi.B200W4Error, match="outside of what the call has"):
        ctx.sync()
    assert (cache.keep[1][1, 0, 2] == 1.0).all() and cache.keep[1].sum() == 64


@pytest.mark.parametrize("dim,news", [(64, None), (192, [5, 9, 6])])
def test_a_length_that_takes_several_launches(ctx, dim, news):
    """A table with room for 2^31 - 1 tokens: eight rows to a launch."""
    g, page = gen(5), 2 ** 20
    lengths = [1 + 11 * i for i in range(20)] if not news else [5, 200, 90]
    starts = starts_of(news or [1] * 20)
    k = torch.randn(1, 1, 256, dim, generator=g).to(BF16)
    v = torch.randn(1, 1, 256, dim, generator=g).to(BF16)
    pools = [torch.zeros(1, 1, page, dim, dtype=BF16, device="cuda") for _ in range(2)]
    for pool, x in zip(pools, (k, v)):
        pool[:, :, :256] = x.cuda()
    q = torch.randn(20, 2 * dim, generator=g)
    tables = torch.zeros(len(lengths), 2048, dtype=torch.int32)
    want, bound = ref.attention(q, k, v, tables, torch.tensor(lengths), page, starts,
                                range(len(lengths)), 2, dim ** -0.5, 0, 0)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = capi.PagedBatch(tables.cuda(), ints(lengths), 2 ** 31 - 1,
                            starts=ints(starts) if news else None, rows=20,
                            max_new=max(news) if news else 1)
    out = torch.full((20, 2 * dim), math.nan, device="cuda")
    work = torch.empty(ctx.paged_attention_work(2, dim), dtype=torch.uint8, device="cuda")
    before = ctx.launches
    ctx.paged_attention(capi.PagedCache(*pools), batch, q.cuda(), 2, out, dim ** -0.5, work)
    ctx.sync()
    assert ctx.launches - before == 6
    assert ((out.cpu().double() - want).abs() <= bound).all()


def test_more_keys_than_a_launch_can_count_are_refused(ctx):
    pool = torch.zeros(1, 16, 2 ** 20, 64, dtype=BF16, device="cuda")
    q = torch.zeros(1, 16 * 64, device="cuda")
    batch = capi.PagedBatch(torch.zeros(1, 2048, dtype=torch.int32, device="cuda"),
                            torch.zeros(1, dtype=torch.int32, device="cuda"), 2 ** 31 - 1)
    work = torch.empty(ctx.paged_attention_work(16, 64), dtype=torch.uint8, device="cuda")
    with pytest.raises(capi.B200W4Error, match="max_length"):
        ctx.paged_attention(capi.PagedCache(pool, pool), batch, q, 16, torch.empty_like(q), 1.0,
                            work)


@pytest.mark.parametrize("news", [None, [130, 20, 77]])
def test_two_streams_at_once(ctx, news):
    """Two contexts with work areas of their own give the bits that each gives alone."""
    case = dict(lengths=[3000, 20, 777], news=news, page=16, heads=8, kv=2, dim=128, dtype=BF16)
    first = run(ctx, case, 31)
    second = run(ctx, dict(case, dtype=F16), 32)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    contexts = [capi.Context(0), capi.Context(0)]
    outs = []
    torch.cuda.synchronize()
    for c, s in zip(contexts, streams):
        c.set_stream(s.cuda_stream)
    for _ in range(20):
        for c, (_, _, _, (cache, batch, qd, out, work, width)) in zip(contexts, (first, second)):
            c.paged_attention(cache, batch, qd, 8, out[:, :width], 128 ** -0.5, work)
    for c, (got, _, _, (_, _, _, out, _, width)) in zip(contexts, (first, second)):
        c.sync()
        outs.append(torch.equal(out.cpu()[:, :width], got))
        c.close()
    assert outs == [True, True]


@pytest.mark.parametrize("news", [None, [2, 3], [150, 150]])
@pytest.mark.parametrize("length,room", [(65, 64), (81, 128), (-1, 64)])
def test_a_length_that_the_call_does_not_have_writes_nothing(ctx, news, length, room):
    """Beyond max_length, beyond the table, negative: the sequence has no token in this call.  Its
    pages stay as they were, its rows are zeros, the other sequence's are what they are alone."""
    g, heads, kv, dim = gen(21), 8, 4, 64
    pools = [torch.randn(16, kv, 16, dim, generator=g).cuda() for _ in range(2)]
    cache = capi.PagedCache(*pools)
    before = [t.clone() for t in pools]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    starts = starts_of(news or [1, 1])
    rows = starts[-1]
    qkv = torch.randn(rows, (heads + 2 * kv) * dim, generator=g).cuda()
    tables = ints([list(range(5)), list(range(8, 13))])
    angle = torch.rand(128, dim // 2, generator=g).cuda()
    q, out = (torch.full((rows, heads * dim), 5.0, device="cuda") for _ in range(2))
    work = torch.empty(ctx.paged_attention_work(heads, dim), dtype=torch.uint8, device="cuda")

    def both(lengths):
        batch = capi.PagedBatch(tables, ints(lengths), room, starts=ints(starts) if news else None,
                                rows=rows, max_new=max(news) if news else 1)
        ctx.paged_prepare(cache, batch, qkv, heads, None, None, 1e-6, angle.cos(), angle.sin(), q)
        ctx.paged_attention(cache, batch, q, heads, out, 0.125, work)
    both([0, 60])
    ctx.sync()
    want, pools_want = out.clone(), [t.clone() for t in pools]
    for pool, x in zip(pools, before):
        pool.copy_(x)
    out.fill_(5.0)
    both([length, 60])
    with pytest.raises(capi.B200W4Error, match="outside of what the call has"):
        ctx.sync()
    assert torch.equal(pools[0], pools_want[0]) and torch.equal(pools[1], pools_want[1])
    assert (q[:starts[1]] == 0).all() and (out[:starts[1]] == 0).all()
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,dim,lengths,news,together", [
    (4, 1, 64, [400, 33], None, False), (8, 1, 128, [400], None, False),
    (16, 1, 128, [400, 200], None, False), (40, 2, 64, [300], None, False),
    (6, 2, 256, [300], None, False), (4, 1, 192, [400], [5], False),
    (16, 4, 128, [2000], [300], True), (16, 4, 64, [2000], [300], True)])
@pytest.mark.parametrize("ahead", [0, 8, 12, 16, 21, 26])
def test_a_first_token_far_ahead_that_holds_zeros(ctx, dtype, heads, kv, dim, lengths, news,
                                                  together, ahead):
    """A sink: the first key's score is `ahead` and more above all others, its value row zero, so that
    the result is made of probabilities that are small against the row's largest.

    Scores are sums of products of small numbers, exact in 32 bits; values are positive, so that
    errors of the probabilities are errors of the result, relative.  In units of eps = 2^-24, with S
    the sink's score and s the others': the factor of the scores (three roundings) 3 (S - s); a
    score's product with it, its difference from the maximum, that one's rounding: S + |s|, S - s,
    S + 15; the exponential 4; its pieces 4; a block's sum, whose products and sums may be truncated:
    at most 24 sums and 17 numbers of each, 82; a rounding of the running sums and of their scale for
    each of at most n / 16 blocks, n / 8; the joins and the division 12.  Beside fp16 a probability is
    a multiple of 2^-51 of the row's largest: 2^-52 of each value more."""
    rule = capi.lib().b2w4_paged_runs_wanted_by
    kind = {F32: capi.F32, F16: capi.F16, BF16: capi.BF16}[dtype]
    rows = sum(news or [1] * len(lengths))
    if news:
        assert rule(148, kind, dim, heads, kv, rows, len(lengths), max(lengths), 0, 0) == together
    g, page, scale = gen(17), 16, 0.125
    q = torch.randint(-1, 2, (rows, heads, dim), generator=g).float()
    q[..., 0] = 1.0
    k, v, tables, held = ref.make_pool(lengths, page, kv, dim, dtype, g)
    k = (torch.randint(-4, 5, k.shape, generator=g) / 4).to(dtype)
    k[..., 0] = 0
    v = (v.float().abs() + 0.25).to(dtype)
    spread = dim ** 0.5 * 0.7 * 4.5 * scale / 2  # of the others' scores, about four sigma either way
    for s in range(len(lengths)):
        k[tables[s, 0], :, 0] = 0
        k[tables[s, 0], :, 0, 0] = round((ahead + spread) / scale)
        v[tables[s, 0], :, 0] = 0
    cache = capi.PagedCache(k.cuda(), v.cuda())
    tables, held = tables[:len(lengths)].cuda(), held[:len(lengths)].cuda()
    starts = starts_of(news or [1] * len(lengths))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = capi.PagedBatch(tables, held, max(lengths), starts=ints(starts) if news else None,
                            rows=rows, max_new=max(news) if news else 1)
    out = torch.empty(rows, heads * dim, device="cuda")
    work = torch.empty(ctx.paged_attention_work(heads, dim), dtype=torch.uint8, device="cuda")
    ctx.paged_attention(cache, batch, q.view(rows, -1).cuda(), heads, out, scale, work)
    ctx.sync()
    eps, group = 2.0 ** -24, heads // kv
    for s, length in enumerate(lengths):
        n = starts[s + 1] - starts[s]
        keys = ref.rows_of(cache.keep[0], tables[s], page, length).double()
        values = ref.rows_of(cache.keep[1], tables[s], page, length).double()
        x = q[starts[s]:starts[s + 1]].cuda().double().view(n, kv, group, dim)
        score = torch.einsum("nhgd,mhd->hgnm", x, keys) * scale
        seen = torch.arange(length)[None] <= torch.arange(length - n, length)[:, None]
        score.masked_fill_(~seen.cuda(), -math.inf)
        top = score[..., :1]
        others = score[..., 1:].masked_fill(~seen.cuda()[:, 1:], 0.0)
        p = (score - score.amax(-1, keepdim=True)).exp()
        weighted = torch.einsum("hgnm,mhd->hgnd", p, values)
        want = weighted / p.sum(-1, keepdim=True)
        size = top.abs()[..., 0] + others.abs().amax(-1)
        rel = (3 * size + 2 * size + size + top.abs()[..., 0] + 15 + 8 + 82 + length / 8 + 12) * eps
        bound = want * rel[..., None]
        if dtype == F16:
            bound = bound + 2.0 ** -52 * values.sum(0)[:, None, None] / p.sum(-1, keepdim=True)
        got = out[starts[s]:starts[s + 1]].double().view(n, kv, group, dim).permute(1, 2, 0, 3)
        off = ((got - want).abs() / bound).max()
        assert off <= 1.0, float(off)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,dim,lengths,news", [
    (4, 1, 128, [300], None), (16, 1, 64, [300], None), (16, 4, 128, [600], [100]),
    (16, 4, 64, [600], [100])])
def test_queries_far_above_the_others_where_keys_are_zero(ctx, dtype, heads, kv, dim, lengths, news):
    """A feature of 2^20 in every row that no key has: the scores are made of the others."""
    def change(q, k, v, tables, held):
        q.view(q.shape[0], heads, dim)[:, :, 5] = 2.0 ** 20
        k[..., 5] = 0
    run(ctx, dict(lengths=lengths, news=news, page=16, heads=heads, kv=kv, dim=dim, dtype=dtype),
        18, change=change)


def test_rows_done_again_behind_a_long_cache(ctx):
    """A key of probability zero whose value is infinite: every row of its kv head is done again key
    by key, behind 400,000 keys, which is longer than a wait may be (2 s).  No row is left out and
    no wait runs out.  A serial sum of n numbers in 32 bits is off by at most n eps of itself."""
    heads, kv, dim, n, page, rows = 32, 2, 64, 400_000, 64, 600
    rule = capi.lib().b2w4_paged_runs_wanted_by
    assert rule(148, capi.F16, dim, heads, kv, rows, 1, n, 0, 0) == 1
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn((n // page, kv, page, dim), device="cuda", generator=g).half()
            for _ in range(2))
    q = torch.randn((rows, heads, dim), device="cuda", generator=g)
    q[..., 0] = 4.0
    k[..., 0] = 0
    k[0, 0, 7] = 0
    k[0, 0, 7, 0] = -2000.0          # a score of -1000
    v[0, 0, 7] = math.inf
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = capi.PagedBatch(torch.arange(n // page, dtype=torch.int32, device="cuda")[None],
                            ints([n]), n, starts=ints([0, rows]), rows=rows, max_new=rows)
    out = torch.full((rows, heads * dim), math.nan, device="cuda")
    work = torch.empty(ctx.paged_attention_work(heads, dim), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    ctx.paged_attention(capi.PagedCache(k, v), batch, q.view(rows, -1), heads, out, 0.125, work)
    ctx.sync()
    assert torch.isfinite(out).all()
    v[0, 0, 7] = 0
    for row in (0, 7, 300, 599):
        for head in (0, 9, 15, 20):
            last = n - rows + row + 1
            keys, values = (t[:, head // 16].reshape(-1, dim)[:last].double() for t in (k, v))
            p = torch.softmax(keys @ q[row, head].double() * 0.125, 0)
            off = (out[row, head * dim:(head + 1) * dim].double() - p @ values).abs()
            assert (off <= 2 * (n + 200) * 2.0 ** -24 * (p @ values.abs())).all()
