"""b2w4_logprobs against 64 bits: log probabilities, entropies and the most likely tokens, over
vocabularies that end anywhere, rows without an answer, ties, orders that a threshold dislikes,
strides, and calls that are refused."""
import math

import pytest
import torch

from __graft_entry__ import load_package

pkg = load_package()
capi = pkg.capi
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = capi.Context(0)
    yield c
    c.close()


def call(ctx, x, target, top):
    rows = x.shape[0]
    out = dict(logprob=torch.full((rows,), 7.0, device="cuda"),
               entropy=torch.full((rows,), 7.0, device="cuda"),
               top_values=torch.full((rows, top), 7.0, device="cuda"),
               top_indices=torch.full((rows, top), -7, dtype=torch.int32, device="cuda"))
    ctx.logprobs(x, target, **out)
    ctx.sync()
    return [out[k].cpu() for k in ("logprob", "entropy", "top_values", "top_indices")]


def check(ctx, x, top=20, target=None):
    """x: on the GPU, finite or -inf.  Tolerances.  Of log S: a sum of n terms in 32 bits by
    threads, warps and blocks, at most n / 2048 + 30 roundings in a row, each term off by its
    exponent's rounding (|d| eps, weighted: at most (H + 2) eps of the sum) and two units of ex2
    (2^-22); the difference x - M, its sum with log S and log itself by eps of their sizes.  The
    entropy adds T / S, whose terms are off by as much of their own size, weighted by |d|."""
    rows, vocab = x.shape
    if target is None:
        g = torch.Generator().manual_seed(1)
        target = torch.randint(0, vocab, (rows,), generator=g).to(torch.int32).cuda()
    lp, ent, values, indices = call(ctx, x, target, top)
    xd = x.double()
    want = torch.log_softmax(xd, -1).cpu()
    p = want.exp()
    wide = torch.where(p > 0, want, torch.zeros(()).double())
    entropy = -(p * wide).sum(-1)
    eps = 2.0 ** -24
    chain = (vocab / 2048 + 34) * eps + (entropy + 2) * eps + 2.0 ** -22
    order = torch.sort(x.cpu(), dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(indices.long(), order)
    t = target.cpu().long()
    for got, ref in ((lp, want.gather(1, t[:, None])[:, 0]),
                     (values, want.gather(1, order))):
        slack = chain if got.dim() == 1 else chain[:, None]
        size = torch.where(torch.isinf(ref), torch.zeros(()).double(), ref.abs())
        same = (got.double() == ref) | ((got.double() - ref).abs() <= slack + 4 * eps * (size + 1))
        assert same.all()
    second = (p * wide * wide).sum(-1)
    assert ((ent.double() - entropy).abs() <= 2 * chain * (entropy + 1) +
            4 * eps * (second + entropy + 1)).all()


def logits(rows, vocab, seed, scale=2.5, ruled_out=0.02):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, vocab), device="cuda", generator=g) * scale
    x[torch.rand((rows, vocab), device="cuda", generator=g) < ruled_out] = -math.inf
    x[:, 0] = 0.5
    return x


@pytest.mark.parametrize("vocab", [1, 2, 3, 31, 32, 1000, 1023, 4096, 4097, 8191, 8192, 8193,
                                   16385, 32768, 50257, 65537, 151936, 200003])
@pytest.mark.parametrize("rows", [1, 3])
def test_vocabularies(ctx, rows, vocab):
    check(ctx, logits(rows, vocab, vocab), top=min(vocab, 20))


@pytest.mark.parametrize("top", [1, 2, 5, 31, 32])
@pytest.mark.parametrize("vocab", [32, 5000, 40000])
def test_tops(ctx, top, vocab):
    check(ctx, logits(40, vocab, top), top=top)


def test_many_rows(ctx):
    check(ctx, logits(700, 9001, 5))


@pytest.mark.parametrize("scale", [1e-3, 30.0, 1e4])
def test_flat_and_sharp_rows(ctx, scale):
    check(ctx, logits(6, 70000, 6, scale))


def test_ties_and_orders_that_fill_the_list(ctx):
    vocab = 40001
    x = torch.empty((8, vocab), device="cuda")
    ramp = torch.arange(vocab, device="cuda", dtype=torch.float32) / 1000
    x[0] = 0.0                                  # all equal
    x[1] = ramp                                 # every tile above the one before
    x[2] = -ramp
    x[3] = (ramp * 10).floor()                  # steps of a hundred equal numbers
    x[4] = -math.inf                            # a single token is left
    x[4, 31234] = -3.0
    x[5] = -0.0                                 # zeros of both signs are equal
    x[5, ::3] = 0.0
    x[6] = -math.inf                            # fewer left than are asked for
    x[6, 77::5001] = torch.arange(8, device="cuda", dtype=torch.float32)
    x[7] = torch.finfo(torch.float32).min       # the type's lowest number as a mask
    x[7, 500:530] = 1.0
    check(ctx, x)
    check(ctx, x, top=32)


def test_rows_without_a_distribution(ctx):
    x = logits(6, 20000, 8, ruled_out=0.0)
    x[0] = -math.inf
    x[1, 333] = math.nan
    x[2, 19999] = math.inf
    x[3] = math.nan
    x[3, 5] = 1.0
    x[3, 17000] = 2.0
    target = torch.tensor([0, 5, 5, 5, 7, 7], dtype=torch.int32, device="cuda")
    lp, ent, values, indices = call(ctx, x, target, 4)
    assert torch.isnan(lp[:4]).all() and torch.isnan(ent[:4]).all()
    assert torch.isnan(values[:4]).all() and torch.isfinite(values[4:]).all()
    assert indices[0].tolist() == [0, 1, 2, 3]
    clean = torch.where(torch.isnan(x[1]), -math.inf, x[1])
    assert indices[1].tolist() == torch.topk(clean, 4).indices.tolist()
    assert indices[2, 0] == 19999
    assert indices[3].tolist() == [17000, 5, 0, 1]  # a NaN only where nothing else is left
    check(ctx, x[4:], top=4, target=target[4:])


def test_targets(ctx):
    x = logits(4, 5000, 9)
    target = torch.tensor([-1, 4999, 17, -5], dtype=torch.int32, device="cuda")
    lp, _, _, _ = call(ctx, x, target, 2)
    want = torch.log_softmax(x.double(), -1).cpu()
    assert lp[0] == 0 and lp[3] == 0
    assert abs(lp[1] - want[1, 4999]) < 1e-5 or lp[1] == want[1, 4999]
    assert abs(lp[2] - want[2, 17]) < 1e-5 or lp[2] == want[2, 17]
    target[2] = 5000
    out = torch.zeros(4, device="cuda")
    ctx.logprobs(x, target, out)
    with pytest.raises(capi.B200W4Error, match="outside of what the call has"):
        ctx.sync()
    assert torch.isnan(out[2]) and not torch.isnan(out[[0, 1, 3]]).any()


def test_strides_and_outputs_left_out(ctx):
    big = logits(5, 30011, 10)
    for x in (big[:, :30000], big[:, 1:], big[:, 3:29001], big[::2], big[:1, 2:]):
        check(ctx, x, top=7)
    x = big.contiguous()
    target = torch.zeros(5, dtype=torch.int32, device="cuda")
    lp, ent, values, indices = call(ctx, x, target, 6)
    for names in (("logprob",), ("entropy",), ("top_values",), ("top_indices",),
                  ("logprob", "top_indices")):
        made = dict(logprob=torch.zeros(5, device="cuda"), entropy=torch.zeros(5, device="cuda"),
                    top_values=torch.zeros(5, 6, device="cuda"),
                    top_indices=torch.zeros(5, 6, dtype=torch.int32, device="cuda"))
        kept = {n: made[n] for n in names}
        ctx.logprobs(x, target if "logprob" in names else None, **kept)
        ctx.sync()
        for n, want in zip(("logprob", "entropy", "top_values", "top_indices"),
                           (lp, ent, values, indices)):
            if n in names:
                assert torch.equal(kept[n].cpu(), want)  # the same bits


def test_the_same_bits_again_and_replayed(ctx):
    x = logits(9, 151936, 11)
    target = torch.arange(9, dtype=torch.int32, device="cuda")
    first = call(ctx, x, target, 20)
    out = [t.cuda().fill_(0) for t in first]
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        ctx.set_stream(side.cuda_stream)
        with torch.cuda.graph(graph, stream=side):
            ctx.logprobs(x, target, *out)
    ctx.set_stream(0)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b.cpu()) for a, b in zip(first, out))


def test_refusals(ctx):
    x = torch.zeros((2, 100), device="cuda")
    z, i = torch.zeros(2, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    tops = torch.zeros((2, 33), device="cuda")
    launches = ctx.launches
    for args in (dict(), dict(targets=i), dict(logprob=z), dict(top_values=tops),
                 dict(logits=x[:, :8], top_values=tops[:, :9].contiguous())):
        with pytest.raises(capi.B200W4Error):
            ctx.logprobs(**{**dict(logits=x), **args})
    for args in (dict(targets=i.long(), logprob=z), dict(entropy=z[:1]),
                 dict(top_values=tops[:, :4]), dict(logits=x.t(), entropy=z),
                 dict(top_indices=tops[:, :4].contiguous())):
        with pytest.raises(ValueError):
            ctx.logprobs(**{**dict(logits=x), **args})
    assert ctx.launches == launches


@pytest.mark.parametrize("vocab", [9000, 151936])
@pytest.mark.parametrize("winner_first", [False, True])
def test_confident_rows(ctx, vocab, winner_first):
    """A winner and a rival 1 to 30 below it, in numbers that one thread meets one after the other
    or that lie anywhere; nothing else is left.  No log probability is above zero, no entropy below.
    With R = e^-gap: log p = -log(1 + R), entropy = log(1 + R) + R gap / (1 + R).  R is off by its
    exponent's roundings (two of a size up to 1.5 gap), two units of ex2 and two of joins: rel =
    (3 gap + 8) eps + 2^-22 of it; the sum 1 + R, its logarithm (two units) and the difference by eps
    of 1 each at most, beside which everything is a share of R or of R gap."""
    gaps = [1.0, 3.0, 5.0, 5.7, 6.5, 7.9, 8.1, 10.0, 14.0, 20.0, 30.0]
    places = [(7, 7 + 4096), (4093, 4093 + 4096), (0, vocab - 1), (100, 101)]
    x = torch.full((len(gaps) * len(places), vocab), -math.inf, device="cuda")
    want_lp, want_h, rel = [], [], []
    for i, (gap, (a, b)) in enumerate((g, p) for g in gaps for p in places):
        win, lose = (a, b) if winner_first else (b, a)
        x[i, win] = 3.25
        x[i, lose] = 3.25 - gap
        gap = 3.25 - float(x[i, lose])
        r = math.exp(-gap)
        want_lp.append((-math.log1p(r), -gap - math.log1p(r)))
        want_h.append(math.log1p(r) + r * gap / (1 + r))
        rel.append((3 * gap + 8) * 2.0 ** -24 + 2.0 ** -22)
    target = x.argmax(-1).to(torch.int32)
    lp, ent, values, indices = call(ctx, x, target, 2)
    want_lp, want_h, rel = (torch.tensor(t, dtype=torch.float64) for t in (want_lp, want_h, rel))
    assert (lp <= 0).all() and (ent >= 0).all() and (values <= 0).all()
    eps = 2.0 ** -24
    slack = 3 * eps + (rel + 4 * eps) * want_h.clamp_min(0)
    assert ((lp.double() - want_lp[:, 0]).abs() <= slack).all()
    assert torch.equal(values[:, 0], lp)
    assert ((values[:, 1].double() - want_lp[:, 1]).abs() <= slack - 2 * eps * want_lp[:, 1]).all()
    assert ((ent.double() - want_h).abs() <= slack).all()
    # many numbers, one far above them
    y = logits(40, vocab, 3)
    y[torch.arange(40), torch.arange(40) * (vocab // 41) + 5] = torch.linspace(10, 40, 40).cuda()
    lp, ent, values, _ = call(ctx, y, y.argmax(-1).to(torch.int32), 20)
    assert (lp <= 0).all() and (ent >= 0).all() and (values <= 0).all()
    check(ctx, y)


@pytest.mark.parametrize("left", [10, 100, 1000])
def test_rows_of_which_a_mask_leaves_few_tokens(ctx, left):
    """Their answers, and that they do not take many times as long as rows of as many tokens: while
    numbers equal to the last of the largest came into the lists, -inf too, they took 21 to 44 times as
    long; 1.5 to 2.4 now."""
    rows, vocab, top = 64, 151936, 20
    x = logits(rows, vocab, 12, ruled_out=0.0)
    masked = torch.full_like(x, -math.inf)
    g = torch.Generator(device="cuda").manual_seed(left)
    kept = torch.rand((rows, vocab), device="cuda", generator=g).topk(left, -1).indices
    masked.scatter_(1, kept, x.gather(1, kept))
    check(ctx, masked, top=top)
    check(ctx, masked, top=32)
    entropy = torch.empty(rows, device="cuda")
    values = torch.empty((rows, top), device="cuda")
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)

    def time(t):
        best = math.inf
        for _ in range(5):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(10):
                ctx.logprobs(t, entropy=entropy, top_values=values)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best
    assert time(masked) < 8 * time(x)
