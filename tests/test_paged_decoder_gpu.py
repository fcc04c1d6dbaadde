"""The paged operators together: a decoder of several sequences against the one-sequence decoder,
token for token, with forks, stops, compaction, replayed steps and a pool that runs out; scores of
a prompt's tokens against the logits in 64 bits."""
import numpy as np
import pytest
import torch

from __graft_entry__ import load_package

pkg = load_package()
capi, dec = pkg.capi, pkg.decoder
pytestmark = pytest.mark.gpu
RULE = capi.ACT_G128  # one rule for every number of rows: the same arithmetic for both decoders


@pytest.fixture(scope="module", params=["dense", "experts"])
def model(request):
    if request.param == "dense":
        cfg, seed = dec.DecoderConfig(2, 256, 4, 2, 64, 512, 1000), 11
    else:
        cfg, seed = dec.DecoderConfig(2, 256, 4, 2, 128, 128, 1000, experts=8, top_k=2), 4
    weights = dec.synthetic_weights(cfg, seed=seed)
    ctx = capi.Context(0)
    ctx.set_moe_rule(RULE)
    rng = np.random.default_rng(5)
    prompts = [rng.integers(0, cfg.vocab, n).tolist() for n in (12, 1, 33, 20, 70)]
    one = dec.DenseDecoder(ctx, cfg, weights, capacity=160, multi_row_rule=RULE)
    want = [sure_tokens(ctx, one, p, one.generate(p, 40), 40 if not cfg.experts else 12)
            for p in prompts]
    assert sum(len(w) for w in want) > 30
    one.free()
    yield cfg, weights, ctx, prompts, want
    ctx.close()


def sure_tokens(ctx, one, prompt, tokens, most):
    """The greedy tokens that a rounding cannot change: those ahead of the first whose logit leads
    by less than 0.05.  The decoders' attention differs by 1e-7, which now and then (3000 codes a
    token, each 127 e-7 steps from its border with probability 3e-5) makes another int8 code of a
    number; that moves the hidden row by up to 1 % (measured 0.5 to 1 %), a logit of size 1.5 by
    0.015 and a lead by 0.02.  With routed experts such a step can also change a route, whose
    effect has no such bound, so only the first tokens are taken."""
    one.reset()
    one.prefill(prompt + tokens[:-1])
    h = one._b("h", len(prompt) + len(tokens) - 1, one.cfg.hidden)[len(prompt) - 1:]
    logits = torch.empty((len(tokens), one.cfg.vocab), device="cuda")
    ctx.matmul(one.lm_head, h, logits, rule=RULE)
    ctx.sync()
    top = torch.topk(logits, 2).values
    close = ((top[:, 0] - top[:, 1]) < 0.05).nonzero()[:1, 0].tolist() + [most]
    return tokens[:min(close[0], most)]


def same(got, want):
    n = min(len(got), len(want))
    return got[:n] == want[:n]


def paged(model, **kw):
    cfg, weights, ctx, _, _ = model
    d = dec.PagedDecoder(ctx, cfg, weights, **{**dict(slots=6, pages=80, page_size=8,
                                                      max_length=160, multi_row_rule=RULE), **kw})
    d.step_ctx.set_moe_rule(RULE)
    return d


@pytest.mark.parametrize("replay", [False, True])
@pytest.mark.parametrize("slots", [5, 11])
def test_tokens_of_several_sequences(model, replay, slots):
    _, _, _, prompts, want = model
    d = paged(model, slots=slots)
    got = d.generate(prompts, 24, replay=replay)
    assert all(map(same, got, want))
    got = d.generate(prompts[::-1], 24, replay=replay)  # the same graph
    assert all(map(same, got[::-1], want))
    used = sum(-(-(len(p) + 23) // 8) for p in prompts)
    assert d.compact() == used and int((d.refs > 0).sum()) == used
    d.free()


def test_forks_stops_and_compaction_change_no_token(model):
    _, _, _, prompts, want = model
    d = paged(model)
    d.add([prompts[2], prompts[0]], [4, 1])
    got = {4: [], 1: []}

    def steps(n, slots):
        for _ in range(n):
            for s in slots:
                got.setdefault(s, []).append(int(d.token[s]))
            d.step(replay=True)
    steps(5, [4, 1])
    d.fork(4, [0, 5, 3])
    for s in (0, 5, 3):
        got[s] = list(got[4])
    steps(4, [4, 1, 0, 5, 3])
    d.drop([4])                # its children keep the shared pages
    d.stop([1, 5])
    steps(3, [0, 3])
    assert d.compact() == int((d.refs > 0).sum())
    held = int((d.refs > 0).sum())
    assert (d.refs[:held] > 0).all() and (d.refs[held:] == 0).all()
    d.running[1], d.running[5] = 1, 5   # go on
    d.drop([0])
    d.add([prompts[3]], [2])
    got[2] = []
    steps(6, [1, 5, 3, 2])
    d.sync()
    for s, tokens in got.items():
        expected = want[{1: 0, 2: 3}.get(s, 2)]
        assert same(tokens, expected), s
    d.drop(range(6))
    d.sync()
    assert int(d.refs.abs().sum()) == 0
    d.free()


def test_a_prompt_in_chunks(model):
    _, _, _, prompts, want = model
    d = paged(model)
    d.add([prompts[4][:31], prompts[2][:9]], [0, 1])
    d.stop([0, 1])
    d.add([prompts[2][9:], prompts[4][31:]], [1, 0])
    tokens = [[], []]
    for _ in range(24):
        tokens[0].append(int(d.token[0]))
        tokens[1].append(int(d.token[1]))
        d.step()
    d.sync()
    assert same(tokens[0], want[4]) and same(tokens[1], want[2])
    d.free()


@pytest.mark.parametrize("cache_type", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (10, 2)])
def test_runs_and_steps_agree(model, cache_type, window, sinks):
    """A window and a cache in 16 bits: the hidden rows of a prompt in one run and token by token
    are the same to the rounding of 32 bits -- attention -- behind which an int8 code may flip, so
    the last layer's rows agree to a code's size."""
    _, _, ctx, prompts, _ = model
    d = paged(model, cache_type=cache_type, window=window, sinks=sinks)
    ids = prompts[4][:40]
    h, _ = d._prompts([ids], [0])
    whole = h.clone()
    for t in ids:
        d._prompts([[t]], [1])
    last = d._b("h", 1, d.cfg.hidden)
    d.sync()
    off = (whole[-1] - last[0]).norm() / last[0].norm()
    assert off < 2e-2
    for li in range(d.cfg.layers):  # what the first layer's matmul sees is the same: its cache too
        k = [d.layers[li]["k_cache"][d.tables[s, :5].long()] for s in (0, 1)]
        if li == 0:
            assert torch.equal(k[0], k[1])
    d.free()


def test_the_pool_runs_out_and_the_decoder_goes_on(model):
    _, _, _, prompts, want = model
    d = paged(model, pages=13)
    d.add([prompts[2]], [0])              # 33 tokens: five pages
    with pytest.raises(capi.B200W4Error, match="out of pages"):
        d.add([prompts[4]], [1])          # 70 tokens: nine
    assert int(d.lengths[1]) == 0 and int((d.refs > 0).sum()) == 5
    d.add([prompts[3]], [1])              # 20 tokens: three
    tokens = []
    for _ in range(10):
        tokens.append(int(d.token[0]))
        d.step(replay=True)
    d.sync()
    assert same(tokens, want[2])
    while True:
        before = d.lengths.tolist()
        d.step(replay=True)
        try:
            d.sync()
        except capi.B200W4Error as e:
            assert "out of pages" in str(e)
            break
    assert d.lengths.tolist()[0] in (before[0], before[0] + 1)
    d.drop([1])                           # room again: the tokens go on where they were
    n = int(d.lengths[0]) - 33
    assert n < 39
    tokens = []
    for _ in range(39 - n):
        tokens.append(int(d.token[0]))
        d.step(replay=True)
    d.sync()
    assert same(tokens, want[2][n:])
    d.free()


def test_a_full_sequence_stays_and_the_others_go_on(model):
    _, _, _, prompts, want = model
    d = paged(model, max_length=35)       # five pages of eight: 40 tokens
    d.add([prompts[2], prompts[0]], [0, 3])
    tokens = [[], []]
    for i in range(12):
        tokens[0].append(int(d.token[0]))
        tokens[1].append(int(d.token[3]))
        d.step(replay=True)
        if i == 6:
            d.sync()
    with pytest.raises(capi.B200W4Error):
        d.sync()
    assert d.lengths.tolist() == [40, 0, 0, 24, 0, 0]
    assert same(tokens[0][:8], want[2]) and tokens[0][7:] == [tokens[0][7]] * 5
    assert same(tokens[1], want[0])
    d.free()


def test_on_a_stream_of_the_callers(model):
    _, _, ctx, prompts, want = model
    d = paged(model)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = d.generate(prompts, 24)
        got_again = d.generate(prompts[::-1], 24, replay=True)
    ctx.set_stream(0)
    assert all(map(same, got, want)) and all(map(same, got_again[::-1], want))
    d.free()


def test_scores_of_a_prompt(model):
    cfg, _, ctx, prompts, _ = model
    d = paged(model)
    ids = prompts[4]
    got = d.score(ids, 3, top=5)
    h = d._b("h", len(ids), cfg.hidden)
    logits = torch.empty((len(ids) - 1, cfg.vocab), device="cuda")
    ctx.matmul(d.lm_head, h[:-1], logits, rule=capi.ACT_G128)
    d.sync()
    want = torch.log_softmax(logits.double(), -1)
    t = torch.tensor(ids[1:], device="cuda")[:, None]
    assert (got["logprob"] - want.gather(1, t)[:, 0]).abs().max() < 1e-5
    assert (got["entropy"] + (want.exp() * want).sum(-1)).abs().max() < 1e-5
    top = torch.topk(logits, 5).indices
    assert torch.equal(got["top_indices"].long(), top)
    assert (got["top_values"] - want.gather(1, top)).abs().max() < 1e-5
    assert int(d.running[3]) == -1 and int(d.lengths[3]) == len(ids)
    d.free()


def test_refusals(model):
    d = paged(model)
    for call in (lambda: d.add([[1]], [6]), lambda: d.add([[1], [2]], [1, 1]),
                 lambda: d.add([[]], [0]), lambda: d.add([[1]], [0, 1]), lambda: d.fork(0, [0]),
                 lambda: d.score([1], 0), lambda: d.drop([-1])):
        with pytest.raises(ValueError):
            call()
    assert int(d.refs.sum()) == 0
    d.free()


def state_of(d):
    return [t.clone() for t in (d.lengths, d.refs, d.running, d.token)]


def test_prompts_that_do_not_all_fit_change_nothing(model):
    """The first prompt fits and the second does not: neither is taken, in an empty slot or in one
    that is running, and what comes behind the refusal is as if it had not been asked for."""
    _, _, _, prompts, want = model
    d = paged(model, pages=13)
    d.add([prompts[0]], [2])              # 12 tokens: two pages
    d.step()
    before = state_of(d)
    for first, slot in ((prompts[2], 0), (prompts[3] + prompts[2], 2)):
        with pytest.raises(capi.B200W4Error, match="out of pages"):
            d.add([first, prompts[4]], [slot, 1])   # five or seven pages, and nine: eleven are left
        assert all(torch.equal(a, b) for a, b in zip(state_of(d), before))
    with pytest.raises(capi.B200W4Error):
        d.add([prompts[1], [1] * 161], [0, 1])      # longer than a sequence may be
    assert all(torch.equal(a, b) for a, b in zip(state_of(d), before))
    d.add([prompts[2]], [0])
    tokens = [[], []]
    for _ in range(10):
        for t, slot in zip(tokens, (2, 0)):
            t.append(int(d.token[slot]))
        d.step(replay=True)
    d.sync()
    assert same(tokens[0], want[0][1:]) and same(tokens[1], want[2])
    d.free()


@pytest.mark.parametrize("top", [-1, 33])
def test_a_score_that_is_refused_takes_no_slot(model, top):
    _, _, _, prompts, _ = model
    d = paged(model)
    with pytest.raises(RuntimeError):
        d.score(prompts[0], 3, top=top)
    assert int(d.refs.sum()) == 0 and int(d.lengths.sum()) == 0
    d.free()


def test_a_fork_with_one_child(model):
    _, _, _, prompts, want = model
    d = paged(model)
    d.add([prompts[0]], [0])
    d.fork(0, [4])
    tokens = {0: [], 4: []}
    for _ in range(6):
        for s, t in tokens.items():
            t.append(int(d.token[s]))
        d.step()
    d.sync()
    assert tokens[0] == tokens[4] and same(tokens[4], want[0])
    d.free()


def test_forks_that_do_not_all_fit_change_nothing(model):
    _, _, _, prompts, want = model
    d = paged(model, pages=5)
    d.add([prompts[0]], [0])              # 12 tokens: a full page and one that every child copies
    before = state_of(d)
    with pytest.raises(capi.B200W4Error, match="out of pages"):
        d.fork(0, [1, 2, 3, 4])
    assert all(torch.equal(a, b) for a, b in zip(state_of(d), before))
    d.fork(0, [1])
    before = state_of(d)
    with pytest.raises(capi.B200W4Error):
        d.fork(0, [3, 1])                 # a child that is not empty
    assert all(torch.equal(a, b) for a, b in zip(state_of(d), before))
    d.fork(0, [3, 4])
    tokens = {s: [] for s in (0, 1, 3, 4)}
    for _ in range(4):
        for s, t in tokens.items():
            t.append(int(d.token[s]))
        d.step()
    d.sync()
    assert all(same(t, want[0]) for t in tokens.values())
    d.free()


def test_steps_and_prompts_take_the_contexts_rule_for_experts(model):
    """Steps have a context of their own: the same rows through both are the same bits, experts that
    hold several rows included."""
    cfg, weights, ctx, prompts, _ = model
    d = dec.PagedDecoder(ctx, cfg, weights, slots=6, pages=80, page_size=8, max_length=160,
                         multi_row_rule=RULE)
    d.add(prompts, [0, 1, 2, 3, 4])
    d.step_ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    d.step_ctx.pages_extend(d.pool, d.running, granted=d.granted)
    rows = [d._rows(c, d.token, d.step_batch, 6).clone() for c in (d.ctx, d.step_ctx)]
    d.sync()
    assert torch.equal(rows[0][:5], rows[1][:5])
    d.free()
