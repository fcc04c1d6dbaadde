"""The paged cache's entry points without a device: what they refuse, how the descriptors lie in
memory, and where the kernels' own arithmetic looks for a token, bad device data included."""
import ctypes as C

import numpy as np
import pytest

from __graft_entry__ import load_package

pkg = load_package()
capi = pkg.capi
ALIGNED = 1 << 20  # an address that nothing dereferences


def cache(**kw):
    c = capi.PagedCache.__new__(capi.PagedCache)
    C.Structure.__init__(c, **{**dict(k_dev=ALIGNED, v_dev=2 * ALIGNED, type=capi.BF16, pages=10,
                                      kv_heads=2, page_size=16, dim=128), **kw})
    return c


def batch(**kw):
    b = capi.PagedBatch.__new__(capi.PagedBatch)
    C.Structure.__init__(b, **{**dict(tables_dev=ALIGNED, lengths_dev=ALIGNED, slots_dev=None,
                                      starts_dev=None, slots=3, table_len=4, sequences=3, rows=3,
                                      max_new=1, max_length=64), **kw})
    return b


def refusal(c, b, heads=8):
    fn = capi.lib().b2w4_paged_refusal
    fn.restype = C.c_char_p
    fn.argtypes = [C.c_void_p, C.c_void_p, C.c_int]
    r = fn(C.addressof(c) if c else None, C.addressof(b) if b else None, heads)
    return r.decode() if r else None


def test_descriptors_lie_as_the_header_says():
    assert C.sizeof(capi.PagedCache) == 40 and capi.PagedCache.type.offset == 16
    assert C.sizeof(capi.PagedBatch) == 56 and capi.PagedBatch.slots.offset == 32


def test_good_descriptors_pass():
    assert refusal(cache(), batch()) is None
    for dim in (64, 128, 192, 256):
        for kind in (capi.F32, capi.F16, capi.BF16):
            assert refusal(cache(dim=dim, type=kind, page_size=1), batch()) is None
    assert refusal(cache(), batch(starts_dev=ALIGNED, rows=77, max_new=70)) is None
    assert refusal(cache(), batch(slots_dev=ALIGNED, sequences=5, rows=5)) is None


@pytest.mark.parametrize("c,b,heads", [
    (None, batch(), 8), (cache(), None, 8),
    (cache(k_dev=None), batch(), 8), (cache(v_dev=ALIGNED + 8), batch(), 8),
    (cache(type=3), batch(), 8), (cache(type=-1), batch(), 8),
    (cache(dim=0), batch(), 8), (cache(dim=80), batch(), 8), (cache(dim=320), batch(), 8),
    (cache(pages=0), batch(), 8), (cache(page_size=0), batch(), 8),
    (cache(kv_heads=0), batch(), 8), (cache(pages=1 << 28, page_size=1 << 10), batch(), 8),
    (cache(), batch(), 0), (cache(), batch(), 7), (cache(), batch(), -2),
    (cache(), batch(tables_dev=None), 8), (cache(), batch(lengths_dev=None), 8),
    (cache(), batch(slots=0), 8), (cache(), batch(table_len=0), 8),
    (cache(), batch(sequences=0), 8), (cache(), batch(max_length=0), 8),
    (cache(), batch(max_new=0), 8), (cache(), batch(sequences=4, rows=4), 8),
    (cache(), batch(rows=4), 8), (cache(), batch(rows=0, starts_dev=ALIGNED), 8),
    (cache(), batch(rows=1 << 30, starts_dev=ALIGNED), 8)])
def test_bad_descriptors_are_refused(c, b, heads):
    assert refusal(c, b, heads)


def test_null_contexts_are_rejected():
    lib = capi.lib()
    assert lib.b2w4_paged_prepare(None, None, None, None, 0, 1, None, None, 1e-6, None, None,
                                  None, 0) == -1
    assert lib.b2w4_paged_attention(None, None, None, None, 0, 1, 1.0, 0, 0, None, 0, None, 0) == -1
    assert lib.b2w4_paged_attention_work(None, 8, 128) == 0


def place(c, tables, lengths, i, j, h, slots=None, starts=None, **kw):
    tables = np.ascontiguousarray(tables, dtype=np.int32)
    arrays = [tables, np.array(lengths, dtype=np.int32)]
    fields = dict(tables_dev=arrays[0].ctypes.data, lengths_dev=arrays[1].ctypes.data,
                  slots=tables.shape[0], table_len=tables.shape[1], sequences=tables.shape[0],
                  rows=tables.shape[0], max_length=1 << 30)
    for name, v in (("slots_dev", slots), ("starts_dev", starts)):
        if v is not None:
            arrays.append(np.array(v, dtype=np.int32))
            fields[name] = arrays[-1].ctypes.data
    b = batch(**{**fields, **kw})
    out = [C.c_int() for _ in range(3)]
    row = capi.lib().b2w4_paged_row(C.byref(c), C.byref(b), i, j, h, *[C.byref(o) for o in out])
    return (row,) + tuple(o.value for o in out)


def test_tokens_lie_in_their_pages():
    tables = [[4, 0, 9], [5, 6, 7]]
    c = cache(page_size=5)
    for j in range(13):
        for h in range(2):
            page = tables[0][j // 5]
            assert place(c, tables, [13, 15], 0, j, h)[0] == (page * 2 + h) * 5 + j % 5
    assert place(c, tables, [13, 15], 0, 13, 0)[0] == -2
    assert place(c, tables, [13, 15], 1, 14, 1)[0] == (7 * 2 + 1) * 5 + 4
    assert place(c, tables, [13, 15], 0, 14, 1, slots=[1, 0])[0] == (7 * 2 + 1) * 5 + 4


def test_bad_device_data_stay_inside_the_arrays():
    c = cache(page_size=5)
    for page in (-1, 10, 1 << 30, -(1 << 31)):
        assert place(c, [[4, page, 9]], [13], 0, 7, 1)[0] == -1
        assert place(c, [[4, page, 9]], [13], 0, 4, 1)[0] == (4 * 2 + 1) * 5 + 4
    # lengths beyond the table, beyond max_length, negative
    assert place(c, [[4, 0, 9]], [16], 0, 0, 0)[:2] == (-2, 15)
    assert place(c, [[4, 0, 9]], [14], 0, 0, 0, max_length=12)[:2] == (-2, 12)
    assert place(c, [[4, 0, 9]], [-3], 0, 0, 0)[:2] == (-2, 0)
    # slots and rows that are not there
    assert place(c, [[4, 0, 9]], [13], 0, 0, 0, slots=[1])[:2] == (-2, 0)
    assert place(c, [[4, 0, 9]], [13], 0, 0, 0, slots=[-1])[:2] == (-2, 0)
    for starts in ([0, 99], [-1, 1], [3, 1], [2, 1 << 31 - 1]):
        got = place(c, [[4, 0, 9]], [13], 0, 0, 0, starts=starts, rows=8)
        assert got[0] == -2 and got[2:] == (0, 0)
    assert place(c, [[4, 0, 9]], [13], 0, 0, 0, starts=[2, 8], rows=8)[2:] == (2, 6)


def test_tensors_of_the_wrong_kind_are_refused():
    import torch
    k = torch.zeros(4, 2, 16, 64)
    with pytest.raises(ValueError):
        capi.PagedCache(k, k.half())
    with pytest.raises(ValueError):
        capi.PagedCache(k, k[:2])
    with pytest.raises(ValueError):
        capi.PagedCache(k.transpose(1, 2), k.transpose(1, 2))
    with pytest.raises(ValueError):
        capi.PagedCache(k.double(), k.double())
    tables, lengths = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    capi.PagedBatch(tables, lengths, 64)
    with pytest.raises(ValueError):
        capi.PagedBatch(tables.long(), lengths, 64)
    with pytest.raises(ValueError):
        capi.PagedBatch(tables, lengths[:2], 64)
    with pytest.raises(ValueError):
        capi.PagedBatch(tables.t(), lengths, 64)
    with pytest.raises(ValueError):
        capi.PagedBatch(tables, lengths, 64, slots=lengths, starts=lengths)


def pages_refusal(pool, planes, wants_pool=1, wants_planes=1):
    fn = capi.lib().b2w4_pages_refusal
    fn.restype = C.c_char_p
    fn.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_int]
    r = fn(C.addressof(pool) if pool else None, C.addressof(planes) if planes else None,
           wants_pool, wants_planes)
    return r.decode() if r else None


def pool(**kw):
    p = capi.PagePool.__new__(capi.PagePool)
    C.Structure.__init__(p, **{**dict(refs_dev=ALIGNED, tables_dev=ALIGNED, lengths_dev=ALIGNED,
                                      pages=9, page_size=4, slots=2, table_len=3), **kw})
    return p


def planes(at=(ALIGNED, 2 * ALIGNED), **kw):
    p = capi.PagePlanes.__new__(capi.PagePlanes)
    array = (C.c_void_p * max(1, len(at)))(*at)
    C.Structure.__init__(p, **{**dict(planes=C.cast(array, C.POINTER(C.c_void_p)), count=len(at),
                                      pages=9, page_bytes=48), **kw})
    p.keep = array
    return p


def test_good_pools_pass():
    assert pages_refusal(pool(), planes()) is None
    assert pages_refusal(None, planes(pages=4), 0, 1) is None
    assert pages_refusal(pool(), None, 1, 0) is None
    assert C.sizeof(capi.PagePool) == 40 and C.sizeof(capi.PagePlanes) == 24


@pytest.mark.parametrize("p,pl", [
    (None, planes()), (pool(), None), (pool(refs_dev=None), planes()),
    (pool(tables_dev=None), planes()), (pool(lengths_dev=None), planes()),
    (pool(pages=0), planes()), (pool(page_size=0), planes()), (pool(slots=0), planes()),
    (pool(table_len=0), planes()), (pool(pages=8), planes()), (pool(), planes(at=())),
    (pool(), planes(page_bytes=0)), (pool(), planes(page_bytes=40)),
    (pool(), planes(at=(ALIGNED, ALIGNED + 8))), (pool(), planes(at=(ALIGNED, None)))])
def test_bad_pools_are_refused(p, pl):
    assert pages_refusal(p, pl)


def test_pages_calls_reject_null_contexts():
    lib = capi.lib()
    assert lib.b2w4_pages_extend(None, None, None, None, 1, None) == -1
    assert lib.b2w4_pages_fork(None, None, None, None, None, 1) == -1
    assert lib.b2w4_pages_free(None, None, None, 1) == -1
    assert lib.b2w4_pages_compact(None, None, None, None, None) == -1
    assert lib.b2w4_pages_copy(None, None, None, None, 1) == -1


@pytest.mark.parametrize("page", [1, 2, 3, 5, 7, 8, 16, 24, 100, 641, 65536, (1 << 30) - 1, 1 << 30])
def test_tokens_by_the_kernels_division(page):
    """Every quotient that a table can hold: pages of any size, positions up to 2^31 - 1."""
    rng = np.random.default_rng(page)
    top = (1 << 31) - 2
    positions = {0, 1, page - 1, page, page + 1, top, top - top % page, top - top % page - 1}
    positions |= {int(x) for x in rng.integers(0, top, 20)}
    for j in sorted(p for p in positions if 0 <= p <= top):
        n = j // page
        if n > 300000:
            continue
        table = np.full((1, n + 1), -1, dtype=np.int32)
        table[0, n] = 0
        c = cache(page_size=page, pages=1, kv_heads=1)
        length = min((n + 1) * page, top + 1)
        assert place(c, table, [length], 0, j, 0, max_length=top + 1)[0] == j - n * page


def test_the_rule_between_runs_and_rows():
    """Prompts go together, a few rows behind a long cache one by one; heads that the former does not
    take never do."""
    rule = capi.lib().b2w4_paged_runs_wanted_by
    wanted = lambda kind, dim, heads, kv, rows, seqs, length, window=0, sinks=0: rule(  # noqa: E731
        148, kind, dim, heads, kv, rows, seqs, length, window, sinks)
    assert wanted(capi.BF16, 128, 32, 8, 6000, 1, 6000, 2048, 4) == 1
    assert wanted(capi.F16, 64, 64, 8, 2100, 6, 3500, 512, 8) == 1
    assert wanted(capi.F32, 128, 32, 8, 333, 1, 1233) == 1
    assert wanted(capi.BF16, 128, 32, 8, 4, 1, 30000) == 0
    assert wanted(capi.BF16, 192, 32, 8, 6000, 1, 6000) == 0
    assert wanted(capi.BF16, 64, 129, 1, 6000, 1, 6000) == 0


def test_how_many_rows_a_launch_takes():
    """Blocks of 16 keys of a launch stay below 2^30, by tiles of eight or sixteen heads of a kv head."""
    items = capi.lib().b2w4_paged_split_items
    items.argtypes = [C.c_int, C.c_double, C.c_int, C.c_int, C.c_int]
    assert items(64, 131072.0, 128, 64, 8) == 64
    assert items(100000, 100000.0, 256, 8, 8) == 2 ** 30 // (6250 * 8)
    assert items(100000, 100000.0, 256, 72, 8) == 2 ** 30 // (6250 * 16)
    assert items(100000, 100000.0, 128, 128, 8) == 2 ** 30 // (6250 * 8)
    assert items(20, 2.0 ** 31 - 1, 64, 1, 1) == 8
    assert items(20, 2.0 ** 31 - 1, 64, 16, 16) == 0


@pytest.mark.parametrize("name,args", [
    ("forward", (None, 1)), ("prefill", ([1],)), ("decode_step", ()), ("capture_decode_step", ()),
    ("replay_decode_step", ()), ("reset", ())])
def test_a_paged_decoder_refuses_the_calls_of_one_sequence(name, args):
    """They take the cache for a contiguous one of 32-bit numbers: in the pages they would write
    over other sequences, and beyond the pool's end where that is of 16 bits."""
    d = pkg.decoder.PagedDecoder.__new__(pkg.decoder.PagedDecoder)
    with pytest.raises(NotImplementedError, match="slots"):
        getattr(d, name)(*args)


def bare_context():
    """A context whose calls get as far as the library, which refuses a context that is none."""
    c = capi.Context.__new__(capi.Context)
    c.handle = None
    return c


def test_logits_that_the_kernel_would_read_past_are_refused():
    """16-bit logits, and rows of a broadcast: read as 32-bit rows of their own they end behind the
    tensor's memory."""
    import torch
    c = bare_context()
    entropy = torch.zeros(4)
    for x in (torch.zeros(4, 100, dtype=torch.bfloat16), torch.zeros(4, 100, dtype=torch.float16),
              torch.zeros(1, 100).expand(4, 100), torch.zeros(500).as_strided((4, 100), (50, 1))):
        with pytest.raises(ValueError, match="logprobs"):
            c.logprobs(x, entropy=entropy)
    with pytest.raises(capi.B200W4Error):   # one row: its stride does not matter
        c.logprobs(torch.zeros(100).as_strided((1, 100), (0, 1)), entropy=entropy[:1])


def test_tensors_that_the_paged_kernels_would_read_or_write_past_are_refused():
    import torch
    c = bare_context()
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    ints = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731
    paged, b = capi.PagedCache(k, k), capi.PagedBatch(ints(3, 4), ints(3), 64)
    rows = lambda n, width, **kw: torch.zeros(n, width, **kw)  # noqa: E731
    half = dict(dtype=torch.bfloat16)
    attend = dict(cache=paged, batch=b, q=rows(3, 256), heads=4, out=rows(3, 256), scale=1.0,
                  work=torch.zeros(8, dtype=torch.uint8))
    prepare = dict(cache=paged, batch=b, qkv=rows(3, 512), heads=4, q_weight=torch.zeros(64),
                   k_weight=None, eps=1e-6, cos=rows(64, 32), sin=rows(70, 32), q_out=rows(3, 256))
    for call, good, bad in (
            (c.paged_attention, attend, dict(q=rows(3, 256, **half))),
            (c.paged_attention, attend, dict(q=rows(2, 256))),
            (c.paged_attention, attend, dict(q=rows(3, 512)[:, ::2])),
            (c.paged_attention, attend, dict(q=rows(1, 768))),
            (c.paged_attention, attend, dict(out=rows(3, 256, **half))),
            (c.paged_attention, attend, dict(out=rows(2, 256))),
            (c.paged_prepare, prepare, dict(qkv=rows(3, 512, **half))),
            (c.paged_prepare, prepare, dict(qkv=rows(2, 512))),
            (c.paged_prepare, prepare, dict(q_out=rows(3, 256, dtype=torch.float64))),
            (c.paged_prepare, prepare, dict(q_weight=torch.zeros(64, **half))),
            (c.paged_prepare, prepare, dict(k_weight=torch.zeros(32))),
            (c.paged_prepare, prepare, dict(cos=rows(63, 32))),
            (c.paged_prepare, prepare, dict(sin=rows(64, 32, **half))),
            (c.paged_prepare, prepare, dict(sin=rows(64, 64)[:, :32]))):
        with pytest.raises(capi.B200W4Error):   # as far as the library
            call(**good)
        with pytest.raises(ValueError, match=next(iter(bad))):
            call(**{**good, **bad})
    for call, good, bad in (   # the last row would end behind the tensor
            (c.paged_attention, attend, dict(q=rows(3, 256)[:, 64:])),
            (c.paged_attention, attend, dict(out=rows(3, 256)[:, 4:])),
            (c.paged_prepare, prepare, dict(qkv=rows(3, 512)[:, 4:])),
            (c.paged_prepare, prepare, dict(q_out=rows(3, 256)[:, 128:]))):
        with pytest.raises(capi.B200W4Error, match="too short"):
            call(**{**good, **bad})


@pytest.mark.parametrize("prompts", [[[5, 100]], [[-1]], [[1, 2], [3, 1 << 40]]])
def test_tokens_beyond_the_vocabulary_are_refused(prompts):
    """Their embedding rows lie outside of the table."""
    import types
    import torch
    d = pkg.decoder.PagedDecoder.__new__(pkg.decoder.PagedDecoder)
    d.cfg, d.slots, d.torch = types.SimpleNamespace(vocab=100), 4, torch
    d.lengths, d.refs = (torch.zeros(4, dtype=torch.int32) for _ in range(2))
    with pytest.raises(ValueError, match="vocabulary of 100"):
        d.add(prompts, list(range(len(prompts))))
    with pytest.raises(ValueError, match="vocabulary of 100"):
        d.score([7] + prompts[-1], 1)


@pytest.mark.parametrize("bad", [dict(slots=1025), dict(slots=0), dict(pages=0), dict(page_size=0)])
def test_a_paged_decoder_that_no_step_could_run_is_refused(bad):
    """More slots than one call of pages_extend takes: every step would raise."""
    cfg = pkg.decoder.DecoderConfig(1, 64, 1, 1, 64, 64, 64)
    with pytest.raises(ValueError, match="1 to 1024 slots"):
        pkg.decoder.PagedDecoder(None, cfg, None, **{**dict(slots=4, pages=4), **bad})


def test_a_loose_bound_of_the_length_does_not_part_prompts_from_their_kernel():
    """Under a window a tile sees few keys, however long the sequences may be."""
    rule = capi.lib().b2w4_paged_runs_wanted_by
    for kind in (capi.F32, capi.F16, capi.BF16):
        for length in (8192, 1 << 24, (1 << 24) + 1, 2 ** 31 - 1):
            assert rule(148, kind, 128, 32, 8, 2000, 1, length, 2048, 4) == 1
        # beyond what a wait's limit leaves time for, and beyond the lists' room
        assert rule(148, kind, 128, 32, 8, 2000, 1, (1 << 24) + 1, 0, 0) == 0
        assert rule(148, kind, 64, 8, 8, 200000, 200000, 4000, 0, 0) == 0
