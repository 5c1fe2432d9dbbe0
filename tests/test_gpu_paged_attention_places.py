"""GPU: attention over a paged cache where it can go wrong beside its numbers: NaNs and infinities in masked places, pages that are
none, padding, layouts, blocks of 256 rows, caches past 32 bits, streams and graphs.  Tolerances as in test_gpu_paged_attention.py."""
import numpy as np
import pytest
import torch

from tests.test_gpu_paged_attention import DEV, DTYPES, FP8, HALF_STEP, Batch, numbers

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


def slot_of(b, i, key):
    page = b.k.shape[1]
    return int(b.table[i, key // page]), key % page


# few rows and many rows, 16-bit and 8-bit caches, split keys and whole ones
FORMS = [dict(lengths=[(100, 2), (70, 1), (40, 3)], dim=64), dict(lengths=[(100, 2), (70, 1), (40, 3)], dim=128, fp8=True),
         dict(lengths=[(150, 60), (90, 90)], dim=128), dict(lengths=[(150, 60), (90, 90)], dim=64, fp8=True),
         dict(lengths=[(150, 60), (90, 90)], dim=256), dict(lengths=[(900, 3)], dim=128, kv_heads=1), dict(lengths=[(900, 40)], dim=80, kv_heads=1),
         dict(lengths=[(100, 14), (200, 15)], dim=256)]


@pytest.mark.parametrize("form", FORMS, ids=[f"{f['lengths']}-{f['dim']}" for f in FORMS])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_behind_a_sequence_and_unused_pages(form, dtype):
    """NaNs in the unused slots of a sequence's last page and in pages of nobody."""
    b = Batch(1, dtype=dtype, **form)
    for c in (b.k, b.v):
        raw = c.view(torch.uint8) if c.dtype == FP8 else c
        special = 0x7f if c.dtype == FP8 else NAN
        raw[torch.from_numpy(b.unused)] = special
        for i, (n, _) in enumerate(b.lengths):
            page, slot = slot_of(b, i, n - 1)
            raw[page, slot + 1:] = special
    b.check(b.call())


@pytest.mark.parametrize("form", FORMS, ids=[f"{f['lengths']}-{f['dim']}" for f in FORMS])
@pytest.mark.parametrize("kind", ["causal", "window", "tree"])
def test_masked_nan_and_infinity(form, kind):
    """A NaN or an infinity of a key or value reaches the queries that see it, in its own column, and no other."""
    window = 30 if kind == "window" else 0
    for what in ("key", "value"):
        b = Batch(2, dtype="bf16", tree_words=2 if kind == "tree" else 0, **form)
        more = dict(window=window) if window else {}
        seen = np.zeros((len(b.q), b.k.shape[2], b.dim), dtype=bool)   # results that may change, a kv head and column each
        from oracle import attention_oracle as ao
        for i, (n, queries) in enumerate(b.lengths):
            first = int(b.starts[i])
            sight = ao.visible(n, queries, window=window, tree=None if b.tree is None else b.tree[first:first + queries].numpy())
            for j, key in enumerate((n - 1, n - queries, max(n - queries - 35, 0), max(n - 33, 0))):
                page, slot = slot_of(b, i, key)
                head, column, value = j % b.k.shape[2], 5 + j, (NAN, INF, -INF, NAN)[j]
                c = b.k if what == "key" else b.v
                if c.dtype == FP8:
                    c.view(torch.uint8)[page, slot, head, column] = 0x7f   # (it has no infinities)
                    value = NAN
                else:
                    c[page, slot, head, column] = value
                for t in range(queries):
                    if sight[t, key]:
                        seen[first + t, head, column if what == "value" else slice(None)] = True
        got = numbers(b.call(**more))
        group = got.shape[1] // b.k.shape[2]
        changed = np.repeat(seen, group, axis=1)
        # what sees none of them is as exact as ever (not the same bits: how far a row's maximum is followed goes by the rows beside it)
        want, limit = b.limits(**more)
        with np.errstate(invalid="ignore"):
            near = np.abs(got - want) <= limit
        assert near[~changed].all(), (what, np.argwhere(~changed & ~near)[:5])
        if what == "value":
            assert not np.isfinite(got[changed]).any()


def test_infinities_of_values_keep_their_sign():
    for queries, dim in ((1, 64), (40, 128), (9, 256)):
        b = Batch(3, [(50, queries)], heads=4, kv_heads=1, dim=dim)
        for key, column, value in ((49, 3, INF), (49, 4, -INF), (10, 6, INF), (10, 7, -INF)):
            page, slot = slot_of(b, 0, key)
            b.v[page, slot, 0, column] = value
        page, slot = slot_of(b, 0, 49)
        b.v[page, slot, 0, 7] = INF
        got = numbers(b.call())
        assert (got[-1, :, 3] == INF).all() and (got[-1, :, 4] == -INF).all() and (got[-1, :, 6] == INF).all() and np.isnan(got[-1, :, 7]).all()
        assert np.isfinite(got[:-1, :, 3:5]).all() and (got[:-1, :, 7] == -INF).all()


@pytest.mark.parametrize("dim,queries", [(64, 1), (128, 1), (128, 7), (128, 60), (256, 20)])
@pytest.mark.parametrize("number", [-1, -2 ** 31, 10 ** 6, 2 ** 31 - 1])
def test_a_page_that_is_none(dim, queries, number):
    """Its sequence's results are NaN; the others' are what they were.  Nothing outside the cache is read."""
    b = Batch(4, [(100, queries), (100, queries), (30, 3)], dim=dim)
    clean = numbers(b.call())
    b.table[1, 2] = number
    got = numbers(b.call())
    first, second = int(b.starts[1]), int(b.starts[2])
    assert np.isnan(got[first:second]).all()
    assert np.array_equal(got[:first], clean[:first]) and np.array_equal(got[second:], clean[second:])
    b.table[1, 2] = len(b.k)   # one past the last
    assert np.isnan(numbers(b.call())[first:second]).all()


@pytest.mark.parametrize("dim,queries,length", [(64, 1, 300), (128, 5, 300), (128, 50, 300), (256, 20, 300), (128, 1, 4000)])
@pytest.mark.parametrize("page", [16, 24, 7])
def test_pages_before_the_window_are_not_read(dim, queries, length, page):
    b = Batch(5, [(length, queries)], dim=dim, page=page)
    window = 60
    first_key = length - queries - window + 1
    b.table[0, :first_key // page] = -1
    b.check(b.call(window=window), window=window)


def test_lengths_out_of_range():
    """More keys than the table has pages for count as many as it has; negative ones as none; starts beyond the tokens end there."""
    b = Batch(6, [(64, 3), (32, 2)], page=16)
    want = numbers(b.call())
    b.lens[0] = 10 ** 9   # the table has four pages a sequence
    assert np.array_equal(numbers(b.call())[:3], want[:3])
    b.lens[0] = -5
    got = numbers(b.call())
    assert (got[:3] == 0).all() and np.array_equal(got[3:], want[3:])
    b.lens[0] = 64
    b.starts[2] = 10 ** 9
    assert np.array_equal(numbers(b.call()), want)


@pytest.mark.parametrize("queries", [1, 40])
def test_tokens_behind_the_last_sequence(queries):
    b = Batch(7, [(100, queries), (50, queries)], dim=128, behind=5)
    got = b.call()
    assert (got[-5:] == 0).all() and not (got[:-5] == 0).all()
    out = torch.full(b.q.shape, 7.0, dtype=b.q.dtype, device=DEV)
    again = b.call(out=out)
    assert again is out and (out[-5:] == 7).all() and torch.equal(out[:-5], got[:-5])
    b.q = b.q[:0]
    b.starts.zero_()
    assert b.call().shape == (0, 4, 128)


def test_no_pages_at_all():
    b = Batch(8, [(0, 3), (0, 1)], dim=64)
    b.k, b.v = b.k[:0], b.v[:0]
    assert (b.call() == 0).all()
    b.table = b.table[:, :0]
    assert (b.call() == 0).all()


@pytest.mark.parametrize("layout", ["projection", "heads first", "odd address", "odd stride", "strided out", "side by side", "one head", "different pages"])
@pytest.mark.parametrize("fp8", [False, True])
def test_layouts(layout, fp8):
    from sonar_amd import ops
    b = Batch(9, [(100, 1), (70, 20), (33, 33)], dim=64, heads=8, kv_heads=1 if layout == "one head" else 4, fp8=fp8)
    want = b.call()
    q, k, v, out = b.q.to(DEV), b.k.to(DEV), b.v.to(DEV), None
    if layout == "projection":
        q = torch.nn.functional.pad(q.flatten(1), (0, 512))[:, :512].unflatten(1, (8, 64))
    if layout == "heads first":
        k, v = ((t.view(torch.uint8) if fp8 else t).transpose(1, 2).contiguous().view(t.dtype).transpose(1, 2) for t in (k, v))
    if layout == "odd address":
        q = torch.nn.functional.pad(q.flatten(), (1, 0))[1:].view(q.shape)
    if layout == "odd stride":
        q = torch.nn.functional.pad(q, (0, 3))[..., :64]
    if layout == "strided out":
        out = torch.zeros((len(q), 8, 96), dtype=q.dtype, device=DEV)[..., 16:80]
    if layout == "side by side":
        raw = [t.view(torch.uint8) if fp8 else t for t in (k, v)]
        both = torch.stack(raw, dim=1)
        k, v = both[:, 0].view(k.dtype), both[:, 1].view(v.dtype)
    if layout == "different pages":   # keys and values with strides of their own
        raw = v.view(torch.uint8) if fp8 else v
        wide = torch.zeros((len(v), 16, 8, 64), dtype=raw.dtype, device=DEV)
        wide[:, :, ::2] = raw
        v = wide[:, :, ::2].view(v.dtype)
    d = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    got = ops.paged_attention(q, k, v, d(b.table), d(b.lens), d(b.starts), k_scale=d(b.k_scale), v_scale=d(b.v_scale), out=out)
    assert torch.equal(got, want)
    wide_table = torch.nn.functional.pad(d(b.table), (3, 5), value=-1)[:, 3:-5]   # rows of a wider table
    assert torch.equal(ops.paged_attention(q, k, v, wide_table, d(b.lens), d(b.starts), k_scale=d(b.k_scale), v_scale=d(b.v_scale)), want)


def double_attention(q, k, v, lengths, table, page, **more):
    """Causal attention in 64 bits on the GPU, a head at a time: (out, mean of |v|, largest score sum)."""
    out, size, most = (torch.zeros(q.shape, dtype=torch.float64, device=DEV) for _ in range(3))
    first = 0
    for i, (n, queries) in enumerate(lengths):
        keys = torch.arange(n, device=DEV)
        slots = table[i].long()[keys // page] * page + keys % page
        seen = keys[None] <= torch.arange(n - queries, n, device=DEV)[:, None]
        for h in range(q.shape[1]):
            g = h // (q.shape[1] // k.shape[2])
            kd, vd = (c.reshape(-1, *c.shape[2:])[slots, g].double() for c in (k, v))
            x = q[first:first + queries, h].double()
            s = (x @ kd.t().contiguous()) * q.shape[2] ** -0.5
            p = torch.softmax(s.masked_fill(~seen, -INF), dim=1)
            out[first:first + queries, h], size[first:first + queries, h] = p @ vd, p @ vd.abs()
            most[first:first + queries, h] = ((x.abs() @ kd.abs().t().contiguous()) * q.shape[2] ** -0.5).masked_fill(~seen, 0).amax(1, keepdim=True)
        first += queries
    return out, size, most


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,lengths", [(128, [(4500, 4100)]), (96, [(700, 700), (3000, 1100), (257, 256), (1, 1), (2600, 2500)])])
def test_blocks_of_256_rows(dtype, dim, lengths):
    b = Batch(10, lengths, heads=32, kv_heads=4, dim=dim, dtype=dtype)
    got = b.call()
    want, size, most = double_attention(b.q.to(DEV), b.k.to(DEV), b.v.to(DEV), lengths, b.table.to(DEV), 16)
    h, u = HALF_STEP[dtype], 2.0 ** -24
    e = (dim + 8) * u * most + 2.0 ** -22
    limit = size * (h + 2 * e + max(n for n, _ in lengths) * u) + want.abs() * h + 2.0 ** -24
    assert ((got.double() - want).abs() <= limit).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("extra", [{}, dict(softcap=20.0), dict(alibi_slopes=True)], ids=["plain", "capped", "sloped"])
def test_256_rows_of_codes_and_scores(dtype, fp8, extra):
    """Every form of 256 rows, against those of 128 rows and of few rows on the same numbers."""
    from sonar_amd import ops
    b = Batch(11, [(4200, 4100)], heads=32, kv_heads=4, dim=128, fp8=fp8, dtype=dtype)
    more = dict(extra)
    if "alibi_slopes" in more:
        more["alibi_slopes"] = torch.linspace(0.001, 0.5, 32, device=DEV)
    got = b.call(**more)
    d = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    for at in (0, 777, 2000, 4000):   # pieces of the same prompt: the queries up to there as a prompt of their own
        for queries in (1, 100):
            n = 100 + at + queries
            part = ops.paged_attention(d(b.q)[at:at + queries], d(b.k), d(b.v), d(b.table), d(torch.tensor([n], dtype=torch.int32)),
                                       d(torch.tensor([0, queries], dtype=torch.int32)), k_scale=d(b.k_scale), v_scale=d(b.v_scale), **more)
            # each is off by less than 2 h of the mean of |v| (see the head of the file) and h of itself: both by 6 h of the largest |v|
            most = b.v.float().abs().max() * (float(b.v_scale) if fp8 else 1.0)
            assert (part.double() - got[at:at + queries].double()).abs().max() <= 6 * HALF_STEP[dtype] * most


def test_a_cache_past_32_bits():
    """Pages that lie more than 2^32 elements, and 2^33 bytes, behind the cache's start."""
    from sonar_amd import ops
    pages, page, kv, dim = (1 << 32) // (16 * 2 * 128) + 40, 16, 2, 128
    k, v = (torch.zeros((pages, page, kv, dim), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    for lengths in ([(90, 1), (60, 2)], [(200, 60), (90, 90)]):
        b = Batch(12, lengths, heads=4, kv_heads=kv, dim=dim)
        k[-len(b.k):], v[-len(b.v):] = b.k.to(DEV), b.v.to(DEV)
        far = torch.where(b.table >= 0, b.table + pages - len(b.k), b.table)
        got = ops.paged_attention(b.q.to(DEV), k, v, far.to(DEV), b.lens.to(DEV), b.starts.to(DEV))
        assert torch.equal(got, b.call(max_seq_len=b.table.shape[1] * 16))
    del k, v
    torch.cuda.empty_cache()


def test_refusals_of_the_ops():
    from sonar_amd import ops
    b = Batch(13, [(40, 3)], heads=4, kv_heads=2, dim=64)
    d = lambda t: t.to(DEV)  # noqa: E731
    args = [d(b.q), d(b.k), d(b.v), d(b.table), d(b.lens), d(b.starts)]
    bad = [(0, args[0].float(), "float16"), (0, args[0][0], "query"), (0, args[0][:, :3], "multiple"), (1, args[1].half(), "type"),
           (2, args[2][:, :8], "one shape"), (1, args[1].repeat_interleave(2, 3)[..., ::2], "behind each other"), (3, args[3].long(), "block_table"), (3, args[3].repeat(2, 1), "block_table"),
           (4, args[4].long(), "seq_lens"), (5, args[5][:-1], "query_start_loc"), (5, b.starts, "query_start_loc")]
    for at, value, message in bad:
        with pytest.raises(RuntimeError, match=message):
            ops.paged_attention(*[value if i == at else a for i, a in enumerate(args)])
    one = torch.ones(1, device=DEV)
    for more, message in ((dict(k_scale=one, v_scale=one), "k_scale"), (dict(window=-1), "window"), (dict(softcap=-1.0), "cap"), (dict(scale=0.0), "scale"),
                          (dict(alibi_slopes=one), "alibi"), (dict(tree_mask=torch.zeros((3, 1), device=DEV)), "tree_mask"),
                          (dict(tree_mask=torch.zeros((3, 1), device=DEV, dtype=torch.int64), window=3), "tree"), (dict(window=3, causal=False), "window"),
                          (dict(out=torch.empty((3, 4, 64), device=DEV)), "out"), (dict(out=args[0]), "(?i)overlap|memory"),
                          (dict(out=torch.empty((3, 1, 64), device=DEV, dtype=torch.bfloat16).expand(3, 4, 64)), "(?i)overlap|memory"),
                          (dict(max_seq_len=-1), "max_seq_len")):
        with pytest.raises(RuntimeError, match=message):
            ops.paged_attention(*args, **more)
    fp8 = [a.to(FP8) if i in (1, 2) else a for i, a in enumerate(args)]
    with pytest.raises(RuntimeError, match="k_scale"):
        ops.paged_attention(*fp8)
    with pytest.raises(RuntimeError, match="k_scale"):
        ops.paged_attention(*fp8, k_scale=torch.ones(3, device=DEV), v_scale=one)
    narrow = torch.zeros((5, 16, 2, 68), device=DEV, dtype=torch.bfloat16)[..., :64]
    with pytest.raises(RuntimeError, match="16"):
        ops.paged_attention(args[0], narrow, narrow, *args[3:])


# ---------------------------------------------------------------- streams and graphs
def test_on_another_stream():
    b = Batch(14, [(900, 2), (500, 40)], dim=128)
    want = b.call()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [b.call() for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_graphs_that_share_a_pool():
    """Two captured calls, both with split keys, in one pool, replayed in turn with other lengths and numbers, eager calls between."""
    from sonar_amd import ops
    pool, held = torch.cuda.graph_pool_handle(), []
    for seed, lengths in ((1, [(3000, 1), (1000, 1)]), (2, [(2000, 50), (700, 30)])):
        b = Batch(seed, lengths, heads=4, kv_heads=1, dim=128)
        t = [x.to(DEV) for x in (b.q, b.k, b.v, b.table, b.lens, b.starts)]
        ops.paged_attention(*t)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            out = ops.paged_attention(*t).clone()
        held.append((graph, t, out))
    for turn in range(4):
        for graph, t, out in held:
            t[0].normal_()
            t[4].sub_(37)   # other lengths than at the capture
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, ops.paged_attention(*t)), turn
            torch.cuda.synchronize()


def test_the_same_bits_every_time():
    b = Batch(15, [(3000, 1), (800, 200), (90, 3)], dim=128)
    want = b.call()
    assert all(torch.equal(b.call(), want) for _ in range(5))


def test_opcheck():
    """Schema, fake results, no autograd formula, dynamic shapes: what the ops declare is what they do."""
    from sonar_amd import ops  # noqa: F401
    utils = ("test_schema", "test_autograd_registration", "test_faketensor", "test_aot_dispatch_dynamic")
    s = torch.ops.sonar_amd
    b = Batch(16, [(40, 3), (30, 1)], heads=4, kv_heads=2, dim=64)
    q, k, v, table, lens, starts = (x.to(DEV) for x in (b.q, b.k, b.v, b.table, b.lens, b.starts))
    for longest in (None, 40):
        args = (q, k, v, table, lens, starts, 0.125, True, 0, 0.0, None, None, None, None, longest)
        torch.library.opcheck(s.paged_attention, args, test_utils=utils)
        torch.library.opcheck(s.paged_attention_out, (*args, torch.zeros_like(q)), test_utils=utils)
    kv, at, cos_sin = torch.randn((4, 2, 64), device=DEV).bfloat16(), torch.arange(4, device=DEV), torch.randn((9, 64), device=DEV)
    w = torch.ones(64, device=DEV, dtype=torch.bfloat16)
    torch.library.opcheck(s.qk_norm_rope, (q, kv, at, cos_sin, w, w, 1e-6, True), test_utils=utils)
    torch.library.opcheck(s.qk_norm_rope, (q, kv, None, None, None, None, 1e-6, True), test_utils=utils)
    torch.library.opcheck(s.qk_norm_rope_append, (q, kv, kv, k, v, at, at, cos_sin, w, None, 1e-6, False, None, None), test_utils=utils)


def test_a_table_that_sequences_share():
    """One row of pages for all sequences, as a view without a copy: drafts of one prompt."""
    from sonar_amd import ops
    b = Batch(19, [(300, 1)], heads=4, kv_heads=2, dim=64)
    d = lambda t: t.to(DEV)  # noqa: E731
    q = torch.cat([b.q] * 5)
    lens, starts = torch.full((5,), 300, dtype=torch.int32), torch.arange(6, dtype=torch.int32)
    got = ops.paged_attention(d(q), d(b.k), d(b.v), d(b.table).expand(5, -1), d(lens), d(starts))
    assert torch.equal(got, ops.paged_attention(d(q), d(b.k), d(b.v), d(b.table.repeat(5, 1)), d(lens), d(starts)))
    b.check(got[:1])


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("seqs", [4, 70], ids=["few", "many"])
def test_starts_that_do_not_rise(seqs, fp8):
    """Not allowed, and then nothing is said of the results; but what lies around them is left alone, and the call ends."""
    rng = np.random.default_rng(20)
    for queries in (1, 30):
        b = Batch(20, [(200, queries)] * seqs, heads=4, kv_heads=2, dim=64, fp8=fp8)
        tokens = len(b.q)
        for starts in (rng.permutation(seqs + 1) * queries, np.full(seqs + 1, tokens), np.arange(seqs, -1, -1) * queries,
                       rng.integers(-1000, 1000, seqs + 1), rng.integers(-2 ** 31, 2 ** 31, seqs + 1)):
            b.starts = torch.from_numpy(starts.astype(np.int32))
            around = torch.full((tokens + 200, 4, 64), 7.0, dtype=torch.bfloat16, device=DEV)
            b.call(out=around[100:100 + tokens])
            assert (around[:100] == 7.0).all() and (around[100 + tokens:] == 7.0).all()


def test_lengths_known_only_on_the_device():
    """A table wide enough for any sequence, and lengths far below it, of one sequence and of more than a wavefront looks at."""
    for lengths in ([(700, 1)], [(3000, 1), (40, 1)], [(1200, 20), (900, 33)], [(40 + 13 * i, 1 + i % 3) for i in range(80)]):
        for fp8 in (False, True):
            b = Batch(21, lengths, heads=4, kv_heads=1, dim=128, fp8=fp8)
            b.check(b.call())
            b.table = torch.nn.functional.pad(b.table, (0, 8192 - b.table.shape[1]), value=-1)
            b.check(b.call())
            b.check(b.call(100))


def test_one_long_sequence_beside_prompts():
    """A single token with 40000 keys beside prompts that fill the card: its keys are split, and the last part is there."""
    from sonar_amd import ops
    lengths = [(400, 400)] * 12 + [(40000, 1)]
    b = Batch(25, lengths, heads=32, kv_heads=8, dim=128)
    got = b.call()
    alone = Batch(25, lengths, heads=32, kv_heads=8, dim=128)
    d = lambda t: t.to(DEV)  # noqa: E731
    one = ops.paged_attention(d(alone.q[-1:]), d(alone.k), d(alone.v), d(alone.table[-1:]), d(alone.lens[-1:]), d(torch.tensor([0, 1], dtype=torch.int32)))
    k = alone.k[alone.table[-1].long()].reshape(-1, 8, 128)[:40000].double().repeat_interleave(4, 1)
    v = alone.v[alone.table[-1].long()].reshape(-1, 8, 128)[:40000].double().repeat_interleave(4, 1)
    weights = (torch.einsum("hd,khd->hk", alone.q[-1].double(), k) * 128 ** -0.5).softmax(1)
    want, size = torch.einsum("hk,khd->hd", weights, v), torch.einsum("hk,khd->hd", weights, v.abs())
    h = HALF_STEP["bf16"]   # (the fp32 sums' share, 40000 keys of 2^-24, is 2^-8.7 of the mean of |v| in the worst order)
    limit = size * (h + 2.0 ** -8.7 + 2.0 ** -12) + want.abs() * h
    for x in (got[-1], one[0]):
        assert ((x.double().cpu() - want).abs() <= limit).all()
