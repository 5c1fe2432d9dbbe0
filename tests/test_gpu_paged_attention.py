"""GPU: attention over a paged cache against the 64-bit oracle.

Tolerances, with h half a step of the type (2^-8 bf16, 2^-11 fp16) and u = 2^-24.  A score's sum of head_dim exact products is off by
at most head_dim u sum|q k|, and by 8 roundings more of its own size (scale, scale of the codes, cap, slope, the exponent); a weight
by that much of itself and 2^-22 (the exponential), so by e = (head_dim + 8) u most + 2^-22 with the largest sum `most` of the row,
and h for its type.  The result is a mean with these weights: off by (h + 2 e + keys u) of the mean of |v|, and by its own rounding,
h of itself.  With a cap c the score passes tanh, formed from an exponential and a reciprocal of 2^-22 each: c 2^-20 more."""
import numpy as np
import pytest
import torch

from oracle import attention_oracle as ao

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}
FP8 = torch.float8_e4m3fn


def numbers(t):
    return t.detach().cpu().double().numpy()


class Batch:
    """A cache with sequences in it; lengths: (tokens, queries) of each."""

    def __init__(self, seed, lengths, heads=4, kv_heads=2, dim=64, page=16, dtype="bf16", fp8=False, tree_words=0, behind=0, scales=1):
        gen = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.dtype, self.lengths, self.dim = dtype, lengths, dim
        counts = [-(-n // page) for n, _ in lengths]
        pages = sum(counts) + 5
        cache = FP8 if fp8 else DTYPES[dtype]
        self.k, self.v = (torch.randn((pages, page, kv_heads, dim), generator=gen).mul_(4 if fp8 else 1).to(cache) for _ in range(2))
        self.k_scale = self.v_scale = None
        if fp8:
            self.k_scale, self.v_scale = torch.rand(scales, generator=gen) * 0.2 + 0.15, torch.rand(scales, generator=gen) * 0.2 + 0.1
        order = rng.permutation(pages)
        self.unused = order[sum(counts):]
        self.table = torch.full((len(lengths), max([*counts, 1])), -1, dtype=torch.int32)
        at = 0
        for i, count in enumerate(counts):
            self.table[i, :count] = torch.from_numpy(order[at:at + count].astype(np.int32))
            at += count
        self.starts = torch.tensor([0, *np.cumsum([q for _, q in lengths])], dtype=torch.int32)
        self.lens = torch.tensor([n for n, _ in lengths], dtype=torch.int32)
        self.q = (torch.randn((int(self.starts[-1]) + behind, heads, dim), generator=gen) * 1.5).to(DTYPES[dtype])
        self.tree = None
        if tree_words:
            words = rng.integers(-2 ** 63, 2 ** 63 - 1, size=(len(self.q), tree_words), dtype=np.int64)
            words[rng.random(len(words)) < 0.2] = 0   # some drafts see no draft, not even themselves
            self.tree = torch.from_numpy(words)

    def call(self, max_seq_len=None, out=None, **more):
        from sonar_amd import ops
        d = lambda t: None if t is None else t.to(DEV)  # noqa: E731
        return ops.paged_attention(d(self.q), d(self.k), d(self.v), d(self.table), d(self.lens), d(self.starts), tree_mask=d(self.tree),
                                   k_scale=d(self.k_scale), v_scale=d(self.v_scale), max_seq_len=max_seq_len, out=out,
                                   **{n: d(v) if isinstance(v, torch.Tensor) else v for n, v in more.items()})

    def want(self, scale=None, causal=True, window=0, softcap=0.0, alibi_slopes=None):
        k, v = numbers(self.k.float()), numbers(self.v.float())
        if self.k_scale is not None:
            k, v = (x * numbers(s)[:, None] for x, s in ((k, self.k_scale), (v, self.v_scale)))
        return ao.paged_attention(numbers(self.q), k, v, self.table.numpy(), self.lens.numpy(), self.starts.numpy(),
                                  self.dim ** -0.5 if scale is None else scale, causal, window, softcap,
                                  None if alibi_slopes is None else numbers(alibi_slopes), None if self.tree is None else self.tree.numpy())

    def limits(self, **more):
        want, size, most = self.want(**more)
        h, u = HALF_STEP[self.dtype], 2.0 ** -24
        e = (self.dim + 8) * u * most + 2.0 ** -22 + more.get("softcap", 0.0) * 2.0 ** -20
        keys = max([n for n, _ in self.lengths] + [1])
        return want, size * (h + 2 * e[:, :, None] + keys * u) + np.abs(want) * h + 2.0 ** -24

    def check(self, got, **more):
        want, limit = self.limits(**more)
        off = np.abs(numbers(got) - want)
        assert got.dtype == DTYPES[self.dtype] and (off <= limit).all(), (off.max(), (off / limit).max(), np.argwhere(~(off <= limit))[:5])


ONES = [(1, 1), (2, 1), (63, 1), (64, 1), (65, 1), (130, 1), (300, 1)]
PIECES = [(5, 5), (64, 64), (70, 33), (200, 7), (1, 1), (129, 128), (150, 150)]
EMPTY = [(3, 3), (0, 0), (0, 2), (17, 0), (40, 1), (2, 5)]   # no keys; no queries; fewer keys than queries


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dim", [16, 64, 80, 96, 128, 192, 256])
@pytest.mark.parametrize("lengths", [ONES, PIECES, EMPTY], ids=["ones", "pieces", "empty"])
def test_widths(dtype, fp8, dim, lengths):
    b = Batch(dim, lengths, dim=dim, dtype=dtype, fp8=fp8)
    b.check(b.call())


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (5, 5), (8, 1), (14, 2), (16, 16), (20, 4), (48, 1), (64, 8)])
@pytest.mark.parametrize("lengths", [ONES, PIECES[:4]], ids=["ones", "pieces"])
def test_heads(heads, kv_heads, lengths):
    b = Batch(heads, lengths, heads=heads, kv_heads=kv_heads, dim=64, scales=kv_heads, fp8=heads % 2 == 1)
    b.check(b.call())


@pytest.mark.parametrize("page", [1, 2, 3, 4, 7, 8, 16, 24, 48, 64, 100, 256])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_pages(page, fp8, dim):
    b = Batch(page, [(1, 1), (90, 1), (131, 40), (64, 64), (257, 1)], page=page, dim=dim, fp8=fp8)
    b.check(b.call())


EXTRAS = [dict(causal=False), dict(window=1), dict(window=5), dict(window=64), dict(window=100), dict(softcap=5.0), dict(softcap=30.0, window=33),
          dict(alibi_slopes=torch.tensor([0.5, 0.1, 0.01, 0.7])), dict(alibi_slopes=torch.tensor([0.5, 0.1, 0.01, 0.7]), causal=False),
          dict(alibi_slopes=torch.tensor([0.2, 0.1, 0.3, -0.1]), softcap=20.0, window=40), dict(scale=0.3)]


@pytest.mark.parametrize("extra", EXTRAS, ids=[",".join(e) for e in EXTRAS])
@pytest.mark.parametrize("dtype,dim,fp8", [("bf16", 128, False), ("fp16", 64, True), ("fp16", 256, False), ("bf16", 64, True)])
@pytest.mark.parametrize("lengths", [ONES, PIECES, EMPTY], ids=["ones", "pieces", "empty"])
def test_masks_and_scores(extra, dtype, dim, fp8, lengths):
    b = Batch(3, lengths, dim=dim, dtype=dtype, fp8=fp8)
    b.check(b.call(**extra), **extra)


@pytest.mark.parametrize("drafts,words", [(2, 1), (8, 1), (16, 1), (33, 1), (64, 1), (65, 2), (100, 2), (70, 1), (130, 3)])
@pytest.mark.parametrize("heads,kv_heads,dim,fp8,softcap", [(4, 2, 128, False, 0.0), (8, 1, 64, True, 0.0), (3, 3, 256, False, 20.0)])
def test_trees(drafts, words, heads, kv_heads, dim, fp8, softcap):
    lengths = [(drafts, drafts), (drafts + 1, drafts), (drafts + 63, drafts), (drafts + 200, drafts // 2), (drafts - 1, drafts), (300, 1)]
    b = Batch(drafts, lengths, heads=heads, kv_heads=kv_heads, dim=dim, fp8=fp8, tree_words=words)
    b.check(b.call(softcap=softcap), softcap=softcap)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lengths", [[(3000, 1)], [(2500, 20), (700, 1), (0, 1), (10, 10)], [(1500, 300)]], ids=["one", "mixed", "piece"])
@pytest.mark.parametrize("fp8", [False, True])
def test_split_keys(dim, lengths, fp8):
    """Few rows, many keys: parts of the keys in workgroups of their own; what max_seq_len says changes the parts only."""
    b = Batch(7, lengths, heads=4, kv_heads=1, dim=dim, fp8=fp8)
    for longest in (None, 1, 512, 3000, 100000):
        b.check(b.call(longest))
    b.check(b.call(3000, window=900), window=900)


def test_random_batches():
    rng = np.random.default_rng(5)
    for seed in range(40):
        lengths = []
        for _ in range(rng.integers(1, 9)):
            n = int(rng.integers(0, 400))
            lengths.append((n, int(rng.integers(0, n + 1)) if rng.random() < 0.6 else min(n, 1)))
        kv_heads = int(rng.integers(1, 4))
        b = Batch(seed, lengths, heads=kv_heads * int(rng.integers(1, 7)), kv_heads=kv_heads, dim=int(rng.choice([32, 64, 112, 128, 160])),
                  page=int(rng.integers(1, 70)), dtype=str(rng.choice(["bf16", "fp16"])), fp8=bool(rng.random() < 0.4))
        more = {}
        if rng.random() < 0.3:
            more["window"] = int(rng.integers(1, 300))
        if rng.random() < 0.3:
            more["softcap"] = 10.0
        if len(b.q):
            print(seed, lengths, more, flush=True)
            b.check(b.call(), **{}) if not more else b.check(b.call(**more), **more)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("extra", [{}, dict(softcap=30.0), dict(alibi_slopes=torch.tensor([0.5, 0.1, 0.01, 0.7]))], ids=["plain", "capped", "sloped"])
def test_every_form(dtype, dim, fp8, extra):
    """Few rows and many, whole and in parts that a wavefront or eight of them join, of every type, width, cache and score."""
    for lengths in (ONES, PIECES, [(3000, 1)], [(1500, 130)]):
        b = Batch(dim, lengths, kv_heads=1, dim=dim, dtype=dtype, fp8=fp8)
        b.check(b.call(**extra), **extra)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("lengths", [ONES, PIECES], ids=["few", "many"])
@pytest.mark.parametrize("cap", [128.0, 129.0, 5e3, 1e7, 1e30])
def test_large_caps(lengths, cap, fp8):
    """A cap far above the scores hardly changes them, and is not off by a share of itself either: from 129 on a score below an eighth
    of the cap is off by 2^-22 of itself (7 roundings of the series more), a larger one by 2^-22 of the cap, so by 2^-19 of itself."""
    b = Batch(17, lengths, kv_heads=2, dim=64, fp8=fp8)
    want, size, most = b.want(softcap=cap)
    h, u = HALF_STEP["bf16"], 2.0 ** -24
    e = (64 + 16) * u * most + 2.0 ** -22 + (cap * 2.0 ** -20 if cap <= 128 else most * 2.0 ** -19)
    keys = max(n for n, _ in lengths)
    limit = size * (h + 2 * e[:, :, None] + keys * u) + np.abs(want) * h + 2.0 ** -24
    assert (np.abs(numbers(b.call(softcap=cap)) - want) <= limit).all()
    if cap > 1e6:   # what is off by 2^-22 of the cap would not be near this
        assert np.abs(want - b.want()[0]).max() < 1e-6


@pytest.mark.parametrize("lengths", [ONES, PIECES], ids=["few", "many"])
@pytest.mark.parametrize("softcap", [0.0, 1e-30, 30.0])
def test_smallest_and_largest_scales(lengths, softcap):
    """Scores next to nothing, whose weights are all one, and a scale of the codes that is 0: means of what is seen."""
    b = Batch(18, lengths, kv_heads=2, dim=64, fp8=True)
    b.check(b.call(scale=1e-30, softcap=softcap), scale=1e-30, softcap=softcap)
    b.k_scale = torch.zeros(1)
    b.check(b.call(scale=1e30), scale=1e30)
    for bad in (-1.0, float("nan")):
        b.k_scale = torch.tensor([bad])
        got = b.call(softcap=softcap)
        seen = torch.cat([torch.arange(n - q, n) >= 0 for n, q in lengths if q]).to(DEV)
        assert got[seen].isnan().all()


# prompts, pieces of them and single tokens: many rows in all, few of some sequences
MIXED = [(150, 150), (700, 1), (300, 130), (9, 1), (260, 33), (520, 8), (129, 129), (64, 1), (200, 140), (33, 32), (0, 0), (321, 1)]


def parts_of_tails(b, kv_heads):
    """How many parts the last rows of a sequence get, from the scratch memory that is asked for (csrc/paged_attention.hip: 32 rows a
    sequence, kv head and part); 0 where none."""
    from sonar_amd import _lib
    lib = _lib.load_attention()
    size = lib.sonar_paged_attention_scratch_bytes(len(b.q), len(b.lengths), b.q.shape[1], kv_heads, b.dim, _lib.CACHE_FP8 if b.k_scale is not None else 1,
                                                   b.table.shape[1] * b.k.shape[1], 0)
    return size / (len(b.lengths) * kv_heads * 32 * (4 * b.dim + 8))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dim", [64, 112, 128, 256])
@pytest.mark.parametrize("extra", [{}, dict(softcap=20.0), dict(window=300), dict(causal=False), dict(alibi_slopes=torch.rand(64, generator=torch.Generator().manual_seed(1)))],
                         ids=["plain", "capped", "window", "all", "sloped"])
def test_few_rows_beside_many(dim, fp8, extra):
    """Workgroups enough without a split: only the last rows of each sequence, where they are few, are split over the keys."""
    b = Batch(22, MIXED, heads=64, kv_heads=64, dim=dim, fp8=fp8, behind=3)
    assert parts_of_tails(b, 64) in (2, 3, 4)
    got = b.call(**extra)
    b.check(got, **extra)
    assert torch.equal(got, b.call(**extra)) and (got[-3:] == 0).all()


@pytest.mark.parametrize("fp8", [False, True])
def test_few_rows_beside_many_trees(fp8):
    b = Batch(23, MIXED, heads=64, kv_heads=32, dim=128, fp8=fp8, tree_words=2)
    assert parts_of_tails(b, 32) in (2, 3, 4)
    b.check(b.call())


def test_few_rows_beside_many_specials():
    """An infinity and a NaN in the values of a sequence's last key, which the last query alone sees, and in a part of its own; a bad page."""
    b = Batch(24, MIXED, heads=64, kv_heads=64, dim=128)
    assert parts_of_tails(b, 64) >= 2
    clean = numbers(b.call())
    want, limit = b.limits()
    at = 519   # of the sixth sequence: 520 keys, 8 queries
    page = int(b.table[5, at // 16])
    b.v[page, at % 16, :, 3], b.v[page, at % 16, :, 5] = float("inf"), float("nan")
    got = numbers(b.call())
    last = int(b.starts[6]) - 1
    assert np.isposinf(got[last, :, 3]).all() and np.isnan(got[last, :, 5]).all()
    others = np.ones(got.shape, dtype=bool)
    others[last, :, 3], others[last, :, 5] = False, False
    assert (np.abs(got - want)[others] <= limit[others]).all()
    b.table[1, 20] = 10 ** 6   # a page of the second sequence
    got = numbers(b.call())
    assert np.isnan(got[150]).all() and not np.isnan(got[:150]).any() and np.isfinite(clean).all()
