"""Attention of many rows over the 4-bit KV cache (ribn_b200.kvq4), where its kernel for them has several key tiles of 128 in one CTA, moves
its references late, or meets what no row may see.  Against the 64-bit reference (tests/kvq4_reference.py), whose keys and values are what the
arena stands for (read back as F32, which is exact); tolerances are those of tests/test_gpu_kvq4.py.

A sequence with more than 64 query rows per kv head takes that kernel (`_MANY`).  `max_keys`, a hint, chooses its form: as 1 a CTA has all of a pair
of query tiles' keys and converts the pages itself, with the true length the keys are shared among CTAs while they leave SMs idle, and
come expanded from the scratch; 75 kv heads leave no SM idle."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
from tests import kvq4_reference as R  # noqa: E402
from tests.test_gpu_kvq4 import TYPES, _check, _host, _rows, _tables  # noqa: E402

pytestmark = pytest.mark.gpu

_MANY = 65   # query rows per kv head


@pytest.fixture(scope="module")
def kvq4(built_library):
    from ribn_b200 import kvq4 as module
    return module


class _Cache:
    """An arena with rows k, v at its first slots, and the values that it stands for."""

    def __init__(self, kvq4, k, v, pages=None):
        rows, heads, d = k.shape
        self.pages = pages or (rows + 15) // 16
        self.bytes = kvq4.empty_cache(self.pages, heads, d)
        slots = torch.arange(self.pages * 16, dtype=torch.int32, device="cuda")
        kvq4.append(self.bytes, k, v, slots[:rows])
        self.k, self.v = (_host(x) for x in kvq4.read(self.bytes, slots, dtype=torch.float32))


def _attend(kvq4, cache, q, tables, lengths, cu, max_keys=None, window=0, scale=None, unit=0.0, check=True):
    cut = [b - a for a, b in zip(cu, cu[1:])]
    got = kvq4.attention(cache.bytes, q, torch.from_numpy(tables).cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                         torch.tensor(cu, dtype=torch.int32, device="cuda"), max_rows=max(cut), max_keys=max(lengths) if max_keys is None else max_keys,
                         window=window, scale=scale)
    if check:
        with np.errstate(invalid="ignore"):
            want, sizes = R.attention(cache.k, cache.v, cache.pages, _host(q), tables, lengths, cu, window, q.shape[2] ** -0.5 if scale is None else scale, np.zeros(q.shape))
        _check(got, want, sizes, q.dtype, unit)
    return got


@pytest.mark.parametrize("type_name", TYPES)
@pytest.mark.parametrize("heads,hint", [(1, 1), (1, 1000), (75, 1000)])
@pytest.mark.parametrize("step", [7.0, -7.0])
def test_scores_that_rise_from_keys_to_keys(kvq4, type_name, heads, hint, step):
    """Scores grow by 2^10 from every 32 keys to the next 32, so that a row's reference moves in both halves of a key tile, tile after tile, and what
    has been summed (results in tensor memory, this tile's earlier probabilities) is scaled again and again; rows of other signs and sizes beside them."""
    dtype, unit = TYPES[type_name]
    rng = np.random.default_rng(21)
    keys, d = 1000, 64
    k = rng.normal(0, 0.05, (keys, heads, d)).astype(np.float32)
    k[:, :, 5] = step * (np.arange(keys) // 32)[:, None]
    cache = _Cache(kvq4, torch.from_numpy(k).cuda(), _rows(rng, keys, heads, d, torch.float32))
    q = rng.normal(0, 1, (_MANY, heads, d)).astype(np.float32)
    q[:, :, 5] = rng.choice([4.0, 4.0, 4.0, 8.0, -4.0, 0.0, 1.0], (_MANY, heads))
    tables = rng.permutation(cache.pages).astype(np.int32)[None]
    # (pages anywhere, the scores by position: the reference's arrays lie by slot, as the arena does)
    order = torch.empty_like(cache.bytes)
    order[torch.from_numpy(tables[0]).long().cuda()] = cache.bytes
    at = (tables[0][:, None] * 16 + np.arange(16)).reshape(-1)
    cache.bytes = order
    cache.k, cache.v = (np.stack([x[i] for i in np.argsort(at)]) for x in (cache.k, cache.v))
    _attend(kvq4, cache, torch.from_numpy(q).to(dtype).cuda(), tables, [keys], [0, _MANY], max_keys=hint, scale=0.25, unit=unit)


@pytest.mark.parametrize("type_name", TYPES)
@pytest.mark.parametrize("heads,d,hint", [(1, 128, 1), (1, 64, 900), (75, 64, 900)])
def test_a_wait_that_runs_out_leaves_nan_and_nothing_else(kvq4, type_name, heads, d, hint):
    """Waits of no or a few polls: the call ends, a row is as it should be or NaN as a whole, rows of the other kernel and the next call know nothing
    of it.  Without a poll every row that sees a key is NaN."""
    from ribn_b200 import lib
    from ribn_b200._lib import KvQ4AttentionArgs
    dtype, _ = TYPES[type_name]
    rng = np.random.default_rng(22)
    lengths, counts = [900, 300, 40], [_MANY, 1, 100]   # (the last one's first 60 rows see nothing)
    cu = [0, *np.cumsum(counts).tolist()]
    k, v = _rows(rng, 80 * 16, heads, d, dtype), _rows(rng, 80 * 16, heads, d, dtype)
    cache, tables = kvq4.empty_cache(80, heads, d), _tables(rng, 80, lengths)
    kvq4.append(cache, k, v, torch.arange(80 * 16, dtype=torch.int32, device="cuda"))
    q = _rows(rng, cu[-1], heads, d, dtype)
    keep = [torch.from_numpy(tables).cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), torch.tensor(cu, dtype=torch.int32, device="cuda")]
    whole = kvq4.attention(cache, q, *keep, max_rows=100, max_keys=hint)
    assert torch.isfinite(whole).all() and not whole[cu[2]:cu[2] + 60].any()
    out = torch.empty_like(q)
    args = KvQ4AttentionArgs(cache.data_ptr(), 80, q.data_ptr(), out.data_ptr(), keep[0].data_ptr(), keep[1].data_ptr(), keep[2].data_ptr(), None, 0,
                             heads * d, heads * d, tables.shape[1], {"f32": 0, "f16": 1, "bf16": 2}[type_name], heads, heads, d, tables.shape[1], 3, cu[-1], 100, hint, 0, 0.0, 0)
    scratch = torch.empty(lib().ribn_b200_kvq4_workspace(args), dtype=torch.uint8, device="cuda")
    args.workspace, args.workspace_bytes = scratch.data_ptr(), scratch.numel()
    for polls in (0, 1, 2, 3, 5, 8, 20, 1 << 30):
        out.fill_(3.0)
        assert lib().ribn_b200_debug_kvq4_attention(0, torch.cuda.current_stream().cuda_stream, args, polls) == 0
        lost = torch.isnan(out).all(dim=2)
        assert torch.equal(out[~lost], whole[~lost])
        assert not lost[cu[1]].any()
        if polls == 0:
            assert lost[:_MANY].all() and lost[cu[2] + 60:].all()
        if polls == 1 << 30:
            assert not lost.any()
        assert torch.equal(kvq4.attention(cache, q, *keep, max_rows=100, max_keys=hint), whole)


@pytest.mark.parametrize("type_name", TYPES)
@pytest.mark.parametrize("rows,length", [(90, 90), (90, 400), (3, 3), (3, 400)])
@pytest.mark.parametrize("window,hint", [(0, 1), (0, 4000), (1, 1), (1, 4000), (2, 1), (30, 4000)])
def test_a_query_that_is_not_finite(kvq4, type_name, rows, length, window, hint):
    """NaN and infinities in queries: NaN wherever the row sees a key, be it one or all, zeros where it sees none, and nothing in other rows."""
    dtype, unit = TYPES[type_name]
    rng = np.random.default_rng(23)
    cache = _Cache(kvq4, _rows(rng, 450, 1, 64, torch.float32), _rows(rng, 450, 1, 64, torch.float32))
    tables = np.arange(cache.pages, dtype=np.int32)[None]
    tables[0, (length - rows) // 16 + 2] = -1   # in a window of one, sixteen rows see nothing
    q = _rows(rng, rows, 2, 64, dtype)
    for row, head, values in ((0, 0, [float("nan")]), (1, 1, [float("inf")]), (0, 1, [float("-inf")]), (2, 0, [float("inf"), float("-inf")]), (4, 0, [float("-inf")]),
                              (17, 1, [float("nan"), float("inf")]), (34, 0, [float("nan")]), (35, 1, [float("inf")]), (65, 0, [float("inf")]), (89, 1, [float("nan")])):
        if row < rows:
            q[row, head, 10:10 + len(values)] = torch.tensor(values).to(dtype)
    got = _attend(kvq4, cache, q, tables, [length], [0, rows], max_keys=hint, window=window, unit=unit)
    assert torch.isnan(got[0, 0]).all() and torch.isnan(got[1, 1]).all() and torch.isfinite(got[0, 1]).logical_not().all()
    if rows > 35 and window == 1 and (length - rows) % 16 == 0:
        assert not got[34, 0].any() and not got[35, 1].any()


def _far_ends(kvq4, dtype, unit, rows, d):
    """Scores so small that every key weighs the same, and so large that one key has all the weight, as queries and scale of the scores come near
    the ends of F32's range (and of the queries' type); masked keys beside them."""
    rng = np.random.default_rng(24)
    length = rows + 130
    cache = _Cache(kvq4, _rows(rng, length, 1, d, torch.float32), _rows(rng, length, 1, d, torch.float32))
    tables = np.arange(cache.pages, dtype=np.int32)[None]
    base = _rows(rng, rows, 2, d, torch.float32).clamp(-3, 3)
    for size, scale in ((1e-30, 1e-12), (1e-30, -1.2e-38), (1e-7, 1.2e-38), (1e-4, -1e-36), (0.0, 1.2e-38)):
        _attend(kvq4, cache, (base * size).to(dtype), tables, [length], [0, rows], scale=scale, unit=unit)
    seen = np.arange(length)[None] <= np.arange(length - rows, length)[:, None]
    for size, scale in ((1e38, 1.0), (1e38, -1e3), (1e38, 3.4e38), (2e4, 3.4e38), (1.0, -3.4e38), (1e-4, 3.4e38), (1e38, 1e-25)):
        q = (base * size).to(dtype)
        if not torch.isfinite(q).all():
            continue   # (F16 ends at 65,504)
        got = _host(_attend(kvq4, cache, q, tables, [length], [0, rows], scale=scale, check=False))
        x = np.einsum("rhd,kd->rhk", _host(q), cache.k[:length, 0]) * scale
        x = np.where(seen[:, None], x, -np.inf)
        order = np.argsort(x, axis=2)
        best, next_best = (np.take_along_axis(x, order[..., [i]], 2)[..., 0] for i in (-1, -2))
        clear = (best - next_best) > 2.0 ** -18 * np.max(np.abs(np.where(seen[:, None], x, 0.0)), axis=2)   # F32 sums of 128 products tell them apart
        assert clear.mean() > 0.9 and np.min((best - next_best)[clear]) > 100.0
        # one key's probability over itself: a polynomial exponential is off by less than 2^-13.7 in the sum, while its binary16 in the product is rounded back
        want = cache.v[:length, 0][order[..., -1]]
        allowed = np.abs(want) * (unit * (1 + 2.0 ** -8) + (2.0 ** -13.6 if dtype is not torch.float32 else 2.0 ** -19))
        assert np.all(np.abs(got - want)[clear] <= allowed[clear]), (size, scale)


@pytest.mark.parametrize("type_name", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_scores_of_a_chunk_at_the_ends_of_the_range(kvq4, type_name, d):
    _far_ends(kvq4, *TYPES[type_name], _MANY, d)


@pytest.mark.parametrize("type_name", TYPES)
@pytest.mark.parametrize("rows,d", [(1, 128), (5, 64), (3, 256), (20, 128)])
def test_scores_of_few_rows_at_the_ends_of_the_range(kvq4, type_name, rows, d):
    _far_ends(kvq4, *TYPES[type_name], rows, d)


def _poisoned(cache, seen):
    """The arena with NaN and infinite scales, and any codes, in every slot but `seen`."""
    d = cache.bytes.shape[2] // 18
    groups, out = d // 32, cache.bytes.clone()
    for slot in sorted(set(range(cache.pages * 16)) - set(seen)):
        page, j = divmod(slot, 16)
        at = torch.tensor([16 * d + (j * groups + G) * 2 for G in range(groups)] + [17 * d + ((j // 2) * groups + G) * 4 + j % 2 * 2 for G in range(groups)], device="cuda")
        out[page, :, at] = 0
        out[page, :, at + 1] = torch.tensor([0x7c, 0x7e, 0xfc, 0xff], dtype=torch.uint8, device="cuda").repeat(d // 32)[:len(at)]
    return out


@pytest.mark.parametrize("type_name", TYPES)
@pytest.mark.parametrize("heads,hint", [(1, 1), (1, 400), (75, 400)])
@pytest.mark.parametrize("window", [0, 37, 200])
def test_bytes_that_no_row_of_a_chunk_may_see_may_be_anything(kvq4, type_name, heads, hint, window):
    dtype, unit = TYPES[type_name]
    rng = np.random.default_rng(25)
    keys, d, rows = 390, 64, _MANY
    cache = _Cache(kvq4, _rows(rng, 448, heads, d, torch.float32), _rows(rng, 448, heads, d, torch.float32))
    tables = rng.permutation(cache.pages).astype(np.int32)[None]
    tables = np.concatenate([tables, tables[:, :2]], axis=1)   # (behind the last key: pages that are in use)
    q = _rows(rng, rows, heads, d, dtype)
    first = max(0, keys - rows + 1 - window) if window else 0
    clean = _attend(kvq4, cache, q, tables, [keys], [0, rows], max_keys=hint, window=window, unit=unit, check=heads == 1 or window == 37)
    cache.bytes = _poisoned(cache, [int(tables[0, p // 16]) * 16 + p % 16 for p in range(first, keys)])
    assert torch.equal(_attend(kvq4, cache, q, tables, [keys], [0, rows], max_keys=hint, window=window, check=False), clean)


@pytest.mark.parametrize("type_name", TYPES)
@pytest.mark.parametrize("hint", [1, 41])
def test_chunks_among_more_sequences_than_threads(kvq4, type_name, hint):
    """Four hundred sequences of none to forty keys, every tenth with twenty rows of four heads, the others with none or one."""
    dtype, unit = TYPES[type_name]
    rng = np.random.default_rng(26)
    cache = _Cache(kvq4, _rows(rng, 480, 1, 64, torch.float32), _rows(rng, 480, 1, 64, torch.float32))
    lengths = rng.integers(0, 41, 400).tolist()
    counts = [20 if i % 10 == 3 else i % 7 % 2 for i in range(400)]
    assert 20 * 4 >= _MANY
    wide = rng.integers(0, 30, (400, 5)).astype(np.int32)
    cu = [0, *np.cumsum(counts).tolist()]
    q = _rows(rng, cu[-1] + 5, 4, 64, dtype)
    got = _attend(kvq4, cache, q, wide[:, :3], lengths, cu, max_keys=hint, unit=unit)
    # the same out of a wider table
    at = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (lengths, cu)]
    assert torch.equal(kvq4.attention(cache.bytes, q, torch.from_numpy(wide).cuda()[:, :3], *at, max_rows=20, max_keys=hint), got)


@pytest.mark.parametrize("type_name", TYPES)
@pytest.mark.parametrize("heads,d,hint", [(1, 128, 1), (1, 64, 2100), (75, 64, 2100)])
@pytest.mark.parametrize("window", [0, 1300])
def test_many_key_tiles_in_one_cta(kvq4, type_name, heads, d, hint, window):
    """Seventeen key tiles behind one pair of query tiles, ten of a window, converted by the CTA, shared, or expanded; a second sequence beside it
    whose pages come behind the first one's."""
    dtype, unit = TYPES[type_name]
    rng = np.random.default_rng(27)
    lengths = [2100, 500]
    cache = _Cache(kvq4, _rows(rng, 2640, heads, d, torch.float32, 1.5), _rows(rng, 2640, heads, d, torch.float32))
    cu = [0, 140, 140 + _MANY] if heads == 1 else [0, _MANY, _MANY + 1]
    q = _rows(rng, cu[-1], heads, d, dtype, 1.5)
    _attend(kvq4, cache, q, _tables(rng, cache.pages, lengths), lengths, cu, max_keys=hint, window=window, unit=unit)


@pytest.mark.parametrize("rows", [5, 90])
def test_rows_beyond_the_most_stay_as_they_are(kvq4, rows):
    """`max_rows` below what a sequence has: its later rows are left alone, the earlier ones keep their positions."""
    rng = np.random.default_rng(28)
    cache = _Cache(kvq4, _rows(rng, 320, 2, 64, torch.float32), _rows(rng, 320, 2, 64, torch.float32))
    most, lengths, cu = rows - 3, [200, 90], [0, rows, rows + 2]
    tables = _tables(rng, cache.pages, lengths)
    q = _rows(rng, rows + 2, 4, 64, torch.float16)
    at = [torch.from_numpy(tables).cuda(), *(torch.tensor(x, dtype=torch.int32, device="cuda") for x in (lengths, cu))]
    out = torch.full_like(q, 5.0)
    kvq4.attention(cache.bytes, q, *at, max_rows=most, max_keys=200, out=out)
    want, sizes = R.attention(cache.k, cache.v, cache.pages, _host(q), tables, lengths, cu, 0, 0.125, np.zeros(q.shape))
    assert (out[most:rows] == 5.0).all()
    keep = [i for i in range(rows + 2) if not most <= i < rows]
    _check(out[keep], want[keep], [x[keep] for x in sizes], torch.float16, 2.0 ** -11)


@pytest.mark.parametrize("type_name", TYPES)
def test_a_mixed_call_captured_and_replayed_as_its_sequences_grow(kvq4, type_name):
    """A chunk beside single rows, captured once with a hint of 64 keys and replayed while lengths, rows per sequence and pages change, up to far more
    keys than the hint; another call's graph with the same tensors replayed between."""
    dtype, unit = TYPES[type_name]
    rng = np.random.default_rng(29)
    cache = _Cache(kvq4, _rows(rng, 1600, 2, 64, torch.float32), _rows(rng, 1600, 2, 64, torch.float32))
    q = _rows(rng, 75, 4, 64, dtype)
    tables, lengths, cu = (torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((3, 40), (3,), (4,)))
    outs, graphs = [torch.zeros_like(q) for _ in range(2)], [torch.cuda.CUDAGraph() for _ in range(2)]
    call = [lambda: kvq4.attention(cache.bytes, q, tables, lengths, cu, max_rows=72, max_keys=64, out=outs[0]),
            lambda: kvq4.attention(cache.bytes, q, tables, lengths, cu, max_rows=72, max_keys=640, window=50, out=outs[1])]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for c in call:
            c()
    torch.cuda.synchronize()
    for c, g in zip(call, graphs):
        with torch.cuda.graph(g, stream=side):
            c()
    for counts, sizes_of in (([72, 1, 2], [72, 9, 33]), ([1, 72, 0], [100, 500, 0]), ([1, 1, 72], [640, 1, 600]), ([30, 1, 40], [640, 640, 3]), ([0, 72, 3], [5, 71, 640])):
        t = rng.integers(0, cache.pages, (3, 40)).astype(np.int32)
        at = [0, *np.cumsum(counts).tolist()]
        for to, x in ((tables, t), (lengths, np.array(sizes_of, np.int32)), (cu, np.array(at, np.int32))):
            to.copy_(torch.from_numpy(x))
        q.copy_(_rows(rng, 75, 4, 64, dtype))
        before = [_host(o) for o in outs]
        for _ in range(2):
            for g in graphs:
                g.replay()
        for o, b, window in zip(outs, before, (0, 50)):
            want, sizes = R.attention(cache.k, cache.v, cache.pages, _host(q), t, sizes_of, at, window, 0.125, b)
            _check(o, want, sizes, dtype, unit)
    for g in graphs:
        g.reset()


@pytest.mark.parametrize("type_name", TYPES)
def test_a_long_range_loses_no_more_than_a_rounding(kvq4, type_name):
    """A chunk whose query tiles fill the GPU, behind 131,072 keys.  Each product of 16 keys cuts the sum it is added to at its last bit, so a sum over n keys
    in tensor memory comes out up to n / 16 x 2^-24 smaller: at most 2^-13 for the 32,768 keys that F16 and BF16 rows add up in one place, on top of what
    rounds either way (probabilities, exponentials, the result), which averages out over 200,000 values.  (Not for BF16 results: the weights e^x of normal x
    leave a standard deviation of sqrt(e / 131,072) = 4.6e-3 around 0.5, nine steps of F16 there but little more than one of BF16, 3.9e-3, whose roundings then go together.)"""
    dtype, unit = TYPES[type_name]
    keys, rows, heads, d = 131072, 1200, 16, 64
    rng = torch.Generator(device="cuda").manual_seed(30)
    cache, slots = kvq4.empty_cache(keys // 16, 1, d), torch.arange(keys, dtype=torch.int32, device="cuda")
    k, v = (torch.randn((keys, 1, d), generator=rng, device="cuda") for _ in range(2))
    kvq4.append(cache, k, v + 0.5, slots)
    k, v = (x[:, 0].double() for x in kvq4.read(cache, slots, dtype=torch.float32))
    q = torch.randn((rows, heads, d), generator=rng, device="cuda").to(dtype)
    at = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([keys], [0, rows])]
    got = kvq4.attention(cache, q, slots[:keys // 16][None], *at, max_rows=rows, max_keys=keys).double()
    some = torch.arange(0, rows, 6, device="cuda")
    x = torch.einsum("rhd,kd->rhk", q[some].double(), k) * d ** -0.5
    x.masked_fill_(slots[None, None] > (keys - rows + some)[:, None, None], -torch.inf)
    want = torch.einsum("rhk,kd->rhd", x.softmax(-1), v)
    off = got[some] - want
    less = -float((off * want).sum() / (want * want).sum())
    assert dtype is torch.bfloat16 or abs(less) < (2.0 ** -13 if dtype is torch.float16 else 2.0 ** -19), less
    assert float(off.norm() / want.norm()) < unit + (2.0 ** -13 if dtype is not torch.float32 else 2.0 ** -18)


@pytest.mark.parametrize("type_name", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hint", [1, 12000])
def test_many_small_probabilities_behind_a_large_one(kvq4, type_name, d, hint):
    """Three keys have e^17.5 = 2^25.2 times the probability of each of 12,000 others: added one by one to a sum in F32 these would all be lost, and
    together they are 1e-4 of it.  (Scores are exact: one dimension, of a few bits.)"""
    dtype, unit = TYPES[type_name]
    rng = np.random.default_rng(33)
    keys = 12000
    k = np.zeros((keys, 1, d), np.float32)
    k[[3, 200, 5000], 0, 5] = 17.5
    v = rng.normal(0.5, 0.5, (keys, 1, d)).astype(np.float32)
    cache = _Cache(kvq4, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda())
    q = np.zeros((_MANY, 2, d), np.float32)
    q[:, :, 5] = rng.choice([4.0, 3.75, 0.0, -4.0], (_MANY, 2))
    tables = np.arange(cache.pages, dtype=np.int32)[None]
    window = keys - 2000   # (the first rows see the key at 5,000 only, whatever the last ones see)
    for w in (0, window):
        _attend(kvq4, cache, torch.from_numpy(q).to(dtype).cuda(), tables, [keys], [0, _MANY], max_keys=hint, window=w, scale=0.25, unit=unit)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("heads,rows", [(4, 1), (4, 4)])
def test_many_small_probabilities_of_single_rows(kvq4, d, heads, rows):
    """The same for F32 rows of the other kernel, whose warps have 15,000 keys each (a hint of one key: one CTA for all).  Here scores are exact, so that what
    may be off is what probabilities as pairs and the sums' order leave (2^-19), and half a step of 2^-24 for each small probability, of the sum of three of 2^7."""
    rng = np.random.default_rng(34)
    keys = 60000
    k = np.zeros((keys, 1, d), np.float32)
    k[[3, 200, 5000], 0, 5] = 17.5
    v = rng.normal(0.5, 0.5, (keys, 1, d)).astype(np.float32)
    cache = _Cache(kvq4, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda())
    q = np.zeros((rows, heads, d), np.float32)
    q[:, :, 5] = 4.0
    q = torch.from_numpy(q).cuda()
    tables = np.arange(cache.pages, dtype=np.int32)[None]
    for hint in (1, keys):
        got = _attend(kvq4, cache, q, tables, [keys], [0, rows], max_keys=hint, scale=0.25, check=False)
        want, (weight, extent, _) = R.attention(cache.k, cache.v, cache.pages, _host(q), tables, [keys], [0, rows], 0, 0.25, np.zeros(q.shape))
        assert np.all(np.abs(_host(got) - want) <= weight * 2.0 ** -19 + extent * 2.0 ** -25 / (3 * 2.0 ** 7)), hint


@pytest.mark.parametrize("type_name", TYPES)
@pytest.mark.parametrize("rows,hint", [(_MANY, 1), (_MANY, 4000), (3, 4000)])
def test_a_row_of_one_key_has_its_value(kvq4, type_name, rows, hint):
    """However its probability is rounded: F16 rows have the cached value exactly, BF16 ones as it rounds, F32 ones but for the probability's rounding
    as a pair (2^-22) and those of the sum, the quotient and the result (2^-24 each)."""
    dtype, unit = TYPES[type_name]
    rng = np.random.default_rng(35)
    cache = _Cache(kvq4, _rows(rng, 200, 2, 128, torch.float32), _rows(rng, 200, 2, 128, torch.float32))
    tables = rng.permutation(cache.pages).astype(np.int32)[None]
    q = _rows(rng, rows, 4, 128, dtype, 2.0)
    got = _host(_attend(kvq4, cache, q, tables, [190], [0, rows], max_keys=hint, window=1, unit=unit))
    at = np.array([tables[0, p // 16] * 16 + p % 16 for p in range(190 - rows, 190)])
    want = cache.v[at][:, [0, 0, 1, 1]]
    if dtype is torch.float16:
        assert np.array_equal(got, want)
    else:
        assert np.all(np.abs(got - want) <= np.abs(want) * (unit * (1 + 2.0 ** -14) if dtype is torch.bfloat16 else 2.0 ** -21))
