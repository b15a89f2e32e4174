"""The 4-bit KV cache on the GPU (ribn_b200.kvq4) against its definition in 64 bits (tests/kvq4_reference.py).

Tolerances.  Writing and reading are exact.  Attention on F16 and BF16 rows rounds each probability to binary16 (2^-11 of it) and
the result to its type; F32 rows carry probabilities as pairs (2^-22), and a warp's sum of at most 32 products per value is cut by
2^-24 of itself each time.  A score of partial sums up to `reach` (scale sum |q k|) is off by at most a few 2^-24 of it, which moves
a probability by that share; 2^-20 covers sixteen such cuts, the two approximate exponentials (2^-22 each) and the sums' order.  So an element may be
off by  weight x (2^-11 or 2^-19, + (reach + 4) x 2^-20) + |result| x half a step of the type,  weight = sum p |v|.
Below the normal range binary16 has steps of 2^-24, whose half is off however small the probability: the largest is held at 2^6
or more (2^7, where the reference is not rounded up to an integer), so each may be off by 2^-25 / 2^6 = 2^-31 of the largest, which is at
most the sum they are divided by: + 2^-31 x sum |v|.
Many F16 or BF16 rows have a quarter of their exponentials from a polynomial of degree 3, whose largest relative error over its
interval is 7.48e-5 (found as the equal ripple of Remez's exchange) < 2^-13.7, so a probability there may be off by (1 + 2^-11)(1 + 2^-13.7) - 1
< 2^-11 + 2^-13.6: weight x 2^-13.6 more."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
from tests import kvq4_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu

TYPES = {"f32": (torch.float32, 2.0 ** -24), "f16": (torch.float16, 2.0 ** -11), "bf16": (torch.bfloat16, 2.0 ** -8)}


@pytest.fixture(scope="module")
def kvq4(built_library):
    from ribn_b200 import kvq4 as module
    return module


def _host(x):
    return x.detach().double().cpu().numpy()


def _rows(rng, n, heads, d, dtype, spread=1.0):
    x = torch.from_numpy(rng.normal(0, spread, (n, heads, d)).astype(np.float32))
    return x.to(dtype).cuda()


def _filled(kvq4, rng, pages, heads, d):
    """An arena whose every slot has a row, on the device and as the reference's."""
    arena = R.Arena(pages, heads, d)
    k, v = _rows(rng, pages * 16, heads, d, torch.float32), _rows(rng, pages * 16, heads, d, torch.float32, 0.7)
    cache = kvq4.empty_cache(pages, heads, d)
    slots = torch.arange(pages * 16, dtype=torch.int32, device="cuda")
    kvq4.append(cache, k, v, slots)
    arena.append(_host(k), _host(v), range(pages * 16))
    return cache, arena


def _check(got, want, sizes, dtype, unit):
    weight, extent, reach = sizes
    p = 2.0 ** -19 if dtype is torch.float32 else 2.0 ** -11 + 2.0 ** -13.6
    tolerance = weight * (p + (reach[:, :, None] + 4) * 2.0 ** -20) + extent * 2.0 ** -31 + np.abs(want) * unit * (1 + 2.0 ** -8) + 1e-7 * (dtype is torch.float16) + 1e-30
    lost = np.isnan(want)   # an infinite query's rows: NaN by the formula, here too
    assert np.array_equal(lost, np.isnan(_host(got)))
    off, tolerance = np.where(lost, 0.0, np.abs(_host(got) - want)), np.where(lost, 1.0, tolerance)
    worst = float(np.max(off / tolerance)) if off.size else 0.0
    assert worst <= 1.0, f"{worst} of what is allowed at {np.unravel_index(np.argmax(off / tolerance), off.shape)}"


# ---- writing and reading ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("type_name", TYPES)
@pytest.mark.parametrize("rows,heads,d", [(1, 8, 128), (19, 2, 64), (37, 3, 128), (5, 1, 256), (300, 2, 64)])
def test_written_bytes_and_values_are_the_definitions(kvq4, rows, heads, d, type_name):
    dtype = TYPES[type_name][0]
    rng = np.random.default_rng(rows * d)
    pages = rows // 16 + 3
    k, v = _rows(rng, rows, heads, d, dtype), _rows(rng, rows, heads, d, dtype, 30.0)
    # NaN and infinities (these in a row of their own: the last), a group of zeros, a tie of two signs, values too large and too small for a scale
    v[0, 0, 0:32] = 0.0
    k[0, 0, 5], k[0, 0, 11] = 9.0, -9.0
    k[0, 0, 33] = float("nan")
    k[-1, -1, 40], v[-1, -1, 3], v[-1, -1, 4] = float("inf"), float("-inf"), float("inf")
    if type_name != "f16":
        v[rows // 2, 0, 32:64] *= 1000.0
    v[rows // 2, -1, d - 32:] *= 1e-6
    slots = rng.permutation(pages * 16)[:rows]
    slots[rows // 3] = -1 if rows > 4 else slots[rows // 3]
    if rows > 10:
        slots[7] = pages * 16   # outside: not written
    cache = kvq4.empty_cache(pages, heads, d)
    at = torch.tensor(slots, dtype=torch.int32, device="cuda")
    kvq4.append(cache, k, v, at)
    arena = R.Arena(pages, heads, d)
    arena.append(_host(k), _host(v), slots)
    assert np.array_equal(cache.cpu().numpy(), arena.bytes)
    for out_name, (out_dtype, _) in TYPES.items():
        got_k, got_v = kvq4.read(cache, at, dtype=out_dtype)
        for got, values in ((got_k, arena.k), (got_v, arena.v)):
            want = np.where(((slots >= 0) & (slots < pages * 16))[:, None, None], values[np.clip(slots, 0, pages * 16 - 1)], 0.0)
            assert torch.equal(got.cpu().double(), torch.from_numpy(want).to(out_dtype).double()), out_name


def test_append_takes_strided_and_unaligned_rows(kvq4):
    rng = np.random.default_rng(3)
    wide = _rows(rng, 21, 5, 64, torch.float16)
    flat = torch.zeros(21 * 2 * 64 + 1, dtype=torch.float16, device="cuda")
    odd = flat[1:].view(21, 2, 64)   # two bytes off a 16-byte border
    odd.copy_(wide[:, :2])
    slots = torch.randperm(64, device="cuda")[:21].to(torch.int32)
    caches = [kvq4.empty_cache(4, 2, 64) for _ in range(3)]
    kvq4.append(caches[0], wide[:, 1:3], wide[:, 3:5], slots)
    kvq4.append(caches[1], wide[:, 1:3].contiguous(), wide[:, 3:5].contiguous(), slots)
    assert torch.equal(caches[0], caches[1])
    kvq4.append(caches[2], odd, odd, slots)
    kvq4.append(caches[0], wide[:, :2].contiguous(), wide[:, :2].contiguous(), slots)
    assert torch.equal(caches[2], caches[0])


def test_a_row_leaves_its_neighbours_in_the_page_alone(kvq4):
    rng = np.random.default_rng(4)
    cache, arena = _filled(kvq4, rng, 3, 2, 128)
    k, v = _rows(rng, 1, 2, 128, torch.bfloat16), _rows(rng, 1, 2, 128, torch.bfloat16)
    kvq4.append(cache, k, v, torch.tensor([21], dtype=torch.int32, device="cuda"))
    arena.append(_host(k), _host(v), [21])
    assert np.array_equal(cache.cpu().numpy(), arena.bytes)


def test_read_slots_may_repeat_and_nothing_is_a_call(kvq4):
    rng = np.random.default_rng(5)
    cache, arena = _filled(kvq4, rng, 2, 1, 256)
    slots = torch.tensor([3, 3, 31, -7, 3, 32], dtype=torch.int32, device="cuda")
    k, v = kvq4.read(cache, slots, dtype=torch.float32)
    want = np.stack([arena.v[3], arena.v[3], arena.v[31], 0 * arena.v[0], arena.v[3], 0 * arena.v[0]])
    assert np.array_equal(_host(v), want) and not k[3].any() and not k[5].any()
    k, v = kvq4.read(cache, slots[:0])
    assert k.shape == (0, 1, 256)
    kvq4.append(cache, k, v, slots[:0])


# ---- attention ----------------------------------------------------------------------------------------------------
def _call(kvq4, cache, arena, q, tables, lengths, cu, max_rows, max_keys=None, window=0, scale=None, out=None, unit=0.0):
    d = q.shape[2]
    total = q.shape[0]
    out = torch.full_like(q, 7.0) if out is None else out
    before = _host(out)
    got = kvq4.attention(cache, q, torch.from_numpy(tables).cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                         torch.tensor(cu, dtype=torch.int32, device="cuda"), max_rows=max_rows, max_keys=max(lengths) if max_keys is None else max_keys,
                         window=window, scale=scale, out=out)
    assert got is out and out.shape[0] == total
    want, sizes = R.attention(arena.k, arena.v, cache.shape[0], _host(q), tables, lengths, cu, window, d ** -0.5 if scale is None else scale, before)
    _check(out, want, sizes, q.dtype, unit)
    return out


def _tables(rng, pages, lengths, extra=1):
    order, width = rng.permutation(pages).astype(np.int32), max((n + 15) // 16 for n in lengths) + extra
    tables, first = np.zeros((len(lengths), width), np.int32), 0
    for i, n in enumerate(lengths):
        count = (n + 15) // 16
        tables[i, :count] = order[first:first + count]
        first += count
    return tables


@pytest.mark.parametrize("type_name", TYPES)
@pytest.mark.parametrize("q_heads,kv_heads,d", [(2, 2, 64), (16, 8, 128), (4, 1, 128), (8, 1, 256), (16, 1, 64), (32, 2, 128), (16, 1, 256), (6, 2, 128), (5, 5, 64)])
def test_single_rows_over_ragged_sequences(kvq4, q_heads, kv_heads, d, type_name):
    dtype, unit = TYPES[type_name]
    rng = np.random.default_rng(q_heads * d)
    lengths = [1, 16, 17, 0, 5, 90, 333]
    cache, arena = _filled(kvq4, rng, 36, kv_heads, d)
    q = _rows(rng, 9, q_heads, d, dtype, 2.0)   # two padding rows
    _call(kvq4, cache, arena, q, _tables(rng, 36, lengths), lengths, list(range(8)), 1, unit=unit)


@pytest.mark.parametrize("type_name", TYPES)
@pytest.mark.parametrize("window", [0, 1, 16, 50])
@pytest.mark.parametrize("q_heads,kv_heads,d", [(8, 2, 128), (3, 1, 64), (32, 2, 64), (2, 1, 256)])
def test_several_rows_and_windows(kvq4, q_heads, kv_heads, d, window, type_name):
    """Rows of one to forty per sequence, some before the sequence's first key, in blocks of columns that end inside a row."""
    dtype, unit = TYPES[type_name]
    rng = np.random.default_rng(q_heads + window)
    counts, lengths = [4, 1, 0, 7, 3, 40], [70, 33, 20, 7, 1, 130]
    cu = [0, *np.cumsum(counts).tolist()]
    cache, arena = _filled(kvq4, rng, 24, kv_heads, d)
    q = _rows(rng, cu[-1] + 1, q_heads, d, dtype)
    _call(kvq4, cache, arena, q, _tables(rng, 24, lengths), lengths, cu, 40, window=window, unit=unit)


@pytest.mark.parametrize("type_name", TYPES)
@pytest.mark.parametrize("d,keys", [(128, 3001), (64, 2000), (256, 1900)])
def test_long_ranges_are_split_and_joined(kvq4, d, keys, type_name):
    dtype, unit = TYPES[type_name]
    rng = np.random.default_rng(keys)
    pages = (keys + 15) // 16 + 1
    cache, arena = _filled(kvq4, rng, pages, 1, d)
    q = _rows(rng, 2, 4, d, dtype, 3.0)
    lengths = [keys, 9]
    out = _call(kvq4, cache, arena, q, _tables(rng, pages, lengths), lengths, [0, 1, 2], 1, unit=unit)
    # the split is the call's own: other hints, the same result but for the order of sums
    for hint in (1, 100, 100000):
        _call(kvq4, cache, arena, q, _tables(np.random.default_rng(1), pages, lengths), lengths, [0, 1, 2], 1, max_keys=hint, unit=unit)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("type_name", TYPES)
@pytest.mark.parametrize("counts,lengths,window,q_heads,kv_heads,d", [
    ([130], [130], 0, 4, 2, 128), ([64], [64], 0, 2, 1, 64), ([300], [1100], 0, 4, 1, 128), ([70, 1, 33, 0, 200], [700, 650, 33, 9, 260], 0, 4, 2, 64),
    ([150], [900], 100, 3, 1, 128), ([257], [300], 1, 2, 1, 64), ([150, 2], [100, 1], 0, 16, 1, 128)])
def test_prompt_chunks_beside_single_rows(kvq4, counts, lengths, window, q_heads, kv_heads, d, type_name):
    """Chunks alone, behind a prefix, over several blocks of rows and keys, longer than their sequence (the first rows see nothing), with
    windows that begin inside a block, and single rows and an empty sequence among them."""
    dtype, unit = TYPES[type_name]
    rng = np.random.default_rng(sum(counts))
    cu = [0, *np.cumsum(counts).tolist()]
    pages = sum((n + 15) // 16 for n in lengths) + 2
    cache, arena = _filled(kvq4, rng, pages, kv_heads, d)
    q = _rows(rng, cu[-1] + 3, q_heads, d, dtype, 1.5)
    _call(kvq4, cache, arena, q, _tables(rng, pages, lengths), lengths, cu, max(counts), window=window, unit=unit)


@pytest.mark.parametrize("rows", [1, 90])
def test_pages_outside_of_the_arena_hide_their_keys(kvq4, rows):
    rng = np.random.default_rng(8)
    cache, arena = _filled(kvq4, rng, 12, 2, 128)
    lengths = [150, 40]
    tables = _tables(rng, 12, [150, 32])
    tables[0, 3], tables[0, 9], tables[1, :] = -1, 12, 1 << 30
    q = _rows(rng, rows + 1, 8, 128, torch.float16)
    out = _call(kvq4, cache, arena, q, tables, lengths, [0, rows, rows + 1], rows, unit=2.0 ** -11)
    assert not out[rows].any()   # every page hidden


@pytest.mark.parametrize("rows", [1, 20])
def test_bytes_that_no_row_may_see_may_be_anything(kvq4, rows):
    """NaN and infinite scales behind the last key, in front of the window and in other pages."""
    rng = np.random.default_rng(9)
    cache, arena = _filled(kvq4, rng, 8, 1, 128)
    keys, window = 70, 37
    tables = np.array([[4, 2, 6, 1, 7, 0]], np.int32)
    q = _rows(rng, rows, 2, 128, torch.bfloat16)
    poisoned = cache.clone()
    seen = [int(tables[0, p // 16]) * 16 + p % 16 for p in range(keys - rows + 1 - window, keys)]
    for slot in set(range(128)) - set(seen):
        page, j = divmod(slot, 16)
        record = poisoned[page, 0]
        record[16 * 128 + j * 8:16 * 128 + j * 8 + 8] = 0x7e
        for G in range(4):
            at = 17 * 128 + ((j // 2) * 4 + G) * 4 + (j % 2) * 2
            record[at], record[at + 1] = 0x00, (0x7c if G % 2 else 0xff)
    outs = [_call(kvq4, c, arena, q, tables, [keys], [0, rows], rows, window=window, unit=2.0 ** -8) for c in (cache, poisoned)]
    assert torch.equal(*outs)


@pytest.mark.parametrize("type_name", TYPES)
def test_large_and_small_queries(kvq4, type_name):
    """Scores that leave one key, queries of the type's far ends, and a score scale of either sign."""
    dtype, unit = TYPES[type_name]
    rng = np.random.default_rng(10)
    cache, arena = _filled(kvq4, rng, 6, 2, 64)
    lengths, tables = [80, 80], np.array([[0, 1, 2, 3, 4], [5, 3, 1, 0, 2]], np.int32)
    base = _rows(rng, 2, 4, 64, torch.float32)
    for size, scale in ((1.0, -0.3), (2e4, 1e-4), (1e-3, 50.0), (1.0, 5.0)) + (((1e30, 2e-31), (1e-30, 1e29)) if type_name != "f16" else ()):
        q = (base * size).to(dtype)
        _call(kvq4, cache, arena, q, tables, lengths, [0, 1, 2], 1, scale=scale, unit=unit)
    _call(kvq4, cache, arena, torch.zeros_like(base).to(dtype), tables, lengths, [0, 1, 2], 1, unit=unit)


@pytest.mark.parametrize("type_name", TYPES)
def test_large_and_small_queries_of_a_chunk(kvq4, type_name):
    """The same where many rows take the other kernel."""
    dtype, unit = TYPES[type_name]
    rng = np.random.default_rng(15)
    cache, arena = _filled(kvq4, rng, 20, 1, 64)
    tables = np.array([rng.permutation(20)], np.int32)
    base = _rows(rng, 50, 2, 64, torch.float32)
    for size, scale in ((1.0, -0.3), (1e-3, 50.0), (1.0, 5.0), (1.0, -40.0)) + (((1e30, 2e-31), (1e-30, 1e29), (1e30, -1.0)) if type_name != "f16" else ()):
        q = (base * size).to(dtype)
        _call(kvq4, cache, arena, q, tables, [300], [0, 50], 50, scale=scale, unit=unit)


def test_an_infinite_query_spoils_its_own_row(kvq4):
    rng = np.random.default_rng(16)
    cache, arena = _filled(kvq4, rng, 20, 1, 128)
    tables = np.array([rng.permutation(20)], np.int32)
    for rows in (2, 60):
        q = _rows(rng, rows, 4, 128, torch.bfloat16)
        q[1, 2, 7], q[0, 3, 100] = float("inf"), float("nan")
        out = _call(kvq4, cache, arena, q, tables, [320], [0, rows], rows, unit=2.0 ** -8)
        lost = torch.isnan(out).all(dim=2)
        assert lost[1, 2] and lost[0, 3] and lost.sum() == 2


def test_more_sequences_than_threads(kvq4):
    """Four hundred sequences of no to forty keys, pages shared among them; every tenth brings ten rows (the other kernel)."""
    rng = np.random.default_rng(17)
    cache, arena = _filled(kvq4, rng, 30, 1, 64)
    lengths = rng.integers(0, 41, 400).tolist()
    counts = [10 if i % 10 == 3 else 1 for i in range(400)]
    cu = [0, *np.cumsum(counts).tolist()]
    tables = rng.integers(0, 30, (400, 3)).astype(np.int32)
    q = _rows(rng, cu[-1] + 5, 4, 64, torch.float16)
    _call(kvq4, cache, arena, q, tables, lengths, cu, 10, unit=2.0 ** -11)


@pytest.mark.parametrize("type_name", ["f32", "bf16"])
def test_less_scratch_gives_the_same_or_a_refusal(kvq4, type_name):
    """The C call with less and less scratch: the operands' part may be missing, what the sums need may not."""
    from ribn_b200 import lib
    from ribn_b200._lib import KvQ4AttentionArgs
    dtype, unit = TYPES[type_name]
    rng = np.random.default_rng(18)
    cache, arena = _filled(kvq4, rng, 50, 2, 128)
    counts, lengths = [40, 1, 60], [400, 90, 200]
    cu, tables = [0, 40, 41, 101], _tables(rng, 50, lengths)
    q = _rows(rng, 101, 4, 128, dtype)
    want, sizes = R.attention(arena.k, arena.v, 50, _host(q), tables, lengths, cu, 0, 128 ** -0.5, np.zeros(q.shape))
    keep = [torch.from_numpy(tables).cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), torch.tensor(cu, dtype=torch.int32, device="cuda")]
    out = torch.empty_like(q)
    args = KvQ4AttentionArgs(cache.data_ptr(), 50, q.data_ptr(), out.data_ptr(), keep[0].data_ptr(), keep[1].data_ptr(), keep[2].data_ptr(), None, 0,
                             512, 512, tables.shape[1], {"f32": 0, "bf16": 2}[type_name], 4, 2, 128, tables.shape[1], 3, 101, 60, 400, 0, 0.0, 0)
    need = lib().ribn_b200_kvq4_workspace(args)
    scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
    args.workspace = scratch.data_ptr()
    accepted = 0
    for size in (need, need - 300000, need * 3 // 4, need // 2, need // 4, need // 8, 0):
        args.workspace_bytes = size
        out.fill_(3.0)
        if lib().ribn_b200_kvq4_attention(0, torch.cuda.current_stream().cuda_stream, args) == 0:
            accepted += 1
            _check(out, want, sizes, dtype, unit)
        else:
            torch.cuda.synchronize()
            assert (out == 3.0).all()
    assert 2 <= accepted < 7


def test_two_streams_at_once(kvq4):
    rng = np.random.default_rng(19)
    cache, arena = _filled(kvq4, rng, 40, 2, 128)
    lengths, tables = [300, 250], _tables(rng, 40, [300, 250])
    device = [torch.from_numpy(tables).cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda")]
    work = []
    for rows in (1, 30, 2, 50):
        q = _rows(rng, 2 * rows, 8, 128, torch.bfloat16)
        work.append((q, rows, torch.tensor([0, rows, 2 * rows], dtype=torch.int32, device="cuda")))
    call = lambda q, rows, cu: kvq4.attention(cache, q, *device, cu, max_rows=rows, max_keys=300)  # noqa: E731
    alone = [call(*w) for w in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    for _ in range(20):
        outs = []
        for s, w in zip(streams, work):
            with torch.cuda.stream(s):
                outs.append(call(*w))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(alone, outs))


def test_strided_and_unaligned_queries_and_results(kvq4):
    rng = np.random.default_rng(11)
    cache, arena = _filled(kvq4, rng, 10, 2, 64)
    lengths, tables = [50, 66], _tables(rng, 10, [50, 66])
    whole = _rows(rng, 2, 12, 64, torch.float16)
    q, out = whole[:, 4:8], torch.zeros((2, 7, 64), dtype=torch.float16, device="cuda")
    _call(kvq4, cache, arena, q, tables, lengths, [0, 1, 2], 1, out=out[:, 1:5], unit=2.0 ** -11)
    assert not out[:, 0].any() and not out[:, 5:].any()
    flat, to = torch.zeros(2 * 4 * 64 + 1, dtype=torch.float16, device="cuda"), torch.zeros(2 * 4 * 64 + 3, dtype=torch.float16, device="cuda")
    odd = flat[1:].view(2, 4, 64)
    odd.copy_(q)
    _call(kvq4, cache, arena, odd, tables, lengths, [0, 1, 2], 1, out=to[3:].view(2, 4, 64), unit=2.0 ** -11)
    assert torch.equal(to[3:].view(2, 4, 64), out[:, 1:5])


def test_a_step_as_it_is_used_and_replayed(kvq4):
    """Prompt rows written, their attention, then decode steps of two sequences: written, attended, read back; the decode step
    captured once into a graph on another stream and replayed with new rows."""
    rng = np.random.default_rng(12)
    heads, kv, d, pages = 8, 2, 128, 24
    cache, arena = kvq4.empty_cache(pages, kv, d), R.Arena(pages, kv, d)
    tables = rng.permutation(pages).astype(np.int32).reshape(2, 12)
    prompts = [45, 130]
    slot = lambda s, p: int(tables[s, p // 16]) * 16 + p % 16  # noqa: E731
    for s, n in enumerate(prompts):
        k, v, q = _rows(rng, n, kv, d, torch.bfloat16), _rows(rng, n, kv, d, torch.bfloat16), _rows(rng, n, heads, d, torch.bfloat16)
        slots = [slot(s, p) for p in range(n)]
        kvq4.append(cache, k, v, torch.tensor(slots, dtype=torch.int32, device="cuda"))
        arena.append(_host(k), _host(v), slots)
        _call(kvq4, cache, arena, q, tables[s:s + 1], [n], [0, n], n, unit=2.0 ** -8)
    k, v, q = _rows(rng, 2, kv, d, torch.bfloat16), _rows(rng, 2, kv, d, torch.bfloat16), _rows(rng, 2, heads, d, torch.bfloat16)
    slots, lengths = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    cu, device_tables, out = torch.arange(3, dtype=torch.int32, device="cuda"), torch.from_numpy(tables).cuda(), torch.empty_like(q)

    def step():
        kvq4.append(cache, k, v, slots)
        return kvq4.attention(cache, q, device_tables, lengths, cu, max_rows=1, max_keys=192, out=out)

    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    slots.fill_(-1)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    assert not out.any()   # no keys yet: lengths of zero
    with torch.cuda.graph(graph, stream=side):
        step()
    for turn in range(20):
        k.copy_(_rows(rng, 2, kv, d, torch.bfloat16)); v.copy_(_rows(rng, 2, kv, d, torch.bfloat16)); q.copy_(_rows(rng, 2, heads, d, torch.bfloat16))
        at = [slot(s, n + turn) for s, n in enumerate(prompts)]
        slots.copy_(torch.tensor(at, dtype=torch.int32)); lengths.copy_(torch.tensor([n + turn + 1 for n in prompts], dtype=torch.int32))
        graph.replay()
        arena.append(_host(k), _host(v), at)
        want, sizes = R.attention(arena.k, arena.v, pages, _host(q), tables, [n + turn + 1 for n in prompts], [0, 1, 2], 0, d ** -0.5, np.zeros(q.shape))
        _check(out, want, sizes, q.dtype, 2.0 ** -8)
    got = kvq4.read(cache, torch.tensor([slot(1, p) for p in range(150)], dtype=torch.int32, device="cuda"), dtype=torch.float32)
    assert np.array_equal(_host(got[0]), arena.k[[slot(1, p) for p in range(150)]])
    graph.reset()


def test_results_do_not_depend_on_neighbours_or_repetition(kvq4):
    rng = np.random.default_rng(13)
    cache, _ = _filled(kvq4, rng, 40, 2, 128)
    lengths = [200, 31, 300]
    tables = _tables(rng, 40, lengths)
    q = _rows(rng, 3, 8, 128, torch.float32)
    run = lambda rows, t, n: kvq4.attention(cache, q[rows], torch.from_numpy(t).cuda(), torch.tensor(n, dtype=torch.int32, device="cuda"),  # noqa: E731
                                            torch.arange(len(n) + 1, dtype=torch.int32, device="cuda"), max_rows=1, max_keys=300)
    whole = run(slice(0, 3), tables, lengths)
    assert all(torch.equal(whole, run(slice(0, 3), tables, lengths)) for _ in range(3))
    moved = tables.copy()
    copied = cache.clone()
    spare = [p for p in range(40) if p not in set(tables[0, :13])][:1][0]
    copied[spare] = cache[int(tables[0, 2])]
    moved[0, 2] = spare
    assert torch.equal(kvq4.attention(copied, q[:1], torch.from_numpy(moved[:1]).cuda(), torch.tensor([200], dtype=torch.int32, device="cuda"),
                                      torch.arange(2, dtype=torch.int32, device="cuda"), max_rows=1, max_keys=300),
                       kvq4.attention(cache, q[:1], torch.from_numpy(tables[:1]).cuda(), torch.tensor([200], dtype=torch.int32, device="cuda"),
                                      torch.arange(2, dtype=torch.int32, device="cuda"), max_rows=1, max_keys=300))


def test_offsets_beyond_32_bits(kvq4):
    """A page whose record begins past 4 GB of the arena."""
    pages = (5 << 30) // (8 * 18 * 128)
    cache = torch.empty((pages, 8, 18 * 128), dtype=torch.uint8, device="cuda")
    rng = np.random.default_rng(14)
    keys, far = 40, [pages - 1, pages // 2, pages - 3]
    k, v, q = _rows(rng, keys, 8, 128, torch.float16), _rows(rng, keys, 8, 128, torch.float16), _rows(rng, 1, 16, 128, torch.float16)
    slots = torch.tensor([far[p // 16] * 16 + p % 16 for p in range(keys)], dtype=torch.int32, device="cuda")
    kvq4.append(cache, k, v, slots)
    arena = R.Arena(3, 8, 128)
    arena.append(_host(k), _host(v), range(keys))
    got = kvq4.read(cache, slots, dtype=torch.float32)
    assert np.array_equal(_host(got[0]), arena.k[:keys]) and np.array_equal(_host(got[1]), arena.v[:keys])
    out = kvq4.attention(cache, q, torch.tensor([far], dtype=torch.int32, device="cuda"), torch.tensor([keys], dtype=torch.int32, device="cuda"),
                         torch.tensor([0, 1], dtype=torch.int32, device="cuda"), max_rows=1, max_keys=keys)
    want, sizes = R.attention(arena.k, arena.v, 3, _host(q), np.array([[0, 1, 2]]), [keys], [0, 1], 0, 128 ** -0.5, np.zeros(q.shape))
    _check(out, want, sizes, q.dtype, 2.0 ** -11)


def test_refusals_of_the_python_calls(kvq4):
    cache = kvq4.empty_cache(4, 2, 64)
    rows = torch.zeros((3, 2, 64), dtype=torch.float16, device="cuda")
    slots = torch.zeros(3, dtype=torch.int32, device="cuda")
    for bad in (lambda: kvq4.append(cache.cpu(), rows, rows, slots), lambda: kvq4.append(cache, rows.double(), rows.double(), slots),
                lambda: kvq4.append(cache, rows, rows.float(), slots), lambda: kvq4.append(cache, rows, rows[:2], slots),
                lambda: kvq4.append(cache, rows, rows, slots[:2]), lambda: kvq4.append(cache, rows, rows, slots.long()),
                lambda: kvq4.append(cache, rows.transpose(1, 2), rows, slots), lambda: kvq4.append(cache, rows.cpu(), rows, slots),
                lambda: kvq4.append(cache, rows[:1].expand(3, 2, 64), rows, slots), lambda: kvq4.read(cache, slots, dtype=torch.float64),
                lambda: kvq4.read(cache[:, :, 1:], slots), lambda: kvq4.empty_cache(4, 2, 96)):
        with pytest.raises(ValueError):
            bad()
    q = torch.zeros((3, 4, 64), dtype=torch.float16, device="cuda")
    tables, lengths, cu = torch.zeros((3, 2), dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"), torch.arange(4, dtype=torch.int32, device="cuda")
    good = dict(max_rows=1, max_keys=32)
    for args, more in (((q[:, :3], tables, lengths, cu), good), ((q, tables[:2], lengths, cu), good), ((q, tables, lengths, cu[:3]), good),
                       ((q, tables.long(), lengths, cu), good), ((q, tables.t(), lengths, cu), good), ((q, tables, lengths, cu), dict(good, scale=0.0)),
                       ((q, tables, lengths, cu), dict(good, scale=float("nan"))), ((q, tables, lengths, cu), dict(good, scale=1e-50)), ((q, tables, lengths, cu), dict(good, scale=-1e39)), ((q, tables, lengths, cu), dict(good, out=q.float())),
                       ((q, tables, lengths, cu), dict(good, out=q[:2]))):
        with pytest.raises(ValueError):
            kvq4.attention(cache, *args, **more)
    with pytest.raises(RuntimeError, match="q_heads"):
        kvq4.attention(cache, torch.zeros((3, 34, 64), dtype=torch.float16, device="cuda"), tables, lengths, cu, **good)
    with pytest.raises(RuntimeError, match="negative"):
        kvq4.attention(cache, q, tables, lengths, cu, max_rows=1, max_keys=-1)
