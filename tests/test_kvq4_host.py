"""The 4-bit KV cache without a device: the reference's byte order against the measured cases' one, and every refusal of the C
boundary, none of which reaches a device."""
import ctypes as C

import numpy as np
import pytest

from tests import kvq4_reference as R


@pytest.fixture(scope="module")
def lib(built_library):
    import ribn_b200
    return ribn_b200.lib()


def _why(lib):
    buf = C.create_string_buffer(512)
    lib.ribn_b200_op_last_error(buf, len(buf))
    return buf.value.decode()


CACHE, OTHER = 1 << 20, 1 << 21   # never looked at: refused before


@pytest.mark.parametrize("change,why", [
    (dict(type=3), "unknown type"), (dict(type=-1), "unknown type"), (dict(head_dim=96), "head_dim"), (dict(head_dim=32), "head_dim"),
    (dict(kv_heads=0), "kv_heads"), (dict(pages=0), "pages"), (dict(pages=1 << 27), "pages"), (dict(cache=None), "cache"), (dict(cache=CACHE + 8), "aligned"),
    (dict(rows=-1), "negative"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(slots=None), "null"), (dict(k=OTHER + 1), "aligned"),
    (dict(v=OTHER + 2), "aligned"), (dict(k_stride=1023), "stride"), (dict(v_stride=1023), "stride"), (dict(device=-1), "device"), (dict(device=64), "device"),
])
def test_append_refusals(lib, change, why):
    a = dict(device=0, cache=CACHE, pages=4, kv_heads=8, head_dim=128, type=0, k=OTHER, k_stride=1024, v=OTHER, v_stride=1024, slots=OTHER, rows=2)
    a.update(change)
    rc = lib.ribn_b200_kvq4_append(a["device"], None, a["cache"], a["pages"], a["kv_heads"], a["head_dim"], a["type"], a["k"], a["k_stride"],
                                   a["v"], a["v_stride"], a["slots"], a["rows"])
    assert rc == -1 and why in _why(lib)


@pytest.mark.parametrize("change,why", [
    (dict(type=3), "unknown type"), (dict(head_dim=0), "head_dim"), (dict(rows=-5), "negative"), (dict(k=None), "null"), (dict(v=OTHER + 8), "aligned"),
    (dict(slots=None), "null"), (dict(device=-1), "device"),
])
def test_read_refusals(lib, change, why):
    a = dict(device=0, cache=CACHE, pages=4, kv_heads=8, head_dim=128, type=1, k=OTHER, v=OTHER, slots=OTHER, rows=2)
    a.update(change)
    rc = lib.ribn_b200_kvq4_read(a["device"], None, a["cache"], a["pages"], a["kv_heads"], a["head_dim"], a["type"], a["slots"], a["rows"], a["k"], a["v"])
    assert rc == -1 and why in _why(lib)


def _args(**change):
    from ribn_b200._lib import KvQ4AttentionArgs
    a = dict(cache=CACHE, pages=64, q=OTHER, out=OTHER, page_tables=OTHER, lengths=OTHER, cu_rows=OTHER, workspace=None, workspace_bytes=0,
             q_stride=2048, out_stride=2048, table_stride=8, type=1, q_heads=16, kv_heads=8, head_dim=128, pages_per_sequence=8, sequences=3,
             rows=3, max_rows=1, max_keys=100, window=0, scale=0.0)
    a.update(change)
    return KvQ4AttentionArgs(**a)


@pytest.mark.parametrize("change,why", [
    (dict(type=7), "unknown type"), (dict(head_dim=80), "head_dim"), (dict(q_heads=12), "q_heads"), (dict(q_heads=136), "q_heads"), (dict(q_heads=0), "q_heads"),
    (dict(rows=-1), "negative"), (dict(sequences=-1), "negative"), (dict(max_keys=-1), "negative"), (dict(window=-1), "negative"), (dict(max_rows=4), "max_rows"),
    (dict(rows=1 << 28), "too large"), (dict(max_keys=2 ** 31 - 1), "too large"), (dict(pages_per_sequence=1 << 28), "too large"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(q=None), "null"), (dict(out=None), "null"), (dict(lengths=None), "null"),
    (dict(cu_rows=None), "null"), (dict(page_tables=None), "null"), (dict(q=OTHER + 1), "aligned"), (dict(out=OTHER + 1), "aligned"),
    (dict(q_stride=2047), "stride"), (dict(out_stride=100), "stride"), (dict(table_stride=7), "stride"), (dict(workspace=OTHER + 4), "aligned"),
    (dict(pages=0), "pages"), (dict(cache=None), "cache"),
])
def test_attention_refusals(lib, change, why):
    assert lib.ribn_b200_kvq4_attention(0, None, _args(**change)) == -1
    assert why in _why(lib)


def test_attention_without_an_argument_is_refused(lib):
    assert lib.ribn_b200_kvq4_attention(0, None, None) == -1 and "null" in _why(lib)
    assert lib.ribn_b200_kvq4_workspace(None) == 0


def test_nothing_to_do_is_not_an_error(lib):
    """Zero rows or sequences enqueue nothing and look at no pointer."""
    assert lib.ribn_b200_kvq4_append(0, None, CACHE, 4, 8, 128, 0, None, 0, None, 0, None, 0) == 0
    assert lib.ribn_b200_kvq4_read(0, None, CACHE, 4, 8, 128, 0, None, 0, None, None) == 0
    assert lib.ribn_b200_kvq4_attention(0, None, _args(rows=0, max_rows=0, q=None)) == 0
    assert lib.ribn_b200_kvq4_attention(0, None, _args(sequences=0, lengths=None)) == 0


def test_workspace_follows_the_call(lib):
    """Scratch for what CTAs share of an item, and for the operands of sequences with many rows; none where one CTA does all."""
    ask = lambda **change: lib.ribn_b200_kvq4_workspace(_args(**change))  # noqa: E731
    assert ask(sequences=1, rows=1, q_heads=1, kv_heads=1, max_keys=16) == 0
    small, long = ask(sequences=1, rows=1, max_keys=1024), ask(sequences=1, rows=1, max_keys=65536, pages_per_sequence=4096)
    assert 0 < small < long < 32 << 20
    # one sequence of 500 rows behind 1,000 keys: K and V of ten blocks of 128 keys as binary16, and no more than half a GB for any call
    assert ask(sequences=1, rows=500, max_rows=500, max_keys=1000) >= 8 * 8 * 128 * 128 * 4
    assert ask(sequences=64, rows=60000, max_rows=2000, max_keys=1 << 20) < 640 << 20


@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_the_two_descriptions_of_the_byte_order_agree(head_dim):
    """The arena written token by token (tests/kvq4_reference.py) is what the measured cases pack whole."""
    torch = pytest.importorskip("torch")
    import perf.operators as O
    rng = np.random.default_rng(head_dim)
    pages, heads = 2, 2
    arena = R.Arena(pages, heads, head_dim)
    codes = rng.integers(0, 16, (2, pages * 16, heads, head_dim)).astype(np.uint8)
    scales = rng.integers(-60, 60, (2, pages * 16, heads, head_dim // 32)) / 64.0
    for slot in range(pages * 16):
        arena.put(slot, codes[0, slot], scales[0, slot], codes[1, slot], scales[1, slot])
    to = lambda x, kind: torch.from_numpy(np.ascontiguousarray(x.reshape(pages, 16, heads, -1).transpose(0, 2, 1, 3)).astype(kind))  # noqa: E731
    packed = O._pack(to(codes[0], np.uint8), to(scales[0], np.float16), to(codes[1], np.uint8), to(scales[1], np.float16))
    assert np.array_equal(packed.numpy(), arena.bytes)


def test_the_quantiser_keeps_the_extreme_value_and_the_first_of_two():
    x = np.zeros((1, 1, 64))
    x[0, 0, 3], x[0, 0, 9], x[0, 0, 40] = 2.0, -2.0, -7.0
    codes, scales = R.quantise(x)
    assert scales[0, 0, 0] == -0.25 and codes[0, 0, 3] == 0 and codes[0, 0, 9] == 15    # -(-2) / 0.25 = 8 is cut to 7
    assert scales[0, 0, 1] == 0.875 and codes[0, 0, 40] == 0 and codes[0, 0, 0] == 8
