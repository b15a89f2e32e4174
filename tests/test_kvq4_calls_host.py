"""Calls of the 4-bit KV cache that are refused, or sized, without a device."""

import random

import pytest

from tests.test_kvq4_host import _args, _why


@pytest.fixture(scope="module")
def lib(built_library):
    import ribn_b200
    return ribn_b200.lib()


def test_a_null_workspace_with_a_size_is_refused(lib):
    assert lib.ribn_b200_kvq4_attention(0, None, _args(workspace=None, workspace_bytes=1 << 20)) == -1
    assert "null workspace" in _why(lib)


def test_sizes_beyond_32_bits_are_not_cut_to_their_low_bits():
    from ribn_b200 import kvq4
    assert [kvq4._size(x, 50) for x in (0, 7, 50, 51, 2 ** 32 + 3, 2 ** 63 - 1)] == [0, 7, 50, 50, 50, 50]
    assert kvq4._size(-1, 50) == kvq4._size(-2 ** 32 + 5, 50) == -1
    with pytest.raises(TypeError):
        kvq4._size(None, 50)


def test_the_workspace_is_enough_on_every_device(lib):
    """A device plans with its own multiprocessors; more of them never need less, so that the most of the machine's devices decide."""
    rng = random.Random(5)
    for _ in range(400):
        d, kv = rng.choice([64, 128, 256]), rng.choice([1, 2, 8, 64])
        sequences, most = rng.choice([1, 3, 64, 500]), rng.choice([1, 4, 70, 2000])
        rows, pages = sequences * rng.randint(1, most), rng.choice([1, 9, 500, 8192])
        heads = kv * rng.choice([1, 4, 16])
        args = _args(type=rng.randint(0, 2), head_dim=d, kv_heads=kv, q_heads=heads, sequences=sequences, rows=rows, max_rows=min(most, rows), pages_per_sequence=pages,
                     table_stride=pages, max_keys=rng.randint(0, pages * 16), window=rng.choice([0, 0, 1000]), q_stride=heads * d, out_stride=heads * d)
        sizes = [lib.ribn_b200_debug_kvq4_workspace(args, sms) for sms in (1, 16, 74, 132, 148, 160, 592)]
        assert sizes == sorted(sizes), sizes
        assert lib.ribn_b200_kvq4_workspace(args) >= sizes[4]   # a B200's, which is also what a machine without a device is told


@pytest.mark.parametrize("change", [dict(sequences=1 << 28), dict(sequences=1 << 24, kv_heads=8, q_heads=128, rows=200, max_rows=4),
                                    dict(sequences=70000, head_dim=256, q_heads=16, kv_heads=1, rows=2000, max_rows=2000, q_stride=4096, out_stride=4096)])
def test_more_work_than_a_grid_has_is_refused_before_anything_is_enqueued(lib, change):
    args = _args(**change)
    assert lib.ribn_b200_kvq4_workspace(args) == 0
    assert lib.ribn_b200_kvq4_attention(0, None, args) == -1 and "too many" in _why(lib)
