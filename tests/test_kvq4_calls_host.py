"""Calls of the 4-bit KV cache that are refused, or sized, without a device."""

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
