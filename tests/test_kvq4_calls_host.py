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
