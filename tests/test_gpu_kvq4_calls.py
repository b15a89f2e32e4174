"""Calls of ribn_b200.kvq4 as its documentation allows them: sizes of any magnitude, gradients, results in place."""
import sys

import numpy as np
import pytest

torch = pytest.importorskip("torch")
from tests.test_gpu_kvq4 import _rows, _tables  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kvq4(built_library):
    from ribn_b200 import kvq4 as module
    return module


class _Call:
    """Two sequences of `rows` rows each over a filled arena; `attention` with whatever a test changes."""

    def __init__(self, kvq4, rows=1, dtype=torch.float16, lengths=(150, 70), seed=31):
        rng = np.random.default_rng(seed)
        self.kvq4, self.rows = kvq4, rows
        self.cache = kvq4.empty_cache(16, 2, 64)
        self.k, self.v = _rows(rng, 256, 2, 64, dtype), _rows(rng, 256, 2, 64, dtype)
        self.slots = torch.arange(256, dtype=torch.int32, device="cuda")
        kvq4.append(self.cache, self.k, self.v, self.slots)
        self.q = _rows(rng, 2 * rows, 4, 64, dtype)
        self.tables = torch.from_numpy(_tables(rng, 16, list(lengths))).cuda()
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        self.cu = torch.tensor([0, rows, 2 * rows], dtype=torch.int32, device="cuda")

    def __call__(self, **change):
        a = dict(q=self.q, max_rows=self.rows, max_keys=150)
        a.update(change)
        return self.kvq4.attention(self.cache, a.pop("q"), self.tables, self.lengths, self.cu, **a)


@pytest.mark.parametrize("rows", [1, 40])
def test_sizes_beyond_32_bits(kvq4, rows):
    call = _Call(kvq4, rows)
    whole = call()
    for window in (150, 2 ** 31 - 1, 2 ** 32 + 100, sys.maxsize):
        assert torch.equal(call(window=window), whole), window
    assert not torch.equal(call(window=100), whole)
    assert torch.equal(call(max_rows=2 ** 32 + 1), call(max_rows=2 * rows))
    for keys in (2 ** 31 - 1, 2 ** 32, sys.maxsize):
        assert torch.allclose(call(max_keys=keys).float(), whole.float(), atol=4e-3), keys   # cut elsewhere: the order of sums
    for bad in (dict(window=-1), dict(window=-2 ** 32 + 5), dict(max_keys=-2 ** 32 + 5), dict(max_rows=-2 ** 32 + 1)):
        with pytest.raises(RuntimeError, match="negative"):
            call(**bad)


def test_a_query_that_wants_a_gradient_is_refused(kvq4):
    call = _Call(kvq4)
    whole = call()
    q = call.q.clone().requires_grad_()
    for change in (dict(q=q), dict(q=q * 2), dict(out=torch.zeros_like(call.q).requires_grad_())):
        with pytest.raises(ValueError, match="no backward"):
            call(**change)
    with torch.no_grad():
        assert torch.equal(call(q=q), whole)
    assert torch.equal(call(q=q.detach()), whole)
