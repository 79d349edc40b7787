"""The exact checks of tests/token_checks.py reject gradients and products with a planted mistake (no device)."""
import pytest
import torch

from tests import token_checks as tc
from tests.token_checks import BF16, F32


def _gradient(dout, ids, V, dtype, drop=None):
    """The gradient as a kernel would leave it, but for the sorted places `drop` of the ids."""
    d = dout.clone()
    if drop is not None:
        d[torch.sort(ids, stable=True).indices[drop]] = 0
    return tc.gradient_sums(d, ids, V).to(F32).to(dtype)


@pytest.mark.parametrize("T,V,E,kind", [(60001, 3000, 16, "one"), (49152, 2, 8, "uniform"), (20001, 999, 72, "one"),
                                        (2**20, 1000, 3, "zipf"), (30011, 50, 8, "runs")])
def test_gradient_check_sees_lost_tokens(T, V, E, kind):
    g = tc.gen(T)
    ids = tc.token_ids(kind, T, V, g)
    hot = int(torch.bincount(ids).argmax())
    first = int((torch.sort(ids).values == hot).nonzero()[0])
    n = int((ids == hot).sum())
    fills = [(tc.counting_dout, F32), (tc.walking_dout, F32), (tc.walking_dout, BF16)]
    for fill, dtype in fills:
        dout = fill(ids, E, g)
        assert torch.equal(dout.to(dtype).double(), dout)
        tc.check_gradient(_gradient(dout, ids, V, dtype), dout, ids, V)
        for a, b in ((0, n), (0, 1), (n - 1, n), (n // 2, n // 2 + 32), (32, 160), (n // 3, n // 3 + 128)):
            with pytest.raises(AssertionError):
                tc.check_gradient(_gradient(dout, ids, V, dtype, slice(first + a, first + b)), dout, ids, V)
