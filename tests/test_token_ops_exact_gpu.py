"""The token operators on the device, on inputs for which fp32 arithmetic is exact (tests/token_checks.py): nothing here
has a tolerance that a lost token, part or plane could hide in."""
import pytest
import torch

from dasa_amd import ops
from tests import token_checks as tc
from tests.token_checks import BF16, F32

pytestmark = pytest.mark.gpu

# few tokens in one launch; the one-launch sort; the two-launch sort (49152 tokens on), both sides of its ends
GRADIENTS = [(20, 992, 256, "uniform"), (1600, 3000, 96, "zipf"), (4099, 1001, 257, "zipf"), (8192, 3, 300, "uniform"),
             (8192, 40, 9, "runs"), (8191, 300, 64, "runs"), (4097, 60000, 40, "one"), (8000, 9, 7, "zipf"),
             (8192, 2, 1030, "one"), (8193, 2, 8, "uniform"), (9000, 300000, 16, "zipf"), (20001, 999, 72, "one"),
             (33000, 40, 520, "zipf"), (49151, 60, 3, "runs"), (30011, 50, 260, "runs"), (49152, 2, 8, "uniform"),
             (60001, 3000, 16, "one"), (50001, 40, 72, "zipf"), (100003, 90, 24, "runs"), (131073, 300000, 8, "zipf"),
             (131072, 1000, 1030, "runs"), (2**22, 1000, 3, "zipf"), (2**22 + 1, 1000, 3, "zipf"), (2**22, 7, 1, "one")]


@pytest.mark.parametrize("T,V,E,kind", GRADIENTS)
def test_embedding_gradient_is_exact(dev, T, V, E, kind):
    """Every sum, with a padding id and added into a gradient, in both types and with both id types."""
    g = tc.gen(T + V + E)
    ids = tc.token_ids(kind, T, V, g)
    pad = int(ids[T // 2])
    old = torch.randint(-3, 4, (V, E), generator=g)
    d64, d32 = ids.to(dev), ids.to(torch.int32).to(dev)
    for fill, dtype in ((tc.counting_dout, F32), (tc.counting_dout, BF16), (tc.walking_dout, F32), (tc.walking_dout, BF16)):
        dout = fill(ids, E, g)
        d = dout.to(dtype).to(dev)
        tc.check_gradient(ops.embedding_bwd(d, d64, V), dout, ids, V)
        tc.check_gradient(ops.embedding_bwd(d, d32, V, scale=0.5, padding_idx=pad), dout, ids, V, scale=0.5, pad=pad)
        acc = old.to(dtype).to(dev)
        ops.embedding_bwd(d, d64, V, scale=2.0, out=acc, accumulate=True)
        tc.check_gradient(acc, dout, ids, V, scale=2.0, old=old)
        acc = old.to(dtype).to(dev)
        ops.embedding_bwd(d, d32, V, padding_idx=pad, out=acc, accumulate=True)
        tc.check_gradient(acc, dout, ids, V, pad=pad, old=old)
