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


def _product(x, codes, scales, K, group, planes=3, lose=None):
    """x W^T as the kernel makes it: planes of 8 significant bits, a group's sum scaled in fp32; `lose` = (from, to) of K."""
    q = torch.stack((codes & 15, codes >> 4), 2).reshape(codes.shape[0], -1)[:, :K].float() - 8
    if lose is not None:
        q[:, lose[0]:lose[1]] = 0
    parts, rest = [], x.float()
    for _ in range(planes):
        cut = (rest.view(torch.int32) & -65536).view(F32)
        parts.append(cut)
        rest = rest - cut
    y = torch.zeros(x.shape[0], codes.shape[0])
    for i, a in enumerate(range(0, K, group)):
        b = min(K, a + group)
        acc = torch.zeros_like(y)
        for part in reversed(parts):
            acc = acc + part[:, a:b] @ (q[:, a:b] / 16).t()
        y = y + scales[:, i] * acc
    return y * 16


@pytest.mark.parametrize("M,N,K,group", [(20, 96, 2240, 64), (64, 100, 2048, 32), (50, 60, 2041, 128), (1, 1, 1, 32)])
def test_product_checks_see_lost_planes_and_lost_columns(M, N, K, group):
    g = tc.gen(M + N + K)
    codes, scales = tc.w4_weight(N, K, group, "powers", g)
    codes[:, 0] |= 9                                          # k = 0 has a code that is not zero in every column
    W = tc.w4_values(codes, scales, K, group)
    x = tc.whole_rows(M, K, g)
    x[:, 0] = 3
    for dtype in (F32, BF16):
        tc.check_rounded(_product(x, codes, scales, K, group).to(dtype), x @ W.t())
    with pytest.raises(AssertionError):
        tc.check_rounded(_product(x, codes, scales, K, group, lose=(0, 1)), x @ W.t())
    one = torch.full_like(scales, 0.25)
    W1 = tc.w4_values(codes, one, K, group)
    x = tc.three_plane_rows(M, K, g)
    tc.check_rounded(_product(x, codes, one, K, group), x @ W1.t())
    codes2, any_ = codes | 0x11, tc.w4_weight(N, K, group, "any", g)[1]
    W2 = tc.w4_values(codes2, any_, K, group)
    ks = torch.randint(0, K, (M,), generator=g)
    s = tc.single_rows(ks, K, g)
    tc.check_single(_product(s, codes2, any_, K, group), s, W2)
    for planes in (1, 2):
        with pytest.raises(AssertionError):
            tc.check_rounded(_product(x, codes, one, K, group, planes), x @ W1.t())
        with pytest.raises(AssertionError):
            tc.check_single(_product(s, codes2, any_, K, group, planes), s, W2)
    with pytest.raises(AssertionError):
        tc.check_single(_product(s, codes2, any_, K, group, lose=(int(ks[0]), int(ks[0]) + 1)), s, W2)
    r = torch.randn(M, K, generator=g).double()
    tc.check_groups(_product(r, codes2, any_, K, group), r, W2, group, 3)
    tc.check_groups(_product(r.to(BF16).double(), codes2, any_, K, group).to(BF16), r.to(BF16).double(), W2, group, 1)
    if K > 1:
        with pytest.raises(AssertionError):
            tc.check_groups(_product(r, codes2, any_, K, group, lose=(0, 32)), r, W2, group, 3)
