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
             (131072, 1000, 1030, "runs"), (2**22, 1000, 3, "zipf"), (2**22 + 1, 1000, 3, "zipf"), (2**22, 7, 1, "one"),
             # the two-launch sort of larger tables, below and above where it begins, and where its counts end it
             (98303, 100000, 5, "zipf"), (98304, 100000, 5, "zipf"), (393215, 300000, 3, "zipf"),
             (393216, 300000, 3, "runs"), (3 * 2**20, 300000, 1, "zipf"), (2**22, 300000, 1, "zipf"),
             (2**22, 102400, 1, "runs")]


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


# each form of the products: 16 rows a workgroup with one, two and four column blocks, on 8 and 16 waves, K split over
# workgroups or not; 32 rows sharing their activations with one and two column blocks a wave, K split or not; 64 rows, K
# split or not; rows, columns and K that end inside a tile
PRODUCTS = [(1, 1, 1, 32), (15, 17, 33, 32), (1, 2048, 256, 64), (16, 992, 1100, 64), (48, 2100, 300, 128),
            (20, 4096, 2240, 64), (7, 7000, 1100, 32), (1, 30522, 768, 32), (16, 12000, 300, 64), (64, 4096, 8192, 128),
            (3, 100, 8000, 32), (1, 1000, 8192, 128), (16, 5000, 6200, 32), (8, 7000, 6200, 64), (20, 30522, 200, 64),
            (33, 30522, 768, 128), (150, 8193, 255, 64), (64, 16384, 2048, 32), (17, 24000, 4100, 64),
            (64, 7000, 8191, 32), (33, 8192, 8192, 128), (40, 65536, 2041, 128), (50, 65536, 2048, 64),
            (64, 12000, 8192, 64), (64, 12000, 8190, 32), (64, 21000, 4096, 128), (50, 21000, 4095, 32)]


@pytest.mark.parametrize("M,N,K,group", PRODUCTS)
def test_linear_w4_is_exact(dev, M, N, K, group):
    """Whole numbers through every form in both types, with either type of scale and a bias; fp32 rows whose second and
    third plane count; single values of 24 bits at many k."""
    g = tc.gen(M + N + K + group)
    codes, scales = tc.w4_weight(N, K, group, "powers", g)
    codes = codes.to(dev)
    W = tc.w4_values(codes, scales.to(dev), K, group)
    bias = torch.randint(-50, 50, (N,), generator=g).to(dev)
    x = tc.whole_rows(M, K, g).to(dev)
    want = x @ W.t()
    for sdt in (F32, BF16):
        w = ops.pack_w4(codes, scales.to(sdt).to(dev), K, group)
        for dtype in (F32, BF16):
            tc.check_rounded(ops.linear_w4(x.to(dtype), w), want)
            tc.check_rounded(ops.linear_w4(x.to(dtype), w, bias.float()), want + bias)
    scales = torch.full_like(scales, 0.25).to(dev)
    W = tc.w4_values(codes, scales, K, group)
    w = ops.pack_w4(codes, scales, K, group)
    x = tc.three_plane_rows(M, K, g).to(dev)
    tc.check_rounded(ops.linear_w4(x.float(), w), x @ W.t())
    scales = tc.w4_weight(N, K, group, "any", g)[1].to(dev)
    W = tc.w4_values(codes, scales, K, group)
    w = ops.pack_w4(codes, scales, K, group)
    for i in range(3):
        x = tc.single_rows(torch.randint(0, K, (M,), generator=g), K, g).to(dev)
        tc.check_single(ops.linear_w4(x.float(), w), x, W)
    for dtype, planes in ((F32, 3), (BF16, 1)):
        x = torch.randn(M, K, generator=g).to(dtype).to(dev)
        tc.check_groups(ops.linear_w4(x, w), x.double(), W, group, planes)


@pytest.mark.parametrize("M,N,K", [(16, 64, 256), (64, 16384, 2048), (64, 12000, 8192)])
def test_linear_w4_range(dev, M, N, K):
    """The ends of the range at which fp32 rows keep fp32 accuracy: 24-bit values of 2^-110, and rows of 2^121, whose
    groups sum up to 2^127 before a small scale."""
    g = tc.gen(K)
    codes = (tc.w4_weight(N, K, 128, "any", g)[0] | 0x11).to(dev)
    scales = torch.ones(N, -(-K // 128), device=dev)
    x = tc.single_rows(torch.randint(0, K, (M,), generator=g), K, g)
    x = (torch.sign(x) * torch.ldexp(2 * torch.frexp(x)[0].abs(), torch.tensor(-110))).to(dev)
    assert torch.equal(x.float().double(), x)
    tc.check_single(ops.linear_w4(x.float(), ops.pack_w4(codes, scales, K, 128)), x, tc.w4_values(codes, scales, K, 128))
    codes = torch.zeros_like(codes)                              # every weight is -8 times its scale
    w = ops.pack_w4(codes, scales * 2.0**-30, K, 128)
    x = torch.full((M, K), 2.0**121, device=dev)
    assert bool((ops.linear_w4(x, w) == -K * 2.0**94).all())
    assert bool((ops.linear_w4(-x.to(BF16), w) == torch.tensor(K * 2.0**94).to(BF16).to(dev)).all())
