"""The token operators on the device (dasa_amd.ops embedding / embedding_bwd, linear_w4, logit_rules) against plain
64-bit implementations. Every tolerance counts roundings: HALF[t] is half a step of type t relative to the value, each
fp32 operation adds at most 2^-24 of its result, and a sum of n terms at most (n - 1) 2^-24 sum |terms|."""
import math

import pytest
import torch

from dasa_amd import functional as DF
from dasa_amd import ops
from dasa_amd._lib import DasaError

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
HALF = {F32: 2.0**-24, BF16: 2.0**-8}
U = 2.0**-24


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _within(got, want, tol, what):
    got, want = got.detach().cpu().double(), want.cpu().double()
    bad = ~((got - want).abs() <= tol) & ~((got == want) | (got.isnan() & want.isnan()))
    assert not bool(bad.any()), (what, int(bad.sum()), got[bad][:4].tolist(), want[bad][:4].tolist())


# ------------------------------------------------------------------------------------------ embedding
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,V,E", [(1, 1, 1), (3, 5, 4), (20, 992, 256), (65, 7, 257), (1000, 301, 24), (4097, 50, 768),
                                   (9000, 1000, 1024)])
def test_embedding(dev, dtype, T, V, E):
    g = _gen(T + V + E)
    table = torch.randn(V, E, generator=g).to(dtype)
    ids = torch.randint(0, V, (T,), generator=g)
    for idt in (torch.int64, torch.int32):
        got = ops.embedding(ids.to(idt).to(dev), table.to(dev))
        assert torch.equal(got.cpu(), table[ids])                  # scale 1: the rows themselves
    got = ops.embedding(ids.to(dev), table.to(dev), scale=math.sqrt(E))
    want = table[ids].double() * torch.tensor(math.sqrt(E), dtype=F32).double()
    _within(got, want, want.abs() * (U + HALF[dtype] * (1 + U)), "embedding")


def test_embedding_shapes_strides_and_ids_outside(dev):
    g = _gen(1)
    wide = torch.randn(40, 100, generator=g).to(dev)
    table = wide[:, 10:74]                                         # row stride 100, rows 8-B aligned only
    ids = torch.randint(0, 40, (3, 5, 2), generator=g).to(dev)
    got = ops.embedding(ids.transpose(0, 1), table)
    assert got.shape == (5, 3, 2, 64) and torch.equal(got, table[ids.transpose(0, 1)])
    buf = torch.full((30, 70), 7.0, device=dev)
    out = ops.embedding(ids.reshape(-1), table, out=buf[:, 3:67])
    assert out.data_ptr() == buf[:, 3:67].data_ptr() and torch.equal(buf[:, 3:67], table[ids.reshape(-1)])
    assert bool((buf[:, :3] == 7).all()) and bool((buf[:, 67:] == 7).all())
    assert ops.embedding(ids[:0], table).shape == (0, 5, 2, 64)
    bad = torch.tensor([0, -1, 39, 40, -2**40, 2**40 + 1, 5], device=dev)
    ops.check_device_errors()
    got = ops.embedding(bad, table)
    assert torch.equal(got[[0, 2, 6]], table[[0, 39, 5]])
    assert bool((got[[1, 4]] == 0).all()) and bool(got[[3, 5]].isnan().all())
    with pytest.raises(DasaError, match="token id"):
        ops.check_device_errors()
    ops.check_device_errors()


def _bwd_reference(dout, ids, V, scale, pad):
    """(gradient, sum of magnitudes, terms) of every table entry, in 64 bits."""
    E = dout.shape[-1]
    d, i = dout.cpu().double().reshape(-1, E), ids.cpu().reshape(-1).long()
    keep = (i >= 0) & (i < V)
    if pad is not None:
        keep &= i != pad
    d, i = d[keep], i[keep]
    s = torch.tensor(scale, dtype=F32).double()
    z = torch.zeros(V, E, dtype=torch.float64)
    n = torch.bincount(i, minlength=V).double()[:, None]
    return z.index_add(0, i, d) * s, z.index_add(0, i, d.abs()) * s.abs(), n


def _check_bwd(got, dout, ids, V, scale, pad, dtype, what, old=None):
    want, mag, n = _bwd_reference(dout, ids, V, scale, pad)
    tol = mag * (n + 1) * U                                  # n - 1 additions, the scale, and one to spare
    if old is not None:
        want = want + old.cpu().double()
        tol = tol + (n > 0) * want.abs() * U
    tol = tol + HALF[dtype] * (want.abs() + tol)
    _within(got, want, tol, what)
    untouched = (n == 0).expand_as(want)
    ref = torch.zeros_like(want) if old is None else old.cpu().double()
    assert torch.equal(got.cpu().double()[untouched], ref[untouched])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,V,E,kind", [(1, 1, 1, "uniform"), (1, 300, 4, "uniform"), (63, 5, 8, "uniform"),
                                        (64, 64, 257, "one"), (65, 1000, 64, "one"), (700, 3, 100, "uniform"),
                                        (1600, 30522, 768, "zipf"), (4099, 1001, 257, "zipf"), (5000, 17, 16, "zipf"),
                                        (20000, 100, 256, "zipf"), (20001, 999, 72, "one"), (8192, 8192, 40, "perm"),
                                        (130, 300000, 8, "uniform"), (9000, 300000, 16, "zipf"),
                                        (8193, 2, 8, "uniform"), (33000, 40, 520, "zipf"),
                                        (49152, 2, 8, "uniform"), (60001, 3000, 16, "one"), (50001, 40, 72, "zipf"),
                                        (131073, 300000, 8, "zipf"), (70000, 70000, 4, "perm"),
                                        (2**22, 1000, 1, "zipf"), (2**22 + 1, 1000, 1, "zipf"),
                                        (8192, 3, 300, "uniform"), (4097, 60000, 40, "one"), (1601, 9000, 129, "one"),
                                        (513, 2, 3, "one"), (8000, 9, 7, "zipf"), (6000, 40, 1030, "zipf")])
def test_embedding_gradient(dev, dtype, T, V, E, kind):
    g = _gen(T * 3 + V + E)
    if kind == "uniform":
        ids = torch.randint(0, V, (T,), generator=g)
    elif kind == "one":                                      # every place the same id: one long run
        ids = torch.full((T,), V // 2)
    elif kind == "perm":
        ids = torch.randperm(V, generator=g)[:T]
    else:
        ids = (torch.pow(float(V), torch.rand(T, generator=g, dtype=torch.float64)).long() - 1).clamp(0, V - 1)
    dout = torch.randn(T, E, generator=g).to(dtype)
    got = ops.embedding_bwd(dout.to(dev), ids.to(dev), V, scale=1.5)
    assert got.shape == (V, E) and got.dtype == dtype
    _check_bwd(got, dout, ids, V, 1.5, None, dtype, "gradient")
    again = ops.embedding_bwd(dout.to(dev), ids.to(torch.int32).to(dev), V, scale=1.5)
    assert torch.equal(got, again)                           # bitwise reproducible, either id type
    pad = int(ids[0])
    _check_bwd(ops.embedding_bwd(dout.to(dev), ids.to(dev), V, padding_idx=pad), dout, ids, V, 1.0, pad, dtype, "pad")
    old = torch.randn(V, E, generator=g).to(dtype)
    acc = old.to(dev)
    ops.embedding_bwd(dout.to(dev), ids.to(dev), V, scale=0.5, out=acc, accumulate=True)
    _check_bwd(acc, dout, ids, V, 0.5, None, dtype, "accumulate", old=old)


def test_embedding_gradient_layouts_and_skipped_ids(dev):
    g = _gen(5)
    V, E = 50, 24
    ids = torch.randint(0, V, (6, 9), generator=g)
    ids[0, 0], ids[2, 3], ids[5, 8] = -1, V, 2**40
    wide = torch.randn(6, 9, 60, generator=g).to(dev)
    d = wide[..., 5:29]                                      # strided rows, not 16-B aligned
    _check_bwd(ops.embedding_bwd(d, ids.to(dev), V), d, ids, V, 1.0, None, F32, "strided")
    t = torch.randn(9, 6, E, generator=g).to(dev).transpose(0, 1)
    _check_bwd(ops.embedding_bwd(t, ids.to(dev), V), t, ids, V, 1.0, None, F32, "transposed")
    one = torch.randn(E, generator=g).to(dev).expand(6, 9, E)
    _check_bwd(ops.embedding_bwd(one, ids.to(dev), V), one, ids, V, 1.0, None, F32, "broadcast rows")
    buf = torch.full((V, 40), 3.0, device=dev)
    ops.embedding_bwd(d, ids.to(dev), V, out=buf[:, 8:32])
    _check_bwd(buf[:, 8:32], d, ids, V, 1.0, None, F32, "strided out")
    assert bool((buf[:, :8] == 3).all()) and bool((buf[:, 32:] == 3).all())
    z = ops.embedding_bwd(torch.empty(0, E, device=dev), torch.empty(0, dtype=torch.int64, device=dev), V)
    assert z.shape == (V, E) and bool((z == 0).all())
    z = ops.embedding_bwd(torch.ones(4, E, device=dev), torch.full((4,), 7, device=dev), V, padding_idx=7)
    assert bool((z == 0).all())


def test_embedding_offsets_past_32_bits(dev):
    """A table and a gradient of more than 2^31 elements: the last rows."""
    V, E = 2_200_003, 1024
    table = torch.empty(V, E, dtype=BF16, device=dev)
    ids = torch.tensor([0, V - 1, V - 2, V - 1, V // 2], device=dev)
    table[ids] = torch.randn(5, E, device=dev).to(BF16)
    assert torch.equal(ops.embedding(ids, table), table[ids])
    dout = torch.randn(5, E, device=dev).to(BF16)
    ops.embedding_bwd(dout, ids, V, out=table)
    assert torch.equal(table[V - 2], dout[2]) and torch.equal(table[0], dout[0]) and torch.equal(table[V // 2], dout[4])
    want = dout[1].double() + dout[3].double()
    _within(table[V - 1], want.cpu(), HALF[BF16] * want.abs().cpu() * (1 + 2 * U) + 2 * U * want.abs().cpu(), "last row")
    assert bool((table[1:1000] == 0).all()) and bool((table[V - 1000:V - 2] == 0).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_embedding_autograd(dev, dtype):
    g = _gen(9)
    table = torch.randn(31, 20, generator=g).to(dtype).to(dev).requires_grad_()
    ids = torch.randint(0, 31, (4, 11), generator=g).to(dev)
    dout = torch.randn(4, 11, 20, generator=g).to(dtype).to(dev)
    y = DF.embedding(ids, table, scale=2.0, padding_idx=3)
    assert y.requires_grad and torch.equal(y, ops.embedding(ids, table.detach(), scale=2.0))
    y.backward(dout)
    _check_bwd(table.grad, dout, ids, 31, 2.0, 3, dtype, "autograd")
    with torch.no_grad():
        assert not DF.embedding(ids, table).requires_grad
    # against differences of the formula: the lookup is linear, so a central difference is exact up to rounding
    if dtype == F32:
        t64 = table.detach().cpu().double()
        e = torch.zeros_like(t64)
        e[7, 3] = 1.0
        f = lambda t: float(((t[ids.cpu()] * 2.0) * dout.cpu().double()).sum())   # noqa: E731
        assert abs((f(t64 + e) - f(t64 - e)) / 2 - float(table.grad[7, 3])) < 1e-4


def test_embedding_in_a_captured_training_region(dev):
    """Forward and backward replayed as graphs on new ids, with an eager graph of the same table alive: the gradients
    are the eager ones, bit for bit."""
    from dasa_amd import graph
    g = _gen(21)
    emb = torch.nn.Embedding(300, 64).to(dev)
    region = graph.AutogradGraphs([emb])
    link = torch.zeros(1, device=dev, requires_grad=True)        # (regions are linked by an input that trains)
    fn = lambda ids, link: (DF.embedding(ids, emb.weight, scale=3.0, padding_idx=0) + link,)   # noqa: E731
    for i in range(4):
        region.new_iteration()
        ids = torch.randint(0, 300, (5, 40), generator=g)
        ids[:, 20 + 4 * i:] = 0
        ids, dy = ids.to(dev), torch.randn(5, 40, 64, generator=g).to(dev)
        eager = DF.embedding(ids, emb.weight, scale=3.0, padding_idx=0)
        emb.weight.grad = link.grad = None
        y, = region.run("rows", fn, (ids, link))
        assert torch.equal(y, eager)
        y.backward(dy)
        got = emb.weight.grad.clone()
        emb.weight.grad = None
        eager.backward(dy)
        assert torch.equal(got, emb.weight.grad)
        _check_bwd(got, dy, ids, 300, 3.0, 0, F32, i)
        with torch.no_grad():
            emb.weight.add_(0.1)                                 # a step between the replays
    assert region.captures == 1


def test_capture_beside_an_eager_graph_of_the_table_is_refused(dev):
    """Before anything is recorded; once the eager graph is gone, forward and backward are captured and replayed."""
    table = torch.randn(50, 16, device=dev).requires_grad_()
    ids = torch.arange(12, device=dev)
    dy = torch.randn(12, 16, device=dev)
    ops.check_device_errors()
    y = DF.embedding(ids, table)
    graph, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=st):
        one = torch.ones(4, device=dev)
        with pytest.raises(DasaError, match="AutogradGraphs"):
            DF.embedding(ids, table)
        with torch.no_grad():
            z = DF.embedding(ids, table)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(z, table.detach()[:12]) and float(one.sum()) == 4.0
    del y
    st.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        grad, = torch.autograd.grad(DF.embedding(ids, table), table, dy)
    for i in range(3):
        ids.copy_(torch.randperm(50, generator=_gen(i))[:12].to(dev))
        want = ops.embedding_bwd(dy, ids, 50)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(grad, want)


# ------------------------------------------------------------------------------------------ 4-bit weights
def _w4(N, K, group, sdt, seed):
    g = _gen(seed)
    codes = torch.randint(0, 256, (N, (K + 1) // 2), generator=g, dtype=torch.uint8)
    scales = (0.01 + 0.1 * torch.rand(N, -(-K // group), generator=g)).to(sdt)
    q = torch.stack((codes & 15, codes >> 4), 2).reshape(N, -1)[:, :K].double() - 8
    return codes, scales, q * scales.double().repeat_interleave(group, 1)[:, :K]


def _check_w4(got, x, W, group, dtype, what, bias=None, extra=None):
    """Products are exact; an fp32 sum adds three planes of every product (an addition off by at most a whole step,
    2^-23), one scaling a group, the joins of the waves and the bias."""
    xd = x.to(got.device).double()
    W = W.to(got.device)
    want, mag = (xd @ W.t()).cpu(), (xd.abs() @ W.abs().t()).cpu()
    K = W.shape[1]
    tol = mag * (3 * K + 2 * (-(-K // group)) + 16) * 2 * U
    if bias is not None:
        want, tol = want + bias.cpu().double(), tol + U * (want.abs() + bias.cpu().double().abs())
    if extra is not None:
        want, tol = want + extra.cpu().double(), tol + U * (want.abs() + extra.cpu().double().abs())
    _within(got, want, tol + HALF[dtype] * (want.abs() + tol), what)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("N,K", [(1, 1), (15, 31), (16, 128), (17, 129), (100, 200), (33, 640)])
def test_w4_weight_values(dev, N, K, group):
    """Every weight lands where it belongs: x = the identity gives W^T, each value one rounding of (q - 8) s."""
    for sdt in (F32, BF16):
        codes, scales, W = _w4(N, K, group, sdt, N + K)
        w = ops.pack_w4(codes.to(dev), scales.to(dev), K, group)
        assert torch.equal(w.dequantize().cpu(), W.float())
        assert torch.equal(ops.linear_w4(torch.eye(K, device=dev), w).cpu(), W.float().t())
        y = ops.linear_w4(torch.eye(K, device=dev, dtype=BF16), w)
        assert torch.equal(y.cpu(), W.float().t().to(BF16))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,N,K,group", [(1, 1, 1, 32), (1, 2048, 256, 64), (2, 1000, 512, 128), (15, 17, 33, 32),
                                         (16, 992, 512, 64), (17, 100, 1000, 128), (20, 4096, 2240, 64),
                                         (31, 50, 2241, 32), (33, 130, 127, 64), (64, 8200, 640, 128), (65, 33, 96, 32),
                                         (150, 8193, 255, 64), (1, 30522, 768, 32), (20, 30522, 200, 64),
                                         (64, 16384, 2100, 64), (40, 65536, 2041, 128), (3, 100, 8000, 32),
                                         (20, 100, 8000, 64), (48, 2100, 300, 128), (20, 30522, 768, 64),
                                         (33, 30522, 128, 128), (64, 16384, 2048, 32), (50, 65536, 2048, 128)])
def test_linear_w4(dev, dtype, M, N, K, group):
    """Every form: 16 rows a workgroup with 1, 2 and 4 column blocks, K split over workgroups, 32 and 64 rows sharing
    their activations, rows and columns that end inside a tile, an inner size that ends inside a group."""
    for sdt in (F32, BF16) if N < 20000 else (F32 if dtype == F32 else BF16,):
        codes, scales, W = _w4(N, K, group, sdt, M + N + K)
        w = ops.pack_w4(codes.to(dev), scales.to(dev), K, group)
        x = torch.randn(M, K, generator=_gen(M)).to(dtype)
        b = torch.randn(N, generator=_gen(N))
        got = ops.linear_w4(x.to(dev), w, b.to(dev))
        assert got.dtype == dtype and got.shape == (M, N)
        _check_w4(got, x, W, group, dtype, "linear_w4", bias=b)
        assert torch.equal(got, ops.linear_w4(x.to(dev), w, b.to(dev)))
        # one row alone: the same sums
        assert torch.equal(ops.linear_w4(x[:1].to(dev), w, b.to(dev)), got[:1]) or M > 16
        _check_w4(ops.linear_w4(x[:1].to(dev), w), x[:1], W, group, dtype, "one row")


def test_linear_w4_epilogue_strides_and_accumulation(dev):
    codes, scales, W = _w4(70, 130, 64, F32, 3)
    w = ops.pack_w4(codes.to(dev), scales.to(dev), 130, 64)
    g = _gen(4)
    wide = torch.randn(5, 3, 150, generator=g).to(dev)
    x = wide[..., 7:137]                                            # strided, unaligned rows
    b = torch.randn(70, generator=g).to(dev)
    y = ops.linear_w4(x, w, b)
    assert y.shape == (5, 3, 70)
    _check_w4(y.view(15, 70), x.reshape(15, 130), W, 64, F32, "strided", bias=b)
    _check_w4(ops.linear_w4(x.transpose(0, 1), w).reshape(15, 70), x.transpose(0, 1).reshape(15, 130), W, 64, F32, "order")
    assert torch.equal(ops.linear_w4(x[0, 0], w, b), y[0, 0])
    for act, f in (("relu", torch.relu), ("tanh", torch.tanh), ("sigmoid", torch.sigmoid),
                   ("gelu", torch.nn.functional.gelu)):
        # the activations change their argument's error by a factor of at most 1.13 (gelu) and add a few steps
        got = ops.linear_w4(x, w, b, act=act)
        assert float((got - f(y)).abs().max()) <= 4e-6
    buf = torch.full((15, 90), 2.0, device=dev)
    old = torch.randn(15, 70, generator=g).to(dev)
    buf[:, 4:74] = old
    ops.linear_w4(x.reshape(15, 130), w, b, out=buf[:, 4:74], beta=1.0)
    _check_w4(buf[:, 4:74], x.reshape(15, 130), W, 64, F32, "beta", bias=b, extra=old)
    assert bool((buf[:, :4] == 2).all()) and bool((buf[:, 74:] == 2).all())
    assert ops.linear_w4(x[:0], w).shape == (0, 3, 70)
    expanded = x[0, 0].expand(4, 130)
    assert torch.equal(ops.linear_w4(expanded, w), ops.linear_w4(expanded.contiguous(), w))


def test_linear_w4_values_that_are_not_finite(dev):
    """Infinities and NaN reach their own row alone, as in the product; the wide range of fp32 survives."""
    codes, scales, W = _w4(40, 96, 32, F32, 8)
    w = ops.pack_w4(codes.to(dev), scales.to(dev), 96, 32)
    x = torch.randn(5, 96, generator=_gen(2))
    x[1, 3], x[2, 5] = float("inf"), float("nan")
    x[3] *= 1e30
    x[4] *= 1e-30
    y = ops.linear_w4(x.to(dev), w).cpu()
    _check_w4(y[[0, 3, 4]], x[[0, 3, 4]], W, 32, F32, "range")
    want = torch.where(W[:, 3] == 0, float("nan"), torch.sign(W[:, 3]) * float("inf"))
    assert torch.equal(y[1].isnan(), want.isnan()) and torch.equal(y[1][~want.isnan()].double(), want[~want.isnan()])
    assert bool(y[2].isnan().all())
    tiny_nan = torch.tensor([0x7f800001], dtype=torch.int32).view(F32)       # a NaN that truncation would make inf
    x = torch.zeros(1, 96)
    x[0, 0] = tiny_nan
    assert bool(ops.linear_w4(x.to(dev), w).isnan().all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,K,group", [(1, 1, 32), (37, 200, 64), (64, 128, 128), (5, 33, 32)])
def test_quantize_w4(dev, dtype, N, K, group):
    """Codes are the nearest values: every weight is within half a scale (a hair more for the division)."""
    g = _gen(N * K)
    W = torch.randn(N, K, generator=g).to(dtype)
    W[0, :min(K, group)] = 0.0                                      # a group of zeros
    for sdt in (F32, BF16):
        w = ops.quantize_w4(W.to(dev), group, scale_dtype=sdt)
        d = w.dequantize().cpu().double()
        pad = torch.nn.functional.pad(W.double().abs(), (0, -K % group)).view(N, -1, group)
        s = pad.amax(2) / 7
        sd = s.repeat_interleave(group, 1)[:, :K]
        assert bool(((d - W.double()).abs() <= sd * (0.5 + 8 * HALF[sdt]) * (1 + 4 * U)).all())
        assert bool((d[0, :min(K, group)] == 0).all())
    again = ops.quantize_w4(W.to(dev), group)
    assert torch.equal(again.dequantize(), ops.quantize_w4(W.to(dev), group).dequantize())


# ------------------------------------------------------------------------------------------ rules on logits
def _rules_reference(logits, history=None, lengths=None, r=1.0, p=0.0, f=0.0, bias=None, open_=None):
    """(values, tolerance before the last rounding) in 64 bits."""
    x = logits.double().clone()
    B, V = x.shape
    tol = torch.zeros_like(x)
    count = torch.zeros_like(x)
    if history is not None:
        for b in range(B):
            h = history[b, :int(lengths[b]) if lengths is not None else None].long()
            h = h[(h >= 0) & (h < V)]
            count[b] = torch.bincount(h, minlength=V)[:V].double()
    col = lambda v: v.double()[:, None] if isinstance(v, torch.Tensor) else torch.tensor(v, dtype=F32).double()  # noqa
    r, p, f = col(r), col(p), col(f)
    y = torch.where(x > 0, x / r, x * r)
    t = U * y.abs()
    z = y - f * count
    t = t + U * (f * count).abs() + U * z.abs()
    w = z - p
    t = t + U * w.abs()
    seen = count > 0
    x, tol = torch.where(seen, w, x), torch.where(seen, t, tol)
    if bias is not None:
        x = x + bias.double()
        tol = tol + U * x.abs()
    if open_ is not None:
        x = x.masked_fill(~open_.expand(B, V), -math.inf)
    tol = torch.where(x.isfinite(), tol * (1 + 8 * U), torch.zeros_like(tol))
    return x, tol


def _words(open_):
    n = -(-open_.shape[-1] // 32)
    b = torch.nn.functional.pad(open_.long(), (0, n * 32 - open_.shape[-1])).view(*open_.shape[:-1], n, 32)
    w = (b << torch.arange(32)).sum(-1)
    return torch.where(w >= 2**31, w - 2**32, w).to(torch.int32)


def _first_best(y):
    y = y.double().cpu()
    key = torch.where(y.isnan(), torch.full_like(y, math.inf), y)
    best = key.amax(1, keepdim=True)
    hit = torch.where(y.isnan().any(1, keepdim=True), y.isnan(), key == best)
    return torch.where(hit, torch.arange(y.shape[1])[None], y.shape[1]).amin(1)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,V,L", [(1, 1, 1), (3, 5, 9), (20, 992, 120), (2, 8192, 300), (2, 8193, 300), (5, 30522, 70),
                                   (1, 100003, 4000), (7, 1025, 20000), (64, 33, 1)])
def test_logit_rules(dev, dtype, B, V, L):
    g = _gen(B + V + L)
    logits = (3 * torch.randn(B, V, generator=g)).to(dtype)
    history = (torch.pow(float(V), torch.rand(B, L, generator=g, dtype=torch.float64)).long() - 1).clamp(0, V - 1)
    lengths = torch.randint(0, L + 1, (B,), generator=g)
    r, p, f = 1 + torch.rand(B, generator=g), torch.rand(B, generator=g), 0.3 * torch.rand(B, generator=g)
    for own in (False, True):
        bias = torch.randn(*((B, V) if own else (V,)), generator=g)
        open_ = torch.rand(*((B, V) if own else (V,)), generator=g) < 0.5
        want, tol = _rules_reference(logits, history, lengths, r, p, f, bias, open_)
        tol = tol + HALF[dtype] * torch.where(want.isfinite(), want.abs() + tol, torch.zeros_like(tol))
        dv = lambda t: t.to(dev)   # noqa: E731
        for mask in (open_, open_.to(torch.uint8) * 3, _words(open_)):
            y, c = ops.logit_rules(dv(logits), dv(history), dv(lengths), repetition=dv(r), presence=dv(p),
                                   frequency=dv(f), bias=dv(bias), allowed=dv(mask), want_choice=True)
            assert y.dtype == dtype
            _within(y, want, tol, "rules")
            assert torch.equal(c.cpu(), _first_best(y))
        y2 = ops.logit_rules(dv(logits), dv(history.to(torch.int32)), dv(lengths.to(torch.int32)), repetition=dv(r),
                             presence=dv(p), frequency=dv(f), bias=dv(bias), allowed=dv(open_))
        assert torch.equal(y, y2)
    want, tol = _rules_reference(logits, history, None, 1.3, 0.25, 0.125)
    y = ops.logit_rules(dv(logits), dv(history), repetition=1.3, presence=0.25, frequency=0.125)
    _within(y, want, tol + HALF[dtype] * (want.abs() + tol), "numbers")
    assert torch.equal(ops.logit_rules(dv(logits)), dv(logits))                  # no rule: the logits
    y = dv(logits).clone()
    z = ops.logit_rules(y, dv(history), repetition=1.3, presence=0.25, frequency=0.125, out=y)     # in place
    assert z.data_ptr() == y.data_ptr()
    _within(y, want, tol + HALF[dtype] * (want.abs() + tol), "in place")


@pytest.mark.parametrize("V", [37, 9001])
def test_logit_rules_rows_that_leave_nothing_and_values_that_are_not_finite(dev, V):
    inf, nan = float("inf"), float("nan")
    logits = torch.zeros(8, V)
    logits[1, 5] = nan
    logits[2, 7], logits[2, 3] = nan, inf
    logits[3, 4], logits[3, 2] = inf, inf
    logits[4] = -inf
    logits[5, 6], logits[5, 8] = 1.0, 1.0
    logits[6] = torch.finfo(F32).min                                 # a mask of the type's lowest value
    logits[7, 0], logits[7, 1] = -0.0, 0.0
    open_ = torch.ones(8, V, dtype=torch.bool)
    open_[0] = False                                                 # nothing allowed
    open_[2, 7] = False                                              # a NaN in a masked place
    hist = torch.tensor([[0], [5], [3], [4], [1], [8], [2], [1]])
    for mask in (open_, _words(open_)):
        y, c = ops.logit_rules(logits.to(dev), hist.to(dev), repetition=2.0, presence=0.5, allowed=mask.to(dev),
                               want_choice=True)
        y = y.cpu()
        assert bool((y[0] == -inf).all())
        assert bool(y[1, 5].isnan()) and float(y[2, 7]) == -inf and float(y[2, 3]) == inf
        assert bool((y[4] == -inf).all()) and float(y[6, 2]) == -inf and float(y[6, 0]) == torch.finfo(F32).min
        assert float(y[5, 8]) == 0.0 and float(y[7, 1]) == -0.5
        assert c.tolist() == [0, 5, 3, 2, 0, 6, 0, 0], c.tolist()
    # strides: rows of a wider buffer, ids to ignore, an empty history
    wide = torch.randn(3, V + 9, generator=_gen(1)).to(dev)
    out = torch.full((3, V + 5), 9.0, device=dev)
    h = torch.tensor([[1, -1, V, 2**40, -2**40, 1], [0, 0, 0, 0, 0, 0], [-1, -1, -1, -1, -1, -1]])
    want, tol = _rules_reference(wide[:, 4:4 + V].cpu(), h, None, 1.5, 0.0, 0.5)
    y = ops.logit_rules(wide[:, 4:4 + V], h.to(dev), repetition=1.5, frequency=0.5, out=out[:, 2:2 + V])
    _within(y, want, tol + HALF[F32] * (want.abs() + tol), "strided")
    assert bool((out[:, :2] == 9).all()) and bool((out[:, 2 + V:] == 9).all())
    x = wide[:, 4:4 + V]
    assert torch.equal(ops.logit_rules(x, h[:, :0].to(dev), repetition=1.5), x)
    assert torch.equal(ops.logit_rules(x, h.to(dev), torch.zeros(3, dtype=torch.int64, device=dev), repetition=1.5), x)
    many = torch.tensor([100, -5, 3], device=dev)                    # lengths outside [0, L] are clipped to it
    full = ops.logit_rules(x, h.to(dev), repetition=1.5, frequency=0.5)
    got = ops.logit_rules(x, h.to(dev), many, repetition=1.5, frequency=0.5)
    assert torch.equal(got[0], full[0]) and torch.equal(got[1], x[1]) and torch.equal(got[2], x[2])
    y, c = ops.logit_rules(x[:0], want_choice=True)
    assert y.shape == (0, V) and c.shape == (0,)


# ------------------------------------------------------------------------------------------ together
def _step_state(dev):
    g = _gen(77)
    V, E, B, L = 992, 256, 20, 12
    s = dict(table=torch.randn(V, E, generator=g).to(dev), word=torch.randint(0, V, (B,), generator=g).to(dev),
             hist=torch.randint(0, V, (B, L), generator=g).to(dev), ban=torch.ones(V, dtype=torch.bool, device=dev))
    s["ban"][3] = False
    s["w"] = ops.quantize_w4(torch.randn(V, E, generator=g).to(dev) * 0.1, 64)
    s["b"] = torch.randn(V, generator=g).to(dev)
    return s


def _step(s):
    x = ops.embedding(s["word"], s["table"], scale=0.5)
    logits = ops.linear_w4(x, s["w"], s["b"])
    y, word = ops.logit_rules(logits, s["hist"], repetition=1.2, frequency=0.1, allowed=s["ban"], want_choice=True)
    return x, logits, y, word


def test_word_step_together(dev):
    """Lookup, 4-bit projection and rules in a row, against the plain step in 64 bits."""
    s = _step_state(dev)
    x, logits, y, word = _step(s)
    W = s["w"].dequantize().cpu().double()
    xe = s["table"].cpu().double()[s["word"].cpu()] * 0.5
    assert torch.equal(x.cpu().double(), xe)
    _check_w4(logits, x, W, 64, F32, "logits", bias=s["b"])
    want, tol = _rules_reference(logits.cpu(), s["hist"].cpu(), None, 1.2, 0.0, 0.1, None, s["ban"].cpu())
    _within(y, want, tol + HALF[F32] * torch.where(want.isfinite(), want.abs() + tol, torch.zeros_like(tol)), "rules")
    assert torch.equal(word.cpu(), _first_best(y)) and bool((y[:, 3] == -float("inf")).all())


def test_word_step_captured_and_on_another_stream(dev):
    """A captured step, replayed on new inputs with eager work between, and two graphs in flight on two streams."""
    s1, s2 = _step_state(dev), _step_state(dev)
    _step(s1)
    graphs = []
    for s in (s1, s2):
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            _step(s)
        torch.cuda.current_stream().wait_stream(st)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            out = _step(s)
            grad = ops.embedding_bwd(out[0], s["word"], 992)
        graphs.append((gr, s, out, grad, st))
    for i in range(4):
        want = []
        for k, (gr, s, out, grad, st) in enumerate(graphs):
            s["word"].copy_(torch.randint(0, 992, (20,), generator=_gen(10 * i + k)).to(dev))
            s["hist"].copy_(torch.randint(0, 992, (20, 12), generator=_gen(10 * i + k + 5)).to(dev))
            w = _step(s)
            want.append((*w, ops.embedding_bwd(w[0], s["word"], 992)))
        torch.cuda.synchronize()
        for gr, s, out, grad, st in graphs:
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for (gr, s, out, grad, st), w in zip(graphs, want):
            for a, b in zip((*out, grad), w):
                assert torch.equal(a, b)


def test_outputs_that_overlap_an_input_are_refused(dev):
    """out may not share bytes with what the call reads (but logit_rules works in place, and column blocks of one
    buffer are apart)."""
    buf = torch.randn(6, 64, device=dev)
    w = ops.quantize_w4(torch.randn(20, 32, device=dev), 32)
    want = ops.linear_w4(buf[:, :32].contiguous(), w)
    got = ops.linear_w4(buf[:, :32], w, out=buf[:, 32:52])
    assert torch.equal(got, want)
    with pytest.raises(DasaError, match="overlaps"):
        ops.linear_w4(buf[:, :32], w, out=buf[:, 31:51])
    with pytest.raises(DasaError, match="overlaps"):
        ops.linear_w4(buf[:, 40:], ops.quantize_w4(torch.randn(24, 24, device=dev), 32), out=buf[:, 30:54])
    x = torch.randn(6, 30, device=dev)
    with pytest.raises(DasaError, match="overlaps"):
        ops.logit_rules(x[:5], out=x[1:])
    with pytest.raises(DasaError, match="overlaps"):
        ops.logit_rules(x[:, :20], out=x[:, 5:25])
    assert torch.equal(ops.logit_rules(x[:, :15], out=x[:, 15:]), x[:, :15])
    with pytest.raises(DasaError, match="overlaps"):
        ops.embedding(torch.tensor([1, 2], device=dev), x, out=x[:2])
    with pytest.raises(DasaError, match="overlaps"):
        ops.embedding_bwd(x, torch.arange(6, device=dev), 6, out=x)
    with pytest.raises(DasaError, match="rows of out"):
        ops.embedding(torch.tensor([1, 2], device=dev), x, out=torch.empty(30, device=dev).expand(2, 30))


def test_refusals_on_the_device(dev):
    x = torch.randn(3, 40, device=dev)
    h = torch.zeros(3, 5, dtype=torch.int64, device=dev)
    for bad in (dict(history=h[:2]), dict(history=h.float()), dict(lengths=h[:, 0]), dict(repetition=0.0),
                dict(repetition=float("nan")), dict(presence=float("inf")), dict(frequency=torch.ones(2, device=dev)),
                dict(repetition=torch.ones(3, device=dev, dtype=torch.float64)), dict(bias=torch.ones(3, device=dev)),
                dict(bias=torch.ones(40, device=dev, dtype=BF16)), dict(allowed=torch.ones(40, device=dev)),
                dict(allowed=torch.ones(41, device=dev, dtype=torch.bool)),
                dict(allowed=torch.ones(40, device=dev, dtype=torch.int32)), dict(out=torch.empty(3, 41, device=dev)),
                dict(out=torch.empty(3, 40, device=dev, dtype=BF16)), dict(history=h, lengths=h[:2, 0]),
                dict(history=h, lengths=torch.ones(3, device=dev)), dict(bias=torch.ones(40)), dict(repetition=torch.ones(3))):
        with pytest.raises(DasaError):
            ops.logit_rules(x, **bad)
    with pytest.raises(DasaError, match="rows of logits"):
        ops.logit_rules(x.t())
    with pytest.raises(DasaError, match="forward only"):
        ops.logit_rules(x.clone().requires_grad_())
    with pytest.raises(DasaError, match="token at least"):
        ops.logit_rules(torch.empty(3, 0, device=dev))
    w = ops.quantize_w4(torch.randn(20, 40, device=dev), 32)
    for bad in (dict(b=torch.ones(19, device=dev)), dict(b=torch.ones(20)), dict(beta=1.0), dict(act="swish"),
                dict(out=torch.empty(3, 21, device=dev)), dict(out=torch.empty(3, 20, device=dev, dtype=BF16))):
        with pytest.raises(DasaError):
            ops.linear_w4(x, w, **bad)
    with pytest.raises(DasaError, match="forward only"):
        ops.linear_w4(x.clone().requires_grad_(), w)
    d = torch.randn(3, 5, 8, device=dev)
    for a, k in (((d[:2], h, 10), {}), ((d, h, 10), dict(padding_idx=10)), ((d, h, 10), dict(accumulate=True)),
                 ((d, h, 10), dict(out=torch.empty(10, 9, device=dev))), ((d, h, -1), {}), ((d, h.float(), 10), {})):
        with pytest.raises(DasaError):
            ops.embedding_bwd(*a, **k)
    with pytest.raises(DasaError, match="no rows"):
        ops.embedding(h, torch.empty(0, 8, device=dev))
    with pytest.raises(DasaError, match="rows must be contiguous"):
        ops.embedding(h, torch.randn(8, 10, device=dev).t())


@pytest.mark.parametrize("dtype,E", [(BF16, 1), (BF16, 8), (F32, 5)])
def test_embedding_gradient_of_more_rows_than_one_launch_takes(dev, dtype, E):
    """2^26 rows and some, four of them to a workgroup of 256 threads: more threads than a launch may have. Whole numbers
    of at most three bits: every sum is exact in fp32, so the gradient is the 64-bit sum, rounded once."""
    V, T = 2**26 + 3, 8200
    g = _gen(E)
    ids = torch.randint(0, V, (T,), generator=g)
    edge = 2**26 - 264 + torch.arange(-40, 40)                   # where the second launch begins
    ids[:80], ids[80:90], ids[90:400] = edge, V - 1 - torch.arange(10), V - 1
    ids[400:500], ids[500] = edge[39], 0
    dout = torch.randint(-3, 4, (T, E), generator=g).to(dtype)
    got = ops.embedding_bwd(dout.to(dev), ids.to(dev), V, scale=2.0)
    rows, at = torch.unique(ids, return_inverse=True)
    want = torch.zeros(len(rows), E, dtype=torch.float64).index_add_(0, at, dout.double()) * 2.0
    assert torch.equal(got[rows.to(dev)].cpu(), want.to(dtype))
    got[rows.to(dev)] = 0
    assert int(torch.count_nonzero(got)) == 0
    again = torch.full((V, E), 3.0, dtype=dtype, device=dev)
    ops.embedding_bwd(dout.to(dev), ids.to(dev), V, out=again, accumulate=True)
    assert torch.equal(again[rows.to(dev)].cpu(), (want / 2.0 + 3.0).to(dtype))
    again[rows.to(dev)] = 3.0
    assert bool((again == 3.0).all())
