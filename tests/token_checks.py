"""Inputs on which the token operators are exact, and the checks that use it. Sums of small whole numbers round nowhere
in fp32, whatever their order, so a kernel's result has to equal the 64-bit one rounded once to its type: one token,
part or plane too few or too many shows, which a tolerance that grows with the number of terms would hide."""
import torch

F32, BF16 = torch.float32, torch.bfloat16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def token_ids(kind, T, V, g):
    """Token ids by kind: uniform, zipf (frequency falls with the rank), one id, or runs whose lengths lie around the
    multiples of 32 and 128 at which long rows are cut."""
    if kind == "uniform":
        return torch.randint(0, V, (T,), generator=g)
    if kind == "one":
        return torch.full((T,), V // 2)
    if kind == "zipf":
        return (torch.pow(float(V), torch.rand(T, generator=g, dtype=torch.float64)).long() - 1).clamp(0, V - 1)
    lengths = [1, 31, 32, 33, 64, 95, 96, 97, 127, 128, 129, 160, 255, 256, 257, 511, 512, 513, 600, 2049, 2176, 3000]
    ids, v = [], 0
    while sum(map(len, ids)) < T:
        ids.append(torch.full((lengths[(v * 7) % len(lengths)],), v % V))
        v += 1
    return torch.cat(ids)[:T][torch.randperm(T, generator=g)]


def counting_dout(ids, E, g):
    """1, 2 or 3 everywhere: a sum misses or gains whatever a row misses or gains (below 2^24 up to 2^22 tokens)."""
    return torch.randint(1, 4, (ids.numel(), E), generator=g).double()


def walking_dout(ids, E, g):
    """The steps of a walk on 0..6 along each id's tokens: every id's sum is its last place, and the sum of any stretch of
    them is small, so bf16 holds it exactly and a lost or doubled stretch shows there too."""
    order = torch.sort(ids, stable=True).indices
    s = ids[order]
    w = torch.randint(0, 7, (ids.numel(), E), generator=g).double()
    before = torch.zeros_like(w)
    before[1:] = w[:-1] * (s[1:] == s[:-1])[:, None]
    d = torch.empty_like(w)
    d[order] = w - before
    return d


def gradient_sums(dout, ids, V, pad=None):
    """The table's gradient in 64 bits."""
    keep = (ids >= 0) & (ids < V)
    if pad is not None:
        keep &= ids != pad
    return torch.zeros(V, dout.shape[-1], dtype=torch.float64).index_add_(0, ids[keep], dout.double()[keep])


def check_gradient(got, dout, ids, V, scale=1.0, pad=None, old=None):
    """got is the exact gradient, rounded once; scale a power of two, old (accumulated into) small whole numbers."""
    want = gradient_sums(dout, ids, V, pad) * scale
    if old is not None:
        want = want + old.double()
    want, got = want.to(got.dtype), got.cpu()
    bad = (got != want).any(1)
    rows = torch.nonzero(bad)[:4, 0].tolist()
    assert not rows, (int(bad.sum()), rows, [int((ids == r).sum()) for r in rows], got[rows][:, :4].tolist(),
                      want[rows][:, :4].tolist())


# ------------------------------------------------------------------------------------------ 4-bit products
def w4_weight(N, K, group, scales, g):
    """(codes [N, ceil(K / 2)], scales [N, groups] fp32); scales: "powers" of two, 1/8 to 1, or "any"."""
    codes = torch.randint(0, 256, (N, (K + 1) // 2), generator=g, dtype=torch.uint8)
    groups = -(-K // group)
    s = torch.exp2(-torch.randint(0, 4, (N, groups), generator=g).float()) if scales == "powers" else \
        0.01 + 0.1 * torch.rand(N, groups, generator=g)
    return codes, s


def w4_values(codes, scales, K, group):
    """The weight in 64 bits, on the codes' device."""
    q = torch.stack((codes & 15, codes >> 4), 2).reshape(codes.shape[0], -1)[:, :K].double() - 8
    return q * scales.double().repeat_interleave(group, 1)[:, :K]


def whole_rows(M, K, g):
    """-4..4: with scales that are powers of two, every partial sum up to K = 2^16 is exact in fp32."""
    return torch.randint(-4, 5, (M, K), generator=g).double()


def three_plane_rows(M, K, g):
    """Up to 8 odd numbers of 17 bits in a row whose three pieces of 8 significant bits are all nonzero: 2^16 + .. + 2^8
    + .. + 1. With codes up to 8 and one power of two as scale, every partial sum is exact in fp32."""
    n = min(8, K)
    x = torch.zeros(M, K, dtype=torch.float64)
    for m in range(M):
        at = torch.randperm(K, generator=g)[:n]
        v = 2**16 + torch.randint(0, 128, (n,), generator=g) * 2**9 + 2**8 + torch.randint(0, 128, (n,), generator=g) * 2 + 1
        x[m, at] = (v * (2 * torch.randint(0, 2, (n,), generator=g) - 1)).double()
    return x


def single_rows(ks, K, g):
    """A row for each k of ks with one value there: 24 significant bits, the third piece at least 2^-16 of the first,
    any sign, exponents -20 to 20."""
    n = len(ks)
    bits = 2**23 + torch.randint(0, 2**23, (n,), generator=g)
    bits = bits | 2**15 | 2**7 | 1                        # the leading bits of the second and the third piece, the last bit
    v = bits.double() * torch.exp2(torch.randint(-43, -2, (n,), generator=g).double())
    x = torch.zeros(n, K, dtype=torch.float64)
    x[torch.arange(n), ks] = v * (2 * torch.randint(0, 2, (n,), generator=g) - 1)
    return x


def check_rounded(got, want):
    """got is want (exact in fp32), rounded once to its type."""
    want = want.to(got.dtype).to(got.device)
    bad = got != want
    assert not bool(bad.any()), (int(bad.sum()), torch.nonzero(bad)[:4].tolist(), got[bad][:4].tolist(),
                                 want[bad][:4].tolist())


def check_single(got, x, W):
    """Outputs of single_rows in fp32: pieces times a code are exact, their sum is at most one step (2^-23) off, the scale
    half a step: less than 2^-22 of the value. Without its third piece a value is at least 2^-17 off."""
    want = x @ W.t()
    bad = ~((got.double() - want).abs() <= want.abs() * 2.0**-22)
    assert not bool(bad.any()), (int(bad.sum()), torch.nonzero(bad)[:4].tolist(), got[bad][:4].tolist(),
                                 want[bad][:4].tolist())


def check_groups(got, x, W, group, planes):
    """Random rows. A group's fp32 sum adds planes * group products, each addition off by at most a step (2^-23) of at
    most the group's sum of magnitudes; a group is scaled and added (half a step of the total each), and 24 joins of
    waves and splits follow. (Not planes * K additions: sums start again with each group.)"""
    K = W.shape[1]
    want, mag = x @ W.t(), x.abs() @ W.abs().t()
    tol = mag * (planes * group * 2.0**-23 + (2 * -(-K // group) + 24) * 2.0**-24) * (1 + 2.0**-10)
    if got.dtype == BF16:
        tol = tol + 2.0**-8 * (want.abs() + tol)
    else:
        tol = tol + 2.0**-24 * want.abs()
    bad = ~((got.double() - want).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float(((got.double() - want).abs() / tol).max()))
