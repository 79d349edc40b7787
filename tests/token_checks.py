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
