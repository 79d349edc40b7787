"""Measured cases of the token operators: the embedding lookup and its gradient, products with 4-bit weights,
and the rules on logits before a token is chosen.

`listed()` names the cases, `prepare()` makes what a program holds before the call, `run()` is one pass (plain
torch operations, or the framework's kernels where `own` is true), `exact()` the same in 64 bits, `work()` the bytes
and operations a pass cannot do without.
"""
import math

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "bf16": 2}


def listed():
    return [
        # ---- embedding lookup, forward
        # the speaker's word step: one word for each of 20 rows, vocabulary 992, --wemb 256
        dict(name="embed_word", op="embed", batch=20, length=1, vocab=992, width=256, dtype="f32", scale=1.0),
        # prompts of a served encoder: 64 sequences of 512 tokens, bf16 table scaled by sqrt(width)
        dict(name="embed_prompts", op="embed", batch=64, length=512, vocab=30522, width=1024, dtype="bf16", scale=32.0),
        # ---- embedding lookup and its gradient (training)
        # the README batch: 20 instructions of 80 tokens, padded, the BERT table
        dict(name="embed_train", op="embed_train", batch=20, length=80, vocab=30522, width=768, dtype="f32", scale=1.0,
             padded=True),
        # one long ragged text, a small vocabulary (every row hit, long runs of one token), odd width
        dict(name="embed_train_odd", op="embed_train", batch=1, length=4099, vocab=1001, width=257, dtype="f32",
             scale=0.5, padded=False),
        # a pretraining batch: 256 sequences of 512, bf16, padded
        dict(name="embed_train_large", op="embed_train", batch=256, length=512, vocab=50021, width=1024, dtype="bf16",
             scale=32.0, padded=True),
        # ---- 4-bit weights
        # the speaker's input gates for one row: latency
        dict(name="w4_gates", op="w4", rows=1, n=2048, k=256, group=64, dtype="f32", scales="f32", bias=True),
        # the policy decoder's input gates at the README batch; the inner size ends inside a group block
        dict(name="w4_decoder", op="w4", rows=20, n=4096, k=2240, group=64, dtype="f32", scales="f32", bias=True),
        # a vocabulary projection over the BERT vocabulary for 64 rows
        dict(name="w4_vocab", op="w4", rows=64, n=30522, k=768, group=128, dtype="bf16", scales="bf16", bias=True),
        # one token through a wide layer: the weights are all there is to read
        dict(name="w4_wide", op="w4", rows=1, n=32768, k=8192, group=128, dtype="bf16", scales="bf16", bias=False),
        # ---- rules on logits
        # the speaker's word step: ban and repetition penalty over --maxDecode 120 words
        dict(name="rules_word", op="rules", rows=20, vocab=992, history=120, dtype="f32", bias="none", own_masks=False,
             own_penalties=False),
        # a served batch with its own settings and grammar for each row
        dict(name="rules_batch", op="rules", rows=64, vocab=30522, history=1024, dtype="f32", bias="shared",
             own_masks=True, own_penalties=True),
        # long contexts, a large odd vocabulary, a bias for each row
        dict(name="rules_long", op="rules", rows=16, vocab=128255, history=16384, dtype="bf16", bias="rows",
             own_masks=True, own_penalties=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embed", "embed_train", "w4", "rules"])
    dtype = rng.choice(["f32", "bf16"])
    if op in ("embed", "embed_train"):
        width = _log_int(rng, 64, 1024)
        case = dict(op=op, vocab=_log_int(rng, 300, 50021), width=width, dtype=dtype,
                    scale=rng.choice([1.0, 0.5, math.sqrt(width)]), batch=_log_int(rng, 1, 64),
                    length=_log_int(rng, 1, 512))
        if op == "embed_train":
            case["padded"] = rng.choice([True, False])
        return case
    if op == "w4":
        return dict(op=op, rows=rng.choice([1, 1, 2, 3, 5, 8, 16, 17, 20, 33, 48, 64]), n=_log_int(rng, 200, 32768),
                    k=_log_int(rng, 65, 8192), group=rng.choice([32, 64, 128]), dtype=dtype,
                    scales=rng.choice(["f32", "bf16"]), bias=rng.choice([True, False]))
    return dict(op=op, rows=_log_int(rng, 1, 64), vocab=_log_int(rng, 300, 32000) if rng.random() < 0.7 else
                _log_int(rng, 32000, 128255), history=_log_int(rng, 1, 16384), dtype=dtype,
                bias=rng.choice(["none", "shared", "rows"]), own_masks=rng.choice([True, False]),
                own_penalties=rng.choice([True, False])) if rng.random() < 0.75 else \
        dict(op=op, rows=_log_int(rng, 1, 16), vocab=_log_int(rng, 300, 128255), history=_log_int(rng, 1, 120),
             dtype=dtype, bias="none", own_masks=False, own_penalties=False)


# ------------------------------------------------------------------------------------------ inputs
def _tokens(g, batch, length, vocab, dev):
    """Token ids whose frequency falls with 1 / rank, as words' does, spread over the table."""
    u = torch.rand(batch, length, generator=g, device=dev, dtype=torch.float64)
    rank = torch.pow(float(vocab), u).long() - 1
    step = next(p for p in (7919, 7927, 7933) if vocab % p)
    return (rank.clamp_(0, vocab - 1) * step) % vocab


def _randn(g, *shape, dev, dtype):
    return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).to(dtype)


def _inputs(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(1000003 * int(seed) + 17)
    dt = _DT[case["dtype"]]
    s = {"op": case["op"]}
    if case["op"] in ("embed", "embed_train"):
        B, L, V, E = case["batch"], case["length"], case["vocab"], case["width"]
        s["ids"] = _tokens(g, B, L, V, dev)
        s["table"] = _randn(g, V, E, dev=dev, dtype=dt)
        s["scale"] = case["scale"]
        s["padding_idx"] = None
        if case["op"] == "embed_train":
            if case["padded"]:      # sequences of 30 % to 100 % of the padded length; id 0 pads
                n = (L * (0.3 + 0.7 * torch.rand(B, 1, generator=g, device=dev))).ceil()
                s["ids"] = s["ids"].masked_fill(torch.arange(L, device=dev)[None] >= n, 0)
                s["padding_idx"] = 0
            s["dout"] = _randn(g, B, L, E, dev=dev, dtype=dt)
    elif case["op"] == "w4":
        M, N, K, G = case["rows"], case["n"], case["k"], case["group"]
        s["x"] = _randn(g, M, K, dev=dev, dtype=dt)
        # two codes a byte, the even one in the low half; a weight is (code - 8) * its group's scale
        s["codes"] = torch.randint(0, 256, (N, (K + 1) // 2), generator=g, device=dev, dtype=torch.uint8)
        groups = -(-K // G)
        s["scales"] = ((0.5 + torch.rand(N, groups, generator=g, device=dev)) * (0.2 / math.sqrt(K))).to(
            _DT[case["scales"]])
        s["k"], s["group"] = K, G
        s["bias"] = _randn(g, N, dev=dev, dtype=torch.float32) if case["bias"] else None
    else:
        B, V, L = case["rows"], case["vocab"], case["history"]
        s["logits"] = (3.0 * torch.randn(B, V, generator=g, device=dev)).to(dt)
        s["history"] = _tokens(g, B, L, V, dev)
        s["lengths"] = (L * (0.5 + 0.5 * torch.rand(B, generator=g, device=dev))).ceil().to(torch.int32)
        if case["own_penalties"]:
            s["repetition"] = 1.0 + 0.3 * torch.rand(B, generator=g, device=dev)
            s["presence"] = 0.5 * torch.rand(B, generator=g, device=dev)
            s["frequency"] = 0.2 * torch.rand(B, generator=g, device=dev)
        else:
            s["repetition"], s["presence"], s["frequency"] = 1.2, 0.0, 0.0
        s["bias"] = None
        if case["bias"] != "none":
            s["bias"] = torch.randn(*([V] if case["bias"] == "shared" else [B, V]), generator=g, device=dev)
        # one bit a token, lowest first; about half of a grammar's tokens are open, every token but some if shared
        words = -(-V // 32)
        w = torch.randint(-2**31, 2**31, (B if case["own_masks"] else 1, words), generator=g, device=dev)
        if not case["own_masks"]:
            w = w | torch.randint(-2**31, 2**31, (1, words), generator=g, device=dev) | ~torch.randint(
                -2**31, 2**31, (1, words), generator=g, device=dev)
            w = w[0]
        s["allowed"] = w.to(torch.int32)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case["op"] == "w4":
        from dasa_amd import ops
        s["weight"] = ops.pack_w4(s.pop("codes"), s.pop("scales"), s["k"], s["group"])
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(s):
    return _RUN_OWN[s["op"]](s) if own else _RUN[s["op"]](s)


def _embed(s):
    return (s["table"][s["ids"]].float() * s["scale"]).to(s["table"].dtype)


def _embed_train(s):
    out = _embed(s)
    V, E = s["table"].shape
    ids, d = s["ids"].reshape(-1), s["dout"].reshape(-1, E).float()
    if s["padding_idx"] is not None:
        d = d * (ids != s["padding_idx"])[:, None]
    dtable = torch.zeros(V, E, dtype=torch.float32, device=d.device).index_add_(0, ids, d)
    return out, (dtable * s["scale"]).to(s["table"].dtype)


def _w4(s):
    K, c = s["k"], s["codes"]
    q = torch.stack((c & 15, c >> 4), 2).reshape(c.shape[0], -1)[:, :K].float() - 8.0
    W = q * s["scales"].float().repeat_interleave(s["group"], 1)[:, :K]
    y = s["x"].float() @ W.t()
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["x"].dtype)


def _col(v, device):
    """A penalty as a column; a number becomes the 32-bit number nearest to it."""
    return v[:, None] if isinstance(v, torch.Tensor) else torch.full((1, 1), v, device=device)


def _allowed(words, V):
    bits = (words[..., None] >> torch.arange(32, device=words.device, dtype=torch.int32)) & 1
    return (bits != 0).flatten(-2)[..., :V]


def _rules(s):
    x = s["logits"].float()
    B, V = x.shape
    hist = s["history"]
    valid = torch.arange(hist.shape[1], device=x.device)[None] < s["lengths"][:, None]
    count = torch.zeros_like(x).scatter_add_(1, hist, valid.float())
    r, p, f = (_col(s[name], x.device) for name in ("repetition", "presence", "frequency"))
    seen = torch.where(x > 0, x / r, x * r) - f * count - p
    x = torch.where(count > 0, seen, x)
    if s["bias"] is not None:
        x = x + s["bias"]
    x = x.masked_fill(~_allowed(s["allowed"], V), -math.inf).to(s["logits"].dtype)
    at = torch.arange(V, device=x.device)
    choice = torch.where(x == x.amax(1, keepdim=True), at, V).amin(1)      # the lowest index of the largest value
    return x, choice


def _own_embed(s):
    from dasa_amd import ops
    return ops.embedding(s["ids"], s["table"], scale=s["scale"])


def _own_embed_train(s):
    from dasa_amd import ops
    out = ops.embedding(s["ids"], s["table"], scale=s["scale"])
    return out, ops.embedding_bwd(s["dout"], s["ids"], s["table"].shape[0], scale=s["scale"],
                                  padding_idx=s["padding_idx"])


def _own_w4(s):
    from dasa_amd import ops
    return ops.linear_w4(s["x"], s["weight"], s["bias"])


def _own_rules(s):
    from dasa_amd import ops
    return ops.logit_rules(s["logits"], s["history"], s["lengths"], repetition=s["repetition"],
                           presence=s["presence"], frequency=s["frequency"], bias=s["bias"], allowed=s["allowed"],
                           want_choice=True)


_RUN = {"embed": _embed, "embed_train": _embed_train, "w4": _w4, "rules": _rules}
_RUN_OWN = {"embed": _own_embed, "embed_train": _own_embed_train, "w4": _own_w4, "rules": _own_rules}


# ------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    e = _SIZE[case["dtype"]]
    if case["op"] in ("embed", "embed_train"):
        T, V, E = case["batch"] * case["length"], case["vocab"], case["width"]
        rows = min(T, V)                       # table rows read at most once each
        b = T * 8 + rows * E * e + T * E * e
        f = T * E
        if case["op"] == "embed_train":
            b += T * E * e + V * E * e
            f += T * E
        return {"bytes": b, "flops": f}
    if case["op"] == "w4":
        M, N, K = case["rows"], case["n"], case["k"]
        b = N * K / 2 + N * (-(-K // case["group"])) * _SIZE[case["scales"]] + (M * K + M * N) * e
        return {"bytes": b + (4 * N if case["bias"] else 0), "flops": 2 * M * N * K}
    B, V = case["rows"], case["vocab"]
    b = 2 * B * V * e + B * case["history"] * 0.75 * 8 + B * 8
    b += {"none": 0, "shared": 4 * V, "rows": 4 * B * V}[case["bias"]]
    b += (B if case["own_masks"] else 1) * V / 8
    return {"bytes": b, "flops": 4 * B * V}


# ------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] in ("embed", "embed_train"):
        V, E = s["table"].shape
        out = torch.index_select(s["table"].double(), 0, s["ids"].reshape(-1)).mul_(s["scale"]).view(*s["ids"].shape, E)
        if case["op"] == "embed":
            return out
        # the gradient from the running sum over the tokens in sorted order
        ids, order = torch.sort(s["ids"].reshape(-1), stable=True)
        total = s["dout"].reshape(-1, E)[order].double()
        if s["padding_idx"] is not None:
            total[ids == s["padding_idx"]] = 0.0
        total = torch.cumsum(total, 0)
        ends = torch.searchsorted(ids, torch.arange(V, device=ids.device), right=True)
        upto = torch.zeros(V + 1, E, dtype=torch.float64, device=ids.device)
        some = ends > 0
        upto[1:][some] = total[ends[some] - 1]
        return out, (upto[1:] - upto[:-1]) * s["scale"]
    if case["op"] == "w4":
        K, G, c = s["k"], s["group"], s["codes"].long()
        y = torch.zeros(s["x"].shape[0], c.shape[0], dtype=torch.float64, device=c.device)
        for g in range(-(-K // G)):             # group by group: integers, then the scale
            k = torch.arange(g * G, min(K, (g + 1) * G), device=c.device)
            q = torch.div(c[:, k // 2], 16 ** (k % 2), rounding_mode="floor") % 16 - 8
            y += (s["x"][:, k].double() @ q.double().t()) * s["scales"][:, g].double()
        return y if s["bias"] is None else y + s["bias"].double()
    x = s["logits"].double()
    B, V = x.shape
    open_ = _allowed(s["allowed"], V).expand(B, V)
    for b in range(B):
        ids = s["history"][b, :int(s["lengths"][b])]
        ids, count = torch.unique(ids, return_counts=True)
        r, p, f = (v[b].double() if isinstance(v, torch.Tensor) else float(v)
                   for v in (s["repetition"], s["presence"], s["frequency"]))
        if not isinstance(s["repetition"], torch.Tensor):   # a number is the 32-bit number nearest to it
            r = float(torch.tensor(r, dtype=torch.float32))
        l = x[b, ids]
        x[b, ids] = torch.maximum(l, torch.zeros_like(l)) / r + torch.minimum(l, torch.zeros_like(l)) * r \
            - count.double() * f - p
    if s["bias"] is not None:
        x = x + s["bias"].double()
    x[~open_] = -math.inf
    return x, None
