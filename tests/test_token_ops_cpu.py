"""Refusals of the token operators (dasa_amd.ops): wrong types, shapes and devices raise DasaError on the host, and the
C entries return hipErrorInvalidValue before anything is launched. No GPU needed."""
import ctypes

import pytest
import torch

from dasa_amd import _lib, functional as DF, ops
from dasa_amd._lib import DasaError

INVALID = 1


def _refused(match, f, *a, **k):
    with pytest.raises(DasaError, match=match):
        f(*a, **k)


def test_host_tensors_are_refused():
    ids, table = torch.zeros(3, dtype=torch.int64), torch.zeros(5, 4)
    _refused("device tensors", ops.embedding, ids, table)
    _refused("device tensors", DF.embedding, ids, table)
    _refused("device tensors", ops.embedding_bwd, torch.zeros(3, 4), ids, 5)
    _refused("device tensors", ops.quantize_w4, torch.zeros(4, 64))
    _refused("device tensors", ops.pack_w4, torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 1), 64, 64)
    w = ops.W4Weight(torch.zeros(256, dtype=torch.int32), torch.zeros(32), (4, 64), 64)
    _refused("device tensors", ops.linear_w4, torch.zeros(2, 64), w)
    _refused("device tensors", ops.logit_rules, torch.zeros(2, 8))


def test_embedding_arguments():
    ids, table = torch.zeros(3, dtype=torch.int64), torch.zeros(5, 4)
    _refused("float32 or bfloat16", ops.embedding, ids, table.double())
    _refused("float32 or bfloat16", ops.embedding, ids, table.half())
    _refused("int64 or int32", ops.embedding, ids.to(torch.int16), table)
    _refused("int64 or int32", ops.embedding, ids.float(), table)
    _refused(r"\[V, E\]", ops.embedding, ids, table[0])
    d = torch.zeros(3, 4)
    _refused("float32 or bfloat16", ops.embedding_bwd, d.double(), ids, 5)
    _refused("padding_idx", DF.embedding, ids, table, 1.0, 5)
    _refused("padding_idx", DF.embedding, ids, table, 1.0, -1)


def test_w4_arguments():
    codes, scales = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 1)
    for group in (0, 16, 48, 256):
        _refused("group", ops.pack_w4, codes, scales, 64, group)
        _refused("group", ops.quantize_w4, torch.zeros(4, 64), group)
    _refused("describe", ops.pack_w4, codes, scales, 66, 64)
    _refused("describe", ops.pack_w4, codes, scales, 64, 32)
    _refused("describe", ops.pack_w4, codes.int(), scales, 64, 64)
    _refused("describe", ops.pack_w4, codes, scales[:3], 64, 64)
    _refused("float32 or bfloat16", ops.pack_w4, codes, scales.half(), 64, 64)
    _refused(r"\[N, K\]", ops.quantize_w4, torch.zeros(4))
    _refused(r"\[N, K\]", ops.quantize_w4, torch.zeros(0, 4))
    _refused("scales are", ops.quantize_w4, torch.zeros(4, 64), 64, torch.float16)
    w = ops.W4Weight(torch.zeros(256, dtype=torch.int32), torch.zeros(32), (4, 64), 64)
    _refused("W4Weight", ops.linear_w4, torch.zeros(2, 64), torch.zeros(4, 64))
    _refused("end in K", ops.linear_w4, torch.zeros(2, 65), w)
    _refused("float32 or bfloat16", ops.linear_w4, torch.zeros(2, 64).double(), w)
    _refused("bias", ops.linear_w4, torch.zeros(2, 64), w, torch.zeros(5))
    _refused("bias", ops.linear_w4, torch.zeros(2, 64), w, torch.zeros(4, dtype=torch.bfloat16))
    _refused("activation", ops.linear_w4, torch.zeros(2, 64), w, None, "swish")


def test_logit_rules_arguments():
    x = torch.zeros(2, 8)
    _refused(r"\[B, V\]", ops.logit_rules, x[0])
    _refused("float32 or bfloat16", ops.logit_rules, x.half())


def test_entry_points_refuse_before_a_launch():
    """Addresses are made up: nothing here may reach a launch."""
    L = _lib.lib()
    P = 0x100000
    assert L.dasa_embedding_fwd(P, 8, P, 8, 0, 10, 8, 1.0, 0, P, 8, None, None) == 0           # no tokens
    for T, V, E, nb, ldt, ldo in ((-1, 10, 8, 8, 8, 8), (4, 0, 8, 8, 8, 8), (4, 10, 8, 2, 8, 8), (4, 10, 8, 8, 7, 8),
                                  (4, 10, 8, 8, 8, 7), (4, -1, 8, 8, 8, 8), (4, 2**30 + 1, 8, 8, 8, 8),
                                  (4, 10, 2**30 + 1, 8, 2**31, 2**31)):
        assert L.dasa_embedding_fwd(P, ldt, P, nb, T, V, E, 1.0, 0, P, ldo, None, None) == INVALID
    assert L.dasa_embedding_fwd(None, 8, P, 8, 4, 10, 8, 1.0, 0, P, 8, None, None) == INVALID
    assert L.dasa_embedding_bwd_workspace(2**31, 50, 8) == 0 and L.dasa_embedding_bwd_workspace(100, 50, 8) == 0
    T0 = 100000
    need = L.dasa_embedding_bwd_workspace(T0, 50, 8)
    assert need >= 4 * (T0 + 51)
    for T, nb, ldd, ldt, ws, n in ((2**31, 8, 8, 8, P, need), (T0, 1, 8, 8, P, need), (T0, 8, 7, 8, P, need),
                                   (T0, 8, 8, 7, P, need), (T0, 8, 8, 8, None, need), (T0, 8, 8, 8, P, need - 1),
                                   (-1, 8, 8, 8, P, need), (100, 8, 7, 8, None, 0), (100, 8, 8, 7, None, 0)):
        assert L.dasa_embedding_bwd(P, ldd, P, nb, T, 50, 8, 1.0, -1, 0, P, ldt, 0, ws, n, None) == INVALID
    assert L.dasa_w4_weight_bytes(17, 129) == 2 * 2 * 1024 and L.dasa_w4_weight_bytes(0, 4) == 0
    assert L.dasa_embedding_bwd(P, 8, P, 8, T0, 2**30 + 1, 8, 1.0, -1, 0, P, 8, 0, P, 2**40, None) == INVALID
    assert L.dasa_w4_weight_bytes(2**30 + 1, 64) == 0 and L.dasa_w4_weight_bytes(64, 2**31 - 1) == 0
    assert L.dasa_gemm_w4(P, 2**31, 0, P, P, 0, 64, None, 0, 0.0, P, 4, 1, 4, 2**31 - 1, None, 0, None) == INVALID
    assert L.dasa_gemm_w4(P, 64, 0, P, P, 0, 64, None, 0, 0.0, P, 4, 65535 * 16 + 1, 4, 64, None, 0, None) == INVALID
    assert L.dasa_w4_scale_count(17, 129, 64) == 2 * 2 * 2 * 16 and L.dasa_w4_scale_count(17, 129, 16) == 0
    assert L.dasa_w4_quantize(P, 64, 0, 4, 64, 16, P, 32, P, 4, 0, None) == INVALID
    assert L.dasa_w4_quantize(P, 63, 0, 4, 64, 64, P, 32, P, 1, 0, None) == INVALID
    assert L.dasa_w4_layout(P, 31, P, 1, 0, 4, 64, 64, P, P, None) == INVALID
    assert L.dasa_gemm_w4(P, 64, 0, P, P, 0, 64, None, 0, 0.0, P, 4, 0, 4, 64, None, 0, None) == 0        # no rows
    for ldx, w, group, act, ldy, M in ((63, P, 64, 0, 4, 2), (64, P + 8, 64, 0, 4, 2), (64, P, 65, 0, 4, 2),
                                       (64, P, 64, 9, 4, 2), (64, P, 64, 0, 3, 2), (64, P, 64, 0, 4, -1)):
        assert L.dasa_gemm_w4(P, ldx, 0, w, P, 0, group, None, act, 0.0, P, ldy, M, 4, 64, None, 0, None) == INVALID
    good = dict(B=2, V=9000, L=4, ids_bytes=8, logits=P, ld=9000, out=P, ldo=9000, history=P, ldh=4, repetition0=1.0)
    def desc(**kw):
        d = _lib.LogitRules()
        for k, v in {**good, **kw}.items():
            setattr(d, k, v)
        return ctypes.byref(d)
    for kw in (dict(V=0), dict(B=-1), dict(B=65536), dict(ld=8999), dict(ldo=8999), dict(ids_bytes=3), dict(ldh=3),
               dict(logits=None), dict(L=-1), dict(bias=P, ldb=8999), dict(allowed_bits=P, ldbits=281),
               dict(allowed_bytes=P, ldbytes=8999), dict(allowed_bits=P, allowed_bytes=P), dict(choice=P),
               dict(V=2**30 + 1, ld=2**31, ldo=2**31), dict(L=2**30 + 1, ldh=2**31)):
        assert L.dasa_logit_rules(desc(**kw), None, 0, None) == INVALID, kw
    assert L.dasa_logit_rules(desc(B=0), None, 0, None) == 0


def test_capture_beside_a_live_eager_graph_is_refused(monkeypatch):
    """functional's record of live eager graphs, with the stream and the capture state of a device played by the host."""
    from dasa_amd import functional as DF
    state = dict(capturing=False, stream=0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])
    monkeypatch.setattr(ops, "_stream", lambda: state["stream"])
    table, other = torch.zeros(4, 2, requires_grad=True), torch.zeros(4, 2, requires_grad=True)
    use = DF._leaf_use((table, torch.zeros(3)))
    state["capturing"] = True
    assert DF._leaf_use((other,)) is None
    _refused("AutogradGraphs", DF._leaf_use, (other, table))
    del use                                                    # the eager graph is gone
    assert DF._leaf_use((table,)) is None
    state.update(capturing=False, stream=7)                    # a warm-up on a side stream
    assert DF._leaf_use((table,)) is None
    state.update(capturing=True)
    assert DF._leaf_use((table,)) is None
    key = id(other)
    state.update(capturing=False, stream=0)
    keep = DF._leaf_use((other,))
    assert key in DF._USES
    del other
    assert key not in DF._USES and keep is not None


class _Codes:
    """Stands for a 4-bit weight where none can be made (no device)."""
    device = torch.device("cpu")


@pytest.mark.parametrize("change", ["in place", "data", "vector", "type and back", "transposed", "address reused",
                                    "object"])
def test_speaker_decoder_refuses_4bit_forms_of_other_weights(monkeypatch, change):
    """quantize_w4() followed by anything that gives a weight other values: forward may not go on with the old codes."""
    from dasa_amd.r2r import model
    monkeypatch.setattr(ops, "quantize_w4", lambda W, group, scale_dtype: _Codes())
    monkeypatch.setattr(ops, "linear_w4", lambda x, q, b, act=None, out=None, beta=0.0: "ran")
    dec = model.SpeakerDecoder(12, 4, 0, 4, 0.0)
    dec.quantize_w4()
    lin = dec.attention_layer.linear_in                     # square: a transposed view keeps its shape
    run = lambda: dec._linear("att_in", lin.weight, None)   # noqa: E731
    with torch.no_grad():
        assert run() == "ran" and run() == "ran"
        if change == "in place":
            lin.weight.mul_(2.0)
        elif change == "data":
            lin.weight.data = lin.weight.data * 2.0
        elif change == "vector":
            v = torch.nn.utils.parameters_to_vector(dec.parameters()) * 2.0
            torch.nn.utils.vector_to_parameters(v, dec.parameters())
        elif change == "type and back":
            dec.half().float()
        elif change == "transposed":
            lin.weight.data = lin.weight.data.t()
        elif change == "address reused":                    # the old values' memory may not come back as new values'
            at = lin.weight.data_ptr()
            for _ in range(50):
                lin.weight.data = torch.empty(0)
                lin.weight.data = torch.randn(4, 4)
                assert lin.weight.data_ptr() != at
        else:
            lin.weight = torch.nn.Parameter(lin.weight.detach().clone())
        _refused("changed since", run)
        dec.quantize_w4()
        assert run() == "ran"
        dec.dequantize_w4()
        assert not dec._w4


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32, torch.int16, torch.uint8, torch.float32])
def test_speaker_decoder_takes_words_of_any_number_type(monkeypatch, dtype):
    """forward converts the words for the lookup, which takes int64 and int32."""
    from dasa_amd.r2r import model
    seen = []

    def lookup(ids, table):
        seen.append(ids)
        raise KeyboardInterrupt                             # the rest of the step needs a device
    monkeypatch.setattr(ops, "embedding", lookup)
    dec = model.SpeakerDecoder(12, 4, 0, 4, 0.0)
    words = torch.tensor([[3], [11], [0]]).to(dtype)
    with torch.no_grad(), pytest.raises(KeyboardInterrupt):
        dec(words, None, None, torch.zeros(1, 3, 4), torch.zeros(1, 3, 4))
    ids, = seen
    assert ids.dtype in (torch.int64, torch.int32) and torch.equal(ids.long(), words.long())


def _double(f, *leaves):
    """A second derivative through f's first gradients, with the upstream gradient itself depending on a leaf."""
    a = torch.ones((), requires_grad=True)
    y = f()
    g = torch.autograd.grad((y * a).sum() + a * a, (*leaves, a), create_graph=True)
    sum(t.sum() for t in g).backward()


@pytest.mark.parametrize("which", ["embedding", "bert_embed"])
def test_second_derivatives_are_refused(monkeypatch, which):
    """The lookups' backward passes are kernels: differentiating through them raises instead of dropping the part that
    goes through them. First gradients under create_graph=True are unharmed."""
    monkeypatch.setattr(DF, "_leaf_use", lambda leaves: None)
    monkeypatch.setattr(ops, "embedding", lambda ids, table, scale=1.0: table.detach()[ids] * scale)
    monkeypatch.setattr(ops, "embedding_bwd", lambda d, ids, V, scale=1.0, padding_idx=None:
                        torch.zeros(V, d.shape[-1]).index_add_(0, ids.reshape(-1), d.detach().reshape(-1, d.shape[-1])) * scale)
    monkeypatch.setattr(ops, "bert_embed", lambda ids, w, p, t, ga, be, eps, pr, seed: w.detach()[ids])
    monkeypatch.setattr(ops, "add2d", lambda a, b: a + b)
    monkeypatch.setattr(ops, "layernorm", lambda x, g, b, eps, save: (x, x))
    monkeypatch.setattr(ops, "layernorm_bwd", lambda dy, saved, g, dg, db: dy.detach())
    ids, table = torch.tensor([[1, 3, 1]]), torch.randn(5, 4, requires_grad=True)
    if which == "embedding":
        f, leaves = (lambda: DF.embedding(ids, table)), (table,)
    else:
        more = [torch.randn(*s, requires_grad=True) for s in ((3, 4), (2, 4), (4,), (4,))]
        f, leaves = (lambda: DF.bert_embed(ids, table, *more, 1e-12)), (table, *more)
    first = torch.autograd.grad(f().sum(), leaves, create_graph=True)
    assert torch.equal(first[0], torch.tensor([0.0, 2, 0, 1, 0])[:, None].expand(5, 4))
    with pytest.raises(RuntimeError, match="once_differentiable"):
        _double(f, *leaves)


def test_lookup_of_a_trained_table_without_a_gradient_is_refused():
    """ops.embedding makes no graph: in grad mode a table that wants a gradient goes through functional.embedding."""
    ids, table = torch.zeros(3, dtype=torch.int64), torch.zeros(5, 4, requires_grad=True)
    _refused("forward only", ops.embedding, ids, table)
    with torch.no_grad():
        _refused("device tensors", ops.embedding, ids, table)          # as far as host tensors come
    _refused("device tensors", ops.embedding, ids, table.detach())


def test_logit_rules_of_arguments_that_want_a_gradient_are_refused(monkeypatch):
    """Not the logits alone: a bias or a penalty in grad mode would lose its gradient as well."""
    monkeypatch.setattr(ops, "_on_device", lambda what, *ts: 0)
    x, leaf = torch.zeros(2, 8), lambda *s: torch.ones(*s, requires_grad=True)   # noqa: E731
    for kw in (dict(bias=leaf(8)), dict(bias=leaf(2, 8)), dict(repetition=leaf(2)), dict(presence=leaf(2)),
               dict(frequency=leaf(2))):
        _refused("forward only", ops.logit_rules, x, **kw)
    _refused("forward only", ops.logit_rules, x.clone().requires_grad_())


def test_embedding_bwd_of_a_gradient_that_wants_one_is_refused():
    d, ids = torch.zeros(3, 4, requires_grad=True), torch.zeros(3, dtype=torch.int64)
    _refused("forward only", ops.embedding_bwd, d, ids, 5)
    with torch.no_grad():
        _refused("device tensors", ops.embedding_bwd, d, ids, 5)


def test_logit_rules_numbers_outside_fp32_are_refused(monkeypatch):
    """The kernel takes the 32-bit number nearest to a penalty: one that becomes 0 or infinite there is none."""
    monkeypatch.setattr(ops, "_on_device", lambda what, *ts: 0)
    x = torch.zeros(2, 8)
    for kw in (dict(repetition=1e-50), dict(repetition=1e39), dict(presence=1e39), dict(frequency=-1e39),
               dict(repetition=0.0), dict(repetition=-1.0), dict(presence=float("nan"))):
        _refused(f"{next(iter(kw))} =", ops.logit_rules, x, **kw)


def test_gradients_that_no_launch_can_hold_are_refused_at_the_check():
    """A launch takes fewer than 2^32 threads in a dimension and 65535 workgroups in the second: such sizes are refused
    before the first kernel. Addresses are made up."""
    L, P = _lib.lib(), 0x100000
    for V, E, bf in ((2**30, 600, 1), (2**30, 260, 0), (2**29 + 1, 1030, 1), (2**28 + 1, 2**20, 0)):
        assert L.dasa_embedding_bwd(P, E, P, 8, 4, V, E, 1.0, -1, bf, P, E, 0, None, 0, None) == INVALID, (V, E)
    T, E = 9000, 16776961
    need = L.dasa_embedding_bwd_workspace(T, 50, E)
    assert L.dasa_embedding_bwd(P, E, P, 8, T, 50, E, 1.0, -1, 0, P, E, 0, P, need, None) == INVALID


def test_4bit_weights_that_no_launch_can_lay_out_are_refused_at_the_check():
    """The layout has 256 threads for 16 x 512 values, and a launch takes fewer than 2^32. Addresses are made up."""
    L, P = _lib.lib(), 0x100000
    for N, K in ((2**28, 64), (2**28 - 15, 512), (2**27, 513), (2**30, 1), (32768, 2**22), (2**20, 2**30)):
        assert L.dasa_w4_weight_bytes(N, K) == 0 and L.dasa_w4_scale_count(N, K, 64) == 0, (N, K)
        g = -(-K // 64)
        assert L.dasa_w4_quantize(P, K, 0, N, K, 64, P, K, P, g, 0, None) == INVALID, (N, K)
        assert L.dasa_w4_layout(P, K, P, g, 0, N, K, 64, P, P, None) == INVALID, (N, K)
        assert L.dasa_gemm_w4(P, K, 0, P, P, 0, 64, None, 0, 0.0, P, N, 1, N, K, None, 0, None) == INVALID, (N, K)
    for N, K in ((2**28 - 16, 512), (2**27 - 16, 1024), (16, 2**30), (32768, 2**22 - 512)):
        assert L.dasa_w4_weight_bytes(N, K) == -(-N // 16) * -(-K // 128) * 1024


def test_entry_points_refuse_buffers_that_are_not_aligned():
    """The header asks for 16-B alignment of tiles, scale tiles and workspaces, which are read in 16-B vectors."""
    L, P = _lib.lib(), 0x100000
    for off in (2, 4, 8):
        assert L.dasa_gemm_w4(P, 64, 0, P, P + off, 0, 32, None, 0, 0.0, P, 4, 2, 4, 64, None, 0, None) == INVALID
        assert L.dasa_gemm_w4(P, 64, 0, P + off, P, 0, 32, None, 0, 0.0, P, 4, 2, 4, 64, None, 0, None) == INVALID
        assert L.dasa_w4_layout(P, 32, P, 2, 0, 4, 64, 32, P + off, P, None) == INVALID
        assert L.dasa_w4_layout(P, 32, P, 2, 0, 4, 64, 32, P, P + off, None) == INVALID
        need = L.dasa_gemm_w4_workspace(1, 1000, 8192, 0)
        assert need > 0
        assert L.dasa_gemm_w4(P, 8192, 0, P, P, 0, 32, None, 0, 0.0, P, 1000, 1, 1000, 8192, P + off, need, None) == INVALID
        need = L.dasa_embedding_bwd_workspace(9000, 50, 8)
        assert L.dasa_embedding_bwd(P, 8, P, 8, 9000, 50, 8, 1.0, -1, 0, P, 8, 0, P + off, need, None) == INVALID
        need = L.dasa_logit_rules_workspace(2, 9000)
        assert need > 0
        d = _lib.LogitRules()
        for k, v in dict(B=2, V=9000, logits=P, ld=9000, out=P, ldo=9000, repetition0=1.0, choice=P).items():
            setattr(d, k, v)
        assert L.dasa_logit_rules(ctypes.byref(d), P + off, need, None) == INVALID


def test_4bit_weight_of_tensors_that_do_not_hold_it_is_refused():
    """linear_w4 reads what the shape says: tiles or scales of another size, type or device never get that far."""
    tiles, scales = torch.zeros(2 * 2 * 256, dtype=torch.int32), torch.zeros(2 * 2 * 2 * 16)
    assert ops.W4Weight(tiles, scales, (17, 129), 64).nbytes == 4 * (tiles.numel() + scales.numel())
    for t, s, shape, group in ((tiles[:-1], scales, (17, 129), 64), (tiles, scales[:-1], (17, 129), 64),
                               (tiles, scales, (33, 129), 64), (tiles, scales, (17, 257), 64),
                               (tiles, scales, (17, 129), 32), (tiles, scales, (17, 129), 48),
                               (tiles.float(), scales, (17, 129), 64), (tiles, scales.half(), (17, 129), 64),
                               (tiles[::2], scales, (1, 129), 64), (tiles, scales, (0, 129), 64),
                               (tiles, scales.to("meta"), (17, 129), 64)):
        _refused("W4Weight", ops.W4Weight, t, s, shape, group)


def test_logit_rules_out_over_a_penalty_is_refused(monkeypatch):
    """Other workgroups may still read a row's penalties when the first has written its slice."""
    monkeypatch.setattr(ops, "_on_device", lambda what, *ts: 0)
    buf = torch.ones(40)
    x, out = torch.zeros(2, 8), buf[10:26].view(2, 8)
    for name in ("repetition", "presence", "frequency"):
        for at in (9, 10, 17, 25):
            _refused("overlaps", ops.logit_rules, x, out=out, **{name: buf[at:at + 2]})


def test_gradient_sort_has_no_step_at_4_million_tokens():
    """The two-launch sort, whose counts are part of the workspace, ends where its counts outweigh the tokens, not at a
    number of tokens: one more token never needs much less workspace, except there."""
    need = lambda T, V: _lib.lib().dasa_embedding_bwd_workspace(T, V, 8)   # noqa: E731
    for V in (2, 1000, 50021, 102400):
        for T in (2**22, 2**23):
            assert 0 <= need(T + 1, V) - need(T, V) < 4096, (T, V)
    assert need(393216, 300000) - need(393215, 300000) > 8 * 300000 * 4      # begins at 1536 tokens an owner
    assert need(2**22, 300000) < 2**22 * 8                                   # and has ended


def test_profile_families_name_kernels_that_exist():
    """The profile looks a family's kernel up by its first word."""
    import glob
    import os
    import re

    from dasa_amd import build, prof
    text = "".join(open(f).read() for f in glob.glob(os.path.join(build.CSRC, "*")))
    for family in ("embed", "embed_bwd", "gemm_w4", "logit_rules"):
        names = re.findall(r"\w+_kernel", prof.FAMILIES[family][1])
        assert names and prof.FAMILIES[family][1].split(" ")[0] == names[0], family
        for n in names:
            assert re.search(rf"void {n}\(", text), (family, n)
