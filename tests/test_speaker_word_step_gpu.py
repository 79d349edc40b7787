"""The word step of the speaker on the token operators: Speaker.infer_batch with rules on its logits, SpeakerDecoder
on 4-bit weights, and BertEmbeddings' gradients (dasa_amd.r2r) against plain forms."""
import contextlib
import io
import os

import numpy as np
import pytest
import torch

from tests import golden_inputs as GI
from tests.helpers import GOLDEN

pytestmark = pytest.mark.gpu


@contextlib.contextmanager
def _speaker():
    cfg = GI.SPEAKER
    from dasa_amd.r2r import param
    param.readme_train(["--maxDecode", str(cfg["max_decode"]), "--batchSize", str(cfg["batch"])])
    try:
        from dasa_amd.r2r import agent_dg, speaker, utils
        from dasa_amd.synth import SynthR2RBatch, SynthWorld, init_params
        tok = utils.Tokenizer(vocab=utils.read_vocab(os.path.join(GOLDEN, "train_vocab.txt")), encoding_length=80)
        world = SynthWorld(cfg["viewpoints"], 0, cfg["graph_seed"])
        env = SynthR2RBatch(world, cfg["batch"], seed=cfg["env_seed"], mode="goal", instr_len=80, variable_len=True)
        with contextlib.redirect_stdout(io.StringIO()):
            listener = agent_dg.Seq2SeqAgent(env, "", None, 5, "Dic")
        spk = speaker.Speaker(env, listener, tok)
        init_params(spk.encoder, cfg["seed_enc"])
        init_params(spk.decoder, cfg["seed_dec"])
        yield spk
    finally:
        param.readme_train(["--d_vl_layers", "1", "--batchSize", "2", "--maxAction", "5"])


def _record(spk):
    """Every word's logits as the decoder returned them (infer_batch writes its rules into them)."""
    seen, fwd = [], spk.decoder.forward

    def wrapped(*a, **k):
        r = fwd(*a, **k)
        seen.append(r[0].detach().cpu().double().squeeze(1).clone())
        return r
    spk.decoder.forward = wrapped
    return seen


def test_infer_batch_with_rules(dev):
    with _speaker() as spk:
        w2i, V = spk.tok.word_to_index, spk.tok.vocab_size()
        spk.env.reset()
        g = torch.Generator().manual_seed(3)
        allowed = torch.rand(V, generator=g) < 0.7
        allowed[w2i["<EOS>"]] = True
        bias = 0.1 * torch.randn(V, generator=g)
        seen = _record(spk)
        insts = spk.infer_batch(repetition=1.5, presence=0.05, frequency=0.02, bias=bias.to(dev), allowed=allowed.to(dev))
        B = insts.shape[0]
        assert len(seen) == insts.shape[1] and not (insts == w2i["<UNK>"]).any()
        # the same choice from the recorded logits by the plain rules in 64 bits; a row that has ended writes <PAD>
        # while its own words go on, so each row is followed up to its end
        words = np.zeros((B, 0), np.int64)
        f32 = lambda v: torch.tensor(v, dtype=torch.float32).double()   # noqa: E731
        ended = np.zeros(B, bool)
        for t, x in enumerate(seen):
            x = x.clone()
            for b in range(B):
                for v in set(words[b].tolist()):
                    c = int((words[b] == v).sum())
                    l = x[b, v]
                    l = l / f32(1.5) if l > 0 else l * f32(1.5)
                    x[b, v] = l - f32(0.02) * c - f32(0.05)
            x = x + bias.double()
            x[:, ~allowed] = -float("inf")
            x[:, w2i["<UNK>"]] = -float("inf")
            top = x.topk(2, 1)
            for b in range(B):
                if not ended[b]:
                    # the gap between the two best is far above fp32 roundings of values below 16 (6 x 2^-21)
                    assert float(top.values[b, 0] - top.values[b, 1]) > 3e-6
                    assert int(insts[b, t]) == int(top.indices[b, 0])
            step = top.indices[:, 0].numpy()
            words = np.concatenate([words, step[:, None]], 1)
            ended |= step == w2i["<EOS>"]
            if ended.all():
                break


def test_infer_batch_neutral_rules_change_nothing(dev):
    with _speaker() as spk:
        spk.env.reset()
        base = spk.infer_batch()
    with _speaker() as spk:
        spk.env.reset()
        assert np.array_equal(base, spk.infer_batch(repetition=1.0))
    with _speaker() as spk:
        spk.env.reset()
        V = spk.tok.vocab_size()
        only = torch.zeros(V, dtype=torch.bool, device=dev)
        only[17] = True
        forced = spk.infer_batch(allowed=only, sampling=True)
        assert (forced == 17).all() and forced.shape[1] == GI.SPEAKER["max_decode"]


def test_speaker_decoder_on_4bit_weights(dev):
    from dasa_amd import ops
    from dasa_amd._lib import DasaError
    from dasa_amd.r2r import model
    torch.manual_seed(5)
    dec = model.SpeakerDecoder(992, 256, 0, 512, 0.0).to(dev).eval()
    with torch.no_grad():
        for name, p in dec.named_parameters():
            p.copy_(torch.randn(p.shape, generator=torch.Generator().manual_seed(len(name))).to(dev) * 0.08)
        words = torch.randint(0, 992, (20, 3), generator=torch.Generator().manual_seed(1)).to(dev)
        ctx = torch.randn(20, 7, 512, generator=torch.Generator().manual_seed(2)).to(dev)
        mask = torch.zeros(20, 7, dtype=torch.bool, device=dev)
        mask[3, 4:] = True
        h = torch.zeros(1, 20, 512, device=dev)
        plain = dec(words, ctx, mask, h, h)
        keys = set(dec.state_dict())
        dec.quantize_w4(32)
        assert set(dec.state_dict()) == keys
        got = dec(words, ctx, mask, h, h)
        one = dec(words[:, :1], ctx, mask, h, h)[0]
        # the same step with the weights replaced by the values the codes stand for: equal up to the fp32 sums of the
        # two products (K <= 1024 terms each, magnitudes below 0.1 sum |x w| = 30: 30 x 1024 x 2^-24 x 2 < 4e-3); the
        # weights' own rounding, up to 0.5 / 7 of a group's largest, moves the logits further than that
        q = {k: v[0].dequantize() for k, v in dec._w4.items()}
        dec.dequantize_w4()
        for k, W in dec._word_linears().items():
            W.copy_(q[k])
        want = dec(words, ctx, mask, h, h)
        for a, b in zip(got, want):
            assert float((a - b).abs().max()) < 4e-3
        assert float((one[:, 0] - got[0][:, 0]).abs().max()) == 0.0
        assert float((got[0] - plain[0]).abs().max()) > 1e-2
        dec.quantize_w4()
        dec.projection.weight.mul_(1.0)
        with pytest.raises(DasaError, match="changed since"):
            dec(words, ctx, mask, h, h)
        dec.quantize_w4()
        dec(words, ctx, mask, h, h)
    with pytest.raises(DasaError, match="infinities"):
        ops.quantize_w4(torch.full((4, 64), float("inf"), device=dev))


@pytest.mark.parametrize("B,L", [(1, 1), (3, 17), (20, 80)])
def test_bert_embeddings_gradients(dev, B, L):
    """BertEmbeddings with its tables trained: outputs as before, gradients of the formula in 64 bits."""
    from dasa_amd.r2r import param, vilmodel
    param.readme_train([])
    cfg = vilmodel.BertConfig(vocab_size=500, hidden_size=768, update_embeddings=True)
    m = vilmodel.BertEmbeddings(cfg).to(dev).eval()
    g = torch.Generator().manual_seed(B * L)
    with torch.no_grad():
        for p in m.parameters():
            p.copy_(torch.randn(p.shape, generator=g).to(dev))
    ids = torch.randint(0, 500, (B, L), generator=g)
    ids[:, L // 2 + 1:] = 0                                     # padding
    with torch.no_grad():
        base = m(ids.to(dev))
    y = m(ids.to(dev))
    assert y.requires_grad and torch.equal(y, base)
    dy = torch.randn(B, L, 768, generator=g)
    y.backward(dy.to(dev))
    t = {k: v.detach().cpu().double().requires_grad_() for k, v in m.named_parameters()}
    e = torch.nn.functional.embedding(ids, t["word_embeddings.weight"], padding_idx=0) + \
        t["position_embeddings.weight"][:L] + t["token_type_embeddings.weight"][0]
    torch.nn.functional.layer_norm(e, (768,), t["LayerNorm.weight"], t["LayerNorm.bias"], cfg.layer_norm_eps).backward(dy.double())
    n = B * L
    for k, p in m.named_parameters():
        want, got = t[k].grad, p.grad.cpu().double()
        # sums of at most n terms of magnitude below 30, each off by a few fp32 steps of LayerNorm's 768-term sums
        assert float((got - want).abs().max()) < 30 * n * 64 * 2.0**-24 + 1e-5, k
    assert bool((m.word_embeddings.weight.grad[0] == 0).all())
    m.trained = False
    assert not m(ids.to(dev)).requires_grad


def test_bert_embeddings_gradients_with_dropout_regenerate_the_mask(dev):
    from dasa_amd import functional as DF
    g = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g).to(dev).requires_grad_()   # noqa: E731
    word, pos, typ, gamma, beta = r(50, 64), r(16, 64), r(2, 64), r(64), r(64)
    ids = torch.randint(0, 50, (4, 16), generator=g).to(dev)
    y = DF.bert_embed(ids, word, pos, typ, gamma, beta, 1e-12, 0.5, True, 0)
    keep = (y != 0).double().cpu()                              # LayerNorm's values are not zero
    y.backward(torch.ones_like(y))
    want = (keep * 2.0).sum((0, 1))                             # d beta: the kept places times 1 / (1 - p)
    assert float((beta.grad.cpu().double() - want).abs().max()) < 1e-4


def test_training_step_reaches_the_tables_on_request(dev):
    """A finetune iteration of the agent with the language stack trained (--d_transformer_update True): with
    --d_update_embeddings the tables and the LayerNorm of BertEmbeddings get gradients, and the loss and every other
    gradient stay as without it."""
    from dasa_amd import functional as DF
    from dasa_amd.r2r import param
    from dasa_amd.r2r.agent_dg import Seq2SeqAgent
    from dasa_amd.synth import SynthR2RBatch, SynthWorld, init_params
    res = {}
    try:
        for on in (False, True):
            param.readme_finetune(["--d_vl_layers", "1", "--batchSize", "2", "--maxAction", "2",
                                   "--d_transformer_update", "True"] + (["--d_update_embeddings"] if on else []))
            torch.manual_seed(3)
            env = SynthR2RBatch(SynthWorld(32, 0, 5), 2, seed=701, mode="wander", instr_len=80, variable_len=True)
            with contextlib.redirect_stdout(io.StringIO()):
                ag = Seq2SeqAgent(env, "", None, 2, "Dic")
            for m, s in ((ag.encoder, 1), (ag.decoder, 2), (ag.critic, 3), (ag.adaIn, 4)):
                init_params(m, s)
                for sub in m.modules():
                    if isinstance(sub, torch.nn.Dropout):
                        sub.p = 0.0
            param.args.ml_weight = param.args.ml_weight_org
            assert ag.encoder.bert.update_lang_bert and ag.encoder.bert.embeddings.trained == on
            table = GI.forced_table(2, 2, seed=GI.FORCED_SEED)
            ag.force_action_fn = lambda t, lens, table=table: GI.forced_actions(table, t, lens, no_stop=True)
            ag.zero_grad()
            ag.accumulate_gradient("sample")
            loss = ag.loss.item()
            with DF.defer_bilstm_backward(), DF.defer_weight_grads():
                ag.loss.backward()
                DF.flush_bilstm_backward()
            DF.flush_weight_grads()
            res[on] = loss, {f"{i}.{k}": p.grad.detach().clone() for i, m in enumerate(ag.models)
                             for k, p in m.named_parameters() if p.grad is not None}
            del ag
    finally:
        param.readme_train(["--d_vl_layers", "1", "--batchSize", "2", "--maxAction", "5"])
    (l0, g0), (l1, g1) = res[False], res[True]
    new = {"0.bert.embeddings." + k for k in ("word_embeddings.weight", "position_embeddings.weight",
                                              "token_type_embeddings.weight", "LayerNorm.weight", "LayerNorm.bias")}
    assert l0 == l1 and set(g1) - set(g0) == new and set(g0) <= set(g1)
    assert any(k.startswith("0.bert.lalayer") for k in g0)
    for k in g0:                              # the same kernels on the same values: equal bit for bit
        assert torch.equal(g0[k], g1[k]), k
    for k in new:
        assert bool(g1[k].isfinite().all()) and float(g1[k].abs().max()) > 0, k
    assert bool((g1["0.bert.embeddings.word_embeddings.weight"][0] == 0).all())
