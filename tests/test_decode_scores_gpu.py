"""The 8-bit cache and the token scores where the framework uses them: greedy decoding with kv_cache="fp8" and scores, teacher-forced
scores with their gradient, the sampling script."""
import math
import os
import sys

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
from helpers import rel_l2  # noqa: E402
from kv8_reference import Cache  # noqa: E402

pytestmark = pytest.mark.gpu


def _vae(arch="trans1x-128", **params):
    from transvae_amd import synth
    from transvae_amd.trans_models import TransVAE
    cd, od, w = synth.load_vocab("zinc")
    vae = TransVAE(params={"CHAR_DICT": cd, "ORG_DICT": od, "CHAR_WEIGHTS": w, **params}, name="s", **synth.ARCHS[arch])
    vae.model.load_state_dict(synth.synth_state_dict(vae.model.state_dict(), 0))
    return vae


def _z(n, seed=2):
    return torch.randn(n, 128, generator=torch.Generator().manual_seed(seed))


def test_fp8_greedy_decode_follows_its_definition():
    """Store, attend and score together, step by step, against the decoder written out in 64 bits over the reference cache.  A key
    within 1e-6 of the middle of two codes may round the other way there (a step of 2^-4 of one of dk values): scores are
    compared to 0.02, tokens up to the first whose two best logits are closer than twice that."""
    vae = _vae()
    n, L = 5, 125
    z = _z(n)
    ids, logp, ent = (t.cpu() for t in vae.greedy_decode(z, kv_cache="fp8", scores=True))
    model, h = vae.model, vae.params["h"]
    model.eval()
    f = lambda t: t.detach().cpu().double()
    with torch.no_grad():
        lens = model.encoder.predict_mask_length(z.cuda())
        mask = (torch.arange(127, device="cuda")[None] < lens)
        from transvae_amd import ops
        mem = f(model.decoder.expand_memory(z.cuda(), ops.MaskSpec(key_mask=mask.to(torch.uint8).contiguous())))
    mask = mask.cpu()
    d = mem.shape[-1]
    dk = d // h
    lin = lambda x, m: x @ f(m.weight).T + f(m.bias)

    def ln(x, m):
        return f(m.a_2) * (x - x.mean(-1, keepdim=True)) / (x.std(-1, keepdim=True) + m.eps) + f(m.b_2)

    layers = list(model.decoder.layers)
    per = 4
    src, own = [], []
    for lyr in layers:
        c = Cache(n * per, h, dk, 32)
        a = lyr.src_attn.linears
        c.store(lin(mem, a[1]).view(n, 127, h, dk), lin(mem, a[2]).view(n, 127, h, dk), [0] * n, [127] * n, None, per)
        src.append(c)
        own.append(Cache(n * per, h, dk, 32))
    lut, pe = f(model.tgt_embed[0].lut.weight), f(model.tgt_embed[1].pe[0])
    alive = torch.ones(n, dtype=torch.bool)
    tok = torch.full((n,), vae.params["CHAR_DICT"]["<start>"])
    compared = 0
    for t in range(40):
        x = lut[tok] * math.sqrt(d) + pe[t]
        for li, lyr in enumerate(layers):
            s, a = lyr.sublayer, lyr.self_attn.linears
            y = ln(x, s[0].norm)
            own[li].store(lin(y, a[1]).view(n, 1, h, dk), lin(y, a[2]).view(n, 1, h, dk), [t] * n, [1] * n, None, per)
            o, _, _ = own[li].attend(lin(y, a[0]).view(n, 1, h, dk), [t + 1] * n, None, per)
            x = x + lin(o.reshape(n, d), a[3])
            a = lyr.src_attn.linears
            y = ln(x, s[1].norm)
            o, _, _ = src[li].attend(lin(y, a[0]).view(n, 1, h, dk), [127] * n, None, per, mask=mask)
            x = x + lin(o.reshape(n, d), a[3])
            y = ln(x, s[2].norm)
            x = x + lin(torch.relu(lin(y, lyr.feed_forward.w_1)), lyr.feed_forward.w_2)
        lp = torch.log_softmax(lin(ln(x, model.decoder.norm), model.generator.proj), -1)
        two = lp.topk(2).values
        got = ids[:, t]
        agree = lp.argmax(-1) + 1 == got
        assert bool((agree | ~alive | (two[:, 0] - two[:, 1] < 0.04)).all()), t
        live = alive & agree
        compared += int(live.sum())
        assert float((lp[torch.arange(n), got - 1] - logp[:, t].double()).abs()[live].max()) < 0.02
        assert float((-(lp.exp() * lp).sum(-1) - ent[:, t].double()).abs()[live].max()) < 0.02
        alive &= agree
        tok = got
    assert compared > 100


@pytest.mark.parametrize("kv", ["fp32", "fp8"])
def test_scores_are_those_of_the_teacher_forced_model(kv):
    "the decoded tokens fed back through the full decoder (fp32 attention): the same log probabilities, to 1e-4 or to the 8 bits"
    from transvae_amd.data import make_std_mask
    from transvae_amd.loss import token_logprobs
    vae = _vae("trans4x-256")
    z = _z(6)
    src_mask = (torch.arange(127)[None] < torch.tensor([20, 33, 127, 1, 64, 90])[:, None]).unsqueeze(-2).cuda()
    ids, logp, ent = vae.greedy_decode(z, src_mask=src_mask, kv_cache=kv, scores=True)
    assert torch.equal(ids, vae.greedy_decode(z, src_mask=src_mask, kv_cache=kv))
    vae.model.eval()
    tgt = torch.cat([torch.zeros_like(ids[:, :1]), ids], 1)                    # start id, then the tokens: position i predicts ids[:, i]
    with torch.no_grad():
        logits = vae.model.generator(vae.model.decode(z.cuda(), src_mask, tgt, make_std_mask(tgt, 10 ** 6)))
    want, went, _, top = token_logprobs(logits[:, :125], ids - 1, top=1)
    lim = 1e-4 if kv == "fp32" else 0.5
    assert float((want - logp).abs().max()) < lim and float((went - ent).abs().max()) < lim
    if kv == "fp32":
        assert float((top[..., 0] + 1 == ids).float().mean()) > 0.999


def test_conditioned_tokens_are_scored_and_graphs_replay():
    vae = _vae()
    z = _z(7, 3)
    for kv in ("fp32", "fp8"):
        cond = ["C", "c"]
        runs = [vae.greedy_decode(z, condition=cond, kv_cache=kv, scores=True) for _ in range(4)]        # plain launches, capture, replays
        for r in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))
        assert runs[0][0][:, :2].cpu().tolist() == [[vae.params["CHAR_DICT"][c] for c in cond]] * 7
        assert bool((runs[0][1] < 0).all()) and bool(torch.isfinite(runs[0][1]).all()) and bool((runs[0][2] > 0).all())
        other = vae.greedy_decode(_z(7, 4), condition=cond, kv_cache=kv, scores=True)
        assert not torch.equal(other[1], runs[0][1])
        again = vae.greedy_decode(z, condition=cond, kv_cache=kv, scores=True)
        assert all(torch.equal(a, b) for a, b in zip(again, runs[0]))


def test_decode_latents_in_pieces_with_fp8_and_scores():
    """four pieces on four streams: bit for bit the pieces one after the other; near the whole (its sums may be taken in another order:
    the 8-bit attention deals keys to waves by the number of rows)"""
    vae = _vae()
    z = _z(9000, 5)
    ids, logp, ent = vae.decode_latents(z, slab=9000, kv_cache="fp8", scores=True)
    assert ids.dtype == torch.uint8 and ids.shape == (9000, 125) and logp.shape == ent.shape == (9000, 125)
    for a in range(0, 9000, 2250):
        part = vae.greedy_decode(z[a:a + 2250], kv_cache="fp8", scores=True)
        assert torch.equal(part[0].to(torch.uint8), ids[a:a + 2250])
        assert torch.equal(part[1], logp[a:a + 2250]) and torch.equal(part[2], ent[a:a + 2250])
    assert torch.equal(vae.decode_latents(z, slab=9000, kv_cache="fp8"), ids)
    whole = vae.greedy_decode(z, kv_cache="fp8")
    assert float((whole.to(torch.uint8) == ids).float().mean()) > 0.99
    one = vae.decode_latents(z[:50], kv_cache="fp8", scores=True)
    assert one[0].shape == (50, 125) and one[1].shape == (50, 125)


@pytest.mark.parametrize("arch", ["trans1x-128", "rnnattn"])
def test_token_scores_and_their_gradient(arch):
    from transvae_amd import synth
    if arch == "rnnattn":
        from transvae_amd.rnn_models import RNNAttn
        cd, od, w = synth.load_vocab("zinc")
        torch.manual_seed(0)
        vae = RNNAttn(params={"CHAR_DICT": cd, "ORG_DICT": od, "CHAR_WEIGHTS": w}, name="r", d_model=128, d_latent=64)
        dl = 64
    else:
        vae, dl = _vae(arch), 128
    vae.model.eval()
    toks = synth.synth_tokens(9, seed=5)
    data = torch.cat([toks.float(), torch.zeros(9, 1)], 1)
    eps = torch.randn(9, dl, generator=torch.Generator().manual_seed(1)).cuda()
    logp, ent, tl, ti = vae.token_scores(data, top=3, eps=eps)
    y = toks[:, 1:].cuda()
    pad = y == vae.pad_idx
    assert logp.shape == (9, 126) and float(logp[pad].abs().max()) == 0 and bool((logp[~pad] < 0).all())
    w = torch.randn(9, 126, generator=torch.Generator().manual_seed(2)).cuda()
    (logp * w).sum().sub(0.3 * (ent * ~pad).sum()).add((tl * w[..., None]).sum() * 0.1).backward()
    got = {k: p.grad.clone() for k, p in vae.model.named_parameters() if p.grad is not None}
    vae.model.zero_grad(set_to_none=True)
    src, tgt, _, sm, tm = vae._chunk_inputs(data.cuda())
    lp = torch.log_softmax(vae._model_forward(src, tgt, sm, tm, eps)[0], -1)
    pick = lp.gather(-1, (y - 1).clamp(min=0)[..., None])[..., 0].masked_fill(pad, 0.0)
    e = -(lp.exp() * lp).sum(-1)
    (pick * w).sum().sub(0.3 * (e * ~pad).sum()).add((lp.gather(-1, ti) * w[..., None]).sum() * 0.1).backward()
    assert rel_l2(logp.detach().cpu(), pick.detach().cpu().double()) < 1e-6 and rel_l2(ent.detach().cpu(), e.detach().cpu().double()) < 1e-6
    names = [k for k, p in vae.model.named_parameters() if p.grad is not None]
    assert set(names) == set(got) and len(names) > 10
    for k, p in vae.model.named_parameters():
        if p.grad is not None and float(p.grad.abs().max()) > 1e-6:
            assert rel_l2(got[k].cpu(), p.grad.cpu().double()) < 2e-4, k


def test_recurrent_models_score_and_refuse_the_cache():
    from transvae_amd import _lib, synth
    from transvae_amd.rnn_models import RNNAttn
    cd, od, w = synth.load_vocab("zinc")
    torch.manual_seed(0)
    vae = RNNAttn(params={"CHAR_DICT": cd, "ORG_DICT": od, "CHAR_WEIGHTS": w}, name="r", d_model=128, d_latent=64)
    z = torch.randn(5, 64)
    ids, logp, ent = vae.greedy_decode(z, condition=["C"], scores=True)
    assert torch.equal(ids, vae.greedy_decode(z, condition=["C"])) and logp.shape == (5, 125) and bool((logp < 0).all()) and bool((ent > 0).all())
    for call in (vae.greedy_decode, vae.decode_latents):
        with pytest.raises(_lib.TvaeError):
            call(z, kv_cache="fp8")
    with pytest.raises(_lib.TvaeError):
        vae.kv_cache_error(z)
    with pytest.raises(_lib.TvaeError):
        _vae().greedy_decode(_z(3), kv_cache="int4")


def test_cache_error_is_that_of_the_codes():
    "relative error of rounding to e4m3: between a quarter of the half step 2^-4 and the half step, for values well inside the scale's range"
    vae = _vae("trans4x-256")
    e = vae.kv_cache_error(_z(40))
    assert e.shape == (len(vae.model.decoder.layers), 2) and bool((e > 2.0 ** -6).all()) and bool((e < 2.0 ** -4).all())
    assert torch.equal(e, vae.kv_cache_error(_z(40)))


@pytest.mark.parametrize("per_batch", ["0", "1"])
def test_sample_script_writes_scores(tmp_path, monkeypatch, per_batch):
    import pandas as pd
    from scripts import parsers, sample
    monkeypatch.chdir(tmp_path)
    monkeypatch.setenv("TVAE_SAMPLE_PER_BATCH", per_batch)
    vae = _vae()
    vae.current_state.update(model_state_dict=vae.model.state_dict(), optimizer_state_dict=vae.optimizer.state_dict, epoch=1, name="s")
    vae.save(vae.current_state, "x.ckpt", path=str(tmp_path), use_name=False)
    sample.sample(parsers.sample_parser().parse_args(
        ["--model", "transvae", "--model_ckpt", "x.ckpt", "--sample_mode", "rand", "--n_samples", "20", "--n_samples_per_batch", "10",
         "--save_path", "out.csv", "--kv_cache", "fp8", "--scores"]))
    t = pd.read_csv("out.csv", keep_default_na=False)
    assert list(t.columns) == ["mol", "logp"] and len(t) == 20 and bool((t["logp"] < 0).all()) and np.isfinite(t["logp"]).all()
