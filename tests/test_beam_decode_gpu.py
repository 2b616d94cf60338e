"""T2S.set_decoding: the decode operators together, as the eval loop runs them - prefill into the 8-bit cache, one row a step, selection, reordering,
then the three passes' scores along the best beam - against the same loop in 64 bits on the CPU over the same cached codes."""
import math

import pytest
import torch

from decode_ref import read_cache, select_ref
from golden_util import Fixture

DEV = "cuda:0"


def _model(case, dtype, beams, fmt, eos=None):
    from vitxt_gqa_amd import registry
    from vitxt_gqa_amd.testing import build_model_for_fixture, to_device
    fx = Fixture(case)
    model = build_model_for_fixture(fx, dtype).to(DEV).eval()
    if eos is not None:
        class P:
            BOS_IDX, EOS_IDX = 1, eos
        model.answer_processor = P()
    s = to_device(fx.batch(), DEV)
    s.grounding_noise, s.grounding_masks = (fx["E1"], fx["E2"]), fx.masks()
    return model.set_decoding(beams, fmt), s


class Loop64:
    """The decoder rows of the "pos" pass in 64 bits: model weights, cached keys / values, pointer keys as the model holds them."""

    def __init__(self, model, fwd):
        self.sd = {k: v.detach().cpu().double() for k, v in model.state_dict().items()}
        self.kv = [read_cache(c) for c in fwd["pos_caches"]]
        self.k_ptr, self.ocr = fwd["pos_k_ptr"].cpu().double(), fwd["ocr_mmt_in"].cpu().double()
        self.mask = fwd["pos_ocr_mask"].cpu().double()
        self.V = self.sd["classifier.module.weight"].shape[0]

    def ln(self, x, name):
        return torch.nn.functional.layer_norm(x, (768,), self.sd[name + ".weight"], self.sd[name + ".bias"], 1e-12)

    def lin(self, x, name):
        return x @ self.sd[name + ".weight"].t() + self.sd[name + ".bias"]

    def row(self, b, token, t, past):
        """Logits of step t of one beam that reads ``token``; past[layer] = (keys, values) [t, 12, 64], extended in place."""
        p = "mmt.prev_pred_embeddings."
        is_ocr = token >= self.V
        raw = self.ln(self.ocr[b, token - self.V], p + "ocr_layer_norm") if is_ocr else self.ln(self.sd["classifier.module.weight"][token], p + "ans_layer_norm")
        x = raw + self.ln(self.sd[p + "position_embeddings.weight"][t] + self.sd[p + "token_type_embeddings.weight"][int(is_ocr)], p + "emb_layer_norm")
        for l in range(len(self.kv)):
            n = "mmt.encoder.layer.%d." % l
            q, k, v = (self.lin(x, n + "attention.self." + w).view(12, 64) for w in ("query", "key", "value"))
            past[l] = tuple(torch.cat([a, c[None]]) for a, c in zip(past[l], (k, v)))
            att = []
            for h in range(12):
                kk, vv = (torch.cat([self.kv[l][b][h][i], past[l][i][:, h]]) for i in range(2))
                att.append(torch.softmax(kk @ q[h] * 0.125, 0) @ vv)
            x = self.ln(x + self.lin(torch.cat(att), n + "attention.output.dense"), n + "attention.output.LayerNorm")
            u = self.lin(x, n + "intermediate.dense")
            x = self.ln(x + self.lin(0.5 * u * (1 + torch.erf(u / math.sqrt(2))), n + "output.dense"), n + "output.LayerNorm")
        ptr = self.k_ptr[b] @ self.lin(x, "ocr_ptr_net.query") / math.sqrt(768) + self.mask[b]
        return torch.cat([self.lin(x, "classifier.module"), ptr])

    def search(self, b, K, D, bos, eos):
        """-> tokens [K, D], scores [K], the smallest gap between a chosen candidate and the next one on the way, the chosen beams' logits."""
        empty = lambda: [(torch.zeros(0, 12, 64, dtype=torch.float64),) * 2 for _ in self.kv]
        toks, total, ended, past, rows, gap = [[] for _ in range(K)], torch.full((K,), -math.inf, dtype=torch.float64), [False] * K, [empty() for _ in range(K)], [[] for _ in range(K)], math.inf
        total[0] = 0.0
        for t in range(D):
            past = [list(p) for p in past]
            logits = torch.stack([self.row(b, toks[n][-1] if t else bos, t, past[n]) for n in range(K)])
            best, par, tok = select_ref(logits[None], total[None], K, torch.tensor([ended]) if eos is not None else None, eos or 0)
            step = (best[0, :-1] - best[0, 1:])
            gap = min([gap] + step[torch.isfinite(step)].tolist())               # (one ended beam: nothing else has a score)
            par, tok = par[0].tolist(), tok[0].tolist()
            total, toks, past, rows = best[0, :K], [toks[p] + [w] for p, w in zip(par, tok)], [past[p] for p in par], [rows[p] + [logits[p]] for p in par]
            ended = [ended[p] or (eos is not None and w == eos) for p, w in zip(par, tok)]
        return torch.tensor(toks), total, gap, rows


@pytest.mark.gpu
@pytest.mark.parametrize("case,beams,fmt,eos", [("tiny_b2_f6_p8", 1, "int8", None), ("tiny_b2_f6_p8", 4, "e4m3", None), ("ptr_b3_f8_p10", 3, "int8", None), ("ptr_b3_f8_p10", 5, "int8", 7), ("tiny_b2_f6_p8", 16, "e4m3", 7),
                                                ("ptr_b3_f8_p10", 1, "int8", 7)])
def test_beam_decode_equals_the_64_bit_loop(case, beams, fmt, eos):
    model, s = _model(case, torch.float32, beams, fmt, eos)
    if eos is not None:                                       # make the end likely enough to be chosen on the way
        with torch.no_grad():
            model.classifier.module.bias[eos] += 3.0
    model.keep_intermediates = True
    with torch.no_grad():
        out = model(s)
    f = model._last_fwd
    loop, D = Loop64(model, f), s.train_prev_inds.size(1)
    B = s.text.size(0)
    assert out["beam_tokens"].shape == (B, beams, D) and out["beam_scores"].shape == (B, beams)
    for b in range(B):
        toks, total, gap, rows = loop.search(b, beams, D, 1, eos)
        # fp32 rows of 3 layers against 64 bits: a logit is off by some 1e-5 (the model's fp32 bound is 1e-3), a score by D of them
        got = out["beam_scores"][b].cpu().double()
        assert (got - total).abs().max() < D * 1e-3, (got, total)
        print("%s sample %d: smallest gap %.2e, score error %.2e" % (case, b, gap, (got - total).abs().max()))
        if gap > 2 * D * 1e-5:
            assert torch.equal(out["beam_tokens"][b].cpu(), toks)
            # the scores of the pass along the best beam
            want = torch.stack(rows[0])
            assert (out["pos_scores"][b].cpu().double() - want).abs().max() < 1e-3
    best = out["beam_tokens"][:, 0]
    assert torch.equal(f["prev_inds"][:, 1:], best[:, :-1]) and bool((f["prev_inds"][:, 0] == 1).all())
    if eos is not None:
        after = (out["beam_tokens"] == eos).cumsum(-1) > 0
        assert bool(after.any()) and bool((out["beam_tokens"][after] == eos).all())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_one_beam_is_the_greedy_loop(fmt):
    """One beam takes the argmax of every step: what the best beam's own scores say, and - the codes being near enough on this fixture, whose winners lead by
    more than the codes move them - what the loop over the operand-type cache takes."""
    model, s = _model("ptr_b3_f8_p10", torch.float32, 1, fmt)
    with torch.no_grad():
        out = model(s)
        tokens = out["beam_tokens"][:, 0].cpu()
        top = out["pos_scores"].cpu().topk(2, dim=-1)
        lead = top.values[..., 0] - top.values[..., 1]
        clear = lead > 1e-3
        assert torch.equal(top.indices[..., 0][clear], tokens[clear]) and clear.float().mean() > 0.9
        ref = model.set_decoding(1, None)(s)
        assert "beam_tokens" not in ref
    prev = model._last_fwd["prev_inds"].cpu()
    moved = max(float((out[k] - ref[k]).abs().max()) for k in ("pos_scores",))
    print("%s: scores of the 8-bit prefix differ by %.3g where both loops took the same words" % (fmt, moved))
    D = tokens.shape[1]
    for b in range(tokens.shape[0]):
        for t in range(D - 1):
            if int(tokens[b, t]) != int(prev[b, t + 1]):
                top = ref["pos_scores"][b, t].topk(2).values
                assert float(top[0] - top[1]) < 0.2, "the loops part at a clear winner"
                break


@pytest.mark.gpu
def test_beam_decode_bf16_and_defaults():
    model, s = _model("cfg1_b2_f20_p30", torch.bfloat16, 5, None)
    assert model.decode_cache == "int8"
    with torch.no_grad():
        out = model(s)
        again = model(s)
        one = model.set_decoding(1, "int8")(s)
    for k in ("beam_tokens", "beam_scores", "pos_scores", "ref_scores", "neg_scores"):
        assert torch.equal(out[k], again[k]), k                                   # nothing depends on an order of arrival
    assert bool((out["beam_scores"][:, :-1] >= out["beam_scores"][:, 1:]).all()) and bool(torch.isfinite(out["beam_scores"]).all())
    seqs = [tuple(x) for x in out["beam_tokens"][0].tolist()]
    assert len(set(seqs)) == len(seqs)
    # five beams find an answer at least as good as the greedy one (up to the rounding of bf16 rows)
    assert bool((out["beam_scores"][:, 0] >= one["beam_scores"][:, 0] - 0.1).all())


def test_set_decoding_refuses():
    from vitxt_gqa_amd.testing import make_model
    m = make_model(6, 8, 64, text_vocab=100, dtype=torch.float32)
    assert (m.decode_beams, m.decode_cache) == (1, None)
    for kw in (dict(beams=0), dict(beams=17), dict(beams=2, cache="fp4"), dict(cache="operand")):
        with pytest.raises(ValueError):
            m.set_decoding(**kw)
    assert m.set_decoding(beams=3).decode_cache == "int8" and m.set_decoding().decode_cache is None
