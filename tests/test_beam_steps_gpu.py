"""Every step of T2S's beam search, as the eval loop ran it, against 64 bits: the logits of each beam along its own words, what was selected from them, where the
beams' words went, and the scores along the answer.  Each step is checked from what the step before it chose, so nothing depends on how close two candidates
came on the way: all steps of all samples are compared.

Tolerances, u = 2^-24: logits 1e-3, the bound of the model's fp32 forward; a selection's score 160 u + u |score| from the logits and scores it was given
(tests/test_decode_gpu.py has the derivation), so candidates further apart than twice that have an order."""
import math

import pytest
import torch

from decode_ref import select_ref
from test_beam_decode_gpu import Loop64, _model

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _follow(monkeypatch, case, beams, fmt, eos):
    """The model's output, its intermediate results and what each step's selection was given and gave."""
    from vitxt_gqa_amd import decode
    model, s = _model(case, torch.float32, beams, fmt, eos)
    if eos is not None:                                       # (likely enough to be chosen on the way)
        with torch.no_grad():
            model.classifier.module.bias[eos] += 3.0
    model.keep_intermediates = True
    steps, select = [], decode.beam_select

    def recorded(logits, scores, n_select, finished=None, pad=0):
        res = select(logits, scores, n_select, finished, pad)
        steps.append([None if t is None else t.detach().cpu().clone() for t in (logits, scores, finished, *res)])
        return res

    monkeypatch.setattr(decode, "beam_select", recorded)
    with torch.no_grad():
        out = model(s)
    return model, s, out, steps


@pytest.mark.parametrize("case,beams,fmt,eos", [("tiny_b2_f6_p8", 1, "int8", None), ("tiny_b2_f6_p8", 4, "e4m3", None), ("ptr_b3_f8_p10", 3, "int8", None), ("ptr_b3_f8_p10", 5, "int8", 7),
                                                ("tiny_b2_f6_p8", 16, "e4m3", 7), ("ptr_b3_f8_p10", 1, "e4m3", 7)])
def test_every_step_of_the_search(monkeypatch, case, beams, fmt, eos):
    from vitxt_gqa_amd import metrics
    model, s, out, steps = _follow(monkeypatch, case, beams, fmt, eos)
    B, D = s.text.size(0), s.train_prev_inds.size(1)
    assert len(steps) == D
    loop = Loop64(model, model._last_fwd)
    words = [[[] for _ in range(beams)] for _ in range(B)]                       # what each beam holds before the step
    past = [[[(torch.zeros(0, 12, 64, dtype=torch.float64),) * 2 for _ in loop.kv] for _ in range(beams)] for _ in range(B)]
    rows = [[[] for _ in range(beams)] for _ in range(B)]
    compared = 0
    for t, (logits, before, ended, after, parents, tokens) in enumerate(steps):
        assert torch.equal(before, steps[t - 1][3] if t else torch.tensor([[0.0] + [-math.inf] * (beams - 1)] * B))
        if eos is None:
            assert ended is None
        else:
            assert ended.tolist() == [[eos in w for w in words[b]] for b in range(B)]
        for b in range(B):
            for n in range(beams):
                if t and before[b, n] == -math.inf:                               # (one ended beam offers a single word: a beam that is none)
                    rows[b][n] = rows[b][n] + [None]
                    past[b][n] = None
                    continue
                kv = [tuple(x) for x in past[b][n]]
                want = loop.row(b, words[b][n][-1] if t else 1, t, kv)
                past[b][n] = kv
                assert (logits[b, n].double() - want).abs().max() < 1e-3, (t, b, n)
                rows[b][n] = rows[b][n] + [want]
                compared += 1
        # the selection from what it was given
        best, rp, rt = select_ref(logits, before, beams, ended, eos or 0)
        ref = best[:, :beams]
        some = ref > -math.inf
        tol = 160 * U + U * ref.abs()
        assert torch.equal(after > -math.inf, some) and bool(((after.double() - ref).abs() <= tol)[some].all())
        V = logits.shape[2]
        full = select_ref(logits, before, beams * V, ended, eos or 0)
        total = torch.empty(B, beams * V, dtype=torch.float64).scatter_(1, full[1] * V + full[2], full[0])
        for b in range(B):
            picked = parents[b] * V + tokens[b]
            assert len(set(picked.tolist())) == beams
            assert bool(((total[b, picked] - ref[b]).abs() <= 2 * tol[b])[some[b]].all())          # the K best, whatever the order of what is that close
            words[b] = [words[b][p] + [w] for p, w in zip(parents[b].tolist(), tokens[b].tolist())]
            past[b] = [past[b][p] for p in parents[b].tolist()]
            rows[b] = [rows[b][p] for p in parents[b].tolist()]
    assert compared >= B * D
    assert out["beam_tokens"].tolist() == words and torch.equal(out["beam_scores"].cpu(), steps[-1][3])
    for b in range(B):                                                            # the "pos" pass along the answer
        assert (out["pos_scores"][b].cpu().double() - torch.stack(rows[b][0])).abs().max() < 1e-3
    assert out["pos_scores"].shape == (B, D, logits.shape[2])
    assert metrics.answer_inds(out).tolist() == [w[0] for w in words]             # what the answer metrics decode
