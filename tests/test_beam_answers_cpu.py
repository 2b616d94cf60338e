"""The answer metrics (vitxt_gqa_amd/metrics.py) over outputs of a beam search (T2S.set_decoding): they score the best beam's words.  Row t of the output's
``pos_scores`` holds the scores of what follows the beam's first t words; its largest need not be the word that the beam took there."""
import pytest
import torch

from vitxt_gqa_amd import SampleList, registry
from vitxt_gqa_amd import metrics as M

WORDS = ["<pad>", "<s>", "</s>", "red", "blue", "car", "stop"]
V, EOS = len(WORDS), 2
TOKENS = [["exit", "main", "st"], ["joe", "diner", "go"], ["x", "y", "z"]]
GTS = [["blue car"] * 10, ["diner stop"] * 10, ["z"] * 10]
# the best beam's words, and the words that are the largest of its rows: another first word; an end that the beam does not take; the same
BEAM = [[4, 5, EOS, EOS], [V + 1, 6, EOS, EOS], [V + 2, EOS, EOS, EOS]]
LARGEST = [[3, 5, EOS, 6], [EOS, 6, EOS, EOS], [V + 2, EOS, EOS, EOS]]


class _Processor:
    class answer_vocab:
        idx2word = staticmethod(lambda i: WORDS[i])
    EOS_IDX, BOS_IDX = EOS, 1

    def get_true_vocab_size(self):
        return V


def _output(beams=True):
    scores = torch.zeros(3, 4, V + 3).scatter_(2, torch.tensor(BEAM).unsqueeze(-1), 4.0).scatter_(2, torch.tensor(LARGEST).unsqueeze(-1), 5.0)
    out = {"pos_scores": scores}
    if beams:
        second = torch.tensor(LARGEST)                                            # (another beam: not the answer)
        out.update(beam_tokens=torch.stack([torch.tensor(BEAM), second], dim=1), beam_scores=torch.tensor([[-1.0, -2.0]] * 3))
    return out


@pytest.mark.parametrize("name", ["textvqa_accuracy", "stvqa_anls"])
def test_the_best_beam_is_the_answer_that_is_scored(name):
    cls = {"textvqa_accuracy": M.TextVQAAccuracy, "stvqa_anls": M.STVQAANLS}[name]
    plain = SampleList({"context_tokens": TOKENS, "gt_answers": GTS})
    assert float(cls(WORDS, EOS).calculate(plain, _output())) == 1.0
    registry.register("beam_answers_answer_processor", _Processor())
    batch = SampleList({"targets": torch.zeros(3, 4, V + 3), "dataset_type": "val", "dataset_name": "beam_answers",
                        "context_tokens_enc": torch.stack([M.enc_obj2bytes(t) for t in TOKENS]), "gt_answers_enc": torch.stack([M.enc_obj2bytes(g) for g in GTS])})
    assert M.Metrics([name])(batch, _output())["val/beam_answers/" + name].tolist() == [1.0]
    # without beams the largest of every row, as before: "red car", nothing, "z"
    entries = [{"pred_answer": a, "gt_answers": g} for a, g in zip(("red car", "", "z"), GTS)]
    want = cls(WORDS, EOS).evaluator.eval_pred_list([], entries)[1]
    assert want < 1.0
    assert float(cls(WORDS, EOS).calculate(plain, _output(beams=False))) == pytest.approx(want)
    assert M.Metrics([name])(batch, _output(beams=False))["val/beam_answers/" + name].item() == pytest.approx(want)
