"""beam_select, mostly past what one workgroup holds: what a row scores depends on its values alone, not on where it lies in memory, so that beams with equal rows and
equal scores tie exactly and go in the order of n V + v.  No tolerance: the order of equal beams is the order of their logits, an integer matter."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _laid_out(rows, at, gap):
    """``rows`` [B, N, V] on the GPU as a view whose first row starts ``at`` elements behind a 16-byte boundary and whose rows are V + gap apart."""
    B, N, V = rows.shape
    buf = torch.full((B * N * (V + gap) + at + 16,), 1e4, dtype=rows.dtype, device="cuda")       # (what is around the rows would win if it were read)
    view = buf.as_strided((B, N, V), (N * (V + gap), V + gap, 1), at)
    view.copy_(rows)
    return view


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("B,N,V,K", [(24, 4, 9001, 16), (24, 8, 15001, 5), (12, 8, 30523, 16), (300, 8, 9003, 8), (2, 32, 16386, 32), (16, 3, 140001, 32), (24, 4, 501, 9), (24, 8, 4001, 16)])
def test_equal_beams_tie_exactly(dtype, B, N, V, K):
    from vitxt_gqa_amd import decode
    g = torch.Generator(device="cuda").manual_seed(V + N)
    row = (torch.randn(B, V, generator=g, device="cuda") * 2).to(DT[dtype])
    logits = row[:, None].expand(B, N, V).contiguous()
    scores = torch.randn(B, 1, generator=g, device="cuda").expand(B, N).contiguous()
    # the best K of N equal rows: by the logit, then the beam, then the word
    best, at = torch.sort(row.float(), dim=1, descending=True, stable=True)
    cand, place = best[:, :K].repeat_interleave(N, 1), (at[:, None, :K] + V * torch.arange(N, device="cuda")[:, None]).transpose(1, 2).reshape(B, -1)
    by_place = torch.argsort(place, dim=1)
    order = by_place.gather(1, torch.sort(cand.gather(1, by_place), dim=1, descending=True, stable=True).indices)[:, :K]
    want = place.gather(1, order)
    for view in (logits, row[:, None].expand(B, N, V), _laid_out(logits, 1, 2), _laid_out(logits, 3, 0)):
        got, parents, tokens = decode.beam_select(view, scores, K)
        assert torch.equal(parents * V + tokens, want), (parents * V + tokens != want).nonzero()[:4]
        assert bool((got[:, 1:] <= got[:, :-1]).all())


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("B,N,V,K", [(6, 5, 15001, 5), (3, 8, 30522, 16), (300, 8, 8189, 8), (1, 2, 140001, 32), (4, 4, 9000, 9)])
def test_scores_do_not_depend_on_the_rows_place(dtype, B, N, V, K):
    from vitxt_gqa_amd import decode
    g = torch.Generator(device="cuda").manual_seed(V)
    x = (torch.randn(B, N, V, generator=g, device="cuda") * 2).to(DT[dtype])
    scores = -torch.rand(B, N, generator=g, device="cuda") * 4
    fin = torch.rand(B, N, generator=g, device="cuda") < 0.2
    want = decode.beam_select(x, scores, K, fin, V // 2)
    for at in range(16 // x.element_size()):
        for gap in (0, 1, 5) if B < 100 else (1,):
            got = decode.beam_select(_laid_out(x, at, gap), scores, K, fin, V // 2)
            for a, b in zip(got, want):
                assert torch.equal(a, b), (at, gap)
