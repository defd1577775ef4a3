"""Routing and 8-bit products at their edges: calls that the documentation allows and that need care, against the same
64-bit restatements as in test_gpu_routing_int8."""
import pytest
import torch

from moe_quant_amd import ops
from test_gpu_routing_int8 import DT, _check_route, _gen, _say

pytestmark = pytest.mark.gpu


# ---- routing: all experts, or all but one, chosen -------------------------------------------------------------
def _rows_with_a_pair(E, near):
    """A row for every distance that is a multiple of four: well separated logits and one pair of equal (near: neighbouring)
    ones that far apart, once at the top, once in the middle and once at the end of the order."""
    rows = []
    for d in range(4, E, 4):
        for a in {0, (E - d) // 2, E - d - 1}:
            for place in (0, E // 2, E - 2):
                order = torch.randperm(E, generator=_gen(E * d + a)).tolist()
                order.remove(a), order.remove(a + d)
                order[place:place] = [a + d, a]
                row = torch.empty(E)
                row[order] = 3.0 - 0.25 * torch.arange(E).float()
                row[a + d] = row[a]
                if near:
                    row[a + d] = torch.nextafter(row[a], torch.tensor(9.0))
                rows.append(row)
    return torch.stack(rows)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("k", [5, 8, 16])
def test_one_tied_pair_and_no_candidate_left(dev, score, k):
    for E in (k, k + 1, k + 2, 2 * k + 1):
        for near in (False, True):
            _say("pair", E, k, score, near)
            l = _rows_with_a_pair(E, near)
            zero, bias = torch.zeros(E), 0.1 * torch.randn(E, generator=_gen(E))
            for kw in (dict(), dict(bias=zero.to(dev)), dict(bias=bias.to(dev))):
                w, i = _check_route(dev, l, k, score=score, **kw)
                assert all(len(set(r)) == k for r in i.tolist())
            for dt in (DT["bf16"], DT["f16"]):
                _check_route(dev, l.to(dt), k, score=score)
                _check_route(dev, l.to(dt), k, score=score, bias=zero.to(dev))
                _check_route(dev, l.to(dt), k, score=score, bias=bias.to(dev))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_one_tied_pair_in_the_groups_that_stay(dev, score):
    for G, per, tg, k in ((4, 8, 1, 8), (4, 9, 1, 8), (8, 8, 2, 16), (32, 8, 1, 8), (4, 6, 1, 5), (64, 16, 1, 16), (20, 17, 1, 16),
                          (8, 32, 1, 16)):
        _say("groups", G, per, tg, k, score)
        pair = _rows_with_a_pair(tg * per, False) + 4.0
        rows = -2.0 + 0.5 * torch.randn(pair.shape[0], G, per, generator=_gen(G * per)).clamp(-2, 2)
        for t in range(rows.shape[0]):
            at = torch.randperm(G, generator=_gen(t))[:tg]
            rows[t, at] = pair[t].view(tg, per)
        l = rows.reshape(-1, G * per)
        bias = torch.zeros(G * per, device=dev)
        for kw in (dict(), dict(bias=bias)):
            w, i = _check_route(dev, l, k, score=score, n_group=G, topk_group=tg, group_top=2, **kw)
            assert all(len(set(r)) == k for r in i.tolist())
        _check_route(dev, l.bfloat16(), k, score=score, n_group=G, topk_group=tg, group_top=1, bias=bias)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,k", [(8, 8), (9, 8), (6, 5), (16, 16), (17, 16), (4, 4), (65, 16)])
def test_all_chosen_from_a_coarse_grid(dev, score, E, k):
    """Logits on a grid of eighths: pairs tie here and there, anywhere in the row."""
    l = (torch.randn(3000, E, generator=_gen(E * k)) * 16).round() / 8
    for kw in (dict(), dict(bias=torch.zeros(E, device=dev)), dict(renormalize=False, scale=2.5)):
        w, i = _check_route(dev, l, k, score=score, **kw)
        assert all(len(set(r)) == k for r in i.tolist())
