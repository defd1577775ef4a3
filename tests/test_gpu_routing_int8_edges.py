"""Routing and 8-bit products at their edges: calls that the documentation allows and that need care, against the same
64-bit restatements as in test_gpu_routing_int8."""
import pytest
import torch

from moe_quant_amd import moe_layer, ops
from test_gpu_routing_int8 import DT, U, _check_route, _experts, _gen, _half, _product64, _say

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


# ---- the experts' weighted sum ----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("S,C,T,k", [(1, 1, 1, 1), (16, 7168, 2, 8), (100, 33, 25, 4), (64, 2048, 64, 1), (30, 1000, 10, 3),
                                     (50, 2056, 7, 9), (5, 64, 0, 2), (0, 64, 3, 2)])
def test_combine_rounds_fp32_outputs_once(dev, dtype, S, C, T, k):
    dt, g = DT[dtype], _gen(S * C + T)
    Y = torch.randn(S, C, generator=g)
    slots = torch.randint(0, max(S, 1), (T, k), generator=g, dtype=torch.int32)
    if T > 2:
        slots[1, 0], slots[2], slots[0, -1] = -1, -1, S
    w = torch.rand(T, k, generator=g) - 0.3
    live = ((slots >= 0) & (slots < S)).double()[..., None]
    terms = (Y.double()[slots.clamp(0, S - 1).long()] if S else torch.zeros(T, k, C, dtype=torch.float64)) * w.double()[..., None] * live
    want, mag = terms.sum(1), terms.abs().sum(1)
    tol = k * U * mag * (1 + _half(dt)) + _half(dt) * want.abs() + (2.0**-25 if dt == torch.float16 else 2.0**-140)
    for view in (Y.to(dev), torch.cat([Y, Y], 1).to(dev)[:, :C], torch.cat([Y[:, :1], Y], 1).to(dev)[:, 1:]):
        out = ops.combine_experts(view, slots.to(dev), w.to(dev), dt)
        assert out.dtype == dt and out.shape == (T, C) and ((out.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T,E,k,C,I", [(4, 16, 8, 256, 64), (64, 24, 8, 512, 128), (700, 8, 4, 264, 96), (5000, 6, 2, 128, 64)])
def test_experts_outputs_are_rounded_after_their_sum(dev, dtype, T, E, k, C, I):
    """The last two stages against 64 bits on what the two before gave.  The outputs of a token's experts are of both signs, so
    their sum is smaller than they are: a rounding of each one to the tokens' type would be off by half a step of the terms,
    not of the sum.  Roundings: five in 32 bits for a product, one for each term and its addition, one for the result."""
    dt, g = DT[dtype], _gen(T + E)
    x = torch.randn(T, C, generator=g).to(dt).to(dev)
    ex = _experts(g, E, C, I, dev)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).to(dev)
    weights = (torch.rand(T, k, generator=g) + 0.1).to(dev)
    y = moe_layer.experts_forward_int8(x, ids, weights, ex)
    rows, offsets, slots = ops.sort_by_expert(ids, E)
    h = ops.matmul_int8_grouped(*ops.quantize_tokens(x), ex.gate_up, ex.gate_up_scale, offsets, rows, dt, True)
    q, s = (t.cpu() for t in ops.quantize_tokens(h))
    each = torch.empty(T * k, C, dtype=torch.float64)
    for e in range(E):
        lo, hi = offsets[e].item(), offsets[e + 1].item()
        each[lo:hi] = _product64(q[lo:hi], s[lo:hi], ex.down[e].cpu(), ex.down_scale[e].cpu())[0]
    terms = each[slots.long().cpu()] * weights.cpu().double()[..., None]
    want, mag = terms.sum(1), terms.abs().sum(1)
    tol = (6 + k) * U * mag * 1.01 + _half(dt) * want.abs() + (2.0**-25 if dt == torch.float16 else 2.0**-140)
    assert y.dtype == dt and ((y.cpu().double() - want).abs() <= tol).all()


# ---- ids that the layer driver's own sort does not take ------------------------------------------------------------
@pytest.mark.parametrize("shape,E", [((5, 0), 4), ((0, 3), 4), ((0, 3), 0), ((0, 0), 2), ((2, 3, 1), 4), ((7, 2), 1025)])
def test_route_tokens_of_any_shape_matches_the_host(dev, shape, E):
    ids = torch.zeros(shape, dtype=torch.int64)
    if ids.dim() == 3:
        ids[1] = 3
    want_rows, want = moe_layer.route_tokens(ids, E)
    rows, offsets = moe_layer.route_tokens(ids.to(dev), E)
    assert rows.dtype == torch.int64 and torch.equal(rows.cpu(), want_rows) and offsets == want


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_experts_of_many_tokens_go_in_parts(dev, dtype, monkeypatch):
    """With the bound on the experts' fp32 outputs brought down: the same bits, and no more scratch memory than it allows."""
    dt, g = DT[dtype], _gen(40)
    T, E, k, C, I = 5001, 12, 4, 512, 64
    x = torch.randn(T, C, generator=g).to(dt).to(dev)
    ex = _experts(g, E, C, I, dev)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).to(dev)
    ids[7, 1], ids[4000] = -1, E
    weights = torch.rand(T, k, generator=g).to(dev)

    def peak(limit):
        monkeypatch.setattr(moe_layer, "_OUTPUTS_AT_ONCE", limit)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        y = moe_layer.experts_forward_int8(x, ids, weights, ex)
        torch.cuda.synchronize()
        return y, torch.cuda.max_memory_allocated() - before

    whole, much = peak(1 << 32)
    assert much >= 4 * T * k * C
    for limit in (T * k * C - 1, 1 << 21, 1 << 20, k * C, 1):
        if limit < 1 << 18:  # a token at a time: a few of them
            monkeypatch.setattr(moe_layer, "_OUTPUTS_AT_ONCE", limit)
            assert torch.equal(moe_layer.experts_forward_int8(x[:9], ids[:9], weights[:9], ex), whole[:9])
            continue
        y, little = peak(limit)
        assert torch.equal(y, whole) and y.is_contiguous()
        # the result, a part of it, and the part's outputs; its codes, activations and places are a quarter of those
        assert little <= 2 * y.nbytes + 1.25 * 4 * limit + (1 << 20)
    strided = torch.randn(C, T, generator=g).to(dt).to(dev).t()
    monkeypatch.setattr(moe_layer, "_OUTPUTS_AT_ONCE", 1 << 20)
    y = moe_layer.experts_forward_int8(strided, ids, weights, ex)
    monkeypatch.setattr(moe_layer, "_OUTPUTS_AT_ONCE", 1 << 32)
    assert torch.equal(y, moe_layer.experts_forward_int8(strided, ids, weights, ex))
