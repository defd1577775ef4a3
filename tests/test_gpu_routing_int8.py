"""Routing to experts and products on 8-bit integers against plain 64-bit restatements on the CPU.

Whole numbers (ids, rows, offsets, slots, codes) have to be equal.  Tolerances count roundings: u = 2^-24 per 32-bit
operation, half a step (finfo.eps / 2, relative) for the result's own rounding."""
import math

import pytest
import torch

from moe_quant_amd import moe_layer, ops, quant_utils
from moe_quant_amd.gptq import GPTQ

pytestmark = pytest.mark.gpu
U = 2.0**-24
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _half(dt):
    return torch.finfo(dt).eps / 2


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _say(*m):
    print(*m, flush=True)


# ---- routing -------------------------------------------------------------------------------------------
def _route64(logits, k, score="softmax", bias=None, n_group=1, topk_group=None, group_top=2, renormalize=True, scale=1.0):
    """Row by row, by sorting (-value, index) pairs."""
    T, E = logits.shape
    l = logits.double()
    l = torch.where(l.isnan(), torch.full_like(l, -math.inf), l)
    ids, ws = torch.empty(T, k, dtype=torch.int64), torch.empty(T, k, dtype=torch.float64)
    for t in range(T):
        row = l[t]
        m = row.max()
        if score == "sigmoid":
            s = 1 / (1 + torch.exp(-row))
        elif m == -math.inf:
            s = torch.zeros_like(row)
        else:
            s = torch.where(row == m, torch.ones_like(row), torch.exp(row - m))
            s = s / s.sum()
        c = s
        if bias is not None:
            b = bias.double()
            c = torch.where(b.isnan(), torch.full_like(s, -math.inf), s + b)
        rank = (row if bias is None else c).tolist()
        allowed = list(range(E))
        if n_group > 1:
            per = E // n_group
            def total(g):
                top = sorted(c[g * per:(g + 1) * per].tolist(), reverse=True)[:group_top]
                v = sum(top)
                return top[0] if v != v else v
            kept = sorted(range(n_group), key=lambda g: (-total(g), g))[:topk_group or n_group]
            allowed = [e for e in allowed if e // per in kept]
        chosen = sorted(allowed, key=lambda e: (-rank[e], e))[:k]
        ids[t] = torch.tensor(chosen)
        w = s[chosen]
        if renormalize:
            w = w / (w.sum() + 1e-20)
        ws[t] = w * scale
    return ws, ids


def _check_route(dev, logits, k, **kw):
    want_w, want_i = _route64(logits, k, **{n: (v.cpu() if isinstance(v, torch.Tensor) else v) for n, v in kw.items()})
    w, i = ops.route_experts(logits.to(dev), k, **kw)
    assert w.dtype == torch.float32 and i.dtype == torch.int64 and w.shape == i.shape == (logits.shape[0], k)
    assert torch.equal(i.cpu(), want_i)
    # exp's argument is rounded once and scaled once: with |l - max| <= 32, 2 * 32 * 1.45 u, and a dozen roundings beside
    # it (sums of up to E positive terms run as trees); results below 2^-126 may be flushed
    err = (w.cpu().double() - want_w).abs()
    assert (err <= 112 * U * want_w.abs() + 2.0**-126).all(), (err / (want_w.abs() + 1e-300)).max()
    return w, i


ROUTE_SHAPES = [(1, 256, 8), (1, 1, 1), (3, 2, 2), (7, 60, 6), (5, 64, 64), (129, 72, 6), (33, 255, 9), (65, 256, 8), (17, 257, 3),
                (9, 1024, 16), (2, 1000, 40), (6, 16, 16), (130, 128, 1)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_plain(dev, dtype, score):
    for T, E, k in ROUTE_SHAPES:
        _say("route", T, E, k, dtype, score)
        logits = (2 * torch.randn(T, E, generator=_gen(T + E))).to(DT[dtype])
        bias = 0.1 * torch.randn(E, generator=_gen(E))
        _check_route(dev, logits, k, score=score)
        _check_route(dev, logits, k, score=score, renormalize=False, scale=2.5)
        _check_route(dev, logits, k, score=score, bias=bias.to(dev), scale=0.5)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("group_top", [1, 2])
def test_route_groups(dev, dtype, score, group_top):
    for T, E, k, G, tg in [(65, 256, 8, 8, 4), (1, 256, 8, 8, 4), (33, 60, 6, 4, 2), (9, 64, 2, 32, 1), (17, 1024, 8, 64, 8),
                           (5, 24, 6, 4, 1), (7, 120, 5, 8, 8), (31, 160, 6, 8, 3), (3, 8, 2, 2, 1)]:
        _say("groups", T, E, k, G, tg, dtype, score, group_top)
        logits = (2 * torch.randn(T, E, generator=_gen(T * E))).to(DT[dtype])
        bias = (0.1 * torch.randn(E, generator=_gen(E))).to(dev)
        kw = dict(score=score, n_group=G, topk_group=tg, group_top=group_top)
        _check_route(dev, logits, k, **kw)
        _check_route(dev, logits, k, bias=bias, scale=2.5, **kw)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_groups_whose_best_cancel(dev, score):
    """Biases of both signs, so that a group's two best almost cancel: their sum is what tells the groups apart."""
    for T, E, k, G, tg in [(40, 64, 4, 8, 3), (40, 60, 3, 4, 2), (17, 256, 8, 8, 4), (9, 1024, 16, 16, 5)]:
        _say("cancel", T, E, k, G, tg, score)
        logits = 2 * torch.randn(T, E, generator=_gen(T + E))
        bias = torch.full((G, E // G), -(2.0**20))
        bias[:, 3] = 2.0**20
        _check_route(dev, logits, k, score=score, bias=bias.reshape(-1).to(dev), n_group=G, topk_group=tg)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_ties_and_near_ties(dev, score):
    """Equal logits everywhere, equal pairs, and neighbours one 32-bit step apart, with and without a bias."""
    E = 256
    rows = [torch.zeros(E), torch.arange(E).float() // 16, torch.arange(E).flip(0).float() // 3 * 0.01]
    near = torch.full((E,), 1.0)
    near[torch.randperm(E, generator=_gen(1))[:40]] = torch.nextafter(torch.tensor(1.0), torch.tensor(2.0)).item()
    rows.append(near)
    walk = [1.5]
    for _ in range(E - 1):
        walk.append(torch.nextafter(torch.tensor(walk[-1]), torch.tensor(9.0)).item())
    rows.append(torch.tensor(walk)[torch.randperm(E, generator=_gen(2))])
    logits = torch.stack(rows)
    _check_route(dev, logits, 8, score=score)
    _check_route(dev, logits, 8, score=score, n_group=8, topk_group=3, group_top=1)
    _check_route(dev, logits.bfloat16(), 8, score=score, n_group=8, topk_group=3, group_top=2)
    _check_route(dev, logits, 8, score=score, bias=torch.zeros(E, device=dev))
    step = (torch.arange(E) % 7).float() * 2.0**-20
    _check_route(dev, logits, 8, score=score, bias=step.to(dev))
    # close values around the border of the choice: differences of 1e-7 relative in the score
    g = _gen(3)
    close = 1.0 + 1e-6 * torch.randn(64, E, generator=g)
    _check_route(dev, close, 8, score=score)
    _check_route(dev, close, 8, score=score, bias=(1e-7 * torch.randn(E, generator=g)).to(dev))
    _check_route(dev, close, 8, score=score, bias=(1e-7 * torch.randn(E, generator=g)).to(dev), n_group=8, topk_group=4)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_masked_and_infinite(dev, dtype, score):
    """Masked experts (-inf and the type's lowest value), rows with nothing left, NaN, +inf."""
    dt, E = DT[dtype], 48
    low = torch.finfo(dt).min
    l = torch.randn(10, E, generator=_gen(4)).to(dt)
    l[0] = -math.inf
    l[1] = low
    l[2, 3:] = -math.inf
    l[3, 5:] = low
    l[4, ::2] = math.nan
    l[5] = math.nan
    l[6, 7] = math.inf
    l[7, [3, 40]] = math.inf
    l[8] = torch.finfo(dt).max
    for kw in (dict(), dict(renormalize=False), dict(n_group=4, topk_group=2), dict(n_group=4, topk_group=2, group_top=1)):
        w, i = _check_route(dev, l, 6, score=score, **kw)
        assert torch.isfinite(w).all()
        assert all(len(set(r)) == 6 and min(r) >= 0 and max(r) < E for r in i.tolist())
    b = torch.zeros(E)
    b[:8], b[9], b[20] = -math.inf, math.nan, math.inf
    for kw in (dict(), dict(n_group=4, topk_group=3)):
        _check_route(dev, l, 6, score=score, bias=b.to(dev), **kw)


def test_route_far_logits(dev):
    """Scores that saturate or vanish in 32 bits: the choice stays by the logits."""
    l = torch.linspace(-200, 200, 96).flip(0).repeat(3, 1)[:, torch.randperm(96, generator=_gen(5))]
    for score in ("softmax", "sigmoid"):
        w, i = ops.route_experts(l.to(dev), 8, score=score)
        assert torch.equal(i.cpu(), _route64(l, 8, score)[1])
    l = l.abs().neg()  # down to e^-200, every value twice
    for score in ("softmax", "sigmoid"):
        w, i = ops.route_experts(l.to(dev), 64, score=score)
        assert torch.equal(i.cpu(), _route64(l, 64, score)[1])


def test_route_strides_and_empty(dev):
    base = torch.randn(37, 100, generator=_gen(6))
    for v in (base[:, 3:75], base[::2, :60], base.t()[:50], base[:1, 1:41], base[:1].expand(4, 100)):
        _check_route(dev, v, 5)
        on_gpu = base.to(dev)
        view = torch.as_strided(on_gpu, v.shape, v.stride(), v.storage_offset())
        w, i = ops.route_experts(view, 5)
        assert torch.equal(i.cpu(), _route64(v, 5)[1])
    w, i = ops.route_experts(torch.zeros(0, 16, device=dev), 4)
    assert w.shape == i.shape == (0, 4)


# ---- sort ------------------------------------------------------------------------------------------------
def _sort64(ids, E):
    flat = ids.reshape(-1)
    key = torch.where((flat < 0) | (flat >= E), torch.full_like(flat, E), flat)
    order = torch.argsort(key, stable=True)
    offsets = torch.zeros(E + 1, dtype=torch.int64)
    offsets[1:] = torch.cumsum(torch.bincount(key, minlength=E + 1)[:E], 0)
    slots = torch.empty(flat.numel(), dtype=torch.int32)
    slots[order] = torch.arange(flat.numel(), dtype=torch.int32)
    slots[key == E] = -1
    return order // max(1, ids.shape[1]), offsets, slots.view(ids.shape)


def _check_sort(dev, ids, E):
    got = ops.sort_by_expert(ids.to(dev), E)
    for g, w in zip(got, _sort64(ids, E)):
        assert g.dtype == w.dtype and torch.equal(g.cpu(), w)


@pytest.mark.parametrize("T,k,E", [(0, 2, 4), (1, 1, 1), (1, 8, 256), (61, 8, 256), (64, 1, 3), (513, 2, 1024), (1023, 8, 60),
                                   (1024, 8, 256), (1025, 8, 256), (8192, 1, 7), (8193, 1, 7), (5000, 3, 1), (40000, 8, 256),
                                   (70001, 6, 1000), (300000, 1, 2)])
def test_sort(dev, T, k, E):
    ids = torch.randint(0, E, (T, k), generator=_gen(T + k))
    _check_sort(dev, ids, E)
    if T > 1:
        skew = (torch.rand(T, k, generator=_gen(T)) ** 4 * E).long()
        _check_sort(dev, skew, E)
        _check_sort(dev, torch.full_like(ids, E - 1), E)  # every choice the same expert
        _check_sort(dev, ids.flip(0), E)
        bad = ids.clone()  # some choices belong to nobody
        bad[:: 3, 0], bad[1::5, -1], bad[-1, 0] = -1, E, torch.iinfo(torch.int64).max
        _check_sort(dev, bad, E)
        _check_sort(dev, torch.full_like(ids, -1), E)
        _check_sort(dev, ids.t().contiguous().t(), E)


def test_route_tokens_matches_the_host(dev):
    ids = torch.randint(0, 9, (5000, 3), generator=_gen(8))
    rows, offsets = moe_layer.route_tokens(ids.to(dev), 9)
    want_rows, want = moe_layer.route_tokens(ids, 9)
    assert torch.equal(rows.cpu(), want_rows) and offsets == want and isinstance(offsets, list)
    with pytest.raises(ValueError):
        moe_layer.route_tokens(ids.to(dev), 8)


# ---- quantize ---------------------------------------------------------------------------------------------
def _codes64(x):
    """Exact codes by whole-number arithmetic in python for every value that is near a border, by 64 bits elsewhere."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    z = torch.where(top > 0, x * 127.0 / torch.where(top > 0, top, torch.ones_like(top)), torch.zeros_like(x))
    return z.round().to(torch.int8), (top / 127).squeeze(-1)


def _check_quantize(dev, x):
    q, s = ops.quantize_tokens(x.to(dev))
    want_q, want_s = _codes64(x)
    assert q.dtype == torch.int8 and s.dtype == torch.float32
    assert torch.equal(q.cpu(), want_q)
    assert ((s.cpu().double() - want_s).abs() <= U * want_s + 2.0**-149).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n,C", [(1, 1), (1, 7168), (3, 5), (4, 64), (7, 2048), (5, 1000), (2, 16384), (33, 100), (300, 512),
                                 (2, 40001), (9, 2304), (1, 8), (2, 18432)])
def test_quantize(dev, dtype, n, C):
    x = torch.randn(n, C, generator=_gen(n * C)) * torch.exp(torch.randn(n, 1, generator=_gen(n)))
    x[:, C // 3] *= 20
    _check_quantize(dev, x.to(DT[dtype]))


@pytest.mark.parametrize("dtype", DT)
def test_quantize_borders(dev, dtype):
    """Rows of exact ties (a row whose largest value is 127 or 254 times a power of two has them everywhere) and of values
    one step beside them."""
    dt = DT[dtype]
    half = torch.arange(-127, 127).float() + 0.5
    rows = []
    for scale in (1.0, 2.0**-9, 2.0**5):
        r = torch.cat([half, torch.tensor([127.0])]) * scale
        rows += [r, torch.cat([2 * half, torch.tensor([254.0])]) * scale]
    x = torch.stack(rows).to(dt)
    _check_quantize(dev, x)
    bits = {2: torch.int16, 4: torch.int32}[x.element_size()]
    for step in (-1, 1):
        y = (x.view(bits) + step).view(dt)
        y[:, -1] = x[:, -1]
        _check_quantize(dev, y)
    z = torch.randn(64, 512, generator=_gen(1)).to(dt)
    z[:, :64] = (z.float().abs().amax(-1, keepdim=True) / 2).to(dt)  # half the largest: 63.5 exactly
    _check_quantize(dev, z)


@pytest.mark.parametrize("dtype", DT)
def test_quantize_zero_tiny_and_not_finite(dev, dtype):
    dt = DT[dtype]
    x = torch.randn(8, 300, generator=_gen(2)).to(dt)
    x[0] = 0
    x[1] = -0.0
    x[2, 17] = math.nan
    x[3, 299] = math.inf
    x[4, 0] = -math.inf
    x[5] = torch.finfo(dt).max
    q, s = ops.quantize_tokens(x.to(dev))
    q, s = q.cpu(), s.cpu()
    assert (q[:2] == 0).all() and (s[:2] == 0).all()
    assert s[2:5].isnan().all() and (q[2:5] == 0).all()
    fine = [5, 6, 7]
    assert torch.equal(q[fine], _codes64(x[fine])[0]) and torch.isfinite(s[fine]).all()
    tiny = torch.zeros(3, 64)
    tiny[0, 3], tiny[1, 5], tiny[1, 6] = torch.finfo(dt).tiny, torch.finfo(dt).tiny, -torch.finfo(dt).tiny / 2
    tiny[2, 1] = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps  # the smallest denormal
    q, s = ops.quantize_tokens(tiny.to(dt).to(dev))
    assert q[0, 3] == 127 and q[1, 5] == 127 and q[1, 6] == -64 and q.cpu()[2].abs().sum() == 127
    assert ops.quantize_tokens(torch.zeros(0, 8, device=dev))[0].shape == (0, 8)


def test_quantize_strides(dev):
    base = torch.randn(50, 200, generator=_gen(3))
    g = base.to(dev)
    for view in (lambda t: t[:, 3:150], lambda t: t[::3, :64], lambda t: t.t()[:40], lambda t: t[:1].expand(3, 200)):
        q, s = ops.quantize_tokens(view(g))
        assert torch.equal(q.cpu(), _codes64(view(base))[0])


# ---- products -----------------------------------------------------------------------------------------------
def _rand_codes(g, *shape):
    return torch.randint(-128, 128, shape, generator=g, dtype=torch.int64).to(torch.int8)


def _product64(A, sa, B, sb, bias=None, swiglu=False):
    """(result, magnitude the 32-bit roundings are relative to, the SwiGLU's extra relative and absolute error).  Absolute:
    below g = -88.7 exp(-g) passes 2^128 and is inf in 32 bits, the quotient 0 instead of g exp(g) < |g| 2^-128; just above
    it the quotient may be flushed from below 2^-126.  Both are at most |g u| 2^-126 off."""
    y = (A.double() @ B.double().t()) * sa.double()[:, None] * sb.double()
    if swiglu:
        g, u = y.chunk(2, dim=1)
        out = g / (1 + torch.exp(-g)) * u
        return out, out.abs(), (64 + 8 * g.abs(), (g * u).abs() * 2.0**-126)
    mag = y.abs()
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    return y, mag, None


def _close(got, want, mag, extra, dt):
    # sum -> float, two scales (one product with another's rounding), bias: 4 roundings; SwiGLU: exp's argument and the
    # errors of its operands on top; then one rounding to dt (and the steps of f16 below its normal range)
    rel, low = (5 * U, 0.0) if extra is None else ((5 + extra[0]) * U, extra[1])
    tol = rel * mag * (1 + _half(dt)) + low + _half(dt) * want.abs() + (2.0**-25 if dt == torch.float16 else 2.0**-140)
    err = (got.cpu().double() - want).abs()
    assert (err <= tol).all(), ((err - tol).max(), err.max())


SHAPES = [(1, 1, 1), (1, 2048, 7168), (1, 7, 33), (2, 64, 64), (3, 100, 500), (4, 576, 1024), (5, 130, 129), (8, 96, 4096),
          (16, 256, 256), (17, 257, 255), (31, 40, 1000), (33, 576, 7168), (64, 192, 96), (65, 129, 640), (100, 1536, 320),
          (127, 128, 64), (128, 128, 128), (129, 384, 192), (255, 255, 257), (256, 256, 128), (257, 300, 384), (300, 1000, 72),
          (333, 576, 7168), (512, 520, 208), (700, 2048, 48), (1025, 264, 1040), (2, 5000, 16), (60, 33, 16400),
          (320, 320, 16), (4100, 4200, 64), (2100, 2600, 130), (2561, 2304, 449), (1500, 5000, 20)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(dev, M, N, K):
    g = _gen(M * N + K)
    A, B = _rand_codes(g, M, K), _rand_codes(g, N, K)
    sa, sb = torch.rand(M, generator=g) + 0.1, (torch.rand(N, generator=g) + 0.1) / (100 * K**0.5)
    for name, dt in DT.items():
        _say("product", M, N, K, name)
        bias = torch.randn(N, generator=g).to(dt)
        want, mag, _ = _product64(A, sa, B, sb)
        _close(ops.matmul_int8(A.to(dev), sa.to(dev), B.to(dev), sb.to(dev), None, dt), want, mag, None, dt)
        want, mag, _ = _product64(A, sa, B, sb, bias)
        _close(ops.matmul_int8(A.to(dev), sa.to(dev), B.to(dev), sb.to(dev), bias.to(dev), dt), want, mag, None, dt)
        if N % 2 == 0:
            want, mag, extra = _product64(A, sa, B, sb, None, True)
            got = ops.matmul_int8(A.to(dev), sa.to(dev), B.to(dev), sb.to(dev), None, dt, swiglu=True)
            _close(got, want, mag, extra, dt)


def test_product_extremes(dev):
    """The longest sum of the largest products stays inside 32 bits; scales of 0 and NaN reach their own row only."""
    K = 131071
    for a, b in ((-128, -128), (-128, 127)):
        A, B = torch.full((3, K), a, dtype=torch.int8), torch.full((5, K), b, dtype=torch.int8)
        y = ops.matmul_int8(A.to(dev), torch.ones(3, device=dev), B.to(dev), torch.ones(5, device=dev), None, torch.float32)
        assert ((y.cpu().double() - float(a) * b * K).abs() <= abs(a * b * K) * U).all()
    g = _gen(9)
    for M in (4, 200):
        A, B = _rand_codes(g, M, 256), _rand_codes(g, 192, 256)
        sa = torch.ones(M)
        sa[1], sa[2] = 0.0, math.nan
        y = ops.matmul_int8(A.to(dev), sa.to(dev), B.to(dev), torch.ones(192, device=dev), None, torch.float32).cpu()
        assert (y[1] == 0).all() and y[2].isnan().all() and y[0].isfinite().all() and y[3:].isfinite().all()


@pytest.mark.parametrize("M", [1, 20, 300])
def test_product_views(dev, M):
    """Pitches and starts off every alignment; rows beside the ones asked for are not touched by reads that matter."""
    g = _gen(M)
    A, B = _rand_codes(g, M, 700), _rand_codes(g, 260, 700)
    sa, sb = torch.rand(M, generator=g), torch.rand(260, generator=g)
    for a0, b0, K in ((0, 0, 640), (16, 32, 256), (1, 0, 512), (0, 3, 130), (5, 7, 333), (4, 4, 64)):
        Av, Bv = A[:, a0:a0 + K], B[:, b0:b0 + K]
        want, mag, _ = _product64(Av, sa, Bv, sb)
        got = ops.matmul_int8(A.to(dev)[:, a0:a0 + K], sa.to(dev), B.to(dev)[:, b0:b0 + K], sb.to(dev), None, torch.float32)
        _close(got, want, mag, None, torch.float32)
    want, mag, _ = _product64(A[:, ::2], sa, B[:, ::2], sb)
    _close(ops.matmul_int8(A.to(dev)[:, ::2], sa.to(dev), B.to(dev)[:, ::2], sb.to(dev), None, torch.float32), want, mag, None,
           torch.float32)
    assert ops.matmul_int8(A.to(dev)[:0], sa.to(dev)[:0], B.to(dev), sb.to(dev)).shape == (0, 260)


@pytest.mark.parametrize("M,N,K", [(1, 2048, 7168), (1, 1, 16), (1, 33, 1000), (2, 70, 1003), (2, 576, 17), (1, 9, 5), (3, 100, 257),
                                   (1, 40, 81920), (2, 24, 90001), (17, 64, 300), (300, 520, 130), (2100, 2600, 133), (2048, 2560, 96)])
def test_linear_equals_its_two_halves(dev, M, N, K):
    """quantize + product in one call: the same bits as the two calls (and their exact codes, for the fused rows too)."""
    g = _gen(M + N + K)
    B, sb = _rand_codes(g, N, K), (torch.rand(N, generator=g) + 0.1) / (100 * K**0.5)
    for name, dt in DT.items():
        _say("linear", M, N, K, name)
        x = torch.randn(M, K, generator=g)
        x[:, K // 3] *= 20
        x[-1, K // 2:] = 0 if M > 1 else x[-1, K // 2:]
        x = x.to(dt)
        bias = torch.randn(N, generator=g).to(dt)
        for b in (None, bias.to(dev)):
            got = ops.linear_int8(x.to(dev), B.to(dev), sb.to(dev), b)
            q, s = ops.quantize_tokens(x.to(dev))
            assert torch.equal(got, ops.matmul_int8(q, s, B.to(dev), sb.to(dev), b, dt))
        q, s = _codes64(x)
        want, mag, _ = _product64(q, s, B, sb, bias)
        _close(got, want, mag * (1 + U), None, dt)


def test_linear_special_rows(dev):
    """Rows of zeros, with a NaN, an infinity, and tiny ones, one and many tokens at a time."""
    g = _gen(77)
    B, sb = _rand_codes(g, 50, 300).to(dev), torch.ones(50, device=dev)
    x = torch.randn(5, 300, generator=g)
    x[0], x[1, 9], x[2, 299] = 0, math.nan, -math.inf
    x[3] *= 2.0**-120
    x = x.to(dev)
    whole = ops.linear_int8(x, B, sb)
    assert (whole[0] == 0).all() and whole[1:3].isnan().all() and whole[3:].isfinite().all()
    for r in range(5):
        for n in (1, 2):
            got = ops.linear_int8(x[r:r + n], B, sb)
            assert torch.equal(got.nan_to_num(7), whole[r:r + n].nan_to_num(7))
    assert ops.linear_int8(x[:0], B, sb).shape == (0, 50)
    y = ops.linear_int8(x.t()[:, :3].t(), B, sb)  # another stride
    assert torch.equal(y.nan_to_num(7), whole[:3].nan_to_num(7))


GROUPS = [([5], 40, 64), ([0, 0, 3], 130, 96), ([1] * 9, 64, 512), ([16, 0, 17, 1, 33], 96, 256), ([130, 0, 64, 1], 200, 128),
          ([300, 5, 0, 257], 264, 320), ([2, 1, 0, 0, 4, 0, 0], 576, 1030), ([700], 300, 144), ([0, 0], 32, 32),
          ([128, 128, 256], 512, 192), ([1] * 70, 48, 80), ([3] * 200, 16, 48), ([600, 256, 0, 513, 77], 9000, 64), ([255, 33, 97, 129], 5200, 452),
          ([40, 70, 0, 300], 64, 10)]


@pytest.mark.parametrize("counts,N,K", GROUPS)
def test_grouped(dev, counts, N, K):
    g = _gen(sum(counts) + N)
    E, S = len(counts), sum(counts)
    tail = 7  # rows behind the last range
    offsets = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)))
    B, sb = _rand_codes(g, E, N, K), (torch.rand(E, N, generator=g) + 0.1) / (100 * K**0.5)
    src = _rand_codes(g, 50, K)
    ssrc = torch.rand(50, generator=g) + 0.1
    rows = torch.randint(0, 50, (S + tail,), generator=g)
    if S > 2:
        rows[1], rows[S - 1] = -1, 50  # nobody's rows
    took = torch.where((rows >= 0) & (rows < 50), rows, torch.zeros_like(rows))
    live = ((rows >= 0) & (rows < 50)).to(torch.int8)
    Ag, sg = src[took] * live[:, None], ssrc[took] * live
    plain, splain = _rand_codes(g, S + tail, K), torch.rand(S + tail, generator=g)
    for dt in DT.values():
        for swiglu in (False, True):
            n = N // 2 if swiglu else N
            for gather in (False, True):
                _say("grouped", counts[:6], N, K, dt, swiglu, gather)
                A, sa = (Ag, sg) if gather else (plain, splain)
                out = torch.full((S + tail, n), 77.0, dtype=dt, device=dev)
                a_in, s_in = (src, ssrc) if gather else (plain, splain)
                got = ops.matmul_int8_grouped(a_in.to(dev), s_in.to(dev), B.to(dev), sb.to(dev), offsets.to(dev),
                                              rows.to(dev) if gather else None, dt, swiglu, out)
                assert got is out and (out[S:] == 77.0).all()
                for e in range(E):
                    lo, hi = offsets[e], offsets[e + 1]
                    if lo == hi:
                        continue
                    want, mag, extra = _product64(A[lo:hi], sa[lo:hi], B[e], sb[e], None, swiglu)
                    _close(out[lo:hi], want, mag, extra, dt)


def test_grouped_strange_offsets(dev):
    """Offsets that leave [0, S] or run backwards are clamped: nothing outside the result is written."""
    g = _gen(5)
    A, B = _rand_codes(g, 40, 64), _rand_codes(g, 3, 32, 64)
    sa, sb = torch.ones(40), torch.ones(3, 32)
    for off in ([-5, 10, 20, 1000], [30, 20, 10, 0], [0, 0, 2**40, 2**41], [50, 60, 70, 80]):
        frame = torch.full((60, 32), 5.0, device=dev)
        out = frame[10:50]
        ops.matmul_int8_grouped(A.to(dev), sa.to(dev), B.to(dev), sb.to(dev), torch.tensor(off, device=dev), None, torch.float32,
                                False, out)
        assert (frame[:10] == 5).all() and (frame[50:] == 5).all()
    out = torch.full((40, 64), 5.0, device=dev)  # a strided result: columns beside it stay
    ops.matmul_int8_grouped(A.to(dev), sa.to(dev), B.to(dev), sb.to(dev), torch.tensor([0, 10, 20, 40], device=dev), None,
                            torch.float32, False, out[:, 16:48])
    assert (out[:, :16] == 5).all() and (out[:, 48:] == 5).all()
    want, mag, _ = _product64(A[20:], sa[20:], B[2], sb[2])
    _close(out[20:, 16:48], want, mag, None, torch.float32)


def test_grouped_strange_offsets_few_rows(dev):
    """The same with fewer rows than experts (rows look their experts up), and rows that leave A altogether."""
    g = _gen(15)
    E, S = 70, 9
    A, B = _rand_codes(g, S, 64), _rand_codes(g, E, 32, 64)
    sa, sb = torch.ones(S), torch.ones(E, 32)
    up = torch.arange(E + 1)
    for off in (up * 0, up * 0 + S, up - 30, up.flip(0), torch.where(up > 40, up * 0 + 5, up * 0), up * 2**35 - 2**36):
        frame = torch.full((S + 20, 32), 5.0, device=dev)
        out = frame[10:10 + S]
        ops.matmul_int8_grouped(A.to(dev), sa.to(dev), B.to(dev), sb.to(dev), off.to(dev), None, torch.float32, False, out)
        assert (frame[:10] == 5).all() and (frame[10 + S:] == 5).all()
    off = torch.where(up > 40, up * 0 + S, up * 0)  # all rows belong to expert 40
    for rows in (None, torch.tensor([-1, 9, 2**40, -2**50, 0, 8, 3, 3, 9])):
        got = ops.matmul_int8_grouped(A.to(dev), sa.to(dev), B.to(dev), sb.to(dev), off.to(dev),
                                      None if rows is None else rows.to(dev), torch.float32)
        took = A if rows is None else torch.stack([A[r] if 0 <= r < S else A[0] * 0 for r in rows.tolist()])
        assert torch.equal(got.cpu().double(), took.double() @ B[40].double().t())
    for n in (S, 700):  # no rows in A at all: without tiles and with them
        off = torch.where(up > 40, up * 0 + n, up * 0)
        none = ops.matmul_int8_grouped(A.to(dev)[:0], sa.to(dev)[:0], B.to(dev), sb.to(dev), off.to(dev),
                                       torch.zeros(n, dtype=torch.int64, device=dev), torch.float32)
        assert none.shape == (n, 32) and (none == 0).all()


@pytest.mark.parametrize("dt,K,swiglu,gather", [("bf16", 64, False, False), ("f16", 449, True, True), ("f32", 204, False, True)])
def test_grouped_many_rows(dev, dt, K, swiglu, gather):
    """Large tiles: many rows an expert, and enough tiles to go round several times."""
    g, dt = _gen(K), DT[dt]
    counts, N, ld = [600, 0, 300, 260, 5, 1000], 18708, (K + 3) // 4 * 4
    E, S = len(counts), sum(counts)
    offsets = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)))
    B = _rand_codes(g, E, N, ld)
    sb = (torch.rand(E, N, generator=g) + 0.1) / (100 * K**0.5)
    A, sa = _rand_codes(g, S, ld), torch.rand(S, generator=g) + 0.1
    rows = torch.randint(0, S, (S,), generator=g) if gather else torch.arange(S)
    if gather:
        rows[0], rows[601], rows[S - 1] = -1, S, 2**40
    out = torch.full((S + 3, N // 2 if swiglu else N), 77.0, dtype=dt, device=dev)
    ops.matmul_int8_grouped(A.to(dev)[:, :K], sa.to(dev), B.to(dev)[:, :, :K], sb.to(dev), offsets.to(dev),
                            rows.to(dev) if gather else None, dt, swiglu, out[:S])
    out = out.cpu()
    assert (out[S:] == 77).all()
    live = (rows >= 0) & (rows < S)
    took = torch.where(live, rows, torch.zeros_like(rows))
    for e in range(E):
        lo, hi = offsets[e], offsets[e + 1]
        for c in range(lo, hi, 256):  # (parts, to keep the 64-bit results small)
            d = min(c + 256, hi)
            r = took[c:d]
            want, mag, extra = _product64(A[r, :K] * live[c:d, None].to(torch.int8), sa[r], B[e, :, :K], sb[e], None, swiglu)
            _close(out[c:d], want, mag, extra, dt)


def test_grouped_one_row_of_weights(dev):
    g = _gen(16)
    full = _rand_codes(g, 4, 3, 96)
    A, sa = _rand_codes(g, 30, 96), torch.rand(30, generator=g)
    off = torch.tensor([0, 7, 7, 20, 30])
    sb = torch.rand(4, 1, generator=g)
    got = ops.matmul_int8_grouped(A.to(dev), sa.to(dev), full.to(dev)[:, 1:2], sb.to(dev), off.to(dev), None, torch.float32)
    for e in range(4):
        lo, hi = off[e], off[e + 1]
        if lo < hi:
            want, mag, _ = _product64(A[lo:hi], sa[lo:hi], full[e, 1:2], sb[e])
            _close(got[lo:hi], want, mag, None, torch.float32)


def test_experts_forward_without_tokens(dev):
    ex = _experts(_gen(17), 4, 64, 16, dev)
    y = moe_layer.experts_forward_int8(torch.zeros(0, 64, device=dev), torch.zeros(0, 2, dtype=torch.int64, device=dev),
                                       torch.zeros(0, 2, device=dev), ex)
    assert y.shape == (0, 64)
    x = torch.randn(3, 64, device=dev)
    nobody = torch.full((3, 2), -1, dtype=torch.int64, device=dev)  # every choice dropped
    assert (moe_layer.experts_forward_int8(x, nobody, torch.ones(3, 2, device=dev), ex) == 0).all()


def test_rows_beyond_one_grid_dimension(dev):
    """More than 65536 workgroups of one row each."""
    x = torch.randn(70001, 1040, generator=_gen(18)).bfloat16()
    q, s = ops.quantize_tokens(x.to(dev))
    want, ws = _codes64(x)
    assert torch.equal(q.cpu(), want) and ((s.cpu().double() - ws).abs() <= U * ws).all()
    Y = torch.randn(50, 16, generator=_gen(19))
    slots = torch.randint(0, 50, (140001, 1), generator=_gen(20), dtype=torch.int32)
    w = torch.rand(140001, 1, generator=_gen(21))
    out = ops.combine_experts(Y.to(dev), slots.to(dev), w.to(dev)).cpu()
    assert torch.equal(out, Y[slots[:, 0].long()] * w)


def test_grouped_weights_with_gaps(dev):
    g = _gen(6)
    full = _rand_codes(g, 6, 80, 160)
    A, sa, sb = _rand_codes(g, 30, 128), torch.rand(30, generator=g), torch.rand(3, 64, generator=g)
    off = torch.tensor([0, 11, 11, 30])
    for view in (lambda t: t[::2, 8:72, 16:144], lambda t: t[1::2, 3:67, 5:133]):
        B = view(full)
        got = ops.matmul_int8_grouped(A.to(dev), sa.to(dev), view(full.to(dev)), sb.to(dev), off.to(dev), None, torch.float32)
        for e, (lo, hi) in enumerate(((0, 11), (11, 11), (11, 30))):
            want, mag, _ = _product64(A[lo:hi], sa[lo:hi], B[e], sb[e])
            _close(got[lo:hi], want, mag, None, torch.float32)


# ---- combine --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("S,C,T,k", [(1, 1, 1, 1), (16, 7168, 2, 8), (100, 33, 25, 4), (64, 2048, 64, 1), (30, 1000, 10, 3),
                                     (50, 2056, 7, 9), (5, 64, 0, 2), (0, 64, 3, 2)])
def test_combine(dev, dtype, S, C, T, k):
    dt, g = DT[dtype], _gen(S * C + T)
    Y = torch.randn(S, C, generator=g).to(dt)
    slots = torch.randint(0, max(S, 1), (T, k), generator=g, dtype=torch.int32)
    if T > 2:
        slots[1, 0], slots[2] = -1, -1
        slots[0, -1] = S  # nobody's
    w = torch.rand(T, k, generator=g)
    out = ops.combine_experts(Y.to(dev), slots.to(dev), w.to(dev))
    want, mag = torch.zeros(T, C, dtype=torch.float64), torch.zeros(T, C, dtype=torch.float64)
    for t in range(T):
        for j in range(k):
            if 0 <= slots[t, j] < S:
                term = w[t, j].double() * Y[slots[t, j]].double()
                want[t] += term
                mag[t] += term.abs()
    tol = k * U * mag * (1 + _half(dt)) + _half(dt) * want.abs() + (2.0**-25 if dt == torch.float16 else 2.0**-140)
    assert out.dtype == dt and ((out.cpu().double() - want).abs() <= tol).all()


def test_combine_views(dev):
    g = _gen(7)
    Y, slots, w = torch.randn(40, 300, generator=g), torch.randint(0, 40, (9, 6), generator=g, dtype=torch.int32), torch.rand(9, 6, generator=g)
    for v in (lambda t: t[:, 3:203], lambda t: t[:, ::2], lambda t: t[:, 4:68]):
        out = ops.combine_experts(v(Y.to(dev)), slots.to(dev)[:, ::2], w.to(dev)[:, ::2])
        want = (v(Y).double()[slots[:, ::2].long()] * w[:, ::2, None].double()).sum(1)
        mag = (v(Y).double()[slots[:, ::2].long()].abs() * w[:, ::2, None].double()).sum(1)
        assert ((out.cpu().double() - want).abs() <= 4 * U * mag).all()


# ---- together ---------------------------------------------------------------------------------------------------
def _experts(g, E, C, I, dev):
    return moe_layer.Int8Experts(_rand_codes(g, E, 2 * I, C).to(dev), ((torch.rand(E, 2 * I, generator=g) + 0.5) / (100 * C**0.5)).to(dev),
                                 _rand_codes(g, E, C, I).to(dev), ((torch.rand(E, C, generator=g) + 0.5) / (100 * I**0.5)).to(dev))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("T,E,k,C,I", [(1, 8, 2, 256, 64), (5, 16, 4, 72, 40), (64, 9, 3, 512, 128), (300, 4, 2, 264, 96),
                                       (700, 3, 1, 128, 200), (33, 24, 6, 100, 36)])
def test_experts_forward_together(dev, dtype, T, E, k, C, I):
    """Router -> sort -> quantize -> SwiGLU product -> quantize -> down product -> combine, as a block runs them; every
    stage against 64 bits on what the stage before it gave."""
    dt, g = DT[dtype], _gen(T + C)
    x = torch.randn(T, C, generator=g).to(dt)
    ex = _experts(g, E, C, I, dev)
    router = moe_layer.Router(torch.randn(E, C, generator=g).to(dev), k, score="sigmoid", bias=torch.zeros(E, device=dev), scale=2.5,
                              rows_per_call=100)
    weights, ids = router(x.to(dev))
    assert weights.shape == ids.shape == (T, k)
    ids[T // 2, 0] = -1  # a dropped choice
    y = moe_layer.experts_forward_int8(x.to(dev), ids, weights, ex)
    assert y.shape == (T, C) and y.dtype == dt
    rows, offsets, slots = _sort64(ids.cpu(), E)
    q, s = _codes64(x)
    h = ops.matmul_int8_grouped(*ops.quantize_tokens(x.to(dev)), ex.gate_up, ex.gate_up_scale, offsets.to(dev), rows.to(dev), dt, True).cpu()
    want, mag = torch.zeros(T * k, C, dtype=torch.float64), torch.zeros(T * k, C, dtype=torch.float64)
    for e in range(E):
        lo, hi = offsets[e], offsets[e + 1]
        if lo == hi:
            continue
        hw, hm, extra = _product64(q[rows[lo:hi]], s[rows[lo:hi]], ex.gate_up[e].cpu(), ex.gate_up_scale[e].cpu(), None, True)
        _close(h[lo:hi], hw, hm, (extra[0] + 2, extra[1]), dt)
        hq, hs = _codes64(h[lo:hi])
        want[lo:hi] = _product64(hq, hs, ex.down[e].cpu(), ex.down_scale[e].cpu())[0]
    sl, w = slots.long(), weights.cpu().double()
    w = torch.where(slots >= 0, w, torch.zeros_like(w))[..., None]
    out = (want[sl.clamp_min(0)] * w).sum(1)
    mag = (want[sl.clamp_min(0)].abs() * w).sum(1)
    # the experts' outputs are held in dt; then k terms in 32 bits and one rounding.  Below f16's normal range a rounding is
    # off by half its smallest step, 2^-25: once for each expert's output, times its weight, and once for the sum
    low = 2.0**-25 if dt == torch.float16 else 2.0**-141
    tol = ((6 + k) * U + _half(dt)) * mag * 1.01 + _half(dt) * out.abs() + low * (1 + w.sum(1))
    assert ((y.cpu().double() - out).abs() <= tol).all()


def test_gptq_codes_through_the_products(dev):
    """GPTQ with 8 bits and one scale per row -> int8_weight -> linear_int8: the layer on its dequantized weights."""
    g = _gen(21)
    lin = torch.nn.Linear(256, 96, bias=True, dtype=torch.bfloat16, device=dev)
    x = torch.randn(3, 50, 256, generator=g).bfloat16()
    h = GPTQ(lin, None, True, 0.01, 128)
    h.update(x.to(dev))
    w, s = quant_utils.int8_weight(*h.quantize(8))
    assert w.shape == (96, 256) and s.shape == (96,)
    y = quant_utils.linear_int8(x.to(dev), w, s, lin.bias.data)
    assert y.shape == (3, 50, 96) and y.dtype == torch.bfloat16
    q, qs = _codes64(x.view(-1, 256))
    want, mag, _ = _product64(q, qs, w.cpu(), s.cpu(), lin.bias.data.cpu())
    _close(y.view(-1, 96), want, mag * 1.2, None, torch.bfloat16)
    assert quant_utils.linear_int8(x.to(dev)[0, 0], w, s).shape == (96,)


def test_quantize_moe_layer_takes_a_router(dev):
    """The layer driver with a Router routes as the ids that Router gives, and its 8-bit codes run."""
    g = _gen(22)
    C, I, E, T = 256, 128, 4, 900
    x = torch.randn(T, C, generator=g).bfloat16().to(dev)
    mk = lambda r, c: (0.05 * torch.randn(r, c, generator=g)).bfloat16().to(dev)
    experts = [moe_layer.ExpertWeights(mk(I, C), mk(I, C), mk(C, I)) for _ in range(E)]
    router = moe_layer.Router(mk(E, C), 2)
    weights, ids = router(x)
    kw = dict(bits=8, group_size=None, keep_outputs=False, keep_codes=list(range(E)), group=2)
    a = moe_layer.quantize_moe_layer(x, router, experts, **kw)
    b = moe_layer.quantize_moe_layer(x, ids, experts, **kw)
    assert a.tokens_per_expert == b.tokens_per_expert == torch.bincount(ids.flatten().cpu(), minlength=E).tolist()
    for n in a.qweight:
        assert torch.equal(a.qweight[n], b.qweight[n]) and torch.equal(a.scales[n], b.scales[n])
    three = lambda e: tuple((a.qweight[f"{e}.{n}"], a.scales[f"{e}.{n}"], torch.full_like(a.scales[f"{e}.{n}"], 128))
                            for n in ("gate_proj", "up_proj", "down_proj"))
    ex = moe_layer.Int8Experts.from_quantized([three(e) for e in range(E)])
    y = moe_layer.experts_forward_int8(x, ids, weights, ex).cpu().double()
    plain = torch.zeros(T, C, dtype=torch.float64)
    xd = x.cpu().double()
    for e in range(E):
        t, j = (ids.cpu() == e).nonzero(as_tuple=True)
        gate, up, down = (w.cpu().double() for w in (experts[e].gate, experts[e].up, experts[e].down))
        hh = xd[t] @ gate.t()
        hh = hh / (1 + torch.exp(-hh)) * (xd[t] @ up.t())
        plain.index_add_(0, t, (hh @ down.t()) * weights.cpu().double()[t, j][:, None])
    # steps of max / 127 on tokens and weights: about 1% a product; an error of wiring would be of order one
    assert ((y - plain).norm() / plain.norm()).item() < 0.1


# ---- streams, graphs ----------------------------------------------------------------------------------------------
def test_replayed_from_graphs_that_share_a_stream(dev):
    """Two captured graphs of the whole run, replayed several times on two streams with eager work in between."""
    g = _gen(30)
    E, k, C, I, T = 12, 3, 256, 64, 1100 * 3
    ex = _experts(g, E, C, I, dev)
    gate = torch.randn(E, C, generator=g).to(dev)
    xs = [torch.randn(T, C, generator=g).bfloat16().to(dev) for _ in range(2)]
    logits = [(x.float() @ gate.t()) for x in xs]

    def step(i):
        w, ids = ops.route_experts(logits[i], k, score="sigmoid", n_group=4, topk_group=2)
        return moe_layer.experts_forward_int8(xs[i], ids, w, ex)

    eager = [step(i).clone() for i in range(2)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for i in range(2):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=side):
                outs.append(step(i))
            graphs.append(gr)
    other = torch.cuda.Stream()
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
        again = step(0)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], eager[0]) and torch.equal(outs[1], eager[1]) and torch.equal(again, eager[0])


def test_two_streams_at_once(dev):
    g = _gen(31)
    ids = [torch.randint(0, 256, (50000, 8), generator=g) for _ in range(2)]
    on = [i.to(dev) for i in ids]
    want = [_sort64(i, 256) for i in ids]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(4):
        for s, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[s].append(ops.sort_by_expert(on[s], 256))
    torch.cuda.synchronize()
    for s in range(2):
        for r in got[s]:
            assert all(torch.equal(a.cpu(), b) for a, b in zip(r, want[s]))


def test_results_repeat(dev):
    """The same call twice gives the same bits (no sum depends on an order of arrival)."""
    g = _gen(32)
    for M, N, K in ((3, 520, 7168), (333, 576, 7168), (700, 300, 512)):
        A, B = _rand_codes(g, M, K).to(dev), _rand_codes(g, N, K).to(dev)
        sa, sb = torch.rand(M, generator=g).to(dev), torch.rand(N, generator=g).to(dev)
        first = ops.matmul_int8(A, sa, B, sb, None, torch.float32)
        assert all(torch.equal(first, ops.matmul_int8(A, sa, B, sb, None, torch.float32)) for _ in range(3))
