"""Routing and 8-bit products, the parts that need no GPU: refusals of the wrappers (arguments are checked before the
device) and of the C ABI, the host helpers around them."""
import ctypes

import pytest
import torch

from moe_quant_amd import _lib, moe_layer, ops, quant_utils

F32, I64, I32, I8 = torch.float32, torch.int64, torch.int32, torch.int8


def test_cpu_tensors_are_refused():
    x, q = torch.zeros(4, 16), torch.zeros(4, 16, dtype=I8)
    with pytest.raises(_lib.MoeQuantHipError):
        ops.route_experts(x, 2)
    with pytest.raises(_lib.MoeQuantHipError):
        ops.sort_by_expert(torch.zeros(4, 2, dtype=I64), 8)
    with pytest.raises(_lib.MoeQuantHipError):
        ops.quantize_tokens(x)
    with pytest.raises(_lib.MoeQuantHipError):
        ops.matmul_int8(q, torch.ones(4), q, torch.ones(4))
    with pytest.raises(_lib.MoeQuantHipError):
        ops.matmul_int8_grouped(q, torch.ones(4), q[None], torch.ones(1, 4), torch.tensor([0, 4]))
    with pytest.raises(_lib.MoeQuantHipError):
        ops.combine_experts(x, torch.zeros(2, 2, dtype=I32), torch.zeros(2, 2))


@pytest.mark.parametrize("kw", [
    dict(top_k=0), dict(top_k=17), dict(top_k=2, score="tanh"), dict(top_k=2, n_group=3), dict(top_k=2, n_group=0),
    dict(top_k=9, n_group=4, topk_group=2), dict(top_k=2, n_group=4, topk_group=5), dict(top_k=2, n_group=4, topk_group=0),
    dict(top_k=2, n_group=16, topk_group=4, group_top=2), dict(top_k=2, n_group=4, topk_group=2, group_top=3),
    dict(top_k=2, bias=torch.zeros(15)), dict(top_k=2, bias=torch.zeros(16, dtype=torch.bfloat16)),
    dict(top_k=2, bias=torch.zeros(32)[::2]),
])
def test_route_refusals(kw):
    with pytest.raises(ValueError):
        ops.route_experts(torch.zeros(3, 16), **kw)


def test_route_refuses_shapes_and_types():
    for bad in (torch.zeros(16), torch.zeros(3, 16, dtype=torch.float64), torch.zeros(3, 0), torch.zeros(3, 1025)):
        with pytest.raises(ValueError):
            ops.route_experts(bad, 1)
    with pytest.raises(ValueError):
        ops.route_experts(torch.zeros(3, 128), 65)


def test_sort_refusals():
    for ids, E in ((torch.zeros(4, dtype=I64), 4), (torch.zeros(4, 2, dtype=I32), 4), (torch.zeros(4, 0, dtype=I64), 4),
                   (torch.zeros(4, 2, dtype=I64), 0), (torch.zeros(4, 2, dtype=I64), 1025),
                   (torch.zeros(1, dtype=I64).expand(1 << 30, 2), 4)):
        with pytest.raises(ValueError):
            ops.sort_by_expert(ids, E)


def test_combine_refusals():
    Y, s, w = torch.zeros(4, 8), torch.zeros(3, 2, dtype=I32), torch.zeros(3, 2)
    for a in ((Y[0], s, w), (Y.double(), s, w), (Y, s.long(), w), (Y, s, w[:2]), (Y, s, w.bfloat16()), (Y, s[:, :0], w[:, :0])):
        with pytest.raises(ValueError):
            ops.combine_experts(*a)


def test_product_refusals():
    A, B, sa, sb = torch.zeros(3, 32, dtype=I8), torch.zeros(6, 32, dtype=I8), torch.zeros(3), torch.zeros(6)
    ok = dict(A=A, a_scale=sa, B=B, b_scale=sb)
    wide = torch.zeros(1, dtype=I8).expand(2, 131072)
    for bad in (dict(A=A.short()), dict(A=A[:, :31]), dict(B=B[None]), dict(B=B.short()), dict(a_scale=sa[:2]),
                dict(a_scale=sa.double()), dict(b_scale=sb[:5]), dict(b_scale=torch.zeros(12)[::2]), dict(out_dtype=torch.int32),
                dict(bias=torch.zeros(6)), dict(bias=torch.zeros(5), out_dtype=F32),
                dict(bias=torch.zeros(3), out_dtype=F32, swiglu=True), dict(B=B[:5], b_scale=sb[:5].clone(), swiglu=True),
                dict(A=A[:, :0], B=B[:, :0]), dict(B=B[:0], b_scale=sb[:0]),
                dict(A=wide, B=wide, a_scale=torch.zeros(2), b_scale=torch.zeros(2))):
        with pytest.raises(ValueError):
            ops.matmul_int8(**{**ok, **bad})
    for bad in (torch.zeros(3), torch.zeros(3, 4, dtype=torch.float64), torch.zeros(3, 0)):
        with pytest.raises(ValueError):
            ops.quantize_tokens(bad)
    x = torch.zeros(3, 32)
    for bad in ((x[0], B, sb), (x.double(), B, sb), (x[:, :31], B, sb), (x, B.short(), sb), (x, B[None], sb), (x, B, sb[:5]),
                (x, B, sb.double()), (x, B, sb, torch.zeros(5)), (x, B, sb, torch.zeros(6).half()), (x[:, :0], B[:, :0], sb)):
        with pytest.raises(ValueError):
            ops.linear_int8(*bad)
    with pytest.raises(ValueError):
        quant_utils.linear_int8(torch.zeros(()), B, sb)
    with pytest.raises(_lib.MoeQuantHipError):
        quant_utils.linear_int8(x, B, sb)


def test_grouped_refusals():
    ok = dict(A=torch.zeros(5, 32, dtype=I8), a_scale=torch.zeros(5), B=torch.zeros(2, 6, 32, dtype=I8),
              b_scale=torch.zeros(2, 6), offsets=torch.tensor([0, 2, 5]))
    for bad in (dict(B=ok["B"][0], b_scale=ok["b_scale"][0]), dict(offsets=torch.tensor([0, 5])),
                dict(offsets=torch.tensor([0, 2, 5], dtype=I32)), dict(rows=torch.zeros(5, dtype=I32)),
                dict(rows=torch.zeros(5, 1, dtype=I64)), dict(out=torch.zeros(5, 6)), dict(out=torch.zeros(4, 6), out_dtype=F32),
                dict(out=torch.zeros(6, 5).t(), out_dtype=F32), dict(B=ok["B"][:0], b_scale=ok["b_scale"][:0])):
        with pytest.raises(ValueError):
            ops.matmul_int8_grouped(**{**ok, **bad})


def test_c_abi_refusals():
    """Bad arguments come back as codes, before anything is launched (no GPU here)."""
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.cast(buf, ctypes.c_void_p)
    ARG, WS = _lib.MQ_ERR_ARG, _lib.MQ_ERR_WORKSPACE

    def route(**k):
        a = dict(l=p, dt=0, ldl=16, T=2, E=16, k=2, score=0, b=None, g=1, tg=1, gt=1, rn=1, s=1.0, w=p, i=p)
        a.update(k)
        return lib.mq_route_experts(*a.values(), None)

    for bad in (dict(E=0), dict(E=1025, ldl=1025), dict(k=0), dict(k=17), dict(ldl=15), dict(score=2), dict(dt=3), dict(g=3),
                dict(g=4, tg=5), dict(g=4, tg=2, gt=3), dict(g=4, tg=1, gt=1, k=5), dict(T=-1), dict(l=None), dict(w=None),
                dict(i=None), dict(g=0)):
        assert route(**bad) == ARG, bad
    assert route(T=0) == _lib.MQ_OK

    def sort(**k):
        a = dict(ids=p, T=2, k=2, E=4, rows=p, off=p, sl=p, ws=None, wsb=0)
        a.update(k)
        return lib.mq_sort_by_expert(*a.values(), None)

    for bad in (dict(T=-1), dict(k=0), dict(E=0), dict(E=1025), dict(T=1 << 30, k=4), dict(ids=None), dict(rows=None),
                dict(off=None)):
        assert sort(**bad) == ARG, bad
    big = lib.mq_sort_by_expert_workspace_bytes(1 << 20, 8, 256)
    assert big > 0 and lib.mq_sort_by_expert_workspace_bytes(16, 8, 256) == 0
    assert sort(T=1 << 20, k=8, E=256) == WS and sort(T=1 << 20, k=8, E=256, ws=p, wsb=big - 1) == WS

    for bad in ((None, 0, 8, 2, 8, p, p, 2, 2, p, 8), (p, 3, 8, 2, 8, p, p, 2, 2, p, 8), (p, 0, 7, 2, 8, p, p, 2, 2, p, 8),
                (p, 0, 8, 2, 8, None, p, 2, 2, p, 8), (p, 0, 8, 2, 8, p, p, 2, 0, p, 8), (p, 0, 8, 2, 8, p, p, 2, 2, p, 7)):
        assert lib.mq_combine_experts(*bad, None) == ARG
    for bad in ((None, 0, 8, 2, 8, p, 8, p), (p, 5, 8, 2, 8, p, 8, p), (p, 0, 8, 2, 8, p, 7, p), (p, 0, 8, 2, 0, p, 8, p),
                (p, 0, 8, -1, 8, p, 8, p)):
        assert lib.mq_quantize_tokens(*bad, None) == ARG

    def product(**k):
        a = dict(A=p, lda=32, sa=p, B=p, ldb=32, sb=p, bias=None, Y=p, ldy=8, dt=1, M=4, N=8, K=32, sw=0, ws=None, wsb=0)
        a.update(k)
        return lib.mq_matmul_int8(*a.values(), None)

    for bad in (dict(A=None), dict(lda=31), dict(ldb=31), dict(ldy=7), dict(dt=9), dict(N=0), dict(K=0), dict(M=-1),
                dict(K=131072, lda=131072, ldb=131072), dict(sw=1, bias=p)):
        assert product(**bad) == ARG, bad
    assert product(M=0) == _lib.MQ_OK

    def linear(**k):
        a = dict(X=p, dt=1, ldx=32, B=p, ldb=32, sb=p, bias=None, Y=p, ldy=8, M=4, N=8, K=32, ws=p, wsb=4096)
        a.update(k)
        return lib.mq_linear_int8(*a.values(), None)

    for bad in (dict(X=None), dict(ldx=31), dict(ldb=31), dict(ldy=7), dict(dt=-1), dict(N=0), dict(K=0), dict(M=-1), dict(Y=None),
                dict(K=131072, ldx=131072, ldb=131072)):
        assert linear(**bad) == ARG, bad
    need = lib.mq_linear_int8_workspace_bytes(4, 8, 32)
    assert need == 4 * 32 + 16 and lib.mq_linear_int8_workspace_bytes(1, 8, 32) == 0 and linear(M=0) == _lib.MQ_OK
    assert linear(ws=None) == WS and linear(wsb=need - 1) == WS
    odd = lib.mq_matmul_int8_workspace_bytes(4096, 4096, 1001, 0)
    assert odd == 8192 * 1008 and lib.mq_matmul_int8_workspace_bytes(4096, 4096, 1004, 0) == 0
    assert product(M=4096, N=4096, K=1001, lda=1001, ldb=1001, ldy=4096) == WS

    def grouped(**k):
        a = dict(A=p, lda=32, sa=p, src=4, rows=None, S=4, B=p, ldb=32, st=256, sb=p, E=2, off=p, Y=p, ldy=8, dt=1, N=8, K=32, sw=0)
        a.update(k)
        return lib.mq_matmul_int8_grouped(*a.values(), None)

    for bad in (dict(off=None), dict(E=0), dict(E=1025), dict(S=5), dict(st=-1), dict(src=-1), dict(K=0), dict(dt=4)):
        assert grouped(**bad) == ARG, bad
    assert grouped(S=0) == _lib.MQ_OK


def test_int8_weight():
    q = torch.tensor([[0, 128, 255], [128, 127, 129]], dtype=torch.uint8)
    w, s = quant_utils.int8_weight(q, torch.tensor([[0.5], [0.25]]).bfloat16(), torch.full((2, 1), 128.0).bfloat16())
    assert w.dtype == I8 and w.tolist() == [[-128, 0, 127], [0, -1, 1]] and s.tolist() == [0.5, 0.25] and s.dtype == F32
    with pytest.raises(ValueError):
        quant_utils.int8_weight(q, torch.ones(2, 3), torch.full((2, 3), 128.0))  # grouped scales
    with pytest.raises(ValueError):
        quant_utils.int8_weight(q, torch.ones(2, 1), torch.zeros(2, 1))  # 255 does not fit
    with pytest.raises(ValueError):
        quant_utils.int8_weight(q.int(), torch.ones(2, 1), torch.zeros(2, 1))


def test_int8_experts_from_quantized():
    z = torch.full((4, 1), 8.0)
    mk = lambda r, c, v: (torch.full((r, c), v, dtype=torch.uint8), torch.full((r, 1), 0.5 * v), torch.full((r, 1), 8.0))
    ex = moe_layer.Int8Experts.from_quantized([(mk(2, 4, 9), mk(2, 4, 10), mk(4, 2, 11)), (mk(2, 4, 1), mk(2, 4, 2), mk(4, 2, 3))])
    assert ex.gate_up.shape == (2, 4, 4) and ex.down.shape == (2, 4, 2) and z.numel() == 4
    assert ex.gate_up[0, :, 0].tolist() == [1, 1, 2, 2] and ex.gate_up_scale[1].tolist() == [0.5, 0.5, 1.0, 1.0]
    assert ex.down[1, 0, 0] == -5 and ex.down_scale[0].tolist() == [5.5] * 4


def test_route_tokens_on_the_host_is_unchanged():
    ids = torch.tensor([[2, 0], [1, 2], [0, 1]])
    rows, offsets = moe_layer.route_tokens(ids, 4)
    assert rows.tolist() == [0, 2, 1, 2, 0, 1] and offsets == [0, 2, 4, 6, 6]


def test_counts_beyond_32_bits_are_refused():
    """Sizes that a 32-bit count would cut: refused before anything is launched (the tensors are one element each)."""
    huge = torch.zeros(1, dtype=I8).expand((1 << 30) + 1, 64)
    small = torch.zeros(8, 64, dtype=I8)
    many = torch.zeros(1).expand((1 << 30) + 1)
    with pytest.raises(ValueError):
        ops.quantize_tokens(torch.zeros(1).expand((1 << 30) + 1, 4))
    with pytest.raises(ValueError):
        ops.matmul_int8(huge, many, small, torch.zeros(8))
    with pytest.raises(ValueError):
        ops.linear_int8(torch.zeros(1).expand((1 << 32) + 1, 64), small, torch.zeros(8))
    with pytest.raises(ValueError):
        ops.route_experts(torch.zeros(1).expand((1 << 25) + 1, 8), 2)
    with pytest.raises(ValueError):
        ops.combine_experts(torch.zeros(1).expand(4, 1 << 27), torch.zeros(1, 1, dtype=I32), torch.zeros(1, 1))
    lib = _lib.load()
    p = ctypes.cast(ctypes.create_string_buffer(64), ctypes.c_void_p)
    top = 0x7fffffff
    assert lib.mq_quantize_tokens(p, 0, 8, top, 8, p, 8, p, None) == _lib.MQ_ERR_ARG
    assert lib.mq_matmul_int8(p, 32, p, p, 32, p, None, p, 8, 1, top, 8, 32, 0, None, 0, None) == _lib.MQ_ERR_ARG
    assert lib.mq_linear_int8(p, 0, 32, p, 32, p, None, p, 8, top, 8, 32, p, 1 << 40, None) == _lib.MQ_ERR_ARG
    assert lib.mq_matmul_int8_grouped(p, 32, p, top, None, top, p, 32, 256, p, 2, p, p, 8, 1, 8, 32, 0, None) == _lib.MQ_ERR_ARG
    assert lib.mq_combine_experts(p, 0, 8, 4, 8, p, p, top, 2, p, 8, None) == _lib.MQ_ERR_ARG
    assert lib.mq_route_experts(p, 0, 16, top, 16, 2, 0, None, 1, 1, 1, 1, 1.0, p, p, None) == _lib.MQ_ERR_TOO_LARGE


def test_experts_forward_refusals():
    z = lambda *s: torch.zeros(*s, dtype=I8)
    ex = moe_layer.Int8Experts(z(3, 8, 16), torch.zeros(3, 8), z(3, 16, 4), torch.zeros(3, 16))
    x, ids, w = torch.zeros(5, 16), torch.zeros(5, 2, dtype=I64), torch.zeros(5, 2)
    for bad in ((x[:, :8], ids, w, ex), (x[0], ids, w, ex), (x, ids[:4], w, ex), (x, ids, w[:, :1], ex), (x, ids[:, 0], w[:, 0], ex),
                (x, ids, w, moe_layer.Int8Experts(z(3, 8, 16), torch.zeros(3, 8), z(3, 15, 4), torch.zeros(3, 15))),
                (x, ids, w, moe_layer.Int8Experts(z(8, 16), torch.zeros(8), z(16, 4), torch.zeros(16)))):
        with pytest.raises(ValueError):
            moe_layer.experts_forward_int8(*bad)


def test_sort_workspace_alignment():
    lib = _lib.load()
    buf = ctypes.create_string_buffer(64)
    p = ctypes.cast(buf, ctypes.c_void_p)
    need = lib.mq_sort_by_expert_workspace_bytes(10000, 1, 4)
    for off in (1, 2, 3):
        at = ctypes.c_void_p((p.value + 3) // 4 * 4 + off)
        assert lib.mq_sort_by_expert(p, 10000, 1, 4, p, p, p, at, need, None) == _lib.MQ_ERR_WORKSPACE
