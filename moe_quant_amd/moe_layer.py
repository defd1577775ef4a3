"""One MoE layer through the engine on one GPU: the expert part of MoE-Quant's per-block flow
(quant.py:241-411) with the model forward replaced by its two ingredients the Hessians need --
the routed token sets and the SwiGLU product that feeds each down projection.

Flow, as in the reference: all Hessians of the block are collected first (gate and up of an expert
share one, quant.py:258-277), then every linear is quantized and packed.  Everything stays resident
in HBM: 256 x 7168^2 fp32 gate/up Hessians (52.6 GB) + 256 x 2048^2 (4.3 GB) + 2M x 7168 bf16 tokens
(30 GB) + bf16 weights (22.5 GB) fit one MI355X.  Routed activations are gathered one expert at a time
(materialising all top-8 copies at once would take 240 GB).
"""
from __future__ import annotations

import time
from dataclasses import dataclass, field
from typing import Dict, List, Optional, Union

import torch
import torch.nn as nn

from . import ops, quant_utils
from .gptq import GPTQ


@dataclass
class ExpertWeights:
    gate: torch.Tensor  # (I, C) bf16
    up: torch.Tensor  # (I, C) bf16
    down: torch.Tensor  # (C, I) bf16


@dataclass
class LayerResult:
    seconds: Dict[str, float] = field(default_factory=dict)
    tokens_per_expert: List[int] = field(default_factory=list)
    packed: Dict[str, torch.Tensor] = field(default_factory=dict)  # "<e>.<proj>" -> int32 words (kept if asked)
    scales: Dict[str, torch.Tensor] = field(default_factory=dict)
    qweight: Dict[str, torch.Tensor] = field(default_factory=dict)  # only for the experts listed in keep_codes
    hessians: Dict[str, torch.Tensor] = field(default_factory=dict)  # idem (undamped copies)
    down_inputs: Dict[int, torch.Tensor] = field(default_factory=dict)  # idem: what the expert's down_proj saw
    issues: Dict[str, int] = field(default_factory=dict)
    issues_by_linear: Dict[str, List[str]] = field(default_factory=dict)  # "<e>.<proj>" -> names of raised flags
    factorizations: int = 0  # Hessian factorisations actually computed (a tied up_proj reuses its gate_proj's)
    overlapped: bool = False  # quantization ran beside the collection of later Hessians (seconds then overlap too)


def route_tokens(expert_ids: torch.Tensor, n_experts: int):
    """expert_ids (T, top_k) -> (order, offsets): order[offsets[e]:offsets[e+1]] are the token rows of expert e."""
    # (what the sort does not take goes the other way: other types and shapes, no choices at all, no experts or too many, more
    # choices than its 32-bit positions hold)
    if (expert_ids.is_cuda and expert_ids.dtype == torch.int64 and expert_ids.dim() == 2 and expert_ids.shape[1] >= 1
            and 1 <= n_experts <= 1024 and expert_ids.numel() < (1 << 31) - 8192):
        rows, offsets, _ = ops.sort_by_expert(expert_ids, n_experts)
        offsets = offsets.tolist()
        if offsets[-1] != rows.numel():
            raise ValueError(f"expert ids must lie in [0, {n_experts})")
        return rows, offsets
    flat = expert_ids.reshape(-1)
    order = torch.argsort(flat, stable=True)
    counts = torch.bincount(flat, minlength=n_experts)
    offsets = torch.zeros(n_experts + 1, dtype=torch.int64, device=flat.device)
    offsets[1:] = torch.cumsum(counts, 0)
    return order // expert_ids.shape[1], offsets.tolist()


@dataclass
class Router:
    """The gate of an MoE block: weight (E, C), the rest as `ops.route_experts` takes it.  Calling it on tokens (T, C) gives
    (weights (T, top_k) fp32, ids (T, top_k) int64); the logits are fp32."""

    weight: torch.Tensor
    top_k: int
    score: str = "softmax"
    bias: Optional[torch.Tensor] = None
    n_group: int = 1
    topk_group: Optional[int] = None
    group_top: int = 2
    renormalize: bool = True
    scale: float = 1.0
    rows_per_call: int = 1 << 18  # tokens whose fp32 copies and logits are alive at a time

    @torch.no_grad()
    def __call__(self, x: torch.Tensor):
        w = self.weight.float().t()
        parts = [ops.route_experts(xs.float() @ w, self.top_k, score=self.score, bias=self.bias, n_group=self.n_group,
                                   topk_group=self.topk_group, group_top=self.group_top, renormalize=self.renormalize,
                                   scale=self.scale) for xs in x.split(self.rows_per_call)]
        if len(parts) == 1:
            return parts[0]
        return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])


@dataclass
class Int8Experts:
    """The SwiGLU experts of a block on 8-bit weights with a scale per output channel."""

    gate_up: torch.Tensor  # (E, 2 I, C) int8: the gate projection's rows, then the up projection's
    gate_up_scale: torch.Tensor  # (E, 2 I) fp32
    down: torch.Tensor  # (E, C, I) int8
    down_scale: torch.Tensor  # (E, C) fp32

    @classmethod
    def from_quantized(cls, experts) -> "Int8Experts":
        """`experts`: for every expert its (gate, up, down), each the (qweight, scale, zero) that
        `GPTQ(..., group_size=None).quantize(bits)` returned."""
        gu, gus, dn, dns = [], [], [], []
        for gate, up, down in experts:
            (g, gs), (u, us), (d, ds) = (quant_utils.int8_weight(*w) for w in (gate, up, down))
            if g.shape != u.shape or d.shape != g.shape[::-1]:
                raise ValueError("an expert's gate and up must be (I, C) and its down (C, I)")
            gu.append(torch.cat([g, u]))
            gus.append(torch.cat([gs, us]))
            dn.append(d)
            dns.append(ds)
        return cls(torch.stack(gu), torch.stack(gus), torch.stack(dn), torch.stack(dns))


# values of the experts' fp32 outputs that are alive at a time (16 GiB): more tokens than that go in equal parts, one after the
# other, with the same results.  A part of 74898 tokens of eight experts of 7168 reads its 11 GB of weights in a twentieth of
# the time it takes in all.
_OUTPUTS_AT_ONCE = 1 << 32


@torch.no_grad()
def experts_forward_int8(x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, experts: Int8Experts) -> torch.Tensor:
    """The expert part of a block's forward on its quantized weights:
    y[t] = sum_j weights[t, j] * down_e(silu(gate_e(x[t])) * up_e(x[t])), e = ids[t, j].  x (T, C) fp32, bf16 or fp16; ids
    (T, top_k) int64 and weights (T, top_k) fp32 as a `Router` gives them (ids outside the experts add nothing).  Tokens and
    the product between the projections, held in x's type, are quantized to 8 bits with a scale per row; the experts' outputs
    are fp32 and rounded once, after their weighted sum (scratch memory for T * top_k * C values, at most 2^32 of them at a
    time).  Nothing is read back to the host."""
    if experts.gate_up.dim() != 3 or experts.down.dim() != 3:
        raise ValueError("gate_up must be (E, 2 I, C) and down (E, C, I)")
    E, C = experts.gate_up.shape[0], experts.gate_up.shape[2]
    if x.dim() != 2 or x.shape[1] != C or ids.shape != weights.shape or ids.dim() != 2 or ids.shape[0] != x.shape[0]:
        raise ValueError("x must be (T, C) with the experts' C, ids and weights (T, top_k)")
    if experts.gate_up.shape[1] % 2 or experts.down.shape != (E, C, experts.gate_up.shape[1] // 2):
        raise ValueError("gate_up must be (E, 2 I, C) and down (E, C, I)")
    T = x.shape[0]
    parts = -(-T // max(1, _OUTPUTS_AT_ONCE // max(1, ids.shape[1] * C)))
    if parts > 1:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
        step = -(-T // parts)
        for t in range(0, T, step):
            part = slice(t, t + step)
            out[part] = experts_forward_int8(x[part], ids[part], weights[part], experts)
        return out
    rows, offsets, slots = ops.sort_by_expert(ids, E)
    codes, scale = ops.quantize_tokens(x)
    h = ops.matmul_int8_grouped(codes, scale, experts.gate_up, experts.gate_up_scale, offsets, rows, x.dtype, swiglu=True)
    codes, scale = ops.quantize_tokens(h)
    y = ops.matmul_int8_grouped(codes, scale, experts.down, experts.down_scale, offsets, None, torch.float32)
    return ops.combine_experts(y, slots, weights, x.dtype)


@torch.no_grad()
def quantize_moe_layer(
    x: torch.Tensor,
    expert_ids: Union[torch.Tensor, Router],
    experts: List[ExpertWeights],
    bits: int = 4,
    group_size: int = 128,
    rel_damp: float = 0.01,
    block_size: int = 128,
    keep_outputs: bool = False,
    keep_codes: Optional[List[int]] = None,
    max_rows_per_update: int = 1 << 17,
    streams: int = 2,
    group: int = 8,
    overlap: bool = True,
) -> LayerResult:
    """x (T, C) bf16 on the GPU, expert_ids (T, top_k) int64 on the GPU, or the block's `Router`, which then chooses.

    `group`, `streams`: one linear is a long chain of dependent launches whose critical path (one-workgroup
    diagonal blocks, 64-row column walks) leaves most of the GPU idle.  Experts are therefore quantized `group` at a
    time -- their factorisations and column loops run as grouped library calls, every launch carrying the work of
    all of them -- and the groups go round-robin onto `streams` HIP streams, so that the short per-linear kernels
    of one group overlap the long launches of another.  Nothing in the path reads a value back to the host, so one
    host thread keeps all streams fed.
    `overlap`: quantize a group as soon as its Hessians are complete, beside the collection of the next group's
    (False: the reference's order, every Hessian of the block first)."""
    dev = x.device
    E = len(experts)
    keep_codes = set(keep_codes or [])
    res = LayerResult()
    sync = lambda: torch.cuda.synchronize(dev)

    def linear(w):
        m = nn.Linear(w.shape[1], w.shape[0], bias=False, dtype=w.dtype, device=dev)
        m.weight.data = w
        return m

    handles = []
    for ew in experts:
        g = GPTQ(linear(ew.gate), group_size, True, rel_damp, block_size)
        u = GPTQ(linear(ew.up), group_size, True, rel_damp, block_size, tied_gptq_handle=g)
        d = GPTQ(linear(ew.down), group_size, True, rel_damp, block_size)
        handles.append((g, u, d))

    sync()
    t0 = time.perf_counter()
    if isinstance(expert_ids, Router):
        expert_ids = expert_ids(x)[1]
    rows, offsets = route_tokens(expert_ids, E)
    sync()
    res.seconds["route"] = time.perf_counter() - t0
    res.tokens_per_expert = [offsets[e + 1] - offsets[e] for e in range(E)]
    main = torch.cuda.current_stream(dev)
    n_lanes = max(1, streams)
    # without overlap the current stream is lane 0; with overlap the Hessians keep the current stream to themselves
    lanes = ([] if overlap else [main]) + [torch.cuda.Stream(device=dev) for _ in range(n_lanes - (0 if overlap else 1))]
    done = []  # (name, handle): verdict words are read after everything is queued
    factor_calls_before = GPTQ.factor_calls
    group = max(1, group)

    # Hessian products wait here until `group` of one width have come together (or the same handle comes again: two
    # products into one H must not share a launch); then they run as one grouped library call.
    pending = {"gate_up": [], "down": []}

    def flush(kind):
        for want_packed in (True, False):
            part = [(h, p) for h, p in pending[kind] if isinstance(p, ops.PackedTokens) == want_packed]
            if part:
                GPTQ.update_many([h for h, _ in part], [p for _, p in part])
        pending[kind].clear()

    def enqueue(kind, h, tokens):
        if any(h is q for q, _ in pending[kind]):
            flush(kind)
        pending[kind].append((h, tokens))
        if len(pending[kind]) >= group:
            flush(kind)

    packable = x.dtype in (torch.bfloat16, torch.float16) and x.shape[1] % 8 == 0 and experts[0].gate.shape[0] % 8 == 0

    def collect_hessians(e):
        """Hessians of expert e (gate and up share one, quant.py:258-277) from its routed tokens: one pass gathers the
        expert's rows of x twice -- token-major for the two GEMMs of the expert's own forward (the model's matmuls,
        rocBLAS/hipBLASLt through torch) and in the packed layout the Hessian kernel reads -- and the SiLU product is
        written straight into that layout, its only reader being the down projection's Hessian."""
        g, u, d = handles[e]
        lo, hi = offsets[e], offsets[e + 1]
        for s in range(lo, hi, max_rows_per_update):
            idx = rows[s : min(hi, s + max_rows_per_update)]
            if packable and idx.numel() >= 256:
                P, xe = ops.pack_tokens(x, idx, also_token_major=True)
                enqueue("gate_up", g, P)
                A = ops.swiglu_packed(xe @ experts[e].gate.t(), xe @ experts[e].up.t())
                enqueue("down", d, A)
                a = ops.unpack_tokens(A) if e in keep_codes else None
            else:  # a handful of tokens: plain tensors
                xe = x.index_select(0, idx)
                enqueue("gate_up", g, xe)
                a = ops.swiglu(torch.cat([xe @ experts[e].gate.t(), xe @ experts[e].up.t()], dim=1))
                enqueue("down", d, a)
            if e in keep_codes:
                prev = res.down_inputs.get(e)
                res.down_inputs[e] = a if prev is None else torch.cat([prev, a])

    def hessians_done():
        flush("gate_up")
        flush("down")

    def quantize_chunk(chunk):
        """Quantize + pack the three linears of every expert of the chunk (on the current stream)."""
        for e in chunk:
            g, u, d = handles[e]
            if e in keep_codes:
                g.symmetrize_hessian()
                d.symmetrize_hessian()
                if g.H is not None:
                    res.hessians[f"{e}.gate_proj"] = g.H.clone()
                if d.H is not None:
                    res.hessians[f"{e}.down_proj"] = d.H.clone()
        # gate and up projections of the chunk (one factor per expert, shared), then the down projections
        gu = [handles[e][i] for e in chunk for i in (0, 1)]
        names = [(e, n) for e in chunk for n in ("gate_proj", "up_proj")] + [(e, "down_proj") for e in chunk]
        dn = [handles[e][2] for e in chunk]
        if group > 1:
            outs = GPTQ.quantize_many(gu, bits) + GPTQ.quantize_many(dn, bits)
        else:
            outs = [h.quantize(bits) for h in gu + dn]
        for (e, name), h, (q, s, z) in zip(names, gu + dn, outs):
            words = h.packed_words()
            done.append((f"{e}.{name}", h))
            if keep_outputs:
                res.packed[f"{e}.{name}"] = words
                res.scales[f"{e}.{name}"] = s
            if e in keep_codes:
                res.qweight[f"{e}.{name}"] = q
                res.scales[f"{e}.{name}"] = s
        for h in gu + dn:  # as quant.py:330: free per-linear state as soon as the linear is done
            h.H = None
            h._hessian_inv = h._loop_factor = None
            h._Qt = None
            h.W = h.layer.weight

    chunks = [list(range(e0, min(E, e0 + group))) for e0 in range(0, E, group)]
    t1 = time.perf_counter()
    ev0, ev1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    ev0.record(main)
    if overlap:
        # The Hessians of a chunk of experts are collected on the current stream; as soon as they are complete the
        # chunk is quantized on a lane of its own while the next chunk's Hessians are collected.  Legal because the
        # expert forward reads the original weights whatever has been quantized meanwhile (this driver never writes
        # quantized weights back), which is all the reference's "collect everything first" order is there for.
        for ci, chunk in enumerate(chunks):
            for e in chunk:
                collect_hessians(e)
            hessians_done()
            ready = torch.cuda.Event()
            ready.record(main)
            lane = lanes[ci % len(lanes)]
            lane.wait_event(ready)
            with torch.cuda.stream(lane):
                quantize_chunk(chunk)
        ev1.record(main)
    else:
        # ---- phase 1: Hessians of the whole block, phase 2: quantize + pack, chunks round-robin over the lanes
        for chunk in chunks:
            for e in chunk:
                collect_hessians(e)
        hessians_done()
        ev1.record(main)
        sync()
        for s_ in lanes:
            if s_ is not main:
                s_.wait_stream(main)
        for ci, chunk in enumerate(chunks):
            with torch.cuda.stream(lanes[ci % len(lanes)]):
                quantize_chunk(chunk)
    for s_ in lanes:
        if s_ is not main:
            main.wait_stream(s_)
    sync()
    t_end = time.perf_counter()
    # time the Hessian work took on its stream (with overlap: while quantization ran beside it), and the rest of the wall
    res.seconds["hessians_incl_gather_and_forward"] = ev0.elapsed_time(ev1) / 1e3
    res.seconds["quantize_and_pack"] = (t_end - t1) - res.seconds["hessians_incl_gather_and_forward"]
    res.overlapped = bool(overlap)
    issues = {"zero_samples": 0, "nan_hessian": 0, "non_invertible": 0}
    for name, h in done:
        raised = [k for k, v in (("zero_samples", h.issue_zero_samples), ("nan_hessian", h.issue_nan_hessian),
                                 ("non_invertible", h.issue_non_invertible)) if v]
        for k in raised:
            issues[k] += 1
        if raised:
            res.issues_by_linear[name] = raised
    res.factorizations = GPTQ.factor_calls - factor_calls_before
    res.seconds["total"] = time.perf_counter() - t0
    res.issues = issues
    return res
