"""CPU oracle of the fused-MoE operator -- TEST INFRASTRUCTURE ONLY.

This module is the checker, never the product: only tests/, the smoke() of
__graft_entry__.py and the CPU-baseline leg of bench.py may import it. The
product path (kernelswift_b200) never calls it and has no CPU fallback.

It restates, in plain torch-CPU fp32 and numpy, the algorithm of the
reference operator kernels/track1-triton/fused_moe/base.py:
  route()            base.py:44-47  softmax(fp32) -> topk -> renormalise
  grouped_topk()     groupedtopk/base.py:31-72 (the grouped top-k routing
                     operator of the same suite)
  fused_experts()    base.py:50-76  replicate, per-expert SwiGLU MLP, weighted
                                    top-k sum (fp32 throughout)
  model_forward()    base.py:35-76
and the pieces the reference leaves implicit:
  moe_align()        the per-expert grouping of base.py:64-68 as the padded,
                     stable counting sort the kernels emit
  quant_*/dequant_*  W8A8 formats (absent from the reference; fp32-dequant
                     semantics), including the power-of-two (UE8M0) block
                     scales and their scale-factor image layout
  regroup_w13()      the gate/up row regrouping of the prepared w1

Parity pin: tests/golden/ holds outputs of the reference base.py itself
(generated by tests/golden/make_golden.py in a container where the reference
is importable); tests/test_oracle.py checks this oracle against them.
"""
from __future__ import annotations

import numpy as np
import torch

FP8_MAX = 448.0
INT8_MAX = 127.0


# ---------------------------------------------------------------------------
# Routing (base.py:44-47)
# ---------------------------------------------------------------------------

def route(router_logits: torch.Tensor, top_k: int, renormalize: bool = True):
    """Returns (topk_weights fp32 [T, k], topk_ids int64 [T, k])."""
    scores = torch.softmax(router_logits.float().cpu(), dim=-1)
    w, ids = torch.topk(scores, top_k, dim=-1)
    if renormalize:
        w = w / w.sum(-1, keepdim=True)
    return w, ids


def grouped_topk(gating_output: torch.Tensor, topk: int, renormalize: bool,
                 num_expert_group: int, topk_group: int, scoring_func: str = "softmax",
                 routed_scaling_factor: float = 1.0):
    """Grouped top-k routing, restating kernels/track1-triton/groupedtopk/
    base.py:31-72 op for op on the CPU: scores (softmax or sigmoid), group
    score = max score in the group, top `topk_group` groups, experts of the
    other groups masked to -inf, top-k, optional renormalisation, scaling.
    Returns (weights fp32 [T, k], ids int32 [T, k])."""
    logits = gating_output.cpu()
    if scoring_func == "softmax":
        scores = torch.softmax(logits, dim=-1)
    elif scoring_func == "sigmoid":
        scores = logits.sigmoid()
    else:
        raise ValueError(f"Unsupported scoring_func: {scoring_func}")
    T, E = scores.shape
    group_scores = scores.view(T, num_expert_group, -1).max(dim=-1).values
    group_idx = torch.topk(group_scores, k=topk_group, dim=-1)[1]
    group_mask = torch.zeros_like(group_scores)
    group_mask.scatter_(1, group_idx, 1)
    score_mask = group_mask.unsqueeze(-1).expand(T, num_expert_group,
                                                 E // num_expert_group).reshape(T, -1)
    masked = scores.masked_fill(~score_mask.bool(), float("-inf"))
    w, ids = torch.topk(masked, k=topk, dim=-1)
    if renormalize:
        w = w / w.sum(dim=-1, keepdim=True)
    if routed_scaling_factor != 1.0:
        w = w * routed_scaling_factor
    return w.to(torch.float32), ids.to(torch.int32)


# ---------------------------------------------------------------------------
# moe_align_block_size (canonical specification)
# ---------------------------------------------------------------------------

def balanced_topk(logits, bias, topk: int, renormalize: bool = True, num_expert_group: int = 1,
                  topk_group: int = 1, scoring_func: str = "sigmoid", group_score: str = "top2",
                  scale: float = 1.0):
    """Routing by score plus bias, in fp64, row by row: the experts of the
    best groups in descending order of c = score + bias, ties to the lower
    index; weights from the unbiased scores (0 when the chosen ones vanish).
    Returns (weights fp64 [T, k], ids int64 [T, k])."""
    l = logits.double()
    T, E = l.shape
    per = E // num_expert_group
    if scoring_func == "sigmoid":
        s = torch.sigmoid(l)
    else:
        s = torch.softmax(l, dim=-1)
        s = torch.where((l == -torch.inf).all(1, keepdim=True), torch.zeros_like(s), s)
    c = s if bias is None else s + bias.double()
    c = torch.where(c.isnan(), torch.full_like(c, -torch.inf), c)
    ids = torch.empty(T, topk, dtype=torch.int64)
    for t in range(T):
        row = c[t].tolist()
        values = []
        for g in range(num_expert_group):
            best = sorted(row[g * per:(g + 1) * per], reverse=True)
            v = sum(best[:2]) if group_score == "top2" else best[0]
            values.append(v if v == v else -float("inf"))
        kept = sorted(range(num_expert_group), key=lambda g: (-values[g], g))[:topk_group]
        pool = [e for e in range(E) if e // per in kept]
        ids[t] = torch.tensor(sorted(pool, key=lambda e: (-row[e], e))[:topk])
    w = s.gather(1, ids)
    if renormalize:
        total = w.sum(-1, keepdim=True)
        w = torch.where(total == 0, torch.zeros_like(w), w / total)
    return w * scale, ids


def align_buffer_len(numel: int, num_experts: int, block_m: int) -> int:
    n = numel + num_experts * (block_m - 1)
    return -(-n // block_m) * block_m


def moe_align(topk_ids, num_experts: int, block_m: int):
    """Stable counting sort of the flat ids by expert, padded to block_m.

    Returns numpy (sorted_ids int32 [L], expert_ids int32 [L/block_m],
    num_post_pad int). sorted_ids lists, per expert in ascending order, the
    flat indices r with ids[r] == e in ascending r (the row order of
    base.py:68 `x_rep[mask]`), then padding slots = numel; expert_ids[b] is
    the expert of block b or -1 past the padded total; ids outside
    [0, num_experts) are dropped.
    """
    flat = np.asarray(topk_ids.reshape(-1).cpu() if isinstance(topk_ids, torch.Tensor)
                      else topk_ids).reshape(-1).astype(np.int64)
    numel = flat.size
    L = align_buffer_len(numel, num_experts, block_m)
    sorted_ids = np.full(L, numel, dtype=np.int32)
    expert_ids = np.full(L // block_m, -1, dtype=np.int32)
    off = 0
    for e in range(num_experts):
        rows = np.nonzero(flat == e)[0]
        cnt = rows.size
        padded = -(-cnt // block_m) * block_m
        sorted_ids[off:off + cnt] = rows
        expert_ids[off // block_m:(off + padded) // block_m] = e
        off += padded
    return sorted_ids, expert_ids, off


# ---------------------------------------------------------------------------
# Expert computation (base.py:50-76), fp32
# ---------------------------------------------------------------------------

def fused_experts(hidden, w1, w2, topk_weights, topk_ids):
    """fp32 restatement of base.py:50-76.

    hidden [T, H], w1 [E, 2I, H] (gate rows first), w2 [E, H, I],
    topk_weights [T, k], topk_ids [T, k]; returns fp32 [T, H]. Slots whose id
    is outside [0, E) contribute nothing.
    """
    hidden = hidden.float().cpu()
    w1 = w1.float().cpu()
    w2 = w2.float().cpu()
    T, H = hidden.shape
    E = w1.shape[0]
    k = topk_ids.shape[1]
    flat_ids = topk_ids.reshape(-1).cpu()
    flat_w = topk_weights.reshape(-1).float().cpu()
    x_rep = hidden.unsqueeze(1).expand(-1, k, -1).reshape(-1, H)
    out = torch.zeros_like(x_rep)
    for e in range(E):
        mask = flat_ids == e
        if not bool(mask.any()):
            continue
        x_e = x_rep[mask]
        gate_up = x_e @ w1[e].T
        gate, up = gate_up.chunk(2, dim=-1)
        out[mask] = (torch.nn.functional.silu(gate) * up) @ w2[e].T
    out = out * flat_w.unsqueeze(-1)
    return out.view(T, k, H).sum(dim=1)


def model_forward(hidden, router_logits, w1, w2, top_k, renormalize=True):
    """Routing + experts (base.py:35-76) in fp32; returns (out, weights, ids)."""
    w, ids = route(router_logits, top_k, renormalize)
    return fused_experts(hidden, w1, w2, w, ids), w, ids


def model_forward_native(hidden, router_logits, w1, w2, top_k, renormalize=True):
    """base.py:35-76 step for step in hidden.dtype, including the per-call
    weight casts of base.py:60-61: the reference's own CPU path, used as the
    timed CPU baseline (not as a checker)."""
    T, H = hidden.shape
    dtype = hidden.dtype
    scores = torch.softmax(router_logits.float(), dim=-1)
    topk_weights, topk_ids = torch.topk(scores, top_k, dim=-1)
    if renormalize:
        topk_weights = topk_weights / topk_weights.sum(-1, keepdim=True)
    topk_weights = topk_weights.to(dtype)
    flat_ids = topk_ids.view(-1)
    flat_w = topk_weights.view(-1)
    x_rep = hidden.unsqueeze(1).expand(-1, top_k, -1).reshape(-1, H)
    w1c = w1.to(dtype)
    w2c = w2.to(dtype)
    out = torch.zeros_like(x_rep)
    for e in range(w1.shape[0]):
        mask = flat_ids == e
        if not bool(mask.any()):
            continue
        gate_up = x_rep[mask] @ w1c[e].T
        gate, up = gate_up.chunk(2, dim=-1)
        out[mask] = (torch.nn.functional.silu(gate) * up) @ w2c[e].T
    out = out * flat_w.unsqueeze(-1)
    return out.view(T, top_k, H).sum(dim=1)


# ---------------------------------------------------------------------------
# W8A8 formats
# ---------------------------------------------------------------------------

def _scale(absmax: torch.Tensor, qmax: float) -> torch.Tensor:
    s = absmax / qmax
    return torch.where(s > 0, s, torch.ones_like(s))


def quant_fp8_block(w: torch.Tensor, block: int = 128):
    """w [..., R, C] -> (e4m3 [..., R, C], fp32 scales [..., ceil(R/b), ceil(C/b)]).

    scale = absmax / 448 per block (1 for an all-zero block);
    q = e4m3_rn(clamp(w / scale, -448, 448)).
    """
    w = w.float().cpu()
    *lead, R, C = w.shape
    RB, CB = -(-R // block), -(-C // block)
    pad = torch.zeros(*lead, RB * block, CB * block)
    pad[..., :R, :C] = w
    blocks = pad.reshape(*lead, RB, block, CB, block)
    amax = blocks.abs().amax(dim=(-3, -1))
    scale = _scale(amax, FP8_MAX)
    s_full = scale.repeat_interleave(block, -2).repeat_interleave(block, -1)[..., :R, :C]
    q = torch.clamp(w / s_full, -FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return q, scale


def dequant_fp8_block(q: torch.Tensor, scale: torch.Tensor, block: int = 128):
    R, C = q.shape[-2:]
    s_full = scale.repeat_interleave(block, -2).repeat_interleave(block, -1)[..., :R, :C]
    return q.float() * s_full


def quant_fp8_group(x: torch.Tensor, group: int = 128):
    """Per-row, per-`group`-column e4m3 quantisation of activations [N, C]:
    scale = absmax / 448 (1 for an all-zero group), inv = 1 / scale,
    q = e4m3_rn(clamp(x * inv, -448, 448)) (multiplication by the reciprocal,
    as the activation quantisers of the GPU path do)."""
    x = x.float().cpu()
    N, C = x.shape
    G = -(-C // group)
    pad = torch.zeros(N, G * group)
    pad[:, :C] = x
    amax = pad.reshape(N, G, group).abs().amax(-1)
    scale = _scale(amax, FP8_MAX)
    inv = (1.0 / scale).repeat_interleave(group, -1)[:, :C]
    q = torch.clamp(x * inv, -FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return q, scale


def dequant_fp8_group(q, scale, group: int = 128):
    C = q.shape[-1]
    return q.float() * scale.repeat_interleave(group, -1)[:, :C]


def quant_int8_rows(w: torch.Tensor, reciprocal: bool = False):
    """Per-row int8: scale = absmax / 127 (1 if zero), q = rint(clamp(w/scale)).
    `reciprocal=True` restates the activation quantiser, which multiplies by
    1 / scale instead of dividing (weights are quantised by division)."""
    w = w.float().cpu()
    amax = w.abs().amax(-1, keepdim=True)
    scale = _scale(amax, INT8_MAX)
    y = w * (1.0 / scale) if reciprocal else w / scale
    q = torch.round(torch.clamp(y, -INT8_MAX, INT8_MAX)).to(torch.int8)
    return q, scale.squeeze(-1)


def dequant_int8_rows(q, scale):
    return q.float() * scale.unsqueeze(-1)


def fused_experts_fp8(hidden, w1, w2, topk_weights, topk_ids, block: int = 128):
    """fp32 oracle of the fp8 W8A8 path: weights quantised per 128x128 block
    and dequantised, activations quantised per token per 128 columns and
    dequantised, then the fp32 expert computation."""
    q1, s1 = quant_fp8_block(w1, block)
    q2, s2 = quant_fp8_block(w2, block)
    xq, xs = quant_fp8_group(hidden, block)
    return fused_experts(dequant_fp8_group(xq, xs, block), dequant_fp8_block(q1, s1, block),
                         dequant_fp8_block(q2, s2, block), topk_weights, topk_ids)


def fused_experts_int8(hidden, w1, w2, topk_weights, topk_ids):
    """fp32 oracle of the int8 W8A8 path: per-output-channel weight scales,
    per-token activation scales, dequantised before the fp32 computation."""
    q1, s1 = quant_int8_rows(w1)
    q2, s2 = quant_int8_rows(w2)
    xq, xs = quant_int8_rows(hidden, reciprocal=True)
    return fused_experts(dequant_int8_rows(xq, xs), dequant_int8_rows(q1, s1),
                         dequant_int8_rows(q2, s2), topk_weights, topk_ids)


# ---------------------------------------------------------------------------
# fp8 with power-of-two (UE8M0) block scales
# ---------------------------------------------------------------------------

def ue8m0_byte(amax: torch.Tensor) -> torch.Tensor:
    """Scale byte b (scale 2^(b - 127)) of groups with absolute maximum `amax`:
    the smallest b with amax <= 448 * 2^(b - 127), read off the fp32 encoding
    of amax (448 = 1.75 * 2^8: b = E - 8 if the significand is <= 1.75, else
    E - 7, E the biased exponent); 127 for all-zero groups, 0 for subnormal
    ones. Returns int64."""
    a = amax.float().contiguous()
    bits = a.view(torch.int32).long() & 0xFFFFFFFF
    e = (bits >> 23) & 0xFF
    b = (e - 8 + ((bits & 0x7FFFFF) > 0x600000).long()).clamp(0, 254)
    return torch.where(a > 0, b, torch.full_like(b, 127))


def ue8m0_value(b: torch.Tensor) -> torch.Tensor:
    """2^(b - 127) as fp32."""
    return torch.ldexp(torch.ones(b.shape), (b.long() - 127).to(torch.int32))


def quant_fp8_block_ue8m0(w: torch.Tensor, block: int = 128):
    """w [..., R, C] (R, C multiples of `block`) -> (e4m3 [..., R, C], scale
    bytes int64 [..., R/b, C/b]); q = e4m3_rn(w / 2^(b - 127)) (exact scaling)."""
    w = w.float().cpu()
    *lead, R, C = w.shape
    blocks = w.reshape(*lead, R // block, block, C // block, block)
    b = ue8m0_byte(blocks.abs().amax(dim=(-3, -1)))
    s_full = ue8m0_value(b).repeat_interleave(block, -2).repeat_interleave(block, -1)
    q = torch.clamp(w / s_full, -FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return q, b


def dequant_fp8_block_ue8m0(q: torch.Tensor, b: torch.Tensor, block: int = 128):
    s_full = ue8m0_value(b).repeat_interleave(block, -2).repeat_interleave(block, -1)
    return q.float() * s_full


def quant_fp8_group_ue8m0(x: torch.Tensor, group: int = 128):
    """Activations [N, C] (C a multiple of `group`): one scale byte per row per
    group; q = e4m3_rn(x * 2^(127 - b)). Returns (e4m3 [N, C], bytes [N, C/g])."""
    x = x.float().cpu()
    N, C = x.shape
    b = ue8m0_byte(x.reshape(N, C // group, group).abs().amax(-1))
    inv = ue8m0_value(254 - b).repeat_interleave(group, -1)  # 2^(127 - b)
    q = torch.clamp(x * inv, -FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return q, b


def dequant_fp8_group_ue8m0(q, b, group: int = 128):
    return q.float() * ue8m0_value(b).repeat_interleave(group, -1)


def sf_image_bytes(groups: int, rows: int, cols: int) -> int:
    """Size of a scale-factor image: one 512-byte chunk per 128 rows and 4
    column blocks of 128."""
    kb = -(-cols // 128)
    return groups * (-(-kb // 4)) * (-(-rows // 128)) * 512


def sf_image_offset(g, r, kb, q_blocks: int, row_slices: int):
    """Byte of the scale of row r, column block kb of matrix group g: chunk
    (g, kb // 4, r // 128) in [g][q][row slice] order; inside the chunk, 32
    rows of 16 bytes where row r % 32 holds four 4-byte cells, cell (r % 128)
    // 32 holding the bytes of column blocks 4q .. 4q + 3 (the tensor-memory
    copy puts cell c of chunk row l at lane l, column c)."""
    return (((g * q_blocks + kb // 4) * row_slices + r // 128) * 512 + 16 * (r % 32)
            + 4 * ((r % 128) // 32) + kb % 4)


def sf_image_encode(row_bytes: torch.Tensor) -> torch.Tensor:
    """Per-row scale bytes [G, R, KB] -> the uint8 image (unused bytes 0)."""
    G, R, KB = row_bytes.shape
    q_blocks, slices = -(-KB // 4), -(-R // 128)
    img = torch.zeros(sf_image_bytes(G, R, KB * 128), dtype=torch.uint8)
    g, r, k = torch.meshgrid(torch.arange(G), torch.arange(R), torch.arange(KB), indexing="ij")
    img[sf_image_offset(g, r, k, q_blocks, slices).reshape(-1)] = \
        row_bytes.reshape(-1).to(torch.uint8)
    return img


def sf_image_decode(img: torch.Tensor, G: int, R: int, KB: int) -> torch.Tensor:
    """The per-row scale bytes [G, R, KB] (int64) held by an image."""
    q_blocks, slices = -(-KB // 4), -(-R // 128)
    g, r, k = torch.meshgrid(torch.arange(G), torch.arange(R), torch.arange(KB), indexing="ij")
    return img.cpu()[sf_image_offset(g, r, k, q_blocks, slices)].long()


def fused_experts_fp8_ue8m0(hidden, w1, w2, topk_weights, topk_ids, block: int = 128):
    """fp32 oracle of the fp8 W8A8 path with power-of-two scales: weights per
    128x128 block, activations per token per 128 columns, dequantised, then
    the fp32 expert computation."""
    q1, b1 = quant_fp8_block_ue8m0(w1, block)
    q2, b2 = quant_fp8_block_ue8m0(w2, block)
    xq, xb = quant_fp8_group_ue8m0(hidden, block)
    return fused_experts(dequant_fp8_group_ue8m0(xq, xb, block),
                         dequant_fp8_block_ue8m0(q1, b1, block),
                         dequant_fp8_block_ue8m0(q2, b2, block), topk_weights, topk_ids)


# ---------------------------------------------------------------------------
# Prepared-weight layout
# ---------------------------------------------------------------------------

def regroup_w13(w1: torch.Tensor) -> torch.Tensor:
    """w1 [E, 2I, H] -> rows regrouped as 16 gate rows, then the 16 matching
    up rows, per 32-row slice (the layout moe_prepare_w13 writes)."""
    E, two_i, H = w1.shape
    inter = two_i // 2
    gate = w1[:, :inter].reshape(E, inter // 16, 16, H)
    up = w1[:, inter:].reshape(E, inter // 16, 16, H)
    return torch.cat([gate, up], dim=2).reshape(E, two_i, H)


def regroup_rows_vec(v: torch.Tensor) -> torch.Tensor:
    """Per-row vector [E, 2I] regrouped like regroup_w13."""
    E, two_i = v.shape
    inter = two_i // 2
    gate = v[:, :inter].reshape(E, inter // 16, 16)
    up = v[:, inter:].reshape(E, inter // 16, 16)
    return torch.cat([gate, up], dim=2).reshape(E, two_i)


def rel_l2(a: torch.Tensor, b: torch.Tensor) -> float:
    a = a.float().cpu()
    b = b.float().cpu()
    return float((a - b).norm() / b.norm().clamp_min(1e-30))


# ---------------------------------------------------------------------------
# Dense block-scaled fp8 (fp64 restatement)
# ---------------------------------------------------------------------------

def e4m3_nearest(v: torch.Tensor) -> torch.Tensor:
    """v (fp64) to the nearest e4m3 value, halves to even, saturating at 448."""
    e = torch.frexp(v.abs().clamp_min(2.0 ** -6)).exponent - 4
    q = torch.ldexp(torch.round(torch.ldexp(v, -e)), e)
    return torch.where(v.isnan(), v, q.clamp(-FP8_MAX, FP8_MAX))


def _fp8_group(part: torch.Tensor, m: torch.Tensor, fmt: str):
    """(q, scale), both fp64, of a group with absolute maximum m."""
    s = torch.where(m > 0, m / FP8_MAX, torch.ones_like(m))
    if fmt == "fp32":
        return e4m3_nearest(part * FP8_MAX / torch.where(m > 0, m, torch.full_like(m, FP8_MAX))), s
    frac, exp = torch.frexp(s)  # s = frac * 2^exp, 0.5 <= frac < 1
    s = torch.ldexp(torch.ones_like(s), torch.where(frac == 0.5, exp - 1, exp))
    return e4m3_nearest(part / s), s


def fp8_rows(x: torch.Tensor, fmt: str):
    """Per row and 128 columns: (q fp64 [T, K], scale fp64 [T, KB])."""
    got = [_fp8_group(p, p.abs().amax(1, keepdim=True), fmt) for p in x.double().split(128, 1)]
    return torch.cat([q for q, _ in got], 1), torch.cat([s for _, s in got], 1)


def fp8_blocks(w: torch.Tensor, fmt: str):
    """Per 128x128 block: (q fp64 [N, K], scale fp64 [NB, KB])."""
    qs, ss = [], []
    for band in w.double().split(128, 0):
        got = [_fp8_group(p, p.abs().max().view(1, 1), fmt) for p in band.split(128, 1)]
        qs.append(torch.cat([q for q, _ in got], 1))
        ss.append(torch.cat([s for _, s in got], 1))
    return torch.cat(qs), torch.cat(ss)


def fp8_scale_values(scale: torch.Tensor) -> torch.Tensor:
    """Stored scales (float32, or UE8M0 bytes) as fp64 numbers."""
    if scale.dtype == torch.uint8:
        return torch.ldexp(torch.ones(scale.shape, dtype=torch.float64), scale.int() - 127)
    return scale.double()


def fp8_dense(x, xs, w, ws):
    """(product fp64 [T, N], sum of the terms' magnitudes [T, N]) of
    block-scaled e4m3 operands with stored scales."""
    (T, K), N = x.shape, w.shape[0]
    a = x.double() * fp8_scale_values(xs).repeat_interleave(128, 1)[:, :K]
    b = w.double() * (fp8_scale_values(ws).repeat_interleave(128, 0)[:N]
                      .repeat_interleave(128, 1)[:, :K])
    return a @ b.t(), a.abs() @ b.abs().t()
