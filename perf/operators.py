"""Cases of the operators around the routed experts: balanced routing, the fp8
quantisers, the block-scaled fp8 product and the shared expert's MLP.

`run` computes a case in plain torch operations, or, where `own` is true,
through the framework's own entry points. `exact` computes it again in 64
bits from the definitions.
"""
import math

import torch

own = False

BLOCK = 128
FP8_MAX = 448.0
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one decode step's routing, 256 experts in 8 groups, sigmoid scores: latency
        route("route one token", 1, 256, 8, 8, 4, "sigmoid", "top2", "f32", False),
        # a prefill chunk through the same router
        route("route prefill", 8192, 256, 8, 8, 4, "sigmoid", "top2", "f32", False),
        # a training step of a 128-expert softmax router with load counts and its backward pass
        route("route train", 4096, 128, 8, 1, 1, "softmax", "max", "bf16", True),
        # the activations of a prefill chunk before the gate-up product
        quant("quantise prefill", 4096, 7168, "bf16", "ue8m0", False),
        # silu(gate) * up of a prefill chunk before the down product
        quant("quantise gated", 4096, 2048, "bf16", "fp32", True),
        # a small ragged batch whose last block of columns is partial
        quant("quantise ragged", 83, 1000, "f16", "fp32", False),
        # one decode token against the shared expert's gate-up weights: the weight stream
        product("product one token", 1, 4096, 7168, "bf16", "ue8m0", False),
        # a ragged mid-sized batch: no size a multiple of a tile, added to another result
        product("product ragged", 333, 1500, 1000, "f16", "fp32", True),
        # a prefill chunk against weights of a checkpoint with fp32 block scales
        product("product prefill", 4096, 4096, 7168, "bf16", "fp32", False),
        # the largest: a long prefill with power-of-two scales
        product("product long prefill", 16384, 4096, 7168, "bf16", "ue8m0", False),
        # the shared expert of a decode batch, added to the routed experts' rows
        mlp("mlp decode", 16, 7168, 2048, "fp32"),
        # the shared expert of a prefill chunk
        mlp("mlp prefill", 2048, 7168, 2048, "ue8m0"),
    ]


def route(name, T, E, k, groups, kept, score, group_score, dtype, train):
    return dict(name=name, op="route", T=T, E=E, k=k, groups=groups, kept=kept, score=score,
                group_score=group_score, dtype=dtype, train=train)


def quant(name, T, K, dtype, fmt, gated):
    return dict(name=name, op="quant", T=T, K=K, dtype=dtype, fmt=fmt, gated=gated)


def product(name, T, N, K, dtype, fmt, add):
    return dict(name=name, op="product", T=T, N=N, K=K, dtype=dtype, fmt=fmt, add=add)


def mlp(name, T, H, I, fmt):
    return dict(name=name, op="mlp", T=T, H=H, I=I, dtype="bf16", fmt=fmt)


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], evenly over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["route", "quant", "product", "product", "mlp"])
    fmt = rng.choice(["fp32", "ue8m0"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        per = rng.randint(2, 64 if groups > 1 else 384)
        kept = rng.randint(1, groups)
        case = route("", _spread(rng, 1, 16384), groups * per, rng.randint(1, min(16, kept * per)),
                     groups, kept, rng.choice(["sigmoid", "softmax"]), rng.choice(["top2", "max"]),
                     rng.choice(["f32", "bf16", "f16"]), rng.random() < 0.5)
    elif op == "quant":
        case = quant("", _spread(rng, 1, 8192), _spread(rng, 64, 8192),
                     rng.choice(["f32", "bf16", "f16"]), fmt, rng.random() < 0.5)
    elif op == "product":
        case = product("", _spread(rng, 1, 8192), _spread(rng, 32, 8192), _spread(rng, 64, 7168),
                       rng.choice(["bf16", "f16"]), fmt, rng.random() < 0.5)
    else:
        case = mlp("", _spread(rng, 1, 4096), 16 * _spread(rng, 8, 448),
                   16 * _spread(rng, 8, 128), fmt)
    del case["name"]
    return case


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _scaled(x, m, fmt):
    """(x / s rounded to e4m3, scale as stored) for groups of x with absolute
    maxima m (of x's shape but for its sizes of 1): q is nearest to
    x * 448 / m and s = m / 448 in 32 bits, or s is the least power of two
    with m / s <= 448, stored as a byte b, s = 2^(b - 127)."""
    m = torch.where(m > 0, m, FP8_MAX * torch.ones_like(m))
    if fmt == "fp32":
        q, scale = x * FP8_MAX / m, (m / FP8_MAX).float()
    else:
        frac, exp = torch.frexp(m)  # m = frac * 2^exp, 448 = 0.875 * 2^9
        power = exp - 9 + (frac > 0.875).int()
        q, scale = torch.ldexp(x, -power), (power + 127).to(torch.uint8)
    return q.clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn), scale


def _values(scale):
    """The scales as fp32 numbers, whichever way they are stored."""
    if scale.dtype == torch.uint8:
        return torch.ldexp(torch.ones(scale.shape, device=scale.device), scale.int() - 127)
    return scale


def _groups(x):
    T, K = x.shape
    return torch.nn.functional.pad(x, (0, -K % BLOCK)).view(T, -1, BLOCK)


def _quantise(x, fmt, most=None):
    """(e4m3 [T, K], scale [T, ceil(K / 128)]) of x [T, K]; `most` [T, ceil(K / 128), 1]
    are the groups' absolute maxima where x does not give them exactly enough."""
    groups = _groups(x)
    q, scale = _scaled(groups, groups.abs().amax(-1, keepdim=True) if most is None else most, fmt)
    return q.flatten(1)[:, :x.shape[1]], scale[..., 0]


def _pitched(q, scale):
    """Operands as the framework's quantiser leaves them: rows start on
    16-byte boundaries, fp32 scales lie token by token, scale bytes in rows
    of a multiple of 4."""
    T, K = q.shape
    rows = torch.zeros(T, -(-K // 16) * 16, dtype=torch.uint8, device=q.device)
    rows[:, :K] = q.view(torch.uint8)
    if scale.dtype == torch.uint8:
        keep = torch.zeros(T, -(-scale.shape[1] // 4) * 4, dtype=torch.uint8, device=q.device)
        keep[:, :scale.shape[1]] = scale
        scale = keep[:, :scale.shape[1]]
    else:
        keep = torch.zeros(scale.shape[1], -(-T // 4) * 4, device=q.device)
        keep[:, :T] = scale.t()
        scale = keep[:, :T].t()
    return rows[:, :K].view(torch.float8_e4m3fn), scale


def _weight(N, K, fmt, gen, dev):
    """e4m3 weights [N, K] ~ N(0, 1/K) with a scale for each 128x128 block."""
    w = torch.randn(N, K, generator=gen, device=dev) / math.sqrt(K)
    nb, kb = -(-N // BLOCK), -(-K // BLOCK)
    padded = torch.nn.functional.pad(w, (0, kb * BLOCK - K, 0, nb * BLOCK - N))
    blocks = padded.view(nb, BLOCK, kb, BLOCK)
    q, scale = _scaled(blocks, blocks.abs().amax((1, 3), keepdim=True), fmt)
    q = q.reshape(nb * BLOCK, kb * BLOCK)[:N, :K]
    rows = torch.zeros(N, -(-K // 16) * 16, dtype=torch.uint8, device=dev)
    rows[:, :K] = q.view(torch.uint8)
    return rows[:, :K].view(torch.float8_e4m3fn), scale[:, 0, :, 0]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    state = {"case": case}
    T = case["T"]
    if case["op"] == "route":
        E = case["E"]
        # logits ~ N(0, 1), skewed by expert; a learnt bias works against the skew
        skew = 0.5 * torch.randn(E, generator=gen, device=dev)
        state["logits"] = (torch.randn(T, E, generator=gen, device=dev) + skew).to(dtype)
        spread = 0.1 if case["score"] == "sigmoid" else 0.5 / E
        state["bias"] = spread * torch.randn(E, generator=gen, device=dev) - 0.1 * spread * skew
        if case["train"]:
            state["logits"].requires_grad_()
            state["grad"] = torch.randn(T, case["k"], generator=gen, device=dev)
    elif case["op"] == "quant":
        wide = case["K"] * (2 if case["gated"] else 1)
        # rows of different magnitudes, as activations have them
        size = torch.exp(torch.randn(T, 1, generator=gen, device=dev))
        state["x"] = (size * torch.randn(T, wide, generator=gen, device=dev)).to(dtype)
    elif case["op"] == "product":
        x = torch.randn(T, case["K"], generator=gen, device=dev)
        state["x"] = _pitched(*_quantise(x, case["fmt"]))
        state["w"] = _weight(case["N"], case["K"], case["fmt"], gen, dev)
        state["add"] = None
        if case["add"]:
            state["add"] = torch.randn(T, case["N"], generator=gen, device=dev).to(dtype)
    else:
        H, I = case["H"], case["I"]
        state["x"] = torch.randn(T, H, generator=gen, device=dev).to(dtype)
        state["w13"] = _weight(2 * I, H, case["fmt"], gen, dev)
        state["w2"] = _weight(H, I, case["fmt"], gen, dev)
        state["add"] = torch.randn(T, H, generator=gen, device=dev).to(dtype)
    return state


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def run(state):
    case = state["case"]
    return (_own if own else _plain)[case["op"]](case, state)


def _own_route(case, s):
    from kernelswift_b200 import fused_moe as fm
    load = None
    if case["train"]:
        load = torch.zeros(case["E"], dtype=torch.int32, device=s["logits"].device)
    w, ids = fm.balanced_topk(s["logits"], s["logits"], s["bias"], case["k"], renormalize=True,
                              num_expert_group=case["groups"], topk_group=case["kept"],
                              scoring_func=case["score"], group_score=case["group_score"],
                              routed_scaling_factor=2.5, expert_load=load)
    if not case["train"]:
        return w, ids
    grad, = torch.autograd.grad(w, s["logits"], s["grad"])
    return w.detach(), ids, load, grad


def _own_quant(case, s):
    from kernelswift_b200 import fp8
    return fp8.quantize_rows(s["x"], scale_format=case["fmt"], gated=case["gated"])


def _own_product(case, s):
    from kernelswift_b200 import fp8
    return fp8.block_matmul(*s["x"], *s["w"], out_dtype=DTYPES[case["dtype"]], addend=s["add"])


def _own_mlp(case, s):
    from kernelswift_b200 import fp8
    return fp8.swiglu_mlp(s["x"], *s["w13"], *s["w2"], addend=s["add"])


def _choose(c, case):
    """The chosen experts' indices [T, k] by the biased scores c [T, E]."""
    T, E = c.shape
    G = case["groups"]
    if G > 1:
        best = c.view(T, G, E // G).sort(dim=-1, descending=True).values
        top = best[..., :2].sum(-1) if case["group_score"] == "top2" else best[..., 0]
        kept = top.sort(dim=-1, descending=True, stable=True).indices[:, :case["kept"]]
        mask = torch.ones(T, G, dtype=torch.bool, device=c.device).scatter_(1, kept, False)
        c = c.masked_fill(mask.repeat_interleave(E // G, 1), -math.inf)
    return c.sort(dim=-1, descending=True, stable=True).indices[:, :case["k"]]


def _plain_route(case, s):
    # in 64 bits: two experts whose scores nearly tie have to come out in their true order
    logits = s["logits"].detach().double()
    scores = torch.sigmoid(logits) if case["score"] == "sigmoid" else torch.softmax(logits, -1)
    ids = _choose(scores + s["bias"].double(), case)
    chosen = scores.gather(1, ids)
    total = chosen.sum(-1, keepdim=True)
    w = 2.5 * chosen / total
    if not case["train"]:
        return w.float(), ids.int()
    g = 2.5 * s["grad"].double()
    ds = (g - (g * chosen).sum(-1, keepdim=True) / total) / total
    dense = torch.zeros_like(scores).scatter_(1, ids, ds)
    if case["score"] == "sigmoid":
        grad = dense * scores * (1 - scores)
    else:
        grad = scores * (dense - (ds * chosen).sum(-1, keepdim=True))
    load = torch.bincount(ids.reshape(-1), minlength=case["E"]).int()
    return w.float(), ids.int(), load, grad.to(s["logits"].dtype)


def _silu_up(both):
    gate, up = both.chunk(2, -1)
    return gate * torch.sigmoid(gate) * up


def _plain_quant(case, s):
    x = s["x"].float()
    if not case["gated"]:
        return _quantise(x, case["fmt"])
    # the maxima in 64 bits: one next to 448 times a power of two decides its group's scale
    most = _groups(_silu_up(s["x"].double())).abs().amax(-1, keepdim=True)
    return _quantise(_silu_up(x), case["fmt"], most if case["fmt"] == "ue8m0" else most.float())


def _product(x, xs, w, ws, add, dtype):
    N, K = w.shape
    a = x.float() * _values(xs).repeat_interleave(BLOCK, 1)[:, :K]
    b = _values(ws).repeat_interleave(BLOCK, 0)[:N].repeat_interleave(BLOCK, 1)[:, :K]
    out = a @ (w.float() * b).t()
    return (out if add is None else out + add.float()).to(dtype)


def _plain_product(case, s):
    return _product(*s["x"], *s["w"], s["add"], DTYPES[case["dtype"]])


def _plain_mlp(case, s):
    dtype = s["x"].dtype
    both = _product(*_quantise(s["x"].float(), case["fmt"]), *s["w13"], None, dtype).float()
    return _product(*_quantise(_silu_up(both), case["fmt"]), *s["w2"], s["add"], dtype)


_own = {"route": _own_route, "quant": _own_quant, "product": _own_product, "mlp": _own_mlp}
_plain = {"route": _plain_route, "quant": _plain_quant, "product": _plain_product,
          "mlp": _plain_mlp}


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    T, b = case["T"], SIZES[case["dtype"]]
    per = 4 if case.get("fmt") == "fp32" else 1  # bytes of a scale

    def blocks(n):
        return -(-n // BLOCK)

    if case["op"] == "route":
        E, k = case["E"], case["k"]
        bytes_ = T * E * b + E * 4 + T * k * 8
        flops = T * E * 8
        if case["train"]:
            bytes_ += T * k * 4 + T * E * b + E * 4  # the gradients of w in, of the logits out
            flops += T * E * 4
    elif case["op"] == "quant":
        K, wide = case["K"], 2 if case["gated"] else 1
        bytes_ = T * K * b * wide + T * K + T * blocks(K) * per
        flops = T * K * (8 if case["gated"] else 3)
    elif case["op"] == "product":
        N, K = case["N"], case["K"]
        bytes_ = T * K + N * K + (T + blocks(N)) * blocks(K) * per
        bytes_ += T * N * b * (2 if case["add"] else 1)
        flops = 2 * T * N * K
    else:
        H, I = case["H"], case["I"]
        bytes_ = 3 * H * I + 3 * blocks(H) * blocks(I) * per + 3 * T * H * b
        flops = 6 * T * H * I
    return {"bytes": bytes_, "flops": flops}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def _power(v):
    """The exponent e of 2^e <= v < 2^(e + 1)."""
    return torch.frexp(v).exponent - 1


def _exact_e4m3(v):
    """v to the nearest e4m3 value, halves to even: 4 significant bits down to 2^-6."""
    e = _power(v.abs().clamp_min(2.0 ** -6)) - 3
    return torch.ldexp(torch.round(torch.ldexp(v, -e)), e)


def _exact_quantise(x, fmt):
    qs, scales = [], []
    for part in x.split(BLOCK, 1):
        m = part.abs().amax(1, keepdim=True)
        s = torch.where(m > 0, m / FP8_MAX, torch.ones_like(m))
        if fmt == "ue8m0":  # up to a power of two
            low = torch.ldexp(torch.ones_like(s), _power(s))
            s = torch.where(FP8_MAX * low >= m, low, 2 * low)
            qs.append(_exact_e4m3(part / s))
        else:
            qs.append(_exact_e4m3(part * FP8_MAX / torch.where(m > 0, m, FP8_MAX)))
        scales.append(s)
    return torch.cat(qs, 1), torch.cat(scales, 1)


def _exact_matrix(q, scale, rows):
    """The matrix that e4m3 values and scales (numbers) of `rows` x 128 blocks stand for."""
    out = q.double().clone()
    for i in range(scale.shape[0]) if rows > 1 else [slice(None)]:
        at = slice(i * rows, (i + 1) * rows) if rows > 1 else slice(None)
        for j in range(scale.shape[1]):
            s = scale[i, j] if rows > 1 else scale[:, j:j + 1]
            out[at, j * BLOCK:(j + 1) * BLOCK] *= s
    return out


def _exact_numbers(scale):
    return torch.exp2(scale.double() - 127) if scale.dtype == torch.uint8 else scale.double()


def _exact_silu(both):
    gate, up = both[:, :both.shape[1] // 2], both[:, both.shape[1] // 2:]
    return gate / (1 + torch.exp(-gate)) * up


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        l = s["logits"].detach().double()
        e = torch.exp(-l) if case["score"] == "sigmoid" else torch.exp(l)
        p = 1 / (1 + e) if case["score"] == "sigmoid" else e / e.sum(1, keepdim=True)
        # rank[t, e]: how many experts of the row come before e
        c = p + s["bias"].double()
        T, E = c.shape
        per = E // case["groups"]
        if case["groups"] > 1:
            top = c.view(T, case["groups"], per).topk(2 if case["group_score"] == "top2" else 1).values
            score = top.sum(-1)
            floor = score.topk(case["kept"]).values[:, -1:]
            c = torch.where((score >= floor).repeat_interleave(per, 1), c, -math.inf * torch.ones_like(c))
        ids = c.topk(case["k"]).indices
        mine = torch.gather(p, 1, ids)
        w = mine / mine.sum(1, keepdim=True) * 2.5
        if not case["train"]:
            return w, None
        leaf = l.clone().requires_grad_()
        q = torch.sigmoid(leaf) if case["score"] == "sigmoid" else torch.softmax(leaf, 1)
        got = q.gather(1, ids)
        (2.5 * got / got.sum(1, keepdim=True) * s["grad"].double()).sum().backward()
        return w, None, None, leaf.grad
    if case["op"] == "quant":
        x = s["x"].double()
        q, scale = _exact_quantise(_exact_silu(x) if case["gated"] else x, case["fmt"])
        return q, scale if case["fmt"] == "fp32" else None
    add = 0 if s["add"] is None else s["add"].double()
    if case["op"] == "product":
        (x, xs), (w, ws) = s["x"], s["w"]
        return _exact_matrix(x, _exact_numbers(xs), 1) @ _exact_matrix(w, _exact_numbers(ws), BLOCK).t() + add
    w13 = _exact_matrix(s["w13"][0], _exact_numbers(s["w13"][1]), BLOCK)
    w2 = _exact_matrix(s["w2"][0], _exact_numbers(s["w2"][1]), BLOCK)
    q, scale = _exact_quantise(s["x"].double(), case["fmt"])
    both = (_exact_matrix(q, scale, 1) @ w13.t()).to(s["x"].dtype).double()
    q, scale = _exact_quantise(_exact_silu(both), case["fmt"])
    return _exact_matrix(q, scale, 1) @ w2.t() + add
