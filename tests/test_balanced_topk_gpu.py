"""GPU: balanced routing (moe_balanced_topk and its backward) against the fp64
restatement of the oracle.

Weights: each is off by at most 2 ulp of an exponential, the roundings of a
sum of up to 1024 terms by lane and tree (37), of the logit's difference to
the maximum (|l - max| < 16 here) and of two divisions and a product, under
64 roundings of 2^-24 in all."""
import pytest
import torch

from kernelswift_b200 import fused_moe as fm
from oracle import moe_oracle as orc

pytestmark = pytest.mark.gpu

RTOL = 64 * 2.0 ** -24
STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}

SHAPES = [
    # T, E, k, groups, kept
    (1, 256, 8, 8, 4),
    (5, 1, 1, 1, 1),
    (33, 8, 2, 1, 1),
    (64, 40, 6, 5, 2),
    (77, 96, 32, 3, 2),
    (130, 128, 8, 1, 1),
    (9, 30, 3, 30, 7),    # groups of one expert
    (19, 32, 4, 32, 5),
    (50, 160, 6, 8, 3),   # experts per group not a power of two
    (21, 384, 8, 1, 1),
    (700, 64, 6, 4, 4),   # several tokens per block
    (13, 1000, 16, 20, 9),
    (7, 1024, 32, 2, 1),
]


def inputs(T, E, dtype, seed, spread=0.2):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(T, E, generator=g) * 1.5).to(dtype)
    return logits, spread * torch.randn(E, generator=g)


def check(logits, bias, w, ids, k, **kw):
    rw, rids = orc.balanced_topk(logits, bias, k, **kw)
    assert torch.equal(ids.cpu().long(), rids)
    torch.testing.assert_close(w.double().cpu(), rw, rtol=RTOL, atol=1e-30)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("T,E,k,G,kept", SHAPES)
def test_matches_fp64(cuda_device, T, E, k, G, kept, score):
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        logits, bias = inputs(T, E, dtype, T + E, 0.2 if score == "sigmoid" else 1.0 / E)
        for group_score, b, renorm in (("top2", bias, True), ("max", bias, False),
                                       ("top2", None, True)):
            kw = dict(renormalize=renorm, num_expert_group=G, topk_group=kept,
                      scoring_func=score, group_score=group_score)
            x = logits.to(cuda_device)
            w, ids = fm.balanced_topk(x, x, None if b is None else b.to(cuda_device), k,
                                      routed_scaling_factor=2.5, **kw)
            assert w.dtype == torch.float32 and ids.dtype == torch.int32
            check(logits, b, w, ids, k, scale=2.5, **kw)


@pytest.mark.parametrize("score,G,kept", [("sigmoid", 1, 1), ("softmax", 1, 1), ("sigmoid", 8, 3),
                                          ("softmax", 4, 2)])
def test_order_of_scores_that_32_bits_cannot_tell_apart(cuda_device, score, G, kept):
    """The bias moves every expert's score to the same number, up to the
    rounding of the bias: the order is that of differences near 2^-26."""
    T, E, k = 40, 128, 8
    g = torch.Generator().manual_seed(11)
    for t in range(4):
        row = torch.randn(1, E, generator=g)
        s = torch.sigmoid(row.double()) if score == "sigmoid" else torch.softmax(row.double(), -1)
        bias = (0.7 - s[0]).float()
        logits = row.repeat(T, 1)
        x = logits.to(cuda_device)
        kw = dict(num_expert_group=G, topk_group=kept, scoring_func=score)
        w, ids = fm.balanced_topk(x, x, bias.to(cuda_device), k, **kw)
        check(logits, bias, w, ids, k, **kw)


def test_true_ties_go_to_the_lower_index(cuda_device):
    x = torch.zeros(3, 64, device=cuda_device)
    x[1, 40] = 1.0
    x[2] = -50.0
    _, ids = fm.balanced_topk(x, x, None, 3)
    assert ids.tolist() == [[0, 1, 2], [40, 0, 1], [0, 1, 2]]
    _, ids = fm.balanced_topk(x, x, None, 3, num_expert_group=4, topk_group=2)
    assert ids.tolist() == [[0, 1, 2], [40, 0, 1], [0, 1, 2]]


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("G,kept", [(1, 1), (4, 2)])
def test_masked_experts_and_empty_rows(cuda_device, score, G, kept):
    """Logits of -inf and of the type's lowest value, biases of -inf, rows
    with nothing left: the ids stay valid, and as the definition says."""
    T, E, k = 6, 32, 4
    logits, bias = inputs(T, E, torch.float32, 3)
    logits[0, ::2] = -torch.inf
    logits[1] = -torch.inf
    logits[2, 1:] = torch.finfo(torch.float32).min
    logits[3, 5] = 60.0
    bias[7] = -torch.inf
    bias[9:30] = -torch.inf
    x = logits.to(cuda_device)
    for renorm in (True, False):
        kw = dict(renormalize=renorm, num_expert_group=G, topk_group=kept, scoring_func=score)
        w, ids = fm.balanced_topk(x, x, bias.to(cuda_device), k, **kw)
        rw, rids = orc.balanced_topk(logits, bias, k, **kw)
        assert torch.equal(ids.cpu().long(), rids)
        # scores below fp32's range vanish; a row of them has no weights
        rw = torch.where(rw < 1e-37, torch.zeros_like(rw), rw)
        got = torch.where(w.cpu().double() < 1e-37, torch.zeros_like(rw), w.cpu().double())
        far = (logits.gather(1, rids) < -87).all(1)  # chosen scores under 2^-126
        torch.testing.assert_close(got[~far], rw[~far], rtol=RTOL, atol=1e-30)
        assert torch.isfinite(w).all()


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("G,per,kept", [(8, 2, 4), (32, 2, 8), (16, 4, 5)])
def test_groups_of_opposite_biases(cuda_device, G, per, kept, score):
    """A group's two largest nearly cancel: their sum is far smaller than what
    each lost when its bias was added in 32 bits. Biases of 1e2 to 1e5, and
    ordinary ones against scores that are small themselves."""
    T, k = 2048, 4
    sign = torch.ones(G, per)
    sign[:, 1] = -1
    sign[:, 2:] = -2
    for size, mean in ((1e2, 0), (1e3, 0), (1e4, 0), (1e5, 0), (0.25, -16), (1.0, -16), (8.0, -12)):
        logits, _ = inputs(T, G * per, torch.float32, int(size) + G)
        logits += mean
        bias = (size * sign).reshape(-1)
        x = logits.to(cuda_device)
        kw = dict(num_expert_group=G, topk_group=kept, scoring_func=score)
        w, ids = fm.balanced_topk(x, x, bias.to(cuda_device), k, **kw)
        check(logits, bias, w, ids, k, **kw)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("G,per,kept", [(8, 2, 4), (32, 2, 12), (16, 3, 6)])
def test_groups_of_opposite_biases_among_others(cuda_device, G, per, kept, score):
    """Some groups' values are in doubt, their neighbours' in the order are not:
    a kept one in doubt need not be the last one kept."""
    T, k = 2048, 6
    for size, mean in ((1e3, 0), (1e4, 0), (117894.359375, 2), (0.25, -16), (8.0, -12)):
        g = torch.Generator().manual_seed(int(size) + G)
        logits = torch.randn(T, G * per, generator=g) * 0.05 + mean
        bias = size * torch.randint(-2, 3, (G, per), generator=g) / 2
        pinned = torch.arange(G) % 3 == 0
        bias[pinned, 0], bias[pinned, 1:] = size, -size
        bias[torch.arange(G) % 3 == 1] = 0
        bias = bias.reshape(-1)
        x = logits.to(cuda_device)
        kw = dict(num_expert_group=G, topk_group=kept, scoring_func=score)
        w, ids = fm.balanced_topk(x, x, bias.to(cuda_device), k, **kw)
        check(logits, bias, w, ids, k, **kw)


@pytest.mark.parametrize("G,kept", [(1, 1), (8, 3), (5, 2)])
def test_biases_of_the_lowest_value(cuda_device, G, kept):
    """Experts masked by the lowest value of fp32 or bf16, of which groups have
    one, two or only such: sums past 32 bits' range keep their 64-bit order."""
    T, E, k = 60, 40, 6
    logits, bias = inputs(T, E, torch.float32, 2)
    low, bf = torch.finfo(torch.float32).min, torch.finfo(torch.bfloat16).min
    for masked in ({0: low, 3: low, 4: low}, {e: low for e in range(0, 20)},
                   {e: (low, bf, -torch.inf)[e % 3] for e in range(2, 40)},
                   {e: (low, bf)[e // 5 % 2] for e in range(40)}):
        b = bias.clone()
        for e, v in masked.items():
            b[e] = v
        x = logits.to(cuda_device)
        for group_score in ("top2", "max"):
            kw = dict(num_expert_group=G, topk_group=kept, group_score=group_score)
            w, ids = fm.balanced_topk(x, x, b.to(cuda_device), k, **kw)
            check(logits, b, w, ids, k, **kw)


@pytest.mark.parametrize("G,kept", [(1, 1), (4, 2)])
def test_scores_below_the_normal_range(cuda_device, G, kept):
    """Logits whose sigmoids lie about 2^-126, with biases of that size: the
    fast 32-bit scores are 0 there, the order is still that of 64 bits."""
    T, E, k = 300, 64, 8
    g = torch.Generator().manual_seed(7)
    logits = -87.5 + 0.5 * torch.randn(T, E, generator=g)
    bias = 1e-38 * torch.randn(E, generator=g)
    x = logits.to(cuda_device)
    kw = dict(num_expert_group=G, topk_group=kept)
    _, ids = fm.balanced_topk(x, x, bias.to(cuda_device), k, **kw)
    assert torch.equal(ids.cpu().long(), orc.balanced_topk(logits, bias, k, **kw)[1])


def test_nan_ranks_last_and_ids_stay_valid(cuda_device):
    x = torch.randn(4, 16, device=cuda_device)
    x[0, 3] = torch.nan
    x[1] = torch.nan
    w, ids = fm.balanced_topk(x, x, None, 4)
    assert ((ids >= 0) & (ids < 16)).all() and 3 not in ids[0].tolist()
    assert ids[1].tolist() == [0, 1, 2, 3] and w[1].isnan().all()
    assert torch.isfinite(w[[0, 2, 3]]).all()
    w, ids = fm.balanced_topk(x, x, None, 4, scoring_func="softmax", renormalize=False)
    assert ((ids >= 0) & (ids < 16)).all() and w[:2].isnan().all()


def test_load_is_added_and_types_are_kept(cuda_device):
    T, E, k = 501, 48, 5
    logits, bias = inputs(T, E, torch.float32, 8)
    x = logits.to(cuda_device)
    load = torch.full((E,), 7, dtype=torch.int32, device=cuda_device)
    w, ids = fm.balanced_topk(x, x, bias.to(cuda_device), k, expert_load=load,
                              weights_dtype=torch.bfloat16, ids_dtype=torch.int64)
    assert w.dtype == torch.bfloat16 and ids.dtype == torch.int64
    rw, rids = orc.balanced_topk(logits, bias, k)
    assert torch.equal(ids.cpu(), rids)
    torch.testing.assert_close(w.double().cpu(), rw, rtol=2.0 ** -8 + RTOL, atol=0)
    assert torch.equal(load.cpu().long(), 7 + torch.bincount(rids.reshape(-1), minlength=E))


def test_no_tokens_and_views(cuda_device):
    x = torch.empty(0, 16, device=cuda_device)
    w, ids = fm.balanced_topk(x, x, None, 2)
    assert w.shape == (0, 2) and ids.shape == (0, 2)
    wide = torch.randn(20, 2 * 24, device=cuda_device)
    for view in (wide[:, 1:25], wide[::2, ::2], wide[:1, :24].expand(20, 24)):
        w, ids = fm.balanced_topk(view, view, None, 3)
        check(view.cpu(), None, w, ids, 3)


def formula(logits, bias, gw, k, score, renorm, scale, ids):
    """fp64 gradient by autograd through the definition, ids given."""
    leaf = logits.double().requires_grad_()
    s = torch.sigmoid(leaf) if score == "sigmoid" else torch.softmax(leaf, -1)
    w = s.gather(1, ids)
    if renorm:
        w = w / w.sum(-1, keepdim=True)
    (scale * w * gw.double()).sum().backward()
    return leaf.grad


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("T,E,k,G,kept", SHAPES)
def test_gradient(cuda_device, T, E, k, G, kept, score, renorm):
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        logits, bias = inputs(T, E, dtype, 3 * T + E, 0.2 if score == "sigmoid" else 1.0 / E)
        x = logits.to(cuda_device).requires_grad_()
        gw = torch.randn(T, k, generator=torch.Generator().manual_seed(1))
        w, ids = fm.balanced_topk(x, x, bias.to(cuda_device), k, renormalize=renorm,
                                  num_expert_group=G, topk_group=kept, scoring_func=score,
                                  routed_scaling_factor=1.5)
        assert w.requires_grad and not ids.requires_grad
        w.backward(gw.to(cuda_device))
        want = formula(logits, bias, gw, k, score, renorm, 1.5, ids.cpu().long())
        assert x.grad.dtype == dtype
        # g_j - mean and the sum over k cancel: the error goes by the row's
        # largest |g| times the largest score, not by each entry
        room = RTOL * 1.5 * gw.abs().amax(1, keepdim=True).double() * k
        err = (x.grad.double().cpu() - want).abs()
        # an fp16 entry below 2^-14 is subnormal: half a step of 2^-24
        tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
        assert (err <= room + STEP[dtype] * want.abs() + tiny).all()


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("T,E,k,G,kept", SHAPES)
def test_gradient_of_each_entry(cuda_device, T, E, k, G, kept, score, renorm):
    """Each entry to its own size. An entry is p_e (g_e - m) (times 1 - s_e for the
    sigmoid) with m = sum_i g_i p_i, p the scores or, renormalised, their shares,
    g_e = 0 for one not chosen, and no m for sigmoids that are not renormalised.
    p_e is off by RTOL of itself, m by RTOL sum_i |g_i p_i|; the difference, the
    products and 1 - s_e (under 8 roundings) fit in as much again."""
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        logits, bias = inputs(T, E, dtype, 5 * T + E, 0.2 if score == "sigmoid" else 1.0 / E)
        x = logits.to(cuda_device).requires_grad_()
        gw = torch.randn(T, k, generator=torch.Generator().manual_seed(3))
        w, ids = fm.balanced_topk(x, x, bias.to(cuda_device), k, renormalize=renorm,
                                  num_expert_group=G, topk_group=kept, scoring_func=score,
                                  routed_scaling_factor=1.5)
        w.backward(gw.to(cuda_device))
        ids = ids.cpu().long()
        want = formula(logits, bias, gw, k, score, renorm, 1.5, ids)
        l = logits.double()
        s = torch.sigmoid(l) if score == "sigmoid" else torch.softmax(l, -1)
        p = s / s.gather(1, ids).sum(1, keepdim=True) if renorm else s
        g = torch.zeros(T, E, dtype=torch.float64).scatter_(1, ids, 1.5 * gw.double())
        chosen = torch.zeros(T, E, dtype=torch.bool).scatter_(1, ids, True)
        m = (g * p).abs().sum(1, keepdim=True)
        if score == "sigmoid":
            p = p * (1 - s)
            m = m if renorm else torch.zeros_like(m)
        if renorm or score == "sigmoid":
            # 0 by the formula for one not chosen; autograd's two terms for it cancel
            # to 2^-53 of themselves
            p, want = (torch.where(chosen, v, torch.zeros_like(v)) for v in (p, want))
        room = 2 * RTOL * p * (g.abs() + m)
        err = (x.grad.double().cpu() - want).abs()
        # an fp16 entry below 2^-14 is subnormal: half a step of 2^-24
        tiny = 2.0 ** -25 * (p > 0) if dtype == torch.float16 else 0.0
        assert (err <= room + STEP[dtype] * want.abs() + tiny).all()


def test_gradient_against_differences(cuda_device):
    """(f(l + h) - f(l - h)) / 2h of the fp64 definition at fixed ids."""
    T, E, k = 3, 24, 4
    for score in ("sigmoid", "softmax"):
        for renorm in (True, False):
            logits, bias = inputs(T, E, torch.float32, 21)
            x = logits.to(cuda_device).requires_grad_()
            w, ids = fm.balanced_topk(x, x, bias.to(cuda_device), k, renormalize=renorm,
                                      scoring_func=score)
            gw = torch.linspace(-1, 2, T * k).view(T, k)
            (w * gw.to(cuda_device)).sum().backward()
            idx = ids.cpu().long()

            def f(l):
                s = torch.sigmoid(l) if score == "sigmoid" else torch.softmax(l, -1)
                v = s.gather(1, idx)
                v = v / v.sum(-1, keepdim=True) if renorm else v
                return (v * gw.double()).sum()

            h, base = 1e-5, logits.double()
            for t in range(T):
                for e in range(E):
                    d = torch.zeros(T, E, dtype=torch.float64)
                    d[t, e] = h
                    diff = (f(base + d) - f(base - d)) / (2 * h)
                    # differences: h^2 / 6 of a third derivative under 10, and
                    # 2^-53 / h of rounding; the kernel: as in test_gradient
                    assert abs(x.grad[t, e].item() - diff.item()) < 1e-9 + 8 * RTOL


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("renorm", [0, 1])
def test_gradient_of_ids_out_of_range(cuda_device, score, renorm):
    """Through the C entry: such an id contributes nothing, in either width.
    2^32 + 3 is 3 in its low 32 bits."""
    from kernelswift_b200 import _lib
    from kernelswift_b200.fused_moe import _ptr, _stream

    T, E, k = 5, 24, 4
    x, _ = inputs(T, E, torch.float32, 6)
    gw = torch.randn(T, k, generator=torch.Generator().manual_seed(2))
    good = torch.tensor([7, 11, 0, 23])
    for dtype, code, bad in ((torch.int64, _lib.DT_I64, (-1, E, 2 ** 32 + 3, -2 ** 32 + 3)),
                             (torch.int32, _lib.DT_I32, (-1, E, 2 ** 31 - 1, -2 ** 31))):
        for at, wrong in enumerate(bad):
            ids = good.repeat(T, 1)
            ids[1:, at] = wrong
            dev = [t.to(cuda_device) for t in (x, ids.to(dtype), gw)]
            grad = torch.full((T, E), 9.0, device=cuda_device)
            _lib.call("moe_balanced_topk_backward", _ptr(dev[0]), _lib.DT_F32, _ptr(dev[1]), code,
                      _ptr(dev[2]), T, E, k, renorm, score, 1.5, _ptr(grad), _stream(cuda_device))
            name = "sigmoid" if score else "softmax"
            rest = [j for j in range(k) if j != at]
            want = formula(x, None, gw[:, rest], k - 1, name, bool(renorm), 1.5, ids[:, rest])
            whole = formula(x, None, gw, k, name, bool(renorm), 1.5, good.repeat(T, 1))
            want[0] = whole[0]
            room = RTOL * 1.5 * gw.abs().amax(1, keepdim=True).double() * k
            assert ((grad.double().cpu() - want).abs() <= room).all(), wrong


def test_gradient_of_expanded_logits(cuda_device):
    row = torch.randn(1, 16, device=cuda_device, requires_grad=True)
    x = row.expand(6, 16)
    w, ids = fm.balanced_topk(x, x, None, 3, renormalize=False)
    w.sum().backward()
    want = formula(row.detach().cpu(), None, torch.full((1, 3), 6.0), 3, "sigmoid", False, 1.0,
                   ids[:1].cpu().long())
    # six equal terms: five more roundings
    torch.testing.assert_close(row.grad.double().cpu(), want, rtol=2 * RTOL, atol=1e-30)


def test_captured_and_on_another_stream(cuda_device):
    T, E, k = 16, 256, 8
    logits, bias = inputs(T, E, torch.float32, 5)
    b = bias.to(cuda_device)
    static = torch.zeros(T, E, device=cuda_device)
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        fm.balanced_topk(static, static, b, k, num_expert_group=8, topk_group=4)
        w, ids = fm.balanced_topk(logits.to(cuda_device), static, b, k)
    torch.cuda.current_stream(cuda_device).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w, ids = fm.balanced_topk(static, static, b, k, num_expert_group=8, topk_group=4)
    for seed in (1, 2):
        logits, _ = inputs(T, E, torch.float32, seed)
        static.copy_(logits)
        graph.replay()
        check(logits, bias, w, ids, k, num_expert_group=8, topk_group=4)


@pytest.mark.parametrize("E,G,kept", [(256, 8, 4), (384, 1, 1), (1024, 32, 9)])
def test_bias_off_alignment(cuda_device, E, G, kept):
    """A bias that is a slice of a larger tensor, strided or off a 16-byte boundary."""
    logits, bias = inputs(40, E, torch.float32, 11)
    x = logits.to(cuda_device)
    wide = torch.zeros(2 * E + 1, device=cuda_device)
    for view in (wide[1:E + 1], wide[1::2]):
        view.copy_(bias)
        w, ids = fm.balanced_topk(x, x, view, 8, num_expert_group=G, topk_group=kept)
        check(logits, bias, w, ids, 8, num_expert_group=G, topk_group=kept)


@pytest.mark.parametrize("score,renorm", [("sigmoid", True), ("softmax", False)])
def test_captured_training_step(cuda_device, score, renorm):
    T, E, k = 70, 64, 6
    logits, bias = inputs(T, E, torch.float32, 3)
    b = bias.to(cuda_device)
    x = torch.zeros(T, E, device=cuda_device, requires_grad=True)
    gw = torch.randn(T, k, generator=torch.Generator().manual_seed(1)).to(cuda_device)
    load = torch.zeros(E, dtype=torch.int32, device=cuda_device)

    def step():
        w, ids = fm.balanced_topk(x, x, b, k, renormalize=renorm, scoring_func=score,
                                  expert_load=load)
        return w, ids, *torch.autograd.grad(w, x, gw)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    with torch.no_grad():
        x.copy_(logits)
    graph.replay()
    graph.replay()
    counts, _ = load.clone(), load.zero_()
    eager = step()
    for g, e in zip(captured, eager):
        assert torch.equal(g, e)
    assert torch.equal(counts, 2 * load)


def test_offsets_past_32_bits(cuda_device):
    E, k = 1024, 8
    T = 2 ** 31 // E + 700
    x = torch.zeros(T, E, dtype=torch.bfloat16, device=cuda_device)
    logits, bias = inputs(3, E, torch.bfloat16, 8)
    rows = torch.tensor([5, T - 2, T - 1], device=cuda_device)
    x[rows] = logits.to(cuda_device)
    x.requires_grad_()
    w, ids = fm.balanced_topk(x, x, bias.to(cuda_device), k)
    check(logits, bias, w[rows], ids[rows], k)
    grad, = torch.autograd.grad(w[rows[1:]].sum() * 2 + w[rows[:1], 0].sum(), x)
    small = logits.to(cuda_device).requires_grad_()
    w, _ = fm.balanced_topk(small, small, bias.to(cuda_device), k)
    want, = torch.autograd.grad(w[1:].sum() * 2 + w[:1, 0].sum(), small)
    assert torch.equal(grad[rows], want)
    assert not grad[6:T - 2].any()


def test_forward_mode_is_refused(cuda_device):
    """A tangent of the logits would be lost; one of the bias has no effect."""
    import torch.autograd.forward_ad as fwd

    x, bias = (t.to(cuda_device) for t in inputs(4, 16, torch.float32, 1))
    want = fm.balanced_topk(x, x, bias, 2)
    with fwd.dual_level():
        for logits in (x, x.clone().requires_grad_()):
            with pytest.raises(ValueError, match="forward"):
                fm.balanced_topk(x, fwd.make_dual(logits, torch.ones_like(x)), bias, 2)
        got = fm.balanced_topk(x, x, fwd.make_dual(bias, torch.ones_like(bias)), 2)
        assert all(torch.equal(g, w) for g, w in zip(got, want))
    with pytest.raises(ValueError, match="forward"):
        torch.func.jvp(lambda l: fm.balanced_topk(x, l, None, 2)[0], (x,), (x,))


def test_refusals(cuda_device):
    from kernelswift_b200._lib import MoeError

    x = torch.randn(4, 32, device=cuda_device)
    with pytest.raises(MoeError):
        fm.balanced_topk(x, x, None, 9, num_expert_group=4, topk_group=1)
    with pytest.raises(MoeError):
        fm.balanced_topk(x, x, None, 33)
    with pytest.raises(MoeError):
        fm.balanced_topk(x, x, None, 2, num_expert_group=5)
    with pytest.raises(ValueError):
        fm.balanced_topk(x, x, torch.zeros(31, device=cuda_device), 2)
    with pytest.raises(ValueError):
        fm.balanced_topk(x, x, torch.zeros(32), 2)
    with pytest.raises(ValueError):
        fm.balanced_topk(x, x, None, 2, expert_load=torch.zeros(32, device=cuda_device))
