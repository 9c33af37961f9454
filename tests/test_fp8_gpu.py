"""GPU: the dense block-scaled fp8 operators (quantize_rows, quantize_blocks,
block_matmul, swiglu_mlp) against their fp64 restatement in the oracle."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from kernelswift_b200 import fp8
from kernelswift_b200 import fused_moe as fm
from fp8_plans import CASES
from oracle import moe_oracle as orc

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
FORMATS = ["fp32", "ue8m0"]


def gen(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def same_e4m3(got, want, share=0.0):
    """Equal e4m3 values but for `share` of them one step aside."""
    got = got.double().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    ok = ~want.isnan()
    off = (got - want).abs()[ok]
    step = torch.ldexp(torch.ones_like(off), torch.frexp(want[ok].abs().clamp_min(2.0 ** -6))
                       .exponent - 4)
    assert (off <= step * 1.001).all()
    assert (off != 0).double().mean().item() <= share if off.numel() else True


# ---------------------------------------------------------------------------
# quantisers
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("T,K", [(1, 1), (1, 128), (3, 100), (9, 129), (17, 1000), (64, 1024),
                                 (5, 1016), (33, 2049), (8, 7168)])
def test_quantize_rows(cuda_device, T, K, fmt):
    for dtype in DTYPES:
        x = gen(T, K, seed=T + K, dtype=dtype)
        x[T // 2, :min(K, 128)] = 0  # an all-zero group
        q, s = fp8.quantize_rows(x.to(cuda_device), fmt)
        assert q.dtype == torch.float8_e4m3fn and q.shape == (T, K)
        assert s.shape == (T, -(-K // 128)) and q.stride(0) % 16 == 0
        wq, ws = orc.fp8_rows(x, fmt)
        if fmt == "ue8m0":
            assert torch.equal(orc.fp8_scale_values(s.cpu()), ws)
            same_e4m3(q, wq)  # a division by a power of two is exact
        else:
            torch.testing.assert_close(s.double().cpu(), ws, rtol=2.0 ** -24, atol=0)
            # 16-bit inputs: exact. fp32: two roundings of 2^-24 move a value
            # across one of the midpoints 2^-5 apart for about 2^-18 of them
            same_e4m3(q, wq, 0.0 if dtype != torch.float32 else 2.0 ** -15 + 1.0 / (T * K) * (T * K > 99))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("T,K", [(1, 1), (2, 100), (7, 384), (21, 1000), (16, 2048)])
def test_quantize_gated(cuda_device, T, K, fmt):
    for dtype in DTYPES:
        x = (2 * gen(T, 2 * K, seed=T * K)).to(dtype)
        g, u = x.double().chunk(2, 1)
        act = g / (1 + torch.exp(-g)) * u
        q, s = fp8.quantize_rows(x.to(cuda_device), fmt, gated=True)
        wq, ws = orc.fp8_rows(act, fmt)
        if fmt == "ue8m0":
            assert torch.equal(orc.fp8_scale_values(s.cpu()), ws)
        else:
            # exp 2 ulp, add, divide, multiply, and the scale's division: 8 half steps
            torch.testing.assert_close(s.double().cpu(), ws, rtol=8 * 2.0 ** -24, atol=0)
        # the activation is off by 8 half steps of 2^-24: as above, and one more
        same_e4m3(q, wq, 2.0 ** -13 + 2.0 / (T * K) * (T * K > 99))


def test_gated_scale_next_to_a_power_of_two(cuda_device):
    """Maxima of silu(g) * u within 32-bit rounding of 448 * 2^k on either
    side: the byte is the one of the 64-bit value."""
    T = 400
    g = 1 + 3 * torch.rand(T, generator=torch.Generator().manual_seed(4))
    silu = g.double() / (1 + torch.exp(-g.double()))
    u = (448 * 2.0 ** torch.arange(-6, 6).repeat(T)[:T] / silu).float()
    x = torch.zeros(T, 256)
    x[:, 5], x[:, 128 + 5] = g, u
    act = silu * u.double()
    assert ((act / 448).log2() % 1 < 0.5).any() and ((act / 448).log2() % 1 > 0.5).any()
    _, s = fp8.quantize_rows(x.to(cuda_device), "ue8m0", gated=True)
    want = orc.fp8_rows(act[:, None], "ue8m0")[1]
    assert torch.equal(orc.fp8_scale_values(s.cpu()), want)


MANY = [(2500, 1030, 0),   # rows off 16-byte boundaries in every type
        (1300, 2048, 0),   # aligned, whole runs
        (1200, 2303, 3),   # the first row too, and the last run partial
        (9500, 200, 1)]    # less than a run


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,K,off", MANY)
def test_quantize_many_rows(cuda_device, T, K, off, dtype, fmt):
    """Rows enough for several runs of 256 columns per warp (from 9473 runs on)."""
    assert T * -(-K // 256) > 148 * 64
    wide = (gen(T, K + off, seed=K) * torch.exp(gen(T, 1, seed=T))).to(dtype)
    wide[T // 2, off:off + min(K, 128)] = 0
    x = wide[:, off:]
    q, s = fp8.quantize_rows(wide.to(cuda_device)[:, off:], fmt)
    wq, ws = orc.fp8_rows(x, fmt)
    if fmt == "ue8m0":
        assert torch.equal(orc.fp8_scale_values(s.cpu()), ws)
        same_e4m3(q, wq)
    else:
        torch.testing.assert_close(s.double().cpu(), ws, rtol=2.0 ** -24, atol=0)
        # as in test_quantize_rows
        same_e4m3(q, wq, 0.0 if dtype != torch.float32 else 2.0 ** -15)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,K,off", MANY)
def test_quantize_gated_many_rows(cuda_device, T, K, off, dtype, fmt):
    wide = (2 * gen(T, 2 * K + off, seed=K)).to(dtype)
    g, u = wide[:, off:].double().chunk(2, 1)
    q, s = fp8.quantize_rows(wide.to(cuda_device)[:, off:], fmt, gated=True)
    wq, ws = orc.fp8_rows(g / (1 + torch.exp(-g)) * u, fmt)
    if fmt == "ue8m0":
        assert torch.equal(orc.fp8_scale_values(s.cpu()), ws)
    else:
        torch.testing.assert_close(s.double().cpu(), ws, rtol=8 * 2.0 ** -24, atol=0)
    same_e4m3(q, wq, 2.0 ** -13)  # as in test_quantize_gated


def test_gated_scales_of_many_rows_next_to_a_power_of_two(cuda_device):
    """As test_gated_scale_next_to_a_power_of_two, in each group that a warp holds
    of rows with several runs."""
    T, K = 2400, 1024
    assert T * -(-K // 256) > 148 * 64
    n = K // 128
    g = 1 + 3 * torch.rand(T, n, generator=torch.Generator().manual_seed(4))
    silu = g.double() / (1 + torch.exp(-g.double()))
    u = (448 * 2.0 ** (torch.arange(T * n).view(T, n) % 12 - 6) / silu).float()
    x = torch.zeros(T, 2 * K)
    at = 128 * torch.arange(n) + 5 + 17 * torch.arange(n) % 123
    x[:, at], x[:, K + at] = g, u
    act = silu * u.double()
    up = (act / 448).log2() % 1 < 0.5
    assert up.any() and not up.all()
    _, s = fp8.quantize_rows(x.to(cuda_device), "ue8m0", gated=True)
    want = torch.cat([orc.fp8_rows(act[:, j:j + 1], "ue8m0")[1] for j in range(n)], 1)
    assert torch.equal(orc.fp8_scale_values(s.cpu()), want)


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_nan_inf_and_extremes(cuda_device, fmt):
    x = gen(6, 256, seed=9)
    x[0, 3] = torch.nan
    x[1, 200] = torch.inf
    x[2] = torch.nan
    x[3, :128] *= 1e-44      # subnormal
    x[4, :128] *= 1e37
    x[5, 0] = torch.finfo(torch.float32).max
    q, s = fp8.quantize_rows(x.to(cuda_device), fmt)
    v = q.double().cpu()
    assert torch.equal(v.isnan()[[0, 2, 3, 4, 5]], x.isnan()[[0, 2, 3, 4, 5]])
    rest = x[0, 4:128]
    assert torch.isfinite(s[0].float()).all()
    sv = orc.fp8_scale_values(s.cpu())
    back = v[0, 4:128] * sv[0, 0]
    assert ((back - rest.double()).abs() <= 2.0 ** -4 * rest.abs().double() + sv[0, 0] * 2.0 ** -10
            ).all()
    assert (v[4:].abs() <= 448).all()
    back = v[4, :128] * sv[4, 0]
    want = x[4, :128].double()
    assert ((back - want).abs() <= 1.001 * (2.0 ** -4 * want.abs() + sv[4, 0] * 2.0 ** -10)).all()
    if fmt == "fp32":
        assert s[1, 1].isinf() and v[1, 200].isnan()  # no finite scale for that group
    else:
        assert v[1, 200] == 448 and torch.equal(v[1, :128].isnan(), torch.zeros(128).bool())


def test_quantize_strided_rows_and_none(cuda_device):
    wide = gen(20, 700, seed=2, dtype=torch.bfloat16).to(cuda_device)
    for view in (wide[:, 3:303], wide[::3, :512], wide.t()[:, :16], wide[:1].expand(5, 700)):
        q, s = fp8.quantize_rows(view, "ue8m0")
        wq, ws = orc.fp8_rows(view.cpu(), "ue8m0")
        same_e4m3(q, wq)
        assert torch.equal(orc.fp8_scale_values(s.cpu()), ws)
    q, s = fp8.quantize_rows(wide[:0], "fp32")
    assert q.shape == (0, 700) and s.shape == (0, 6)


def test_rows_behind_the_matrix_stay(cuda_device):
    """Through the C entry: only rows [0, T) of larger buffers are written,
    and of a row no more than its 16-byte padded length."""
    from kernelswift_b200 import _lib
    from kernelswift_b200.fused_moe import _ptr, _stream

    T, K = 5, 200
    x = gen(T, K, seed=1).to(cuda_device)
    q = torch.full((T + 3, 256), 7, dtype=torch.uint8, device=cuda_device)
    s = torch.full((T + 3, 4), 9, dtype=torch.uint8, device=cuda_device)
    _lib.call("moe_fp8_quantize_rows", _ptr(x), _lib.DT_F32, T, K, K, 0, 1, _ptr(q), 256, _ptr(s),
              4, 1, _stream(cuda_device))
    assert (q[T:] == 7).all() and (q[:, 208:] == 7).all()
    assert (s[T:] == 9).all() and (s[:, 2:] == 9).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("N,K", [(1, 1), (128, 128), (130, 100), (300, 700), (576, 1000)])
def test_quantize_blocks(cuda_device, N, K, fmt):
    for dtype in DTYPES:
        w = gen(N, K, seed=N, dtype=dtype)
        q, s = fp8.quantize_blocks(w.to(cuda_device), fmt)
        wq, ws = orc.fp8_blocks(w, fmt)
        assert q.shape == (N, K) and s.shape == ws.shape and q.stride(0) % 16 == 0
        if fmt == "ue8m0":
            assert torch.equal(orc.fp8_scale_values(s.cpu()), ws)
            same_e4m3(q, wq)
        else:
            torch.testing.assert_close(s.double().cpu(), ws, rtol=2.0 ** -24, atol=0)
            same_e4m3(q, wq, 0.0 if dtype != torch.float32 else 2.0 ** -15 + 1.0 / (N * K) * (N * K > 99))


# ---------------------------------------------------------------------------
# product
# ---------------------------------------------------------------------------

def operands(T, N, K, fmt, dev, seed=0):
    x = fp8.quantize_rows((gen(T, K, seed=seed) * torch.exp(gen(T, 1, seed=seed + 1))).to(dev), fmt)
    w = fp8.quantize_blocks(gen(N, K, seed=seed + 2).to(dev) / K ** 0.5, fmt)
    return x, w


def check_product(out, x, w, addend=None):
    """Each MMA step adds 32 products to the sum: its alignment costs at most
    2^-23 of the magnitudes summed, as does each addition of a scaled block;
    then one rounding to the output's type."""
    K = x[0].shape[1]
    want, mag = orc.fp8_dense(*(t.cpu() for t in x), *(t.cpu() for t in w))
    if addend is not None:
        want, mag = want + addend.double().cpu(), mag + addend.double().cpu().abs()
    room = HALF[out.dtype] * want.abs() + (4 + K / 32) * 2.0 ** -23 * mag
    tiny = 2.0 ** -25 if out.dtype == torch.float16 else 0.0
    err = (out.double().cpu() - want).abs()
    assert (err <= room + tiny).all(), (err - room).max()


SIZES = [(1, 1, 1), (1, 128, 128), (3, 17, 100), (16, 130, 129), (17, 256, 640), (31, 300, 1000),
         (33, 129, 2000), (64, 576, 512), (65, 384, 300), (100, 77, 4000), (128, 640, 1536),
         (129, 257, 130), (200, 1024, 1000), (257, 513, 999), (333, 1500, 1000), (600, 2049, 256),
         (1, 4096, 7168), (5, 7168, 2048), (513, 1032, 2000), (1000, 4104, 384), (2049, 1544, 700)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("T,N,K", SIZES)
def test_product(cuda_device, T, N, K, fmt):
    x, w = operands(T, N, K, fmt, cuda_device, T + N + K)
    for dtype in DTYPES:
        check_product(fp8.block_matmul(*x, *w, out_dtype=dtype), x, w)
    add = gen(T, N, seed=5, dtype=torch.bfloat16).to(cuda_device)
    want = fp8.block_matmul(*x, *w, addend=add)
    check_product(want, x, w, add)
    got = fp8.block_matmul(*x, *w, addend=add, out=add)  # in place
    assert got is add and torch.equal(got, want)


def dense64(x, w):
    """orc.fp8_dense on the GPU, in torch's fp64: (product, sum of magnitudes)."""
    def values(s):
        return torch.exp2(s.double() - 127) if s.dtype == torch.uint8 else s.double()

    (T, K), N = x[0].shape, w[0].shape[0]
    a = x[0].double() * values(x[1]).repeat_interleave(128, 1)[:, :K]
    b = w[0].double() * (values(w[1]).repeat_interleave(128, 0)[:N]
                         .repeat_interleave(128, 1)[:, :K])
    return a @ b.t(), a.abs() @ b.abs().t()


@pytest.mark.parametrize("fmt,plan,size", CASES)
def test_every_plan(cuda_device, fmt, plan, size):
    """Each tile and split, plain and with an addend, into a tensor of its own, in
    place and into columns of a wider one; bounds as in check_product."""
    T, N, K = size
    x, w = operands(T, N, K, fmt, cuda_device, 11)
    want, mag = dense64(x, w)

    def check(out, add=0.0):
        room = (HALF[out.dtype] * (want + add).abs()
                + (4 + K / 32) * 2.0 ** -23 * (mag + abs(add)))
        tiny = 2.0 ** -25 if out.dtype == torch.float16 else 0.0
        err = (out.double() - want - add).abs()
        assert (err <= room + tiny).all(), (err - room).max()

    check(fp8.block_matmul(*x, *w, out_dtype=torch.float32))
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        add = gen(T, N, seed=5, dtype=dtype).to(cuda_device)
        got = fp8.block_matmul(*x, *w, addend=add, out_dtype=dtype)
        check(got, add.double())
        wide = torch.full((T + 1, N + 16), 7.0, dtype=dtype, device=cuda_device)
        inner = wide[:-1, 8:N + 8]
        inner.copy_(add)
        assert torch.equal(fp8.block_matmul(*x, *w, addend=inner, out=inner), got)
        assert (wide[-1] == 7).all() and (wide[:, :8] == 7).all() and (wide[:, N + 8:] == 7).all()
        assert torch.equal(fp8.block_matmul(*x, *w, addend=add, out=add), got)


@pytest.mark.parametrize("fmt", FORMATS)
def test_large_products_by_rows(cuda_device, fmt):
    """Many tiles per CTA: rows drawn from a product too large for the oracle."""
    T, N, K = 5000, 4104, 1100
    x, w = operands(T, N, K, fmt, cuda_device)
    out = fp8.block_matmul(*x, *w)
    rows = torch.cat([torch.arange(0, T, 37), torch.tensor([T - 1])])
    xq = x[0].view(torch.uint8)[rows.to(cuda_device)].view(torch.float8_e4m3fn)
    check_product(out[rows.to(cuda_device)], (xq, x[1][rows.to(cuda_device)]), w)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_large_products_off_alignment(cuda_device, dtype, fmt):
    """Output and addend rows of odd pitch, inside larger buffers."""
    T, N, K = 1300, 2403, 520
    assert fp8.block_matmul_plan(T, N, K, fmt)["cta_pairs"] == 1
    x, w = operands(T, N, K, fmt, cuda_device, 9)
    add = gen(T, N + 2, seed=5, dtype=dtype).to(cuda_device)[:, 1:-1]
    check_product(fp8.block_matmul(*x, *w, addend=add, out_dtype=dtype), x, w, add)
    wide = torch.full((T + 1, N + 4), 7.0, dtype=dtype, device=cuda_device)
    out = fp8.block_matmul(*x, *w, out=wide[:-1, 3:-1])
    assert torch.equal(out, fp8.block_matmul(*x, *w, out_dtype=dtype))
    check_product(out, x, w)
    assert (wide[-1] == 7).all() and (wide[:, :3] == 7).all() and (wide[:, -1] == 7).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_operand_layouts(cuda_device, fmt):
    """Row-major and padded scales, rows of a wider matrix, unaligned views,
    an output inside a larger one whose other columns stay."""
    T, N, K = 40, 200, 700
    x, w = operands(T, N, K, fmt, cuda_device, 3)
    want = fp8.block_matmul(*x, *w, out_dtype=torch.float32)
    dense_q = x[0].view(torch.uint8).contiguous().view(torch.float8_e4m3fn)  # pitch 700
    dense_w = w[0].view(torch.uint8).contiguous().view(torch.float8_e4m3fn)
    off = torch.zeros(T * 704 + 5, dtype=torch.uint8, device=cuda_device)
    off_q = off[5:].view(T, 704)[:, :K]
    off_q.copy_(x[0].view(torch.uint8))
    rowmajor = x[1].contiguous()
    wide = torch.zeros(T, 3 * x[1].shape[1], dtype=x[1].dtype, device=cuda_device)
    wide[:, ::3] = x[1]
    for q, s, wq in ((dense_q, rowmajor, w[0]), (x[0], wide[:, ::3], dense_w),
                     (off_q.view(torch.float8_e4m3fn), x[1], w[0])):
        assert torch.equal(fp8.block_matmul(q, s, wq, w[1], out_dtype=torch.float32), want)
    big = torch.full((T, N + 9), 3.0, device=cuda_device)
    fp8.block_matmul(*x, *w, out=big[:, 4:4 + N])
    assert torch.equal(big[:, 4:4 + N], want) and (big[:, :4] == 3).all() and (big[:, 4 + N:] == 3).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("T,N,K", [(5, 130, 700), (200, 264, 1100), (2100, 1290, 700)])
def test_parts_of_operands(cuda_device, T, N, K, fmt):
    """Rows and k-blocks of larger operands, scales repeated or transposed, a
    status word that stays 0."""
    x, w = operands(T + 3, N, K, fmt, cuda_device, 6)
    status = torch.zeros(2, dtype=torch.int32, device=cuda_device)

    def run(xq, xs, wq, ws):
        return fp8.block_matmul(xq, xs, wq, ws, out_dtype=torch.float32, status=status[1:])

    def check(got, xq, xs, wq, ws):
        want, mag = dense64((xq, xs), (wq, ws))
        room = 2.0 ** -24 * want.abs() + (4 + K / 32) * 2.0 ** -23 * mag
        assert ((got.double() - want).abs() <= room).all()

    rows = x[0][2:T + 2], x[1][2:T + 2], *w
    check(run(*rows), *rows)
    blocks = x[0][:, 128:], x[1][:, 1:], w[0][:, 128:], w[1][:, 1:]
    check(run(*blocks), *blocks)
    one = x[0], x[1][:1].expand(T + 3, -1), w[0], w[1].t().contiguous().t()
    check(run(*one), *one)
    assert not status.any()


def test_scales_at_the_ends_of_their_range(cuda_device):
    """Powers of two far from 1 on one side and back on the other."""
    for T in (7, 40, 300, 2100):
        x, w = operands(T, 1290, 256, "ue8m0", cuda_device, 8)
        want = fp8.block_matmul(*x, *w, out_dtype=torch.float32)
        for up in (-100, -20, 20, 100):
            xs = (x[1].int() + up).to(torch.uint8)
            ws = (w[1].int() - up).to(torch.uint8)
            got = fp8.block_matmul(x[0], xs, w[0], ws, out_dtype=torch.float32)
            assert torch.equal(got, want), (T, up)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("T", [1, 20, 150])
def test_nan_and_inf_stay_in_their_rows(cuda_device, T, fmt):
    x0 = gen(T, 300, seed=1)
    x, w = operands(T, 150, 300, fmt, cuda_device, 3)
    clean = fp8.quantize_rows(x0.to(cuda_device), fmt)
    x0[T // 2, 7] = torch.nan
    dirty = fp8.quantize_rows(x0.to(cuda_device), fmt)
    a = fp8.block_matmul(*clean, *w)
    b = fp8.block_matmul(*dirty, *w)
    keep = torch.arange(T) != T // 2
    assert torch.equal(a[keep], b[keep]) and b[T // 2].isnan().all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_offsets_past_32_bits(cuda_device, fmt):
    """Rows far behind the first: inputs and outputs of more than 2^32 bytes and
    2^31 elements."""
    K, N = 100, 40000
    T = 2 ** 31 // N + 500
    x = torch.zeros(T, K, dtype=torch.bfloat16, device=cuda_device)
    rows = torch.tensor([0, T // 2, T - 2, T - 1], device=cuda_device)
    x[rows] = gen(4, K, dtype=torch.bfloat16).to(cuda_device)
    w = fp8.quantize_blocks(gen(N, K, seed=1).to(cuda_device) / 10, fmt)
    q, scale = fp8.quantize_rows(x, fmt)
    out = fp8.block_matmul(q, scale, *w)
    alone = fp8.quantize_rows(x[rows], fmt)
    check_product(out[rows], alone, w)
    assert not out[T // 2 + 1:T - 2].any()
    del out
    big, two = fp8.quantize_rows(x.expand(2, T, K).reshape(2 * T, K), fmt)
    assert torch.equal(big.view(torch.uint8)[rows + T], alone[0].view(torch.uint8))
    assert torch.equal(two[rows + T], alone[1])


def test_long_quantised_rows(cuda_device):
    """One call over more than 2^32 elements."""
    T, K = 66000, 65600
    x = torch.zeros(T, K, dtype=torch.bfloat16, device=cuda_device)
    x[-1] = gen(K, dtype=torch.bfloat16).to(cuda_device)
    q, scale = fp8.quantize_rows(x)
    one, s1 = fp8.quantize_rows(x[-1:])
    assert torch.equal(q.view(torch.uint8)[-1:], one.view(torch.uint8))
    assert torch.equal(scale[-1:], s1)
    assert not q[-2].view(torch.uint8).any()


@pytest.mark.parametrize("T,N,K", [(100003, 8, 64), (1, 128, 100000), (2, 100001, 32),
                                   (7, 300, 40001)])
@pytest.mark.parametrize("fmt", FORMATS)
def test_lopsided_products(cuda_device, T, N, K, fmt):
    x, w = operands(T, N, K, fmt, cuda_device, 4)
    rows = torch.arange(0, T, max(1, T // 40), device=cuda_device)
    xq = x[0].view(torch.uint8)[rows].view(torch.float8_e4m3fn)
    check_product(fp8.block_matmul(*x, *w, out_dtype=torch.float32)[rows], (xq, x[1][rows]), w)


def test_first_calls_of_a_process_captured(cuda_device):
    """Nothing has to run eagerly before a capture."""
    code = """
import torch
from kernelswift_b200 import fp8, fused_moe as fm
dev = torch.device("cuda", 0)
x = torch.randn(300, 640, device=dev).bfloat16()
logits = torch.randn(300, 64, device=dev)
def layer(fmt):
    w13 = fp8.quantize_blocks(a, fmt)
    w2 = fp8.quantize_blocks(b, fmt)
    return fp8.swiglu_mlp(x, *w13, *w2), fm.balanced_topk(x, logits, None, 4)[0]
a = torch.randn(768, 640, device=dev) / 25
b = torch.randn(640, 384, device=dev) / 20
for fmt in ("fp32", "ue8m0"):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer(fmt)
    graph.replay()
    want = layer(fmt)
    assert all(torch.equal(g, w) for g, w in zip(got, want)), fmt
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True,
                          timeout=120)
    assert done.returncode == 0, done.stderr[-2000:]


def test_two_streams_at_once(cuda_device):
    """Calls on two streams share nothing."""
    work = []
    for seed in range(2):
        x = gen(500, 640, seed=seed, dtype=torch.bfloat16).to(cuda_device)
        w13 = fp8.quantize_blocks(gen(768, 640, seed=2 + seed).to(cuda_device) / 25)
        w2 = fp8.quantize_blocks(gen(640, 384, seed=4 + seed).to(cuda_device) / 20)
        work.append((x, *w13, *w2))
    want = [fp8.swiglu_mlp(*w) for w in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    for _ in range(20):
        got = []
        for w, s in zip(work, streams):
            with torch.cuda.stream(s):
                got.append(fp8.swiglu_mlp(*w))
        torch.cuda.synchronize()
        assert all(torch.equal(g, v) for g, v in zip(got, want))


def test_no_rows_and_zero_scales(cuda_device):
    x, w = operands(4, 64, 256, "fp32", cuda_device)
    out = fp8.block_matmul(x[0][:0], x[1][:0], *w)
    assert out.shape == (0, 64)
    zero = fp8.quantize_rows(torch.zeros(4, 256, device=cuda_device), "ue8m0")
    wu = fp8.quantize_blocks(torch.zeros(64, 256, device=cuda_device), "ue8m0")
    assert (fp8.block_matmul(*zero, *wu) == 0).all()


def test_same_bits_every_time_and_captured(cuda_device):
    """A fixed order of summation: equal bits on a repeated call, on another
    stream, and replayed from a graph next to another captured product."""
    for fmt in FORMATS:
        for T, N, K in ((1, 4096, 7168), (48, 1024, 4096), (300, 512, 2048)):
            x, w = operands(T, N, K, fmt, cuda_device)
            want = fp8.block_matmul(*x, *w)
            side = torch.cuda.Stream(cuda_device)
            side.wait_stream(torch.cuda.current_stream(cuda_device))
            with torch.cuda.stream(side):
                other = fp8.block_matmul(*x, *w)
            torch.cuda.current_stream(cuda_device).wait_stream(side)
            graphs, outs = [], []
            for _ in range(2):
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    outs.append(fp8.block_matmul(*x, *w))
                graphs.append(g)
            for g in graphs * 2:
                g.replay()
            torch.cuda.synchronize()
            for got in [other, fp8.block_matmul(*x, *w)] + outs:
                assert torch.equal(got, want)


@pytest.mark.parametrize("fmt", FORMATS)
def test_products_right_behind_each_other(cuda_device, fmt):
    """A product's last arrivals are on barriers of its own shared memory: the
    products launched behind it, which take the same memory for theirs, give the
    same bits every time."""
    sizes = [(2048, 1280, 640), (20, 512, 1000), (1300, 2403, 520), (1, 1024, 2000)]
    plans = [fp8.block_matmul_plan(*size, fmt)["cta_pairs"] for size in sizes]
    assert plans == [1, 0, 1, 0]
    work = [operands(*size, fmt, cuda_device, 5) for size in sizes]
    want = []
    for x, w in work:
        want.append(fp8.block_matmul(*x, *w))
        torch.cuda.synchronize()
        check_product(want[-1], x, w)
    got = [[fp8.block_matmul(*x, *w) for x, w in work] for _ in range(60)]
    for outs in got:
        assert all(torch.equal(g, v) for g, v in zip(outs, want))


# ---------------------------------------------------------------------------
# the MLP, and the layer: balanced routing, routed experts, shared expert
# ---------------------------------------------------------------------------

def mlp_reference(x, w13, w2, fmt, addend):
    """The chain in fp64, activations quantised and the gate-up product
    rounded as the operator states."""
    q, s = orc.fp8_rows(x, fmt)
    s = s.float().double()
    K = x.shape[1]

    def dense(w):
        (N, K), ws = w[0].shape, orc.fp8_scale_values(w[1].cpu())
        return (w[0].cpu().double() * ws.repeat_interleave(128, 0)[:N]
                .repeat_interleave(128, 1)[:, :K])

    both = (q * s.repeat_interleave(128, 1)[:, :K]) @ dense(w13).t()
    g, u = both.to(x.dtype).double().chunk(2, 1)
    q, s = orc.fp8_rows(g / (1 + torch.exp(-g)) * u, fmt)
    out = (q * s.repeat_interleave(128, 1)[:, :w2[0].shape[1]]) @ dense(w2).t()
    return out + addend.double()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("T,H,I", [(1, 256, 128), (19, 512, 200), (300, 640, 384)])
def test_swiglu_mlp(cuda_device, T, H, I, fmt):
    x = gen(T, H, seed=1, dtype=torch.bfloat16)
    add = gen(T, H, seed=2, dtype=torch.bfloat16)
    w13 = fp8.quantize_blocks(gen(2 * I, H, seed=3).to(cuda_device) / H ** 0.5, fmt)
    w2 = fp8.quantize_blocks(gen(H, I, seed=4).to(cuda_device) / I ** 0.5, fmt)
    out = fp8.swiglu_mlp(x.to(cuda_device), *w13, *w2, addend=add.to(cuda_device))
    want = mlp_reference(x, w13, w2, fmt, add)
    # a gate-up value next to a rounding border may fall the other way, by a
    # bf16 step (2^-7), then its fp8 value by a step (2^-3): a few of the I
    # terms; the rest as one rounding of the result
    assert orc.rel_l2(out.double().cpu(), want) < 2.0 ** -8
    err = (out.double().cpu() - want).abs()
    assert (err <= 2.0 ** -8 * want.abs() + 2.0 ** -3 * want.abs().amax()).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,H,I", [(1, 250, 100), (33, 512, 200), (300, 648, 384)])
def test_swiglu_mlp_types_and_places(cuda_device, T, H, I, dtype, fmt):
    """Each type, with no addend, rows of a wider tensor, the result in place of
    the input, of the addend, or beside it."""
    wide = gen(T, H + 5, seed=1, dtype=dtype).to(cuda_device)
    x = wide[:, 3:H + 3]
    w13 = fp8.quantize_blocks(gen(2 * I, H, seed=3).to(cuda_device) / H ** 0.5, fmt)
    w2 = fp8.quantize_blocks(gen(H, I, seed=4).to(cuda_device) / I ** 0.5, fmt)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    out = fp8.swiglu_mlp(x, *w13, *w2, status=status)
    want = mlp_reference(x.cpu(), w13, w2, fmt, torch.zeros(T, H))
    assert out.dtype == dtype and not status.any()
    assert orc.rel_l2(out.double().cpu(), want) < 2.0 ** -8  # as in test_swiglu_mlp
    add = gen(T, H, seed=2, dtype=dtype).to(cuda_device)
    added = fp8.swiglu_mlp(x, *w13, *w2, addend=add)
    assert orc.rel_l2(added.double().cpu(), want + add.double().cpu()) < 2.0 ** -8
    got = fp8.swiglu_mlp(x, *w13, *w2, addend=add, out=add)
    assert got is add and torch.equal(got, added)
    both = fp8.swiglu_mlp(x, *w13, *w2, addend=x)
    buf = wide.clone()
    place = buf[:, 3:H + 3]
    assert torch.equal(fp8.swiglu_mlp(place, *w13, *w2, addend=place, out=place), both)
    assert torch.equal(buf[:, :3], wide[:, :3]) and torch.equal(buf[:, H + 3:], wide[:, H + 3:])
    buf = wide.clone()
    assert torch.equal(fp8.swiglu_mlp(buf[:, 3:H + 3], *w13, *w2, out=buf[:, 3:H + 3]), out)
    none = fp8.swiglu_mlp(x[:0], *w13, *w2, addend=x[:0])
    assert none.shape == (0, H) and none.dtype == dtype


def test_layer_of_routed_and_shared_experts(cuda_device):
    """Balanced routing -> routed experts (fp8) -> shared expert added, eager
    and replayed from one graph, against the fp32 layer of the same weights."""
    T, H, I, E, k = 40, 512, 256, 16, 4
    hidden = gen(T, H, seed=1, dtype=torch.bfloat16).to(cuda_device)
    logits = gen(T, E, seed=2).to(cuda_device)
    bias = 0.1 * gen(E, seed=3).to(cuda_device)
    w1 = (gen(E, 2 * I, H, seed=4) / H ** 0.5).to(cuda_device)
    w2 = (gen(E, H, I, seed=5) / I ** 0.5).to(cuda_device)
    sw13 = gen(2 * I, H, seed=6).to(cuda_device) / H ** 0.5
    sw2 = gen(H, I, seed=7).to(cuda_device) / I ** 0.5
    routed = fm.prepare_weights(w1, w2, "fp8-ue8m0")
    s13, s2 = fp8.quantize_blocks(sw13), fp8.quantize_blocks(sw2)

    def layer(h, l):
        w, ids = fm.balanced_topk(h, l, bias, k, num_expert_group=4, topk_group=2)
        r = fm.fused_experts(h, routed, None, w, ids, use_fp8_w8a8=True)
        return fp8.swiglu_mlp(h, *s13, *s2, addend=r)

    with torch.no_grad():
        out = layer(hidden, logits)
        step = fm.CapturedMoE(layer, T, H, E)
        assert torch.equal(step(hidden, logits), out)
    w, ids = orc.balanced_topk(logits.cpu(), bias.cpu(), k, num_expert_group=4, topk_group=2)
    x = hidden.double().cpu()
    want = orc.fused_experts(x.float(), w1.cpu(), w2.cpu(), w.float(), ids).double()
    g, u = (x @ sw13.double().cpu().t()).chunk(2, 1)
    want = want + (g / (1 + torch.exp(-g)) * u) @ sw2.double().cpu().t()
    # e4m3 operands on both sides of four products: the layer's fp8 bound
    assert orc.rel_l2(out.double().cpu(), want) < 8e-2


def test_addend_beside_the_output(cuda_device):
    """Columns of one buffer that share no element with the output."""
    x, w = operands(40, 64, 256, "ue8m0", cuda_device)
    wide = gen(40, 200, dtype=torch.bfloat16).to(cuda_device)
    for at, to in ((100, 3), (0, 64), (64, 0)):
        buf = wide.clone()
        want = fp8.block_matmul(*x, *w, addend=wide[:, at:at + 64].contiguous())
        fp8.block_matmul(*x, *w, addend=buf[:, at:at + 64], out=buf[:, to:to + 64])
        assert torch.equal(buf[:, to:to + 64], want)


@pytest.mark.parametrize("fmt", FORMATS)
def test_one_token_added_in_place(cuda_device, fmt):
    """A row of a wider buffer as output and, under another stride, as addend."""
    x, w = operands(1, 64, 256, fmt, cuda_device)
    buf = gen(3, 80, dtype=torch.bfloat16).to(cuda_device)
    want = fp8.block_matmul(*x, *w, addend=buf[1:2, :64].clone())
    before = buf.clone()
    got = fp8.block_matmul(*x, *w, out=buf[1:2, :64], addend=buf[1, :64].unsqueeze(0))
    assert torch.equal(got, want)
    before[1, :64] = want[0]
    assert torch.equal(buf, before)


def test_forward_mode_is_refused(cuda_device):
    """No tangent is lost silently."""
    import torch.autograd.forward_ad as fwd

    x, w = operands(4, 64, 256, "fp32", cuda_device)
    w13, w2 = operands(1, 256, 64, "fp32", cuda_device)[1], operands(1, 64, 128, "fp32", cuda_device)[1]
    rows = gen(4, 64).to(cuda_device)
    add = gen(4, 64, dtype=torch.bfloat16).to(cuda_device)
    with fwd.dual_level():
        def dual(t):
            return fwd.make_dual(t, torch.ones_like(t))

        for call in (lambda: fp8.quantize_rows(dual(rows)), lambda: fp8.quantize_blocks(dual(rows)),
                     lambda: fp8.block_matmul(x[0], dual(x[1]), *w),
                     lambda: fp8.block_matmul(*x, w[0], dual(w[1])),
                     lambda: fp8.block_matmul(*x, *w, addend=dual(add)),
                     lambda: fp8.block_matmul(*x, *w, out=dual(add)),
                     lambda: fp8.swiglu_mlp(dual(rows), *w13, *w2),
                     lambda: fp8.swiglu_mlp(rows, w13[0], dual(w13[1]), *w2),
                     lambda: fp8.swiglu_mlp(rows, *w13, w2[0], dual(w2[1])),
                     lambda: fp8.swiglu_mlp(rows, *w13, *w2, addend=dual(rows))):
            with pytest.raises(ValueError, match="forward"):
                call()
        fp8.block_matmul(*x, *w, addend=add)


def test_refusals(cuda_device):
    x, w = operands(4, 64, 256, "fp32", cuda_device)
    xu, wu = operands(4, 64, 256, "ue8m0", cuda_device)
    both = torch.zeros(5, 65, dtype=torch.bfloat16, device=cuda_device)
    bad = [
        lambda: fp8.block_matmul(x[0], x[1], w[0], wu[1]),            # mixed formats
        lambda: fp8.block_matmul(x[0], x[1][:3], *w),
        lambda: fp8.block_matmul(x[0], x[1][:, :1], *w),
        lambda: fp8.block_matmul(x[0], x[1], w[0][:, :128], w[1]),
        lambda: fp8.block_matmul(x[0].float(), x[1], *w),
        lambda: fp8.block_matmul(*x, *w, out_dtype=torch.int32),
        lambda: fp8.block_matmul(*x, *w, addend=torch.zeros(4, 64, device=cuda_device)),
        lambda: fp8.block_matmul(*x, *w, out=torch.zeros(4, 63, device=cuda_device)),
        lambda: fp8.block_matmul(*x, *w, out=torch.zeros(64, 4, device=cuda_device).t()),
        lambda: fp8.block_matmul(x[0].cpu(), *x[1:], *w),
        lambda: fp8.quantize_rows(torch.zeros(4, device=cuda_device)),
        lambda: fp8.quantize_rows(torch.zeros(4, 5, device=cuda_device), gated=True),
        lambda: fp8.quantize_rows(torch.zeros(4, 4, device=cuda_device), "int8"),
        lambda: fp8.quantize_rows(torch.zeros(4, 4, device=cuda_device, requires_grad=True)),
        lambda: fp8.quantize_blocks(torch.zeros(4, 4, device=cuda_device).int()),
        lambda: fp8.swiglu_mlp(torch.zeros(4, 256, device=cuda_device), *w, *w),
        lambda: fp8.block_matmul(*x, *w, status=torch.zeros(1, dtype=torch.int32)),
        lambda: fp8.block_matmul(*x, *w, status=torch.zeros(1, device=cuda_device)),
        lambda: fp8.block_matmul(x[0], x[1].clone().requires_grad_(), *w),
        lambda: fp8.block_matmul(*x, *w, addend=torch.zeros(1, 64, device=cuda_device,
                                                            dtype=torch.bfloat16).expand(4, 64)),
        lambda: fp8.block_matmul(*x, *w, out=both[:4, :64], addend=both[:4, 1:]),
        lambda: fp8.block_matmul(*x, *w, out=both[:4, :64], addend=both[1:, :64]),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
