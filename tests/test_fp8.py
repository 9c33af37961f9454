"""CPU: refusals of the dense fp8 entry points (on the host, before any
launch), the plan of the product, and the oracle's roundings."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from kernelswift_b200 import _lib, fp8
from fp8_plans import CASES, PLANS
from oracle import moe_oracle as orc

F32, BF16, I8 = _lib.DT_F32, _lib.DT_BF16, _lib.DT_I8
INVALID, UNSUPPORTED = _lib.MOE_ERR_INVALID_ARG, _lib.MOE_ERR_UNSUPPORTED


def quantize(x_dtype=BF16, T=4, K=256, ld=None, gated=0, fmt=1, q=0x1000, ld_q=256):
    ld = (2 * K if gated else K) if ld is None else ld
    return _lib.load().moe_fp8_quantize_rows(0x1000, x_dtype, T, K, ld, gated, fmt, q, ld_q,
                                             0x1000, 4, 1, None)


def matmul(x=0x1000, ld_x=256, w=0x1000, ld_w=256, fmt=1, T=4, N=64, K=256, add=None, ld_add=0,
           ld_out=64, out_dtype=BF16):
    return _lib.load().moe_fp8_matmul(x, ld_x, 0x1000, 4, 1, w, ld_w, 0x1000, fmt, T, N, K, add,
                                      ld_add, 0x1000, ld_out, out_dtype, None, None)


@pytest.mark.parametrize("bad,status", [
    (dict(x_dtype=I8), INVALID), (dict(T=-1), INVALID), (dict(K=0), INVALID),
    (dict(ld=255), INVALID), (dict(gated=1, ld=511), INVALID), (dict(fmt=2), INVALID),
    (dict(q=0x1008), INVALID), (dict(ld_q=250), INVALID), (dict(K=257, ld_q=256), INVALID),
    (dict(T=1 << 31), UNSUPPORTED),
])
def test_quantizer_refusals(bad, status):
    assert quantize(**bad) == status
    assert "fp8_quantize_rows" in _lib.load().moe_last_error().decode()


@pytest.mark.parametrize("bad,status", [
    (dict(x=0x1008), INVALID), (dict(w=0x1004), INVALID), (dict(ld_x=250, K=250), INVALID),
    (dict(ld_w=264), INVALID), (dict(ld_x=240), INVALID), (dict(fmt=3), INVALID),
    (dict(T=-1), INVALID), (dict(N=0), INVALID), (dict(K=0), INVALID),
    (dict(ld_out=63), INVALID), (dict(add=0x1000, ld_add=63), INVALID),
    (dict(out_dtype=I8), INVALID), (dict(T=1 << 31), UNSUPPORTED), (dict(N=1 << 31), UNSUPPORTED),
    (dict(T=1 << 30, N=1 << 30, ld_out=1 << 30), UNSUPPORTED),
])
def test_product_refusals(bad, status):
    assert matmul(**bad) == status
    assert "fp8_matmul" in _lib.load().moe_last_error().decode()


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError):
        fp8.quantize_rows(torch.zeros(2, 128))
    with pytest.raises(ValueError):
        fp8.quantize_blocks(torch.zeros(2, 128))


def test_import_with_a_torch_without_cuda():
    """The host's queries need no CUDA in torch, and tensors are refused as ever."""
    code = """
import torch
for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"):
    if hasattr(torch._C, name):
        delattr(torch._C, name)
from kernelswift_b200 import fp8, fused_moe as fm
assert fm.fused_experts_plan(16, 256, 128, 8, 2)
assert fp8.block_matmul_plan(1, 128, 128)["splits"] == 1
try:
    fm.balanced_topk(torch.zeros(2, 8), torch.zeros(2, 8), None, 2)
except ValueError:
    print("refused")
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parents[1],
                          capture_output=True, text=True, timeout=300)
    assert done.stdout == "refused\n", done.stderr[-2000:]


def test_calls_run_on_their_operands_device(monkeypatch):
    """With another device current, the call is made with the operands' device
    current and on its current stream; a failing status raises."""
    from kernelswift_b200 import fused_moe as fm

    current, seen = [0], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.before

    status = [0]
    monkeypatch.setattr(fm, "_get_device", lambda: current[0])
    monkeypatch.setattr(fm, "_raw_stream", lambda index: 100 + index)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setitem(fm._bound, "moe_fp8_matmul",
                        lambda *a: seen.append((current[0], a)) or status[0])
    fm._enqueue("moe_fp8_matmul", 1, "x")
    fm._enqueue("moe_fp8_matmul", 0, "y")
    assert seen == [(1, ("x", 101)), (0, ("y", 100))] and current == [0]
    status[0] = INVALID
    with pytest.raises(_lib.MoeError):
        fm._enqueue("moe_fp8_matmul", 1, "z")
    assert current == [0]


def apart(out, addend):
    """Whether fp8 takes `addend` for `out`."""
    try:
        fp8._addend(addend, *out.shape, out.dtype, -1, out)
    except ValueError:
        return False
    return True


def test_a_single_row_or_column_in_place():
    """The strides of one row, or one column, mean nothing."""
    buf = torch.zeros(8, 80)
    one = buf[:1, :64]
    assert apart(one, one) and apart(one, buf[0, :64].unsqueeze(0))  # strides 80 and 64
    assert apart(one, buf[0, 64:].repeat(4)[None]) and not apart(one, buf[0, 1:65].unsqueeze(0))
    row = torch.as_strided(buf, (1, 64), (0, 1), 0)
    assert apart(row, row) and apart(row, one) and apart(one, row)
    assert not apart(row, torch.as_strided(buf, (1, 64), (0, 1), 63))
    assert apart(row, torch.as_strided(buf, (1, 64), (0, 1), 64))
    column = torch.as_strided(buf, (8, 1), (80, 8), 3)
    assert apart(column, column) and apart(column, buf[:, 3:4]) and apart(column, buf[:, 4:5])
    assert not apart(column, torch.as_strided(buf, (8, 1), (40, 1), 3))


def test_overlaps_are_refused():
    """Every accepted pair of layouts is the same elements or shares none; the
    same elements, columns of one matrix and runs behind each other are accepted."""
    import random

    rng, buf = random.Random(5), torch.zeros(400)
    taken = 0
    for _ in range(4000):
        rows, cols = rng.choice((1, 1, 2, 3, 5)), rng.choice((1, 2, 4, 7))
        def view():
            strides = (rng.choice((0, cols, cols, cols + 1, 2 * cols, 16)), rng.choice((1, 1, 1, 3)))
            return torch.as_strided(buf, (rows, cols), strides, rng.randint(0, 40))
        out, addend = view(), view()
        if rows > 1 and out.stride(0) < cols or cols > 1 and out.stride(1) != 1:
            continue  # not an output
        cells = []
        for t in (out, addend):
            cells.append([t.storage_offset() + r * t.stride(0) + c * t.stride(1)
                          for r in range(rows) for c in range(cols)])
        if apart(out, addend):
            taken += 1
            assert cells[0] == cells[1] or not set(cells[0]) & set(cells[1])
        else:
            dense = (rows == 1 or addend.stride(0) >= cols) and (cols == 1 or addend.stride(1) == 1)
            assert not dense or cells[0] != cells[1]
    assert taken > 500


@pytest.mark.parametrize("fmt", ["fp32", "ue8m0"])
def test_plan_covers_the_product(fmt):
    """Every plan's tiles cover the output, K splits leave no CTA empty and
    clusters stay within 8 CTAs."""
    for T in (1, 2, 15, 16, 17, 64, 100, 128, 129, 300, 1000, 4096, 16384):
        for N in (1, 100, 576, 4096, 7168, 100000):
            for K in (1, 100, 1024, 2048, 7168, 20000):
                p = fp8.block_matmul_plan(T, N, K, fmt)
                kb = -(-K // 128)
                assert 1 <= p["splits"] <= min(8, kb)
                assert p["tile_cols"] in (16, 32, 64, 128, 256)
                if p["cta_pairs"]:
                    tiles = 2 * (-(-T // 256) * -(-N // 256))
                else:
                    tiles = -(-T // p["tile_cols"]) * -(-N // 128)
                if p["splits"] > 1:
                    assert p["ctas"] == tiles * p["splits"]
                else:
                    assert 1 <= p["ctas"] <= min(tiles, 296)
    assert fp8.block_matmul_plan(0, 64, 64, fmt)["ctas"] == 0


def plan_of(T, N, K, fmt):
    p = fp8.block_matmul_plan(T, N, K, fmt)
    return p["cta_pairs"], p["tile_cols"], p["splits"]


def test_listed_sizes_take_their_plans():
    for fmt, plan, size in CASES:
        assert plan_of(*size, fmt) == plan, (fmt, size)
        T, N, K = size
        assert T % (256 if plan[0] else plan[1]) and N % (256 if plan[0] else 128) and K % 128


@pytest.mark.parametrize("fmt", ["fp32", "ue8m0"])
def test_no_plan_goes_unlisted(fmt):
    """Every plan that sizes drawn over the whole range take is one that the GPU
    tests run."""
    import math
    import random

    rng, seen = random.Random(2), set()

    def draw(lo, hi):
        return int(math.exp(rng.uniform(math.log(lo), math.log(hi))))

    for _ in range(60000):
        seen.add(plan_of(draw(1, 30000), draw(1, 60000), draw(1, 60000), fmt))
    assert seen == set(PLANS[fmt])


def test_oracle_roundings():
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    every = every[~every.isnan()]
    assert torch.equal(orc.e4m3_nearest(every), every)
    v = torch.randn(10000, generator=torch.Generator().manual_seed(0)).double() * 100
    assert torch.equal(orc.e4m3_nearest(v), v.clamp(-448, 448).to(torch.float8_e4m3fn).double())
    q, s = orc.fp8_rows(torch.tensor([[448.0, 1.0], [449.0, 0.0], [0.0, 0.0]]), "ue8m0")
    assert s.tolist() == [[1.0], [2.0], [1.0]]
    assert q.tolist() == [[448.0, 1.0], [224.0, 0.0], [0.0, 0.0]]
