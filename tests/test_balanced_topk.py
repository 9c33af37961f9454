"""CPU: refusals of balanced routing, on the host before any launch, and the
oracle's restatement on cases small enough to check by hand."""
import pytest
import torch

from kernelswift_b200 import _lib
from kernelswift_b200 import fused_moe as fm
from oracle import moe_oracle as orc

F32, BF16, I32, I8 = _lib.DT_F32, _lib.DT_BF16, _lib.DT_I32, _lib.DT_I8


def call(logits_dtype=F32, T=4, E=32, k=2, groups=1, kept=1, group_score=1, scoring=1,
         w_dtype=F32, ids_dtype=I32):
    # the pointers are never followed: every case is refused on the host
    return _lib.load().moe_balanced_topk(0x1000, logits_dtype, None, T, E, k, 1, groups, kept,
                                         group_score, scoring, 1.0, 0x1000, w_dtype, 0x1000,
                                         ids_dtype, None, None)


@pytest.mark.parametrize("bad,status", [
    (dict(T=-1), _lib.MOE_ERR_INVALID_ARG),
    (dict(E=0), _lib.MOE_ERR_UNSUPPORTED),
    (dict(E=1025), _lib.MOE_ERR_UNSUPPORTED),
    (dict(k=0), _lib.MOE_ERR_UNSUPPORTED),
    (dict(k=33, E=64), _lib.MOE_ERR_UNSUPPORTED),
    (dict(k=9, E=8), _lib.MOE_ERR_UNSUPPORTED),
    (dict(groups=5), _lib.MOE_ERR_UNSUPPORTED),
    (dict(groups=33, E=66), _lib.MOE_ERR_UNSUPPORTED),
    (dict(groups=0), _lib.MOE_ERR_UNSUPPORTED),
    (dict(groups=4, kept=5), _lib.MOE_ERR_INVALID_ARG),
    (dict(groups=4, kept=0), _lib.MOE_ERR_INVALID_ARG),
    (dict(groups=4, kept=1, k=9), _lib.MOE_ERR_UNSUPPORTED),
    (dict(group_score=2), _lib.MOE_ERR_INVALID_ARG),
    (dict(scoring=2), _lib.MOE_ERR_INVALID_ARG),
    (dict(w_dtype=I32), _lib.MOE_ERR_INVALID_ARG),
    (dict(ids_dtype=F32), _lib.MOE_ERR_INVALID_ARG),
    (dict(logits_dtype=I8), _lib.MOE_ERR_INVALID_ARG),
])
def test_refused_arguments(bad, status):
    assert call(**bad) == status
    assert "balanced_topk" in _lib.load().moe_last_error().decode()


def test_backward_refuses_a_misaligned_gradient():
    st = _lib.load().moe_balanced_topk_backward(0x1000, F32, 0x1000, I32, 0x1000, 4, 32, 2, 1, 1,
                                                1.0, 0x1004, None)
    assert st == _lib.MOE_ERR_INVALID_ARG


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 8)
    with pytest.raises(ValueError):
        fm.balanced_topk(x, x, None, 2)


def test_oracle_by_hand():
    logits = torch.tensor([[0.0, 1.0, 2.0, 3.0], [0.0, 0.0, 0.0, 0.0]])
    bias = torch.tensor([1.0, 0.0, 0.0, 0.0])
    w, ids = orc.balanced_topk(logits, bias, 2)
    assert ids.tolist() == [[0, 3], [0, 1]]
    s = torch.sigmoid(logits.double())
    assert torch.allclose(w[0], torch.stack([s[0, 0], s[0, 3]]) / (s[0, 0] + s[0, 3]))
    # groups {0, 1} and {2, 3}: by the sum of two 1.5 + 0.73 > 0.88 + 0.95; by the
    # largest 1.5 > 0.95
    _, ids = orc.balanced_topk(logits[:1], bias, 2, num_expert_group=2)
    assert ids.tolist() == [[0, 1]]
    bias = torch.tensor([0.3, -0.5, 0.0, 0.0])  # group 0: 0.8 + 0.23
    _, ids = orc.balanced_topk(logits[:1], bias, 2, num_expert_group=2)
    assert ids.tolist() == [[3, 2]]
