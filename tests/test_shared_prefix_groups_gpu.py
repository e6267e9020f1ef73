"""Attention over a shared prefix with more groups than members, and with values that only some members see."""

import math

import pytest
import torch

from socrates_b200.kernels import KernelError, ops
from test_several_answers_gpu import PAGE, Case, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads", [(32, 8, 128), (4, 2, 16), (12, 4, 96), (20, 1, 128)], ids=str)
@pytest.mark.parametrize("families,spare", [([(0, []), (32, [1, 40]), (16, []), (0, []), (48, []), (0, [])], 6),
                                            ([(16, [])] * 20 + [(3300, [1] * 20)] + [(32, [])] * 20 + [(0, [7])], 40),
                                            ([(16, [])] * 150 + [(64, [3])] + [(16, [])] * 450, 700)], ids=["two", "twenty", "one_of_601"])
def test_more_groups_than_members(families, spare, heads, dtype):
    """Groups may be empty anywhere, as many as there are tokens; scratch is allocated by the call, or by its size."""
    case = Case(families, *heads, dtype, spare_tokens=spare)
    want = case.want()
    check(case, case.run(), want)
    M, R = len(case.members), len(case.lens)
    assert M < R <= case.N
    floats, counts = ops.attention_shared_scratch_size(M, *heads, PAGE, dtype, R)
    part, lists = torch.full((floats,), math.nan, device="cuda"), torch.full((counts,), -9, dtype=torch.int32, device="cuda")
    check(case, case.run(part=part, lists=lists), want)
    assert ops.attention_shared_scratch_size(M, *heads, PAGE, dtype) == ops.attention_shared_scratch_size(M, *heads, PAGE, dtype, M)


def test_more_groups_than_tokens_are_refused():
    case = Case([(16, [])] * 3 + [(32, [1, 2])], 8, 2, 32, torch.bfloat16)
    with pytest.raises(KernelError):
        case.run()
