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


@pytest.mark.parametrize("window", [0, 60])
@pytest.mark.parametrize("heads,dtype", [((8, 2, 32), torch.float32), ((32, 8, 128), torch.float32), ((12, 4, 96), torch.bfloat16)], ids=str)
def test_shared_values_that_some_members_see(heads, dtype, window):
    """The kernel on the CUDA cores keeps a value from those who do not see it, whatever it is: behind a token's position, or before
    its window.  (The tensor-core kernels weigh it with 0, so there it has to be finite.)"""
    case = Case([(96, [0, 40, 70])], *heads, dtype, seed=4)
    a, b, c = case.members
    row, at = int(case.token_rows[a]), {0: 90, 60: 40}[window]
    case.positions[a] = 80                                  # sees neither; b and c end at 135 and 165, their windows begin at 76 and 106
    case.v[int(case.table[row, at // PAGE]), :, at % PAGE] = math.inf
    got = case.run(window).double().cpu()
    want = case.want(window)
    sees = [n for n in case.members if at <= int(case.positions[n]) and (not window or at > int(case.positions[n]) - window)]
    assert sees == ([b, c] if not window else [a])
    for n in case.members:
        if n in sees:
            assert not bool(torch.isfinite(got[n]).any())
    others = [n for n in case.members if n not in sees]
    assert bool(torch.isfinite(got[others]).all())
    check(case, got[others], want[others])
