"""The penalty for repeated tokens is the formula's quotient, rounded once."""

import pytest
import torch

from socrates_b200.kernels import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [1000, 20001])
def test_repetition_divides(V):
    """l / r of two float32 numbers has one nearest float32 number, and so has l * r: nothing may be off by a bit."""
    g = torch.Generator().manual_seed(V)
    M, W = 6, 4000
    logits = 5 * torch.randn(M, V, generator=g)
    r = torch.tensor([1.1, 1.3, 0.7, 3.0, 1.000001, 1e-3])
    told = torch.randint(0, V, (M, W), generator=g).to(torch.int32)
    met = torch.zeros(M, V, dtype=torch.bool).scatter_(1, told.long(), True)
    want = torch.where(met, torch.where(logits > 0, logits / r[:, None], logits * r[:, None]), logits)
    out, new = torch.zeros(M, dtype=torch.int32, device="cuda"), torch.empty(M, V, device="cuda")
    each = lambda values: torch.tensor(values, dtype=torch.int32, device="cuda")  # noqa: E731
    ops.sample_adjusted(out, logits.cuda(), history=told.cuda(), history_rows=each(list(range(M))), prompt_lens=each([W // 2] * M),
                        lengths=each([W] * M), penalties=torch.stack([r, torch.zeros(M), torch.zeros(M)], 1).cuda(), adjusted=new)
    assert torch.equal(new.cpu(), want) and torch.equal(out.cpu().long(), want.argmax(1))
