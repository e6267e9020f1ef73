"""Answers that are drawn, so that rows behind a shared prefix differ, against the plain implementation token by token."""

import pytest
import torch

import plain_qwen3 as plain
from socrates_b200 import Engine
from socrates_b200.engine.runner import ModelRunner
from socrates_b200.parts import attention
from test_engine_gpu import check_teacher_forced
from tiny_configs import make_folder

pytestmark = pytest.mark.gpu


def prompt(n, seed=0, vocab=256):
    return torch.randint(1, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("extra", [dict(), dict(compile=False), dict(run_ahead=False, warmup=True), dict(num_blocks=24)], ids=str)
@pytest.mark.parametrize("length", [70, 33, 96])
def test_drawn_answers_of_a_family_are_the_plain_implementations(tmp_path, monkeypatch, length, extra):
    """bfloat16, shared keys read once: each drawn token has the best plain score (logit / T + noise) up to bfloat16's gap."""
    monkeypatch.setattr(attention, "SHARED_PAYS_FROM", 1)
    folder = make_folder(tmp_path, "A")
    cfg, w = plain.load_folder(folder)
    eng = Engine(str(folder), dtype="bfloat16", max_batch=6, max_len=128, token_budget=64, **extra)
    steps = []
    families = ModelRunner._families
    monkeypatch.setattr(ModelRunner, "_families", lambda self, entries: steps.append(families(self, entries)[0]) or families(self, entries))
    ids = prompt(length)
    answers = eng.generate([ids], 20, temperature=0.7, seed=11, n=6)[0]
    assert sum(f is not None for f in steps) >= 10          # most steps read the prompt's keys once
    assert len(set(map(tuple, answers))) > 1
    for i, a in enumerate(answers):
        assert len(a) == 20
        check_teacher_forced(cfg, w, ids, a, 2e-2, temperature=0.7, seed=11 + i)
    # what the check can tell: another prefix of as many tokens, or another answer's noise, are not what was computed
    for wrong, seed in ((prompt(length, 1), 11), (ids, 12)):
        with pytest.raises(AssertionError):
            for i, a in enumerate(answers):
                check_teacher_forced(cfg, w, wrong, a, 2e-2, temperature=0.7, seed=seed + i)
