"""Steps with and without adjusted logits side by side: what is recorded stays recorded, and rows keep their own tokens."""

import gc

import pytest
import torch

from socrates_b200 import Engine
from tiny_configs import make_folder

pytestmark = pytest.mark.gpu


def prompt(n, seed=0, vocab=256):
    return torch.randint(1, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("kw", [dict(logit_bias={3: 1.0}), dict(allowed=range(3, 200)), dict(repetition_penalty=1.2)], ids=str)
def test_warmed_steps_stay_recorded_behind_adjusted_ones(tmp_path, kw):
    """Only penalties look at the rows' tokens, and steps without them launch what they did before."""
    folder = str(make_folder(tmp_path, "A"))
    eng = Engine(folder, dtype="float32", max_batch=3, max_len=128, token_budget=32, warmup=True)
    warmed = dict(eng.runner._graphs)

    def plain_answers():
        steps, launches = eng.runner.steps_run, eng.runner.kernel_launches
        out = eng.generate([prompt(20), prompt(7, 1)], 10)
        return out, eng.runner.steps_run - steps, eng.runner.kernel_launches - launches

    before = plain_answers()
    assert eng.runner._graphs.keys() == warmed.keys()
    eng.generate([prompt(9, 2), prompt(8, 3)], 8, **kw)
    assert (eng.cache.tokens is not None) == ("repetition_penalty" in kw)
    new = eng.runner._graphs.keys() - warmed.keys()
    assert new and all("adjust" in key and ("penalize" in key) == ("repetition_penalty" in kw) for key in new)
    assert plain_answers() == before
    assert eng.runner._graphs.keys() - warmed.keys() == new
    assert all(eng.runner._graphs[key][0] is graph[0] for key, graph in warmed.items())


def test_a_penalized_request_is_sampled_from_its_own_tokens_beside_others(tmp_path):
    """Steps of plain requests alone note nothing; rows that such steps used before are taken over by penalized ones, and rows move."""
    folder = str(make_folder(tmp_path, "A"))
    kw, ask = dict(dtype="float32", max_batch=3, max_len=128, token_budget=32), dict(repetition_penalty=3.0, frequency_penalty=0.5)
    want = [Engine(folder, **kw).generate([prompt(12, i)], 16, 0.5, i, **ask)[0] for i in range(2)]
    eng = Engine(folder, **kw)
    late = [eng.submit(prompt(12, 0), 16, 0.5, 0, **ask)]
    plain = [eng.submit(prompt(30, 7), 4), eng.submit(prompt(6, 8), 30)]
    eng.run()                                               # (the last of them goes on without a penalized request)
    plain += [eng.submit(prompt(9, 9), 5), eng.submit(prompt(8, 10), 12)]
    for _ in range(4):
        eng.step()
    late.append(eng.submit(prompt(12, 1), 16, 0.5, 1, **ask))
    eng.run()
    assert [r.output for r in late] == want
    lone = Engine(folder, **kw)
    for r, (ids, new) in zip(plain, ((prompt(30, 7), 4), (prompt(6, 8), 30), (prompt(9, 9), 5), (prompt(8, 10), 12))):
        assert r.output == lone.generate([ids], new)[0]


def test_bad_grammars_beside_other_requests(tmp_path):
    folder = str(make_folder(tmp_path, "A"))
    kw = dict(dtype="float32", max_batch=3, max_len=128, token_budget=32)
    eng = Engine(folder, **kw)
    free = eng.submit(prompt(12, 4), 12)
    raises = eng.submit(prompt(20), 12, 0.8, 3, allowed=lambda out: range(48, 58) if len(out) < 3 else 1 // 0)
    beyond = eng.submit(prompt(5), 12, allowed=lambda out: None if len(out) < 2 else [256])
    eng.run()
    assert isinstance(raises.error, ZeroDivisionError) and len(raises.output) == 3 and all(48 <= t < 58 for t in raises.output)
    assert isinstance(beyond.error, ValueError) and len(beyond.output) == 2 and beyond.done and beyond.event.is_set()
    assert free.error is None and free.output == Engine(folder, **kw).generate([prompt(12, 4)], 12)[0]
    assert set(eng.cache.free_pages()) == {eng.num_blocks}


def test_a_warm_up_beside_live_requests_is_refused(tmp_path):
    folder = str(make_folder(tmp_path, "A"))
    kw = dict(dtype="float32", max_batch=3, max_len=128, token_budget=32)
    ask = dict(temperature=0.0, repetition_penalty=3.0)
    want = Engine(folder, **kw).generate([prompt(12)], 16, **ask)[0]
    eng = Engine(folder, **kw)
    req = eng.submit(prompt(12), 16, **ask)
    for _ in range(4):
        eng.step()
    with pytest.raises(RuntimeError, match="live"):
        eng.warmup()
    eng.run()
    assert req.output == want
    eng.warmup()                                            # nobody is live: nothing is disturbed
    assert eng.generate([prompt(12)], 16, **ask)[0] == want


def test_garbage_with_recorded_steps_does_not_end_a_recording(tmp_path, monkeypatch):
    """What collects garbage while a step is recorded (any allocation may) would reset the recorded steps of an engine that is among
    it, which is not permitted then."""
    folder = str(make_folder(tmp_path, "A"))
    kw = dict(dtype="float32", max_batch=2, max_len=64, token_budget=16)
    eng = Engine(folder, **kw)
    want = Engine(folder, **kw).generate([prompt(9)], 12)
    gc.disable()
    try:
        old = Engine(folder, **kw)
        assert old.generate([prompt(9)], 12) == want and old.runner._graphs
        old.itself = old
        del old
        forward, recorded = type(eng.model).forward, []

        def collecting(self, ctx, cache):
            if torch.cuda.is_current_stream_capturing():
                recorded.append(1)
                if gc.isenabled():
                    gc.collect()
            return forward(self, ctx, cache)

        monkeypatch.setattr(type(eng.model), "forward", collecting)
        gc.enable()
        gc.freeze()                                         # young garbage waits for the collection above
        gc.unfreeze()
        assert eng.generate([prompt(9)], 12) == want and recorded and gc.isenabled()
    finally:
        gc.enable()
