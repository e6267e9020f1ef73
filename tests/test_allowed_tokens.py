"""Sets of allowed tokens: what is a mask and what is ids, from the caller to the step."""

import numpy as np
import pytest

from host_engine import allowed_by, host_engine
from socrates_b200.engine.scheduler import Request
from socrates_b200.sampling import AllowedMask, SamplingParams, pack_allowed
from test_scheduler import STOP, VOCAB


@pytest.mark.parametrize("vocab", [1, 31, 32, 64, 256, 383])
def test_as_many_ids_as_a_mask_has_words_are_ids(vocab):
    words = -(-vocab // 32)
    ids = np.arange(vocab - words, vocab, dtype=np.int32)
    assert ids.shape == (words,)
    assert allowed_by(pack_allowed(ids, vocab), vocab) == ids.tolist()
    assert np.array_equal(pack_allowed(ids, vocab), pack_allowed(ids.tolist(), vocab))


def test_masks_stay_masks():
    a, b = pack_allowed([1, 3, 40], VOCAB), pack_allowed([3, 49], VOCAB)
    assert isinstance(a, AllowedMask) and isinstance(pack_allowed(a, VOCAB), AllowedMask)
    assert allowed_by(pack_allowed(a & b, VOCAB)) == [3] and allowed_by(pack_allowed(a | b, VOCAB)) == [1, 3, 40, 49]
    words = np.array([2 + 8, 1 << 8], dtype=np.int32)
    assert allowed_by(pack_allowed(words.view(AllowedMask), VOCAB)) == [1, 3, 40]
    for wrong in (a[:1], np.concatenate([a, a]).view(AllowedMask), a.astype(np.int64).view(AllowedMask)):
        with pytest.raises(ValueError):
            pack_allowed(wrong, VOCAB)


@pytest.mark.parametrize("form", ["ids", "words", "step by step"])
def test_answers_hold_allowed_tokens_alone(form):
    """A fixed mask is not walked as ids, ids of a mask's length are no mask, and what becomes of the caller's array does not matter."""
    ids = np.array([7, 31], dtype=np.int32) if form != "words" else pack_allowed([7, 31], VOCAB)
    e = host_engine()
    reqs = e.submit_answers([5, 6], 2, 6, allowed=(lambda out: ids) if form == "step by step" else ids)
    if form != "step by step":
        ids[:] = 0
    e.run()
    for r in reqs:
        assert len(r.output) == 6 and set(r.output) <= {7, 31}
    assert STOP not in (7, 31)


@pytest.mark.parametrize("make", [lambda: [7, 31], lambda: iter([7, 31]), lambda: pack_allowed([7, 31], VOCAB), lambda: {7, 31}],
                         ids=["list", "iterator", "mask", "set"])
def test_requests_at_the_schedulers_door_keep_to_their_tokens(make):
    e = host_engine()
    req = e.scheduler.submit(Request([5, 6], 6, SamplingParams(allowed=make())))
    e.run()
    assert len(req.output) == 6 and set(req.output) <= {7, 31}


@pytest.mark.parametrize("bad", [dict(allowed=[VOCAB]), dict(allowed=[]), dict(allowed=iter([-1])), dict(logit_bias={VOCAB: 1.0})], ids=str)
def test_the_schedulers_door_refuses_tokens_that_are_none(bad):
    e = host_engine()
    with pytest.raises(ValueError):
        e.scheduler.submit(Request([5, 6], 6, SamplingParams(**bad)))
    assert not e.scheduler.has_work()


def test_parameters_keep_what_they_were_given():
    bias, mask, ids = {3: 1.0}, pack_allowed([7], VOCAB), [7]
    p, q = SamplingParams(logit_bias=bias, allowed=mask), SamplingParams(allowed=ids)
    bias.clear(), ids.clear()
    mask[:] = 0
    assert p.logit_bias == {3: 1.0} and allowed_by(p.allowed) == [7] and q.allowed == [7]
