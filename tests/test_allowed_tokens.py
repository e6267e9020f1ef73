"""Sets of allowed tokens: what is a mask and what is ids, from the caller to the step."""

import numpy as np
import pytest

from host_engine import allowed_by, host_engine
from socrates_b200.sampling import AllowedMask, pack_allowed
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
