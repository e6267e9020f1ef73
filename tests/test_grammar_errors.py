"""A grammar that raises, or names a token that there is not, ends its own request and no other."""

import numpy as np
import pytest

from host_engine import host_engine
from socrates_b200.sampling import AllowedMask
from test_scheduler import VOCAB, expected_output

BAD = {"raises": lambda: [][0], "beyond the vocabulary": lambda: [3, VOCAB], "negative": lambda: [-1], "no set": lambda: 7,
       "another vocabulary's mask": lambda: np.ones(7, np.int32).view(AllowedMask)}


@pytest.mark.parametrize("at", [0, 3])
@pytest.mark.parametrize("bad", BAD.values(), ids=BAD)
def test_a_bad_grammar_ends_its_request_alone(bad, at):
    e = host_engine()
    before, asked = e.submit([9, 8, 7], 12), []

    def grammar(out):
        asked.append(len(out))
        return range(1, VOCAB) if len(out) < at else bad()

    req = e.submit([5, 6], 12, stream=True, allowed=grammar)
    after = e.submit([4, 4], 12)
    e.run()
    assert req.done and req.error is not None and len(req.output) == at and req.event.is_set()
    assert [req.stream.get_nowait() for _ in range(at + 1)] == req.output + [None]
    assert asked == list(range(at + 1))                     # once a step, and not again when it has failed
    for other, ids in ((before, [9, 8, 7]), (after, [4, 4])):
        assert other.error is None and other.output == expected_output(ids, 12)
    e.cache.check()
    assert e.cache.free_pages() == [64]


def test_a_grammar_that_fails_for_one_answer():
    e = host_engine()
    calls = []

    def grammar(out):
        calls.append(1)
        if len(calls) == 4:
            raise RuntimeError("once")
        return range(1, VOCAB)

    reqs = e.submit_answers([5, 6], 3, 4, allowed=grammar)
    e.run()
    failed = [r for r in reqs if r.error is not None]
    assert len(failed) == 1 and all(len(r.output) == 4 for r in reqs if r.error is None)


def test_generate_raises_what_a_grammar_raised_when_all_are_done():
    e = host_engine()
    for n in (1, 2):
        with pytest.raises(KeyError, match="lost"):
            e.generate([[5, 6], [7, 8]], 4, n=n, allowed=lambda out: {}["lost"] if len(out) == 2 else range(1, VOCAB))
        assert not e.scheduler.has_work()
    assert len(e.generate([[5, 6]], 4, allowed=range(1, VOCAB))[0]) == 4
