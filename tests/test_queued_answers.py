"""Answers of one prompt: queued all or none, whatever other threads do at the queue's door, and forked where a fork has what they need."""

import sys
import threading

import pytest

from host_engine import host_engine
from socrates_b200 import QueueFull, TooLong
from socrates_b200.engine.scheduler import Request
from socrates_b200.sampling import SamplingParams
from test_scheduler import expected_output


def test_answers_are_queued_all_or_none_beside_other_threads():
    every = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        for _ in range(60):
            e, taken, start = host_engine(max_queue=7), [], threading.Barrier(4)

            def put(first):
                start.wait()
                try:
                    taken.append(e.submit_answers([first, 5, 6], 3, 4))
                except QueueFull:
                    pass

            threads = [threading.Thread(target=put, args=(i,)) for i in range(1, 5)]
            for t in threads:
                t.start()
            for t in threads:
                t.join()
            waiting = list(e.scheduler.pending)
            assert len(taken) == 2 and len(waiting) == 6    # seven places hold two prompts' answers
            for i in (0, 3):                                # together, and somebody's
                assert any(all(a is b for a, b in zip(reqs, waiting[i:i + 3])) for reqs in taken)
    finally:
        sys.setswitchinterval(every)


def test_refused_answers_leave_the_queue_alone():
    e = host_engine(max_queue=3)
    with pytest.raises(QueueFull):
        e.submit_answers([1, 2], 4, 3)
    with pytest.raises(TooLong):
        e.submit_answers([1] * 250, 2, 30)
    assert not e.scheduler.pending
    reqs = e.submit_answers([1, 2], 3, 3)
    with pytest.raises(QueueFull):
        e.submit([1, 2])
    assert list(e.scheduler.pending) == reqs and all(r.siblings == reqs for r in reqs)


@pytest.mark.parametrize("first,second,forked", [(1.0, 1.0, True), (1.5, 1.5, True), (1.5, 1.0, True), (1.0, 1.5, False)])
def test_a_row_whose_tokens_are_not_kept_has_no_penalized_fork(first, second, forked):
    e = host_engine()
    reqs = [Request([5, 6, 7], 4, SamplingParams(repetition_penalty=r)) for r in (first, second)]
    for r in reqs:
        r.siblings = reqs
        e.scheduler.submit(r)
    assert e.step() and e.step()
    assert (e.cache.family[reqs[1].row] > 0) == forked
    e.run()
    assert all(r.output == expected_output([5, 6, 7], 4) for r in reqs)
