"""Forks of cache rows and answers of one prompt, on the host."""

import random

import numpy as np
import pytest
import torch

from socrates_b200.cache import CacheManager, CacheNeeds, PageAllocator, PagedKVSpec, StateSpec
from socrates_b200.engine.scheduler import Request, Scheduler
from socrates_b200.kernels.library import library
from socrates_b200.sampling import MAX_BIASES, SamplingParams, pack_allowed
from test_scheduler import STOP, VOCAB, FakeEngine, next_token


# ------------------------------------------------------------------ pages with several holders
def test_allocator_counts_holders():
    a = PageAllocator(4)
    assert a.alloc(2) == [1, 2] and a.holders(1) == 1 and a.holders(3) == 0
    a.share([1])
    a.share([1, 2])
    assert a.holders(1) == 3 and a.holders(2) == 2 and a.n_used == 2
    a.check()
    a.free([1, 2])
    assert a.holders(1) == 2 and a.holders(2) == 1 and a.n_free == 2
    a.free([1])
    a.free([2, 1])
    assert a.n_free == 4 and a.holders(1) == 0
    with pytest.raises(ValueError):
        a.free([1])
    for bad in (0, 1, 9, -1):
        with pytest.raises(ValueError):
            a.share([bad])                                  # nobody holds it
    assert a.alloc(1) == [2]
    with pytest.raises(ValueError):
        a.share([2, 3])
    assert a.holders(2) == 1                                # a failed share changes nothing
    with pytest.raises(ValueError):
        a.free([2, 2])
    a.check()


def manager(num_pages=24, max_rows=6, window=None, state=False):
    needs = [CacheNeeds(PagedKVSpec(2, 16, None)), CacheNeeds(PagedKVSpec(1, 16, window), StateSpec((3,)) if state else None)]
    return CacheManager(needs, max_rows, 128, 16, num_pages, torch.float32, "cpu")


def written(m, row, value):
    """Fill the row's pages with numbers of (value, position)."""
    for g in m.groups:
        for pos in range(m.lengths[row]):
            page = int(g.host_table[row, pos // 16])
            if page:
                g.k[:, page, :, pos % 16] = value * 1000 + pos
                g.v[:, page, :, pos % 16] = -(value * 1000 + pos)


@pytest.mark.parametrize("length", [1, 15, 16, 17, 31, 32, 47])
def test_fork_shares_whole_pages_and_copies_the_last(length):
    m = manager()
    m.assign(0)
    assert m.reserve(0, 50)
    m.commit(0, 50)
    written(m, 0, 3)
    before = m.free_pages()
    assert m.can_fork(0, length) and m.fork(0, 2, length)
    m.check()
    m.flush()
    assert m.free_pages() == [n - (length % 16 != 0) for n in before]
    for g in m.groups:
        whole = length // 16
        assert g.row_pages[2][:whole] == g.row_pages[0][:whole]
        if length % 16:
            a, b = g.row_pages[0][whole], g.row_pages[2][whole]
            assert a != b and torch.equal(g.k[:, a], g.k[:, b]) and torch.equal(g.v[:, a], g.v[:, b])
    assert m.lengths[2] == length and m.families([2, 0, 1])[2] == ([length // 16 * 16, 0] if length >= 16 else [0, 0, 0])
    # both go on in pages of their own
    assert m.reserve(2, length + 20) and m.reserve(0, 60)
    for g in m.groups:
        assert not set(g.row_pages[2][length // 16:]) & set(g.row_pages[0])
    m.check()
    m.release(0)
    m.check()
    assert m.lengths[2] == length
    m.release(2)
    m.check()
    assert m.free_pages() == [24, 24]


def test_forks_of_forks_moves_and_families():
    m = manager(num_pages=40)
    m.assign(0)
    assert m.reserve(0, 70)
    m.commit(0, 70)
    assert m.fork(0, 1, 60) and m.fork(1, 2, 40) and m.fork(0, 3, 65)
    m.check()
    assert m.families([0, 1, 2, 3]) == ([0, 1, 2, 3], [0, 4], [32])
    assert m.families([3, 0]) == ([0, 1], [0, 2], [48])     # what the family shares, not what the two might
    assert m.families([2]) == ([0], [0, 1], [0])
    m.assign(4)
    assert m.families([4, 1, 0]) == ([1, 2, 0], [0, 2, 3], [48, 0])
    m.release(0)
    m.move_row(3, 0)
    m.check()
    assert m.families([0, 2]) == ([0, 1], [0, 2], [32]) and m.family[3] == 0
    assert not m.can_fork(3, 5) and not m.can_fork(0, 66) and not m.can_fork(0, 0)
    with pytest.raises(ValueError):
        m.fork(0, 1, 10)                                    # in use
    with pytest.raises(ValueError):
        m.fork(0, 5, 90)                                    # longer than the row
    for r in (0, 1, 2, 4):
        m.release(r)
    m.check()
    assert m.free_pages() == [40, 40]


def test_fork_without_a_free_page_changes_nothing():
    m = manager(num_pages=3)
    m.assign(0)
    assert m.reserve(0, 48)
    m.commit(0, 48)
    assert not m.fork(0, 1, 47)
    assert not m.active[1] and m.families([0])[2] == [0]
    m.check()
    assert m.fork(0, 1, 32)                                 # whole pages need none
    m.check()


def test_forks_of_windowed_rows_and_of_state():
    m = manager(window=20)
    m.assign(0)
    assert m.reserve(0, 64)
    m.commit(0, 64)                                         # the windowed group holds positions 45 and up: blocks 2 and 3
    assert not m.can_fork(0, 40) and m.can_fork(0, 60)
    assert m.fork(0, 1, 60)
    m.check()
    win = m.groups[1]
    assert win.row_pages[1][:2] == [0, 0] and win.row_pages[1][2] == win.row_pages[0][2] and win.row_pages[1][3] != win.row_pages[0][3]
    assert m.reserve(0, 100)
    m.commit(0, 100)                                        # row 0 gives block 2 back; row 1 holds it still
    m.check()
    assert win.allocator.holders(win.row_pages[1][2]) == 1
    m.release(1)
    m.release(0)
    m.check()

    m = manager(state=True)
    m.assign(0)
    assert m.reserve(0, 20)
    m.commit(0, 20)
    m.state(1)[0] = 7.0
    assert not m.can_fork(0, 19) and m.fork(0, 1, 20)       # the state is the one behind all 20 tokens
    assert bool((m.state(1)[1] == 7.0).all())


def test_copies_that_wait_follow_their_pages():
    """Between a fork and the flush that makes its copy, pages leave and come back."""
    m = manager(num_pages=6, max_rows=6)
    m.assign(0)
    assert m.reserve(0, 20)
    m.commit(0, 20)
    written(m, 0, 1)
    assert m.fork(0, 1, 18)
    m.release(1)                                            # nobody wants the copy any more
    assert all(not g.copies for g in m.groups)
    assert m.fork(0, 1, 18) and m.fork(1, 2, 17)            # the second goes back to the page that is written
    m.check()
    m.release(0)                                            # its last page may become a copy of another one
    m.assign(3)
    assert m.reserve(3, 10)
    m.commit(3, 10)
    assert m.fork(3, 4, 5)
    m.flush()
    m.check()
    for g in m.groups:
        for row, n in ((1, 18), (2, 17)):
            page = g.row_pages[row][1]
            assert g.k[0, page, 0, :n - 16, 0].tolist() == [1000.0 + p for p in range(16, n)]


# ------------------------------------------------------------------ the scheduler
class Answers(FakeEngine):
    """FakeEngine that knows forks: a row that is opened as one holds the prompt but for its last token."""

    forks = 0

    def submit_answers(self, ids, n, max_new=8):
        reqs = [Request(ids=list(ids), max_new_tokens=max_new, sampling=SamplingParams(seed=i)) for i in range(n)]
        for r in reqs:
            self.s.submit(r)
            r.siblings = reqs
        return reqs

    def step(self):
        plan = self.s.plan
        def planned():
            p = plan()
            for e in (p.entries if p is not None else ()):
                if e.start and id(e.request) not in self.fed:
                    self.forks += 1
                    assert e.start == len(e.request.ids) - 1 and self.cache.family[e.row]
                    self.fed[id(e.request)] = list(e.request.ids[:-1])
            return p
        self.s.plan = planned
        try:
            return super().step()
        finally:
            del self.s.plan


def expected(ids, max_new):
    seq, out = list(ids), []
    while len(out) < max_new:
        t = next_token(seq)
        if t == STOP:
            break
        out.append(t)
        seq.append(t)
    return out


@pytest.mark.parametrize("window", [None, 20])
@pytest.mark.parametrize("seed", range(4))
def test_answers_do_not_depend_on_forks(seed, window):
    rng = random.Random(seed)
    e = Answers(num_pages=40 if seed else 200, max_batch=5, budget=rng.choice([7, 32, 100]), window=window)
    groups = []
    for _ in range(6):
        ids = [rng.randrange(1, VOCAB) for _ in range(rng.choice([1, 2, 16, 17, rng.randint(3, 70)]))]
        groups.append((ids, e.submit_answers(ids, rng.randint(1, 6), rng.randint(1, 14))))
    e.run()
    for ids, reqs in groups:
        for r in reqs:
            assert r.done and r.output == expected(ids, r.max_new_tokens)
    assert e.forks > 0 and set(e.cache.free_pages()) == {40 if seed else 200}
    e.cache.check()


def test_answers_wait_for_their_prompt_and_others_pass():
    e = Answers(max_batch=4, budget=16)
    long = [1 + i % 40 for i in range(60)]
    answers = e.submit_answers(long, 3, 4)
    other = e.submit([5, 6, 7], 4)
    e.step()                                                # the first 16 tokens of the prompt: nothing is left of the budget
    e.step()
    assert answers[0].row >= 0 and answers[1].row < 0 and answers[2].row < 0
    while answers[0].cached < 59:
        e.step()
    assert other in e.s.pending or other.row >= 0 or other.done
    e.run()
    assert e.forks == 2 and all(r.output == expected(long, 4) for r in answers) and other.output == expected([5, 6, 7], 4)


def test_an_answer_whose_siblings_are_gone_computes_the_prompt():
    e = Answers(max_batch=1)
    reqs = e.submit_answers([3, 4, 5, 6], 3, 3)
    e.run()
    assert e.forks == 0 and all(r.output == expected([3, 4, 5, 6], 3) for r in reqs)


# ------------------------------------------------------------------ sampling parameters
def test_params_are_checked():
    SamplingParams(0.5, 1, 1.2, -0.1, 0.3, {3: 2.0, 4: -float("inf")}, [1, 2]).validate(10)
    for bad in (dict(repetition_penalty=0.0), dict(repetition_penalty=float("nan")), dict(presence_penalty=float("inf")),
                dict(frequency_penalty=float("nan")), dict(logit_bias={10: 1.0}), dict(logit_bias={-1: 1.0}),
                dict(logit_bias={1: float("nan")}), dict(logit_bias={1: float("inf")}), dict(allowed=[]), dict(allowed=[10]),
                dict(allowed=[-1]), dict(logit_bias={i: 0.0 for i in range(MAX_BIASES + 1)}), dict(temperature=-1.0)):
        with pytest.raises(ValueError):
            SamplingParams(**bad).validate(10 if "logit_bias" not in bad or len(bad["logit_bias"]) == 1 else 10 ** 6)
    assert not SamplingParams(0.7).adjusts and SamplingParams(allowed=[1]).adjusts and SamplingParams(presence_penalty=0.1).penalizes


@pytest.mark.parametrize("bad", [dict(repetition_penalty=1e-46), dict(repetition_penalty=1e-40), dict(repetition_penalty=1e39),
                                 dict(presence_penalty=1e39), dict(frequency_penalty=-1e39), dict(logit_bias={1: 1e39}),
                                 dict(logit_bias={1: -1e39})], ids=str)
def test_numbers_that_float32_does_not_hold_are_refused(bad):
    with pytest.raises(ValueError):
        SamplingParams(**bad).validate(10)


@pytest.mark.parametrize("vocab", [1, 31, 32, 33, 100])
def test_masks(vocab):
    ids = sorted({0, vocab - 1, vocab // 2})
    mask = pack_allowed(ids, vocab)
    assert mask.dtype == np.int32 and mask.shape == (-(-vocab // 32),)
    assert [t for t in range(vocab) if (int(mask[t // 32]) >> (t % 32)) & 1] == ids
    assert np.array_equal(pack_allowed(mask, vocab), mask) and np.array_equal(pack_allowed(iter(ids), vocab), mask)
    assert pack_allowed([], vocab) is None and pack_allowed(np.zeros_like(mask), vocab) is None
    behind = np.zeros_like(mask)
    behind[-1] = -1 << (vocab % 32) if vocab % 32 else 0    # bits behind the vocabulary allow nothing
    assert pack_allowed(behind, vocab) is None


# ------------------------------------------------------------------ refusals at the C entries, before any device is touched
def test_c_entries_refuse():
    from array import array
    lib, p = library(), 0x10000                             # an address that is never followed

    def copy(src, dst, runs=2, pages=6, kb=1024, vb=1024, k=p):
        a, b = array("i", src), array("i", dst)
        return lib.sb_copy_pages(k, p, a.buffer_info()[0], b.buffer_info()[0], len(src), runs, pages, kb, vb, None)

    for bad in (([1], [6]), ([6], [1]), ([-1], [2]), ([1, 2], [3, 3]), ([1, 2], [2, 3]), ([1], [1])):
        assert copy(*bad) == 100001
    many = list(range(40))
    assert copy(many, [40 + i for i in range(39)] + [40], pages=100) == 100001          # twice, found in the map
    assert copy(many, [40 + i for i in range(39)] + [0], pages=100) == 100001           # read and written
    assert copy(many, many, pages=30) == 100001 and copy([1], [2], kb=3) == 100001 and copy([1], [2], runs=0) == 100001
    assert copy([1], [2], kb=0) == 100001 and copy([1], [2], k=None) == 100001 and copy([], []) == 0

    def attention(**kw):
        a = dict(out=p, part=p, floats=1 << 40, lists=p, ints=1 << 30, q=p, k=p, v=p, pages=10, table=p, width=4, rows=p, pos=p,
                 members=p, M=2, starts=p, lens=p, R=1, N=2, Hq=4, Hkv=2, D=64, BS=16, window=0, scale=1.0, dtype=1, status=None, stream=None)
        return lib.sb_attention_shared(*{**a, **kw}.values())

    for bad in (dict(Hq=3), dict(Hkv=0), dict(D=24), dict(D=272), dict(D=0), dict(BS=0), dict(width=0), dict(window=-1), dict(M=3),
                dict(M=0), dict(R=0), dict(R=3), dict(N=0), dict(dtype=2), dict(part=None), dict(floats=10), dict(ints=3),
                dict(q=p + 2), dict(lists=None), dict(dtype=0, floats=10)):
        assert attention(**bad) == 100001, bad

    def sample(**kw):
        a = dict(out=p, logits=p, t=None, seeds=None, counters=None, M=2, V=100, scratch=p, ints=1000, history=None, width=0, rows=None,
                 prompt=None, lengths=None, penalties=None, starts=None, ids=None, values=None, mask=None, words=0, mask_rows=None,
                 adjusted=None, stream=None)
        return lib.sb_sample_adjusted(*{**a, **kw}.values())

    for bad in (dict(V=0), dict(M=-1), dict(V=262145), dict(t=p), dict(scratch=None), dict(ints=11), dict(penalties=p),
                dict(penalties=p, history=p, width=0, rows=p, prompt=p, lengths=p), dict(starts=p), dict(mask=p, words=4),
                dict(mask=p, words=3, mask_rows=p)):
        assert sample(**bad) == 100001, bad
    assert sample(M=0) == 0
    assert lib.sb_note_tokens(p, 0, 4, p, p, p, 1, None, 0, None) == 100001 and lib.sb_note_tokens(p, 2, 4, p, p, p, 0, None, 0, None) == 0


@pytest.mark.parametrize("scale", [0.0, -0.125, float("nan"), float("inf")])
def test_attention_shared_refuses_scales_that_turn_masks_round(scale):
    lib, p = library(), 0x10000
    assert lib.sb_attention_shared(p, p, 1 << 40, p, 1 << 30, p, p, p, 10, p, 4, p, p, p, 2, p, p, 1, 2, 4, 2, 64, 16, 0, scale, 1,
                                   None, None) == 100001


def test_shapes_that_the_engine_reads_shared_keys_with():
    """The tensor-core kernels' shapes, and head sizes up to 128 that have no tensor-core kernel for rows one by one."""
    from socrates_b200.kernels import ops
    from socrates_b200.parts.attention import reads_shared_keys
    good = dict(members=64, num_heads=32, num_kv_heads=8, head_dim=128, page_size=16)
    assert ops.attention_shared_supports(**good) and reads_shared_keys(**good)
    for other in (dict(head_dim=24), dict(head_dim=96), dict(num_heads=136), dict(num_heads=33)):
        assert not ops.attention_shared_supports(**{**good, **other}) and reads_shared_keys(**{**good, **other}), other
    for bad in (dict(head_dim=256), dict(page_size=8), dict(members=513)):
        assert not ops.attention_shared_supports(**{**good, **bad}) and not reads_shared_keys(**{**good, **bad}), bad
    for wrong in (dict(members=0), dict(num_kv_heads=0)):
        assert not ops.attention_shared_supports(**{**good, **wrong})
