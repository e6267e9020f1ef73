"""An Engine whose steps run on the host: the scheduler, the cache manager and Engine's own code are the real ones, the model is
`next_token` of test_scheduler, sampled among the tokens that the step's masks allow."""

from types import SimpleNamespace

import numpy as np
import torch

from socrates_b200.cache import CacheManager, CacheNeeds, PagedKVSpec
from socrates_b200.engine.engine import Engine
from socrates_b200.engine.scheduler import Scheduler
from test_scheduler import STOP, VOCAB, next_token


class HostRunner:
    """Keeps the tokens in the rows' pages and answers a step with the first allowed token from `next_token` on."""

    def __init__(self, cache):
        self.cache, self.sampled, self.steps = cache, [], []

    def place(self, row, pos):
        g = self.cache.groups[0]
        page = int(g.host_table[row, pos // 16])
        assert page
        return g.k[0, page, 0, pos % 16]

    def step(self, entries, sampling=None, ahead=0, **kw):
        self.cache.flush()
        self.steps.append((entries, sampling, kw))
        before, self.sampled = self.sampled, []
        args = iter(sampling)
        for e in entries:
            end = e.start + len(e.tokens)
            for pos, t in zip(range(e.start, end), e.tokens):
                self.place(e.row, pos)[:] = before[-1 - t] if t < 0 else t
            if e.want:
                held = [int(self.place(e.row, pos)[0]) for pos in range(end)]
                mask = getattr(next(args).adjust, "mask", None)
                t = next_token(held)
                while mask is not None and not int(mask[t // 32]) >> t % 32 & 1:
                    t = (t + 1) % VOCAB
                self.sampled.append(t)
        return SimpleNamespace(tokens=self.sampled)

    def begin_read(self, count):
        return list(self.sampled[:count])

    def finish_read(self, handle):
        return handle

    def check_status(self):
        pass


def host_engine(max_batch=4, max_queue=100, num_pages=64, token_budget=64):
    e = Engine.__new__(Engine)
    e.model, e.tok, e.max_new_tokens, e.max_len = SimpleNamespace(plan=SimpleNamespace(vocab_size=VOCAB)), None, 8, 256
    e.cache = CacheManager([CacheNeeds(PagedKVSpec(1, 16, None))], max_batch, 256, 16, num_pages, torch.float32, "cpu")
    e.runner = HostRunner(e.cache)
    e.scheduler = Scheduler(e.cache, max_batch, 256, token_budget, max_queue, [STOP], VOCAB)
    e.run_ahead, e._ahead, e._planned, e.steps, e.ahead_launched, e.ahead_discarded = True, None, None, 0, 0, 0
    return e


def allowed_by(mask, vocab=VOCAB):
    return [t for t in range(vocab) if int(np.asarray(mask)[t // 32]) >> t % 32 & 1]
