"""Several answers of one prompt through the engine: forked rows, attention that reads the prompt once, penalties, biases and
grammars."""

import math

import pytest
import torch

import plain_qwen3 as plain
from socrates_b200 import Engine
from socrates_b200.cache import CacheManager
from socrates_b200.config import config_from_dict
from socrates_b200.engine.engine import build_random_model
from socrates_b200.engine.runner import ModelRunner, SamplingArgs, StepEntry
from socrates_b200.parts import attention
from tiny_configs import make_folder

pytestmark = pytest.mark.gpu

# heads as the 4B shape's, so that every kernel of the shared-prefix attention serves them
WIDE = {"architectures": ["Qwen3ForCausalLM"], "vocab_size": 512, "hidden_size": 128, "intermediate_size": 192,
        "num_hidden_layers": 4, "num_attention_heads": 16, "num_key_value_heads": 4, "head_dim": 128, "rms_norm_eps": 1e-6,
        "rope_theta": 10000.0, "tie_word_embeddings": True, "max_position_embeddings": 4096}


def prompt(n, seed=0, vocab=256):
    return torch.randint(1, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.fixture
def always_shared(monkeypatch):
    monkeypatch.setattr(attention, "SHARED_PAYS_FROM", 1)


# ------------------------------------------------------------------ the same answers as from requests of their own
@pytest.mark.parametrize("name", ["A", "B"])
@pytest.mark.parametrize("length", [1, 2, 16, 17, 50, 90])
def test_answers_are_those_of_single_requests(tmp_path, name, length):
    """float32: a request's numbers do not depend on the batch, and a forked page holds the same bits."""
    folder = str(make_folder(tmp_path, name))
    kw = dict(dtype="float32", max_batch=4, max_len=128, max_new_tokens=9, token_budget=32)
    alone = Engine(folder, **kw)
    want = [alone.generate([prompt(length)], temperature=0.9, seed=5 + i)[0] for i in range(6)]
    eng = Engine(folder, **kw)
    got = eng.generate([prompt(length)], temperature=0.9, seed=5, n=6)[0]
    assert got == want and len(set(map(tuple, got))) > 1
    eng.cache.check()
    assert set(eng.cache.free_pages()) == {eng.num_blocks}
    prompts = eng.scheduler.prompt_tokens
    assert prompts <= length * 6 and (length < 3 or prompts < length * 6)       # forks computed less


def test_answers_under_few_pages(tmp_path):
    folder = str(make_folder(tmp_path, "A"))
    want = Engine(folder, dtype="float32", max_batch=6, max_len=128, token_budget=16).generate(
        [prompt(40), prompt(33, 1)], 20, 0.8, 3, n=4)
    eng = Engine(folder, dtype="float32", max_batch=6, max_len=128, token_budget=16, num_blocks=6)
    assert eng.generate([prompt(40), prompt(33, 1)], 20, 0.8, 3, n=4) == want
    assert eng.scheduler.preemptions > 0
    eng.cache.check()


# ------------------------------------------------------------------ attention of families inside a step
class Rows:
    """A runner over a random model whose row 0 holds a prompt and rows 1.. are forks of it, all gone on by some tokens."""

    def __init__(self, rows, length, shape=WIDE, dtype=torch.bfloat16, graphs=True, more=3, page=16):
        config = config_from_dict(shape)
        _, model = build_random_model(config, 7, dtype, torch.device("cuda:0"))
        self.cache = CacheManager(model.cache_needs(), rows + 2, 2048, page, 500, dtype, "cuda:0")
        self.runner = ModelRunner(model, self.cache, dtype, "cuda:0", max_tokens=1600, max_seqs=rows + 2, use_graphs=graphs)
        self.vocab = config.plan().vocab_size
        self.ids = {0: prompt(length, 3, self.vocab)}
        self.cache.assign(0)
        self.feed({0: self.ids[0]})
        for r in range(1, rows):
            assert self.cache.fork(0, r, length - 1)
            self.ids[r] = self.ids[0][:-1]
        for r in range(1, rows):
            for t in prompt(r % (more + 1), 40 + r, self.vocab):
                self.feed({r: [t]})

    def feed(self, new):
        """One step; returns its logits, a row for the last token of each request."""
        entries = []
        for r, tokens in new.items():
            start = self.cache.lengths[r]
            assert self.cache.reserve(r, start + len(tokens))
            entries.append(StepEntry(r, tokens, start, [len(tokens) - 1]))
        logits = self.runner.step(entries).logits.clone()
        self.runner.check_status()
        for e in entries:
            self.cache.commit(e.row, e.start + len(e.tokens))
        return logits


@pytest.mark.parametrize("rows,length", [(2, 100), (5, 33), (14, 500), (3, 17), (48, 1500)])
def test_a_step_with_families_gives_the_step_without(always_shared, monkeypatch, rows, length):
    both = []
    for on in (True, False):
        monkeypatch.setattr(attention, "SHARED_PAYS_FROM", 1 if on else 1 << 60)
        r = Rows(rows, length)
        out = [r.feed({i: [11 + i + 7 * k] for i in range(rows)}) for k in range(3)]      # eager, recorded, replayed
        # some of the rows, in another order, beside a prompt portion and a row that shares nothing
        r.cache.assign(rows)
        out.append(r.feed({rows: prompt(40, 9, r.vocab), rows - 1: [5], 0: [6]}))
        out.append(r.feed({0: [8], rows: [3], rows - 1: [4]}))
        if on:
            assert any("families" in key for key in r.runner._graphs)
            assert any("large" in key for key in r.runner._graphs) == (rows == 48)
        both.append(out)
    for a, b in zip(*both):
        # bfloat16 activations: a few roundings of 2^-9 of values that add up over four layers, as far as two correct kernels differ
        scale = float(b.abs().max())
        assert float((a - b).abs().max()) <= 2e-2 * scale


@pytest.mark.parametrize("shape,page,reads", [(dict(head_dim=96), 16, True), (dict(num_attention_heads=20, num_key_value_heads=1), 16, True),
                                              (dict(head_dim=256), 16, False), (dict(), 8, False), (dict(), 16, True)], ids=str)
def test_shapes_whose_shared_keys_are_read_once(always_shared, monkeypatch, shape, page, reads):
    both = []
    for least in (1, 1 << 60):
        monkeypatch.setattr(attention, "SHARED_PAYS_FROM", least)
        r = Rows(4, 50, {**WIDE, **shape}, page=page)
        out = [r.feed({i: [11 + i + 7 * k] for i in range(4)}) for k in range(3)]
        assert any("families" in key for key in r.runner._graphs) == (reads and least == 1)
        both.append(out)
    for a, b in zip(*both):                                 # (as far as two correct kernels differ, see above)
        assert float((a - b).abs().max()) <= 2e-2 * float(b.abs().max())


def test_a_recorded_step_follows_its_families(always_shared):
    """The graph of a width is recorded with one set of families and replayed with others."""
    r, fresh = Rows(6, 80), Rows(6, 80)
    # from here on (the steps of one row before it choose their kernels' partitions by whether they may be recorded)
    fresh.runner.use_graphs = False
    replays = r.runner.graph_replays
    for k in range(6):
        if k == 3:                                          # row 2 leaves, another prompt comes into its place
            for x in (r, fresh):
                x.cache.release(2)
                x.cache.assign(2)
                x.feed({2: prompt(30, 5, x.vocab)})
        if k == 4:
            for x in (r, fresh):
                x.cache.release(5)
                assert x.cache.fork(4, 5, x.cache.lengths[4])
        step = {i: [20 + i + k] for i in range(6)}
        assert torch.equal(r.feed(step), fresh.feed(step))
    assert r.runner.graph_replays >= replays + 4


def test_engine_with_families_answers_like_one_without(always_shared, monkeypatch, tmp_path):
    """Greedy answers of one prompt are one answer; with different first tokens they are what the plain implementation says."""
    folder = make_folder(tmp_path, "A")
    cfg, w = plain.load_folder(folder)
    eng = Engine(str(folder), dtype="bfloat16", max_batch=6, max_len=128, token_budget=64, warmup=True)
    answers = eng.generate([prompt(70)], 12, temperature=0.7, seed=11, n=6)[0]
    assert any("families" in key for key in eng.runner._graphs)
    assert len(set(map(tuple, answers))) > 1
    for a in answers:
        logits = plain.logits(w, cfg, prompt(70) + a[:-1])
        assert all(0 <= t < 256 for t in a) and len(a) == 12 and bool(torch.isfinite(logits).all())
    monkeypatch.setattr(attention, "SHARED_PAYS_FROM", 1 << 60)
    greedy = Engine(str(folder), dtype="bfloat16", max_batch=6, max_len=128, token_budget=64).generate([prompt(70)], 12, n=4)[0]
    monkeypatch.setattr(attention, "SHARED_PAYS_FROM", 1)
    shared = eng.generate([prompt(70)], 12, n=4)[0]
    for a, b in zip(shared, greedy):
        for i, (x, y) in enumerate(zip(a, b)):
            if x != y:                                      # two near-equal logits: 2 % of the largest
                row = plain.logits(w, cfg, prompt(70) + a[:i])[-1]
                assert float((row[x] - row[y]).abs()) <= 2e-2 * float(row.abs().max())
                break


# ------------------------------------------------------------------ adjusted logits in the engine
def greedy_adjusted(w, cfg, ids, new, adjust):
    """The plain implementation's greedy answer with adjusted logits, and by how much each token won."""
    out, margins = [], []
    for _ in range(new):
        row = adjust(plain.logits(w, cfg, ids + out)[-1].double(), out)
        top = torch.topk(row, 2)
        out.append(int(top.indices[0]))
        margins.append(float(top.values[0] - top.values[1]))
    return out, margins


def penalties(ids, r=1.0, presence=0.0, frequency=0.0, bias=None, allowed=None):
    def adjust(row, out):
        for t in set(ids) | set(out):
            row[t] = row[t] / r if row[t] > 0 else row[t] * r
        for t in set(out):
            row[t] -= presence + frequency * out.count(t)
        for t, b in (bias or {}).items():
            row[t] += b
        if allowed is not None:
            keep = torch.full_like(row, -math.inf)
            keep[list(allowed)] = row[list(allowed)]
            row = keep
        return row
    return adjust


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("kw", [dict(repetition_penalty=1.6), dict(presence_penalty=0.7, frequency_penalty=0.2),
                                dict(logit_bias={3: 1.5, 200: -2.0}), dict(allowed=[9, 40, 41, 200, 255]),
                                dict(repetition_penalty=0.8, frequency_penalty=0.4, logit_bias={7: 0.5}, allowed=range(0, 256, 3))],
                         ids=["repetition", "presence_frequency", "bias", "allowed", "all"])
def test_greedy_answers_with_adjusted_logits(tmp_path, kw, graphs):
    folder = make_folder(tmp_path, "A")
    cfg, w = plain.load_folder(folder)
    eng = Engine(str(folder), dtype="float32", max_batch=3, max_len=128, token_budget=16, compile=graphs)
    ids = prompt(37, 2)
    plainly = {"r": kw.get("repetition_penalty", 1.0), "presence": kw.get("presence_penalty", 0.0),
               "frequency": kw.get("frequency_penalty", 0.0), "bias": kw.get("logit_bias"), "allowed": kw.get("allowed")}
    want, margins = greedy_adjusted(w, cfg, ids, 14, penalties(ids, **plainly))
    assert min(margins) > 1e-4                              # no tie that rounding decides
    # beside requests without and with other adjustments, forked and alone
    others = [eng.submit(prompt(20, 8), 14), eng.submit(prompt(9, 9), 14, 0.8, 3, presence_penalty=0.4)]
    answers = eng.submit_answers(ids, 2, 14, **kw)
    eng.run()
    assert [r.output for r in answers] == [want, want]
    lone = Engine(str(folder), dtype="float32", max_batch=3, max_len=128, token_budget=16)
    assert others[0].output == lone.generate([prompt(20, 8)], 14)[0]
    assert others[1].output == lone.generate([prompt(9, 9)], 14, 0.8, 3, presence_penalty=0.4)[0]


def test_running_ahead_and_preemption_keep_adjusted_answers(tmp_path):
    folder = str(make_folder(tmp_path, "A"))
    kw = dict(repetition_penalty=1.3, frequency_penalty=0.3, logit_bias={5: 1.0}, allowed=range(0, 250))
    outs = []
    for extra in (dict(), dict(run_ahead=False), dict(num_blocks=6), dict(compile=False, token_budget=7)):
        eng = Engine(folder, dtype="float32", max_batch=4, max_len=128, **{"token_budget": 32, **extra})
        outs.append(eng.generate([prompt(30), prompt(45, 1)], 25, 0.7, 2, n=3, **kw))
        if "num_blocks" in extra:
            assert eng.scheduler.preemptions > 0
        if not extra:
            assert eng.ahead_launched > 0
    assert all(o == outs[0] for o in outs)


def test_a_grammar_decides_step_by_step(tmp_path):
    """A function of the output: digits (ids 48 to 57) in turn with one of two others, five tokens at most."""
    folder = str(make_folder(tmp_path, "A"))

    def grammar(out):
        if len(out) == 5:
            return []                                       # nothing more: the request ends
        if len(out) == 4:
            return None                                     # anything
        return range(48, 58) if len(out) % 2 == 0 else [10, 11]

    for n in (1, 3):
        eng = Engine(folder, dtype="bfloat16", max_batch=3, max_len=128, token_budget=32)
        free = eng.submit(prompt(12, 4), 20)
        reqs = eng.submit_answers(prompt(20), n, 20, temperature=1.0, seed=4, allowed=grammar)
        eng.run()
        for r in reqs:
            assert r.done and len(r.output) == 5
            assert all((48 <= t < 58) if i % 2 == 0 else t in (10, 11) for i, t in enumerate(r.output[:4]))
        assert len(free.output) == 20


def test_penalties_beside_rows_that_were_there_before(tmp_path):
    """The rows' tokens are kept from the first penalized request on; it may come while others decode, recorded, running ahead,
    and what the caller does to its biases later changes nothing."""
    folder = str(make_folder(tmp_path, "A"))
    kw = dict(dtype="float32", max_batch=4, max_len=128, token_budget=32)
    eng, bias = Engine(folder, **kw), {7: 2.0, 9: -1.0}
    first = eng.submit(prompt(20), 40)
    for _ in range(8):
        eng.step()
    assert eng.cache.tokens is None and first.output
    late = eng.submit_answers(prompt(37, 2), 2, 20, 0.6, 5, repetition_penalty=1.5, frequency_penalty=0.2, logit_bias=bias)
    bias.clear()
    eng.run()
    assert eng.cache.tokens is not None
    lone = Engine(folder, **kw)
    assert first.output == lone.generate([prompt(20)], 40)[0]
    assert [r.output for r in late] == lone.generate([prompt(37, 2)], 20, 0.6, 5, n=2, repetition_penalty=1.5, frequency_penalty=0.2,
                                                     logit_bias={7: 2.0, 9: -1.0})[0]


def test_what_is_refused(tmp_path):
    folder = str(make_folder(tmp_path, "A"))
    eng = Engine(folder, dtype="float32", max_batch=2, max_len=64, token_budget=16, max_queue=3)
    for bad in (dict(repetition_penalty=0), dict(presence_penalty=math.nan), dict(logit_bias={256: 1.0}), dict(allowed=[]),
                dict(allowed=[256]), dict(logit_bias={1: math.inf})):
        with pytest.raises(ValueError):
            eng.submit([1, 2], **bad)
    with pytest.raises(TypeError):
        eng.submit([1, 2], top_k=3)
    with pytest.raises(ValueError):
        eng.submit_answers([1, 2], 0)
    from socrates_b200 import QueueFull, TooLong
    with pytest.raises(QueueFull):
        eng.submit_answers([1, 2], 4, 3)
    with pytest.raises(TooLong):
        eng.submit_answers([1] * 60, 2, 30)
    assert not eng.scheduler.pending
    assert eng.generate([[1, 2]], 3, n=1) == [eng.generate([[1, 2]], 3, n=2)[0][0]]


def test_the_command_line_takes_answers(tmp_path, capsys):
    from socrates_b200.inference_paged import main
    folder = str(make_folder(tmp_path, "A"))
    assert main(["--model", folder, "--prompt-ids", "5,17,3", "--answers", "3", "--max-new-tokens", "4", "--temperature", "0.9",
                 "--max-len", "64", "--max-batch", "3", "--repetition-penalty", "1.2", "--dtype", "float32"]) == 0
    out = capsys.readouterr().out
    assert out.count("> 5 17 3") == 3 and "12 tok" in out
