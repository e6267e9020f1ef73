"""What the operators for several answers of one prompt are measured on: copies of cache pages (a fork of a row), decode
attention of rows that share a prefix, and sampling with penalties, biases and grammar masks.

A case is a dict of plain values.  kind "pages": `copies` pages of each of `runs` layer runs, keys and values.  kind
"attention": one token of each of `rows` requests over its paged keys; the rows are dealt to `families` families, each of
which shares its first `shared` keys (page by page the same ones), and `loners` rows share nothing; behind the shared keys
a row has up to `tail` keys of its own.  kind "sampling": one token for each of `rows` rows of `vocab` logits.

Sizes: heads, widths, page size and vocabularies of the Qwen3-4B and 32B shapes and of the tests' tiny configurations.
Queries, keys and values are N(0, 1) (what normed keys and projected values measure), logits N(0, 2.5), token ids of
histories skewed towards a few that come again and again, as text is.
"""

import math

import torch

own = False

PAGE = 16
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ------------------------------------------------------------------ cases
def _pages(name, copies, runs, kv_heads, key_dim, value_dim, dtype="bfloat16"):
    return {"name": name, "kind": "pages", "copies": copies, "runs": runs, "kv_heads": kv_heads, "key_dim": key_dim,
            "value_dim": value_dim, "dtype": dtype}


def _attention(name, rows, shared, tail, heads, kv_heads, dim, families=1, loners=0, window=0, dtype="bfloat16"):
    return {"name": name, "kind": "attention", "rows": rows, "shared": shared, "tail": tail, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "families": families, "loners": loners, "window": window, "dtype": dtype}


def _sampling(name, rows, vocab, history, penalties=True, biases=0, masked="none", temperature=0.0, adjusted=False):
    return {"name": name, "kind": "sampling", "rows": rows, "vocab": vocab, "history": history, "penalties": penalties,
            "biases": biases, "masked": masked, "temperature": temperature, "adjusted": adjusted}


def listed():
    return [
        # one more answer for one prompt: the partly filled page of every layer of the 4B shape
        _pages("fork_1", 1, 36, 8, 128, 128),
        # a full server's worth of answers forked from one prompt, 32B shape
        _pages("fork_63_32b", 63, 64, 8, 128, 128),
        # whole rows copied, small float32 pages with values of another size
        _pages("copy_501_float32", 501, 3, 2, 32, 48, dtype="float32"),
        # two answers of one chat prompt
        _attention("answers_2", 2, 512, 60, 32, 8, 128),
        # eight answers of one long prompt
        _attention("answers_8", 8, 4096, 300, 32, 8, 128),
        # a full server behind one system prompt, answers of all lengths
        _attention("system_prompt_64", 64, 6144, 2048, 32, 8, 128),
        # several families and some requests of their own, 32B heads
        _attention("families_27_32b", 27, 2000, 500, 64, 8, 128, families=3, loners=5),
        # the tests' size in the 32-bit engine, a window that leaves some rows little or nothing of the prefix
        _attention("window_float32", 9, 145, 70, 8, 2, 32, families=2, window=37, dtype="float32"),
        # one chat request with all penalties
        _sampling("penalties_1", 1, 151936, 800, temperature=0.8),
        # a full server, penalties and biases, half of the rows greedy
        _sampling("penalties_64", 64, 151936, 4096, biases=40, temperature=0.7),
        # structured output: a grammar allows few tokens; the adjusted logits are asked for
        _sampling("grammar_16", 16, 151936, 300, biases=5, masked="few", adjusted=True),
        # the tests' size, an odd vocabulary, most tokens allowed
        _sampling("tiny_5", 5, 383, 40, biases=3, masked="most", temperature=0.9, adjusted=True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["pages", "attention", "sampling"])
    if kind == "pages":
        dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
        key_dim, kv_heads = rng.choice([16, 32, 64, 96, 128]), rng.choice([1, 2, 4, 8])
        value_dim = key_dim if rng.random() < 0.7 else rng.choice([16, 48, 64, 128])
        runs = _log_uniform(rng, 1, 64)
        page = kv_heads * PAGE * (key_dim + value_dim) * (2 if dtype == "bfloat16" else 4)
        most = max(2, min(600, 250_000_000 // (page * runs)))
        case = _pages("", _log_uniform(rng, 1, most), runs, kv_heads, key_dim, value_dim, dtype)
    elif kind == "attention":
        dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
        heads, kv_heads, dim = rng.choice([(32, 8, 128), (64, 8, 128), (16, 8, 64), (8, 2, 32), (4, 2, 16), (12, 4, 96), (32, 2, 128)])
        rows = _log_uniform(rng, 2, 64)
        most = min(8192, 64 * 8192 // rows, 8192 if dtype == "bfloat16" else 2048)
        shared = _log_uniform(rng, 16, most * 3 // 4)
        tail = _log_uniform(rng, 1, max(1, most // 4))
        families = rng.randint(1, max(1, rows // 3))
        loners = rng.randint(0, max(0, min(rows - families, rows // 4)))
        window = rng.choice([0, 0, 0, _log_uniform(rng, 8, most)])
        case = _attention("", rows, shared, tail, heads, kv_heads, dim, families, loners, window, dtype)
    else:
        vocab = rng.choice([151936, 151936, 32000, 256, 384, rng.randint(200, 150000)])
        masked = rng.choice(["none", "none", "few", "most"])
        case = _sampling("", _log_uniform(rng, 1, 64), vocab, _log_uniform(rng, 1, 8000), rng.random() < 0.8,
                         rng.choice([0, _log_uniform(rng, 1, min(300, vocab // 2))]), masked, rng.choice([0.0, round(rng.uniform(0.3, 1.5), 2)]),
                         rng.random() < 0.3)
    del case["name"]
    return case


# ------------------------------------------------------------------ inputs
def _attention_layout(case, g):
    """(shared keys of each family, family of each row (-1: none), length of each row), fixed by the generator."""
    rows, families, loners = case["rows"], case["families"], case["loners"]
    pages = max(1, case["shared"] // PAGE)
    shared = [PAGE * pages if f == 0 else PAGE * int(torch.randint(max(1, pages // 4), pages + 1, (1,), generator=g)) for f in range(families)]
    sharing = rows - loners
    family = [i if i < families else int(torch.randint(0, families, (1,), generator=g)) for i in range(sharing)] + [-1] * loners
    order = torch.randperm(rows, generator=g).tolist()
    family = [family[i] for i in order]
    tails = torch.randint(1, case["tail"] + 1, (rows,), generator=g).tolist()
    alone = torch.randint(1, case["shared"] + 1, (rows,), generator=g).tolist()
    lengths = [tails[r] + (shared[family[r]] if family[r] >= 0 else alone[r]) for r in range(rows)]
    return shared, family, lengths


def _prepare_attention(case, seed):
    g = torch.Generator().manual_seed(1000 + case["rows"])          # the layout is the case's; values are the seed's
    shared, family, lengths = _attention_layout(case, g)
    rows, Hkv, D, dtype = case["rows"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    width = -(-max(lengths) // PAGE)
    page, prefix_pages = 1, []
    for s in shared:
        prefix_pages.append(list(range(page, page + s // PAGE)))
        page += s // PAGE
    tables = []
    for r in range(rows):
        pages = list(prefix_pages[family[r]]) if family[r] >= 0 else []
        need = -(-lengths[r] // PAGE) - len(pages)
        pages += range(page, page + need)
        page += need
        tables.append(pages + [0] * (width - len(pages)))
    shuffle = torch.randperm(page - 1, generator=g) + 1             # pages of a row lie anywhere in the pool
    shuffle = torch.cat([torch.zeros(1, dtype=torch.int64), shuffle])
    table = shuffle[torch.tensor(tables)].to(torch.int32)
    members, starts, lens = [], [0], []
    for f, s in enumerate(shared):
        members += [r for r in range(rows) if family[r] == f]
        starts.append(len(members))
        lens.append(s)
    for r in range(rows):
        if family[r] < 0:
            members.append(r)
            starts.append(len(members))
            lens.append(0)
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda").to(dtype)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    return {"kind": "attention", "case": case, "q": normal(rows, case["heads"] * D), "k": normal(page, Hkv, PAGE, D),
            "v": normal(page, Hkv, PAGE, D), "table": table.cuda(), "token_rows": ints(list(range(rows))),
            "positions": ints([n - 1 for n in lengths]), "members": ints(members), "starts": ints(starts), "lens": ints(lens),
            "out": torch.zeros(rows, case["heads"] * D, dtype=dtype, device="cuda")}


def _prepare_pages(case, seed):
    g = torch.Generator().manual_seed(seed)
    dtype, copies, runs, Hkv = DTYPES[case["dtype"]], case["copies"], case["runs"], case["kv_heads"]
    pages = 2 * copies + 2                                          # the null page and a page that nobody copies
    order = (torch.randperm(pages - 1, generator=g) + 1).tolist()
    src = order[:copies]
    if copies > 1:
        src[-1] = src[0]                                            # one page copied twice
    dst = order[copies:2 * copies]
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def pool(dim):
        return torch.randn((runs, pages, Hkv, PAGE, dim), generator=gen, device="cuda", dtype=dtype)

    return {"kind": "pages", "k": pool(case["key_dim"]), "v": pool(case["value_dim"]), "src": src, "dst": dst}


def _prepare_sampling(case, seed):
    M, V, W = case["rows"], case["vocab"], case["history"]
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device="cuda")

    rows = M + 2                                                    # the table has rows that are not sampled
    history = (uniform(rows, W) ** 3 * V).to(torch.int32).clamp_(0, V - 1)
    row = torch.randperm(rows, generator=gen, device="cuda")[:M].to(torch.int32)
    lengths = (1 + uniform(M) * W).to(torch.int32).clamp_(1, W)
    prompt = (uniform(M) * lengths).to(torch.int32)
    s = {"kind": "sampling", "case": case, "logits": 2.5 * torch.randn((M, V), generator=gen, device="cuda"),
         "history": history, "rows": row, "prompt_lens": prompt, "lengths": lengths, "penalties": None,
         "bias_starts": None, "bias_ids": None, "bias_values": None, "mask": None, "mask_rows": None,
         "temperature": None, "seeds": None, "counters": None,
         "out": torch.zeros(M, dtype=torch.int32, device="cuda"),
         "adjusted": torch.empty((M, V), device="cuda") if case["adjusted"] else None}
    if case["penalties"]:
        s["penalties"] = torch.stack([1.0 + 0.5 * uniform(M), 0.8 * uniform(M), 0.4 * uniform(M)], dim=1).contiguous()
    if case["biases"]:
        per = case["biases"]
        s["bias_starts"] = torch.arange(0, M * per + 1, per, dtype=torch.int32, device="cuda")
        s["bias_ids"] = torch.stack([torch.randperm(V, generator=gen, device="cuda")[:per] for _ in range(M)]).reshape(-1).to(torch.int32)
        s["bias_values"] = 3.0 * torch.randn(M * per, generator=gen, device="cuda")
    if case["masked"] != "none":
        words = -(-V // 32)
        if case["masked"] == "few":                                 # a few dozen tokens are allowed
            bits = torch.zeros((M, words * 32), dtype=torch.bool, device="cuda")
            bits.scatter_(1, (uniform(M, 40) * V).to(torch.int64).clamp_(0, V - 1), True)
        else:
            bits = uniform(M, words * 32) < 0.9
        weights = (2 ** torch.arange(32, dtype=torch.int64, device="cuda"))
        packed = (bits.reshape(M, words, 32).to(torch.int64) * weights).sum(-1)
        s["mask"] = torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32).contiguous()
        mask_rows = torch.arange(M, dtype=torch.int32, device="cuda")
        if M > 2:
            mask_rows[1] = -1                                       # a row without a grammar
        s["mask_rows"] = mask_rows
    if case["temperature"] > 0:
        t = torch.full((M,), case["temperature"], device="cuda")
        t[1::2] = 0.0
        s["temperature"] = t
        s["seeds"] = torch.randint(-2 ** 31, 2 ** 31 - 1, (M,), generator=gen, device="cuda").to(torch.int32)
        s["counters"] = (lengths - prompt).to(torch.int32)
    return s


def prepare(case, seed):
    return {"pages": _prepare_pages, "attention": _prepare_attention, "sampling": _prepare_sampling}[case["kind"]](case, seed)


# ------------------------------------------------------------------ the framework's calls
def _run_own(s):
    from socrates_b200.kernels import ops
    if s["kind"] == "pages":
        ops.copy_pages(s["k"], s["v"], s["src"], s["dst"])
        return {"k": s["k"], "v": s["v"]}
    if s["kind"] == "attention":
        c = s["case"]
        if "scratch" not in s:                                      # kept, as a step's buffers are
            floats, ints = ops.attention_shared_scratch_size(c["rows"], c["heads"], c["kv_heads"], c["dim"], PAGE, s["q"].dtype)
            s["scratch"] = (torch.empty(floats, device="cuda"), torch.zeros(ints, dtype=torch.int32, device="cuda"))
            s["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        ops.attention_shared(s["out"], s["q"], s["k"], s["v"], s["table"], s["token_rows"], s["positions"], s["members"],
                             s["starts"], s["lens"], c["heads"], c["dim"] ** -0.5, c["window"], *s["scratch"], s["status"])
        return s["out"]
    if "scratch" not in s:
        s["scratch"] = torch.zeros(ops.sample_scratch_size(*s["logits"].shape), dtype=torch.int32, device="cuda")
    ops.sample_adjusted(s["out"], s["logits"], s["temperature"], s["seeds"], s["counters"], s["scratch"],
                        history=s["history"], history_rows=s["rows"], prompt_lens=s["prompt_lens"], lengths=s["lengths"],
                        penalties=s["penalties"], bias_starts=s["bias_starts"], bias_ids=s["bias_ids"],
                        bias_values=s["bias_values"], mask=s["mask"], mask_rows=s["mask_rows"], adjusted=s["adjusted"])
    return {"tokens": s["out"], "adjusted": s["adjusted"]} if s["adjusted"] is not None else s["out"]


# ------------------------------------------------------------------ the plain forms
def _plain_pages(s):
    src, dst = (torch.tensor(x, device="cuda") for x in (s["src"], s["dst"]))
    for pool in (s["k"], s["v"]):
        pool[:, dst] = pool[:, src]
    return {"k": s["k"], "v": s["v"]}


def _plain_attention(s):
    c = s["case"]
    N, Hq, Hkv, D = c["rows"], c["heads"], c["kv_heads"], c["dim"]
    table = s["table"][s["token_rows"].long()].long()
    keys = table.shape[1] * PAGE
    k = s["k"][table].float().permute(0, 2, 1, 3, 4).reshape(N, Hkv, keys, D)
    q = s["q"].float().reshape(N, Hkv, Hq // Hkv, D)
    scores = torch.matmul(q, k.transpose(2, 3)) * D ** -0.5
    del k
    at = torch.arange(keys, device="cuda")
    pos = s["positions"][:, None]
    seen = (at <= pos) & ((at > pos - c["window"]) if c["window"] else (at >= 0))
    scores = torch.where(seen[:, None, None, :], scores, torch.tensor(-math.inf, device="cuda"))
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    v = s["v"][table].float().permute(0, 2, 1, 3, 4).reshape(N, Hkv, keys, D)
    v = torch.where(seen[:, None, :, None], v, torch.tensor(0.0, device="cuda"))
    out = torch.matmul(weights, v) / weights.sum(-1, keepdim=True)
    s["out"].copy_(out.reshape(N, Hq * D))
    return s["out"]


def _mix(x):
    x = (x ^ (x >> 16)) * 0x7FEB352D & 0xFFFFFFFF
    x = (x ^ (x >> 15)) * 0x846CA68B & 0xFFFFFFFF
    return x ^ (x >> 16)


def _uniforms(seeds, counters, V):
    """The counter-based uniforms of the sampler: a function of (seed, counter, vocabulary index)."""
    seeds, counters = (x.long() & 0xFFFFFFFF for x in (seeds, counters))
    key = _mix(_mix(seeds ^ 0x9E3779B9) ^ _mix((counters + 0x85EBCA6B) & 0xFFFFFFFF))
    at = (torch.arange(V, device=seeds.device) + 0x165667B1) & 0xFFFFFFFF
    return ((_mix(at[None, :] ^ key[:, None]) >> 9).double() + 0.5) / 2.0 ** 23


def _plain_sampling(s):
    l = s["logits"].clone()
    M, V = l.shape
    if s["penalties"] is not None:
        tokens = s["history"][s["rows"].long()].long()
        at = torch.arange(tokens.shape[1], device="cuda")
        in_prompt = at < s["prompt_lens"][:, None]
        in_output = ~in_prompt & (at < s["lengths"][:, None])
        prompt = torch.zeros((M, V), device="cuda").scatter_add_(1, tokens, in_prompt.float())
        output = torch.zeros((M, V), device="cuda").scatter_add_(1, tokens, in_output.float())
        r, presence, frequency = (s["penalties"][:, i:i + 1] for i in range(3))
        l = torch.where((prompt > 0) | (output > 0), torch.where(l > 0, l / r, l * r), l)
        l = l - frequency * output - presence * (output > 0).float()
    if s["bias_ids"] is not None:
        per = s["case"]["biases"]
        l.scatter_add_(1, s["bias_ids"].reshape(M, per).long(), s["bias_values"].reshape(M, per))
    if s["mask"] is not None:
        words = s["mask"][s["mask_rows"].clamp(min=0).long()]
        bits = (words[:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        allowed = (bits.reshape(M, -1)[:, :V] == 1) | (s["mask_rows"] < 0)[:, None]
        l = torch.where(allowed, l, torch.tensor(-math.inf, device="cuda"))
    scores = l
    if s["temperature"] is not None:
        t = s["temperature"][:, None]
        noise = -torch.log(-torch.log(_uniforms(s["seeds"], s["counters"], V).float()))
        scores = torch.where(t > 0, l / torch.where(t > 0, t, torch.ones_like(t)) + noise, l)
    best = scores.amax(-1, keepdim=True)
    tokens = torch.where(scores == best, torch.arange(V, device="cuda"), V).amin(-1)
    s["out"].copy_(tokens)
    if s["adjusted"] is None:
        return s["out"]
    s["adjusted"].copy_(l)
    return {"tokens": s["out"], "adjusted": s["adjusted"]}


def run(state):
    if own:
        return _run_own(state)
    return {"pages": _plain_pages, "attention": _plain_attention, "sampling": _plain_sampling}[state["kind"]](state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["kind"] == "pages":
        page = case["kv_heads"] * PAGE * (case["key_dim"] + case["value_dim"]) * (2 if case["dtype"] == "bfloat16" else 4)
        sources = max(1, case["copies"] - 1)                        # one of them is copied twice
        return {"bytes": page * case["runs"] * (sources + case["copies"]), "flops": 0}
    if case["kind"] == "attention":
        shared, family, lengths = _attention_layout(case, torch.Generator().manual_seed(1000 + case["rows"]))
        item = 2 if case["dtype"] == "bfloat16" else 4
        keys = products = 0
        seen = [max(shared) + 1] * len(shared)
        for f, n in zip(family, lengths):
            first = max(0, n - case["window"]) if case["window"] else 0
            products += n - first
            if f < 0:
                keys += n - first
            else:
                keys += n - max(first, shared[f])
                seen[f] = min(seen[f], first)                       # the first key that somebody sees
        keys += sum(max(0, s - f) for s, f in zip(shared, seen))
        rows = case["rows"] * case["heads"] * case["dim"]
        return {"bytes": 2 * keys * case["kv_heads"] * case["dim"] * item + 2 * rows * item,
                "flops": 4 * products * case["heads"] * case["dim"]}
    M, V = case["rows"], case["vocab"]
    n = M * V * 4 + M * 4
    if case["penalties"]:
        n += M * case["history"] * 4 // 2                           # rows are half full on average
    n += M * case["biases"] * 8
    if case["masked"] != "none":
        n += M * V // 8
    if case["masked"] == "few" and not (M > 2):
        n -= M * V * 4                                              # places that are not allowed need not be read
    elif case["masked"] == "few":
        n -= (M - 1) * V * 4
    if case["adjusted"]:
        n += M * V * 4
    return {"bytes": n, "flops": 0}


# ------------------------------------------------------------------ from the definitions, in 64 bits
def _exact_attention(s):
    c = s["case"]
    D, G = c["dim"], c["heads"] // c["kv_heads"]
    k, v, q = (s[x].double() for x in ("k", "v", "q"))
    rows = []
    for n, (row, pos) in enumerate(zip(s["token_rows"].tolist(), s["positions"].tolist())):
        first = max(0, pos + 1 - c["window"]) if c["window"] else 0
        at = torch.arange(first, pos + 1, device="cuda")
        page, slot = s["table"][row].long()[at // PAGE], at % PAGE
        heads = []
        for h in range(c["kv_heads"]):
            kh, vh = k[page, h, slot], v[page, h, slot]
            qh = q[n].reshape(c["heads"], D)[h * G:(h + 1) * G]
            heads.append(torch.softmax(qh @ kh.T / math.sqrt(D), dim=-1) @ vh)
        rows.append(torch.cat(heads).reshape(-1))
    return torch.stack(rows)


def _exact_sampling(s):
    M, V = s["logits"].shape
    adjusted, tokens = [], []
    for m in range(M):
        l = s["logits"][m].double()
        if s["penalties"] is not None:
            r, presence, frequency = s["penalties"][m].double().tolist()
            told = s["history"][int(s["rows"][m])].long()
            p, n = int(s["prompt_lens"][m]), int(s["lengths"][m])
            counts = torch.bincount(told[p:n], minlength=V).double()
            met = torch.bincount(told[:n], minlength=V) > 0
            l[met] = torch.where(l[met] > 0, l[met] / r, l[met] * r)
            l = l - frequency * counts
            l[counts > 0] -= presence
        if s["bias_ids"] is not None:
            a, b = int(s["bias_starts"][m]), int(s["bias_starts"][m + 1])
            l[s["bias_ids"][a:b].long()] += s["bias_values"][a:b].double()
        if s["mask"] is not None and int(s["mask_rows"][m]) >= 0:
            word = s["mask"][int(s["mask_rows"][m])].long() & 0xFFFFFFFF
            at = torch.arange(V, device="cuda")
            l[(word[at // 32] >> (at % 32)) % 2 == 0] = -math.inf
        adjusted.append(l.clone())
        if s["temperature"] is not None and float(s["temperature"][m]) > 0:
            u = _uniforms(s["seeds"][m:m + 1], s["counters"][m:m + 1], V)[0]
            l = l / float(s["temperature"][m]) - torch.log(-torch.log(u))
        tokens.append(int(torch.nonzero(l == l.max())[0]))
    tokens = torch.tensor(tokens, dtype=torch.int32, device="cuda")
    return {"tokens": tokens, "adjusted": torch.stack(adjusted)} if s["adjusted"] is not None else tokens


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attention":
        return _exact_attention(s)
    if case["kind"] == "sampling":
        return _exact_sampling(s)
    k, v = s["k"].clone(), s["v"].clone()
    for a, b in zip(s["src"], s["dst"]):
        k[:, b], v[:, b] = s["k"][:, a], s["v"][:, a]
    return {"k": k.double(), "v": v.double()}
