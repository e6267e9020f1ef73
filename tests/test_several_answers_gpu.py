"""The operators that several answers of one prompt take: page copies, attention over a shared prefix, sampling with
penalties, biases and grammar masks.  References in 64 bits, from the formulas."""

import math

import pytest
import torch

from socrates_b200.kernels import KernelError, ops

pytestmark = pytest.mark.gpu

PAGE = 16


def ints(v):
    return torch.tensor(list(v), dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ page copies
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("runs,heads,slots,dim,value_dim,copies", [
    (1, 1, 16, 16, 16, 1),
    (3, 2, 16, 32, 48, 33),          # more pairs than the small launch holds
    (2, 8, 16, 128, 128, 5),
    (5, 1, 4, 6, 2, 7),              # pages that are no multiple of 16 bytes
    (2, 3, 1, 1, 1, 2),              # pages of six bytes (bfloat16)
    (1, 1, 2, 8, 8, 2500),           # more pairs than one launch holds
])
def test_copy_pages(dtype, runs, heads, slots, dim, value_dim, copies):
    g = torch.Generator().manual_seed(copies)
    pages = 2 * copies + 3
    order = torch.randperm(pages, generator=g).tolist()
    src, dst = order[:copies], order[copies:2 * copies]
    src[-1] = src[0]                                        # one page to several places
    k = torch.randn(runs, pages, heads, slots, dim, generator=g).to(dtype)
    v = torch.randn(runs, pages, heads, slots, value_dim, generator=g).to(dtype)
    k[0, src[0], 0, 0, 0] = math.nan                        # bits are copied, whatever they mean
    want_k, want_v = k.clone(), v.clone()
    for a, b in zip(src, dst):
        want_k[:, b], want_v[:, b] = k[:, a], v[:, a]
    kd, vd = k.cuda(), v.cuda()
    ops.copy_pages(kd, vd, src, dst)
    bits = torch.int16 if dtype == torch.bfloat16 else torch.int32
    assert torch.equal(kd.cpu().view(bits), want_k.view(bits))
    assert torch.equal(vd.cpu().view(bits), want_v.view(bits))


def test_copy_pages_at_an_odd_address_and_of_nothing():
    flat = torch.randn(2 * 5 * 16 + 1, device="cuda").to(torch.bfloat16)
    k, v = flat[1:81].view(1, 5, 1, 4, 4), flat[81:161].view(1, 5, 1, 4, 4)     # 2 bytes behind a multiple of 16
    want = k.clone()
    want[:, 4] = want[:, 1]
    ops.copy_pages(k, v, [1], [4])
    assert torch.equal(k, want)
    ops.copy_pages(k, v, [], [])
    assert torch.equal(k, want)


def test_copy_pages_past_two_to_the_31():
    """A pool of more than 2^31 elements: offsets in 64 bits."""
    k = torch.zeros(2, 4200, 8, 16, 2048, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros(2, 4200, 8, 16, 1, dtype=torch.bfloat16, device="cuda")
    k[1, 4199].fill_(3.0)
    v[1, 4199].fill_(5.0)
    ops.copy_pages(k, v, [4199], [4198])
    assert bool((k[1, 4198] == 3.0).all()) and bool((k[0, 4198] == 0).all()) and bool((k[1, 4197] == 0).all())
    assert bool((v[1, 4198] == 5.0).all())


def test_copies_recorded_and_replayed_on_another_stream():
    k, v = (torch.randn(2, 6, 2, 16, 32, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ops.copy_pages(k, v, [1, 1], [2, 3])
        ops.copy_pages(k, v, [3], [4])                      # a chain in two calls
    k[:, 1].fill_(7.0)
    graph.replay()
    torch.cuda.synchronize()
    for page in (2, 3, 4):
        assert torch.equal(k[:, page], k[:, 1]) and torch.equal(v[:, page], v[:, 1])


def test_copy_pages_refusals():
    k, v = (torch.zeros(2, 6, 2, 16, 32, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    for src, dst in (([1], [6]), ([6], [1]), ([-1], [1]), ([1], [-1]), ([1, 2], [3, 3]), ([1, 2], [2, 3]), ([1], [1]),
                     ([1, 2], [3]), ([2 ** 31], [1]), (["1"], [2]), ([1.5], [2])):
        with pytest.raises(KernelError):
            ops.copy_pages(k, v, src, dst)
    with pytest.raises(KernelError):
        ops.copy_pages(k, v.float(), [1], [2])
    with pytest.raises(KernelError):
        ops.copy_pages(k, v[:1], [1], [2])
    with pytest.raises(KernelError):
        ops.copy_pages(k.transpose(2, 3), v, [1], [2])
    with pytest.raises(KernelError):
        ops.copy_pages(k.cpu(), v.cpu(), [1], [2])
    assert not bool(k.any())


# ------------------------------------------------------------------ attention over a shared prefix
class Case:
    """Rows in families: `families` is a list of (shared keys, [own keys of each member]); a family of shared length 0 shares
    nothing.  Pages lie anywhere; a row's pages end inside its last key's page."""

    def __init__(self, families, heads, kv_heads, dim, dtype, page=PAGE, seed=0, spare_tokens=0):
        g = torch.Generator().manual_seed(seed)
        self.heads, self.kv_heads, self.dim, self.dtype, self.page = heads, kv_heads, dim, dtype, page
        rows, self.members, starts, lens, lengths = [], [], [0], [], []
        next_page = 1
        for shared, owns in families:
            prefix = list(range(next_page, next_page + -(-shared // page)))
            next_page += len(prefix)
            for own in owns:
                # the page in which the prefix ends is the row's own (a copy) where the row goes on behind it
                whole = shared // page
                pages = prefix[:whole]
                need = -(-(shared + own) // page) - len(pages)
                if shared % page and own == 0:
                    pages, need = prefix, 0
                pages = pages + list(range(next_page, next_page + need))
                next_page += need
                rows.append((pages, prefix, shared))
                lengths.append(shared + own)
            starts.append(starts[-1] + len(owns))
            lens.append(shared)
        N = len(rows) + spare_tokens
        order = torch.randperm(N, generator=g).tolist()             # member i of the families is token order[i]
        self.N, self.members = N, order[:len(rows)]
        places = torch.cat([torch.zeros(1, dtype=torch.int64), torch.randperm(next_page, generator=g) + 1])
        width = max(len(p) for p, _, _ in rows) + 2
        table = torch.zeros(N, width, dtype=torch.int32)
        self.positions = torch.zeros(N, dtype=torch.int32)
        self.token_rows = torch.randperm(N, generator=g).to(torch.int32)
        k = torch.randn(next_page + 2, kv_heads, page, dim, generator=g)
        v = torch.randn(next_page + 2, kv_heads, page, dim, generator=g)
        for i, (pages, prefix, shared) in enumerate(rows):
            n = self.members[i]
            row = int(self.token_rows[n])
            table[row, :len(pages)] = places[torch.tensor(pages, dtype=torch.int64)].to(torch.int32)
            self.positions[n] = lengths[i] - 1
            if shared % page and pages[:len(prefix)] != prefix:     # its own copy of the prefix's last page
                a, b = int(places[prefix[-1]]), int(places[pages[len(prefix) - 1]])
                k[b], v[b] = k[a], v[a]
        self.q = torch.randn(N, heads * dim, generator=g).to(dtype)
        self.k, self.v, self.table = k.to(dtype), v.to(dtype), table
        self.starts, self.lens = starts, lens
        self.unused = [int(places[next_page])] if next_page < len(places) else []

    def poison(self):
        """NaN in every slot that no member holds, the null page's included."""
        held = torch.zeros(self.k.shape[0], self.page, dtype=torch.bool)
        for n in self.members:
            for j in range(int(self.positions[n]) + 1):
                held[int(self.table[int(self.token_rows[n]), j // self.page]), j % self.page] = True
        for t in (self.k, self.v):
            t.permute(0, 2, 1, 3)[~held] = math.nan
        return self

    def run(self, window=0, status=True, out=None, **kw):
        out = torch.full((self.N, self.heads * self.dim), 77.0, dtype=self.dtype, device="cuda") if out is None else out
        word = torch.zeros(1, dtype=torch.int32, device="cuda") if status else None
        self.device = [t.cuda() for t in (self.q, self.k, self.v, self.table, self.token_rows, self.positions)]
        self.lists = [ints(self.members), ints(self.starts), ints(self.lens)]
        ops.attention_shared(out, *self.device, *self.lists, self.heads, self.dim ** -0.5, window, status=word, **kw)
        if status:
            assert int(word.item()) == 0
        return out

    def want(self, window=0):
        G, want = self.heads // self.kv_heads, torch.full((self.N, self.heads * self.dim), 77.0, dtype=torch.float64)
        for n in self.members:
            pos, row = int(self.positions[n]), int(self.token_rows[n])
            at = torch.arange(max(0, pos - window + 1) if window else 0, pos + 1)
            pages = self.table[row].long()[at // self.page]
            for h in range(self.heads):
                k = self.k[pages, h // G, at % self.page].double()
                v = self.v[pages, h // G, at % self.page].double()
                s = k @ self.q[n, h * self.dim:(h + 1) * self.dim].double() * self.dim ** -0.5
                want[n, h * self.dim:(h + 1) * self.dim] = torch.softmax(s, -1) @ v
        return want


def check(case, got, want):
    """float32: sums of up to some thousand terms of weights that add up to 1; a term's error is a few 2^-24 of the value's
    size (scores up to about 6: their error of 2^-24 x 6 x sqrt(dim) terms moves a weight as much), so 2e-5 absolute for
    values of size 1.  bfloat16: the result's rounding (2^-8 of its size, at most 4) and weights in two terms of bfloat16
    (2^-16), exponentials of 2^-21: 2^-8 |want| + 1e-3."""
    got = got.double().cpu()
    if case.dtype == torch.float32:
        assert bool(((got - want).abs() <= 2e-5).all()), float((got - want).abs().max())
    else:
        assert bool(((got - want).abs() <= want.abs() * 2.0 ** -8 + 1e-3).all()), float((got - want).abs().max())


HEADS = [(4, 2, 16), (8, 2, 32), (16, 8, 64), (32, 8, 128), (8, 8, 128), (24, 2, 64), (12, 4, 96), (20, 1, 128), (4, 1, 256), (5, 1, 64)]
FAMILIES = {
    "one_token": [(0, [1])],
    "two_answers": [(32, [1, 40])],
    "nothing_shared": [(0, [5]), (0, [64]), (0, [130])],
    "several": [(16, [3, 1, 17]), (0, [33]), (144, [9] * 11), (80, [70])],
    "an_odd_prefix": [(77, [1, 2, 30, 3]), (63, [1, 5])],
    "no_own_keys": [(48, [0, 0, 5]), (37, [0, 3])],
    "more_rows_than_a_tile": [(100, list(range(1, 41)))],
    "long": [(1000, [1, 300, 64]), (500, [2, 2])],
    "large_families": [(130, [3] * 20), (0, [9]), (1000, [1, 64] * 15), (16, [2] * 9)],
    "a_hundred": [(400, [1, 30] * 50)],
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("families", FAMILIES)
def test_attention_shared(families, heads, dtype):
    case = Case(FAMILIES[families], *heads, dtype, seed=len(families), spare_tokens=2).poison()
    check(case, case.run(), case.want())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("window", [1, 20, 100, 5000])
@pytest.mark.parametrize("heads", [(8, 2, 32), (32, 8, 128), (12, 4, 96)], ids=str)
def test_attention_shared_windows(heads, window, dtype):
    """A window of 1 or 20 leaves most rows nothing of the prefix, one of 100 a part that differs by row."""
    case = Case([(96, [1, 5, 50, 200]), (160, [7] * 6 + [90]), (0, [40])], *heads, dtype, seed=window)
    check(case, case.run(window), case.want(window))


def test_attention_shared_of_more_members_than_the_lists_in_shared_memory_hold():
    case = Case([(32, [1, 3] * 300), (48, [2] * 3)], 4, 2, 32, torch.bfloat16, seed=8).poison()
    check(case, case.run(), case.want())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_shared_of_more_families_than_a_block_has_threads(dtype):
    case = Case([(16, [1, 2]), (0, [3])] * 150 + [(40, [5] * 9)] + [(0, [7])] * 270, 4, 2, 32, dtype, seed=4).poison()
    check(case, case.run(), case.want())


def test_attention_shared_of_one_family_where_as_many_families_as_members_have_no_place():
    """512 members of one large family; the lists of 512 families would not fit beside that kernel's tiles."""
    case = Case([(200, [1, 5] * 256)], 16, 1, 64, torch.bfloat16, seed=6).poison()
    check(case, case.run(), case.want())


def test_attention_shared_on_two_streams_at_once():
    """Two calls with scratch of their own, large families in both, beside one another again and again."""
    cases = [Case([(3500, [1, 70, 9] * 8), (64, [40, 3])], 32, 8, 128, torch.bfloat16, seed=s) for s in (1, 2)]
    outs, calls = [], []
    for case in cases:
        want = case.run()
        sizes = ops.attention_shared_scratch_size(len(case.members), case.heads, case.kv_heads, case.dim, case.page, case.dtype)
        part, lists = torch.empty(sizes[0], device="cuda"), torch.empty(sizes[1], dtype=torch.int32, device="cuda")
        outs.append((want, [torch.zeros_like(want) for _ in range(6)]))
        calls.append((case, part, lists, torch.zeros(1, dtype=torch.int32, device="cuda"), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for i in range(6):
        for (case, part, lists, word, stream), (_, got) in zip(calls, outs):
            with torch.cuda.stream(stream):
                ops.attention_shared(got[i], *case.device, *case.lists, case.heads, case.dim ** -0.5, 0, part, lists, word)
    torch.cuda.synchronize()
    for (want, got), (_, _, _, word, _) in zip(outs, calls):
        assert int(word.item()) == 0 and all(torch.equal(want, x) for x in got)


def test_attention_shared_large_families_with_windows():
    case = Case([(3300, [1, 5, 50, 200] * 5), (160, [7] * 7 + [90])], 32, 8, 128, torch.bfloat16, seed=2)
    for window in (3, 150, 2900):
        check(case, case.run(window), case.want(window))


@pytest.mark.parametrize("heads,shared", [((32, 8, 128), 4160), ((16, 8, 64), 6000), ((24, 2, 64), 1001)], ids=str)
@pytest.mark.parametrize("own", [1, 60, 100, 200, 300, 420, 900])
def test_attention_shared_beside_large_families(heads, shared, own):
    """A family large enough for the kernel of its own, beside own keys of all lengths: few tiles and many, chunks that are
    claimed one after the other and in advance; a small family and a lone token besides."""
    n = -(-(1 << 18) // (shared * (heads[0] // heads[1]))) + 1
    case = Case([(shared, [max(1, own - 7 * (i % 5)) for i in range(n)]), (64, [own, 3]), (0, [own])], *heads, torch.bfloat16, seed=own)
    first = case.run()
    check(case, first, case.want())
    assert torch.equal(case.run(), first)


@pytest.mark.parametrize("status", [True, False])
def test_attention_shared_twice_is_the_same_bits(status):
    """Nothing is added in the order in which blocks come; with and without the kernel for large families."""
    case = Case([(3500, [1, 70, 9] * 8), (64, [40, 3])], 32, 8, 128, torch.bfloat16, seed=9)
    first = case.run(status=status).clone()
    for _ in range(20):
        assert torch.equal(case.run(status=status), first)
    check(case, first, case.want())


@pytest.mark.parametrize("page", [1, 4, 32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_shared_page_sizes(page, dtype):
    case = Case([(128, [1, 77, 30]), (0, [50])], 16, 8, 64, dtype, page=page, seed=page).poison()
    check(case, case.run(), case.want())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_shared_large_scores(dtype):
    """Scores of some hundreds: the parts' maxima differ by far more than float32's exponent of e^x allows."""
    case = Case([(200, [3, 90]), (64, [1, 1])], 8, 2, 64, dtype, seed=3)
    case.q *= 30.0
    want = case.want()
    got = case.run().double().cpu()
    # a score's error is 2^-24 x 64 terms x |q k| ~ 2^-24 x 64 x 100, which weights follow: 5e-4 of values up to 4
    limit = want.abs() * (2.0 ** -8 if dtype == torch.bfloat16 else 0.0) + (4e-3 if dtype == torch.bfloat16 else 2e-3)
    assert bool(((got - want).abs() <= limit).all()), float((got - want).abs().max())


def test_attention_shared_nan_reaches_its_rows():
    """A NaN among a row's own keys makes that row NaN, and no other row of the family."""
    for dtype in (torch.bfloat16, torch.float32):
        case = Case([(64, [20, 20, 20])], 4, 2, 32, dtype, seed=1)
        n = case.members[1]
        case.k[int(case.table[int(case.token_rows[n]), 4]), :, 3] = math.nan
        got = case.run().cpu()
        assert bool(got[n].isnan().all())
        assert not bool(got[[case.members[0], case.members[2]]].isnan().any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_shared_replayed_with_other_families(dtype):
    """A recorded call follows the lists it is given at the time of the replay, and two graphs share one scratch."""
    first = Case([(64, [5, 9, 30, 2]), (0, [50]), (32, [1])], 32, 8, 128, dtype, seed=5)
    first.run()
    members, starts, lens = first.lists
    floats, counts = ops.attention_shared_scratch_size(6, 32, 8, 128, PAGE, dtype)
    part, lists = torch.empty(floats, device="cuda"), torch.zeros(counts, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    outs = [torch.zeros(6, 32 * 128, dtype=dtype, device="cuda") for _ in range(2)]
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph, out in zip(graphs, outs):
        with torch.cuda.graph(graph):
            ops.attention_shared(out, *first.device, *first.lists, 32, 128 ** -0.5, 0, part, lists, status)
    want = first.want()
    for graph, out in zip(graphs, outs):
        graph.replay()
        graph.replay()
        check(first, out, want)
    # the same rows as six families of their own
    starts.copy_(ints([0, 6, 6, 6]))
    lens.copy_(ints([0, 0, 0]))
    for graph, out in zip(graphs, outs):
        out.zero_()
        graph.replay()
        check(first, out, want)
    assert int(status.item()) == 0


def test_attention_shared_refusals():
    case = Case([(32, [1, 2])], 8, 2, 32, torch.bfloat16)
    case.run()
    q, k, v, table, rows, pos = case.device
    members, starts, lens = case.lists
    out = torch.zeros_like(q)
    good = dict(out=out, q=q, k_pool=k, v_pool=v, block_table=table, token_rows=rows, positions=pos, members=members,
                group_starts=starts, shared_lens=lens, num_heads=8, scale=1.0)
    ops.attention_shared(**good)
    floats, _ = ops.attention_shared_scratch_size(2, 8, 2, 32, PAGE, torch.bfloat16)
    for bad in (dict(out=out.float()), dict(v_pool=v[:, :1].contiguous()), dict(q=q[:, ::2]), dict(positions=pos.long()),
                dict(group_starts=starts[:1]), dict(num_heads=7), dict(window=-1), dict(members=ints([0, 1, 0])),
                dict(k_pool=k.half(), v_pool=v.half(), q=q.half(), out=out.half()), dict(token_rows=rows[:1]),
                dict(part=torch.empty(8, device="cuda")), dict(k_pool=k.cpu()), dict(block_table=table[0]),
                dict(part=torch.empty(floats, device="cuda"), lists=torch.zeros(9, device="cuda"))):
        with pytest.raises(KernelError):
            ops.attention_shared(**{**good, **bad})
    wide = torch.zeros(2, 2 * 264, dtype=torch.bfloat16, device="cuda")
    pool = torch.zeros(4, 2, 16, 264, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(KernelError):
        ops.attention_shared(**{**good, "out": wide, "q": wide, "k_pool": pool, "v_pool": pool, "num_heads": 2})


# ------------------------------------------------------------------ sampling
MIX = (0x7FEB352D, 0x846CA68B)


def mix(x):
    x = (x ^ (x >> 16)) * MIX[0] & 0xFFFFFFFF
    x = (x ^ (x >> 15)) * MIX[1] & 0xFFFFFFFF
    return x ^ (x >> 16)


def uniforms(seed, counter, V):
    key = mix(mix((seed & 0xFFFFFFFF) ^ 0x9E3779B9) ^ mix(((counter & 0xFFFFFFFF) + 0x85EBCA6B) & 0xFFFFFFFF))
    at = (torch.arange(V) + 0x165667B1) & 0xFFFFFFFF
    return ((mix(at ^ key) >> 9).double() + 0.5) / 2.0 ** 23


def pack(allowed):
    M, V = allowed.shape
    words = -(-V // 32)
    bits = torch.zeros(M, words * 32, dtype=torch.int64)
    bits[:, :V] = allowed.long()
    bits[:, V:] = 1                                         # what stands behind the vocabulary does not matter
    packed = (bits.view(M, words, 32) << torch.arange(32)).sum(-1)
    return torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32)


def adjust_64(logits, m, s):
    V = logits.shape[1]
    l = logits[m].double()
    if "history" in s:
        r, presence, frequency = s["penalties"][m].double().tolist()
        told, n, p = s["history"][int(s["history_rows"][m])], int(s["lengths"][m]), int(s["prompt_lens"][m])
        for t in sorted(set(told[:n].tolist())):
            if not 0 <= t < V:
                continue
            c = int((told[p:n] == t).sum())
            x = float(l[t])
            x = x / r if x > 0 else x * r
            l[t] = x - frequency * c - presence * (c > 0)
    if "bias_starts" in s:
        for i in range(int(s["bias_starts"][m]), int(s["bias_starts"][m + 1])):
            if 0 <= int(s["bias_ids"][i]) < V:
                l[int(s["bias_ids"][i])] += float(s["bias_values"][i])
    if "mask" in s and int(s["mask_rows"][m]) >= 0:
        word = s["mask"][int(s["mask_rows"][m])].long() & 0xFFFFFFFF
        at = torch.arange(V)
        l[(word[at // 32] >> (at % 32)) & 1 == 0] = -math.inf
    return l


def settings(M, V, W, g, biases=6, masks=True):
    lengths = torch.randint(1, W + 1, (M,), generator=g).to(torch.int32)
    prompt = (torch.rand(M, generator=g) * (lengths + 1)).to(torch.int32)
    s = {"history": (torch.rand(M + 3, W, generator=g) ** 3 * V).to(torch.int32),
         "history_rows": torch.randperm(M + 3, generator=g)[:M].to(torch.int32), "prompt_lens": prompt, "lengths": lengths,
         "penalties": torch.stack([0.6 + torch.rand(M, generator=g), torch.rand(M, generator=g) - 0.3, torch.rand(M, generator=g)], 1)}
    counts = torch.randint(0, biases + 1, (M,), generator=g)
    s["bias_starts"] = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).to(torch.int32)
    s["bias_ids"] = torch.randint(0, V, (int(counts.sum()),), generator=g).to(torch.int32)
    s["bias_values"] = 4 * torch.randn(int(counts.sum()), generator=g)
    if masks:
        s["mask"] = pack(torch.rand(M + 1, V, generator=g) < 0.5)
        s["mask_rows"] = (torch.randint(-1, M + 1, (M,), generator=g)).to(torch.int32)
    return s


def sample(logits, s, adjusted=True, **kw):
    M = logits.shape[0]
    out = torch.full((M,), -5, dtype=torch.int32, device="cuda")
    new = torch.full(logits.shape, 5.0, device="cuda") if adjusted else None
    ops.sample_adjusted(out, logits.cuda(), **{k: t.cuda() for k, t in kw.items()}, **{k: t.cuda() for k, t in s.items()}, adjusted=new)
    return out.cpu(), None if new is None else new.cpu()


@pytest.mark.parametrize("V", [1, 5, 31, 32, 33, 383, 8192, 8196, 9001, 151936])
@pytest.mark.parametrize("M,W", [(1, 1), (3, 700), (9, 64)])
@pytest.mark.parametrize("parts", ["all", "penalties", "biases", "masks", "none"])
def test_sample_adjusted(M, W, V, parts):
    g = torch.Generator().manual_seed(V + M)
    logits = 3 * torch.randn(M, V, generator=g)
    s = settings(M, V, W, g)
    names = {"all": tuple(s), "none": (), "biases": ("bias_starts", "bias_ids", "bias_values"), "masks": ("mask", "mask_rows"),
             "penalties": ("history", "history_rows", "prompt_lens", "lengths", "penalties")}[parts]
    s = {k: s[k] for k in names}
    T = torch.tensor([0.0 if m % 2 else 0.9 for m in range(M)])
    seeds, counters = torch.arange(M, dtype=torch.int32) * 77 - 5, torch.arange(M, dtype=torch.int32)
    tokens, adjusted = sample(logits, s, temperature=T, seeds=seeds, counters=counters)
    alone, _ = sample(logits, s, adjusted=False, temperature=T, seeds=seeds, counters=counters)
    assert torch.equal(tokens, alone)
    for m in range(M):
        want = adjust_64(logits, m, s)
        # five float32 operations on values of size 12 and below (counts of up to 700 times a number of size 1): half a step each
        limit = 5 * 2.0 ** -24 * (want.abs().clamp(min=12.0) + (700 if "history" in s else 0))
        same = (adjusted[m].double() == want) | (want.isfinite() & ((adjusted[m].double() - want).abs() <= limit))
        assert bool(same.all()), (m, float((adjusted[m].double() - want).abs().max()))
        got = adjusted[m].double()
        if float(T[m]) > 0:
            got = got / float(T[m]) - torch.log(-torch.log(uniforms(int(seeds[m]), int(counters[m]), V)))
        # the best of the scores as the kernel saw them, up to the float32 error of a score of size 40
        t = int(tokens[m])
        if bool((want == -math.inf).all()):
            assert t == 0
        else:
            assert float(got[t]) >= float(got.max()) - (0 if float(T[m]) == 0 else 2e-5)


def test_sample_adjusted_is_sample_where_nothing_is_adjusted():
    g = torch.Generator().manual_seed(0)
    logits = torch.randn(6, 32000, generator=g).cuda()
    kw = dict(temperature=torch.tensor([0.0, 0.5, 1.0, 0.0, 2.0, 0.7]).cuda(), seeds=ints(range(6)), counters=ints(range(6)))
    a, b = (torch.zeros(6, dtype=torch.int32, device="cuda") for _ in range(2))
    ops.sample(a, logits, **kw)
    ops.sample_adjusted(b, logits, **kw)
    assert torch.equal(a, b)


@pytest.mark.parametrize("V", [7, 1000, 32000, 151936, 151937])
@pytest.mark.parametrize("spread", [0.0, 1e-3, 2.5, 300.0])
def test_sample_adjusted_draws_as_sample_at_any_temperature(V, spread):
    """Which logits' noise is looked at changes no draw: all temperatures, flat and steep rows, the same scratch for both."""
    g = torch.Generator().manual_seed(V)
    M = 64
    logits = (spread * torch.randn(M, V, generator=g)).cuda()
    logits[5, ::3] = -math.inf
    logits[6] = -math.inf
    logits[7, V // 2] = math.inf
    logits[9, ::2] = math.nan
    T = torch.exp(6 * torch.rand(M, generator=g) - 3)
    T[:4] = torch.tensor([0.0, 1e-6, 1e-38, 1e30])
    kw = dict(temperature=T.cuda(), seeds=ints(torch.randint(-2 ** 31, 2 ** 31, (M,), generator=g).tolist()), counters=ints(range(M)),
              scratch=torch.zeros(ops.sample_scratch_size(M, V), dtype=torch.int32, device="cuda"))
    a, b, c = (torch.zeros(M, dtype=torch.int32, device="cuda") for _ in range(3))
    ops.sample(a, logits, **kw)
    ops.sample_adjusted(b, logits, **kw)
    ops.sample(c[:3], logits[:3], **{k: t if k == "scratch" else t[:3] for k, t in kw.items()})
    assert torch.equal(a, b) and torch.equal(a[:3], c[:3])


@pytest.mark.parametrize("W", [4096, 4097, 9001])
def test_sample_adjusted_long_histories_and_many_biases(W):
    """Histories beyond what a block holds in registers, hundreds of biases, tokens named again and again by both."""
    g = torch.Generator().manual_seed(W)
    M, V = 3, 20000
    logits = 3 * torch.randn(M, V, generator=g)
    s = settings(M, V, W, g, masks=False)
    s["lengths"][:] = torch.tensor([W, W - 3, W // 2], dtype=torch.int32)
    s["prompt_lens"][:] = torch.tensor([0, W // 2, W], dtype=torch.int32)
    s["history"] %= 300
    s["penalties"][:, 2] = 0.001
    s["bias_starts"] = torch.tensor([0, 700, 700, 1800], dtype=torch.int32)
    s["bias_ids"] = torch.randint(0, 400, (1800,), generator=g).to(torch.int32)
    s["bias_values"] = torch.randn(1800, generator=g)
    tokens, adjusted = sample(logits, s)
    for m in range(M):
        want = adjust_64(logits, m, s)
        # one division or product, two subtractions (9 for a count of 9,000), a sum of up to 30 biases of size 3 in their order: 40 roundings
        # of values of size 40
        assert bool(((adjusted[m].double() - want).abs() <= 40 * 2.0 ** -24 * 40).all())
        assert int(tokens[m]) == int(adjusted[m].argmax())


def test_sample_adjusted_ties_nothing_left_and_values_that_are_not_finite():
    V, inf = 300, math.inf
    logits = torch.zeros(5, V)
    logits[0, 7:] = 2.0                                     # a tie: the lowest index
    logits[1, 3], logits[1, 9] = math.nan, inf              # both masked away: the tie of what is left
    logits[2] = -inf
    logits[2, 250] = -1e38
    logits[3, 5] = inf
    allowed = torch.ones(3, V, dtype=torch.bool)
    allowed[0, [3, 9, 0]] = False
    allowed[1] = False                                      # nothing is left: 0
    s = {"mask": pack(allowed), "mask_rows": torch.tensor([-1, 0, 2, 2, 1], dtype=torch.int32)}
    tokens, adjusted = sample(logits, s)
    assert tokens.tolist() == [7, 1, 250, 5, 0]
    assert bool((adjusted[4] == -inf).all()) and adjusted[1, 3] == -inf and adjusted[3, 5] == inf
    # a bias of -inf takes a token out, one named twice gets both, an id outside the vocabulary is passed over
    s = {"bias_starts": torch.tensor([0, 1, 1, 4, 6, 6], dtype=torch.int32),
         "bias_ids": torch.tensor([7, 250, 4, 4, -1, 300], dtype=torch.int32),
         "bias_values": torch.tensor([-inf, -inf, 1.0, 0.5, 9.0, 9.0])}
    tokens, adjusted = sample(logits.nan_to_num(nan=0.0, posinf=50.0, neginf=-1.0), s)
    assert tokens.tolist() == [8, 9, 4, 5, 0] and adjusted[2, 4] == 0.5


def test_sample_adjusted_in_place_replayed_and_on_another_stream():
    g = torch.Generator().manual_seed(4)
    M, V = 4, 20000
    s = {k: t.cuda() for k, t in settings(M, V, 50, g).items()}
    logits = torch.randn(M, V, generator=g).cuda()
    want, keep = torch.zeros(M, dtype=torch.int32, device="cuda"), torch.empty(M, V, device="cuda")
    ops.sample_adjusted(want, logits, **s, adjusted=keep)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    out, work = torch.zeros_like(want), logits.clone()
    scratch = torch.zeros(ops.sample_scratch_size(M, V), dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ops.sample_adjusted(out, work, None, None, None, scratch, **s, adjusted=work)
    for _ in range(2):
        work.copy_(logits)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(work, keep)
    s["history"].fill_(V + 5)                               # tokens of no vocabulary: no penalties
    s["mask_rows"].fill_(-1)
    s["bias_values"].zero_()
    work.copy_(logits)
    graph.replay()
    assert torch.equal(work, logits) and torch.equal(out.long(), logits.argmax(-1))


def test_sample_adjusted_refusals():
    g = torch.Generator().manual_seed(4)
    logits = torch.zeros(3, 100, device="cuda")
    s = {k: t.cuda() for k, t in settings(3, 100, 8, g).items()}
    out = torch.zeros(3, dtype=torch.int32, device="cuda")
    ops.sample_adjusted(out, logits, **s)
    for bad in ({"penalties": s["penalties"][:, :2].contiguous()}, {"history": None}, {"lengths": s["lengths"].long()},
                {"bias_starts": s["bias_starts"][:3]}, {"bias_values": s["bias_values"][1:]}, {"bias_ids": None},
                {"mask": s["mask"][:, :3].contiguous()}, {"mask_rows": None}, {"adjusted": torch.zeros(3, 99, device="cuda")},
                {"temperature": torch.zeros(3, device="cuda")}, {"scratch": torch.zeros(2, dtype=torch.int32, device="cuda")},
                {"prompt_lens": s["prompt_lens"].cpu()}, {"history": s["history"][0]}):
        with pytest.raises(KernelError):
            ops.sample_adjusted(out, logits, **{**s, **bad})
    wide = torch.zeros(1, 262145, device="cuda")
    with pytest.raises(KernelError):
        ops.sample_adjusted(out[:1], wide)


def test_bytes_are_no_page_numbers():
    k, v = (torch.zeros(2, 6, 2, 16, 32, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    for n in (4, 5):
        with pytest.raises(KernelError):
            ops.copy_pages(k, v, bytes(n), bytes(n))


def test_sample_adjusted_of_no_rows():
    ops.sample_adjusted(ints([]), torch.zeros(0, 100, device="cuda"))
    ops.note_tokens(torch.zeros(2, 3, dtype=torch.int32, device="cuda"), ints([]), ints([]), ints([]))


@pytest.mark.parametrize("N", [1, 300, 3000])
@pytest.mark.parametrize("feedback", [True, False])
def test_note_tokens(N, feedback):
    g = torch.Generator().manual_seed(N)
    rows, width = 37, 90
    place = torch.randperm(rows * width, generator=g)[:N]
    ids = torch.randint(0, 1000, (N,), generator=g)
    fed = torch.randint(0, 1000, (50,), generator=g) if feedback else None
    if feedback:
        ids[::3] = -1 - torch.randint(0, 50, ids[::3].shape, generator=g)
    r, p = place // width, place % width
    want = torch.full((rows, width), 5)
    want[r, p] = torch.where(ids < 0, fed[(-1 - ids).clamp(0)], ids) if feedback else ids
    # places outside: nothing is written, and nothing behind the table either
    outside = [(-1, 0), (rows, 0), (0, -1), (0, width), (2 ** 31 - 1, 2 ** 31 - 1), (-2 ** 31, 5)]
    for a, b in outside:
        ids, r, p = (torch.cat([t, torch.tensor([x])]) for t, x in ((ids, 9), (r, a), (p, b)))
    flat = torch.full((rows * width + 200,), 5, dtype=torch.int32, device="cuda")
    ops.note_tokens(flat[100:-100].view(rows, width), ints(ids.tolist()), ints(r.tolist()), ints(p.tolist()),
                    None if fed is None else ints(fed.tolist()))
    assert torch.equal(flat[100:-100].view(rows, width).cpu().long(), want)
    assert bool((flat[:100] == 5).all()) and bool((flat[-100:] == 5).all())


def test_note_tokens_refusals():
    h, one = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), ints([1])
    for bad in ((h.float(), one, one, one), (h[0], one, one, one), (h.t(), one, one, one), (h, one, ints([1, 2]), one),
                (h, one, one, one.float()), (h.cpu(), one, one, one), (h, one.cpu(), one, one), (h, one, one, one, one.float())):
        with pytest.raises(KernelError):
            ops.note_tokens(*bad)
    assert not bool(h.any())
