"""A step's metadata laid out on the GPU from the requests' lengths, against lists."""

import random

import pytest

torch = pytest.importorskip("torch")

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]

DEV = "cuda:0"


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


class Case:
    def __init__(self, q, context, page, seed=0, window=0, keep_first=0, shared=None, padding=(), spare=5, width=None, rows=None,
                 use_rows=True):
        rng = random.Random(seed)
        n = len(q)
        self.q, self.context, self.page, self.window, self.keep_first = list(q), list(context), page, window, keep_first
        self.padding = set(padding)
        have = [-(-c // page) for c in context]
        need = [-(-(c + t) // page) - h for c, t, h in zip(context, q, have)]
        self.width = width or max(1, max(h + k for h, k in zip(have, need)) + 2)
        n_rows = n + 4
        self.rows = rows or (rng.sample(range(n_rows), n) if use_rows else list(range(n)))
        self.use_rows = use_rows
        self.shared = shared or [(-1, 0)] * n          # (leader's sequence, pages)
        pages = list(range(sum(have) + sum(need) + 7))
        rng.shuffle(pages)
        self.n_pages = len(pages)
        self.tables = [[-1] * self.width for _ in range(n_rows)]
        for s in range(n):
            for k in range(have[s]):
                self.tables[self.rows[s]][k] = pages.pop()
        self.free = pages
        self.n_tokens = sum(q) + spare

    def expected(self):
        cu, positions, tok_seq, slots, at = [0], [], [], [], 0
        tables = [list(row) for row in self.tables]
        for s, (q, context) in enumerate(zip(self.q, self.context)):
            row = tables[self.rows[s]]
            for k in range(-(-context // self.page), -(-(context + q) // self.page)):
                row[k] = self.free[at]
                at += 1
            for p in range(context, context + q):
                positions.append(p)
                tok_seq.append(s)
                slots.append(row[p // self.page] * self.page + p % self.page)
            cu.append(cu[-1] + q)
        block = []
        for s, (q, context) in enumerate(zip(self.q, self.context)):
            out = [-1] * self.width
            leader, pages = self.shared[s]
            low = 0
            if self.window > 0:
                low = max(0, context - self.window + 1) // self.page
            elif self.window < 0:
                low = (context - context % -self.window) // self.page
            kept = -(-self.keep_first // self.page) if self.window > 0 else 0
            for k in range(-(-(context + q) // self.page)):
                if k < kept or k >= low:
                    out[k] = (tables[self.rows[leader]] if k < pages and leader >= 0 else tables[self.rows[s]])[k]
            block.append(out)
        pad = self.n_tokens - len(positions)
        return {"cu_q": cu, "positions": positions + [0] * pad, "tok_seq": tok_seq + [-1] * pad, "slots": slots + [-1] * pad,
                "block_tables": block, "taken": [at], "tables": tables}

    def device(self):
        n = len(self.q)
        self.inputs = {"q_lens": ints(self.q), "context_lens": ints(self.context), "rows": ints(self.rows) if self.use_rows else None,
                       "tables": ints(self.tables), "free_pages": ints(self.free), "n_free": ints([len(self.free)])}
        self.outputs = {"positions": ints([77] * self.n_tokens), "tok_seq": ints([77] * self.n_tokens), "cu_q": ints([77] * (n + 1)),
                        "slots": ints([77] * self.n_tokens), "block_tables": ints([[77] * self.width] * n), "taken": ints([77])}
        self.status = ints([0])
        self.more = {"window": self.window, "keep_first": self.keep_first}
        if any(leader >= 0 for leader, _ in self.shared):
            self.more["shared_rows"] = ints([self.rows[leader] if leader >= 0 else -1 for leader, _ in self.shared])
            self.more["shared_pages"] = ints([pages for _, pages in self.shared])
        return self

    def run(self):
        from matricxon_b200.ops import kernels

        i, o = self.inputs, self.outputs
        kernels.step_tables(i["q_lens"], i["context_lens"], i["rows"], i["tables"], i["free_pages"], i["n_free"], self.page,
                            self.n_pages, o["positions"], o["tok_seq"], o["cu_q"], o["slots"], o["block_tables"], o["taken"],
                            self.status, **self.more)
        return {**{k: v.tolist() for k, v in o.items()}, "tables": i["tables"].tolist()}

    def empty(self):
        n = len(self.q)
        return {"cu_q": [0] * (n + 1), "positions": [0] * self.n_tokens, "tok_seq": [-1] * self.n_tokens,
                "slots": [-1] * self.n_tokens, "block_tables": [[-1] * self.width] * n, "taken": [0], "tables": self.tables}


def random_case(n, page, seed, most=500, **more):
    rng = random.Random(seed)
    return Case([rng.choice((0, 1, 1, 1, rng.randrange(1, 70))) for _ in range(n)], [rng.randrange(most) for _ in range(n)], page, seed, **more)


@pytest.mark.parametrize("n", [1, 2, 31, 33, 255, 256, 257, 600, 1300])
@pytest.mark.parametrize("page", [1, 8, 16, 24, 32])
def test_lengths_of_all_kinds(n, page):
    case = random_case(n, page, n + page).device()
    expected = case.expected()
    for _ in range(2):                                  # laid out again: the same
        assert case.run() == expected
    assert case.status.item() == 0


@pytest.mark.parametrize("use_rows", [True, False])
@pytest.mark.parametrize("q,context", [([1], [0]), ([0], [0]), ([0], [37]), ([16], [0]), ([16], [16]), ([17], [15]), ([1], [31]), ([1], [32])])
def test_ends_of_pages(q, context, use_rows):
    case = Case(q, context, 16, use_rows=use_rows).device()
    assert case.run() == case.expected() and case.status.item() == 0


@pytest.mark.parametrize("window,keep_first", [(1, 0), (16, 0), (17, 0), (100, 0), (100, 5), (64, 33), (10000, 4), (-64, 0), (-17, 0), (0, 9)])
def test_pages_out_of_sight(window, keep_first):
    case = random_case(40, 16, 5, window=window, keep_first=keep_first).device()
    assert case.run() == case.expected() and case.status.item() == 0


def test_the_cache_managers_rule():
    """The entries are those that the host's manager keeps for the same lengths."""
    from matricxon_b200.cache.manager import CacheManager, GroupRule

    for window, keep_first, block in ((None, 0, None), (40, 0, None), (40, 20, None), (None, 0, 48)):
        manager = CacheManager([GroupRule(window, keep_first, block)], 400, 16, 8)
        lengths = [0, 1, 15, 16, 100, 129]
        for s, length in enumerate(lengths):
            manager.add_request(str(s))
            for part in (length // 2, length - length // 2):
                if part:
                    manager.reserve(str(s), part)
                    manager.commit(str(s), part)
        q = [1, 16, 1, 1, 33, 2]
        case = Case(q, lengths, 16, window=-block if block else window or 0, keep_first=keep_first, rows=list(range(6)), width=12)
        case.n_pages = 400
        case.tables = [list(manager.table_row(str(s), 0, 12)) for s in range(6)] + [[-1] * 12] * 4
        case.tables = [[int(v) for v in row] for row in case.tables]
        before = [len(manager.record(str(s)).tables[0]) for s in range(6)]
        for s in range(6):
            manager.reserve(str(s), q[s])
        case.free = [page for s in range(6) for page in manager.record(str(s)).tables[0][before[s]:]] + [399]
        case.device()
        got = case.run()
        assert case.status.item() == 0
        at = 0
        for s in range(6):
            assert got["block_tables"][s] == manager.table_row(str(s), 0, 12).tolist()
            assert got["slots"][at:at + q[s]] == manager.slot_ids(str(s), 0, lengths[s], q[s]).tolist()
            at += q[s]


def test_shared_pages():
    """Sequences that read their first pages through another one's row, one that is not in the step's order among them."""
    context = [100, 64, 80, 33, 200]
    shared = [(-1, 0), (0, 4), (4, 5), (-1, 0), (0, 6)]
    case = Case([1, 1, 20, 1, 1], context, 16, shared=shared, seed=2).device()
    assert case.run() == case.expected() and case.status.item() == 0


def test_padding_sequences_bring_nothing():
    case = Case([1, 0, 1, 0], [5, 0, 40, 0], 16, seed=3)
    case.device()
    expected = case.expected()
    case.inputs["rows"][1] = case.inputs["rows"][3] = -1
    assert case.run() == expected and case.status.item() == 0


@pytest.mark.parametrize("width", [9000, 40000])
def test_tables_wider_than_a_blocks_share(width):
    case = Case([1, 3], [70000, 10], 16, width=width).device()
    assert case.run() == case.expected() and case.status.item() == 0


@pytest.mark.parametrize("fault", ["rows", "pages", "width", "negative", "context", "row", "shared", "padding"])
@pytest.mark.parametrize("n", [3, 700])
def test_a_step_that_does_not_fit_comes_out_empty(fault, n):
    case = Case([1 + (s % 5 == 0) * 30 for s in range(n)], [s % 90 for s in range(n)], 16, seed=1)
    if fault == "shared":
        case.shared = [(0, 0) if s else (-1, 0) for s in range(n)]
    case.device()
    i, last = case.inputs, n - 1
    if fault == "rows":
        case.n_tokens = sum(case.q) - 1
        for name in ("positions", "tok_seq", "slots"):
            case.outputs[name] = case.outputs[name][:case.n_tokens].clone()
    elif fault == "pages":
        i["n_free"].fill_(case.expected()["taken"][0] - 1)
    elif fault == "width":
        i["context_lens"][last] = case.width * 16
    elif fault == "negative":
        i["q_lens"][last] = -1
    elif fault == "context":
        i["context_lens"][last] = -16
    elif fault == "row":
        i["rows"][last] = len(case.tables)
    elif fault == "padding":
        i["rows"][last] = -1
    else:
        case.more["shared_pages"][last] = 1000
    assert case.run() == case.empty()
    assert case.status.item() == 16


def test_a_row_listed_twice():
    """The first sequence of a row is laid out, the later one is empty and reported."""
    case = Case([1, 1, 1], [20, 40, 20], 16, seed=1).device()
    case.inputs["rows"][2] = case.inputs["rows"][0]
    got = case.run()
    assert case.status.item() == 16
    expected = case.expected()
    assert got["block_tables"][:2] == expected["block_tables"][:2] and got["slots"][:2] == expected["slots"][:2]
    assert got["block_tables"][2] == [-1] * case.width and got["slots"][2] == -1 and got["tok_seq"][2] == -1


def test_a_page_outside_the_pool_is_reported():
    case = Case([1, 1], [20, 40], 16, seed=1).device()
    case.inputs["tables"][case.rows[1], 0] = case.n_pages
    got = case.run()
    assert case.status.item() == 4 and got["block_tables"][1][0] == -1 and got["block_tables"][0] == case.expected()["block_tables"][0]


def test_captured_with_other_lengths():
    a, b = random_case(40, 16, 1, spare=3000, width=64).device(), random_case(40, 16, 2, width=64)
    b.n_tokens = a.n_tokens
    a.run()
    from matricxon_b200.ops import kernels

    i, o = a.inputs, a.outputs
    free = torch.zeros(4000, dtype=torch.int32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        kernels.step_tables(i["q_lens"], i["context_lens"], i["rows"], i["tables"], free, i["n_free"], 16, 8000, o["positions"],
                            o["tok_seq"], o["cu_q"], o["slots"], o["block_tables"], o["taken"], a.status)
    i["q_lens"].copy_(ints(b.q))
    i["context_lens"].copy_(ints(b.context))
    i["rows"].copy_(ints(b.rows))
    i["tables"].copy_(ints(b.tables))
    free[:len(b.free)] = ints(b.free)
    i["n_free"].fill_(len(b.free))
    graph.replay()
    assert {**{k: v.tolist() for k, v in o.items()}, "tables": i["tables"].tolist()} == b.expected()
    assert a.status.item() == 0


def test_refusals():
    from matricxon_b200.ops.library import KernelLibraryError

    def broken(**changes):
        case = Case([1, 2], [5, 6], 16).device()
        for name, value in changes.items():
            where = case.inputs if name in case.inputs else case.outputs if name in case.outputs else case.more
            where[name] = value(where.get(name)) if callable(value) else value
        with pytest.raises(KernelLibraryError):
            case.run()

    broken(q_lens=lambda t: t.long())
    broken(context_lens=lambda t: t[:1])
    broken(tables=lambda t: t.t())
    broken(tables=lambda t: t.cpu())
    broken(slots=lambda t: t[:1])
    broken(block_tables=lambda t: t[:, :-1].contiguous())
    broken(shared_rows=ints([-1, -1]))
    broken(keep_first=-1)
    case = Case([1, 2], [5, 6], 16, use_rows=False).device()      # the step's tables in place of the requests'
    case.inputs["tables"] = case.outputs["block_tables"]
    with pytest.raises(KernelLibraryError):
        case.run()
    case = Case([1, 2], [5, 6], 16).device()
    case.page = 0
    with pytest.raises(KernelLibraryError):
        case.run()
    case.page, case.n_pages = 1 << 16, 1 << 16
    with pytest.raises(KernelLibraryError):
        case.run()


@pytest.mark.parametrize("n", [4, 70, 700])
@pytest.mark.parametrize("n_rows", [None, 70000])
def test_a_row_listed_twice_takes_nothing(n, n_rows):
    """The later sequences of a row bring no rows and take no pages; the others come out as without them."""
    rng = random.Random(n)
    case = Case([rng.choice((1, 1, 17)) for _ in range(n)], [16 * rng.randrange(4) for _ in range(n)], 16, seed=n, spare=40 * n)
    if n_rows:                                            # rows far apart
        case.rows = [r * (n_rows // len(case.tables)) for r in case.rows]
        tables = [[-1] * case.width for _ in range(n_rows)]
        for s, row in enumerate(case.rows):
            for k in range(-(-case.context[s] // 16)):
                tables[row][k] = s * 4 + k
        case.tables, case.n_pages = tables, 4 * n + n * 2
        case.free = list(range(4 * n, 6 * n))
    again = sorted(rng.sample(range(1, n), max(1, n // 9)))
    without = list(case.q)
    for s in again:
        without[s] = 0
    case.device()
    for s in again:
        case.inputs["rows"][s] = case.rows[rng.choice([0] + [r for r in range(s) if r not in again])]
    got = case.run()
    assert case.status.item() == 16
    case.q = without
    expected = case.expected()
    for s in again:
        expected["block_tables"][s] = [-1] * case.width
    assert got == expected
    case.status.zero_()
    assert case.run() == expected and case.status.item() == 16


def test_rows_far_apart_that_are_not_the_same():
    """Rows 65,536 apart, which the kernel cannot tell apart at first."""
    rows = [5, 5 + 65536, 9, 131081, 70000, 65545]
    case = Case([1, 2, 1, 17, 1, 1], [5, 40, 16, 0, 31, 100], 16, seed=1)
    case.rows = rows
    tables = [[-1] * case.width for _ in range(131100)]
    at = 0
    for s, row in enumerate(rows):
        for k in range(-(-case.context[s] // 16)):
            tables[row][k], at = at, at + 1
    case.tables, case.free, case.n_pages = tables, list(range(at, at + 20)), at + 20
    case.device()
    assert case.run() == case.expected() and case.status.item() == 0


def stale(case, seed):
    """Valid page numbers of an earlier tenant behind what each row holds."""
    rng = random.Random(seed)
    for s, row in enumerate(case.rows):
        for k in range(-(-case.context[s] // case.page), case.width):
            case.tables[row][k] = rng.randrange(case.n_pages)
    return case


@pytest.mark.parametrize("n", [3, 40, 700])
@pytest.mark.parametrize("use_rows", [True, False])
def test_shared_pages_that_the_leader_takes_in_the_same_step(n, use_rows):
    """A prompt portion fills the prefix's pages in the step in which others begin behind them."""
    rng = random.Random(n)
    lead = n // 2
    context = [160 + rng.randrange(40) for _ in range(n)]
    q = [rng.choice((1, 1, 9)) for _ in range(n)]
    context[lead], q[lead] = 40, 130
    shared = [(lead, rng.randrange(1, 11)) if s != lead and rng.random() < 0.8 else (-1, 0) for s in range(n)]
    shared[0], shared[-1] = (lead, 10), (lead, 7)
    if lead in (0, n - 1):
        shared[lead] = (-1, 0)
    case = stale(Case(q, context, 16, seed=n, shared=shared, use_rows=use_rows), n).device()
    expected = case.expected()
    for _ in range(5):
        assert case.run() == expected
        assert case.status.item() == 0


def test_more_shared_pages_than_the_leader_has():
    """Pages that the leader neither holds nor takes are none, and reported, whatever stands in its row."""
    case = stale(Case([1, 3, 1], [200, 20, 200], 16, seed=4, shared=[(1, 2), (-1, 0), (1, 5)]), 4).device()
    expected = case.expected()
    expected["block_tables"][2][2:5] = [-1] * 3
    assert case.run() == expected and case.status.item() == 4


def test_a_leader_that_is_listed_twice():
    """The first sequence of a row is the leader, and what the later ones would take is not counted before it."""
    case = stale(Case([5, 17, 20, 1], [16, 30, 30, 90], 16, seed=4, shared=[(-1, 0), (-1, 0), (-1, 0), (2, 3)]), 4).device()
    case.inputs["rows"][1] = case.rows[0]
    got = case.run()
    assert case.status.item() == 16
    case.q[1] = 0
    expected = case.expected()
    expected["block_tables"][1] = [-1] * case.width
    assert got == expected


def test_tables_that_lie_in_one_another_are_refused():
    """The step's block tables in a part of the requests' tables, or over their end."""
    from matricxon_b200.ops.library import KernelLibraryError

    for begin in (1, 4, 11):
        case = Case([1, 2], [5, 6], 16, width=3).device()
        memory = torch.full((6 * 3 + 20,), -1, dtype=torch.int32, device=DEV)
        memory[:18] = case.inputs["tables"].view(-1)
        case.inputs["tables"] = memory[:18].view(6, 3)
        case.outputs["block_tables"] = memory[begin:begin + 6].view(2, 3)
        with pytest.raises(KernelLibraryError):
            case.run()
        case = Case([1, 2], [5, 6], 16, width=3).device()
        memory[6:24] = case.inputs["tables"].view(-1)
        case.inputs["tables"] = memory[6:24].view(6, 3)
        case.outputs["block_tables"] = memory[1:7].view(2, 3)
        with pytest.raises(KernelLibraryError):
            case.run()
    case = Case([1, 2], [5, 6], 16, width=3).device()             # side by side: fine
    memory[:18] = case.inputs["tables"].view(-1)
    case.inputs["tables"], case.outputs["block_tables"] = memory[:18].view(6, 3), memory[18:24].view(2, 3)
    assert case.run() == case.expected() and case.status.item() == 0


def test_calls_queued_on_two_streams():
    """Calls with inputs and outputs of their own, queued on two streams without reading back in between."""
    cases = [random_case(300, 16, s).device() for s in range(8)]
    expected = [case.expected() for case in cases]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    from matricxon_b200.ops import kernels

    for _ in range(20):
        for i, case in enumerate(cases):
            with torch.cuda.stream(streams[i % 2]):
                a, o = case.inputs, case.outputs
                for out in o.values():
                    out.fill_(77)
                kernels.step_tables(a["q_lens"], a["context_lens"], a["rows"], a["tables"], a["free_pages"], a["n_free"], 16, case.n_pages,
                                    o["positions"], o["tok_seq"], o["cu_q"], o["slots"], o["block_tables"], o["taken"], case.status)
    torch.cuda.synchronize()
    for case, want in zip(cases, expected):
        assert {**{k: v.tolist() for k, v in case.outputs.items()}, "tables": case.inputs["tables"].tolist()} == want
        assert case.status.item() == 0


def test_leaders_among_many_rows():
    """More rows of tables than the kernel keeps notes of."""
    shared = [(2, 10), (2, 7), (-1, 0), (4, 9), (-1, 0), (1, 12)]
    case = Case([1, 1, 130, 3, 1, 1], [160, 200, 40, 171, 300, 200], 16, seed=5, shared=shared)
    rows = [r * 900 for r in case.rows]
    tables = [[-1] * case.width for _ in range(10000)]
    for old, new in zip(case.rows, rows):
        tables[new] = case.tables[old]
    case.rows, case.tables = rows, tables
    case = stale(case, 5).device()
    assert case.run() == case.expected() and case.status.item() == 0


@pytest.mark.parametrize("n", [4, 300])
@pytest.mark.parametrize("use_rows", [True, False])
@pytest.mark.parametrize("n_rows", [None, 5000])
def test_a_leader_that_brings_nothing_is_read_as_it_is(n, use_rows, n_rows):
    """A finished request that the batch still has a place for: its lengths are 0, its row still holds the prefix."""
    context = [0] + [80 + s % 40 for s in range(n - 1)]
    shared = [(-1, 0)] + [(0, 1 + s % 5) for s in range(n - 1)]
    case = Case([0] + [1] * (n - 1), context, 16, seed=n, shared=shared, use_rows=use_rows)
    case.n_pages += 5
    case.tables[case.rows[0]][:5] = range(case.n_pages - 5, case.n_pages)
    if n_rows:
        case.tables += [[-1] * case.width for _ in range(n_rows - len(case.tables))]
    case.device()
    assert case.run() == case.expected() and case.status.item() == 0
