"""Attention over keys that the sequences of a group have in common, against a plain implementation in float64."""

import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]

DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


class Step:
    """A step on the device: ``groups`` lists (shared keys, [(own keys before the step, tokens), ...]). Every slot of the
    cache that holds no key of a sequence is NaN; ``spare`` rows behind the last sequence's belong to nobody."""

    def __init__(self, groups, heads, kv_heads, dim, page, dtype, seed=0, spare=0, extra_pages=0, spread=1.0):
        gen = torch.Generator().manual_seed(seed)
        self.heads, self.kv_heads, self.dim, self.page, self.dtype = heads, kv_heads, dim, page, dtype
        self.groups = groups
        seqs = [(g, shared, before, q) for g, (shared, members) in enumerate(groups) for before, q in members]
        self.q_lens = [q for _, _, _, q in seqs]
        self.lens = [shared for _, shared, _, _ in seqs]
        self.context = [shared + before for _, shared, before, _ in seqs]
        totals = [c + q for c, q in zip(self.context, self.q_lens)]
        first, at = [0], 0
        for _, members in groups:
            at += len(members)
            first.append(at)
        self.first = first
        width = max(-(-t // page) for t in totals)
        count = sum(-(-(s + page) // page) for s, _ in groups) + sum(-(-t // page) + 1 for t in totals) + extra_pages
        order = torch.randperm(count, generator=gen).tolist()
        self.tables = [[-1] * width for _ in seqs]
        cache = torch.full((count, 2, kv_heads, page, dim), float("nan"))
        keys, values = cache[:, 0], cache[:, 1].view(count, kv_heads, dim, page)
        self.dense = []
        shared_of = {}
        for s, (g, shared, _, _) in enumerate(seqs):
            total = totals[s]
            k, v = torch.randn(total, kv_heads, dim, generator=gen) * spread, torch.randn(total, kv_heads, dim, generator=gen)
            k, v = k.to(dtype).float(), v.to(dtype).float()
            if g in shared_of:
                leader, lk, lv = shared_of[g]
                k[:shared], v[:shared] = lk[:shared], lv[:shared]
            else:
                shared_of[g] = (s, k, v)
            whole = shared // page                      # a page that the shared keys fill in part is everybody's own copy
            for i in range(-(-total // page)):
                if i < whole and shared_of[g][0] != s:
                    self.tables[s][i] = self.tables[shared_of[g][0]][i]
                    continue
                self.tables[s][i] = order.pop()
                a, b = i * page, min(total, (i + 1) * page)
                keys[self.tables[s][i], :, :b - a] = k[a:b].transpose(0, 1)
                values[self.tables[s][i], :, :, :b - a] = v[a:b].permute(1, 2, 0)
            self.dense.append((k.double(), v.double()))
        n = sum(self.q_lens)
        self.n = n + spare
        self.q = (torch.randn(self.n, heads * dim, generator=gen) * 1.5).to(dtype)
        cu = [0]
        for q in self.q_lens:
            cu.append(cu[-1] + q)
        self.cu = cu
        self.d = {"q": self.q.to(DEV), "cache": cache.to(dtype).to(DEV), "tables": ints(self.tables), "cu": ints(cu),
                  "context": ints(self.context), "first": ints(first), "lens": ints(self.lens),
                  "tok_seq": ints([s for s, q in enumerate(self.q_lens) for _ in range(q)] + [-1] * spare),
                  "positions": ints([c + i for c, q in zip(self.context, self.q_lens) for i in range(q)] + [0] * spare),
                  "status": ints([0])}

    def bounds(self):
        return {"max_q_len": max(self.q_lens), "max_shared_len": max(self.lens),
                "max_own_len": max(c + q - s for c, q, s in zip(self.context, self.q_lens, self.lens))}

    def run(self, window=None, softcap=None, sink=None, out=None, **more):
        from matricxon_b200.ops import kernels

        d = self.d
        if out is None:
            out = torch.full((self.n, self.heads * self.dim), float("nan"), dtype=self.dtype, device=DEV)
        kernels.paged_attention_shared(d["q"], d["q"].stride(0), d["cache"], d["tables"], d["cu"], d["context"], d["tok_seq"],
                                       d["positions"], d["first"], d["lens"], self.n, self.heads, self.kv_heads, self.dim, window,
                                       self.dim ** -0.5, out, d["status"], softcap=softcap, sink=sink, **{**self.bounds(), **more})
        return out

    def plain(self, window=None, softcap=None, sink=None):
        """(result, how far the kernels may be off it), both float64 [tokens, heads * dim].

        A score of d terms is off by at most (d + 4) half steps of float of the sum of its terms' sizes, twice that with the
        cap's tanh; a weight relatively by that much and the exponential's own few steps, the quotient of two sums of n weights
        by twice it and 2 n half steps. In bfloat16 a weight is rounded once more before it meets its value; the result is
        rounded once."""
        group, half = self.heads // self.kv_heads, torch.finfo(F32).eps / 2
        out_half = torch.finfo(self.dtype).eps / 2
        rows, bounds = [], []
        for s, (k, v) in enumerate(self.dense):
            a, b = self.cu[s], self.cu[s + 1]
            q = self.q[a:b].double().view(b - a, self.kv_heads, group, self.dim)
            score = torch.einsum("tkgd,jkd->tkgj", q, k) * self.dim ** -0.5
            size = torch.einsum("tkgd,jkd->tkgj", q.abs(), k.abs()) * self.dim ** -0.5
            if softcap:
                score = softcap * torch.tanh(score / softcap)
            p = torch.arange(self.context[s], self.context[s] + b - a)[:, None]
            j = torch.arange(k.shape[0])[None]
            seen = j <= p
            if window:
                seen = seen & ((j > p - window) if window > 0 else (j >= p - p % -window))
            score = score.masked_fill(~seen[:, None, None], -math.inf)
            size = size.masked_fill(~seen[:, None, None], 0.0)
            if sink is not None:
                extra = sink.double().cpu().view(1, self.kv_heads, group, 1).expand(b - a, -1, -1, -1)
                weights = torch.softmax(torch.cat([score, extra], -1), -1)[..., :-1]
            else:
                weights = torch.softmax(score, -1)
            result = torch.einsum("tkgj,jkd->tkgd", weights, v)
            sizes = torch.einsum("tkgj,jkd->tkgd", weights, v.abs())
            off = (2 * (self.dim + 4) * half * size.amax(-1) + 32 * half)[..., None] * 2 + (2 * k.shape[0] + 16) * half
            if softcap:
                off = off + 8e-7 * softcap          # the caps' own tanh: a few 1e-7 of the cap (common.cuh)
            rounded = torch.finfo(BF16).eps / 2 if self.dtype == BF16 else 0.0
            rows.append(result.reshape(b - a, self.heads * self.dim))
            bounds.append(((off + rounded) * sizes + out_half * result.abs()).reshape(b - a, self.heads * self.dim))
        return torch.cat(rows), torch.cat(bounds)


def close(step, out, **masks):
    ref, bound = step.plain(**masks)
    got = out[:ref.shape[0]].double().cpu()
    worst = ((got - ref).abs() / bound).max().item()
    assert worst <= 1.0, worst
    assert step.d["status"].item() == 0


# heads, KV heads, dim, page, dtype: tcgen05, mma.sync and the FP32 cores, groups of 1 to 130 heads
SHAPES = [(24, 2, 128, 16, BF16), (9, 1, 128, 32, BF16), (4, 4, 128, 16, BF16), (130, 1, 128, 16, BF16), (8, 2, 128, 8, BF16),
          (16, 4, 64, 16, BF16), (6, 2, 64, 8, BF16), (5, 1, 64, 32, BF16), (6, 2, 80, 16, BF16), (4, 2, 256, 8, BF16),
          (24, 2, 128, 16, F32), (6, 3, 48, 8, F32), (17, 1, 16, 24, F32), (4, 2, 192, 16, F32)]
STEPS = {
    "one token": [(0, [(0, 1)])],
    "one request": [(160, [(3, 1)])],
    "decoding": [(384, [(0, 1), (1, 1), (40, 1), (300, 1)])],
    "groups": [(0, [(5, 1), (700, 1)]), (128, [(64, 1)]), (1040, [(0, 1)] * 7 + [(129, 1)] * 5), (24, [(0, 1)])],
    "portions": [(256, [(0, 1), (7, 33), (130, 2)]), (0, [(0, 40)]), (512, [(100, 5), (0, 17)])],
    "shared keys that fill no page": [(133, [(0, 1), (9, 3), (50, 1)]), (5, [(1, 1), (90, 1)])],
}


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("name", STEPS)
def test_every_kind_of_step(shape, name):
    step = Step(STEPS[name], *shape, seed=len(name))
    close(step, step.run())


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[5], SHAPES[10]], ids=str)
@pytest.mark.parametrize("masks", [{"window": 1}, {"window": 100}, {"window": 300}, {"window": -64}, {"softcap": 5.0}, {"sink": True},
                                   {"window": 150, "softcap": 20.0, "sink": True}], ids=str)
def test_masks_caps_and_sinks(shape, masks):
    """Windows that leave a request none of its group's keys, some of them, and all; blocks."""
    step = Step([(256, [(0, 1), (60, 1), (290, 1), (33, 20)]), (0, [(90, 2)]), (40, [(0, 9)])], *shape, seed=3)
    masks = dict(masks, sink=torch.randn(shape[0]).to(DEV)) if "sink" in masks else masks
    close(step, step.run(**masks), **masks)


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[4], SHAPES[10]], ids=str)
@pytest.mark.parametrize("shared", [1, 31, 32, 33, 127, 128, 129, 255, 257])
def test_every_end_of_the_shared_keys(shape, shared):
    step = Step([(shared, [(0, 1), (1, 1), (127, 1)])], *shape, seed=shared)
    close(step, step.run())


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[6], SHAPES[11]], ids=str)
def test_more_groups_and_requests_than_a_warp(shape):
    groups = [(16 * (g % 5), [(g % 7, 1 + (g % 3 == 0))] * (1 + g % 4)) for g in range(70)]
    step = Step(groups, *shape, seed=9)
    close(step, step.run())


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[5], SHAPES[10]], ids=str)
def test_rows_behind_the_last_sequence_stay(shape):
    step = Step([(64, [(0, 1), (5, 1)])], *shape, spare=6)
    out = step.run()
    close(step, out)
    assert torch.isnan(out[2:]).all()


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[5], SHAPES[10]], ids=str)
def test_a_step_without_sequences_rows_and_with_empty_ones(shape):
    """Sequences that bring nothing, between others, at either end, and a whole group of them."""
    step = Step([(64, [(0, 0), (3, 1), (9, 0)]), (32, [(1, 0), (1, 0)]), (96, [(40, 1), (40, 0)])], *shape, seed=4)
    close(step, step.run())


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[5], SHAPES[10]], ids=str)
def test_scores_far_apart(shape):
    """Large scores: the maxima of the parts differ by hundreds, in either direction."""
    for flip in (False, True):
        step = Step([(300, [(50, 1), (200, 3)])], *shape, seed=6, spread=30.0)
        if flip:
            step = Step([(16, [(50, 1), (200, 3)])], *shape, seed=7, spread=30.0)
        close(step, step.run())


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[5], SHAPES[10]], ids=str)
def test_sizing_numbers_change_no_result_beyond_rounding(shape):
    step = Step(STEPS["groups"], *shape, seed=2)
    for more in ({"max_shared_len": 0}, {"max_shared_len": 100000, "max_own_len": 1}, {"max_own_len": 50000}):
        close(step, step.run(**more))


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[5], SHAPES[10]], ids=str)
def test_repeats_bit_by_bit(shape):
    step = Step(STEPS["portions"], *shape, seed=1)
    first = step.run().clone()
    for _ in range(5):
        assert torch.equal(step.run()[:step.cu[-1]], first[:step.cu[-1]])


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[5], SHAPES[10]], ids=str)
@pytest.mark.parametrize("chained", [False, True])
def test_captured_and_replayed_with_other_lengths_and_groups(shape, chained):
    """Two captured steps, replayed in turn on other lengths, groups and keys; each has parts of its own."""
    from matricxon_b200.ops import kernels

    other = [Step([(16, [(0, 1)]), (400, [(30, 1), (100, 1), (2, 1)])], *shape, seed=s) for s in (3, 4)]
    wide = [Step([(128, [(0, 1), (5, 1), (90, 1)]), (400, [(100, 1)])], *shape, seed=s, extra_pages=200) for s in (5, 6)]
    graphs, outs = [], []
    for step in wide:
        kernels.set_chained_launch(chained)
        step.run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step.run(max_shared_len=512, max_own_len=512))
        kernels.set_chained_launch(False)
        graphs.append(graph)
    for step, new in zip(wide, other):
        d, e = step.d, new.d
        for name in ("q", "cu", "context", "first", "lens", "tok_seq", "positions"):
            d[name].copy_(e[name])
        d["cache"][:e["cache"].shape[0]].copy_(e["cache"])
        d["tables"].fill_(-1)
        d["tables"][:, :e["tables"].shape[1]].copy_(e["tables"])
    for _ in range(3):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for step, new, out in zip(wide, other, outs):
        new.d["status"] = step.d["status"]
        close(new, out)


def test_on_another_stream():
    step = Step(STEPS["groups"], *SHAPES[0], seed=2)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        out = step.run()
    side.synchronize()
    close(step, out)


def test_strided_queries_and_results():
    """Queries in the rows of a fused product, results in columns of a wider buffer; a row start that is no multiple of 16
    bytes takes the kernels that need none."""
    for shape, offset in ((SHAPES[0], 64), (SHAPES[0], 3), (SHAPES[10], 5)):
        step = Step(STEPS["portions"], *shape, seed=5)
        width = step.heads * step.dim
        wide = torch.randn(step.n, width + 200, device=DEV).to(step.dtype)
        wide[:, offset:offset + width] = step.d["q"]
        step.d["q"] = wide[:, offset:offset + width]
        result = torch.full((step.n, width + 77), float("nan"), dtype=step.dtype, device=DEV)
        out = step.run(out=result[:, 11:11 + width])
        close(step, out)
        assert torch.isnan(result[:, :11]).all() and torch.isnan(result[:, 11 + width:]).all()


def test_pages_beyond_32_bits_of_elements():
    """A cache of 2.2 billion numbers whose last pages are read."""
    step = Step([(64, [(3, 1), (40, 1)])], 24, 2, 128, 16, BF16, seed=8)
    used = step.d["cache"]
    per_page = used[0].numel()
    pages = (1 << 31) // per_page + 20000 // 2
    big = torch.empty((pages, *used.shape[1:]), dtype=BF16, device=DEV)
    shift = pages - used.shape[0]
    big[shift:] = used
    step.d["cache"] = big
    step.d["tables"] = torch.where(step.d["tables"] >= 0, step.d["tables"] + shift, step.d["tables"])
    close(step, step.run())


def test_a_page_that_is_none_is_reported():
    for shape in (SHAPES[0], SHAPES[5], SHAPES[10]):
        for entry, value in ((0, -1), (0, 1 << 20), (5, -1)):
            step = Step([(64, [(30, 1), (30, 1)])], *shape, seed=3)
            entry = entry if entry == 0 else -(-94 // step.page) - 1
            step.d["tables"][0, entry] = value
            step.run()
            assert step.d["status"].item() == 4


def test_a_request_with_more_tokens_than_said_is_reported():
    step = Step([(64, [(30, 1), (30, 9)])], *SHAPES[0], seed=3)
    step.run(max_q_len=1)
    assert step.d["status"].item() == 16


def test_sequences_beyond_the_rows_are_cut_off_and_reported():
    """Sequences that together bring more tokens than there are rows: the rows that there are come out as ever, nothing is
    written behind them."""
    for shape in (SHAPES[0], SHAPES[5], SHAPES[10]):
        step = Step([(64, [(30, 3), (9, 4)])], *shape, seed=3)
        out = step.run().clone()
        step.d["status"].zero_()
        rows, step.n = step.n, 5
        scratch = torch.full((1 << 22,), 7.0, device=DEV)
        short = step.run(out=torch.full((rows, step.heads * step.dim), float("nan"), dtype=step.dtype, device=DEV), scratch=scratch)
        assert step.d["status"].item() == 16
        assert torch.isnan(short[5:]).all() and (short[:5].float() - out[:5].float()).abs().max() <= 4 * 2 ** -8 * 5.0
        used = (5 * step.heads * 32 * 2) * (step.dim + 2)            # at most 32 parts of either kind
        assert (scratch[used:] == 7).all()


def test_refusals():
    from matricxon_b200.ops import kernels
    from matricxon_b200.ops.library import KernelLibraryError

    step = Step(STEPS["decoding"], *SHAPES[0])
    good = dict(step.d)
    for name, value in (("tok_seq", good["tok_seq"].long()), ("tok_seq", good["tok_seq"][:1]), ("lens", good["lens"][:1]),
                        ("first", good["first"][:1]), ("cu", good["cu"][:2]), ("positions", good["positions"].cpu()),
                        ("cache", good["cache"].float()), ("cache", good["cache"][:, :1]), ("q", good["q"][:1]),
                        ("tables", good["tables"][:1])):
        step.d = dict(good, **{name: value})
        with pytest.raises(KernelLibraryError):
            step.run()
    step.d = good
    with pytest.raises(KernelLibraryError):
        step.run(scratch=torch.empty(16, device=DEV))
    with pytest.raises(KernelLibraryError):
        step.run(max_q_len=0)
    with pytest.raises(KernelLibraryError):
        step.run(out=torch.empty(step.n, 5, dtype=BF16, device=DEV))
    odd = Step(STEPS["decoding"], 4, 2, 24, 16, F32)                        # heads of 24 numbers
    with pytest.raises(KernelLibraryError):
        odd.run()
    assert kernels.describe_status(16) != "no error"


def out_of_sight(step, window):
    """The step's tables without what no query of a sequence sees any more, as the cache manager and step_tables leave them."""
    tables = [list(row) for row in step.tables]
    for row, context in zip(tables, step.context):
        low = max(0, context - window + 1) if window > 0 else context - context % -window
        row[:low // step.page] = [-1] * (low // step.page)
    step.d["tables"] = ints(tables)
    return step


WINDOWED = {
    "longest first": [(512, [(900, 1), (0, 1), (300, 1), (80, 1)])],
    "longest in the middle": [(512, [(100, 1), (900, 1), (20, 1)]), (0, [(40, 1)])],
    "portions": [(512, [(500, 20), (3, 1), (0, 33), (130, 2)])],
    "nobody sees the first pages": [(1056, [(310, 1), (120, 1), (200, 1)])],
    "shared keys that fill no page": [(517, [(40, 1), (0, 1), (90, 3)])],
    "first ones without tokens": [(512, [(900, 0), (0, 0), (600, 1), (10, 1)])],
    "more requests than a warp": [(256, [(700 - 13 * i, 1) for i in range(50)])],
}


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[1], SHAPES[4], SHAPES[5], SHAPES[7], SHAPES[8], SHAPES[10], SHAPES[12]], ids=str)
@pytest.mark.parametrize("window", [300, 77, -256])
@pytest.mark.parametrize("name", WINDOWED)
def test_pages_that_the_first_sequence_no_longer_holds(shape, window, name):
    """Tables of a window: the group's first sequence has given pages back that others of the group still see."""
    groups = WINDOWED[name]
    if shape[3] == 24:
        groups = [(shared // 24 * 24, members) for shared, members in groups]
    step = out_of_sight(Step(groups, *shape, seed=len(name)), window)
    close(step, step.run(window=window), window=window)


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[5], SHAPES[10]], ids=str)
def test_pages_between_that_nobody_sees(shape):
    """Shared lengths that differ within a group: under a window its sequences see stretches with a gap between them."""
    step = out_of_sight(Step([(96, [(404, 1), (4, 1), (20, 1)])], *shape, seed=2), 50)
    step.d["lens"] = ints([500, 96, 96])
    close(step, step.run(window=50, max_shared_len=500), window=50)


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[5], SHAPES[10]], ids=str)
def test_a_page_that_all_have_lost_is_reported(shape):
    step = out_of_sight(Step([(512, [(900, 1), (0, 1), (80, 1)])], *shape, seed=3), 300)
    step.d["tables"][1:, 300 // step.page] = -1
    step.run(window=300)
    assert step.d["status"].item() == 4


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[5], SHAPES[10]], ids=str)
def test_a_lost_page_that_the_shared_keys_fill_in_part_is_reported(shape):
    """Only the first sequence's page holds them; the others have a copy of their own, of which nobody says what is in it."""
    step = out_of_sight(Step([(517, [(900, 1), (0, 1)])], *shape, seed=3), 300)
    step.run(window=300)
    assert step.d["status"].item() == 4


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[5]], ids=str)
def test_lost_pages_beyond_what_a_block_keeps_of_its_table(shape):
    """More pages in one part than a block reads ahead."""
    step = out_of_sight(Step([(40000, [(30000, 1), (0, 1), (7, 1)])], *shape, seed=5), 39000)
    close(step, step.run(window=39000, max_shared_len=1), window=39000)


def forget_tails(step):
    """The slots of a sequence's first own page that lie before its own keys, NaN in all but the group's first sequence's."""
    cache = step.d["cache"]
    keys, values = cache[:, 0], cache[:, 1].view(cache.shape[0], step.kv_heads, step.dim, step.page)
    for s, shared in enumerate(step.lens):
        tail = shared % step.page
        if tail and s not in step.first and shared // step.page < len(step.tables[s]) and step.tables[s][shared // step.page] >= 0:
            page = step.tables[s][shared // step.page]
            keys[page, :, :tail] = float("nan")
            values[page, :, :, :tail] = float("nan")
    return step


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("masks", [{}, {"window": 40}, {"softcap": 5.0}], ids=str)
@pytest.mark.parametrize("groups", [[(133, [(0, 1), (9, 1), (50, 1), (0, 1)])], [(133, [(0, 1), (9, 3), (50, 21), (0, 70)]), (5, [(1, 1), (90, 1)])],
                                    [(257, [(0, 2)] * 9), (1, [(300, 1)] * 3)]], ids=["narrow", "portions", "one key over"])
def test_slots_before_a_sequences_own_keys_hold_anything(shape, masks, groups):
    step = forget_tails(Step(groups, *shape, seed=11))
    close(step, step.run(**masks), **masks)


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[5], SHAPES[10]], ids=str)
@pytest.mark.parametrize("first,lost", [([0, 2], (2, 3)), ([1, 4], (0,)), ([0, 1, 3], (3,)), ([0, 3, 1, 4], (0, 1, 2, 3)), ([2, 2], (0, 1, 2, 3)),
                                        ([0, 2, 9], ()), ([-3, 2, 4], ())], ids=str)
def test_sequences_of_no_group_are_reported_and_left_alone(shape, first, lost):
    """Lists of groups that leave sequences out, or whose starts fall: rows of such sequences stay, the status word is set,
    whatever the scratch memory holds. Starts outside the sequences are taken for their ends, as ever."""
    step = Step([(64, [(30, 1), (9, 2), (0, 1), (5, 1)])], *shape, seed=3)
    whole = step.run().clone()
    assert step.d["status"].item() == 0
    step.d["first"] = ints(first)
    out = step.run(scratch=torch.full((1 << 22,), 1e6, device=DEV))
    assert step.d["status"].item() == (16 if lost else 0)
    seq = step.d["tok_seq"].tolist()
    ref, bound = step.plain()
    for row, s in enumerate(seq):
        if s in lost:
            assert torch.isnan(out[row]).all()
        else:
            assert ((out[row].double().cpu() - ref[row]).abs() <= bound[row]).all()
    assert not torch.isnan(whole).any()


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[5], SHAPES[10]], ids=str)
def test_sequences_without_tokens_may_be_of_no_group(shape):
    """The padding of a batch of a fixed size, behind the groups or before them."""
    step = Step([(64, [(30, 1), (9, 1), (0, 0), (5, 0)])], *shape, seed=3)
    step.d["first"] = ints([0, 2])
    close(step, step.run())
    step = Step([(64, [(30, 0), (9, 1), (0, 1)])], *shape, seed=3)
    step.d["first"] = ints([1, 3])
    step.d["tables"][1, :4] = step.d["tables"][0, :4]
    close(step, step.run())


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[5], SHAPES[10]], ids=str)
def test_rows_with_another_sequences_number_are_reported_and_left_alone(shape):
    step = Step([(64, [(30, 1), (9, 1), (0, 1)])], *shape, seed=3)
    step.d["tok_seq"] = ints([0, -1, 0])
    out = step.run(scratch=torch.full((1 << 22,), 1e6, device=DEV))
    assert step.d["status"].item() == 16
    ref, bound = step.plain()
    assert ((out[0].double().cpu() - ref[0]).abs() <= bound[0]).all() and torch.isnan(out[1:]).all()


def test_tokens_beyond_what_was_said_are_left_alone():
    """Two of a sequence's nine tokens fit the sixteen rows of its tile."""
    step = Step([(64, [(30, 1), (30, 9)])], 16, 2, 128, 16, BF16, seed=3)
    out = step.run(max_q_len=2, scratch=torch.full((1 << 22,), 1e6, device=DEV))
    assert step.d["status"].item() == 16
    ref, bound = step.plain()
    assert ((out[:3].double().cpu() - ref[:3]).abs() <= bound[:3]).all() and torch.isnan(out[3:]).all()


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_results_do_not_hang_on_the_scratch_memory(shape):
    for name in ("groups", "portions"):
        step = Step(STEPS[name], *shape, seed=4)
        outs = [step.run(scratch=torch.full((1 << 23,), value, device=DEV)) for value in (0.0, 1e30, float("nan"))]
        close(step, outs[0])
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_rows_that_lie_in_one_another_or_too_far_apart_are_refused():
    from matricxon_b200.ops.library import KernelLibraryError

    step = Step(STEPS["decoding"], *SHAPES[0])
    width = step.heads * step.dim
    with pytest.raises(KernelLibraryError):
        step.run(out=torch.zeros(1, width, dtype=BF16, device=DEV).expand(step.n, width))
    with pytest.raises(KernelLibraryError):
        step.run(out=torch.zeros(step.n * width, dtype=BF16, device=DEV).as_strided((step.n, width), (width - 16, 1)))
    one = Step(STEPS["one token"], *SHAPES[0])
    one.d["q"] = one.d["q"].as_strided((1, width), (1 << 31, 1))       # strides are 32-bit numbers further down
    with pytest.raises(KernelLibraryError):
        one.run()
    one = Step(STEPS["one token"], *SHAPES[0])
    with pytest.raises(KernelLibraryError):
        one.run(out=torch.zeros(width, dtype=BF16, device=DEV).as_strided((1, width), (1 << 31, 1)))
    close(one, one.run(out=torch.zeros(width, dtype=BF16, device=DEV).as_strided((1, width), (1, 1))))     # one row lies in no other


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[5], SHAPES[10]], ids=str)
@pytest.mark.parametrize("first,lost", [([0, 2, 4, 0, 0], ()), ([0, 2, 4, 4, 4, 4], ()), ([0] * 40 + [2] + [4] * 40, ()), ([0, 0, 2, 4, 1, 0], ()),
                                        ([0, 3, 2, 4], (0, 1, 2, 3)), ([0, 1, 0, 1, 4], (0, 1, 2, 3))], ids=str)
def test_lists_of_groups_that_are_filled_up(shape, first, lost):
    """Places without a group behind, between and before the groups; groups that overlap."""
    step = Step([(64, [(30, 1), (9, 2), (0, 1), (5, 1)])], *shape, seed=3)
    step.d["first"] = ints(first)
    if lost:
        out = step.run(scratch=torch.full((1 << 23,), 1e6, device=DEV))
        assert step.d["status"].item() == 16 and torch.isnan(out).all()
    else:
        close(step, step.run(scratch=torch.full((1 << 23,), 1e6, device=DEV)))


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[5], SHAPES[10]], ids=str)
def test_overlapping_groups_beside_sequences_of_none(shape):
    """As many tokens in groups as there are, but one sequence in two of them and one in none."""
    step = Step([(64, [(30, 1), (9, 1), (0, 1), (5, 1)])], *shape, seed=3)
    step.d["first"] = ints([0, 2, 1, 3])
    out = step.run(scratch=torch.full((1 << 23,), 1e6, device=DEV))
    assert step.d["status"].item() == 16 and torch.isnan(out[[1, 3]]).all()
    ref, bound = step.plain()
    assert ((out[[0, 2]].double().cpu() - ref[[0, 2]]).abs() <= bound[[0, 2]]).all()
