"""Penalties, biases and masks on rows of scores, against a plain implementation in float64."""

import math
import random

import pytest

torch = pytest.importorskip("torch")

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]

DEV = "cuda:0"


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def floats(values):
    return torch.tensor(values, dtype=torch.float32, device=DEV)


def words_of(allowed, vocab):
    """Mask words of a set of tokens."""
    words = [0] * ((vocab + 31) // 32)
    for v in allowed:
        words[v // 32] |= 1 << (v % 32)
    return [w - (1 << 32) if w >= 1 << 31 else w for w in words]


class Case:
    def __init__(self, rows, vocab, tokens=50, biases=5, masked=0.5, dtype=torch.float32, seed=0, pending=True):
        rng = random.Random(seed)
        self.rows, self.vocab, self.dtype = rows, vocab, dtype
        self.logits = (4 * torch.randn(rows, vocab, generator=torch.Generator().manual_seed(seed))).to(dtype)
        self.tokens = [[min(vocab - 1, int(vocab * rng.random() ** 3)) for _ in range(rng.randrange(tokens + 1))] for _ in range(rows)]
        self.pending = [rng.randrange(-1, vocab) if pending else -1 for _ in range(rows)]
        self.biases = [[(rng.randrange(vocab), rng.gauss(0, 5)) for _ in range(rng.randrange(biases + 1))] for _ in range(rows)]
        self.repeat = [rng.uniform(0.8, 1.5) for _ in range(rows)]
        self.presence = [rng.uniform(-0.5, 1.0) for _ in range(rows)]
        self.frequency = [rng.uniform(-0.2, 0.3) for _ in range(rows)]
        self.masks = [None if rng.random() >= masked else {v for v in range(vocab) if rng.random() < 0.3} for _ in range(rows)]

    def device(self):
        offsets, ids = [0], []
        for row in self.tokens:
            ids += row
            offsets.append(len(ids))
        b_offsets, b_ids, b_values = [0], [], []
        for row in self.biases:
            b_ids += [v for v, _ in row]
            b_values += [x for _, x in row]
            b_offsets.append(len(b_ids))
        masks = [m for m in self.masks if m is not None]
        rows, at = [], 0
        for m in self.masks:
            rows.append(-1 if m is None else at)
            at += m is not None
        return {"token_offsets": ints(offsets), "token_ids": ints(ids), "repeat_penalty": floats(self.repeat),
                "presence_penalty": floats(self.presence), "frequency_penalty": floats(self.frequency), "bias_offsets": ints(b_offsets),
                "bias_ids": ints(b_ids), "bias_values": floats(b_values),
                "mask_words": ints([words_of(m, self.vocab) for m in masks] or [[0] * ((self.vocab + 31) // 32)]), "mask_rows": ints(rows),
                "pending_ids": ints(self.pending)}

    def plain(self):
        """(result, how far off a float result may be): every operation of the formula rounds once, by half a step of its
        result: the quotient or product, the penalty's product and sum, and two sums."""
        out = self.logits.double().clone()
        size = out.abs()
        as_float = lambda x: float(torch.tensor(x, dtype=torch.float32))  # noqa: E731
        for r in range(self.rows):
            counts = {}
            for v in self.tokens[r] + ([self.pending[r]] if self.pending[r] >= 0 else []):
                counts[v] = counts.get(v, 0) + 1
            repeat, presence, frequency = as_float(self.repeat[r]), as_float(self.presence[r]), as_float(self.frequency[r])
            for v, c in counts.items():
                if not 0 <= v < self.vocab:
                    continue
                x = float(out[r, v])
                x = x / repeat if x > 0 else x * repeat
                out[r, v] = x - frequency * c - presence
                size[r, v] = abs(x) * 2 + 3 * (abs(frequency) * c + abs(presence))
            for v, x in dict(self.biases[r]).items():
                out[r, v] += as_float(x)
                size[r, v] += abs(as_float(x)) * 2
            if self.masks[r] is not None:
                banned = torch.ones(self.vocab, dtype=torch.bool)
                banned[list(self.masks[r])] = False
                out[r][banned] = -math.inf
        return out, size * torch.finfo(torch.float32).eps / 2 * 4

    def check(self, got):
        ref, bound = self.plain()
        got = got.double().cpu()
        finite = torch.isfinite(ref)
        assert torch.equal(finite, torch.isfinite(got)) and torch.equal(ref[~finite], got[~finite])
        assert ((got - ref).abs() <= bound)[finite].all()
        untouched = finite & (ref == self.logits.double())
        assert torch.equal(got[untouched], ref[untouched])


def adjust(logits, out, **args):
    from matricxon_b200.ops import kernels

    kernels.adjust_logits(logits, out, **args)
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 31), (3, 32), (5, 33), (7, 1000), (2, 4095), (3, 4096), (2, 4097), (4, 20001),
                                        (300, 129), (40, 9000)])
def test_all_of_it(rows, vocab, dtype):
    case = Case(rows, vocab, dtype=dtype, seed=rows + vocab)
    case.check(adjust(case.logits.to(DEV), torch.full((rows, vocab), float("nan"), device=DEV), **case.device()))


@pytest.mark.parametrize("tokens", [0, 1, 300, 5000])
@pytest.mark.parametrize("biases", [0, 1, 700])
def test_lists_of_all_lengths(tokens, biases):
    """Long histories in a small vocabulary (counts of hundreds), biases that name a token several times."""
    case = Case(6, 500, tokens=tokens, biases=biases, seed=tokens + biases)
    case.check(adjust(case.logits.to(DEV), torch.empty(6, 500, device=DEV), **case.device()))


def test_counts_beyond_16_bits():
    case = Case(2, 40, tokens=0, biases=0, masked=0, pending=False)
    case.tokens = [[7] * 70000 + [3], [0]]
    case.check(adjust(case.logits.to(DEV), torch.empty(2, 40, device=DEV), **case.device()))


def test_each_part_alone():
    """What is left out changes nothing."""
    for kept in (("token_offsets", "token_ids", "repeat_penalty"), ("token_offsets", "token_ids", "presence_penalty"),
                 ("token_offsets", "token_ids", "frequency_penalty"), ("bias_offsets", "bias_ids", "bias_values"),
                 ("mask_words", "mask_rows"), ("pending_ids", "presence_penalty"), ()):
        case = Case(5, 777, seed=len(kept))
        args = {name: value for name, value in case.device().items() if name in kept}
        if "token_ids" not in kept:
            case.tokens = [[]] * 5
        if "pending_ids" not in kept:
            case.pending = [-1] * 5
        if "bias_ids" not in kept:
            case.biases = [[]] * 5
        if "mask_words" not in kept:
            case.masks = [None] * 5
        for name in ("repeat", "presence", "frequency"):
            if f"{name}_penalty" not in kept:
                setattr(case, name, [1.0 if name == "repeat" else 0.0] * 5)
        case.check(adjust(case.logits.to(DEV), torch.empty(5, 777, device=DEV), **args))


def test_a_mask_a_row_without_mask_rows_and_one_mask_for_many():
    case = Case(4, 100, masked=1.0, seed=2)
    args = case.device()
    del args["mask_rows"]
    case.check(adjust(case.logits.to(DEV), torch.empty(4, 100, device=DEV), **args))
    args = case.device()
    case.masks = [case.masks[2], None, case.masks[2], case.masks[0]]
    args["mask_rows"] = ints([2, -1, 2, 0])
    case.check(adjust(case.logits.to(DEV), torch.empty(4, 100, device=DEV), **args))


def test_masks_that_allow_nothing_and_everything():
    case = Case(3, 5000, masked=1.0, seed=2)
    case.masks = [set(), set(range(5000)), {4999}]
    got = adjust(case.logits.to(DEV), torch.empty(3, 5000, device=DEV), **case.device())
    case.check(got)
    assert torch.isinf(got[0]).all()


def test_infinities_and_nan_stand_where_they_stood_unless_masked():
    case = Case(2, 300, tokens=0, biases=0, masked=0, pending=False)
    case.logits[:, 5], case.logits[:, 6], case.logits[:, 7] = math.inf, -math.inf, math.nan
    case.logits[:, 8], case.logits[:, 9] = math.nan, torch.finfo(torch.float32).min
    case.masks = [None, set(range(300)) - {5, 8}]
    case.tokens = [[5, 6, 9], [6]]
    case.repeat = [1.25, 2.0]
    got = adjust(case.logits.to(DEV), torch.empty(2, 300, device=DEV), **case.device()).cpu()
    assert got[0, 5] == math.inf and got[0, 6] == -math.inf and torch.isnan(got[0, 7]) and torch.isnan(got[0, 8])
    assert got[1, 5] == -math.inf and got[1, 8] == -math.inf and torch.isnan(got[1, 7]) and got[1, 6] == -math.inf
    assert got[0, 9] == -math.inf          # the lowest value times 1.25


def test_ids_outside_the_vocabulary_are_passed_over():
    case = Case(2, 100, seed=1)
    case.tokens[0] += [-1, 100, 2 ** 31 - 1, -2 ** 31]
    case.pending = [-7, 100]
    args = case.device()
    args["bias_ids"] = args["bias_ids"].clone()
    case.check(adjust(case.logits.to(DEV), torch.empty(2, 100, device=DEV), **args))


def test_in_place_and_strided():
    case = Case(4, 1001, seed=4)
    buffer = torch.full((4, 1300), 7.0, device=DEV)
    buffer[:, 3:1004] = case.logits.to(DEV)
    view = buffer[:, 3:1004]
    case.check(adjust(view, view, **case.device()))
    assert (buffer[:, :3] == 7).all() and (buffer[:, 1004:] == 7).all()
    wide = torch.full((4, 2500), 7.0, device=DEV)
    wide[:, :1001] = case.logits.to(DEV)
    case.check(adjust(wide[:, :1001], wide[:, 1200:2201], **case.device()))
    assert torch.equal(wide[:, :1001].cpu(), case.logits)


def test_repeats_bit_by_bit_and_on_another_stream():
    case = Case(8, 3001, tokens=2000, biases=900, seed=4)
    args, logits = case.device(), case.logits.to(DEV)
    first = adjust(logits, torch.empty(8, 3001, device=DEV), **args).clone()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        second = adjust(logits, torch.empty(8, 3001, device=DEV), **args)
    side.synchronize()
    assert torch.equal(first, second)


def test_captured_with_other_lists():
    case = Case(3, 700, tokens=40, seed=4)
    args, logits, out = case.device(), case.logits.to(DEV), torch.empty(3, 700, device=DEV)
    args["token_ids"] = torch.zeros(500, dtype=torch.int32, device=DEV)
    adjust(logits, out, **args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        adjust(logits, out, **args)
    case.tokens = [[1, 2, 2], [], [699] * 50]
    args["token_offsets"].copy_(ints([0, 3, 3, 53]))
    args["token_ids"][:53] = ints([1, 2, 2] + [699] * 50)
    graph.replay()
    case.check(out)


def test_more_elements_than_32_bits_of_bytes():
    """Rows beyond 2^31 bytes of the scores."""
    rows, vocab = 5, 140_000_000
    logits = torch.zeros(rows, vocab, device=DEV)
    out = torch.empty_like(logits)
    adjust(logits, out, pending_ids=ints([vocab - 1] * rows), presence_penalty=floats([1, 2, 3, 4, 5]))
    assert out[:, -1].tolist() == [-1, -2, -3, -4, -5] and not out[:, :-1].any()


def test_refusals():
    from matricxon_b200.ops.library import KernelLibraryError

    case = Case(3, 100)
    good, logits, out = case.device(), case.logits.to(DEV), torch.empty(3, 100, device=DEV)
    for name, value in (("token_offsets", good["token_offsets"][:2]), ("token_ids", good["token_ids"].long()), ("token_ids", None),
                        ("bias_values", None), ("bias_ids", good["bias_ids"][:1]), ("mask_words", good["mask_words"][:, :3].contiguous()),
                        ("mask_words", None), ("mask_rows", good["mask_rows"][:1]), ("repeat_penalty", good["repeat_penalty"].double()),
                        ("presence_penalty", good["presence_penalty"][:1]), ("pending_ids", good["pending_ids"].cpu())):
        with pytest.raises(KernelLibraryError):
            adjust(logits, out, **dict(good, **{name: value}))
    for bad_logits, bad_out in ((logits.half(), out), (logits, out[:2]), (logits, out.bfloat16()), (logits.t(), out.t()), (logits.cpu(), out)):
        with pytest.raises(KernelLibraryError):
            adjust(bad_logits, bad_out, **good)
    buffer = torch.zeros(400, device=DEV)
    with pytest.raises(KernelLibraryError):                 # a few columns along in the same memory
        adjust(buffer[:300].view(3, 100), buffer[4:304].view(3, 100))
    with pytest.raises(KernelLibraryError):                 # rows that lie in one another
        adjust(logits, out[:1].expand(3, 100))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,tokens", [(3, 20001, 8000), (5, 9000, 3000), (37, 70001, 4500), (37, 70001, 60), (2, 40000, 30000)])
def test_lists_over_several_stretches(rows, vocab, tokens, dtype):
    """Ids dealt out to ten stretches of a turn and to nine of four turns, and lists short enough not to be."""
    case = Case(rows, vocab, tokens=tokens, biases=40, dtype=dtype, seed=rows)
    case.check(adjust(case.logits.to(DEV), torch.empty(rows, vocab, device=DEV), **case.device()))


@pytest.mark.parametrize("rows,vocab,tokens", [(4, 700, 60), (4, 20001, 8000)])
@pytest.mark.parametrize("which", ["token", "bias"])
@pytest.mark.parametrize("bad", [(-5, 10, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1), (0, 70, 30, 90, 100), (2 ** 31 - 1, 0, -2 ** 31, 50, 20),
                                 (90, 60, 40, 20, 0), (0, 10 ** 6, 10 ** 6 + 1, 10 ** 6 + 2, 10 ** 6 + 3), (100, 100, 100, 100, 10 ** 6)], ids=str)
def test_offsets_outside_their_list(rows, vocab, tokens, which, bad):
    """A row takes what lies inside the list, whether ids are dealt out first or not; parts may overlap."""
    case = Case(rows, vocab, tokens=tokens, biases=90, seed=3)
    args = case.device()
    lists = {"token": [v for row in case.tokens for v in row], "bias": [pair for row in case.biases for pair in row]}
    size = len(lists[which])
    scale = max(1, size // 100)
    bad = [o if abs(o) > 1000 else o * scale for o in bad]
    inside = [min(max(o, 0), size) for o in bad]
    parts = [lists[which][a:b] for a, b in zip(inside, inside[1:])]
    if which == "token":
        case.tokens = parts
    else:
        case.biases = parts
    args[f"{which}_offsets"].copy_(ints(bad))
    out = torch.empty(rows, vocab, device=DEV)
    for _ in range(3):
        case.check(adjust(case.logits.to(DEV), out.fill_(float("nan")), **args))


def test_captured_with_offsets_that_fall_and_rise_again():
    case = Case(4, 20001, tokens=8000, seed=6)
    args, logits, out = case.device(), case.logits.to(DEV), torch.empty(4, 20001, device=DEV)
    adjust(logits, out, **args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        adjust(logits, out, **args)
    ids = [v for row in case.tokens for v in row]
    for offsets in ([0, 9000, 3000, 12000, 10], [0, 50, 8000, 8000, len(ids)], [5, 4, 3, 2, 1 << 30]):
        args["token_offsets"].copy_(ints(offsets))
        graph.replay()
        case.tokens = [ids[a:b] for a, b in zip(offsets, offsets[1:])]
        case.check(out)
