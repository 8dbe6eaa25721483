"""The operators of a serving step as they are used: through the engine's sampling options, and one after another."""

import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]

DEV = "cuda:0"


def plain_scores(row, config, generated):
    """The adjusted scores of one row, float64."""
    out = row.double().cpu().clone()
    counts = {}
    for token in generated:
        counts[token] = counts.get(token, 0) + 1
    as_float = lambda x: float(torch.tensor(x, dtype=torch.float32))  # noqa: E731
    for token, c in counts.items():
        x = float(out[token])
        x = x / as_float(config.repeat_penalty) if x > 0 else x * as_float(config.repeat_penalty)
        out[token] = x - as_float(config.frequency_penalty) * c - as_float(config.presence_penalty)
    for token, value in config.logit_bias:
        out[token] += as_float(value)
    if config.allowed_token_ids is not None:
        banned = torch.ones(out.shape[0], dtype=torch.bool)
        banned[list(config.allowed_token_ids)] = False
        out[banned] = -math.inf
    return out


def test_sampler_rows_with_and_without_adjustments():
    """A batch of both: greedy rows take the best adjusted score, drawn rows an allowed token, rows without options what they
    take in a batch of their own."""
    from matricxon_b200.sampling.config import SamplingConfig
    from matricxon_b200.sampling.sampler import BatchSampler, RequestSampler

    vocab = 1003
    logits = (3 * torch.randn(6, vocab, generator=torch.Generator().manual_seed(1))).to(DEV)
    before = logits.clone()
    configs = [SamplingConfig(temperature=0.0, repeat_penalty=1.3, presence_penalty=1.0, frequency_penalty=0.5),
               SamplingConfig(temperature=0.0, repeat_penalty=1.0, logit_bias={5: 40.0, 6: -40.0}),
               SamplingConfig(temperature=0.0, repeat_penalty=1.5),
               SamplingConfig(temperature=1.0, top_k=0, top_p=1.0, repeat_penalty=1.0, allowed_token_ids=(3, 500, 1002), seed=5),
               SamplingConfig(temperature=0.9, top_k=20, top_p=0.9, repeat_penalty=1.2, seed=6),
               SamplingConfig(temperature=0.7, top_k=2, top_p=0.5, repeat_penalty=1.2, allowed_token_ids=(77,), seed=7)]
    samplers = [RequestSampler(config) for config in configs]
    top = [int(v) for v in logits[0].topk(3).indices]
    for sampler in samplers:
        for token in top + [top[0]] * 4 + [9]:
            sampler.accept(token)
    batch = BatchSampler(DEV, vocab)
    chosen = batch.sample(logits, samplers)
    assert torch.equal(logits, before)                     # the model's scores stay as they are
    for r in (0, 1):
        scores = plain_scores(logits[r], configs[r], samplers[r].generated)
        assert float(scores[chosen[r]]) >= float(scores.max()) - 1e-5
    assert chosen[1] == 5 and chosen[3] in (3, 500, 1002) and chosen[5] == 77
    for r in (2, 4):
        assert batch.sample(logits[r:r + 1], [samplers[r]]) == [chosen[r]]
    # a token that the host has not seen yet counts like the others
    pending = torch.tensor([top[1]] * 6, dtype=torch.int32, device=DEV)
    ahead = batch.read(batch.launch(logits, samplers, pending=pending))
    scores = plain_scores(logits[0], configs[0], samplers[0].generated + [top[1]])
    assert float(scores[ahead[0]]) >= float(scores.max()) - 1e-5


@pytest.mark.parametrize("look_ahead", [True, False])
def test_engine_with_adjusted_requests(look_ahead):
    """Requests with and without options generated together: those without give what they give alone; masks hold for every
    token; steps queued ahead, whose newest token is still on the device, choose the same tokens."""
    from test_gpu_generation import random_ids, tiny_config, tiny_tensors

    from matricxon_b200 import ChatEngine, GenerationRequest, SamplingConfig
    from matricxon_b200.engine.core import model_from_tensors
    from matricxon_b200.engine.scheduler import RequestRefused

    model = model_from_tensors(tiny_config("A"), tiny_tensors("A", torch.float32), dtype="float32", device=DEV)
    vocab = model.spec.vocab_size
    allowed = tuple(range(0, vocab, 7))
    configs = [SamplingConfig(temperature=0.0, repeat_penalty=1.0, num_predict=24, num_ctx=128),
               SamplingConfig(temperature=0.0, repeat_penalty=1.0, frequency_penalty=5.0, num_predict=24, num_ctx=128),
               SamplingConfig(temperature=0.8, top_k=0, top_p=1.0, repeat_penalty=1.1, allowed_token_ids=allowed, seed=3, num_predict=24, num_ctx=128),
               SamplingConfig(temperature=0.0, repeat_penalty=1.0, logit_bias={11: 1e4}, num_predict=5, num_ctx=128)]
    prompts = [random_ids(9 + 3 * i, vocab, seed=i) for i in range(4)]
    engine = ChatEngine(model, max_cache_tokens=2048, max_active=4, prefill_chunk=32, max_model_len=128, look_ahead=look_ahead)
    results = engine.generate_batch([GenerationRequest(p, c) for p, c in zip(prompts, configs)])
    assert engine.generate(GenerationRequest(prompts[0], configs[0])).token_ids == results[0].token_ids
    counts = [results[1].token_ids.count(token) for token in set(results[1].token_ids)]
    plain = engine.generate(GenerationRequest(prompts[1], configs[0])).token_ids
    assert max(counts) <= max(plain.count(token) for token in set(plain))
    assert all(token in allowed for token in results[2].token_ids) and len(results[2].token_ids) == 24
    assert results[3].token_ids == [11] * 5
    step_by_step = ChatEngine(model, max_cache_tokens=2048, max_active=4, prefill_chunk=32, max_model_len=128, look_ahead=False)
    again = step_by_step.generate_batch([GenerationRequest(p, c) for p, c in zip(prompts, configs)])
    assert [r.token_ids for r in again] == [r.token_ids for r in results]
    with pytest.raises(RequestRefused):
        engine.add_request(prompts[0], SamplingConfig(allowed_token_ids=(vocab,)))


@pytest.mark.parametrize("chained", [False, True])
def test_a_decoding_loop_of_all_three(chained):
    """Eight requests on one prefix, six steps: tables on the GPU, keys and values into the slots they name, attention over the
    shared and own keys, adjusted scores, a draw. Against the same requests without sharing, on tables laid out on the host;
    as one captured step that is replayed, its lengths moved on by the device alone."""
    from matricxon_b200.cache.manager import CacheManager, GroupRule
    from matricxon_b200.ops import kernels
    from matricxon_b200.sampling.config import SamplingConfig
    from matricxon_b200.sampling.sampler import BatchSampler, RequestSampler

    heads, kv_heads, dim, page, n, vocab, steps = 8, 2, 128, 16, 8, 515, 6
    prefix, width, n_pages = 48, 16, 200
    gen = torch.Generator(device=DEV).manual_seed(4)
    ints = lambda values: torch.tensor(values, dtype=torch.int32, device=DEV)  # noqa: E731
    cache = torch.randn(n_pages, 2, kv_heads, page, dim, generator=gen, device=DEV).bfloat16()
    plain_cache = cache.clone()
    head = (0.3 * torch.randn(vocab, heads * dim, generator=gen, device=DEV)).bfloat16()
    rows = torch.randn(steps, n, (heads + 2 * kv_heads) * dim, generator=gen, device=DEV).bfloat16()
    inv_freq = 1.0 / (10000.0 ** (torch.arange(0, dim, 2, device=DEV).float() / dim))
    own = [0, 1, 15, 14, 17, 29, 2, 9]                               # keys of each request behind the prefix
    context = [prefix + k for k in own]

    # the host's tables: every request holds pages of its own; what they hold of the prefix is the leader's content
    manager = CacheManager([GroupRule(None)], n_pages, page, n)
    for s in range(n):
        manager.add_request(str(s))
        manager.reserve(str(s), context[s])
        manager.commit(str(s), context[s])
    host_tables = [manager.table_row(str(s), 0, width).tolist() for s in range(n)]
    for s in range(1, n):
        for k in range(prefix // page):
            plain_cache[host_tables[s][k]] = plain_cache[host_tables[0][k]]
    cache.copy_(plain_cache)
    # on the device the others read the prefix through the leader's row
    tables = ints(host_tables)
    tables[1:, :prefix // page] = -1
    first_free = n_pages - manager.pools[0].free_count
    free = ints(list(range(first_free, n_pages)))
    shared_rows, shared_pages = ints([-1] + [0] * (n - 1)), ints([0] + [prefix // page] * (n - 1))
    lengths, q_lens, n_free = ints(context), ints([1] * n), ints([n_pages - first_free])
    status = ints([0])
    out = {name: torch.empty(size, dtype=torch.int32, device=DEV) for name, size in
           (("positions", n), ("tok_seq", n), ("cu_q", n + 1), ("slots", n), ("taken", 1))}
    block_tables = torch.empty(n, width, dtype=torch.int32, device=DEV)
    row_in = torch.empty_like(rows[0])
    attended = torch.empty(n, heads * dim, dtype=torch.bfloat16, device=DEV)
    configs = [SamplingConfig(temperature=0.0, repeat_penalty=1.3, presence_penalty=0.5, allowed_token_ids=range(s % 3, vocab, 3)) for s in range(n)]

    def step():
        kernels.step_tables(q_lens, lengths, None, tables, free, n_free, page, n_pages, out["positions"], out["tok_seq"], out["cu_q"],
                            out["slots"], block_tables, out["taken"], status, shared_rows=shared_rows, shared_pages=shared_pages)
        qkv = row_in.clone()
        kernels.rope_kv_write(qkv, out["positions"], inv_freq, out["slots"], cache, heads, kv_heads, dim, dim, page, status)
        kernels.paged_attention_shared(qkv, qkv.stride(0), cache, block_tables, out["cu_q"], lengths, out["tok_seq"],
                                       out["positions"], ints_first, shared_lens, n, heads, kv_heads, dim, None, dim ** -0.5, attended,
                                       status, max_q_len=1, max_shared_len=prefix, max_own_len=64)
        scores = attended.float() @ head.float().t()
        lengths.add_(1)                                              # the next step's lengths and free pages
        free.copy_(torch.roll(free, -1, 0).where(out["taken"] == 1, free))
        return scores

    ints_first, shared_lens = ints([0, n]), ints([prefix] * n)
    row_in.copy_(rows[0])
    keep = [t.clone() for t in (tables, free, lengths, cache)]
    step()                                                            # once, for what is built at the first call
    for tensor, value in zip((tables, free, lengths, cache), keep):
        tensor.copy_(value)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    kernels.set_chained_launch(chained)
    try:
        with torch.cuda.graph(graph):
            scores = step()
    finally:
        kernels.set_chained_launch(False)
    samplers, plain_samplers = ([RequestSampler(c) for c in configs] for _ in range(2))
    batch = BatchSampler(DEV, vocab)
    for i in range(steps):
        # a step takes at most one page here, so that rolling the list by one is what giving them out does
        need = [s for s in range(n) if (context[s] + i) % page == 0]
        if len(need) > 1:
            pytest.fail("the lengths above let two requests need a page at once")
        row_in.copy_(rows[i])
        graph.replay()
        got = batch.sample(scores, samplers)
        # the same step with the host's tables and nothing shared
        for s in range(n):
            manager.reserve(str(s), 1)
        slots = ints([int(manager.slot_ids(str(s), 0, context[s] + i, 1)[0]) for s in range(n)])
        assert torch.equal(out["slots"], slots) and out["positions"].tolist() == [c + i for c in context]
        full = ints([manager.table_row(str(s), 0, width).tolist() for s in range(n)])
        qkv = rows[i].clone()
        kernels.rope_kv_write(qkv, out["positions"], inv_freq, slots, plain_cache, heads, kv_heads, dim, dim, page, status)
        alone = torch.empty_like(attended)
        kernels.paged_attention(qkv, qkv.stride(0), plain_cache, full, ints(list(range(n))), out["positions"], n, heads, kv_heads, dim,
                                None, dim ** -0.5, alone, status)
        for s in range(n):
            manager.commit(str(s), 1)
        # both round weights and results to bfloat16 on their own ways: two half steps each of what a softmax of these values gives
        assert (attended.float() - alone.float()).abs().max() <= 4 * 2 ** -8 * 5.0
        for s in range(n):
            expected = plain_scores(scores[s], configs[s], samplers[s].generated)
            assert float(expected[got[s]]) >= float(expected.max()) - 1e-4 and got[s] % 3 == s % 3
            samplers[s].accept(got[s])
    assert status.item() == 0


def test_two_streams_at_once():
    """Calls of all three queued on two streams, many times over: each gives, bit by bit, what it gives alone."""
    from test_gpu_adjust_logits import Case as Scores
    from test_gpu_adjust_logits import adjust
    from test_gpu_attention_shared import SHAPES, STEPS, Step
    from test_gpu_step_tables import random_case

    attention = [Step(STEPS["groups"], *SHAPES[0], seed=1), Step(STEPS["portions"], *SHAPES[5], seed=2),
                 Step([(2048, [(k * 37 % 300, 1) for k in range(20)])], *SHAPES[0], seed=3), Step(STEPS["groups"], *SHAPES[10], seed=4)]
    scores = [Scores(30, 9001, tokens=400, seed=s) for s in (1, 2)]
    arguments = [(case.logits.to(DEV), case.device()) for case in scores]
    tables = [random_case(60, 16, s).device() for s in (3, 4)]
    expected_tables = [case.expected() for case in tables]
    alone = [step.run().clone() for step in attention]
    alone_scores = [adjust(logits, torch.empty_like(logits), **args) for logits, args in arguments]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(25):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got += [(k, attention[k].run()) for k in (i, 2 + i)]
                got.append((4 + i, adjust(arguments[i][0], torch.empty_like(arguments[i][0]), **arguments[i][1])))
    torch.cuda.synchronize()
    for k, out in got:
        if k < 4:
            rows = attention[k].cu[-1]
            assert torch.equal(out[:rows], alone[k][:rows])
        else:
            assert torch.equal(out, alone_scores[k - 4])
    for case, expected in zip(tables, expected_tables):
        for stream in streams:
            with torch.cuda.stream(stream):
                assert case.run() == expected
            torch.cuda.synchronize()
    assert all(step.d["status"].item() == 0 for step in attention)


@pytest.mark.parametrize("chained", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype,window", [(8, 2, 128, 16, torch.bfloat16, 64), (8, 2, 128, 16, torch.bfloat16, -96),
                                                                  (16, 4, 64, 8, torch.bfloat16, 40), (6, 2, 80, 16, torch.bfloat16, 64),
                                                                  (24, 2, 128, 16, torch.float32, 50), (8, 2, 128, 16, torch.bfloat16, 0),
                                                                  (24, 2, 128, 16, torch.float32, 0)])
def test_a_decoding_loop_under_a_window(chained, heads, kv_heads, dim, page, dtype, window):
    """Requests on one prefix, the longest first: attention on the tables that the step's kernel writes, which leave out what a
    request no longer sees. Against one softmax over each request's keys, in 64 bits, by its bounds."""
    from matricxon_b200.ops import kernels

    prefix, n, steps = 160, 6, 8
    own = [150, 30, 0, 70, 15, 1]
    context = [prefix + k for k in own]
    width, n_pages = 45, 400
    gen = torch.Generator(device=DEV).manual_seed(9)
    ints = lambda values: torch.tensor(values, dtype=torch.int32, device=DEV)  # noqa: E731
    history = [(torch.randn(context[s] + steps, kv_heads, dim, generator=gen, device=DEV).to(dtype),
                torch.randn(context[s] + steps, kv_heads, dim, generator=gen, device=DEV).to(dtype)) for s in range(n)]
    for k, v in history[1:]:
        k[:prefix], v[:prefix] = history[0][0][:prefix], history[0][1][:prefix]
    cache = torch.full((n_pages, 2, kv_heads, page, dim), float("nan"), dtype=dtype, device=DEV)
    values = cache[:, 1].view(n_pages, kv_heads, dim, page)
    pages = torch.randperm(n_pages, generator=torch.Generator().manual_seed(1)).tolist()
    tables = [[-1] * width for _ in range(n)]
    for s in range(n):
        for k in range(prefix // page if s else 0, -(-context[s] // page)):
            tables[s][k] = pages.pop()
    for s in range(n):
        for p in range(prefix if s else 0, context[s]):
            cache[tables[s][p // page], 0, :, p % page] = history[s][0][p]
            values[tables[s][p // page], :, :, p % page] = history[s][1][p]
    tables, free = ints(tables), ints(pages)
    shared_rows, shared_pages = ints([-1] + [0] * (n - 1)), ints([0] + [prefix // page] * (n - 1))
    lengths, status = ints(context), ints([0])
    out = {name: torch.empty(size, dtype=torch.int32, device=DEV) for name, size in
           (("positions", n), ("tok_seq", n), ("cu_q", n + 1), ("slots", n), ("taken", 1))}
    block_tables, taken_all = torch.empty(n, width, dtype=torch.int32, device=DEV), ints([0])
    q, key, value = (torch.zeros(n, h * dim, dtype=dtype, device=DEV) for h in (heads, kv_heads, kv_heads))
    attended = torch.empty(n, heads * dim, dtype=dtype, device=DEV)
    q_lens, n_free, first, shared_lens = ints([1] * n), ints([len(pages)]), ints([0, n]), ints([prefix] * n)
    places = torch.arange(free.numel(), device=DEV)

    def step():
        kernels.step_tables(q_lens, lengths, None, tables, free, n_free, page, n_pages, out["positions"], out["tok_seq"], out["cu_q"],
                            out["slots"], block_tables, out["taken"], status, shared_rows=shared_rows, shared_pages=shared_pages, window=window)
        at, inside = out["slots"].long() // page, out["slots"].long() % page
        cache[:, 0].transpose(1, 2)[at, inside] = key.view(n, kv_heads, dim)
        values.permute(0, 3, 1, 2)[at, inside] = value.view(n, kv_heads, dim)
        kernels.paged_attention_shared(q, q.stride(0), cache, block_tables, out["cu_q"], lengths, out["tok_seq"], out["positions"],
                                       first, shared_lens, n, heads, kv_heads, dim, window, dim ** -0.5, attended, status, max_q_len=1,
                                       max_shared_len=prefix, max_own_len=256)
        lengths.add_(1)
        free.copy_(free[(places + out["taken"]) % free.numel()])
        taken_all.add_(out["taken"])

    keep = [t.clone() for t in (tables, free, lengths, cache)]
    step()
    for tensor, kept in zip((tables, free, lengths, cache), keep):
        tensor.copy_(kept)
    status.zero_()
    taken_all.zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    kernels.set_chained_launch(chained)
    try:
        with torch.cuda.graph(graph):
            step()
    finally:
        kernels.set_chained_launch(False)
    half, out_half = torch.finfo(torch.float32).eps / 2, torch.finfo(dtype).eps / 2
    for i in range(steps):
        q.copy_((1.5 * torch.randn(n, heads * dim, generator=gen, device=DEV)).to(dtype))
        for s in range(n):
            key[s], value[s] = history[s][0][context[s] + i].view(-1), history[s][1][context[s] + i].view(-1)
        graph.replay()
        for s in range(n):
            position = context[s] + i
            low = 0 if window == 0 else max(0, position - window + 1) if window > 0 else position - position % -window
            k, v = (t[low:position + 1].double() for t in history[s])
            rows = q[s].double().view(kv_heads, heads // kv_heads, dim)
            weights = torch.softmax(torch.einsum("kgd,jkd->kgj", rows, k) * dim ** -0.5, -1)
            size = torch.einsum("kgd,jkd->kgj", rows.abs(), k.abs()) * dim ** -0.5
            ref = torch.einsum("kgj,jkd->kgd", weights, v)
            sizes = torch.einsum("kgj,jkd->kgd", weights, v.abs())
            # the bound of test_gpu_attention_shared.py: scores, exponentials, two sums of n weights; a weight rounded to
            # bfloat16 before it meets its value; the result rounded once
            off = (2 * (dim + 4) * half * size.amax(-1) + 32 * half)[..., None] * 2 + (2 * k.shape[0] + 16) * half
            bound = (off + (out_half if dtype == torch.bfloat16 else 0.0)) * sizes + out_half * ref.abs()
            assert ((attended[s].double().view_as(ref) - ref).abs() <= bound).all()
            assert block_tables[s, :low // page].max().item() < 0 if low >= page else True
    assert status.item() == 0
    assert taken_all.item() == sum(-(-(c + steps) // page) - -(-c // page) for c in context)


@pytest.mark.parametrize("look_ahead", [True, False])
def test_engine_penalties_change_what_is_chosen(look_ahead):
    """Greedy requests whose plain text repeats itself: with a penalty above every score no token comes twice, with a bonus the
    first one comes again and again, and a bias of its own size takes its token out."""
    from test_gpu_generation import random_ids, tiny_config, tiny_tensors

    from matricxon_b200 import ChatEngine, GenerationRequest, SamplingConfig
    from matricxon_b200.engine.core import model_from_tensors

    model = model_from_tensors(tiny_config("A"), tiny_tensors("A", torch.float32), dtype="float32", device=DEV)
    vocab = model.spec.vocab_size
    engine = ChatEngine(model, max_cache_tokens=4096, max_active=8, prefill_chunk=32, max_model_len=128, look_ahead=look_ahead)

    def generate(prompts, **options):
        config = SamplingConfig(temperature=0.0, repeat_penalty=1.0, num_predict=24, num_ctx=128, **options)
        return [r.token_ids for r in engine.generate_batch([GenerationRequest(p, config) for p in prompts])]

    prompts = [random_ids(7 + i, vocab, seed=i) for i in range(8)]
    plain = generate(prompts)
    prompts, plain = zip(*[(p, t) for p, t in zip(prompts, plain) if len(t) == 24 and len(set(t)) < 20])
    assert prompts                                        # the plain choice repeats itself, or this shows nothing
    for options in ({"frequency_penalty": 1e4}, {"presence_penalty": 1e4}):
        for text, before in zip(generate(prompts, **options), plain):
            assert text[0] == before[0] and len(text) == 24 and len(set(text)) == 24
    for text, before in zip(generate(prompts, frequency_penalty=-1e4), plain):
        assert text == [before[0]] * len(text)
    for prompt, before in zip(prompts, plain):
        assert before[0] not in generate([prompt], logit_bias={before[0]: -1e4})[0]
