"""Beam search through the entry point (`Model.generate_beams`): the host's decisions against a search over all beams written out plainly, and
whole searches of every architecture against the same search over logits of prompts that are run anew for every text."""
import json
import math
import random

import pytest
import torch

import plain_beams as P
import test_buludra
import test_forisun
import test_mibezen
import test_mugedra
import test_ramolix
import test_zivitar
from helpers import TINY_A, TINY_B, make_model_dir, random_tokens
from janus_b200.engine.beams import _Search, beam_pages, room_for_beams, take_step, text_value, texts_of

gpu = pytest.mark.gpu
NONE = -math.inf


def plain_search(logits_of, beams, limit, stops, length_penalty, early_stopping):
    """(texts as (tokens, score, value, reason), the best first; the smallest distance of two numbers that were compared).  logits_of(texts):
    [len(texts), V] behind each of them."""
    texts, scores, ended, gap = [[]] * beams, [0.0] + [NONE] * (beams - 1), [], math.inf
    for n in range(1, limit + 1):
        logits = logits_of([t if s > NONE else None for t, s in zip(texts, scores)])
        parents, tokens, nxt, ep, _, es, near = P.select(logits, torch.tensor([scores]), stops)
        gap = min(gap, near)
        for b, s in zip(ep[0], es[0]):
            if b >= 0:
                ended.append((texts[b], s, text_value(s, n, length_penalty), "stop"))
        texts = [texts[p] + [t] if p >= 0 else [] for p, t in zip(parents[0], tokens[0])]
        scores = [float(torch.tensor(s, dtype=torch.float32)) for s in nxt[0]]
        live = [(t, s) for t, s in zip(texts, scores) if s > NONE]
        if n == limit:
            ended += [(t, s, text_value(s, n, length_penalty), "length") for t, s in live]
        ended.sort(key=lambda e: -e[2])
        for a, b in zip(ended[: beams + 1], ended[1:]):
            if a[2] != b[2]:
                gap = min(gap, a[2] - b[2])
        ended = ended[:beams]
        if not live:
            break
        if len(ended) == beams:
            reach = max(s for _, s in live) / (limit if length_penalty > 0 else n + 1) ** length_penalty
            gap = min(gap, abs(reach - ended[-1][2])) if not early_stopping else gap
            if early_stopping or reach <= ended[-1][2]:
                break
    return ended, gap


# -- the host's part, without a device ---------------------------------------------------------------------------------------
class Tables:
    """A language of fixed random tables: the logits behind a text depend on its last two tokens."""

    def __init__(self, V, seed):
        g = torch.Generator().manual_seed(seed)
        self.V, self.rows = V, torch.randn(V * V + V + 1, V, generator=g) * 2.0

    def __call__(self, texts):
        return torch.stack([torch.zeros(self.V) if t is None else self.rows[self.place(t)] for t in texts])

    def place(self, t):
        return 0 if not t else 1 + t[-1] if len(t) == 1 else 1 + self.V + t[-2] * self.V + t[-1]


def host_search(logits_of, beams, limit, stops, length_penalty, early_stopping):
    q = _Search(0, limit)
    texts, scores = [[]] * beams, [0.0] + [NONE] * (beams - 1)
    while not q.done:
        logits = logits_of([t if s > NONE else None for t, s in zip(texts, scores)])
        parents, tokens, nxt, ep, _, es, _ = P.select(logits, torch.tensor([scores]), stops)
        texts = [texts[p] + [t] if p >= 0 else [] for p, t in zip(parents[0], tokens[0])]
        scores = [float(torch.tensor(s, dtype=torch.float32)) for s in nxt[0]]
        take_step(q, parents[0], tokens[0], scores, ep[0], es[0], beams, length_penalty, early_stopping)
    return texts_of(q)


@pytest.mark.parametrize("seed", range(12))
def test_host_search_against_the_plain_one(seed):
    rnd = random.Random(seed)
    V, beams, limit = rnd.choice([2, 5, 11]), rnd.choice([1, 2, 4, 7]), rnd.choice([1, 2, 6, 15])
    stops = rnd.sample(range(V), rnd.choice([0, 1, 2]))
    penalty, early = rnd.choice([0.0, 1.0, 0.6, 2.0, -0.5]), rnd.random() < 0.4
    lm = Tables(V, seed)
    want, _ = plain_search(lm, beams, limit, stops, penalty, early)
    got = host_search(lm, beams, limit, stops, penalty, early)
    assert [(t.tokens, t.reason) for t in got] == [(w[0], w[3]) for w in want]
    assert all(t.score == w[1] and t.value == w[2] for t, w in zip(got, want))


def test_host_search_finds_the_best_text_of_all():
    """With as many beams as texts nothing is lost: the best of all texts of three tokens comes first."""
    V, stops = 3, [2]
    lm = Tables(V, 5)
    every = []

    def walk(text, score):
        logp = lm([text])[0].double().log_softmax(0)
        every.append((text, score + float(logp[2]), len(text) + 1))
        for v in (0, 1):
            if len(text) == 2:
                every.append((text + [v], score + float(logp[v]), 3))
            else:
                walk(text + [v], score + float(logp[v]))

    walk([], 0.0)
    best = max(every, key=lambda e: e[1] / e[2])
    got = host_search(lm, 9, 3, stops, 1.0, False)
    assert got[0].tokens == best[0] and abs(got[0].value - best[1] / best[2]) < 1e-6


def _cache(slots, groups=()):
    from types import SimpleNamespace
    groups = [SimpleNamespace(pool=SimpleNamespace(n_free=n, n_pages=n)) for n in groups]
    return SimpleNamespace(n_free_slots=slots, groups=groups)


def _runner(cache):
    from types import SimpleNamespace
    from janus_b200.engine.beams import BeamRunner
    return BeamRunner(SimpleNamespace(cache=cache, max_seq_len=1 << 30, model=SimpleNamespace(vocab_size=100)))


@pytest.mark.parametrize("requests, beams, length, limit", [(64, 4, 40, 66000), (1024, 1, 3, 70), (32, 32, 1000, 130000), (1, 32, 1, (1 << 25) - 64)])
def test_batches_of_models_that_keep_only_states(requests, beams, length, limit):
    """Their tables are of pages that hold nothing; whatever a batch's slots have room for, they are what `ops.fork_pages` takes."""
    from janus_b200.engine.beams import position_pages, table_width
    from janus_b200.kernels import ops
    prompts, searches = [[1] * length] * requests, [_Search(i, limit) for i in range(requests)]
    n = _runner(_cache(1024))._batch_size(prompts, searches, 0, beams, requests)
    assert n == requests
    size, pages = position_pages(n, beams, table_width(-(-(length + limit) // 64)))
    assert size >= length + limit and pages <= ops.MOST_FORK_PAGES and size * pages <= ops.MOST_FORK_TOKENS


def test_batches_stop_where_tables_end():
    """Texts so long that their tokens pass what tables count: fewer requests a batch; one that is alone too long is refused."""
    from janus_b200.cache import CacheFull
    limit = 1 << 22
    prompts, searches = [[1]] * 300, [_Search(i, limit) for i in range(300)]
    n = _runner(_cache(4096))._batch_size(prompts, searches, 0, 4, 300)
    assert n == 50                                          # pages of 2^23 tokens, 255 of them: 1 + 5 n
    with pytest.raises(CacheFull, match="tables"):
        _runner(_cache(4096))._batch_size(prompts, [_Search(0, 1 << 29)], 0, 4, 1)
    with pytest.raises(CacheFull, match="1 pages"):
        _runner(_cache(4096, [1]))._batch_size(prompts, searches[:1], 0, 1, 1)


def test_a_cache_of_more_pages_than_tables_count_is_refused_before_the_prompts():
    from janus_b200.kernels import ops
    with pytest.raises(ValueError, match="pages"):
        _runner(_cache(64, [10, ops.MOST_FORK_PAGES + 1])).generate([[1, 2]], 2, 10)


def test_room_for_beams():
    assert beam_pages(64, 1) == 1 and beam_pages(63, 1) == 1 and beam_pages(63, 2) == 2 and beam_pages(130, 70) == 2
    assert room_for_beams([10, 64], 1, 3, 2) == (1 + 3 + 1 + 3 + 1) * 64
    assert room_for_beams([10, 64, 640], 1, 3, 1) == (10 + 3 + 1) * 64


# -- whole searches ------------------------------------------------------------------------------------------------------------
def by_prompts(model, prompt):
    """Logits behind prompt + text, each from a prompt of its own."""
    from janus_b200.engine import StepEntry

    def logits_of(texts):
        rows = []
        for t in texts:
            if t is None:
                rows.append(torch.zeros(model.engine.model.vocab_size))
                continue
            slot = model.alloc_slot()
            ids = list(prompt) + list(t)
            rows.append(model.step([StepEntry(slot, ids, [len(ids) - 1])])[0].cpu())
            model.free_slot(slot)
        return torch.stack(rows)

    return logits_of


def clear_cases(model, vocab, lengths, beams, limit, stops, penalty, early, wanted, seed, least):
    """Prompts whose plain search has no two numbers nearer than `least`, with the search's texts."""
    found = []
    for i in range(60):
        prompt = random_tokens(lengths[len(found)], vocab, seed + i)
        texts, gap = plain_search(by_prompts(model, prompt), beams, limit, stops, penalty, early)
        if gap > least:
            found.append((prompt, texts))
            if len(found) == wanted:
                return found
    raise AssertionError("no prompts with a clear ranking")


LLAMA_C = {**TINY_A, "max_position_embeddings": 512, "eos_token_id": [3]}
DESIGNS = {"llama A": LLAMA_C, "llama B": TINY_B, "zivitar A": test_zivitar.CFG_A, "zivitar B": test_zivitar.CFG_B, "zivitar C": test_zivitar.CFG_C,
           "ramolix A": test_ramolix.CONFIGS["A"], "ramolix B": test_ramolix.CONFIGS["B"], "mugedra A": test_mugedra.CFG_A,
           "mugedra B": test_mugedra.CFG_B, "buludra A": test_buludra.CONFIGS["A"], "buludra B": test_buludra.CONFIGS["B"],
           "forisun A": test_forisun.CONFIGS["A"], "forisun B": test_forisun.CONFIGS["B"], "mibezen A": test_mibezen.CONFIGS["A"],
           "mibezen B": test_mibezen.CONFIGS["B"]}


def random_model(cfg, dtype, seed=3, max_tokens=16384, **kw):
    import janus_b200
    return janus_b200.load_random(cfg, seed, dtype=dtype, max_tokens=max_tokens, max_slots=64, std=0.15, **kw)


@gpu
@pytest.mark.parametrize("name", list(DESIGNS))
def test_every_architecture_searches_as_the_plain_search(name):
    """float32.  Logits of a text by single tokens and by a prompt differ by some 1e-5 of their size at most; rankings nearer than 1e-3 are
    not asked for."""
    model = random_model(DESIGNS[name], "float32")
    V = model.engine.model.vocab_size
    stops = [7, 11]
    cases = clear_cases(model, V, [66, 5, 31], 4, 9, stops, 1.0, False, 3, 100, 1e-3)
    got, stats = model.generate_beams([c[0] for c in cases], beams=4, max_tokens=9, stop_token_ids=stops, ignore_eos=True, return_all=True)
    for texts, (_, want) in zip(got, cases):
        assert [(t.tokens, t.reason) for t in texts] == [(w[0], w[3]) for w in want]
        assert all(abs(t.score - w[1]) < 1e-3 * max(1.0, abs(w[1])) for t, w in zip(texts, want))
    assert stats.requests == 3 and stats.batches == 1
    model.engine.cache.check()
    assert model.engine.cache.n_free_slots == 64 and all(g.pool.n_held == 0 for g in model.engine.cache.groups)


STATES_ONLY = {
    "lightning": dict(architecture="Zivitar", vocab=120, width=64, norm=dict(eps=1e-5), streams=2,
                      layers=[test_zivitar.layer("lightning", dict(heads=2, dim=16, vdim=40, decay=[0.9, 0.999]), 96, 1.0),
                              test_zivitar.layer("lightning", dict(heads=4, dim=8, vdim=16, decay=[0.5, 0.8, 0.95, 0.99]), 72, 0.5)]),
    "mamba2": test_ramolix.config(140, 96, 1e-6, 1.0, 1.0, [test_ramolix.layer("mamba2", test_ramolix.mamba(3, 16, 24, 3, 4, 3), 40),
                                                            test_ramolix.layer("mamba2", test_ramolix.mamba(2, 24, 8, 1, 2, 1), 72)])}


@gpu
@pytest.mark.parametrize("name", list(STATES_ONLY))
def test_models_that_keep_only_states(name):
    """No pages at all: states move with their beams, positions and lengths with tables that hold nothing."""
    model = random_model(STATES_ONLY[name], "float32")
    assert not model.engine.cache.groups
    stops = [7, 11]
    cases = clear_cases(model, model.engine.model.vocab_size, [66, 5, 31], 4, 9, stops, 1.0, False, 3, 100, 1e-3)
    for _ in range(2):                                       # (the second time from the captured step)
        got, stats = model.generate_beams([c[0] for c in cases], beams=4, max_tokens=9, stop_token_ids=stops, ignore_eos=True, return_all=True)
        for texts, (_, want) in zip(got, cases):
            assert [(t.tokens, t.reason) for t in texts] == [(w[0], w[3]) for w in want]
    assert stats.graph_captures == 0
    # texts across what would be pages of 64 tokens, alone and in a batch
    whole, _ = model.generate_beams([c[0] for c in cases], beams=3, max_tokens=100, ignore_eos=True, return_all=True)
    for (prompt, _), texts in zip(cases, whole):
        alone, _ = model.generate_beams([prompt], beams=3, max_tokens=100, ignore_eos=True, return_all=True)
        assert [t.tokens for t in alone[0]] == [t.tokens for t in texts] and all(len(t.tokens) == 100 for t in texts)
    model.engine.cache.check()
    assert model.engine.cache.n_free_slots == 64


@gpu
def test_many_long_requests_of_a_model_that_keeps_only_states(monkeypatch):
    """64 requests of 4 beams with tables for texts of 70,000 tokens, more than 2^19 pages of 64: the first 30 tokens of them."""
    import janus_b200
    from janus_b200.engine.beams import BeamRunner
    model = janus_b200.load_random(STATES_ONLY["mamba2"], 3, dtype="float32", max_tokens=1 << 20, max_slots=256, std=0.15)
    prompts = [random_tokens(2 + n % 5, 140, n) for n in range(64)]
    want, _ = model.generate_beams(prompts, beams=4, max_tokens=30, ignore_eos=True, return_all=True)
    run_batch, step_for, widths = BeamRunner._run_batch, BeamRunner._step_for, []

    def shortened(self, prompts, searches, *args):
        def cut(self, *sizes):
            step = step_for(self, *sizes)
            widths.append(step.W)
            for q in searches:
                q.limit = 30
            return step

        monkeypatch.setattr(BeamRunner, "_step_for", cut)
        return run_batch(self, prompts, searches, *args)

    monkeypatch.setattr(BeamRunner, "_run_batch", shortened)
    got, stats = model.generate_beams(prompts, beams=4, max_tokens=70000, ignore_eos=True, return_all=True)
    assert stats.batches == 1 and widths == [2048]
    assert [[t.tokens for t in row] for row in got] == [[t.tokens for t in row] for row in want]


@gpu
@pytest.mark.parametrize("beams, penalty, early", [(1, 1.0, False), (2, 0.0, True), (5, 2.0, False), (8, -0.5, True), (16, 0.7, False)])
def test_numbers_of_beams_and_penalties(beams, penalty, early):
    model = random_model(LLAMA_C, "float32")
    stops = [3, 40, 77, 110]
    cases = clear_cases(model, 256, [64, 130], beams, 12, stops, penalty, early, 2, 500, 2e-4)
    got, _ = model.generate_beams([c[0] for c in cases], beams=beams, max_tokens=12, stop_token_ids=stops[1:], length_penalty=penalty,
                                  early_stopping=early, return_all=True)
    for texts, (_, want) in zip(got, cases):
        assert [(t.tokens, t.reason) for t in texts] == [(w[0], w[3]) for w in want]


@gpu
def test_long_texts_cross_pages_and_batches_follow_one_another():
    """Texts of 150 tokens (three pages), twice through a cache that holds one batch; pages and slots are used again."""
    model = random_model(LLAMA_C, "float32", max_tokens=64 * 40)
    prompts = [random_tokens(n, 256, n) for n in (61, 3, 64, 100)]
    whole, stats = model.generate_beams(prompts, beams=3, max_tokens=150, ignore_eos=True, return_all=True, batch_size=2)
    assert stats.batches >= 2
    for prompt, texts in zip(prompts, whole):
        alone, _ = model.generate_beams([prompt], beams=3, max_tokens=150, ignore_eos=True, return_all=True)
        assert [t.tokens for t in alone[0]] == [t.tokens for t in texts] and len({tuple(t.tokens) for t in texts}) == len(texts)
        for t in texts:
            assert len(t.tokens) == 150 and t.reason == "length"
            # the text's score is the sum of its tokens' log-probabilities in one prompt
            from janus_b200.engine import StepEntry
            slot, ids = model.alloc_slot(), prompt + t.tokens
            logits = model.step([StepEntry(slot, ids[:-1], range(len(prompt) - 1, len(ids) - 1))]).cpu().double()
            model.free_slot(slot)
            want = float(logits.log_softmax(1).gather(1, torch.tensor(t.tokens)[:, None]).sum())
            assert abs(want - t.score) < 1e-4 * abs(want)
    model.engine.cache.check()


@gpu
@pytest.mark.parametrize("shared", [True, False])
@pytest.mark.parametrize("name", ["llama A", "llama B", "zivitar A", "mugedra A"])
def test_bfloat16_scores_are_the_texts_own(name, shared, monkeypatch):
    """bfloat16, with pages that beams share read once for all and by every row: logits of a text by single tokens and by a prompt differ by the
    engine's tolerance (3e-2 of the largest), every token's log-probability by twice that at most."""
    from janus_b200.kernels import ops
    calls, attention = [], ops.attention_beams
    monkeypatch.setattr(ops, "beams_pay", lambda *sizes: shared)
    monkeypatch.setattr(ops, "attention_beams", lambda *a, **kw: (calls.append(1), attention(*a, **kw)))
    model = random_model(DESIGNS[name], "bfloat16")
    V = model.engine.model.vocab_size
    prompts = [random_tokens(n, V, n) for n in (200, 64, 9)]
    got, _ = model.generate_beams(prompts, beams=4, max_tokens=30, ignore_eos=True, return_all=True)
    for prompt, texts in zip(prompts, got):
        assert len(texts) == 4 and len({tuple(t.tokens) for t in texts}) == 4
        assert [t.value for t in texts] == sorted((t.value for t in texts), reverse=True)
        for t in texts:
            rows = torch.cat([by_prompts(model, prompt)([t.tokens[:i]]) for i in range(len(t.tokens))]).double()
            want = float(rows.log_softmax(1).gather(1, torch.tensor(t.tokens)[:, None]).sum())
            assert abs(want - t.score) <= 30 * 2 * 3e-2 * float(rows.abs().max())
    assert bool(calls) == (shared and name.startswith("llama"))


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_one_beam_is_greedy_generation(dtype):
    model = random_model(LLAMA_C, dtype)
    prompts = [random_tokens(n, 256, n) for n in (70, 1, 33)]
    if dtype == "float32":
        # (the first text that ends is enough; without that a beam goes on while a longer text may become better)
        got, _ = model.generate_beams(prompts, beams=1, max_tokens=40, early_stopping=True)
        want, _ = model.generate(prompts, max_tokens=40)
        assert got == want
    again = [model.generate_beams(prompts, beams=3, max_tokens=20)[0] for _ in range(2)]
    assert dtype == "bfloat16" or again[0] == again[1]


@gpu
@pytest.mark.parametrize("lengths", [(70, 1, 33), (64, 128, 5)])
def test_one_beam_in_bfloat16_takes_what_a_prompt_prefers(lengths):
    """Every token of the one text is within the engine's tolerance (3e-2 of the largest logit, for the step and for the prompt) of the best, and the
    score is the sum of those log-probabilities."""
    model = random_model(LLAMA_C, "bfloat16")
    prompts = [random_tokens(n, 256, n) for n in lengths]
    got, _ = model.generate_beams(prompts, beams=1, max_tokens=40, ignore_eos=True, return_all=True)
    for prompt, (text,) in zip(prompts, got):
        assert len(text.tokens) == 40 and text.reason == "length"
        rows = torch.cat([by_prompts(model, prompt)([text.tokens[:i]]) for i in range(40)]).double()
        taken = rows.gather(1, torch.tensor(text.tokens)[:, None])[:, 0]
        tolerance = 2 * 3e-2 * rows.abs().max(1).values
        assert torch.all(taken >= rows.max(1).values - tolerance)
        assert abs(float((taken - rows.logsumexp(1)).sum()) - text.score) <= float(tolerance.sum())


@gpu
@pytest.mark.parametrize("name, beams, lengths", [("llama A", 4, (200, 64, 9)), ("llama A", 16, (130, 63)), ("llama B", 7, (128, 1, 100))])
def test_attention_within_a_search_is_each_rows_own(name, beams, lengths, monkeypatch):
    """Every call of `attention_beams` that a search makes, in every layer of every step, against the definition over the rows' own pages in 64 bits: pages
    said to be shared that are not, tables or copies a step behind would show in it."""
    import plain_beams
    from janus_b200.kernels import ops
    from test_beams import attention_bound
    calls, attention = [], ops.attention_beams
    monkeypatch.setattr(ops, "beams_pay", lambda *sizes: True)

    def compared(q, k, v, out, table, kv_len, shared, K, nh, nkv, hd, page_size, scale, workspace, bound):
        attention(q, k, v, out, table, kv_len, shared, K, nh, nkv, hd, page_size, scale, workspace, bound)
        want, size = plain_beams.attention(q, k, v, table.tolist(), kv_len.tolist(), nh, nkv, hd, scale)
        off = (out.cpu().double().view(want.shape) - want).abs()
        calls.append((float((off / attention_bound(want, size)).max()), int(shared.max())))

    monkeypatch.setattr(ops, "attention_beams", compared)
    model = random_model(DESIGNS[name], "bfloat16", use_graphs=False)
    prompts = [random_tokens(n, model.engine.model.vocab_size, n) for n in lengths]
    model.generate_beams(prompts, beams=beams, max_tokens=24, ignore_eos=True)
    layers = DESIGNS[name]["num_hidden_layers"]
    assert len(calls) == 23 * layers and max(c[0] for c in calls) <= 1.0 and max(c[1] for c in calls) == max(lengths) // 64


@gpu
def test_with_and_without_graphs():
    out = []
    for graphs in (True, False):
        model = random_model(LLAMA_C, "float32", use_graphs=graphs)
        prompts = [random_tokens(n, 256, n) for n in (90, 20)]
        texts, stats = model.generate_beams(prompts, beams=4, max_tokens=70, ignore_eos=True, return_all=True)
        out.append([[(t.tokens, t.reason) for t in row] for row in texts])
        assert (stats.graph_captures > 0) == graphs
    assert out[0] == out[1]


@gpu
def test_a_captured_step_serves_later_calls():
    """Batches of as many requests and beams, lengths up to as many pages (a power of two) and no more prompt tokens record one step."""
    model = random_model(LLAMA_C, "float32")
    first = [random_tokens(n, 256, n) for n in (90, 20)]
    _, stats = model.generate_beams(first, beams=4, max_tokens=30, ignore_eos=True)
    assert stats.graph_captures == 1
    for lengths in ((30, 70), (3, 98)):
        prompts = [random_tokens(n, 256, n) for n in lengths]
        got, stats = model.generate_beams(prompts, beams=4, max_tokens=30, ignore_eos=True)
        assert stats.graph_captures == 0
        assert got == random_model(LLAMA_C, "float32").generate_beams(prompts, beams=4, max_tokens=30, ignore_eos=True)[0]


@gpu
def test_requests_of_unequal_limits_and_the_longest_length():
    """A prompt near the longest length ends earlier than its neighbours."""
    model = random_model(LLAMA_C, "float32", max_seq_len=128)
    prompts = [random_tokens(n, 256, n) for n in (128, 120, 12)]
    texts, _ = model.generate_beams(prompts, beams=3, max_tokens=30, ignore_eos=True, return_all=True)
    assert [[len(t.tokens) for t in row] for row in texts] == [[1] * 3, [9] * 3, [30] * 3]
    for prompt, row in zip(prompts, texts):
        alone, _ = model.generate_beams([prompt], beams=3, max_tokens=30, ignore_eos=True, return_all=True)
        assert [t.tokens for t in alone[0]] == [t.tokens for t in row]


@gpu
def test_plain_generation_beside_beams():
    """Slots and pages of a caller stay as they were, and what ran before gives the same afterwards."""
    from janus_b200.engine import StepEntry
    model = random_model(LLAMA_C, "float32")
    prompts = [random_tokens(n, 256, n) for n in (70, 30)]
    before, _ = model.generate(prompts, max_tokens=30)
    slot = model.alloc_slot()
    model.step([StepEntry(slot, prompts[0], [])])
    want = model.step([StepEntry(slot, [5], [0])]).clone()
    model.free_slot(slot)
    slot = model.alloc_slot()
    model.step([StepEntry(slot, prompts[0], [])])
    model.generate_beams(prompts, beams=5, max_tokens=30)
    assert torch.equal(model.step([StepEntry(slot, [5], [0])]), want)
    model.free_slot(slot)
    assert model.generate(prompts, max_tokens=30)[0] == before


@gpu
def test_prompts_in_pieces_of_limited_size():
    model = random_model(LLAMA_C, "float32", max_step_tokens=33)
    prompts = [random_tokens(n, 256, n) for n in (70, 1, 1, 64)]
    got, _ = model.generate_beams(prompts, beams=2, max_tokens=10, ignore_eos=True)
    model.engine.options.max_step_tokens = None
    assert model.generate_beams(prompts, beams=2, max_tokens=10, ignore_eos=True)[0] == got


@gpu
def test_refusals():
    from janus_b200.cache import CacheFull
    from janus_b200.engine.step import StepError
    model = random_model(LLAMA_C, "float32", max_tokens=64 * 8)
    ok = [[1, 2, 3]]
    for bad, kw in ((ValueError, dict(beams=0)), (ValueError, dict(beams=33)), (ValueError, dict(max_tokens=-1)), (ValueError, dict(length_penalty=math.nan)),
                    (ValueError, dict(length_penalty=1e3)), (ValueError, dict(length_penalty=-1e3)),
                    (ValueError, dict(stop_token_ids=range(33))), (ValueError, dict(batch_size=0)), (CacheFull, dict(beams=8, max_tokens=200))):
        with pytest.raises(bad):
            model.generate_beams(ok, **kw)
    for bad, prompts in ((ValueError, [[]]), (StepError, [[256]]), (StepError, [[-1]]), (ValueError, [[1] * 513])):
        with pytest.raises(bad):
            model.generate_beams(prompts)
    assert model.generate_beams([], beams=2)[0] == [] and model.generate_beams(ok, max_tokens=0)[0] == [[]]
    model.engine.cache.check()
    assert model.engine.cache.n_free_slots == 64


@gpu
def test_what_ends_a_search_in_the_middle_gives_everything_back(monkeypatch):
    from janus_b200.engine.beams import BeamRunner
    model = random_model(LLAMA_C, "float32")
    prompts = [random_tokens(n, 256, n) for n in (70, 30)]
    want, _ = model.generate_beams(prompts, beams=3, max_tokens=20, ignore_eos=True)
    free = model.engine.cache.n_free_slots, [g.pool.n_free for g in model.engine.cache.groups]
    take, calls = BeamRunner._take, []

    def stops(self, *args):
        calls.append(1)
        if len(calls) == 5:
            raise KeyboardInterrupt
        return take(self, *args)

    monkeypatch.setattr(BeamRunner, "_take", stops)
    with pytest.raises(KeyboardInterrupt):
        model.generate_beams(prompts, beams=3, max_tokens=20, ignore_eos=True)
    monkeypatch.undo()
    assert free == (model.engine.cache.n_free_slots, [g.pool.n_free for g in model.engine.cache.groups])
    model.engine.cache.check()
    assert model.generate_beams(prompts, beams=3, max_tokens=20, ignore_eos=True)[0] == want


@gpu
def test_on_another_stream_and_with_the_most_beams():
    model = random_model(LLAMA_C, "float32", max_tokens=64 * 200)
    prompts = [random_tokens(n, 256, n) for n in (64, 1)]
    want, _ = model.generate_beams(prompts, beams=32, max_tokens=70, ignore_eos=True)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        got, _ = random_model(LLAMA_C, "float32", max_tokens=64 * 200).generate_beams(prompts, beams=32, max_tokens=70, ignore_eos=True)
    assert got == want


@gpu
def test_command_line(tmp_path, capsys):
    from janus_b200.cli import main
    d = make_model_dir(LLAMA_C, str(tmp_path / "m"), 1, "float32")
    assert main([d, "1,2,3", "4 5", "--beams", "3", "--max-tokens", "8", "--dtype", "fp32", "--json", "--ignore-eos"]) == 0
    out = json.loads(capsys.readouterr().out)
    assert [len(t) for t in out["tokens"]] == [8, 8] and out["finish_reasons"] == ["length"] * 2


def test_command_line_refuses_what_does_not_go_together(capsys):
    from janus_b200.cli import main
    for more in (["--temperature", "0.5"], ["--shared-prefix", "1,2"], ["--top-k", "3"], ["--repetition-penalty", "1.1"], ["--beams", "33"], ["--beams=-1"]):
        with pytest.raises(SystemExit):
            main(["nowhere", "1,2", "--beams", "2", *more])
    capsys.readouterr()
