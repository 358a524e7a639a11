"""Beam search: for each request the most probable texts, several kept at a time.

The prompt runs once, in the slot of a request's first row.  From then on every request has K rows of a step, one a beam, which share
its pages as far as their texts agree.  A step is one CUDA graph: the forward pass of all rows, the choice of continuations over
all beams and the vocabulary (`ops.beam_select`), block tables of the rows that go on (`ops.fork_pages`), copies of partly filled pages
(`ops.copy_pages`) and states of a fixed size moved with their beams (`ops.reorder_rows`).  Tokens, scores and tables stay on the
device; the host reads what was chosen one step later, keeps the history, and ends requests.

The reference names a beam width among its sampling options and has no loop for it
(crates/janus-engine/src/model/sampler.rs:20-39,804-847).
"""
from __future__ import annotations

import gc
import math
import time
from dataclasses import dataclass, field
from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

from ..cache import PAGE_SIZE, CacheFull, GroupStepView
from ..kernels import ops
from .generate import GenerationStats, plan_prompt_steps
from .step import Engine, StepContext, StepEntry, StepError

MOST_GRAPHS = 16       # captured steps that are kept


@dataclass
class BeamText:
    """One of a request's texts."""
    tokens: List[int]
    score: float               # the sum of its tokens' log-probabilities, the stop token's among them
    value: float               # score / length ** length_penalty, by which texts are compared
    reason: str                # "stop" or "length"


@dataclass
class _Search:
    """A request's history and the texts that have ended."""
    index: int
    limit: int                                         # tokens at most
    parents: List[List[int]] = field(default_factory=list)
    tokens: List[List[int]] = field(default_factory=list)
    ended: List[Tuple[float, float, int, int, str]] = field(default_factory=list)    # value, score, tokens, row, reason
    done: bool = False


def text_value(score: float, length: int, length_penalty: float) -> float:
    return score / max(1, length) ** length_penalty


def take_step(q: _Search, parents: Sequence[int], tokens: Sequence[int], scores: Sequence[float], ended_parents: Sequence[int],
              ended_scores: Sequence[float], beams: int, length_penalty: float, early_stopping: bool) -> None:
    """What a step chose for one request: texts that ended are kept, the best `beams` of them; the request is done when its length is reached,
    when no beam is left, or when it has as many texts as beams and (unless `early_stopping` is enough) no beam can become better than
    the worst of them: a score only falls, and the length it is divided by is at most the limit."""
    n = len(q.tokens) + 1
    for b, s in zip(ended_parents, ended_scores):
        if b >= 0:
            q.ended.append((text_value(s, n, length_penalty), s, n - 1, b, "stop"))
    q.parents.append(list(parents))
    q.tokens.append(list(tokens))
    live = [(s, k) for k, (p, s) in enumerate(zip(parents, scores)) if p >= 0]
    if n >= q.limit:
        q.ended += [(text_value(s, n, length_penalty), s, n, k, "length") for s, k in live]
    q.ended.sort(key=lambda t: -t[0])                  # (equal ones as they were found)
    del q.ended[beams:]
    if n >= q.limit or not live:
        q.done = True
    elif len(q.ended) == beams:
        best = max(s for s, _ in live)
        longest = q.limit if length_penalty > 0 else n + 1
        q.done = early_stopping or text_value(best, longest, length_penalty) <= q.ended[-1][0]


def texts_of(q: _Search) -> List[BeamText]:
    out = []
    for value, score, n, row, reason in q.ended:
        tokens = []
        for step in range(n - 1, -1, -1):
            tokens.append(q.tokens[step][row])
            row = q.parents[step][row]
        out.append(BeamText(tokens[::-1], score, value, reason))
    return out


def beam_pages(prompt_len: int, limit: int) -> int:
    """Pages of its own that a beam takes at most behind the whole pages of its prompt.  (The last token is never fed back, but a place for
    it is made ready.)"""
    return -(-(prompt_len + limit) // PAGE_SIZE) - prompt_len // PAGE_SIZE


def room_for_beams(prompt_lens: Sequence[int], max_tokens: int, beams: int, batch_size: int) -> int:
    """Cache tokens, in whole pages, with room for any `batch_size` of the requests."""
    pages = sorted((-(-n // PAGE_SIZE) + beams * beam_pages(n, max_tokens) for n in prompt_lens), reverse=True)
    return (sum(pages[:batch_size]) + 1) * PAGE_SIZE


def table_width(pages: int) -> int:
    """Pages that a step's tables have room for a row: a power of two, so that a captured step serves texts of about as many."""
    W = 1
    while W < pages:
        W *= 2
    return W


def position_pages(R: int, K: int, W: int) -> Tuple[int, int]:
    """(tokens of a page, pages) of the table of a model whose mixers keep only states.  Nobody stores anything in its pages: they carry positions
    and lengths, and one is as long as the longest text.  Page 0 for rows without a beam, one a prompt, one a beam."""
    return W * PAGE_SIZE, 1 + R + R * K


class _Tables:
    """One cache group's tables on the device."""

    def __init__(self, R: int, K: int, W: int, n_pages: int, device: torch.device):
        z = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=device)      # noqa: E731
        self.table, self.refs, self.free, self.n_free = z(R * K, W), z(n_pages), z(n_pages), z(1)
        self.positions, self.dest_rows, self.shared = z(R, K), z(R, K), z(R)
        self.copy_src, self.copy_dst, self.copy_rows = z(R, K), z(R, K), z(R, K)


class _BeamStep:
    """The buffers of a step of R requests of K beams with room for W pages a row, and the step's kernels as a captured graph."""

    def __init__(self, engine: Engine, R: int, K: int, W: int, stops: int):
        self.engine, self.R, self.K, self.W = engine, R, K, W
        cache, device, N = engine.cache, engine.device, R * K
        i32 = dict(dtype=torch.int32, device=device)
        G = max(1, len(cache.groups))
        # what the host reads: six arrays of the choice, and rows for which a page was missing, a number a group
        self.result = torch.zeros(6 * N + G, **i32)
        part = lambda i: self.result[i * N: (i + 1) * N].view(R, K)      # noqa: E731
        self.parents, self.tokens, self.ended_parents, self.ended_tokens = part(0), part(1), part(2), part(3)
        self.scores, self.ended_scores = part(4).view(torch.float32), part(5).view(torch.float32)
        self.missing = [self.result[6 * N + g: 6 * N + g + 1] for g in range(G)]
        self.stops = torch.full((stops,), -1, **i32)
        self.page_size, self.pages = PAGE_SIZE, [g.pool.n_pages for g in cache.groups]
        if not cache.groups:
            self.page_size, n = position_pages(R, K, W)
            self.pages = [n]
        self.tables = [_Tables(R, K, W if cache.groups else 1, n, device) for n in self.pages]
        self.lengths = torch.zeros((R, K), **i32)
        self.other_lengths = torch.zeros((R, K), **i32)
        self.spares = torch.zeros(G, **i32)
        self.spare = [0] * G
        self.slots = torch.zeros(N, **i32)
        self.rows, self.starts = torch.arange(N, **i32), torch.arange(N + 1, **i32)
        self.logits, _ = engine._graph_output_buffers(N)
        self.states = list(cache.states.values())
        self.storage = []
        for g in cache.groups:
            tensors = {t.data_ptr(): t for place in g.places for t in (g.k[place], g.v[place])}
            self.storage.append(list(tensors.values()))
        self.graph, self.generation, self.launches = None, -1, 0
        ctx = StepContext()
        ctx.n_tokens, ctx.n_seqs, ctx.is_decode, ctx.max_q_len = N, N, True, 1
        ctx.max_kv_len_bound = W * PAGE_SIZE
        ctx.token_ids, ctx.positions, ctx.token_seq = self.tokens.view(N), self.tables[0].positions.view(N), self.rows
        ctx.q_start, ctx.kv_len, ctx.seq_slot = self.starts, self.lengths.view(N), self.slots
        ctx.groups = [GroupStepView(t.dest_rows.view(N), t.table, PAGE_SIZE, t.shared) for t in self.tables[: len(cache.groups)]]
        ctx.workspace, ctx.cache, ctx.dtype = engine.workspace, cache, engine.dtype
        ctx.beams = K
        self.ctx = ctx

    def choose(self) -> None:
        """From the logits to tables that are ready for the next step."""
        with ops.stream_scope():
            ops.beam_select(self.logits, self.scores, self.stops, parents=self.parents, tokens=self.tokens, next_scores=self.scores,
                            ended_parents=self.ended_parents, ended_tokens=self.ended_tokens, ended_scores=self.ended_scores,
                            workspace=self.engine.workspace)
            for i, t in enumerate(self.tables):
                last = i == len(self.tables) - 1           # (all groups start from the same lengths)
                ops.fork_pages(self.parents, self.lengths, t.table, t.refs, t.free, t.n_free,
                               kv_len=self.lengths if last else self.other_lengths, positions=t.positions, dest_rows=t.dest_rows,
                               new_table=t.table, new_refs=t.refs, new_free=t.free, new_n_free=t.n_free, copy_src=t.copy_src,
                               copy_dst=t.copy_dst, copy_rows=t.copy_rows, shared=t.shared, missing=self.missing[i], spare=self.spare[i],
                               page_size=self.page_size)
                if i < len(self.storage):
                    N = self.R * self.K
                    ops.copy_pages(self.storage[i], t.copy_src.view(N), t.copy_dst.view(N), t.copy_rows.view(N))
            ops.reorder_rows(self.states, self.slots, self.parents)

    def forward_and_choose(self) -> None:
        self.engine.model.forward(self.ctx, self.rows, self.logits)
        self.choose()

    def begin(self, slots: List[int], prompt_lens: List[int], pages: List[List[List[int]]], mine: List[List[int]], spare: List[int],
              stops: List[int]) -> None:
        """A batch's first tables: row 0 of each request holds its prompt (pages[group][request]), which its slot keeps as well; mine[group]
        are the pages that beams may take, spare[group] the one that rows without a beam use."""
        R, K = self.R, self.K
        if spare != self.spare:
            self.spare, self.graph = list(spare), None       # a captured launch knows it by number
        copy = lambda t, values: t.copy_(torch.from_numpy(np.asarray(values, dtype=np.int32).reshape(t.shape)))      # noqa: E731
        copy(self.slots, slots)
        copy(self.stops, stops)
        lengths = np.ones((R, K), dtype=np.int32)
        lengths[:, 0] = prompt_lens
        copy(self.lengths, lengths)
        self.scores.copy_(torch.tensor([[0.0] + [-math.inf] * (K - 1)] * R))
        for g, t in enumerate(self.tables):
            table, refs = np.full((R, K, t.table.shape[1]), -1, dtype=np.int32), np.zeros(self.pages[g], dtype=np.int32)
            table[:, 1:, 0] = spare[g]
            for r, held in enumerate(pages[g]):
                table[r, 0, : len(held)] = held
                refs[[p for p in held if p >= 0]] = 2        # the row and the slot
            free = np.full(self.pages[g], -1, dtype=np.int32)
            free[: len(mine[g])] = mine[g][::-1]             # (taken from the back)
            for to, values in ((t.table, table), (t.refs, refs), (t.free, free), (t.n_free, [len(mine[g])])):
                copy(to, values)

    def end_request(self, r: int) -> None:
        """The rows of a request that is over go on as rows without a beam."""
        K = self.K
        self.scores[r].fill_(-math.inf)
        self.lengths[r].fill_(1)
        self.tokens[r].zero_()
        for g, t in enumerate(self.tables):
            rows = t.table[r * K: r * K + K]
            rows.fill_(-1)
            rows[:, 0].fill_(self.spare[g])
            t.positions[r].zero_()
            t.dest_rows[r].fill_(self.spare[g] * self.page_size)
            t.shared[r].zero_()

    def run(self) -> None:
        """One step, from the graph if there is one; a step that finds none runs its kernels directly and records them for the next."""
        engine = self.engine
        if not engine.options.use_graphs:
            self.forward_and_choose()
            return
        if self.graph is not None and self.generation == engine.workspace.generation:
            self.graph.replay()
            return
        self.graph = None
        self.forward_and_choose()
        torch.cuda.synchronize(engine.device)
        graph, before = torch.cuda.CUDAGraph(), ops.launch_count()
        gc_was_on = gc.isenabled()
        gc.disable()              # (see Engine._graph_decode: a collection in the middle of a capture may destroy another graph)
        try:
            if engine._capture_stream is None:
                engine._capture_stream = torch.cuda.Stream(device=engine.device)
            side = engine._capture_stream
            side.wait_stream(torch.cuda.current_stream(engine.device))
            with torch.cuda.stream(side), ops.unchecked():
                graph.capture_begin()
                try:
                    self.forward_and_choose()
                finally:
                    graph.capture_end()
            torch.cuda.current_stream(engine.device).wait_stream(side)
        finally:
            if gc_was_on:
                gc.enable()
        self.graph, self.generation, self.launches = graph, engine.workspace.generation, ops.launch_count() - before
        engine.graph_captures += 1


class BeamRunner:
    def __init__(self, engine: Engine):
        self.engine = engine
        self.steps: Dict[Tuple[int, int, int, int], _BeamStep] = {}
        self.staging: List[torch.Tensor] = []

    def generate(self, prompts: Sequence[Sequence[int]], beams: int, max_tokens: int, stop: Sequence[int] = (), length_penalty: float = 1.0,
                 early_stopping: bool = False, batch_size: Optional[int] = None):
        """Returns (texts per request, the best first; stats)."""
        engine = self.engine
        V = engine.model.vocab_size
        stop = sorted({int(t) for t in stop if 0 <= int(t) < V})
        if not 1 <= beams <= ops.MOST_BEAMS:
            raise ValueError(f"{beams} beams: 1 to {ops.MOST_BEAMS} are taken")
        if len(stop) > ops.MOST_BEAM_STOPS:
            raise ValueError(f"{len(stop)} stop tokens: beam search takes up to {ops.MOST_BEAM_STOPS}")
        if max_tokens < 0 or not math.isfinite(length_penalty) or (batch_size is not None and batch_size < 1):
            raise ValueError(f"max_tokens {max_tokens}, length_penalty {length_penalty}, batch_size {batch_size}")
        if abs(length_penalty) * math.log(max(2, min(max_tokens, engine.max_seq_len))) > 600.0:      # (scores times that power stay numbers)
            raise ValueError(f"length_penalty {length_penalty} is too large for {max_tokens} tokens")
        prompts = [np.asarray(p, dtype=np.int64).reshape(-1) for p in prompts]
        for i, p in enumerate(prompts):
            if len(p) == 0:
                raise ValueError(f"prompt {i} is empty")
            if len(p) > engine.max_seq_len:
                raise ValueError(f"prompt {i} has {len(p)} tokens, the longest sequence allowed is {engine.max_seq_len}")
            if p.min() < 0 or p.max() >= V:
                raise StepError(f"a token id of prompt {i} is outside the vocabulary of {V}")
        for g in engine.cache.groups:
            if g.pool.n_pages > ops.MOST_FORK_PAGES:
                raise ValueError(f"beam search takes caches of up to {ops.MOST_FORK_PAGES} pages of {PAGE_SIZE} tokens, this one has {g.pool.n_pages}")
        stats = GenerationStats(requests=len(prompts))
        if max_tokens == 0:
            return [[BeamText([], 0.0, 0.0, "length")] for _ in prompts], stats
        # the last token of a text is not fed back: a text may pass the longest length by that one
        searches = [_Search(i, min(max_tokens, engine.max_seq_len - len(p) + 1)) for i, p in enumerate(prompts)]
        captures = engine.graph_captures
        first = 0
        while first < len(searches):
            n = self._batch_size(prompts, searches, first, beams, batch_size or len(prompts))
            stats.batches += 1
            self._run_batch([prompts[q.index] for q in searches[first: first + n]], searches[first: first + n], beams, stop, length_penalty,
                            early_stopping, stats)
            first += n
        stats.graph_captures = engine.graph_captures - captures
        ops.check_kernel_status(engine.device)
        return [texts_of(q) for q in searches], stats

    def _batch_size(self, prompts, searches, first: int, beams: int, most: int) -> int:
        """Requests of the next batch: as many as slots and every group's free pages have room for."""
        cache = self.engine.cache
        free = min((g.pool.n_free for g in cache.groups), default=0) - 1                  # one for rows without a beam
        n = pages = longest = 0
        for q in searches[first: first + most]:
            length = len(prompts[q.index])
            pages += -(-length // PAGE_SIZE) + beams * beam_pages(length, q.limit)
            longest = max(longest, -(-(length + q.limit) // PAGE_SIZE))
            if (n + 1) * beams > cache.n_free_slots:
                break
            if cache.groups:
                if pages > free:
                    break
            else:
                size, count = position_pages(n + 1, beams, table_width(longest))
                if count > ops.MOST_FORK_PAGES or size * count > ops.MOST_FORK_TOKENS:
                    break
            n += 1
        if n == 0:
            what = f"request {searches[first].index} with {beams} beams needs {beams} slots"
            if cache.groups:
                raise CacheFull(f"{what} and {pages + 1} pages of {PAGE_SIZE} tokens; the cache has {cache.n_free_slots} free slots and {free + 1} pages")
            raise CacheFull(f"{what} and texts of {longest * PAGE_SIZE} tokens; the cache has {cache.n_free_slots} free slots, tables of positions "
                            f"count {ops.MOST_FORK_TOKENS} tokens")
        return n

    def _step_for(self, R: int, K: int, pages: int, stops: int) -> _BeamStep:
        W = table_width(pages)
        key = (R, K, W, stops)
        step = self.steps.pop(key, None)
        logits, _ = self.engine._graph_output_buffers(R * K)
        if step is None or step.logits.data_ptr() != logits.data_ptr():
            step = _BeamStep(self.engine, R, K, W, stops)
        while len(self.steps) >= MOST_GRAPHS:
            del self.steps[next(iter(self.steps))]
        self.steps[key] = step                               # used last: at the end of the line
        return step

    def _run_batch(self, prompts, searches: List[_Search], beams: int, stop: List[int], length_penalty: float, early_stopping: bool,
                   stats: GenerationStats) -> None:
        engine = self.engine
        cache, R, K = engine.cache, len(prompts), beams
        slots: List[int] = []
        mine: List[List[int]] = [[] for _ in cache.groups]
        # rows without a beam use a page that is taken first and given back last, so that it is the same one batch after batch: a
        # captured step knows it by number
        spare: List[int] = []
        try:
            t0 = time.perf_counter()
            for group in cache.groups:
                spare.append(group.pool.take())
            for _ in range(R * K):
                slots.append(engine.alloc_slot())
            step = self._step_for(R, K, max(-(-(len(p) + q.limit) // PAGE_SIZE) for p, q in zip(prompts, searches)), len(stop))
            heads, last = slots[::K], {}
            for pieces in plan_prompt_steps([len(p) for p in prompts], engine.options.max_step_tokens):
                logits = engine.step([StepEntry(heads[i], prompts[i][a:b], (b - a - 1,) if b == len(prompts[i]) else ())
                                      for i, a, b in pieces])
                for row, i in enumerate(i for i, _, b in pieces if b == len(prompts[i])):
                    last[i] = logits[row]
            for i, row in last.items():                      # (only now: steps of single tokens leave their logits in the same buffer)
                step.logits[i * K].copy_(row)
            own = sum(beam_pages(len(p), q.limit) for p, q in zip(prompts, searches)) * K
            for g, group in enumerate(cache.groups):
                for _ in range(own):
                    mine[g].append(group.pool.take())
            pages = [[g.pages[s] for s in heads] for g in cache.groups]
            if cache.groups:
                step.begin(slots, [len(p) for p in prompts], pages, mine, spare, stop)
            else:                                            # pages of no storage: 0 spare, then the prompts', then the beams'
                step.begin(slots, [len(p) for p in prompts], [[[1 + r] for r in range(R)]], [list(range(1 + R, 1 + R + R * K))], [0], stop)
            torch.cuda.synchronize(engine.device)
            stats.prefill_tokens += sum(len(p) for p in prompts)
            stats.prefill_ms += (time.perf_counter() - t0) * 1e3
            t0 = time.perf_counter()
            self._search(step, searches, K, length_penalty, early_stopping, stats)
            stats.decode_ms += (time.perf_counter() - t0) * 1e3
        finally:
            # whatever ended the batch: wait for what is still in flight, then all that it holds comes back
            try:
                torch.cuda.synchronize(engine.device)
            finally:
                for group, pages in zip(cache.groups, mine):
                    for p in reversed(pages):
                        group.pool.give_back(p)
                for s in slots:
                    engine.free_slot(s)
                for group, p in zip(cache.groups, spare):
                    group.pool.give_back(p)

    def _search(self, step: _BeamStep, searches: List[_Search], K: int, length_penalty: float, early_stopping: bool, stats) -> None:
        """Steps until every request is done.  A step is launched before the host has read what the one before chose; a request that turns out
        to be done had its rows computed once in vain."""
        R, N = step.R, step.R * K
        over = [False] * R                                   # rows already go on without a beam
        step.choose()
        handle, launched = self._fetch(step), 1              # tokens chosen so far, by what was launched
        while True:
            for r, q in enumerate(searches):
                if not over[r] and (q.done or launched >= q.limit):
                    step.end_request(r)
                    over[r] = True
            following = None
            if not all(over):
                step.run()
                following = self._fetch(step)
                launched += 1
            self._take(handle, searches, N, K, length_penalty, early_stopping, stats)
            if following is None or all(q.done for q in searches):
                return
            handle = following

    def _fetch(self, step: _BeamStep):
        n = step.result.numel()
        if len(self.staging) < 3 or self.staging[0].numel() < n:
            torch.cuda.synchronize(self.engine.device)
            self.staging = [torch.zeros(n, dtype=torch.int32, pin_memory=True) for _ in range(3)]
        to = self.staging[0][:n]
        self.staging.append(self.staging.pop(0))
        to.copy_(step.result, non_blocking=True)             # (a copy between two steps: kernels of the next wait for all of this one)
        done = torch.cuda.Event()
        done.record()
        return to, done

    def _take(self, handle, searches: List[_Search], N: int, K: int, length_penalty: float, early_stopping: bool, stats) -> None:
        values, done = handle
        done.synchronize()
        values = values.numpy()
        if values[6 * N:].any():
            raise CacheFull(f"{int(values[6 * N:].sum())} pages are missing for a step of {N} beams")
        parents, tokens, ended_parents, _ = (values[i * N: (i + 1) * N].reshape(-1, K).tolist() for i in range(4))
        scores, ended_scores = (values[i * N: (i + 1) * N].view(np.float32).reshape(-1, K).tolist() for i in (4, 5))
        for r, q in enumerate(searches):
            if not q.done:
                take_step(q, parents[r], tokens[r], scores[r], ended_parents[r], ended_scores[r], K, length_penalty, early_stopping)
                if len(q.tokens) > 1:
                    stats.decode_tokens += 1
        if any(len(q.tokens) > 1 for q in searches):
            stats.decode_steps += 1
