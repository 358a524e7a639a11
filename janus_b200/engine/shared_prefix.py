"""Generation for a batch of requests that begin with the same tokens, several tokens a request and step.

The prefix runs once and its pages lie once in the cache; every request's table of pages begins with them.  A step brings, for
each request, its last token and a few drafted ones; the index tables are made on the device (`ops.step_tables`), attention reads
the prefix once for all requests (`ops.attention_prefix`), and the step's logits verify the drafts (`ops.verify_drafts`): what a
request gets follows the target model's distribution (at temperature 0: its argmax), whatever was drafted.

The reference runs one token per row and step and each row's whole prompt
(crates/janus-engine/src/model/transformer/generation.rs:673-876); its sampler knows no drafts.
"""
from __future__ import annotations

import itertools
import time
from dataclasses import dataclass, field
from typing import Callable, Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

from ..cache import PAGE_SIZE, CacheFull, GroupStepView
from ..kernels import ops
from ..parts.attention import GQAttention
from .generate import GenerationStats, plan_prompt_steps
from .step import Engine, StepContext, StepEntry, StepError


@dataclass
class SharedPrefixStats(GenerationStats):
    drafted: int = 0            # drafted tokens that were verified
    accepted: int = 0           # ... and kept


class LookupDrafter:
    """Drafts for one request from its own text: the tokens that followed the last time its last two tokens stood there."""

    def __init__(self, tokens: Sequence[int], before: Optional["LookupDrafter"] = None):
        """`before`: a drafter of the text in front of `tokens`, whose places are looked up where its own have no answer (requests behind
        one prefix share the prefix's)."""
        self.tokens: List[int] = list(before.tokens) if before is not None else []
        self.seen: Dict[Tuple[int, int], int] = {}       # a pair -> the place behind its latest occurrence but the last
        self.seen_before = before.seen if before is not None else {}
        self.extend(tokens)

    def extend(self, tokens: Sequence[int]) -> None:
        for t in tokens:
            if len(self.tokens) >= 2:
                self.seen[(self.tokens[-2], self.tokens[-1])] = len(self.tokens)
            self.tokens.append(int(t))

    def draft(self, most: int) -> List[int]:
        if len(self.tokens) < 2:
            return []
        pair = (self.tokens[-2], self.tokens[-1])
        at = self.seen.get(pair, self.seen_before.get(pair))
        return self.tokens[at: at + most] if at is not None else []


def pages_behind_prefix(prefix_len: int, prompt_len: int, max_tokens: int, drafts: int, shared: int, longest: Optional[int] = None) -> int:
    """Pages of its own that a request takes at most, behind `shared` whole pages of the prefix.  (The last token is never fed back;
    drafts behind it are.)"""
    held = prefix_len + prompt_len + max(0, max_tokens - 1) + drafts
    return -(-(held if longest is None else min(longest, held)) // PAGE_SIZE) - shared


def room_for_batch(prefix_len: int, prompt_lens: Sequence[int], max_tokens: int, drafts: int, batch_size: int) -> int:
    """Cache tokens, in whole pages, with room for the prefix once and beside it any `batch_size` of the requests (none of whose prompts is
    empty)."""
    shared = prefix_len // PAGE_SIZE
    own = sorted((pages_behind_prefix(prefix_len, n, max_tokens, drafts, shared) for n in prompt_lens), reverse=True)
    return (shared + sum(own[:batch_size])) * PAGE_SIZE


def _random(seed: int, request: int) -> np.random.Generator:
    """A request's random numbers.  A negative seed stands for its 64 bits, as the plain generation's sampler takes it."""
    return np.random.default_rng((int(seed) if seed >= 0 else int(seed) % (1 << 64), request))


@dataclass
class _Request:
    index: int
    own: List[int]              # its tokens that are not in the cache yet: the prompt, then the token it ended with
    length: int                 # tokens in the cache
    row: int                    # row of the last step's table, -1 before the first
    drafter: object
    random: np.random.Generator
    limit: int                  # tokens that its pages have room for
    held: int                   # pages of its row, the shared ones among them
    drafts: List[int] = field(default_factory=list)    # of the step that is running


class SharedPrefixRunner:
    """Runs an engine's model by the steps described above.  The model's mixers are grouped-query attention without a window,
    all of one cache group (the Llama decoder)."""

    def __init__(self, engine: Engine):
        model, cache = engine.model, engine.cache
        mixers = [part for objs in model._layer_part_objs for part in objs.values() if hasattr(part, "cache_spec")]
        if len(cache.groups) != 1 or cache.states or any(type(m) is not GQAttention or m.window for m in mixers):
            raise ValueError("a shared prefix needs a model whose mixers are all grouped-query attention over one kind of cache, "
                             "without a window")
        self.engine, self.model, self.group = engine, model, cache.groups[0]
        self.device = engine.device

    def generate(self, prefix: Sequence[int], prompts: Sequence[Sequence[int]], max_tokens: int, stop: Sequence[int] = (),
                 drafts: int = 4, temperature: float = 0.0, seed: int = 0, batch_size: Optional[int] = None,
                 callback: Optional[Callable[[int, int], bool]] = None, drafter: Callable[[List[int]], object] = LookupDrafter):
        """Returns (tokens per request, finish reasons, stats).  `drafter(tokens)` makes an object with `draft(most)` and
        `extend(tokens)` for a request."""
        if drafts < 0 or max_tokens < 0 or not 0.0 <= temperature < float("inf"):
            raise ValueError(f"drafts {drafts}, max_tokens {max_tokens} and temperature {temperature} cannot be negative")
        prefix = [int(t) for t in prefix]
        prompts = [[int(t) for t in p] for p in prompts]
        V = self.model.vocab_size
        if any(not 0 <= t < V for t in prefix):
            raise StepError(f"a token id of the prefix is outside the vocabulary of {V}")
        for i, p in enumerate(prompts):
            if not prefix and not p:
                raise ValueError(f"prompt {i} is empty")
            if len(prefix) + len(p) > self.engine.max_seq_len:
                raise StepError(f"prompt {i} has {len(prefix) + len(p)} tokens with the prefix, the longest sequence allowed is "
                                f"{self.engine.max_seq_len}")
            if any(not 0 <= t < V for t in p):
                raise StepError(f"a token id of prompt {i} is outside the vocabulary of {V}")
        outputs: List[List[int]] = [[] for _ in prompts]
        reasons = ["length"] * len(prompts)
        stats = SharedPrefixStats(requests=len(prompts))
        if max_tokens == 0 or not prompts:
            return outputs, reasons, stats
        # whole pages are shared, and every request keeps a token of its own; the rest of the prefix goes with each prompt
        shared = len(prefix) // PAGE_SIZE
        while shared and shared * PAGE_SIZE == len(prefix) and any(not p for p in prompts):
            shared -= 1
        if drafter is LookupDrafter:
            before = LookupDrafter(prefix)
            begin = lambda prompt: LookupDrafter(prompt, before)      # noqa: E731
        else:
            begin = lambda prompt: drafter(prefix + prompt)           # noqa: E731
        slot = self.engine.alloc_slot()
        try:
            self._run_prefix(slot, prefix[: shared * PAGE_SIZE], stats)
            pending = list(range(len(prompts)))
            while pending:
                pending = self._run_batch(slot, shared, prefix, prompts, pending, outputs, reasons, max_tokens, set(int(t) for t in stop),
                                          drafts, temperature, seed, batch_size or len(prompts), callback, begin, stats)
        finally:
            torch.cuda.synchronize(self.device)
            self.engine.free_slot(slot)
        ops.check_kernel_status(self.device)
        return outputs, reasons, stats

    def _run_prefix(self, slot: int, tokens: List[int], stats) -> None:
        t0 = time.perf_counter()
        most = self.engine.options.max_step_tokens or len(tokens)
        for a in range(0, len(tokens), max(1, most)):
            self.engine.step([StepEntry(slot, tokens[a: a + most])])
        torch.cuda.synchronize(self.device)
        stats.prefill_ms += (time.perf_counter() - t0) * 1e3
        stats.prefill_tokens += len(tokens)

    def _run_batch(self, slot, shared, prefix, prompts, pending, outputs, reasons, max_tokens, stop, drafts, temperature, seed,
                   batch_size, callback, drafter, stats) -> List[int]:
        """One batch from its prompts to its last token; returns the requests that are left."""
        group, longest = self.group, self.engine.max_seq_len
        rest = prefix[shared * PAGE_SIZE:]
        chosen, own_pages, width = [], 0, 0
        for r in pending:
            pages = pages_behind_prefix(len(prefix), len(prompts[r]), max_tokens, drafts, shared, longest)
            if len(chosen) == batch_size or own_pages + pages > group.pool.n_free:
                break
            chosen.append(r)
            own_pages, width = own_pages + pages, max(width, shared + pages)
        if not chosen:
            raise CacheFull(f"request {pending[0]} needs {pages} pages of {PAGE_SIZE} tokens behind the shared prefix, the cache has "
                            f"{group.pool.n_free} free ones")
        live = []
        for r in chosen:
            own = rest + prompts[r]
            held = min(longest, len(prefix) + len(prompts[r]) + max_tokens - 1 + drafts)
            live.append(_Request(r, own, shared * PAGE_SIZE, -1, drafter(prompts[r]), _random(seed, r), held,
                                 shared))
        mine = [group.pool.take() for _ in range(own_pages)]
        stats.batches += 1
        try:
            new = lambda *shape: torch.empty(shape, dtype=torch.int32, device=self.device)      # noqa: E731
            prefix_pages = torch.tensor(group.pages[slot][:shared], dtype=torch.int32).to(self.device)
            state = dict(table=new(0, width), held=new(0), free_pages=torch.tensor(mine, dtype=torch.int32).to(self.device),
                         n_free=torch.tensor([own_pages], dtype=torch.int32).to(self.device))
            first = True
            while live:
                t0 = time.perf_counter()
                if first:
                    # prompts in as many steps as the limit asks for; every request is in every one of them (the pages of a row
                    # that nobody goes on with are given back), with no tokens where its turn is over or still to come
                    tokens: List[List[int]] = [[] for _ in live]
                    for pieces in plan_prompt_steps([len(q.own) for q in live], self.engine.options.max_step_tokens):
                        brought, judged = [[] for _ in live], [0] * len(live)
                        for i, begin, end in pieces:
                            brought[i], judged[i] = live[i].own[begin:end], int(end == len(live[i].own))
                        state, got = self._step(live, brought, judged, state, prefix_pages, shared, width, temperature)
                        tokens = [t + more for t, more in zip(tokens, got)]
                else:
                    for q in live:
                        room = q.limit - q.length - len(q.own)
                        wanted = max_tokens - len(outputs[q.index]) - 1
                        q.drafts = self._drafts(q.drafter, max(0, min(drafts, room, wanted)))
                    brought = [q.own + q.drafts for q in live]
                    state, tokens = self._step(live, brought, [len(t) for t in brought], state, prefix_pages, shared, width, temperature)
                still = []
                for q, got in zip(live, tokens):
                    n = len(got) - 1
                    stats.drafted += len(q.drafts)
                    stats.accepted += n
                    q.length -= len(q.drafts) - n       # refused drafts
                    q.own = [got[-1]]
                    if self._accept(q, got, outputs, reasons, max_tokens, stop, callback, longest):
                        still.append(q)
                    if not first:
                        stats.decode_tokens += n + 1
                if first:
                    stats.prefill_tokens += sum(len(rest) + len(prompts[r]) for r in chosen)
                    stats.prefill_ms += (time.perf_counter() - t0) * 1e3
                else:
                    stats.decode_steps += 1
                    stats.decode_ms += (time.perf_counter() - t0) * 1e3
                live, first = still, False
        finally:
            torch.cuda.synchronize(self.device)
            for p in mine:
                group.pool.give_back(p)
        return pending[len(chosen):]

    def _drafts(self, drafter, most: int) -> List[int]:
        """What a drafter says, no more than it was asked for (the request's pages have no room for more), up to the first id outside
        the vocabulary: verification would refuse that one and with it all behind, but the step looks embeddings up before it
        verifies."""
        tokens: List[int] = []
        for t in drafter.draft(most):
            if len(tokens) == most or not 0 <= int(t) < self.model.vocab_size:
                break
            tokens.append(int(t))
        return tokens

    @staticmethod
    def _accept(q, got, outputs, reasons, max_tokens, stop, callback, longest) -> bool:
        """Take a step's tokens one by one, as the plain generation loop does; True if the request goes on."""
        out = outputs[q.index]
        for t in got:
            if t in stop:
                reasons[q.index] = "stop"
                return False
            out.append(t)
            if callback is not None and callback(q.index, t) is False:
                reasons[q.index] = "stop"
                return False
            if len(out) >= max_tokens:
                return False
        q.drafter.extend(got)
        return q.length + 1 <= longest

    def _step(self, live: List[_Request], brought: List[List[int]], judged: List[int], state, prefix_pages, shared: int, width: int,
              temperature: float):
        """One step: request i brings the tokens brought[i], and the logits behind its last judged[i] tokens verify the drafts among them
        and give one more (none behind a prompt's part that is not its last).  Returns the next state and each request's new tokens;
        the requests' lengths, rows and pages are those after the step, refused drafts still counted."""
        B = len(live)
        lens = [len(t) for t in brought]
        T = sum(lens)
        # a step whose tokens have no page must not run: its tables would send them to a row in front of the cache
        held = [max(q.held, -(-(q.length + n) // PAGE_SIZE)) for q, n in zip(live, lens)]
        lacking = sum(held) - B * shared - state["free_pages"].shape[0]
        if lacking > 0 or max(held) > width:
            raise CacheFull(f"a step of {T} tokens needs {max(lacking, max(held) - width)} pages more than its requests have room for")
        for q, n in zip(live, held):
            q.held = n
        all_tokens, at = np.fromiter(itertools.chain.from_iterable(brought), np.int64, T), np.arange(T)
        wanted = at[at >= np.repeat(np.cumsum(lens) - judged, lens)]
        W = len(wanted)
        starts = np.concatenate([[0], np.cumsum(judged)])
        u = np.concatenate([q.random.random(1 + n) if n else np.zeros(1) for q, n in zip(live, judged)]).astype(np.float32)
        u = np.minimum(u, np.float32(1.0 - 2.0 ** -24))            # (rounding may have made it one)
        first_u = starts[:-1] + np.arange(B)                       # a request's numbers: one for its draw, one for each row's test
        tests = np.delete(u, first_u)
        parts = [[q.length for q in live], lens, [q.row for q in live], all_tokens, wanted, all_tokens[wanted], starts, u[first_u].view(np.int32),
                 tests.view(np.int32)]
        sizes = [len(p) for p in parts]
        offsets = np.concatenate([[0], np.cumsum([(n + 3) // 4 * 4 for n in sizes])])
        host = np.zeros(offsets[-1], dtype=np.int32)
        for p, at in zip(parts, offsets):
            host[at: at + len(p)] = p
        dev = torch.from_numpy(host).pin_memory().to(self.device, non_blocking=True)
        lengths, fresh, rows, ids, want, verified, starts, u_draw, u_accept = (dev[a: a + n] for a, n in zip(offsets, sizes))

        new = lambda *shape: torch.empty(shape, dtype=torch.int32, device=self.device)      # noqa: E731
        made = dict(q_start=new(B + 1), kv_len=new(B), positions=new(T), token_seq=new(T), dest_rows=new(T), table=new(B, width), held=new(B),
                    free_pages=new(state["free_pages"].shape[0]), n_free=new(1), missing=new(1))
        ops.step_tables(lengths, fresh, rows, state["table"], state["held"], prefix_pages, state["free_pages"], state["n_free"],
                        **made, page_size=PAGE_SIZE)
        engine = self.engine
        ctx = StepContext()
        ctx.n_tokens, ctx.n_seqs, ctx.max_q_len = T, B, max(lens)
        ctx.max_kv_len_bound = max(q.length + n for q, n in zip(live, lens))
        ctx.token_ids, ctx.positions, ctx.token_seq = ids, made["positions"], made["token_seq"]
        ctx.q_start, ctx.kv_len = made["q_start"], made["kv_len"]
        ctx.groups = [GroupStepView(made["dest_rows"], made["table"], PAGE_SIZE)]
        ctx.workspace, ctx.cache, ctx.dtype = engine.workspace, engine.cache, engine.dtype
        ctx.prefix_pages = prefix_pages
        logits = torch.empty((W, self.model.vocab_size), dtype=torch.float32, device=self.device)
        self.model.forward(ctx, want, logits)

        for b, (q, n) in enumerate(zip(live, lens)):
            q.length, q.row = q.length + n, b
        tokens_of = [[] for _ in live]
        if W:
            most = max(judged)
            result = new(B, 1 + most)
            accepted, tokens, kept = new(B), new(B, most), new(B)
            logprobs = torch.empty((B, most), dtype=torch.float32, device=self.device)
            ops.verify_drafts(logits, verified, starts, made["kv_len"], accepted, tokens, logprobs, kept, temperature,
                              u_accept.view(torch.float32), u_draw.view(torch.float32), None, engine.workspace)
            result[:, 0].copy_(accepted)
            result[:, 1:].copy_(tokens)
            tokens_of = [row[1: 2 + row[0]] if n else [] for row, n in zip(result.cpu().tolist(), judged)]
        missing = int(made["missing"])
        if missing:
            raise CacheFull(f"{missing} pages are missing for a step of {T} tokens")
        return made, tokens_of
