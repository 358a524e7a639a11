"""Generation behind a shared prefix without a device: the real runner over stand-ins for the engine and the three faces, which answer
on the host (the index tables and the verification by their definitions) and note every step's tokens.  The model's next token
goes by the last one alone, so what has to come out is known.
"""
import types

import pytest
import torch

from janus_b200.cache import PAGE_SIZE, CacheFull
from janus_b200.cache.pages import PagePool
from janus_b200.engine import shared_prefix
from janus_b200.engine.shared_prefix import SharedPrefixRunner
from janus_b200.engine.step import StepError
from janus_b200.kernels import ops
from test_shared_prefix import tables_oracle, verify_oracle

V = 50


def next_token(t):
    return (3 * t + 1) % V


def continuation(last, n):
    out = []
    for _ in range(n):
        last = next_token(last)
        out.append(last)
    return out


class Host:
    """A runner whose steps are noted in `steps` (token ids, positions, cache rows, rows of the table)."""

    def __init__(self, monkeypatch, pages=64, longest=4096, max_step_tokens=None):
        self.steps, self.prefix_steps = [], []
        pool, held = PagePool(pages), []

        def step(entries):
            (e,) = entries
            self.prefix_steps.append(len(e.tokens))
            need = -(-sum(self.prefix_steps) // PAGE_SIZE)
            while len(held) < need:
                held.append(pool.take())

        def free_slot(slot):
            while held:
                pool.give_back(held.pop())

        def forward(ctx, want, logits):
            ids, rows = ctx.token_ids.tolist(), ctx.groups[0].dest_rows.tolist()
            assert all(0 <= t < V for t in ids), ids
            assert min(rows) >= 0 and len(set(rows)) == len(rows), rows
            assert max(ctx.positions.tolist()) < longest
            self.steps.append(types.SimpleNamespace(ids=ids, positions=ctx.positions.tolist(), rows=rows, most=ctx.max_q_len,
                                                    lengths=ctx.kv_len.tolist(), bound=ctx.max_kv_len_bound))
            logits[:] = -1.0
            for i, w in enumerate(want.tolist()):
                logits[i, next_token(ids[w])] = 30.0

        group = types.SimpleNamespace(pool=pool, pages=[held])
        engine = types.SimpleNamespace(max_seq_len=longest, options=types.SimpleNamespace(max_step_tokens=max_step_tokens), workspace=None,
                                       cache=None, dtype=torch.float32, alloc_slot=lambda: 0, free_slot=free_slot, step=step)
        runner = SharedPrefixRunner.__new__(SharedPrefixRunner)
        runner.engine, runner.group, runner.device = engine, group, torch.device("cpu")
        runner.model = types.SimpleNamespace(vocab_size=V, forward=forward)
        self.runner, self.pool = runner, pool
        monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
        monkeypatch.setattr(torch.Tensor, "pin_memory", lambda t: t)
        monkeypatch.setattr(ops, "check_kernel_status", lambda device: None)
        monkeypatch.setattr(ops, "step_tables", self._tables)
        monkeypatch.setattr(ops, "verify_drafts", self._verify)

    @staticmethod
    def _tables(lengths, new, rows, old_table, old_held, prefix, old_free, old_n_free, *, page_size, **out):
        got = tables_oracle(lengths.tolist(), new.tolist(), rows.tolist(), old_table.tolist(), old_held.tolist(), prefix.tolist(),
                            old_free.tolist(), int(old_n_free), out["table"].shape[1], out["positions"].shape[0], page_size)
        for k, v in out.items():
            v.copy_(torch.tensor(got[k], dtype=torch.int32).reshape(v.shape))

    @staticmethod
    def _verify(logits, tokens, q_start, kv_len, accepted, out, logprobs, kept, heat, u_accept, u_draw, probs, workspace):
        got = verify_oracle(dict(logits=logits, tokens=tokens, q_start=q_start, kv_len=kv_len, heat=heat, width=out.shape[1], probs=probs,
                                 u_accept=u_accept, u_draw=u_draw))
        for mine, theirs in zip((accepted, out, logprobs, kept), got):
            mine.copy_(torch.as_tensor(theirs).reshape(mine.shape))

    def generate(self, prefix, prompts, n, **more):
        out, reasons, stats = self.runner.generate(prefix, prompts, n, **more)
        self.pool.check()
        assert self.pool.n_held == 0
        return out, reasons, stats


def drafting(answer):
    """A drafter whose answer is answer(tokens so far, how many were asked for)."""
    class Drafter:
        def __init__(self, tokens):
            self.tokens = list(tokens)

        def extend(self, tokens):
            self.tokens += tokens

        def draft(self, most):
            return answer(self.tokens, most)
    return Drafter


@pytest.mark.parametrize("prefix", [0, 5, 64, 150])
def test_generation_on_the_host_gives_what_the_model_says(monkeypatch, prefix):
    prompts = [[7, 8], [9], [1, 2, 3] * 30]
    for drafter in (drafting(lambda t, most: continuation(t[-1], most)), drafting(lambda t, most: [3] * most), drafting(lambda t, most: [])):
        host = Host(monkeypatch)
        out, reasons, stats = host.generate([4] * prefix, prompts, 20, drafts=3, drafter=drafter)
        assert out == [continuation(p[-1], 20) for p in prompts] and reasons == ["length"] * 3
        assert stats.prefill_tokens == prefix // PAGE_SIZE * PAGE_SIZE + sum(prefix % PAGE_SIZE + len(p) for p in prompts)


@pytest.mark.parametrize("bad", [-1, V, 2 ** 31 - 1, -2 ** 31, 2 ** 40])
def test_a_draft_outside_the_vocabulary_ends_the_drafts(monkeypatch, bad):
    """Verification refuses such a draft; the step, which reads its embedding first, must not see it."""
    host = Host(monkeypatch)
    drafter = drafting(lambda t, most: (continuation(t[-1], 2) + [bad] + [0] * most)[:most])
    out, _, stats = host.generate([4] * 70, [[7], [9, 2]], 12, drafts=4, drafter=drafter)
    assert out == [continuation(7, 12), continuation(2, 12)]
    assert stats.accepted == stats.drafted > 0
    assert max(s.most for s in host.steps[1:]) == 3


@pytest.mark.parametrize("right", [True, False])
def test_more_drafts_than_were_asked_for_are_left_out(monkeypatch, right):
    """They would pass the request's pages and the longest length."""
    asked = []

    def answer(tokens, most):
        asked.append(most)
        return continuation(tokens[-1], 200) if right else [3] * 200
    host = Host(monkeypatch, pages=1 + 2 * 2, longest=64 + 70)
    out, reasons, stats = host.generate([4] * 64, [[7, 8, 9], [5]], 60, drafts=3, drafter=drafting(answer))
    assert out == [continuation(9, 60), continuation(5, 60)] and reasons == ["length"] * 2
    assert max(s.most for s in host.steps[1:]) == 4 and stats.drafted <= sum(asked)
    host = Host(monkeypatch, longest=64 + 70)                       # up to the longest length
    out, reasons, _ = host.generate([4] * 64, [[7, 8, 9]], 999, drafts=5, drafter=drafting(answer))
    assert out == [continuation(9, 70 - 3 + 1)]


@pytest.mark.parametrize("prompts,pages", [([[7, 8, 9]], 2), ([[7], [8], [9, 9]], 4)])
def test_a_step_without_pages_for_its_tokens_is_not_launched(monkeypatch, prompts, pages):
    """Should anything count wrong: the request's row is too narrow, or the others' pages would go."""
    host = Host(monkeypatch, pages=pages)
    host.runner._drafts = lambda drafter, most: [3] * (200 if len(prompts) == 1 else 64)
    with pytest.raises(CacheFull, match="pages more"):
        host.generate([4] * 64, prompts, 30, drafts=3)
    assert len(host.steps) == 1 and host.pool.n_held == 0


@pytest.mark.parametrize("most", [1, 7, 64, 100, 1000, None, 0])
@pytest.mark.parametrize("prefix", [0, 70, 128])
def test_prompts_run_in_steps_of_at_most_the_limit(monkeypatch, most, prefix):
    host = Host(monkeypatch, max_step_tokens=most)
    prompts = [[7] * 40 + [8], [9], [1, 2, 3] * 30, [5] * 64, [11]]
    out, reasons, stats = host.generate([4] * prefix, prompts, 9, drafts=3, drafter=drafting(lambda t, n: continuation(t[-1], n)))
    assert out == [continuation(p[-1], 9) for p in prompts] and reasons == ["length"] * 5
    brought = sum(prefix % PAGE_SIZE + len(p) for p in prompts)
    limit = most or brought
    steps = host.steps[:-(-brought // limit)]
    assert all(len(s.ids) <= limit for s in steps) and sum(len(s.ids) for s in steps) == brought
    assert stats.prefill_tokens == prefix // PAGE_SIZE * PAGE_SIZE + brought
    assert max(host.prefix_steps, default=0) <= (most or prefix)
    for s in host.steps:
        assert s.bound >= max(s.lengths)


def test_draws_do_not_go_by_how_prompts_were_cut(monkeypatch):
    prompts = [[7] * 40 + [8], [9], [1, 2, 3] * 30]
    more = dict(drafts=2, temperature=9.0, seed=5, drafter=drafting(lambda t, n: [3] * n))
    want = Host(monkeypatch).generate([4] * 70, prompts, 9, **more)[0]
    assert Host(monkeypatch, max_step_tokens=13).generate([4] * 70, prompts, 9, **more)[0] == want
    assert any(w != continuation(p[-1], 9) for w, p in zip(want, prompts))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_prompts_cut_in_steps_give_the_same_tokens(tmp_path, dtype):
    import janus_b200
    from helpers import BF16_TOL, TINY_A, make_model_dir, random_tokens
    folder = make_model_dir(TINY_A, str(tmp_path), seed=2, dtype=dtype)
    prefix = random_tokens(70, 256, 5)
    prompts = [random_tokens(n, 256, n) for n in (1, 29, 2, 17, 40)]
    out = []
    for most in (11, 64, 32768):
        model = janus_b200.load(folder, dtype=dtype, max_tokens=2048, max_step_tokens=most)
        tokens, counts, forward = [], [], model.engine.model.forward
        model.engine.model.forward = lambda ctx, want, logits: (counts.append(ctx.n_tokens), forward(ctx, want, logits))[1]
        tokens, _ = model.generate_shared(prefix, prompts, max_tokens=10, drafts=3, ignore_eos=True)
        assert max(counts) <= max(most, 5 * 4) and counts[0] <= most
        out.append(tokens)
        want, _ = model.generate([prefix + p for p in prompts], max_tokens=10, ignore_eos=True)
        if dtype == "float32":
            assert tokens == want
    if dtype == "bfloat16":              # sums in another order: a token may differ where two logits nearly tie
        import plain_llama as P
        cfg, w = P.read_model_dir(folder)
        for tokens in out:
            for p, o in zip(prompts, tokens):
                logits = P.forward(cfg, w, prefix + p + o)
                for j, t in enumerate(o):
                    row = logits[len(prefix) + len(p) - 1 + j]
                    assert float(row.max() - row[t]) <= BF16_TOL * float(row.abs().max())


def run_command(monkeypatch, tmp_path, args):
    """The command line over a model that notes how it was asked for and what it was called with."""
    import json
    import janus_b200
    from janus_b200 import cli
    asked = {}

    class Model:
        def generate_shared(self, prefix, prompts, **more):
            asked.update(prefix=prefix, prompts=prompts, **{f"call_{k}": v for k, v in more.items()})
            return [[1]] * len(prompts), ["length"] * len(prompts), shared_prefix.SharedPrefixStats()

        def generate(self, prompts, **more):
            return self.generate_shared(None, prompts, **more)

    def load_random(config, **more):
        asked.update(more)
        return Model()
    monkeypatch.setattr(janus_b200, "load_random", load_random)
    (tmp_path / "config.json").write_text(json.dumps({}))
    assert cli.main([str(tmp_path)] + args + ["--random-weights", "--json"]) == 0
    return asked


@pytest.mark.parametrize("prefix,lens,batch,n,drafts", [(8192, [100] * 64, 64, 50, 4), (5, [3], 1, 1, 0), (64, [1, 200, 7], 2, 65, 9),
                                                         (191, [64] * 5, 3, 1, 0), (1, [1, 1], 9, 0, 4)])
def test_command_line_makes_room_for_the_prefix_once(monkeypatch, tmp_path, prefix, lens, batch, n, drafts):
    """What it makes room for is what the requests of a batch hold: they run together, and a page less would not do."""
    prompts = [[7 + i % 9] * m for i, m in enumerate(lens)]
    text = [" ".join(map(str, p)) for p in prompts]
    asked = run_command(monkeypatch, tmp_path, text + ["--shared-prefix", " ".join(["4"] * prefix), "--drafts", str(drafts), "--max-tokens", str(n),
                                                       "--batch-size", str(batch), "--max-step-tokens", "777"])
    assert asked["prefix"] == [4] * prefix and asked["prompts"] == prompts and asked["call_drafts"] == drafts
    assert asked["max_step_tokens"] == 777 and asked["call_batch_size"] == min(batch, len(lens))
    pages = asked["max_tokens"] // PAGE_SIZE
    assert asked["max_tokens"] % PAGE_SIZE == 0
    own = sorted((-(-(prefix + m + max(0, n - 1) + drafts) // PAGE_SIZE) - prefix // PAGE_SIZE for m in lens), reverse=True)
    assert pages == prefix // PAGE_SIZE + sum(own[:batch])
    if n == 0:
        return
    drafter = drafting(lambda t, most: [3] * most)
    host = Host(monkeypatch, pages=pages, longest=1 << 20)
    out, _, stats = host.generate([4] * prefix, prompts, n, drafts=drafts, drafter=drafter, batch_size=asked["call_batch_size"])
    assert out == [continuation(p[-1], n) for p in prompts] and stats.batches == -(-len(lens) // batch)


def test_command_line_without_a_prefix_is_as_it_was(monkeypatch, tmp_path):
    asked = run_command(monkeypatch, tmp_path, ["1 2 3", "4", "5 6", "--max-tokens", "63", "--batch-size", "2"])
    assert asked["max_tokens"] == 128 + 64 and asked["max_slots"] == 2 and asked["prefix"] is None


@pytest.mark.gpu
def test_command_line_behind_a_prefix(tmp_path, capsys):
    import json
    import janus_b200
    from helpers import TINY_A, make_model_dir, random_tokens
    from janus_b200 import cli
    folder = make_model_dir(TINY_A, str(tmp_path), seed=2, dtype="float32")
    prefix, prompts = random_tokens(70, 256, 5), [random_tokens(n, 256, n) for n in (3, 20, 1)]
    text = [" ".join(map(str, p)) for p in prompts]
    assert cli.main([folder] + text + ["--shared-prefix", " ".join(map(str, prefix)), "--drafts", "3", "--max-tokens", "12", "--dtype", "fp32",
                                       "--ignore-eos", "--json"]) == 0
    got = json.loads(capsys.readouterr().out.strip().splitlines()[-1])["tokens"]
    want, _ = janus_b200.load(folder, dtype="float32", max_tokens=1024).generate([prefix + p for p in prompts], max_tokens=12, ignore_eos=True)
    assert got == want


def test_any_whole_number_is_a_seed(monkeypatch):
    """As for the plain generation; a seed repeats its numbers, another one has others."""
    more = dict(drafts=2, temperature=9.0, drafter=drafting(lambda t, n: [3] * n))
    seen = [Host(monkeypatch).generate([4] * 70, [[7], [8]], 20, seed=seed, **more)[0] for seed in (-1, -1, -2, 0, 1, 2 ** 40)]
    assert seen[0] == seen[1] and all(a != b for i, a in enumerate(seen[1:]) for b in seen[2 + i:])


def test_the_prefix_is_looked_through_once_for_all_requests(monkeypatch):
    """Its pairs of tokens lie in one table: a table of each request's own made 256 requests behind 16,384 tokens wait for 1.5 s and took
    half a gigabyte of the host."""
    looked_at = []
    extend = shared_prefix.LookupDrafter.extend
    monkeypatch.setattr(shared_prefix.LookupDrafter, "extend", lambda self, tokens: (looked_at.append(len(tokens)), extend(self, tokens))[1])
    prompts = [[7 + i, 8] for i in range(30)]
    out, _, stats = Host(monkeypatch, pages=200).generate([4] * 1000, prompts, 30)
    assert out == [continuation(8, 30)] * 30 and stats.accepted > 0
    assert sum(looked_at) <= 1000 + 30 * (2 + 30)


def test_drafts_behind_a_shared_text_are_those_of_the_whole_text():
    import random
    rng = random.Random(5)
    for _ in range(400):
        text = lambda n: [rng.randrange(4) for _ in range(n)]      # noqa: E731
        prefix, prompt = text(rng.randrange(30)), text(rng.randrange(6))
        before = shared_prefix.LookupDrafter(prefix)
        whole, behind = shared_prefix.LookupDrafter(prefix + prompt), shared_prefix.LookupDrafter(prompt, before)
        other = shared_prefix.LookupDrafter(text(9), before)       # (another request does not change it)
        for _ in range(12):
            assert behind.draft(3) == whole.draft(3)
            more = text(rng.randrange(1, 4))
            whole.extend(more), behind.extend(more), other.extend(text(2))
        assert before.tokens == prefix


def test_the_prefix_is_checked_once(monkeypatch):
    """16,384 tokens for each of 256 requests took 0.15 s."""
    class Counted(int):
        looks = 0

        def __ge__(self, other):                 # 0 <= id
            Counted.looks += 1
            return int(self) >= other
    host = Host(monkeypatch)
    monkeypatch.setattr(shared_prefix, "int", lambda t: t if isinstance(t, Counted) else int(t), raising=False)
    with pytest.raises(StepError, match="prompt 19"):
        host.generate([Counted(4)] * 500, [[1]] * 19 + [[V]], 5)
    assert Counted.looks == 500
    with pytest.raises(StepError, match="prefix"):
        host.generate([4, V], [[1]], 5)
    with pytest.raises(StepError, match="prefix"):
        host.generate([-1], [[1]], 5)
    assert not host.steps and not host.prefix_steps
