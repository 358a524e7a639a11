"""The operators of beam search over a paged cache, each against its definition in 64 bits (`plain_beams.py`).

Tolerances.  A score is the beam's own plus a log-probability, rounded once to float32 (2^-24 of it).  The sum of exponentials is made of
float32 terms exp(d), d = x - max: d and its product with log2(e) are each within 2^-24 |d|, the power within 2^-22, short sums in float32
within 2^-22; weighted by the terms themselves |d| is at most the logarithm of the vocabulary plus 1, below 13 here: 26 / 2^24 + 2^-21 < 2.1e-6.
Whole numbers are equal; where rankings are compared, the smallest distance of two neighbours of different beams is above twice that.

Attention is sum(p v) / sum(p) with weights p (1 + d), |d| <= 2^-8 (their rounding to bfloat16), above and below: off by sum(p d (v - result)) /
sum(p), at most 2^-8 of the weighted mean of |v - result|, which is at most S + |result|, S the weighted mean of the values' magnitudes.  The
result's own rounding is 2^-8 of it: 2^-7 |result| + 2^-8 S together.  Scores are float32 sums over a head's numbers, whose errors (d 2^-24 of their
terms, below 2^-12 for scores below 30) and the rounding of the power change weights by less than 2^-11 of S.
"""
import math
import random

import pytest
import torch

import plain_beams as P
from janus_b200.engine.workspace import Workspace
from janus_b200.kernels import ops

gpu = pytest.mark.gpu
PAGE, NONE = 64, -math.inf
LSE_TOL = 2.1e-6


def ints(values, shape=None):
    t = torch.tensor(values, dtype=torch.int32, device="cuda")
    return t if shape is None else t.reshape(shape)


def empty(*shape, dtype=torch.int32):
    return torch.full(shape, 12345, dtype=dtype, device="cuda")


# -- which continuations go on -----------------------------------------------------------------------------------------
def run_select(logits, scores, stops, in_place=False):
    R, K = scores.shape
    scores = scores.float().cuda()
    out = dict(parents=empty(R, K), tokens=empty(R, K), next_scores=scores if in_place else empty(R, K, dtype=torch.float32),
               ended_parents=empty(R, K), ended_tokens=empty(R, K), ended_scores=empty(R, K, dtype=torch.float32))
    ops.beam_select(logits, scores, ints(list(stops)), **out, workspace=Workspace(torch.device("cuda")))
    return out


def check_select(logits, scores, stops, in_place=False, gap_needed=True):
    out = run_select(logits.cuda(), scores, stops, in_place)
    parents, tokens, nxt, ep, et, es, gap = P.select(logits.cpu(), scores, stops)
    if gap_needed:
        assert gap > 2 * LSE_TOL, "this seed's ranking is too close to call"
    assert out["parents"].tolist() == parents
    assert out["tokens"].tolist() == tokens
    assert out["ended_parents"].tolist() == ep and out["ended_tokens"].tolist() == et
    for got, want in ((out["next_scores"], nxt), (out["ended_scores"], es)):
        got, want = got.cpu().double(), torch.tensor(want, dtype=torch.float64)
        assert torch.equal(got == NONE, want == NONE)
        fine = want > NONE
        assert torch.all((got - want)[fine].abs() <= LSE_TOL + 2.0 ** -24 * want[fine].abs())


def random_logits(rows, vocab, seed, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * spread
    return x, g


@gpu
@pytest.mark.parametrize("R, K, V, S", [(1, 1, 1, 0), (1, 1, 5, 1), (1, 4, 7, 2), (2, 3, 4095, 1), (3, 4, 4096, 0), (2, 5, 4097, 3), (1, 8, 32000, 1),
                                        (3, 2, 20001, 2), (1, 32, 9001, 32), (2, 16, 12290, 1), (40, 2, 1003, 1), (300, 3, 130, 1)])
def test_select_small_to_large(R, K, V, S):
    x, g = random_logits(R * K, V, 17 * R + K + V)
    scores = -torch.rand(R, K, generator=g) * 3.0 - 1.0
    stops = torch.randperm(V, generator=g)[:S].tolist()
    for s in stops:
        x[:, s] += 9.0
    check_select(x, scores, stops)


@gpu
@pytest.mark.parametrize("V", [1001, 8192, 50002, 128256])
def test_select_equal_logits_lowest_token_first(V):
    x, g = random_logits(4, V, V)
    x = (x * 2).round() / 2                         # many are equal, the largest too
    x[1] = 0.25                                     # all of a row are
    x[2, ::7] = 0.0
    x[2, 1::7] = -0.0                               # equal to 0
    check_select(x, torch.tensor([[0.0, -0.3], [-0.7, -0.1]]), [0, V - 1])


@gpu
def test_select_rising_and_falling_rows():
    """Every number passes all in front of it, or none does."""
    V = 70000
    up = torch.arange(V, dtype=torch.float32) * 1e-4
    check_select(torch.stack([up, up.flip(0), up * -3, up * 0.5]), torch.tensor([[0.0, -1.01, -0.4, -0.2]]), [V - 2, 3])


@gpu
def test_select_dead_beams_and_masked_rows():
    V = 5000
    x, g = random_logits(12, V, 3)
    low = torch.finfo(torch.float32).min
    x[0] = NONE                                     # nothing is left of a row
    x[1, 10:] = NONE                                # ten numbers are
    x[2, 1:] = low                                  # masked by the type's lowest value
    x[3] = float("nan")
    x[4, ::3] = float("nan")
    x[5, 7] = math.inf                              # one token has all the weight
    x[6, [8, 20]] = math.inf                        # two share it
    x[7] = low
    scores = torch.tensor([[0.0, -1.0, -2.0, -0.5], [NONE, float("nan"), -3.0, -2.0], [-0.1, NONE, NONE, NONE]])
    check_select(x, scores, [7, 4999])
    check_select(x, torch.full((3, 4), NONE), [1])          # nobody is left
    check_select(x[:4], scores[:1], [], in_place=True)


@gpu
def test_select_fewer_continuations_than_beams():
    x, _ = random_logits(8, 3, 5)
    check_select(x, torch.tensor([[0.0, NONE, NONE, NONE, NONE, NONE, NONE, NONE]]), [1])
    check_select(x, torch.tensor([[0.0, -0.5, NONE, NONE, NONE, NONE, NONE, NONE]]), [0, 1, 2])


@gpu
def test_select_stop_tokens_given_twice_or_outside():
    x, _ = random_logits(4, 999, 8)
    x[:, 5] += 12.0
    check_select(x, torch.tensor([[0.0, -0.5, -0.25, -1.0]]), [5, 5, 998])
    out = run_select(x.cuda(), torch.tensor([[0.0, -0.5, -0.25, -1.0]]), [5, -1, 999, 2 ** 31 - 1])
    want = run_select(x.cuda(), torch.tensor([[0.0, -0.5, -0.25, -1.0]]), [5])
    assert all(torch.equal(out[k], want[k]) for k in out)


@gpu
def test_select_equal_beams_and_large_scores():
    x, _ = random_logits(1, 40000, 9)
    check_select(x.repeat(4, 1), torch.full((1, 4), -2.0), [77], gap_needed=False)      # totals are equal: the lowest beam first
    check_select(x.repeat(4, 1), torch.tensor([[-1e4, -1e4 - 8, -2e4, -3e30]]), [77])


@gpu
def test_select_rows_at_any_address():
    V = 4099
    x, g = random_logits(9, V, 12)
    flat = torch.zeros(10 * V + 8, device="cuda")
    scores = -torch.rand(2, 2, generator=g)
    for shift in range(4):
        view = flat[shift: shift + 4 * V].view(4, V)
        view.copy_(x[:4])
        check_select(view, scores, [4])


@gpu
def test_select_sums_against_64_bits():
    """The smallest errors that rankings rest on: rows of very different spreads."""
    V = 128256
    g = torch.Generator().manual_seed(1)
    x = torch.cat([torch.randn(1, V, generator=g) * s + t for s, t in ((0.0, 5.0), (0.1, -300.0), (1.0, 80.0), (2.5, 0.0), (6.0, 1e4), (30.0, 0.0))])
    out = run_select(x.cuda(), torch.zeros(6, 1), [])
    want = x.double().max(1).values - x.double().logsumexp(1)
    got = out["next_scores"].cpu().double()[:, 0]
    assert torch.all((got - want).abs() <= LSE_TOL + 2.0 ** -24 * want.abs())


@gpu
def test_select_within_a_beam_the_logits_decide():
    """Scores so large that 64 bits hold no logarithm beside them: totals of a beam are equal, its logits are not."""
    V = 9000
    x = torch.zeros(4, V)
    for row, best in enumerate(([70, 20, 8999], [5, 4, 3], [8000, 12, 13], [1, 2, 0])):
        x[row, best] = torch.tensor([9.0, 8.0, 7.0])
    out = run_select(x.cuda(), torch.tensor([[-1e17, NONE], [-1e30, -2e30]]), [])
    assert out["parents"].tolist() == [[0, 0], [0, 0]] and out["tokens"].tolist() == [[70, 20], [8000, 12]]
    # a stop token in front of others, and behind one, of its beam
    out = run_select(x[:2].cuda(), torch.tensor([[-1e17, NONE]]), [20])
    assert out["tokens"].tolist() == [[70, 8999]] and out["ended_tokens"].tolist() == [[20, -1]] and out["ended_parents"].tolist() == [[0, -1]]
    out = run_select(x[:2].cuda(), torch.tensor([[-1e17, NONE]]), [8999])
    assert out["tokens"].tolist() == [[70, 20]] and out["ended_tokens"].tolist() == [[-1, -1]]


@gpu
@pytest.mark.parametrize("V", [130, 4099, 50001, 50257, 128257])
def test_select_equal_beams_at_any_address(V):
    """Rows of the same logits begin at different places of a vector where the vocabulary is no multiple of 8, or where the tensor begins off one;
    totals are equal all the same, and the lowest beam comes first."""
    x, g = random_logits(3, V, V)
    x = x.repeat_interleave(4, 0)
    flat = torch.zeros(12 * V + 8, device="cuda")
    order = x[::4].sort(dim=1, descending=True, stable=True).indices[:, :4].tolist()
    for shift in (0, 1, 6):
        view = flat[shift: shift + 12 * V].view(12, V)
        view.copy_(x)
        # the four beams' best, which are equal: every beam goes on with its own
        out = run_select(view, torch.full((3, 4), -2.0), [])
        assert out["parents"].tolist() == [[0, 1, 2, 3]] * 3 and out["tokens"].tolist() == [[o[0]] * 4 for o in order]
        assert all(len(set(row)) == 1 for row in out["next_scores"].tolist())
        # ... which all end: then their second ones; of eight equal beams' two best tokens each the first four stand in front
        out = run_select(view, torch.full((3, 4), -2.0), [o[0] for o in order])
        for r, o in enumerate(order):
            others = [t for t in o if t not in [p[0] for p in order]]
            assert out["ended_parents"][r].tolist() == [0, 1, 2, 3] and out["ended_tokens"][r].tolist() == [o[0]] * 4
            assert out["parents"][r].tolist() == [0, 1, 2, 3] and out["tokens"][r].tolist() == [others[0]] * 4


def near_beams(R, K, V, seed):
    """Logits and scores whose rows' sums of exponentials are the same number: the beams of a request have the same logits at other places, above
    one another by what float32 holds exactly.  Totals of the best tokens differ by the scores alone: steps of 2^-23."""
    g = torch.Generator().manual_seed(seed)
    x = torch.empty(R * K, V)
    scores = torch.empty(R, K)
    for r in range(R):
        one = (torch.randn(V, generator=g) * 2.5 * 4096).round() / 4096
        if r % 3 == 0:
            one[:] = 0.0                                # one number stands out of a flat row
            one[0], one[1] = 27.0, 26.5
        elif r % 3 == 1:
            one = 26.9921875 + (one / 64 * 4096).round() / 4096
            one[::9] = 0.0
        for b in range(K):
            x[r * K + b] = one[torch.randperm(V, generator=g)] + [0.0, 64.0, -777.0, 3.5][(b + r) % 4]
        scores[r] = -1.0 - torch.randperm(K, generator=g) * 2.0 ** -23
    return x, scores


@gpu
@pytest.mark.parametrize("R, K, V", [(12, 4, 9001), (30, 2, 40000), (6, 8, 50257), (3, 32, 4100)])
def test_select_beams_that_float32_sums_do_not_tell_apart(R, K, V):
    """Totals 2^-23 apart, less than sums of float32 terms are off (2.1e-6): the order is that of 64 bits, among stop tokens as well."""
    x, scores = near_beams(R, K, V, R + V)
    for stops in ([], [int(t) for t in x[::K].argmax(1)[:16]] + [int(t) for t in x[1::K].argmax(1)[:16]]):
        gap = P.select(x, scores, stops)[-1]
        assert gap > 2.0 ** -24
        for in_place in (False, True):
            check_select(x, scores, stops, in_place, gap_needed=False)


@gpu
def test_select_beams_that_float32_sums_do_not_tell_apart_replayed():
    """The same from a graph on another stream, scores changed in place from step to step: rows are summed again in some replays and not in others."""
    x, scores = near_beams(6, 8, 50257, 6 + 50257)
    R, K = scores.shape
    logits, stops, far = x.cuda(), ints([int(t) for t in x[::K].argmax(1)]), -torch.rand(R, K, generator=torch.Generator().manual_seed(3))

    def outputs():
        return dict(parents=empty(R, K), tokens=empty(R, K), ended_parents=empty(R, K), ended_tokens=empty(R, K),
                    ended_scores=empty(R, K, dtype=torch.float32))

    want, given = [], (scores, far, scores - 1.0, far - 3.0)
    for start in given:
        held, out = start.cuda(), outputs()
        for _ in range(2):
            ops.beam_select(logits, held, stops, next_scores=held, **out, workspace=Workspace(torch.device("cuda")))
        want.append([held] + list(out.values()))
    torch.cuda.synchronize()
    side, workspace, held, out = torch.cuda.Stream(), Workspace(torch.device("cuda")), scores.cuda(), outputs()
    with torch.cuda.stream(side):
        ops.beam_select(logits, held, stops, next_scores=held, **out, workspace=workspace)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        graph.capture_begin()
        ops.beam_select(logits, held, stops, next_scores=held, **out, workspace=workspace)
        graph.capture_end()
        for start, w in zip(given, want):
            held.copy_(start)
            graph.replay()
            graph.replay()
            side.synchronize()
            assert all(torch.equal(a, b) for a, b in zip([held] + list(out.values()), w))


def log_weight_of_the_largest(x):
    """log softmax(x) of each row's largest number, from the distances to it (far from 0 their difference is all that 64 bits hold)."""
    return -(x.double() - x.double().max(1, keepdim=True).values).exp().sum(1).log()


@gpu
@pytest.mark.parametrize("edge", [1e4, 1e6, 6.9314716e7, 1e8, 1e12, 3e38])
def test_select_sums_of_far_logits(edge):
    """Numbers on both sides of -edge and of edge, as near to one another as float32 has them, in every thread's share of a row; beside them rows with a
    few such numbers among ordinary ones, and among masked ones."""
    V = 16 * 4096 + 700
    g = torch.Generator().manual_seed(11)
    near = torch.tensor([float(torch.nextafter(torch.tensor(edge), torch.tensor(math.inf if up else 0.0))) for up in (True, False)] + [edge])
    pick = near[torch.randint(0, 3, (2, V), generator=g)]
    few = torch.where(torch.arange(V) % 176 == 5, near.max(), near.min())          # one of a thread's largest, all others a step below
    masked = torch.full((2, V), torch.finfo(torch.float32).min)
    masked[:, ::7] = torch.randn(2, len(range(0, V, 7)), generator=g)
    masked[0, ::11] = -edge
    x = torch.cat([-pick, pick[:1], -few[None], few[None], masked])
    rows, want = x.shape[0], log_weight_of_the_largest(x)
    out = run_select(x.cuda(), torch.zeros(rows, 1), [])
    got = out["next_scores"].cpu().double()[:, 0]
    assert torch.all((got - want).abs() <= LSE_TOL + 2.0 ** -24 * want.abs()), (got - want).tolist()


@gpu
def test_select_a_thread_with_numbers_on_both_sides_of_a_power():
    """Some of a thread's vectors have numbers only below -1e8 in powers of two, others a number above; 8 apart, float32's spacing there."""
    V, step = 32 * 4096, 8.0
    for top in (-69314720.0, -69314712.0, -69314728.0):
        x = torch.full((3, V), top - step)
        x[0, ::176] = top
        x[1, V // 2:] = top
        x[2, :4096] = top
        out = run_select(x.cuda(), torch.zeros(3, 1), [])
        want = log_weight_of_the_largest(x)
        assert torch.all((out["next_scores"].cpu().double()[:, 0] - want).abs() <= LSE_TOL + 2.0 ** -24 * want.abs())


# -- tables ----------------------------------------------------------------------------------------------------------------
def run_fork(parents, lengths, table, refs, free, F=None, spare=0, page=PAGE, in_place=False):
    (R, K), (N, W), Pn = (len(parents), len(parents[0])), (len(table), len(table[0])), len(refs)
    F = len(free) if F is None else F
    given = dict(parents=ints(parents), lengths=ints(lengths), table=ints(table), refs=ints(refs),
                 free_pages=ints((list(free) + [-1] * F)[:F]) if F else empty(0), n_free=ints([len(free)]))
    out = dict(kv_len=empty(R, K), positions=empty(R, K), dest_rows=empty(R, K), new_table=empty(N, W), new_refs=empty(Pn), new_free=empty(F),
               new_n_free=empty(1), copy_src=empty(R, K), copy_dst=empty(R, K), copy_rows=empty(R, K), shared=empty(R), missing=empty(1))
    if in_place:
        out.update(kv_len=given["lengths"], new_table=given["table"], new_refs=given["refs"], new_free=given["free_pages"],
                   new_n_free=given["n_free"])
    ops.fork_pages(*given.values(), **out, spare=spare, page_size=page)
    return out


def check_fork(parents, lengths, table, refs, free, F=None, spare=0, page=PAGE):
    F = len(free) if F is None else F
    want = P.fork(parents, lengths, table, refs, free[:F], spare, page)
    left = want.pop("free")
    want.update(new_free=(left + [-1] * F)[:F], new_n_free=[min(len(left), F)], missing=[want["missing"] + max(0, len(left) - F)])
    for in_place in (False, True):
        out = run_fork(parents, lengths, table, refs, free, F, spare, page, in_place)
        for name, w in want.items():
            assert out[name].tolist() == w, (name, in_place)
    return want


class Cache:
    """Tables that beam search could have left, by running it: rows of groups fork and grow at random, the counts kept by `plain_beams`."""

    def __init__(self, R, K, n_pages, W, prompts, seed, outside=True, page=PAGE):
        self.R, self.K, self.W, self.page, self.rnd = R, K, W, page, random.Random(seed)
        self.table, self.refs = [[-1] * W for _ in range(R * K)], [0] * n_pages
        self.free = list(range(1, n_pages))
        self.rnd.shuffle(self.free)
        self.lengths = []
        for r in range(R):
            n = prompts[r % len(prompts)]
            for c in range(-(-n // page)):
                p = self.free.pop()
                self.table[r * K][c] = p
                self.refs[p] = 2 if outside else 1
            self.lengths.append([n] + [1] * (K - 1))
            for k in range(1, K):
                self.table[r * K + k][0] = 0

    def parents(self, dead=0.1, first=False):
        if first:
            return [[0] * self.K for _ in range(self.R)]
        pick = [[self.rnd.choice(row) for _ in range(self.K)] for row in
                ([k for k in range(self.K) if self.table[r * self.K + k][0] > 0] or [-1] for r in range(self.R))]
        return [[p if self.rnd.random() >= dead else -1 for p in row] for row in pick]

    def take(self, want):
        self.table, self.refs, self.lengths = want["new_table"], want["new_refs"], want["kv_len"]
        self.free = want["new_free"][: want["new_n_free"][0]]


@gpu
@pytest.mark.parametrize("R, K, prompts, page, outside", [(1, 1, [1], 64, True), (1, 4, [63, 64], 64, True), (3, 2, [64, 130, 1], 64, False),
                                                          (5, 5, [200, 640, 3], 64, True), (2, 32, [70, 190], 64, True), (7, 16, [31, 5], 4, True),
                                                          (130, 8, [10, 77, 300], 64, False), (3, 6, [9], 8, False), (1, 3, [5], 1, True)])
def test_fork_steps(R, K, prompts, page, outside):
    W = -(-max(prompts) // page) + -(-20 // page) + 1
    pages = 1 + R * (-(-max(prompts) // page) + K * (-(-20 // page) + 2))
    c = Cache(R, K, pages, W, prompts, R * 100 + K, outside, page)
    for step in range(18):
        free = c.free + [-1] * (pages - len(c.free))
        want = check_fork(c.parents(first=step == 0, dead=0.0 if step < 3 else 0.1), c.lengths, c.table, c.refs, c.free, F=pages, page=page)
        assert want["missing"] == [0] and len(free) == pages
        for src, dst in zip(sum(want["copy_src"], []), sum(want["copy_dst"], [])):
            assert (src < 0) == (dst < 0) and (src < 0 or src != dst)
        c.take(want)
        held = [p for row, n in zip(c.table, sum(c.lengths, [])) for p in row[: -(-n // page)] if p > 0]
        assert not set(held) & set(c.free)
        written = [r // page for r in sum(want["dest_rows"], []) if r >= page]
        assert len(written) == len(set(written)) and all(held.count(p) == 1 and c.refs[p] == 1 for p in written)


@gpu
def test_fork_without_enough_pages():
    c = Cache(2, 4, 12, 3, [70], 4)
    want = check_fork([[0] * 4] * 2, c.lengths, c.table, c.refs, c.free[:3], F=3)
    assert want["missing"] == [8 - 3]
    c = Cache(2, 4, 12, 3, [64], 4, outside=False)
    assert check_fork([[0] * 4, [-1] * 4], c.lengths, c.table, c.refs, [], F=0)["missing"] == [4 - 1]      # (the other row's page comes back)
    assert check_fork([[-1] * 4] * 2, c.lengths, c.table, c.refs, [], F=1)["missing"] == [1]               # two pages back, place for one


@gpu
def test_fork_tables_too_narrow_and_odd_entries():
    c = Cache(2, 3, 30, 2, [128], 4)
    assert check_fork([[0, 0, 0], [0, -1, 0]], c.lengths, c.table, c.refs, c.free)["missing"] == [5]
    c.lengths = [[100, 0, 0], [0, 0, 0]]                     # rows without tokens
    check_fork([[0, 1, 2], [2, 1, 0]], c.lengths, c.table, c.refs, c.free)
    c.table[0][0] = -1                                       # a page that a window has passed
    check_fork([[0, 0, 0], [5, -7, 2 ** 30]], [[100, 1, 1], [1, 1, 1]], c.table, c.refs, c.free)


@gpu
def test_fork_far_pages_and_spare():
    """Numbers of pages above 2^16, a spare page that is not the first."""
    n = 200_000
    table = [[199_999, 150_000, -1], [199_999, 150_001, -1], [70_001, -1, -1], [70_001, -1, -1]]
    refs = [0] * n
    for row in table:
        for p in row:
            if p >= 0:
                refs[p] += 1
    want = check_fork([[1, 1], [1, -1]], [[100, 101], [64, 64]], table, refs, [5, 131_072, 77], F=6, spare=123_456)
    # page 150,000 comes back and is taken again at once, by the row that gives up 150,001; the row at the end of 70,001 takes 77
    assert want["copy_src"] == [[-1, 150_001], [-1, -1]] and want["copy_dst"] == [[-1, 150_000], [-1, -1]]
    assert want["new_table"][2] == [70_001, 77, -1] and want["new_free"] == [5, 131_072, -1, -1, -1, -1]


# -- copies ----------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shapes, page", [([(1, 8)], 64), ([(3, 5), (2, 64)], 64), ([(8, 128)] * 3 + [(1, 576)], 64), ([(2, 1)], 64),
                                          ([(4, 80), (4, 40)], 16), ([(1, 7)] * 130, 64)])
def test_copy_pages(dtype, shapes, page):
    n = 23
    g = torch.Generator().manual_seed(len(shapes))
    tensors = [torch.randn(n, h, page, d, generator=g).to(dtype).cuda() for h, d in shapes]
    src, dst, rows = [3, -1, 5, 3, 9, 40, 2, 7], [20, 19, 18, 17, -1, 16, 15, 14], [1, 9, page, page - 1, 3, 3, 0, page + 9]
    want = [t.clone() for t in tensors]
    for t in want:
        for s, d, r in zip(src, dst, rows):
            if 0 <= s < n and d >= 0:
                t[d, :, : min(r, page)] = t[s, :, : min(r, page)].clone()
    ops.copy_pages(tensors, ints(src), ints(dst), ints(rows))
    assert all(torch.equal(a, b) for a, b in zip(tensors, want))


@gpu
def test_copy_pages_beyond_32_bits():
    """Pages whose first byte lies past 2^32."""
    t = torch.zeros(5000, 8, 64, 1024, dtype=torch.bfloat16, device="cuda")
    t[4998] = 3.0
    ops.copy_pages([t], ints([4998]), ints([4999]), ints([40]))
    assert bool((t[4999, :, :40] == 3.0).all()) and not bool(t[4999, :, 40:].any()) and not bool(t[:4998].any())


# -- states ----------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("R, K, slots", [(1, 1, 1), (2, 4, 9), (3, 5, 15), (1, 8, 30), (2, 16, 40), (2, 32, 64)])
@pytest.mark.parametrize("numbers", [(1,), (3, 1000), (4096, 8, 20), (5,) * 70])
def test_reorder_rows(R, K, slots, numbers):
    g = torch.Generator().manual_seed(R * K)
    matrices = [torch.randn(slots, n, generator=g).cuda() for n in numbers]
    at = torch.randperm(slots, generator=g)[: R * K]
    parents = torch.randint(-1, K + 1, (R, K), generator=g)
    if K > 1:
        parents[0] = torch.arange(K).roll(1)                # a cycle through all rows
    want = [m.clone() for m in matrices]
    for a, b in zip(want, matrices):
        for r in range(R):
            for k in range(K):
                p = int(parents[r, k])
                if 0 <= p < K:
                    a[at[r * K + k]] = b[at[r * K + p]]
    ops.reorder_rows(matrices, at.int().cuda(), parents.int().cuda())
    assert all(torch.equal(a, b) for a, b in zip(matrices, want))


@gpu
def test_reorder_rows_slots_outside():
    m = torch.arange(12.0, device="cuda").view(4, 3)
    want = m.clone()
    want[2] = m[1]
    ops.reorder_rows([m], ints([1, 2, 9, -3]), ints([[3, 0, 0, 1]]))
    assert torch.equal(m, want)


# -- attention ---------------------------------------------------------------------------------------------------------------
def attention_case(R, K, kv_len, shared, nkv, group, hd, seed, extra=1):
    """Pages of a pool in random order; rows of a group share their first shared[r] pages."""
    g = torch.Generator().manual_seed(seed)
    W = max(-(-n // PAGE) for n in kv_len) + extra
    table, pages = [[-1] * W for _ in range(R * K)], 0
    for r in range(R):
        common = list(range(pages, pages + shared[r]))
        pages += shared[r]
        for k in range(K):
            n = -(-kv_len[r * K + k] // PAGE)
            mine = common[:n] + list(range(pages, pages + max(0, n - shared[r])))
            pages += max(0, n - shared[r])
            table[r * K + k][:n] = mine
    pages += 2
    order = torch.randperm(pages, generator=g).tolist()
    table = [[order[p] if p >= 0 else -1 for p in row] for row in table]
    nh = nkv * group
    q = (torch.randn(R * K, nh * hd, generator=g) * 2).bfloat16()
    k, v = (torch.randn(pages, nkv, PAGE, hd, generator=g).bfloat16() for _ in range(2))
    seen = torch.zeros(pages, PAGE, dtype=torch.bool)
    for row, n in zip(table, kv_len):
        for i in range(n):
            seen[row[i // PAGE], i % PAGE] = True
    for t in (k, v):                                        # what nobody may look at is no number
        t.masked_fill_(~seen[:, None, :, None], float("nan"))
    return q, k, v, table, nh


def attention_bound(want, size):
    return 2.0 ** -7 * want.abs() + (2.0 ** -8 + 2.0 ** -11) * size + 1e-30


def check_attention(R, K, kv_len, shared, nkv, group, hd, seed=1, extra=1, bound=None):
    q, k, v, table, nh = attention_case(R, K, kv_len, shared, nkv, group, hd, seed, extra)
    out = empty(R * K, nh * hd, dtype=torch.bfloat16)
    scale = 1.0 / math.sqrt(hd)
    ops.attention_beams(q.cuda(), k.cuda(), v.cuda(), out, ints(table), ints(kv_len), ints(shared), K, nh, nkv, hd, PAGE, scale,
                        Workspace(torch.device("cuda")), bound or max(kv_len))
    want, size = P.attention(q, k, v, table, kv_len, nh, nkv, hd, scale)
    off = (out.cpu().double().view(R * K, nh, hd) - want).abs()
    worst = (off / attention_bound(want, size)).max()
    assert worst <= 1.0, float(worst)


@gpu
@pytest.mark.parametrize("hd", [8, 16, 40, 64, 80, 96, 128, 256])
@pytest.mark.parametrize("K, group", [(1, 1), (4, 4), (5, 7), (8, 8)])
def test_attention_heads_and_groups(hd, K, group):
    check_attention(2, K, [130] * K + [700] * K, [2, 9], 2, group, hd)


@gpu
@pytest.mark.parametrize("lengths, shared", [([1, 1, 1], 0), ([63, 64, 65], 0), ([64, 64, 64], 1), ([65, 65, 65], 1), ([200, 200, 200], 3),
                                             ([129, 140, 190], 2), ([0, 70, 0], 0), ([0, 0, 0], 0), ([1, 500, 500], 7), ([1000, 3, 64], 1),
                                             ([2000, 2000, 2000], 0)])
def test_attention_lengths(lengths, shared):
    for group, hd in ((4, 128), (1, 64)):
        check_attention(1, 3, lengths, [min(shared, max(lengths) // PAGE)], 2, group, hd)


@gpu
def test_attention_many_groups_ragged():
    kv_len, shared = [], []
    for r in range(9):
        n = [1, 64, 300, 1030, 4000, 65, 2, 127, 900][r]
        kv_len += [n, n, n, n]
        shared.append([0, 1, 3, 16, 10, 0, 0, 1, 14][r])
    check_attention(9, 4, kv_len, shared, 2, 4, 128)
    check_attention(9, 4, kv_len, shared, 1, 7, 64, bound=64 * 64, extra=3)


@gpu
@pytest.mark.parametrize("K, group", [(32, 1), (32, 8), (16, 4), (3, 40)])
def test_attention_many_rows(K, group):
    check_attention(2, K, [190] * K + [500] * K, [1, 7], 1, group, 64)


@gpu
@pytest.mark.parametrize("R, K, group, hd", [(1300, 2, 1, 64), (40, 32, 5, 72), (70, 3, 2, 160)])
def test_attention_of_many_groups(R, K, group, hd):
    """More blocks of rows than places that a block counts them in."""
    rnd = random.Random(R)
    kv_len, shared = [], []
    for _ in range(R):
        n = [rnd.randrange(0, 150) for _ in range(K)]
        shared.append(rnd.randrange(0, 1 + min(n) // PAGE))
        kv_len += n
    check_attention(R, K, kv_len, shared, 1, group, hd, seed=R)


@gpu
def test_attention_pages_beyond_32_bits():
    """Numbers of a cache that 32 bits cannot count, rows of 16 bytes up to the last that its rows' number has bits for."""
    for nkv, hd, pages in ((1, 128, 300000), (8, 8, 2 ** 31 // (8 * PAGE) - 1)):
        q, k, v, table, nh = attention_case(1, 2, [300, 290], [2], nkv, 2, hd, 4)
        far = torch.tensor([pages - 1 - 7 * i if i % 2 else 3 * i for i in range(k.shape[0])])
        big = [torch.empty(pages, nkv, PAGE, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        for to, t in zip(big, (k, v)):
            to[far.cuda()] = t.cuda()
        moved = [[int(far[p]) if p >= 0 else -1 for p in row] for row in table]
        out = empty(2, nh * hd, dtype=torch.bfloat16)
        ops.attention_beams(q.cuda(), *big, out, ints(moved), ints([300, 290]), ints([2]), 2, nh, nkv, hd, PAGE, 0.3, Workspace(torch.device("cuda")), 300)
        want, size = P.attention(q, k, v, table, [300, 290], nh, nkv, hd, 0.3)
        off = (out.cpu().double().view(2, nh, hd) - want).abs()
        assert float((off / attention_bound(want, size)).max()) <= 1.0
        del big
    with pytest.raises(ops.KernelError, match="attention_beams"):
        args = _attention_args(K=1, nh=1, nkv=1, hd=8, device="cuda")
        cache = torch.empty(2 ** 31 // PAGE, 1, PAGE, 8, dtype=torch.bfloat16, device="cuda")
        ops.attention_beams(**{**args, "k_cache": cache, "v_cache": cache, "workspace": Workspace(torch.device("cuda"))})


@gpu
def test_select_logits_beyond_32_bits():
    """The last of 2,100 rows of 1,050,000 logits (8.8 GB)."""
    rows, V = 2100, 1050000
    logits = torch.full((rows, V), NONE, device="cuda")
    x, _ = random_logits(3, V, 9)
    logits[-3:] = x.cuda()
    scores = torch.full((rows // 3, 3), NONE)
    scores[-1] = torch.tensor([-1.0, -1.2, -0.7])
    out = run_select(logits, scores, [5])
    parents, tokens, nxt, ep, et, es, gap = P.select(x, scores[-1:], [5])
    assert gap > 2 * LSE_TOL
    assert out["parents"][-1].tolist() == parents[0] and out["tokens"][-1].tolist() == tokens[0]
    assert (out["parents"][:-1] == -1).all() and (out["next_scores"][:-1] == NONE).all() and (out["ended_tokens"][:-1] == -1).all()


@gpu
@pytest.mark.parametrize("hd", [40, 64, 128, 256])
@pytest.mark.parametrize("K, group", [(4, 4), (5, 16), (11, 2)])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_attention_numbers_that_are_not_finite_stay_with_their_readers(hd, K, group, what):
    """In pages that only some beams read: the others' answers are as if they were not there."""
    kv_len = [130] + [700] * (K - 2) + [650] + [700] * K
    q, k, v, table, nh = attention_case(2, K, kv_len, [9, 9], 2, group, hd, 7)
    v[table[1][5], 1, 17, hd - 3] = what                    # a page that all but the first beam share
    k[table[2][10], 0, 3, 5] = what                         # own pages
    v[table[K - 1][9], 0, 60, 0] = what
    out = empty(2 * K, nh * hd, dtype=torch.bfloat16)
    scale = 1.0 / math.sqrt(hd)
    ops.attention_beams(q.cuda(), k.cuda(), v.cuda(), out, ints(table), ints(kv_len), ints([9, 9]), K, nh, 2, hd, PAGE, scale,
                        Workspace(torch.device("cuda")), 700)
    got = out.cpu().double().view(2 * K, 2, group, hd)
    want, size = P.attention(q, k, v, table, kv_len, nh, 2, hd, scale)
    want, size = want.view(2 * K, 2, group, hd), size.view(2 * K, 2, group, -1)
    clean = torch.ones(2 * K, 2, dtype=torch.bool)
    clean[1:K, 1] = clean[2, 0] = clean[K - 1, 0] = False
    off = (got - want).abs() / attention_bound(want, size)
    assert float(off[clean].max()) <= 1.0
    bad = ~torch.isfinite(want)
    assert bad[1, 1, :, hd - 3].all() and bad[K - 1, 0, :, 0].all() and not torch.isfinite(got[bad]).any()


@gpu
@pytest.mark.parametrize("hd", [40, 64, 128, 136, 256])
@pytest.mark.parametrize("K, group", [(4, 4), (5, 6), (5, 12), (11, 2)])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_attention_a_value_that_is_not_finite_is_one_number_of_a_row(hd, K, group, what):
    """Whether a stage is read by all rows of a tile or by some: the other numbers of the rows that read the value are those of the definition, and so
    are the rows that do not."""
    kv_len = [130] + [700] * (K - 2) + [650] + [700] * K
    q, k, v, table, nh = attention_case(2, K, kv_len, [9, 9], 2, group, hd, 7)
    v[table[1][5], 1, 17, hd - 3] = what                    # a page that all but the first beam share
    v[table[1][5], 1, 18, 2] = v[table[1][6], 1, 40, 2] = what
    v[table[2][10], 0, 3, 5] = what                         # own pages
    v[table[2][10], 0, 3, 6] = v[table[2][10], 0, 59, 7] = what
    v[table[K - 1][9], 0, 60, 0] = what
    v[table[K + 1][3], 0, 11, 9] = what                     # a page that all of a request share
    out = empty(2 * K, nh * hd, dtype=torch.bfloat16)
    scale = 1.0 / math.sqrt(hd)
    ops.attention_beams(q.cuda(), k.cuda(), v.cuda(), out, ints(table), ints(kv_len), ints([9, 9]), K, nh, 2, hd, PAGE, scale,
                        Workspace(torch.device("cuda")), 700)
    got = out.cpu().double().view(2 * K, nh, hd)
    want, size = P.attention(q, k, v, table, kv_len, nh, 2, hd, scale)
    bad = ~torch.isfinite(want)
    assert int(bad.sum()) == group * (2 * (K - 1) + 3 + 1 + K) and not torch.isfinite(got[bad]).any()
    off = (got - want).abs() / attention_bound(want, size)
    assert float(off[~bad].max()) <= 1.0


def climbing_case(R, K, kv_len, shared, nkv, group, hd, seed):
    """Scores that climb (or fall, or stay) along the keys, each beam's and head's by a slope of its own: -48 to 48 from the first key to the last,
    69 powers of two.  A query has 16 numbers that are not 0."""
    q, k, v, table, nh = attention_case(R, K, kv_len, shared, nkv, group, hd, seed)
    g = torch.Generator().manual_seed(seed + 1)
    longest = max(kv_len)
    fine = torch.isfinite(k[:, 0, :, 0])
    place = torch.zeros(k.shape[0], PAGE)                    # of a key in its row, as far as rows agree
    for row, n in zip(table, kv_len):
        for i in range(-(-n // PAGE)):
            place[row[i]] = torch.arange(i * PAGE, (i + 1) * PAGE) / longest
    slope = (torch.arange(R * K * nh).view(R * K, nh) % 7 - 3) * 16.0
    q = torch.zeros(R * K, nh, hd)
    q[:, :, 8:16] = torch.randn(R * K, nh, 8, generator=g) * 0.3
    q[:, :, :8] = slope[:, :, None] / 8 * math.sqrt(hd)
    k = torch.where(fine[:, None, :, None], torch.randn(k.shape, generator=g), k.float())
    k[..., :8] = torch.where(fine[:, None, :, None], place[:, None, :, None] + torch.randn(*k.shape[:-1], 8, generator=g) * 0.01, k[..., :8])
    return q.view(R * K, nh * hd).bfloat16(), k.bfloat16(), v, table, nh


@gpu
@pytest.mark.parametrize("blocks", [2, 7, 74])
@pytest.mark.parametrize("K, group, hd", [(4, 4, 64), (4, 4, 128), (4, 4, 256), (4, 7, 64), (4, 7, 128), (4, 7, 256), (8, 8, 64), (8, 8, 128), (8, 8, 256),
                                          (16, 8, 64), (16, 8, 128), (16, 8, 256)])
def test_attention_scores_that_climb(K, group, hd, blocks, monkeypatch):
    """Sums and results are scaled down in the middle of a run of keys again and again, by factors between 0 and 1 that differ from row to row; tiles of 16 to
    128 rows, the list cut into few shares (runs of many stages) and many.  Errors: 16 products of a query, |q k| scale below 64 together, summed
    in float32 within 16 * 64 / 2^24 = 2^-14; scaled by log2(e) and rounded below 128, 2^-18, and once more as a distance: with the power's 2^-22
    less than 2^-11 of a weight."""
    plan = ops.beam_attention_plan
    monkeypatch.setattr(ops, "beam_attention_plan", lambda *sizes: (blocks, plan(*sizes)[1]))
    kv_len = [1300 - 20 * (k % 3) for k in range(K)] + [1700] * K
    shared = [14, 26]
    q, k, v, table, nh = climbing_case(2, K, kv_len, shared, 2, group, hd, K + hd)
    out = empty(2 * K, nh * hd, dtype=torch.bfloat16)
    scale = 1.0 / math.sqrt(hd)
    ops.attention_beams(q.cuda(), k.cuda(), v.cuda(), out, ints(table), ints(kv_len), ints(shared), K, nh, 2, hd, PAGE, scale,
                        Workspace(torch.device("cuda")), max(kv_len))
    want, size = P.attention(q, k, v, table, kv_len, nh, 2, hd, scale)
    off = (out.cpu().double().view(2 * K, nh, hd) - want).abs()
    assert float((off / attention_bound(want, size)).max()) <= 1.0


@gpu
@pytest.mark.parametrize("size", [1e3, 1e15, 1e18])
@pytest.mark.parametrize("K, group, hd", [(4, 4, 128), (5, 2, 64), (16, 4, 64), (3, 2, 256)])
def test_attention_scores_far_below_zero(K, group, hd, size):
    """All scores of some rows lie at -size^2 and below, of some at size^2 and above: the largest of them share the weight, in one part and in several."""
    R = 2
    kv_len = [130] * K + [1500] * K
    q, k, v, table, nh = attention_case(R, K, kv_len, [1, 9], 2, group, hd, 5)
    sign = torch.where(torch.arange(R * K * nh) % 3 == 0, 1.0, -1.0).view(R * K, nh, 1)
    q = torch.zeros(R * K, nh, hd)
    q[:, :, 1:2] = sign * size
    q = q.view(R * K, nh * hd).bfloat16()
    fine = torch.isfinite(k)
    k = torch.where(fine, torch.zeros(()), k.float())
    # a key in seven has the least, one in five the most: numbers that bfloat16 holds
    step = torch.arange(k.shape[0] * PAGE).view(k.shape[0], 1, PAGE)
    k[..., 1] = torch.where(fine[..., 1], torch.where(step % 7 == 0, 0.5, torch.where(step % 5 == 0, 2.0, 1.0)) * size, k[..., 1])
    k = k.bfloat16()
    out = empty(R * K, nh * hd, dtype=torch.bfloat16)
    ops.attention_beams(q.cuda(), k.cuda(), v.cuda(), out, ints(table), ints(kv_len), ints([1, 9]), K, nh, 2, hd, PAGE, 0.25,
                        Workspace(torch.device("cuda")), 1500)
    want, weight = P.attention(q, k, v, table, kv_len, nh, 2, hd, 0.25)
    off = (out.cpu().double().view(R * K, nh, hd) - want).abs()
    assert float((off / attention_bound(want, weight)).max()) <= 1.0


@gpu
def test_attention_shared_pages_said_too_many():
    """More pages said to be shared than the rows have."""
    q, k, v, table, nh = attention_case(1, 2, [100, 100], [2], 1, 4, 64, 3)
    out = [empty(2, nh * 64, dtype=torch.bfloat16) for _ in range(2)]
    for o, shared in zip(out, (1, 9)):
        ops.attention_beams(q.cuda(), k.cuda(), v.cuda(), o, ints(table), ints([100, 100]), ints([shared]), 2, nh, 1, 64, PAGE, 0.125,
                            Workspace(torch.device("cuda")), 100)
    assert torch.equal(out[0], out[1])


# -- together ----------------------------------------------------------------------------------------------------------------
class Step:
    """A step's operators as a search has them: beams chosen, pages forked and copied, states moved, attention over the new tables."""

    def __init__(self, R, K, V, seed, hd=64, prompt=200):
        g = torch.Generator().manual_seed(seed)
        W, own = 8, 3 * K * R
        held = -(-prompt // PAGE)
        pages = 1 + R * held + own
        table = torch.full((R, K, W), -1, dtype=torch.int32)
        table[:, 1:, 0] = 0                                  # page 0 is the spare one
        refs = torch.zeros(pages, dtype=torch.int32)
        for r in range(R):
            table[r, 0, :held] = torch.arange(1 + r * held, 1 + (r + 1) * held)
            refs[1 + r * held: 1 + (r + 1) * held] = 2
        free = torch.full((pages,), -1, dtype=torch.int32)
        free[:own] = torch.arange(pages - own, pages).flip(0)
        lengths = torch.ones(R, K, dtype=torch.int32)
        lengths[:, 0] = prompt
        scores = torch.full((R, K), NONE)
        scores[:, 0] = 0.0
        z = lambda *s: torch.zeros(s, dtype=torch.int32)      # noqa: E731
        t = dict(logits=torch.randn(R * K, V, generator=g) * 2, scores=scores, stops=torch.tensor([1, 5], dtype=torch.int32), parents=z(R, K),
                 tokens=z(R, K), ep=z(R, K), et=z(R, K), es=torch.zeros(R, K), lengths=lengths, table=table.view(R * K, W), refs=refs, free=free,
                 n_free=torch.tensor([own], dtype=torch.int32), positions=z(R, K), dest=z(R, K), src=z(R * K), dst=z(R * K), rows=z(R * K),
                 shared=z(R), missing=z(1), k=torch.randn(pages, 2, PAGE, hd, generator=g).bfloat16(),
                 v=torch.randn(pages, 2, PAGE, hd, generator=g).bfloat16(), state=torch.randn(R * K, 24, generator=g), slots=torch.arange(R * K).int(),
                 q=torch.randn(R * K, 8 * hd, generator=g).bfloat16(), out=torch.zeros(R * K, 8 * hd, dtype=torch.bfloat16))
        self.t = {name: x.cuda() for name, x in t.items()}
        self.R, self.K, self.hd, self.workspace = R, K, hd, Workspace(torch.device("cuda"))

    def run(self):
        t, R, K, hd = self.t, self.R, self.K, self.hd
        ops.beam_select(t["logits"], t["scores"], t["stops"], parents=t["parents"], tokens=t["tokens"], next_scores=t["scores"],
                        ended_parents=t["ep"], ended_tokens=t["et"], ended_scores=t["es"], workspace=self.workspace)
        ops.fork_pages(t["parents"], t["lengths"], t["table"], t["refs"], t["free"], t["n_free"], kv_len=t["lengths"], positions=t["positions"],
                       dest_rows=t["dest"], new_table=t["table"], new_refs=t["refs"], new_free=t["free"], new_n_free=t["n_free"],
                       copy_src=t["src"].view(R, K), copy_dst=t["dst"].view(R, K), copy_rows=t["rows"].view(R, K), shared=t["shared"],
                       missing=t["missing"], spare=0, page_size=PAGE)
        ops.copy_pages([t["k"], t["v"]], t["src"], t["dst"], t["rows"])
        ops.reorder_rows([t["state"]], t["slots"], t["parents"])
        ops.attention_beams(t["q"], t["k"], t["v"], t["out"], t["table"], t["lengths"].view(-1), t["shared"], K, 8, 2, hd, PAGE, 0.125,
                            self.workspace, 8 * PAGE)
        t["logits"].mul_(-0.97).add_(0.01)                   # the next step's

    def same(self, other):
        for name, x in self.t.items():
            if not torch.equal(x.view(torch.uint8) if name in ("k", "v") else x, other.t[name].view(torch.uint8) if name in ("k", "v") else other.t[name]):
                return name
        return None


@gpu
@pytest.mark.parametrize("R, K, V, hd", [(1, 4, 300, 64), (3, 32, 5000, 128), (5, 3, 40000, 256)])
def test_steps_replayed_on_another_stream(R, K, V, hd):
    """Ten steps launched one by one, and the same captured once on another stream and replayed."""
    plain, captured, other = (Step(R, K, V, 3, hd) for _ in range(3))
    for _ in range(10):
        plain.run()
    assert int(plain.t["missing"]) == 0
    side = torch.cuda.Stream()
    captured.workspace = other.workspace
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        other.run()                                          # (makes the workspace)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        graph.capture_begin()
        captured.run()
        graph.capture_end()
        for _ in range(10):
            graph.replay()
    side.synchronize()
    assert captured.same(plain) is None


@gpu
def test_steps_of_two_streams_at_once():
    """Two searches, each with a stream and a workspace of its own."""
    want = [Step(4, 8, 50000, seed) for seed in (1, 2)]
    got = [Step(4, 8, 50000, seed) for seed in (1, 2)]
    for s in want:
        for _ in range(8):
            s.run()
    streams = [torch.cuda.Stream() for _ in got]
    torch.cuda.synchronize()
    for _ in range(8):
        for s, stream in zip(got, streams):
            with torch.cuda.stream(stream):
                s.run()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert a.same(b) is None


# -- refusals --------------------------------------------------------------------------------------------------------------
def _select_args(R=1, K=2, V=9, S=1, device="cpu"):
    i, f = dict(dtype=torch.int32, device=device), dict(dtype=torch.float32, device=device)
    return dict(logits=torch.zeros(R * K, V, **f), scores=torch.zeros(R, K, **f), stop_tokens=torch.zeros(S, **i), parents=torch.zeros(R, K, **i),
                tokens=torch.zeros(R, K, **i), next_scores=torch.zeros(R, K, **f), ended_parents=torch.zeros(R, K, **i),
                ended_tokens=torch.zeros(R, K, **i), ended_scores=torch.zeros(R, K, **f), workspace=None)


def _fork_args(R=1, K=2, W=3, n=8, device="cpu"):
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device=device)      # noqa: E731
    return dict(parents=z(R, K), lengths=z(R, K), table=z(R * K, W), refs=z(n), free_pages=z(n), n_free=z(1), kv_len=z(R, K),
                positions=z(R, K), dest_rows=z(R, K), new_table=z(R * K, W), new_refs=z(n), new_free=z(n), new_n_free=z(1), copy_src=z(R, K),
                copy_dst=z(R, K), copy_rows=z(R, K), shared=z(R), missing=z(1), spare=0, page_size=64)


def _attention_args(K=2, R=1, nh=4, nkv=2, hd=64, W=2, device="cpu"):
    b, i = dict(dtype=torch.bfloat16, device=device), dict(dtype=torch.int32, device=device)
    return dict(q=torch.zeros(R * K, nh * hd, **b), k_cache=torch.zeros(3, nkv, 64, hd, **b), v_cache=torch.zeros(3, nkv, 64, hd, **b),
                out=torch.zeros(R * K, nh * hd, **b), block_table=torch.zeros(R * K, W, **i), kv_len=torch.zeros(R * K, **i),
                shared=torch.zeros(R, **i), beams=K, nh=nh, nkv=nkv, hd=hd, page_size=64, scale=1.0, workspace=None, max_kv_len=64)


def test_a_wait_that_ran_out_names_who_waited():
    """Every code that a bounded wait of the kernels gives ends in the digit of one of the three that a message names, and in attention of beams in
    that of the warp it stands in."""
    import os
    import re
    folder = os.path.join(os.path.dirname(ops.__file__), "..", "csrc")
    for name in sorted(os.listdir(folder)):
        if name.endswith((".cu", ".cuh")):
            text = open(os.path.join(folder, name)).read()
            codes = [int(c) for c in re.findall(r"mbar_wait\([^;]*?status, (\d+)\)", text)]
            assert all(c % 10 in (1, 2, 3) for c in codes), (name, codes)
    text = open(os.path.join(folder, "beam_attention.cu")).read()
    text = text[text.index("beam_attention_kernel"):]
    roles = [text.index(s) for s in ("if (warp == 0) {", "} else if (warp == 1) {", "} else if (warp >= 4) {", "// The parts of a (beam, head)")]
    for role, (begin, end) in enumerate(zip(roles, roles[1:]), 1):
        codes = [int(c) for c in re.findall(r"status, (\d+)\)", text[begin:end])]
        assert codes and all(c % 10 == role for c in codes), (role, codes)
    for code, who in ((511, "TMA producer"), (552, "MMA issuer"), (583, "epilogue")):
        ops.kernel_status(torch.device("cpu")).fill_(code)
        with pytest.raises(ops.KernelError, match=f"{who}, code {code}"):
            ops.check_kernel_status(torch.device("cpu"))
        ops.check_kernel_status(torch.device("cpu"))            # told once


def test_refused_off_the_device():
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.beam_select(**_select_args())
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.fork_pages(**_fork_args())
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.attention_beams(**_attention_args())
    z = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.copy_pages([torch.zeros(2, 1, 64, 8)], z, z, z)
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.reorder_rows([torch.zeros(2, 8)], z, z.view(1, 2))


@pytest.mark.parametrize("change", [dict(K=33), dict(S=33), dict(R=0)])
def test_select_sizes_refused(change):
    with pytest.raises(ops.KernelError, match="beam_select"):
        ops.beam_select(**_select_args(**change))


@pytest.mark.parametrize("change", [dict(K=33), dict(R=0)])
def test_fork_sizes_refused(change):
    with pytest.raises(ops.KernelError, match="fork_pages"):
        ops.fork_pages(**_fork_args(**change))


@pytest.mark.parametrize("change", [dict(spare=8), dict(spare=-1), dict(page_size=0)])
def test_fork_spare_page_refused(change):
    with pytest.raises(ops.KernelError, match="fork_pages"):
        ops.fork_pages(**{**_fork_args(), **change})


def test_fork_more_pages_than_are_counted_refused():
    with pytest.raises(ops.KernelError, match="fork_pages"):
        ops.fork_pages(**_fork_args(n=ops.MOST_FORK_PAGES + 1))
    with pytest.raises(ops.KernelError, match="fork_pages"):
        ops.fork_pages(**{**_fork_args(n=8), "page_size": 1 << 28})


@pytest.mark.parametrize("change", [dict(beams=33), dict(beams=3), dict(page_size=32), dict(hd=60), dict(hd=264), dict(nh=3), dict(nkv=0)])
def test_attention_sizes_refused(change):
    with pytest.raises(ops.KernelError, match="attention_beams"):
        ops.attention_beams(**{**_attention_args(), **change})


def test_reorder_sizes_refused():
    z = torch.zeros(1, 33, dtype=torch.int32)
    with pytest.raises(ops.KernelError, match="reorder_rows"):
        ops.reorder_rows([torch.zeros(2, 8)], z[0], z)


@gpu
def test_wrong_types_and_shapes_refused():
    for name in ("logits", "scores", "stop_tokens", "parents", "ended_scores"):
        args = _select_args(device="cuda")
        args[name] = args[name].double()
        with pytest.raises(ops.KernelError, match="beam_select"):
            ops.beam_select(**args)
    for name in ("table", "new_table", "refs", "new_free", "missing", "kv_len"):
        args = _fork_args(device="cuda")
        args[name] = torch.zeros((*args[name].shape[:-1], args[name].shape[-1] + 1), dtype=torch.int32, device="cuda")
        with pytest.raises(ops.KernelError, match="fork_pages"):
            ops.fork_pages(**args)
    for name in ("q", "k_cache", "out"):
        args = _attention_args(device="cuda")
        args[name] = args[name].float()
        with pytest.raises(ops.KernelError, match="attention_beams"):
            ops.attention_beams(**args)
    i = torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in (torch.zeros(2, 1, 64, 8, dtype=torch.float64), torch.zeros(2, 64, 8), torch.zeros(3, 1, 64, 8), torch.zeros(2, 1, 32, 8)):
        with pytest.raises(ops.KernelError, match="copy_pages"):
            ops.copy_pages([torch.zeros(2, 1, 64, 8, device="cuda"), bad.cuda()], i, i, i)
    for bad in (torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(3, 8), torch.zeros(8, 2).t()):
        with pytest.raises(ops.KernelError, match="reorder_rows"):
            ops.reorder_rows([torch.zeros(2, 8, device="cuda"), bad.cuda()], i, i.view(1, 2))


@gpu
@pytest.mark.parametrize("name, other", [("parents", "tokens"), ("next_scores", "ended_scores"), ("ended_tokens", "stop_tokens"),
                                         ("ended_scores", "scores"), ("next_scores", "logits")])
def test_select_outputs_over_others_refused(name, other):
    args = _select_args(R=1, K=2, V=2, S=2, device="cuda")
    args[name] = args[other].view(-1)[:2].view(args[name].shape)
    args["workspace"] = Workspace(torch.device("cuda"))
    with pytest.raises(ops.KernelError, match="10004"):
        ops.beam_select(**args)


@gpu
def test_attention_addresses_refused():
    args = _attention_args(device="cuda")
    args["workspace"] = Workspace(torch.device("cuda"))
    for name in ("q", "out", "k_cache", "v_cache"):
        t = args[name]
        odd = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape)
        with pytest.raises(ops.KernelError, match="attention_beams"):
            ops.attention_beams(**{**args, name: odd})
    with pytest.raises(ops.KernelError, match="10004"):
        ops.attention_beams(**{**args, "out": args["q"]})


@gpu
@pytest.mark.parametrize("name", ["block_table", "kv_len", "shared"])
def test_attention_output_over_the_tables_refused(name):
    args = _attention_args(device="cuda")
    args["workspace"] = Workspace(torch.device("cuda"))
    words = args["out"].view(torch.int32).view(-1)
    args[name] = words[128: 128 + args[name].numel()].view(args[name].shape)
    with pytest.raises(ops.KernelError, match="10004"):
        ops.attention_beams(**args)


@gpu
def test_copies_and_moves_over_one_another_refused():
    """Views that share some of their memory; a tensor of pages given twice, of which both copies are the same, is taken."""
    i = torch.zeros(2, dtype=torch.int32, device="cuda")
    some = torch.arange(4 * 64 * 8, dtype=torch.float32, device="cuda")
    a, b = some[: 2 * 64 * 8].view(2, 1, 64, 8), some[64 * 8: 3 * 64 * 8].view(2, 1, 64, 8)
    lists = [torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0], [1], [3])]
    with pytest.raises(ops.KernelError, match="10004"):
        ops.copy_pages([a, b], *lists)
    with pytest.raises(ops.KernelError, match="10004"):
        ops.copy_pages([a], some[:1].view(torch.int32), lists[1], lists[2])
    before = a.clone()
    ops.copy_pages([a, a], *lists)
    assert torch.equal(a[1, :, :3], before[0, :, :3]) and torch.equal(a[1, :, 3:], before[1, :, 3:])
    m, n = some[:32].view(4, 8), some[8:40].view(4, 8)
    with pytest.raises(ops.KernelError, match="10004"):
        ops.reorder_rows([m, n], i, i.view(1, 2))
    with pytest.raises(ops.KernelError, match="10004"):
        ops.reorder_rows([m], m.view(-1)[4:6].view(torch.int32), i.view(1, 2))
    # lists are read: they may be one another
    slots = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    before = m.clone()
    ops.reorder_rows([m], slots, slots.view(1, 2))              # row 1 becomes row 0, and row 0 row 1
    assert torch.equal(m[:2], before[:2].flip(0)) and torch.equal(m[2:], before[2:])


@gpu
def test_reorder_a_matrix_twice_refused():
    m, i = torch.zeros(2, 8, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(ops.KernelError, match="twice"):
        ops.reorder_rows([m, m], i, i.view(1, 2))


@gpu
@pytest.mark.parametrize("name, other", [("new_table", "refs"), ("positions", "lengths"), ("kv_len", "positions"), ("missing", "n_free"),
                                         ("new_refs", "free_pages"), ("copy_src", "copy_dst")])
def test_fork_outputs_over_others_refused(name, other):
    args = _fork_args(R=2, K=2, W=2, n=8, device="cuda")
    args[name] = args[other].view(args[name].shape)
    with pytest.raises(ops.KernelError, match="10004"):
        ops.fork_pages(**args)
