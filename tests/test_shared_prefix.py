"""A step of sequences that share a prefix, with drafted tokens: the index tables made on the device, attention over the
shared pages and each sequence's own, the verification of drafts; each against its definition in 64 bits.

Tolerances, from the number formats: a bfloat16 result differs from the exact one by its own rounding (relative 2^-9) and by the
weights' rounding to bfloat16 for the tensor cores (2^-9 each, which adds up like noise over a row's keys): 2^-7 of a row's
largest value bounds both with room.  float32 sums of up to some thousands of terms: 2^-24 a term, in trees: 2e-6 of the largest; and a
score s is itself rounded, which changes its weight by 2^-24 s twice (the product's sum, the change to units of log2): 2^-23 s where
scores are large.
"""
import math

import numpy as np
import pytest
import torch

from janus_b200.kernels import ops

gpu = pytest.mark.gpu
PAGE = 64
TOL = {torch.bfloat16: 2.0 ** -7, torch.float32: 2e-6}


def ints(values, shape=None):
    t = torch.tensor(values, dtype=torch.int32, device="cuda")
    return t if shape is None else t.reshape(shape)


# -- index tables ----------------------------------------------------------------------------------------------------
def tables_oracle(lengths, new, rows, old_table, held, prefix, free, n_free, width, places, page):
    pool = list(free[:n_free])
    for r in range(len(old_table)):
        if r not in rows:
            pool += [int(p) for p in old_table[r][len(prefix):held[r]]]
    at, missing = 0, 0
    out = dict(q_start=[0], kv_len=[], positions=[], token_seq=[], dest_rows=[], table=[], held=[])
    for b, (n, t, r) in enumerate(zip(lengths, new, rows)):
        mine = [int(p) for p in (prefix if r < 0 else old_table[r][:held[r]])]
        want = -(-(n + t) // page)
        while len(mine) < min(want, width) and at < len(pool):
            mine.append(pool[at])
            at += 1
        missing += max(0, want - len(mine))
        for p in range(n, n + t):
            out["positions"].append(p)
            out["token_seq"].append(b)
            out["dest_rows"].append(mine[p // page] * page + p % page if p // page < len(mine) else -1)
        out["q_start"].append(out["q_start"][-1] + t)
        out["kv_len"].append(n + t)
        out["table"].append(mine + [-1] * (width - len(mine)))
        out["held"].append(len(mine))
    for k in ("positions", "token_seq", "dest_rows"):
        out[k] = (out[k] + [-1] * places)[:places]
    left, N = pool[at:], len(free)
    out.update(free_pages=(left + [-1] * N)[:N], n_free=[min(len(left), N)], missing=[missing + max(0, len(left) - N)])
    return out


def run_tables(lengths, new, rows, old_table, held, prefix, free, n_free, width, places, page=PAGE):
    B = len(lengths)
    empty = lambda *shape: torch.full(shape, 12345, dtype=torch.int32, device="cuda")      # noqa: E731
    out = dict(q_start=empty(B + 1), kv_len=empty(B), positions=empty(places), token_seq=empty(places), dest_rows=empty(places),
               table=empty(B, width), held=empty(B), free_pages=empty(len(free)), n_free=empty(1), missing=empty(1))
    ops.step_tables(ints(lengths), ints(new), ints(rows), ints(old_table, (len(old_table), -1 if old_table else width)), ints(held),
                    ints(prefix), ints(free), ints([n_free]), **out, page_size=page)
    return {k: v.cpu().tolist() for k, v in out.items()}


def tables_case(seed, B, B0, prefix_pages, width, longest, most_new, page=PAGE, spare=None, free_share=1.0, places_more=3):
    rng = np.random.default_rng(seed)
    ids = rng.permutation(100000).tolist()
    take = lambda n: [ids.pop() for _ in range(n)]       # noqa: E731
    prefix = take(prefix_pages)
    old, held = [], []
    for _ in range(B0):
        h = int(rng.integers(prefix_pages, width + 1))
        held.append(h)
        old.append(prefix + take(h - prefix_pages) + [-7] * (width - h))
    rows = [-1] * B
    some = rng.permutation(B0)[: min(B, int(B0 * 0.7))]
    for b, r in zip(rng.permutation(B).tolist(), some.tolist()):
        rows[b] = r
    lengths = [int(rng.integers(0, longest + 1)) if r >= 0 else prefix_pages * page for r in rows]
    new = [int(v) for v in rng.integers(0, most_new + 1, B)]
    need = sum(max(0, -(-(n + t) // page)) for n, t in zip(lengths, new))
    n_free = int(need * free_share)
    free = take(n_free) + [-5] * int(rng.integers(0, 9))
    return lengths, new, rows, old, held, prefix, free, n_free, width, sum(new) + places_more


@gpu
@pytest.mark.parametrize("args", [
    dict(seed=1, B=1, B0=0, prefix_pages=0, width=1, longest=0, most_new=1),
    dict(seed=2, B=1, B0=1, prefix_pages=0, width=3, longest=100, most_new=70),
    dict(seed=3, B=3, B0=9, prefix_pages=2, width=8, longest=400, most_new=5),
    dict(seed=4, B=33, B0=20, prefix_pages=1, width=31, longest=1900, most_new=6),
    dict(seed=5, B=700, B0=650, prefix_pages=5, width=40, longest=2500, most_new=60),
    dict(seed=6, B=2000, B0=2300, prefix_pages=0, width=9, longest=500, most_new=2),
    dict(seed=7, B=64, B0=64, prefix_pages=3, width=12, longest=700, most_new=9, free_share=0.2),      # the pool runs dry
    dict(seed=8, B=50, B0=40, prefix_pages=0, width=4, longest=900, most_new=300),                     # rows too narrow
    dict(seed=9, B=17, B0=17, prefix_pages=2, width=90, longest=500, most_new=7, page=7),              # another page size
    dict(seed=10, B=5, B0=6, prefix_pages=1, width=6, longest=300, most_new=0, places_more=1),         # nobody brings anything
])
def test_step_tables_against_lists(args):
    case = tables_case(**args)
    page = args.get("page", PAGE)
    assert run_tables(*case, page=page) == tables_oracle(*case, page=page)


@gpu
def test_step_tables_chain_keeps_every_page():
    """Steps one after another, sequences that end and begin: no page is lost, held twice or given out twice."""
    rng = np.random.default_rng(3)
    width, N = 12, 90
    prefix, free = [0, 1], list(range(2, N))
    table, held, lengths, n_free = [], [], [], len(free)
    for step in range(40):
        on = [r for r in range(len(table)) if rng.random() < 0.8]
        rng.shuffle(on)
        rows = on + [-1] * int(rng.integers(0, 3))
        lens = [lengths[r] for r in on] + [2 * PAGE] * (len(rows) - len(on))
        new = [int(rng.integers(0, 90)) for _ in rows]
        new = [min(t, width * PAGE - n) for t, n in zip(new, lens)]
        need = sum(max(0, -(-(n + t) // PAGE) - (held[r] if r >= 0 else 2)) for n, t, r in zip(lens, new, rows))
        back = sum(h - 2 for r, h in enumerate(held) if r not in on)
        if not rows or need > n_free + back:
            rows, lens, new = on[:1] or [-1], [lengths[on[0]] if on else 2 * PAGE], [0]
        out = run_tables(lens, new, rows, table, held, prefix, free, n_free, width, sum(new) + 1)
        assert out["missing"] == [0]
        table, held, free, n_free, lengths = out["table"], out["held"], out["free_pages"], out["n_free"][0], out["kv_len"]
        seen = free[:n_free] + [p for t, h in zip(table, held) for p in t[2:h]]
        assert sorted(seen) == list(range(2, N))
        free = free + [-1] * (N - len(free))


# -- attention -------------------------------------------------------------------------------------------------------
def attention_case(seed, dtype, heads, kv_heads, dim, prefix, new, owned, extra_columns=0, page_offset=0, n_pages=None, sharp=1.0):
    """`owned`: own keys of each sequence with its new tokens (its length is prefix + owned)."""
    g = torch.Generator().manual_seed(seed)
    d = torch.Generator(device="cuda").manual_seed(seed)
    first = -(-prefix // PAGE)
    width = max(1, max(-(-max(o, 0) // PAGE) for o in owned))
    total = first + sum(-(-max(o, 0) // PAGE) for o in owned) + 3
    ids = (torch.randperm(total, generator=g) + page_offset).tolist()
    table = torch.full((len(new), width + extra_columns), -1, dtype=torch.int32)
    at = first
    for b, o in enumerate(owned):
        k = -(-max(o, 0) // PAGE)
        table[b, extra_columns:extra_columns + k] = torch.tensor(ids[at:at + k], dtype=torch.int32)
        at += k
    starts = np.concatenate([[0], np.cumsum(new)]).tolist()
    positions = [prefix + o - n + j for o, n in zip(owned, new) for j in range(n)]
    n_pages = n_pages or total
    make = lambda *shape: torch.randn(shape, generator=d, device="cuda").to(dtype)      # noqa: E731
    k = make(n_pages, kv_heads, PAGE, dim)
    return dict(q=(sharp * torch.randn((max(1, starts[-1]), heads * dim), generator=d, device="cuda")).to(dtype), k=k,
                v=make(n_pages, kv_heads, PAGE, dim), prefix_pages=ints(ids[:first]), prefix=prefix,
                table=table.cuda()[:, extra_columns:], q_start=ints(starts), kv_len=ints([prefix + o for o in owned]),
                positions=ints(positions or [-1]), heads=heads, kv_heads=kv_heads, dim=dim, scale=dim ** -0.5, most_new=max(new),
                most=prefix + max(0, max(owned)))


def attention(c, out=None):
    from janus_b200.engine.workspace import Workspace
    out = torch.full_like(c["q"], 7.0) if out is None else out
    ops.attention_prefix(c["q"], c["k"], c["v"], out, c["prefix_pages"], c["prefix"], c["table"], c["q_start"], c["kv_len"], c["positions"],
                         c["heads"], c["kv_heads"], c["dim"], PAGE, c["scale"], c.get("workspace") or Workspace(torch.device("cuda")),
                         c["most_new"], c["most"])
    return out


def attention_oracle(c):
    G, D, P = c["kv_heads"], c["dim"], c["prefix"]
    starts, lens = c["q_start"].tolist(), c["kv_len"].tolist()
    out = torch.zeros(c["q"].shape, dtype=torch.float64, device="cuda")
    flat = lambda x, pages: x[pages.long()].double().permute(1, 0, 2, 3).reshape(G, -1, D)       # noqa: E731
    for b, length in enumerate(lens):
        n = starts[b + 1] - starts[b]
        for j in range(n):
            see = length - n + j + 1
            own = max(0, see - P)
            k = torch.cat([flat(c["k"], c["prefix_pages"])[:, :min(see, P)], flat(c["k"], c["table"][b, :-(-own // PAGE)])[:, :own]], 1) if see > 0 else None
            if k is None or k.shape[1] == 0:
                continue
            v = torch.cat([flat(c["v"], c["prefix_pages"])[:, :min(see, P)], flat(c["v"], c["table"][b, :-(-own // PAGE)])[:, :own]], 1)
            q = c["q"][starts[b] + j].double().view(G, -1, D)
            p = torch.softmax(torch.einsum("grd,gkd->grk", q, k) * c["scale"], -1)
            out[starts[b] + j] = torch.einsum("grk,gkd->grd", p, v).reshape(-1)
    return out


def close(got, want, dtype, rows=slice(None), largest_score=0.0):
    got, want = got[rows].double(), want[rows]
    assert torch.isfinite(got).all()
    err = (got - want).abs() / want.abs().amax(1, keepdim=True).clamp_min(1e-30)
    assert float(err.max()) <= TOL[dtype] + 2.0 ** -23 * largest_score, float(err.max())


BF, F32 = torch.bfloat16, torch.float32


@gpu
@pytest.mark.parametrize("dtype,heads,kv_heads,dim,prefix,new,owned", [
    (BF, 4, 1, 64, 64, [1], [1]),                                        # the smallest
    (BF, 8, 2, 128, 130, [1, 1, 1], [1, 64, 65]),                        # page edges
    (BF, 32, 8, 128, 1000, [1] * 9, [1, 5, 63, 64, 65, 127, 128, 129, 700]),
    (BF, 6, 2, 64, 300, [1, 6, 2, 3], [30, 6, 2, 90]),                   # groups of three; all own keys new
    (BF, 20, 4, 80, 777, [3, 1, 4], [200, 1, 40]),                       # head sizes between the builds'
    (BF, 14, 2, 96, 127, [5, 2], [5, 400]),
    (BF, 2, 2, 8, 100, [2, 1], [9, 80]),
    (BF, 4, 2, 256, 500, [1, 3], [70, 3]),
    (BF, 4, 4, 200, 129, [40, 3], [90, 3]),
    (BF, 16, 1, 72, 65, [1, 1], [33, 200]),                              # one key head for sixteen
    (BF, 128, 1, 64, 70, [1], [5]),                                      # as many rows as a tile has
    (BF, 33, 1, 40, 200, [2, 1], [60, 3]),
    (BF, 8, 2, 128, 700, [200, 31, 90], [230, 31, 500]),                 # tiles of prompts
    (BF, 32, 8, 64, 129, [300], [300]),
    (BF, 8, 4, 128, 0, [1, 1], [1, 300]),                                # no prefix
    (BF, 8, 4, 64, 0, [70, 3], [70, 200]),
    (BF, 4, 1, 128, 20000, [1], [3]),                                    # a long one for one sequence
    (BF, 4, 2, 64, 100, [0, 1, 0, 2, 0], [50, 20, 0, 2, 7]),             # sequences that bring nothing
    (BF, 8, 2, 128, 200, [3, 2], [-10, 1]),                              # tokens inside the prefix, and across its end
    (BF, 4, 1, 64, 64, [1] * 300, [1 + i % 70 for i in range(300)]),     # many sequences
    (BF, 8, 8, 128, 100, [1] * 40, [3000] + [2] * 39),                   # one that is much longer
    (F32, 4, 1, 64, 64, [1], [1]),
    (F32, 16, 4, 128, 500, [1, 3, 2], [1, 65, 300]),
    (F32, 6, 2, 40, 130, [2, 1], [2, 129]),
    (F32, 4, 2, 256, 100, [1, 20], [64, 30]),
    (F32, 3, 3, 37, 70, [1, 2], [5, 66]),                                # no multiple of four
    (F32, 8, 2, 128, 100, [70, 5], [70, 150]),
    (F32, 4, 2, 64, 0, [1, 2], [1, 200]),
    (F32, 8, 2, 64, 200, [0, 3, 2], [4, -10, 1]),
])
def test_attention_against_formula(dtype, heads, kv_heads, dim, prefix, new, owned):
    c = attention_case(5, dtype, heads, kv_heads, dim, prefix, new, owned)
    close(attention(c), attention_oracle(c), dtype, slice(0, sum(new)))


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [[1, 1, 1], [4, 1, 3], [60, 90, 70]])
def test_attention_masked_values_that_are_not_numbers(dtype, new):
    """What lies behind a sequence's end in its last page, behind the prefix's end, and in later tokens of the same step stays
    out of a row, whatever it is; and a row with such a value of its own shows it."""
    owned = [n + b * 40 for b, n in enumerate(new)]
    c = attention_case(7, dtype, 8, 2, 64, 100, new, owned)
    want = attention_oracle(c)
    bad = [float("nan"), float("inf"), -float("inf")]
    for b, o in enumerate(owned):
        if o % PAGE:
            page = int(c["table"][b, o // PAGE])
            c["k"][page, :, o % PAGE:], c["v"][page, :, o % PAGE:] = bad[b % 3], bad[(b + 1) % 3]
    last = int(c["prefix_pages"][-1])
    c["k"][last, :, 36:], c["v"][last, :, 36:] = float("nan"), float("nan")
    close(attention(c), want, dtype)
    if max(new) == 1:
        return
    # the last token of the first sequence: its key and value are not numbers, the rows before it do not see them
    o, n = owned[0], new[0]
    page = int(c["table"][0, (o - 1) // PAGE])
    c["v"][page, :, (o - 1) % PAGE] = float("nan")
    got = attention(c)
    close(got, want, dtype, [t for t in range(sum(new)) if t != n - 1])
    assert torch.isnan(got[n - 1]).all()


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [[1, 1, 1], [4, 1, 3], [130, 90, 70]])
def test_attention_stale_numbers_and_keys_that_are_not_numbers(dtype, new):
    """Finite numbers of any size behind a sequence's end weigh nothing at all; a key of the prefix that is not a number, wherever
    it lies in a block of keys, shows in every row."""
    owned = [n + b * 40 for b, n in enumerate(new)]
    c = attention_case(8, dtype, 8, 2, 128, 1400, new, owned)
    want = attention_oracle(c)
    for b, o in enumerate(owned):
        if o % PAGE:
            page = int(c["table"][b, o // PAGE])
            c["k"][page, :, o % PAGE:], c["v"][page, :, o % PAGE:] = 0.0, 3e38
    last = int(c["prefix_pages"][-1])
    c["k"][last, :, 1400 % PAGE:], c["v"][last, :, 1400 % PAGE:] = 0.0, -3e38
    close(attention(c), want, dtype)
    for at in (0, 15, 30, 63, 1399):
        page, row = int(c["prefix_pages"][at // PAGE]), at % PAGE
        kept = c["k"][page, 0, row].clone()
        c["k"][page, 0, row] = float("nan")
        got = attention(c)
        assert torch.isnan(got[:, :4 * 128]).all()                       # the query heads of kv head 0
        close(torch.cat([torch.zeros_like(got[:, :4 * 128]), got[:, 4 * 128:]], 1), torch.cat([0 * want[:, :4 * 128], want[:, 4 * 128:]], 1), dtype)
        c["k"][page, 0, row] = kept


@gpu
@pytest.mark.parametrize("n,prefix,longest,new", [(400, 16000, 1000, 1), (64, 3000, 900, 1), (40, 2500, 130, 4), (12, 6000, 60, 100), (9, 1900, 60, 130)])
def test_attention_of_many_sequences(n, prefix, longest, new):
    """Steps whose prefix is cut in ranges, by one and by two tiles a block, beside long own keys."""
    c = attention_case(11, BF, 16, 4, 128, prefix, [new] * n, [new + i * 37 % longest for i in range(n)])
    close(attention(c), attention_oracle(c), BF)


@gpu
@pytest.mark.parametrize("n,prefix,new,heads,kv_heads,dim", [
    (66, 6001, 2, 32, 8, 64),       # ranges of 13 key blocks that go from one row tile to the next
    (300, 60, 1, 16, 8, 64),        # one block of 64 keys, for the first of two groups only
    (300, 190, 1, 16, 8, 40),       # three
    (700, 900, 1, 8, 8, 48),        # a last tile with few rows
    (90, 2500, 3, 8, 1, 32),
])
def test_attention_of_narrow_heads_behind_a_prefix(n, prefix, new, heads, kv_heads, dim):
    c = attention_case(12, BF, heads, kv_heads, dim, prefix, [new] * n, [new + i * 37 % 90 for i in range(n)], sharp=3.0)
    close(attention(c), attention_oracle(c), BF)


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_loud_keys_and_rows_that_see_nothing(dtype):
    c = attention_case(9, dtype, 8, 2, 128, 300, [2, 1, 3], [2, 90, 40], sharp=40.0)      # weights of nearly one key each
    largest = float(c["q"].float().view(-1, 128).norm(dim=1).max() * c["k"].float().norm(dim=-1).max()) * c["scale"]
    close(attention(c), attention_oracle(c), dtype, largest_score=largest)
    c = attention_case(9, dtype, 8, 2, 128, 300, [2, 1, 3], [2, 90, 40])
    c["kv_len"][1], c["positions"][2] = 0, -1
    got = attention(c)
    assert (got[2] == 0).all()
    close(got, attention_oracle(c), dtype, [0, 1, 3, 4, 5])


@gpu
def test_attention_rows_of_no_sequence_are_left_alone():
    for dtype in (BF, F32):
        c = attention_case(3, dtype, 8, 2, 64, 200, [1, 2], [40, 70])
        want = attention_oracle(c)
        pad = lambda t, v: torch.cat([t, t.new_full((5,) + t.shape[1:], v)])     # noqa: E731
        c["q"], c["positions"] = pad(c["q"], 1.0), pad(c["positions"], -1)
        got = attention(c)
        close(got[:3], want, dtype)
        assert (got[3:] == 7.0).all()


@gpu
def test_attention_takes_whole_tables_as_a_view_and_runs_in_a_graph_on_another_stream():
    c = attention_case(4, BF, 8, 2, 128, 256, [1, 2, 1], [3, 200, 64], extra_columns=4)
    assert not c["table"].is_contiguous()
    from janus_b200.engine.workspace import Workspace
    c["workspace"] = Workspace(torch.device("cuda"))
    want, plain = attention_oracle(c), attention(c)
    close(plain, want, BF)
    out = torch.zeros_like(c["q"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            attention(c, out)
        out.zero_()
        graph.replay()
    side.synchronize()
    assert torch.equal(out, plain)      # the same sums in the same order


@gpu
def test_attention_of_a_cache_beyond_32_bit_offsets():
    pages = (1 << 32) // (2 * PAGE * 128) + 400                # more than 2^32 numbers a tensor
    c = attention_case(6, BF, 4, 2, 128, 300, [1, 2], [100, 30], page_offset=pages - 12, n_pages=None)
    k = torch.zeros((pages, 2, PAGE, 128), dtype=BF, device="cuda")
    need = torch.cat([c["prefix_pages"], c["table"].reshape(-1)])
    need = need[need >= 0].long()
    k[need] = torch.randn((len(need), 2, PAGE, 128), device="cuda").to(BF)
    c["k"] = c["v"] = k
    close(attention(c), attention_oracle(c), BF)


@gpu
def test_attention_refusals():
    c = attention_case(1, BF, 8, 2, 64, 100, [1, 2], [5, 9])
    for change, text in ((dict(q=c["q"].half()), "float32 or bfloat16"), (dict(q=c["q"].float()), "expected"), (dict(dim=60), "multiples of 8"),
                         (dict(k=c["k"][:, :1]), "expected shape|contiguous"), (dict(prefix=200), "do not hold a prefix"),
                         (dict(most=100 + 65), "do not hold"), (dict(kv_len=c["kv_len"].long()), "int32"),
                         (dict(table=c["table"].long()), "block table"), (dict(table=c["table"][:1]), "block table"),
                         (dict(positions=c["positions"][:2]), "shape"), (dict(q=c["q"].cpu()), "CUDA")):
        with pytest.raises(ops.KernelError, match=text):
            attention({**c, **change}, out=torch.empty_like(c["q"]))


# -- verification ----------------------------------------------------------------------------------------------------
def verify(c):
    from janus_b200.engine.workspace import Workspace
    B, width = c["q_start"].shape[0] - 1, c["width"]
    empty = lambda *shape: torch.full(shape, 99, dtype=torch.int32, device="cuda")         # noqa: E731
    accepted, tokens, kept = empty(B), empty(B, width), empty(B)
    logprobs = torch.full((B, width), 99.0, device="cuda")
    ops.verify_drafts(c["logits"], c["tokens"], c["q_start"], c["kv_len"], accepted, tokens, logprobs, kept, c["heat"], c["u_accept"],
                      c["u_draw"], c["probs"], Workspace(torch.device("cuda")))
    return accepted.tolist(), tokens.tolist(), logprobs.cpu().double(), kept.tolist()


def verify_oracle(c, adjust=False):
    """The definition, in 64 bits.  `adjust`: numbers near an edge are moved away from it first (two right sums may differ there)."""
    starts, ids, lens = c["q_start"].tolist(), c["tokens"].tolist(), c["kv_len"].tolist()
    V, heat, width = c["logits"].shape[1], c["heat"], c["width"]
    accepted, tokens, kept = [], [], []
    logprobs = torch.zeros((len(lens), width), dtype=torch.float64)
    for b, (lo, hi) in enumerate(zip(starts, starts[1:])):
        rows = min(hi - lo, width)
        tokens.append([-1] * width)
        if rows == 0:
            accepted.append(0)
            kept.append(lens[b])
            continue
        x = c["logits"][lo:lo + rows].double()
        x = torch.where(torch.isnan(x), -math.inf, x)
        top = x.amax(1, keepdim=True)
        w = torch.where(x == top, 1.0, torch.exp((x - top) / (heat or 1.0)))
        w = torch.where(x == -math.inf, 0.0, w)
        S = w.sum(1)
        a = 0
        for a in range(rows):
            if a == rows - 1:
                break
            d = ids[lo + a + 1]
            if not 0 <= d < V:
                break
            if heat > 0:
                q = float(c["probs"][lo + a + 1, d]) if c["probs"] is not None else 1.0
                p = float(w[a, d] / S[a]) if S[a] > 0 else 0.0
                if adjust and abs(float(c["u_accept"][lo + a + 1]) * q - p) < 1e-4 * p:
                    c["u_accept"][lo + a + 1] *= 0.9
                if not float(c["u_accept"][lo + a + 1]) * q < p:
                    break
            elif int(torch.where(x[a] == top[a], 1, 0).argmax()) != d:
                break
        m = w[a].clone()
        if heat > 0:
            if a < rows - 1:
                d = ids[lo + a + 1]
                r = (w[a] / S[a] - c["probs"][lo + a + 1].double()).clamp_min(0) if c["probs"] is not None else m.clone()
                if c["probs"] is None and 0 <= d < V:
                    r[d] = 0.0
                if float(r.sum()) > 0:
                    m = r
            cum = torch.cumsum(m, 0)
            if adjust and float(cum[-1]) > 0:
                v = int(torch.searchsorted(cum, float(c["u_draw"][b]) * cum[-1:], right=True).clamp_max(V - 1))
                low, high = float((cum[v] - m[v]) / cum[-1]), float(cum[v] / cum[-1])
                if min(float(c["u_draw"][b]) - low, high - float(c["u_draw"][b])) < 1e-4:
                    v = int(m.argmax())
                    c["u_draw"][b] = float((cum[v] - 0.5 * m[v]) / cum[-1])
            t = int(torch.searchsorted(cum, float(c["u_draw"][b]) * cum[-1:], right=True)) if float(cum[-1]) > 0 else 0
        else:
            t = int(torch.where(x[a] == top[a], 1, 0).argmax())
        mine = ids[lo + 1:lo + 1 + a] + [t]
        for k, v in enumerate(mine):
            tokens[-1][k] = v
            logprobs[b, k] = math.log(float(w[k, v] / S[k])) if float(S[k]) > 0 and float(w[k, v]) > 0 else -math.inf
        accepted.append(a)
        kept.append(lens[b] - (hi - lo - 1) + a)
    return accepted, tokens, logprobs, kept


def verify_case(seed, V, drafts, heat, probs, width=None, agree=0.7):
    d = torch.Generator(device="cuda").manual_seed(seed)
    g = torch.Generator().manual_seed(seed)
    starts = np.concatenate([[0], np.cumsum([n + 1 if n >= 0 else 0 for n in drafts])]).tolist()
    T = max(1, starts[-1])
    logits = 2.0 * torch.randn((T, V), generator=d, device="cuda")
    logits[:, : min(V, 7)] += 5.0
    p = torch.zeros((T, V), device="cuda")
    p[1:] = torch.softmax((logits[:-1] + (1.0 - agree) * torch.randn((T - 1, V), generator=d, device="cuda")) / (heat or 0.5), 1)
    tokens = torch.cat([torch.zeros(1, dtype=torch.long, device="cuda"), torch.multinomial(p[1:] + 1e-12, 1, generator=d)[:, 0]]) if T > 1 else \
        torch.zeros(1, dtype=torch.long, device="cuda")
    c = dict(logits=logits, tokens=tokens.int(), q_start=ints(starts), kv_len=ints([100 + n for n in range(len(drafts))]), heat=heat,
             probs=p if probs else None, u_accept=torch.rand(T, generator=g).cuda(), u_draw=torch.rand(len(drafts), generator=g).cuda(),
             width=width or max(max(drafts) + 1, 1))
    return c


def check_verify(c):
    want = verify_oracle(c, adjust=True)
    got = verify(c)
    assert got[0] == want[0] and got[1] == want[1] and got[3] == want[3]
    a, b = got[2], want[2]
    same = (a == b) | ((a - b).abs() <= 2e-6 * (1.0 + b.abs()))       # sums of float32 in trees, and a logarithm's rounding
    assert same.all(), (a, b)


@gpu
@pytest.mark.parametrize("V", [1, 2, 5, 127, 4096, 8191, 8192, 8193, 32000, 50257, 300001])
@pytest.mark.parametrize("heat,probs", [(0.0, False), (0.8, False), (1.0, True), (0.6, True)])
def test_verify_against_definition(V, heat, probs):
    check_verify(verify_case(V, V, [0, 4, 1, 7, 2], heat, probs))


@gpu
@pytest.mark.parametrize("drafts", [[3], [0], [2] * 100, [6] * 400, [-1, 3, -1, 0, 5]])
@pytest.mark.parametrize("probs", [False, True])
def test_verify_batches(drafts, probs):
    """One request and hundreds (a cluster of blocks each, or a block), and requests that bring no rows."""
    check_verify(verify_case(11, 20011, drafts, 0.9, probs))


@gpu
def test_verify_drafts_of_the_same_distribution_are_always_accepted():
    c = verify_case(5, 5000, [5] * 20, 1.0, True, agree=1.0)
    c["probs"][1:] = torch.softmax(c["logits"][:-1], 1)
    c["u_accept"] *= 0.999
    assert verify(c)[0] == [5] * 20


@gpu
@pytest.mark.parametrize("heat", [0.0, 0.7])
@pytest.mark.parametrize("probs", [False, True])
def test_verify_filtered_rows_strange_numbers_and_strange_drafts(heat, probs):
    V = 10007
    c = verify_case(8, V, [3, 3, 3, 3, 3, 3, 2], heat, probs)
    c["logits"][:, 11:9000] = -math.inf                        # filtered
    c["tokens"][1::4] = torch.tensor([-1, V, 2 ** 31 - 1, -5, 10, 20, 3][:len(c["tokens"][1::4])], dtype=torch.int32)
    c["logits"][4] = -math.inf                                 # a row that leaves nothing
    c["logits"][8, 5] = math.nan
    c["logits"][9, 9500:9510] = math.inf                       # ten tokens share everything
    c["logits"][12:16] = 3.0                                   # ties: the lowest index
    check_verify(c)


@gpu
def test_verify_nothing_left_after_a_refusal_draws_from_the_target():
    c = verify_case(2, 3000, [2, 2], 1.0, True)
    c["probs"][:] = 2.0                                        # not a distribution: max(p - q, 0) is zero everywhere
    c["u_accept"][:] = 0.99
    check_verify(c)


@gpu
def test_verify_more_drafts_than_places():
    check_verify(verify_case(3, 4000, [6, 1, 9], 0.8, True, width=4))


@gpu
def test_verify_refusals():
    c = verify_case(1, 1000, [2, 1], 1.0, True)
    for change, text in ((dict(heat=-1.0), "temperature"), (dict(heat=math.nan), "temperature"), (dict(logits=c["logits"].bfloat16()), "float32"),
                         (dict(tokens=c["tokens"].long()), "int32"), (dict(probs=c["probs"][:, :-1].contiguous()), "shape"),
                         (dict(u_accept=c["u_accept"][:-1]), "shape"), (dict(logits=c["logits"][:, ::2]), "contiguous"),
                         (dict(u_draw=c["u_draw"].cpu()), "CUDA")):
        with pytest.raises(ops.KernelError, match=text):
            verify({**c, **change})


# -- refusals that need no device ------------------------------------------------------------------------------------
def test_tables_refuse_what_does_not_fit():
    z = lambda *shape: torch.zeros(shape, dtype=torch.int32)      # noqa: E731
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.step_tables(z(2), z(2), z(2), z(2, 4), z(2), z(1), z(5), z(1), q_start=z(3), kv_len=z(2), positions=z(4), token_seq=z(4),
                        dest_rows=z(4), table=z(2, 4), held=z(2), free_pages=z(5), n_free=z(1), missing=z(1), page_size=64)


@gpu
def test_tables_refusals():
    z = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")      # noqa: E731
    ins = [z(2), z(2), z(2), z(2, 4), z(2), z(1), z(5), z(1)]
    outs = dict(q_start=z(3), kv_len=z(2), positions=z(4), token_seq=z(4), dest_rows=z(4), table=z(2, 4), held=z(2), free_pages=z(5),
                n_free=z(1), missing=z(1))
    for i, change, text in ((0, z(3), "shape"), (3, z(2, 4).long(), "int32"), (3, z(2, 9), "take over")):
        with pytest.raises(ops.KernelError, match=text):
            ops.step_tables(*ins[:i], change, *ins[i + 1:], **outs, page_size=64)
    for name, change, text in (("table", ins[3], "cannot lie"), ("free_pages", ins[6], "cannot lie"), ("q_start", z(2), "shape"),
                               ("dest_rows", z(5), "shape")):
        with pytest.raises(ops.KernelError, match=text):
            ops.step_tables(*ins, **{**outs, name: change}, page_size=64)


def test_plans_cover_what_they_cut():
    """A row's ranges over the prefix are never more than the plan says: counted for every tile of many sizes."""
    rng = np.random.default_rng(1)
    for _ in range(300):
        group, nkv, hd = int(rng.integers(1, 17)), int(rng.integers(1, 17)), int(rng.choice([64, 128, 256]))
        n = int(rng.integers(1, 300))
        q = int(rng.choice([1, 1, 2, 7, 100]))
        T, prefix, own = n * q, int(rng.integers(1, 30000)), int(rng.integers(1, 4000))
        tiles, per, ranges, own_tiles, own_ctas, fewest, own_most = ops.attention_prefix_plan(T, n, q, prefix, own, group * nkv, nkv, hd)
        assert 0 <= ranges <= 64 and own_most <= 64 and (own_tiles or own_ctas >= 1)
        if not per:
            continue
        keys = 64 if hd > 128 else 128
        blocks, step = -(-prefix // keys), 128 // group * tiles
        items = -(-T // step) * nkv
        owner = np.arange(items * blocks) // per
        for i in range(items):
            assert owner[(i + 1) * blocks - 1] - owner[i * blocks] + 1 <= ranges


# -- the three together: generation behind a shared prefix -----------------------------------------------------------
def test_lookup_drafts():
    from janus_b200.engine.shared_prefix import LookupDrafter
    d = LookupDrafter([1, 2, 3, 4, 1, 2])
    assert d.draft(3) == [3, 4, 1] and d.draft(0) == []
    d.extend([3])
    assert d.draft(2) == [4, 1]
    d.extend([9])
    assert d.draft(2) == [] and LookupDrafter([5]).draft(4) == [] and LookupDrafter([]).draft(4) == []
    assert LookupDrafter([7, 7, 7]).draft(4) == [7]


class EveryToken:
    """Drafts that are mostly wrong."""

    def __init__(self, tokens):
        self.n = len(tokens)

    def extend(self, tokens):
        self.n += len(tokens)

    def draft(self, most):
        return [(self.n * 7 + j) % 200 for j in range(most)]


@gpu
@pytest.mark.parametrize("which", ["A", "B"])
@pytest.mark.parametrize("prefix_len", [0, 3, 64, 70])
def test_generate_shared_equals_generate_in_float32(tmp_path, which, prefix_len):
    """Greedy tokens behind a shared prefix are those of whole prompts, with drafts that are right, wrong or none, in batches."""
    import janus_b200
    from helpers import TINY, make_model_dir, random_tokens
    cfg = TINY[which]
    model = janus_b200.load(make_model_dir(cfg, str(tmp_path), seed=2, dtype="float32"), dtype="float32", max_tokens=2048)
    prefix = random_tokens(prefix_len, cfg["vocab_size"], 5)
    prompts = [random_tokens(n, cfg["vocab_size"], n) for n in (1, 9, 2, 17)]
    prompts.append(prompts[1][:4] * 3)
    n = 24
    want, _ = model.generate([prefix + p for p in prompts], max_tokens=n, ignore_eos=True)
    for drafts, batch, drafter in ((0, None, None), (4, None, None), (3, 2, None), (5, None, EveryToken)):
        more = {} if drafter is None else dict(drafter=drafter)
        got, reasons, stats = model.generate_shared(prefix, prompts, max_tokens=n, drafts=drafts, batch_size=batch, ignore_eos=True,
                                                    return_reasons=True, **more)
        assert got == want and reasons == ["length"] * len(prompts)
        assert stats.drafted >= stats.accepted and (drafts == 0) == (stats.drafted == 0)
        model.engine.cache.check()
        assert model.engine.cache.groups[0].pool.n_held == 0
    stop = want[1][5]
    got, reasons, _ = model.generate_shared(prefix, prompts, max_tokens=n, stop_token_ids=[stop], return_reasons=True, ignore_eos=True)
    for g, w, r in zip(got, want, reasons):
        assert g == (w[: w.index(stop)] if stop in w else w) and r == ("stop" if stop in w else "length")


@gpu
def test_generate_shared_in_bfloat16_stays_with_the_plain_model(tmp_path):
    import janus_b200
    import plain_llama as P
    from helpers import BF16_TOL, TINY_A, make_model_dir, random_tokens
    d = make_model_dir(TINY_A, str(tmp_path), seed=1, dtype="bfloat16")
    cfg, w = P.read_model_dir(d)
    model = janus_b200.load(d, dtype="bfloat16", max_tokens=2048)
    prefix = random_tokens(70, cfg["vocab_size"], 1)
    prompts = [random_tokens(n, cfg["vocab_size"], 10 + n) for n in (1, 4, 8)]
    out, stats = model.generate_shared(prefix, prompts, max_tokens=16, drafts=3, ignore_eos=True, drafter=EveryToken)
    assert stats.drafted > 0
    for p, o in zip(prompts, out):
        logits = P.forward(cfg, w, prefix + p + o)
        for j, t in enumerate(o):
            row = logits[len(prefix) + len(p) - 1 + j]
            assert float(row.max() - row[t]) <= BF16_TOL * float(row.abs().max())


@gpu
def test_generate_shared_draws_like_the_model(tmp_path):
    """At a temperature the first tokens of many requests follow the model's distribution, drafts or not, and a seed repeats them."""
    import janus_b200
    import plain_llama as P
    from helpers import TINY_A, make_model_dir, random_tokens
    d = make_model_dir(TINY_A, str(tmp_path), seed=4, dtype="float32")
    cfg, w = P.read_model_dir(d)
    model = janus_b200.load(d, dtype="float32", max_tokens=65536, max_slots=1024)
    prefix, n = random_tokens(64, cfg["vocab_size"], 3), 900
    p = torch.softmax(P.forward(cfg, w, prefix + [5])[-1].double() / 0.05, 0).numpy()
    one, _ = model.generate_shared(prefix, [[5]] * n, max_tokens=3, drafts=2, temperature=0.05, seed=7, ignore_eos=True, drafter=EveryToken)
    two, _ = model.generate_shared(prefix, [[5]] * n, max_tokens=3, drafts=2, temperature=0.05, seed=7, ignore_eos=True, drafter=EveryToken)
    assert one == two
    count = np.bincount([o[0] for o in one], minlength=len(p))
    # n draws: a token's count has standard deviation sqrt(n p (1 - p)); five of them, and a little for the rarest
    assert (np.abs(count - n * p) <= 5.0 * np.sqrt(n * p * (1.0 - p)) + 2.0).all()


@gpu
def test_generate_shared_refusals(tmp_path):
    import janus_b200
    from helpers import TINY_A, make_model_dir
    from janus_b200.cache import CacheFull
    from janus_b200.engine.step import StepError
    folder = make_model_dir(TINY_A, str(tmp_path), seed=0, dtype="float32")
    model = janus_b200.load(folder, dtype="float32", max_tokens=192)
    for error, args in ((ValueError, dict(prefix=[], prompts=[[]])), (StepError, dict(prefix=[1] * 100, prompts=[[1] * 40])),
                        (StepError, dict(prefix=[1], prompts=[[999]])), (ValueError, dict(prefix=[1], prompts=[[1]], drafts=-1)),
                        (ValueError, dict(prefix=[1], prompts=[[1]], temperature=-0.5))):
        with pytest.raises(error):
            model.generate_shared(**{**dict(max_tokens=4), **args})
    small = janus_b200.load(folder, dtype="float32", max_tokens=64, max_slots=2)     # one page: the prefix takes it
    with pytest.raises(CacheFull):
        small.generate_shared([1] * 64, [[1, 2]], max_tokens=4)
    for m in (model, small):
        m.engine.cache.check()
        assert m.engine.cache.groups[0].pool.n_held == 0
    with pytest.raises(ValueError, match="grouped-query attention"):
        from janus_b200.engine.shared_prefix import SharedPrefixRunner
        model.engine.cache.states[0] = torch.zeros(1)
        SharedPrefixRunner(model.engine)
