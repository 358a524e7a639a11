"""The operators of beam search over a paged cache, as cases that can be timed and compared: every request keeps several
continuations (beams), whose pages are shared as long as their tokens are.

select     the beams that go on and the ones that end, from a step's logits over all beams and the whole vocabulary
           (`ops.beam_select`)
fork       the block tables of the beams that go on: pages shared, given back and taken, and the copies that rows on
           partly filled pages need (`ops.fork_pages`)
copy       those copies, in the key and value pages of all layers (`ops.copy_pages`)
reorder    fixed-size states of layers that keep some, moved to the rows of the beams that go on (`ops.reorder_rows`)
attention  one query token for each beam, pages that the beams of a request share read once for all of them
           (`ops.attention_beams`)

The plain forms are elementary torch operations: 64 bits where continuations are compared with one another (a sum over a
vocabulary in 32 bits could turn two of them round), 32 bits in attention, whole numbers elsewhere.
"""
import math

import numpy as np
import torch

own = False

PAGE = 64
NONE = -math.inf


# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------
def _select(name, requests, beams, vocab, stops, first=False, rounded=False, masked=0.0):
    return dict(name=name, op="select", requests=requests, beams=beams, vocab=vocab, stops=stops, first=first, rounded=rounded,
                masked=masked)


def _fork(name, requests, beams, len_lo, len_hi, width, tail, dead):
    return dict(name=name, op="fork", requests=requests, beams=beams, len_lo=len_lo, len_hi=len_hi, width=width, tail=tail, dead=dead)


def _copy(name, rows, copies, tensors, heads, dim, dtype="bfloat16"):
    return dict(name=name, op="copy", rows=rows, copies=copies, tensors=tensors, heads=heads, dim=dim, dtype=dtype)


def _reorder(name, requests, beams, matrices, numbers, spare):
    return dict(name=name, op="reorder", requests=requests, beams=beams, matrices=matrices, numbers=numbers, spare=spare)


def _attention(name, requests, beams, len_lo, len_hi, tail, heads, kv_heads, dim):
    return dict(name=name, op="attention", requests=requests, beams=beams, len_lo=len_lo, len_hi=len_hi, tail=tail, heads=heads,
                kv_heads=kv_heads, dim=dim)


def listed():
    return [
        # one request, four beams, the smallest vocabulary of the benchmarks; latency
        _select("select_1x4", 1, 4, 32000, 1),
        # a batch's first step: one live beam a request; an odd vocabulary, two stop tokens, logits rounded as bfloat16
        # models leave them (many ties) and a tenth of them masked
        _select("select_12x5_first", 12, 5, 50001, 2, first=True, rounded=True, masked=0.1),
        # the largest batch on the large vocabulary
        _select("select_64x8", 64, 8, 128256, 1),
        # one request in the middle of a page; latency
        _fork("fork_1x4", 1, 4, 700, 700, 16, 90, 0.0),
        # a full server behind long prompts, some beams without a continuation
        _fork("fork_64x8", 64, 8, 900, 16000, 256, 400, 0.05),
        # what one request's fork leaves to be copied, the 1B layers' pages; latency
        _copy("copy_4_rows", 4, 2, 32, 8, 64),
        # what a full server's fork leaves, the 8B layers' pages in 16 of the layers
        _copy("copy_512_rows", 512, 220, 32, 8, 128),
        # one request, six layers with a matrix state a head; latency
        _reorder("reorder_1x4", 1, 4, 6, 16 * 64 * 64, 3),
        # a batch, twelve layers of 16 heads with a 64 x 128 state each, five beams a request; slots that are not in use beside
        _reorder("reorder_40x5", 40, 5, 12, 16 * 64 * 128, 20),
        # one request, four beams behind a short prompt, the 8B layers' heads; latency
        _attention("attention_1x4", 1, 4, 300, 300, 60, 32, 8, 128),
        # ragged requests of an odd number of beams that parted long ago, groups of seven heads of 64
        _attention("attention_6x5_parted", 6, 5, 150, 5000, 700, 14, 2, 64),
        # the largest batch: eight beams each behind long prompts
        _attention("attention_16x8_long", 16, 8, 6000, 24000, 150, 32, 8, 128),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    """A case of the ranges above: 1 to 64 requests of 1 to 16 beams over vocabularies of 1,000 to 128,256; tables of up to 256 pages;
    up to 512 rows of pages to copy; up to 40 requests' states; attention over 1 to 24,000 tokens."""
    op = rng.choice(["select", "fork", "copy", "reorder", "attention", "attention"])
    beams = rng.choice([1, 2, 3, 4, 5, 6, 8, 8, 10, 16])
    if op == "select":
        vocab = rng.choice([32000, 128256, _log_int(rng, 1000, 128256)])
        return _select("", _log_int(rng, 1, max(1, 512 // beams)), beams, vocab, rng.randint(0, 3), rng.random() < 0.3, rng.random() < 0.5,
                       rng.choice([0.0, 0.0, 0.3]))
    if op == "fork":
        lo = _log_int(rng, 1, 8000)
        hi = lo + _log_int(rng, 1, 8000)
        return _fork("", _log_int(rng, 1, max(1, 512 // beams)), beams, lo, hi, hi // PAGE + rng.randint(1, 6), _log_int(rng, 1, 400),
                     rng.choice([0.0, 0.1]))
    if op == "copy":
        rows = _log_int(rng, 1, 512)
        return _copy("", rows, rng.randint(0, max(1, 2 * rows // 5)), rng.randint(2, 32), rng.choice([1, 2, 4, 8]),
                     rng.choice([64, 128, 80, 96, 40]), rng.choice(["bfloat16", "bfloat16", "float32"]) if rows < 200 else "bfloat16")
    if op == "reorder":
        return _reorder("", _log_int(rng, 1, max(1, 200 // beams)), beams, rng.randint(1, 12), _log_int(rng, 64, 16 * 64 * 128),
                        rng.randint(0, 20))
    kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 4, 7, 8])
    lo = _log_int(rng, 1, 6000)
    return _attention("", _log_int(rng, 1, max(1, 128 // beams)), beams, lo, lo + _log_int(rng, 1, 18000), _log_int(rng, 1, 700),
                      kv_heads * group, kv_heads, rng.choice([64, 128, 128, 80, 96]))


def _spread(n, lo, hi):
    """n lengths from lo to hi, spread evenly over their logarithms (the same for every seed: what a pass costs is fixed)."""
    return [min(hi, lo + round(math.expm1(math.log1p(hi - lo) * (i + 0.5) / n))) if n > 1 else (lo + hi + 1) // 2 for i in range(n)]


def _pages(n):
    return (n + PAGE - 1) // PAGE


def prepare(case, seed):
    return {"select": _prepare_select, "fork": _prepare_fork, "copy": _prepare_copy, "reorder": _prepare_reorder,
            "attention": _prepare_attention}[case["op"]](case, seed)


def run(state):
    op = state["case"]["op"]
    if own:
        return {"select": _own_select, "fork": _own_fork, "copy": _own_copy, "reorder": _own_reorder, "attention": _own_attention}[op](state)
    return {"select": _plain_select, "fork": _plain_fork, "copy": _plain_copy, "reorder": _plain_reorder,
            "attention": _plain_attention}[op](state)


def exact(case, seed):
    make = {"select": _exact_select, "fork": _exact_fork, "attention": _exact_attention}.get(case["op"])
    return make(prepare(case, seed)) if make is not None else None      # (copies have nothing that is computed)


def work(case):
    return {"select": _work_select, "fork": _work_fork, "copy": _work_copy, "reorder": _work_reorder,
            "attention": _work_attention}[case["op"]](case)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _workspace():
    from janus_b200.engine.workspace import Workspace
    return Workspace(torch.device("cuda", torch.cuda.current_device()))


def _new(*shape, dtype=torch.int32):
    return torch.empty(shape, dtype=dtype, device="cuda")


def _survivors(beams, g, lost=0.4):
    """A parent for each beam of a request, as a step of beam search leaves them: beams that go on keep their row, the rows of the
    others take second continuations."""
    stays = torch.rand(beams, generator=g) >= lost
    if not bool(stays.any()):
        stays[int(torch.randint(0, beams, (1,), generator=g))] = True
    alive = stays.nonzero()[:, 0]
    pick = alive[torch.randint(0, len(alive), (beams,), generator=g)]
    return torch.where(stays, torch.arange(beams), pick)


# ---------------------------------------------------------------------------------------------
# select: log-probabilities log softmax(x) of every beam's row; a continuation's total is its beam's score plus its
# log-probability.  Continuations are ordered by total, then by beam and token.  The K best that are no stop token go on; a
# stop token among the K best of all ends.  A beam's best continuation keeps the beam's row, the others take the rows left.
# ---------------------------------------------------------------------------------------------
def _prepare_select(case, seed):
    R, K, V = case["requests"], case["beams"], case["vocab"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.Generator().manual_seed(seed + 1)
    logits = torch.randn((R * K, V), generator=g, device="cuda") * 2.5
    # a row's text prefers some tokens by far
    favourites = torch.randint(0, V, (R * K, 12), generator=g, device="cuda")
    logits.scatter_(1, favourites, torch.randn((R * K, 12), generator=g, device="cuda") * 2.0 + 11.0)
    stops = torch.randperm(V, generator=h)[: case["stops"]].sort().values
    if len(stops):
        logits[:, stops.cuda()] = torch.randn((R * K, len(stops)), generator=g, device="cuda") * 3.0 + 10.0
    if case["rounded"]:
        logits = logits.bfloat16().float()
    if case["masked"]:
        out = torch.rand((R * K, V), generator=g, device="cuda") < case["masked"]
        logits.masked_fill_(out, NONE)
        logits[0].clamp_min_(torch.finfo(torch.float32).min)       # ... one row by the type's lowest value
    scores = -torch.rand((R, K), generator=h).cumsum(1) * 2.0 - 20.0 * torch.rand((R, 1), generator=h)
    if case["first"]:
        scores[:, 0], scores[:, 1:] = 0.0, NONE
    return dict(case=case, logits=logits, scores=scores.float().cuda(), stops=stops.int().cuda(), workspace=_workspace() if own else None)


def _own_select(s):
    from janus_b200.kernels import ops
    R, K = s["scores"].shape
    out = dict(parents=_new(R, K), tokens=_new(R, K), next_scores=_new(R, K, dtype=torch.float32), ended_parents=_new(R, K),
               ended_tokens=_new(R, K), ended_scores=_new(R, K, dtype=torch.float32))
    ops.beam_select(s["logits"], s["scores"], s["stops"], **out, workspace=s["workspace"])
    return out


def _best(flat, count):
    """The `count` largest of each row in order, the lowest index first among equals: (values, indices)."""
    flat = flat.clone()
    values, indices = [], []
    for _ in range(count):
        i = flat.argmax(1, keepdim=True)
        values.append(flat.gather(1, i))
        indices.append(i)
        flat.scatter_(1, i, NONE)
    return torch.cat(values, 1), torch.cat(indices, 1)


def _plain_select(s):
    R, K = s["scores"].shape
    x = s["logits"].view(R, K, -1).double()
    V = x.shape[2]
    x = torch.where(torch.isnan(x), NONE, x)
    top = x.amax(2, keepdim=True)
    z = torch.where(top == math.inf, torch.where(x == math.inf, 0.0, NONE), torch.where(top == NONE, NONE, x - top))
    logp = z - z.exp().sum(2, keepdim=True).log()
    total = s["scores"].double()[:, :, None] + logp
    total = torch.where(torch.isnan(total), NONE, total)
    is_stop = torch.zeros(V, dtype=torch.bool, device=x.device)
    is_stop[s["stops"].long()] = True
    on, on_at = _best(torch.where(is_stop, NONE, total).view(R, K * V), K)
    end, end_at = _best(torch.where(is_stop, total, NONE).view(R, K * V), K)
    # how many continuations that go on stand in front of each stop token
    before = (on[:, None, :] > end[:, :, None]) | ((on[:, None, :] == end[:, :, None]) & (on_at[:, None, :] < end_at[:, :, None]))
    ends = (before.sum(2) + torch.arange(K, device=x.device) < K) & (end > NONE)
    parent, token = on_at // V, on_at % V
    live = on > NONE
    # rows: the first continuation of a beam keeps its row
    earlier = torch.ones((K, K), dtype=torch.bool, device=x.device).tril(-1)
    first = live & ~((parent[:, :, None] == parent[:, None, :]) & live[:, None, :] & earlier).any(2)
    rows = torch.arange(K, device=x.device)
    kept = ((parent[:, :, None] == rows) & first[:, :, None]).any(1)                     # [R, row]
    free = torch.where(kept, K, rows).sort(1).values                                     # rows left, in order
    nth = (~first).long().cumsum(1) - 1
    row = torch.where(first, parent, free.gather(1, nth.clamp_min(0)))
    put = lambda v: torch.zeros_like(v).scatter_(1, row, v)      # noqa: E731
    i32 = lambda v: v.to(torch.int32)      # noqa: E731
    return dict(parents=i32(put(torch.where(live, parent, -1))), tokens=i32(put(torch.where(live, token, 0))),
                next_scores=put(on).float(), ended_parents=i32(torch.where(ends, end_at // V, -1)),
                ended_tokens=i32(torch.where(ends, end_at % V, -1)), ended_scores=torch.where(ends, end, NONE).float())


def _exact_select(s):
    logits, scores, stops = s["logits"].cpu().numpy(), s["scores"].cpu().numpy().astype(np.float64), set(s["stops"].tolist())
    R, K = scores.shape
    V = logits.shape[1]
    made = {k: np.zeros((R, K), np.int64) for k in ("parents", "tokens", "ended_parents", "ended_tokens")}
    made.update(next_scores=np.full((R, K), NONE), ended_scores=np.full((R, K), NONE))
    made["parents"] -= 1
    made["ended_parents"] -= 1
    made["ended_tokens"] -= 1
    for r in range(R):
        found = []
        for k in range(K):
            x = logits[r * K + k].astype(np.float64)
            if not scores[r, k] > NONE or not x.max() > NONE:
                continue
            m = x.max()
            base = scores[r, k] - m - math.log(np.exp(x - m).sum())
            n = min(V, K + len(stops))
            edge = np.partition(x, V - n)[V - n]
            for t in np.nonzero(x >= max(edge, -1e308))[0]:
                found.append((-(base + x[t]), k * V + int(t)))
        found.sort()
        on = [f for f in found if f[1] % V not in stops][:K]
        ended = [f for f in found[:K] if f[1] % V in stops]
        for j, (total, at) in enumerate(ended):
            made["ended_parents"][r, j], made["ended_tokens"][r, j], made["ended_scores"][r, j] = at // V, at % V, -total
        taken, later = set(), []
        for total, at in on:
            if at // V in taken:
                later.append((total, at))
                continue
            taken.add(at // V)
            made["parents"][r, at // V], made["tokens"][r, at // V], made["next_scores"][r, at // V] = at // V, at % V, -total
        for row, (total, at) in zip([k for k in range(K) if k not in taken], later):
            made["parents"][r, row], made["tokens"][r, row], made["next_scores"][r, row] = at // V, at % V, -total
    return made


def _work_select(case):
    n = case["requests"] * case["beams"]
    return {"bytes": 4 * n * case["vocab"] + 28 * n + 4 * case["stops"], "flops": 4 * n * case["vocab"]}


# ---------------------------------------------------------------------------------------------
# fork: row r K + k goes on with the pages of row r K + parents[r, k].  Full pages are shared.  A partly filled page stays with
# the lowest row that holds it if nobody else holds it; other rows take a page of their own and a copy.  Rows at the end of a
# page take a new one.  refs counts the holders of a page; at 0 it comes back, behind the free pages, in order of number.
# ---------------------------------------------------------------------------------------------
def _prepare_fork(case, seed):
    R, K, W = case["requests"], case["beams"], case["width"]
    g = torch.Generator().manual_seed(seed)
    lengths = _spread(R, case["len_lo"], case["len_hi"])
    parents = torch.stack([_survivors(K, g) for _ in range(R)])
    parents[torch.rand((R, K), generator=g) < case["dead"]] = -1
    if case["dead"]:
        parents[R // 2] = -1                                          # a request that is over
    # pages that all beams of a request share, then those since the beams parted, some of them shared by two
    n_pages, plan = 1, []                                             # page 0: where rows that do not go on lie
    for r, n in enumerate(lengths):
        common = max(0, n - 1 - (37 * r + 11) % case["tail"]) // PAGE
        plan.append((n_pages, common))
        n_pages += common + K * (_pages(n) - common)
    spare = 2 * R * K
    order = torch.cat([torch.zeros(1, dtype=torch.long), 1 + torch.randperm(n_pages + spare - 1, generator=g)])
    table = np.full((R, K, W), -1, np.int64)
    refs = np.zeros(n_pages + spare, np.int64)
    for r, (n, (at, common)) in enumerate(zip(lengths, plan)):
        pages = _pages(n)
        table[r, :, :common] = np.arange(at, at + common)
        own_pages = np.arange(at + common, at + common + K * (pages - common)).reshape(K, pages - common)
        if K > 1 and pages - common > 1:
            own_pages[1, :-1] = own_pages[0, :-1]                     # the first two beams parted in their last page
        table[r, :, common:pages] = own_pages
        refs[at: at + common // 2] += 1                               # the prompt's whole pages are the request's own as well
    flat = order.numpy()[table] * (table >= 0) - (table < 0)
    refs_of = np.zeros_like(refs)
    refs_of[order.numpy()] = refs
    np.add.at(refs_of, flat[flat >= 0], 1)
    free = np.nonzero(refs_of[1:] == 0)[0] + 1
    free = free[torch.randperm(len(free), generator=g).numpy()]
    free_pages = np.full(n_pages + spare, -1, np.int64)
    free_pages[: len(free)] = free
    return dict(case=case, parents=parents.int().cuda(), lengths=_ints([[n] * K for n in lengths]), table=_ints(flat.reshape(R * K, W)),
                refs=_ints(refs_of), free_pages=_ints(free_pages), n_free=_ints([len(free)]))


def _own_fork(s):
    from janus_b200.kernels import ops
    (R, K), W, P, F = s["parents"].shape, s["table"].shape[1], s["refs"].shape[0], s["free_pages"].shape[0]
    out = dict(kv_len=_new(R, K), positions=_new(R, K), dest_rows=_new(R, K), new_table=_new(R * K, W), new_refs=_new(P), new_free=_new(F),
               new_n_free=_new(1), copy_src=_new(R, K), copy_dst=_new(R, K), copy_rows=_new(R, K), shared=_new(R), missing=_new(1))
    ops.fork_pages(s["parents"], s["lengths"], s["table"], s["refs"], s["free_pages"], s["n_free"], **out, spare=0, page_size=PAGE)
    return out


def _plain_fork(s):
    (R, K), W, P, F = s["parents"].shape, s["table"].shape[1], s["refs"].shape[0], s["free_pages"].shape[0]
    dev = s["parents"].device
    N, spare = R * K, 0
    parent = s["parents"].long()
    live = ((parent >= 0) & (parent < K)).view(N)
    source = (parent.clamp(0, K - 1) + K * torch.arange(R, device=dev)[:, None]).view(N)
    before = s["lengths"].long().view(N)
    length = torch.where(live, before[source], 0)
    cols = torch.arange(W, device=dev)
    old = s["table"].long()
    table = torch.where(live[:, None] & (cols < ((length + PAGE - 1) // PAGE)[:, None]), old[source], -1)
    count = lambda t: torch.zeros(P + 1, dtype=torch.long, device=dev).index_add_(      # noqa: E731
        0, torch.where((t >= 0) & (t < P) & (t != spare), t, P).reshape(-1), torch.ones(t.numel(), dtype=torch.long, device=dev))[:P]
    refs_before = s["refs"].long()
    refs = refs_before + count(table) - count(torch.where(cols < ((before + PAGE - 1) // PAGE)[:, None], old, -1))
    # pages that nobody holds any longer follow the free ones, in order of number
    freed = (refs == 0) & (refs_before > 0)
    n0 = s["n_free"].long().clamp(0, F)
    places = torch.where(freed, n0 + freed.long().cumsum(0) - 1, F + P).clamp_max(F + P)
    pool = torch.full((F + P + 1,), -1, dtype=torch.long, device=dev)
    pool[:F] = torch.where(torch.arange(F, device=dev) < n0, s["free_pages"].long(), -1)
    pool.scatter_(0, places, torch.arange(P, device=dev))
    pool[F + P] = -1
    total = n0 + freed.sum()
    # who keeps a partly filled page
    at, part = length // PAGE, length % PAGE
    fits = at < W
    held = table.gather(1, at.clamp_max(W - 1)[:, None])[:, 0]
    held = torch.where(live & fits & (part > 0) & (held >= 0) & (held < P), held, -1)
    same = (held.view(R, K)[:, :, None] == held.view(R, K)[:, None, :]) & (held.view(R, K) >= 0)[:, :, None]
    lowest = ~(same & torch.ones((K, K), dtype=torch.bool, device=dev).tril(-1)).any(2)
    alone = same.sum(2).view(N) == refs[held.clamp_min(0)]
    keeps = (held >= 0) & lowest.view(N) & alone
    needs = live & fits & ~keeps
    i = total - needs.long().cumsum(0)
    fresh = torch.where(needs & (i >= 0), pool[i.clamp_min(0)], -1)
    gives = needs & (held >= 0)
    refs = refs - count(torch.where(gives, held, -1))
    refs = torch.cat([refs, refs.new_zeros(1)]).scatter_(0, torch.where(fresh >= 0, fresh, P), 1)[:P]
    page = torch.where(keeps, held, fresh)
    first = torch.where(live, page, spare)
    column = torch.where(live, at, 0)
    table = torch.where((cols == column[:, None]) & (fits | ~live)[:, None], first[:, None], table)
    left = (total - needs.sum()).clamp_min(0)
    n_free = left.clamp_max(F)
    lacking = (needs & (fresh < 0)).sum() + (live & ~fits).sum() + (left - F).clamp_min(0)
    copies = gives & (fresh >= 0)
    ok = live & (page >= 0)
    # leading whole pages that all live beams of a request have in common
    lead = torch.where(live, at.clamp_max(W), W).view(R, K).amin(1)
    head = live.view(R, K).long().argmax(1) + K * torch.arange(R, device=dev)
    differs = ((table != table[head].repeat_interleave(K, 0)) & live[:, None]).view(R, K, W).any(1)
    lead = torch.minimum(lead, torch.where(differs, cols, W).amin(1))
    lead = torch.where(live.view(R, K).any(1), lead, 0)
    i32 = lambda v, *shape: v.to(torch.int32).view(*shape)      # noqa: E731
    return dict(kv_len=i32(torch.where(live, length + 1, 1), R, K), positions=i32(torch.where(live, length, 0), R, K),
                dest_rows=i32(torch.where(ok, page * PAGE + part, spare * PAGE), R, K), new_table=i32(table, N, W), new_refs=i32(refs, P),
                new_free=i32(torch.where(torch.arange(F, device=dev) < n_free, pool[:F], -1), F), new_n_free=i32(n_free, 1),
                copy_src=i32(torch.where(copies, held, -1), R, K), copy_dst=i32(torch.where(copies, fresh, -1), R, K),
                copy_rows=i32(torch.where(copies, part, 0), R, K), shared=i32(lead, R), missing=i32(lacking, 1))


def _exact_fork(s):
    parents, lengths, old = s["parents"].tolist(), s["lengths"].tolist(), s["table"].tolist()
    R, K, W = len(parents), len(parents[0]), len(old[0])
    refs, free = s["refs"].tolist(), s["free_pages"].tolist()
    F, pool = len(free), free[: s["n_free"].item()]
    table, dead = [], [[not 0 <= p < K for p in row] for row in parents]
    for r in range(R):
        for k in range(K):
            row = [-1] * W
            if not dead[r][k]:
                n = _pages(lengths[r][parents[r][k]])
                row[:n] = old[r * K + parents[r][k]][:n]
            table.append(row)
    before = list(refs)
    for row in table:
        for p in row:
            if p > 0:
                refs[p] += 1
    for i, row in enumerate(old):
        for p in row[: _pages(lengths[i // K][i % K])]:
            if p > 0:
                refs[p] -= 1
    pool += [p for p in range(len(refs)) if refs[p] == 0 and before[p] > 0]
    out = {k: [[0] * K for _ in range(R)] for k in ("kv_len", "positions", "dest_rows", "copy_src", "copy_dst", "copy_rows")}
    missing, gave = 0, []
    shared = [0] * R
    for r in range(R):
        rows = table[r * K: r * K + K]
        ends = [0 if dead[r][k] else lengths[r][parents[r][k]] for k in range(K)]
        held = [rows[k][ends[k] // PAGE] if not dead[r][k] and ends[k] % PAGE and ends[k] // PAGE < W else -1 for k in range(K)]
        for k in range(K):
            out["copy_src"][r][k] = out["copy_dst"][r][k] = -1
            if dead[r][k]:
                rows[k][0] = 0
                out["kv_len"][r][k] = 1
                continue
            at, part = ends[k] // PAGE, ends[k] % PAGE
            out["kv_len"][r][k], out["positions"][r][k] = ends[k] + 1, ends[k]
            if at >= W:
                missing += 1
                continue
            if held[k] >= 0 and held.index(held[k]) == k and held.count(held[k]) == refs[held[k]]:
                page = held[k]
            else:
                page = pool.pop() if pool else -1
                missing += page < 0
                if held[k] >= 0:
                    gave.append(held[k])
                    if page >= 0:
                        out["copy_src"][r][k], out["copy_dst"][r][k], out["copy_rows"][r][k] = held[k], page, part
                if page >= 0:
                    gave.append(-page)
            rows[k][at] = page
            out["dest_rows"][r][k] = page * PAGE + part if page >= 0 else 0
        alive = [k for k in range(K) if not dead[r][k]]
        if alive:
            while shared[r] < min(min(ends[k] // PAGE for k in alive), W) and len({rows[k][shared[r]] for k in alive}) == 1:
                shared[r] += 1
    for p in gave:
        if p < 0:
            refs[-p] = 1
        else:
            refs[p] -= 1
    out.update(new_table=table, new_refs=refs, new_free=(pool + [-1] * F)[:F], new_n_free=[min(len(pool), F)],
               shared=shared, missing=[missing + max(0, len(pool) - F)])
    return {k: np.array(v) for k, v in out.items()}


def _work_fork(case):
    # entries that change are the rows of beams that do not stay, from the shared pages on; counted as two fifths of the rows' tails;
    # every row of the new table is an output of its own, as are the pages' counts and the free list
    n = case["requests"] * case["beams"]
    pages = sum(_pages(x) * case["beams"] for x in _spread(case["requests"], case["len_lo"], case["len_hi"]))
    return {"bytes": 8 * n * case["width"] + 16 * pages + 40 * n, "flops": 0}


# ---------------------------------------------------------------------------------------------
# copy: for every row with a page to copy, the first tokens of every head of the page, in all tensors
# ---------------------------------------------------------------------------------------------
def _prepare_copy(case, seed):
    g, h = torch.Generator(device="cuda").manual_seed(seed), torch.Generator().manual_seed(seed + 1)
    N, C = case["rows"], case["copies"]
    pages = N + C + 3
    shape, dtype = (pages, case["heads"], PAGE, case["dim"]), getattr(torch, case["dtype"])
    tensors = [torch.randn(shape, generator=g, device="cuda", dtype=dtype) for _ in range(case["tensors"])]
    order = torch.randperm(pages, generator=h)
    src, dst, rows = (torch.full((N,), v, dtype=torch.long) for v in (-1, -1, 0))
    which = torch.randperm(N, generator=h)[:C]
    # two rows in three are copied from a page that another row copies too
    src[which], dst[which] = order[torch.randint(0, max(1, (2 * C + 2) // 3), (C,), generator=h)], order[N: N + C]
    # ends of pages, evenly over their tokens (the same for every seed)
    rows[which] = torch.tensor([1 + (i * 62) // max(1, C - 1) for i in range(C)], dtype=torch.long)
    return dict(case=case, tensors=tensors, src=src.int().cuda(), dst=dst.int().cuda(), rows=rows.int().cuda())


def _own_copy(s):
    from janus_b200.kernels import ops
    ops.copy_pages(s["tensors"], s["src"], s["dst"], s["rows"])
    return s["tensors"]


def _plain_copy(s):
    some = (s["src"] >= 0).nonzero()[:, 0]
    src, dst, rows = s["src"][some].long(), s["dst"][some].long(), s["rows"][some]
    taken = (torch.arange(PAGE, device=rows.device) < rows[:, None])[:, None, :, None]
    for t in s["tensors"]:
        t[dst] = torch.where(taken, t[src], t[dst])
    return s["tensors"]


def _work_copy(case):
    rows = sum(1 + (i * 62) // max(1, case["copies"] - 1) for i in range(case["copies"]))
    size = 2 if case["dtype"] == "bfloat16" else 4
    return {"bytes": (2 * rows * case["heads"] * case["dim"] * size) * case["tensors"] + 12 * case["rows"], "flops": 0}


# ---------------------------------------------------------------------------------------------
# reorder: the state in row slots[r K + k] becomes the one in row slots[r K + parents[r, k]], in every matrix
# ---------------------------------------------------------------------------------------------
def _prepare_reorder(case, seed):
    R, K = case["requests"], case["beams"]
    g, h = torch.Generator(device="cuda").manual_seed(seed), torch.Generator().manual_seed(seed + 1)
    n = R * K + case["spare"]
    matrices = [torch.randn((n, case["numbers"]), generator=g, device="cuda") for _ in range(case["matrices"])]
    parents = torch.stack([_survivors(K, h) for _ in range(R)])
    return dict(case=case, matrices=matrices, parents=parents.int().cuda(), slots=torch.randperm(n, generator=h)[: R * K].int().cuda())


def _own_reorder(s):
    from janus_b200.kernels import ops
    ops.reorder_rows(s["matrices"], s["slots"], s["parents"])
    return s["matrices"]


def _plain_reorder(s):
    R, K = s["parents"].shape
    parents = s["parents"].long()
    rows = torch.arange(K, device=parents.device)
    parents = torch.where((parents >= 0) & (parents < K), parents, rows)
    source = (parents + K * torch.arange(R, device=parents.device)[:, None]).view(-1)
    slots = s["slots"].long()
    for m in s["matrices"]:
        m[slots] = m[slots[source]]
    return s["matrices"]


def _work_reorder(case):
    # two rows in five change, each from a row that is read once
    moved = 0.4 * (1 if case["beams"] > 1 else 0) * case["requests"] * case["beams"]
    return {"bytes": int(1.8 * 4 * moved * case["numbers"]) * case["matrices"] + 8 * case["requests"] * case["beams"], "flops": 0}


# ---------------------------------------------------------------------------------------------
# attention: softmax(q K' / sqrt(d)) V of every beam's one query over its kv_len keys; the first shared[r] pages of a request's beams
# are the same
# ---------------------------------------------------------------------------------------------
def _lengths(case):
    lengths = _spread(case["requests"], case["len_lo"], case["len_hi"])
    tails = [(37 * r + 11) % case["tail"] + 1 for r in range(case["requests"])]
    return lengths, [max(0, n - t) // PAGE for n, t in zip(lengths, tails)]


def _prepare_attention(case, seed):
    R, K, nkv, hd = case["requests"], case["beams"], case["kv_heads"], case["dim"]
    g, h = torch.Generator(device="cuda").manual_seed(seed), torch.Generator().manual_seed(seed + 1)
    lengths, shared = _lengths(case)
    width = max(_pages(n) for n in lengths) + 1
    n_pages, table = 0, np.full((R, K, width), -1, np.int64)
    for r, (n, common) in enumerate(zip(lengths, shared)):
        table[r, :, :common] = np.arange(n_pages, n_pages + common)
        n_pages += common
        rest = _pages(n) - common
        table[r, :, common: common + rest] = np.arange(n_pages, n_pages + K * rest).reshape(K, rest)
        n_pages += K * rest
    order = torch.randperm(n_pages, generator=h).numpy()
    table = order[table] * (table >= 0) - (table < 0)
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)      # noqa: E731
    return dict(case=case, q=normal(R * K, case["heads"] * hd) * 2, k=normal(n_pages, nkv, PAGE, hd), v=normal(n_pages, nkv, PAGE, hd),
                table=_ints(table.reshape(R * K, width)), kv_len=_ints([n for n in lengths for _ in range(K)]), shared=_ints(shared),
                workspace=_workspace() if own else None)


def _own_attention(s):
    from janus_b200.kernels import ops
    c, q = s["case"], s["q"]
    out = torch.empty_like(q)
    ops.attention_beams(q, s["k"], s["v"], out, s["table"], s["kv_len"], s["shared"], c["beams"], c["heads"], c["kv_heads"], c["dim"], PAGE,
                        1.0 / math.sqrt(c["dim"]), s["workspace"], PAGE * s["table"].shape[1])
    return out


def _plain_attention(s):
    c = s["case"]
    K, nh, nkv, hd = c["beams"], c["heads"], c["kv_heads"], c["dim"]
    out = torch.empty_like(s["q"])
    lengths, _ = _lengths(c)
    for r, n in enumerate(lengths):
        rows = slice(r * K, r * K + K)
        pages = s["table"][rows, : _pages(n)].long()
        k, v = (t[pages].permute(0, 2, 1, 3, 4).reshape(K, nkv, -1, hd).float() for t in (s["k"], s["v"]))
        q = s["q"][rows].float().view(K, nkv, nh // nkv, hd)
        scores = (q @ k.transpose(2, 3)) * (1.0 / math.sqrt(hd))
        seen = torch.arange(k.shape[2], device=k.device) < s["kv_len"][rows, None]
        scores = torch.where(seen[:, None, None, :], scores, NONE)
        weights = torch.exp(scores - scores.amax(3, keepdim=True))
        out[rows] = ((weights @ v) / weights.sum(3, keepdim=True)).reshape(K, nh * hd).to(out.dtype)
    return out


def _exact_attention(s):
    c = s["case"]
    K, nh, nkv, hd = c["beams"], c["heads"], c["kv_heads"], c["dim"]
    out = torch.empty(s["q"].shape, dtype=torch.float64)
    for i in range(s["q"].shape[0]):
        n = int(s["kv_len"][i])
        at = torch.arange(n, device="cuda")
        page = s["table"][i].long()[at // PAGE]
        q = s["q"][i].double().view(nkv, nh // nkv, hd)
        for j in range(nkv):
            keys, values = s["k"][page, j, at % PAGE].double(), s["v"][page, j, at % PAGE].double()
            weights = torch.softmax(q[j] @ keys.T / math.sqrt(hd), 1)
            out[i, j * (nh // nkv) * hd: (j + 1) * (nh // nkv) * hd] = (weights @ values).reshape(-1).cpu()
    return out


def _work_attention(case):
    lengths, shared = _lengths(case)
    K = case["beams"]
    keys = sum(c * PAGE + K * (n - c * PAGE) for n, c in zip(lengths, shared))
    return {"bytes": 4 * keys * case["kv_heads"] * case["dim"] + 4 * case["requests"] * K * case["heads"] * case["dim"],
            "flops": 4 * sum(lengths) * K * case["heads"] * case["dim"]}
