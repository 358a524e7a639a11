"""Three operators of one serving step, as cases that can be timed and compared: many requests that share one long prompt
in front of their own tokens, each with a few drafted tokens that the step verifies.

tables     the step's index arrays on the device, from request lengths: pages taken from the free list and given back,
           block tables, the cache row of every new token (`ops.step_tables`)
attention  the step's queries over the shared prompt's pages, read once for all requests, and over each request's own
           pages, joined (`ops.attention_prefix`)
verify     drafted tokens accepted or refused against the target's logits from given random numbers, and the token
           that follows the accepted ones (`ops.verify_drafts`)

The plain forms are elementary torch operations in 32 bits; requests of unequal lengths are padded there.  Uniform
numbers that fall so near an edge that two correctly rounded sums may answer differently are moved when inputs are made.
"""
import math

import torch

own = False

PAGE = 64


# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------
def _tables(name, requests, new_lo, new_hi, len_lo, len_hi, width, prefix_pages, spare):
    return dict(name=name, op="tables", requests=requests, new_lo=new_lo, new_hi=new_hi, len_lo=len_lo, len_hi=len_hi, width=width,
                prefix_pages=prefix_pages, spare=spare)


def _attention(name, requests, new_lo, new_hi, prefix, own_lo, own_hi, heads, kv_heads, dim, dtype="bfloat16"):
    return dict(name=name, op="attention", requests=requests, new_lo=new_lo, new_hi=new_hi, prefix=prefix, own_lo=own_lo,
                own_hi=own_hi, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype)


def _verify(name, requests, drafts_lo, drafts_hi, vocab, temperature, probs):
    return dict(name=name, op="verify", requests=requests, drafts_lo=drafts_lo, drafts_hi=drafts_hi, vocab=vocab,
                temperature=temperature, probs=probs)


def listed():
    return [
        # the smallest decode step: four requests, one token each; latency
        _tables("tables_4_requests", 4, 1, 1, 70, 900, 16, 1, 0),
        # a decode step of a full server: one to six tokens each (the last one and its drafts), a quarter of the requests new
        _tables("tables_256_drafted", 256, 1, 6, 1030, 7900, 128, 16, 64),
        # prompts of very many requests beside each other behind long contexts, buffers laid out for more tokens
        _tables("tables_1024_prompts", 1024, 3, 190, 2100, 31000, 512, 32, 1000),
        # a handful of chats behind a short system prompt; latency
        _attention("attention_4_requests", 4, 1, 1, 1000, 5, 130, 32, 8, 128),
        # a full batch of single tokens behind a long system prompt, the 8B layers' heads
        _attention("attention_64_single_tokens", 64, 1, 1, 8192, 30, 700, 32, 8, 128),
        # drafted tokens, one to six a request, the 1B layers' heads; the prompt ends inside a page
        _attention("attention_48_drafted", 48, 1, 6, 6001, 20, 400, 32, 8, 64),
        # the largest batch: very many requests behind a long document, own contexts of very unequal lengths
        _attention("attention_256_long", 256, 1, 1, 16384, 3, 2500, 32, 8, 128),
        # the requests' own prompts behind the shared one, ragged, in one step
        _attention("attention_8_prompts", 8, 65, 510, 4100, 0, 3, 32, 8, 128),
        # the true 32-bit engine, a few drafted tokens
        _attention("attention_float32", 16, 1, 3, 2050, 9, 300, 16, 4, 128, "float32"),
        # one request whose drafts were looked up in its own text (no probabilities of a drafting model); latency
        _verify("verify_1_request", 1, 4, 4, 128256, 0.7, False),
        # a batch with the probabilities of a drafting model, a small vocabulary
        _verify("verify_64_requests", 64, 0, 6, 32000, 0.9, True),
        # the largest batch on the large vocabulary
        _verify("verify_256_requests", 256, 1, 5, 128256, 1.0, True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    """A case of the ranges above: 1 to 1,024 requests and 30,000 tokens for the tables, 1 to 256 requests behind prompts of 100 to
    16,384 tokens for attention, 1 to 256 requests of up to six drafts over vocabularies of 1,000 to 128,256 for verification."""
    op = rng.choice(["tables", "attention", "attention", "verify"])
    if op == "tables":
        requests = _log_int(rng, 1, 1024)
        new_hi = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 8, 190)])
        prefix_pages = rng.choice([0, rng.randint(1, 32)])
        len_lo = prefix_pages * PAGE + rng.randint(1, 300)
        len_hi = len_lo + _log_int(rng, 1, 28000)
        return _tables("", requests, rng.randint(0, 1) if new_hi < 9 else rng.randint(1, new_hi), new_hi, len_lo, len_hi,
                       (len_hi + new_hi + PAGE - 1) // PAGE + rng.randint(0, 40), prefix_pages, rng.choice([0, rng.randint(1, 1000)]))
    if op == "attention":
        kv_heads = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 3, 4, 5, 8])
        dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
        dim = rng.choice([64, 128, 128, 80, 96])
        prefix = _log_int(rng, 100, 16384 if dtype == "bfloat16" else 2100)
        if rng.random() < 0.25 and dtype == "bfloat16":
            requests, new_hi = rng.randint(1, 8), _log_int(rng, 20, 500)
            prefix = min(prefix, 4100)
            own_hi = rng.randint(1, 300)
        else:
            requests = _log_int(rng, 1, 256 if dtype == "bfloat16" else 16)
            new_hi = rng.choice([1, 1, rng.randint(2, 6)]) if requests <= 64 else 1
            own_hi = _log_int(rng, 2, 2500 if dtype == "bfloat16" else 300)
        return _attention("", requests, rng.randint(1, new_hi), new_hi, prefix, rng.randint(0, own_hi), own_hi, kv_heads * group,
                          kv_heads, dim, dtype)
    drafts_hi = rng.randint(1, 6)
    vocab = rng.choice([32000, 128256, _log_int(rng, 1000, 100000)])
    return _verify("", _log_int(rng, 1, 200 if drafts_hi > 4 else 256), rng.randint(0, drafts_hi), drafts_hi, vocab,
                   rng.choice([0.0, 0.6, 0.8, 1.0, 1.3]), rng.random() < 0.6)


def _spread(n, lo, hi):
    """n lengths from lo to hi, spread evenly over their logarithms (the same for every seed: what a pass costs is fixed)."""
    return [min(hi, lo + round(math.expm1(math.log1p(hi - lo) * (i + 0.5) / n))) if n > 1 else (lo + hi + 1) // 2 for i in range(n)]


def _pages(n):
    return (n + PAGE - 1) // PAGE


def _held(case, length):
    """Pages of a row of the last step's table: now and then one more than its tokens need, for drafts that were refused."""
    return min(case["width"], max(case["prefix_pages"], _pages(length) + (length % 3 == 0)))


def _room(case):
    """Places of the free list: every page of the pool fits."""
    lengths, new = _spread(case["requests"], case["len_lo"], case["len_hi"]), _spread(case["requests"], case["new_lo"], case["new_hi"])
    return sum(_held(case, n) + _pages(n) for n in lengths) + sum(_pages(n) + 1 for n in new) + case["prefix_pages"] + 7


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def prepare(case, seed):
    return {"tables": _prepare_tables, "attention": _prepare_attention, "verify": _prepare_verify}[case["op"]](case, seed)


def _shuffled(values, g):
    return [values[i] for i in torch.randperm(len(values), generator=g).tolist()]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _prepare_tables(case, seed):
    g = torch.Generator().manual_seed(seed)
    B, width, P0 = case["requests"], case["width"], case["prefix_pages"]
    new = _shuffled(_spread(B, case["new_lo"], case["new_hi"]), g)
    # three quarters go on from a row of the last step's table, in another order; the others begin behind the prefix
    requests = _shuffled([(n, i % 4 == 3) for i, n in enumerate(_spread(B, case["len_lo"], case["len_hi"]))], g)
    rows = _shuffled(list(range(B)), g)
    held = [0] * B
    for r, (n, _) in zip(rows, requests):
        held[r] = _held(case, n)
    lengths = [P0 * PAGE if begins else n for n, begins in requests]
    rows = [-1 if begins else r for r, (_, begins) in zip(rows, requests)]
    room = _room(case)
    ids = torch.randperm(room, generator=g).tolist()
    prefix, at = ids[:P0], P0
    table = torch.full((B, width), -1, dtype=torch.int32)
    for r in range(B):
        more = held[r] - P0
        table[r, :held[r]] = torch.tensor(prefix + ids[at:at + more], dtype=torch.int32)
        at += more
    free = ids[at:]
    total = sum(new) + case["spare"]
    return dict(op="tables", total=max(1, total), width=width, lengths=_ints(lengths), new=_ints(new), rows=_ints(rows), table=table.cuda(),
                held=_ints(held), prefix=_ints(prefix), free=_ints(free + [-1] * (room - len(free))), n_free=_ints([len(free)]))


def _prepare_attention(case, seed):
    g = torch.Generator().manual_seed(seed)
    d = torch.Generator(device="cuda").manual_seed(seed)
    B, H, G, D = case["requests"], case["heads"], case["kv_heads"], case["dim"]
    dtype = getattr(torch, case["dtype"])
    new = _shuffled(_spread(B, case["new_lo"], case["new_hi"]), g)
    before = _shuffled(_spread(B, case["own_lo"], case["own_hi"]), g)
    owned = [a + b for a, b in zip(new, before)]
    first, width = _pages(case["prefix"]), max(_pages(n) for n in owned)
    n_pages = first + sum(_pages(n) for n in owned) + 5
    ids = torch.randperm(n_pages, generator=g).tolist()
    table, at = torch.full((B, width), -1, dtype=torch.int32), first
    for b in range(B):
        k = _pages(owned[b])
        table[b, :k] = torch.tensor(ids[at:at + k], dtype=torch.int32)
        at += k
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    positions = [case["prefix"] + o - n + j for o, n in zip(owned, new) for j in range(n)]
    make = lambda *shape: torch.randn(shape, generator=d, device="cuda").to(dtype)      # noqa: E731
    return dict(op="attention", q=(1.5 * torch.randn((starts[-1], H * D), generator=d, device="cuda")).to(dtype), k=make(n_pages, G, PAGE, D),
                v=make(n_pages, G, PAGE, D), prefix_pages=_ints(ids[:first]), prefix=case["prefix"], table=table.cuda(),
                q_start=_ints(starts), kv_len=_ints([case["prefix"] + n for n in owned]), positions=_ints(positions),
                heads=H, kv_heads=G, dim=D, most_new=max(new), most_own=max(owned), scale=D ** -0.5)


def _prepare_verify(case, seed):
    g = torch.Generator().manual_seed(seed)
    d = torch.Generator(device="cuda").manual_seed(seed)
    B, V, heat = case["requests"], case["vocab"], case["temperature"]
    drafts = _shuffled(_spread(B, case["drafts_lo"], case["drafts_hi"]), g)
    starts = [0]
    for n in drafts:
        starts.append(starts[-1] + n + 1)
    T = starts[-1]
    # logits as language models give them: a broad floor and a few tokens that carry nearly all of the mass; some filtered out
    logits = 1.5 * torch.randn((T, V), generator=d, device="cuda")
    heads = torch.randint(0, V, (T, 16), generator=d, device="cuda")
    logits.scatter_(1, heads, math.log(V) + 1.2 + 2.0 * torch.randn((T, 16), generator=d, device="cuda"))
    logits[:, 5::97] = -math.inf
    # the drafting model: the row before's logits with noise, its probabilities, and a token drawn from them
    tokens = torch.randint(0, V, (T,), generator=d, device="cuda")
    starts_t = torch.tensor(starts, device="cuda")
    drafted = torch.ones(T, dtype=torch.bool, device="cuda")
    drafted[starts_t[:-1]] = False
    probs = torch.zeros((T, V), device="cuda") if case["probs"] else None
    temper = heat if heat > 0 else 0.5
    for lo in range(1, T, 256):         # rows in portions: noise for all at once would be large
        hi = min(T, lo + 256)
        rough = logits[lo - 1:hi - 1] + 0.5 * torch.randn((hi - lo, V), generator=d, device="cuda")
        p = torch.softmax(rough / temper, 1)
        noise = -torch.log(torch.rand((hi - lo, V), generator=d, device="cuda").clamp_min(1e-30))
        tokens[lo:hi] = torch.where(drafted[lo:hi], (p / noise).argmax(1), tokens[lo:hi])
        if probs is not None:
            probs[lo:hi] = p * drafted[lo:hi, None]
    u_accept = torch.rand(T, generator=d, device="cuda")
    u_draw = torch.rand((B, 24), generator=d, device="cuda")
    if heat > 0:
        # away from the edges: a draft's test by a ten-thousandth, the drawn number by more than what sums of float32 differ by
        at = torch.arange(T, device="cuda") - 1
        p_d = torch.zeros(T, dtype=torch.float64, device="cuda")
        for lo in range(0, T, 256):
            rows = at[lo:lo + 256].clamp_min(0)
            x = logits[rows].double() / heat
            p_d[lo:lo + 256] = torch.exp(x.gather(1, tokens[lo:lo + 256, None])[:, 0] - torch.logsumexp(x, 1))
        q_d = probs.gather(1, tokens[:, None])[:, 0].double() if probs is not None else torch.ones_like(p_d)
        near = (u_accept.double() * q_d - p_d).abs() < 1e-4 * p_d
        u_accept = torch.where(near, u_accept * 0.99, u_accept)
        yes = u_accept.double() * q_d < p_d
        picked = []
        for lo in range(0, B, 32):
            hi = min(B, lo + 32)
            rows = []
            for b in range(lo, hi):
                ok = yes[starts[b] + 1:starts[b + 1]].long()
                rows.append(starts[b] + ok.cumprod(0).sum())
            rows = torch.stack([torch.as_tensor(r, device="cuda") for r in rows])
            refused = rows + 1 < starts_t[lo + 1:hi + 1]
            w = torch.softmax(logits[rows].double() / heat, 1)
            nxt = (rows + 1).clamp_max(T - 1)
            if probs is not None:
                w = torch.where(refused[:, None], (w - probs[nxt].double()).clamp_min(0), w)
            else:
                w = torch.where(refused[:, None], w.scatter(1, tokens[nxt][:, None], 0.0), w)
            c = torch.cumsum(w, 1)
            mass = c[:, -1:].contiguous()
            u = u_draw[lo:hi].double()
            v = torch.searchsorted(c, u * mass, right=True).clamp_max(V - 1)
            top = c.gather(1, v) / mass
            low = top - w.gather(1, v) / mass
            good = torch.minimum(u - low, top - u) > 2e-5 + 4e-6 / mass
            first = good.float().argmax(1)
            v_max = w.argmax(1)[:, None]
            middle = ((c.gather(1, v_max) - 0.5 * w.gather(1, v_max)) / mass)[:, 0]
            picked.append(torch.where(good.any(1), u.gather(1, first[:, None])[:, 0], middle).float())
        u_draw = torch.cat(picked)
    else:
        u_draw = u_draw[:, 0].contiguous()
    cached = torch.randint(1, 9000, (B,), generator=g)
    return dict(op="verify", logits=logits, tokens=tokens.int(), q_start=_ints(starts), width=max(drafts) + 1, heat=heat, probs=probs,
                u_accept=u_accept, u_draw=u_draw, kv_len=(cached + torch.tensor(drafts) + 1).int().cuda())


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
_KEPT = {}


def run(state):
    if own:
        from janus_b200.engine.workspace import Workspace
        from janus_b200.kernels import ops
        if "workspace" not in _KEPT:         # scratch that an engine keeps from step to step
            _KEPT["workspace"] = Workspace(torch.device("cuda"))
        return {"tables": _own_tables, "attention": _own_attention, "verify": _own_verify}[state["op"]](state, ops, _KEPT["workspace"])
    return {"tables": _plain_tables, "attention": _plain_attention, "verify": _plain_verify}[state["op"]](state)


def _own_tables(s, ops, workspace):
    B, T = s["lengths"].shape[0], s["total"]
    new = lambda *shape: torch.empty(shape, dtype=torch.int32, device="cuda")            # noqa: E731
    out = dict(q_start=new(B + 1), kv_len=new(B), positions=new(T), token_seq=new(T), dest_rows=new(T), table=new(B, s["width"]),
               held=new(B), free_pages=new(s["free"].shape[0]), n_free=new(1), missing=new(1))
    ops.step_tables(s["lengths"], s["new"], s["rows"], s["table"], s["held"], s["prefix"], s["free"], s["n_free"], **out, page_size=PAGE)
    return out


def _own_attention(s, ops, workspace):
    out = torch.empty_like(s["q"])
    ops.attention_prefix(s["q"], s["k"], s["v"], out, s["prefix_pages"], s["prefix"], s["table"], s["q_start"], s["kv_len"],
                         s["positions"], s["heads"], s["kv_heads"], s["dim"], PAGE, s["scale"], workspace, max_q_len=s["most_new"],
                         max_kv_len=s["prefix"] + s["most_own"])
    return out


def _own_verify(s, ops, workspace):
    B = s["q_start"].shape[0] - 1
    accepted, kept = (torch.empty(B, dtype=torch.int32, device="cuda") for _ in range(2))
    tokens = torch.empty((B, s["width"]), dtype=torch.int32, device="cuda")
    logprobs = torch.empty((B, s["width"]), device="cuda")
    ops.verify_drafts(s["logits"], s["tokens"], s["q_start"], s["kv_len"], accepted, tokens, logprobs, kept, s["heat"], s["u_accept"],
                      s["u_draw"], s["probs"], workspace)
    return dict(accepted=accepted, tokens=tokens, logprobs=logprobs, kept=kept)


def _plain_tables(s):
    B, T, width, dev = s["lengths"].shape[0], s["total"], s["width"], s["lengths"].device
    P0, N = s["prefix"].shape[0], s["free"].shape[0]
    lengths, new, rows = s["lengths"].long(), s["new"].long(), s["rows"].long()
    begins = rows < 0
    at = rows.clamp_min(0)
    column = torch.arange(width, device=dev)
    # pages of rows that nobody goes on with, behind the free ones
    goes_on = torch.zeros(s["held"].shape[0], dtype=torch.int32, device=dev).index_add_(0, at, (~begins).int()) > 0
    back = ~goes_on[:, None] & (column >= P0) & (column < s["held"].long()[:, None])
    given = back.sum()
    n_free = s["n_free"].long()
    place = torch.where(back, n_free + back.reshape(-1).cumsum(0).reshape(back.shape) - 1, N)
    pool = torch.cat([s["free"].long(), s["free"].new_zeros(1).long()])
    pool = pool.scatter(0, place.reshape(-1), s["table"].long().reshape(-1))[:N]
    have = n_free + given
    # the requests' rows
    kv_len = lengths + new
    held = torch.where(begins, P0, s["held"].long()[at])
    want = torch.minimum((kv_len + PAGE - 1) // PAGE, torch.full_like(kv_len, width))
    need = (want - held).clamp_min(0)
    ends = need.cumsum(0)
    begin = ends - need
    got = torch.minimum(need, (have - begin).clamp_min(0))
    took = torch.minimum(ends[-1:], have)
    missing = ends[-1:] - took + ((kv_len + PAGE - 1) // PAGE - width).clamp_min(0).sum()
    before = torch.where(begins[:, None], torch.cat([s["prefix"].long(), s["prefix"].new_full((width,), -1).long()])[:width][None],
                         s["table"].long()[at])
    fresh = column - held[:, None]
    taken = pool[(begin[:, None] + fresh).clamp(0, N - 1)]
    table = torch.where(column < held[:, None], before, torch.where(fresh < got[:, None], taken, -1))
    left = torch.arange(N, device=dev)
    free = torch.where(left < have - took, pool[(left + took).clamp_max(N - 1)], -1)
    # the tokens
    q_start = torch.cat([new.new_zeros(1), new.cumsum(0)])
    t = torch.arange(T, device=dev)
    inside = t < q_start[-1]
    seq = torch.searchsorted(q_start[1:], t, right=True).clamp_max(B - 1)
    position = lengths[seq] + t - q_start[seq]
    page = table[seq, (position // PAGE).clamp_max(width - 1)]
    dest = torch.where(inside & (position < width * PAGE) & (page >= 0), page * PAGE + position % PAGE, -1)
    out = dict(q_start=q_start, kv_len=kv_len, positions=torch.where(inside, position, -1), token_seq=torch.where(inside, seq, -1),
               dest_rows=dest, table=table, held=held + got, free_pages=free, n_free=have - took, missing=missing)
    return {k: v.int() for k, v in out.items()}


def _plain_attention(s):
    q, G, D, P, L = s["q"].float(), s["kv_heads"], s["dim"], s["prefix"], s["most_own"]
    T, B = q.shape[0], s["q_start"].shape[0] - 1
    q = q.view(T, G, -1, D)
    flat = lambda pages, x: x[pages].float().transpose(-3, -2).reshape(*pages.shape[:-1], -1, G, D)      # noqa: E731
    keys, values = (flat(s["prefix_pages"].long(), x)[:P] for x in (s["k"], s["v"]))
    position = s["positions"].long()
    shared = torch.einsum("tgrd,kgd->tgrk", q, keys) * s["scale"]
    shared = torch.where((torch.arange(P, device=q.device) <= position[:, None])[:, None, None], shared, -math.inf)
    # every request's own keys and queries, padded to the longest
    table = s["table"][:, :(L + PAGE - 1) // PAGE].long().clamp_min(0)
    k_own, v_own = (flat(table, x)[:, :L] for x in (s["k"], s["v"]))
    start = s["q_start"].long()
    seq = torch.searchsorted(start[1:], torch.arange(T, device=q.device), right=True)
    place = torch.arange(T, device=q.device) - start[seq]
    q_own = q.new_zeros((B, s["most_new"]) + q.shape[1:])
    q_own[seq, place] = q
    mine = (torch.einsum("bjgrd,bkgd->bjgrk", q_own, k_own) * s["scale"])[seq, place]
    mine = torch.where((P + torch.arange(L, device=q.device) <= position[:, None])[:, None, None], mine, -math.inf)
    top = torch.maximum(shared.amax(-1, keepdim=True), mine.amax(-1, keepdim=True))
    shared, mine = torch.exp(shared - top), torch.exp(mine - top)
    total = shared.sum(-1, keepdim=True) + mine.sum(-1, keepdim=True)
    w_own = q.new_zeros((B, s["most_new"]) + mine.shape[1:])
    w_own[seq, place] = mine
    out = torch.einsum("tgrk,kgd->tgrd", shared, values) + torch.einsum("bjgrk,bkgd->bjgrd", w_own, v_own)[seq, place]
    return (out / total).reshape(T, -1).to(s["q"].dtype)


def _plain_verify(s):
    logits, start, heat, W = s["logits"], s["q_start"].long(), s["heat"], s["width"]
    B, (T, V) = start.shape[0] - 1, logits.shape
    n = start[1:] - start[:-1] - 1                                  # drafts of each request
    place = torch.arange(W - 1, device=logits.device)
    row = (start[:-1, None] + place).clamp_max(T - 1)               # the row whose logits judge a draft
    at = (row + 1).clamp_max(T - 1)                                 # the draft's own row
    draft = s["tokens"].long()[at]
    top = logits.amax(1)
    total = torch.exp((logits - top[:, None]) / (heat or 1.0)).sum(1)
    if heat > 0:
        weight = torch.exp((logits[row, draft] - top[row]) / heat)
        q = s["probs"][at, draft] if s["probs"] is not None else 1.0
        yes = s["u_accept"][at] * q * total[row] < weight
    else:
        yes = logits.argmax(1)[row] == draft
    accepted = ((yes & (place < n[:, None])).int().cumprod(1)).sum(1)
    last = start[:-1] + accepted                                    # the row that gives the next token
    refused = accepted < n
    x = logits[last]
    if heat > 0:
        w = torch.exp((x - top[last, None]) / heat)
        behind = (last + 1).clamp_max(T - 1)
        if s["probs"] is not None:
            left = (w / total[last, None] - s["probs"][behind]).clamp_min(0)
        else:
            left = w.scatter(1, s["tokens"].long()[behind][:, None], 0.0)
        w = torch.where((refused & (left.sum(1) > 0))[:, None], left, w)
        c = torch.cumsum(w, 1)
        token = (c <= s["u_draw"][:, None] * c[:, -1:]).sum(1).clamp_max(V - 1)
    else:
        token = x.argmax(1)
    k = torch.arange(W, device=logits.device)
    kept = s["tokens"].long()[(start[:-1, None] + 1 + k).clamp_max(T - 1)]
    tokens = torch.where(k < accepted[:, None], kept, torch.where(k == accepted[:, None], token[:, None], -1))
    judge = (start[:-1, None] + k).clamp_max(T - 1)
    logprobs = (logits[judge, tokens.clamp_min(0)] - top[judge]) / (heat or 1.0) - torch.log(total[judge])
    logprobs = torch.where(tokens >= 0, logprobs, 0.0)
    return dict(accepted=accepted.int(), tokens=tokens.int(), logprobs=logprobs, kept=(s["kv_len"] - n + accepted).int())


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    B = case["requests"]
    if case["op"] == "tables":
        new = _spread(B, case["new_lo"], case["new_hi"])
        total = sum(new) + case["spare"]
        # three arrays a token; the old rows' pages and the free list in, the new ones out
        held = sum(_held(case, n) for n in _spread(B, case["len_lo"], case["len_hi"]))
        return {"bytes": 4 * (3 * total + held + B * case["width"] + 2 * _room(case) - held + 8 * B), "flops": 0}
    if case["op"] == "attention":
        size = 2 if case["dtype"] == "bfloat16" else 4
        H, G, D, P = case["heads"], case["kv_heads"], case["dim"], case["prefix"]
        new, before = _spread(B, case["new_lo"], case["new_hi"]), _spread(B, case["own_lo"], case["own_hi"])
        T = sum(new)
        cached = P + sum(before) + T
        # pairs of tokens and keys that see each other: own lengths and new tokens meet in an order of their own per seed
        pairs = T * P + T * sum(before) / B + sum(n * (n + 1) / 2 for n in new)
        return {"bytes": size * (2 * T * H * D + 2 * cached * G * D), "flops": 4 * H * D * pairs}
    drafts = _spread(B, case["drafts_lo"], case["drafts_hi"])
    rows, V = sum(drafts) + B, case["vocab"]
    refused = sum(n > 0 for n in drafts) if case["probs"] and case["temperature"] > 0 else 0
    return {"bytes": 4 * (rows * V + refused * V), "flops": 3 * rows * V}


# ---------------------------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"tables": _exact_tables, "attention": _exact_attention, "verify": _exact_verify}[case["op"]](s)


def _exact_tables(s):
    lengths, new, rows, held0 = (s[k].tolist() for k in ("lengths", "new", "rows", "held"))
    old, prefix, width = s["table"].tolist(), s["prefix"].tolist(), s["width"]
    pool = s["free"].tolist()[:int(s["n_free"])]
    for r, row in enumerate(old):
        if r not in rows:
            pool += row[len(prefix):held0[r]]
    taken, missing = 0, 0
    table, held, q_start, positions, token_seq, dest = [], [], [0], [], [], []
    for b, (n, t, r) in enumerate(zip(lengths, new, rows)):
        pages = list(prefix) if r < 0 else old[r][:held0[r]]
        while len(pages) * PAGE < n + t and len(pages) < width:
            if taken == len(pool):
                missing += min(width, -(-(n + t) // PAGE)) - len(pages)
                break
            pages.append(pool[taken])
            taken += 1
        missing += max(0, -(-(n + t) // PAGE) - width)
        held.append(len(pages))
        for p in range(n, n + t):
            positions.append(p)
            token_seq.append(b)
            dest.append(pages[p // PAGE] * PAGE + p % PAGE if p // PAGE < len(pages) else -1)
        q_start.append(q_start[-1] + t)
        table.append(pages + [-1] * (width - len(pages)))
    left = pool[taken:]
    fill = [-1] * (s["total"] - len(positions))
    out = dict(q_start=q_start, kv_len=[n + t for n, t in zip(lengths, new)], positions=positions + fill, token_seq=token_seq + fill,
               dest_rows=dest + fill, table=table, held=held, free_pages=left + [-1] * (s["free"].shape[0] - len(left)),
               n_free=[len(left)], missing=[missing])
    return {k: torch.tensor(v, dtype=torch.int32) for k, v in out.items()}


def _exact_attention(s):
    G, D, P = s["kv_heads"], s["dim"], s["prefix"]
    rows = lambda x, pages, n: x[pages.long()].double().permute(1, 0, 2, 3).reshape(G, -1, D)[:, :n]     # noqa: E731
    k0, v0 = rows(s["k"], s["prefix_pages"], P), rows(s["v"], s["prefix_pages"], P)
    starts, lens = s["q_start"].tolist(), s["kv_len"].tolist()
    out = []
    for b, length in enumerate(lens):
        n = starts[b + 1] - starts[b]
        pages = s["table"][b, :_pages(length - P)]
        k = torch.cat([k0, rows(s["k"], pages, length - P)], 1)
        v = torch.cat([v0, rows(s["v"], pages, length - P)], 1)
        q = s["q"][starts[b]:starts[b + 1]].double().view(n, G, -1, D).permute(1, 2, 0, 3)
        score = torch.matmul(q, k[:, None].transpose(-1, -2)) * s["scale"]
        hidden = torch.arange(length, device=q.device)[None] > torch.arange(length - n, length, device=q.device)[:, None]
        share = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
        out.append(torch.matmul(share, v[:, None]).permute(2, 0, 1, 3).reshape(n, -1))
    return torch.cat(out)


def _exact_verify(s):
    starts, ids, cached = s["q_start"].tolist(), s["tokens"].tolist(), s["kv_len"].tolist()
    heat, V = s["heat"], s["logits"].shape[1]
    u_accept, u_draw = s["u_accept"].tolist(), s["u_draw"].tolist()
    all_accepted, all_tokens, all_logprobs, all_kept = [], [], [], []
    for b, (lo, hi) in enumerate(zip(starts, starts[1:])):
        x = s["logits"][lo:hi].double()
        p = torch.softmax(x / heat, 1) if heat > 0 else torch.nn.functional.one_hot(x.argmax(1), V).double()
        drafts = ids[lo + 1:hi]
        p_draft = [float(v) for v in p[torch.arange(len(drafts)), torch.tensor(drafts, dtype=torch.long)].tolist()]
        accepted = 0
        for j, d in enumerate(drafts):
            q = float(s["probs"][lo + 1 + j, d]) if s["probs"] is not None and heat > 0 else 1.0
            if not (u_accept[lo + 1 + j] * q < p_draft[j] if heat > 0 else p_draft[j] == 1.0):
                break
            accepted += 1
        w = p[accepted].clone()
        if heat > 0 and accepted < len(drafts):
            if s["probs"] is not None:
                w = (w - s["probs"][lo + 1 + accepted].double()).clamp_min(0)
            else:
                w[drafts[accepted]] = 0.0
        c = torch.cumsum(w, 0)
        token = int(torch.searchsorted(c, u_draw[b] * c[-1:], right=True)) if heat > 0 else int(w.argmax())
        all_accepted.append(accepted)
        all_tokens.append(drafts[:accepted] + [token] + [-1] * (s["width"] - accepted - 1))
        given = torch.log_softmax(x[:accepted + 1] / (heat or 1.0), 1)
        chosen = given[torch.arange(accepted + 1), torch.tensor(drafts[:accepted] + [token])].tolist()
        all_logprobs.append(chosen + [0.0] * (s["width"] - accepted - 1))
        all_kept.append(cached[b] - len(drafts) + accepted)
    whole = lambda v: torch.tensor(v, dtype=torch.int32)      # noqa: E731
    return dict(accepted=whole(all_accepted), tokens=whole(all_tokens), kept=whole(all_kept),
                logprobs=torch.tensor(all_logprobs, dtype=torch.float64))
