"""The operators of beam search written down once more, in 64 bits and plain loops: what `test_beams.py` compares the kernels with."""
import math

import torch

PAGE = 64
NONE = -math.inf


def select(logits, scores, stops):
    """(parents, tokens, scores, ended parents, ended tokens, ended scores, the smallest distance between two neighbours of the ranking of any
    request that could change an answer).  logits [R K, V], scores [R, K]; lists [R][K]."""
    R, K = scores.shape
    V = logits.shape[1]
    stops = {int(s) for s in stops}
    out = [[], [], [], [], [], []]
    gap = math.inf
    for r in range(R):
        ranked = []
        for b in range(K):
            score = float(scores[r, b])
            if not score > NONE:
                continue
            x = logits[r * K + b].double()
            x = torch.where(torch.isnan(x), NONE, x)
            top = float(x.max())
            if top == NONE:
                continue
            z = torch.where(x == math.inf, 0.0, NONE) if top == math.inf else x - top
            logp = z - math.log(float(z.exp().sum()))
            best = x.sort(descending=True, stable=True).indices[: K + len(stops)].tolist()
            ranked += [(score + float(logp[v]), b, v) for v in best if float(logp[v]) > NONE]
        ranked.sort(key=lambda t: (-t[0], t[1], t[2]))
        for (s, b, _), (t, c, _) in zip(ranked[: 2 * K + len(stops)], ranked[1:]):
            if b != c and s != t:
                gap = min(gap, s - t)
        on = [t for t in ranked if t[2] not in stops][:K]
        ended = [t for t in ranked[:K] if t[2] in stops]
        rows = [None] * K
        later = []
        for t in on:
            if rows[t[1]] is None:
                rows[t[1]] = t
            else:
                later.append(t)
        for t in later:
            rows[rows.index(None)] = t
        rows = [t if t is not None else (NONE, -1, 0) for t in rows]
        ended += [(NONE, -1, -1)] * (K - len(ended))
        for o, v in zip(out, ([t[1] for t in rows], [t[2] for t in rows], [t[0] for t in rows], [t[1] for t in ended], [t[2] for t in ended],
                              [t[0] for t in ended])):
            o.append(v)
    return (*out, gap)


def fork(parents, lengths, table, refs, free, spare=0, page=PAGE):
    """As `ops.fork_pages`, on lists: parents and lengths [R][K], table [R K][W], refs [P], free: the free pages.  Returns a dict; `free` in
    it are the free pages that are left."""
    R, K, W = len(parents), len(parents[0]), len(table[0])
    pages_of = lambda n: -(-n // page)      # noqa: E731
    counted = lambda p: 0 <= p < len(refs) and p != spare      # noqa: E731
    goes = [[0 <= p < K for p in row] for row in parents]
    new = []
    for r in range(R):
        for k in range(K):
            row = [-1] * W
            if goes[r][k]:
                p = parents[r][k]
                n = min(W, pages_of(lengths[r][p]))
                row[:n] = table[r * K + p][:n]
            new.append(row)
    before, refs, free = list(refs), list(refs), list(free)
    for i, (old, row) in enumerate(zip(table, new)):
        for p in row:
            refs[p] += counted(p)
        for p in old[: pages_of(lengths[i // K][i % K])]:
            refs[p] -= counted(p)
    free += [p for p in range(len(refs)) if refs[p] == 0 and before[p] > 0]
    out = dict(kv_len=[], positions=[], dest_rows=[], copy_src=[], copy_dst=[], copy_rows=[], shared=[])
    gives, takes, missing = [], [], 0
    for r in range(R):
        rows = new[r * K: r * K + K]
        ends = [lengths[r][parents[r][k]] if goes[r][k] else 0 for k in range(K)]
        held = [rows[k][ends[k] // page] if goes[r][k] and ends[k] % page and ends[k] // page < W else -1 for k in range(K)]
        made = {k: [] for k in ("kv_len", "positions", "dest_rows", "copy_src", "copy_dst", "copy_rows")}
        for k in range(K):
            at, part = ends[k] // page, ends[k] % page
            src, dst, copied, next_page = -1, -1, 0, -1
            if not goes[r][k]:
                rows[k][0] = spare
            elif at >= W:
                missing += 1
            elif held[k] >= 0 and held.index(held[k]) == k and held.count(held[k]) == refs[held[k]]:
                next_page = held[k]
            else:
                next_page = free.pop() if free else -1
                missing += next_page < 0
                if held[k] >= 0:
                    gives.append(held[k])
                    if next_page >= 0:
                        src, dst, copied = held[k], next_page, part
                if next_page >= 0:
                    takes.append(next_page)
                rows[k][at] = next_page
            for name, v in (("kv_len", ends[k] + 1 if goes[r][k] else 1), ("positions", ends[k]),
                            ("dest_rows", next_page * page + part if next_page >= 0 else spare * page), ("copy_src", src), ("copy_dst", dst),
                            ("copy_rows", copied)):
                made[name].append(v)
        for name, v in made.items():
            out[name].append(v)
        alive = [k for k in range(K) if goes[r][k]]
        lead = min((min(ends[k] // page, W) for k in alive), default=0)
        out["shared"].append(next((c for c in range(lead) if len({rows[k][c] for k in alive}) > 1), lead))
    for p in gives:
        refs[p] -= 1
    for p in takes:
        refs[p] = 1
    return dict(out, new_table=new, new_refs=refs, free=free, missing=missing)


def attention(q, k, v, table, kv_len, nh, nkv, hd, scale):
    """(result, weighted sum of the values' magnitudes), [rows, nh, hd] in 64 bits; a row without keys is 0."""
    out = torch.zeros(q.shape[0], nh, hd, dtype=torch.float64)
    size = torch.zeros_like(out)
    q, k, v = q.double().cpu().view(-1, nh, hd), k.double().cpu(), v.double().cpu()
    for i, n in enumerate(kv_len):
        if n <= 0:
            continue
        at = torch.arange(n)
        page = torch.tensor(table[i])[at // PAGE]
        for h in range(nh):
            j = h // (nh // nkv)
            w = torch.softmax(k[page, j, at % PAGE] @ q[i, h] * scale, 0)
            out[i, h], size[i, h] = w @ v[page, j, at % PAGE], w @ v[page, j, at % PAGE].abs()
    return out, size
