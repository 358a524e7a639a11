"""How attention behind a shared prefix shares its work out, replayed on the host: a row's shares of the list of own keys and its
ranges over the prefix, as the kernels count them, against the room and the counts that they are kept in.

On the device, steps whose groups of heads do not divide a block of 16 rows, against the formula; the tolerance is the one that
test_shared_prefix.py derives for bfloat16.
"""
import numpy as np
import pytest
import torch

from janus_b200.kernels import ops
from test_shared_prefix import attention, attention_case, attention_oracle, close

gpu = pytest.mark.gpu


def own_shares(plan, new, owned, prefix, nkv, group, apart, bound=None):
    """[(first token, kv head, first row, rows, shares)] of every block of 16 rows: the list of (sequence, kv head, 16 rows) and their
    tiles of 32 keys, cut in even shares."""
    _, _, _, _, own_ctas, fewest, _ = plan
    shared = 0 if apart else -(-prefix // 32)
    tiles = [shared + min(max(-(-o // 32), 1), bound or 1 << 30) for o in owned]
    blocks = [-(-n * group // 16) for n in new]
    total = sum(nkv * b * t for b, t in zip(blocks, tiles))
    per = max(fewest, -(-total // (own_ctas * 4)))
    out, place, token = [], 0, 0
    for n, b, t in zip(new, blocks, tiles):
        for kvh in range(nkv):
            for rb in range(b):
                out.append((token, kvh, 16 * rb, min(16, n * group - 16 * rb), (place + t - 1) // per - place // per + 1))
                place += t
        token += n
    return out


def cases(count):
    rng = np.random.default_rng(2)
    for _ in range(count):
        group, nkv, hd = int(rng.integers(1, 17)), int(rng.integers(1, 9)), int(rng.choice([64, 128, 256]))
        n, most = int(rng.integers(1, 80)), max(1, min(int(rng.choice([1, 2, 4, 6])), 64 // group))
        new = [int(v) for v in rng.integers(0, most + 1, n)]
        new[0] = most
        owned = [v + int(rng.integers(0, int(rng.choice([2, 300, 3000])))) for v in new]
        yield new, owned, int(rng.integers(1, 9000)), nkv, group, hd
    yield [6] * 48, [206] * 48, 4096, 8, 3, 128
    yield [4] * 48, [204] * 48, 4096, 8, 5, 128


def test_rows_that_share_a_count_have_as_many_shares():
    split = 0
    for new, owned, prefix, nkv, group, hd in cases(400):
        T, nh = sum(new), nkv * group
        plan = ops.attention_prefix_plan(T, len(new), max(new), prefix, max(owned), nh, nkv, hd)
        assert not plan[3]
        _, floats, _ = ops._attention_prefix_sizes(prefix, 99, 99, T, 999, len(new), nh, nkv, hd, 64, max(new), prefix + max(owned), 1.0, False)
        counts = floats - (plan[2] + plan[6]) * T * nh * (hd + 2)
        assert counts % T == 0
        of_head = nh // (counts // T)                          # query heads that one count stands for
        kept = {}
        for token, kvh, row0, rows, shares in own_shares(plan, new, owned, prefix, nkv, group, plan[1] > 0):
            assert shares <= plan[6]
            for r in range(row0, row0 + rows):
                where = (token + r // group, (kvh * group + r % group) // of_head)
                assert kept.setdefault(where, shares) == shares, (new[0], group, nkv)
            split += row0 % group != 0
    assert split > 100


def test_ranges_of_the_prefix_as_they_are_launched():
    """The list as the C entry makes it: ranges that cut a tile evenly pad it, tiles of narrow heads count blocks of 64 keys."""
    for new, owned, prefix, nkv, group, hd in cases(400):
        T, nh = sum(new), nkv * group
        tiles, per, ranges, *_ = ops.attention_prefix_plan(T, len(new), max(new), prefix, max(owned), nh, nkv, hd)
        if not per:
            continue
        keys, step = (64 if hd > 128 else 128), 128 // group * tiles
        blocks, items = -(-prefix // keys), -(-T // step) * nkv
        even = -(-blocks // per)
        if per < blocks and items * even <= 148:
            blocks = even * per
        finer = 2 if hd <= 64 and tiles == 1 else 1
        blocks, per = blocks * finer, per * finer
        real = -(-prefix // (keys // finer))
        for i in range(items):
            first, last = i * blocks // per, (i * blocks + blocks - 1) // per
            assert last - first + 1 <= ranges
            for c in range(first, last + 1):                   # every range of a tile has a block with keys in it
                assert max(c * per, i * blocks) - i * blocks < real


def test_lengths_beyond_the_bound_take_no_places_beyond_the_scratch():
    """A caller's bound that is too low: shares counted by the device's lengths have more results than places, by the bound they fit."""
    beyond = 0
    for new, owned, prefix, nkv, group, hd in cases(200):
        bound = max(1, max(owned) // 5)
        plan = ops.attention_prefix_plan(sum(new), len(new), max(new), prefix, bound, nkv * group, nkv, hd)
        args = (plan, new, owned, prefix, nkv, group, plan[1] > 0)
        beyond += max(b[4] for b in own_shares(*args)) > plan[6]
        assert max(b[4] for b in own_shares(*args, bound=max(1, -(-bound // 32)))) <= plan[6]
    assert beyond > 10


@pytest.mark.parametrize("n,new,prefix,heads,kv_heads,dim,together", [
    (4, 1, 1000, 32, 8, 128, True), (16, 1, 400, 32, 8, 64, True), (8, 1, 600, 32, 8, 128, True), (8, 1, 1400, 32, 8, 64, True),
    (4, 4, 1000, 32, 8, 128, False), (4, 4, 1600, 32, 8, 128, False), (8, 1, 1800, 32, 8, 128, False), (64, 2, 1146, 2, 2, 80, False),
    (4, 1, 903, 32, 16, 256, False), (32, 1, 400, 32, 8, 128, False)])
def test_who_walks_the_prefix_is_the_faster_form_by_calls(n, new, prefix, heads, kv_heads, dim, together):
    """Shapes on both sides of the line whose forms were timed 0.9 to 5 us apart."""
    plan = ops.attention_prefix_plan(n * new, n, new, prefix, 60, heads, kv_heads, dim)
    assert (plan[1] == 0) == together


def test_scratch_of_float32_goes_by_the_rows():
    """Two results a row where rows alone fill the machine; where they do not, no more than 64 rows each of ranges that fill it eight
    times (and of the prefix twice), whatever the lengths."""
    rng = np.random.default_rng(4)
    for _ in range(2000):
        group, nkv, hd = int(rng.integers(1, 17)), int(rng.integers(1, 33)), int(rng.choice([64, 128, 256]))
        n, new = int(rng.integers(1, 65)), int(2 ** rng.uniform(0, 12))
        T, prefix, own = max(new, int(n * new * rng.uniform(0.3, 1.0))), int(2 ** rng.uniform(0, 14)), new + int(2 ** rng.uniform(0, 14))
        _, floats, _ = ops._attention_prefix_sizes(prefix, 99, 99, T, 999, n, nkv * group, nkv, hd, 64, new, prefix + own, 1.0, True)
        rows = T * nkv * group
        assert floats <= (2 * rows + 64 * (8 * 296 + 2 * 296 + nkv * n * 2)) * (hd + 2) + rows, (group, nkv, hd, n, new, T)
    _, floats, _ = ops._attention_prefix_sizes(1000, 99, 99, 32000, 999, 8, 32, 8, 128, 64, 4000, 5000, 1.0, True)
    assert floats * 4 < 1.1e9


@gpu
def test_attention_of_float32_prompts_beside_single_tokens():
    c = attention_case(15, torch.float32, 8, 2, 64, 200, [700, 1, 300, 0, 1], [900, 2000, 300, 50, 1])
    close(attention(c), attention_oracle(c), torch.float32)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("prefix,n,new", [(0, 5, 1), (100, 5, 1), (3000, 40, 2), (3000, 6, 90)])
def test_bounds_that_are_too_low_write_nothing_beyond_the_scratch(dtype, prefix, n, new):
    from janus_b200.engine.workspace import Workspace
    c = attention_case(14, dtype, 8, 2, 64, prefix, [new] * n, [new + 400 + 97 * i for i in range(n)])
    c["workspace"], c["most"] = Workspace(torch.device("cuda")), prefix + 40
    _, floats, _ = ops._attention_prefix_sizes(prefix, c["table"].stride(0), c["table"].shape[1], n * new, c["k"].shape[0], n, 8, 2, 64, 64, new,
                                               c["most"], float(c["scale"]), dtype is torch.float32)
    scratch = c["workspace"].get("prefix_parts", (40 * floats,), torch.float32).fill_(3.0)
    attention(c)
    assert (scratch[floats:] == 3.0).all()
    ops.check_kernel_status(torch.device("cuda"))


@gpu
@pytest.mark.parametrize("heads,kv_heads,dim,n,new,before,prefix", [
    (24, 8, 128, 48, 6, 200, 4096),      # heads of a group that do not divide 16 rows
    (40, 8, 128, 48, 4, 200, 4096),
    (28, 4, 64, 60, 5, 333, 3000),
    (6, 2, 80, 90, 6, 517, 2500),
    (9, 1, 256, 40, 5, 260, 2000),
    (24, 8, 128, 64, 6, 40, 16000),
])
def test_attention_of_groups_that_do_not_divide_a_block_of_rows(heads, kv_heads, dim, n, new, before, prefix):
    from janus_b200.engine.workspace import Workspace
    counts = [new if i % 5 else 1 + i % new for i in range(n)]
    owned = [c + before + i * 37 % 101 for i, c in enumerate(counts)]
    c = attention_case(13, torch.bfloat16, heads, kv_heads, dim, prefix, counts, owned)
    c["workspace"] = Workspace(torch.device("cuda"))
    plan = ops.attention_prefix_plan(sum(counts), n, new, prefix, max(owned), heads, kv_heads, dim)
    assert plan[1] > 0 and not plan[3]
    # results that an earlier step left in the scratch: as large as real ones
    c["workspace"].get("prefix_parts", (65 * sum(counts) * heads * (dim + 3),), torch.float32).fill_(3.0)
    got = attention(c)
    close(got, attention_oracle(c), torch.bfloat16)
    for _ in range(3):
        assert torch.equal(attention(c), got)
