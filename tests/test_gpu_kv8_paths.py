"""The 8-bit cache's cross, shared-prefix and weighing attention and its eviction where a
size of the call chooses another kernel or another way through one."""
from __future__ import annotations

import numpy as np
import pytest

import _kv8 as kv8
from test_gpu_kv8 import Batch, Pair, check_attention, device, lists_for, rows
from test_gpu_kv8_cross import check_cross, cross
from test_gpu_kv8_evict import check_evict, evict, model_evict, snapshot, some_weights
from test_gpu_kv8_shared import Prefix, check_shared, shared
from test_gpu_kv8_weigh import check_weights, model_weights, sums, weigh

pytestmark = pytest.mark.gpu


def wide(heads, kv, dim, new):
    """Whether 16-bit rows go to the kernel of 256 rows a workgroup (kv8_cross.hip)."""
    most = max(new) * (heads // kv)
    return dim <= 128 and most > 128 and -(-most // 256) * kv * len(new) >= 256


WIDE = [
    # heads, kv heads, dim, page, tokens of a list, query tokens
    (32, 32, 128, 16, [0, 1, 63, 64, 65, 300, 1000, 17], [129, 40, 300, 1, 0, 257, 130, 256]),
    (32, 32, 64, 32, [257, 40, 0, 700, 31, 32, 33, 5], [3, 129, 150, 200, 1, 16, 0, 255]),
    (32, 32, 96, 48, [100, 47, 480, 1, 49, 0, 97, 11], [129, 1, 140, 33, 32, 31, 64, 2]),
    (24, 24, 80, 16, [77, 129, 400, 16, 15, 1, 900, 64, 65, 2, 0], [2] * 10 + [200]),
    (32, 32, 48, 64, [64, 130, 1, 200, 63, 65, 0, 5], [131, 1, 2, 132, 128, 127, 0, 9]),
    (64, 32, 16, 256, [256, 700, 3, 255, 257, 1, 30, 512], [65, 100, 1, 70, 64, 2, 0, 33]),
    (16, 8, 128, 64, [(37 * r) % 400 for r in range(32)], [65 + r % 7 if r % 3 else r for r in range(32)]),
    # more requests than are taken by length
    (12, 4, 64, 16, [(53 * r) % 500 for r in range(70)], [43 if r % 9 == 4 else r % 5 for r in range(70)]),
]


@pytest.mark.parametrize("fmt", [kv8.E4M3, kv8.INT8])
@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("case", WIDE, ids=lambda c: "%dx%dx%d_p%d_%d" % (c[:4] + (len(c[4]),)))
def test_cross_wide(gpu, case, kind, fmt):
    import torch
    heads, kv, dim, page, held, new = case
    assert wide(heads, kv, dim, new)
    rng = np.random.default_rng(heads * dim + page + sum(new))
    capacity = sum(-(-n // page) for n in held) + 1
    pair = Pair(gpu, kv, dim, page, capacity, fmt)
    pair.fill(dim + fmt)
    lists = lists_for(rng, held, page, capacity)
    for l, n in zip(lists, held):
        if n % page:
            pair.set_counts(l[-1], n % page)
    q = rows(rng, kind, sum(new) + 2, heads, dim)
    out = torch.full_like(q, 9.0)
    fail = torch.zeros(1, dtype=torch.int64, device="cuda")
    batch = Batch(gpu, lists, [0] * len(new), new)
    cross(pair, batch, kind, q, out, fail=fail)
    assert int(fail) == 0
    check_cross(pair, lists, new, kind, q, out)
    assert bool((out[sum(new):] == 9.0).all())  # rows behind the last request
    again = torch.full_like(q, 9.0)
    cross(pair, Batch(gpu, lists, [0] * len(new), new, strided=max(len(l) for l in lists) + 1,
                      max_pages=1), kind, q, again, scale=-0.21, fail=fail)
    assert int(fail) == 0
    check_cross(pair, lists, new, kind, q, again, scale=-0.21)


@pytest.mark.parametrize("dim", [16, 64])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_cross_wide_any_list(gpu, kind, dim):
    """Pages out of order, half-full and empty ones in the middle, one twice, some outside
    the cache; a stage of pages that holds such ones after stages that hold none."""
    import torch
    rng = np.random.default_rng(12)
    pair = Pair(gpu, 32, dim, 16, 600)
    pair.fill(2)
    for page, count in ((3, 5), (7, 0), (11, 1), (12, 15), (30, 0), (580, 4), (581, 0)):
        pair.set_counts(page, count)
        if count == 0:
            pair.key_scales[page] = float("nan")
            pair.value_scales[page] = float("inf")
    lists = [[3, 9, 7, 11], [12, 12, 5], [7, 30], [], [39, 3, 38, 7, 37, 12, 36, 11, 1, 2, 3, 3],
             list(range(40, 600)), [3] + list(range(41, 590)), [600, 4, -1, 5]]
    new = [130, 1, 129, 5, 140, 33, 2, 150]
    assert wide(32, 32, dim, new)
    q = rows(rng, kind, sum(new), 32, dim)
    out = torch.full_like(q, 9.0)
    fail = torch.zeros(1, dtype=torch.int64, device="cuda")
    cross(pair, Batch(gpu, lists, [0] * 8, new), kind, q, out, fail=fail)
    assert int(fail) & 0xffffffff == 3
    lists[7] = [4, 5]
    check_cross(pair, lists, new, kind, q, out)
    # a NaN value: its dim of all rows of the request, and no other
    fail.zero_()
    cross(pair, Batch(gpu, lists, [0] * 8, new), kind, q, out, fail=fail)
    want = out.clone()
    pair.values[300, 3, 0, 5, 3] = 0x7f  # in the lists of requests 5 and 6
    cross(pair, Batch(gpu, lists, [0] * 8, new), kind, q, out, fail=fail)
    assert int(fail) == 0
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[sum(new[:5]):sum(new[:7]), 3, 5] = True
    assert bool(out[hit].isnan().all()) and torch.equal(out[~hit], want[~hit])
    # an infinite query: its row alone, and where the list holds no token not even that
    row = sum(new[:4]) + 10
    q[row, 7, 0] = q[200, 7, 0] = float("inf")
    assert sum(new[:2]) <= 200 < sum(new[:3]) and not bool(want[200].any())
    pair.values[300, 3, 0, 5, 3] = 0x31
    cross(pair, Batch(gpu, lists, [0] * 8, new), kind, q, out)
    hit.zero_()
    hit[row, 7] = True
    keep = ~hit
    keep[sum(new[:5]):sum(new[:7]), 3, 5] = False  # (the value is another one now)
    assert bool(out[hit].isnan().all()) and torch.equal(out[keep], want[keep])


def holed(rng, pages, page):
    """Counts of a list's pages: one in eight holds fewer tokens than it has places."""
    counts = np.full(pages, page)
    some = rng.choice(pages, pages // 8, replace=False)
    counts[some] = rng.integers(0, page, len(some))
    counts[[pages // 9, pages - pages // 7]] = page // 2  # (where the first and the last end)
    return counts


@pytest.mark.parametrize("fmt", [kv8.E4M3, kv8.INT8])
@pytest.mark.parametrize("style", ["spread", "ties", "any"])
@pytest.mark.parametrize("pages,hint", [(530, None), (1100, None), (2100, None), (530, 3), (1100, 400)])
def test_evict_long_lists_with_holes(gpu, pages, hint, style, fmt):
    """Lists of more places than a wave holds of the shortest form (8192) and of the longest
    (32768), more pages than a workgroup has threads, whose inner pages are half-full or
    empty; the first tokens and the last ones end inside such pages."""
    import torch
    rng = np.random.default_rng(pages)
    page, room = 16, 520
    counts = holed(rng, pages, page)
    pair = Pair(gpu, 2, 16, page, pages + room, fmt)
    pair.fill(3 + fmt)
    order = rng.permutation(pages + room).tolist()
    whole, new = order[:pages], [order[pages:]]
    for p, n in zip(whole, counts):
        if n < page:
            pair.set_counts(p, int(n))
    i, j = pages // 9, pages - pages // 7
    first = int(counts[:i].sum()) + 3
    recent = int(counts[j + 1:].sum()) + 5
    keep = first + recent + 300
    lists = [whole]
    weights = some_weights(rng, pair.model, style)
    given, before = weights.clone(), snapshot(pair)
    fail = torch.zeros(1, dtype=torch.int64, device="cuda")
    got = evict(pair, Batch(gpu, lists, max_pages=hint), keep, first, recent, weights, device(new),
                fail=fail)
    assert int(fail) == 0
    want = model_evict(pair, lists, keep, first, recent, given, new)
    check_evict(pair, lists, new, (weights,) + got, want, before)
    # one of its pages lies outside the cache
    lists[0][pages // 2] = pages + room
    weights, before = given.clone(), snapshot(pair)
    got = evict(pair, Batch(gpu, lists, max_pages=hint), 333, 4, 40, weights, device(new), fail=fail)
    assert int(fail) & 0xffffffff == 3
    want = model_evict(pair, lists, 333, 4, 40, given, new)
    check_evict(pair, lists, new, (weights,) + got, want, before)


@pytest.mark.parametrize("fmt", [kv8.E4M3, kv8.INT8])
@pytest.mark.parametrize("kv,dim,page", [(2, 64, 16), (1, 128, 64), (3, 80, 112), (1, 256, 256)])
def test_evict_without_summaries(gpu, kv, dim, page, fmt):
    rng = np.random.default_rng(dim)
    pair = Pair(gpu, kv, dim, page, 20, fmt, summaries=False)
    pair.fill(5)
    pair.set_counts(4, page // 2)
    lists, new = [[0, 1, 2, 3, 4], [5], [6, 7]], [[8, 9, 10], [11, 12, 13], [14, 15, 16]]
    keep = 2 * page + 3
    weights = some_weights(rng, pair.model, "spread")
    given, before = weights.clone(), snapshot(pair)
    got = evict(pair, Batch(gpu, lists), keep, 2, page // 3, weights, device(new))
    want = model_evict(pair, lists, keep, 2, page // 3, given, new)
    check_evict(pair, lists, new, (weights,) + got, want, before)


@pytest.mark.parametrize("heads,kv,dim,requests,groups,pre", [
    (32, 8, 64, 48, [0, 40], [3000]),                       # 1536 rows: fewer slots a row
    (32, 1, 16, 1100, [0, 2, 4, 6, 8], [900, 300, 64, 1]),  # 35200: two a row, blocks of 16 rows
    (32, 1, 16, 1100, [5, 1090], [700]),                    # and of 128
    (2, 1, 32, 200, [2 * g for g in range(70)] + [150], [20 * (g % 4) for g in range(70)]),
])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_shared_many_rows_and_groups(gpu, heads, kv, dim, requests, groups, pre, kind):
    """Rows enough that each has fewer places for pieces; more groups than a wave has lanes,
    empty ones among them."""
    import torch
    rng = np.random.default_rng(requests + dim)
    page = 16
    held = [int(n) for n in rng.integers(0, 40, requests)]
    if requests == 48:
        held[3] = 2500
    capacity = sum(-(-n // page) for n in held + pre) + 1
    pair = Pair(gpu, kv, dim, page, capacity)
    pair.fill(dim)
    lists = lists_for(rng, held + pre, page, capacity)
    for l, n in zip(lists, held + pre):
        if n % page:
            pair.set_counts(l[-1], n % page)
    lists, prefixes = lists[:requests], lists[requests:]
    q = rows(rng, kind, requests, heads, dim)
    out = torch.full_like(q, 9.0)
    fail = torch.zeros(1, dtype=torch.int64, device="cuda")
    shared(pair, Batch(gpu, lists), Prefix(gpu, groups, prefixes), kind, q, out, fail=fail)
    assert int(fail) == 0
    check_shared(pair, lists, groups, prefixes, kind, q, out)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_caches_of_different_sizes_side_by_side(gpu, kind):
    """Handles share kernels, whose LDS goes by each cache's own sizes: the larger ones run
    as before after smaller ones were made."""
    import torch
    rng = np.random.default_rng(44)
    shapes = [(1, 256, 256), (2, 144, 16), (1, 128, 48), (2, 80, 16), (1, 64, 256), (1, 16, 16)]
    pairs = [Pair(gpu, kv, dim, page, 12) for kv, dim, page in shapes]
    for i, pair in enumerate(pairs):
        pair.fill(i)
    lists = [[0, 1], [2], [3, 4, 5]]
    for pair in pairs + pairs[::-1]:
        m = pair.model
        heads = 3 * m.heads
        for new in ([2, 5, 1], [70, 3, 33]):
            q = rows(rng, kind, sum(new), heads, m.dim)
            out = torch.full_like(q, 9.0)
            cross(pair, Batch(gpu, lists, [0] * 3, new), kind, q, out)
            check_cross(pair, lists, new, kind, q, out)
        for users in (3, 33):
            mine = [lists[r % 3] for r in range(users)]
            q = rows(rng, kind, users, heads, m.dim)
            out = torch.full_like(q, 9.0)
            shared(pair, Batch(gpu, mine), Prefix(gpu, [0, users], [[6, 7]]), kind, q, out)
            check_shared(pair, mine, [0, users], [[6, 7]], kind, q, out)
        q = rows(rng, kind, 3, heads, m.dim)
        before, out = sums(pair, rng), torch.full_like(q, 9.0)
        weights = before.clone()
        weigh(pair, Batch(gpu, lists), kind, q, out, weights)
        check_attention(pair, Batch(gpu, lists), kind, q, out)
        check_weights(before, weights, *model_weights(pair, lists, kind, q))
        given, before, new = weights.clone(), snapshot(pair), [[8], [9], [10]]
        got = evict(pair, Batch(gpu, lists), m.page - 1, 1, 2, weights, device(new))
        want = model_evict(pair, lists, m.page - 1, 1, 2, given, new)
        check_evict(pair, lists, new, (weights,) + got, want, before)
