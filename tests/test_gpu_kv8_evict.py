"""dsd_kv8_evict: lists cut to a budget by accumulated weights, against its definition:
the kept places, scales and codes are equal, means within their roundings."""
from __future__ import annotations

import numpy as np
import pytest

import _kv8 as kv8
from test_gpu_kv8 import (TYPES, Batch, Pair, append, attend, check_attention, device, inv_freq,
                          lists_for, model_append, rows)
from test_gpu_kv8_weigh import weigh

pytestmark = pytest.mark.gpu


def evict(pair, batch, keep, first, recent, weights, new_ids, fail=None, stream=0, fill=7):
    """Returns (new counts, kept)."""
    import torch
    B = new_ids.shape[0]
    counts = torch.full((B,), fill, dtype=torch.int32, device="cuda")
    kept = torch.full((B, pair.model.heads, max(keep, 1)), fill, dtype=torch.int32, device="cuda")
    size = pair.cache.evict_workspace_bytes(batch.batch, keep)
    ws = torch.full((size,), 0xff, dtype=torch.uint8, device="cuda")
    pair.cache.evict(batch.batch, keep, first, recent, weights.data_ptr(), new_ids.data_ptr(),
                     new_ids.shape[1], counts.data_ptr(), kept.data_ptr(), workspace=ws.data_ptr(),
                     workspace_bytes=size, fail=0 if fail is None else fail.data_ptr(), stream=stream)
    return counts, kept[..., :keep]


def scale_of(fmt, most):
    """The least scale whose codes reach `most`, from the definition."""
    if fmt == kv8.INT8:
        return np.float32(max(np.float32(most / 127.0), kv8.TINY))
    if not most > 0:
        return kv8.TINY
    fraction, exponent = np.frexp(most)
    return np.float32(2.0 ** max(exponent - 9 + (fraction > 0.875), -126))


def model_evict(pair, lists, keep, first, recent, weights, new_ids):
    """The call on pair.model; returns the weights after it, the counts and kept."""
    m = pair.model
    weights = weights.cpu().numpy().copy()
    kept = np.full((len(lists), m.heads, keep), -1)
    counts = np.zeros(len(lists), int)
    for r, pages in enumerate(lists):
        where = np.array([(p, t, s * m.page + t) for s, p in enumerate(pages)
                          if 0 <= p < m.capacity for t in range(m.counts[p])], int).reshape(-1, 3)
        n = len(where)
        count = min(n, keep)
        counts[r] = -(-count // m.page)
        for h in range(m.heads):
            chosen = np.arange(n)
            if n > keep:
                inner = np.arange(first, n - recent)
                w = weights[where[inner, 0], h, where[inner, 1]].astype(np.float64)
                w = np.where(np.isnan(w), np.inf, w) + 0.0
                top = np.isnan(weights[where[inner, 0], h, where[inner, 1]])
                order = np.lexsort((inner, -w, ~top))[:keep - first - recent]
                chosen = np.sort(np.concatenate([np.arange(first), inner[order],
                                                 np.arange(n - recent, n)]))
            kept[r, h, :count] = where[chosen, 2]
            for i in range(counts[r]):
                new, at = new_ids[r][i], where[chosen[i * m.page:(i + 1) * m.page]]
                moved = weights[at[:, 0], h, at[:, 1]].copy()
                weights[new, h] = 0
                weights[new, h, :len(at)] = moved
                for side in range(2):
                    x = (m.codes[side][at[:, 0], h, at[:, 1]]
                         * m.scales[side][at[:, 0], h].astype(np.float64)[:, None])
                    with np.errstate(invalid="ignore"):
                        s = scale_of(m.fmt, np.abs(np.where(np.isnan(x), 0, x)).max())
                        got = kv8.nearest(m.fmt, x / np.float64(s))
                    m.codes[side][new, h] = 0
                    m.codes[side][new, h, :len(at)] = got
                    m.scales[side][new, h] = s
                m.summaries[new].reshape(m.heads, m.dim)[h] = (
                    m.codes[0][new, h, :len(at)].mean(0) * np.float64(m.scales[0][new, h]))
                m.counts[new] = len(at)
    return weights, counts, kept


def check_evict(pair, lists, new_ids, got, want, before):
    """got: (weights, counts, kept) of the call, want: model_evict's; before: the cache's
    tensors before the call."""
    import torch
    weights, counts, kept = got
    assert np.array_equal(counts.cpu().numpy(), want[1])
    assert np.array_equal(kept.cpu().numpy(), want[2])
    assert np.array_equal(weights.cpu().numpy(), want[0], equal_nan=True)
    written = sorted({p for l, n in zip(new_ids, want[1]) for p in l[:n]})
    pair.check_pages(written)
    k, v = pair.stored()
    for page in written:  # codes behind the tokens
        n = pair.model.counts[page]
        assert not k[page][:, n:].any() and not v[page][:, n:].any()
    rest = np.setdiff1d(np.arange(pair.model.capacity), written)
    for was, now in zip(before, (pair.keys, pair.values, pair.key_scales, pair.value_scales,
                                 pair.counts)):
        index = torch.from_numpy(rest).cuda()
        assert torch.equal(was[index].view(torch.uint8), now[index].view(torch.uint8))


def snapshot(pair):
    return [t.clone() for t in (pair.keys, pair.values, pair.key_scales, pair.value_scales, pair.counts)]


def some_weights(rng, m, style):
    import torch
    shape = (m.capacity, m.heads, m.page)
    if style == "spread":
        w = np.exp(3 * rng.standard_normal(shape))
    elif style == "ties":
        w = rng.integers(0, 4, shape) * 0.25
    elif style == "zero":
        w = np.zeros(shape) * np.where(rng.random(shape) < 0.5, 1, -1)
    else:  # any float: signs, denormals, infinities, NaN
        w = rng.integers(0, 2 ** 32, shape, dtype=np.uint64).astype(np.uint32).view(np.float32)
    return torch.from_numpy(w.astype(np.float32)).cuda()


CASES = [
    # kv heads, dim, page, tokens of a list, keep, first, recent
    (2, 64, 16, [40, 1, 0, 16, 17], 16, 2, 4),
    (1, 128, 16, [300], 33, 0, 0),
    (8, 128, 16, [1000, 900, 100], 256, 4, 64),
    (3, 80, 48, [500, 47], 100, 50, 50),        # nothing by weight
    (2, 256, 64, [700], 129, 1, 1),
    (2, 16, 256, [2000, 256], 300, 0, 7),
    (5, 96, 128, [600, 3], 1, 0, 0),
    (1, 192, 80, [400], 399, 3, 0),             # one goes
    (2, 64, 32, [9000, 5000], 640, 16, 100),    # more than a wave holds of the shortest form
    (1, 32, 16, [40000], 333, 4, 10),           # and of the longest
    (2, 64, 16, [30], 0, 0, 0),
    (4, 64, 112, [1200], 500, 500, 0),
]


@pytest.mark.parametrize("fmt", [kv8.E4M3, kv8.INT8])
@pytest.mark.parametrize("style", ["spread", "ties", "zero", "any"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "%dx%d_p%d_%d_to_%d" % (c[:3] + (sum(c[3]), c[4])))
def test_evict(gpu, case, style, fmt):
    import torch
    kv, dim, page, held, keep, first, recent = case
    rng = np.random.default_rng(dim * page + keep)
    used = sum(-(-n // page) for n in held)
    room = max(-(-keep // page), 1)
    pair = Pair(gpu, kv, dim, page, used + len(held) * room + 2, fmt)
    pair.fill(dim + fmt)
    order = rng.permutation(pair.model.capacity).tolist()
    at, lists = 0, []
    for n in held:
        need = -(-n // page)
        lists.append(order[at:at + need])
        at += need
        if n % page:
            pair.set_counts(lists[-1][-1], n % page)
    new = [order[at + r * room:at + (r + 1) * room] for r in range(len(held))]
    # powers of two and other numbers as the scales before
    if fmt == kv8.E4M3 and style != "ties":
        m = pair.model
        for side, t in ((0, pair.key_scales), (1, pair.value_scales)):
            m.scales[side] = np.exp2(rng.integers(-8, 8, m.scales[side].shape)).astype(np.float32)
            t.copy_(torch.from_numpy(m.scales[side]))
    weights = some_weights(rng, pair.model, style)
    before = snapshot(pair)
    batch = Batch(gpu, lists)
    fail = torch.zeros(1, dtype=torch.int64, device="cuda")
    given = weights.clone()
    counts, kept = evict(pair, batch, keep, first, recent, weights, device(new), fail=fail)
    assert int(fail) == 0
    want = model_evict(pair, lists, keep, first, recent, given, new)
    check_evict(pair, lists, new, (weights, counts, kept), want, before)
    # again, with a hint that is too small and the lists at a stride: the same
    after = snapshot(pair)
    for which in (Batch(gpu, lists, max_pages=1), Batch(gpu, lists, strided=max(len(l) for l in lists) + 1)):
        weights = given.clone()
        counts2, kept2 = evict(pair, which, keep, first, recent, weights, device(new), fail=fail)
        assert int(fail) == 0
        assert torch.equal(counts, counts2) and torch.equal(kept, kept2)
        for was, now in zip(after, snapshot(pair)):
            assert torch.equal(was.view(torch.uint8), now.view(torch.uint8))


@pytest.mark.parametrize("held", [0, 1, 16, 500, 9000, 40000])
def test_evict_keeps_nothing_or_one(gpu, held):
    """A budget of no token empties every list, one of a token keeps one, whatever the
    lists' lengths; neither writes more than it says."""
    import torch
    pages = -(-held // 16)
    rng = np.random.default_rng(held)
    pair = Pair(gpu, 1, 16, 16, pages + 2)
    pair.fill(1)
    if held % 16:
        pair.set_counts(pages - 1, held % 16)
    lists, new = [list(range(pages)), []], [[pages], [pages + 1]]
    for keep, recent in ((0, 0), (1, 0), (1, 1)):
        weights = some_weights(rng, pair.model, "spread")
        given, before = weights.clone(), snapshot(pair)
        counts, kept = evict(pair, Batch(gpu, lists), keep, 0, recent, weights, device(new))
        want = model_evict(pair, lists, keep, 0, recent, given, new)
        check_evict(pair, lists, new, (weights, counts, kept), want, before)
        assert counts.tolist() == [min(held, keep), 0]


@pytest.mark.parametrize("fmt", [kv8.E4M3, kv8.INT8])
def test_evict_any_list(gpu, fmt):
    """Half-full and empty pages in the middle of a list, pages that two lists share; the
    first and last tokens are counted in tokens, not places."""
    import torch
    rng = np.random.default_rng(12)
    pair = Pair(gpu, 2, 64, 16, 60, fmt)
    pair.fill(2)
    for page, count in ((3, 5), (7, 0), (11, 1), (12, 15), (30, 0)):
        pair.set_counts(page, count)
        if count == 0:
            pair.key_scales[page] = float("nan")
            pair.value_scales[page] = float("inf")
    lists = [[3, 9, 7, 11], [30, 12, 12, 5, 7], [7, 30], [], [30, 7, 39, 3, 38, 7, 37, 12, 36, 11, 1, 2, 3, 7]]
    new = [[40 + 4 * r + i for i in range(4)] for r in range(5)]
    for keep, first, recent in ((20, 7, 6), (64, 20, 20), (3, 1, 2)):
        weights = some_weights(rng, pair.model, "spread")
        given, before = weights.clone(), snapshot(pair)
        counts, kept = evict(pair, Batch(gpu, lists), keep, first, recent, weights, device(new))
        want = model_evict(pair, lists, keep, first, recent, given, new)
        check_evict(pair, lists, new, (weights, counts, kept), want, before)


def test_evict_values_at_borders(gpu):
    """NaN codes stay NaN, pages of zeros zero; scales at float32's ends."""
    import torch
    rng = np.random.default_rng(3)
    for fmt in (kv8.E4M3, kv8.INT8):
        pair = Pair(gpu, 1, 64, 16, 16, fmt)
        pair.fill(9)
        m = pair.model
        for side, codes, scales in ((0, pair.keys, pair.key_scales), (1, pair.values, pair.value_scales)):
            ends = [2.0 ** -126, 2.0 ** 119, 1.0, 2.0 ** -100, 3.3, 2.0 ** -126, 1.0, 2.0 ** 119]
            for page, s in enumerate(ends):
                m.scales[side][page] = s
            m.codes[side][6] = 0.0
            codes[6] = 0
            if fmt == kv8.E4M3:
                m.codes[side][2, 0, 5, 7] = np.nan
                if side == 0:
                    codes[2, 0, 5, 7] = 0x7f
                else:
                    codes[2, 0, 0, 7, 5] = 0xff
            scales.copy_(torch.from_numpy(m.scales[side]))
        lists = [[0], [0, 1], [2, 4], [5, 6], [6], [3, 0], [7, 6]]
        new = [[8 + r, 15] for r in range(7)]
        weights = torch.zeros(16, 1, 16, device="cuda")
        given, before = weights.clone(), snapshot(pair)
        counts, kept = evict(pair, Batch(gpu, lists), 16, 0, 7, weights, device(new))
        want = model_evict(pair, lists, 16, 0, 7, given, new)
        check_evict(pair, lists, new, (weights, counts, kept), want, before)


def test_evict_reports_what_does_not_fit(gpu):
    import torch
    rng = np.random.default_rng(16)
    pair = Pair(gpu, 2, 64, 16, 12)
    pair.fill(3)
    lists, new = [[0, 1, 2], [3, 4]], [[8, 9], [10, 11]]
    for bad in (99, -2):
        # a listed page outside the cache holds no token
        weights = some_weights(rng, pair.model, "spread")
        given, before = weights.clone(), snapshot(pair)
        fail = torch.zeros(1, dtype=torch.int64, device="cuda")
        wrong = [[0, bad, 2], [3, 4]]
        counts, kept = evict(pair, Batch(gpu, wrong), 20, 1, 2, weights, device(new), fail=fail)
        assert int(fail) & 0xffffffff == 3
        want = model_evict(pair, wrong, 20, 1, 2, given, new)
        check_evict(pair, wrong, new, (weights, counts, kept), want, before)
        # such a new page takes none
        weights, before = given.clone(), snapshot(pair)
        fail.zero_()
        counts, kept = evict(pair, Batch(gpu, lists), 20, 1, 2, weights, device([[8, bad], [10, 11]]),
                             fail=fail)
        assert int(fail) & 0xffffffff == 3
        want = model_evict(pair, lists, 20, 1, 2, given, new)
        assert np.array_equal(kept.cpu().numpy(), want[2]) and counts.tolist() == [2, 2]
        pair.check_pages([8, 10, 11])
        assert torch.equal(pair.keys[9], before[0][9])
    batch = Batch(gpu, lists)
    for offsets in ([0, 3, 50], [0, -1, 5], [3, 1, 5]):
        batch.keep["page_offsets"].copy_(device(offsets))
        weights = some_weights(rng, pair.model, "spread")
        given, before = weights.clone(), snapshot(pair)
        fail = torch.zeros(1, dtype=torch.int64, device="cuda")
        counts, kept = evict(pair, batch, 20, 1, 2, weights, device(new), fail=fail)
        assert int(fail) & 0xffffffff == 2, offsets
        if offsets[1] == 3:
            want = model_evict(pair, lists[:1], 20, 1, 2, given, new)
            assert np.array_equal(kept[:1].cpu().numpy(), want[2]) and counts.tolist() == [2, 0]
            assert bool((kept[1] == 7).all())
            assert torch.equal(pair.keys[10:], before[0][10:])
            assert torch.equal(weights[10:], given[10:])


def test_evict_refusals(gpu):
    import torch
    pair = Pair(gpu, 2, 64, 16, 8)
    w = torch.zeros(8, 2, 16, device="cuda")
    ids = device([[4, 5], [6, 7]])
    counts, kept = device([0, 0]), device(np.zeros((2, 2, 20)))
    ws = torch.empty(64, dtype=torch.uint8, device="cuda")
    batch = Batch(gpu, [[0], [1]])
    base = dict(keep=20, first=1, recent=2, weights=w.data_ptr(), new_page_ids=ids.data_ptr(),
                new_stride=2, new_page_counts=counts.data_ptr(), kept=kept.data_ptr(),
                workspace=ws.data_ptr(), workspace_bytes=64)
    for bad, what in [(dict(keep=-1), "non-negative"), (dict(first=-1), "non-negative"),
                      (dict(recent=-4), "non-negative"), (dict(first=10, recent=11), "at most keep"),
                      (dict(first=2 ** 31 - 1, recent=2 ** 31 - 1), "at most keep"),
                      (dict(new_stride=1), "new_stride"), (dict(weights=0), "weights"),
                      (dict(weights=w.data_ptr() + 1), "weights"), (dict(new_page_ids=0), "new_page_ids"),
                      (dict(kept=0), "kept"), (dict(new_page_counts=0), "new_page_counts"),
                      (dict(keep=2 ** 31 - 1, new_stride=2 ** 31 - 1), "too large"),
                      (dict(workspace=0), "workspace"), (dict(workspace=ws.data_ptr() + 4), "16-byte"),
                      (dict(workspace_bytes=4), "smaller")]:
        with pytest.raises(gpu.InvalidArgument, match=what):
            pair.cache.evict(batch.batch, **{**base, **bad})
    pair.cache.evict(gpu.Kv8Batch(0), **{**base, "weights": 0, "kept": 0, "workspace": 0})
    torch.cuda.synchronize()


def test_serving_with_a_budget(gpu):
    """Prompts in, steps that weigh, an eviction, steps over what is kept, one more
    eviction: every output against the model's cache; then the eviction replayed."""
    import torch
    rng = np.random.default_rng(21)
    heads, kv, dim, page, keep = 8, 2, 64, 16, 48
    freq = inv_freq(dim)
    order = rng.permutation(60).tolist()
    lists = [order[0:8], order[8:16], order[16:24]]
    spare = [order[24 + 8 * r:32 + 8 * r] for r in range(3)]
    pair = Pair(gpu, kv, dim, page, 60)
    pair.cache.set_rotation(dim, freq)
    weights = torch.zeros(60, kv, page, device="cuda")
    tokens = [100, 5, 64]  # seen so far: positions
    held = [100, 5, 64]    # in the cache
    prompt = Batch(gpu, lists, [0] * 3, held)
    k, v = (rows(rng, "bf16", sum(held), kv, dim) for _ in range(2))
    append(pair, prompt, "bf16", None, k, v, None)
    model_append(pair, prompt, k, v, freq)
    for round_ in range(2):
        for _ in range(3):
            batch = Batch(gpu, lists, held, [1] * 3, positions=tokens)
            qkv = rows(rng, "bf16", 3, heads + 2 * kv, dim)
            q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
            turned = torch.empty(3, heads, dim, device="cuda", dtype=qkv.dtype)
            append(pair, batch, "bf16", q, k, v, turned)
            model_append(pair, batch, k, v, freq, tokens)
            tokens, held = [t + 1 for t in tokens], [t + 1 for t in held]
            mine = Batch(gpu, [l[:-(-n // page)] for l, n in zip(lists, held)])
            out = torch.empty_like(turned)
            weigh(pair, mine, "bf16", turned, out, weights)
            check_attention(pair, mine, "bf16", turned, out)
        mine = [l[:-(-n // page)] for l, n in zip(lists, held)]
        given, before = weights.clone(), snapshot(pair)
        counts, kept = evict(pair, Batch(gpu, mine), keep, 4, 8, weights, device(spare))
        want = model_evict(pair, mine, keep, 4, 8, given, spare)
        check_evict(pair, mine, spare, (weights, counts, kept), want, before)
        held = [min(n, keep) for n in held]
        lists, spare = spare, lists
        pair.counts[device(spare, np.int64).view(-1)] = 0  # the old pages are handed back
        weights[device(spare, np.int64).view(-1)] = 0
        for l in spare:
            pair.model.counts[l] = 0
        q = rows(rng, "bf16", 3, heads, dim)
        out = torch.empty_like(q)
        mine = Batch(gpu, [l[:n] for l, n in zip(lists, counts.tolist())])
        attend(pair, mine, "bf16", q, out)
        check_attention(pair, mine, "bf16", q, out)
    # a replayed eviction reads the weights of its time
    mine = Batch(gpu, [l[:n] for l, n in zip(lists, counts.tolist())])
    ids = device(spare)
    new_counts, kept = device([0] * 3), device(np.zeros((3, kv, 20)))
    ws = torch.empty(pair.cache.evict_workspace_bytes(mine.batch, 20), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pair.cache.evict(mine.batch, 20, 1, 2, weights.data_ptr(), ids.data_ptr(), 8,
                         new_counts.data_ptr(), kept.data_ptr(), workspace=ws.data_ptr(),
                         workspace_bytes=ws.numel(), stream=torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        weights.copy_(some_weights(rng, pair.model, "spread"))
        given, before = weights.clone(), snapshot(pair)
        graph.replay()
        torch.cuda.synchronize()
        want = model_evict(pair, mine.lists, 20, 1, 2, given, spare)
        check_evict(pair, mine.lists, spare, (weights, new_counts, kept), want, before)


def test_evict_new_pages_behind_the_filled_ones(gpu):
    """Entries of new_page_ids behind a list's filled pages may hold anything, and the
    array may end behind the last list's."""
    import torch
    rng = np.random.default_rng(5)
    pair = Pair(gpu, 2, 64, 16, 40)
    pair.fill(6)
    pair.set_counts(9, 3)
    pair.set_counts(12, 15)
    lists = [list(range(0, 5)), list(range(5, 10)), [10], [], [11, 12]]
    new = [[20, 21, 22, 23], [24, 25, 26, 27], [28, -1, 1 << 30, -7], [99, 99, 99, 99], [29, 30, 77, -5]]
    weights = some_weights(rng, pair.model, "spread")
    given, before = weights.clone(), snapshot(pair)
    fail = torch.zeros(1, dtype=torch.int64, device="cuda")
    counts, kept = evict(pair, Batch(gpu, lists), 50, 1, 2, weights, device(new), fail=fail)
    assert int(fail) == 0
    want = model_evict(pair, lists, 50, 1, 2, given, new)
    check_evict(pair, lists, new, (weights, counts, kept), want, before)
    assert counts.tolist() == [4, 4, 1, 0, 2]
