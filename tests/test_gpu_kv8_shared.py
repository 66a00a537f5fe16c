"""dsd_kv8_attend_shared: one token a request over its group's prefix and its own list,
against its definition in 64 bits (the roundings are _kv8.allowed's)."""
from __future__ import annotations

import numpy as np
import pytest

import _kv8 as kv8
from test_gpu_kv8 import (TYPES, Batch, Pair, append, as64, attend, check_attention, device,
                          inv_freq, lists_for, model_append, rows)

pytestmark = pytest.mark.gpu


class Prefix:
    """A Kv8Prefix from host lists; keeps its tensors."""

    def __init__(self, gpu, starts, lists, max_requests=None, max_pages=None):
        self.starts, self.lists = starts, lists
        flat = [p for l in lists for p in l]
        self.keep = {"request_offsets": device(starts), "page_ids": device(flat if flat else [0]),
                     "page_offsets": device(np.concatenate([[0], np.cumsum([len(l) for l in lists])]))}
        longest = max([len(l) for l in lists] + [0])
        most = max([b - a for a, b in zip(starts, starts[1:])] + [0])
        self.prefix = gpu.Kv8Prefix(len(lists), max_requests=most if max_requests is None else max_requests,
                                    max_pages=longest if max_pages is None else max_pages,
                                    total_pages=len(flat),
                                    **{n: t.data_ptr() for n, t in self.keep.items()})


def shared(pair, batch, prefix, kind, q, out, scale=0.0, fail=None, stream=0, ws=None):
    import torch
    size = pair.cache.shared_workspace_bytes(batch.batch, prefix.prefix, q.shape[1])
    if ws is None:
        ws = torch.full((max(size, 1),), 0xff, dtype=torch.uint8, device="cuda")
    pair.cache.attend_shared(batch.batch, prefix.prefix, TYPES[kind], q.shape[1], q.data_ptr(),
                             q.stride(0), out.data_ptr(), out.stride(0), scale,
                             workspace=ws.data_ptr(), workspace_bytes=size,
                             fail=0 if fail is None else fail.data_ptr(), stream=stream)
    return ws


def check_shared(pair, lists, starts, prefixes, kind, q, out, scale=0.0):
    m = pair.model
    G = q.shape[1] // m.heads
    q64, got = as64(q), as64(out)
    scale = scale or 1.0 / np.sqrt(m.dim)
    for r, pages in enumerate(lists):
        mine = [g for g in range(len(prefixes)) if starts[g] <= r < starts[g + 1]]
        parts = [m.rows(np.asarray(l, int)) for l in [prefixes[g] for g in mine] + [pages]]
        keys, values, most = (np.concatenate([p[i] for p in parts], 1) for i in range(3))
        for h in range(m.heads):
            rows_ = q64[r, h * G:(h + 1) * G]
            want, weighted, size, peak = kv8.attend(rows_, keys[h], values[h], scale, None, most[h])
            have = got[r, h * G:(h + 1) * G]
            may = kv8.allowed(want, weighted, size, peak, m.dim, keys.shape[1], kind)
            bad = ~(np.abs(have - want) <= may)
            assert not bad.any(), (r, h, np.argwhere(bad)[:3], have[bad][:3], want[bad][:3], may[bad][:3])


CASES = [
    # heads, kv heads, dim, page, own tokens, first requests of groups, prefix tokens
    (8, 2, 128, 16, [5, 0, 17, 300], [0, 4], [100]),
    (8, 2, 128, 16, [1, 33], [0, 2], [1]),
    (4, 4, 128, 16, [40], [0, 1], [3000]),                         # a group of one
    (8, 2, 64, 32, [7, 100, 0, 0, 65, 1, 2], [1, 3, 3, 6], [50, 70, 0]),  # alone, empty groups
    (8, 1, 128, 16, [20 + i for i in range(9)], [0, 9], [5000]),   # 72 rows: blocks of 128
    (8, 1, 128, 16, [20 + i for i in range(40)], [3, 38], [1000]),  # 280 rows
    (20, 1, 128, 64, [5, 700, 64, 0], [0, 2, 4], [129, 1000]),
    (7, 1, 96, 48, [100, 47], [0, 2], [300]),
    (3, 3, 80, 16, [77, 30] * 40, [0, 40, 80], [400, 17]),
    (2, 2, 16, 16, [33, 1], [0, 2], [90]),
    (6, 2, 256, 128, [128, 130, 513], [0, 3], [600]),
    (12, 1, 192, 256, [255, 60] * 4, [0, 8], [900]),
    (32, 8, 128, 16, [200, 900, 30], [0, 3], [20000]),             # long
    (32, 8, 128, 16, [9000, 20, 50], [0, 3], [200]),
    (16, 4, 64, 16, [30] * 20, [0, 20], [0]),                      # a prefix of nothing
]


@pytest.mark.parametrize("fmt", [kv8.E4M3, kv8.INT8])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "%dx%dx%d_p%d_%d_%d" % (c[:4] + (len(c[4]), sum(c[6]))))
def test_shared(gpu, case, kind, fmt):
    import torch
    heads, kv, dim, page, held, starts, pre = case
    rng = np.random.default_rng(heads * dim + page + sum(held))
    capacity = sum(-(-n // page) for n in held + pre) + 1
    pair = Pair(gpu, kv, dim, page, capacity, fmt)
    pair.fill(dim + fmt)
    lists = lists_for(rng, held + pre, page, capacity)
    for l, n in zip(lists, held + pre):
        if n % page:
            pair.set_counts(l[-1], n % page)
    lists, prefixes = lists[:len(held)], lists[len(held):]
    q = rows(rng, kind, len(held) + 1, heads, dim)
    out = torch.full_like(q, 9.0)
    fail = torch.zeros(1, dtype=torch.int64, device="cuda")
    batch, prefix = Batch(gpu, lists), Prefix(gpu, starts, prefixes)
    shared(pair, batch, prefix, kind, q, out, fail=fail)
    assert int(fail) == 0
    check_shared(pair, lists, starts, prefixes, kind, q, out)
    assert bool((out[len(held)] == 9.0).all())  # a row behind the last request
    again = torch.full_like(q, 9.0)
    shared(pair, batch, prefix, kind, q, again)
    assert torch.equal(out, again)
    # hints of pages that are too small, lists at a stride
    for b, p in ((Batch(gpu, lists, max_pages=1), Prefix(gpu, starts, prefixes, max_pages=1)),
                 (Batch(gpu, lists, strided=max(len(l) for l in lists) + 1),
                  Prefix(gpu, starts, prefixes, max_requests=1000))):
        out.fill_(9.0)
        shared(pair, b, p, kind, q, out, fail=fail)
        assert int(fail) == 0
        check_shared(pair, lists, starts, prefixes, kind, q, out)


@pytest.mark.parametrize("requests", [3, 30])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_shared_any_list(gpu, kind, requests):
    """Half-full and empty pages in the middle of prefixes and lists, pages twice; a
    request's list may name its prefix's pages too."""
    import torch
    rng = np.random.default_rng(12)
    pair = Pair(gpu, 2, 128, 16, 40)
    pair.fill(2)
    for page, count in ((3, 5), (7, 0), (11, 1), (12, 15), (30, 0)):
        pair.set_counts(page, count)
        if count == 0:
            pair.key_scales[page] = float("nan")
            pair.value_scales[page] = float("inf")
    some = [[3, 9, 7, 11], [12, 12, 5], [7, 30], [], [39, 3, 38]]
    lists = [some[r % 5] for r in range(requests)]
    prefixes = [[30, 12, 36, 11, 1, 2, 3, 3], [7, 7], [9, 20, 12, 21]]
    starts = [0, requests - 2, requests - 1, requests]
    q = rows(rng, kind, requests, 8, 128)
    out = torch.full_like(q, 9.0)
    shared(pair, Batch(gpu, lists), Prefix(gpu, starts, prefixes), kind, q, out)
    check_shared(pair, lists, starts, prefixes, kind, q, out)
    # nothing anywhere: zeros
    empty = Prefix(gpu, [0, requests], [[7, 30]])
    shared(pair, Batch(gpu, [[30]] * requests), empty, kind, q, out)
    assert not bool(out.any())


@pytest.mark.parametrize("requests", [4, 40])
def test_shared_scales_that_differ_widely(gpu, requests):
    """Logits of hundreds and value scales 2^40 apart between prefix and lists."""
    import torch
    rng = np.random.default_rng(13)
    for fmt in (kv8.E4M3, kv8.INT8):
        pair = Pair(gpu, 1, 64, 16, 24, fmt)
        pair.fill(5)
        factor = np.exp2(rng.permutation(24) * 2.0 - 24).astype(np.float32)[:, None]
        pair.model.scales[1] = pair.model.scales[1] * factor
        pair.value_scales.copy_(torch.from_numpy(pair.model.scales[1]))
        for kind in ("f32", "f16"):
            q = rows(rng, kind, requests, 4, 64) * 20
            out = torch.empty_like(q)
            lists = [[int(rng.integers(12, 24))] for _ in range(requests)]
            shared(pair, Batch(gpu, lists), Prefix(gpu, [0, requests], [list(range(12))]), kind, q, out,
                   scale=1.5)
            check_shared(pair, lists, [0, requests], [list(range(12))], kind, q, out, scale=1.5)


@pytest.mark.parametrize("requests", [3, 30])
def test_shared_nonfinite_and_unaligned(gpu, requests):
    """A NaN query reaches its row alone, a NaN value of the prefix its dim of all rows of
    the group and of no other; rows start on any element."""
    import torch
    rng = np.random.default_rng(14)
    pair = Pair(gpu, 1, 64, 16, 12)
    pair.fill(7)
    lists = [[4 + r % 7] for r in range(requests)]
    prefix = Prefix(gpu, [0, requests - 1], [[0, 1, 2]])
    width = 4 * 64 + 3
    flat = rows(rng, "bf16", 1, 1, requests * width + 1).view(-1)[1:].view(requests, width)
    q = flat[:, 1:1 + 256].unflatten(1, (4, 64))
    wide = torch.full((requests, width), 9.0, device="cuda", dtype=q.dtype)
    out = wide[:, 1:1 + 256].unflatten(1, (4, 64))
    shared(pair, Batch(gpu, lists), prefix, "bf16", q, out)
    check_shared(pair, lists, prefix.starts, prefix.lists, "bf16", q, out)
    assert bool((wide[:, 0] == 9.0).all()) and bool((wide[:, 257:] == 9.0).all())
    want = out.clone()
    q[0, 1, 3] = float("nan")
    shared(pair, Batch(gpu, lists), prefix, "bf16", q, out)
    assert bool(out[0, 1].isnan().all())
    keep = torch.ones(requests, 4, dtype=torch.bool)
    keep[0, 1] = False
    assert torch.equal(out[keep], want[keep])
    pair.values[1, 0, 0, 5, 3] = 0x7f
    shared(pair, Batch(gpu, lists), prefix, "bf16", q, out)
    assert bool(out[:requests - 1, :, 5].isnan().all())
    keep[0, 0] = True
    assert torch.equal(out[1:requests - 1, :, 6], want[1:requests - 1, :, 6])
    assert torch.equal(out[requests - 1], want[requests - 1])


@pytest.mark.parametrize("requests", [4, 40])
def test_shared_reports_what_does_not_fit(gpu, requests):
    import torch
    rng = np.random.default_rng(16)
    pair = Pair(gpu, 2, 64, 16, 12)
    pair.fill(3)
    q = rows(rng, "bf16", requests, 4, 64)
    lists, half = [[4 + r % 8] for r in range(requests)], requests // 2
    starts, prefixes = [0, half, requests], [[0, 1], [2, 3]]

    def run(batch, prefix, code):
        out = torch.full_like(q, 9.0)
        fail = torch.zeros(1, dtype=torch.int64, device="cuda")
        shared(pair, batch, prefix, "bf16", q, out, fail=fail)
        assert int(fail) & 0xffffffff == code
        return out

    for bad in (99, -2):  # a page outside the cache holds no token
        out = run(Batch(gpu, lists), Prefix(gpu, starts, [[0, bad, 1], [2, 3]]), 3)
        check_shared(pair, lists, starts, prefixes, "bf16", q, out)
    for wrong in ([0, 2, 50], [0, -1, 4], [3, 1, 4]):  # a prefix list that does not fit holds none
        prefix = Prefix(gpu, starts, prefixes)
        prefix.keep["page_offsets"].copy_(device(wrong))
        out = run(Batch(gpu, lists), prefix, 2)
        if wrong[1] == 2:
            check_shared(pair, lists, starts, [[0, 1], []], "bf16", q, out)
    for wrong, first in (([0, half, 70000], True), ([0, -5, requests], False), ([-1, half, requests], None),
                         ([0, half, half - 1], True)):
        prefix = Prefix(gpu, starts, prefixes)
        prefix.keep["request_offsets"].copy_(device(wrong))
        out = run(Batch(gpu, lists), prefix, 2)
        if first is True:
            check_shared(pair, lists, starts, [[0, 1], []], "bf16", q, out)
        elif first is None:
            check_shared(pair, lists, starts, [[], [2, 3]], "bf16", q, out)
    # ranges that overlap: such requests have no prefix, others theirs
    prefix = Prefix(gpu, [0, requests - 1, 1, requests], [[0, 1], [], [2, 3]], max_requests=requests)
    out = run(Batch(gpu, lists), prefix, 2)
    no = [[], [], [], []]
    check_shared(pair, lists[:1], [0, 1], [[0, 1]], "bf16", q, out)
    check_shared(pair, lists[1:requests - 1], [0], [], "bf16", q[1:requests - 1], out[1:requests - 1])
    check_shared(pair, lists[-1:], [0, 1], [[2, 3]], "bf16", q[-1:], out[-1:])
    # a group of more requests than max_requests
    out = run(Batch(gpu, lists), Prefix(gpu, [0, 1, requests], prefixes, max_requests=1), 2)
    check_shared(pair, lists, [0, 1, requests], [[0, 1], []], "bf16", q, out)
    # an own list that does not fit holds no token
    batch = Batch(gpu, lists)
    offsets = list(range(requests + 1))
    offsets[-1] = 4000
    batch.keep["page_offsets"].copy_(device(offsets))
    out = run(batch, Prefix(gpu, starts, prefixes), 2)
    check_shared(pair, lists[:-1] + [[]], starts, prefixes, "bf16", q, out)


def test_shared_refusals(gpu):
    import torch
    pair = Pair(gpu, 2, 64, 16, 4)
    q = torch.zeros(4, 4, 64, device="cuda", dtype=torch.bfloat16)
    batch, prefix = Batch(gpu, [[0], [1]]), Prefix(gpu, [0, 2], [[2, 3]])
    size = pair.cache.shared_workspace_bytes(batch.batch, prefix.prefix, 4)
    ws = torch.empty(size + 16, dtype=torch.uint8, device="cuda")
    base = dict(dtype=1, num_q_heads=4, q=q.data_ptr(), q_stride=256, out=q.data_ptr(), out_stride=256,
                workspace=ws.data_ptr(), workspace_bytes=size)
    for bad, what in [(dict(dtype=3), "type"), (dict(num_q_heads=3), "multiple"), (dict(q=0), "non-null"),
                      (dict(workspace=0), "smaller"), (dict(workspace_bytes=64), "smaller"),
                      (dict(workspace=ws.data_ptr() + 8), "16-byte"), (dict(scale=float("nan")), "scale")]:
        with pytest.raises(gpu.InvalidArgument, match=what):
            pair.cache.attend_shared(batch.batch, prefix.prefix, **{**base, **bad})
    given = dict(groups=1, max_requests=2, max_pages=2, total_pages=2,
                 **{n: t.data_ptr() for n, t in prefix.keep.items()})
    for bad, what in [(dict(groups=-1), "non-negative"), (dict(groups=70000), "65535"),
                      (dict(max_requests=-1), "non-negative"), (dict(request_offsets=0), "request_offsets"),
                      (dict(page_offsets=0), "page_offsets"), (dict(page_ids=0), "page_ids"),
                      (dict(max_requests=1 << 30), "31 bits")]:
        with pytest.raises(gpu.InvalidArgument, match=what):
            pair.cache.attend_shared(batch.batch, gpu.Kv8Prefix(**{**given, **bad}), **base)
    pair.cache.attend_shared(gpu.Kv8Batch(0), prefix.prefix, **{**base, "workspace": 0})
    # without groups it is attend
    pair.fill(3)
    q = rows(np.random.default_rng(1), "bf16", 2, 4, 64)
    out, want = torch.empty_like(q), torch.empty_like(q)
    pair.cache.attend_shared(batch.batch, gpu.Kv8Prefix(0), 1, 4, q.data_ptr(), 256, out.data_ptr(), 256,
                             workspace=ws.data_ptr(), workspace_bytes=size)
    attend(pair, batch, "bf16", q, want)
    assert torch.equal(out, want)
    # a workspace of a larger batch does, whatever the prefixes
    for B in (1, 4, 64, 700):
        most = pair.cache.shared_workspace_bytes(gpu.Kv8Batch(B, max_pages=100), gpu.Kv8Prefix(0), 4)
        for b in (1, 2, 30, 64, 500):
            if b <= B:
                less = pair.cache.shared_workspace_bytes(gpu.Kv8Batch(b, max_pages=1000),
                                                         gpu.Kv8Prefix(3, max_pages=5000), 4)
                assert less <= most


def test_serving_behind_a_prompt(gpu):
    """A system prompt goes in once, its users' turns behind it: the prompt's pages lead
    each user's list for append, and are the group's prefix for attention.  Eagerly, as a
    replayed graph, and on streams of their own."""
    import torch
    rng = np.random.default_rng(21)
    heads, kv, dim, page, users = 8, 2, 64, 16, 5
    freq = inv_freq(dim)
    order = rng.permutation(40).tolist()
    prompt, turns = order[:6], [order[6 + 4 * u:10 + 4 * u] for u in range(users)]
    pair = Pair(gpu, kv, dim, page, 40)
    pair.cache.set_rotation(dim, freq)
    first = Batch(gpu, [prompt], [0], [96])
    k, v = (rows(rng, "bf16", 96, kv, dim) for _ in range(2))
    append(pair, first, "bf16", None, k, v, None)
    model_append(pair, first, k, v, freq)
    past, new = [0] * users, [20, 1, 16, 40, 7]
    prefix = Prefix(gpu, [0, users], [prompt])
    for step in range(4):
        batch = Batch(gpu, turns, past, new, positions=[96 + p + i for p, n in zip(past, new) for i in range(n)])
        qkv = rows(rng, "bf16", batch.tokens, heads + 2 * kv, dim)
        q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
        turned = torch.empty(batch.tokens, heads, dim, device="cuda", dtype=qkv.dtype)
        append(pair, batch, "bf16", q, k, v, turned)
        model_append(pair, batch, k, v, freq, [96 + p + i for p, n in zip(past, new) for i in range(n)])
        past = [p + n for p, n in zip(past, new)]
        new = [1] * users
        if step == 0:
            continue
        mine = [l[:-(-p // page)] for l, p in zip(turns, past)]
        out = torch.empty_like(turned)
        shared(pair, Batch(gpu, mine), prefix, "bf16", turned, out)
        check_shared(pair, mine, [0, users], [prompt], "bf16", turned, out)
        whole = torch.empty_like(turned)  # the same from lists that name the prompt's pages
        attend(pair, Batch(gpu, [prompt + l for l in mine]), "bf16", turned, whole)
        check_attention(pair, Batch(gpu, [prompt + l for l in mine]), "bf16", turned, whole)
    batch = Batch(gpu, mine)
    size = pair.cache.shared_workspace_bytes(batch.batch, prefix.prefix, heads)
    inputs = [rows(rng, "bf16", users, heads, dim) for _ in range(3)]
    q, out = torch.empty_like(inputs[0]), torch.empty_like(inputs[0])
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    want = []
    for x in inputs:
        q.copy_(x)
        shared(pair, batch, prefix, "bf16", q, out)
        torch.cuda.synchronize()
        want.append(out.clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        shared(pair, batch, prefix, "bf16", q, out, ws=ws, stream=torch.cuda.current_stream().cuda_stream)
    for i in (0, 2, 1, 1):
        q.copy_(inputs[i])
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])
    streams, outs = [torch.cuda.Stream() for _ in inputs], [torch.empty_like(q) for _ in inputs]
    spaces = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in inputs]
    torch.cuda.synchronize()
    for x, o, w, s in zip(inputs, outs, spaces, streams):
        shared(pair, batch, prefix, "bf16", x, o, ws=w, stream=s.cuda_stream)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)
