"""dsd_kv8_attend_cross: query tokens over all tokens of their request's list,
against its definition in 64 bits (the roundings are _kv8.allowed's)."""
from __future__ import annotations

import numpy as np
import pytest

import _kv8 as kv8
from test_gpu_kv8 import (TYPES, Batch, Pair, append, as64, device, inv_freq, lists_for,
                          model_append, rows)

pytestmark = pytest.mark.gpu


def cross(pair, batch, kind, q, out, scale=0.0, workspace=True, fail=None, stream=0):
    import torch
    size = pair.cache.workspace_bytes(batch.batch, q.shape[1]) if workspace else 0
    ws = torch.full((max(size, 1),), 0xff, dtype=torch.uint8, device="cuda")
    pair.cache.attend_cross(batch.batch, TYPES[kind], q.shape[1], q.data_ptr(), q.stride(0),
                            out.data_ptr(), out.stride(0), scale,
                            workspace=ws.data_ptr() if size else 0, workspace_bytes=size,
                            fail=0 if fail is None else fail.data_ptr(), stream=stream)
    return ws


def check_cross(pair, lists, new, kind, q, out, scale=0.0):
    m = pair.model
    G = q.shape[1] // m.heads
    q64, got = as64(q), as64(out)
    scale = scale or 1.0 / np.sqrt(m.dim)
    at = 0
    for r, (pages, n) in enumerate(zip(lists, new)):
        keys, values, most = m.rows(np.asarray(pages, int))
        for h in range(m.heads):
            rows_ = q64[at:at + n, h * G:(h + 1) * G].reshape(n * G, m.dim)
            want, weighted, size, peak = kv8.attend(rows_, keys[h], values[h], scale, None, most[h])
            have = got[at:at + n, h * G:(h + 1) * G].reshape(n * G, m.dim)
            may = kv8.allowed(want, weighted, size, peak, m.dim, keys.shape[1], kind)
            bad = ~(np.abs(have - want) <= may)
            assert not bad.any(), (r, h, np.argwhere(bad)[:3], have[bad][:3], want[bad][:3], may[bad][:3])
        at += n


CASES = [
    # heads, kv heads, dim, page, tokens of a list, query tokens
    (8, 2, 128, 16, [33], [1]),
    (8, 2, 128, 16, [1, 0, 17, 64, 65], [3, 2, 0, 5, 16]),
    (8, 2, 128, 16, [0, 300, 15, 1000], [40, 33, 64, 17]),   # many rows, no token for some
    (4, 4, 64, 32, [257, 40], [200, 90]),
    (5, 1, 96, 48, [100, 47], [20, 61]),
    (2, 2, 256, 64, [130, 400], [70, 2]),
    (3, 3, 80, 16, [129], [129]),
    (32, 1, 128, 16, [2000, 31], [9, 3]),
    (20, 20, 64, 16, [1500], [5]),
    (12, 4, 128, 64, [515], [300]),
    (8, 1, 128, 16, [9000], [40]),                           # in pieces, many rows
    (2, 2, 64, 16, [9000, 16], [5, 2]),                      # and few
    (2, 1, 16, 256, [256, 700], [100, 1]),
]


@pytest.mark.parametrize("fmt", [kv8.E4M3, kv8.INT8])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "%dx%dx%d_p%d_%d" % (c[:4] + (sum(c[5]),)))
def test_cross(gpu, case, kind, fmt):
    import torch
    heads, kv, dim, page, held, new = case
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
    # whole lists, and a hint of pages that is too small
    out2 = torch.full_like(q, 9.0)
    cross(pair, batch, kind, q, out2, workspace=False)
    check_cross(pair, lists, new, kind, q, out2)
    small = Batch(gpu, lists, [0] * len(new), new, max_pages=1)
    cross(pair, small, kind, q, out2)
    check_cross(pair, lists, new, kind, q, out2)
    # the lists side by side at a stride
    strided = Batch(gpu, lists, [0] * len(new), new, strided=max(len(l) for l in lists) + 1)
    out2.fill_(9.0)
    cross(pair, strided, kind, q, out2, fail=fail)
    assert int(fail) == 0
    check_cross(pair, lists, new, kind, q, out2)


@pytest.mark.parametrize("new", [3, 70])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_cross_any_list(gpu, kind, new):
    """Pages out of order, half-full and empty ones in the middle, one twice; a stage
    of pages that holds such a one after stages that hold none."""
    import torch
    rng = np.random.default_rng(12)
    pair = Pair(gpu, 2, 128, 16, 700)
    pair.fill(2)
    for page, count in ((3, 5), (7, 0), (11, 1), (12, 15), (30, 0), (650, 4), (651, 0)):
        pair.set_counts(page, count)
        if count == 0:
            pair.key_scales[page] = float("nan")
            pair.value_scales[page] = float("inf")
    lists = [[3, 9, 7, 11], [12, 12, 5], [7, 30], [], [39, 3, 38, 7, 37, 12, 36, 11, 1, 2, 3, 3],
             list(range(40, 700)), [3] + list(range(41, 600))]
    counts = [new, 1, new, 5, new, new, 2]
    q = rows(rng, kind, sum(counts), 8, 128)
    out = torch.full_like(q, 9.0)
    for workspace in (True, False):
        cross(pair, Batch(gpu, lists, [0] * 7, counts), kind, q, out, workspace=workspace)
        check_cross(pair, lists, counts, kind, q, out)
    assert not bool(out[new + 1:2 * new + 6].any())


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_cross_unaligned_rows_and_negative_scale(gpu, kind):
    import torch
    rng = np.random.default_rng(17)
    pair = Pair(gpu, 2, 64, 16, 16)
    pair.fill(11)
    lists, new = [[0, 1, 2], [3, 4, 5, 6], [7]], [3, 40, 1]
    for heads in (4, 18):
        width = heads * 64 + 7
        flat = rows(rng, kind, 1, 1, 44 * width + 1).view(-1)[1:].view(44, width)
        q = flat[:, 3:3 + heads * 64].unflatten(1, (heads, 64))
        wide = torch.full((44, width + 2), 9.0, device="cuda", dtype=q.dtype)
        out = wide[:, 1:1 + heads * 64].unflatten(1, (heads, 64))
        cross(pair, Batch(gpu, lists, [0] * 3, new), kind, q, out, scale=-0.21)
        check_cross(pair, lists, new, kind, q, out, scale=-0.21)
        assert bool((wide[:, 0] == 9.0).all()) and bool((wide[:, 1 + heads * 64:] == 9.0).all())


@pytest.mark.parametrize("new", [4, 60])
def test_cross_nonfinite(gpu, new):
    """A NaN or infinite query reaches its row alone, a NaN value its dim of all rows
    of the request, NaN codes behind a page's tokens nothing."""
    import torch
    rng = np.random.default_rng(14)
    pair = Pair(gpu, 1, 64, 16, 8)
    pair.fill(7)
    pair.set_counts(2, 7)
    batch = Batch(gpu, [[0, 1, 2], [3, 4, 5]], [0, 0], [new, new])
    clean = rows(rng, "bf16", 2 * new, 4, 64)
    q = clean.clone()
    q[0, 1, 3] = float("nan")
    q[new + 1, 2, 0] = float("inf")
    out, want = torch.empty_like(q), torch.empty_like(q)
    cross(pair, batch, "bf16", clean, want)
    assert not bool(want.isnan().any())
    cross(pair, batch, "bf16", q, out)
    assert bool(out[0, 1].isnan().all()) and bool(out[new + 1, 2].isnan().all())
    keep = torch.ones(2 * new, 4, dtype=torch.bool)
    keep[0, 1] = keep[new + 1, 2] = False
    assert torch.equal(out[keep], want[keep])
    pair.values[1, 0, 0, 5, 3] = 0x7f
    cross(pair, batch, "bf16", clean, out)
    assert bool(out[:new, :, 5].isnan().all()) and not bool(out[:new, :, 6].isnan().any())
    assert torch.equal(out[new:], want[new:])


@pytest.mark.parametrize("new", [4, 60])
def test_cross_reports_bad_lists(gpu, new):
    import torch
    rng = np.random.default_rng(16)
    pair = Pair(gpu, 2, 64, 16, 6)
    pair.fill(3)
    q = rows(rng, "bf16", new + 2, 4, 64)
    for bad in (99, -2):
        out = torch.full_like(q, 9.0)
        fail = torch.zeros(1, dtype=torch.int64, device="cuda")
        cross(pair, Batch(gpu, [[0, bad, 1], [2]], [0, 0], [new, 2]), "bf16", q, out, fail=fail)
        assert int(fail) & 0xffffffff == 3
        check_cross(pair, [[0, 1], [2]], [new, 2], "bf16", q, out)  # such a page holds no token
    for name, wrong in (("page_offsets", [0, 2, 50]), ("page_offsets", [0, -1, 3]),
                        ("token_offsets", [0, new, 4000]), ("token_offsets", [0, -1, new + 2]),
                        ("token_offsets", [new + 2, 3, 1])):
        batch = Batch(gpu, [[0, 1], [2]], [0, 0], [new, 2])
        batch.keep[name].copy_(device(wrong))
        out = torch.full_like(q, 9.0)
        fail = torch.zeros(1, dtype=torch.int64, device="cuda")
        cross(pair, batch, "bf16", q, out, fail=fail)
        assert int(fail) & 0xffffffff == 2, (name, wrong)
        if wrong[:2] in ([0, 2], [0, new]):  # the first request is whole, the second left as it was
            check_cross(pair, [[0, 1]], [new], "bf16", q, out)
            assert bool((out[new:] == 9.0).all())


def test_cross_refusals(gpu):
    import torch
    pair = Pair(gpu, 2, 64, 16, 4)
    q = torch.zeros(4, 4, 64, device="cuda", dtype=torch.bfloat16)
    base = dict(dtype=1, num_q_heads=4, q=q.data_ptr(), q_stride=256, out=q.data_ptr(), out_stride=256)
    batch = Batch(gpu, [[0], [1]], [0, 0], [1, 1])
    for bad, what in [(dict(dtype=3), "type"), (dict(num_q_heads=3), "multiple"),
                      (dict(num_q_heads=0), "positive"), (dict(q=0), "non-null"),
                      (dict(q_stride=255), "stride"), (dict(out=q.data_ptr() + 1), "aligned"),
                      (dict(scale=float("inf")), "scale"),
                      (dict(workspace=q.data_ptr() + 2, workspace_bytes=64), "16-byte")]:
        with pytest.raises(gpu.InvalidArgument, match=what):
            pair.cache.attend_cross(batch.batch, **{**base, **bad})
    good = dict(batch=2, tokens=2, max_tokens=1, max_pages=1, total_pages=2,
                **{n: t.data_ptr() for n, t in batch.keep.items()})
    for bad, what in [(dict(token_offsets=0), "token_offsets"), (dict(max_tokens=0), "max_tokens"),
                      (dict(tokens=1 << 30, max_tokens=1 << 30), "31 bits")]:
        with pytest.raises(gpu.InvalidArgument, match=what):
            pair.cache.attend_cross(gpu.Kv8Batch(**{**good, **bad}), **base)
    pair.cache.attend_cross(gpu.Kv8Batch(**{**good, "past_tokens": 0}), **base)
    pair.cache.attend_cross(gpu.Kv8Batch(0), **base)
    torch.cuda.synchronize()


def test_encoder_then_decoder(gpu):
    """An encoder's states go into the cache, its own rows look at all of them, then a
    decoder's tokens do, eagerly and as a replayed graph."""
    import torch
    rng = np.random.default_rng(23)
    heads, kv, dim, page = 8, 2, 64, 16
    held = [150, 33, 16]
    capacity = sum(-(-n // page) for n in held)
    lists = lists_for(rng, held, page, capacity)
    pair = Pair(gpu, kv, dim, page, capacity)
    states = Batch(gpu, lists, [0] * 3, held)
    k, v = (rows(rng, "bf16", sum(held), kv, dim) for _ in range(2))
    append(pair, states, "bf16", None, k, v, None)
    model_append(pair, states, k, v, inv_freq(0))
    q = rows(rng, "bf16", sum(held), heads, dim)
    out = torch.empty_like(q)
    cross(pair, states, "bf16", q, out)
    check_cross(pair, lists, held, "bf16", q, out)
    new = [4, 1, 6]
    batch = Batch(gpu, lists, [0] * 3, new)
    inputs = [rows(rng, "bf16", sum(new), heads, dim) for _ in range(3)]
    size = pair.cache.workspace_bytes(batch.batch, heads)
    ws = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    q, out = torch.empty_like(inputs[0]), torch.empty_like(inputs[0])

    def step():
        pair.cache.attend_cross(batch.batch, 1, heads, q.data_ptr(), q.stride(0), out.data_ptr(),
                                out.stride(0), workspace=ws.data_ptr(), workspace_bytes=size,
                                stream=torch.cuda.current_stream().cuda_stream)

    want = []
    for x in inputs:
        q.copy_(x)
        step()
        torch.cuda.synchronize()
        check_cross(pair, lists, new, "bf16", q, out)
        want.append(out.clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in (0, 2, 1, 1):
        q.copy_(inputs[i])
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])
