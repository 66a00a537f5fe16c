"""dsd_kv8_attend_weigh: attention of one token a request that adds up what each cached
token weighed, against its definition in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import _kv8 as kv8
from test_gpu_kv8 import (ATTEND, TYPES, Batch, Pair, as64, attend, check_attention, device,
                          lists_for, rows)

pytestmark = pytest.mark.gpu


def weigh(pair, batch, kind, q, out, weights, scale=0.0, fail=None, stream=0, ws=None):
    import torch
    size = pair.cache.weigh_workspace_bytes(batch.batch, q.shape[1])
    if ws is None:
        ws = torch.full((max(size, 1),), 0xff, dtype=torch.uint8, device="cuda")
    pair.cache.attend_weigh(batch.batch, TYPES[kind], q.shape[1], q.data_ptr(), q.stride(0),
                            out.data_ptr(), out.stride(0), scale, weights=weights.data_ptr(),
                            workspace=ws.data_ptr(), workspace_bytes=size,
                            fail=0 if fail is None else fail.data_ptr(), stream=stream)
    return ws


def model_weights(pair, lists, kind, q, scale=0.0):
    """What a call adds, and how far a call's sum may be from it.

    A logit is off by (dim + 8) 2^-24 + 2^-21 of sum |q k| (_kv8.allowed), held in
    float32 for the second launch (2^-24 of it) and so is its row's maximum; a weight's
    relative error is twice that for the logit and its row's maximum and sum, 2^-21 for
    two exponentials, tokens 2^-24 for the row's sum, 8 2^-24 for the divisions and
    products; group 2^-24 more for the sum over heads.  2^-126: what exp2 gives nothing
    of, a head each."""
    m = pair.model
    G = q.shape[1] // m.heads
    q64 = as64(q)
    scale = scale or 1.0 / np.sqrt(m.dim)
    add = np.zeros((m.capacity, m.heads, m.page))
    may = np.zeros_like(add)
    for r, pages in enumerate(lists):
        pages = np.asarray(pages, int)
        keys, _, _ = m.rows(pages)
        n = keys.shape[1]
        if n == 0:
            continue
        where = [(p, t) for p in pages for t in range(m.counts[p])]
        p_, t_ = np.array([w[0] for w in where]), np.array([w[1] for w in where])
        for h in range(m.heads):
            x = q64[r, h * G:(h + 1) * G]
            s = scale * (x @ keys[h].T)
            size = np.abs(scale) * (np.abs(x) @ np.abs(keys[h]).T)
            w = np.exp(s - s.max(1, keepdims=True))
            w /= w.sum(1, keepdims=True)
            off = ((m.dim + 9) * 2.0 ** -24 + 2.0 ** -21) * size.max(1, keepdims=True)
            rel = 4 * off + 2 * 2.0 ** -21 + (n + 8 + G) * 2.0 ** -24
            np.add.at(add, (p_, h, t_), w.sum(0))
            np.add.at(may, (p_, h, t_), (w * rel).sum(0) + G * 2.0 ** -126)
    return add, may


def check_weights(before, got, add, may):
    """Adding rounds once a list that names the page: at most 4 here."""
    want = as64(before) + add
    slack = may + 4 * 2.0 ** -24 * np.abs(want)
    slack[add == 0] = 0.0
    bad = ~(np.abs(as64(got) - want) <= slack)
    assert not bad.any(), (np.argwhere(bad)[:3], as64(got)[bad][:3], want[bad][:3], slack[bad][:3])


def sums(pair, rng):
    import torch
    m = pair.model
    return torch.from_numpy(rng.uniform(0, 3, (m.capacity, m.heads, m.page)).astype(np.float32)).cuda()


@pytest.mark.parametrize("fmt", [kv8.E4M3, kv8.INT8])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", ATTEND + [(70, 1, 64, 16, [40, 900])],
                         ids=lambda c: "%dx%dx%d_p%d_%d" % (c[:4] + (sum(c[4]),)))
def test_weigh(gpu, case, kind, fmt):
    import torch
    heads, kv, dim, page, lengths = case
    rng = np.random.default_rng(heads * dim + page)
    capacity = sum(-(-n // page) for n in lengths) + 2
    pair = Pair(gpu, kv, dim, page, capacity, fmt)
    pair.fill(dim + fmt)
    lists = lists_for(rng, lengths, page, capacity)
    for l, n in zip(lists, lengths):
        if n % page:
            pair.set_counts(l[-1], n % page)
    q = rows(rng, kind, len(lengths), heads, dim)
    add, may = model_weights(pair, lists, kind, q)
    batch = Batch(gpu, lists)
    fail = torch.zeros(1, dtype=torch.int64, device="cuda")
    plain = torch.full_like(q, 9.0)
    attend(pair, batch, kind, q, plain)
    strided = Batch(gpu, lists, strided=max(len(l) for l in lists) + 1)
    small = Batch(gpu, lists, max_pages=1)  # a hint that is too small
    for which in (batch, strided, small):
        before = sums(pair, rng)
        weights, out = before.clone(), torch.full_like(q, 9.0)
        weigh(pair, which, kind, q, out, weights, fail=fail)
        assert int(fail) == 0
        check_attention(pair, batch, kind, q, out)
        check_weights(before, weights, add, may)
        if which is batch:
            assert torch.equal(out, plain)
            again = before.clone()
            weigh(pair, which, kind, q, out, again)
            assert torch.equal(again, weights)  # the same from run to run


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_weigh_any_list(gpu, kind):
    """Pages out of order, half-full and empty ones in the middle, one twice, one in
    several lists: each of them counts."""
    import torch
    rng = np.random.default_rng(12)
    pair = Pair(gpu, 2, 128, 16, 40)
    pair.fill(2)
    for page, count in ((3, 5), (7, 0), (11, 1), (12, 15), (30, 0)):
        pair.set_counts(page, count)
        if count == 0:
            pair.key_scales[page] = float("nan")
            pair.value_scales[page] = float("inf")
    lists = [[3, 9, 7, 11], [12, 12, 5], [7, 30], [], [39, 3, 38, 7, 37, 12, 36, 11, 1, 2, 3, 3]]
    q = rows(rng, kind, len(lists), 8, 128)
    out, before = torch.full_like(q, 9.0), sums(pair, rng)
    weights = before.clone()
    batch = Batch(gpu, lists)
    weigh(pair, batch, kind, q, out, weights)
    check_attention(pair, batch, kind, q, out)
    check_weights(before, weights, *model_weights(pair, lists, kind, q))
    assert not bool(out[2].any()) and not bool(out[3].any())


def test_weigh_far_logits_and_nonfinite(gpu):
    """Logits of thousands leave one token; a NaN query makes its key head's tokens NaN
    and no other's."""
    import torch
    rng = np.random.default_rng(13)
    pair = Pair(gpu, 2, 64, 16, 6)
    pair.fill(5)
    lists = [[0, 1, 2], [3, 4, 5]]
    q = rows(rng, "f32", 2, 4, 64) * 400
    out, before = torch.empty_like(q), torch.zeros(6, 2, 16, device="cuda")
    weights = before.clone()
    weigh(pair, Batch(gpu, lists), "f32", q, out, weights)
    check_weights(before, weights, *model_weights(pair, lists, "f32", q))
    total = weights.double().sum((0, 2)).cpu().numpy()
    assert np.abs(total - 4.0).max() < 1e-4  # two requests of two heads
    q[0, 3, 5] = float("nan")
    want = weights.clone()
    weights.zero_()
    weigh(pair, Batch(gpu, lists), "f32", q, out, weights)
    assert bool(weights[:3, 1].isnan().all())
    assert torch.equal(weights[3:], want[3:]) and torch.equal(weights[:3, 0], want[:3, 0])


def test_weigh_reports_bad_lists(gpu):
    import torch
    rng = np.random.default_rng(16)
    pair = Pair(gpu, 2, 64, 16, 6)
    pair.fill(3)
    q = rows(rng, "bf16", 2, 4, 64)
    for bad in (99, -2):
        out, before = torch.full_like(q, 9.0), sums(pair, rng)
        weights = before.clone()
        fail = torch.zeros(1, dtype=torch.int64, device="cuda")
        weigh(pair, Batch(gpu, [[0, bad, 1], [2]]), "bf16", q, out, weights, fail=fail)
        assert int(fail) & 0xffffffff == 3
        check_attention(pair, Batch(gpu, [[0, 1], [2]]), "bf16", q, out)
        check_weights(before, weights, *model_weights(pair, [[0, 1], [2]], "bf16", q))
    batch = Batch(gpu, [[0, 1], [2]])
    for offsets in ([0, 2, 50], [0, -1, 3], [2, 1, 3]):
        batch.keep["page_offsets"].copy_(device(offsets))
        out, before = torch.full_like(q, 9.0), sums(pair, rng)
        weights = before.clone()
        fail = torch.zeros(1, dtype=torch.int64, device="cuda")
        weigh(pair, batch, "bf16", q, out, weights, fail=fail)
        assert int(fail) & 0xffffffff == 2, offsets
        if offsets == [0, 2, 50]:  # zeros, and no weight, for that request alone
            assert not bool(out[1].any())
            check_weights(before, weights, *model_weights(pair, [[0, 1], []], "bf16", q))


def test_weigh_refusals(gpu):
    import torch
    pair = Pair(gpu, 2, 64, 16, 4)
    q = torch.zeros(4, 4, 64, device="cuda", dtype=torch.bfloat16)
    w = torch.zeros(4, 2, 16, device="cuda")
    batch = Batch(gpu, [[0], [1]])
    size = pair.cache.weigh_workspace_bytes(batch.batch, 4)
    ws = torch.empty(size + 16, dtype=torch.uint8, device="cuda")
    base = dict(dtype=1, num_q_heads=4, q=q.data_ptr(), q_stride=256, out=q.data_ptr(), out_stride=256,
                weights=w.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=size)
    for bad, what in [(dict(dtype=3), "type"), (dict(num_q_heads=3), "multiple"), (dict(q=0), "non-null"),
                      (dict(weights=0), "weights"), (dict(weights=w.data_ptr() + 2), "weights"),
                      (dict(workspace=0), "smaller"), (dict(workspace_bytes=64), "smaller"),
                      (dict(workspace=ws.data_ptr() + 8), "16-byte"), (dict(scale=float("nan")), "scale")]:
        with pytest.raises(gpu.InvalidArgument, match=what):
            pair.cache.attend_weigh(batch.batch, **{**base, **bad})
    pair.cache.attend_weigh(gpu.Kv8Batch(0), **{**base, "weights": 0, "workspace": 0})
    # a workspace of a larger batch does
    for B in (1, 3, 40, 200):
        larger = gpu.Kv8Batch(B, max_pages=3000, total_pages=3000 * B)
        most = pair.cache.weigh_workspace_bytes(larger, 4)
        for b in (1, 2, 9, 40, 150):
            for pages in (1, 80, 3000):
                if b <= B:
                    less = gpu.Kv8Batch(b, max_pages=pages, total_pages=pages * b)
                    assert pair.cache.weigh_workspace_bytes(less, 4) <= most


def test_weigh_replayed_and_on_streams(gpu):
    """Steps of a graph add up as eager ones do; two streams with a workspace each."""
    import torch
    rng = np.random.default_rng(31)
    lengths = [4000, 17, 900]
    capacity = sum(-(-n // 16) for n in lengths)
    pair = Pair(gpu, 2, 128, 16, capacity)
    pair.fill(4)
    lists = lists_for(rng, lengths, 16, capacity)
    for l, n in zip(lists, lengths):
        if n % 16:
            pair.set_counts(l[-1], n % 16)
    batch = Batch(gpu, lists)
    inputs = [rows(rng, "bf16", 3, 8, 128) for _ in range(3)]
    q, out = torch.empty_like(inputs[0]), torch.empty_like(inputs[0])
    size = pair.cache.weigh_workspace_bytes(batch.batch, 8)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    weights = torch.zeros(capacity, 2, 16, device="cuda")
    want, outs = [], []
    for x in inputs:
        q.copy_(x)
        weigh(pair, batch, "bf16", q, out, weights)
        want.append(weights.clone())
        outs.append(out.clone())
    weights.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        weigh(pair, batch, "bf16", q, out, weights, ws=ws,
              stream=torch.cuda.current_stream().cuda_stream)
    for x, w, o in zip(inputs, want, outs):
        q.copy_(x)
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(weights, w) and torch.equal(out, o)
    streams = [torch.cuda.Stream() for _ in inputs]
    spaces = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in inputs]
    got = [(torch.empty_like(q), torch.zeros_like(weights)) for _ in inputs]
    torch.cuda.synchronize()
    for x, (o, w), space, s in zip(inputs, got, spaces, streams):
        weigh(pair, batch, "bf16", x, o, w, ws=space, stream=s.cuda_stream)
    torch.cuda.synchronize()
    for i, (o, w) in enumerate(got):
        assert torch.equal(o, outs[i])
        add, may = model_weights(pair, lists, "bf16", inputs[i])
        check_weights(torch.zeros_like(w), w, add, may)


@pytest.mark.parametrize("fmt", [kv8.E4M3, kv8.INT8])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv,dim,page", [(8, 2, 128, 16), (70, 1, 64, 48), (4, 2, 256, 64)])
def test_weigh_beside_malformed_offsets(gpu, heads, kv, dim, page, kind, fmt):
    """page_offsets that fall: the request they fall in is reported and has no token, all
    others get their outputs and add their weights, though their lists overlap.  The logits
    of one behind a fall are formed from the codes in 64 bits and rounded once, which
    model_weights' bound holds."""
    import torch
    rng = np.random.default_rng(dim)
    pair = Pair(gpu, kv, dim, page, 126, fmt)
    pair.fill(dim + fmt)
    for at, count in ((3, 5), (40, 0), (70, 1), (90, page - 1)):
        pair.set_counts(at, count)
    ids = rng.permutation(126)[:120].tolist()
    ids[65] = 500  # (a page outside the cache)
    for offsets in ([0, 100, 60, 120], [60, 120, 0, 50, 40, 120], [0, 500, 30, 80], [3, 3, 1, 120],
                    [0] + [7 * i for i in range(1, 9)] + [119, 63, 70, 80, 120, 120]):
        lists = [ids[a:b] if 0 <= a <= b <= 120 else [] for a, b in zip(offsets, offsets[1:])]
        lists = [[p for p in l if p != 500] for l in lists]
        batch = Batch(gpu, [ids] + [[]] * (len(lists) - 1))
        batch.keep["page_offsets"].copy_(device(offsets))
        q = rows(rng, kind, len(lists), heads, dim)
        add, may = model_weights(pair, lists, kind, q)
        before = sums(pair, rng)
        weights, out = before.clone(), torch.full_like(q, 9.0)
        fail = torch.zeros(1, dtype=torch.int64, device="cuda")
        weigh(pair, batch, kind, q, out, weights, fail=fail)
        assert int(fail) & 0xffffffff in (2, 3), offsets
        check_attention(pair, Batch(gpu, lists), kind, q, out)
        check_weights(before, weights, add, may)


def test_weigh_many_requests_beside_a_malformed_one(gpu):
    """More requests than a workgroup has threads, an entry far before the last too large
    and one near it too small."""
    import torch
    rng = np.random.default_rng(77)
    pair = Pair(gpu, 1, 64, 16, 700)
    pair.fill(1)
    ids = rng.permutation(700)[:600].tolist()
    for wrong in ({5: 300}, {299: 0}, {2: 9000, 290: 100}):
        offsets = [2 * i for i in range(301)]
        for at, x in wrong.items():
            offsets[at] = x
        lists = [ids[a:b] if 0 <= a <= b <= 600 else [] for a, b in zip(offsets, offsets[1:])]
        batch = Batch(gpu, [ids] + [[]] * 299)
        batch.keep["page_offsets"].copy_(device(offsets))
        q = rows(rng, "bf16", 300, 4, 64)
        before = sums(pair, rng)
        weights, out = before.clone(), torch.full_like(q, 9.0)
        fail = torch.zeros(1, dtype=torch.int64, device="cuda")
        weigh(pair, batch, "bf16", q, out, weights, fail=fail)
        assert int(fail) & 0xffffffff == 2, wrong
        check_attention(pair, Batch(gpu, lists), "bf16", q, out)
        check_weights(before, weights, *model_weights(pair, lists, "bf16", q))
