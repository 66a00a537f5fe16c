"""Calls of the 8-bit cache that the documentation allows, at its edges: what a
workspace does for, requests beside malformed ones, how weights are held, caches beside each other."""
from __future__ import annotations

import numpy as np
import pytest

import _kv8 as kv8
from test_gpu_kv8 import (Batch, Pair, append, as64, attend, check_attention, device, inv_freq,
                          lists_for, model_append, rows)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,fmt", [("bf16", kv8.E4M3), ("f32", kv8.INT8)])
@pytest.mark.parametrize("heads,new", [(71, 1), (64, 1), (200, 1), (16, 4), (16, 5), (3, 40), (1, 90)])
def test_workspace_lets_long_lists_spread(gpu, heads, new, kind, fmt):
    """dsd_kv8_workspace_bytes of a batch is enough for it, however its rows come
    about: a list of 8000 tokens for one key head is spread, so the workspace is
    written, and the result is the one without."""
    import torch
    rng = np.random.default_rng(heads)
    pages = 500
    pair = Pair(gpu, 1, 64, 16, pages, fmt)
    pair.fill(12)
    batch = Batch(gpu, [rng.permutation(pages).tolist()], [16 * pages - new], [new])
    q = rows(rng, kind, new, heads, 64)
    out = torch.full_like(q, 9.0)
    space = attend(pair, batch, kind, q, out, causal=True)
    assert bool((space != 0xff).any())
    check_attention(pair, batch, kind, q, out, causal=True)
    attend(pair, batch, kind, q, out, causal=True, workspace=False)
    check_attention(pair, batch, kind, q, out, causal=True)
    # and the workspace of a larger batch does for this one
    larger = Batch(gpu, [list(range(pages))] * 3, [0] * 3, [new + 7] * 3)
    assert (pair.cache.workspace_bytes(larger.batch, heads)
            >= pair.cache.workspace_bytes(batch.batch, heads))


@pytest.mark.parametrize("requests", [4, 9, 64, 65, 150])
@pytest.mark.parametrize("wrong", [700000, -5, 0, 1, 2147483647, -2147483648])
def test_append_beside_malformed_offsets(gpu, wrong, requests):
    """One entry of token_offsets is wrong: the two requests that it bounds are
    reported and skipped, all others are appended."""
    import torch
    rng = np.random.default_rng(requests)
    page, at = 16, requests // 2
    new = [int(n) for n in rng.integers(3, 40, requests)]
    past = [int(p) for p in rng.integers(0, 16, requests)]
    need = [-(-(p + n) // page) for p, n in zip(past, new)]
    ends = np.cumsum(need)
    lists = [list(range(e - n, e)) for e, n in zip(ends, need)]
    pair = Pair(gpu, 2, 64, page, int(ends[-1]), rubbish=False)
    batch = Batch(gpu, lists, past, new)
    k, v = (rows(rng, "bf16", batch.tokens, 2, 64) for _ in range(2))
    first = Batch(gpu, lists, [0] * requests, past)
    k0, v0 = (rows(rng, "bf16", max(first.tokens, 1), 2, 64) for _ in range(2))
    append(pair, first, "bf16", None, k0, v0, None)
    model_append(pair, first, k0, v0, [])
    offsets = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    offsets[at] = wrong
    batch.keep["token_offsets"].copy_(device(offsets))
    fail = torch.zeros(1, dtype=torch.int64, device="cuda")
    append(pair, batch, "bf16", None, k, v, None, fail)
    assert int(fail) & 0xffffffff == 2
    for r in range(requests):
        rows_of = slice(int(sum(new[:r])), int(sum(new[:r + 1])))
        if r not in (at - 1, at):
            one = Batch(gpu, [lists[r]], [past[r]], [new[r]])
            model_append(pair, one, k[rows_of], v[rows_of], [])
    pair.check_pages([p for r, l in enumerate(lists) if r not in (at - 1, at) for p in l])
    # the two are as they were
    pair.check_pages([l[0] for r, l in enumerate(lists) if r in (at - 1, at) and past[r]])


@pytest.mark.parametrize("fmt", [kv8.E4M3, kv8.INT8])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv,dim,page,lengths", [
    (8, 2, 128, 16, [1, 65, 300, 2000]), (20, 1, 64, 64, [500, 129]), (6, 2, 256, 128, [130, 700]),
])
def test_weights_of_one_token(gpu, heads, kv, dim, page, lengths, kind, fmt):
    """Attention of one token with page scales 2^24 apart, by a bound of its own: its
    weights, times their page's scale, are held so that the row's largest is 2^15
    (_kv8.allowed has 2^11, which is the many-rows form's).  A half's numbers end in
    steps of 2^-24, so each is off by 2^-25 / 2^15 = 2^-40 of the largest."""
    import torch
    rng = np.random.default_rng(dim)
    capacity = sum(-(-n // page) for n in lengths)
    pair = Pair(gpu, kv, dim, page, capacity, fmt)
    pair.fill(13)
    m = pair.model
    m.scales[1] = (m.scales[1] * np.exp2(rng.integers(-18, 7, m.scales[1].shape))).astype(np.float32)
    pair.value_scales.copy_(torch.from_numpy(m.scales[1]))
    lists = lists_for(rng, lengths, page, capacity)
    for l, n in zip(lists, lengths):
        if n % page:
            pair.set_counts(l[-1], n % page)
    q = rows(rng, kind, len(lengths), heads, dim)
    batch = Batch(gpu, lists)
    G = heads // kv
    for workspace in (True, False):
        out = torch.full_like(q, 9.0)
        attend(pair, batch, kind, q, out, workspace=workspace)
        for r, pages in enumerate(lists):
            keys, values, most = m.rows(np.asarray(pages))
            tokens = keys.shape[1]
            for h in range(kv):
                x, have = as64(q[r, h * G:(h + 1) * G]), as64(out[r, h * G:(h + 1) * G])
                want, weighted, size, peak = kv8.attend(x, keys[h], values[h], dim ** -0.5, None, most[h])
                may = (kv8.allowed(want, weighted, size, peak, dim, tokens, kind)
                       - (tokens * (2.0 ** -36 - 2.0 ** -40) * peak)[:, None])
                assert (np.abs(have - want) <= may).all(), (r, h)


def test_caches_of_different_sizes_side_by_side(gpu):
    """Handles share kernels, whose LDS goes by each cache's own sizes: the larger
    ones run as before after smaller ones were made."""
    import torch
    rng = np.random.default_rng(44)
    shapes = [(1, 256, 64), (2, 144, 16), (1, 128, 48), (2, 80, 16), (1, 64, 256), (1, 16, 16)]
    pairs = [Pair(gpu, kv, dim, page, 6) for kv, dim, page in shapes]
    for pair in pairs:
        pair.cache.set_rotation(pair.model.dim // 32 * 32, inv_freq(pair.model.dim // 32 * 32))
    for pair in pairs + pairs[::-1]:
        m = pair.model
        lists, new = [[4, 2]], [m.page + 9]
        batch = Batch(gpu, lists, [0], new)
        x = rows(rng, "f32", new[0], 3 * m.heads, m.dim)
        k, v = x[:, :m.heads], x[:, m.heads:2 * m.heads]
        out = torch.empty_like(x)
        append(pair, batch, "f32", x, k, v, out)
        model_append(pair, batch, k, v, inv_freq(m.dim // 32 * 32))
        pair.check_pages([4, 2])
        for q, causal in ((x[:1].contiguous(), False), (x, True)):
            out = torch.full_like(q, 9.0)
            attend(pair, batch if causal else Batch(gpu, lists), "f32", q, out, causal=causal)
            check_attention(pair, batch if causal else Batch(gpu, lists), "f32", q, out, causal=causal)
