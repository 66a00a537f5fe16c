"""Attention over the 8-bit cache where value scales are extreme: values that are
all zero, whose page scale is the least there is, 2^-126, values as small and as
large as float32 has, and both in one list."""
from __future__ import annotations

import numpy as np
import pytest

import _kv8 as kv8
from test_gpu_kv8 import (TYPES, Batch, Pair, append, attend, check_attention, inv_freq, rows)

pytestmark = pytest.mark.gpu


def set_values(pair, pages, codes=None, scale=None):
    """Pages' value codes (0 where not given: zeros) and value scale."""
    import torch
    m = pair.model
    pages = np.asarray(pages, int)
    if codes is None:
        m.codes[1][pages] = 0.0
        pair.values[torch.from_numpy(pages).cuda()] = 0
    if scale is not None:
        m.scales[1][pages] = np.asarray(scale, np.float32).reshape(-1, 1)
        pair.value_scales.copy_(torch.from_numpy(m.scales[1]))


# The calls that attend: one token a request, several with few rows a key head
# (one form of the kernel each), several with many.
FORMS = {"one": None, "few": 5, "many": 90}


def check_form(pair, form, kind, lists, rng, heads, spread=1.0):
    """Every list attended in the form, with its list whole and in pieces."""
    import torch
    page = pair.model.page
    if FORMS[form] is None:
        batch = Batch(pair.gpu, lists)
        count = len(lists)
    else:
        new = [min(FORMS[form], page * len(l)) for l in lists]
        past = [page * len(l) - n for l, n in zip(lists, new)]
        batch = Batch(pair.gpu, lists, past, new)
        count = sum(new)
    q = rows(rng, kind, count, heads, pair.model.dim) * spread
    for workspace in (True, False):
        out = torch.full_like(q, 9.0)
        attend(pair, batch, kind, q, out, causal=form != "one", workspace=workspace)
        check_attention(pair, batch, kind, q, out, causal=form != "one")
    return out


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("fmt", [kv8.E4M3, kv8.INT8])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim,page", [(64, 16), (80, 48), (128, 64), (256, 16)])
def test_zero_values(gpu, dim, page, kind, fmt, form):
    """Values that are zero throughout a page: alone, before, between and behind
    others, over a wave's first group of 64 tokens and over whole pieces."""
    rng = np.random.default_rng(dim + page)
    per_group = max(64 // page, 1)
    zero = 8 * per_group  # pages of zero values
    capacity = zero + 24 * per_group
    pair = Pair(gpu, 2, dim, page, capacity, fmt)
    pair.fill(dim)
    set_values(pair, range(zero), scale=np.full(zero, 2.0 ** -126))
    z, v = list(range(zero)), list(range(zero, capacity))
    g = per_group
    lists = [z[:1], z, z[:1] + v[:2], z[:g] + v[:5 * g], v[:g] + z[:g] + v[g:6 * g], v[:5 * g] + z[:2],
             [p for pair_ in zip(z, v) for p in pair_], (z + v) * 3, (v + z) * 2]
    out = check_form(pair, form, kind, lists, rng, 4)
    if form == "one":  # exactly zero, not only within the roundings
        assert not bool(out[:2].any())
    # scales of zero (cleared memory): the same
    pair.value_scales[:zero] = 0.0
    check_form(pair, form, kind, lists, rng, 4)


@pytest.mark.parametrize("fmt", [kv8.E4M3, kv8.INT8])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_zero_values_through_append_and_sparse_step(gpu, kind, fmt):
    """A head that writes zeros, and a request that starts with zero rows: the
    cache that append leaves, attended in every form and by the sparse step."""
    import torch
    rng = np.random.default_rng(5)
    heads, kv, dim, page = 8, 2, 64, 16
    n = [300, 20]
    need = [-(-t // page) for t in n]
    pair = Pair(gpu, kv, dim, page, sum(need), fmt)
    pair.cache.set_rotation(dim, inv_freq(dim))
    lists = [list(range(need[0])), list(range(need[0], sum(need)))]
    key, value = (rows(rng, kind, sum(n), kv, dim) for _ in range(2))
    value[:, 1] = 0  # the second head's values
    value[:100] = 0
    key[:80] = 0
    value[n[0]:] = 0  # all of the second request's
    append(pair, Batch(gpu, lists, [0, 0], n), kind, None, key, value, None)
    stored = pair.stored()
    pair.model.codes = [np.nan_to_num(x) for x in stored]
    pair.model.scales = [pair.key_scales.cpu().numpy(), pair.value_scales.cpu().numpy()]
    pair.model.counts = pair.counts.cpu().numpy()
    assert float(pair.value_scales[0, 0]) == 2.0 ** -126
    q = rows(rng, kind, 2, heads, dim)
    out = torch.full_like(q, 9.0)
    batch = Batch(gpu, lists)
    attend(pair, batch, kind, q, out)
    check_attention(pair, batch, kind, q, out)
    assert not bool(out[0, heads // kv:].any()) and not bool(out[1].any()) and bool(out[0].any())
    for new in ([3, 2], [120, 20]):
        past = [t - m for t, m in zip(n, new)]
        prompt = Batch(gpu, lists, past, new)
        x = rows(rng, kind, sum(new), heads, dim)
        y = torch.full_like(x, 9.0)
        attend(pair, prompt, kind, x, y, causal=True)
        check_attention(pair, prompt, kind, x, y, causal=True)
    with gpu.Kv8SparseStep(pair.cache, heads, 6, 2, sum(need)) as step:
        selected = torch.full((2, 6), -1, dtype=torch.int32, device="cuda")
        counts = torch.zeros(2, dtype=torch.int32, device="cuda")
        out.fill_(9.0)
        step.run(2, sum(need), max(need), TYPES[kind], q.data_ptr(), q.stride(0),
                 batch.keep["page_offsets"].data_ptr(), batch.keep["page_ids"].data_ptr(),
                 out.data_ptr(), out.stride(0), selected=selected.data_ptr(),
                 selected_counts=counts.data_ptr())
        step.status()
        kept = Batch(gpu, [selected[r, :int(counts[r])].tolist() for r in range(2)])
        check_attention(pair, kept, kind, q, out)
        assert not bool(out[0, heads // kv:].any()) and not bool(out[1].any())


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("fmt", [kv8.E4M3, kv8.INT8])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("spread", [1.0, 40.0])
def test_value_scales_far_apart(gpu, spread, kind, fmt, form):
    """Value scales from 2^-126 to 2^100 in one list and in lists of their own,
    with logits that differ by little and by more than a hundred."""
    rng = np.random.default_rng(6)
    page, heads, capacity = 16, 4, 48
    pair = Pair(gpu, 2, 64, page, capacity, fmt)
    pair.fill(8)
    powers = rng.permutation(np.linspace(-126, 100, capacity).round())
    set_values(pair, range(capacity), codes=True, scale=np.exp2(powers))
    order = np.argsort(powers).tolist()
    lists = [list(range(capacity)), order, order[::-1], order[:5], order[:20], order[14:18], order[24:30],
             order[40:], order[:1], order[-1:], order[:8] + order[28:36], order[30:34] + order[:12]]
    check_form(pair, form, kind, lists, rng, heads, spread)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("fmt", [kv8.E4M3, kv8.INT8])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("power", [-126, -120, 117])
def test_smallest_and_largest_values(gpu, power, kind, fmt, form):
    """Every value scale next to the ends of float32: numbers that float32 and
    bf16 hold come out, and the sum before its division does not overflow."""
    rng = np.random.default_rng(7)
    page, capacity = 16, 130
    pair = Pair(gpu, 2, 64, page, capacity, fmt)
    pair.fill(9)
    set_values(pair, range(capacity), codes=True, scale=np.exp2(power + rng.integers(0, 3, capacity)))
    lists = [list(range(capacity)), [4, 7, 9, 1, 2], [5], list(range(40)) * 4]
    check_form(pair, form, kind, lists, rng, 4, 0.1)
