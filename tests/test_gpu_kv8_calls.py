"""Calls of the 8-bit cache that the documentation allows, at its edges: what a
workspace does for."""
from __future__ import annotations

import numpy as np
import pytest

import _kv8 as kv8
from test_gpu_kv8 import Batch, Pair, attend, check_attention, rows

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
