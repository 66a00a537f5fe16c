"""Attention over the 8-bit cache where logits are so large that float32 holds
no fraction of them: the largest takes all the weight, and nothing overflows."""
from __future__ import annotations

import numpy as np
import pytest

import _kv8 as kv8
from test_gpu_kv8 import Batch, Pair, as64, attend, check_attention, half_step, rows
from test_gpu_kv8_scales import FORMS

pytestmark = pytest.mark.gpu


def check_winners(pair, batch, kind, q, out, causal):
    """Rows whose largest logit leads by more than its error and 60: the value of
    that token, up to the roundings of one weight (_kv8.allowed) and of the
    output.  Returns how many rows there were."""
    m, G = pair.model, q.shape[1] // pair.model.heads
    q64, got, checked, at = as64(q), as64(out), 0, 0
    for r, pages in enumerate(batch.lists):
        n = batch.new[r] if causal else 1
        tokens = batch.past[r] + n if causal else None
        keys, values, _ = m.rows(np.asarray(pages, int), tokens)
        sees = np.repeat(batch.past[r] + 1 + np.arange(n), G) if causal else np.full(G, keys.shape[1])
        for h in range(m.heads):
            x = q64[at:at + n, h * G:(h + 1) * G].reshape(n * G, m.dim) / np.sqrt(m.dim)
            s = x @ keys[h].T
            error = 2 * ((m.dim + 8) * 2.0 ** -24 + 2.0 ** -21) * (np.abs(x) @ np.abs(keys[h]).T).max(1)
            s = np.where(np.arange(s.shape[1]) < sees[:, None], s, -np.inf)
            order = np.sort(s, 1)
            clear = order[:, -1] - order[:, -2] > error + 60 if s.shape[1] > 1 else np.ones(n * G, bool)
            want = values[h][s.argmax(1)][clear]
            have = got[at:at + n, h * G:(h + 1) * G].reshape(n * G, m.dim)[clear]
            weight = 2.0 ** -11 if kind == "bf16" else 2.0 ** -21
            slack = (half_step(kind) + weight + 2.0 ** -19) * np.abs(want)
            # (60 in the exponent: e^-60 of the others' values)
            floor = (2.0 ** -24 if kind == "f16" else 2.0 ** -126) + 2.0 ** -80 * np.abs(values[h]).max()
            assert (np.abs(have - want) <= slack + floor).all(), (r, h)
            checked += int(clear.sum())
        at += n
    return checked


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("fmt", [kv8.E4M3, kv8.INT8])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("power", [16, 20, 24, 30, 60])
def test_large_logits(gpu, power, kind, fmt, form):
    import torch
    rng = np.random.default_rng(power)
    page, heads, capacity, dim = 16, 4, 140, 64
    pair = Pair(gpu, 2, dim, page, capacity, fmt)
    pair.fill(10)
    m = pair.model
    m.scales[0] = (m.scales[0] * np.float32(2.0 ** power)).astype(np.float32)
    m.scales[1] = (m.scales[1] * np.exp2(rng.integers(-10, 11, m.scales[1].shape))).astype(np.float32)
    pair.key_scales.copy_(torch.from_numpy(m.scales[0]))
    pair.value_scales.copy_(torch.from_numpy(m.scales[1]))
    lists = [list(range(capacity)), [3, 1, 9, 120], [7], list(range(60, 20, -1))]
    new = None if FORMS[form] is None else [min(FORMS[form], page * len(l)) for l in lists]
    past = None if new is None else [page * len(l) - n for l, n in zip(lists, new)]
    batch = Batch(gpu, lists, past, new)
    q = rows(rng, kind, len(lists) if new is None else sum(new), heads, dim)
    if kind != "f16":  # (there is room for ordinary rows beside the others)
        q[:, 1] *= 2.0 ** -power
        q[:, 3] *= -2.0 ** 10
    for workspace in (True, False):
        out = torch.full_like(q, 9.0)
        attend(pair, batch, kind, q, out, causal=new is not None, workspace=workspace)
        assert bool(out.isfinite().all())
        check_attention(pair, batch, kind, q, out, causal=new is not None)
        assert check_winners(pair, batch, kind, q, out, new is not None) > 0 or power < 20
