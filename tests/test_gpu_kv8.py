"""The 8-bit paged cache (dsd_kv8_*) against its definition in 64 bits: the
append's codes and scales are equal, attention is within the roundings that
_kv8.allowed derives."""
from __future__ import annotations

import numpy as np
import pytest

import _kv8 as kv8

pytestmark = pytest.mark.gpu

TYPES = {"f32": 0, "bf16": 1, "f16": 2}


def torch_type(kind):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[kind]


def as64(t):
    return t.double().cpu().numpy()


def inv_freq(rotary, base=10000.0):
    return base ** (-np.arange(rotary // 2) * 2.0 / max(rotary, 1))


class Pair:
    """A cache in the library and the model of it, over tensors the test owns.
    Their memory starts as rubbish (NaN codes, wild scales) where the
    definition says that it does not matter."""

    def __init__(self, gpu, heads, dim, page, capacity, fmt=0, rubbish=True, summaries=True):
        import torch
        self.gpu, self.fmt = gpu, fmt
        self.model = kv8.Cache(heads, dim, page, capacity, fmt)
        fill = 0xff if rubbish else 0
        self.keys = torch.full((capacity, heads, page, dim), fill, dtype=torch.uint8, device="cuda")
        self.values = torch.full((capacity, heads, page // 16, dim, 16), fill, dtype=torch.uint8,
                                 device="cuda")
        wild = float("nan") if rubbish else 0.0
        self.key_scales = torch.full((capacity, heads), wild, device="cuda")
        self.value_scales = torch.full((capacity, heads), wild, device="cuda")
        self.summaries = torch.zeros(capacity, heads * dim, device="cuda") if summaries else None
        self.counts = torch.zeros(capacity, dtype=torch.int32, device="cuda")
        arrays = {"keys": self.keys, "values": self.values, "key_scales": self.key_scales,
                  "value_scales": self.value_scales, "token_counts": self.counts}
        if summaries:
            arrays["summaries"] = self.summaries
        self.cache = gpu.Kv8Cache(heads, dim, page, capacity, fmt,
                                  arrays={n: t.data_ptr() for n, t in arrays.items()})

    def fill(self, seed):
        """Full pages of random codes and scales, without an append."""
        import torch
        m, rng = self.model, np.random.default_rng(seed)
        for side, codes, scales in ((0, self.keys, self.key_scales), (1, self.values, self.value_scales)):
            raw = rng.integers(0, 256, m.codes[side].shape, dtype=np.uint8)
            if self.fmt == kv8.E4M3:
                raw[raw & 127 == 127] = 0x31
            else:
                raw[raw == 128] = 127
            m.codes[side] = kv8.numbers(self.fmt, raw)
            m.scales[side] = (rng.uniform(0.2, 3.0, m.scales[side].shape) / kv8.LARGEST[self.fmt]
                              ).astype(np.float32)
            stored = raw
            if side == 1:
                c, h, p, d = raw.shape
                stored = raw.reshape(c, h, p // 16, 16, d).swapaxes(-1, -2)
            codes.copy_(torch.from_numpy(np.ascontiguousarray(stored)))
            scales.copy_(torch.from_numpy(m.scales[side]))
        m.counts[:] = m.page
        self.counts.fill_(m.page)

    def set_counts(self, page, count):
        """Only `count` tokens of a page; what lies behind them is rubbish."""
        self.model.counts[page] = count
        self.counts[page] = count
        self.keys[page, :, count:] = 0xff
        v = self.values[page]  # [heads][groups][dim][16]
        for t in range(count, self.model.page):
            v[:, t // 16, :, t % 16] = 0xff

    def stored(self):
        m = self.model
        k = kv8.numbers(self.fmt, self.keys.cpu().numpy())
        v = self.values.cpu().numpy()
        v = kv8.numbers(self.fmt, np.ascontiguousarray(v.swapaxes(-1, -2)).reshape(k.shape))
        return k, v

    def check_pages(self, pages):
        m = self.model
        k, v = self.stored()
        for page in pages:
            n = m.counts[page]
            assert int(self.counts[page]) == n
            for side, got, scales in ((0, k, self.key_scales), (1, v, self.value_scales)):
                assert np.array_equal(scales[page].cpu().numpy(), m.scales[side][page]), (page, side)
                assert np.array_equal(got[page][:, :n], m.codes[side][page][:, :n],
                                      equal_nan=True), (page, side)
            if self.summaries is not None:
                with np.errstate(over="ignore"):  # (a mean beyond float32 is infinite there)
                    want = m.summaries[page].astype(np.float32).astype(np.float64)
                got = as64(self.summaries[page])
                ends = ~np.isfinite(want)
                assert np.array_equal(got[ends], want[ends], equal_nan=True)
                got, want = np.where(ends, 0.0, got), np.where(ends, 0.0, want)
                # float32 sums of at most 256 codes (exact up to 2^24 of their
                # last place), one rounding
                bound = 2.0 ** -23 * np.nan_to_num(
                    np.abs(m.codes[0][page][:, :n]).sum(1) * m.scales[0][page][:, None] / n).reshape(-1)
                assert (np.abs(got - want) <= bound + 2.0 ** -149).all()


def device(a, dtype=np.int32):
    import torch
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, dtype))).cuda()


class Batch:
    """A Kv8Batch from host lists; keeps its tensors."""

    def __init__(self, gpu, lists, past=None, new=None, positions=None, strided=0, max_pages=None):
        import torch
        B = len(lists)
        self.lists, self.past, self.new = lists, past, new
        flat = [p for l in lists for p in l]
        self.keep = {}
        args = {}
        if strided:
            ids = np.full((B, strided), -7, np.int32)
            for r, l in enumerate(lists):
                ids[r, :len(l)] = l
            self.keep["page_ids"] = device(ids)
            self.keep["page_counts"] = device([len(l) for l in lists])
            args["list_stride"], total = strided, B * strided
        else:
            self.keep["page_ids"] = device(flat if flat else [0])
            self.keep["page_offsets"] = device(np.concatenate([[0], np.cumsum([len(l) for l in lists])]))
            total = len(flat)
        tokens, most = B, 1
        if new is not None:
            self.keep["token_offsets"] = device(np.concatenate([[0], np.cumsum(new)]))
            self.keep["past_tokens"] = device(past)
            tokens, most = int(sum(new)), int(max(list(new) + [1]))
        if positions is not None:
            self.keep["positions"] = device(positions)
        self.tokens = tokens
        longest = max([len(l) for l in lists] + [0])
        self.batch = gpu.Kv8Batch(B, tokens=tokens, max_tokens=most,
                                  max_pages=longest if max_pages is None else max_pages,
                                  total_pages=total,
                                  **args, **{n: t.data_ptr() for n, t in self.keep.items()})


def rows(rng, kind, tokens, heads, dim, spread=1.0):
    """Rows [tokens][heads][dim] of a type, whose tokens differ in size."""
    import torch
    x = rng.standard_normal((tokens, heads, dim)) * np.exp2(rng.uniform(-spread, spread, (tokens, 1, 1)))
    return torch.from_numpy(x).to(torch_type(kind)).cuda()


def append(pair, batch, kind, q, k, v, out, fail=None, stream=0):
    pair.cache.append(batch.batch, TYPES[kind], 0 if q is None else q.shape[1],
                      0 if q is None else q.data_ptr(), 0 if q is None else q.stride(0),
                      k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0),
                      0 if q is None else out.data_ptr(), 0 if q is None else out.stride(0),
                      fail=0 if fail is None else fail.data_ptr(), stream=stream)


def half_step(kind):
    return {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[kind]


def close_to(got, want, kind):
    """One rounding of the type; 2^-24 more for the way there through float32."""
    got = as64(got)
    slack = np.abs(want) * half_step(kind) * (1 + 2.0 ** -10) + np.abs(want) * 2.0 ** -24
    floor = 2.0 ** -25 * 1.001 if kind == "f16" else 2.0 ** -149
    return (np.abs(got - want) <= slack + floor).all()


def model_append(pair, batch, k, v, freq, positions=None, interleaved=False, magnitude=1.0):
    at = 0
    for r, n in enumerate(batch.new):
        where = np.arange(batch.past[r], batch.past[r] + n)
        if positions is not None:
            where = np.asarray(positions[at:at + n])
        pair.model.append(batch.lists[r], batch.past[r],
                          kv8.rotate(as64(k[at:at + n]), where, freq, interleaved, magnitude),
                          as64(v[at:at + n]))
        at += n


APPEND = [
    # heads, kv heads, dim, page, rotary, interleaved, past, new
    (8, 2, 128, 16, 128, False, [0], [1]),
    (8, 2, 128, 16, 128, False, [0, 15, 16, 17, 5], [1, 1, 1, 1, 1]),
    (8, 2, 128, 16, 128, False, [0, 3, 16, 31], [17, 16, 1, 0]),
    (4, 4, 64, 32, 64, True, [0, 20, 31, 33], [70, 1, 2, 100]),
    (6, 3, 80, 48, 32, False, [0, 1, 40], [1, 130, 9]),
    (5, 1, 96, 64, 96, False, [63, 0], [2, 64]),
    (2, 2, 256, 128, 128, True, [100, 0], [60, 300]),
    (7, 7, 16, 16, 16, False, [2, 0], [40, 5]),
    (3, 1, 192, 256, 0, False, [250, 3], [20, 500]),
    (40, 8, 128, 16, 64, True, list(range(70)), [1 + i % 3 for i in range(70)]),
]


@pytest.mark.parametrize("fmt", [kv8.E4M3, kv8.INT8])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", APPEND, ids=lambda c: "%dx%dx%d_p%d_r%d" % (c[0], c[1], c[2], c[3], c[4]))
def test_append(gpu, case, kind, fmt):
    import torch
    heads, kv, dim, page, rotary, interleaved, past, new = case
    rng = np.random.default_rng(dim * page + len(past))
    lists, at = [], 0
    order = rng.permutation(sum((p + n) // page + 1 for p, n in zip(past, new)))
    for p, n in zip(past, new):
        need = (p + n) // page + 1
        lists.append(order[at:at + need].tolist())
        at += need
    pair = Pair(gpu, kv, dim, page, at, fmt)
    freq = inv_freq(rotary)
    pair.cache.set_rotation(rotary, freq, interleaved)
    # what the requests have already: one append of its own, smaller numbers
    begin = Batch(gpu, lists, [0] * len(past), past)
    k, v = (rows(rng, kind, begin.tokens, kv, dim) * 0.25 for _ in range(2))
    append(pair, begin, kind, None, k, v, None)
    model_append(pair, begin, k, v, freq, interleaved=interleaved)
    used = [p for l, n in zip(lists, past) for p in l[:-(-n // page)]]
    pair.check_pages(used)
    # then the case: q, k and v side by side in one projection
    batch = Batch(gpu, lists, past, new)
    qkv = rows(rng, kind, batch.tokens, heads + 2 * kv, dim, spread=2.0)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    out = torch.full((batch.tokens, heads, dim), 7.0, device="cuda", dtype=qkv.dtype)
    fail = torch.zeros(1, dtype=torch.int64, device="cuda")
    before = pair.stored()
    append(pair, batch, kind, q, k, v, out, fail)
    torch.cuda.synchronize()
    assert int(fail) == 0
    model_append(pair, batch, k, v, freq, interleaved=interleaved)
    used = sorted({p for l, n, m in zip(lists, past, new) for p in l[:-(-(n + m) // page)]})
    pair.check_pages(used)
    where = np.concatenate([np.arange(p, p + n) for p, n in zip(past, new)])
    assert close_to(out, kv8.rotate(as64(q), where, freq, interleaved), kind)
    # codes behind the last token stay
    for was, now in zip(before, pair.stored()):
        for page_id in range(pair.model.capacity):
            n = pair.model.counts[page_id]
            assert np.array_equal(was[page_id][:, n:], now[page_id][:, n:], equal_nan=True)
    # the same call again changes nothing
    state = [t.clone() for t in (pair.keys, pair.values, pair.key_scales, pair.value_scales, pair.counts)]
    append(pair, batch, kind, q, k, v, out)
    for was, now in zip(state, (pair.keys, pair.values, pair.key_scales, pair.value_scales, pair.counts)):
        assert torch.equal(was.view(torch.uint8), now.view(torch.uint8))


def test_append_far_positions_and_magnitude(gpu):
    """Positions of millions: angles from 32-bit products would be off by 0.1."""
    import torch
    rng = np.random.default_rng(3)
    pair = Pair(gpu, 2, 128, 16, 3)
    freq = inv_freq(128, 500000.0)
    pair.cache.set_rotation(128, freq, magnitude=1.25)
    positions = [3000001, 0, 2147483647, 16777217, 5] * 4
    batch = Batch(gpu, [[2, 0]], [3], [20], positions=positions)
    first = Batch(gpu, [[2, 0]], [0], [3], positions=[9, 9, 9])
    q, k, v = (rows(rng, "f32", 20, h, 128) for h in (4, 2, 2))
    append(pair, first, "f32", None, k, v, None)
    model_append(pair, first, k, v, freq, [9, 9, 9], magnitude=1.25)
    out = torch.empty_like(q)
    append(pair, batch, "f32", q, k, v, out)
    model_append(pair, batch, k, v, freq, positions, magnitude=1.25)
    pair.check_pages([2, 0])
    want = kv8.rotate(as64(q), positions, freq, magnitude=1.25)
    # a 64-bit angle of 2^31 radians is known to 2^-21, the model's own to 2^-22
    assert np.abs(as64(out) - want).max() <= 2.0 ** -20 * np.abs(want).max()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_append_unaligned_rows_and_in_place(gpu, kind):
    import torch
    rng = np.random.default_rng(8)
    heads, kv, dim = 4, 2, 64
    pair = Pair(gpu, kv, dim, 32, 4)
    freq = inv_freq(64)
    pair.cache.set_rotation(64, freq)
    batch = Batch(gpu, [[1, 3], [0]], [0, 7], [40, 9])
    append(pair, Batch(gpu, [[1, 3], [0]], [0, 0], [0, 7]), kind, None,
           *(rows(np.random.default_rng(1), kind, 7, kv, dim) for _ in range(2)), None)
    model_append(pair, Batch(gpu, [[1, 3], [0]], [0, 0], [0, 7]),
                 *(rows(np.random.default_rng(1), kind, 7, kv, dim) for _ in range(2)), freq)
    width = (heads + 2 * kv) * dim + 5
    flat = rows(rng, kind, 1, 1, 49 * width + 3).view(-1)[3:]  # an odd start and an odd stride
    view = flat.view(49, width)
    q = view[:, :heads * dim].unflatten(1, (heads, dim))
    k = view[:, heads * dim:(heads + kv) * dim].unflatten(1, (kv, dim))
    v = view[:, (heads + kv) * dim:(heads + 2 * kv) * dim].unflatten(1, (kv, dim))
    was = view.clone()
    want = kv8.rotate(as64(q), np.concatenate([np.arange(40), 7 + np.arange(9)]), freq)
    k64, v64 = k.clone(), v.clone()
    append(pair, batch, kind, q, k, v, q)
    model_append(pair, batch, k64, v64, freq)
    pair.check_pages([1, 3, 0])
    assert close_to(q, want, kind)
    assert torch.equal(view[:, heads * dim:], was[:, heads * dim:])  # nothing else written


@pytest.mark.parametrize("fmt", [kv8.E4M3, kv8.INT8])
def test_append_values_at_borders(gpu, fmt):
    """Numbers half way between codes, zero pages, the largest and smallest
    floats, infinities and NaN."""
    import torch
    inf, nan = float("inf"), float("nan")
    dim = 64
    lines = [np.zeros(dim), np.full(dim, 1e-45), np.full(dim, 3e38), np.linspace(-3.4e38, 3.4e38, dim),
             np.arange(dim) + 0.5, -(np.arange(dim) + 0.5) / 7, np.full(dim, 448.0), np.full(dim, 449.0),
             np.concatenate([[inf, -inf, nan], np.linspace(-2, 2, dim - 3)]), np.full(dim, nan),
             np.full(dim, inf), np.linspace(0, 381, dim).round() * 0.5,
             2.0 ** -np.arange(dim).astype(np.float64)]
    x = torch.tensor(np.array(lines), dtype=torch.float32, device="cuda")
    pair = Pair(gpu, 1, dim, 16, len(lines) + 1, fmt)
    # a page each
    batch = Batch(gpu, [[i] for i in range(len(lines))], [0] * len(lines), [1] * len(lines))
    k = x.view(-1, 1, dim)
    append(pair, batch, "f32", None, k, k.flip(0).contiguous(), None)
    model_append(pair, batch, k, k.flip(0), [])
    pair.check_pages(range(len(lines)))
    # and all in one page, a token at a time: the scale grows on the way
    for i in range(len(lines)):
        one = Batch(gpu, [[len(lines)]], [i], [1])
        append(pair, one, "f32", None, k[i:i + 1], k[i:i + 1], None)
        model_append(pair, one, k[i:i + 1], k[i:i + 1], [])
        pair.check_pages([len(lines)])


def test_append_without_summaries_and_own_memory(gpu):
    import torch
    rng = np.random.default_rng(4)
    k, v = (rows(rng, "bf16", 21, 2, 64) for _ in range(2))
    pair = Pair(gpu, 2, 64, 16, 2, summaries=False)
    batch = Batch(gpu, [[1, 0]], [0], [21])
    append(pair, batch, "bf16", None, k, v, None)
    model_append(pair, batch, k, v, [])
    pair.check_pages([0, 1])
    with gpu.Kv8Cache(2, 64, 16, 2) as own:
        arrays = own.device_arrays()
        assert all(arrays.values())
        own.append(batch.batch, TYPES["bf16"], 0, 0, 0, k.data_ptr(), k.stride(0), v.data_ptr(),
                   v.stride(0), 0, 0)
        q = rows(rng, "f32", 1, 4, 64)
        outs = [torch.empty_like(q) for _ in range(2)]
        lists = Batch(gpu, [[1, 0]])
        own.attend(lists.batch, 0, 4, q.data_ptr(), q.stride(0), outs[0].data_ptr(), 256)
        pair.cache.attend(lists.batch, 0, 4, q.data_ptr(), q.stride(0), outs[1].data_ptr(), 256)
        assert torch.equal(*outs) and bool(outs[0].abs().sum() > 0)
        own.reset()
        own.attend(lists.batch, 0, 4, q.data_ptr(), q.stride(0), outs[0].data_ptr(), 256)
        assert not bool(outs[0].any())


def test_append_skips_what_does_not_fit(gpu):
    """Malformed requests are reported and write nothing; the others go on."""
    import torch
    rng = np.random.default_rng(6)
    for what, lists, past, new, code in [
        ("page id", [[0], [9]], [0, 0], [3, 3], 3),
        ("negative id", [[0], [-1]], [0, 0], [3, 3], 3),
        ("short list", [[0], [1]], [0, 14], [3, 3], 2),
        ("negative past", [[0], [1]], [0, -1], [3, 3], 2),
    ]:
        pair = Pair(gpu, 2, 64, 16, 3)
        batch = Batch(gpu, lists, past, new)
        k, v = (rows(rng, "bf16", 6, 2, 64) for _ in range(2))
        fail = torch.zeros(1, dtype=torch.int64, device="cuda")
        append(pair, batch, "bf16", None, k, v, None, fail)
        assert int(fail) & 0xffffffff == code, what
        assert pair.counts.tolist() == [3, 0, 0], what
        assert bool((pair.keys[1:] == 0xff).all()) and bool((pair.values[1:] == 0xff).all()), what
    # offsets that leave the rows: more tokens than the call has
    pair = Pair(gpu, 2, 64, 16, 3)
    batch = Batch(gpu, [[0], [1]], [0, 0], [3, 3])
    for bad in ([0, 3, 700], [0, -5, 6], [0, 7, 6]):
        batch.keep["token_offsets"].copy_(device(bad))
        fail = torch.zeros(1, dtype=torch.int64, device="cuda")
        append(pair, batch, "bf16", None, k, v, None, fail)
        assert int(fail) & 0xffffffff == 2, bad
    assert int(pair.counts[1]) == 0


# ---- attention -------------------------------------------------------------------

def attend(pair, batch, kind, q, out, causal=False, scale=0.0, workspace=True, fail=None, stream=0):
    import torch
    size = pair.cache.workspace_bytes(batch.batch, q.shape[1]) if workspace else 0
    ws = torch.full((max(size, 1),), 0xff, dtype=torch.uint8, device="cuda")
    call = pair.cache.attend_prompt if causal else pair.cache.attend
    call(batch.batch, TYPES[kind], q.shape[1], q.data_ptr(), q.stride(0), out.data_ptr(),
         out.stride(0), scale, workspace=ws.data_ptr() if size else 0, workspace_bytes=size,
         fail=0 if fail is None else fail.data_ptr(), stream=stream)
    return ws


def check_attention(pair, batch, kind, q, out, causal=False, scale=0.0):
    m = pair.model
    heads = q.shape[1]
    G = heads // m.heads
    q64, got = as64(q), as64(out)
    scale = scale or 1.0 / np.sqrt(m.dim)
    at = 0
    for r, pages in enumerate(batch.lists):
        n = batch.new[r] if causal else 1
        tokens = batch.past[r] + n if causal else None
        keys, values, most = m.rows(np.asarray(pages, int), tokens)
        sees = np.repeat(batch.past[r] + 1 + np.arange(n), G) if causal else None
        for h in range(m.heads):
            rows_ = q64[at:at + n, h * G:(h + 1) * G].reshape(n * G, m.dim)
            want, weighted, size, peak = kv8.attend(rows_, keys[h], values[h], scale, sees, most[h])
            have = got[at:at + n, h * G:(h + 1) * G].reshape(n * G, m.dim)
            may = kv8.allowed(want, weighted, size, peak, m.dim, keys.shape[1], kind)
            bad = ~(np.abs(have - want) <= may)
            assert not bad.any(), (r, h, np.argwhere(bad)[:3], have[bad][:3], want[bad][:3], may[bad][:3])
        at += n


def lists_for(rng, lengths, page, capacity):
    """A list of distinct pages for each length, and the tokens of its last page."""
    order, at, lists = rng.permutation(capacity), 0, []
    for n in lengths:
        need = -(-n // page)
        lists.append(order[at:at + need].tolist())
        at += need
    assert at <= capacity
    return lists


ATTEND = [
    # heads, kv heads, dim, page, lengths
    (8, 2, 128, 16, [1, 0, 15, 16, 17, 63, 64, 65, 300]),
    (4, 4, 128, 16, [129, 1, 700]),
    (32, 2, 64, 32, [50, 257]),            # 16 query heads a key head
    (20, 1, 128, 64, [5, 1000]),           # 20: two tiles of rows
    (7, 1, 96, 48, [100, 47, 48, 49]),
    (3, 3, 80, 16, [77, 400]),
    (2, 2, 16, 16, [33]),
    (6, 2, 256, 128, [128, 130, 513]),
    (2, 1, 192, 256, [255, 600]),
    (8, 8, 128, 16, [9000, 20]),           # spread over workgroups
]


@pytest.mark.parametrize("fmt", [kv8.E4M3, kv8.INT8])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", ATTEND, ids=lambda c: "%dx%dx%d_p%d" % c[:4])
def test_attend(gpu, case, kind, fmt):
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
    batch = Batch(gpu, lists)
    out = torch.full_like(q, 9.0)
    attend(pair, batch, kind, q, out)
    check_attention(pair, batch, kind, q, out)
    # unspread, and from a strided list: the same within the roundings
    out2 = torch.full_like(q, 9.0)
    longest = max(len(l) for l in lists)
    attend(pair, Batch(gpu, lists, strided=longest + 3), kind, q, out2, workspace=False)
    check_attention(pair, batch, kind, q, out2)
    # a hint that is too short still reads whole lists
    out3 = torch.full_like(q, 9.0)
    attend(pair, Batch(gpu, lists, max_pages=3), kind, q, out3)
    check_attention(pair, batch, kind, q, out3)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_attend_any_list(gpu, kind):
    """Lists that a top-k leaves: pages out of order, half-full and empty ones
    in the middle, one twice."""
    import torch
    rng = np.random.default_rng(12)
    pair = Pair(gpu, 2, 128, 16, 40)
    pair.fill(2)
    for page, count in ((3, 5), (7, 0), (11, 1), (12, 15), (30, 0)):
        pair.set_counts(page, count)
        if count == 0:  # no append has set its scales
            pair.key_scales[page] = float("nan")
            pair.value_scales[page] = float("inf")
    lists = [[3, 9, 7, 11], [12, 12, 5], [7, 30], [30], [39, 3, 38, 7, 37, 12, 36, 11, 1, 2, 3, 3]]
    q = rows(rng, kind, len(lists), 8, 128)
    out = torch.empty_like(q)
    batch = Batch(gpu, lists)
    attend(pair, batch, kind, q, out)
    check_attention(pair, batch, kind, q, out)
    assert not bool(out[2].any()) and not bool(out[3].any())


def test_attend_scales_that_differ_widely(gpu):
    """Value scales 2^40 apart and logits of hundreds: no weight overflows or
    is lost."""
    import torch
    rng = np.random.default_rng(13)
    for fmt in (kv8.E4M3, kv8.INT8):
        pair = Pair(gpu, 1, 64, 16, 12, fmt)
        pair.fill(5)
        factor = np.exp2(rng.permutation(12) * 2.0 - 12).astype(np.float32)[:, None]
        pair.model.scales[1] = pair.model.scales[1] * factor
        pair.value_scales.copy_(torch.from_numpy(pair.model.scales[1]))
        for kind in ("f32", "f16"):
            q = rows(rng, kind, 3, 4, 64) * 20
            out = torch.empty_like(q)
            batch = Batch(gpu, [list(range(12)), [3], [5, 1, 2, 8]])
            attend(pair, batch, kind, q, out, scale=1.5)
            check_attention(pair, batch, kind, q, out, scale=1.5)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_attend_unaligned_rows_and_negative_scale(gpu, kind):
    """Rows that start on any element, at any stride; a negative scale."""
    import torch
    rng = np.random.default_rng(17)
    pair = Pair(gpu, 2, 64, 16, 16)
    pair.fill(11)
    for causal, past, new in ((False, None, None), (True, [30, 7, 0], [3, 40, 1])):
        tokens = 3 if not causal else sum(new)
        lists = [[0, 1, 2], [3, 4, 5, 6], [7]]
        batch = Batch(gpu, lists, past, new)
        for heads in (4, 18):
            width = heads * 64 + 7
            flat = rows(rng, kind, 1, 1, tokens * width + 1).view(-1)[1:].view(tokens, width)
            q = flat[:, 3:3 + heads * 64].unflatten(1, (heads, 64))
            wide = torch.full((tokens, width + 2), 9.0, device="cuda", dtype=q.dtype)
            out = wide[:, 1:1 + heads * 64].unflatten(1, (heads, 64))
            attend(pair, batch, kind, q, out, causal=causal, scale=-0.21)
            check_attention(pair, batch, kind, q, out, causal=causal, scale=-0.21)
            assert bool((wide[:, 0] == 9.0).all()) and bool((wide[:, 1 + heads * 64:] == 9.0).all())


@pytest.mark.parametrize("kind,fmt", [("bf16", kv8.E4M3), ("f32", kv8.INT8)])
@pytest.mark.parametrize("heads,kv,dim,page,past,new", [
    (8, 1, 128, 16, [9000], [40]),       # one block of rows, its list in pieces
    (8, 2, 128, 64, [5000, 40], [70, 130]),
    (4, 1, 64, 16, [12000], [33]),
    (8, 1, 256, 128, [6000], [20]),
])
def test_prompt_chunk_behind_a_long_context(gpu, heads, kv, dim, page, past, new, kind, fmt):
    import torch
    rng = np.random.default_rng(dim + past[0])
    lengths = [p + n for p, n in zip(past, new)]
    capacity = sum(-(-n // page) for n in lengths)
    pair = Pair(gpu, kv, dim, page, capacity, fmt)
    pair.fill(dim)
    lists = lists_for(rng, lengths, page, capacity)
    q = rows(rng, kind, sum(new), heads, dim)
    batch = Batch(gpu, lists, past, new)
    assert pair.cache.workspace_bytes(batch.batch, heads) > 0
    for workspace in (True, False):
        out = torch.full_like(q, 9.0)
        attend(pair, batch, kind, q, out, causal=True, workspace=workspace)
        check_attention(pair, batch, kind, q, out, causal=True)
    # a NaN value in the middle of a piece, seen by the last rows only
    if fmt == kv8.E4M3:
        token = past[0] + new[0] - 5
        page_id = lists[0][token // page]
        want = torch.full_like(q, 9.0)
        attend(pair, batch, kind, q, want, causal=True)
        pair.values[page_id, 0, token % page // 16, 3, token % 16] = 0x7f
        attend(pair, batch, kind, q, out, causal=True)
        G = heads // kv
        assert bool(out[new[0] - 5:new[0], :G, 3].isnan().all())
        assert torch.equal(out[:new[0] - 5], want[:new[0] - 5])


def test_attend_nonfinite(gpu):
    """Infinite and NaN queries give what the formula gives; other rows of the
    tile are untouched by them."""
    import torch
    rng = np.random.default_rng(14)
    for kind in ("f32", "bf16", "f16"):
        pair = Pair(gpu, 1, 64, 16, 8)
        pair.fill(7)
        clean = rows(rng, kind, 2, 4, 64)
        q = clean.clone()
        q[0, 1, 3] = float("nan")
        q[1, 2, 0] = float("inf")
        out, want = torch.empty_like(q), torch.empty_like(q)
        batch = Batch(gpu, [[0, 1, 2], [3, 4, 5, 6, 7]])
        attend(pair, batch, kind, q, out)
        attend(pair, batch, kind, clean, want)
        assert bool(out[0, 1].isnan().all()) and bool(out[1, 2].isnan().all())
        keep = torch.ones(2, 4, dtype=torch.bool)
        keep[0, 1] = keep[1, 2] = False
        assert torch.equal(out[keep], want[keep])
        # a NaN value code of a page: every row that weighs it
        pair.values[1, 0, 0, 5, 3] = 0x7f
        attend(pair, batch, kind, clean, out)
        assert bool(out[0, :, 5].isnan().all()) and not bool(out[0, :, 6].isnan().any())
        assert torch.equal(out[1], want[1])


PROMPT = [
    # heads, kv heads, dim, page, past, new
    (8, 2, 128, 16, [0], [1]),
    (8, 2, 128, 16, [0, 0, 0, 0], [1, 16, 17, 0]),
    (8, 2, 128, 16, [5, 100, 0, 31], [3, 4, 150, 33]),
    (4, 4, 64, 32, [0, 7], [200, 90]),
    (5, 1, 96, 48, [50, 0], [20, 61]),
    (2, 2, 256, 64, [0, 130], [70, 2]),
    (3, 3, 80, 16, [1], [129]),
    (32, 1, 128, 16, [40, 2000], [9, 3]),
    (12, 4, 128, 64, [0], [515]),
    (2, 1, 16, 16, [3, 0, 8], [0, 0, 1]),
]


@pytest.mark.parametrize("fmt", [kv8.E4M3, kv8.INT8])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", PROMPT, ids=lambda c: "%dx%dx%d_p%d_%s" % (c[:4] + (sum(c[5]),)))
def test_attend_prompt(gpu, case, kind, fmt):
    import torch
    heads, kv, dim, page, past, new = case
    rng = np.random.default_rng(heads * dim + page + sum(new))
    lengths = [p + n for p, n in zip(past, new)]
    capacity = sum(-(-n // page) for n in lengths) + 2
    pair = Pair(gpu, kv, dim, page, capacity, fmt)
    pair.fill(dim + fmt)
    lists = lists_for(rng, lengths, page, capacity)
    for l, n in zip(lists, lengths):
        if n % page:
            pair.set_counts(l[-1], n % page)
    pair.counts.fill_(-5)  # (not read)
    q = rows(rng, kind, max(sum(new), 1), heads, dim)
    batch = Batch(gpu, lists, past, new)
    spare = torch.full((q.shape[0] + 2, heads, dim), 9.0, device="cuda", dtype=q.dtype)
    for workspace in (True, False):
        out = spare[:q.shape[0]]
        out.fill_(9.0)
        attend(pair, batch, kind, q, out, causal=True, workspace=workspace)
        check_attention(pair, batch, kind, q, out, causal=True)
        assert bool((spare[sum(new):] == 9.0).all())  # rows of no request


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_prompt_rows_do_not_see_later_tokens(gpu, kind):
    """NaN keys and values of later tokens leave earlier rows as they were."""
    import torch
    rng = np.random.default_rng(15)
    pair = Pair(gpu, 1, 64, 16, 8)
    pair.fill(9)
    q = rows(rng, kind, 100, 2, 64)
    batch = Batch(gpu, [list(range(8))], [20], [100])
    want, out = torch.empty_like(q), torch.empty_like(q)
    attend(pair, batch, kind, q, want, causal=True)
    for token in (75, 119):
        k, v = pair.keys.clone(), pair.values.clone()
        pair.keys[token // 16, :, token % 16] = 0x7f
        attend(pair, batch, kind, q, out, causal=True)
        assert torch.equal(out[:token - 20], want[:token - 20])
        assert bool(out[token - 20:].isnan().all())
        pair.keys.copy_(k)
        pair.values[token // 16, :, 0, 7, token % 16] = 0xff
        attend(pair, batch, kind, q, out, causal=True)
        assert torch.equal(out[:token - 20], want[:token - 20])
        assert bool(out[token - 20:, :, 7].isnan().all())
        assert torch.equal(out[:, :, :7], want[:, :, :7])
        pair.values.copy_(v)


def test_attend_reports_bad_lists(gpu):
    import torch
    rng = np.random.default_rng(16)
    pair = Pair(gpu, 2, 64, 16, 6)
    pair.fill(3)
    q = rows(rng, "bf16", 2, 4, 64)
    for lists, code in (([[0, 99, 1], [2]], 3), ([[0, -2, 1], [2]], 3)):
        out = torch.full_like(q, 9.0)
        fail = torch.zeros(1, dtype=torch.int64, device="cuda")
        attend(pair, Batch(gpu, lists), "bf16", q, out, fail=fail)
        assert int(fail) & 0xffffffff == code
        good = Batch(gpu, [[0, 1], [2]])  # a page outside the cache holds no token
        check_attention(pair, good, "bf16", q, out)
    batch = Batch(gpu, [[0, 1], [2]])
    for offsets in ([0, 2, 50], [0, -1, 3], [2, 1, 3]):
        batch.keep["page_offsets"].copy_(device(offsets))
        out = torch.full_like(q, 9.0)
        fail = torch.zeros(1, dtype=torch.int64, device="cuda")
        attend(pair, batch, "bf16", q, out, fail=fail)
        assert int(fail) & 0xffffffff == 2, offsets
        assert not bool(out[1].any()) or offsets != [0, 2, 50]
    # a prompt whose list does not hold its tokens: skipped, rows as they were
    batch = Batch(gpu, [[0, 1], [2]], [30, 3], [4, 5])
    q = rows(rng, "bf16", 9, 4, 64)
    out = torch.full_like(q, 9.0)
    fail = torch.zeros(1, dtype=torch.int64, device="cuda")
    attend(pair, batch, "bf16", q, out, causal=True, fail=fail)
    assert int(fail) & 0xffffffff == 2
    assert bool((out[:4] == 9.0).all()) and not bool((out[4:] == 9.0).any())


def test_refusals(gpu):
    import torch
    pair = Pair(gpu, 2, 64, 16, 4)
    q = torch.zeros(4, 4, 64, device="cuda", dtype=torch.bfloat16)
    base = dict(dtype=1, num_q_heads=4, q=q.data_ptr(), q_stride=256, out=q.data_ptr(), out_stride=256)
    batch = Batch(gpu, [[0], [1]], [0, 0], [1, 1])
    for bad, what in [(dict(dtype=3), "type"), (dict(num_q_heads=3), "multiple"),
                      (dict(num_q_heads=0), "positive"), (dict(q=0), "non-null"),
                      (dict(q_stride=255), "stride"), (dict(out_stride=-256), "stride"),
                      (dict(q=q.data_ptr() + 1), "aligned"), (dict(scale=float("nan")), "scale"),
                      (dict(workspace=q.data_ptr() + 2, workspace_bytes=64), "16-byte")]:
        for call in (pair.cache.attend, pair.cache.attend_prompt):
            with pytest.raises(gpu.InvalidArgument, match=what):
                call(batch.batch, **{**base, **bad})
    for bad, what in [(dict(batch=-1), "non-negative"), (dict(batch=70000), "65535"),
                      (dict(page_offsets=0), "page_offsets"), (dict(page_ids=0), "page_ids"),
                      (dict(list_stride=4), "page_counts")]:
        good = dict(batch=2, tokens=2, max_tokens=1, max_pages=1, total_pages=2,
                    **{n: t.data_ptr() for n, t in batch.keep.items()})
        with pytest.raises(gpu.InvalidArgument, match=what):
            pair.cache.attend(gpu.Kv8Batch(**{**good, **bad}), **base)
    with pytest.raises(gpu.InvalidArgument, match="31 bits"):
        huge = dict(good, tokens=1 << 30, max_tokens=1 << 30)
        pair.cache.attend_prompt(gpu.Kv8Batch(**huge), **base)
    with pytest.raises(gpu.InvalidArgument, match="token_offsets"):
        good = dict(good, token_offsets=0)
        pair.cache.attend_prompt(gpu.Kv8Batch(**good), **base)
    for rotary in (8, 80, -16):
        with pytest.raises(gpu.InvalidArgument):
            pair.cache.set_rotation(rotary, np.ones(max(rotary // 2, 0)))
    with pytest.raises(gpu.InvalidArgument, match="finite"):
        pair.cache.set_rotation(16, [np.inf] * 8)
    with pytest.raises(gpu.InvalidArgument, match="pair"):
        pair.cache.set_rotation(16, [1.0])
    pair.cache.attend(gpu.Kv8Batch(0), 1, 4, 0, 256, 0, 256)  # nothing to do
    pair.cache.attend_prompt(gpu.Kv8Batch(2, token_offsets=batch.keep["token_offsets"].data_ptr(),
                                          past_tokens=batch.keep["past_tokens"].data_ptr(),
                                          page_offsets=batch.keep["page_offsets"].data_ptr()),
                             1, 4, 0, 256, 0, 256)
    torch.cuda.synchronize()


# ---- a run of them together --------------------------------------------------------

@pytest.mark.parametrize("kind,fmt", [("bf16", kv8.E4M3), ("f16", kv8.INT8), ("f32", kv8.E4M3)])
def test_serving_run(gpu, kind, fmt):
    """Prompts in, a chunk behind one of them, then tokens one at a time: every
    output against the model's cache."""
    import torch
    rng = np.random.default_rng(21)
    heads, kv, dim, page = 8, 2, 64, 16
    freq = inv_freq(dim)
    lists = [rng.permutation(30)[:0].tolist() for _ in range(3)]
    order = rng.permutation(30).tolist()
    lists = [order[0:10], order[10:20], order[20:30]]
    pair = Pair(gpu, kv, dim, page, 30, fmt)
    pair.cache.set_rotation(dim, freq)
    past = [0, 0, 0]
    for new in ([37, 1, 64], [0, 20, 3], [1, 1, 1], [1, 1, 1], [1, 0, 1], [2, 3, 1], [1, 1, 1]):
        batch = Batch(gpu, lists, past, new)
        qkv = rows(rng, kind, batch.tokens, heads + 2 * kv, dim)
        q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
        turned = torch.empty(batch.tokens, heads, dim, device="cuda", dtype=qkv.dtype)
        append(pair, batch, kind, q, k, v, turned)
        model_append(pair, batch, k, v, freq)
        out = torch.empty_like(turned)
        attend(pair, batch, kind, turned, out, causal=True)
        check_attention(pair, batch, kind, turned, out, causal=True)
        if all(n == 1 for n in new):  # the decode form gives the same
            mine = [l[:-(-(p + 1) // page)] for l, p in zip(lists, past)]
            out = torch.empty_like(turned)
            attend(pair, Batch(gpu, mine), kind, turned, out)
            check_attention(pair, Batch(gpu, mine), kind, turned, out)
        past = [p + n for p, n in zip(past, new)]


def test_streams_and_graph(gpu):
    """A decode step (append, attention spread over workgroups) on two streams
    at once and as a replayed graph: the eager step's bits."""
    import torch
    rng = np.random.default_rng(31)
    heads, kv, dim, page, B = 8, 2, 128, 16, 3
    lengths = [4000, 17, 900]
    need = [n // page + 1 for n in lengths]
    pair = Pair(gpu, kv, dim, page, sum(need))
    pair.fill(4)
    pair.cache.set_rotation(dim, inv_freq(dim))
    lists = lists_for(rng, [n * page for n in need], page, sum(need))
    for l, n in zip(lists, lengths):
        pair.counts[l[-1]] = n % page
    batch = Batch(gpu, lists, lengths, [1] * B)
    size = pair.cache.workspace_bytes(batch.batch, heads)
    assert size > 0
    state = [t.clone() for t in (pair.keys, pair.values, pair.key_scales, pair.value_scales, pair.counts)]

    def restore():
        for t, was in zip((pair.keys, pair.values, pair.key_scales, pair.value_scales, pair.counts), state):
            t.copy_(was)

    def step(qkv, turned, out, ws, stream):
        append(pair, batch, "bf16", qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:],
               turned, stream=stream)
        pair.cache.attend(batch.batch, 1, heads, turned.data_ptr(), turned.stride(0), out.data_ptr(),
                          out.stride(0), workspace=ws.data_ptr(), workspace_bytes=size, stream=stream)

    inputs = [rows(rng, "bf16", B, heads + 2 * kv, dim) for _ in range(4)]
    turned = torch.empty(B, heads, dim, device="cuda", dtype=torch.bfloat16)
    out, ws = torch.empty_like(turned), torch.empty(size, dtype=torch.uint8, device="cuda")
    want = []
    for x in inputs:
        restore()
        step(x, turned, out, ws, 0)
        torch.cuda.synchronize()
        want.append((out.clone(), pair.keys.clone()))
    # a graph of the step on a fixed input
    x = inputs[0].clone()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(x, turned, out, ws, torch.cuda.current_stream().cuda_stream)
    for i in (0, 2, 1, 3, 0):
        restore()
        x.copy_(inputs[i])
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i][0]) and torch.equal(pair.keys, want[i][1])
        torch.ones(1000, device="cuda").sum()
    # attention of four inputs at once on streams of their own, a workspace each
    restore()
    step(inputs[0], turned, out, ws, 0)
    torch.cuda.synchronize()
    queries = [rows(rng, "bf16", B, heads, dim) for _ in range(4)]
    want, outs = [], [torch.empty_like(q) for q in queries]
    spaces = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in queries]
    for q in queries:
        attend(pair, batch, "bf16", q, out)
        torch.cuda.synchronize()
        want.append(out.clone())
    streams = [torch.cuda.Stream() for _ in queries]
    torch.cuda.synchronize()
    for _ in range(3):
        for q, o, w, s in zip(queries, outs, spaces, streams):
            pair.cache.attend(batch.batch, 1, heads, q.data_ptr(), q.stride(0), o.data_ptr(),
                              o.stride(0), workspace=w.data_ptr(), workspace_bytes=size,
                              stream=s.cuda_stream)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)


# ---- the sparse step ----------------------------------------------------------------

def group_sums(q, kv):
    """Each key head's queries added in order in float32, as rows [batch][kv * dim]."""
    q = q.float().cpu().numpy()
    B, H, D = q.shape
    q = q.reshape(B, kv, H // kv, D)
    total = q[:, :, 0].copy()
    for g in range(1, H // kv):
        total = (total + q[:, :, g]).astype(np.float32)
    return total.reshape(B, kv * D)


@pytest.mark.parametrize("heads,kv,dim,page,kind,fmt,k,lengths", [
    (8, 2, 64, 16, "bf16", kv8.E4M3, 4, [300, 16, 1, 900]),
    (4, 4, 128, 32, "f32", kv8.INT8, 8, [2000, 77]),
    (32, 8, 128, 16, "f16", kv8.E4M3, 8, [700, 512, 2048]),
    (6, 2, 80, 64, "f32", kv8.E4M3, 3, [1000, 64]),
    (8, 2, 64, 16, "bf16", kv8.E4M3, 40, [9000, 8000]),  # beyond the certified helper's 256
])
def test_sparse_step(gpu, heads, kv, dim, page, kind, fmt, k, lengths):
    """Prompts appended, then the step: the selection is the sequential float32
    order's over the cache's own summaries, the output that of attention over
    the selected pages."""
    import torch
    import _oracle as orc
    rng = np.random.default_rng(dim + k)
    need = [-(-n // page) for n in lengths]
    pair = Pair(gpu, kv, dim, page, sum(need), fmt)
    pair.cache.set_rotation(dim, inv_freq(dim))
    lists = lists_for(rng, lengths, page, sum(need))
    prompt = Batch(gpu, lists, [0] * len(lengths), lengths)
    key, value = (rows(rng, kind, sum(lengths), kv, dim) for _ in range(2))
    append(pair, prompt, kind, None, key, value, None)
    # the model takes the cache as it is (the append has tests of its own)
    stored = pair.stored()
    pair.model.codes = [np.nan_to_num(x) for x in stored]
    pair.model.scales = [pair.key_scales.cpu().numpy(), pair.value_scales.cpu().numpy()]
    pair.model.counts = pair.counts.cpu().numpy()
    q = rows(rng, kind, len(lengths), heads, dim)
    out = torch.full_like(q, 9.0)
    cand = Batch(gpu, lists)
    offsets = np.concatenate([[0], np.cumsum(need)]).astype(np.int32)
    ids = np.concatenate(lists).astype(np.int32)
    selected = torch.full((len(lengths), k), -1, dtype=torch.int32, device="cuda")
    counts = torch.zeros(len(lengths), dtype=torch.int32, device="cuda")
    with gpu.Kv8SparseStep(pair.cache, heads, k, len(lengths), len(ids)) as step:
        args = (len(lengths), len(ids), max(need), TYPES[kind], q.data_ptr(), q.stride(0),
                cand.keep["page_offsets"].data_ptr(), cand.keep["page_ids"].data_ptr(),
                out.data_ptr(), out.stride(0))
        step.run(*args, selected=selected.data_ptr(), selected_counts=counts.data_ptr())
        step.status()
        summaries = pair.summaries.cpu().numpy()
        E = kv * dim
        zeros = np.zeros((sum(need), page, E), np.float32)
        _, want, _ = orc.sparse_batch(group_sums(q, kv), zeros, zeros, summaries, pair.model.counts,
                                      offsets, ids, kv, dim, page, k)
        for r in range(len(lengths)):
            n = int(counts[r])
            assert selected[r, :n].tolist() == list(want[r]), r
        kept = Batch(gpu, [list(w) for w in want])
        check_attention(pair, kept, kind, q, out)
        # without the caller's id buffers, on another stream, and as a graph
        want_out = out.clone()
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        for stream in (side.cuda_stream, 0, side.cuda_stream):
            out.fill_(9.0)
            torch.cuda.synchronize()
            step.run(*args, stream=stream)
            torch.cuda.synchronize()
            assert torch.equal(out, want_out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step.run(*args, stream=torch.cuda.current_stream().cuda_stream)
        for _ in range(3):
            out.fill_(9.0)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want_out)


def test_sparse_step_refuses(gpu):
    import torch
    pair = Pair(gpu, 2, 64, 16, 4, rubbish=False)
    q = torch.zeros(2, 4, 64, device="cuda")
    with pytest.raises(gpu.InvalidArgument, match="summaries"):
        gpu.Kv8SparseStep(Pair(gpu, 2, 64, 16, 4, summaries=False).cache, 4, 2, 2, 4)
    with pytest.raises(gpu.InvalidArgument, match="head_dim"):
        gpu.Kv8SparseStep(Pair(gpu, 2, 256, 16, 4).cache, 4, 2, 2, 4)
    for args in ((3, 2, 2, 4), (4, -1, 2, 4), (4, 2, -1, 4), (4, 2, 70000, 4)):
        with pytest.raises(gpu.InvalidArgument):
            gpu.Kv8SparseStep(pair.cache, *args)
    lists = Batch(gpu, [[0, 9], [1]])
    with gpu.Kv8SparseStep(pair.cache, 4, 2, 2, 4) as step:
        good = [2, 3, 2, 0, q.data_ptr(), 256, lists.keep["page_offsets"].data_ptr(),
                lists.keep["page_ids"].data_ptr(), q.data_ptr(), 256]
        for i, bad in ((0, 3), (1, 5), (3, 7), (4, 0), (5, 3), (6, 0), (7, 0), (8, 0)):
            args = list(good)
            args[i] = bad
            with pytest.raises(gpu.InvalidArgument):
                step.run(*args)
        step.run(*good)  # page 9 is outside the cache
        with pytest.raises(gpu.OutOfRange):
            step.status()
        step.status()
        assert not bool(q.any())


# ---- calls at the edges ---------------------------------------------------------------

@pytest.mark.parametrize("kind,fmt", [("bf16", kv8.E4M3), ("f32", kv8.INT8)])
@pytest.mark.parametrize("dim,page,past,new,spread", [
    (128, 16, 30, 150, False),
    (96, 48, 0, 200, False),
    (64, 16, 9000, 70, True),  # the list in pieces, and beyond the pages staged at once
])
def test_prompt_skips_pages_outside_the_cache(gpu, dim, page, past, new, spread, kind, fmt):
    """A page id outside the cache holds no token, whatever page 0 holds."""
    import torch
    rng = np.random.default_rng(dim + new)
    kv, G = 2, 2
    need = -(-(past + new) // page)
    pair = Pair(gpu, kv, dim, page, need, fmt)
    pair.fill(dim)
    if fmt == kv8.E4M3:
        pair.values[0] = 0x7f  # (page 0 is in no list)
    ids = np.roll(np.arange(need), -1)  # 1, 2, .., 0
    gone = sorted({0, need // 2, need - 1})
    for where in ([need - 1], [0, need - 1], gone):
        lists = ids.copy()
        lists[where] = -3
        q = rows(rng, kind, new, kv * G, dim)
        out = torch.full_like(q, 9.0)
        fail = torch.zeros(1, dtype=torch.int64, device="cuda")
        batch = Batch(gpu, [lists.tolist()], [past], [new])
        attend(pair, batch, kind, q, out, causal=True, workspace=spread, fail=fail)
        assert int(fail) & 0xffffffff == 3
        held = np.repeat(~np.isin(np.arange(need), where), page)[:past + new]
        keys, values, most = pair.model.rows(np.maximum(lists, 0), past + new)
        sees = np.repeat(np.cumsum(held)[past:past + new], G)
        for h in range(kv):
            mine = as64(q)[:, h * G:(h + 1) * G].reshape(new * G, dim)
            have = as64(out)[:, h * G:(h + 1) * G].reshape(new * G, dim)
            some = sees > 0
            want, weighted, size, peak = kv8.attend(
                mine[some], keys[h][held], values[h][held], 1 / np.sqrt(dim), sees[some],
                most[h][held])
            may = kv8.allowed(want, weighted, size, peak, dim, int(held.sum()), kind)
            assert (np.abs(have[some] - want) <= may).all(), (where, h)
            assert not have[~some].any()


def test_head_counts_and_closed_caches_are_refused(gpu):
    import torch
    pair = Pair(gpu, 1, 16, 16, 2, rubbish=False)
    lists = Batch(gpu, [[0]], [0], [1])
    x = torch.zeros(1, 8200, 16, device="cuda")
    with pytest.raises(gpu.InvalidArgument, match="8192"):
        append(pair, lists, "f32", x, x[:, :1], x[:, :1], x)
    with pytest.raises(gpu.InvalidArgument, match="8192"):
        attend(pair, lists, "f32", x, x, workspace=False)
    with pytest.raises(gpu.InvalidArgument, match="8192"):
        gpu.Kv8SparseStep(pair.cache, 8193, 1, 1, 1)
    wide = torch.randn(1, 8192, 16, device="cuda")  # the most that are taken
    turned, out = torch.empty_like(wide), torch.empty_like(wide)
    append(pair, lists, "f32", wide, wide[:, :1], wide[:, :1], turned)
    assert torch.equal(turned, wide)
    attend(pair, lists, "f32", wide, out)
    assert int(pair.counts[0]) == 1
    # (not the token's value bit for bit: its weight is 2^(s - m) with m = s rounded,
    # which is 1 to 2^-24 of s, held to 2^-22 in the product and as it is in the sum)
    model_append(pair, lists, wide[:, :1], wide[:, :1], [])
    check_attention(pair, Batch(gpu, [[0]]), "f32", wide, out)
    step = gpu.Kv8SparseStep(pair.cache, 1, 1, 1, 1)
    pair.cache.close()
    with pytest.raises(gpu.InvalidArgument, match="closed"):
        step.run(1, 1, 1, 0, x.data_ptr(), 16, lists.keep["page_offsets"].data_ptr(),
                 lists.keep["page_ids"].data_ptr(), x.data_ptr(), 16)
    with pytest.raises(gpu.InvalidArgument, match="non-null"):
        append(pair, lists, "f32", None, x[:, :1], x[:, :1], None)
    step.close()


def test_captured_append_outlives_other_rotations(gpu):
    import torch
    rng = np.random.default_rng(41)
    pair = Pair(gpu, 1, 128, 16, 4)
    pair.cache.set_rotation(16, inv_freq(16))
    batch = Batch(gpu, [[2, 1]], [0], [20])
    q, k = rows(rng, "bf16", 20, 3, 128), rows(rng, "bf16", 20, 1, 128)
    want, out = torch.empty_like(q), torch.empty_like(q)
    append(pair, batch, "bf16", q, k, k, want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        append(pair, batch, "bf16", q, k, k, out, stream=torch.cuda.current_stream().cuda_stream)
    for rotary in (128, 0, 64):
        pair.cache.set_rotation(rotary, inv_freq(rotary) if rotary else [])
        pair.cache.set_rotation(16, inv_freq(16))
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_sparse_step_without_pages_and_beside_captures(gpu):
    import torch
    rng = np.random.default_rng(43)
    heads, kv, dim, page = 4, 2, 64, 16
    pair = Pair(gpu, kv, dim, page, 40, rubbish=False)
    pair.cache.set_rotation(dim, inv_freq(dim))
    lists = [list(range(40)), []]
    prompt = Batch(gpu, lists, [0, 0], [630, 0])
    k = rows(rng, "bf16", 630, kv, dim)
    append(pair, prompt, "bf16", None, k, k, None)
    q = rows(rng, "bf16", 2, heads, dim)
    cand = Batch(gpu, lists)
    none = Batch(gpu, [[], []])
    out = torch.full_like(q, 9.0)

    def args(b, total):
        return (2, total, total, 1, q.data_ptr(), q.stride(0), b.keep["page_offsets"].data_ptr(),
                b.keep["page_ids"].data_ptr(), out.data_ptr(), out.stride(0))

    for top_k, b, total in ((0, cand, 40), (5, none, 0), (0, none, 0)):
        with gpu.Kv8SparseStep(pair.cache, heads, top_k, 2, 40) as step:
            out.fill_(9.0)
            step.run(*args(b, total))
            step.status()
            assert not bool(out.any()), (top_k, total)
    with gpu.Kv8SparseStep(pair.cache, heads, 5, 2, 40) as step:
        step.run(*args(cand, 40))
        step.status()
        want = out.clone()
        assert bool(want[0].any()) and not bool(want[1].any())
        side, other = torch.cuda.Stream(), torch.cuda.Stream()
        torch.cuda.synchronize()
        step.run(*args(cand, 40), stream=side.cuda_stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step.run(*args(cand, 40), stream=torch.cuda.current_stream().cuda_stream)
            # a step elsewhere cannot follow a stream that is being captured
            with pytest.raises(gpu.InvalidArgument, match="captured"):
                step.run(*args(cand, 40), stream=other.cuda_stream)
        for stream in (other.cuda_stream, 0, side.cuda_stream):
            out.fill_(9.0)
            torch.cuda.synchronize()
            step.run(*args(cand, 40), stream=stream)
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            out.fill_(9.0)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
        step.status()
