"""The operators of the 8-bit paged cache, each one call through the package's
public entry points, beside the same in plain torch.

The cache holds a page's keys and values as 8-bit codes with one float32 scale
for each page and head (value = code * scale).  The scale is the least that the
page's largest number fits: of e4m3 codes a power of two, of int8 codes the
largest number / 127.

  keys        uint8 [pages][kv heads][page size][dim]
  values      uint8 [pages][kv heads][page size / 16][dim][16]
  key_scales, value_scales   float32 [pages][kv heads]
  summaries   float32 [pages][kv heads * dim], the mean of the page's keys
  token_counts int32 [pages]

A case is a dict of plain values:

  kind      "append": rotate queries and keys, write keys and values
            "attend": one query token a request over its list of pages
            "prompt": several query tokens a request, each over what precedes it
  batch     requests
  lo, hi    tokens that a request has in the cache before the call
  new_lo, new_hi  new tokens of a request (append, prompt)
  heads, kv_heads, dim, page, type, format
  kept      pages a request's list holds (attend; 0: all of its pages)

`own` says which of the two run() computes.
"""
from __future__ import annotations

import importlib
import math
import random

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_LARGEST = {"e4m3": 448.0, "int8": 127.0}
_TINY = 2.0 ** -126  # the least scale


def _case(name, kind, batch, lo, hi, new_lo=1, new_hi=1, heads=32, kv_heads=8, dim=128, page=16,
          type="bf16", format="e4m3", kept=0):
    return {"name": name, "kind": kind, "batch": batch, "lo": lo, "hi": hi, "new_lo": new_lo,
            "new_hi": new_hi, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "type": type, "format": format, "kept": kept}


def listed():
    return [
        # One user's next token goes into the cache: the smallest call, all latency.
        _case("append_one_token", "append", 1, 1000, 1000),
        # A serving batch's next tokens, each into its request's last page.
        _case("append_batch64", "append", 64, 200, 8000),
        # A long prompt is admitted.
        _case("append_prompt_8k", "append", 1, 0, 0, 8192, 8192),
        # Ragged prompts behind what the cache holds (shared beginnings), float32,
        # as many key heads as query heads, large pages that start half full.
        _case("append_ragged_f32", "append", 16, 0, 500, 100, 1500, kv_heads=32, page=64,
              type="f32"),
        # One user's decode step at a short context.
        _case("attend_one_1k", "attend", 1, 1000, 1000),
        # The benchmark's batch: 16 ragged contexts, 32 x 128, float32 queries.
        _case("attend_batch16_f32", "attend", 16, 512, 2048, kv_heads=32, type="f32"),
        # A full batch of long contexts: the largest decode step.
        _case("attend_batch32_32k", "attend", 32, 32768, 32768),
        # A few very long documents, small heads, int8 codes, half-precision queries.
        _case("attend_4x128k_int8", "attend", 4, 65536, 131072, kv_heads=4, dim=64, page=32,
              type="f16", format="int8"),
        # What a top-k of 32 pages of 64 tokens keeps of each request.
        _case("attend_kept32", "attend", 64, 4096, 16384, page=64, kept=32),
        # A batch of ragged prompts, no context before them.
        _case("prompt_ragged", "prompt", 16, 0, 0, 1, 700),
        # One long prompt.
        _case("prompt_8k", "prompt", 1, 0, 0, 8192, 8192),
        # Drafted tokens checked against long contexts, four a request.
        _case("prompt_drafts", "prompt", 16, 2000, 8000, 4, 4, format="int8"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    what = rng.choice(["token", "tokens", "prompt_in", "decode", "decode", "long", "kept",
                       "prompts", "chunk", "drafts"])
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (32, 32, 128), (40, 8, 128), (8, 1, 128),
                                       (32, 4, 64), (12, 12, 64), (16, 8, 256), (28, 4, 128),
                                       (8, 8, 96), (32, 32, 80)])
    form = {"heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": rng.choice([16, 16, 32, 64, 128]), "type": rng.choice(["bf16", "bf16", "f16", "f32"]),
            "format": rng.choice(["e4m3", "int8"])}
    if what in ("token", "tokens", "prompt_in"):
        form["format"] = "e4m3"

    def spread(least, most):
        a, b = _log_int(rng, least, most), _log_int(rng, least, most)
        return min(a, b), max(a, b)

    if what == "token":
        lo, hi = spread(1, 3000)
        return _case("", "append", rng.randint(1, 8), lo, hi, **form)
    if what == "tokens":
        lo, hi = spread(10, 9000)
        return _case("", "append", _log_int(rng, 9, 256), lo, hi, rng.randint(1, 2), 5, **form)
    if what == "prompt_in":
        lo, hi = spread(1, 900)
        new_lo, new_hi = spread(1, 4000)
        return _case("", "append", _log_int(rng, 1, 12), lo - 1, hi, new_lo, new_hi, **form)
    if what == "decode":
        lo, hi = spread(1, 9000)
        return _case("", "attend", _log_int(rng, 1, 24), lo, hi, **form)
    if what == "long":
        lo, hi = spread(10000, 60000)
        return _case("", "attend", _log_int(rng, 1, 4), lo, hi, **form)
    if what == "kept":
        lo, hi = spread(300, 9000)
        return _case("", "attend", _log_int(rng, 4, 24), lo, hi, kept=rng.randint(4, 64), **form)
    if what == "prompts":
        new_lo, new_hi = spread(1, 1500)
        return _case("", "prompt", _log_int(rng, 1, 12), 0, rng.randint(0, 40), new_lo, new_hi, **form)
    if what == "chunk":
        lo, hi = spread(1000, 12000)
        return _case("", "prompt", 1, lo, hi, 200, rng.randint(256, 1024), **form)
    lo, hi = spread(100, 9000)
    return _case("", "prompt", _log_int(rng, 1, 24), lo, hi, 1, rng.randint(2, 8), **form)


# ---- the shape of a case -------------------------------------------------------

def _lengths(case):
    """(tokens before, new tokens) of each request: the case's own, whatever the seed."""
    rng = random.Random("%(batch)d %(lo)d %(hi)d %(new_lo)d %(new_hi)d" % case)
    past = [rng.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
    past[0] = case["hi"]
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["batch"])]
    new[-1] = case["new_hi"]
    return past, new


def _ceil(a, b):
    return -(-a // b)


def _frequencies(case):
    """The rotation's angles per position, base 500000, over all of a head's dims."""
    half = case["dim"] // 2
    return 500000.0 ** (-np.arange(half, dtype=np.float64) / half)


def _layout(case, seed):
    """Page lists: (CSR offsets, page ids, pages in the cache).  Pages lie
    scattered over the cache, as one that has served for a while hands them out.
    An append's cache holds the pages that its call writes; the earlier entries
    of a list, which it does not look at, are other pages of the cache."""
    past, new = _lengths(case)
    ps, rng = case["page"], np.random.RandomState(seed % (1 << 31))
    if case["kind"] == "attend":
        counts = [_ceil(c, ps) for c in past]
        written = counts
        if case["kept"]:
            counts = [min(case["kept"], c) for c in counts]
    else:
        counts = [_ceil(c + n, ps) for c, n in zip(past, new)]
        first = [c // ps if case["kind"] == "append" else 0 for c in past]
        written = [c - f for c, f in zip(counts, first)]
    offsets = np.zeros(len(counts) + 1, np.int32)
    offsets[1:] = np.cumsum(counts)
    capacity = sum(written)
    order = rng.permutation(capacity).astype(np.int32)
    ids, w = np.empty(int(offsets[-1]), np.int32), 0
    last = np.full(capacity, ps, np.int32)  # tokens in each page
    for r, (n, take) in enumerate(zip(counts, written)):
        mine, w = order[w:w + take], w + take
        if case["kind"] == "append":
            ids[offsets[r]:offsets[r + 1] - take] = rng.randint(0, capacity, n - take)
            ids[offsets[r + 1] - take:offsets[r + 1]] = mine
            last[mine] = 0
            if take:
                last[mine[0]] = past[r] % ps
            continue
        tokens = past[r] if case["kind"] == "attend" else past[r] + new[r]
        if take:
            last[mine[-1]] = tokens - (take - 1) * ps
        if case["kept"]:
            mine = mine[np.sort(rng.permutation(take)[:n])]
        ids[offsets[r]:offsets[r + 1]] = mine
    return offsets, ids, last


def _normal(seed, salt, *shape):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 16 + salt)
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _codes(case, seed, salt, *shape):
    """Codes of N(0, 1) rows whose largest reaches the format's largest value."""
    flat = torch.empty(math.prod(shape), dtype=torch.uint8, device="cuda")
    step = 1 << 28
    for i in range(0, flat.numel(), step):
        x = _normal(seed + i // step, salt, min(step, flat.numel() - i))
        x = (x * (_LARGEST[case["format"]] / 4)).clamp_(-_LARGEST[case["format"]],
                                                         _LARGEST[case["format"]])
        flat[i:i + step] = _to_codes(case, x)
    return flat.view(shape)


def _to_codes(case, x):
    """The nearest codes of x (within the format's range), as bytes: rounded
    once, in x's own type, so that what lies next to a border falls on its side."""
    if case["format"] == "int8":
        return torch.nan_to_num(x).round().to(torch.int8).view(torch.uint8)
    step = torch.exp2((torch.frexp(x).exponent - 1).clamp(min=-6).to(x.dtype) - 3)
    return ((x / step).round() * step).float().to(torch.float8_e4m3fn).view(torch.uint8)


def _of_codes(case, codes):
    """The numbers that bytes stand for."""
    kind = torch.int8 if case["format"] == "int8" else torch.float8_e4m3fn
    return codes.view(kind).float()


def _scale_for(format, most):
    """The scale, in 32 bits, of a page whose largest number is `most` (numpy)."""
    most = np.asarray(most, np.float32)
    if format == "int8":
        scale = (most.astype(np.float64) / 127).astype(np.float32)
    else:
        fraction, exponent = np.frexp(most)  # most = fraction * 2^exponent, 448 = 0.875 * 2^9
        scale = np.ldexp(np.float32(1), exponent - 9 + (fraction > 0.875))
    return np.maximum(scale, np.float32(_TINY)).astype(np.float32)


def _device(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def prepare(case, seed):
    past, new = _lengths(case)
    H, K, D, ps, B = case["heads"], case["kv_heads"], case["dim"], case["page"], case["batch"]
    offsets, ids, counts = _layout(case, seed)
    capacity = len(counts)
    spread = np.random.RandomState(seed % (1 << 31) + 1)
    state = {
        "case": case,
        "keys": _codes(case, seed, 1, capacity, K, ps, D),
        "values": _codes(case, seed, 2, capacity, K, ps // 16, D, 16),
        # a page's largest key and value differ from page to page and head to head
        "key_scales": _device(_scale_for(case["format"], spread.uniform(2, 6, (capacity, K)))),
        "value_scales": _device(_scale_for(case["format"], spread.uniform(2, 6, (capacity, K)))),
        "summaries": torch.zeros(capacity, K * D, device="cuda"),
        "token_counts": _device(counts),
        "page_offsets": _device(offsets), "page_ids": _device(ids),
        "past": _device(np.asarray(past, np.int32)),
        "most_pages": int(np.diff(offsets).max()),
    }
    T = B if case["kind"] == "attend" else sum(new)
    state["tokens"], state["most_new"] = T, 1 if case["kind"] == "attend" else max(new)
    starts = np.zeros(B + 1, np.int32)
    starts[1:] = np.arange(1, B + 1) if case["kind"] == "attend" else np.cumsum(new)
    state["token_offsets"] = _device(starts)
    if case["kind"] == "append":
        # one projection's output: a token's queries, keys and values side by side
        qkv = _normal(seed, 3, T, (H + 2 * K) * D).to(_TYPES[case["type"]])
        state["q"] = qkv[:, :H * D].view(T, H, D)
        state["k"] = qkv[:, H * D:(H + K) * D].view(T, K, D)
        state["v"] = qkv[:, (H + K) * D:].view(T, K, D)
        state["frequencies"] = _device(_frequencies(case))
        state["rotated"] = torch.empty(T, H, D, device="cuda", dtype=qkv.dtype)
    else:
        state["q"] = _normal(seed, 3, T, H, D).to(_TYPES[case["type"]])
        state["outputs"] = torch.empty_like(state["q"])
    if own:
        _own_handles(case, state)
    return state


def _own_handles(case, state):
    """What a program that uses the package keeps beside its tensors: the
    cache's handle over them and the batch's description."""
    dsd = importlib.import_module("15-618_dynamic_sparse_decode_amd")
    names = ("keys", "values", "key_scales", "value_scales", "token_counts") + (
        ("summaries",) if case["kind"] == "append" else ())
    cache = dsd.Kv8Cache(case["kv_heads"], case["dim"], case["page"], len(state["token_counts"]),
                         {"e4m3": dsd.KV8_E4M3, "int8": dsd.KV8_INT8}[case["format"]],
                         arrays={n: state[n].data_ptr() for n in names})
    if case["kind"] == "append":
        cache.set_rotation(case["dim"], _frequencies(case))
    state["type"] = {"f32": dsd.TYPE_F32, "bf16": dsd.TYPE_BF16, "f16": dsd.TYPE_F16}[case["type"]]
    state["cache"] = cache
    state["batch"] = dsd.Kv8Batch(
        case["batch"], tokens=state["tokens"], max_tokens=state["most_new"],
        max_pages=state["most_pages"], total_pages=len(state["page_ids"]),
        page_offsets=state["page_offsets"].data_ptr(), page_ids=state["page_ids"].data_ptr(),
        token_offsets=state["token_offsets"].data_ptr(), past_tokens=state["past"].data_ptr())
    if case["kind"] != "append":
        size = cache.workspace_bytes(state["batch"], case["heads"])
        state["workspace"] = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
        state["workspace_bytes"] = size


def run(state):
    kind = state["case"]["kind"]
    if own:
        return _OWN[kind](state)
    return _PLAIN[kind](state)


# ---- the package's calls -----------------------------------------------------------

def _written(state):
    """What an append leaves: the codes as the numbers that they stand for, in
    units of their scale."""
    kind = torch.int8 if state["case"]["format"] == "int8" else torch.float8_e4m3fn
    return {"rotated": state["rotated"], "keys": state["keys"].view(kind),
            "values": state["values"].view(kind), "key_scales": state["key_scales"],
            "value_scales": state["value_scales"], "summaries": state["summaries"],
            "token_counts": state["token_counts"]}


def _own_append(state):
    q, k, v, out = state["q"], state["k"], state["v"], state["rotated"]
    state["cache"].append(
        state["batch"], state["type"], state["case"]["heads"], q.data_ptr(), q.stride(0),
        k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), out.data_ptr(), out.stride(0),
        stream=torch.cuda.current_stream().cuda_stream)
    return _written(state)


def _own_attend(state):
    q, out = state["q"], state["outputs"]
    state["cache"].attend(
        state["batch"], state["type"], state["case"]["heads"], q.data_ptr(), q.stride(0),
        out.data_ptr(), out.stride(0), workspace=state["workspace"].data_ptr(),
        workspace_bytes=state["workspace_bytes"], stream=torch.cuda.current_stream().cuda_stream)
    return {"outputs": out}


def _own_prompt(state):
    q, out = state["q"], state["outputs"]
    state["cache"].attend_prompt(
        state["batch"], state["type"], state["case"]["heads"], q.data_ptr(), q.stride(0),
        out.data_ptr(), out.stride(0), workspace=state["workspace"].data_ptr(),
        workspace_bytes=state["workspace_bytes"], stream=torch.cuda.current_stream().cuda_stream)
    return {"outputs": out}


_OWN = {"append": _own_append, "attend": _own_attend, "prompt": _own_prompt}


# ---- the plain forms ---------------------------------------------------------------

def _token_places(state):
    """Each new token's request and its index in the request's tokens."""
    at = torch.arange(state["tokens"], device="cuda")
    request = torch.bucketize(at, state["token_offsets"][1:].long(), right=True)
    return request, state["past"][request] + at - state["token_offsets"][request]


def _rotate(x, cos, sin):
    """x [tokens][heads][dim] with the pairs (i, i + dim / 2) turned, in 64 bits."""
    a, b = x.double().chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _finite_largest(x):
    return torch.where(x.isfinite(), x.abs(), 0).amax(-1)


def _page_scale(case, most):
    """The scales of pages whose largest numbers are `most`, in 64 bits."""
    if case["format"] == "int8":
        return (most.float().double() / 127).float().clamp(min=_TINY)
    fraction, exponent = torch.frexp(most.float())
    power = torch.where(most > 0, exponent - 9 + (fraction > 0.875), -126).clamp(min=-126)
    return ((power + 127) << 23).int().view(torch.float32)  # 2^power


def _store(case, old, old_scale, scale, new, slot, first):
    """A page's codes [pages][heads][page size][dim] with the tokens before
    `first` brought to the new scale and the new rows put in their places."""
    page, offset = slot
    pages, K, ps, D = old.shape
    ratio = (old_scale.double() / scale.double()).view(pages, K, 1, 1)
    kept = _to_codes(case, _of_codes(case, old).double() * ratio)
    is_old = torch.arange(ps, device="cuda").view(1, 1, ps, 1) < first.view(pages, 1, 1, 1)
    codes = torch.where(is_old, kept, old)
    largest = _LARGEST[case["format"]]
    codes[page, :, offset] = _to_codes(
        case, (new.double() / scale[page].double().unsqueeze(-1)).clamp(-largest, largest))
    return codes


def _plain_append(state):
    case = state["case"]
    K, D, ps = case["kv_heads"], case["dim"], case["page"]
    request, index = _token_places(state)
    angle = index.double().unsqueeze(-1) * state["frequencies"]
    cos, sin = angle.cos().unsqueeze(1), angle.sin().unsqueeze(1)
    state["rotated"].copy_(_rotate(state["q"], cos, sin))
    key, value = _rotate(state["k"], cos, sin), state["v"].double()
    ids = state["page_ids"][state["page_offsets"][request] + index // ps].long()
    pages, page = torch.unique(ids, return_inverse=True)
    offset = index % ps
    first = torch.full_like(pages, ps).scatter_reduce(0, page, offset, "amin")
    count = torch.zeros_like(pages).scatter_reduce(0, page, offset, "amax") + 1
    codes = {}
    for name, scales, new in (("keys", "key_scales", key), ("values", "value_scales", value)):
        had = torch.where(first.unsqueeze(-1) > 0, state[scales][pages], 0.0)
        most = torch.zeros(len(pages), K, dtype=torch.float64, device="cuda").scatter_reduce(
            0, page.unsqueeze(-1).expand(-1, K), _finite_largest(new), "amax")
        scale = torch.maximum(had, _page_scale(case, most))
        old = state[name][pages]
        if name == "values":
            old = old.transpose(-1, -2).reshape(len(pages), K, ps, D)
        got = codes[name] = _store(case, old, had, scale, new, (page, offset), first)
        if name == "values":
            got = got.view(len(pages), K, ps // 16, 16, D).transpose(-1, -2)
        state[name][pages] = got
        state[scales][pages] = scale
    there = torch.arange(ps, device="cuda").view(1, 1, ps, 1) < count.view(-1, 1, 1, 1)
    total = torch.where(there, _of_codes(case, codes["keys"]).double(), 0).sum(2)
    mean = total * state["key_scales"][pages].double().unsqueeze(-1) / count.view(-1, 1, 1)
    state["summaries"][pages] = mean.float().view(len(pages), K * D)
    state["token_counts"][pages] = count.int()
    return _written(state)


def _rows(state):
    """(keys, values [batch][kv heads][tokens][dim], tokens valid [batch][tokens])
    of every request's list, padded to the longest."""
    case = state["case"]
    K, D, ps, n = case["kv_heads"], case["dim"], case["page"], state["most_pages"]
    B = case["batch"]
    begin, end = state["page_offsets"][:-1].unsqueeze(-1), state["page_offsets"][1:].unsqueeze(-1)
    at = begin + torch.arange(n, device="cuda")
    listed_ = at < end
    ids = state["page_ids"][torch.where(listed_, at, 0)].long()
    keys = _of_codes(case, state["keys"][ids]) * state["key_scales"][ids].view(B, n, K, 1, 1)
    values = _of_codes(case, state["values"][ids]) * state["value_scales"][ids].view(B, n, K, 1, 1, 1)
    keys = keys.transpose(1, 2).reshape(B, K, n * ps, D)
    values = values.permute(0, 2, 1, 3, 5, 4).reshape(B, K, n * ps, D)
    there = torch.where(listed_, state["token_counts"][ids], 0)
    valid = torch.arange(ps, device="cuda") < there.unsqueeze(-1)
    return keys, values, valid.view(B, n * ps)


def _attention(q, keys, values, valid):
    """softmax(q K^T / sqrt(dim)) V over the valid tokens, in 32 bits; zeros
    where there is none."""
    logits = torch.matmul(q * (1.0 / math.sqrt(q.shape[-1])), keys.transpose(-1, -2))
    logits.masked_fill_(~valid, -math.inf)
    most = logits.amax(-1, keepdim=True)
    p = logits.sub_(torch.where(most == -math.inf, 0.0, most)).exp_()
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, values) / torch.where(valid.any(-1, keepdim=True), total, 1.0)


def _plain_attend(state):
    case = state["case"]
    B, H, K, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    keys, values, valid = _rows(state)
    q = state["q"].float().view(B, K, H // K, D)
    out = _attention(q, keys, values, valid.view(B, 1, 1, -1))
    state["outputs"].copy_(out.view(B, H, D))
    return {"outputs": state["outputs"]}


def _plain_prompt(state):
    case = state["case"]
    B, H, K, D, n = case["batch"], case["heads"], case["kv_heads"], case["dim"], state["most_new"]
    request, index = _token_places(state)
    place = index - state["past"][request]
    q = torch.zeros(B, n, H, D, device="cuda")
    q[request, place] = state["q"].float()
    q = q.view(B, n, K, H // K, D).permute(0, 2, 3, 1, 4).reshape(B, K, H // K * n, D)
    keys, values, _ = _rows(state)
    sees = state["past"].view(B, 1, 1) + torch.arange(n, device="cuda").view(1, n, 1)
    valid = torch.arange(keys.shape[2], device="cuda") <= sees
    out = _attention(q, keys, values, valid.repeat(1, H // K, 1).unsqueeze(1))
    out = out.view(B, K, H // K, n, D).permute(0, 3, 1, 2, 4).reshape(B, n, H, D)
    state["outputs"].copy_(out[request, place])
    return {"outputs": state["outputs"]}


_PLAIN = {"append": _plain_append, "attend": _plain_attend, "prompt": _plain_prompt}


# ---- what a pass cannot do without -------------------------------------------------

def work(case):
    past, new = _lengths(case)
    H, K, D, ps, B = case["heads"], case["kv_heads"], case["dim"], case["page"], case["batch"]
    size = 4 if case["type"] == "f32" else 2
    if case["kind"] == "append":
        T = sum(new)
        pages = sum(_ceil(c + n, ps) - c // ps for c, n in zip(past, new))
        held = sum(c % ps for c in past)  # key codes of half-full pages: the means need them
        moved = T * (2 * H + 2 * K) * D * size + 2 * T * K * D + held * K * D
        moved += pages * K * (8 + 4 * D) + 4 * pages
        return {"bytes": moved, "flops": T * (6 * H + 10 * K) * D}
    if case["kind"] == "attend":
        offsets, ids, counts = _layout(case, 0)
        tokens, pages, rows, pairs = int(counts[ids].sum()), len(ids), B, int(counts[ids].sum())
    else:
        tokens = sum(past) + sum(new)
        pages = sum(_ceil(c + n, ps) for c, n in zip(past, new))
        rows, pairs = sum(new), sum(c * n + n * (n + 1) // 2 for c, n in zip(past, new))
    moved = 2 * tokens * K * D + pages * (8 * K + 4) + 2 * rows * H * D * size
    return {"bytes": moved, "flops": 4 * pairs * H * D}


# ---- the same from the definition, in 64 bits --------------------------------------

def _nearest(format, x):
    """The format's value next to x, halves to the even code; NaN stays NaN in
    e4m3 and is 0 in int8."""
    if format == "int8":
        return np.clip(np.rint(np.where(np.isnan(x), 0.0, x)), -127, 127)
    x = np.clip(x, -448.0, 448.0)
    with np.errstate(all="ignore"):
        exponent = np.frexp(np.where(np.isnan(x), 0.0, x))[1] - 1
    step = np.exp2(np.maximum(exponent, -6) - 3.0)
    return np.rint(x / step) * step


def _values(format, codes):
    """The numbers that a uint8 array's codes stand for, from the format's own rule."""
    if format == "int8":
        return codes.astype(np.int64) - 256.0 * (codes > 127)
    code = np.arange(256)
    exponent, fraction = (code >> 3) & 15, code & 7
    table = np.where(exponent == 0, fraction * 2.0 ** -9, (8 + fraction) * np.exp2(exponent - 10.0))
    table = np.where(code & 127 == 127, np.nan, table) * np.where(code >= 128, -1.0, 1.0)
    return table[codes]


def _exact_append(case, seed):
    state = prepare(case, seed)
    past, new = _lengths(case)
    K, D, ps, form = case["kv_heads"], case["dim"], case["page"], case["format"]
    host = {n: t.cpu().numpy() for n, t in state.items()
            if n in ("keys", "values", "key_scales", "value_scales", "summaries", "token_counts",
                     "page_offsets", "page_ids", "token_offsets")}
    rows = {n: state[n].double().cpu().numpy() for n in ("q", "k", "v")}
    index = np.concatenate([c + np.arange(n) for c, n in zip(past, new)])
    turn = np.exp(1j * index[:, None, None] * _frequencies(case))  # a complex number a pair

    def rotated(x):
        z = (x[..., :D // 2] + 1j * x[..., D // 2:]) * turn
        return np.concatenate([z.real, z.imag], -1)

    key = rotated(rows["k"])
    codes = {"keys": _values(form, host["keys"]),
             "values": _values(form, host["values"]).swapaxes(-1, -2).reshape(-1, K, ps, D)}
    for r, (c, n) in enumerate(zip(past, new)):
        for slot in range(c // ps, _ceil(c + n, ps)):
            page = host["page_ids"][host["page_offsets"][r] + slot]
            o0, o1 = max(c - slot * ps, 0), min(c + n - slot * ps, ps)
            at = host["token_offsets"][r] + slot * ps - c
            for name, scales, x in (("keys", "key_scales", key), ("values", "value_scales", rows["v"])):
                x = x[at + o0:at + o1].swapaxes(0, 1)  # [heads][tokens][dim]
                size = np.abs(np.where(np.isfinite(x), x, 0)).max((1, 2))
                had = host[scales][page] if o0 else np.zeros(K, np.float32)
                # the scale is held in 32 bits: the codes are those for the scale as it is held
                scale = np.maximum(had, _scale_for(form, size))
                wide = scale.astype(np.float64)[:, None, None]
                mine = codes[name][page]
                mine[:, :o0] = _nearest(form, mine[:, :o0] * had.astype(np.float64)[:, None, None] / wide)
                mine[:, o0:o1] = _nearest(form, x / wide)
                host[scales][page] = scale
            mean = codes["keys"][page][:, :o1].mean(1) * host["key_scales"][page].astype(np.float64)[:, None]
            host["summaries"] = host["summaries"].astype(np.float64, copy=False)
            host["summaries"][page] = mean.reshape(-1)
    return {"rotated": torch.from_numpy(rotated(rows["q"])), "keys": torch.from_numpy(codes["keys"]),
            "values": torch.from_numpy(codes["values"].reshape(-1, K, ps // 16, 16, D).swapaxes(-1, -2).copy()),
            "key_scales": torch.from_numpy(host["key_scales"].astype(np.float64)),
            "value_scales": torch.from_numpy(host["value_scales"].astype(np.float64)),
            "summaries": torch.from_numpy(host["summaries"]), "token_counts": None}


def _exact_rows(case, state, r, head):
    """One request's keys and values of one head, [tokens][dim], 64 bits."""
    a, b = state["page_offsets"][r].item(), state["page_offsets"][r + 1].item()
    ids = state["page_ids"][a:b].long()
    kind = torch.int8 if case["format"] == "int8" else torch.float8_e4m3fn
    D = case["dim"]
    k = state["keys"][ids, head].view(kind).double() * state["key_scales"][ids, head].double()[:, None, None]
    v = state["values"][ids, head].view(kind).double() * state["value_scales"][ids, head].double()[:, None, None, None]
    there = torch.arange(case["page"], device="cuda") < state["token_counts"][ids][:, None]
    return k.reshape(-1, D)[there.view(-1)], v.transpose(-1, -2).reshape(-1, D)[there.view(-1)]


def _exact_attention(case, seed):
    state = prepare(case, seed)
    past, new = _lengths(case)
    H, K, D, G = case["heads"], case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"]
    if case["kind"] == "attend":
        new = [1] * case["batch"]
    out = torch.zeros(state["tokens"], H, D, dtype=torch.float64, device="cuda")
    at = 0
    for r, n in enumerate(new):
        for head in range(K):
            k, v = _exact_rows(case, state, r, head)
            if not len(k):
                continue
            for g in range(head * G, (head + 1) * G):
                for i in range(0, n, 2048):
                    rows = slice(at + i, at + min(n, i + 2048))
                    s = state["q"][rows, g].double() @ k.t() / math.sqrt(D)
                    if case["kind"] == "prompt":
                        sees = past[r] + i + torch.arange(s.shape[0], device="cuda")
                        s.masked_fill_(torch.arange(len(k), device="cuda") > sees[:, None], -math.inf)
                    out[rows, g] = torch.softmax(s, -1) @ v
        at += n
    return {"outputs": out}


def exact(case, seed):
    if case["kind"] == "append":
        return _exact_append(case, seed)
    return _exact_attention(case, seed)
