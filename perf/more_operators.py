"""More operators over the 8-bit paged cache, each one call through the package's
public entry points, beside the same in plain torch.

The cache holds a page's keys and values as 8-bit codes with one float32 scale
for each page and key head (value = code * scale).

  keys        uint8 [pages][kv heads][page size][dim]
  values      uint8 [pages][kv heads][page size / 16][dim][16]
  key_scales, value_scales   float32 [pages][kv heads]
  summaries   float32 [pages][kv heads * dim], the mean of the page's keys
  token_counts int32 [pages]

A case is a dict of plain values:

  kind      "cross": several query tokens a request, each over all tokens of the
                     request's list (an encoder's states)
            "shared": one query token a request over a prefix that a group of
                     requests shares, then over the request's own list
            "weigh": one query token a request over its list; each token's softmax
                     weight, summed over the query heads of its key head, is added
                     to what it had before
            "evict": of a list's tokens each key head keeps `keep`: the first
                     `first`, the last `recent`, of the others those of the largest
                     weights (the lower place among equals); they go to new pages
  batch     requests
  lo, hi    tokens of a request's list
  new_lo, new_hi        query tokens of a request (cross)
  groups, pre_lo, pre_hi, alone   groups that share a prefix, a prefix's tokens,
            requests behind the last group, which have none (shared)
  keep, first, recent   (evict)
  heads, kv_heads, dim, page, type, format

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


def _case(name, kind, batch, lo, hi, new_lo=1, new_hi=1, groups=0, pre_lo=0, pre_hi=0, alone=0,
          keep=0, first=0, recent=0, heads=32, kv_heads=8, dim=128, page=16, type="bf16",
          format="e4m3"):
    return {"name": name, "kind": kind, "batch": batch, "lo": lo, "hi": hi, "new_lo": new_lo,
            "new_hi": new_hi, "groups": groups, "pre_lo": pre_lo, "pre_hi": pre_hi, "alone": alone,
            "keep": keep, "first": first, "recent": recent, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "page": page, "type": type, "format": format}


def listed():
    return [
        # One utterance's decoder step: five beams over 1500 encoder states, a key
        # head per query head.  All latency.
        _case("cross_beams_1500", "cross", 1, 1500, 1500, 5, 5, heads=20, kv_heads=20, dim=64,
              type="f16"),
        # A batch of ragged targets over ragged sources, int8 codes.
        _case("cross_ragged_int8", "cross", 16, 200, 3000, 1, 300, format="int8"),
        # One long target over a long source (a document's states): the largest.
        _case("cross_4k_over_8k", "cross", 1, 8192, 8192, 4096, 4096),
        # A few users of one assistant: a system prompt of 2000 tokens, short turns.
        _case("shared_8_behind_2k", "shared", 8, 1, 100, groups=1, pre_lo=2000, pre_hi=2000),
        # A full batch of questions about one long document.
        _case("shared_64_behind_32k", "shared", 64, 200, 2000, groups=1, pre_lo=32768,
              pre_hi=32768),
        # Four prompts with samples of each, some requests that share none; float32,
        # as many key heads as query heads, pages of 64.
        _case("shared_4_groups_f32", "shared", 16, 512, 2048, groups=4, pre_lo=4096, pre_hi=16384,
              alone=2, kv_heads=32, page=64, type="f32"),
        # One user's decode step at a short context, its weights kept.
        _case("weigh_one_1k", "weigh", 1, 1000, 1000),
        # The benchmark's batch: 16 ragged contexts, 32 x 128, float32 queries.
        _case("weigh_batch16_f32", "weigh", 16, 512, 2048, kv_heads=32, type="f32", format="int8"),
        # A full batch of long contexts.
        _case("weigh_batch32_32k", "weigh", 32, 32768, 32768),
        # One user's cache goes back to its budget.
        _case("evict_one_4k", "evict", 1, 4300, 4300, keep=2048, first=4, recent=256),
        # Ragged requests, large pages, int8 codes, small heads.
        _case("evict_ragged_int8", "evict", 16, 2000, 30000, keep=2000, first=16, recent=500,
              kv_heads=4, dim=64, page=64, format="int8"),
        # A full batch of long contexts brought to an eighth.
        _case("evict_batch32_32k", "evict", 32, 32768, 32768, keep=4096, first=64, recent=1024),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    what = rng.choice(["beams", "cross", "cross", "shared", "shared", "groups", "weigh", "weigh",
                       "evict", "evict", "long"])
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (32, 32, 128), (40, 8, 128), (8, 1, 128),
                                       (32, 4, 64), (12, 12, 64), (16, 8, 256), (28, 4, 128),
                                       (8, 8, 96), (32, 32, 80)])
    form = {"heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": rng.choice([16, 16, 32, 64, 128]),
            "type": rng.choice(["bf16", "bf16", "f16", "f32"]),
            "format": rng.choice(["e4m3", "int8"])}

    def spread(least, most):
        a, b = _log_int(rng, least, most), _log_int(rng, least, most)
        return min(a, b), max(a, b)

    if what == "beams":
        lo, hi = spread(1, 3000)
        return _case("", "cross", rng.randint(1, 16), lo, hi, 1, rng.randint(2, 8), **form)
    if what == "cross":
        lo, hi = spread(1, 5000)
        new_lo, new_hi = spread(1, 600)
        return _case("", "cross", _log_int(rng, 1, 12), lo, hi, new_lo, new_hi, **form)
    if what == "shared":
        lo, hi = spread(1, 1500)
        pre = _log_int(rng, 100, 20000)
        return _case("", "shared", _log_int(rng, 2, 48), lo, hi, groups=1, pre_lo=pre, pre_hi=pre,
                     **form)
    if what == "groups":
        lo, hi = spread(1, 2000)
        pre_lo, pre_hi = spread(1, 6000)
        return _case("", "shared", rng.randint(4, 32), lo - 1, hi, groups=rng.randint(2, 6),
                     pre_lo=pre_lo, pre_hi=pre_hi, alone=rng.randint(0, 3), **form)
    if what == "weigh":
        lo, hi = spread(1, 9000)
        return _case("", "weigh", _log_int(rng, 1, 24), lo, hi, **form)
    if what == "long":
        lo, hi = spread(10000, 60000)
        return _case("", rng.choice(["weigh", "evict"]), _log_int(rng, 1, 4), lo, hi, keep=5000,
                     first=4, recent=333, **form)
    lo, hi = spread(1, 9000)
    keep = _log_int(rng, 30, 3000)
    return _case("", "evict", _log_int(rng, 1, 16), lo, hi, keep=keep, first=rng.randint(0, keep // 8),
                 recent=rng.randint(0, keep // 2), **form)


# ---- the shape of a case -------------------------------------------------------

def _ceil(a, b):
    return -(-a // b)


def _lengths(case):
    """Tokens of each list, query tokens of each request: the case's own, whatever
    the seed."""
    rng = random.Random("%(batch)d %(lo)d %(hi)d %(new_lo)d %(new_hi)d" % case)
    held = [rng.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
    held[0] = case["hi"]
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["batch"])]
    new[-1] = case["new_hi"]
    return held, new


def _groups(case):
    """Of a shared case: each prefix's tokens, and the first request of each group
    with the end of the last."""
    rng = random.Random("%(groups)d %(pre_lo)d %(pre_hi)d %(batch)d" % case)
    prefix = [rng.randint(case["pre_lo"], case["pre_hi"]) for _ in range(case["groups"])]
    if prefix:
        prefix[0] = case["pre_hi"]
    end = max(case["batch"] - case["alone"], 0)
    cuts = sorted(rng.randint(0, end) for _ in range(case["groups"] - 1))
    return prefix, [0] + cuts + [end]


def _lists(case, seed):
    """Page lists of the requests, then of the prefixes, each (CSR offsets, ids);
    tokens in each page; pages that lists name.  Pages lie scattered over the cache,
    as one that has served for a while hands them out."""
    held, _ = _lengths(case)
    prefix = _groups(case)[0] if case["kind"] == "shared" else []
    ps, rng = case["page"], np.random.RandomState(seed % (1 << 31))
    counts = [_ceil(c, ps) for c in held + prefix]
    used = sum(counts)
    order = rng.permutation(used).astype(np.int32)
    tokens = np.full(used, ps, np.int32)
    ends = np.concatenate([[0], np.cumsum(counts)])
    for c, a, b in zip(held + prefix, ends[:-1], ends[1:]):
        if b > a:
            tokens[order[b - 1]] = c - (b - a - 1) * ps
    B = case["batch"]
    own_lists = (ends[:B + 1].astype(np.int32), order[:ends[B]])
    prefixes = ((ends[B:] - ends[B]).astype(np.int32), order[ends[B]:])
    return own_lists, prefixes, tokens


def _normal(seed, salt, *shape):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 16 + salt)
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _codes(case, seed, salt, out):
    """Codes of N(0, 1) rows whose largest reaches the format's largest value."""
    flat = out.view(-1)
    step, most = 1 << 28, _LARGEST[case["format"]]
    for i in range(0, flat.numel(), step):
        x = _normal(seed + i // step, salt, min(step, flat.numel() - i))
        flat[i:i + step] = _to_codes(case, (x * (most / 4)).clamp_(-most, most))


def _to_codes(case, x):
    """The nearest codes of x (within the format's range), as bytes, rounded once."""
    if case["format"] == "int8":
        return x.round().to(torch.int8).view(torch.uint8)
    step = torch.exp2((torch.frexp(x).exponent - 1).clamp(min=-6).to(x.dtype) - 3)
    return ((x / step).round() * step).float().to(torch.float8_e4m3fn).view(torch.uint8)


def _kind(case):
    return torch.int8 if case["format"] == "int8" else torch.float8_e4m3fn


def _of_codes(case, codes):
    """The numbers that bytes stand for."""
    return codes.view(_kind(case)).float()


def _scales(case, rng, pages):
    """Scales of pages whose largest numbers differ from page to page and head to head."""
    most = rng.uniform(2, 6, (pages, case["kv_heads"])).astype(np.float32)
    if case["format"] == "int8":
        return (most.astype(np.float64) / 127).astype(np.float32)
    fraction, exponent = np.frexp(most)
    return np.ldexp(np.float32(1), exponent - 9 + (fraction > 0.875)).astype(np.float32)


def _device(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def prepare(case, seed):
    held, new = _lengths(case)
    H, K, D, ps, B = case["heads"], case["kv_heads"], case["dim"], case["page"], case["batch"]
    (offsets, ids), (pre_offsets, pre_ids), tokens = _lists(case, seed)
    used = len(tokens)
    # an eviction's new pages lie behind the lists' ones
    room = _ceil(case["keep"], ps) if case["kind"] == "evict" else 0
    capacity = used + B * room
    rng = np.random.RandomState(seed % (1 << 31) + 1)
    keys = torch.zeros(capacity, K, ps, D, dtype=torch.uint8, device="cuda")
    values = torch.zeros(capacity, K, ps // 16, D, 16, dtype=torch.uint8, device="cuda")
    _codes(case, seed, 1, keys[:used])
    _codes(case, seed, 2, values[:used])
    counts = np.zeros(capacity, np.int32)
    counts[:used] = tokens
    state = {
        "case": case, "keys": keys, "values": values, "token_counts": _device(counts),
        "key_scales": _device(_scales(case, rng, capacity)),
        "value_scales": _device(_scales(case, rng, capacity)),
        "page_offsets": _device(offsets), "page_ids": _device(ids if len(ids) else np.zeros(1, np.int32)),
        "total_pages": len(ids), "used": used, "most_pages": int(np.diff(offsets).max()),
    }
    if case["kind"] == "evict":
        state["summaries"] = torch.zeros(capacity, K * D, device="cuda")
        # sums of many steps' weights: most tokens next to nothing, a few a lot, and
        # some that no step has looked at
        w = torch.exp(2 * _normal(seed, 4, capacity, K, ps))
        w[_normal(seed, 5, capacity, K, ps) > 1.5] = 0.0
        state["weights"] = w
        state["new_ids"] = _device(used + rng.permutation(B * room).astype(np.int32).reshape(B, room))
        state["new_counts"] = torch.zeros(B, dtype=torch.int32, device="cuda")
        state["kept"] = torch.zeros(B, K, case["keep"], dtype=torch.int32, device="cuda")
    else:
        rows = sum(new) if case["kind"] == "cross" else B
        state["q"] = _normal(seed, 3, rows, H, D).to(_TYPES[case["type"]])
        state["outputs"] = torch.empty_like(state["q"])
        if case["kind"] == "cross":
            state["token_offsets"] = _device(np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
            state["tokens"], state["most_new"] = rows, max(new)
        if case["kind"] == "shared":
            prefix, starts = _groups(case)
            state["starts"] = _device(np.asarray(starts, np.int32))
            state["pre_offsets"], state["pre_ids"] = _device(pre_offsets), _device(pre_ids)
            state["most_requests"] = max(b - a for a, b in zip(starts, starts[1:]))
        if case["kind"] == "weigh":
            # the sums before the step, which a program keeps until the step's token
            # is accepted
            state["before"] = torch.exp(_normal(seed, 4, capacity, K, ps))
            state["weights"] = torch.empty_like(state["before"])
    if own:
        _own_handles(case, state)
    return state


def _own_handles(case, state):
    """What a program that uses the package keeps beside its tensors: the cache's
    handle over them, the batch's description and a workspace."""
    dsd = importlib.import_module("15-618_dynamic_sparse_decode_amd")
    names = ("keys", "values", "key_scales", "value_scales", "token_counts") + (
        ("summaries",) if case["kind"] == "evict" else ())
    cache = dsd.Kv8Cache(case["kv_heads"], case["dim"], case["page"], len(state["token_counts"]),
                         {"e4m3": dsd.KV8_E4M3, "int8": dsd.KV8_INT8}[case["format"]],
                         arrays={n: state[n].data_ptr() for n in names})
    state["type"] = {"f32": dsd.TYPE_F32, "bf16": dsd.TYPE_BF16, "f16": dsd.TYPE_F16}[case["type"]]
    state["cache"] = cache
    more = {}
    if case["kind"] == "cross":
        more = {"tokens": state["tokens"], "max_tokens": state["most_new"],
                "token_offsets": state["token_offsets"].data_ptr()}
    state["batch"] = dsd.Kv8Batch(
        case["batch"], max_pages=state["most_pages"], total_pages=state["total_pages"],
        page_offsets=state["page_offsets"].data_ptr(), page_ids=state["page_ids"].data_ptr(), **more)
    if case["kind"] == "shared":
        state["prefix"] = dsd.Kv8Prefix(
            case["groups"], max_requests=state["most_requests"],
            max_pages=int(state["pre_offsets"].diff().max()), total_pages=len(state["pre_ids"]),
            request_offsets=state["starts"].data_ptr(), page_offsets=state["pre_offsets"].data_ptr(),
            page_ids=state["pre_ids"].data_ptr())
        size = cache.shared_workspace_bytes(state["batch"], state["prefix"], case["heads"])
    elif case["kind"] == "weigh":
        size = cache.weigh_workspace_bytes(state["batch"], case["heads"])
    elif case["kind"] == "evict":
        size = cache.evict_workspace_bytes(state["batch"], case["keep"])
    else:
        size = cache.workspace_bytes(state["batch"], case["heads"])
    state["workspace"] = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    state["workspace_bytes"] = size


def run(state):
    kind = state["case"]["kind"]
    return (_OWN if own else _PLAIN)[kind](state)


# ---- the package's calls -----------------------------------------------------------

def _space(state):
    return {"workspace": state["workspace"].data_ptr(), "workspace_bytes": state["workspace_bytes"],
            "stream": torch.cuda.current_stream().cuda_stream}


def _rows_of(state):
    q, out = state["q"], state["outputs"]
    return (state["type"], state["case"]["heads"], q.data_ptr(), q.stride(0), out.data_ptr(),
            out.stride(0))


def _own_cross(state):
    state["cache"].attend_cross(state["batch"], *_rows_of(state), **_space(state))
    return {"outputs": state["outputs"]}


def _own_shared(state):
    state["cache"].attend_shared(state["batch"], state["prefix"], *_rows_of(state), **_space(state))
    return {"outputs": state["outputs"]}


def _own_weigh(state):
    state["weights"].copy_(state["before"])
    state["cache"].attend_weigh(state["batch"], *_rows_of(state),
                                weights=state["weights"].data_ptr(), **_space(state))
    return {"outputs": state["outputs"], "weights": state["weights"]}


def _evicted(state):
    """What an eviction writes: the new pages' codes as the numbers that they stand
    for, in units of their scale, and all that goes with them."""
    case, used = state["case"], state["used"]
    return {"keys": state["keys"][used:].view(_kind(case)),
            "values": state["values"][used:].view(_kind(case)),
            "key_scales": state["key_scales"][used:], "value_scales": state["value_scales"][used:],
            "summaries": state["summaries"][used:], "token_counts": state["token_counts"][used:],
            "weights": state["weights"][used:], "new_counts": state["new_counts"],
            "kept": state["kept"]}


def _own_evict(state):
    case = state["case"]
    state["cache"].evict(
        state["batch"], case["keep"], case["first"], case["recent"], state["weights"].data_ptr(),
        state["new_ids"].data_ptr(), state["new_ids"].stride(0), state["new_counts"].data_ptr(),
        state["kept"].data_ptr(), **_space(state))
    return _evicted(state)


_OWN = {"cross": _own_cross, "shared": _own_shared, "weigh": _own_weigh, "evict": _own_evict}


# ---- the plain forms ---------------------------------------------------------------

def _padded(state, offsets, ids, most):
    """Lists padded to the longest: (page ids, listed, token valid), [lists][most],
    [lists][most] and [lists][most * page]."""
    ps = state["case"]["page"]
    at = offsets[:-1].long().unsqueeze(-1) + torch.arange(most, device="cuda")
    there = at < offsets[1:].unsqueeze(-1)
    pages = ids[torch.where(there, at, 0)].long()
    held = torch.where(there, state["token_counts"][pages], 0)
    valid = torch.arange(ps, device="cuda") < held.unsqueeze(-1)
    return pages, there, valid.view(len(pages), most * ps)


def _rows(state, pages):
    """(keys, values) [lists][kv heads][tokens][dim] of padded lists."""
    case = state["case"]
    K, D, ps = case["kv_heads"], case["dim"], case["page"]
    B, n = pages.shape
    keys = _of_codes(case, state["keys"][pages]) * state["key_scales"][pages].view(B, n, K, 1, 1)
    values = _of_codes(case, state["values"][pages]) * state["value_scales"][pages].view(B, n, K, 1, 1, 1)
    return (keys.transpose(1, 2).reshape(B, K, n * ps, D),
            values.permute(0, 2, 1, 3, 5, 4).reshape(B, K, n * ps, D))


def _logits(q, keys, valid):
    """q K^T / sqrt(dim) where a token is valid, in 32 bits."""
    s = torch.matmul(q * (1.0 / math.sqrt(q.shape[-1])), keys.transpose(-1, -2).contiguous())
    return s.masked_fill_(~valid, -math.inf)


def _weights(s, most):
    """exp(s - most) in place; zeros where there is no token."""
    return s.sub_(torch.where(most == -math.inf, 0.0, most)).exp_()


def _plain_cross(state):
    case = state["case"]
    B, H, K, D, n = case["batch"], case["heads"], case["kv_heads"], case["dim"], state["most_new"]
    at = torch.arange(state["tokens"], device="cuda")
    request = torch.bucketize(at, state["token_offsets"][1:].long(), right=True)
    place = at - state["token_offsets"][request]
    q = torch.zeros(B, n, H, D, device="cuda")
    q[request, place] = state["q"].float()
    q = q.view(B, n, K, H // K, D).permute(0, 2, 3, 1, 4).reshape(B, K, H // K * n, D)
    pages, _, valid = _padded(state, state["page_offsets"], state["page_ids"], state["most_pages"])
    keys, values = _rows(state, pages)
    s = _logits(q, keys, valid.view(B, 1, 1, -1))
    p = _weights(s, s.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, values) / torch.where(valid.any(-1).view(B, 1, 1, 1), total, 1.0)
    out = out.view(B, K, H // K, n, D).permute(0, 3, 1, 2, 4).reshape(B, n, H, D)
    state["outputs"].copy_(out[request, place])
    return {"outputs": state["outputs"]}


def _plain_shared(state):
    case = state["case"]
    B, H, K, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    q = state["q"].float().view(B, K, H // K, D)
    pages, _, valid = _padded(state, state["page_offsets"], state["page_ids"], state["most_pages"])
    keys, values = _rows(state, pages)
    own_s = _logits(q, keys, valid.view(B, 1, 1, -1))
    most = own_s.amax(-1, keepdim=True)
    starts, ends = state["starts"].tolist(), state["pre_offsets"].tolist()
    parts = []
    for g in range(case["groups"]):
        a, b = starts[g], starts[g + 1]
        if b == a or ends[g + 1] == ends[g]:
            continue
        listed_ = state["pre_ids"][ends[g]:ends[g + 1]].long().unsqueeze(0)
        there = torch.arange(case["page"], device="cuda") < state["token_counts"][listed_].unsqueeze(-1)
        pre_k, pre_v = _rows(state, listed_)
        rows = q[a:b].transpose(0, 1).reshape(1, K, (b - a) * (H // K), D)
        s = _logits(rows, pre_k, there.view(1, 1, 1, -1))
        s = s.view(K, b - a, H // K, -1).transpose(0, 1)
        most[a:b] = torch.maximum(most[a:b], s.amax(-1, keepdim=True))
        parts.append((a, b, s, pre_v[0]))
    p = _weights(own_s, most)
    total, out = p.sum(-1, keepdim=True), torch.matmul(p, values)
    for a, b, s, pre_v in parts:
        p = _weights(s, most[a:b])
        total[a:b] += p.sum(-1, keepdim=True)
        n = b - a
        add = torch.matmul(p.transpose(0, 1).reshape(K, n * (H // K), -1), pre_v)
        out[a:b] += add.view(K, n, H // K, D).transpose(0, 1)
    state["outputs"].copy_((out / torch.where(total > 0, total, 1.0)).view(B, H, D))
    return {"outputs": state["outputs"]}


def _plain_weigh(state):
    case = state["case"]
    B, H, K, D, ps = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    state["weights"].copy_(state["before"])
    q = state["q"].float().view(B, K, H // K, D)
    pages, there, valid = _padded(state, state["page_offsets"], state["page_ids"], state["most_pages"])
    keys, values = _rows(state, pages)
    s = _logits(q, keys, valid.view(B, 1, 1, -1))
    p = _weights(s, s.amax(-1, keepdim=True))
    p /= torch.where(valid.any(-1).view(B, 1, 1, 1), p.sum(-1, keepdim=True), 1.0)
    state["outputs"].copy_(torch.matmul(p, values).view(B, H, D))
    add = p.sum(2).view(B, K, -1, ps).transpose(1, 2)  # [lists][pages][kv heads][page]
    state["weights"][pages[there]] += add[there]
    return {"outputs": state["outputs"], "weights": state["weights"]}


def _plain_evict(state):
    case = state["case"]
    B, K, D, ps, keep = case["batch"], case["kv_heads"], case["dim"], case["page"], case["keep"]
    pages, _, valid = _padded(state, state["page_offsets"], state["page_ids"], state["most_pages"])
    T = valid.shape[1]
    held = valid.sum(-1, keepdim=True)
    rank = valid.cumsum(-1) - 1
    always = valid & ((rank < case["first"]) | (rank >= held - case["recent"]))
    w = state["weights"][pages].permute(0, 2, 1, 3).reshape(B, K, T).clone()
    w.masked_fill_(always.unsqueeze(1), math.inf).masked_fill_(~valid.unsqueeze(1), -math.inf)
    place = w.sort(dim=-1, descending=True, stable=True)[1][..., :keep]
    if place.shape[-1] < keep:
        place = torch.cat([place, place.new_full((B, K, keep - place.shape[-1]), T)], -1)
    count = held.clamp(max=keep)
    there = (torch.arange(keep, device="cuda") < count).unsqueeze(1).expand(B, K, keep)
    place = torch.where(there, place, T).sort(-1)[0]
    state["kept"].copy_(torch.where(there, place, -1))
    n = state["new_ids"].shape[1]
    full = torch.full((B, K, n * ps), T, device="cuda")
    full[..., :keep] = place
    there = full < T
    full = torch.where(there, full, 0)
    page = pages.unsqueeze(1).expand(B, K, -1).gather(-1, full // ps)
    head, slot = torch.arange(K, device="cuda").view(1, K, 1), full % ps
    new = state["new_ids"].long()
    counts = (count - torch.arange(n, device="cuda") * ps).clamp(0, ps)
    live = counts > 0
    w = torch.where(there, state["weights"][page, head, slot], 0.0).view(B, K, n, ps)
    state["weights"][new[live]] = w.transpose(1, 2)[live]
    state["token_counts"][new[live]] = counts[live].int()
    state["new_counts"].copy_(live.sum(-1))
    for name, scales in (("keys", "key_scales"), ("values", "value_scales")):
        if name == "keys":
            codes = state["keys"][page, head, slot]
        else:
            codes = state["values"][page, head, slot // 16, :, slot % 16]
        x = _of_codes(case, codes).double() * state[scales][page, head].double().unsqueeze(-1)
        x = torch.where(there.unsqueeze(-1), x, 0.0).view(B, K, n, ps, D)
        most = x.abs().amax((-1, -2))
        if case["format"] == "int8":
            scale = (most / 127).float().clamp(min=_TINY)
        else:
            fraction, exponent = torch.frexp(most)
            power = torch.where(most > 0, exponent - 9 + (fraction > 0.875), -126).clamp(min=-126)
            scale = ((power + 127) << 23).int().view(torch.float32)
        codes = _to_codes(case, x / scale.double().view(B, K, n, 1, 1)).transpose(1, 2)
        scale = scale.transpose(1, 2)
        state[scales][new[live]] = scale[live]
        if name == "keys":
            mean = _of_codes(case, codes).sum(-2) * scale.unsqueeze(-1) / counts.clamp(min=1).view(B, n, 1, 1)
            state["summaries"][new[live]] = mean[live].view(-1, K * D)
        else:
            codes = codes.reshape(B, n, K, ps // 16, 16, D).transpose(-1, -2)
        state[name][new[live]] = codes[live]
    return _evicted(state)


_PLAIN = {"cross": _plain_cross, "shared": _plain_shared, "weigh": _plain_weigh,
          "evict": _plain_evict}


# ---- what a pass cannot do without -------------------------------------------------

def work(case):
    held, new = _lengths(case)
    H, K, D, ps, B = case["heads"], case["kv_heads"], case["dim"], case["page"], case["batch"]
    size = 4 if case["type"] == "f32" else 2
    tokens, pages, rows, pairs = sum(held), sum(_ceil(c, ps) for c in held), B, sum(held)
    if case["kind"] == "evict":
        kept = sum(min(c, case["keep"]) for c in held)
        new_pages = sum(_ceil(min(c, case["keep"]), ps) for c in held)
        # every weight; the kept codes, weights and places; the new pages' scales, means
        moved = 4 * K * tokens + kept * K * (4 * D + 8)
        moved += new_pages * (K * (8 + 4 * D) + 4) + pages * (8 * K + 8)
        return {"bytes": moved, "flops": kept * K * 8 * D}
    if case["kind"] == "cross":
        rows, pairs = sum(new), sum(c * n for c, n in zip(held, new))
    more = 0
    if case["kind"] == "weigh":
        more = 8 * K * tokens
    if case["kind"] == "shared":
        prefix, starts = _groups(case)
        for c, a, b in zip(prefix, starts, starts[1:]):
            if b > a:
                tokens += c
                pages += _ceil(c, ps)
                pairs += c * (b - a)
    moved = 2 * tokens * K * D + pages * (8 * K + 8) + 2 * rows * H * D * size + more
    return {"bytes": moved, "flops": 4 * pairs * H * D}


# ---- the same from the definition, in 64 bits --------------------------------------

def _places(state, ids):
    """Where the tokens of a list of pages are: (page, offset in it) of each."""
    ids = ids.long()
    counts = state["token_counts"][ids].long()
    page = ids.repeat_interleave(counts)
    begin = counts.cumsum(0) - counts
    return page, torch.arange(len(page), device="cuda") - begin.repeat_interleave(counts)


def _numbers(case, codes):
    """The numbers that bytes stand for, from the format's own rule, in 64 bits."""
    code = torch.arange(256, dtype=torch.float64, device="cuda")
    if case["format"] == "int8":
        table = torch.where(code > 127, code - 256, code)
    else:
        low = code % 128
        exponent, fraction = torch.div(low, 8, rounding_mode="floor"), low % 8
        table = torch.where(exponent == 0, fraction / 512, (8 + fraction) * torch.exp2(exponent - 10))
        table = torch.where(code > 127, -table, table)
    return table[codes.long()]


def _tokens(state, head, page, offset):
    """One head's keys and values of tokens, [tokens][dim], 64 bits."""
    case = state["case"]
    k = _numbers(case, state["keys"][page, head, offset]) * state["key_scales"][page, head].double()[:, None]
    v = _numbers(case, state["values"][page, head, offset // 16, :, offset % 16])
    return k, v * state["value_scales"][page, head].double()[:, None]


def _exact_attention(case, seed):
    state = prepare(case, seed)
    H, K, D, G = case["heads"], case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"]
    q = state["q"].double().view(-1, K, G, D) / math.sqrt(D)
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    ends = state["page_offsets"].tolist()
    group = [-1] * case["batch"]
    if case["kind"] == "shared":
        starts, pre = state["starts"].tolist(), state["pre_offsets"].tolist()
        for g in range(case["groups"]):
            group[starts[g]:starts[g + 1]] = [g] * (starts[g + 1] - starts[g])
    sums = state["before"].double().clone() if case["kind"] == "weigh" else None
    at = state["token_offsets"].tolist() if case["kind"] == "cross" else list(range(case["batch"] + 1))
    for r in range(case["batch"]):
        ids = state["page_ids"][ends[r]:ends[r + 1]]
        if group[r] >= 0:
            ids = torch.cat([state["pre_ids"][pre[group[r]]:pre[group[r] + 1]], ids])
        page, offset = _places(state, ids)
        if not len(page):
            continue
        for head in range(K):
            k, v = _tokens(state, head, page, offset)
            rows = q[at[r]:at[r + 1], head].reshape(-1, D)
            blocks = []
            for i in range(0, len(rows), 4096):
                p = torch.softmax(rows[i:i + 4096] @ k.t(), -1)
                blocks.append(p @ v)
                if sums is not None:
                    sums[page, head, offset] += p.sum(0)
            out[at[r]:at[r + 1], head] = torch.cat(blocks).view(-1, G, D)
    got = {"outputs": out.view(-1, H, D)}
    if sums is not None:
        got["weights"] = sums
    return got


def _nearest(case, x):
    """The format's value next to x, halves to the even code."""
    if case["format"] == "int8":
        return x.round().clamp(-127, 127)
    size = x.abs().clamp(min=2.0 ** -9)
    step = torch.exp2(torch.log2(size).floor().clamp(min=-6) - 3)
    step = torch.where(size >= 16 * step, 2 * step, step)  # (a logarithm that was rounded up or down)
    step = torch.where((size < 8 * step) & (step > 2.0 ** -9), step / 2, step)
    return (x / step).round() * step


def _exact_evict(case, seed):
    state = prepare(case, seed)
    B, K, D, ps, keep = case["batch"], case["kv_heads"], case["dim"], case["page"], case["keep"]
    n = state["new_ids"].shape[1]
    cap = B * n
    like = {"dtype": torch.float64, "device": "cuda"}
    keys, values = torch.zeros(cap, K, ps, D, **like), torch.zeros(cap, K, ps // 16, D, 16, **like)
    scales = [state[s][state["used"]:].double().clone() for s in ("key_scales", "value_scales")]
    summaries = torch.zeros(cap, K * D, **like)
    weights = state["weights"][state["used"]:].double().clone()
    counts = torch.zeros(cap, dtype=torch.int32)
    kept = torch.full((B, K, keep), -1, dtype=torch.int32)
    new_counts = torch.zeros(B, dtype=torch.int32)
    ends, new_ids = state["page_offsets"].tolist(), (state["new_ids"] - state["used"]).tolist()
    for r in range(B):
        ids = state["page_ids"][ends[r]:ends[r + 1]]
        page, offset = _places(state, ids)
        held, count = len(page), min(len(page), keep)
        new_counts[r] = _ceil(count, ps)
        weights[new_ids[r][:_ceil(count, ps)]] = 0.0
        for i in range(_ceil(count, ps)):
            counts[new_ids[r][i]] = min(count - i * ps, ps)
        for head in range(K):
            w = state["weights"][page, head, offset].cpu().numpy()
            order = np.arange(held)
            inside = order[min(case["first"], held):max(held - case["recent"], min(case["first"], held))]
            must = np.setdiff1d(order, inside, assume_unique=True)[:count]
            best = inside[np.lexsort((inside, -w[inside]))][:count - len(must)]
            chosen = torch.from_numpy(np.sort(np.concatenate([must, best])).astype(np.int64))
            kept[r, head, :count] = chosen.int()
            chosen = chosen.cuda()
            rows = _tokens(state, head, page[chosen], offset[chosen])
            for i in range(_ceil(count, ps)):
                at, m = new_ids[r][i], min(count - i * ps, ps)
                weights[at, head, :m] = state["weights"][page[chosen], head, offset[chosen]][i * ps:i * ps + m].double()
            for side in range(2):
                x = torch.zeros(_ceil(count, ps) * ps, D, **like)
                x[:count] = rows[side]
                x = x.view(-1, ps, D)
                most = x.abs().amax((1, 2))
                if case["format"] == "int8":
                    s = (most / 127).float().double().clamp(min=_TINY)
                else:
                    s = torch.exp2(torch.ceil(torch.log2(most.clamp(min=2.0 ** -120) / 448)))
                    s = torch.where(most > 448 * s, 2 * s, torch.where(most <= 224 * s, s / 2, s))
                    s = torch.where(most > 0, s, _TINY)
                code = _nearest(case, x / s[:, None, None])
                at = torch.tensor(new_ids[r][:len(s)], device="cuda", dtype=torch.long)
                scales[side][at, head] = s
                if side == 0:
                    keys[at, head] = code
                    m = torch.tensor([min(count - i * ps, ps) for i in range(len(s))], **like)
                    summaries.view(cap, K, D)[at, head] = code.sum(1) * s[:, None] / m[:, None]
                else:
                    values[at, head] = code.view(-1, ps // 16, 16, D).transpose(-1, -2)
    if case["format"] == "int8":
        keys, values = keys.to(torch.int8), values.to(torch.int8)
    return {"keys": keys, "values": values, "key_scales": scales[0], "value_scales": scales[1],
            "summaries": summaries, "token_counts": counts, "weights": weights,
            "new_counts": new_counts, "kept": kept}


def exact(case, seed):
    if case["kind"] == "evict":
        return _exact_evict(case, seed)
    return _exact_attention(case, seed)
