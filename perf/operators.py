"""The calls that the speed of the serving operators is measured on.

Four operators that belong together: attention of prompts with a sliding window
and first tokens that stay visible (`window_attention`), attention of new
tokens over a paged key-value cache (`paged_attention`), the writing of new
keys and values into the cache's pages (`cache_write`), and the copying of
whole pages that a fork or a compaction needs (`copy_pages`).

`run` computes them in elementary torch operations in fp32, rounded once at the
end, or, where `own` is true, through the library's entry points. All of them
are forward only, as the library is. Types: bf16, fp16 and fp32.

The visibility rule of both attentions, for a query at position p and a key at
position j of a sequence of `length` tokens: j < length, j <= p, and, with a
window, p - j < window or j < sinks.
"""

from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def _library():
    # The package directory is not a Python identifier; the working folder is
    # the repository's root.
    path = os.path.join(os.getcwd(), "dnn-flash_amd", "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    import onednn_flash_hip as F
    return F


# --- cases -----------------------------------------------------------------

def _window(dtype, batch, heads, kv_heads, tokens, dim, window, sinks, shortest=0, softcap=0.0):
    """A prompt batch of `tokens` padded rows; with `shortest` the sequences have
    lengths from there to `tokens`, else all are full."""
    return {"op": "window", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "tokens": tokens,
            "dim": dim, "window": window, "sinks": sinks, "shortest": shortest, "softcap": softcap}


def _paged(dtype, batch, heads, kv_heads, shortest, longest, dim, page, new=1, window=0, sinks=0, softcap=0.0):
    """`new` tokens for each of `batch` sequences of `shortest` to `longest` tokens."""
    return {"op": "paged", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "shortest": shortest, "longest": longest, "dim": dim, "page": page, "new": new, "window": window,
            "sinks": sinks, "softcap": softcap}


def _write(dtype, batch, kv_heads, shortest, longest, dim, page, new, fewest=0):
    """`new` padded rows per sequence, of which `fewest` to `new` are tokens (all
    of them with 0); the sequences then have `shortest` to `longest` tokens."""
    return {"op": "write", "dtype": dtype, "batch": batch, "kv_heads": kv_heads, "shortest": shortest,
            "longest": longest, "dim": dim, "page": page, "new": new, "fewest": fewest}


def _copy(dtype, kv_heads, dim, page, pages, moved, layers):
    """`moved` of a pool's `pages` pages, in the K and V pools of `layers` layers."""
    return {"op": "copy", "dtype": dtype, "kv_heads": kv_heads, "dim": dim, "page": page, "pages": pages,
            "moved": moved, "layers": layers}


def listed():
    cases = {
        # A chat turn of a small model: one short prompt. Latency counts.
        "prompt_short": _window("bf16", 1, 8, 2, 200, 64, 128, 4),
        # A padded batch of prompts of ordinary length, grouped heads.
        "prompt_batch": _window("bf16", 4, 32, 8, 2048, 128, 1024, 4, shortest=300),
        # The library's block-sparse workload (one long document, a window of
        # 1024 tokens and 256 first ones), by tokens.
        "prompt_long": _window("f16", 1, 16, 16, 16384, 64, 1024, 256),
        # An fp32 encoder-decoder's prompt at the library's ordinary fp32 sizes.
        "prompt_f32": _window("f32", 2, 8, 8, 2047, 64, 512, 16, shortest=1000),
        # The smallest step: one user, one new token, about a thousand cached.
        "decode_one": _paged("bf16", 1, 32, 8, 1001, 1001, 128, 16),
        # A serving batch of sequences of all ages.
        "decode_batch": _paged("bf16", 64, 32, 8, 65, 4096, 128, 16),
        # One very long document: the split over the cache's length carries it.
        "decode_long": _paged("f16", 1, 32, 8, 131000, 131000, 128, 64),
        # Draft tokens checked together, fp32, window and sinks: a bounded read
        # of caches that may be long.
        "decode_window": _paged("f32", 16, 16, 8, 700, 8192, 64, 32, new=3, window=1024, sinks=64),
        # Every decode step writes one row per sequence.
        "write_step": _write("bf16", 64, 8, 33, 1024, 128, 16, 1),
        # A batch of prompts goes into the cache.
        "write_prompts": _write("f16", 8, 8, 1000, 2048, 128, 16, 2048, fewest=700),
        # A few forked sequences take copies of their last, shared page.
        "fork": _copy("bf16", 8, 128, 16, 1024, 5, 4),
        # A pool compacted after many sequences ended.
        "compact": _copy("bf16", 8, 128, 16, 4096, 1700, 2),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _log(rng, low, high):
    """A whole number spread over [low, high] by its logarithm."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["window", "window", "paged", "paged", "paged", "write", "copy"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    page = rng.choice([16, 32, 64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 192, 256])
    window = rng.choice([0, _log(rng, 16, 4096), _log(rng, 16, 4096)])
    sinks = rng.choice([0, _log(rng, 1, 256)]) if window else 0
    softcap = rng.choice([0.0, 0.0, 0.0, 30.0])
    if op == "window":
        tokens = _log(rng, 1, 8192)
        # at most what the long listed prompt costs
        batch = _log(rng, 1, max(1, min(8, (1 << 31) // (heads * dim * tokens * min(tokens, 2048)))))
        if heads * dim * tokens * tokens > 1 << 37:
            tokens = int(math.sqrt((1 << 37) / (heads * dim)))
        if dtype == "f32":
            tokens = min(tokens, 2048)
        shortest = rng.choice([0, rng.randint(1, tokens)])
        return _window(dtype, batch, heads, kv_heads, tokens, dim, window, sinks, shortest, softcap)
    if op == "paged":
        longest = _log(rng, 1, 65536)
        # at most what the long listed cache holds
        batch = _log(rng, 1, max(1, min(128, (1 << 27) // (kv_heads * dim * longest))))
        shortest = rng.randint(1, longest)
        new = rng.choice([1, 1, rng.randint(2, 8)])
        return _paged(dtype, batch, heads, kv_heads, shortest, longest, dim, page, new, window, sinks, softcap)
    if op == "write":
        new = rng.choice([1, _log(rng, 1, 2048)])
        longest = new + _log(rng, 1, 1024)
        batch = _log(rng, 1, max(1, min(128, (1 << 24) // (kv_heads * dim * longest))))
        fewest = rng.choice([0, rng.randint(1, new)])
        return _write(dtype, batch, kv_heads, rng.randint(new, longest), longest, dim, page, new, fewest)
    pages = _log(rng, 16, max(16, min(4096, (1 << 26) // (kv_heads * dim * page))))
    return _copy(dtype, kv_heads, dim, page, pages, rng.randint(1, pages // 2), rng.randint(1, 4))


def _spread(low, high, count):
    """`count` whole numbers from low to high in no order, the last one high."""
    golden = (math.sqrt(5.0) - 1.0) / 2.0
    return [low + int((high - low) * ((i + 1) * golden % 1.0)) for i in range(count - 1)] + [high]


def _lengths(case):
    if case["op"] == "window":
        low = case["shortest"] or case["tokens"]
        return _spread(low, case["tokens"], case["batch"])
    return _spread(case["shortest"], case["longest"], case["batch"])


def _counts(case):
    return _spread(case["fewest"] or case["new"], case["new"], case["batch"])


def _visible(position, length, window, sinks):
    """Keys that a query at `position` sees."""
    last = min(position + 1, length)
    if last <= 0:
        return 0
    if not window:
        return last
    first = max(0, position + 1 - window)
    return max(0, last - first) + min(sinks, first, last)


def _read(first_position, last_position, length, window, sinks):
    """Keys that queries at these positions see together."""
    last = min(last_position + 1, length)
    if last <= 0:
        return 0
    if not window:
        return last
    first = max(0, first_position + 1 - window)
    return max(0, last - first) + min(sinks, first, last)


def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] == "copy":
        page = case["kv_heads"] * case["page"] * case["dim"] * size
        return {"bytes": 2 * 2 * case["layers"] * case["moved"] * page, "flops": 0}
    if case["op"] == "write":
        row = case["kv_heads"] * case["dim"] * size
        return {"bytes": 2 * 2 * sum(_counts(case)) * row + 8 * case["batch"], "flops": 0}
    pairs, keys, rows = 0, 0, 0
    for length in _lengths(case):
        if case["op"] == "window":
            first, last = 0, length - 1
        else:
            first, last = max(0, length - case["new"]), length - 1
        pairs += sum(_visible(p, length, case["window"], case["sinks"]) for p in range(first, last + 1))
        keys += _read(first, last, length, case["window"], case["sinks"])
        rows += case["tokens"] if case["op"] == "window" else case["new"]
    row = case["dim"] * size
    return {"bytes": 2 * row * (keys * case["kv_heads"] + rows * case["heads"]),
            "flops": 4 * case["dim"] * pairs * case["heads"]}


# --- inputs ----------------------------------------------------------------

def _normal(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(DTYPES[dtype])


def _token_major(gen, batch, heads, tokens, dim, dtype):
    """[B, H, T, D] over the [B, T, H, D] storage that a projection makes."""
    return _normal(gen, (batch, tokens, heads, dim), dtype).transpose(1, 2)


def _pages_of(case, lengths):
    """Pages that hold the sequences, and a table row's width."""
    per = [-(-n // case["page"]) for n in lengths]
    return sum(per), max(per)


def _table(case, lengths, pages, seed):
    """The page table of a pool that has been in use for long: pages in no order.
    Entries past a sequence's end are -1."""
    used, width = _pages_of(case, lengths)
    order = np.random.default_rng(seed).permutation(pages)[:used].astype(np.int32)
    table = np.full((len(lengths), width), -1, np.int32)
    at = 0
    for row, n in enumerate(lengths):
        per = -(-n // case["page"])
        table[row, :per] = order[at:at + per]
        at += per
    return table


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    dtype, dim = case["dtype"], case["dim"]
    if case["op"] == "window":
        state["q"] = _token_major(gen, case["batch"], case["heads"], case["tokens"], dim, dtype)
        state["k"] = _token_major(gen, case["batch"], case["kv_heads"], case["tokens"], dim, dtype)
        state["v"] = _token_major(gen, case["batch"], case["kv_heads"], case["tokens"], dim, dtype)
        state["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32).cuda() if case["shortest"] else None
        return state
    if case["op"] == "copy":
        shape = (case["pages"], case["kv_heads"], case["page"], dim)
        state["pools"] = [_normal(gen, shape, dtype) for _ in range(2 * case["layers"])]
        order = np.random.default_rng(seed).permutation(case["pages"])[:2 * case["moved"]].astype(np.int32)
        # the bookkeeping that decides on moves runs on the host
        state["src"], state["dst"] = (torch.from_numpy(part.copy()) for part in np.split(order, 2))
        state["src_gpu"], state["dst_gpu"] = state["src"].cuda(), state["dst"].cuda()
        return state
    lengths = _lengths(case)
    used, _ = _pages_of(case, lengths)
    pages = used + used // 4 + 1
    shape = (pages, case["kv_heads"], case["page"], dim)
    state["k_pages"], state["v_pages"] = _normal(gen, shape, dtype), _normal(gen, shape, dtype)
    state["table"] = torch.from_numpy(_table(case, lengths, pages, seed)).cuda()
    state["lengths"] = torch.tensor(lengths, dtype=torch.int32).cuda()
    if case["op"] == "write":
        state["k"] = _token_major(gen, case["batch"], case["kv_heads"], case["new"], dim, dtype)
        state["v"] = _token_major(gen, case["batch"], case["kv_heads"], case["new"], dim, dtype)
        state["counts"] = torch.tensor(_counts(case), dtype=torch.int32).cuda() if case["fewest"] else None
        if own:
            # the cache's tensors live as long as the program, and so does this
            state["writer"] = _library().CacheWriter(state["k_pages"], state["v_pages"], state["table"],
                                                     state["lengths"], counts=state["counts"])
        return state
    state["q"] = _token_major(gen, case["batch"], case["heads"], case["new"], dim, dtype)
    if own:
        state["attend"] = _library().PagedAttention(
            state["k_pages"], state["v_pages"], state["table"], state["lengths"], heads=case["heads"],
            query_tokens=case["new"], window=case["window"], sink_tokens=case["sinks"], softcap=case["softcap"])
    return state


# --- the plain forms --------------------------------------------------------

def _attend_plain(q, k, v, first_position, length, case):
    """q [Hkv, G, M, D] at positions first_position, ... against k, v [Hkv, N, D];
    positions and length are one-element tensors or numbers. fp32."""
    scores = torch.matmul(q, k.transpose(1, 2).contiguous()[:, None]) * (1.0 / math.sqrt(q.shape[-1]))
    if case["softcap"]:
        scores = case["softcap"] * torch.tanh(scores / case["softcap"])
    position = (torch.arange(q.shape[2], device=q.device) + first_position)[:, None]
    key = torch.arange(k.shape[1], device=q.device)[None, :]
    seen = (key <= position) & (key < length)
    if case["window"]:
        seen &= (position - key < case["window"]) | (key < case["sinks"])
    scores = torch.where(seen, scores, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    weight = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, v[:, None])
    return torch.where(total > 0, out / total, torch.zeros_like(out))


def _window_plain(state):
    case, q, k, v = state["case"], state["q"], state["k"], state["v"]
    batch, heads, tokens, dim = q.shape
    group = heads // k.shape[1]
    out = torch.empty((batch, heads, tokens, dim), dtype=q.dtype, device=q.device)
    for b in range(batch):
        length = tokens if state["lengths"] is None else state["lengths"][b]
        for h in range(k.shape[1]):
            part = slice(h * group, (h + 1) * group)
            res = _attend_plain(q[b, part].float()[None], k[b, h].float()[None], v[b, h].float()[None], 0, length, case)
            rows = torch.arange(tokens, device=q.device)[None, :, None]
            out[b, part] = torch.where(rows < length, res[0], torch.zeros_like(res[0])).to(q.dtype)
    return out


def _paged_plain(state):
    case, q = state["case"], state["q"]
    batch, heads, new, dim = q.shape
    kv_heads, page = case["kv_heads"], case["page"]
    table = state["table"].clamp(min=0).long()
    out = torch.empty((batch, heads, new, dim), dtype=q.dtype, device=q.device)
    for b in range(batch):
        k, v = (state[name][table[b]].float().transpose(0, 1).reshape(kv_heads, -1, dim) for name in ("k_pages", "v_pages"))
        rows = q[b].float().reshape(kv_heads, heads // kv_heads, new, dim)
        length = state["lengths"][b]
        out[b] = _attend_plain(rows, k, v, length - new, length, case).reshape(heads, new, dim).to(q.dtype)
    return out


def _write_plain(state):
    case, k, v = state["case"], state["k"], state["v"]
    counts = state["counts"] if state["counts"] is not None else torch.full_like(state["lengths"], case["new"])
    token = torch.arange(case["new"], device=k.device)[None, :]
    position = state["lengths"][:, None] - counts[:, None] + token
    # rows past a sequence's count repeat its last token (which is there: counts are 1 or more)
    token = torch.minimum(token, counts[:, None] - 1)
    position = torch.minimum(position, state["lengths"][:, None] - 1).long()
    page = torch.gather(state["table"].long(), 1, position // case["page"])
    for pool, rows in ((state["k_pages"], k), (state["v_pages"], v)):
        rows = rows.transpose(1, 2)
        rows = torch.gather(rows, 1, token.long()[:, :, None, None].expand(-1, -1, rows.shape[2], rows.shape[3]))
        pool[page, :, position % case["page"]] = rows
    return [state["k_pages"], state["v_pages"]]


def _copy_plain(state):
    for pool in state["pools"]:
        pool[state["dst_gpu"].long()] = pool[state["src_gpu"].long()]
    return state["pools"]


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return {"window": _window_plain, "paged": _paged_plain, "write": _write_plain, "copy": _copy_plain}[op](state)
    if op == "paged":
        return state["attend"](state["q"])
    if op == "write":
        state["writer"](state["k"], state["v"])
        return [state["k_pages"], state["v_pages"]]
    F = _library()
    if op == "copy":
        F.copy_pages(state["pools"], state["src"], state["dst"])
        return state["pools"]
    return F.window_attention(state["q"], state["k"], state["v"], window=case["window"], sink_tokens=case["sinks"],
                              softcap=case["softcap"], lengths=state["lengths"])


# --- the definitions in 64 bits ----------------------------------------------

def _exact_rows(q, k, v, position, length, case):
    """One block of queries q [G, M, D] at `position` (M numbers) against k, v
    [N, D] in 64 bits, over the keys that some of them may see."""
    last = min(int(position[-1]) + 1, length)
    first = max(0, int(position[0]) + 1 - case["window"]) if case["window"] else 0
    sinks = min(case["sinks"], first, max(last, 0))
    index = torch.cat([torch.arange(0, sinks), torch.arange(first, max(first, last))]).to(q.device)
    out = torch.zeros(q.shape[:2] + v.shape[-1:], dtype=torch.float64, device=q.device)
    if index.numel() == 0:
        return out
    x = torch.tensordot(q, k[index], dims=([2], [1])) / math.sqrt(q.shape[-1])
    if case["softcap"]:
        x = torch.tanh(x / case["softcap"]) * case["softcap"]
    at = position.to(q.device)
    hidden = index[None, :] > at[:, None]
    if case["window"]:
        hidden |= (index[None, :] <= at[:, None] - case["window"]) & (index[None, :] >= case["sinks"])
    x = x.masked_fill(hidden[None], float("-inf"))
    some = ~hidden.all(1)
    out[:, some] = torch.tensordot(torch.softmax(x[:, some], -1), v[index], dims=([2], [0]))
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "copy":
        for pool in state["pools"]:
            for s, d in zip(state["src"].tolist(), state["dst"].tolist()):
                pool[d].copy_(pool[s])
        return state["pools"]
    lengths = _lengths(case)
    if case["op"] == "write":
        table = state["table"].cpu().tolist()
        counts = _counts(case)
        for b, (length, count) in enumerate(zip(lengths, counts)):
            start, token = length - count, 0
            while token < count:  # a page at a time
                page, row = divmod(start + token, case["page"])
                n = min(case["page"] - row, count - token)
                for pool, rows in ((state["k_pages"], state["k"]), (state["v_pages"], state["v"])):
                    pool[table[b][page], :, row:row + n].copy_(rows[b, :, token:token + n])
                token += n
        return [state["k_pages"], state["v_pages"]]
    q = state["q"]
    kv_heads, group, dim = case["kv_heads"], case["heads"] // case["kv_heads"], case["dim"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b, length in enumerate(lengths):
        for h in range(kv_heads):
            if case["op"] == "window":
                k, v, rows, offset = state["k"][b, h], state["v"][b, h], length, 0
            else:
                pages = state["table"][b, :-(-length // case["page"])].long()
                k, v = (state[name][pages, h].reshape(-1, dim) for name in ("k_pages", "v_pages"))
                rows, offset = case["new"], length - case["new"]
            k, v = k.double(), v.double()
            for r in range(0, rows, 1024):
                e = min(rows, r + 1024)
                part = slice(h * group, (h + 1) * group)
                out[b, part, r:e] = _exact_rows(q[b, part, r:e].double(), k, v, torch.arange(r + offset, e + offset),
                                                length, case)
    return out
