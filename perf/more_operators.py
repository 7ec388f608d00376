"""The calls that the speed of the decode-step operators is measured on.

Operators that a program needs next to attention over a paged key-value cache:
rotary positions (`Rotary`), the appending of new keys and values to the cache
with that rotation on the way (`CacheAppender`), attention of a batch whose
sequences share a long prefix, read once for all (`SharedPrefixAttention`),
and sparse attention over pages that a cheap score selects (`PageBounds` keeps
what the score reads, `SelectedAttention` selects and attends).

`run` computes them in elementary torch operations, in fp32 (angles and
selection scores, whose ranks count, in fp64), rounded once at the end; or,
where `own` is true, through the library's entry points. Types: bf16, fp16 and
fp32. Forward only as the library is; the rotation's transposed form is its
gradient.

Rotary positions: pair i of a row (columns i and i + R / 2, or interleaved 2 i
and 2 i + 1, of the first R) turns by the angle position f_i, and is scaled by
a magnitude: (x cos - y sin, y cos + x sin). The transposed form turns back.

Selection: page i of a sequence, for key-value head h, has the bounds lo and hi
of its keys, column by column. Its score for a token is the largest, over the
query heads of h, of sum_d q_d (q_d > 0 ? hi_d : lo_d), rounded to fp32; of the
pages with keys up to the token's position, the first and the recent ones are
always taken, and the others by score, ties to the lower page, until there are
`pages`.
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
FIRST_PAGES, RECENT_PAGES = 1, 2


def _library():
    # The package directory is not a Python identifier; the working folder is
    # the repository's root.
    path = os.path.join(os.getcwd(), "dnn-flash_amd", "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    import onednn_flash_hip as F
    return F


# --- cases -----------------------------------------------------------------

def _rotary(dtype, batch, heads, tokens, dim, part, interleaved, scaling="", farthest=0, transpose=False):
    """[B,H,T,D] rows, the first `part` columns rotated. Positions 0 .. T - 1, or
    with `farthest` a position per token from 0 to there (packed documents, the
    middles of long ones)."""
    return {"op": "rotary", "dtype": dtype, "batch": batch, "heads": heads, "tokens": tokens, "dim": dim, "part": part,
            "interleaved": interleaved, "scaling": scaling, "farthest": farthest, "transpose": transpose}


def _append(dtype, batch, heads, kv_heads, shortest, longest, dim, part, interleaved, page, new, fewest=0, scaling=""):
    """`new` padded rows per sequence, of which `fewest` to `new` are tokens (all
    of them with 0); the sequences then have `shortest` to `longest` tokens."""
    return {"op": "append", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "shortest": shortest,
            "longest": longest, "dim": dim, "part": part, "interleaved": interleaved, "page": page, "new": new,
            "fewest": fewest, "scaling": scaling}


def _prefix(dtype, batch, groups, heads, kv_heads, shared, fewest, most, dim, page, new=1, softcap=0.0):
    """`batch` sequences in `groups` groups. The sequences of a group share about
    `shared` tokens (whole pages) and have `fewest` to `most` of their own."""
    return {"op": "prefix", "dtype": dtype, "batch": batch, "groups": groups, "heads": heads, "kv_heads": kv_heads,
            "shared": shared, "fewest": fewest, "most": most, "dim": dim, "page": page, "new": new, "softcap": softcap}


def _bounds(dtype, batch, kv_heads, shortest, longest, dim, page, new):
    """`new` tokens were written to each of `batch` sequences."""
    return {"op": "bounds", "dtype": dtype, "batch": batch, "kv_heads": kv_heads, "shortest": shortest,
            "longest": longest, "dim": dim, "page": page, "new": new}


def _select(dtype, batch, heads, kv_heads, shortest, longest, dim, page, pages, new=1):
    """`new` tokens for each sequence, that attend to `pages` of its pages each."""
    return {"op": "select", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "shortest": shortest, "longest": longest, "dim": dim, "page": page, "pages": pages, "new": new}


def listed():
    cases = {
        # A batch of prompts before attention without a cache.
        "rotary_prompt": _rotary("bf16", 4, 32, 2048, 128, 128, False),
        # The gradient's way back in fp32: interleaved pairs, a part of an odd
        # head, far positions.
        "rotary_back": _rotary("f32", 2, 8, 1001, 96, 64, True, scaling="linear", farthest=1000000, transpose=True),
        # Every layer of every decode step: one row per sequence. Latency counts.
        "append_step": _append("bf16", 64, 32, 8, 33, 4096, 128, 128, False, 16, 1),
        # A batch of prompts goes into the cache, frequencies stretched for long
        # contexts, half of the head turned.
        "append_prompts": _append("f16", 8, 16, 8, 1000, 2048, 128, 64, True, 16, 2048, fewest=700, scaling="parts"),
        # Four answers to one question, just begun.
        "prefix_few": _prefix("bf16", 4, 1, 32, 8, 1024, 1, 200, 128, 16),
        # A serving batch under one long system prompt.
        "prefix_batch": _prefix("bf16", 64, 1, 32, 8, 16384, 33, 1024, 128, 16),
        # Draft tokens in fp32, three long documents with questions to each.
        "prefix_groups": _prefix("f32", 15, 3, 8, 8, 4000, 10, 300, 64, 32, new=3),
        # What the selection reads is kept up to date after a decode step ...
        "bounds_step": _bounds("bf16", 64, 8, 33, 4096, 128, 16, 1),
        # ... and made for a batch of prompts.
        "bounds_prompts": _bounds("f16", 8, 8, 1500, 2048, 128, 32, 1500),
        # One very long document.
        "select_long": _select("f16", 1, 32, 8, 131000, 131000, 128, 64, 64),
        # A serving batch of long sequences, 2048 keys each.
        "select_batch": _select("bf16", 32, 32, 8, 2000, 32768, 128, 32, 64),
        # Draft tokens in fp32, each with pages of its own.
        "select_drafts": _select("f32", 4, 8, 8, 1000, 8192, 64, 16, 40, new=3),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _log(rng, low, high):
    """A whole number spread over [low, high] by its logarithm."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "append", "prefix", "prefix", "prefix", "bounds", "select", "select", "select"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    page = rng.choice([16, 32, 64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 192, 256])
    part = rng.choice([dim, dim, dim // 2, dim // 4, 2 * rng.randint(1, dim // 2)])
    interleaved = rng.random() < 0.5
    scaling = rng.choice(["", "linear", "parts"])
    if op == "rotary":
        tokens = _log(rng, 1, 8192)
        batch = _log(rng, 1, max(1, min(64, (1 << 24) // (heads * dim * tokens))))
        return _rotary(dtype, batch, heads, tokens, dim, part, interleaved, scaling,
                       rng.choice([0, _log(rng, 100, 2000000)]), rng.random() < 0.5)
    if op == "append":
        new = rng.choice([1, _log(rng, 1, 2048)])
        longest = new + _log(rng, 1, 1024)
        batch = _log(rng, 1, max(1, min(128, (1 << 24) // (heads * dim * longest))))
        fewest = rng.choice([0, rng.randint(1, new)])
        return _append(dtype, batch, heads, kv_heads, rng.randint(new, longest), longest, dim, part, interleaved, page,
                       new, fewest, scaling)
    if op == "prefix":
        # at most what the serving batch holds and computes
        shared = _log(rng, 16, max(16, min(32768, (1 << 24) // (kv_heads * dim))))
        most = _log(rng, 1, 2048)
        new = rng.choice([1, 1, rng.randint(2, 8)])
        pairs = (1 << 30) if dtype == "f32" else (1 << 32)
        room = min((1 << 25) // (kv_heads * dim * (most + 8)), pairs // (heads * dim * new * (shared + most)))
        batch = _log(rng, 1, max(1, min(128, room)))
        groups = _log(rng, 1, max(1, min(8, batch, (1 << 24) // (kv_heads * dim * shared))))
        return _prefix(dtype, batch, groups, heads, kv_heads, shared, rng.randint(1, most), most, dim, page, new,
                       rng.choice([0.0, 0.0, 0.0, 30.0]))
    if op == "bounds":
        longest = _log(rng, 1, 4096)
        batch = _log(rng, 1, max(1, min(128, (1 << 25) // (kv_heads * dim * longest))))
        shortest = rng.randint(1, longest)
        return _bounds(dtype, batch, kv_heads, shortest, longest, dim, page, rng.choice([1, rng.randint(1, shortest)]))
    longest = _log(rng, 16, 65536)
    pages = _log(rng, 4, 128)
    # a pool that prepares quickly, and at most the pages that the serving batch reads
    room = min((1 << 28) // (kv_heads * dim * longest), (1 << 25) // (kv_heads * dim * min(longest, pages * page)))
    batch = _log(rng, 1, max(1, min(64, room)))
    return _select(dtype, batch, heads, kv_heads, rng.randint(1, longest), longest, dim, page, pages,
                   rng.choice([1, 1, rng.randint(2, 4)]))


def _spread(low, high, count):
    """`count` whole numbers from low to high in no order, the last one high."""
    golden = (math.sqrt(5.0) - 1.0) / 2.0
    return [low + int((high - low) * ((i + 1) * golden % 1.0)) for i in range(count - 1)] + [high]


def _groups(case):
    """(sequences, shared tokens) of each group; shared tokens are whole pages."""
    n, g, page = case["batch"], case["groups"], case["page"]
    sizes = [n // g + (i < n % g) for i in range(g)]
    return [(size, max(1, (case["shared"] - 37 * i) // page) * page) for i, size in enumerate(sizes)]


def _lengths(case):
    if case["op"] == "prefix":
        low = max(case["fewest"], case["new"])
        mine = _spread(low, max(low, case["most"]), case["batch"])
        shared = [tokens for size, tokens in _groups(case) for _ in range(size)]
        return [a + b for a, b in zip(shared, mine)]
    return _spread(case["shortest"], case["longest"], case["batch"])


def _counts(case):
    return _spread(case["fewest"] or case["new"], case["new"], case["batch"])


def _base(case):
    """Frequencies in fp64, radians per position, and the magnitude. `linear`
    divides the angles by 4; `parts` (8 times a length of 4096) leaves pairs that
    turn often over that length, divides those that turn less than once by 8, and
    goes from one to the other in between, linear in the number of turns."""
    part = case["part"]
    f = 10000.0 ** (-np.arange(0, part, 2, dtype=np.float64) / part)
    if case["scaling"] == "linear":
        return f / 4.0, 1.0
    if case["scaling"] == "parts":
        turns = 4096.0 * f / (2.0 * math.pi)
        keep = np.clip((turns - 1.0) / (32.0 - 1.0), 0.0, 1.0)
        return f * keep + f / 8.0 * (1.0 - keep), 0.1 * math.log(8.0) + 1.0
    return f, 1.0


def _library_scaling(case):
    """The same as the library's arguments."""
    if case["scaling"] == "linear":
        return {"scaling": {"type": "linear", "factor": 4.0}}
    if case["scaling"] == "parts":
        return {"scaling": {"type": "parts", "factor": 8.0, "original_tokens": 4096, "low": 1.0, "high": 32.0},
                "magnitude": 0.1 * math.log(8.0) + 1.0}
    return {}


def _pages(tokens, page):
    return -(-tokens // page)


def work(case):
    size, dim = BYTES[case["dtype"]], case["dim"]
    if case["op"] == "rotary":
        rows = case["batch"] * case["heads"] * case["tokens"]
        positions = 4 * case["batch"] * case["tokens"] if case["farthest"] else 0
        return {"bytes": 2 * rows * dim * size + positions, "flops": 3 * rows * case["part"]}
    if case["op"] == "append":
        new = sum(_counts(case))
        padded = case["batch"] * case["new"]
        row = dim * size
        return {"bytes": row * (case["heads"] * (new + padded) + 4 * case["kv_heads"] * new) + 8 * case["batch"],
                "flops": 3 * case["part"] * new * (case["heads"] + case["kv_heads"])}
    lengths = _lengths(case)
    if case["op"] == "bounds":
        keys = pages = 0
        for n in lengths:
            first = max(0, n - case["new"]) // case["page"]
            keys += n - first * case["page"]
            pages += _pages(n, case["page"]) - first
        return {"bytes": case["kv_heads"] * dim * size * (keys + 2 * pages), "flops": 2 * case["kv_heads"] * dim * keys}
    rows = case["batch"] * case["heads"] * case["new"]
    if case["op"] == "prefix":
        groups = _groups(case)
        pairs = sum(n * case["new"] - case["new"] * (case["new"] - 1) // 2 for n in lengths)
        keys = sum(lengths) - sum((count - 1) * tokens for count, tokens in groups)
        return {"bytes": 2 * dim * size * (case["kv_heads"] * keys + rows), "flops": 4 * dim * case["heads"] * pairs}
    scored = pairs = keys = 0
    for n in lengths:
        for t in range(case["new"]):
            seen = n - case["new"] + t + 1
            have = _pages(max(seen, 0), case["page"])
            taken = max(0, seen if have <= case["pages"] else case["pages"] * case["page"] - (-seen % case["page"]))
            pairs += taken
            scored += have if have > case["pages"] else 0
        keys += taken  # (the last token's: others may take the same pages)
    scored_pages = sum(_pages(n, case["page"]) for n in lengths if _pages(n, case["page"]) > case["pages"])
    return {"bytes": 2 * dim * size * (case["kv_heads"] * (keys + scored_pages) + rows),
            "flops": dim * case["heads"] * (4 * pairs + 2 * scored)}


# --- inputs ----------------------------------------------------------------

def _normal(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(DTYPES[dtype])


def _token_major(gen, batch, heads, tokens, dim, dtype):
    """[B, H, T, D] over the [B, T, H, D] storage that a projection makes."""
    return _normal(gen, (batch, tokens, heads, dim), dtype).transpose(1, 2)


def _table(case, lengths, seed):
    """The page table of a pool that has been in use for long, pages in no order
    (entries past a sequence's end are -1), and the pool's pages. The sequences
    of a group have its shared pages in common."""
    page = case["page"]
    groups = _groups(case) if case["op"] == "prefix" else [(len(lengths), 0)]
    used = sum(_pages(n, page) for n in lengths) - sum((count - 1) * (tokens // page) for count, tokens in groups)
    pool = used + used // 4 + 1
    order = np.random.default_rng(seed).permutation(pool)[:used].astype(np.int32)
    table = np.full((len(lengths), max(_pages(n, page) for n in lengths)), -1, np.int32)
    at = row = 0
    for count, tokens in groups:
        shared = order[at:at + tokens // page]
        at += shared.size
        for _ in range(count):
            mine = _pages(lengths[row], page) - shared.size
            table[row, :shared.size] = shared
            table[row, shared.size:shared.size + mine] = order[at:at + mine]
            at += mine
            row += 1
    return torch.from_numpy(table).cuda(), pool


def _bounds_of(state, pages):
    """Bounds [P, Hkv, 2, D] of the first `pages` pages of each sequence (a number
    for each)."""
    case, k_pages = state["case"], state["k_pages"]
    size = case["page"]
    row = torch.arange(size, device=k_pages.device)
    low = float("inf")
    for b, n in enumerate(_lengths(case)):
        ids = state["table"][b, :pages[b]].long()
        seen = (torch.arange(pages[b], device=ids.device)[:, None] * size + row < n)[:, None, :, None]
        keys = k_pages[ids]
        state["bounds"][ids, :, 0] = torch.where(seen, keys, low).amin(2)
        state["bounds"][ids, :, 1] = torch.where(seen, keys, -low).amax(2)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    dtype, dim, op = case["dtype"], case["dim"], case["op"]
    if op in ("rotary", "append"):
        frequencies, state["magnitude"] = _base(case)
        state["frequencies"] = torch.from_numpy(frequencies).cuda()
        if own:
            state["rotary"] = _library().Rotary(dim, rotary_dim=case["part"], interleaved=case["interleaved"],
                                                **_library_scaling(case))
    if op == "rotary":
        state["x"] = _token_major(gen, case["batch"], case["heads"], case["tokens"], dim, dtype)
        state["positions"] = None
        if case["farthest"]:
            state["positions"] = torch.randint(0, case["farthest"] + 1, (case["batch"], case["tokens"]), generator=gen,
                                               device="cuda", dtype=torch.int32)
        return state
    lengths = _lengths(case)
    state["lengths"] = torch.tensor(lengths, dtype=torch.int32).cuda()
    state["table"], pool = _table(case, lengths, seed)
    shape = (pool, case["kv_heads"], case["page"], dim)
    state["k_pages"] = _normal(gen, shape, dtype)
    if op == "bounds":
        # pages that are not touched keep what they had: what was right a step before
        state["bounds"] = torch.zeros((pool, case["kv_heads"], 2, dim), dtype=DTYPES[dtype], device="cuda")
        _bounds_of(state, [_pages(max(n - case["new"], 0), case["page"]) for n in lengths])
        if own:
            state["update"] = _library().PageBounds(state["k_pages"], state["bounds"], state["table"],
                                                    state["lengths"], tokens=case["new"])
        return state
    state["v_pages"] = _normal(gen, shape, dtype)
    state["q"] = _token_major(gen, case["batch"], case["heads"], case["new"], dim, dtype)
    if op == "append":
        state["k"] = _token_major(gen, case["batch"], case["kv_heads"], case["new"], dim, dtype)
        state["v"] = _token_major(gen, case["batch"], case["kv_heads"], case["new"], dim, dtype)
        state["counts"] = torch.tensor(_counts(case), dtype=torch.int32).cuda() if case["fewest"] else None
        if own:
            state["append"] = _library().CacheAppender(state["k_pages"], state["v_pages"], state["table"],
                                                       state["lengths"], state["rotary"], counts=state["counts"])
    elif op == "prefix":
        if own:
            state["attend"] = _library().SharedPrefixAttention(
                state["k_pages"], state["v_pages"], state["table"], state["lengths"], groups=_groups(case),
                heads=case["heads"], query_tokens=case["new"], softcap=case["softcap"])
    else:
        state["bounds"] = torch.zeros((pool, case["kv_heads"], 2, dim), dtype=DTYPES[dtype], device="cuda")
        _bounds_of(state, [_pages(n, case["page"]) for n in lengths])
        if own:
            state["attend"] = _library().SelectedAttention(
                state["k_pages"], state["v_pages"], state["bounds"], state["table"], state["lengths"],
                heads=case["heads"], query_tokens=case["new"], pages=case["pages"], first_pages=FIRST_PAGES,
                recent_pages=RECENT_PAGES)
    return state


# --- the plain forms --------------------------------------------------------

def _rotate_plain(x, positions, state):
    """x [B,H,T,D] at positions [B,T] or [1,T] (fp64): fp32."""
    case, part = state["case"], state["case"]["part"]
    angle = (positions[:, None, :, None] * state["frequencies"]).remainder(2.0 * math.pi)
    c, s = (f(angle).float() * state["magnitude"] for f in (torch.cos, torch.sin))
    if case.get("transpose"):
        s = -s
    x = x.float()
    turned = x[..., :part]
    if case["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = turned[..., :part // 2], turned[..., part // 2:]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([turned, x[..., part:]], -1)


def _rotary_plain(state):
    x, positions = state["x"], state["positions"]
    if positions is None:
        positions = torch.arange(x.shape[2], device=x.device)[None]
    return _rotate_plain(x, positions.double(), state).to(x.dtype)


def _append_plain(state):
    case, q, k, v = state["case"], state["q"], state["k"], state["v"]
    counts = state["counts"] if state["counts"] is not None else torch.full_like(state["lengths"], case["new"])
    token = torch.arange(case["new"], device=k.device)[None, :]
    position = state["lengths"][:, None] - counts[:, None] + token
    q_out = _rotate_plain(q, position.double(), state).to(q.dtype)
    q_out = torch.where((token < counts[:, None])[:, None, :, None], q_out, torch.zeros_like(q_out))
    k = _rotate_plain(k, position.double(), state).to(k.dtype)
    # rows past a sequence's count repeat its last token (which is there: counts are 1 or more)
    token = torch.minimum(token, counts[:, None] - 1)
    position = torch.minimum(position, state["lengths"][:, None] - 1).long()
    page = torch.gather(state["table"].long(), 1, position // case["page"])
    for pool, rows in ((state["k_pages"], k), (state["v_pages"], v)):
        rows = rows.transpose(1, 2)
        rows = torch.gather(rows, 1, token.long()[:, :, None, None].expand(-1, -1, rows.shape[2], rows.shape[3]))
        pool[page, :, position % case["page"]] = rows
    return [q_out, state["k_pages"], state["v_pages"]]


def _softmax_plain(scores, seen, v):
    """softmax of the seen scores [.., M, N] times v [.., N, D]; 0 where nothing is seen."""
    scores = torch.where(seen, scores, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    weight = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, v)
    return torch.where(total > 0, out / total, torch.zeros_like(out))


def _paged_rows(state, b):
    """K and V of sequence b, [Hkv, 1, N, D] in fp32."""
    ids = state["table"][b].clamp(min=0).long()
    return (state[name][ids].float().transpose(0, 1).flatten(1, 2)[:, None] for name in ("k_pages", "v_pages"))


def _prefix_plain(state):
    case, q = state["case"], state["q"]
    batch, heads, new, dim = q.shape
    out = torch.empty((batch, heads, new, dim), dtype=q.dtype, device=q.device)
    for b in range(batch):
        k, v = _paged_rows(state, b)
        rows = q[b].float().reshape(case["kv_heads"], -1, new, dim)
        scores = torch.matmul(rows, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(dim))
        if case["softcap"]:
            scores = case["softcap"] * torch.tanh(scores / case["softcap"])
        position = (state["lengths"][b] - new + torch.arange(new, device=q.device))[:, None]
        seen = torch.arange(k.shape[2], device=q.device)[None, :] <= position
        out[b] = _softmax_plain(scores, seen, v).reshape(heads, new, dim).to(q.dtype)
    return out


def _bounds_plain(state):
    case, lengths, table, k_pages = state["case"], state["lengths"], state["table"], state["k_pages"]
    size = case["page"]
    touched = (case["new"] + size - 2) // size + 1
    first = (lengths - case["new"]).clamp(min=0) // size
    last = (lengths - 1) // size
    # pages past the last touched one repeat it
    page = torch.minimum(first[:, None] + torch.arange(touched, device=table.device), last[:, None]).long()
    ids = torch.gather(table, 1, page).long()
    keys = k_pages[ids]  # [B, touched, Hkv, S, D]
    seen = page[:, :, None] * size + torch.arange(size, device=table.device) < lengths[:, None, None]
    seen = seen[:, :, None, :, None]
    state["bounds"][ids, :, 0] = torch.where(seen, keys, float("inf")).amin(3)
    state["bounds"][ids, :, 1] = torch.where(seen, keys, float("-inf")).amax(3)
    return [state["bounds"]]


def _select_plain(state):
    case, q, table = state["case"], state["q"], state["table"]
    batch, heads, new, dim = q.shape
    kv_heads, size, most = case["kv_heads"], case["page"], case["pages"]
    selected = torch.full((batch, kv_heads, new, most), -1, dtype=torch.int32, device=q.device)
    out = torch.empty((batch, heads, new, dim), dtype=q.dtype, device=q.device)
    index = torch.arange(table.shape[1], device=q.device)
    for b in range(batch):
        rows = q[b].reshape(kv_heads, -1, new, dim)
        bounds = state["bounds"][table[b].clamp(min=0).long()].double().transpose(0, 1)  # [Hkv, pages, 2, D]
        up, down = (rows.double().clamp(min=0.0), rows.double().clamp(max=0.0))
        score = (torch.matmul(up, bounds[:, None, :, 1].transpose(2, 3).contiguous())
                 + torch.matmul(down, bounds[:, None, :, 0].transpose(2, 3).contiguous())).float().amax(1)
        position = state["lengths"][b] - new + torch.arange(new, device=q.device)
        have = ((position + size) // size).clamp(min=0)[:, None]  # pages of each token
        score = torch.where((index < FIRST_PAGES) | (index >= have - RECENT_PAGES), float("inf"), score)
        score = torch.where(index < have, score, float("-inf"))
        taken = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :most]
        taken = torch.where(taken < have, taken, table.shape[1]).sort(-1).values
        taken = torch.where(taken < table.shape[1], taken, -1)
        selected[b, :, :, :taken.shape[-1]] = taken.to(torch.int32)
        k, v = _paged_rows(state, b)
        scores = torch.matmul(rows.float(), k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(dim))
        # (one place more, where the -1 go)
        mine = torch.zeros((kv_heads, new, table.shape[1] + 1), dtype=torch.bool, device=q.device)
        mine.scatter_(2, torch.where(taken >= 0, taken, table.shape[1]), True)
        seen = mine[..., :-1].repeat_interleave(size, -1) & \
            (torch.arange(k.shape[2], device=q.device)[None, :] <= position[:, None])
        out[b] = _softmax_plain(scores, seen[:, None], v).reshape(heads, new, dim).to(q.dtype)
    return [selected, out]


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return {"rotary": _rotary_plain, "append": _append_plain, "prefix": _prefix_plain, "bounds": _bounds_plain,
                "select": _select_plain}[op](state)
    if op == "rotary":
        return state["rotary"](state["x"], positions=state["positions"], transpose=case["transpose"])
    if op == "append":
        return [state["append"](state["k"], state["v"], state["q"]), state["k_pages"], state["v_pages"]]
    if op == "prefix":
        return state["attend"](state["q"])
    if op == "bounds":
        state["update"]()
        return [state["bounds"]]
    selected = state["attend"].select(state["q"])
    return [selected, state["attend"](state["q"], selected=selected)]


# --- the definitions in 64 bits ----------------------------------------------

def _exact_rotate(x, position, case):
    """Rows x [.., D] at `position` [..]: as complex numbers."""
    f, magnitude = _base(case)
    part = case["part"]
    sign = -1.0 if case.get("transpose") else 1.0
    angle = position.double()[..., None] * torch.from_numpy(f).to(x.device)
    turn = torch.polar(torch.full_like(angle, magnitude), sign * angle)
    out = x.double().clone()
    first, second = (slice(0, part, 2), slice(1, part, 2)) if case["interleaved"] else \
        (slice(0, part // 2), slice(part // 2, part))
    z = torch.complex(out[..., first].contiguous(), out[..., second].contiguous()) * turn
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _exact_append(case, state):
    q, k, v = state["q"], state["k"], state["v"]
    size = case["page"]
    q_out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    k_pages, v_pages = state["k_pages"].double(), state["v_pages"].double()
    table = state["table"].cpu().tolist()
    for b, (length, count) in enumerate(zip(_lengths(case), _counts(case))):
        position = torch.arange(length - count, length, device=q.device)
        q_out[b, :, :count] = _exact_rotate(q[b, :, :count], position, case)
        turned = _exact_rotate(k[b, :, :count], position, case)
        token = 0
        while token < count:  # a page at a time
            page, row = divmod(length - count + token, size)
            n = min(size - row, count - token)
            k_pages[table[b][page], :, row:row + n] = turned[:, token:token + n]
            v_pages[table[b][page], :, row:row + n] = v[b, :, token:token + n].double()
            token += n
    return [q_out, k_pages, v_pages]


def _exact_row(q, k, v, case):
    """Queries q [G, D] that see all of k, v [N, D]."""
    x = q.double() @ k.double().T.contiguous() / math.sqrt(q.shape[-1])
    if case.get("softcap"):
        x = torch.tanh(x / case["softcap"]) * case["softcap"]
    return torch.softmax(x, -1) @ v.double()


def _exact_attend(case, state, keys_of):
    """Every token's rows over the pages keys_of(b, h, t) names (None: all)."""
    q = state["q"]
    size, group = case["page"], case["heads"] // case["kv_heads"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b, length in enumerate(_lengths(case)):
        for h in range(case["kv_heads"]):
            for t in range(case["new"]):
                seen = length - case["new"] + t + 1
                if seen <= 0:
                    continue
                pages = keys_of(b, h, t)
                pages = torch.arange(_pages(seen, size)) if pages is None else pages
                last = (int(pages[-1]) + 1) * size - seen  # rows of the last page that are not seen
                ids = state["table"][b, pages.to(q.device)].long()
                k, v = (state[name][ids, h].flatten(0, 1) for name in ("k_pages", "v_pages"))
                n = k.shape[0] - max(0, last)
                out[b, h * group:(h + 1) * group, t] = _exact_row(q[b, h * group:(h + 1) * group, t], k[:n], v[:n], case)
    return out


def _exact_select(case, state):
    q = state["q"]
    size, group, most = case["page"], case["heads"] // case["kv_heads"], case["pages"]
    selected = torch.full((case["batch"], case["kv_heads"], case["new"], most), -1, dtype=torch.int32)
    for b, length in enumerate(_lengths(case)):
        for h in range(case["kv_heads"]):
            bounds = state["bounds"][state["table"][b].clamp(min=0).long(), h].double()  # [pages, 2, D]
            for t in range(case["new"]):
                have = _pages(max(0, length - case["new"] + t + 1), size)
                if have > most:
                    rows = q[b, h * group:(h + 1) * group, t].double()
                    best = None
                    for row in rows:
                        s = (row * torch.where(row > 0, bounds[:have, 1], bounds[:have, 0])).sum(-1).float()
                        best = s if best is None else torch.maximum(best, s)
                    best = best.cpu().numpy()
                    always = set(range(FIRST_PAGES)) | set(range(have - RECENT_PAGES, have))
                    rest = [int(i) for i in np.argsort(-best, kind="stable") if int(i) not in always]
                    pages = sorted(always | set(rest[:most - len(always)]))
                else:
                    pages = list(range(have))
                selected[b, h, t, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
    return selected


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "rotary":
        x, positions = state["x"], state["positions"]
        if positions is None:
            positions = torch.arange(x.shape[2], device=x.device)[None]
        return _exact_rotate(x, positions[:, None].expand(x.shape[0], x.shape[1], -1), case)
    if op == "append":
        return _exact_append(case, state)
    if op == "bounds":
        table = state["table"].cpu().tolist()
        for b, n in enumerate(_lengths(case)):
            for page in range(max(0, n - case["new"]) // case["page"], _pages(n, case["page"])):
                keys = state["k_pages"][table[b][page], :, :n - page * case["page"]]
                state["bounds"][table[b][page], :, 0] = keys.min(1).values
                state["bounds"][table[b][page], :, 1] = keys.max(1).values
        return [state["bounds"].double()]
    if op == "prefix":
        return _exact_attend(case, state, lambda b, h, t: None)
    selected = _exact_select(case, state)
    out = _exact_attend(case, state, lambda b, h, t: selected[b, h, t][selected[b, h, t] >= 0].long())
    return [selected.to(state["q"].device), out]
