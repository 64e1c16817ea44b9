"""Performance cases of the paged 4-bit key/value cache: the operators that a serving program
runs next to the draft, each from its smallest call to its largest.

  plan    ``KV4Cache.step``: the block table, the free pages and the slot map of one step, made
          on the GPU from the lengths that the requests keep and the rows that they grow by;
  append  ``KV4Cache.append`` and ``KV4Cache.read``: rows of keys and values quantised into
          their slots, and the values that those slots then stand for;
  attend  ``KV4Cache.attend``: attention of ragged query rows over the cached keys, for single
          tokens, draft blocks (every row sees every key) and prompts (causal).

A row of one head (128 values) is held as four groups of 32: a shared exponent byte b and 32
four-bit codes (sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6), standing for code * 2^(b - 127).
b is the smallest exponent for which the group's largest magnitude is at most 7 * 2^(b - 127)
(0 at least), codes round to nearest with ties to the even code; a group with an infinity or a
NaN has b = 255 and stands for NaN.

``own`` selects the package's kernels; where it is false the same results come from elementary
torch operations in 32 bits.
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

D = 128          # head dimension
G = D // 32      # groups of a row
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # One speculative step of eight requests: 21 of the last block's 32 rows were rejected,
        # the next block of 32 takes their place; launches count.
        {"name": "plan_draft_8", "kind": "plan", "page": 64, "width": 128, "seqs": 8,
         "keep": "4114 4422 6280 7780 747 1587 6801 7766", "grow": "32"},
        # A decode step of a server's 256 requests, some idle, a few crossing into a new page.
        {"name": "plan_token_256", "kind": "plan", "page": 32, "width": 512, "seqs": 256,
         "keep": "mix 1 16000", "grow": "mix 0 2"},
        # A server that replaces all of its 1024 requests at once: every page put back and
        # handed out again, two million rows mapped.
        {"name": "plan_admit_1024", "kind": "plan", "page": 64, "width": 128, "seqs": 1024,
         "keep": "0", "grow": "mix 1 4096"},
        # The new rows of a decode step: eight sequences, one token each.
        {"name": "append_tokens_8", "kind": "append", "rows": 8, "kv": 8, "page": 64,
         "dtype": "float16"},
        # The benchmark's context length as one prompt.
        {"name": "append_prompt_4096", "kind": "append", "rows": 4096, "kv": 8, "page": 64,
         "dtype": "float16"},
        # Several long prompts admitted in one step, ragged in all.
        {"name": "append_prompts_65521", "kind": "append", "rows": 65521, "kv": 8, "page": 128,
         "dtype": "bfloat16"},
        # One token of one conversation: latency.
        {"name": "attend_token_500", "kind": "attend", "heads": 32, "kv": 8, "page": 64,
         "q": "1", "len": "500", "causal": True, "dtype": "float16"},
        # A draft block over a long document, the 27B draft's heads.
        {"name": "attend_block_32768", "kind": "attend", "heads": 40, "kv": 8, "page": 64,
         "q": "32", "len": "32800", "causal": False, "dtype": "float16"},
        # The batched benchmark's blocks: eight sequences of ragged contexts, 32 rows each.
        {"name": "attend_blocks_8", "kind": "attend", "heads": 32, "kv": 8, "page": 64,
         "q": "32 32 32 32 32 32 32 32",
         "len": "4178 4475 6344 7844 811 1651 6865 7830", "causal": False, "dtype": "float16"},
        # A decode step of 64 ragged requests, one of them idle.
        {"name": "attend_tokens_64", "kind": "attend", "heads": 32, "kv": 8, "page": 32,
         "q": " ".join(["1"] * 41 + ["0"] + ["1"] * 22),
         "len": " ".join(str(17 + (i * i * 37) % 12007) for i in range(64)), "causal": True,
         "dtype": "bfloat16"},
        # Prompts: a fresh one of 4096 rows and a follow-up of 777 behind 2048 cached rows.
        {"name": "attend_prompts_2", "kind": "attend", "heads": 32, "kv": 8, "page": 128,
         "q": "4096 777", "len": "4096 2825", "causal": True, "dtype": "bfloat16"},
        # Sixteen long documents, one token each: a million cached rows.
        {"name": "attend_tokens_1m", "kind": "attend", "heads": 64, "kv": 8, "page": 64,
         "q": " ".join(["1"] * 16),
         "len": " ".join(str(65536 - 31 * i) for i in range(16)), "causal": True,
         "dtype": "bfloat16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "append", "attend", "attend", "attend", "attend"])
    page = rng.choice([32, 64, 128])
    if kind == "plan":
        seqs = _log_int(rng, 1, 1024)
        longest = _log_int(rng, 32, 4096)
        fresh = rng.random() < 0.4
        return {"kind": kind, "page": page, "width": _pages(2 * longest + 64, page), "seqs": seqs,
                "keep": "0" if fresh else "mix 1 %d" % longest,
                "grow": "mix 1 %d" % longest if fresh else "mix 0 %d" % _log_int(rng, 1, 64)}
    if kind == "append":
        return {"kind": kind, "rows": _log_int(rng, 1, 65536), "kv": rng.choice([1, 2, 4, 5, 8]),
                "page": page, "dtype": rng.choice(sorted(DTYPES))}
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 3, 4, 5, 7, 8])
    seqs = _log_int(rng, 1, 64)
    shape = rng.choice(["token", "token", "block", "block", "prompt"])
    total = _log_int(rng, 64 * seqs, 1 << (19 if shape == "token" else 16))   # cached rows in all
    lens = [max(1, int(2 * rng.random() * total / seqs)) for _ in range(seqs)]
    if shape == "token":
        q = [1 if rng.random() < 0.9 else 0 for _ in lens]
        q[0] = 1
    elif shape == "block":
        b = rng.randint(2, 32)
        q = [min(b, n) for n in lens]
    else:                                           # prompts or parts of them
        lens = [min(n, 2200) for n in lens[:2]]
        q = [rng.randint(max(1, n // 3), n) for n in lens]
    return {"kind": kind, "heads": heads, "kv": kv, "page": page, "q": " ".join(map(str, q)),
            "len": " ".join(map(str, lens)), "causal": shape != "block" or rng.random() < 0.3,
            "dtype": rng.choice(sorted(DTYPES))}


# ---------------------------------------------------------------------------- inputs


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mirror-sd_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from mirror_sd_amd.kv4 import KV4Cache
    return KV4Cache


def _counts(text, n, seed):
    """n counts: "mix lo hi" (spread over lo .. hi, in the seed's order), one for all, or each."""
    words = text.split()
    if words[0] == "mix":
        lo, hi = int(words[1]), int(words[2])
        rng = random.Random(lo * 31 + hi)
        mix = [rng.randint(lo, hi) for _ in range(n)]
        random.Random(seed).shuffle(mix)
        return mix
    return [int(w) for w in words] if len(words) > 1 else [int(words[0])] * n


def _plan_sizes(case, seed):
    keep = _counts(case["keep"], case["seqs"], seed)
    grow = _counts(case["grow"], case["seqs"], seed + 1)
    return keep, grow


def _pages(n, page):
    return -(-n // page)


def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed(seed * 1000003 + salt)


def _kv_rows(n, kv, dtype, seed, salt):
    """Keys and values [n, 2, kv, 128] as projections leave them: keys after their norm and its
    channel gains, a few channels much larger than the rest; values of row-dependent size."""
    g = _gen(seed, salt)
    x = torch.randn((n, 2, kv, D), generator=g, device="cuda")
    gain = torch.exp(0.4 * torch.randn((kv, D), generator=_gen(seed, 1), device="cuda"))
    gain[:, ::41] *= 4.0
    x[:, 0] *= gain
    x[:, 1] *= torch.exp(0.5 * torch.randn((n, 1, 1), generator=g, device="cuda"))
    return x.to(dtype)


def _q_rows(n, heads, dtype, seed):
    return torch.randn((n, heads, D), generator=_gen(seed, 2), device="cuda").to(dtype)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    torch.cuda.set_device(0)
    kind, page = case["kind"], case["page"]
    if kind == "plan":
        keep, grow = _plan_sizes(case, seed)
        lens = [a + b for a, b in zip(keep, grow)]
        pool = sum(_pages(n, page) for n in keep + grow) + 8
        order = list(range(pool))
        random.Random(seed).shuffle(order)
        table, at = [], 0
        for n in lens:
            p = _pages(n, page)
            table.append(order[at:at + p] + [-1] * (case["width"] - p))
            at += p
        st = {"case": case, "keep": _ints(keep), "grow": _ints(grow), "rows": sum(grow)}
        lens, table = _ints(lens), _ints(table)
        free, n_free = _ints(order[at:] + [-1] * at), _ints([pool - at])
        if own:
            c = _package()(n_kv_heads=1, n_pages=pool, max_seqs=case["seqs"],
                           max_len=case["width"] * page, page=page)
            for dst, src in ((c.lens, lens), (c.table, table), (c.free, free), (c.n_free, n_free)):
                dst.copy_(src)
            st["cache"] = c
        else:
            st.update(lens=lens, table=table, free=free, n_free=n_free)
        return st
    dtype, kv = DTYPES[case["dtype"]], case["kv"]
    if kind == "append":
        n = case["rows"]
        held = _pages(n, page)
        order = torch.randperm(held + 3, generator=_gen(seed, 3), device="cuda")[:held]
        slots = (order[:, None] * page + torch.arange(page, device="cuda")).reshape(-1)[:n]
        st = {"case": case, "kv": _kv_rows(n, kv, dtype, seed, 4), "slots": slots.to(torch.int32)}
        if own:
            st["cache"] = _package()(n_kv_heads=kv, n_pages=held + 3, max_seqs=1,
                                     max_len=(held + 3) * page, page=page)
        else:
            st["codes"], st["scales"] = _pool(held + 3, kv, page)
        return st
    q, lens = _counts(case["q"], 1, 0), _counts(case["len"], 1, 0)
    held = [_pages(n, page) for n in lens]
    pool = sum(held) + 2
    order = torch.randperm(pool, generator=_gen(seed, 3), device="cuda").to(torch.int32)
    st = {"case": case, "q": _q_rows(sum(q), case["heads"], dtype, seed), "q_lens": q, "lens": lens}
    if own:
        c = _package()(n_kv_heads=kv, n_pages=pool, max_seqs=len(lens), max_len=max(held) * page,
                       page=page)
        c.free.copy_(order)
        slots = c.step(grow=_ints(lens), max_rows=sum(lens)).slots
        at = 0
        for s, n in enumerate(lens):
            x = _kv_rows(n, kv, dtype, seed, 16 + s)
            c.append(x[:, 0], x[:, 1], slots[at:at + n])
            at += n
        st["cache"] = c
        st["starts"] = _ints([sum(q[:i]) for i in range(len(q) + 1)])
        return st
    codes, scales = _pool(pool, kv, page)
    table, at = [], 0
    for s, n in enumerate(lens):
        mine = order[at:at + held[s]].long()
        at += held[s]
        c, b = _quantise(_kv_rows(n, kv, dtype, seed, 16 + s))
        slots = (mine[:, None] * page + torch.arange(page, device="cuda")).reshape(-1)[:n]
        _write(codes, scales, slots, c, b)
        table.append(mine)
    st.update(codes=codes, scales=scales, table=table)
    return st


# ---------------------------------------------------------------------------- the plain form


def _pool(pages, kv, page):
    """Codes [pages, 2, kv, page, 64] (two values a byte, the even one low) and exponent bytes
    [pages, 2, kv, page, 4]."""
    return (torch.zeros((pages, 2, kv, page, D // 2), dtype=torch.uint8, device="cuda"),
            torch.zeros((pages, 2, kv, page, G), dtype=torch.uint8, device="cuda"))


def _power(e):
    """2^e in fp32, exact, for -127 <= e <= 127 (2^-127 is subnormal)."""
    return torch.where(e > -127, (e + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _quantise(x):
    """x [..., 128] -> code bytes [..., 64], exponent bytes [..., 4]."""
    x = x.float().unflatten(-1, (G, 32))
    top = x.abs().amax(-1)
    bits = top.view(torch.int32)
    e = (bits >> 23) - 129 + ((bits & 0x7FFFFF) > 0x600000).int()
    bad = ~torch.isfinite(x).all(-1)
    e = torch.where(bad, 0, e.clamp(min=-127))
    y = x * _power(-e)[..., None]
    a = y.abs()
    code = torch.zeros_like(a, dtype=torch.uint8)
    for edge, tie_up in ((0.25, 0), (0.75, 1), (1.25, 0), (1.75, 1), (2.5, 0), (3.5, 1), (5.0, 0)):
        code += (a >= edge) if tie_up else (a > edge)
    code = code | ((y < 0).to(torch.uint8) << 3)
    code = torch.where(bad[..., None], 0, code).to(torch.uint8).flatten(-2)
    byte = torch.where(bad, 255, e + 127).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte


def _values(codes, scales):
    """The fp32 values [..., 128] of code and exponent bytes."""
    grid = torch.tensor(GRID, device=codes.device)
    both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    v = grid[(both & 7).long()] * torch.where(both > 7, -1.0, 1.0)
    s = torch.where(scales == 255, float("nan"), _power(scales.int() - 127))
    return (v.unflatten(-1, (G, 32)) * s[..., None]).flatten(-2)


def _write(codes, scales, slots, c, b):
    page = codes.shape[3]
    p, o = slots.long() // page, slots.long() % page
    codes[p, :, :, o] = c
    scales[p, :, :, o] = b


def _plan(st):
    case, page = st["case"], st["case"]["page"]
    lens, table, free, n_free = (st[k].long() for k in ("lens", "table", "free", "n_free"))
    keep, grow = st["keep"].long(), st["grow"].long()
    p_old, p_keep = -(-lens // page), -(-keep // page)
    p_new = -(-(keep + grow) // page)
    freed, taken = p_old - p_keep, p_new - p_keep
    f_at, t_at = torch.cumsum(freed, 0) - freed, torch.cumsum(taken, 0) - taken
    n_freed, n_taken = freed.sum(), taken.sum()
    col = torch.arange(table.shape[1], device="cuda")[None]
    pool = free.numel()
    # what is put back, from the top of the free pages down
    gone = (col >= p_keep[:, None]) & (col < p_old[:, None])
    back = torch.full((pool + 1,), -1, dtype=torch.long, device="cuda")
    back.scatter_(0, torch.where(gone, f_at[:, None] + col - p_keep[:, None], pool).reshape(-1),
                  table.reshape(-1))
    def from_top(i):
        below = (n_free - 1 - (i - n_freed)).clamp(0, pool - 1)
        return torch.where(i < n_freed, back[i.clamp(0, pool - 1)], free[below])
    new = (col >= p_keep[:, None]) & (col < p_new[:, None])
    table = torch.where(new, from_top(t_at[:, None] + col - p_keep[:, None]),
                        torch.where(col < p_keep[:, None], table, -1))
    idx = torch.arange(pool, device="cuda")
    left = n_free + n_freed - n_taken
    free = torch.where(idx < left, from_top(n_free + n_freed - 1 - idx), -1)
    lens = keep + grow
    starts = torch.cat((torch.zeros_like(grow[:1]), torch.cumsum(grow, 0)))
    row = torch.arange(st["rows"], device="cuda")
    seq = torch.searchsorted(starts[1:], row, right=True)
    pos = keep[seq] + row - starts[seq]
    slots = table[seq, pos // page] * page + pos % page
    st["lens"], st["table"], st["free"], st["n_free"] = (
        t.to(torch.int32) for t in (lens, table, free, left))
    return [starts.to(torch.int32), slots.to(torch.int32), pos.to(torch.int32), st["lens"],
            st["table"], st["free"], st["n_free"]]


def _append(st):
    kv = st["kv"]
    c, b = _quantise(kv)
    _write(st["codes"], st["scales"], st["slots"], c, b)
    page = st["case"]["page"]
    p, o = st["slots"].long() // page, st["slots"].long() % page
    v = _values(st["codes"][p, :, :, o], st["scales"][p, :, :, o]).to(kv.dtype)
    return [v[:, 0], v[:, 1]]


def _attend(st):
    case, q = st["case"], st["q"]
    kv, heads = case["kv"], case["heads"]
    out = torch.zeros_like(q)
    at = 0
    for s, (m, n) in enumerate(zip(st["q_lens"], st["lens"])):
        if not m:
            continue
        x = _values(st["codes"][st["table"][s]], st["scales"][st["table"][s]])
        x = x.permute(1, 2, 0, 3, 4).reshape(2, kv, -1, D)[:, :, :n]     # [2, kv, n, 128]
        mine = q[at:at + m].float().reshape(m, kv, heads // kv, D)
        for h in range(kv):
            rows = mine[:, h].reshape(-1, D)                              # [m * ratio, 128]
            sc = (rows @ x[0, h].T) * (D ** -0.5)
            if case["causal"]:
                pos = torch.arange(m, device="cuda").repeat_interleave(heads // kv) + (n - m)
                sc = torch.where(torch.arange(n, device="cuda")[None] <= pos[:, None], sc,
                                 -float("inf"))
            w = torch.exp(sc - sc.amax(-1, keepdim=True))
            o = (w @ x[1, h]) / w.sum(-1, keepdim=True)
            r = heads // kv
            out[at:at + m, h * r:(h + 1) * r] = o.reshape(m, r, D).to(q.dtype)
        at += m
    return out


def run(state):
    """One call of the case's operator and its outputs."""
    kind = state["case"]["kind"]
    if not own:
        return {"plan": _plan, "append": _append, "attend": _attend}[kind](state)
    c = state["cache"]
    if kind == "plan":
        s = c.step(grow=state["grow"], keep=state["keep"], max_rows=state["rows"])
        return [s.starts, s.slots, s.positions, c.lens, c.table, c.free, c.n_free]
    if kind == "append":
        x = state["kv"]
        c.append(x[:, 0], x[:, 1], state["slots"])
        k, v = c.read(state["slots"], dtype=x.dtype)
        return [k, v]
    return c.attend(state["q"], state["starts"], causal=state["case"]["causal"])


def work(case):
    """Bytes and operations that one pass cannot do without."""
    page = case["page"]
    row = D // 2 + G     # bytes of one head's row in the cache
    if case["kind"] == "plan":
        keep, grow = _plan_sizes(case, 0)
        pages = sum(_pages(a + b, page) - _pages(a, page) for a, b in zip(keep, grow))
        # lengths in and out, starts; pages put back and taken; slots and positions
        return {"bytes": 20 * case["seqs"] + 12 * pages + 8 * sum(grow), "flops": 0}
    if case["kind"] == "append":
        n = case["rows"] * case["kv"] * 2
        # rows in and codes out, codes in and values out
        return {"bytes": n * (2 * D + row) + n * (row + 2 * D) + 8 * case["rows"],
                "flops": 2 * n * D}
    q, lens = _counts(case["q"], 1, 0), _counts(case["len"], 1, 0)
    seen = sum(sum(min(n, n - m + i + 1) for i in range(m)) if case["causal"] else m * n
               for m, n in zip(q, lens))
    rows = sum(n for m, n in zip(q, lens) if m)
    return {"bytes": rows * case["kv"] * 2 * row + 2 * sum(q) * case["heads"] * D * 2,
            "flops": 4 * D * seen * case["heads"]}


# ---------------------------------------------------------------------------- 64 bits


def _near64(x):
    """What the cache holds for x [..., 128], from its definition: the nearest grid value at the
    group's power of two."""
    x = x.double().unflatten(-1, (G, 32))
    top = x.abs().amax(-1, keepdim=True)
    mant, ex = torch.frexp(top)                       # top = mant * 2^ex, mant in [0.5, 1)
    e = torch.where(mant <= 0.875, ex - 3, ex - 2).clamp(min=-127)   # 7 * 2^-3 = 0.875
    unit = ((e.long() + 1023) << 52).view(torch.float64)              # 2^e, to the bit
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    a = x.abs() / unit
    hi = torch.searchsorted(grid, a.contiguous()).clamp(1, 7)
    lo = hi - 1
    up, down = grid[hi] - a, a - grid[lo]
    take = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), grid[hi], grid[lo])
    return (torch.sign(x) * take * unit).flatten(-2)


def exact(case, seed):
    if case["kind"] == "plan":
        return None
    dtype, kv = DTYPES[case["dtype"]], case["kv"]
    if case["kind"] == "append":
        x = _near64(_kv_rows(case["rows"], kv, dtype, seed, 4))
        return [x[:, 0], x[:, 1]]
    q_lens, lens = _counts(case["q"], 1, 0), _counts(case["len"], 1, 0)
    ratio = case["heads"] // kv
    q = _q_rows(sum(q_lens), case["heads"], dtype, seed)
    parts = []
    at = 0
    for s, (m, n) in enumerate(zip(q_lens, lens)):
        rows = q[at:at + m].double()
        at += m
        if not m:
            continue
        x = _near64(_kv_rows(n, kv, dtype, seed, 16 + s))
        heads = []
        for h in range(case["heads"]):
            logit = rows[:, h] @ x[:, 0, h // ratio].T / math.sqrt(D)
            if case["causal"]:
                ahead = torch.ones((m, n), dtype=torch.bool, device="cuda").triu(n - m + 1)
                logit = logit.masked_fill(ahead, -math.inf)
            heads.append(torch.softmax(logit, -1) @ x[:, 1, h // ratio])
        parts.append(torch.stack(heads, 1))
    return torch.cat(parts)
