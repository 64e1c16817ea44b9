"""Performance cases of several candidates of one request: what a serving program runs when it
drafts, forks and verifies more than one continuation of the same context.

  verify  ``verify_draft``: drafted blocks judged against the target's distributions by given
          uniform numbers, and each sequence's next token drawn from what is left;
  fork    ``KV4Cache.step`` with ``parent`` on a cache whose sequences share pages: continuations
          of other sequences without copying them, pages counted, a shared page copied for the
          sequence that writes into it;
  shared  ``KV4Cache.attend`` with ``groups``: the pages that a group's sequences share are
          attended once for all of the group's rows, each sequence's own rows after that.

Verification.  Rows starts[s] .. starts[s + 1] - 1 of the logits are sequence s's block: row 0
holds the last verified token, the others drafted ones.  With p the softmax of the target's row
over its temperature and q that of the draft's (all weight on the largest logit, the first of
equals, for a temperature of zero; all of q's weight on the drafted token where there are no
draft logits), the token x of row t is accepted with the chance min(1, p(x) / q(x)) of row t - 1's
p and row t's q: if u[t] q(x) < p(x).  Behind the accepted rows a token is drawn: from
max(p - q, 0) after a rejection, from p after none, as the first i whose running sum exceeds
u[row 0] times the whole.

``own`` selects the package's kernels; where it is false the same results come from elementary
torch operations.
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

D = 128          # head dimension
G = D // 32      # groups of a cached row
BLOCK = 4352     # bytes of 32 cached rows of one head
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # One request, the 8B draft's block of 16: latency.
        {"name": "verify_block_16", "kind": "verify", "rows": "16", "vocab": 151936,
         "target": "bfloat16", "draft": "float32", "temps": "1.0"},
        # The batched benchmark: eight sequences, blocks of 32, drafted greedily.
        {"name": "verify_greedy_8", "kind": "verify", "rows": "32 32 32 32 32 32 32 32",
         "vocab": 128256, "target": "float16", "draft": "none", "temps": "0.7"},
        # A batch of requests with settings of their own (some greedy), ragged blocks, one idle
        # sequence, a vocabulary whose rows begin at odd addresses.
        {"name": "verify_ragged_48", "kind": "verify",
         "rows": " ".join(str(0 if i == 7 else 1 + (5 * i) % 16) for i in range(48)), "vocab": 32003,
         "target": "bfloat16", "draft": "bfloat16", "temps": "mix"},
        # A server's 64 requests with blocks of 32.
        {"name": "verify_batch_64", "kind": "verify", "rows": " ".join(["32"] * 64),
         "vocab": 151936, "target": "bfloat16", "draft": "bfloat16", "temps": "1.0"},
        # Eight candidate blocks behind one context: the others continue the first.
        {"name": "fork_candidates_8", "kind": "fork", "page": 64, "kv": 8, "layers": 5,
         "groups": 1, "size": 8, "len": 4114, "forked": 1.0, "grow": 32},
        # A decode step of 256 sequences that share pages of old, of which none forks.
        {"name": "fork_none_256", "kind": "fork", "page": 32, "kv": 4, "layers": 1,
         "groups": 64, "size": 4, "len": 1500, "forked": 0.0, "grow": 1},
        # Beams: 16 requests of 4, each step some beams continue others.
        {"name": "fork_beams_64", "kind": "fork", "page": 64, "kv": 8, "layers": 2,
         "groups": 16, "size": 4, "len": 2777, "forked": 0.5, "grow": 1},
        # Sixteen samples of each of 64 long prompts, all begun in one step.
        {"name": "fork_samples_1024", "kind": "fork", "page": 128, "kv": 2, "layers": 1,
         "groups": 64, "size": 16, "len": 6000, "forked": 1.0, "grow": 8},
        # Eight candidates' first tokens behind one context, the 27B draft's heads: latency.
        {"name": "shared_tokens_8", "kind": "shared", "heads": 40, "kv": 8, "page": 64,
         "sizes": "8", "prefix": "4096", "own": "mix 1 40", "q": 1, "causal": True,
         "dtype": "float16"},
        # Draft blocks of 8 rows for four candidates each of four requests.
        {"name": "shared_blocks_16", "kind": "shared", "heads": 32, "kv": 8, "page": 64,
         "sizes": "4 4 4 4", "prefix": "4178 811 7844 1651", "own": "mix 8 300", "q": 8,
         "causal": False, "dtype": "float16"},
        # A decode step of 64 requests behind three system prompts, a few without one.
        {"name": "shared_tokens_64", "kind": "shared", "heads": 32, "kv": 8, "page": 32,
         "sizes": "33 17 10 1 1 1 1", "prefix": "2048 8000 5001 0 0 0 0", "own": "mix 1 2000",
         "q": 1, "causal": True, "dtype": "bfloat16"},
        # 128 questions about one long document.
        {"name": "shared_tokens_128", "kind": "shared", "heads": 64, "kv": 8, "page": 64,
         "sizes": "128", "prefix": "32768", "own": "mix 16 1000", "q": 1, "causal": True,
         "dtype": "bfloat16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["verify", "verify", "fork", "shared", "shared"])
    if kind == "verify":
        seqs, block = _log_int(rng, 1, 64), rng.randint(1, 32)
        ragged = rng.random() < 0.5
        rows = [rng.randint(0 if i else 1, block) if ragged else block for i in range(seqs)]
        return {"kind": kind, "rows": " ".join(map(str, rows)), "vocab": _log_int(rng, 1000, 151936),
                "target": rng.choice(sorted(DTYPES)), "draft": rng.choice(sorted(DTYPES) + ["none"]),
                "temps": rng.choice(["mix", "%.2f" % rng.uniform(0.2, 1.5)])}
    page = rng.choice([32, 64, 128])
    if kind == "fork":
        groups, size = _log_int(rng, 1, 64), _log_int(rng, 1, 16)
        longest = min(8000, 100000 // groups)
        return {"kind": kind, "page": page, "kv": rng.choice([1, 2, 3, 4]),
                "layers": rng.randint(1, 3), "groups": groups, "size": size,
                "len": _log_int(rng, 40, longest), "forked": rng.choice([0.0, 0.3, 0.7, 1.0]),
                "grow": _log_int(rng, 1, 64)}
    kv = rng.choice([1, 2, 4, 8])
    sizes = [_log_int(rng, 1, 32) for _ in range(rng.randint(1, 4))]
    prefix = [_log_int(rng, 100, 20000) if n > 1 else 0 for n in sizes]
    q = rng.choice([1, 1, 1, rng.randint(2, 16)])
    return {"kind": kind, "heads": kv * rng.choice([1, 3, 4, 5, 7, 8]), "kv": kv, "page": page,
            "sizes": " ".join(map(str, sizes)), "prefix": " ".join(map(str, prefix)),
            "own": "mix %d %d" % (q, q + _log_int(rng, 1, 1500)), "q": q,
            "causal": q == 1 or rng.random() < 0.5, "dtype": rng.choice(["float16", "bfloat16"])}


# ---------------------------------------------------------------------------- inputs


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mirror-sd_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import mirror_sd_amd
    return mirror_sd_amd


def _numbers(text):
    return [int(w) for w in text.split()]


def _pages(n, page):
    return -(-n // page)


def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed(seed * 1000003 + salt)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _ends(x):
    return [sum(x[:i]) for i in range(len(x) + 1)]


# ---- verification


def _verify_inputs(case, seed):
    """Target logits with a few likely tokens in each row, a draft near them, tokens drawn from
    the draft (or its likeliest), uniform numbers, and a temperature for each sequence."""
    rows, vocab = _numbers(case["rows"]), case["vocab"]
    n, seqs = sum(rows), len(rows)
    g = _gen(seed, 1)
    starts = _ints(_ends(rows))
    seq = torch.repeat_interleave(torch.arange(seqs, device="cuda"), _ints(rows).long(),
                                  output_size=n)
    if case["temps"] == "mix":   # some greedy, the rest from cool to warm
        temps = 0.3 + 1.1 * torch.rand(seqs, generator=g, device="cuda")
        temps = torch.where(torch.arange(seqs, device="cuda") % 5 == 3, 0.0, temps)
    else:
        temps = torch.full((seqs,), float(case["temps"]), device="cuda")
    target = 1.5 * torch.randn((n, vocab), generator=g, device="cuda")
    likely = torch.randint(vocab, (n, 12), generator=g, device="cuda")
    peaks = 6.0 + 6.0 * torch.rand((n, 12), generator=g, device="cuda")
    target.scatter_add_(1, likely, peaks)
    near = torch.randn((n, vocab), generator=g, device="cuda").mul_(0.6)
    near[1:] += target[:-1]        # row t's draft is of what row t - 1's target goes on with
    target = target.to(DTYPES[case["target"]])
    draft = None
    if case["draft"] == "none":
        ids = near.argmax(1)
    else:
        draft = near.to(DTYPES[case["draft"]])
        noise = torch.rand((n, vocab), generator=g, device="cuda").clamp_(min=1e-30).log_().neg_().log_()
        t = temps[seq].clamp(min=1e-6)[:, None]
        ids = (near.copy_(draft).div_(t) - noise).argmax(1)
    u = torch.rand(n, generator=g, device="cuda")
    return target, ids.to(torch.int32), starts, u, temps, draft


def _prepare_verify(case, seed):
    target, ids, starts, u, temps, draft = _verify_inputs(case, seed)
    st = {"case": case, "target": target, "ids": ids, "starts": starts, "u": u, "draft": draft}
    one = case["temps"] != "mix"
    st["temp"] = float(case["temps"]) if one else temps
    if own:
        st["call"] = _package().verify_draft
    return st


def _chances(logits, temp):
    """Rows of softmax(logits / temp) in 64 bits; all weight on the first largest for temp 0."""
    x = logits.double()
    top = x.amax(1, keepdim=True)
    w = torch.exp((x - top) / torch.where(temp < 1e-5, 1.0, temp)[:, None])
    w = w / w.sum(1, keepdim=True)
    at = torch.arange(x.shape[1], device="cuda")
    first = torch.where(x == top, at, x.shape[1]).amin(1, keepdim=True)
    return torch.where((temp < 1e-5)[:, None], (at == first).double(), w)


def _verify(st):
    target, ids, starts, u = st["target"], st["ids"].long(), st["starts"].long(), st["u"].double()
    n, seqs = ids.shape[0], starts.shape[0] - 1
    row = torch.arange(n, device="cuda")
    seq = torch.searchsorted(starts, row, right=True) - 1
    first = row == starts[seq]
    temp = st["temp"]
    temp = (temp[seq] if isinstance(temp, torch.Tensor) else torch.full((n,), temp, device="cuda")).double()
    p = _chances(target, temp)
    before = (row - 1).clamp(min=0)
    px = p[before, ids]
    q = None if st["draft"] is None else _chances(st["draft"], temp)
    qx = torch.ones_like(px) if q is None else q[row, ids]
    chance = torch.where(px > 0, (px / qx.clamp(min=1e-300)).clamp(max=1.0), 0.0)
    chance = torch.where(first, 1.0, chance)
    ok = first | (u * qx < px)
    # each sequence's first rejected row, or its end
    stop = starts[1:].scatter_reduce(0, seq, torch.where(ok, n, row), "amin")
    idle = starts[1:] == starts[:-1]
    some = (stop < starts[1:]) & ~idle                   # a row was rejected
    last = (stop - 1).clamp(0, n - 1)
    at = stop.clamp(max=n - 1)
    r = p[last]
    if q is None:
        hit = torch.arange(r.shape[1], device="cuda") == ids[at][:, None]
        left = torch.where(hit, 0.0, r)
    else:
        left = (r - q[at]).clamp(min=0.0)
    left = torch.where((left.sum(1) > 0)[:, None], left, r)
    r = torch.where(some[:, None], left, r)
    sums = torch.cumsum(r, 1)
    v = u[starts[:-1].clamp(max=n - 1)] * sums[:, -1]
    i = torch.searchsorted(sums, v[:, None], right=True)[:, 0]
    cols = torch.arange(r.shape[1], device="cuda")
    i = torch.minimum(i, torch.where(r > 0, cols, 0).amax(1))
    return [torch.where(idle, 0, stop - 1 - starts[:-1]).to(torch.int32),
            torch.where(idle, -1, i).to(torch.int32), chance.float()]


def _verify_exact(case, seed):
    target, ids, starts, u, temps, draft = _verify_inputs(case, seed)
    rows = _numbers(case["rows"])
    n = sum(rows)
    seq = torch.repeat_interleave(torch.arange(len(rows), device="cuda"), _ints(rows).long())
    t = temps.double()[seq]
    greedy = t < 1e-5
    x = ids.long()[:, None]
    def log_of(z, tokens):       # log softmax(z / t) at the tokens
        z = z.double()
        best = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :1]   # first of equals
        hard = torch.where(best == tokens, 0.0, -math.inf)[:, 0]
        z = z / torch.where(greedy, 1.0, t)[:, None]
        return torch.where(greedy, hard, (z.gather(1, tokens) - torch.logsumexp(z, 1, keepdim=True))[:, 0])
    behind = log_of(target, torch.roll(x, -1, 0)).roll(1)    # of row t's token under row t - 1
    if draft is not None:
        behind = behind - log_of(draft, x)
    out = torch.exp(behind.clamp(max=0.0))
    out[starts[:-1][_ints(rows) > 0].long()] = 1.0
    return [None, None, out]


# ---- the cache


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


def _fork_sizes(case, seed):
    """Groups of sequences, each of which continues its group's first or another that goes on:
    (parent, kept rows) of every sequence.  A step puts back and copies the same pages again when
    it is repeated."""
    rng, sizes = random.Random(seed), random.Random(case["len"])
    parent, keep = [], []
    for g in range(case["groups"]):
        first = g * case["size"]
        n = max(1, case["len"] - sizes.randint(0, case["len"] // 4))
        stay = [first]
        for s in range(first, first + case["size"]):
            if s > first and rng.random() < case["forked"]:
                parent.append(rng.choice(stay))
            else:
                parent.append(s)
                stay.append(s)
            keep.append(n)
    return parent, keep


def _prepare_fork(case, seed):
    """A cache in which the sequences of a group share all but their last page, with codes of
    random bits (a copy takes them as they are)."""
    page, kv, layers, size = case["page"], case["kv"], case["layers"], case["size"]
    parent, keep = _fork_sizes(case, seed)
    grow = [case["grow"]] * len(keep)
    lens = [k + n for k, n in zip(keep, grow)]
    width = _pages(max(lens) + 1, page) + 1
    held = [_pages(n, page) for n in lens]
    need = sum(held[s] if s % size == 0 else held[s] - k // page for s, k in enumerate(keep))
    pool = need + 9
    order = list(range(pool))
    random.Random(seed + 1).shuffle(order)
    table, at = [], 0
    for s, k in enumerate(keep):
        shared = [] if s % size == 0 else table[s - s % size][:k // page]
        new = held[s] - len(shared)
        table.append(shared + order[at:at + new] + [-1] * (width - held[s]))
        at += new
    tab = _ints(table)
    refs = torch.bincount(torch.where(tab < 0, pool, tab).reshape(-1), minlength=pool + 1)[:pool]
    shape = (layers, pool + 1, kv, page // 32, BLOCK)    # (one for what the plain form does not copy)
    bits = torch.randint(256, shape, generator=_gen(seed, 2), device="cuda", dtype=torch.uint8)
    st = {"case": case, "parent": _ints(parent), "keep": _ints(keep), "grow": _ints(grow),
          "rows": sum(grow)}
    state = {"lens": _ints(lens), "table": tab, "refs": refs.to(torch.int32),
             "n_free": _ints([pool - at])}
    if own:
        c = _package().KV4Cache(n_kv_heads=kv, n_pages=pool, max_seqs=len(keep),
                                max_len=width * page, page=page, n_layers=layers, shared=True)
        for name, t in state.items():
            getattr(c, name).copy_(t)
        c.pool.copy_(bits[:, :pool])
        st["cache"] = c
    else:
        st.update(state, pool=bits)
    return st


def _fork(st):
    case, page = st["case"], st["case"]["page"]
    table, parent, keep, grow = (st[k].long() for k in ("table", "parent", "keep", "grow"))
    seqs, width = table.shape
    pool = st["refs"].numel()
    col = torch.arange(width, device="cuda")[None]
    s = torch.arange(seqs, device="cuda")
    p_keep, p_new = -(-keep // page), -(-(keep + grow) // page)
    held = torch.where(col < p_keep[:, None], table[parent], pool)
    count = torch.bincount(held.reshape(-1), minlength=pool + 1)
    count[pool] = 0
    # sequences that write into their last kept page, and who copies it
    writes = (grow > 0) & (keep % page != 0)
    edge = torch.where(writes, held.gather(1, (p_keep - 1).clamp(min=0)[:, None])[:, 0], pool)
    writers = torch.bincount(edge, minlength=pool + 1)
    first = torch.full((pool + 1,), seqs, device="cuda").scatter_reduce(0, edge, s, "amin")
    stays = (count[edge] == writers[edge]) & (first[edge] == s)
    copies = writes & ~stays
    # free pages, the lowest first
    free = count[:pool] == 0
    rank = torch.cumsum(free.long(), 0) - 1
    taken = p_new - p_keep + copies
    at = torch.cumsum(taken, 0) - taken
    page_of = torch.full((pool + 1,), -1, device="cuda").scatter_(
        0, torch.where(free, rank, pool), torch.arange(pool, device="cuda"))
    fresh = page_of[(at[:, None] + copies[:, None] + col - p_keep[:, None]).clamp(0, pool - 1)]
    new = torch.where(col < p_keep[:, None], held, torch.where(col < p_new[:, None], fresh, -1))
    mine = page_of[at.clamp(max=pool - 1)]
    new = torch.where(copies[:, None] & (col == p_keep[:, None] - 1), mine[:, None], new)
    # the copied pages, blocks that hold kept rows whole
    blocks = torch.arange(page // 32, device="cuda")[None] * 32 < (keep % page)[:, None]
    src, dst = torch.where(copies, edge, pool), torch.where(copies, mine, pool)
    bits = st["pool"]
    bits[:, dst] = torch.where(blocks[None, :, None, :, None], bits[:, src], bits[:, dst])
    ends = torch.cat((torch.zeros_like(grow[:1]), torch.cumsum(grow, 0)))
    row = torch.arange(st["rows"], device="cuda")
    seq = torch.searchsorted(ends[1:], row, right=True)
    pos = keep[seq] + row - ends[seq]
    slots = new[seq, pos // page] * page + pos % page
    refs = torch.bincount(torch.where(new < 0, pool, new).reshape(-1), minlength=pool + 1)[:pool]
    st["lens"], st["table"], st["refs"], st["n_free"] = (
        t.to(torch.int32) for t in (keep + grow, new, refs, (refs == 0).sum()[None]))
    return [ends.to(torch.int32), slots.to(torch.int32), pos.to(torch.int32), st["lens"],
            st["table"], st["refs"], st["n_free"], bits[:, :pool]]


# ---- attention


def _shared_sizes(case):
    """(group, shared rows, rows in all) of every sequence."""
    sizes, prefix = _numbers(case["sizes"]), _numbers(case["prefix"])
    lo, hi = _numbers(case["own"][4:])
    rng = random.Random(lo * 31 + hi)
    return [(g, prefix[g], prefix[g] + rng.randint(lo, hi))
            for g, n in enumerate(sizes) for _ in range(n)]


def _shared_rows(case, seed):
    """Each group's shared rows, and each sequence's own."""
    kv, dtype = case["kv"], DTYPES[case["dtype"]]
    prefix = [_kv_rows(n, kv, dtype, seed, 16 + g) for g, n in enumerate(_numbers(case["prefix"]))]
    mine = [_kv_rows(n - m, kv, dtype, seed, 1000 + s)
            for s, (_, m, n) in enumerate(_shared_sizes(case))]
    return prefix, mine


def _q_rows(case, seed):
    n = sum(_numbers(case["sizes"])) * case["q"]
    return torch.randn((n, case["heads"], D), generator=_gen(seed, 2),
                       device="cuda").to(DTYPES[case["dtype"]])


def _prepare_shared(case, seed):
    page, kv = case["page"], case["kv"]
    sizes, seqs = _numbers(case["sizes"]), _shared_sizes(case)
    prefix, mine = _shared_rows(case, seed)
    q = case["q"]
    st = {"case": case, "q": _q_rows(case, seed)}
    pool = sum(_pages(len(x), page) + 1 for x in prefix) + sum(_pages(n, page) - m // page + 1 for _, m, n in seqs)
    if own:
        c = _package().KV4Cache(n_kv_heads=kv, n_pages=pool, max_seqs=len(seqs),
                                max_len=max(n for _, _, n in seqs), page=page, shared=True)
        ends = _ends(sizes)
        first = [ends[g] for g, _, _ in seqs]
        grow = [m if s == first[s] else 0 for s, (_, m, _) in enumerate(seqs)]
        rows = torch.cat(prefix)
        c.append(rows[:, 0], rows[:, 1], c.step(grow=grow).slots)
        rows = torch.cat(mine)
        slots = c.step(grow=[n - m for _, m, n in seqs], keep=[m for _, m, _ in seqs],
                       parent=first).slots
        c.append(rows[:, 0], rows[:, 1], slots)
        st.update(cache=c, starts=_ints([q * s for s in range(len(seqs) + 1)]), groups=_ints(ends))
        return st
    codes, scales = _pool(pool, kv, page)
    heads, tables, at = [], [], 0
    def place(rows, at):         # rows into pages from number `at` on
        slots = at * page + torch.arange(len(rows), device="cuda")
        _write(codes, scales, slots, *_quantise(rows))
        return list(range(at, at + _pages(len(rows), page)))
    for x in prefix:
        heads.append(place(x, at))
        at += len(heads[-1])
    for s, (g, m, n) in enumerate(seqs):
        full = m // page
        rest = place(torch.cat((prefix[g][full * page:], mine[s])), at)
        at += len(rest)
        tables.append(torch.tensor(heads[g][:full] + rest, device="cuda"))
    st.update(codes=codes, scales=scales, tables=tables, lens=[n for _, _, n in seqs])
    return st


def _pool(pages, kv, page):
    """Codes [pages, 2, kv, page, 64] (two values a byte, the even one low) and exponent bytes
    [pages, 2, kv, page, 4]."""
    return (torch.zeros((pages, 2, kv, page, D // 2), dtype=torch.uint8, device="cuda"),
            torch.zeros((pages, 2, kv, page, G), dtype=torch.uint8, device="cuda"))


def _power(e):
    """2^e in fp32, exact, for -127 <= e <= 127 (2^-127 is subnormal)."""
    return torch.where(e > -127, (e + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _quantise(x):
    """x [..., 128] -> code bytes [..., 64], exponent bytes [..., 4]: the smallest exponent with the
    group's largest magnitude at most 7 units, codes to the nearest, ties to the even one."""
    x = x.float().unflatten(-1, (G, 32))
    bits = x.abs().amax(-1).view(torch.int32)
    e = ((bits >> 23) - 129 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp(min=-127)
    y = x * _power(-e)[..., None]
    a = y.abs()
    code = torch.zeros_like(a, dtype=torch.uint8)
    for edge, tie_up in ((0.25, 0), (0.75, 1), (1.25, 0), (1.75, 1), (2.5, 0), (3.5, 1), (5.0, 0)):
        code += (a >= edge) if tie_up else (a > edge)
    code = (code | ((y < 0).to(torch.uint8) << 3)).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8)


def _values(codes, scales):
    """The fp32 values [..., 128] of code and exponent bytes."""
    grid = torch.tensor(GRID, device=codes.device)
    both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    v = grid[(both & 7).long()] * torch.where(both > 7, -1.0, 1.0)
    return (v.unflatten(-1, (G, 32)) * _power(scales.int() - 127)[..., None]).flatten(-2)


def _write(codes, scales, slots, c, b):
    page = codes.shape[3]
    p, o = slots.long() // page, slots.long() % page
    codes[p, :, :, o] = c
    scales[p, :, :, o] = b


def _shared(st):
    case = st["case"]
    kv, heads, q = case["kv"], case["heads"], case["q"]
    ratio = heads // kv
    held = _values(st["codes"], st["scales"])                          # every page once
    out = torch.empty_like(st["q"])
    for s, (tab, n) in enumerate(zip(st["tables"], st["lens"])):
        x = held[tab].permute(1, 2, 0, 3, 4).reshape(2, kv, -1, D)[:, :, :n]
        mine = st["q"][q * s:q * s + q].float().reshape(q, kv, ratio, D).transpose(0, 1)
        sc = (mine.reshape(kv, q * ratio, D) @ x[0].transpose(1, 2).contiguous()) * (D ** -0.5)
        if case["causal"]:
            pos = torch.arange(q, device="cuda").repeat_interleave(ratio) + (n - q)
            sc = torch.where(torch.arange(n, device="cuda") <= pos[:, None], sc, -float("inf"))
        w = torch.exp(sc - sc.amax(-1, keepdim=True))
        o = (w @ x[1]) / w.sum(-1, keepdim=True)
        out[q * s:q * s + q] = o.reshape(kv, q, ratio, D).transpose(0, 1).reshape(q, heads, D).to(out.dtype)
    return out


def _near64(x):
    """What the cache holds for x [..., 128], from its definition: the nearest grid value at the
    group's power of two."""
    x = x.double().unflatten(-1, (G, 32))
    mant, ex = torch.frexp(x.abs().amax(-1, keepdim=True))   # mant * 2^ex, mant in [0.5, 1)
    e = torch.where(mant <= 0.875, ex - 3, ex - 2).clamp(min=-127)   # 7 * 2^-3 = 0.875
    unit = ((e.long() + 1023) << 52).view(torch.float64)              # 2^e, to the bit
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    a = x.abs() / unit
    hi = torch.searchsorted(grid, a.contiguous()).clamp(1, 7)
    lo = hi - 1
    up, down = grid[hi] - a, a - grid[lo]
    take = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), grid[hi], grid[lo])
    return (torch.sign(x) * take * unit).flatten(-2)


def _shared_exact(case, seed):
    kv, heads, m = case["kv"], case["heads"], case["q"]
    rows = _q_rows(case, seed).double()
    prefix, mine = _shared_rows(case, seed)
    prefix = [_near64(x) for x in prefix]
    parts = []
    for s, (g, _, n) in enumerate(_shared_sizes(case)):
        x = torch.cat((prefix[g], _near64(mine[s])))
        k, v = (x[:, i].repeat_interleave(heads // kv, 1).permute(1, 0, 2).contiguous() for i in (0, 1))
        logit = rows[m * s:m * s + m].permute(1, 0, 2) @ k.transpose(1, 2).contiguous() / math.sqrt(D)
        if case["causal"]:
            ahead = torch.ones((m, n), dtype=torch.bool, device="cuda").triu(n - m + 1)
            logit = logit.masked_fill(ahead, -math.inf)
        parts.append((torch.softmax(logit, -1) @ v).permute(1, 0, 2))
    return torch.cat(parts)


# ---------------------------------------------------------------------------- the interface


def prepare(case, seed):
    torch.cuda.set_device(0)
    return {"verify": _prepare_verify, "fork": _prepare_fork, "shared": _prepare_shared}[case["kind"]](case, seed)


def run(state):
    """One call of the case's operator and its outputs."""
    kind = state["case"]["kind"]
    if not own:
        return {"verify": _verify, "fork": _fork, "shared": _shared}[kind](state)
    if kind == "verify":
        v = state["call"](state["target"], state["ids"], state["starts"], state["u"],
                          temperature=state["temp"], draft_logits=state["draft"])
        return [v.accepted, v.next_ids, v.chances]
    c = state["cache"]
    if kind == "fork":
        s = c.step(grow=state["grow"], keep=state["keep"], parent=state["parent"],
                   max_rows=state["rows"])
        return [s.starts, s.slots, s.positions, c.lens, c.table, c.refs, c.n_free, c.pool]
    return c.attend(state["q"], state["starts"], causal=state["case"]["causal"],
                    groups=state["groups"])


def work(case):
    """Bytes and operations that one pass cannot do without."""
    if case["kind"] == "verify":
        rows, vocab = _numbers(case["rows"]), case["vocab"]
        size = {"float32": 4, "float16": 2, "bfloat16": 2, "none": 0}
        n = sum(rows)
        drafted = sum(max(0, r - 1) for r in rows)
        # the logits, ids, numbers and starts in; two numbers a sequence and the chances out
        return {"bytes": vocab * (n * size[case["target"]] + drafted * size[case["draft"]]) +
                12 * n + 12 * len(rows), "flops": 4 * vocab * (n + (drafted if size[case["draft"]] else 0))}
    page = case["page"]
    if case["kind"] == "fork":
        parent, keep = _fork_sizes(case, 0)
        grow, size = case["grow"], case["size"]
        moved = copied = 0
        for s, (p, k) in enumerate(zip(parent, keep)):
            forks = p != s
            # places of the table that change, pages counted up and down; blocks copied
            moved += 2 * _pages(k, page) if forks else 0
            moved += 2 * (_pages(k + grow, page) - _pages(k, page))
            if forks and k % page:
                copied += _pages(k % page, 32) * case["kv"] * case["layers"] * BLOCK
        n = len(keep)
        return {"bytes": 28 * n + 12 * moved + 8 * n * grow + 2 * copied, "flops": 0}
    row = 2 * case["kv"] * (D // 2 + G)     # bytes of a cached row's keys and values
    seqs, q = _shared_sizes(case), case["q"]
    seen = sum(sum(n - q + i + 1 for i in range(q)) if case["causal"] else q * n for _, _, n in seqs)
    rows = sum(_numbers(case["prefix"])) + sum(n - m for _, m, n in seqs)
    return {"bytes": rows * row + 4 * len(seqs) * q * case["heads"] * D,
            "flops": 4 * D * seen * case["heads"]}


def exact(case, seed):
    """The outputs' values from their definition in 64 bits (None: whole numbers)."""
    if case["kind"] == "verify":
        return _verify_exact(case, seed)
    if case["kind"] == "shared":
        return _shared_exact(case, seed)
    return None
