"""The operators of a serving step over many requests, as cases that can be timed
and checked: page tables and slot maps from request lengths, rows of keys and
values appended to an 8-bit paged cache, attention over that cache, and tokens
sampled from logits.

Sizes are those of the BitNet-2B shape that bench.py measures (20 query and 5
key/value heads of 128, vocab 128256), of the tests' smaller shape (16 and 4
heads of 64), or generic.  Random numbers are inputs, made from the seed.

With `own` false, `run` is the plain form in elementary torch operations; with
`own` true it makes the calls of loom_amd.paged and loom_amd.transformer that
a user makes.
"""
import math

import numpy as np
import torch

own = False

SHAPES = {"2b": (20, 5, 128), "small": (16, 4, 64)}
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # the tables of a decode step: one new token for each of 64 requests
        dict(name="plan_decode", kind="plan", requests=64, longest=4096, new=1, page=16, fresh=False),
        # a scheduler that rebuilds every table: 1000 prompts of ragged length
        dict(name="plan_admit", kind="plan", requests=1000, longest=400, new=0, page=16, fresh=True),
        # one decode step's keys and values of 64 requests, amid their pages
        dict(name="append_decode", kind="append", requests=64, longest=1, shape="2b", page=16, dtype="fp32"),
        # the keys and values of prompts, whole pages at a time
        dict(name="append_prompts", kind="append", requests=9, longest=2048, shape="2b", page=32, dtype="bf16"),
        # one request's next token after a 2048-token prompt
        dict(name="attend_row", kind="attend", chunks=0, chunk=0, rows=1, context=2177, ragged=False, shape="2b",
             page=16, dtype="fp32"),
        # one decode step of 64 requests at all lengths
        dict(name="attend_decode", kind="attend", chunks=0, chunk=0, rows=64, context=4096, ragged=True, shape="2b",
             page=16, dtype="bf16"),
        # a few requests with very long contexts, where the bytes of the cache count
        dict(name="attend_long", kind="attend", chunks=0, chunk=0, rows=7, context=65536, ragged=False, shape="2b",
             page=64, dtype="fp32"),
        # four prompts at once, where the products count
        dict(name="attend_prompts", kind="attend", chunks=4, chunk=2048, rows=0, context=2048, ragged=False,
             shape="2b", page=16, dtype="fp32"),
        # a chunk of a long prompt in the same step as the decode rows of others, small heads
        dict(name="attend_mixed", kind="attend", chunks=1, chunk=509, rows=31, context=3000, ragged=True,
             shape="small", page=16, dtype="bf16"),
        # one request's token from a full vocabulary, all filters on
        dict(name="sample_row", kind="sample", rows=1, vocab=128256, filters="all"),
        # a batch whose requests each ask for something else
        dict(name="sample_mixed", kind="sample", rows=63, vocab=128256, filters="mixed"),
        # many rows of a nucleus over the full vocabulary
        dict(name="sample_nucleus", kind="sample", rows=256, vocab=128256, filters="nucleus"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["plan", "append", "attend", "attend", "attend", "sample", "sample"])
    if kind == "plan":
        fresh = rng.random() < 0.5
        return dict(kind=kind, requests=_log(rng, 1, 1000), longest=_log(rng, 20, 400) if fresh else _log(rng, 50, 4096),
                    new=0 if fresh else rng.choice([1, 1, 4]), page=rng.choice([16, 32, 64]), fresh=fresh)
    if kind == "append":
        longest = rng.choice([1, 1, 5, _log(rng, 2, 2048)])
        return dict(kind=kind, requests=_log(rng, 1, 64 if longest < 8 else 8), longest=longest,
                    shape=rng.choice(["2b", "small"]), page=rng.choice([16, 32, 64]),
                    dtype=rng.choice(["fp32", "bf16"]))
    if kind == "attend":
        chunked = rng.random() < 0.5
        return dict(kind=kind, chunks=rng.choice([1, 1, 2, 3]) if chunked else 0,
                    chunk=_log(rng, 2, 1500) if chunked else 0, rows=rng.choice([0, 7, 20]) if chunked else _log(rng, 1, 64),
                    context=_log(rng, 20, 2048) if chunked else _log(rng, 20, 7000), ragged=rng.random() < 0.6,
                    shape=rng.choice(["2b", "small"]), page=rng.choice([16, 32, 64]),
                    dtype=rng.choice(["fp32", "bf16"]))
    return dict(kind=kind, rows=_log(rng, 1, 200), vocab=rng.choice([128256, 32000, _log(rng, 300, 128256)]),
                filters=rng.choice(["all", "mixed", "nucleus", "topk", "none"]))


# ---- inputs -----------------------------------------------------------------

def _gen(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(seed)


def _ints(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def _order(n, seed):
    return np.random.default_rng(seed).permutation(n)


# Lengths are the case's own, so that outputs have one shape and a pass one
# size of work; the seed says which request has which.

def _plan_lengths(case, seed):
    """(tokens held before, new tokens) of each request."""
    n = case["requests"]
    lens = np.random.default_rng(n).integers(1, case["longest"] + 1, n)[_order(n, seed)]
    if case["fresh"]:
        return np.zeros(n, np.int64), lens
    return lens, np.full(n, case["new"], np.int64)


def _append_lengths(case, seed):
    n = case["requests"]
    r, order = np.random.default_rng(n), _order(n, seed)
    if case["longest"] < 8:  # decode rows fall anywhere in their pages
        return r.integers(0, 500, n)[order], np.full(n, case["longest"], np.int64)
    before = r.integers(0, 3 * case["page"], n)
    return before[order], r.integers(case["longest"] // 2, case["longest"] + 1, n)[order]


def _attend_lengths(case, seed):
    """(context with the new rows, new rows) of each request."""
    r = np.random.default_rng(case["context"])
    ctx, new = [], []
    for _ in range(case["chunks"]):
        new.append(case["chunk"])
        ctx.append(max(case["chunk"], case["context"]))
    for _ in range(case["rows"]):
        new.append(1)
        ctx.append(int(r.integers(1, case["context"] + 1)) if case["ragged"] else case["context"])
    order = _order(len(ctx), seed)
    return np.array(ctx)[order], np.array(new)[order]


def _page_ids(pages_of, seed):
    """Shuffled page ids of each request as a padded table, and the pool's size."""
    total = int(pages_of.sum())
    ids = np.random.default_rng(seed + 1).permutation(total + 3)[:total]
    table = np.full((len(pages_of), max(1, int(pages_of.max()))), -1, np.int64)
    at = 0
    for i, n in enumerate(pages_of):
        table[i, :n] = ids[at:at + n]
        at += n
    return table, total + 3


def _slots(table, page, start, stop):
    """Cache slots of positions start..stop of each request, one after another."""
    out = []
    for i in range(len(start)):
        p = np.arange(start[i], stop[i])
        out.append(table[i, p // page] * page + p % page)
    return np.concatenate(out)


def _codes(shape, g):
    """Codes of normal values under their block's largest, in pieces."""
    out = torch.empty(shape, dtype=torch.int8, device="cuda")
    flat = out.view(-1)
    step = 1 << 27
    for a in range(0, flat.numel(), step):
        n = min(step, flat.numel() - a)
        flat[a:a + n] = (torch.randn(n, generator=g, device="cuda") * 30).round_().clamp_(-127, 127).to(torch.int8)
    return out


def _cache(pages, page, kv_heads, hd, seed):
    g = _gen(seed)
    k = _codes((pages, kv_heads, page, hd), g)
    v = _codes((pages, kv_heads, hd, page), g)
    ks = torch.exp(0.3 * torch.randn(pages, kv_heads, generator=g, device="cuda")) / 30
    vs = torch.exp(0.3 * torch.randn(pages, kv_heads, generator=g, device="cuda")) / 30
    return k, v, ks, vs


def _append_inputs(case, seed):
    heads, kv, hd = SHAPES[case["shape"]]
    before, new = _append_lengths(case, seed)
    page = case["page"]
    table, pages = _page_ids(-(-(before + new) // page), seed)
    slots = _slots(table, page, before, before + new)
    first = before // page * page  # from the first token of the first page that is touched
    g = _gen(seed + 2)
    rows = len(slots)
    # some rows larger than what their page holds, so that its scale has to grow
    size = torch.exp(0.4 * torch.randn(rows, 1, 1, generator=g, device="cuda"))
    dt = DTYPES[case["dtype"]]
    k = (torch.randn(rows, kv, hd, generator=g, device="cuda") * size).to(dt)
    v = (torch.randn(rows, kv, hd, generator=g, device="cuda") * size).to(dt)
    return dict(slots=_ints(slots), seen=_ints(_slots(table, page, first, before + new)), k=k, v=v,
                cache=_cache(pages, page, kv, hd, seed + 3))


def _attend_inputs(case, seed):
    heads, kv, hd = SHAPES[case["shape"]]
    ctx, new = _attend_lengths(case, seed)
    page = case["page"]
    table, pages = _page_ids(-(-ctx // page), seed)
    pos = np.concatenate([np.arange(c - n, c) for c, n in zip(ctx, new)])
    g = _gen(seed + 2)
    q = torch.randn(len(pos), heads, hd, generator=g, device="cuda").to(DTYPES[case["dtype"]])
    start = np.concatenate([[0], np.cumsum(new)])
    return dict(q=q, table=_ints(table), start=_ints(start), positions=_ints(pos), ctx=ctx.tolist(), new=new.tolist(),
                cache=_cache(pages, page, kv, hd, seed + 3), scale=1 / math.sqrt(hd))


def _sample_inputs(case, seed):
    g = _gen(seed)
    rows, vocab = case["rows"], case["vocab"]
    # a broad body, a thin upper tail, and a hundredth of the tokens banned
    x = torch.randn(rows, vocab, generator=g, device="cuda") * 2
    x += 3 * torch.relu(torch.randn(rows, vocab, generator=g, device="cuda") - 2.5)
    x.masked_fill_(torch.rand(rows, vocab, generator=g, device="cuda") < 0.01, float("-inf"))
    r = np.random.default_rng(seed)
    f = case["filters"]

    def pick(options):
        return r.choice(options, rows)

    temp, k, p, mp = np.full(rows, 0.8), np.zeros(rows, np.int64), np.ones(rows), np.zeros(rows)
    if f == "all":
        k, p, mp = np.full(rows, 50), np.full(rows, 0.95), np.full(rows, 0.02)
    elif f == "nucleus":
        p = np.full(rows, 0.9)
    elif f == "topk":
        k = pick([1, 20, 40, 64, 1000])
    elif f == "mixed":
        temp, k = pick([0.0, 0.6, 1.0, 1.3]), pick([0, 0, 20, 50, 500])
        p, mp = pick([1.0, 0.9, 0.95]), pick([0.0, 0.0, 0.05])
    f32 = dict(dtype=torch.float32, device="cuda")
    return dict(logits=x, temperature=torch.tensor(temp, **f32), top_k=_ints(k), top_p=torch.tensor(p, **f32),
                min_p=torch.tensor(mp, **f32), uniform=torch.rand(rows, generator=g, device="cuda"))


def prepare(case, seed):
    if case["kind"] == "plan":
        before, new = _plan_lengths(case, seed)
        page, n = case["page"], case["requests"]
        pages_of = -(-(before + new) // page)
        rows, pages, most = int(new.sum()), int(pages_of.sum()) + 5, int(pages_of.max()) + 1
        state = dict(case=case, lens=_ints(before), new=_ints(new), rows=rows, page=page)
        if own:
            from loom_amd import paged
            state["table"] = paged.PageTable(n, most, pages, page)
            if not case["fresh"]:  # the pages of the tokens that are there
                state["table"].plan(_ints(np.zeros(n)), state["lens"], int(before.sum()))
        else:
            state.update(pages=torch.full((n, most), -1, dtype=torch.int32, device="cuda"),
                         held=_ints(np.zeros(n)), free=torch.arange(pages - 1, -1, -1, dtype=torch.int32, device="cuda"),
                         free_count=_ints([pages]))
            if not case["fresh"]:
                _plan_plain(state, _ints(np.zeros(n)), state["lens"], int(before.sum()))
        return state
    if case["kind"] == "sample":
        return dict(_sample_inputs(case, seed), case=case)
    state = _append_inputs(case, seed) if case["kind"] == "append" else _attend_inputs(case, seed)
    if own:
        from loom_amd import paged
        state["cache"] = paged.PagedCache.from_tensors(*state["cache"])
    return dict(state, case=case)


# ---- plain forms --------------------------------------------------------------

def _plan_plain(s, lens, new, rows):
    page, table = s["page"], s["pages"]
    n, most = table.shape
    i64 = torch.int64
    after = lens.to(i64) + new
    row_upto = torch.cumsum(new, 0)
    fits = (after <= most * page) & (row_upto <= rows)
    want = torch.where(fits, torch.clamp((after + page - 1) // page - s["held"], min=0), 0)
    upto = torch.cumsum(want, 0)
    fits &= (want == 0) | (upto <= s["free_count"])
    want = torch.where(fits, want, 0)
    first = torch.cumsum(want, 0) - want
    col = torch.arange(most, device="cuda")[None, :]
    fill = (col >= s["held"][:, None]) & (col < (s["held"] + want)[:, None])
    rank = first[:, None] + col - s["held"][:, None]
    src = (s["free_count"].to(i64) - 1 - rank).clamp(0, s["free"].numel() - 1)
    table.copy_(torch.where(fill, s["free"][src], table))
    s["held"].copy_(s["held"] + want)
    s["free_count"].copy_(s["free_count"] - want.sum())
    start = torch.cat([torch.zeros(1, dtype=i64, device="cuda"), row_upto]).clamp(max=rows)
    t = torch.arange(rows, device="cuda")
    req = torch.searchsorted(start[1:], t, right=True)
    live = req < n
    r = req.clamp(max=n - 1)
    pos = lens[r] + t - start[r]
    good = live & fits[r]
    slot = table[r, (pos // page).clamp(0, most - 1)] * page + pos % page
    minus = torch.full_like(t, -1)
    return dict(start=start.int(), request=torch.where(live, req, minus).int(), positions=torch.where(good, pos, minus).int(),
                slots=torch.where(good, slot, minus).int(), lens=torch.where(fits, after, lens.to(i64)).int(),
                pages=table, held=s["held"], free_count=s["free_count"])


def _half_away(x):
    return torch.sign(x) * torch.floor(x.abs() + 0.5)


def _append_plain(codes, scales, x, slots, page, tokens_last):
    """One side of the cache.  codes is updated in place; x rows x heads x dims."""
    pages, heads = scales.shape
    slots = slots.long()
    pg, off = slots // page, slots % page
    big = torch.zeros(pages, heads, device="cuda")
    big.scatter_reduce_(0, pg[:, None].expand(-1, heads), x.float().abs().amax(2), "amax")
    touched = torch.zeros(pages, dtype=torch.bool, device="cuda").index_fill_(0, pg, True)
    fresh = torch.zeros(pages, dtype=torch.bool, device="cuda").index_fill_(0, pg[off == 0], True)
    old = torch.where(fresh[:, None], torch.zeros_like(scales), scales)
    new = torch.where(touched[:, None], torch.maximum(old, (big.double() / 127).float()), scales)
    ids = touched.nonzero()[:, 0]
    ratio = (old[ids].double(), new[ids].double())
    c = codes[ids].double() * ratio[0][:, :, None, None]
    codes[ids] = _half_away(torch.where(ratio[1][:, :, None, None] > 0, c / ratio[1][:, :, None, None], 0)).to(torch.int8)
    q = _half_away(x.double() / new[pg].double()[:, :, None]).nan_to_num(0).to(torch.int8)
    if tokens_last:
        codes[pg, :, :, off] = q
    else:
        codes[pg, :, off] = q
    scales.copy_(new)


def _read_plain(codes, scales, slots, page, tokens_last):
    slots = slots.long()
    pg, off = slots // page, slots % page
    c = codes[pg, :, :, off] if tokens_last else codes[pg, :, off]
    return c.float() * scales[pg][:, :, None]


def _attend_plain(s):
    q, (kc, vc, ks, vs) = s["q"], s["cache"]
    page = kc.shape[2]
    heads, hd = q.shape[1:]
    kv = kc.shape[1]
    out = torch.empty_like(q)
    at = 0
    for i, (ctx, new) in enumerate(zip(s["ctx"], s["new"])):
        ids = s["table"][i, :-(-ctx // page)].long()
        k = kc[ids].float() * ks[ids][:, :, None, None]
        v = vc[ids].float() * vs[ids][:, :, None, None]
        kt = k.permute(1, 3, 0, 2).reshape(kv, hd, -1)[:, :, :ctx].contiguous()
        vt = v.permute(1, 0, 3, 2).reshape(kv, -1, hd)[:, :ctx].contiguous()
        x = q[at:at + new].float().reshape(new, kv, heads // kv, hd).permute(1, 2, 0, 3).reshape(kv, -1, hd).contiguous()
        score = torch.matmul(x, kt).mul_(s["scale"]).view(kv, heads // kv, new, ctx)
        if new > 1:
            pos = s["positions"][at:at + new]
            score.masked_fill_(torch.arange(ctx, device="cuda")[None, :] > pos[:, None], float("-inf"))
        score -= score.amax(3, keepdim=True)
        p = torch.exp(score)
        o = torch.matmul(p.view(kv, -1, ctx), vt).view(kv, heads // kv, new, hd) / p.sum(3, keepdim=True)
        out[at:at + new] = o.permute(2, 0, 1, 3).reshape(new, heads, hd).to(q.dtype)
        at += new
    return out


def _sample_plain(s):
    x = s["logits"]
    rows, vocab = x.shape
    greedy = s["temperature"] <= 0
    t = torch.where(greedy, 1.0, s["temperature"]).double()
    order = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((order.values.double() - order.values[:, :1].double()) / t[:, None])
    rank = torch.arange(vocab, device="cuda")[None, :]
    k = torch.where(s["top_k"] > 0, s["top_k"], vocab)[:, None]
    w = torch.where(rank < k, w, 0)
    upto = torch.cumsum(w, 1)
    p = s["top_p"].double()[:, None]
    keep = (rank < k) & ((p >= 1) | (upto - w < p * upto[:, -1:])) & (w >= s["min_p"].double()[:, None])
    keep[:, 0] = True
    w = torch.zeros_like(w).scatter_(1, order.indices, torch.where(keep, w, 0))
    upto = torch.cumsum(w, 1)
    drawn = (upto > s["uniform"].double()[:, None] * upto[:, -1:]).to(torch.int8).argmax(1)
    return torch.where(greedy, order.indices[:, 0], drawn).int()


def run(state):
    kind = state["case"]["kind"]
    if own:
        from loom_amd import paged, transformer
        if kind == "plan":
            table = state["table"]
            if state["case"]["fresh"]:
                table.reset()
            plan = table.plan(state["lens"], state["new"], state["rows"])
            return dict(start=plan.row_start, request=plan.request, positions=plan.positions, slots=plan.slots,
                        lens=plan.lens, pages=table.pages, held=table.held, free_count=table.free_count)
        if kind == "append":
            state["cache"].append(state["k"], state["v"], state["slots"])
            return state["cache"].read(state["seen"])
        if kind == "attend":
            return paged.attention(state["q"], state["cache"], state["table"], state["start"], state["positions"])
        return transformer.sample(state["logits"], state["uniform"], temperature=state["temperature"],
                                  top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"])
    if kind == "plan":
        if state["case"]["fresh"]:
            n = state["free"].numel()
            state["pages"].fill_(-1)
            state["held"].zero_()
            state["free_count"].fill_(n)
            state["free"].copy_(torch.arange(n - 1, -1, -1, device="cuda"))
        return _plan_plain(state, state["lens"], state["new"], state["rows"])
    if kind == "append":
        kc, vc, ks, vs = state["cache"]
        page = state["case"]["page"]
        _append_plain(kc, ks, state["k"], state["slots"], page, False)
        _append_plain(vc, vs, state["v"], state["slots"], page, True)
        return (_read_plain(kc, ks, state["seen"], page, False), _read_plain(vc, vs, state["seen"], page, True))
    if kind == "attend":
        return _attend_plain(state)
    return _sample_plain(state)


# ---- what a pass cannot do without -----------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "plan":
        before, new = _plan_lengths(case, 1)
        pages = -(-(before + new) // case["page"]) - (0 if case["fresh"] else -(-before // case["page"]))
        rows, n = int(new.sum()), case["requests"]
        return {"bytes": 4 * (2 * n + 2 * int(pages.sum()) + 3 * rows + 3 * n), "flops": 4 * rows}
    if kind == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n, "flops": 8 * n}
    heads, kv, hd = SHAPES[case["shape"]]
    size = 4 if case["dtype"] == "fp32" else 2
    if kind == "append":
        before, new = _append_lengths(case, 1)
        page, rows = case["page"], int(new.sum())
        seen = int((before + new - before // page * page).sum())
        # values in, codes out, and the codes read again as fp32 values
        return {"bytes": 2 * kv * hd * (rows * (size + 1) + seen * 5), "flops": 2 * kv * hd * (3 * rows + seen)}
    ctx, new = _attend_lengths(case, 1)
    pairs = int((new * ctx - new * (new - 1) // 2).sum())
    return {"bytes": int(ctx.sum()) * 2 * kv * hd + 2 * int(new.sum()) * heads * hd * size,
            "flops": 4 * pairs * heads * hd}


# ---- the definition in 64 bits ------------------------------------------------------

def _plan_exact(case, seed):
    before, new = _plan_lengths(case, seed)
    page, n = case["page"], case["requests"]
    pages_of = -(-(before + new) // page)
    total, most, rows = int(pages_of.sum()) + 5, int(pages_of.max()) + 1, int(new.sum())
    table = np.full((n, most), -1)
    taken = 0
    # pages come off the pool in request order: first those of the tokens that
    # are there, then those of the new ones
    for goal in ([pages_of] if case["fresh"] else [-(-before // page), pages_of]):
        for i in range(n):
            have = int((table[i] >= 0).sum())
            for j in range(have, int(goal[i])):
                table[i, j] = taken
                taken += 1
    req = np.repeat(np.arange(n), new)
    pos = np.concatenate([np.arange(b, b + m) for b, m in zip(before, new)])
    return dict(start=_ints(np.concatenate([[0], np.cumsum(new)])), request=_ints(req), positions=_ints(pos),
                slots=_ints(table[req, pos // page] * page + pos % page), lens=_ints(before + new), pages=_ints(table),
                held=_ints(pages_of), free_count=_ints([total - taken]))


def _append_exact(case, seed):
    s = _append_inputs(case, seed)
    page = case["page"]
    slots, seen = s["slots"].cpu().numpy(), s["seen"].cpu().numpy()
    out = []
    for codes, scales, x, last in ((s["cache"][0], s["cache"][2], s["k"], False), (s["cache"][1], s["cache"][3], s["v"], True)):
        codes, scales = codes.cpu().numpy(), scales.cpu().numpy()
        if last:
            codes = codes.transpose(0, 1, 3, 2)
        codes, x = codes.astype(np.float64), x.double().cpu().numpy()
        order = np.argsort(slots, kind="stable")
        ids, first = np.unique(slots[order] // page, return_index=True)
        for pg, rows in zip(ids, np.split(order, first[1:])):
            for h in range(scales.shape[1]):
                old = np.float32(0) if (slots[rows] % page).min() == 0 else scales[pg, h]
                new = max(old, np.float32(np.abs(x[rows, h]).max() / 127))
                c = codes[pg, h] * float(old) / float(new)
                codes[pg, h] = np.sign(c) * np.floor(np.abs(c) + 0.5)
                c = x[rows, h] / float(new)
                codes[pg, h, slots[rows] % page] = np.sign(c) * np.floor(np.abs(c) + 0.5)
                scales[pg, h] = new
        val = codes[seen // page, :, seen % page] * scales[seen // page].astype(np.float64)[:, :, None]
        out.append(torch.from_numpy(val).cuda())
    return tuple(out)


def _attend_exact(case, seed):
    s = _attend_inputs(case, seed)
    kc, vc, ks, vs = s["cache"]
    page, group = case["page"], s["q"].shape[1] // kc.shape[1]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for i, (ctx, new) in enumerate(zip(s["ctx"], s["new"])):
        tok = torch.arange(ctx, device="cuda")
        pg = s["table"][i].long()[tok // page]
        for h in range(kc.shape[1]):
            k = kc[pg, h, tok % page].double() * ks[pg, h].double()[:, None]
            v = vc[pg, h, :, tok % page].double() * vs[pg, h].double()[:, None]
            for j in range(h * group, h * group + group):
                score = s["q"][at:at + new, j].double() @ k.T / math.sqrt(k.shape[1])
                late = tok[None, :] > torch.arange(ctx - new, ctx, device="cuda")[:, None]
                out[at:at + new, j] = torch.softmax(score.masked_fill(late, -math.inf), 1) @ v
        at += new
    return out


def _sample_exact(case, seed):
    s = {n: v.cpu().numpy() for n, v in _sample_inputs(case, seed).items()}
    ids = []
    for x, t, k, p, mp, u in zip(s["logits"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], s["uniform"]):
        if t <= 0:
            ids.append(int(x.argmax()))
            continue
        w = np.exp((x.astype(np.float64) - float(x.max())) / float(t))
        # ranked by value, equal values by index; a filter keeps a first part of the ranking
        rank = np.lexsort((np.arange(len(x)), -x.astype(np.float64)))
        n = len(x) if k <= 0 else min(int(k), len(x))
        mass = np.cumsum(w[rank[:n]])
        if p < 1:
            n = min(n, int(np.searchsorted(mass, float(p) * mass[-1])) + 1)
        n = max(1, min(n, int((w >= float(mp)).sum())))
        kept = np.sort(rank[:n])
        mass = np.cumsum(w[kept])
        ids.append(int(kept[np.searchsorted(mass, float(u) * mass[-1], side="right")]))
    return _ints(ids)


def exact(case, seed):
    return {"plan": _plan_exact, "append": _append_exact, "attend": _attend_exact, "sample": _sample_exact}[case["kind"]](
        case, seed)
