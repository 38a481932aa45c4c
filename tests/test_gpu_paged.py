"""Page tables, the 8-bit paged cache and attention over it on the GPU against
plain restatements in 64 bits (tests/paged_ref.py)."""
import numpy as np
import pytest

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def paged(amd_lib):
    from loom_amd import paged as m
    return m


def ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def same(t, want, what):
    got = t.cpu().numpy()
    assert np.array_equal(got, want), f"{what}: {got} != {want}"


def check_plan(table, tables, plan, want):
    for f in ("row_start", "lens", "request", "positions", "slots"):
        same(getattr(plan, f), want[f], f)
    same(table.pages, tables.pages, "pages")
    same(table.held, tables.held, "held")
    n = int(table.free_count[0])
    assert n == len(tables.free)
    same(table.free[:n], np.array(tables.free, np.int64).reshape(-1), "free")


# (5000 requests pass the fold of the row fill into the one-workgroup kernel,
# 9000 rows its row count)
@pytest.mark.parametrize("requests,longest,page,seed", [(1, 1, 16, 0), (3, 40, 16, 1), (64, 5, 32, 2), (130, 90, 64, 3),
                                                        (1025, 7, 16, 4), (5000, 3, 16, 5), (9, 2500, 128, 6)])
def test_plans_of_a_run_of_steps(paged, requests, longest, page, seed):
    r = np.random.default_rng(seed)
    most, pool = -(-longest * 6 // page) + 1, requests * (-(-longest * 3 // page) + 1)
    table = paged.PageTable(requests, most, pool, page)
    tables = ref.Tables(requests, most, pool, page)
    lens = np.zeros(requests, np.int64)
    for step in range(6):
        new = r.integers(0, longest + 1, requests)
        if step == 2:
            new[r.random(requests) < 0.5] = 0
        rows = int(new.sum()) + (step % 3) * 5  # some rows behind the last request
        plan = table.plan(ints(lens), ints(new), rows)
        want = tables.plan(lens, new, rows)
        check_plan(table, tables, plan, want)
        # the same lengths again: the pages are there, the slots stay
        again = table.plan(ints(lens), ints(new), rows)
        same(again.slots, tables.plan(lens, new, rows)["slots"], "slots again")
        lens = want["lens"]
        if step in (1, 3):
            done = r.random(requests) < 0.4
            flags = torch.tensor(done, device="cuda")
            table.release(flags if step == 1 else flags.to(torch.uint8))
            tables.release(done)
            lens = np.where(done, 0, lens)


def test_plan_refuses_what_does_not_fit(paged):
    # request 1 is past its table, 3 past the pool (and so 4, which needs a page,
    # but not 5, which needs none), 6 past the rows
    table, tables = paged.PageTable(7, 4, 6, 16), ref.Tables(7, 4, 6, 16)
    lens0 = np.array([0, 0, 0, 0, 0, 3, 0])
    new0 = np.array([20, 0, 0, 0, 0, 3, 0])
    for t in (0, 1):
        if t == 0:
            lens, new, rows = np.zeros(7, np.int64), new0, 23
        else:
            lens, new, rows = np.array([20, 0, 5, 0, 0, 3, 1]), np.array([1, 65, 11, 60, 17, 2, 9]), 160
        plan = table.plan(ints(lens), ints(new), rows)
        check_plan(table, tables, plan, tables.plan(lens, new, rows))
    # negative lengths and counts are none, huge ones refused
    lens, new = np.array([-5, 2**31 - 1, 0, 0, 0, 0, 0]), np.array([3, 2**31 - 1, -7, 0, 2**31 - 1, 1, 1])
    plan = table.plan(ints(lens), ints(new), 40)
    check_plan(table, tables, plan, tables_plan_capped(tables, lens, new, 40))


def tables_plan_capped(tables, lens, new, rows):
    """tables.plan with counts of billions cut to just past every limit."""
    cut = np.minimum(new, 10 * rows)
    want = tables.plan(np.minimum(lens, 10**6), cut, rows)
    want["lens"] = np.where(np.asarray(lens) > 10**6, lens, want["lens"])
    return want


def test_plan_of_no_rows(paged):
    table, tables = paged.PageTable(5, 2, 4, 16), ref.Tables(5, 2, 4, 16)
    z = np.zeros(5, np.int64)
    plan = table.plan(ints(z), ints(z), 0)
    check_plan(table, tables, plan, tables.plan(z, z, 0))


def new_cache(paged, pages, page, heads, hd, seed):
    """A cache of random codes, and the same in numpy (tokens before dimensions)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = paged.PagedCache(pages, page, heads, hd)
    for t in (c.k, c.v):
        t.copy_(torch.randint(-127, 128, t.shape, generator=g, device="cuda"))
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.exp(torch.randn(t.shape, generator=g, device="cuda")) / 60)
    return c


def snapshot(c):
    return (*(t.cpu().numpy().astype(np.float64) for t in c.codes()), c.k_scale.cpu().numpy(), c.v_scale.cpu().numpy())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("page,heads,hd", [(16, 5, 128), (32, 1, 64), (64, 3, 32), (128, 2, 256), (16, 4, 64)])
def test_append_and_read(paged, page, heads, hd, dtype):
    r = np.random.default_rng(page + hd)
    pages = 12
    c = new_cache(paged, pages, page, heads, hd, 7)
    want = snapshot(c)
    # runs: a single row, one from inside a page over two more, a whole page, the
    # start of one, rows with no slot, a last token
    runs = [[5 * page + 3], list(range(7 * page - 2, 7 * page)) , list(range(2 * page, 3 * page)), [-1],
            list(range(9 * page, 9 * page + 5)), [pages * page, -7], [page - 1], [11 * page]]
    slots = np.array(sum(runs, []) + [8 * page + i for i in range(page // 2, page)] + [3 * page + i for i in range(page)])
    rows = len(slots)
    size = np.exp(r.normal(0, 1.5, (rows, 1, 1)))
    wide = torch.tensor(r.normal(0, 1, (rows, 2 * heads * hd + 6)) , device="cuda").to(dtype)
    k = (wide[:, 3:3 + heads * hd].view(rows, heads, hd) * torch.tensor(size, device="cuda")).to(dtype)
    wide[:, 5:5 + heads * hd] = k.reshape(rows, -1)
    k, v = wide[:, 5:5 + heads * hd].view(rows, heads, hd), wide[:, -heads * hd:].view(rows, heads, hd)
    x = [t.double().cpu().numpy() for t in (k, v)]
    c.append(k, v, ints(slots))
    ref.append(want[0], want[2], x[0], slots)
    ref.append(want[1], want[3], x[1], slots)
    got = snapshot(c)
    seen = []  # what the pages are known to hold: the runs and the tokens before them
    for s in slots[(slots >= 0) & (slots < pages * page)]:
        seen += list(range(s // page * page, s + 1))
    seen += [4 * page + 1, 6 * page]  # an untouched page
    seen = np.unique(seen)
    for i, name in ((0, "k"), (1, "v")):
        same_codes = got[i][seen // page, :, seen % page] == want[i][seen // page, :, seen % page]
        assert same_codes.all(), f"{name} codes differ at slots {seen[~same_codes.all((1, 2))]}"
        assert np.array_equal(got[2 + i], want[2 + i]), f"{name} scales"
    seen = np.concatenate([seen, [-1, pages * page]])
    ka, va = c.read(ints(seen))
    inside = seen[:-2]
    for t, i in ((ka, 0), (va, 1)):
        val = want[i][inside // page, :, inside % page].astype(np.float32) * want[2 + i][inside // page][:, :, None]
        assert np.array_equal(t[:-2].cpu().numpy(), val)
        assert not t[-2:].any()


def test_append_not_finite_and_tiny(paged):
    c = paged.PagedCache(3, 16, 2, 32)
    x = torch.zeros(4, 2, 32, device="cuda")
    x[0, 0, 0], x[0, 0, 1], x[0, 0, 2], x[0, 0, 3] = float("nan"), float("inf"), -float("inf"), 2.0
    x[1, 0, 5] = -1.0
    x[2, 0, 4] = float("inf")  # a page of nothing finite but zeros
    x[2, 1, 4] = 1e-38  # under 2^-100
    x[3, 1, 4] = 3.4e38
    slots = np.array([0, 1, 16, 32])
    c.append(x, x, ints(slots))
    k, v = c.read(ints(slots))
    want = np.zeros((4, 2, 32), np.float32)
    s = np.float32(2.0) / np.float32(127)
    want[0, 0, 1:4] = np.float32(127) * s, -np.float32(127) * s, np.float32(127) * s
    want[1, 0, 5] = -np.float32(64) * s  # -63.5: half away from zero
    want[3, 1, 4] = np.float32(127) * (np.float32(3.4e38) / np.float32(127))
    for t in (k, v):
        assert np.array_equal(t.cpu().numpy(), want)


def attention_bound(q, kc, vc, ks, vs, scale, longest, dtype):
    """How far a row may be off, from its scores' and sums' roundings.

    Scores: q in fixed point is off by at most half a unit of amax / 8355000;
    the digits' sums are exact, their join and factors take 7 roundings, the
    difference to the maximum 1 more of up to twice the score: 9 * 2^-24 |s| in
    all.
    A probability is off by that, 2^-23 of exp2 and its fp16 form (2^-22 as a
    pair, 2^-12 as one); numerator and denominator both: twice.  The sums: 16
    terms and 4 products a step of 64 tokens, and the join, each 2^-23 at most.
    The result is rounded to its type."""
    big_k = np.abs(kc).astype(np.float64).sum(-1).max(initial=0) * np.nanmax(ks)
    big_q = np.abs(q[np.isfinite(q)]).max(initial=0)
    s = big_q * scale * big_k * 0.5  # (a loose bound of |q.k|)
    unit = 0.5 / 8355000
    d = big_q * unit * scale * big_k + 9 * 2.0 ** -24 * s + 2.0 ** -23
    d += 2.0 ** -22 if dtype != torch.bfloat16 else 2.0 ** -12
    d = 2 * d + (longest / 64 * 20 + 40) * 2.0 ** -23
    if dtype == torch.bfloat16:
        d += 2.0 ** -8 / 2
    elif dtype == torch.float64:
        d += 2.0 ** -24
    return d * 127 * vs.max()


def run_attention(paged, hd, kv, group, page, dtype, ctx, new, seed=0, pad=0, slack=0, qscale=1.0, max_context=None,
                  spoil=None):
    """Requests of ctx tokens of which the last `new` are rows of the call."""
    r = np.random.default_rng(seed)
    ctx, new = np.array(ctx), np.array(new)
    pages_of = -(-ctx // page)
    pool = int(pages_of.sum()) + 2
    c = new_cache(paged, pool, page, kv, hd, seed)
    ids = r.permutation(pool)
    table = np.full((len(ctx), max(1, int(pages_of.max())) + slack), -1)
    at = 0
    for i, n in enumerate(pages_of):
        table[i, :n] = ids[at:at + n]
        at += n
    start = np.concatenate([[0], np.cumsum(new)])
    pos = np.concatenate([np.arange(x - n, x) for x, n in zip(ctx, new)] + [np.full(pad, 10 ** 6)])
    rows = len(pos)
    q = (torch.randn(rows, kv * group, hd, generator=torch.Generator().manual_seed(seed)) * qscale).to(dtype)
    if spoil:
        spoil(c, table, pos, q)
    dq = q.cuda()
    out = torch.full_like(dq, 7.0)
    got = paged.attention(dq, c, ints(table), ints(start), ints(pos), out=out, max_context=max_context)
    assert got is out
    scale = hd ** -0.5
    kc, vc = (t.cpu().numpy() for t in c.codes())
    vc = vc.transpose(0, 1, 3, 2)
    ks, vs = c.k_scale.cpu().numpy(), c.v_scale.cpu().numpy()
    qn = q.double().numpy()
    want = ref.attention(qn, kc, vc, ks, vs, table, start, pos, scale)
    tol = attention_bound(qn, kc, vc, ks, vs, scale, max(1, int(ctx.max())), dtype)
    got = got.double().cpu().numpy()
    if pad:
        assert (got[rows - pad:] == 7.0).all(), "rows of no request were written"
        got, want = got[:rows - pad], want[:rows - pad]
    bad = ~(np.abs(got - want) <= tol)
    both_nan = np.isnan(got) & np.isnan(want)
    bad &= ~both_nan
    assert not bad.any(), (f"{bad.sum()} of {bad.size} off, first {np.argwhere(bad)[0]}: {got[bad][0]} != "
                           f"{want[bad][0]} (tolerance {tol})")
    return got, want, tol


DTYPES = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,kv,group,page", [(128, 5, 4, 16), (64, 4, 4, 32), (32, 2, 1, 64), (256, 1, 3, 128),
                                              (128, 1, 16, 64), (64, 1, 23, 16)])
def test_attention_decode_rows(paged, hd, kv, group, page, dtype):
    run_attention(paged, hd, kv, group, page, dtype, [1, 2, 15, 16, 17, 63, 64, 65, 255, 300], [1] * 10, pad=3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,kv,group,page", [(128, 2, 4, 16), (64, 2, 2, 64), (32, 1, 5, 16), (256, 1, 2, 32)])
def test_attention_chunks_and_decode_rows(paged, hd, kv, group, page, dtype):
    # whole prompts, chunks behind a context, single rows, a request without rows
    run_attention(paged, hd, kv, group, page, dtype, [70, 1, 200, 33, 90, 5, 130], [70, 1, 41, 1, 0, 5, 17], pad=2)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_split_contexts(paged, dtype):
    # one request: its context is cut into parts, for decode rows and for a chunk
    run_attention(paged, 128, 1, 4, 16, dtype, [3001], [1], slack=70)
    run_attention(paged, 64, 2, 2, 32, dtype, [2500, 3, 700], [90, 3, 1], pad=1)
    run_attention(paged, 128, 1, 4, 16, dtype, [3001], [2], max_context=3010, slack=9)


@pytest.mark.parametrize("requests", [64, 65, 129, 4097])
def test_attention_finds_requests(paged, requests):
    # the search over row starts: steps of one and of many requests, empty ones among them
    r = np.random.default_rng(requests)
    new = r.integers(0, 2, requests)
    new[-1] = 1
    run_attention(paged, 32, 1, 2, 16, torch.float32, np.maximum(new, r.integers(1, 20, requests)), new)


def test_codes_in_and_out(paged):
    g = torch.Generator(device="cuda").manual_seed(0)
    for pages, heads, page, hd in ((3, 2, 16, 32), (2, 1, 128, 64), (1, 3, 32, 256)):
        k = torch.randint(-127, 128, (pages, heads, page, hd), generator=g, device="cuda").to(torch.int8)
        v = torch.randint(-127, 128, (pages, heads, hd, page), generator=g, device="cuda").to(torch.int8)
        ks, vs = (torch.rand(pages, heads, generator=g, device="cuda") for _ in range(2))
        c = paged.PagedCache.from_tensors(k, v, ks, vs)
        kc, vc = c.codes()
        assert torch.equal(kc, k) and torch.equal(vc, v.transpose(2, 3))
        a, b = c.read(torch.arange(pages * page, dtype=torch.int32, device="cuda"))
        assert torch.equal(a, (k.float() * ks[:, :, None, None]).transpose(1, 2).reshape(pages * page, heads, hd))
        assert torch.equal(b, (v.float() * vs[:, :, None, None]).permute(0, 3, 1, 2).reshape(pages * page, heads, hd))


def test_attention_float64_rows(paged):
    run_attention(paged, 128, 5, 4, 16, torch.float64, [100, 64, 7], [1, 20, 7])


def test_attention_of_rows_and_pages_that_are_not_there(paged):
    def spoil(c, table, pos, q):
        pos[0] = -1                       # a row without a place
        table[1, 1] = -1                  # a page taken away
        table[2, 0] = c.num_pages         # not one of the cache's
        table[3, :] = -5
        pos[4] = 2 ** 31 - 2              # past the table: its last position
        # codes of the pages nobody attends to are whatever they are
        c.k_scale[int(table[4, 2])] = float("nan")
        table[4, 2] = 2 ** 31 - 1

    for dtype in DTYPES:
        got, want, tol = run_attention(paged, 64, 2, 2, 16, dtype, [40, 40, 40, 40, 48], [1, 1, 1, 1, 1], spoil=spoil)
        assert not got[0].any() and not got[3].any()


def test_attention_not_finite_queries(paged):
    def spoil(c, table, pos, q):
        q[0, 1, 3] = float("nan")
        q[1, 2, 0] = float("inf")
        q[2] = 0.0
        q[3] = 1e30   # scores past fp32's exponent differences: one-hot rows
        q[3, 0] = 1e-30

    for dtype in DTYPES:
        c_new = [1, 1, 1, 1]
        for ctx in ([40, 40, 40, 40], [2000, 40, 40, 40]):
            r = np.random.default_rng(1)
            got = attention_raw(paged, 64, 2, 2, 16, dtype, ctx, c_new, spoil)
            nan = np.isnan(got).all(2)
            assert np.isnan(got).any(2).sum() == 2 and nan[0, 1] and nan[1, 2]
            assert np.isfinite(got[2]).all() and np.isfinite(got[3]).all()


def attention_raw(paged, hd, kv, group, page, dtype, ctx, new, spoil):
    ctx, new = np.array(ctx), np.array(new)
    n = -(-ctx // page)
    c = new_cache(paged, int(n.sum()), page, kv, hd, 3)
    table = np.full((len(ctx), int(n.max())), -1)
    at = 0
    for i, m in enumerate(n):
        table[i, :m] = np.arange(at, at + m)
        at += m
    pos = ctx - 1
    q = torch.randn(len(ctx), kv * group, hd, generator=torch.Generator().manual_seed(5)).to(dtype)
    spoil(c, table, pos, q)
    out = paged.attention(q.cuda(), c, ints(table), ints(np.arange(len(ctx) + 1)), ints(pos))
    return out.double().cpu().numpy()


def test_attention_scales_apart(paged):
    # pages whose scales differ by many orders, zero scales among them
    def spoil(c, table, pos, q):
        f = torch.tensor(10.0 ** np.random.default_rng(0).integers(-9, 3, c.num_pages), device="cuda").float()
        c.v_scale.copy_(f[:, None].expand_as(c.v_scale))
        c.v_scale[int(table[0, 0])] = 0.0
        c.k_scale[int(table[1, 0])] = 0.0
        c.v_scale[table[2, table[2] >= 0]] = 0.0

    got, want, tol = run_attention(paged, 64, 2, 2, 16, torch.float32, [90, 90, 90, 200], [1, 1, 1, 30], spoil=spoil)
    assert not got[2].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_strided_rows_and_out(paged, dtype):
    hd, kv, group, page = 64, 2, 2, 16
    c = new_cache(paged, 8, page, kv, hd, 1)
    table, start, pos = ints([[0, 1, 2], [5, 4, 3]]), ints([0, 2, 5]), ints([30, 31, 40, 41, 42])
    for off, width in ((0, 800), (3, 777), (8, 840)):
        wide = torch.randn(5, width, device="cuda").to(dtype)
        q = wide[:, off:off + kv * group * hd].view(5, kv * group, hd)
        dense = paged.attention(q.contiguous(), c, table, start, pos)
        buf = torch.zeros(5, width, device="cuda", dtype=dtype)
        out = buf[:, off:off + kv * group * hd].view(5, kv * group, hd)
        paged.attention(q, c, table, start, pos, out=out)
        assert torch.equal(out, dense)
        buf[:, off:off + kv * group * hd] = 0
        assert not buf.any()


def test_long_cache_passes_32_bits(paged):
    # codes past 2^31 and 2^32 bytes from the start of their tensors
    page, kv, hd = 64, 8, 128
    pages = (2 ** 32 // (page * kv * hd)) + 40
    c = paged.PagedCache(pages, page, kv, hd)
    r = np.random.default_rng(0)
    ids = np.array([0, pages // 2 + 5, pages - 1, pages - 30])
    slots = np.concatenate([np.arange(i * page, i * page + page) for i in ids])
    x = torch.randn(len(slots), kv, hd, device="cuda")
    y = torch.randn(len(slots), kv, hd, device="cuda")
    c.append(x, y, ints(slots))
    k, v = c.read(ints(slots))
    assert ((k - x).abs() <= x.abs().amax((0, 2), keepdim=True) / 127).all()
    assert ((v - y).abs() <= y.abs().amax((0, 2), keepdim=True) / 127).all()
    n = len(slots) - 3
    q = torch.randn(1, kv * 2, hd, device="cuda")
    out = paged.attention(q, c, ints(ids[None]), ints([0, 1]), ints([n - 1]))
    s = (k[:n].double().repeat_interleave(2, 1) * q.double()).sum(2) * hd ** -0.5
    want = (torch.softmax(s, 0)[:, :, None] * v[:n].double().repeat_interleave(2, 1)).sum(0)
    tol = attention_bound(q.double().cpu().numpy(), np.array([127.0 * hd]), None, c.k_scale[ids].cpu().numpy(),
                          c.v_scale[ids].cpu().numpy(), hd ** -0.5, n, torch.float32)
    assert float((out[0].double() - want).abs().max()) <= tol


def test_streams_and_graphs(paged):
    """A step captured once and replayed while lengths advance on the device,
    with eager work on other streams between, equals the eager steps."""
    kv, group, hd, page, n = 2, 2, 64, 16, 5
    steps = 40

    def setup():
        t = paged.PageTable(n, 8, 40, page)
        c = paged.PagedCache(40, page, kv, hd)
        return t, c, ints([0, 3, 15, 16, 31])

    g = torch.Generator(device="cuda").manual_seed(1)
    data = torch.randn(steps, 3, n, kv * group, hd, generator=g, device="cuda")

    def step(t, c, lens, q, k, v):
        plan = t.plan(lens, torch.ones_like(lens), n)
        c.append(k, v, plan.slots)
        out = paged.attention(q, c, t.pages, plan.row_start, plan.positions)
        lens.copy_(plan.lens)
        return out

    t, c, lens = setup()
    t.plan(ints([0] * n), lens, 65)
    eager = [step(t, c, lens, data[i, 0], data[i, 1, :, :kv].contiguous(), data[i, 2, :, :kv].contiguous()).clone()
             for i in range(steps)]

    t2, c2, lens2 = setup()
    t2.plan(ints([0] * n), lens2, 65)
    q, k, v = (torch.empty(n, kv * group, hd, device="cuda"), torch.empty(n, kv, hd, device="cuda"),
               torch.empty(n, kv, hd, device="cuda"))
    for x in (q, k, v):
        x.zero_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    saved = [x.clone() for x in (t2.pages, t2.held, t2.free, t2.free_count, lens2, c2.k, c2.v, c2.k_scale, c2.v_scale)]
    with torch.cuda.stream(side):
        step(t2, c2, lens2, q, k, v)  # warm up on the capture stream
    torch.cuda.synchronize()
    for x, y in zip((t2.pages, t2.held, t2.free, t2.free_count, lens2, c2.k, c2.v, c2.k_scale, c2.v_scale), saved):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(t2, c2, lens2, q, k, v)
    for i in range(steps):
        q.copy_(data[i, 0])
        k.copy_(data[i, 1, :, :kv])
        v.copy_(data[i, 2, :, :kv])
        graph.replay()
        if i % 7 == 0:
            torch.cuda.synchronize()
            with torch.cuda.stream(side):  # an eager call of its own meanwhile
                step(t, c, lens.clone(), data[i, 0], k, v)
            torch.cuda.synchronize()
        assert torch.equal(out, eager[i]), f"replay {i}"
    assert lens2.tolist() == [40, 43, 55, 56, 71]
