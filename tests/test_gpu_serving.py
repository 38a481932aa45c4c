"""The serving operators together on the GPU: a block over ragged requests with
a paged cache, stage by stage, and a serving loop of tables, block, LM head and
sampling."""
import numpy as np
import pytest

from tests import paged_ref as ref
from tests.stages import BITNET_2B, SMALL, Shape, Weights, _quant, _rel_rows, f64_inner_norm
from tests.test_gpu_paged import attention_bound, ints

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def tf(amd_lib):
    from loom_amd import transformer
    return transformer


@pytest.mark.parametrize("norm", ["strict", "fast"])
@pytest.mark.parametrize("shape,page,act,bias,qk", [(SMALL, 16, 6, False, None), (SMALL, 32, 1, True, "per_head"),
                                                    (Shape(128, 4, 4, 32, 256, 64), 16, 6, False, "shared"),
                                                    (BITNET_2B, 64, 1, False, None)])
def test_block_forward_paged_stages(orc, tf, norm, shape, page, act, bias, qk):
    """Three steps of ragged requests: the projection equals the ring block's
    bit for bit (each request run alone through it), the cache holds those K and
    V rows as append stores them, attention is within its bound of the formula,
    and the stages behind it are the block's own of that attention."""
    from loom_amd import paged
    w = Weights(orc, shape, seed=701, act=act, bias=bias, qk=qk)
    blk = tf.BitNetBlock(w.cfg(tf, norm), w.gpu(tf))
    n = 5
    table = paged.PageTable(n, 4, 4 * n, page)
    cache = paged.PagedCache(4 * n, page, shape.kv, shape.hd)
    kc, vc, ks, vs = (np.zeros((4 * n, shape.kv, page, shape.hd)), np.zeros((4 * n, shape.kv, page, shape.hd)),
                      np.zeros((4 * n, shape.kv), np.float32), np.zeros((4 * n, shape.kv), np.float32))
    lens = np.zeros(n, np.int64)
    g = torch.Generator().manual_seed(3)
    xs = [torch.randn(40, shape.hidden, generator=g) for _ in range(n)]
    # the ring block over each request's whole sequence: Q, K, V of every position
    q_all, k_all, v_all = [], [], []
    for x in xs:
        _, taps = blk.forward(x.cuda(), taps=True)
        q_all.append(taps.q.cpu().numpy())
        ck, cv = blk.kv_cache(0)
        k_all.append(ck[:40].cpu().numpy().reshape(40, shape.kv, shape.hd))
        v_all.append(cv[:40].cpu().numpy().reshape(40, shape.kv, shape.hd))
    for new, pad in (([17, 1, 0, 30, 5], 2), ([1, 1, 1, 1, 1], 0), ([3, 9, 1, 0, 16], 1)):
        new = np.array(new)
        rows = int(new.sum()) + pad
        plan = table.plan(ints(lens), ints(new), rows)
        at = [(r, lens[r] + j) for r in range(n) for j in range(new[r])]
        x_in = torch.cat([torch.stack([xs[r][p] for r, p in at]), torch.zeros(pad, shape.hidden)])
        x, taps = blk.forward_paged(x_in.cuda(), cache, table.pages, plan, taps=True)
        plain, _ = blk.forward_paged(x_in.cuda(), cache, table.pages, plan, max_context=64)
        T = taps.numpy()
        live = len(at)
        q = np.stack([q_all[r][p] for r, p in at])
        assert np.array_equal(T["q"][:live], q), "Q rows"
        slots = plan.slots.cpu().numpy()
        k, v = (np.stack([a[r][p] for r, p in at]).astype(np.float64) for a in (k_all, v_all))
        ref.append(kc, ks, k, slots[:live])
        ref.append(vc, vs, v, slots[:live])
        got = cache.codes()
        pages = table.pages.cpu().numpy()
        lens = lens + new
        assert np.array_equal(plan.lens.cpu().numpy(), lens)
        for r in range(n):
            p = np.arange(lens[r])
            s = pages[r, p // page] * page + p % page
            for c, want, sc, wsc in ((got[0], kc, cache.k_scale, ks), (got[1], vc, cache.v_scale, vs)):
                assert np.array_equal(c.cpu().numpy()[s // page, :, s % page], want[s // page, :, s % page]), "codes"
                assert np.array_equal(sc.cpu().numpy()[s // page], wsc[s // page]), "scales"
        start = plan.row_start.cpu().numpy()
        want = ref.attention(q.astype(np.float32).astype(np.float64).reshape(live, shape.heads, shape.hd), kc,
                             vc.transpose(0, 1, 3, 2), ks, vs, pages, start, plan.positions.cpu().numpy(), shape.hd ** -0.5)
        tol = attention_bound(q, kc, vc, ks, vs, shape.hd ** -0.5, 48, torch.float64)
        assert np.abs(T["attn"][:live].reshape(want.shape) - want).max() <= tol, "attention"
        an = f64_inner_norm(orc, T["attn"][:live], w.an)
        if norm == "strict":
            assert np.array_equal(T["attn_norm"][:live], an)
        else:
            _rel_rows(T["attn_norm"][:live], an, 1e-13, "inner norm")
        _quant(orc, T["attn_norm"][:live], T["aq"][:live], T["aamax"][:live], "attention int8")
        o = orc.dense_quantized(w.o, T["aq"][:live], T["aamax"][:live], bias=w.bias[3] if w.bias else None)
        assert np.array_equal(T["mid"][:live], (o + x_in[:live].numpy()).astype(np.float32)), "O projection"
        dn = orc.dense_quantized(w.d, T["hq"][:live], T["hamax"][:live])
        assert np.array_equal(x[:live].cpu().numpy(), (dn + T["mid"][:live]).astype(np.float32)), "down"
        # the same rows again (their slots are rewritten with the same values), fewer workgroups
        assert float((plain[:live] - x[:live]).abs().max()) <= 1e-2 * float(x[:live].abs().max())
    blk.release()


def test_serving_loop(orc, tf):
    """Requests come, decode at their own lengths and go: tokens, lengths and
    pages follow the plain restatement of tables and sampling, from the same
    logits; a request's tokens do not depend on its neighbours."""
    from loom_amd import paged
    sh = SMALL
    ws = [Weights(orc, sh, seed=801 + 20 * i) for i in range(2)]
    blocks = [tf.BitNetBlock(w.cfg(tf, "fast"), w.gpu(tf)) for w in ws]
    vocab, slots, page = 500, 4, 16
    g = torch.Generator().manual_seed(9)
    emb = torch.randn(vocab, sh.hidden, generator=g).cuda()
    prompts = [torch.randint(0, vocab, (m,), generator=g) for m in (5, 21, 1, 33, 12, 8)]
    steps = [9, 4, 14, 3, 6, 10]
    u_all = torch.rand(len(prompts), 20, generator=g)
    opts = dict(temperature=[0.7, 0.0, 1.2, 0.9, 1.0, 0.5], top_k=[20, 0, 0, 5, 0, 50], top_p=[0.9, 1, 0.8, 1, 1, 0.95],
                min_p=[0, 0, 0, 0, 0.1, 0.02])

    def serve(order, width):
        table, tables = paged.PageTable(width, 4, 3 * width + 1, page), ref.Tables(width, 4, 3 * width + 1, page)
        caches = [paged.PagedCache(3 * width + 1, page, sh.kv, sh.hd) for _ in blocks]
        waiting, active = list(order), [None] * width
        out = {r: [] for r in order}
        lens = np.zeros(width, np.int64)
        while waiting or any(a is not None for a in active):
            feed = []
            for s in range(width):
                if active[s] is None and waiting:
                    active[s] = waiting.pop(0)
                    lens[s] = 0
                    feed.append(prompts[active[s]])
                elif active[s] is not None:
                    feed.append(torch.tensor([out[active[s]][-1]]))
                else:
                    feed.append(torch.zeros(0, dtype=torch.long))
            new = np.array([len(f) for f in feed])
            rows = int(new.sum())
            plan = table.plan(ints(lens), ints(new), rows)
            want = tables.plan(lens, new, rows)
            assert np.array_equal(plan.slots.cpu().numpy(), want["slots"])
            x = emb[torch.cat(feed).cuda()].contiguous()
            for b, c in zip(blocks, caches):
                b.forward_paged(x, c, table.pages, plan)
            lens = want["lens"]
            live = [s for s in range(width) if active[s] is not None]
            last = plan.row_start[1:].long()[torch.tensor(live).cuda()] - 1
            logits = tf.lm_head(emb, x[last].contiguous()) * 0.05
            rs = [active[s] for s in live]
            u = torch.stack([u_all[r, len(out[r])] for r in rs]).cuda()
            args = {k: torch.tensor([v[r] for r in rs], dtype=torch.int32 if k == "top_k" else torch.float32,
                                    device="cuda") for k, v in opts.items()}
            ids = tf.sample(logits, u, **args).tolist()
            lg = logits.cpu().numpy()
            for i, r in enumerate(rs):
                assert ids[i] == ref.sample(lg[i], np.float32(opts["temperature"][r]), opts["top_k"][r],
                                            np.float32(opts["top_p"][r]), np.float32(opts["min_p"][r]),
                                            np.float32(u_all[r, len(out[r])]))
                out[r].append(ids[i])
            done = np.array([active[s] is not None and len(out[active[s]]) >= steps[active[s]] for s in range(width)])
            table.release(torch.tensor(done, device="cuda"))
            tables.release(done)
            for s in np.nonzero(done)[0]:
                active[s], lens[s] = None, 0
        assert int(table.free_count[0]) == 3 * width + 1
        return out

    together = serve([0, 1, 2, 3, 4, 5], slots)
    assert [len(together[r]) for r in range(6)] == steps
    assert serve([0, 1, 2, 3, 4, 5], slots) == together
    for b in blocks:
        b.release()


def test_block_forward_paged_in_a_graph(orc, tf):
    from loom_amd import paged
    w = Weights(orc, SMALL, seed=811)
    blk = tf.BitNetBlock(w.cfg(tf, "fast"), w.gpu(tf))
    n, page = 3, 16

    def fresh():
        t, c = paged.PageTable(n, 4, 12, page), paged.PagedCache(12, page, SMALL.kv, SMALL.hd)
        lens = ints([0, 0, 0])
        plan = t.plan(lens, ints([5, 17, 1]), 23)
        x = torch.randn(23, SMALL.hidden, generator=torch.Generator().manual_seed(1)).cuda()
        blk.forward_paged(x, c, t.pages, plan)
        return t, c, plan.lens.clone()

    data = torch.randn(20, n, SMALL.hidden, generator=torch.Generator().manual_seed(2)).cuda()

    def step(t, c, lens, x):
        plan = t.plan(lens, torch.ones_like(lens), n)
        blk.forward_paged(x, c, t.pages, plan)
        lens.copy_(plan.lens)

    t, c, lens = fresh()
    eager = []
    for i in range(20):
        x = data[i].clone()
        step(t, c, lens, x)
        eager.append(x)
    t, c, lens = fresh()
    x = data[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(t, c, lens, x)
    for i in range(20):
        x.copy_(data[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(x, eager[i]), f"replay {i}"
    blk.release()


def test_block_forward_paged_growing_and_refusals(orc, tf):
    """A larger call after a capture leaves the captured one good; a cache of
    another shape and tensors of other types are refused."""
    from loom_amd import _lib, paged
    w = Weights(orc, SMALL, seed=821)
    blk = tf.BitNetBlock(w.cfg(tf, "fast"), w.gpu(tf))
    t, c = paged.PageTable(2, 8, 16, 16), paged.PagedCache(16, 16, SMALL.kv, SMALL.hd)
    lens, one = ints([0, 0]), ints([1, 1])
    plan = t.plan(lens, one, 2)
    x0 = torch.randn(2, SMALL.hidden, generator=torch.Generator().manual_seed(3)).cuda()
    x = x0.clone()
    blk.forward_paged(x, c, t.pages, plan)
    want = x.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        blk.forward_paged(x, c, t.pages, plan)
    big = t.plan(ints([1, 1]), ints([100, 90]), 200)
    y = torch.randn(200, SMALL.hidden, generator=torch.Generator().manual_seed(4)).cuda()
    blk.forward_paged(y, c, t.pages, big)
    for _ in range(3):
        x.copy_(x0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(x, want)
    with pytest.raises(_lib.AMDError, match="heads"):
        blk.forward_paged(x, paged.PagedCache(16, 16, SMALL.kv + 1, SMALL.hd), t.pages, plan)
    with pytest.raises(_lib.AMDError, match="max_context"):
        blk.forward_paged(x, c, t.pages, plan, max_context=1000)
    for bad in (x.half(), x[:1], x[:, :8], x.t()):
        with pytest.raises(ValueError):
            blk.forward_paged(bad, c, t.pages, plan)
    with pytest.raises(ValueError, match="slots"):
        blk.forward_paged(x, c, t.pages, paged.StepPlan(plan.row_start, plan.lens, plan.request, plan.positions,
                                                        plan.slots.long()))
    blk.release()


def test_refusals_of_device_tensors(tf):
    from loom_amd import paged
    c = paged.PagedCache(4, 16, 2, 64)
    q, k = torch.zeros(3, 4, 64, device="cuda"), torch.zeros(3, 2, 64, device="cuda")
    pages, start, pos = ints([[0, 1]]), ints([0, 3]), ints([0, 1, 2])
    good = dict(q=q, cache=c, pages=pages, row_start=start, positions=pos)
    assert not paged.attention(**good).any()
    for kw in (dict(q=q.half()), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q.cpu()), dict(q=q[:1].expand(3, 4, 64)),
               dict(q=torch.zeros(3, 64, 4, device="cuda").transpose(1, 2)), dict(pages=pages.long()), dict(pages=pages[0]),
               dict(pages=pages[:, :0]), dict(row_start=start[:1]), dict(positions=pos[:2]), dict(positions=pos.cpu()),
               dict(max_context=33), dict(max_context=-1), dict(out=torch.zeros(3, 4, 64)), dict(out=q[:2]),
               dict(out=torch.zeros(1, 4, 64, device="cuda").expand(3, 4, 64))):
        with pytest.raises(ValueError):
            paged.attention(**{**good, **kw})
    slots = ints([0, 1, 2])
    for a in ((k, k.bfloat16(), slots), (k.half(), k.half(), slots), (k, k, slots.long()), (k[:2], k, slots),
              (k.cpu(), k.cpu(), slots), (k[:1].expand(3, 2, 64), k, slots)):
        with pytest.raises(ValueError):
            c.append(*a)
    for a in (slots.long(), slots.cpu(), slots[None]):
        with pytest.raises(ValueError):
            c.read(a)
    t = paged.PageTable(2, 3, 4)
    for a in ((ints([0]), ints([1, 1]), 2), (ints([0, 0]), ints([1, 1]).long(), 2), (ints([0, 0]), ints([1, 1]).cpu(), 2),
              (ints([0, 0]), ints([1, 1]), -1)):
        with pytest.raises(ValueError):
            t.plan(*a)
    with pytest.raises(ValueError):
        t.release(ints([0, 1]))
    lg, u = torch.zeros(2, 10, device="cuda"), torch.zeros(2, device="cuda")
    for a, kw in (((lg.half(), u), {}), ((lg[0], u), {}), ((lg.t(), u), {}), ((lg, u[:1]), {}), ((lg, u.cpu()), {}),
                  ((lg, None), {}), ((lg, u), dict(top_k=u)), ((lg, u), dict(temperature=u.double())),
                  ((lg[:1].expand(2, 10), u), {})):
        with pytest.raises(ValueError):
            tf.sample(*a, **kw)
    # no rows at all
    none = ints([])
    assert paged.attention(q[:0], c, pages, ints([0, 0]), none).shape == (0, 4, 64)
    c.append(k[:0], k[:0], none)
    assert c.read(none)[0].shape == (0, 2, 64)
    assert tf.sample(lg[:0], u[:0]).shape == (0,)


def test_calls_on_two_streams_at_once(tf):
    """Attention and sampling with their workspaces on two streams at once give
    what each gives alone (contexts long enough to be cut into parts)."""
    from loom_amd import paged
    c = paged.PagedCache(400, 16, 2, 64)
    g = torch.Generator(device="cuda").manual_seed(1)
    for t in (c.k, c.v):
        t.copy_(torch.randint(-127, 128, t.shape, generator=g, device="cuda"))
    c.k_scale.fill_(0.01)
    c.v_scale.fill_(0.02)
    pages = torch.randperm(400, generator=g, device="cuda").to(torch.int32).view(2, 200)
    start, pos = ints([0, 1, 2]), ints([3100, 2400])
    qs = torch.randn(8, 2, 8, 64, generator=g, device="cuda")
    lg = torch.randn(8, 3, 30000, generator=g, device="cuda")
    u = torch.rand(8, 3, generator=g, device="cuda")
    p = torch.tensor([0.9, 0.5, 1.0], device="cuda")
    want = [(paged.attention(qs[i], c, pages, start, pos), tf.sample(lg[i], u[i], top_p=p)) for i in range(8)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None] * 8
    for rep in range(4):
        for i in range(8):
            with torch.cuda.stream(streams[i % 2]):
                got[i] = (paged.attention(qs[i], c, pages, start, pos), tf.sample(lg[i], u[i], top_p=p))
        torch.cuda.synchronize()
        for i in range(8):
            assert torch.equal(got[i][0], want[i][0]) and torch.equal(got[i][1], want[i][1]), (rep, i)


def test_two_graphs_replayed_in_turn_and_at_once(tf):
    from loom_amd import paged
    c = paged.PagedCache(300, 32, 1, 128)
    g = torch.Generator(device="cuda").manual_seed(2)
    for t in (c.k, c.v):
        t.copy_(torch.randint(-127, 128, t.shape, generator=g, device="cuda"))
    c.k_scale.fill_(0.01)
    c.v_scale.fill_(0.02)
    pages = torch.randperm(300, generator=g, device="cuda").to(torch.int32).view(2, 150)
    calls = []
    for i, (start, pos) in enumerate(((ints([0, 1, 2]), ints([4000, 3500])), (ints([0, 40, 41]), torch.cat(
            [torch.arange(1000, 1040, device="cuda"), torch.tensor([4500], device="cuda")]).to(torch.int32)))):
        q = torch.randn(pos.shape[0], 4, 128, generator=g, device="cuda")
        want = paged.attention(q, c, pages, start, pos).clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = paged.attention(q, c, pages, start, pos)
        calls.append((graph, out, want, (q, start, pos)))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for rep in range(5):
        for graph, out, want, _ in calls:
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
        for (graph, out, _, _), s in zip(calls, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for _, out, want, _ in calls:
            assert torch.equal(out, want), rep
