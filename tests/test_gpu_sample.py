"""Sampling on the GPU against the plain restatement in 64 bits
(tests/paged_ref.py): ids are whole numbers and have to be equal."""
import numpy as np
import pytest

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def tr(amd_lib):
    from loom_amd import transformer
    return transformer


def check(tr, x, u, t=None, k=None, p=None, mp=None):
    rows = len(x)

    def dev(a, dt):
        return None if a is None else torch.tensor(np.broadcast_to(np.asarray(a), rows).copy(), dtype=dt, device="cuda")

    f = torch.float32
    got = tr.sample(torch.tensor(x, device="cuda"), dev(u, f), dev(t, f), dev(k, torch.int32), dev(p, f), dev(mp, f))
    got = got.cpu().numpy()

    def at(a, i, off):
        return off if a is None else np.broadcast_to(np.asarray(a), rows)[i]

    want = [ref.sample(x[i], np.float32(at(t, i, 1.0)), at(k, i, 0), np.float32(at(p, i, 1.0)),
                       np.float32(at(mp, i, 0.0)), np.float32(np.broadcast_to(u, rows)[i])) for i in range(rows)]
    bad = np.nonzero(got != want)[0]
    assert not len(bad), f"rows {bad[:5]}: {got[bad[:5]]} != {np.array(want)[bad[:5]]}"


def logits(rows, vocab, seed, spread=2.0):
    return (np.random.default_rng(seed).normal(0, spread, (rows, vocab))).astype(np.float32)


@pytest.mark.parametrize("vocab", [1, 2, 7, 1000, 8191, 8192, 8193, 32000, 128256])
def test_filters(tr, vocab):
    rows = 24
    r = np.random.default_rng(vocab)
    x = logits(rows, vocab, vocab)
    u = r.random(rows).astype(np.float32)
    check(tr, x, u)
    check(tr, x, u, t=0.7)
    check(tr, x, u, k=r.choice([1, 2, 40, 5000], rows))
    check(tr, x, u, t=0.8, p=r.choice([0.1, 0.5, 0.9, 0.999], rows))
    check(tr, x, u, mp=r.choice([0.001, 0.05, 0.5, 1.0], rows))
    check(tr, x, u, t=r.choice([0.0, 0.3, 1.0, 2.0, -1.0], rows), k=r.choice([0, 1, 50, 1500, vocab, vocab + 5], rows),
          p=r.choice([1.0, 0.95, 0.6], rows), mp=r.choice([0.0, 0.02], rows))


def test_edges_of_the_random_number(tr):
    x = logits(8, 300, 1)
    x[:, 0] = -np.inf
    for u in (0.0, np.nextafter(np.float32(1), np.float32(0)), 1.0):
        check(tr, x, u)
        check(tr, x, u, k=5, p=0.9, mp=0.01)


def test_equal_logits(tr):
    # every filter ends among tokens of one value: the lowest indexes stay
    for vocab in (10, 3000, 20000):
        x = np.zeros((16, vocab), np.float32)
        x[8:, ::3] = 1.5
        x[4:8] = np.where(np.arange(vocab) % 2, np.float32(0.0), np.float32(-0.0))
        u = np.linspace(0, 0.999, 16).astype(np.float32)
        check(tr, x, u)
        check(tr, x, u, k=7)
        check(tr, x, u, k=vocab // 2 + 1)
        check(tr, x, u, p=0.5)
        check(tr, x, u, k=vocab - 2, p=0.25)
        check(tr, x, u, mp=0.9)
        check(tr, x, u, k=vocab // 3 + 2, mp=0.2, p=0.7)


def test_crowded_buckets(tr):
    # temperatures that put many tokens into one bucket, or a few nats over all of them
    x = logits(12, 50000, 3)
    u = np.random.default_rng(3).random(12).astype(np.float32)
    for t in (8.0, 60.0, 1e4, 1e30, np.inf):
        check(tr, x, u, t=t, k=[0, 1, 900, 1025, 30000, 49999] * 2, p=[1.0, 0.3] * 6)
        check(tr, x, u, t=t, mp=0.5, p=0.77)
    # values quantized to a few levels (as logits of 16 bits are)
    check(tr, np.round(x * 2) / 2, u, k=[3, 100, 2000] * 4, p=[0.9, 1.0] * 6)


def test_sharp_and_far(tr):
    x = logits(12, 9000, 4)
    u = np.random.default_rng(4).random(12).astype(np.float32)
    for t in (1e-2, 1e-4, 1e-6, 1e-30):
        check(tr, x, u, t=t, p=0.9)
    for off in (1e4, -1e4, 1e9, 3e38):
        y = (x + np.float32(off)).astype(np.float32)
        check(tr, y, u)
        check(tr, y, u, t=0.5, k=3, p=0.9, mp=0.1)
        y[:, 77] = y.max(1)
        check(tr, y, u, k=2)


def test_not_finite(tr):
    x = logits(10, 700, 5)
    x[0, :] = -np.inf
    x[1, :] = np.nan
    x[2, 0] = np.nan
    x[3, 5:600] = np.nan
    x[4, 9] = np.inf
    x[5, [9, 99]] = np.inf
    x[6, 1:] = -np.inf
    x[7, :350] = -np.inf
    u = np.full(10, 0.6, np.float32)
    check(tr, x, u)
    check(tr, x, u, k=3, p=0.8, mp=0.05)
    check(tr, x, u, t=0.0)
    for bad in (np.nan,):
        check(tr, x, u, t=bad)
        check(tr, x, u, p=bad)


def test_strided_rows_and_repeats(tr):
    x = logits(6, 5003, 6)
    u = torch.rand(6, device="cuda")
    args = dict(top_k=torch.tensor([0, 5, 0, 1200, 9, 0], dtype=torch.int32, device="cuda"),
                top_p=torch.tensor([0.9, 1, 0.5, 0.8, 1, 1], device="cuda"))
    base = tr.sample(torch.tensor(x, device="cuda"), u, **args)
    for off, width in ((1, 5010), (4, 5012)):
        wide = torch.full((6, width), 50.0, device="cuda")
        wide[:, off:off + 5003] = torch.tensor(x, device="cuda")
        for _ in range(3):
            assert torch.equal(tr.sample(wide[:, off:off + 5003], u, **args), base)


def test_many_rows_and_graph(tr):
    rows, vocab = 70000, 40
    x = logits(rows, vocab, 8)
    u = np.random.default_rng(8).random(rows).astype(np.float32)
    check(tr, x, u, k=7, p=0.9)
    lg, ud = torch.tensor(x[:64], device="cuda"), torch.rand(64, device="cuda")
    tr.sample(lg, ud)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ids = tr.sample(lg, ud)
    for i in range(5):
        lg.copy_(torch.randn(64, vocab, device="cuda"))
        ud.copy_(torch.rand(64, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ids, tr.sample(lg, ud))


def test_drawn_as_often_as_likely(tr):
    n = 40000
    x = torch.tensor([[0.0, 1.0, -1.0, 2.0, 0.5]], device="cuda").expand(n, 5).contiguous()
    u = (torch.arange(n, device="cuda") + 0.5) / n
    ids = tr.sample(x, u, temperature=torch.full((n,), 1.5, device="cuda"))
    got = torch.bincount(ids, minlength=5).double() / n
    want = torch.softmax(x[0].double() / 1.5, 0)
    # the random numbers are a grid: each count is off by less than two of them
    assert float((got - want).abs().max()) < 2.0 / n
