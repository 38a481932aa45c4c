"""Refusals of the serving entry points, which all come before any GPU call:
the C functions with plain numbers for pointers, and the Python wrappers with
CPU tensors.  No compute runs here."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

P16 = 1 << 20  # stands for a 16-byte aligned device pointer; never read


@pytest.fixture
def L(amd_lib):
    from loom_amd import _lib
    return _lib


def refused(lib, rc, part):
    assert rc == -1
    msg = lib.loom_amd_last_error().decode()
    assert part in msg, msg


def table(L, **kw):
    d = dict(pages=P16, held=P16, free_pages=P16, free_count=P16, requests=4, max_pages=8, num_pages=20, page_size=16)
    d.update(kw)
    return C.byref(L.PageTable(*(d[f] for f, _ in L.PageTable._fields_)))


def cache(L, **kw):
    d = dict(k=P16, v=P16, k_scale=P16, v_scale=P16, num_pages=20, page_size=16, kv_heads=2, head_dim=64)
    d.update(kw)
    return C.byref(L.KvPages(*(d[f] for f, _ in L.KvPages._fields_)))


@pytest.mark.parametrize("bad,part", [(dict(pages=0), "null"), (dict(free_count=0), "null"), (dict(requests=0), "positive"),
                                      (dict(max_pages=-1), "positive"), (dict(num_pages=0), "positive"),
                                      (dict(page_size=24), "page_size"), (dict(page_size=8), "page_size"),
                                      (dict(num_pages=2 ** 27), "2^31"), (dict(max_pages=2 ** 27), "2^31")])
def test_page_table_refusals(amd_lib, L, bad, part):
    plan = L.PagePlan(P16, P16, P16, P16, P16, P16)
    refused(amd_lib, amd_lib.loom_amd_page_table_reset(table(L, **bad), None), part)
    refused(amd_lib, amd_lib.loom_amd_page_table_plan(table(L, **bad), P16, P16, 3, C.byref(plan), None), part)
    refused(amd_lib, amd_lib.loom_amd_page_table_release(table(L, **bad), P16, None), part)


def test_plan_refusals(amd_lib, L):
    def plan(i=None, v=0):
        f = [P16] * 6
        if i is not None:
            f[i] = v
        return C.byref(L.PagePlan(*f))

    fn = amd_lib.loom_amd_page_table_plan
    refused(amd_lib, fn(None, P16, P16, 3, plan(), None), "null")
    refused(amd_lib, fn(table(L), None, P16, 3, plan(), None), "null")
    refused(amd_lib, fn(table(L), P16, None, 3, plan(), None), "null")
    refused(amd_lib, fn(table(L), P16, P16, 3, None, None), "null")
    refused(amd_lib, fn(table(L), P16, P16, -1, plan(), None), "shape")
    for i in range(6):
        refused(amd_lib, fn(table(L), P16, P16, 3, plan(i), None), "null")
    refused(amd_lib, fn(table(L), P16, P16, 3, plan(5, P16 + 4), None), "aligned")
    refused(amd_lib, amd_lib.loom_amd_page_table_release(table(L), None, None), "null")


@pytest.mark.parametrize("bad,part", [(dict(k=0), "null"), (dict(v_scale=0), "null"), (dict(num_pages=0), "positive"),
                                      (dict(kv_heads=0), "positive"), (dict(kv_heads=70000), "heads"),
                                      (dict(page_size=48), "page_size"), (dict(head_dim=96), "head_dim"),
                                      (dict(head_dim=512), "head_dim"), (dict(num_pages=2 ** 27), "2^31"),
                                      (dict(k=P16 + 8), "aligned"), (dict(v=P16 + 1), "aligned")])
def test_cache_refusals(amd_lib, L, bad, part):
    c = cache(L, **bad)
    refused(amd_lib, amd_lib.loom_amd_kv_append(c, P16, P16, 0, 3, 128, 128, P16, None), part)
    refused(amd_lib, amd_lib.loom_amd_kv_read(c, P16, 3, P16, P16, None), part)
    refused(amd_lib, amd_lib.loom_amd_paged_attention(c, P16, 4, 8, P16, P16, P16, 0, 3, 4, 256, 0.1, 100, P16, 256, P16,
                                                      1 << 30, None), part)


def test_append_and_read_refusals(amd_lib, L):
    c, fn = cache(L), amd_lib.loom_amd_kv_append
    refused(amd_lib, fn(None, P16, P16, 0, 3, 128, 128, P16, None), "null")
    refused(amd_lib, fn(c, P16, P16, 2, 3, 128, 128, P16, None), "fp32 or bf16")
    refused(amd_lib, fn(c, P16, P16, 0, -1, 128, 128, P16, None), "shape")
    refused(amd_lib, fn(c, None, P16, 0, 3, 128, 128, P16, None), "null")
    refused(amd_lib, fn(c, P16, P16, 0, 3, 128, 128, None, None), "null")
    refused(amd_lib, fn(c, P16, P16, 0, 3, 127, 128, P16, None), "strides")
    refused(amd_lib, fn(c, P16, P16, 0, 3, 128, 0, P16, None), "strides")
    assert fn(c, None, None, 0, 0, 0, 0, None, None) == 0  # no rows: nothing to do
    rd = amd_lib.loom_amd_kv_read
    refused(amd_lib, rd(c, P16, 3, P16 + 4, P16, None), "aligned")
    refused(amd_lib, rd(c, None, 3, P16, P16, None), "null")
    refused(amd_lib, rd(c, P16, -3, P16, P16, None), "shape")
    assert rd(c, None, 0, None, None, None) == 0


def test_attention_refusals(amd_lib, L):
    good = dict(cache=cache(L), pages=P16, requests=4, max_pages=8, row_start=P16, positions=P16, q=P16, type=0, rows=3,
                heads=4, q_stride=256, scale=0.1, max_context=100, out=P16, out_stride=256, ws=P16, bytes=1 << 30)

    def call(**kw):
        a = dict(good, **kw)
        return amd_lib.loom_amd_paged_attention(*a.values(), None)

    for kw, part in ((dict(cache=None), "null"), (dict(requests=0), "shape"), (dict(rows=-1), "shape"),
                     (dict(heads=0), "shape"), (dict(heads=3), "divide"), (dict(rows=2 ** 30), "2^31"),
                     (dict(max_pages=0), "max_pages"), (dict(max_pages=2 ** 27), "max_pages"),
                     (dict(max_context=129), "max_context"), (dict(max_context=-1), "max_context"),
                     (dict(type=3), "fp32, bf16 or fp64"), (dict(scale=float("inf")), "finite"),
                     (dict(scale=float("nan")), "finite"), (dict(pages=None), "null"), (dict(row_start=None), "null"),
                     (dict(positions=None), "null"), (dict(q=None), "null"), (dict(out=None), "null"),
                     (dict(q_stride=255), "strides"), (dict(out_stride=0), "strides"), (dict(ws=P16 + 8), "aligned")):
        refused(amd_lib, call(**kw), part)
    assert call(rows=0, q=None, out=None) == 0
    n = C.c_size_t()
    size = amd_lib.loom_amd_paged_attention_workspace
    assert size(1, 20, 5, 128, 1, 4096, C.byref(n)) == 0 and n.value > 0
    long = dict(cache=cache(L, num_pages=2000, kv_heads=5, head_dim=128), max_pages=256, max_context=4096, rows=1, requests=1,
                heads=20, q_stride=2560, out_stride=2560)
    refused(amd_lib, call(**long, bytes=n.value - 1), "workspace")
    refused(amd_lib, call(**long, ws=None, bytes=0), "workspace")
    refused(amd_lib, size(1, 20, 5, 96, 1, 4096, C.byref(n)), "head_dim")
    refused(amd_lib, size(1, 20, 3, 128, 1, 4096, C.byref(n)), "divide")
    refused(amd_lib, size(1, 20, 5, 128, 1, 4096, None), "null")


def test_sample_refusals(amd_lib):
    n = C.c_size_t()
    size, fn = amd_lib.loom_amd_sample_workspace, amd_lib.loom_amd_sample
    refused(amd_lib, size(0, 3, C.byref(n)), "shape")
    refused(amd_lib, size(8388609, 3, C.byref(n)), "vocab")
    refused(amd_lib, size(10, 3, None), "null")
    assert size(1000, 3, C.byref(n)) == 0
    o = (None, None, None, None)
    refused(amd_lib, fn(P16, 1000, 1000, -1, *o, P16, P16, P16, n.value, None), "shape")
    refused(amd_lib, fn(None, 1000, 1000, 3, *o, P16, P16, P16, n.value, None), "null")
    refused(amd_lib, fn(P16, 1000, 1000, 3, *o, None, P16, P16, n.value, None), "null")
    refused(amd_lib, fn(P16, 1000, 1000, 3, *o, P16, None, P16, n.value, None), "null")
    refused(amd_lib, fn(P16, 999, 1000, 3, *o, P16, P16, P16, n.value, None), "stride")
    refused(amd_lib, fn(P16, 1000, 1000, 3, *o, P16, P16, P16, n.value - 1, None), "workspace")
    refused(amd_lib, fn(P16, 1000, 1000, 3, *o, P16, P16, None, n.value, None), "workspace")
    refused(amd_lib, fn(P16, 1000, 1000, 3, *o, P16, P16, P16 + 4, n.value, None), "aligned")
    assert fn(None, 0, 1000, 0, *o, None, None, None, 0, None) == 0


def test_block_forward_paged_refusals(amd_lib, L):
    refused(amd_lib, amd_lib.loom_amd_block_forward_paged(None, P16, 3, cache(L), P16, 4, 8, P16, P16, P16, 100, None, None),
            "block is null")


def test_python_refusals(amd_lib):
    from loom_amd import paged, transformer
    for kw in (dict(page_size=20), dict(requests=0), dict(max_pages=0), dict(num_pages=-1)):
        with pytest.raises(ValueError):
            paged.PageTable(**{**dict(requests=2, max_pages=3, num_pages=4, page_size=16), **kw})
    with pytest.raises(ValueError):
        paged.PageTable(2, 3, 4, 16, device="cpu")
    for a in ((4, 20, 2, 64), (4, 16, 2, 96), (0, 16, 2, 64), (4, 16, 0, 64)):
        with pytest.raises(ValueError):
            paged.PagedCache(*a)
    k, s = torch.zeros(2, 1, 16, 64, dtype=torch.int8), torch.zeros(2, 1)
    with pytest.raises(ValueError, match="device"):
        paged.PagedCache.from_tensors(k, k.transpose(2, 3).contiguous(), s, s)
    with pytest.raises(ValueError):
        paged.PagedCache.from_tensors(k[0], k, s, s)
    with pytest.raises(ValueError, match="device tensor"):
        transformer.sample(torch.zeros(2, 10), torch.zeros(2))


def test_sampling_restatement():
    """The restatement that the GPU tests rely on, on cases worked by hand."""
    import numpy as np

    from tests import paged_ref as ref
    x = np.log(np.array([1, 4, 2, 4, 1], np.float64)).astype(np.float32)  # ranked 1, 3, 2, 0, 4; masses 1 4 2 4 1
    big = 1e9

    def s(u, t=1.0, k=0, p=1.0, mp=0.0):
        return ref.sample(x, t, k, np.float32(p), np.float32(mp), np.float32(u))

    assert [s(u) for u in (0.0, 0.08, 0.09, 0.41, 0.42, 0.58, 0.59, 0.91, 0.92)] == [0, 0, 1, 1, 2, 2, 3, 3, 4]
    assert [s(u, k=1) for u in (0.0, 0.99)] == [1, 1]
    assert [s(u, k=2) for u in (0.4, 0.6)] == [1, 3]
    assert [s(u, k=4) for u in (0.05, 0.99)] == [0, 3]  # of the two equal last ones the lower index
    assert [s(u, p=0.3) for u in (0.0, 0.99)] == [1, 1]
    assert [s(u, p=0.6) for u in (0.4, 0.6)] == [1, 3]
    assert [s(u, mp=0.4) for u in (0.0, 0.5, 0.9)] == [1, 2, 3]
    assert s(0.9, t=0.0) == 1 and s(0.2, t=big) == 1 and s(0.99, t=big) == 4
    assert [s(u, k=3, p=0.75) for u in (0.4, 0.6)] == [1, 3]  # 8 of 10 of the first three


def test_table_restatement():
    from tests import paged_ref as ref
    t = ref.Tables(3, 2, 3, 16)
    a = t.plan([0, 0, 0], [17, 1, 1], 20)
    assert a["slots"][:18].tolist() == list(range(17)) + [32] and a["slots"][18:].tolist() == [-1, -1]
    assert a["lens"].tolist() == [17, 1, 0] and a["request"].tolist() == [0] * 17 + [1, 2, -1]
    t.release([True, False, False])
    assert t.free == [0, 1]
    assert t.plan([0, 1, 0], [0, 0, 1], 1)["slots"].tolist() == [16]
