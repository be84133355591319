"""The key/value cache without a GPU: the reference's own closed forms, the
Python checks, and the C entries over the stand-in HIP runtime (refusals, which
launches a call makes, what it allocates and what it does under capture)."""
from __future__ import annotations

import ctypes as C
import subprocess
import sys
from pathlib import Path
from types import SimpleNamespace

import numpy as np
import pytest

sys.path.insert(0, str(Path(__file__).resolve().parent))
import kv_reference as ref  # noqa: E402
import test_host_dispatch as host  # noqa: E402


# ---- the reference against brute force -------------------------------------------

@pytest.mark.parametrize("elem", ["bf16", "f16"])
def test_reference_quantizes_to_the_nearest_code_of_the_least_scale(elem):
    r = np.random.default_rng(1)
    x = r.standard_normal((40, 64)) * 2.0 ** r.integers(-12, 12, (40, 1))
    code, e = ref.quantize(x, elem)
    v = ref.values(code, e)
    g = x.reshape(40, 2, 32)
    top = np.abs(g).max(-1)
    lo, hi = ref.LIMITS[elem]
    fits = (e > lo) & (e < hi)
    assert (top <= 6 * 2.0 ** e)[fits].all() and (top > 6 * 2.0 ** (e - 1.0))[fits].all()
    grid = np.concatenate((ref.GRID, -ref.GRID))
    best = np.abs(g[..., None] - grid * 2.0 ** e[..., None, None]).min(-1)
    assert np.array_equal(np.abs(g - v.reshape(g.shape)), best)


def test_reference_ties_go_to_the_even_code():
    x = np.zeros((1, 32))
    x[0, :8] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0]
    code, e = ref.quantize(x, "bf16")
    assert e[0, 0] == 0 and list(code[0, :8]) == [0, 2, 2, 4, 4, 6, 6, 7]


def test_reference_box_holds_every_key():
    b = ref.Batch(32, [50], [0])
    c = ref.Cache(b.pages, 2, 32, 64, "bf16")
    ref.fill(c, b, magnitude=3.0)
    for j, n in ((0, 32), (1, 18)):
        pid = b.table[0, j]
        unit = 2.0 ** (c.box_scale[pid].astype(float) - 127)[:, None]
        for t in range(n):
            k = c.read(pid, t)[0]
            assert (k <= c.box[pid, :, 0] * unit).all() and (k >= c.box[pid, :, 1] * unit).all()


def test_reference_attention_is_a_softmax():
    b = ref.Batch(32, [40], [1])
    c = ref.Cache(b.pages, 1, 32, 64, "bf16")
    ref.fill(c, b)
    q = np.random.default_rng(3).standard_normal((1, 2, 64))
    kv = [c.read(b.table[0, t // 32], t % 32) for t in range(40)]
    k, v = np.array([x[0][0] for x in kv]), np.array([x[1][0] for x in kv])
    p = np.exp(q[0] @ k.T)
    out, lse, _ = ref.attend(c, b, q, 1.0)
    assert np.allclose(out[0], p / p.sum(-1, keepdims=True) @ v, rtol=1e-12)
    assert np.allclose(lse[0], np.log(p.sum(-1)), rtol=1e-12)


# ---- Python checks ----------------------------------------------------------------

def _cpu_cache(**kw):
    import torch
    from gofann_amd import kvcache
    shapes = kvcache._shapes(4, 2, 64, 128)
    t = {n: torch.zeros(s, dtype=torch.int8 if n == "box" else torch.uint8) for n, s in shapes.items()}
    t.update(kw)
    return kvcache.KvCache(SimpleNamespace(lib=None, handle=None, stream=0), **t)


def test_batches_that_are_refused():
    import torch
    from gofann_amd.kvcache import KvBatch
    table, lens = torch.zeros(3, 4, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    off = torch.arange(4, dtype=torch.int32)
    KvBatch(table, lens, max_length=9)
    KvBatch(table, lens, off, queries=3, max_queries=1, max_length=9)
    for args, kw in [((table[0], lens), {}), ((table, lens[:2]), {}), ((table.long(), lens), {}),
                     ((table, lens, off[:3]), dict(queries=3, max_queries=1)), ((table, lens, off), {}),
                     ((table, lens), dict(queries=4)), ((table, lens), dict(max_queries=2)),
                     ((table.t(), torch.ones(4, dtype=torch.int32)), {}),
                     ((table[:1].expand(3, 4), lens), {}),
                     ((table, lens), dict(visible=torch.zeros(2, 4, dtype=torch.int32))),
                     ((table, lens), dict(visible=torch.zeros(3, 4)))]:
        with pytest.raises(ValueError):
            KvBatch(*args, max_length=9, **kw)
    with pytest.raises(ValueError):
        KvBatch(table, lens, max_length=-1)


def test_caches_and_rows_that_are_refused():
    import torch
    from gofann_amd import kvcache
    d = _cpu_cache()
    assert (d.pages, d.kv_heads, d.page, d.dim) == (4, 2, 64, 128) and d.boxed
    assert not _cpu_cache(box=None, box_scale=None).boxed
    for kw in (dict(k_codes=torch.zeros(4, 2, 64, 48, dtype=torch.uint8)),
               dict(k_codes=torch.zeros(4, 2, 48, 64, dtype=torch.uint8)),
               dict(v_codes=torch.zeros(4, 2, 8, 16, 8, 2, dtype=torch.uint8)),
               dict(k_scales=torch.zeros(4, 2, 64, 4, dtype=torch.int8)),
               dict(v_scales=torch.zeros(8, 2, 8, 4, 8, dtype=torch.uint8)[::2]),
               dict(box=None), dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            _cpu_cache(**kw)
    with pytest.raises(ValueError):
        kvcache.KvCache.empty(SimpleNamespace(device=0), pages=1, kv_heads=1, dim=96)
    q = torch.zeros(5, 8, 128, dtype=torch.bfloat16)
    r = d._rows("q", q, 5, 8)
    assert (r.token_stride, r.head_stride) == (1024, 128)
    r = d._rows("q", q.transpose(0, 1).contiguous().transpose(0, 1), 5, 8)
    assert (r.token_stride, r.head_stride) == (128, 640)
    assert d._rows("q", q[:1].expand(5, 8, 128), 5, 8).token_stride == 0  # may be read
    for t, n, h, written in ((q, 4, 8, False), (q, 5, 4, False), (q.float(), 5, 8, False),
                             (q[..., :64], 5, 8, False), (q.transpose(1, 2), 5, 128, False),
                             (q[0], 5, 8, False), (q[:1].expand(5, 8, 128), 5, 8, True),
                             (q[:, :1].expand(5, 8, 128), 5, 8, True)):
        with pytest.raises(ValueError):
            d._rows("x", t, n, h, written)


# ---- C entries over the stand-in runtime ------------------------------------------

class Kv(host.Fake):
    def cache(self, **kw):
        p = self.p
        c = dict(k_codes=p, k_scales=p, v_codes=p, v_scales=p, box=p, box_scale=p, pages=1000,
                 kv_heads=8, page_size=64, dim=128, elem=self.L.ELEM_BF16)
        c.update(kw)
        return self.L.KvCacheView(*[c[n] for n, _ in self.L.KvCacheView._fields_])

    def batch(self, **kw):
        p = self.p
        c = dict(page_table=p, lengths=p, query_offsets=p, visible=None, sequences=4, table_width=512,
                 table_stride=512, visible_stride=0, queries=4, max_queries=1, max_length=32768)
        c.update(kw)
        return self.L.KvBatchView(*[c[n] for n, _ in self.L.KvBatchView._fields_])

    def rows(self, data=-1):
        return self.L.KvRows(self.p if data == -1 else data, 4096, 128)

    def attend(self, h, cache=None, batch=None, heads=32, scale=0.1, blocks=None, width=0, q=None, out=None):
        return self.lib.gofann_kv_attention(h, cache or self.cache(), batch or self.batch(), q or self.rows(),
                                            heads, scale, blocks, width, out or self.rows(), None)

    def select(self, h, cache=None, batch=None, heads=32, width=8, first=1, last=2, out=-1):
        return self.lib.gofann_kv_select(h, cache or self.cache(), batch or self.batch(), self.rows(), heads,
                                         width, first, last, self.p if out == -1 else out)

    def append(self, h, cache=None, batch=None, k=None, v=None):
        return self.lib.gofann_kv_append(h, cache or self.cache(), batch or self.batch(), k or self.rows(),
                                         v or self.rows(), None, None)


def case_refusals(f: Kv):
    h, L, p = f.context(), f.L, f.p
    inv, uns = L.ERR_INVALID, L.ERR_UNSUPPORTED
    bad = [(uns, f.cache(dim=96)), (uns, f.cache(page_size=16)), (uns, f.cache(elem=L.ELEM_F32)),
           (inv, f.cache(kv_heads=0)), (inv, f.cache(k_codes=None)), (inv, f.cache(v_codes=p + 8)),
           (inv, f.cache(v_scales=p + 4)), (inv, f.cache(box=p + 4)), (inv, f.cache(box=None)),
           (uns, f.cache(pages=2 ** 31)), (uns, f.cache(pages=2 ** 30, kv_heads=8))]
    for rc, c in bad:
        assert f.attend(h, cache=c) == f.append(h, cache=c) == f.select(h, cache=c) == rc
    bad = [(inv, f.batch(lengths=None)), (inv, f.batch(page_table=None)), (inv, f.batch(table_stride=8)),
           (inv, f.batch(max_queries=5)), (inv, f.batch(query_offsets=None, queries=3)),
           (uns, f.batch(sequences=65536)), (uns, f.batch(max_length=2 ** 31)), (uns, f.batch(queries=2 ** 31))]
    for rc, b in bad:
        assert f.attend(h, batch=b) == f.append(h, batch=b) == f.select(h, batch=b) == rc
    for s in (0.0, -0.5, float("nan"), float("inf")):
        assert f.attend(h, scale=s) == inv
    for n in (0, 12, 8 * 1025):
        assert f.attend(h, heads=n) == f.select(h, heads=n) == inv
    assert f.attend(h, blocks=p, width=0) == inv and f.attend(h, q=f.rows(None)) == inv
    assert f.attend(h, out=f.rows(p + 1)) == inv and f.append(h, k=f.rows(None)) == inv
    assert f.select(h, width=2) == f.select(h, width=0) == f.select(h, out=None) == inv
    assert f.select(h, first=2 ** 32 - 1, last=2) == inv
    assert f.select(h, cache=f.cache(box=None, box_scale=None)) == inv
    assert f.append(h, cache=f.cache(box=None, box_scale=None)) == L.OK
    for call in (f.attend, f.select, f.append):
        assert call(None) == inv
    many = f.batch(queries=2 ** 24, max_queries=2 ** 24)
    assert f.select(h, batch=many) == uns and f.attend(h, batch=many) == uns
    assert not [n for n, _ in f.launched() if "append" not in n]


def case_nothing_to_do(f: Kv):
    h = f.context()
    for b in (f.batch(sequences=0), f.batch(queries=0), f.batch(max_queries=0)):
        assert f.attend(h, batch=b) == f.select(h, batch=b) == f.append(h, batch=b) == f.L.OK
    assert not f.launched()


def case_launches(f: Kv):
    """Which kernels a call takes: splits joined within the launch up to 16, by
    a launch of their own past it; long chunks, and the few rows beside them."""
    h = f.context()

    def names(**kw):
        assert f.attend(h, batch=f.batch(**kw)) == f.L.OK
        return [n.split("kernel")[0].split("kv_")[-1] for n, _ in f.launched()]

    one = dict(sequences=1, queries=1)
    assert names(**one, max_length=30) == ["attention_"]
    assert names(**one, max_length=2000) == ["attention_"]
    assert names(**one, max_length=32768) == ["attention_", "join_"]
    chunk = dict(sequences=1, queries=2048, max_queries=2048)
    assert names(**chunk) == ["attention_wide_"]
    assert names(sequences=3, queries=2050, max_queries=2048, max_length=256) == ["attention_wide_", "attention_"]
    # as many rows, none of them long: not wide
    assert "attention_wide_" not in names(sequences=2048, queries=2048, max_queries=2)
    assert f.select(h, batch=f.batch(max_length=64 * 256)) == f.L.OK
    assert len(f.launched()) == 1
    assert f.select(h, batch=f.batch(queries=8, max_queries=2)) == f.L.OK
    assert ["pick" in n for n, _ in f.launched()] == [False, True]


def case_workspace_under_capture(f: Kv):
    """A captured call needs a workspace of its size from before; the buffer
    that a graph may keep outlives a later growth."""
    h = f.context(host.SIDE)
    f.hip.fake_capture(host.SIDE)
    big, small = f.batch(), f.batch(max_length=4096)
    assert f.attend(h, batch=small) == f.L.ERR_NOMEM
    assert b"before capturing" in f.lib.gofann_last_error(h)
    assert not f.hip.fake_capture_broken() and not f.launched()
    f.hip.fake_capture(None)
    assert f.attend(h, batch=small) == f.L.OK
    used = f.hip.fake_used()
    f.hip.fake_capture(host.SIDE)
    assert f.attend(h, batch=small) == f.L.OK and f.hip.fake_used() == used
    f.hip.fake_capture(None)
    assert f.attend(h, batch=big) == f.L.OK
    grown = f.hip.fake_used()
    assert grown > 2 * used - 4096  # the old buffers are still there
    f.lib.gofann_destroy(h)
    assert f.hip.fake_used() < used


def case_another_streams_capture_is_left_intact(f: Kv):
    f.hip.fake_capture(0x2000)
    assert f.attend(f.context(host.SIDE)) == f.L.OK
    assert not f.hip.fake_capture_broken()
    f.hip.fake_capture(None)


def case_out_of_memory(f: Kv):
    h = f.context()
    f.hip.fake_limit(f.hip.fake_used() + 1024)
    assert f.attend(h) == f.select(h, batch=f.batch(queries=8, max_queries=2)) == f.L.ERR_NOMEM
    assert not f.launched()
    f.hip.fake_limit(host.GIB)
    assert f.attend(h) == f.L.OK


CASES = sorted(k[5:] for k in globals() if k.startswith("case_"))


@pytest.mark.parametrize("case", CASES)
def test_c_entries(case, hip_lib_path, tmp_path_factory):
    base = tmp_path_factory.getbasetemp() / "fake_hip_kv"
    base.mkdir(exist_ok=True)
    res = subprocess.run([sys.executable, __file__, case, str(host._stub(base))], timeout=120,
                         capture_output=True, text=True)
    assert res.returncode == 0, res.stdout[-2000:] + res.stderr[-2000:]


if __name__ == "__main__":
    globals()["case_" + sys.argv[1]](Kv(sys.argv[2]))
