"""Edges of the key/value cache without a GPU: what the views hand to the C ABI,
and the C entries over the stand-in HIP runtime."""
from __future__ import annotations

import ctypes as C
import subprocess
import sys
from pathlib import Path
from types import SimpleNamespace

import pytest

sys.path.insert(0, str(Path(__file__).resolve().parent))
import test_host_dispatch as host  # noqa: E402
from test_kvcache import Kv, _cpu_cache  # noqa: E402


def _batch(sequences=3, blocks=4, **kw):
    import torch
    from gofann_amd.kvcache import KvBatch
    table = torch.zeros(sequences, blocks, dtype=torch.int32)
    return KvBatch(table, torch.full((sequences,), 200, dtype=torch.int32), max_length=200, **kw)


# ---- views ------------------------------------------------------------------------

def test_a_column_slice_of_a_filter_ends_at_its_words():
    import torch
    big = torch.full((3, 16), -1, dtype=torch.int32)
    v = _batch(visible=big[:, 12:]).view
    assert (v.visible_stride, v.visible_width) == (16, 4)
    assert v.visible == big.data_ptr() + 48
    v = _batch(visible=big).view
    assert (v.visible_stride, v.visible_width) == (16, 16)
    v = _batch(1, visible=big[:1, 3:5]).view
    assert v.visible_width == 2 <= v.visible_stride
    assert _batch().view.visible_width == 0


@pytest.mark.parametrize("sequences", [1, 3])
def test_a_filter_without_words_is_not_no_filter(sequences):
    import torch
    for t in (torch.empty((sequences, 0), dtype=torch.int32),
              torch.zeros((sequences, 8), dtype=torch.int32)[:, 3:3]):
        v = _batch(sequences, visible=t).view
        assert v.visible and v.visible_stride == v.visible_width == 0


def test_the_batch_view_is_the_header_struct():
    """visible_width is the struct's last member, where the other fields' padding is."""
    from gofann_amd import _lib
    assert C.sizeof(_lib.KvBatchView) == 4 * 8 + 8 * 4
    v = _lib.KvBatchView()
    v.max_length, v.visible_width = 5, 7
    assert bytes(v)[-8:] == bytes([5, 0, 0, 0, 7, 0, 0, 0]) and v.visible_width == 7


@pytest.mark.parametrize("name", ["queries", "max_queries", "max_length"])
def test_bounds_past_32_bits_are_refused(name):
    """ctypes would hand on their low bits: a bound of 2^32 as one of 0."""
    import torch
    from gofann_amd.kvcache import KvBatch
    table, off = torch.zeros((3, 4), dtype=torch.int32), torch.arange(4, dtype=torch.int32)
    kw = dict(queries=3, max_queries=1, max_length=9)
    for wrong in (2 ** 32, 2 ** 32 + 9, -2 ** 32 + 9, -1):
        with pytest.raises(ValueError, match=name):
            KvBatch(table, off[1:], off, **{**kw, name: wrong})
    assert getattr(KvBatch(table, off[1:], off, **{**kw, name: 2 ** 32 - 1}).view, name) == 2 ** 32 - 1


@pytest.mark.parametrize("name", ["width", "first", "last"])
def test_counts_of_blocks_past_32_bits_are_refused(name, monkeypatch):
    import torch
    d = _cpu_cache()
    monkeypatch.setattr(d, "_ready", lambda batch: None)
    kw = dict(width=4, first=1, last=2)
    for wrong in (2 ** 32 + 1, -2 ** 32 + 4, -1):
        with pytest.raises(ValueError, match=name):
            d.select(_batch(), torch.zeros((3, 8, 128), dtype=d.dtype), **{**kw, name: wrong})


def _calls(cache, batch):
    import torch
    n, h = batch.queries, cache.kv_heads
    k, q = (torch.zeros(n, m, cache.dim, dtype=cache.dtype) for m in (h, 4 * h))
    return (lambda: cache.append(batch, k, k), lambda: cache.select(batch, q, 4),
            lambda: cache.attend(batch, q))


def test_arrays_on_another_device_than_the_contexts_are_refused(monkeypatch):
    """Host arrays, or another GPU's, would be addresses that the kernels cannot read."""
    from gofann_amd import _lib, kvcache
    monkeypatch.setattr(kvcache, "_raw_stream", lambda i: 0)
    d = _cpu_cache()
    d.ctx.device = 0
    for call in _calls(d, _batch()):
        with pytest.raises(ValueError, match="context's device"):
            call()
    # arrays in place, but torch's current device another: so is the default stream's
    monkeypatch.setattr(kvcache, "_current_device", lambda: 1, raising=False)
    d._index = 0
    for call in _calls(d, _batch()):
        with pytest.raises(_lib.GofannError, match="current device"):
            call()


@pytest.mark.parametrize("fails", ["append", "select", "attend"])
def test_a_refused_step_of_the_example_leaves_its_lengths(fails):
    import torch
    from gofann_amd.longcontext import Session
    s = Session.__new__(Session)
    s.sequences, s.capacity, s.filled = 2, 100, 10
    s.table = torch.zeros((2, 4), dtype=torch.int32)
    s.lengths = torch.full((2,), 10, dtype=torch.int32)
    s.visible = torch.full((2, 4), -1, dtype=torch.int32)

    def call(name):
        def f(batch, *a, **kw):
            assert batch.max_length == 13 and s.lengths.tolist() == [13, 13]
            if name == fails:
                raise ValueError("refused")
        return f

    s.cache = SimpleNamespace(**{n: call(n) for n in ("append", "select", "attend")})
    q = torch.zeros((6, 4, 64))
    with pytest.raises(ValueError, match="refused"):
        s.step(q, q, q, 8)
    assert s.filled == 10 and s.lengths.tolist() == [10, 10]
    with pytest.raises(ValueError, match="sequences"):
        s.step(q[:5], q[:5], q[:5], 8)
    assert s.filled == 10 and s.lengths.tolist() == [10, 10]
    fails = None
    s.step(q, q, q, 8)
    assert s.filled == 13


# ---- C entries over the stand-in runtime ------------------------------------------

def case_filter_width(f: Kv):
    h = f.context()

    def batch(stride, width):
        b = f.batch(visible=f.p, visible_stride=stride)
        b.visible_width = width
        return b

    for call in (f.attend, f.select, f.append):
        assert call(h, batch=batch(16, 17)) == f.L.ERR_INVALID
        assert call(h, batch=batch(16, 16)) == call(h, batch=batch(16, 0)) == f.L.OK
        assert call(h, batch=batch(0, 0)) == f.L.OK


def case_scales_past_the_range(f: Kv):
    """A scale is taken times log2(e): past 2.36e38 that is infinite, and 0 times it no number."""
    h = f.context()
    for scale, rc in ((2.4e38, f.L.ERR_INVALID), (3.0e38, f.L.ERR_INVALID), (2.3e38, f.L.OK), (1e-40, f.L.OK)):
        assert f.attend(h, scale=scale) == rc, scale


def case_append_without_a_page_table(f: Kv):
    h = f.context()
    for table in (None, f.p):
        assert f.append(h, batch=f.batch(page_table=table, table_width=0, table_stride=0)) == f.L.OK
    assert not f.launched()  # a grid of no workgroups is an error of the runtime


def _mixed(f: Kv, **kw):
    """63 sequences of one token beside a chunk of 512, under a far bound on the length."""
    b = dict(sequences=64, queries=63 + 512, max_queries=512, max_length=131072, table_width=2048,
             table_stride=2048)
    b.update(kw)
    return f.batch(**b)


def case_workspace_by_the_rows_there_are(f: Kv):
    f.hip.fake_workgroups.restype = C.c_uint64
    f.hip.fake_limit(8 * host.GIB)  # the arrays are never touched
    before = f.hip.fake_used()
    # one token each: 64 x 32 rows of 86 splits of 130 floats
    h = f.context()
    b = f.batch(sequences=64, queries=64, max_length=131072, table_width=2048, table_stride=2048)
    assert f.attend(h, batch=b) == f.L.OK
    assert f.hip.fake_used() - before <= 64 * 32 * 86 * 130 * 4
    f.lib.gofann_destroy(h)
    for kw in ({}, dict(blocks=f.p, width=64), dict(batch=_mixed(f, max_length=1 << 20, table_width=1 << 14,
                                                                table_stride=1 << 14))):
        h = f.context()
        f.launched()
        assert f.attend(h, batch=kw.pop("batch", _mixed(f)), **kw) == f.L.OK
        assert f.hip.fake_used() - before <= 520 << 20
        # 135 tiles of 32 rows, listed 575 of 16, of 8 heads in at most 56 splits
        assert f.hip.fake_workgroups(0) <= 575 * 8 * 56
        f.lib.gofann_destroy(h)


def case_workspace_beside_long_chunks(f: Kv):
    """What the wide launch leaves, however many rows it has itself."""
    f.hip.fake_limit(8 * host.GIB)
    before = f.hip.fake_used()
    h = f.context()
    assert f.attend(h, batch=_mixed(f, queries=63 + 4096, max_queries=4096)) == f.L.OK
    assert ["wide" in n for n, _ in f.launched()] == [True, False, False]
    assert f.hip.fake_used() - before <= 520 << 20


CASES = sorted(k[5:] for k in globals() if k.startswith("case_"))


@pytest.mark.parametrize("case", CASES)
def test_c_entries(case, hip_lib_path, tmp_path_factory):
    base = tmp_path_factory.getbasetemp() / "fake_hip_kv_edges"
    base.mkdir(exist_ok=True)
    res = subprocess.run([sys.executable, __file__, case, str(host._stub(base))], timeout=120,
                         capture_output=True, text=True)
    assert res.returncode == 0, res.stdout[-2000:] + res.stderr[-2000:]


if __name__ == "__main__":
    globals()["case_" + sys.argv[1]](Kv(sys.argv[2]))
