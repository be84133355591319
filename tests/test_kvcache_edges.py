"""Edges of the key/value cache without a GPU: what the views hand to the C ABI,
and the C entries over the stand-in HIP runtime."""
from __future__ import annotations

import ctypes as C
import subprocess
import sys
from pathlib import Path

import pytest

sys.path.insert(0, str(Path(__file__).resolve().parent))
import test_host_dispatch as host  # noqa: E402
from test_kvcache import Kv  # noqa: E402


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


def case_append_without_a_page_table(f: Kv):
    h = f.context()
    for table in (None, f.p):
        assert f.append(h, batch=f.batch(page_table=table, table_width=0, table_stride=0)) == f.L.OK
    assert not f.launched()  # a grid of no workgroups is an error of the runtime


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
