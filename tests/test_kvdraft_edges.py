"""Edges of drafts and cross attention without a GPU: the example's bounds, and plans
of calls with large ones over the stand-in HIP runtime."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path
from types import SimpleNamespace

import pytest

sys.path.insert(0, str(Path(__file__).resolve().parent))
import test_host_dispatch as host  # noqa: E402
from test_kvdraft import Drafts  # noqa: E402


# ---- the example ------------------------------------------------------------------

def test_settled_drafts_leave_the_room_that_they_did_not_take(monkeypatch):
    """A session is full when its longest sequence is, not when its drafts could have made it so."""
    import torch
    from gofann_amd import longcontext
    s = longcontext.Session.__new__(longcontext.Session)
    s.sequences, s.capacity, s.filled = 2, 40, 0
    s.table = torch.zeros((2, 2), dtype=torch.int32)
    s.lengths = torch.zeros(2, dtype=torch.int32)
    s.visible = torch.full((2, 2), -1, dtype=torch.int32)
    kept = [1, 2]  # tokens of each draft

    def accept(ctx, batch, parents, drafted, chosen, width):
        return None, s.lengths - batch.max_queries + torch.tensor(kept, dtype=torch.int32), None

    monkeypatch.setattr(longcontext, "draft_tree", lambda ctx, batch, parents: (None, None))
    monkeypatch.setattr(longcontext, "draft_accept", accept)
    bounds = []

    def attend(batch, q, **kw):
        bounds.append(batch.max_length)
        assert batch.max_length >= int(s.lengths.max())

    s.cache = SimpleNamespace(ctx=None, append=lambda *a: None, attend=attend, keep=lambda *a: None)
    q = torch.zeros((16, 4, 64))
    for i in range(17):  # 8 tokens of 40, two of them kept: 17 drafts, not 5
        s.draft(q, q, q, None)
        s.settle(None, None, 8)
        assert s.lengths.tolist() == [i + 1, 2 * i + 2]
    with pytest.raises(ValueError, match="full"):
        s.draft(q, q, q, None)
    assert s.lengths.tolist() == [17, 34] and s.filled == 34 and s.pending is None
    s.grow(6)
    assert s.lengths.tolist() == [23, 40] and max(bounds) <= 40
    with pytest.raises(ValueError, match="full"):
        s.grow(1)


def test_a_refused_draft_keeps_the_renewed_bound(monkeypatch):
    import torch
    from gofann_amd import longcontext
    s = longcontext.Session.__new__(longcontext.Session)
    s.sequences, s.capacity, s.filled, s.loose = 1, 40, 38, True
    s.table, s.visible = torch.zeros((1, 2), dtype=torch.int32), torch.zeros((1, 2), dtype=torch.int32)
    s.lengths = torch.full((1,), 9, dtype=torch.int32)

    def refuse(*a):
        raise ValueError("refused")

    monkeypatch.setattr(longcontext, "draft_tree", refuse)
    s.cache = SimpleNamespace(ctx=None)
    q = torch.zeros((8, 4, 64))
    with pytest.raises(ValueError, match="refused"):
        s.draft(q, q, q, None)
    assert s.filled == 9 and s.lengths.tolist() == [9] and s.pending is None


# ---- C entries over the stand-in runtime ------------------------------------------

def case_bounds_past_a_count_of_tiles(f: Drafts):
    """Tiles are counted in 32 bits.  From 2^30 on, by the call's bounds, the 128-row kernel takes a row
    tile a workgroup, which counts nothing, and few rows go by splits."""
    h = f.context()

    def names(call, heads=32, dim=128, length=2 ** 20, **kw):
        width = -(-length // 64)
        b = f.batch(table_width=width, table_stride=width, max_length=length, **kw)
        assert call(h, heads=heads, cache=f.cache(dim=dim), batch=b) == f.L.OK
        grids = [f.hip.fake_workgroups(i) for i in range(f.hip.fake_launches())]
        return [(n.split("kernel")[0].split("kv_")[-1], g) for (n, _), g in zip(f.launched(), grids)]

    for call in (f.draft, f.cross):
        # so many row tiles that each is a workgroup's, whatever the bound
        many = dict(sequences=64, queries=64 * 2048, max_queries=2048)
        for length in (2 ** 14, 2 ** 19, 2 ** 20, 2 ** 24):
            assert names(call, length=length, **many) == [("attention_shared_", 64 * 64 * 8)]
        # 256 channels are shared out up to (4096 + 64) x 8 x (tiles + 16) = 2^30
        for tiles, shared in ((32247, True), (32248, False)):
            got = names(call, dim=256, length=tiles * 32, **many)
            assert [n for n, _ in got] == ["attention_shared_", "join_pieces_"][:1 + shared]
            assert got[0][1] == (256 if shared else 64 * 64 * 8)
        # one long chunk among decoding sequences: counted through the sequences, or a grid
        mixed = dict(sequences=1000, queries=999 + 700, max_queries=700)
        assert [n for n, _ in names(call, **mixed)] == ["attention_shared_", "join_pieces_"]
        assert names(call, length=2 ** 24, **mixed) == [("attention_shared_", 22 * 1000 * 8)]
        # more rows than 65,535 tiles of 32
        long = dict(sequences=1, queries=600_000, max_queries=600_000)
        assert names(call, **long) == [("attention_shared_", 18750 * 8)]
        few = dict(sequences=1000, queries=16000, max_queries=16)
        assert [n for n, _ in names(call, **few)] == ["attention_shared_few_", "join_pieces_"]
        assert names(call, length=2 ** 22, **few)[0][0] == "attention_"


CASES = sorted(k[5:] for k in globals() if k.startswith("case_"))


@pytest.mark.parametrize("case", CASES)
def test_c_entries(case, hip_lib_path, tmp_path_factory):
    base = tmp_path_factory.getbasetemp() / "fake_hip_kv_draft_edges"
    base.mkdir(exist_ok=True)
    res = subprocess.run([sys.executable, __file__, case, str(host._stub(base))], timeout=120,
                         capture_output=True, text=True)
    assert res.returncode == 0, res.stdout[-2000:] + res.stderr[-2000:]


if __name__ == "__main__":
    globals()["case_" + sys.argv[1]](Drafts(sys.argv[2]))
