"""Drafts, cross attention and reading back over the key/value cache without a
GPU: the reference's closed forms, the Python checks, and the C entries over the
stand-in HIP runtime (refusals, launches, workspaces)."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path
from types import SimpleNamespace

import numpy as np
import pytest

sys.path.insert(0, str(Path(__file__).resolve().parent))
import kv_draft_reference as draft  # noqa: E402
import kv_reference as ref  # noqa: E402
import test_host_dispatch as host  # noqa: E402
from test_kvcache import Kv, _cpu_cache  # noqa: E402


# ---- the reference --------------------------------------------------------------

def test_reference_trees_are_closed_under_parents():
    new = [9, 0, 40]
    p = draft.trees(new, seed=1, bad=0.2)
    sees, depths = draft.tree(new, p)
    at = 0
    for n in new:
        for i in range(n):
            q = draft.parent_of(int(p[at + i]), i)
            want = np.zeros(sees.shape[1], bool)
            if q >= 0:
                want |= sees[at + q]
            want[i] = True
            assert np.array_equal(sees[at + i], want) and depths[at + i] == want.sum() - 1
        at += n


def test_reference_paths_are_walks_from_token_zero():
    p = np.array([-1, 0, 0, 1, 2, 2, 0], np.int32)
    drafted = np.array([9, 1, 2, 5, 3, 3, 2], np.int32)
    chosen = np.array([2, 5, 3, 0, 7, 8, 4], np.int32)
    path, lengths, answer = draft.accept([20], [7], p, drafted, chosen, 5)
    assert path.tolist() == [[0, 2, 4, -1, -1]] and lengths[0] == 16 and answer[0] == 7
    path, lengths, answer = draft.accept([20], [7], p, drafted, chosen, 2)
    assert path.tolist() == [[0, 2]] and lengths[0] == 15 and answer[0] == 3
    path, lengths, answer = draft.accept([4], [0], p[:0], drafted[:0], chosen[:0], 2)
    assert path.tolist() == [[-1, -1]] and lengths[0] == 4 and answer[0] == -1


def test_reference_keep_is_an_append_of_the_kept_tokens():
    b = ref.Batch(32, [75], [20], seed=1)
    whole, some = (ref.Cache(b.pages, 2, 32, 64, "f16", seed=1) for _ in range(2))
    r = np.random.default_rng(2)
    k, v = r.standard_normal((2, 20, 2, 64))
    for i in range(20):
        whole.write(b.table[0, (55 + i) // 32], (55 + i) % 32, k[i], v[i])
    path = np.array([[0, 2, 3, 11, 17, 19, -1]], np.int32)
    draft.keep(whole, b, path)
    for i, at in enumerate(path[0][:6]):
        some.write(b.table[0, (55 + i) // 32], (55 + i) % 32, k[at], v[at])
    for t in range(55, 61):
        for x, y in zip(whole.read(b.table[0, 1], t - 32), some.read(b.table[0, 1], t - 32)):
            assert np.array_equal(x, y)


def test_reference_attention_of_a_chain_is_causal():
    b = ref.Batch(32, [50, 9], [7, 9])
    c = ref.Cache(b.pages, 1, 32, 64, "bf16")
    ref.fill(c, b)
    q = np.random.default_rng(3).standard_normal((16, 2, 64))
    sees = np.concatenate((np.tril(np.ones((7, 9), bool)), np.tril(np.ones((9, 9), bool))))
    for x, y in zip(draft.attend(c, b, q, 0.1, sees), ref.attend(c, b, q, 0.1)):
        assert np.allclose(x, y, rtol=1e-12, atol=1e-12)


def test_reference_cross_attention_sees_all():
    b = ref.Batch(32, [50, 0], [3, 2])
    c = ref.Cache(b.pages, 1, 32, 64, "bf16")
    ref.fill(c, b)
    q = np.random.default_rng(3).standard_normal((5, 2, 64))
    out, lse, _ = draft.attend(c, b, q, 0.1)
    kv = [c.read(b.table[0, t // 32], t % 32) for t in range(50)]
    k, v = np.array([x[0][0] for x in kv]), np.array([x[1][0] for x in kv])
    p = np.exp(0.1 * q[:3] @ k.T)
    assert np.allclose(out[:3], p / p.sum(-1, keepdims=True) @ v, rtol=1e-12)
    assert (out[3:] == 0).all() and np.isneginf(lse[3:]).all()


# ---- Python checks ----------------------------------------------------------------

def _batch(new=(3, 2), **kw):
    import torch
    from gofann_amd.kvcache import KvBatch
    n = len(new)
    off = torch.tensor([sum(new[:i]) for i in range(n + 1)], dtype=torch.int32)
    return KvBatch(torch.zeros(n, 4, dtype=torch.int32), torch.full((n,), 200, dtype=torch.int32), off,
                   queries=sum(new), max_queries=max(new), max_length=200, **kw)


@pytest.fixture
def cache(monkeypatch):
    """A cache on the CPU whose C calls are noted."""
    d = _cpu_cache()
    calls = []

    class Lib:
        def __getattr__(self, name):
            return lambda *a: calls.append((name, a)) or 0

    d.lib = Lib()
    d.ctx = SimpleNamespace(lib=d.lib, handle=None, check=lambda rc: None, device=0, stream=0)
    monkeypatch.setattr(d, "_ready", lambda batch: None)
    d.calls = calls
    return d


def test_bits_that_are_refused(cache):
    import torch
    b, q = _batch(), torch.zeros(5, 4, 128, dtype=cache.dtype)
    good = torch.zeros(5, 1, dtype=torch.int32)
    cache.attend(b, q, sees=good)
    cache.attend(b, q, sees=torch.zeros(5, 9, dtype=torch.int32)[:, 2:4])
    assert cache.calls[-1][0] == "gofann_kv_draft_attention" and cache.calls[-1][1][7:9] == (2, 9)
    cache.attend(b, q, sees=torch.zeros(5, 0, dtype=torch.int32))
    assert cache.calls[-1][1][6] and cache.calls[-1][1][7] == 0  # an address that is not read
    n = len(cache.calls)
    for bad in (good[:4], good.long(), good[0], good[:, 0], torch.zeros(5, 4, dtype=torch.int32)[:, ::2],
                torch.zeros(1, 2, dtype=torch.int32).expand(5, 2), torch.zeros(2, 5, dtype=torch.int32).t()):
        with pytest.raises(ValueError, match="sees"):
            cache.attend(b, q, sees=bad)
    assert len(cache.calls) == n


def test_rows_of_bits_too_far_apart_are_refused(cache):
    import torch

    class Far(torch.Tensor):  # a view into more words than a 32-bit stride spans
        def stride(self, *axis):
            return 1 if axis == (1,) else 1 << 32

    b, q = _batch(), torch.zeros(5, 4, 128, dtype=cache.dtype)
    far = torch.zeros(5, 2, dtype=torch.int32).as_subclass(Far)
    with pytest.raises(ValueError, match="sees"):
        cache.attend(b, q, sees=far)


def test_rows_and_paths_that_are_refused(cache):
    import torch
    b = _batch()
    rows = torch.zeros(5, 2, 128, dtype=cache.dtype)
    cache.read(b)
    cache.read(b, k=rows)
    cache.keep(b, torch.zeros(2, 7, dtype=torch.int32))
    n = len(cache.calls)
    for kw in (dict(k=rows[:4]), dict(v=rows.float()), dict(k=rows, v=rows[:, :1].expand(5, 2, 128)),
               dict(k=torch.zeros(5, 4, 128, dtype=cache.dtype))):
        with pytest.raises(ValueError):
            cache.read(b, **kw)
    for path in (torch.zeros(3, 7, dtype=torch.int32), torch.zeros(2, 7), torch.zeros(14, dtype=torch.int32),
                 torch.zeros(2, 14, dtype=torch.int32)[:, ::2]):
        with pytest.raises(ValueError, match="path"):
            cache.keep(b, path)
    for q in (torch.zeros(4, 4, 128, dtype=cache.dtype), torch.zeros(5, 4, 64, dtype=cache.dtype),
              torch.zeros(5, 4, 128)):
        with pytest.raises(ValueError):
            cache.cross(b, q)
    with pytest.raises(ValueError, match="lse"):
        cache.cross(b, torch.zeros(5, 4, 128, dtype=cache.dtype), lse=torch.zeros(5, 3))
    assert len(cache.calls) == n


def test_drafts_on_another_device_are_refused():
    import torch
    from gofann_amd import kvcache
    ints = torch.zeros(5, dtype=torch.int32)
    ctx = SimpleNamespace(device=0, stream=0, lib=None, handle=None)
    with pytest.raises(ValueError, match="device"):
        kvcache.draft_tree(ctx, _batch(), ints)
    with pytest.raises(ValueError, match="device"):
        kvcache.draft_accept(ctx, _batch(), ints, ints, ints, 3)


def test_draft_rows_that_are_refused(monkeypatch):
    import torch
    from gofann_amd import kvcache
    monkeypatch.setattr(kvcache, "_current", lambda ctx: None)
    b = _batch()
    device = SimpleNamespace(type="cuda", index=0)
    monkeypatch.setattr(b, "device", device)
    ctx = SimpleNamespace(device=0)
    good = torch.zeros(5, dtype=torch.int32)

    def at(t):  # as if it were there
        return SimpleNamespace(shape=t.shape, dtype=t.dtype, device=device, is_contiguous=t.is_contiguous)

    kvcache._draft(ctx, b, parents=at(good))
    for bad in (at(good[:4]), at(good.long()), at(torch.zeros(10, dtype=torch.int32)[::2]), good):
        with pytest.raises(ValueError, match="parents"):
            kvcache._draft(ctx, b, parents=bad)
        with pytest.raises(ValueError, match="chosen"):
            kvcache._draft(ctx, b, parents=at(good), drafted=at(good), chosen=bad)


# ---- C entries over the stand-in runtime ------------------------------------------

class Drafts(Kv):
    def draft(self, h, cache=None, batch=None, heads=32, scale=0.1, sees=-1, words=4, stride=4, blocks=None,
              width=0, q=None, out=None):
        return self.lib.gofann_kv_draft_attention(
            h, cache or self.cache(), batch or self.batch(), q or self.rows(), heads, scale,
            self.p if sees == -1 else sees, words, stride, blocks, width, out or self.rows(), None)

    def cross(self, h, cache=None, batch=None, heads=32, scale=0.1, q=None, out=None):
        return self.lib.gofann_kv_cross_attention(h, cache or self.cache(), batch or self.batch(),
                                                  q or self.rows(), heads, scale, out or self.rows(), None)

    def read(self, h, cache=None, batch=None, k=-1, v=-1):
        return self.lib.gofann_kv_read(h, cache or self.cache(), batch or self.batch(),
                                       self.rows() if k == -1 else k, self.rows() if v == -1 else v)

    def keep(self, h, cache=None, batch=None, path=-1, width=8):
        return self.lib.gofann_kv_keep(h, cache or self.cache(), batch or self.batch(),
                                       self.p if path == -1 else path, width)

    def tree(self, h, batch=None, parents=-1, words=1, sees=-1, depths=-1):
        p = lambda x: self.p if x == -1 else x  # noqa: E731
        return self.lib.gofann_kv_draft_tree(h, batch or self.batch(), p(parents), words, p(sees), p(depths))

    def accept(self, h, batch=None, parents=-1, drafted=-1, chosen=-1, width=8, path=-1, lengths=-1, answer=-1):
        p = lambda x: self.p if x == -1 else x  # noqa: E731
        return self.lib.gofann_kv_draft_accept(h, batch or self.batch(), p(parents), p(drafted), p(chosen),
                                               width, p(path), p(lengths), p(answer))


def case_refusals(f: Drafts):
    h, L, p = f.context(), f.L, f.p
    inv, uns = L.ERR_INVALID, L.ERR_UNSUPPORTED
    bad = [(uns, f.cache(dim=96)), (uns, f.cache(page_size=16)), (uns, f.cache(elem=L.ELEM_F32)),
           (inv, f.cache(kv_heads=0)), (inv, f.cache(k_codes=None)), (inv, f.cache(v_codes=p + 8)),
           (inv, f.cache(box=None)), (uns, f.cache(pages=2 ** 31))]
    for rc, c in bad:
        assert f.draft(h, cache=c) == f.cross(h, cache=c) == f.read(h, cache=c) == f.keep(h, cache=c) == rc
    bad = [(inv, f.batch(lengths=None)), (inv, f.batch(page_table=None)), (inv, f.batch(table_stride=8)),
           (inv, f.batch(max_queries=5)), (inv, f.batch(query_offsets=None, queries=3)),
           (uns, f.batch(sequences=65536)), (uns, f.batch(max_length=2 ** 31)), (uns, f.batch(queries=2 ** 31))]
    for rc, b in bad:
        assert f.draft(h, batch=b) == f.cross(h, batch=b) == f.read(h, batch=b) == f.keep(h, batch=b) == rc
        assert f.tree(h, batch=b) == f.accept(h, batch=b) == rc
    for s in (0.0, -0.5, float("nan"), float("inf")):
        assert f.draft(h, scale=s) == f.cross(h, scale=s) == inv
    for n in (0, 12, 8 * 1025):
        assert f.draft(h, heads=n) == f.cross(h, heads=n) == inv
    for call in (f.draft, f.cross):
        assert call(h, q=f.rows(None)) == call(h, out=f.rows(p + 1)) == inv
    assert f.draft(h, sees=None) == f.draft(h, sees=p + 2) == f.draft(h, words=5) == inv
    assert f.draft(h, words=2 ** 28, stride=2 ** 28) == f.draft(h, blocks=p, width=0) == inv
    assert f.read(h, k=None, v=None) == f.read(h, k=f.rows(p + 1)) == f.read(h, v=f.rows(None)) == inv
    assert f.keep(h, path=None) == f.keep(h, path=p + 2) == f.keep(h, width=2 ** 24 + 1) == inv
    assert f.tree(h, parents=None) == f.tree(h, parents=p + 1) == f.tree(h, sees=p + 2) == inv
    assert f.tree(h, sees=None, depths=None) == f.tree(h, words=2 ** 27) == inv
    assert f.accept(h, width=0) == f.accept(h, width=2 ** 24 + 1) == f.accept(h, path=None) == inv
    for name in ("parents", "drafted", "chosen"):
        assert f.accept(h, **{name: None}) == f.accept(h, **{name: p + 1}) == inv
    for name in ("lengths", "answer"):
        assert f.accept(h, **{name: p + 2}) == inv
    many = dict(queries=2 ** 24, max_queries=2 ** 24)
    assert f.tree(h, batch=f.batch(**many)) == uns and f.read(h, batch=f.batch(**many)) == uns
    assert f.tree(h, batch=f.batch(queries=8193, max_queries=8193)) == uns
    for call in (f.draft, f.cross, f.read, f.keep, f.tree, f.accept):
        assert call(None) == inv
    assert f.lib.gofann_kv_draft_tree(h, None, p, 1, p, p) == inv
    assert f.lib.gofann_kv_draft_accept(h, None, p, p, p, 1, p, p, p) == inv
    assert not f.launched()


def case_what_may_be_missing(f: Drafts):
    h, ok = f.context(), f.L.OK
    assert f.read(h, k=None) == f.read(h, v=None) == f.tree(h, sees=None) == f.tree(h, depths=None) == ok
    assert f.accept(h, lengths=None) == f.accept(h, answer=None) == f.keep(h, path=None, width=0) == ok
    assert f.keep(h, cache=f.cache(box=None, box_scale=None)) == f.draft(h, words=0, stride=0) == ok
    assert len(f.launched()) >= 8


def case_nothing_to_do(f: Drafts):
    h = f.context()
    for b in (f.batch(sequences=0), f.batch(queries=0), f.batch(max_queries=0)):
        assert f.draft(h, batch=b, sees=None) == f.cross(h, batch=b) == f.read(h, batch=b) == f.L.OK
        assert f.keep(h, batch=b) == f.tree(h, batch=b) == f.L.OK
    assert f.accept(h, batch=f.batch(sequences=0)) == f.L.OK
    assert not f.launched()
    # sequences without tokens have paths too, empty ones
    assert f.accept(h, batch=f.batch(max_queries=0), parents=None, drafted=None, chosen=None) == f.L.OK
    assert len(f.launched()) == 1


def case_launches(f: Drafts):
    """Which kernels a call takes, by its rows, what there is to read, and its sequences."""
    h = f.context()

    def names(call, heads=32, dim=128, **kw):
        assert call(h, heads=heads, cache=f.cache(dim=dim), batch=f.batch(**kw)) == f.L.OK
        return [n.split("kernel")[0].split("kv_")[-1] for n, _ in f.launched()]

    shared, few = ["attention_shared_", "join_pieces_"], ["attention_shared_few_", "join_pieces_"]
    for call in (f.draft, f.cross):
        one = dict(sequences=1, queries=1)
        assert names(call, **one, max_length=2000) == ["attention_"]
        assert names(call, **one, max_length=32768) == ["attention_", "join_"]
        # more than 16 rows: shared out where there is something to share
        some = dict(sequences=1, queries=16, max_queries=16)
        assert names(call, **some, max_length=1000) == ["attention_"]
        assert names(call, **some, max_length=4000) == few
        assert names(call, **some, max_length=4000, dim=256) == few
        assert names(call, sequences=64, queries=1024, max_queries=16, max_length=1000) == few
        # 128 rows a workgroup, and enough of them
        many = dict(sequences=1, queries=128, max_queries=128)
        assert names(call, **many, max_length=4000) == shared
        assert names(call, **many, max_length=4000, dim=256) == few
        assert names(call, sequences=2, queries=256, max_queries=128, max_length=4000, dim=256) == shared
        # 288 rows: a third tile of 128 would be mostly empty
        assert names(call, sequences=1, queries=72, max_queries=72, max_length=4000) == few
        assert names(call, sequences=4, queries=4096, max_queries=1024) == ["attention_shared_"]
        # a filter's tiles are listed first, unless the list would be too long
        p = dict(visible=f.p, visible_stride=1024, visible_width=1024)
        assert names(call, **some, max_length=4000, **p) == ["live_", *few]
        assert names(call, sequences=1000, queries=16000, max_queries=16, max_length=2 ** 18,
                     table_width=4096, table_stride=4096, **p) == few
        # sequences past those that tiles are shared out over
        assert "attention_shared_few_" not in names(call, sequences=1025, queries=1025 * 16, max_queries=16)
    assert names(f.draft, **some, max_length=4000) == few
    assert f.draft(h, blocks=f.p, width=64, batch=f.batch(**some)) == f.L.OK
    assert [n for n, _ in f.launched() if "shared" in n] == []


def case_workspace_under_capture(f: Drafts):
    few, many = dict(queries=64, max_queries=16), dict(queries=512, max_queries=128)
    for call, kw in ((f.draft, {}), (f.cross, {}), (f.draft, few), (f.cross, few), (f.draft, many), (f.cross, many)):
        h = f.context(host.SIDE)
        big = f.batch(**kw)
        call = lambda h, to=call: to(h, batch=big)  # noqa: E731
        f.hip.fake_capture(host.SIDE)
        assert call(h) == f.L.ERR_NOMEM
        assert b"before capturing" in f.lib.gofann_last_error(h)
        assert not f.hip.fake_capture_broken() and not f.launched()
        # the others need none
        assert f.read(h) == f.keep(h) == f.tree(h) == f.accept(h) == f.L.OK
        f.hip.fake_capture(None)
        f.launched()
        assert call(h) == f.L.OK
        used = f.hip.fake_used()
        f.hip.fake_capture(host.SIDE)
        assert call(h) == f.L.OK and f.hip.fake_used() == used
        f.hip.fake_capture(None)
        f.launched()
        f.lib.gofann_destroy(h)


def case_out_of_memory(f: Drafts):
    h = f.context()
    f.hip.fake_limit(f.hip.fake_used() + 1024)
    assert f.draft(h) == f.cross(h) == f.L.ERR_NOMEM
    assert not f.launched()
    f.hip.fake_limit(host.GIB)
    assert f.draft(h) == f.cross(h) == f.L.OK


CASES = sorted(k[5:] for k in globals() if k.startswith("case_"))


@pytest.mark.parametrize("case", CASES)
def test_c_entries(case, hip_lib_path, tmp_path_factory):
    base = tmp_path_factory.getbasetemp() / "fake_hip_kv_draft"
    base.mkdir(exist_ok=True)
    res = subprocess.run([sys.executable, __file__, case, str(host._stub(base))], timeout=120,
                         capture_output=True, text=True)
    assert res.returncode == 0, res.stdout[-2000:] + res.stderr[-2000:]


if __name__ == "__main__":
    globals()["case_" + sys.argv[1]](Drafts(sys.argv[2]))
