"""Register budgets of the kernels for drafts and cross attention, from the
compiler's resource report: the waves a SIMD that they were measured at, and the
spills that they were measured with.  CPU only."""
from __future__ import annotations

import re
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

import pytest

sys.path.insert(0, str(Path(__file__).resolve().parent))
import test_kernel_resources as res  # noqa: E402

pytestmark = res.pytestmark
SOURCES = [f"kv_{kind}_{dim}.hip" for kind in ("draft", "cross") for dim in (64, 128, 256)] + \
    ["kv_settle.hip", "kv_read.hip", "kv_cache.hip"]


@pytest.fixture(scope="module")
def report(tmp_path_factory):
    d = tmp_path_factory.mktemp("kvdraft_res")
    with ThreadPoolExecutor(max_workers=4) as ex:
        return dict(zip(SOURCES, ex.map(lambda s: res._resources(s, d), SOURCES)))


@pytest.mark.parametrize("kind", ["draft", "cross"])
@pytest.mark.parametrize("dim,waves", [(64, {1: 5, 2: 3}), (128, {1: 4, 2: 2}), (256, {1: 2, 2: 1})])
def test_attention_of_few_rows(report, kind, dim, waves):
    """A draft's 16 rows of 128 channels leave one register too few."""
    seen = set()
    for label in ("19kv_attention_kernel", "30kv_attention_shared_few_kernel"):
        for name, r in res._kernels(report[f"kv_{kind}_{dim}.hip"], label).items():
            tiles = int(re.search(r"Li(\d)EEE", name).group(1))
            seen.add((label, tiles))
            spills = 1 if (kind, dim, tiles) == ("draft", 128, 1) else 0
            assert r["occupancy"] >= waves[tiles] and r["vgpr_spill"] <= spills, (name, r)
    assert seen >= {("30kv_attention_shared_few_kernel", 2), ("19kv_attention_kernel", 1)}


@pytest.mark.parametrize("kind", ["draft", "cross"])
@pytest.mark.parametrize("dim,waves", [(64, 3), (128, 2), (256, 1)])
def test_attention_of_many_rows_spills_nothing(report, kind, dim, waves):
    kernels = res._kernels(report[f"kv_{kind}_{dim}.hip"], "26kv_attention_shared_kernel")
    assert len(kernels) == 2
    for name, r in kernels.items():
        assert r["occupancy"] >= waves and r["vgpr_spill"] == r["scratch"] == 0, (name, r)


def test_the_others_spill_nothing(report):
    for source, label, waves in (("kv_settle.hip", "kv_tree_kernel", 5), ("kv_settle.hip", "kv_accept_kernel", 8),
                                 ("kv_settle.hip", "kv_keep_kernel", 6), ("kv_read.hip", "kv_read_kernel", 8),
                                 ("kv_cache.hip", "kv_live_kernel", 8)):
        kernels = res._kernels(report[source], label)
        assert kernels
        for name, r in kernels.items():
            assert r["occupancy"] >= waves and r["vgpr_spill"] == r["scratch"] == 0, (name, r)
