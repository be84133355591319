"""Register budgets of the key/value cache's kernels, from the compiler's
resource report: the waves a SIMD that they were measured at, and the spills
that they were measured with.  CPU only: hipcc cross-compiles without a GPU."""
from __future__ import annotations

import re
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

import pytest

sys.path.insert(0, str(Path(__file__).resolve().parent))
import test_kernel_resources as res  # noqa: E402

pytestmark = res.pytestmark
SOURCES = ("kv_attention_64.hip", "kv_attention_128.hip", "kv_attention_256.hip", "kv_select.hip", "kv_append.hip")


@pytest.fixture(scope="module")
def report(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv_res")
    with ThreadPoolExecutor(max_workers=len(SOURCES)) as ex:
        return dict(zip(SOURCES, ex.map(lambda s: res._resources(s, d), SOURCES)))


@pytest.mark.parametrize("dim,tiles,waves", [(64, 1, 5), (64, 2, 3), (128, 1, 4), (128, 2, 2), (256, 1, 2)])
def test_attention_of_few_rows_spills_nothing(report, dim, tiles, waves):
    for name, r in res._kernels(report[f"kv_attention_{dim}.hip"], "19kv_attention_kernel").items():
        if int(re.search(r"Li(\d)EEE", name).group(1)) == tiles:
            assert r["occupancy"] >= waves and r["vgpr_spill"] == r["scratch"] == 0, (name, r)


@pytest.mark.parametrize("dim,waves,spills", [(64, 3, 0), (128, 2, 0), (256, 2, 29)])
def test_attention_of_long_chunks(report, dim, waves, spills):
    """256 channels: eight tiles of output and the queries leave 29 registers too few."""
    for name, r in res._kernels(report[f"kv_attention_{dim}.hip"], "24kv_attention_wide_kernel").items():
        assert r["occupancy"] >= waves and r["vgpr_spill"] <= spills, (name, r)


def test_choice_of_blocks(report):
    """Kernels for one token spill nothing; for several, those of 128 channels
    spill 6 registers, 29 where a token has one or two heads."""
    for name, r in res._kernels(report["kv_select.hip"], "kv_select_kernel").items():
        dim, quads, many = re.search(r"Li(\d+)ELb(\d)ELb(\d)EEE", name).groups()
        spills = (6 if quads == "1" else 29) if dim == "128" and many == "1" else 0
        assert r["occupancy"] >= (2 if dim == "256" else 3) and r["vgpr_spill"] <= spills, (name, r)
    for name, r in res._kernels(report["kv_select.hip"], "kv_pick_kernel").items():
        assert r["occupancy"] == 8 and r["vgpr_spill"] == 0, (name, r)


def test_append(report):
    for name, r in res._kernels(report["kv_append.hip"], "kv_append_kernel").items():
        assert r["occupancy"] >= 7 and r["vgpr_spill"] == 0, (name, r)
