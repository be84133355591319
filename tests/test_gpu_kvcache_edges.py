"""Edges of the 4-bit key/value cache on the GPU against its plain 64-bit
definition: filters that are slices, sequences longer than their page table,
batches of very unequal chunks, long chunks under filters and holes."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kv_reference as ref
from test_gpu_kvcache import check_attend, device_cache, rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(gpu_ctx):
    return gpu_ctx


def with_filter(b: ref.Batch, visible: torch.Tensor, **kw):
    """The batch on the device under another filter tensor."""
    from gofann_amd import kvcache
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    return kvcache.KvBatch(dev(b.table), dev(np.array(b.lens, np.int32)), dev(b.offsets),
                           queries=b.queries, max_queries=max(b.new), max_length=max(b.lens),
                           visible=visible, **kw)


# ---- filters ------------------------------------------------------------------

@pytest.mark.parametrize("new", [[1, 1, 1], [1, 9, 3]])
@pytest.mark.parametrize("width", [1, 4, 16])
def test_a_sliced_filter_hides_what_lies_past_its_words(ctx, width, new):
    """Columns of a larger tensor whose other bits are all set: positions past
    the slice are hidden, in the last row as in the others."""
    lens = [200, 130, 490]
    b = ref.Batch(32, lens, new, seed=5, visible=lambda s, n, r: r.random(n) < 0.7)
    b.bits[:, 32 * width:] = False
    big = torch.full((3, 20), -1, dtype=torch.int32, device="cuda")
    part = big[:, 20 - width:]
    words = np.packbits(b.bits[:, :32 * width].reshape(3, width, 32), axis=-1, bitorder="little")
    part.copy_(torch.from_numpy(words.view(np.int32)[..., 0].copy()))
    c = ref.Cache(b.pages, 2, 32, 64, "bf16", seed=1)
    ref.fill(c, b, seed=2)
    q, q64 = rows(np.random.default_rng(3), b.queries, 6, 64, "bf16")
    d, db = device_cache(ctx, c), with_filter(b, part)
    lse = torch.empty((b.queries, 6), device="cuda")
    check_attend(d.attend(db, q, lse=lse), lse, *ref.attend(c, b, q64, 64 ** -0.5))
    got = d.select(db, q, 5)
    assert np.array_equal(got.cpu().numpy(), ref.select(c, b, q64, 5, 1, 2))
    check_attend(d.attend(db, q, blocks=got, lse=lse), lse,
                 *ref.attend(c, b, q64, 64 ** -0.5, got.cpu().numpy()))


def test_a_filter_without_words_hides_everything(ctx):
    b = ref.Batch(32, [70, 40], [1, 3], seed=5)
    c = ref.Cache(b.pages, 1, 32, 64, "bf16", seed=1)
    ref.fill(c, b, seed=2)
    q, _ = rows(np.random.default_rng(3), b.queries, 2, 64, "bf16")
    d, db = device_cache(ctx, c), with_filter(b, torch.empty((2, 0), dtype=torch.int32, device="cuda"))
    lse = torch.zeros((b.queries, 2), device="cuda")
    assert (d.attend(db, q, lse=lse) == 0).all() and torch.isneginf(lse).all()
    assert (d.select(db, q, 4) == -1).all()
