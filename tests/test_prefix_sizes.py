"""CPU tier: the shared-prefix attention's sizes near the ends of their 32-bit ranges, by its plan's workspace."""

from __future__ import annotations

import pytest

from pallas_flash import _lib
from test_prefix_validation import args

MOST = 0x7fffffff - (1 << 20)  # keys that a call counts


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def long_prefix(prefix_len, **over):
    a = dict(page_size=1024, prefix_len=prefix_len, prefix_pages=-(-prefix_len // 1024), num_pages=2, head_dim=64,
             pages_per_seq=0)  # no own keys: the workspace is the prefix's partials
    return args(**{**a, **over})


# Items for every CU by rows or heads alone: one chunk holds the whole prefix, and its length and the keys together pass
# 2^31; and the float32 streams' (at most 128 rows), whose waves are four to a workgroup.
@pytest.mark.parametrize("shape", [
    dict(batch=128, num_heads=256, num_kv_heads=1, dtype=1), dict(batch=1, num_heads=256, num_kv_heads=256, dtype=2),
    dict(batch=1, num_heads=2048, num_kv_heads=1024, dtype=0), dict(batch=1, num_heads=1030, num_kv_heads=1030, dtype=0),
    dict(batch=300, num_heads=512, num_kv_heads=256, dtype=0),
])
@pytest.mark.parametrize("prefix_len", [1 << 20, (1 << 30) + 5, 1_500_000_000, MOST])
def test_partials_of_a_long_prefix(L, shape, prefix_len):
    """One row of float32 partials for each query at least: no length leaves the prefix without a chunk."""
    need = L.pf_paged_prefix_attn_workspace_size(long_prefix(prefix_len, **shape))
    rows = shape["batch"] * shape["num_heads"]
    assert rows * (64 + 2) * 4 <= need <= 64 * rows * (64 + 2) * 4 + (1 << 28)


def test_lengths_past_the_range_are_refused(L):
    shape = dict(batch=128, num_heads=256, num_kv_heads=1, dtype=1)
    assert L.pf_paged_prefix_attn_workspace_size(long_prefix(MOST + 1, **shape)) == 0
    assert L.pf_paged_prefix_attn(long_prefix(MOST + 1, **shape), None) == _lib.PF_ERR_UNSUPPORTED


@pytest.mark.parametrize("batch,heads", [(600_000, 32), (1 << 24, 1)])
def test_batches_past_the_launch_are_refused(L, batch, heads):
    """A launch has fewer than 2^32 threads: the merge's 256 for each sequence and KV head, at least."""
    a = dict(batch=batch, num_heads=heads, num_kv_heads=heads, dtype=1)
    assert L.pf_paged_prefix_attn_workspace_size(long_prefix(2048, **a)) == 0
    assert L.pf_paged_prefix_attn(long_prefix(2048, **a), None) == _lib.PF_ERR_UNSUPPORTED
    a["batch"] = (1 << 24) // heads - 1
    assert L.pf_paged_prefix_attn_workspace_size(long_prefix(2048, **a)) > 0
