"""GPU tier: the shared-prefix attention at the ends of its ranges, against float64."""

from __future__ import annotations

import pytest
import torch

from gpu_util import note
from pallas_flash import paged_flash_attention_prefix
from test_gpu_prefix import check, make, reference

pytestmark = pytest.mark.gpu


def within(got, want, bound):
    eps = torch.finfo(got.dtype).eps
    return ((got.double() - want).abs() <= bound + eps / 2 * (want.abs() + bound) + 2.0 ** -25).all()


@pytest.mark.parametrize("dt,heads,page", [("bf16", 256, 256), ("f32", 1024, 64)])
def test_short_prefix_in_a_table_past_2_30_tokens(dt, heads, page):
    """The table's reach and its one chunk's length together pass 2^31; the prefix on the device has 300 tokens."""
    note(f"prefix {dt} {heads} heads, a table of 1.6e9 tokens, 300 of them the prefix")
    q, k, v, ptab, prefix, table, lens = make(dt, 1, heads, heads, 64, page, 300, [page // 2])
    far = ptab[:1].expand(1_600_000_000 // page).clone()
    far[:ptab.shape[0]] = ptab
    n = torch.tensor(prefix, dtype=torch.int32, device="cuda")
    got = paged_flash_attention_prefix(q, k, v, far, n, table, lens)
    want, bound = reference(q, k, v, ptab, prefix, table, lens)
    assert within(got, want, bound)
