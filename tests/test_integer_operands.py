"""Numbers past 32 bits in the calls of the shared-prefix attention, the rotation and the rotating paged write: never
taken by their low bits."""

from __future__ import annotations

import pytest
import torch

from pallas_flash import _lib, paged_flash_attention_prefix


# CPU tier: the argument blocks.
@pytest.mark.parametrize("block,field", [
    (_lib.PagedPrefixArgs, "prefix_len"), (_lib.PagedPrefixArgs, "prefix_pages"), (_lib.PagedPrefixArgs, "num_pages"),
    (_lib.RopeAxesArgs, "rope_len"), (_lib.RopeAxesArgs, "seq_len"), (_lib.RopePagedWriteArgs, "pages_per_seq"),
    (_lib.RopePagedWriteArgs, "num_pages"),
])
def test_blocks_refuse_numbers_past_32_bits(block, field):
    at = [name for name, _ in block._fields_].index(field)
    front = [kind() if hasattr(kind, "_length_") else None if kind is _lib.c_ptr else 0
             for _, kind in block._fields_[:at]]
    for n in (1 << 31, (1 << 32) + 1024, -(1 << 31) - 1):
        with pytest.raises(NotImplementedError, match=field):
            block(**{field: n})
        with pytest.raises(NotImplementedError, match=field):
            block(*front, n)
    for n in ((1 << 31) - 1, -(1 << 31), 0):
        assert getattr(block(**{field: n}), field) == getattr(block(*front, n), field) == n


# GPU tier: the calls.
@pytest.fixture
def cache():
    gen = torch.Generator("cuda").manual_seed(0)
    q = torch.randn(2, 4, 1, 64, device="cuda", generator=gen, dtype=torch.float32)
    k, v = (torch.randn(6, 2, 16, 64, device="cuda", generator=gen) for _ in range(2))
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    return q, k, v, ints(0, 1), 20, ints(2, 3, 4, 5).view(2, 2), ints(32, 7)


@pytest.mark.gpu
def test_reach_and_prefix_past_32_bits(cache):
    """A table past 2^31 tokens: a length on the device cannot count up to its reach; one on the host can be served."""
    q, k, v, pre, prefix, table, lens = cache
    want = paged_flash_attention_prefix(*cache)
    for pages in ((1 << 27) + 3, (1 << 28) + 1):  # 16-token pages: past 2^31, and 2^32 + 16
        far = pre[:1].expand(pages).clone()
        far[:2] = pre
        assert torch.equal(want, paged_flash_attention_prefix(q, k, v, far, prefix, table, lens))
        with pytest.raises(NotImplementedError):
            paged_flash_attention_prefix(q, k, v, far, torch.tensor(20, device="cuda"), table, lens)
        with pytest.raises(NotImplementedError):
            paged_flash_attention_prefix(q, k, v, far, torch.tensor(20, device="cuda", dtype=torch.int32), table, lens)
        with pytest.raises(NotImplementedError):
            paged_flash_attention_prefix(q, k, v, far, pages * 16, table, lens)
