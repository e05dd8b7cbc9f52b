"""Numbers past 32 bits in the calls of the shared-prefix attention, the rotation and the rotating paged write: never
taken by their low bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from pallas_flash import _lib, paged_flash_attention_prefix, precompute_rope, write_to_paged_cache_rope


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


def test_wide_integers_stay_out_of_bounds():
    for n, want in ((5, 5), (-1, -1), ((1 << 32) + 5, 0x7fffffff), (1 << 31, 0x7fffffff), ((1 << 63) - 1, 0x7fffffff),
                    (-(1 << 63), -0x80000000), (5 - (1 << 32), -0x80000000)):
        t = _lib.device_ints(torch.tensor([n, 3]), "cpu")
        assert t.dtype == torch.int32 and t.tolist() == [want, 3]
    for dt in (torch.int8, torch.uint8, torch.int16, torch.int32):
        assert _lib.device_ints(torch.tensor([7, 100], dtype=dt), "cpu").tolist() == [7, 100]


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


@pytest.mark.gpu
def test_attention_of_wide_integers(cache):
    q, k, v, pre, _, table, lens = cache
    wide = lambda *x: torch.tensor(x, dtype=torch.int64, device="cuda")  # noqa: E731
    for n, same in (((1 << 32) + 5, 32), ((1 << 31) + 1, 32), (-(1 << 32) + 5, 0), (11, 11)):
        want = paged_flash_attention_prefix(q, k, v, pre, same, table, lens)
        assert torch.equal(want, paged_flash_attention_prefix(q, k, v, pre, wide(n), table, lens))
    small = torch.tensor(11, dtype=torch.int8, device="cuda")
    assert torch.equal(paged_flash_attention_prefix(q, k, v, pre, 11, table, lens),
                       paged_flash_attention_prefix(q, k, v, pre, small, table, lens))
    want = paged_flash_attention_prefix(q, k, v, pre, 20, table, lens * 0 + 32)
    assert torch.equal(want, paged_flash_attention_prefix(q, k, v, pre, 20, table, wide((1 << 31) + 4, (1 << 63) - 1)))
    want = paged_flash_attention_prefix(q, k, v, pre, 20, table, lens * 0)
    assert torch.equal(want, paged_flash_attention_prefix(q, k, v, pre, 20, table, wide(-(1 << 63), 9 - (1 << 32))))
    # entries outside the pool read the nearest page
    near, far = table.clone(), table.long()
    near[0, 0], near[1, 0] = 5, 0
    far[0, 0], far[1, 0] = (1 << 32) + 1, -(1 << 63)
    assert torch.equal(paged_flash_attention_prefix(q, k, v, pre, 20, near, lens),
                       paged_flash_attention_prefix(q, k, v, pre, 20, far, lens.long()))
    assert torch.equal(paged_flash_attention_prefix(q, k, v, wide(0, 5).int(), 20, table, lens),
                       paged_flash_attention_prefix(q, k, v, wide(0, (1 << 32) + 2), 20, table, lens))


@pytest.mark.gpu
def test_append_of_wide_integers():
    rng = np.random.default_rng(0)
    x = torch.as_tensor(rng.standard_normal((2, 8, 3, 64))).float().cuda()
    q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
    cos, sin = precompute_rope(64, 64, 10000.0, device="cuda")
    ints = lambda *x: torch.tensor(x, dtype=torch.int64)  # noqa: E731

    def write(table, position, lens=None):
        kp, vp = (torch.full((6, 2, 16, 64), 7.0, device="cuda") for _ in range(2))
        out, _, _ = write_to_paged_cache_rope(kp, vp, q, k, v, table, position, cos, sin, seq_lens=lens)
        return out, kp, vp

    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))  # noqa: E731
    table = ints(2, 3, 4, 5).view(2, 2)
    want = write(table, ints(5, 0))
    # no row of the first sequence is padding, every one of the second is
    assert same(write(table, ints(5, 0), ints(3, 0)), write(table, ints(5, 0), ints((1 << 63) - 1, 2 - (1 << 32))))
    # pages outside the pool are not written; the other sequence's are
    for entry in ((1 << 32) + 1, -(1 << 63), (1 << 31)):
        bad = table.clone()
        bad[0, 0] = entry
        got = write(bad, ints(5, 0))
        assert torch.equal(got[0], want[0]) and (got[1][:4] == 7).all() and (got[2][:4] == 7).all()
        assert torch.equal(got[1][4:], want[1][4:]) and torch.equal(got[2][4:], want[2][4:])
        assert same(got, write(bad.cuda(), ints(5, 0).cuda()))
    # positions outside the tables: no write, q zero
    for at in ((1 << 32) + 5, 1 << 40, -(1 << 63), 5 - (1 << 32)):
        got = write(table, ints(at, 0))
        assert (got[0][0] == 0).all() and (got[1][:4] == 7).all() and (got[2][:4] == 7).all()
        assert torch.equal(got[0][1], want[0][1]) and torch.equal(got[1][4:], want[1][4:])
        got = write(table, at)
        assert (got[0] == 0).all() and (got[1] == 7).all() and (got[2] == 7).all()
