"""CPU tier: what the shared-prefix attention refuses, before any device work, and its workspace."""

from __future__ import annotations

import pytest
import torch

from pallas_flash import _lib, paged_flash_attention_prefix


def z(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def call(**over):
    a = dict(q=z(2, 4, 1, 64), k_pages=z(6, 2, 8, 64), v_pages=z(6, 2, 8, 64), prefix_table=ints(3), prefix_len=20,
             block_tables=ints(2, 2), context_lens=ints(2))
    a.update(over)
    return paged_flash_attention_prefix(**a)


@pytest.mark.parametrize("over", [
    dict(q=z(2, 4, 64)), dict(q=z(2, 4, 2, 64)), dict(q=z(2, 3, 1, 64)), dict(q=z(2, 0, 1, 64)), dict(q=z(2, 4, 1, 32)),
    dict(k_pages=z(6, 2, 8)), dict(v_pages=z(6, 2, 4, 64)), dict(k_pages=z(0, 2, 8, 64), v_pages=z(0, 2, 8, 64)),
    dict(k_pages=z(6, 0, 8, 64), v_pages=z(6, 0, 8, 64)), dict(prefix_table=ints(1, 3)), dict(prefix_table=z(3)),
    dict(prefix_len=-1), dict(prefix_len=25), dict(block_tables=ints(2)), dict(block_tables=ints(3, 2)),
    dict(block_tables=z(2, 2)), dict(context_lens=ints(3)), dict(context_lens=ints(2, 1)), dict(context_lens=z(2)),
])
def test_refuses(over):
    with pytest.raises(ValueError):
        call(**over)


def test_prefix_len_is_an_integer_and_cpu_tensors_are_refused():
    with pytest.raises(TypeError):
        call(prefix_len=3.5)
    for n in (0, 24, torch.tensor(7)):
        with pytest.raises(RuntimeError, match="ROCm device"):
            call(prefix_len=n)


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def args(**over):
    a = dict(q=256, k_pages=256, v_pages=256, prefix_table=256, block_tables=256, context_lens=256, o=256, batch=4,
             num_heads=8, num_kv_heads=2, num_pages=50, page_size=16, head_dim=128, prefix_pages=20, prefix_len=300,
             pages_per_seq=5, sm_scale=0.1, dtype=1, workspace=256, workspace_bytes=1 << 40)
    a.update(over)
    return _lib.PagedPrefixArgs(**a)


@pytest.mark.parametrize("over,status", [
    (dict(batch=-1), _lib.PF_ERR_INVALID), (dict(num_heads=0), _lib.PF_ERR_INVALID),
    (dict(num_kv_heads=3), _lib.PF_ERR_INVALID), (dict(num_kv_heads=0), _lib.PF_ERR_INVALID),
    (dict(num_pages=0), _lib.PF_ERR_INVALID), (dict(page_size=0), _lib.PF_ERR_INVALID),
    (dict(pages_per_seq=-1), _lib.PF_ERR_INVALID), (dict(prefix_pages=-1), _lib.PF_ERR_INVALID),
    (dict(prefix_len=-1), _lib.PF_ERR_INVALID), (dict(prefix_len=321), _lib.PF_ERR_INVALID),
    (dict(sm_scale=float("nan")), _lib.PF_ERR_INVALID), (dict(dtype=5), _lib.PF_ERR_UNSUPPORTED),
    (dict(head_dim=130), _lib.PF_ERR_UNSUPPORTED), (dict(head_dim=264), _lib.PF_ERR_UNSUPPORTED),
    (dict(head_dim=256, dtype=0), _lib.PF_ERR_UNSUPPORTED),
])
def test_c_refuses(L, over, status):
    assert L.pf_paged_prefix_attn(args(**over), None) == status
    assert L.pf_paged_prefix_attn_workspace_size(args(**over)) == 0


@pytest.mark.parametrize("missing", ["q", "k_pages", "v_pages", "o", "context_lens", "block_tables", "prefix_table"])
def test_c_needs_its_buffers(L, missing):
    assert L.pf_paged_prefix_attn(args(**{missing: None}), None) == _lib.PF_ERR_INVALID


def test_c_workspace(L):
    need = L.pf_paged_prefix_attn_workspace_size(args())
    assert need > 0 and need % 256 == 0
    for over in (dict(workspace=None), dict(workspace=264), dict(workspace_bytes=need - 1)):
        assert L.pf_paged_prefix_attn(args(**over), None) == _lib.PF_ERR_WORKSPACE
    assert L.pf_paged_prefix_attn(args(batch=0), None) == _lib.PF_OK
    assert L.pf_paged_prefix_attn(None, None) == _lib.PF_ERR_INVALID


@pytest.mark.parametrize("dtype,d", [(0, 64), (0, 128), (1, 64), (1, 128), (2, 256), (1, 96)])
def test_c_workspace_is_bounded(L, dtype, d):
    """What the partials take: in proportion to the queries, not to the prefix."""
    for batch in (1, 7, 128, 1000):
        for hq, hkv in ((1, 1), (32, 8), (64, 1)):
            for prefix in (64, 6000, 1 << 20):
                a = args(batch=batch, num_heads=hq, num_kv_heads=hkv, head_dim=d, dtype=dtype, prefix_len=prefix,
                         prefix_pages=-(-prefix // 16), num_pages=1 << 17, pages_per_seq=64)
                need = L.pf_paged_prefix_attn_workspace_size(a)
                assert 0 < need <= (1 << 28) + batch * hq * 64 * (d + 64) * 4, (batch, hq, prefix, need)


@pytest.mark.parametrize("dtype,d,page", [(0, 64, 16), (0, 128, 20), (1, 128, 16), (2, 256, 50), (1, 96, 12)])
@pytest.mark.parametrize("batch,hq,hkv", [(1, 8, 1), (16, 16, 4), (40, 64, 4), (9, 34, 2)])
def test_c_workspace_wherever_the_operands_lie(L, dtype, d, page, batch, hq, hkv):
    a = dict(batch=batch, num_heads=hq, num_kv_heads=hkv, head_dim=d, dtype=dtype, page_size=page, prefix_len=5000,
             prefix_pages=-(-5000 // page), num_pages=4000, pages_per_seq=30)
    need = L.pf_paged_prefix_attn_workspace_size(args(**a))
    for over in (dict(q=264), dict(k_pages=264), dict(v_pages=258), dict(q=None, k_pages=None, v_pages=None)):
        assert L.pf_paged_prefix_attn_workspace_size(args(**a, **over)) == need > 0
