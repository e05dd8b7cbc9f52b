"""CPU tier: what the multi-axis rotation and the rotating paged write refuse, before any device work."""

from __future__ import annotations

import pytest
import torch

from pallas_flash import _lib, apply_rope_axes, write_to_paged_cache_rope


def z(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def pos(*shape):
    return torch.zeros(shape, dtype=torch.int64)


COS = z(10, 64)


@pytest.mark.parametrize("q,k,positions,cos,sections", [
    (z(4, 8, 64), z(1, 4, 8, 64), pos(8), COS, None),              # rank
    (z(1, 4, 8, 64), z(1, 4, 9, 64), pos(8), COS, None),           # seq
    (z(1, 4, 8, 64), z(2, 4, 8, 64), pos(8), COS, None),           # batch
    (z(1, 4, 8, 64), z(1, 4, 8, 32), pos(8), COS, None),           # head_dim
    (z(1, 4, 8, 64), z(1, 0, 8, 64), pos(8), COS, None),           # no heads
    (z(1, 4, 8, 64), z(1, 4, 8, 64, dtype=torch.float16), pos(8), COS, None),
    (z(1, 4, 8, 63), None, pos(8), z(10, 63), None),               # odd head_dim
    (z(1, 4, 8, 64), None, pos(8), z(10, 32), None),               # tables
    (z(1, 4, 8, 64), None, pos(8), z(0, 64), None),
    (z(1, 4, 8, 64), None, pos(7), COS, None),                     # positions
    (z(1, 4, 8, 64), None, pos(3, 1, 8), COS, None),
    (z(2, 4, 8, 64), None, pos(3, 8), COS, None),
    (z(2, 4, 8, 64), None, pos(2, 3, 8), COS, (16, 16)),
    (z(2, 4, 8, 64), None, pos(8), COS, (16, 16)),
    (z(1, 4, 8, 64), None, z(8), COS, None),
    (z(1, 4, 8, 64), None, pos(8).bool(), COS, None),
    (z(1, 4, 8, 64), None, pos(2, 8), COS, (16, 15)),              # sections
    (z(1, 4, 8, 64), None, pos(2, 8), COS, (0, 32)),
    (z(1, 4, 8, 64), None, pos(2, 8), COS, (33, -1)),
    (z(1, 4, 8, 64), None, pos(5, 8), COS, (16, 4, 4, 4, 4)),
    (z(1, 4, 8, 64), None, pos(0, 8), COS, ()),
])
def test_rotation_refuses(q, k, positions, cos, sections):
    with pytest.raises(ValueError):
        apply_rope_axes(q, k, positions, cos, cos, sections)


def test_cpu_tensors_refused():
    with pytest.raises(RuntimeError, match="ROCm device"):
        apply_rope_axes(z(1, 4, 8, 64), z(1, 2, 8, 64), pos(3, 8), COS, COS, (8, 12, 12))
    with pytest.raises(RuntimeError, match="ROCm device"):
        write_to_paged_cache_rope(z(4, 2, 8, 64), z(4, 2, 8, 64), z(1, 4, 3, 64), z(1, 2, 3, 64), z(1, 2, 3, 64),
                                  pos(2), 0, COS, COS)


def append(**over):
    a = dict(k_pages=z(4, 2, 8, 64), v_pages=z(4, 2, 8, 64), q=z(2, 4, 3, 64), k=z(2, 2, 3, 64), v=z(2, 2, 3, 64),
             block_table=pos(2, 2), position=0, cos=COS, sin=COS)
    a.update(over)
    return write_to_paged_cache_rope(**a)


@pytest.mark.parametrize("over", [
    dict(k_pages=z(4, 2, 64)), dict(v_pages=z(4, 2, 8, 32)), dict(q=z(2, 4, 64)), dict(v=z(2, 2, 4, 64)),
    dict(k_pages=z(0, 2, 8, 64), v_pages=z(0, 2, 8, 64)), dict(k_pages=z(4, 1, 8, 64), v_pages=z(4, 1, 8, 64)),
    dict(q=z(2, 3, 3, 64)), dict(q=z(2, 0, 3, 64)), dict(q=z(1, 4, 3, 64)), dict(q=z(2, 4, 2, 64)),
    dict(q=z(2, 4, 3, 32)), dict(q=z(2, 4, 3, 64, dtype=torch.float16)), dict(v_pages=z(4, 2, 8, 64, dtype=torch.float16)),
    dict(block_table=pos(3, 2)), dict(block_table=pos(2)), dict(position=pos(3)), dict(position=0.5),
    dict(position=pos(2, 1)), dict(cos=z(10, 32)), dict(sin=z(9, 64)), dict(sections=(16, 16)),
    dict(sections=(16, 8)), dict(rope_positions=pos(2, 3), sections=(32,), q=z(1, 4, 3, 64)),
    dict(rope_positions=pos(3, 2, 3), sections=(16, 16)), dict(seq_lens=pos(3)), dict(seq_lens=z(2)),
])
def test_append_refuses(over):
    with pytest.raises(ValueError):
        append(**over)


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def axes_args(**over):
    a = dict(q=8, k=8, q_out=8, k_out=8, positions=8, axes=2, sections=(_lib.c_i32 * 4)(20, 12), cos=8, sin=8,
             rope_len=10, batch=1, num_heads=4, num_kv_heads=2, seq_len=3, head_dim=64, dtype=1)
    a.update(over)
    return _lib.RopeAxesArgs(**a)


def write_args(**over):
    a = dict(q=8, k=8, v=8, q_out=8, k_pages=8, v_pages=8, block_tables=8, positions=8, rope_positions=8, axes=2,
             sections=(_lib.c_i32 * 4)(20, 12), cos=8, sin=8, rope_len=10, batch=1, num_heads=4, num_kv_heads=2,
             seq_len=3, num_pages=2, page_size=4, head_dim=64, pages_per_seq=2, dtype=1)
    a.update(over)
    return _lib.RopePagedWriteArgs(**a)


BAD = [dict(axes=0), dict(axes=5), dict(sections=(_lib.c_i32 * 4)(20, 13)), dict(sections=(_lib.c_i32 * 4)(32, 0)),
       dict(sections=(_lib.c_i32 * 4)(2 ** 31 - 1, 2 ** 31 - 1)), dict(cos=None), dict(sin=None), dict(rope_len=0),
       dict(batch=-1), dict(seq_len=-1), dict(head_dim=63), dict(head_dim=0), dict(num_heads=0), dict(q=None),
       dict(q_out=None), dict(k=None)]


@pytest.mark.parametrize("over", BAD + [dict(positions_i64=2), dict(positions=None), dict(inverse=2),
                                        dict(num_kv_heads=-1), dict(k_out=None)])
def test_c_rotation_refuses(L, over):
    assert L.pf_rope_axes(axes_args(**over), None) == _lib.PF_ERR_INVALID


@pytest.mark.parametrize("over", BAD + [
    dict(rope_positions_i64=2), dict(rope_positions=None), dict(positions=None), dict(block_tables=None), dict(v=None),
    dict(k_pages=None), dict(v_pages=None), dict(num_kv_heads=0), dict(num_pages=0), dict(page_size=0),
    dict(pages_per_seq=-1), dict(positions_stride=2)])
def test_c_append_refuses(L, over):
    assert L.pf_rope_paged_cache_write(write_args(**over), None) == _lib.PF_ERR_INVALID


def test_c_dtypes_empty_and_null(L):
    assert L.pf_rope_axes(axes_args(dtype=3), None) == _lib.PF_ERR_UNSUPPORTED
    assert L.pf_rope_paged_cache_write(write_args(dtype=3), None) == _lib.PF_ERR_UNSUPPORTED
    assert L.pf_rope_axes(None, None) == _lib.PF_ERR_INVALID
    assert L.pf_rope_paged_cache_write(None, None) == _lib.PF_ERR_INVALID
    for empty in (dict(batch=0), dict(seq_len=0)):
        assert L.pf_rope_axes(axes_args(**empty), None) == _lib.PF_OK
        assert L.pf_rope_paged_cache_write(write_args(**empty), None) == _lib.PF_OK


@pytest.mark.parametrize("over", [dict(num_heads=65536), dict(num_heads=65532, num_kv_heads=4),
                                  dict(batch=1 << 26, seq_len=1)])
def test_c_sizes_past_the_grid_refused(L, over):
    assert L.pf_rope_axes(axes_args(**over), None) == _lib.PF_ERR_UNSUPPORTED
    assert L.pf_rope_paged_cache_write(write_args(**over), None) == _lib.PF_ERR_UNSUPPORTED
