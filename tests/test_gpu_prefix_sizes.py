"""GPU tier: the shared-prefix attention at the ends of its ranges, against float64."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from gpu_util import note
from pallas_flash import _lib, apply_rope_axes, paged_flash_attention_prefix, precompute_rope
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


@pytest.mark.parametrize("dt,batch,hq,hkv,d", [("bf16", 16, 32, 8, 128), ("f16", 3, 40, 2, 64), ("f32", 4, 8, 2, 64),
                                               ("f32", 200, 2, 1, 128), ("bf16", 8, 8, 4, 256)])
def test_device_length_far_below_its_table(dt, batch, hq, hkv, d):
    """Chunks go by the table's reach: a short prefix fills a few of them, the others' partials are not read."""
    note(f"prefix {dt} B={batch} {hq}/{hkv} D={d}, a table of 65536 tokens")
    q, k, v, ptab, prefix, table, lens = make(dt, batch, hq, hkv, d, 16, 1000, [(9 * i) % 50 for i in range(batch)])
    far = torch.full((4096,), -1, dtype=torch.int32, device="cuda")
    far[:ptab.shape[0]] = ptab
    for n in (1000, 0, 1, 15, 64, 385, 999):
        check((q, k, v, far, torch.tensor(n, dtype=torch.int32, device="cuda"), table, lens), dt)


@pytest.mark.parametrize("dt,hq,hkv,d", [
    ("bf16", 8, 2, 80), ("f16", 40, 2, 96), ("f32", 8, 2, 36), ("f32", 40, 2, 96), ("bf16", 8, 1, 256),
    ("f16", 20, 1, 200)])
@pytest.mark.parametrize("page", [18, 50])
def test_straddled_pages_at_the_end_of_4_gib(dt, hq, hkv, d, page):
    """The largest pool whose pages a lane picks by 32-bit offsets, its last pages live: the bits of a small pool's."""
    note(f"prefix {dt} {hq}/{hkv} D={d} page={page}, pools of 4 GiB")
    q, k, v, ptab, prefix, table, lens = make(dt, 4, hq, hkv, d, page, 333, [0, page, 200, 1])
    pages = 0xffffffe0 // (k[0].numel() * k.element_size())
    far = pages - k.shape[0]
    assert far > 0 and pages * k[0].numel() * k.element_size() > 0xffff0000 - k[0].numel() * k.element_size()
    kf, vf = (torch.empty(pages, *k.shape[1:], dtype=k.dtype, device="cuda") for _ in range(2))
    kf[far:], vf[far:] = k, v
    # half of them at the front, so that one stage's two pages lie 4 GiB apart
    front = k.shape[0] // 2
    kf[:front], vf[:front] = k[:front], v[:front]
    move = lambda t: torch.where((t < 0) | (t < front), t, t + far)  # noqa: E731
    near = check((q, k, v, ptab, prefix, table, lens), dt)
    assert torch.equal(near, paged_flash_attention_prefix(q, kf, vf, move(ptab), prefix, move(table), lens))
    assert torch.equal(near, paged_flash_attention_prefix(q, kf, vf, ptab + far, prefix,
                                                          torch.where(table < 0, table, table + far), lens))


@pytest.mark.parametrize("hq", [8, 48])
@pytest.mark.parametrize("prefix,hi", [(300, 900), (5000, 500), (9000, 700), (40000, 700), (40000, 3000), (0, 3000)])
@pytest.mark.parametrize("dt,d", [("f16", 256), ("f32", 128)])
def test_own_keys_over_few_workgroups(dt, d, prefix, hi, hq):
    """Rows of 512 bytes: the own keys have what the prefix leaves of the CUs, so that a wave or workgroup has many
    stages and sequences are cut wherever its share ends."""
    note(f"prefix {dt} {hq}/2 D={d} prefix={prefix} lens to {hi}")
    lens = np.random.default_rng(prefix + hi).integers(0, hi + 1, 7).tolist()
    lens[2], lens[4] = hi, 0
    check(make(dt, 7, hq, 2, d, 16, prefix, lens, poison=False), dt)


@pytest.mark.parametrize("dt,batch,hq,hkv,d,page", [("bf16", 24, 32, 8, 128, 16), ("f16", 5, 48, 2, 64, 50),
                                                    ("f32", 9, 8, 2, 64, 16), ("f32", 200, 2, 1, 128, 12)])
def test_repeats_itself(dt, batch, hq, hkv, d, page):
    """The same bits from call to call, on two streams at once too: nothing depends on the order of the workgroups."""
    note(f"prefix {dt} B={batch} {hq}/{hkv} D={d} page={page}, again and again")
    args = make(dt, batch, hq, hkv, d, page, 3000, [(37 * i) % 700 for i in range(batch)])
    want = check(args, dt)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        got = [paged_flash_attention_prefix(*args) for _ in range(3)]
        with torch.cuda.stream(side):
            got += [paged_flash_attention_prefix(*args) for _ in range(3)]
        torch.cuda.synchronize()
        assert all(torch.equal(x, want) for x in got)


@pytest.mark.parametrize("dt,hq", [("bf16", 8), ("f16", 40), ("f32", 8), ("f32", 40)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_live_keys_without_a_finite_score(dt, hq, bad):
    """A key of NaN or infinities, or a value of NaN, reaches the rows that attend it and no others."""
    args = q, k, v, ptab, prefix, table, lens = make(dt, 4, hq, 2, 64, 16, 200, [30, 0, 70, 5], poison=False)
    want = paged_flash_attention_prefix(*args)
    g = hq // 2
    for pool in (k, v) if math.isnan(bad) else (k,):
        keep = pool.clone()
        pool[ptab[3], 1, 5] = bad  # a prefix token of one KV head: its heads in every sequence
        got = paged_flash_attention_prefix(*args)
        assert torch.isnan(got[:, g:]).all() and torch.equal(got[:, :g], want[:, :g])
        pool.copy_(keep)
        pool[table[2, 4], 0, 3] = bad  # an own token of sequence 2
        got = paged_flash_attention_prefix(*args)
        assert torch.isnan(got[2, :g]).all() and torch.equal(got[2, g:], want[2, g:])
        assert torch.equal(got[[0, 1, 3]], want[[0, 1, 3]])
        pool.copy_(keep)


def test_result_has_no_graph():
    """Inference only, as the paged decode: in either path, whatever requires a gradient."""
    q, k, v, ptab, prefix, table, lens = make("f32", 2, 4, 2, 64, 16, 50, [3, 30])
    want = paged_flash_attention_prefix(q, k, v, ptab, prefix, table, lens)
    q, k, v = (x.requires_grad_() for x in (q, k, v))
    for t in (table, table.long()):
        out = paged_flash_attention_prefix(q, k, v, ptab, prefix, t, lens)
        assert not out.requires_grad and torch.equal(out, want)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("seq", [5, 6000])
def test_rotation_in_place_through_the_c_entry(dt, seq):
    """pf_rope_axes with q_out and k_out the inputs themselves: a head a thread, and four with non-temporal accesses."""
    gen = torch.Generator("cuda").manual_seed(0)
    q, k = (torch.randn(2, h, seq, 128, device="cuda", generator=gen).to(dt) for h in (14, 3))
    cos, sin = precompute_rope(300, 128, 10000.0, device="cuda")
    pos = torch.randint(-1, 301, (3, 2, seq), device="cuda", generator=gen)
    sections = (16, 24, 24)
    want = apply_rope_axes(q, k, pos, cos, sin, sections)
    stride = lambda t: (_lib.c_i64 * 3)(*t.stride()[:3])  # noqa: E731
    args = _lib.RopeAxesArgs(_lib.ptr(q), _lib.ptr(k), _lib.ptr(q), _lib.ptr(k), stride(q), stride(k), _lib.ptr(pos),
                             stride(pos), 1, 3, (_lib.c_i32 * 4)(*sections), _lib.ptr(cos), _lib.ptr(sin), 300, 2, 14,
                             3, seq, 128, 0, _lib.dtype_tag(q))
    assert _lib.lib().pf_rope_axes(args, _lib.stream_of(q)) == _lib.PF_OK
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_no_prefix_and_no_sequences_as_lists():
    q, k, v, _, _, table, lens = make("f32", 2, 4, 2, 64, 16, 0, [3, 30])
    want = check((q, k, v, table[0, :0], 0, table, lens), "f32")
    assert torch.equal(want, paged_flash_attention_prefix(q, k, v, [], 0, table, lens))
    pre = table[0, :1]
    want = check((q, k, v, pre, 3, table[:, :0], lens * 0), "f32")
    assert torch.equal(want, paged_flash_attention_prefix(q, k, v, pre, 3, [[], []], lens * 0))
    assert paged_flash_attention_prefix(q[:0], k, v, pre, 3, table[:0], []).shape == (0, 4, 1, 64)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_rotation_with_its_gradient_captured(dt):
    """Forward and backward in one graph, replayed with new positions, inputs and gradients between eager steps."""
    gen = torch.Generator("cuda").manual_seed(3)
    new = lambda h: torch.randn(2, 33, h, 64, device="cuda", generator=gen).to(dt).transpose(1, 2)  # noqa: E731
    cos, sin = precompute_rope(200, 64, 10000.0, device="cuda")
    pos = torch.zeros(3, 2, 33, dtype=torch.int64, device="cuda")
    x, y, gx, gy = new(6), new(2), new(6), new(2)

    def step():
        q, k = (t.detach().requires_grad_() for t in (x, y))
        out = apply_rope_axes(q, k, pos, cos, sin, (8, 12, 12))
        return [*(t.detach() for t in out), *torch.autograd.grad(out, (q, k), (gx, gy))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(4):
        pos.random_(-1, 201, generator=gen)
        for t in (x, y, gx, gy):
            t.copy_(new(t.shape[1]))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
