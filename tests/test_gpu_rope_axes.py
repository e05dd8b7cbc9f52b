"""GPU tier: multi-axis rotary positions and the rotating paged write against float64."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from gpu_util import TORCH_DT, dev, host, note
from pallas_flash import (apply_rope, apply_rope_axes, flash_attention, precompute_rope, write_to_paged_cache,
                          write_to_paged_cache_rope)
from pallas_flash.fused_rope import _rope
from rope_axes_ref import rotate, tolerance, write

pytestmark = pytest.mark.gpu
EPS = {k: torch.finfo(v).eps for k, v in TORCH_DT.items()}


def tables(rows, d, seed=5):
    """Tables whose halves differ, as no frequency table's do: the rotation reads all four values of a pair."""
    rng = np.random.default_rng(seed)
    return (torch.as_tensor(rng.uniform(-1, 1, (rows, d))).float().cuda() for _ in range(2))


def close(got, want, bound, dt, name=""):
    got = host(got)
    assert np.isfinite(got).all(), name
    off = np.abs(got - want) - tolerance(want, bound, EPS[dt])
    assert off.max() <= 0, f"{name}: {off.max():.3e} past the tolerance"


def projected(rng, b, s, heads, d, dt, strided):
    x = dev(rng.standard_normal((b, s, heads, d) if strided else (b, heads, s, d)), dt)
    return x.transpose(1, 2) if strided else x


CASES = [  # b, hq, hk, s, d, sections
    (1, 1, 1, 1, 2, (1,)),
    (2, 4, 2, 1, 128, (16, 24, 24)),
    (1, 32, 8, 1, 128, (64,)),
    (3, 5, 1, 37, 64, (8, 12, 12)),
    (2, 7, 7, 130, 80, (10, 15, 15)),
    (1, 8, 2, 300, 256, (3, 100, 20, 5)),
    (2, 3, 1, 19, 72, (1, 1, 33, 1)),
    (2, 2, 2, 41, 6, (1, 2)),
    (1, 9, 3, 2049, 96, (24, 24)),
    (5, 16, 4, 257, 128, (32, 32)),
]


@pytest.mark.parametrize("strided", [True, False])
@pytest.mark.parametrize("pos_dt", [torch.int32, torch.int64])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("b,hq,hk,s,d,sections", CASES)
def test_rotation(b, hq, hk, s, d, sections, dt, pos_dt, strided):
    note(f"rope axes {dt} {b} {hq}/{hk} S={s} D={d} {sections}")
    rng = np.random.default_rng(s)
    q, k = projected(rng, b, s, hq, d, dt, strided), projected(rng, b, s, hk, d, dt, strided)
    rows = 50
    cos, sin = tables(rows, d)
    pos = rng.integers(0, rows, (len(sections), b, s))
    qr, kr = apply_rope_axes(q, k, torch.as_tensor(pos).to("cuda", pos_dt), cos, sin, sections)
    assert qr.shape == q.shape and qr.is_contiguous() and qr.dtype == q.dtype and kr.is_contiguous()
    for x, y in ((q, qr), (k, kr)):
        close(y, *rotate(host(x), pos, host(cos), host(sin), sections), dt)


def test_positions_forms():
    """[seq], [batch, seq], [axes, seq], expanded and strided tensors, other integer types, lists."""
    rng = np.random.default_rng(1)
    q = dev(rng.standard_normal((2, 3, 5, 64)), "f32")
    cos, sin = tables(9, 64)
    one = torch.tensor([3, 8, 0, 1, 1])
    per = torch.tensor([[3, 8, 0, 1, 1], [2, 2, 7, 4, 5]])
    want = [rotate(host(q), p.numpy(), host(cos), host(sin), (32,))[0] for p in (one.expand(1, 2, 5), per[None])]
    wide = torch.zeros(2, 10, dtype=torch.int64, device="cuda")
    wide[:, ::2] = per.cuda()
    for form, w in ((one.cuda(), want[0]), (one, want[0]), (one.tolist(), want[0]), (one[None].cuda(), want[0]),
                    (one.to(torch.int16).cuda(), want[0]), (per.cuda(), want[1]), (per[None].cuda(), want[1]),
                    (wide[:, ::2], want[1]), (one.cuda()[None].expand(2, 5), want[0])):
        qr, none = apply_rope_axes(q, None, form, cos, sin)
        assert none is None
        close(qr, w, 1e-6, "f32")
    two = torch.stack([one, per[1]])
    qr, _ = apply_rope_axes(q, None, two.cuda(), cos, sin, (20, 12))
    close(qr, *rotate(host(q), two[:, None].expand(2, 2, 5).numpy(), host(cos), host(sin), (20, 12)), "f32")


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_one_axis_is_rope(dt):
    """At positions 0 .. S - 1 what pf_rope gives. Not to the bit: which of a pair's two products is fused
    into the sum is each kernel's own, so both are held to the bound of either order against float64."""
    rng = np.random.default_rng(2)
    q, k = dev(rng.standard_normal((2, 4, 100, 128)), dt), dev(rng.standard_normal((2, 2, 100, 128)), dt)
    cos, sin = precompute_rope(100, 128, 10000.0, device="cuda")
    qr, kr = apply_rope_axes(q, k, torch.arange(100, device="cuda"), cos, sin)
    at = np.broadcast_to(np.arange(100), (1, 2, 100))
    for x, y in ((q, qr), (k, kr)):
        want = rotate(host(x), at, host(cos), host(sin), (64,))
        close(y, *want, dt)
        close(_rope(x, cos, sin, False), *want, dt)
    if dt == "f32":
        assert torch.allclose(qr, apply_rope(q, cos, sin), atol=1e-5)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_positions_outside_the_tables(dt):
    rng = np.random.default_rng(3)
    q, k = projected(rng, 2, 8, 4, 64, dt, True), projected(rng, 2, 8, 1, 64, dt, True)
    cos, sin = tables(20, 64)
    pos = rng.integers(0, 20, (2, 2, 8))
    pos[0, 0, 1], pos[1, 1, 2], pos[1, 0, 7], pos[0, 1, 0] = -1, 20, 1 << 40, -(1 << 33)
    q.requires_grad_(), k.requires_grad_()
    qr, kr = apply_rope_axes(q, k, torch.as_tensor(pos).cuda(), cos, sin, (16, 16))
    for x, y in ((q, qr), (k, kr)):
        close(y, *rotate(host(x), pos, host(cos), host(sin), (16, 16)), dt)
    dq, dk = torch.autograd.grad(qr.float().sum() + kr.float().sum(), (q, k))
    for g in (dq, dk):
        for b, s in ((0, 1), (1, 2), (0, 7), (1, 0)):
            assert (g[b, :, s] == 0).all()


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("b,hq,hk,s,d,sections", CASES[1:])
def test_gradient(b, hq, hk, s, d, sections, dt):
    rng = np.random.default_rng(s + 1)
    q, k = (projected(rng, b, s, h, d, dt, True).requires_grad_() for h in (hq, hk))
    cos, sin = tables(60, d)
    pos = rng.integers(0, 60, (len(sections), b, s))
    gq, gk = dev(rng.standard_normal(q.shape), dt), projected(rng, b, s, hk, d, dt, True)
    out = apply_rope_axes(q, k, torch.as_tensor(pos).cuda(), cos, sin, sections)
    dq, dk = torch.autograd.grad(out, (q, k), (gq, gk))
    for g, got in ((gq, dq), (gk, dk)):
        close(got, *rotate(host(g), pos, host(cos), host(sin), sections, inverse=True), dt)


def test_gradient_against_differences():
    """The rotation is linear: <g, R(x + u) - R(x)> = <R^T g, u> for any u, to float32's rounding."""
    rng = np.random.default_rng(4)
    q, u, g = (dev(rng.standard_normal((1, 2, 9, 64)), "f32") for _ in range(3))
    cos, sin = tables(30, 64)
    pos = torch.as_tensor(rng.integers(0, 30, (3, 1, 9))).cuda()
    turn = lambda x: apply_rope_axes(x, None, pos, cos, sin, (8, 12, 12))[0]  # noqa: E731
    leaf = q.clone().requires_grad_()
    (dq,) = torch.autograd.grad(turn(leaf), leaf, g)
    diff = (host(g) * (host(turn(q + u)) - host(turn(q)))).sum()
    # n terms, each off by a few roundings of values of up to about 10
    assert abs(diff - (host(dq) * host(u)).sum()) < q.numel() * 10 * 4 * 2.0 ** -24


def test_gradient_of_one_input_of_sums_and_twice():
    rng = np.random.default_rng(5)
    q, k = (dev(rng.standard_normal((2, 2, 7, 64)), "f32").requires_grad_() for _ in range(2))
    cos, sin = tables(30, 64)
    pos = rng.integers(0, 30, (1, 2, 7))
    tp = torch.as_tensor(pos[0]).cuda()
    back = lambda g: rotate(g, pos, host(cos), host(sin), (32,), inverse=True)  # noqa: E731
    ones = np.ones(q.shape)
    qr, kr = apply_rope_axes(q, k, tp, cos, sin)
    (dk,) = torch.autograd.grad(kr.sum(), k)  # an expanded gradient, and none for q
    close(dk, *back(ones), "f32")
    qr, kr = apply_rope_axes(q.detach(), k, tp, cos, sin)
    (dk,) = torch.autograd.grad(qr.sum() + 2 * kr.sum(), k)
    close(dk, *back(2 * ones), "f32")
    # q . R q: gradient R q + R^T q, and its own gradient through both
    qr, _ = apply_rope_axes(q, None, tp, cos, sin)
    (dq,) = torch.autograd.grad((q * qr).sum(), q, create_graph=True)
    want = rotate(host(q), pos, host(cos), host(sin), (32,))[0] + back(host(q))[0]
    close(dq, want, 1e-5, "f32")
    (ddq,) = torch.autograd.grad(dq.sum(), q)
    want = rotate(ones, pos, host(cos), host(sin), (32,))[0] + back(ones)[0]
    close(ddq, want, 1e-5, "f32")


def test_through_attention():
    """q and k of a projection, rotated, attended: gradients reach the projection as through the plain rotation."""
    rng = np.random.default_rng(6)
    b, s, hq, hk, d = 1, 130, 4, 2, 64
    x = dev(rng.standard_normal((b, s, (hq + 2 * hk) * d)), "f32")
    cos, sin = precompute_rope(s, d, 10000.0, device="cuda")
    g = dev(rng.standard_normal((b, hq, s, d)), "f32")

    def step(turn):
        leaf = x.clone().requires_grad_()
        h = leaf.view(b, s, hq + 2 * hk, d).transpose(1, 2)
        q, k = turn(h[:, :hq], h[:, hq:hq + hk])
        o = flash_attention(q, k, h[:, hq + hk:], causal=True)
        return o.detach(), torch.autograd.grad(o, leaf, g)[0]

    at = torch.arange(s, device="cuda")
    got = step(lambda q, k: apply_rope_axes(q, k, at, cos, sin))
    want = step(lambda q, k: (apply_rope(q, cos, sin), apply_rope(k, cos, sin)))
    for a, c in zip(got, want):
        # both in float32: the rotations differ in the order of one rounding
        assert (a - c).abs().max() <= 2e-5 * c.abs().max()


def test_streams_and_graph():
    rng = np.random.default_rng(7)
    q, k = projected(rng, 2, 33, 4, 128, "bf16", True), projected(rng, 2, 33, 2, 128, "bf16", True)
    cos, sin = precompute_rope(200, 128, 10000.0, device="cuda")
    pos = torch.as_tensor(rng.integers(0, 200, (3, 2, 33))).cuda()
    call = lambda: apply_rope_axes(q, k, pos, cos, sin, (16, 24, 24))  # noqa: E731
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for shift in (0, 3, 50):
        pos.copy_((pos + shift) % 200)
        want = call()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_empty():
    cos, sin = precompute_rope(4, 64, 10000.0, device="cuda")
    q = torch.zeros(2, 4, 0, 64, device="cuda")
    qr, kr = apply_rope_axes(q, q, torch.zeros(1, 0, dtype=torch.int64), cos, sin)
    assert qr.shape == kr.shape == q.shape
    q = torch.zeros(0, 4, 3, 64, device="cuda")
    qr, _ = apply_rope_axes(q, None, torch.zeros(3, dtype=torch.int64), cos, sin)
    assert qr.shape == q.shape


# ---------------------------------------------------------------------------
# the rotating paged write
# ---------------------------------------------------------------------------
WRITES = [  # b, hq, hk, L, d, page, sections, padded
    (1, 2, 2, 1, 64, 16, (32,), False),
    (5, 8, 2, 1, 128, 64, (64,), False),
    (3, 4, 1, 50, 128, 16, (16, 24, 24), True),
    (4, 7, 1, 33, 96, 5, (48,), True),
    (2, 6, 3, 20, 80, 1, (20, 20), True),
    (3, 2, 2, 129, 256, 32, (128,), True),
    (2, 2, 1, 11, 10, 4, (3, 2), True),
]


def append_inputs(b, hq, hk, L, d, page, sections, padded, dt, seed=0):
    rng = np.random.default_rng(seed + L)
    per = (40 + L) // page + 2
    pool = b * per + 3
    x = dev(rng.standard_normal((b, L, (hq + 2 * hk), d)), dt).transpose(1, 2)
    kp, vp = (dev(rng.standard_normal((pool, hk, page, d)), dt) for _ in range(2))
    table = rng.permutation(pool)[:b * per].reshape(b, per).astype(np.int32)
    own = rng.integers(0, 40, b)
    lens = rng.integers(0, L + 1, b) if padded else None
    rope = None if len(sections) == 1 and b % 2 else rng.integers(0, 90, (len(sections), b, L))
    cos, sin = tables(200, d)
    return x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:], kp, vp, table, own, lens, rope, cos, sin


def check_append(args, sections, dt):
    q, k, v, kp, vp, table, own, lens, rope, cos, sin = args
    L = q.shape[2]
    at = own[:, None] + np.arange(L)
    rpos = at[None] if rope is None else rope
    live = np.ones(at.shape, bool) if lens is None else np.arange(L) < lens[:, None]
    bad = ((rpos < 0) | (rpos >= cos.shape[0])).any(0)
    live &= ~bad
    before = [kp.clone(), vp.clone()]
    t = lambda a, dtype=torch.int32: None if a is None else torch.as_tensor(a).to("cuda", dtype)  # noqa: E731
    qr, ko, vo = write_to_paged_cache_rope(kp, vp, q, k, v, t(table), t(own), cos, sin,
                                           rope_positions=t(rope, torch.int64), sections=sections, seq_lens=t(lens))
    assert ko is kp and vo is vp and qr.is_contiguous() and qr.shape == q.shape
    wq, bq = rotate(host(q), rpos, host(cos), host(sin), sections)
    keep = live[:, None, :, None]
    close(qr, wq * keep, bq * keep, dt, "q")
    wk, bk = rotate(host(k), rpos, host(cos), host(sin), sections)
    close(kp, write(host(before[0]), wk, table, at, live), write(0 * host(kp), bk, table, at, live), dt, "k")
    assert np.array_equal(host(vp), write(host(before[1]), host(v), table, at, live))
    # what is not written keeps its bits
    mark = write(np.zeros(host(kp).shape, np.int64), np.ones(host(k).shape, np.int64), table, at, live) == 0
    mark = torch.as_tensor(mark).cuda()
    assert torch.equal(kp[mark], before[0][mark])


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("b,hq,hk,L,d,page,sections,padded", WRITES)
def test_append(b, hq, hk, L, d, page, sections, padded, dt):
    note(f"append {dt} {b} {hq}/{hk} L={L} D={d} page={page} {sections}")
    check_append(append_inputs(b, hq, hk, L, d, page, sections, padded, dt), sections, dt)


@pytest.mark.parametrize("dt", ["bf16"])
def test_append_rows_without_a_page(dt):
    """-1 entries, entries past the pool, positions before and past the table: not written; q still rotated."""
    args = list(append_inputs(4, 4, 2, 30, 64, 8, (16, 16), False, dt))
    args[5][0, 2], args[5][1, 1] = -1, args[3].shape[0]
    args[6] = np.array([0, 4, -3, 8 * args[5].shape[1] - 5])
    check_append(tuple(args), (16, 16), dt)


def test_append_rope_positions_outside_the_tables():
    args = list(append_inputs(2, 4, 2, 9, 64, 8, (16, 16), False, "f32"))
    args[8][0, 0, 3], args[8][1, 1, 4], args[8][1, 1, 0] = -1, 200, 200
    check_append(tuple(args), (16, 16), "f32")
    # without rotary positions of their own the rows' positions are looked up
    args = list(append_inputs(3, 4, 2, 9, 64, 8, (32,), False, "f32"))
    args[6] = np.array([3, -2, 1])
    args[9], args[10] = args[9][:8].contiguous(), args[10][:8].contiguous()
    check_append(tuple(args), (32,), "f32")


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_append_is_rotation_and_write(dt):
    """The same bits as apply_rope_axes followed by write_to_paged_cache; an int and a one-entry position."""
    q, k, v, kp, vp, table, own, _, _, cos, sin = append_inputs(3, 8, 2, 21, 128, 16, (64,), False, dt)
    table = torch.as_tensor(table).cuda()
    for position in (7, torch.tensor(7), torch.tensor([7], device="cuda", dtype=torch.int32)):
        k1, v1 = kp.clone(), vp.clone()
        q1, _, _ = write_to_paged_cache_rope(k1, v1, q, k, v, table, position, cos, sin)
        qr, kr = apply_rope_axes(q, k, torch.arange(7, 28, device="cuda"), cos, sin)
        k2, v2 = write_to_paged_cache(kp.clone(), vp.clone(), kr, v, table, 7)
        assert torch.equal(q1, qr) and torch.equal(k1, k2) and torch.equal(v1, v2)


def test_append_captured():
    """One captured step, replayed while the positions move on."""
    q, k, v, kp, vp, table, own, _, _, cos, sin = append_inputs(3, 8, 2, 1, 128, 16, (64,), False, "bf16")
    table, pos = torch.as_tensor(table).cuda(), torch.as_tensor(own).to("cuda", torch.int32)
    graph = torch.cuda.CUDAGraph()
    k1, v1 = kp.clone(), vp.clone()
    write_to_paged_cache_rope(k1, v1, q, k, v, table, pos, cos, sin)
    k1.copy_(kp), v1.copy_(vp)
    with torch.cuda.graph(graph):
        q1, _, _ = write_to_paged_cache_rope(k1, v1, q, k, v, table, pos, cos, sin)
    for _ in range(4):
        q2, _, _ = write_to_paged_cache_rope(kp, vp, q, k, v, table, pos, cos, sin)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(q1, q2) and torch.equal(k1, kp) and torch.equal(v1, vp)
        pos += 1


def test_append_empty():
    q, k, v, kp, vp, table, own, _, _, cos, sin = append_inputs(2, 4, 2, 3, 64, 8, (32,), False, "f32")
    before = kp.clone()
    q1, _, _ = write_to_paged_cache_rope(kp, vp, q[:, :, :0], k[:, :, :0], v[:, :, :0], table, 0, cos, sin)
    assert q1.shape == (2, 4, 0, 64) and torch.equal(kp, before)


@pytest.mark.parametrize("dt,hq,hk,d", [("bf16", 15, 5, 128), ("f32", 6, 3, 64), ("f16", 7, 7, 256)])
def test_large_calls(dt, hq, hk, d):
    """Past 48 MB a thread takes four heads: the bits of the same call in short pieces, head counts that four does not divide."""
    s = 26000000 // ((hq + hk) * d * 2 * torch.finfo(TORCH_DT[dt]).bits // 8) + 7
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(2, s, hq + 2 * hk, d, device="cuda", generator=gen).to(TORCH_DT[dt]).transpose(1, 2)
    q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    cos, sin = tables(300, d)
    sections = (d // 8, d // 4, d // 8)
    pos = torch.randint(-1, 300, (3, 2, s), device="cuda", generator=gen)
    page, per = 64, -(-(s + 5) // 64)
    table = torch.randperm(2 * per, device="cuda", generator=gen).to(torch.int32).view(2, per)
    pools = [torch.zeros(2 * per, hk, page, d, device="cuda", dtype=x.dtype) for _ in range(4)]
    lens = torch.tensor([s - 11, 1500], device="cuda", dtype=torch.int32)
    qr, kr = apply_rope_axes(q, k, pos, cos, sin, sections)
    qa, _, _ = write_to_paged_cache_rope(*pools[:2], q, k, v, table, 5, cos, sin, rope_positions=pos,
                                         sections=sections, seq_lens=lens)
    for lo in range(0, s, 1000):
        at = slice(lo, lo + 1000)
        q1, k1 = apply_rope_axes(q[:, :, at], k[:, :, at], pos[:, :, at], cos, sin, sections)
        assert torch.equal(q1, qr[:, :, at]) and torch.equal(k1, kr[:, :, at])
        q1, _, _ = write_to_paged_cache_rope(*pools[2:], q[:, :, at], k[:, :, at], v[:, :, at], table, 5 + lo, cos,
                                             sin, rope_positions=pos[:, :, at], sections=sections, seq_lens=lens - lo)
        assert torch.equal(q1, qa[:, :, at])
    assert torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])
    keep = (pos >= 0).all(0)[:, None, :, None] & (torch.arange(s, device="cuda") < lens[:, None])[:, None, :, None]
    assert torch.equal(qa, torch.where(keep, qr, torch.zeros_like(qr))) and pools[0].any()


def test_rotation_past_32_bits():
    """Heads behind 2^32 bytes: the bits of the same heads alone, forward and backward, dense and strided."""
    b, h, s, d = 2, 20, 220000, 256
    cos, sin = tables(300, d)
    pos = torch.randint(0, 300, (2, b, s), device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    last = torch.randn(b, 1, s, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).half()
    for dims in ((b, h, s, d), (b, s, h, d)):
        x = torch.zeros(dims, dtype=torch.float16, device="cuda")
        assert x.numel() > 1 << 31
        x = x if dims[1] == h else x.transpose(1, 2)
        x[:, -1:] = last
        out, _ = apply_rope_axes(x, None, pos, cos, sin, (50, 78))
        want, _ = apply_rope_axes(last, None, pos, cos, sin, (50, 78))
        assert torch.equal(out[:, -1:], want) and not out[:, :-1].any()
        y = last.clone().requires_grad_()
        want, = torch.autograd.grad(apply_rope_axes(y, None, pos, cos, sin, (50, 78))[0], y, last)
        del out
        z = torch.zeros_like(x).requires_grad_()
        got, = torch.autograd.grad(apply_rope_axes(z, None, pos, cos, sin, (50, 78))[0], z, x)
        assert torch.equal(got[:, -1:], want)
        del x, z, got
