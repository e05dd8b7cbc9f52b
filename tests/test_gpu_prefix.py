"""GPU tier: single-query attention over a shared prefix and the sequences' own pages, against float64."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from gpu_util import TORCH_DT, check_fwd, host, note
from pallas_flash import (_lib, apply_rope_axes, paged_flash_attention, paged_flash_attention_prefix, precompute_rope,
                          write_to_paged_cache_rope)

pytestmark = pytest.mark.gpu


def make(dt, batch, hq, hkv, d, page, prefix, lens, *, seed=0, extra=1, poison=True):
    """q, pools, prefix table, own table, lengths: scrambled pages, -1 behind the live ones, NaN in every slot no sequence has."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    pre, need = -(-prefix // page), [-(-n // page) for n in lens]
    per = max(need) + extra if need else extra
    pool = pre + sum(need) + 2
    ids = rng.permutation(pool)
    table = np.full((batch, per), -1)
    at = pre
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    q = torch.randn(batch, hq, 1, d, device="cuda", generator=gen).to(TORCH_DT[dt])
    k, v = (torch.randn(pool, hkv, page, d, device="cuda", generator=gen).to(TORCH_DT[dt]) for _ in range(2))
    if poison:
        live = np.zeros((pool, page), bool)
        for row, n in [(ids[:pre], prefix)] + list(zip(table, lens)):
            for i in range(-(-n // page)):
                live[row[i], :min(page, n - i * page)] = True
        dead = torch.as_tensor(~live).cuda()[:, None, :, None].expand_as(k)
        k[dead], v[dead] = math.nan, math.nan
    t = lambda a: torch.as_tensor(np.asarray(a), device="cuda", dtype=torch.int32)  # noqa: E731
    return q, k, v, t(ids[:pre]), prefix, t(table).view(batch, per), t(lens).view(batch)


def rows(pages, table, n):
    """[hkv, n, d] in float64: the first n tokens of a table."""
    page = pages.shape[2]
    x = pages[table[:-(-n // page)].long()].double()
    return x.transpose(0, 1).reshape(pages.shape[1], -1, pages.shape[3])[:, :n]


def reference(q, k, v, ptab, prefix, table, lens, scale=None):
    """(o, bound of the kernel's error before the output's rounding), float64. With e = 2^-24 and P the weights:
    a score is a sum of d products in at least 16-wide steps (float32: 2-wide), scaled, shifted and put through
    exp2 -- relative error of a weight at most 2 e ((d / w + 4) S + 8), S its largest sum of |q k| in log2 units;
    sums of n weights in steps of w add (n / w + 64) e to numerator and denominator; 16-bit weights are rounded,
    half a step each."""
    batch, hq, _, d = q.shape
    hkv, g = k.shape[1], hq // k.shape[1]
    scale = 1 / math.sqrt(d) if scale is None else scale
    e, w = 2.0 ** -24, 2 if q.dtype == torch.float32 else 16
    half = 0.0 if q.dtype == torch.float32 else torch.finfo(q.dtype).eps / 2
    out, bound = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64,
                                                                                       device="cuda")
    pk, pv = rows(k, ptab, prefix), rows(v, ptab, prefix)
    for b, n in enumerate(lens.tolist()):
        n = min(max(n, 0), table.shape[1] * k.shape[2])
        kk, vv = torch.cat([pk, rows(k, table[b], n)], 1), torch.cat([pv, rows(v, table[b], n)], 1)
        if kk.shape[1] == 0:
            continue
        qb = q[b].double().view(hkv, g, d)
        p = torch.softmax(torch.matmul(qb, kk.transpose(1, 2).contiguous()) * scale, -1)
        s_abs = torch.matmul(qb.abs(), kk.abs().transpose(1, 2).contiguous()).amax(-1, keepdim=True) * abs(scale) * 1.4427
        rel = 2 * (2 * e * ((d / w + 4) * s_abs + 8) + (kk.shape[1] / w + 64) * e) + half
        out[b] = torch.matmul(p, vv).view(hq, 1, d)
        bound[b] = (torch.matmul(p, vv.abs()) * rel).view(hq, 1, d)
    return out, bound


def check(args, dt, scale=None, **kw):
    out = paged_flash_attention_prefix(*args, **({} if scale is None else dict(sm_scale=scale)), **kw)
    q, k, v, ptab, prefix, table, lens = args
    if isinstance(prefix, torch.Tensor):
        prefix = min(max(int(prefix), 0), ptab.shape[0] * k.shape[2])
    want, bound = reference(q, k, v, ptab, prefix, table, lens, scale)
    assert out.shape == q.shape and out.dtype == q.dtype and torch.isfinite(out).all()
    eps = torch.finfo(q.dtype).eps
    tiny = 2.0 ** -25 if dt == "f16" else 0.0
    off = (out.double() - want).abs() - (bound + eps / 2 * (want.abs() + bound) + tiny)
    assert off.max() <= 0, f"{float(off.max()):.3e} past the bound"
    if scale is None:
        check_fwd(host(out), want.cpu().numpy(), dt)
    return out


CASES = [  # batch, hq, hkv, d, page, prefix, lens
    (1, 1, 1, 64, 8, 1, [0]),
    (1, 1, 1, 64, 8, 0, [1]),
    (2, 4, 2, 128, 64, 0, [0, 3]),
    (1, 8, 8, 128, 16, 65, [1]),
    (3, 4, 2, 128, 64, 100, [0, 5, 200]),
    (4, 32, 8, 128, 64, 500, [1, 64, 65, 30]),
    (3, 16, 1, 64, 16, 333, [17, 0, 90]),
    (40, 8, 1, 128, 16, 700, [(7 * i) % 50 for i in range(40)]),
    (33, 8, 2, 64, 32, 129, [i for i in range(33)]),
    (2, 20, 1, 128, 32, 260, [70, 33]),
    (2, 20, 1, 64, 32, 260, [70, 33]),
    (2, 7, 1, 128, 4, 400, [500, 900]),
    (5, 12, 4, 96, 16, 190, [3, 77, 0, 16, 300]),
    (5, 3, 3, 80, 100, 190, [3, 77, 0, 16, 300]),
    (2, 4, 2, 8, 24, 77, [3, 40]),
    (3, 4, 1, 128, 1, 70, [3, 0, 20]),
    (3, 4, 1, 64, 5, 70, [3, 0, 20]),
    (3, 6, 2, 128, 50, 1111, [49, 50, 51]),
    (2, 14, 2, 64, 12, 1000, [1000, 12]),
    (6, 16, 4, 64, 16, 2000, [0, 300, 1, 16, 15, 17]),
    (3, 8, 1, 128, 12, 90, [1, 40, 200]),
    (3, 16, 2, 64, 8, 90, [1, 40, 200]),
    (2, 14, 2, 64, 12, 90, [33, 40]),
    (2, 9, 1, 128, 16, 90, [33, 400]),
    (2, 260, 2, 64, 16, 90, [33, 400]),
    (70, 5, 5, 128, 20, 33, [i % 7 for i in range(70)]),
]


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("batch,hq,hkv,d,page,prefix,lens", CASES)
def test_against_float64(batch, hq, hkv, d, page, prefix, lens, dt):
    note(f"prefix {dt} B={batch} {hq}/{hkv} D={d} page={page} prefix={prefix} lens={lens[:8]}")
    check(make(dt, batch, hq, hkv, d, page, prefix, lens), dt)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("batch,hq,hkv,d,page,prefix,lens", [
    (3, 4, 2, 256, 32, 333, [0, 5, 200]),
    (17, 16, 1, 256, 2, 260, [9 * i for i in range(17)]),
    (2, 4, 2, 200, 32, 333, [70, 129]),
    (2, 4, 2, 136, 7, 100, [70, 13]),
    (5, 8, 1, 256, 4, 100, [70, 13, 0, 1, 300]),
    (5, 8, 1, 256, 6, 100, [70, 13, 0, 1, 300]),
])
def test_wide_heads(batch, hq, hkv, d, page, prefix, lens, dt):
    note(f"prefix {dt} B={batch} {hq}/{hkv} D={d} page={page} prefix={prefix}")
    check(make(dt, batch, hq, hkv, d, page, prefix, lens), dt)


@pytest.mark.parametrize("dt,batch,hq,hkv,d,page,prefix,hi", [
    ("bf16", 2, 8, 8, 128, 64, 9000, 3000),    # few sequences in many pieces
    ("bf16", 300, 32, 8, 128, 16, 200, 500),   # more sequences than waves: whole ones and cut ones
    ("f16", 200, 8, 8, 64, 32, 64, 700),
    ("f32", 64, 16, 4, 64, 16, 300, 500),      # 16-key stages
    ("f32", 9, 4, 4, 128, 16, 1500, 900),
    ("bf16", 70, 2, 1, 64, 32, 20000, 40),     # long prefix, a tile and a bit of rows
])
def test_work_lists(dt, batch, hq, hkv, d, page, prefix, hi):
    note(f"prefix {dt} B={batch} {hq}/{hkv} D={d} page={page} prefix={prefix} lens to {hi}")
    lens = np.random.default_rng(hi).integers(0, hi + 1, batch).tolist()
    lens[0], lens[-1] = hi, 0
    check(make(dt, batch, hq, hkv, d, page, prefix, lens, poison=False), dt)


@pytest.mark.parametrize("batch,hq,hkv,d,page,prefix", [
    (1, 1, 1, 64, 16, 3000), (16, 1, 1, 128, 16, 1000), (17, 2, 2, 64, 64, 777), (5, 21, 3, 36, 50, 640),
    (8, 16, 1, 128, 32, 5000), (43, 6, 2, 80, 4, 100), (64, 8, 4, 64, 16, 65), (2, 24, 24, 64, 32, 33),
])
def test_few_rows_in_float32(batch, hq, hkv, d, page, prefix):
    """Row groups of 16 that rows and heads do not divide, chunks that end inside a page; and the length on the device."""
    note(f"prefix f32 B={batch} {hq}/{hkv} D={d} page={page} prefix={prefix}")
    args = make("f32", batch, hq, hkv, d, page, prefix, [(5 * i) % 33 for i in range(batch)])
    out = check(args, "f32")
    n = torch.tensor(prefix, dtype=torch.int32, device="cuda")
    if -(-prefix // page) * page == prefix:
        assert torch.equal(out, paged_flash_attention_prefix(*args[:4], n, *args[5:]))
    n -= 20
    check((*args[:4], n, *args[5:]), "f32")


@pytest.mark.parametrize("dt,hq,hkv,d,page", [("bf16", 32, 2, 128, 16), ("f16", 18, 2, 64, 32), ("f32", 8, 2, 64, 20),
                                              ("bf16", 24, 2, 256, 16), ("f32", 13, 1, 128, 4)])
def test_runs_of_short_sequences(dt, hq, hkv, d, page):
    """A wave's run of several sequences of one stage, and of one and two and three."""
    rng = np.random.default_rng(5)
    lens = rng.integers(0, 17, 1400).tolist()
    lens[700:] = rng.integers(0, 40, 700).tolist()
    note(f"prefix {dt} {hq}/{hkv} D={d} page={page} short sequences")
    check(make(dt, 1400, hq, hkv, d, page, 40, lens, poison=False), dt)


@pytest.mark.parametrize("page", [17, 18, 31, 50, 100])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (20, 2), (36, 2)])
@pytest.mark.parametrize("dt,d", [("bf16", 64), ("f16", 128), ("bf16", 256), ("bf16", 80), ("f32", 64), ("f32", 128),
                                  ("f32", 36)])
def test_pages_that_a_stage_straddles(dt, d, hq, hkv, page):
    note(f"prefix {dt} {hq}/{hkv} D={d} page={page}")
    check(make(dt, 6, hq, hkv, d, page, 333, [0, 1, page, 15 * page + 3, 16, 200]), dt)


@pytest.mark.parametrize("dt,batch,hq,hkv,d,page,prefix,lens", [
    ("bf16", 1, 4, 1, 128, 16, 0, [30000]),        # one sequence over every wave
    ("f16", 1, 20, 1, 64, 16, 77, [30000]),        # ... over every workgroup
    ("f32", 2, 16, 1, 128, 16, 9000, [5000, 3]),   # one workgroup per CU
    ("f16", 2, 16, 1, 256, 16, 9000, [40, 900]),
    ("bf16", 48, 64, 2, 128, 64, 1300, [5] * 48),  # 12 tiles of rows, few keys
    ("bf16", 300, 16, 16, 64, 64, 3, [0] * 300),   # more items than CUs, nothing of one's own
])
def test_splits(dt, batch, hq, hkv, d, page, prefix, lens):
    note(f"prefix {dt} B={batch} {hq}/{hkv} D={d} page={page} prefix={prefix} lens={lens[:4]}")
    check(make(dt, batch, hq, hkv, d, page, prefix, lens, poison=False), dt)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("waves,stages", [(1, 2), (7, 3), (64, 4)])
def test_tuned_grids(dt, waves, stages):
    lens = [0, 5, 700, 33, 64, 1]
    with _lib.tuning(decode_waves=waves, decode_stages=stages):
        check(make(dt, 6, 8, 2, 128, 16, 150, lens), dt)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_scales(dt, scale):
    check(make(dt, 3, 4, 2, 64, 16, 100, [0, 5, 90]), dt, scale)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_unaligned_operands(dt):
    """Pools and queries between two 16-byte boundaries. Both calls lie within their bound of one float64 result, so
    they differ by at most twice it (their sums run in other orders: float32 sums of 430 weights, not 4 steps)."""
    args = list(make(dt, 3, 4, 2, 128, 16, 300, [7, 0, 130]))
    want = paged_flash_attention_prefix(*args)
    exact, bound = reference(*args)
    tol = 2 * (bound + torch.finfo(want.dtype).eps / 2 * (exact.abs() + bound) + 2.0 ** -25)
    for i in range(3):
        x = args[i]
        flat = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")
        flat[1:] = x.reshape(-1)
        args[i] = flat[1:].view(x.shape)
        got = check(tuple(args), dt)
        assert ((got.double() - want.double()).abs() <= tol).all()


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_equals_paged_attention_of_joined_tables(dt):
    """A prefix of whole pages in front of every table: each within its bound of the same float64 result."""
    q, k, v, ptab, prefix, table, lens = make(dt, 5, 8, 2, 128, 16, 320, [0, 3, 64, 100, 17], poison=False)
    joined = torch.cat([ptab.expand(5, -1), table], 1)
    one = paged_flash_attention(q, k, v, joined, lens + prefix).double()
    two = check((q, k, v, ptab, prefix, table, lens), dt).double()
    want, bound = reference(q, k, v, ptab, prefix, table, lens)
    tol = 2 * (bound + torch.finfo(q.dtype).eps / 2 * (want.abs() + bound) + 2.0 ** -25)
    assert ((one - two).abs() <= tol).all()


def test_lengths_past_the_table_and_negative():
    args = list(make("bf16", 3, 4, 2, 64, 16, 50, [32, 20, 48], extra=0, poison=False))
    args[6] = torch.tensor([32, -5, 1000], dtype=torch.int32, device="cuda")
    args[5] = args[5].clamp(min=0)
    check(tuple(args), "bf16")


def test_table_entries_are_clamped():
    """A live entry outside the pool reads the nearest page, as the paged decode's does."""
    q, k, v, ptab, prefix, table, lens = make("bf16", 2, 4, 2, 128, 16, 64, [20, 33], poison=False)
    far_p, far_t = ptab.clone(), table.clone()
    far_p[1], far_t[0, 0] = 1 << 30, -7
    near_p, near_t = far_p.clamp(0, k.shape[0] - 1), far_t.clamp(0, k.shape[0] - 1)
    got = paged_flash_attention_prefix(q, k, v, far_p, prefix, far_t, lens)
    assert torch.equal(got, paged_flash_attention_prefix(q, k, v, near_p, prefix, near_t, lens))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_scores_without_weight(dt):
    """Keys whose scores are -inf weigh nothing; with no other key the row is zero, as in the paged decode."""
    q, k, v, ptab, prefix, table, lens = make(dt, 2, 2, 1, 64, 16, 70, [20, 0], poison=False)
    q = q.abs() + 0.1
    k[ptab[2].long()] = -math.inf  # a page of the prefix
    got = paged_flash_attention_prefix(q, k, v, ptab, prefix, table, lens)
    keep = torch.cat([ptab[:2], ptab[3:]])
    want = paged_flash_attention_prefix(q, k, v, keep, prefix - 16, table, lens)
    assert torch.isfinite(got).all()
    assert (got.double() - want.double()).abs().max() <= 2 * torch.finfo(q.dtype).eps * want.abs().max() + 1e-6
    k[ptab.long()] = -math.inf
    got = paged_flash_attention_prefix(q, k, v, ptab, prefix, table, lens)
    assert (got[1] == 0).all()
    want = paged_flash_attention(q, k, v, table, lens)
    assert (got[0].double() - want[0].double()).abs().max() <= 2 * torch.finfo(q.dtype).eps * want.abs().max() + 1e-6


@pytest.mark.parametrize("page", [16, 12])
def test_pools_past_32_bits(page):
    """Pages behind 2^32 elements of a pool: the bits of a small pool's, for the append and the attention."""
    q, k, v, ptab, prefix, table, lens = make("bf16", 3, 8, 2, 128, page, 200, [30, 0, 55], poison=False)
    far = (1 << 32) // k[0].numel() + 3
    kf, vf = (torch.empty(far + x.shape[0], *x.shape[1:], dtype=x.dtype, device="cuda") for x in (k, v))
    kf[far:], vf[far:] = k, v
    move = lambda t: torch.where(t < 0, t, t + far)  # noqa: E731
    cos, sin = precompute_rope(100, 128, 10000.0, device="cuda")
    x = torch.randn(3, 12, 4, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(q.dtype)
    at = torch.tensor([30, 0, 55], device="cuda", dtype=torch.int32)
    for kp, vp, tab in ((k, v, table), (kf, vf, move(table))):
        write_to_paged_cache_rope(kp, vp, x[:, :8], x[:, 8:10], x[:, 10:], tab, at, cos, sin)
    assert torch.equal(kf[far:], k) and torch.equal(vf[far:], v)
    near = check((q, k, v, ptab, prefix, table, lens), "bf16")
    assert torch.equal(near, paged_flash_attention_prefix(q, kf, vf, move(ptab), prefix, move(table), lens))


@pytest.mark.parametrize("page", [20, 50])
def test_straddled_pages_past_32_bits(page):
    """Past 4 GiB a pool's pages are not picked by the lane: the attention within its bound all the same."""
    q, k, v, ptab, prefix, table, lens = make("bf16", 3, 8, 2, 128, page, 200, [30, 0, 55], poison=False)
    want, bound = reference(q, k, v, ptab, prefix, table, lens)
    far = (1 << 32) // k[0].numel() + 3
    kf, vf = (torch.empty(far + x.shape[0], *x.shape[1:], dtype=x.dtype, device="cuda") for x in (k, v))
    kf[far:], vf[far:] = k, v
    got = paged_flash_attention_prefix(q, kf, vf, ptab + far, prefix, torch.where(table < 0, table, table + far), lens)
    assert ((got.double() - want).abs() <= bound + torch.finfo(q.dtype).eps / 2 * (want.abs() + bound)).all()


def test_prefix_length_on_the_device_captured():
    """One captured call follows a prefix and contexts that grow; replays on a side stream, eager work between them."""
    q, k, v, ptab, _, table, lens = make("bf16", 6, 8, 2, 128, 16, 640, [30, 0, 500, 64, 10, 1], poison=False)
    table = table.clamp(min=0)
    n = torch.tensor([100], dtype=torch.int32, device="cuda")
    paged_flash_attention_prefix(q, k, v, ptab, n, table, lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_flash_attention_prefix(q, k, v, ptab, n, table, lens)
    for prefix in (100, 0, 640, 1, 5000, -3, 333):
        n.fill_(prefix)
        lens.add_(1)
        want = check((q, k, v, ptab, n, table, lens), "bf16")
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_streams_and_forms_of_arguments():
    args = make("bf16", 4, 8, 2, 64, 16, 200, [30, 0, 50, 64])
    want = paged_flash_attention_prefix(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = paged_flash_attention_prefix(*args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    q, k, v, ptab, prefix, table, lens = args
    for p in (ptab.long(), ptab.cpu(), ptab.tolist()):
        for n in (prefix, torch.tensor(prefix), torch.tensor(prefix, device="cuda"), np.int64(prefix)):
            assert torch.equal(want, paged_flash_attention_prefix(q, k, v, p, n, table.long(), lens.cpu()))
    strided = torch.empty(4, 1, 8, 64, dtype=q.dtype, device="cuda").transpose(1, 2)
    strided.copy_(q)
    assert torch.equal(want, paged_flash_attention_prefix(strided, *args[1:]))
    none = paged_flash_attention_prefix(q[:0], k, v, ptab, prefix, table[:0], lens[:0])
    assert none.shape == (0, 8, 1, 64)


def test_mixed_dtypes_and_odd_head_dim():
    """Computed in float32 as the paged decode does; a head_dim that is not whole chunks goes through copies."""
    q, k, v, ptab, prefix, table, lens = make("bf16", 2, 4, 2, 64, 16, 50, [3, 30])
    with pytest.warns(RuntimeWarning, match="copied"):
        out = paged_flash_attention_prefix(q.float(), k, v, ptab, prefix, table, lens)
    want, bound = reference(q.float(), k, v, ptab, prefix, table, lens)
    assert out.dtype == torch.float32 and ((out.double() - want).abs() <= bound + 2.0 ** -23 * want.abs()).all()
    check(make("bf16", 2, 4, 2, 30, 16, 50, [3, 30]), "bf16")


def test_serving_step_of_a_batch_behind_a_shared_prompt():
    """The three operators as one layer uses them: the shared image prompt is rotated by three axes and appended
    once, then every sequence appends and attends token after token; against float64 over all that was appended."""
    rng = np.random.default_rng(0)
    batch, hq, hkv, d, page, prompt, steps = 5, 8, 2, 64, 16, 150, 20
    sections = (8, 12, 12)
    cos, sin = precompute_rope(400, d, 10000.0, device="cuda")
    dt = torch.bfloat16
    pool = 64
    kp, vp = (torch.zeros(pool, hkv, page, d, device="cuda", dtype=dt) for _ in range(2))
    ids = torch.as_tensor(rng.permutation(pool), device="cuda", dtype=torch.int32)
    ptab, table = ids[:10], ids[10:10 + batch * 3].view(batch, 3)

    def fused(b, n):
        x = torch.as_tensor(rng.standard_normal((b, n, (hq + 2 * hkv) * d))).cuda().to(dt)
        x = x.view(b, n, hq + 2 * hkv, d).transpose(1, 2)
        return x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]

    image = torch.as_tensor(rng.integers(0, 300, (3, 1, prompt)), device="cuda")
    q, k, v = fused(1, prompt)
    write_to_paged_cache_rope(kp, vp, q, k, v, ptab, 0, cos, sin, rope_positions=image, sections=sections)
    keys, values = apply_rope_axes(k, None, image, cos, sin, sections)[0], v
    keys, values = (x.expand(batch, -1, -1, -1) for x in (keys, values))
    own = torch.zeros(batch, dtype=torch.int32, device="cuda")
    lens = torch.as_tensor(rng.integers(0, steps, batch), device="cuda", dtype=torch.int32)  # tokens still padded
    ks, vs = [keys[b] for b in range(batch)], [values[b] for b in range(batch)]
    for step in range(steps):
        q, k, v = fused(batch, 1)
        take = (lens <= step).to(torch.int32)  # a sequence joins once its padding is over
        at = (own + 300)[None, :, None].expand(3, batch, 1)
        qr, _, _ = write_to_paged_cache_rope(kp, vp, q, k, v, table, own, cos, sin, rope_positions=at,
                                             sections=sections, seq_lens=take)
        kr, _ = apply_rope_axes(k, None, at, cos, sin, sections)
        own = own + take
        out = paged_flash_attention_prefix(qr, kp, vp, ptab, prompt, table, own)
        want, bound = reference(qr, kp, vp, ptab, prompt, table, own)
        eps = torch.finfo(dt).eps
        assert ((out.double() - want).abs() <= bound + eps / 2 * (want.abs() + bound)).all()
        for b in range(batch):
            if take[b]:
                ks[b], vs[b] = torch.cat([ks[b], kr[b]], 1), torch.cat([vs[b], v[b]], 1)
            assert torch.equal(rows(kp, table[b], int(own[b])), ks[b][:, prompt:].double())
            assert torch.equal(rows(vp, ptab, prompt), vs[b][:, :prompt].double())
            s = torch.matmul(qr[b].double().view(hkv, hq // hkv, d), ks[b].double().transpose(1, 2).contiguous())
            o = torch.matmul(torch.softmax(s / math.sqrt(d), -1), vs[b].double()).view(hq, 1, d)
            assert torch.allclose(o, want[b], atol=1e-12)
