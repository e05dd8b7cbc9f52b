"""GPU tier: the C++ host side of the multi-axis rotation, the rotating paged write and the shared-prefix attention
against their general path: the same bits, and what it takes and declines."""

from __future__ import annotations

import contextlib

import pytest
import torch

from pallas_flash import (_lib, apply_rope_axes, paged_flash_attention_prefix, precompute_rope,
                          write_to_paged_cache_rope)

pytestmark = pytest.mark.gpu


@contextlib.contextmanager
def general_path():
    real, _lib._calls = _lib.calls(), _lib._Declining
    try:
        yield
    finally:
        _lib._calls = real


def r(*shape, dt=torch.bfloat16, seed=0):
    return torch.randn(shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda").to(dt)


def rope_args(dt=torch.bfloat16, b=2, s=33):
    q, k = r(b, s, 6, 64, dt=dt).transpose(1, 2), r(b, s, 2, 64, dt=dt, seed=1).transpose(1, 2)
    cos, sin = precompute_rope(100, 64, 10000.0, device="cuda")
    pos = torch.randint(0, 100, (3, b, s), generator=torch.Generator("cuda").manual_seed(2), device="cuda")
    return [q, k, pos, cos, sin, (8, 12, 12)]


def write_args(dt=torch.bfloat16, b=2, s=5):
    q, k, pos, cos, sin, sections = rope_args(dt, b, s)
    kp, vp = torch.zeros(12, 2, 16, 64, device="cuda", dtype=dt), torch.zeros(12, 2, 16, 64, device="cuda", dtype=dt)
    table = torch.randperm(12, generator=torch.Generator("cuda").manual_seed(3), device="cuda").to(torch.int32)
    at = torch.tensor([3, 30][:b], dtype=torch.int32, device="cuda")
    return [kp, vp, q, k, k + 1, table.view(b, -1), at, cos, sin, pos, sections,
            torch.tensor([s, 2][:b], dtype=torch.int32, device="cuda")]


def write(a):
    return write_to_paged_cache_rope(*a[:9], rope_positions=a[9], sections=a[10], seq_lens=a[11])


def prefix_args(dt=torch.bfloat16):
    table = torch.randperm(30, generator=torch.Generator("cuda").manual_seed(3), device="cuda").to(torch.int32)
    return [r(3, 6, 1, 64, dt=dt), r(30, 2, 16, 64, dt=dt, seed=4), r(30, 2, 16, 64, dt=dt, seed=5), table[:15], 230,
            table[15:].view(3, 5), torch.tensor([0, 33, 80], dtype=torch.int32, device="cuda"), None]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("with_k,want_q,want_k", [(1, 1, 1), (1, 1, 0), (1, 0, 1), (0, 1, 0), (1, 0, 0)])
def test_rotation(dt, with_k, want_q, want_k):
    def go():
        q, k, *rest = rope_args(dt)
        q.requires_grad_(bool(want_q)), k.requires_grad_(bool(want_k))
        out = [x for x in apply_rope_axes(q, k if with_k else None, *rest) if x is not None]
        leaves = [x for x in (q, k) if x.requires_grad]
        grads = torch.autograd.grad([o for o in out if o.requires_grad], leaves,
                                    [o.detach() * 2 for o in out if o.requires_grad], allow_unused=True) if leaves else ()
        return [o.detach() for o in out] + [g for g in grads if g is not None]
    got = go()
    with general_path():
        want = go()
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(a.is_contiguous() for a in got)


def test_rotation_gradients_twice_and_alone():
    q, k, *rest = rope_args(torch.float32)
    q.requires_grad_(), k.requires_grad_()

    def go():
        qr, kr = apply_rope_axes(q, k, *rest)
        (dk,) = torch.autograd.grad(kr.sum(), k, retain_graph=True)  # q's output has no gradient, k's is expanded
        dq, dk2 = torch.autograd.grad((qr * qr * q).sum() + (kr * k).sum(), (q, k), create_graph=True)
        ddq, ddk = torch.autograd.grad((dq * dq).sum() + (dk2 * k).sum(), (q, k))
        return [x.detach() for x in (dk, dq, dk2, ddq, ddk)]
    got = go()
    with general_path():
        want = go()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert got[3].abs().max() > 0


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
def test_write_and_prefix(dt):
    a, b = write_args(dt), write_args(dt)
    got = write(a)
    with general_path():
        want = write(b)
    assert all(torch.equal(x, y) for x, y in zip(got, want)) and got[1].any()
    p = prefix_args(dt)
    got = paged_flash_attention_prefix(*p[:7])
    with general_path():
        want = paged_flash_attention_prefix(*p[:7])
    assert torch.equal(got, want)
    p[4] = torch.tensor(230, dtype=torch.int32, device="cuda")
    assert torch.equal(paged_flash_attention_prefix(*p[:7]), want)


def test_takes_the_plain_case():
    c = _lib.calls()
    assert hasattr(c, "__file__"), "the extension is not built"
    a = rope_args()
    for positions, sections in ((a[2], a[5]), (a[2], list(a[5])), (a[2][:, :1], a[5]), (a[2][:, 0], a[5]),
                                (a[2][0, 0], None), (a[2][0], None), (a[2][:1], (32,)), (a[2].int(), a[5])):
        assert c.rope_axes(a[0], a[1], positions, a[3], a[4], sections) is not None
    assert c.rope_axes(a[0], None, *a[2:])[1] is None
    a = write_args()
    assert c.rope_write(*a) is not None
    assert c.rope_write(*a[:9], None, None, None) is not None
    assert c.rope_write(*a[:6], a[6][:1], *a[7:]) is not None
    assert c.prefix(*prefix_args()) is not None


def test_declines_the_rest():
    c = _lib.calls()
    a = rope_args()
    other = {0: (a[0].double(), a[0][0], a[0].cpu(), a[0][:, :, :0], r(2, 64, 6, 33).transpose(1, 3), r(2, 6, 33, 63)),
             1: (a[1].float(), a[1][:, :, 1:], a[1][:1], a[1][..., :32], 3),
             2: (a[2][:2], a[2][:, :, 1:], a[2].float(), a[2].cpu(), a[2][0, 0], a[2].tolist(), a[2].short()),
             3: (a[3].half(), a[3][:, :32], a[3].cpu(), a[3].clone().requires_grad_(), a[3][0]),
             4: (a[4][:50],),
             5: ((8, 12, 11), (8, 24), (32, 0, 0), (33, -1), (1, 1, 1, 1, 28), "aaa", (8.0, 12, 12), None)}
    for i, bad in other.items():
        for x in bad:
            assert c.rope_axes(*a[:i], x, *a[i + 1:]) is None, (i, x)
    a = write_args()
    other = {0: (a[0].float(), a[0][:, :1], a[0].transpose(0, 1)), 1: (a[1][:3],), 2: (a[2][:1], a[2][..., :32], a[2][:, :3]),
             3: (a[3].float(), a[3][:, :, 1:]), 4: (a[4][:, :1],),
             5: (a[5].long(), a[5][:1], a[5][0], a[5][:, :0]), 6: (a[6].long(), 3, a[6][:, None], a[6][:0]),
             7: (a[7][:, :32],), 9: (None, a[9][:, :, 1:]), 10: ((8, 12), None), 11: (a[11].long(), a[11][:1], [5, 2])}
    for i, bad in other.items():
        for x in bad:
            assert c.rope_write(*a[:i], x, *a[i + 1:]) is None, (i, x)
    assert not a[0].any() and not a[1].any()
    a = prefix_args()
    other = {0: (a[0].float(), a[0][:, :5], a[0][..., :32], a[0].cpu()), 1: (a[1][:5], a[1].transpose(0, 1)),
             3: (a[3].long(), a[3][None], a[3][:0], a[3].cpu()), 4: (0, -1, 241, 3.0, torch.tensor(3),
                                                                     torch.tensor(3, device="cuda")),
             5: (a[5][:2], a[5].long(), a[5][:, :0]), 6: (a[6][:2], a[6].long()), 7: (1, "a", float("nan"))}
    for i, bad in other.items():
        for x in bad:
            assert c.prefix(*a[:i], x, *a[i + 1:]) is None, (i, x)


@pytest.mark.parametrize("grad", [False, True])
def test_sizes_past_the_grid(grad):
    """Refused before any launch, by the extension and by the general path."""
    q = r(1, 65536, 1, 2).requires_grad_(grad)
    t = torch.ones(4, 2, device="cuda")
    at = torch.zeros(1, dtype=torch.int32, device="cuda")
    with pytest.raises(NotImplementedError):
        apply_rope_axes(q, None, at, t, t)
    with general_path(), pytest.raises(NotImplementedError):
        apply_rope_axes(q, None, at, t, t)
    assert torch.equal(apply_rope_axes(q[:, :65535], None, at, t, 0 * t)[0], q[:, :65535])
