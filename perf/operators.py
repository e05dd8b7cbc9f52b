"""Multi-axis rotary positions, the rotating paged append and attention over a shared prefix, as timed cases.

``listed`` holds the standing cases, ``draw`` gives more of the same ranges,
``prepare`` makes what a program has in hand before the call, ``run`` is one
pass -- in elementary torch operations, or through ``pallas_flash`` where
``own`` is true --, ``work`` its unavoidable bytes and operations and ``exact``
its result in float64.

The three operators are what one layer of a server for text and image prompts
does around its projections:

* ``rope``: q and k rotated by positions with several axes (time, height,
  width), with the gradients where the case is a training step;
* ``append``: the new tokens' q and k rotated, k and v written to their pages;
* ``prefix``: one query token per sequence over a prefix that the whole batch
  shares and over the sequence's own pages.
"""

import math
import os
import random
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
POS = {"i32": torch.int32, "i64": torch.int64}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # The rotation of one decode step of a small batch: latency.
        dict(name="rope_step", kind="rope", dtype="bf16", batch=8, heads=32, kv_heads=8, seq=1, dim=128, axes=3,
             grid=0, pos="i64", train=False),
        # Training step over image prompts: text, then a grid of patches; the
        # heads are those of the package's long training shape.
        dict(name="rope_train", kind="rope", dtype="bf16", batch=2, heads=16, kv_heads=4, seq=8192, dim=128, axes=3,
             grid=64, pos="i64", train=True),
        # Prefill of a long video prompt.
        dict(name="rope_video", kind="rope", dtype="f16", batch=1, heads=32, kv_heads=8, seq=32768, dim=128, axes=3,
             grid=32, pos="i32", train=False),
        # Full-precision training step, multi-head, a length that no tile divides.
        dict(name="rope_f32", kind="rope", dtype="f32", batch=3, heads=12, kv_heads=12, seq=1001, dim=64, axes=2,
             grid=17, pos="i32", train=True),
        # One token of each sequence of a full decode batch.
        dict(name="append_step", kind="append", dtype="bf16", batch=64, heads=32, kv_heads=8, dim=128, page=64,
             new_lo=1, new_hi=1, old=900, axes=1, lens_seed=0),
        # Prompts of different lengths written behind what the pages hold, image positions.
        dict(name="append_prompts", kind="append", dtype="bf16", batch=8, heads=32, kv_heads=8, dim=128, page=64,
             new_lo=256, new_hi=2048, old=300, axes=3, lens_seed=1),
        # A small service with small heads in float32 (the pool's default type) and small pages.
        dict(name="append_f32", kind="append", dtype="f32", batch=16, heads=16, kv_heads=4, dim=64, page=16,
             new_lo=1, new_hi=100, old=50, axes=1, lens_seed=2),
        # A few short conversations behind a short instruction: latency.
        dict(name="prefix_small", kind="prefix", dtype="bf16", batch=4, heads=32, kv_heads=8, dim=128, page=64,
             prefix=500, lo=1, hi=64, lens_seed=3),
        # A chat service: a long instruction, conversations of up to a thousand tokens.
        dict(name="prefix_chat", kind="prefix", dtype="bf16", batch=32, heads=32, kv_heads=8, dim=128, page=64,
             prefix=6000, lo=16, hi=1024, lens_seed=4),
        # Many questions about one long document.
        dict(name="prefix_document", kind="prefix", dtype="bf16", batch=128, heads=32, kv_heads=8, dim=128, page=64,
             prefix=32768, lo=64, hi=2048, lens_seed=5),
        # Wide heads, half precision.
        dict(name="prefix_wide", kind="prefix", dtype="f16", batch=16, heads=16, kv_heads=8, dim=256, page=32,
             prefix=5003, lo=1, hi=500, lens_seed=6),
        # Small heads in float32, small pages.
        dict(name="prefix_f32", kind="prefix", dtype="f32", batch=16, heads=16, kv_heads=4, dim=64, page=16,
             prefix=2000, lo=0, hi=300, lens_seed=7),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        kind = rng.choice(["rope", "append", "prefix", "prefix"])
        kv = rng.choice([1, 2, 4, 8])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        c = dict(kind=kind, dtype=dtype, batch=_spread(rng, 1, 128), heads=kv * rng.choice([1, 2, 4, 7, 8]),
                 kv_heads=kv, dim=rng.choice([64, 80, 128, 128] if dtype == "f32" else [64, 96, 128, 128, 256]))
        if kind == "rope":
            c.update(seq=_spread(rng, 1, 32768), axes=rng.choice([1, 2, 3, 3]), grid=rng.choice([0, 9, 24, 50]),
                     pos=rng.choice(["i32", "i64"]), train=rng.random() < 0.5)
        elif kind == "append":
            new = rng.choice([1, 1, _spread(rng, 2, 4096)])
            c.update(page=rng.choice([16, 32, 64, 100]), new_lo=max(1, new // 8), new_hi=new,
                     old=_spread(rng, 1, 2000) - 1, axes=rng.choice([1, 1, 3]), lens_seed=rng.randrange(1 << 30))
        else:
            hi = _spread(rng, 1, 4096)
            c.update(page=rng.choice([16, 16, 32, 64, 64, 128, 50]), prefix=_spread(rng, 32, 65536), lo=hi // 16, hi=hi,
                     lens_seed=rng.randrange(1 << 30))
        w = work(c)
        # No dearer than the listed ones: float32 products run at about a
        # sixteenth of the 16-bit rate. A pool of at most 1 GiB each for K and V.
        if w["bytes"] > 6.5e8 or w["flops"] * (16 if dtype == "f32" else 1) > 7e10:
            continue
        if kind != "rope" and _pages(c)[0] * kv * c["page"] * c["dim"] * _size(c) > 1 << 30:
            continue
        return c


# ---------------------------------------------------------------------------
# sizes that follow from a case
# ---------------------------------------------------------------------------
def _size(case):
    return 4 if case["dtype"] == "f32" else 2


def _sections(case):
    """The rotated pairs of each axis: halves, or a quarter for time and the rest for height and width."""
    half, axes = case["dim"] // 2, case["axes"]
    if axes == 1:
        return [half]
    if axes == 2:
        return [half // 2, half - half // 2]
    time, height = half // 4, (half - half // 4) // 2
    return [time, height, half - time - height]


def _lengths(case):
    """The sequences' lengths: part of the case, so that its work is known."""
    lo, hi = (case["new_lo"], case["new_hi"]) if case["kind"] == "append" else (case["lo"], case["hi"])
    return np.random.default_rng(case["lens_seed"]).integers(lo, hi + 1, case["batch"])


def _pages(case):
    """Pages in the pool, in a sequence's table row, and in the prefix's table."""
    page, batch = case["page"], case["batch"]
    if case["kind"] == "append":
        per = -(-(case["old"] + case["new_hi"]) // page)
        return batch * per, per, 0
    per, pre = max(1, -(-case["hi"] // page)), -(-case["prefix"] // page)
    return pre + int(sum(-(-int(n) // page) for n in _lengths(case))), per, pre


def _axis_of(case):
    """The axis of each rotated pair, [dim / 2]."""
    return torch.as_tensor(np.repeat(np.arange(case["axes"]), _sections(case)), device="cuda")


def work(case):
    es, b, d = _size(case), case["batch"], case["dim"]
    hq, hkv = case["heads"], case["kv_heads"]
    if case["kind"] == "rope":
        tokens = b * case["seq"]
        passes = 2 if case["train"] else 1
        table = 2 * 4 * d * min(_reach(case), tokens * case["axes"])
        pos = tokens * case["axes"] * (4 if case["pos"] == "i32" else 8)
        values = tokens * (hq + hkv) * d
        return {"bytes": passes * (2 * values * es + table + pos), "flops": passes * 3 * values}
    if case["kind"] == "append":
        tokens = int(_lengths(case).sum())
        table = 2 * 4 * d * min(_reach(case), tokens * case["axes"])
        return {"bytes": 2 * tokens * (hq + 2 * hkv) * d * es + table + 4 * tokens * case["axes"],
                "flops": 3 * tokens * (hq + hkv) * d}
    keys = int(_lengths(case).sum())
    n = b * case["prefix"] + keys
    return {"bytes": 2 * (case["prefix"] + keys) * hkv * d * es + 2 * b * hq * d * es + 4 * sum(_pages(case)[1:]),
            "flops": 4 * n * hq * d}


def _reach(case):
    """Rows of the rotary tables."""
    return case["seq"] + 64 if case["kind"] == "rope" else case["old"] + case["new_hi"] + 64


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _tables(rows, dim):
    """cos and sin, [rows, dim] float32, of position / 10000^(pair / (dim / 2)), the halves alike."""
    half = dim // 2
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    angle = torch.outer(torch.arange(rows, dtype=torch.float64, device="cuda"), freq)
    return (torch.cat([angle.cos(), angle.cos()], 1).float(), torch.cat([angle.sin(), angle.sin()], 1).float())


def _positions(case, count, gen):
    """[axes, batch, count]: text counts on in every axis; behind it a grid of patches, row by row, frame by frame."""
    b, axes = case["batch"], case["axes"]
    start = torch.randint(0, 33, (b, 1), generator=gen, device="cuda")
    i = torch.arange(count, device="cuda")[None] + start
    grid = case.get("grid", 24)
    if axes == 1 or grid == 0 or count < 2:
        return i[None].expand(axes, b, count).contiguous()
    patch = (torch.arange(count, device="cuda") - count // 4).clamp(min=0)
    cols = min(grid, max(1, count // 4))
    frame, row, col = patch // (cols * cols), patch // cols % cols, patch % cols
    at = start + count // 4
    image = (torch.arange(count, device="cuda") >= count // 4)[None]
    of = [at + frame, at + row, at + col] if axes == 3 else [at + patch // cols, at + col]
    top = case["seq"] + 64 if case["kind"] == "rope" else case["new_hi"] + 64
    return torch.stack([torch.where(image, p.clamp(max=top - 1), i) for p in of])


def _prepare_rope(case, gen):
    dt, b, s, d = DTYPES[case["dtype"]], case["batch"], case["seq"], case["dim"]

    def projected(heads):  # [batch, heads, seq, dim], a view of a projection's [batch, seq, heads * dim]
        x = torch.randn((b, s, heads * d), generator=gen, device="cuda", dtype=dt)
        return x.view(b, s, heads, d).transpose(1, 2)

    q, k = projected(case["heads"]), projected(case["kv_heads"])
    st = dict(q=q.requires_grad_(case["train"]), k=k.requires_grad_(case["train"]),
              positions=_positions(case, s, gen).to(POS[case["pos"]]))
    if case["train"]:
        st["dq"], st["dk"] = (torch.randn(x.shape, generator=gen, device="cuda", dtype=dt) for x in (q, k))
    st["cos"], st["sin"] = _tables(_reach(case), d)
    return st


def _prepare_append(case, gen):
    dt, b, d, page = DTYPES[case["dtype"]], case["batch"], case["dim"], case["page"]
    hq, hkv, n = case["heads"], case["kv_heads"], case["new_hi"]
    pool, per, _ = _pages(case)
    x = torch.randn((b, n, (hq + 2 * hkv) * d), generator=gen, device="cuda", dtype=dt)  # one fused projection
    x = x.view(b, n, hq + 2 * hkv, d).transpose(1, 2)
    st = dict(q=x[:, :hq], k=x[:, hq:hq + hkv], v=x[:, hq + hkv:])
    for name in ("k_pages", "v_pages"):
        st[name] = torch.randn((pool, hkv, page, d), generator=gen, device="cuda", dtype=dt)
    st["table"] = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32).view(b, per)
    new = torch.as_tensor(_lengths(case)).to("cuda", torch.int32)
    st["lens"] = new if case["new_hi"] > 1 else None
    # each sequence holds another number of tokens already
    held = torch.randint(0, case["old"] + 1, (b,), generator=gen, device="cuda")
    st["position"] = held.to(torch.int32)
    st["rope"] = None
    if case["axes"] > 1:
        st["rope"] = (_positions(case, n, gen) + held[None, :, None]).clamp(max=_reach(case) - 1).to(torch.int32)
    st["cos"], st["sin"] = _tables(_reach(case), d)
    return st


def _prepare_prefix(case, gen):
    dt, b, d, page = DTYPES[case["dtype"]], case["batch"], case["dim"], case["page"]
    hq, hkv = case["heads"], case["kv_heads"]
    pool, per, pre = _pages(case)
    st = dict(q=torch.randn((b, hq, 1, d), generator=gen, device="cuda", dtype=dt))
    for name in ("k_pages", "v_pages"):
        st[name] = torch.randn((pool, hkv, page, d), generator=gen, device="cuda", dtype=dt)
    ids = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    st["prefix_table"], st["prefix_len"] = ids[:pre].clone(), case["prefix"]
    lens = _lengths(case)
    need = -(-lens // page)
    table = np.full((b, per), -1, np.int64)  # -1 behind a sequence's last page
    at = np.arange(per)[None] < need[:, None]
    table[at] = np.arange(int(need.sum())) + pre
    t = torch.as_tensor(table, device="cuda")
    st["table"] = torch.where(t >= 0, ids[t.clamp(min=0)], -1).to(torch.int32)
    st["lens"] = torch.as_tensor(lens).to("cuda", torch.int32)
    return st


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    make = {"rope": _prepare_rope, "append": _prepare_append, "prefix": _prepare_prefix}[case["kind"]]
    st = dict(make(case, gen), case=case)
    if case["kind"] != "prefix":
        st["axis"] = _axis_of(case)
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _calls():
    # The package's folder is not an importable name.
    path = os.path.abspath("tpu-native-pallas-flashattention_amd")
    if path not in sys.path:
        sys.path.insert(1, path)
    import pallas_flash
    return pallas_flash


def _rows(axis, table, positions):
    """The rows of a rotary table for positions [axes, batch, seq]: [batch, 1, seq, dim]."""
    at = positions.long()[axis].permute(1, 2, 0)  # [batch, seq, dim / 2]
    at = torch.cat([at, at], -1)
    return table[at, torch.arange(table.shape[1], device=table.device)][:, None]


def _rotated(x, cos, sin):
    x = x.float()
    half = x.shape[-1] // 2
    return x * cos + torch.cat([-x[..., half:], x[..., :half]], -1) * sin


def _run_rope(st):
    case, q, k = st["case"], st["q"], st["k"]
    if own:
        pf = _calls()
        qr, kr = pf.apply_rope_axes(q, k, st["positions"], st["cos"], st["sin"], _sections(case))
    else:
        cos, sin = (_rows(st["axis"], st[t], st["positions"]) for t in ("cos", "sin"))
        qr, kr = (_rotated(x, cos, sin).to(x.dtype) for x in (q, k))
    if not case["train"]:
        return qr, kr
    dq, dk = torch.autograd.grad((qr, kr), (q, k), (st["dq"], st["dk"]))
    return qr.detach(), kr.detach(), dq, dk


def _run_append(st):
    case = st["case"]
    if own:
        pf = _calls()
        qr, kp, vp = pf.write_to_paged_cache_rope(
            st["k_pages"], st["v_pages"], st["q"], st["k"], st["v"], st["table"], st["position"], st["cos"], st["sin"],
            rope_positions=st["rope"], sections=_sections(case), seq_lens=st["lens"])
        return qr, kp, vp
    q, k, v, page = st["q"], st["k"], st["v"], case["page"]
    n = q.shape[2]
    i = torch.arange(n, device=q.device)[None].expand(q.shape[0], n)
    live = i < (n if st["lens"] is None else st["lens"][:, None])
    # a padded row writes its sequence's last token once more
    i = i if st["lens"] is None else torch.minimum(i, st["lens"][:, None].long() - 1)
    at = st["position"].long()[:, None] + i
    rope = at[None] if st["rope"] is None else st["rope"].long()
    cos, sin = (_rows(st["axis"], st[t], rope) for t in ("cos", "sin"))
    qr = torch.where(live[:, None, :, None], _rotated(q, cos, sin), 0.0).to(q.dtype)
    kr = _rotated(k, cos, sin).to(k.dtype)
    last = i[:, None, :, None].expand(k.shape)
    pages = torch.gather(st["table"].long(), 1, at // page)
    for pool, rows in ((st["k_pages"], kr), (st["v_pages"], v)):
        pool[pages, :, at % page] = torch.gather(rows, 2, last).transpose(1, 2)
    return qr, st["k_pages"], st["v_pages"]


def _run_prefix(st):
    q, kp, vp = st["q"], st["k_pages"], st["v_pages"]
    if own:
        pf = _calls()
        return pf.paged_flash_attention_prefix(q, kp, vp, st["prefix_table"], st["prefix_len"], st["table"], st["lens"])
    b, hq, _, d = q.shape
    hkv, page = kp.shape[1], kp.shape[2]
    g = hq // hkv
    qf = q.float().view(b, hkv, g, d) * d ** -0.5
    pre = st["prefix_table"].long()
    kf, vf = (x[pre].transpose(0, 1).reshape(hkv, -1, d)[:, :st["prefix_len"]].float() for x in (kp, vp))
    rows = qf.transpose(0, 1).reshape(hkv, b * g, d)
    sp = torch.matmul(rows, kf.transpose(1, 2).contiguous())  # [hkv, b g, prefix]
    tab = st["table"].long().clamp(min=0)
    ko, vo = (x[tab].transpose(1, 2).reshape(b, hkv, -1, d).float() for x in (kp, vp))
    so = torch.matmul(qf, ko.transpose(2, 3).contiguous())  # [b, hkv, g, own]
    keep = torch.arange(so.shape[3], device=q.device)[None] < st["lens"][:, None]
    so = torch.where(keep[:, None, None], so, -math.inf)
    top = torch.maximum(sp.amax(2).view(hkv, b, g).transpose(0, 1), so.amax(3))
    pp = torch.exp(sp - top.transpose(0, 1).reshape(hkv, b * g, 1))
    po = torch.exp(so - top[..., None])
    total = pp.sum(2).view(hkv, b, g).transpose(0, 1) + po.sum(3)
    out = torch.matmul(pp, vf).view(hkv, b, g, d).transpose(0, 1) + torch.matmul(po, vo)
    return (out / total[..., None]).reshape(b, hq, 1, d).to(q.dtype)


def run(state):
    return {"rope": _run_rope, "append": _run_append, "prefix": _run_prefix}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------
# the definition, in float64
# ---------------------------------------------------------------------------
def _turn(x, positions, st, case, back=False):
    """Each pair (x[i], x[i + dim / 2]) of token t turned by the table row of its axis' position; back: the transpose."""
    half, out, at = case["dim"] // 2, torch.empty(x.shape, dtype=torch.float64, device=x.device), 0
    x = x.detach().double()
    for axis, count in enumerate(_sections(case)):
        p, lo, hi = positions[axis].long(), slice(at, at + count), slice(half + at, half + at + count)
        c, s = (st[t].double()[p][:, None] for t in ("cos", "sin"))  # [batch, 1, seq, dim]
        if back:
            out[..., lo] = x[..., lo] * c[..., lo] + x[..., hi] * s[..., hi]
            out[..., hi] = x[..., hi] * c[..., hi] - x[..., lo] * s[..., lo]
        else:
            out[..., lo] = x[..., lo] * c[..., lo] - x[..., hi] * s[..., lo]
            out[..., hi] = x[..., hi] * c[..., hi] + x[..., lo] * s[..., hi]
        at += count
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "rope":
        out = tuple(_turn(st[n], st["positions"], st, case) for n in ("q", "k"))
        if case["train"]:
            out += tuple(_turn(st[n], st["positions"], st, case, back=True) for n in ("dq", "dk"))
        return out
    if case["kind"] == "append":
        n, held = case["new_hi"], st["position"].long()
        rope = st["rope"] if st["rope"] is not None else (held[:, None] + torch.arange(n, device="cuda"))[None]
        rope = rope.clamp(max=_reach(case) - 1)
        qr, kr, v = _turn(st["q"], rope, st, case), _turn(st["k"], rope, st, case), st["v"].double()
        kp, vp = st["k_pages"].double(), st["v_pages"].double()
        for b, count in enumerate(_lengths(case).tolist()):
            qr[b, :, count:] = 0
            at = held[b] + torch.arange(count, device="cuda")
            page, slot = st["table"][b].long()[at // case["page"]], at % case["page"]
            kp[page, :, slot] = kr[b, :, :count].transpose(0, 1)
            vp[page, :, slot] = v[b, :, :count].transpose(0, 1)
        return qr, kp, vp
    q = st["q"].double()
    hkv, d, g = case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"]
    out = torch.empty_like(q)
    page, pre = case["page"], st["prefix_table"].long()
    kf, vf = (st[n][pre].double().transpose(0, 1).reshape(hkv, -1, d)[:, :case["prefix"]] for n in ("k_pages", "v_pages"))
    for b, count in enumerate(_lengths(case).tolist()):
        t = st["table"][b, :-(-count // page)].long()
        ko, vo = (st[n][t].double().transpose(0, 1).reshape(hkv, -1, d)[:, :count] for n in ("k_pages", "v_pages"))
        keys, values = torch.cat([kf, ko], 1), torch.cat([vf, vo], 1)
        scores = torch.matmul(q[b].view(hkv, g, d) / math.sqrt(d), keys.transpose(1, 2).contiguous())
        out[b] = torch.matmul(torch.softmax(scores, -1), values).view(case["heads"], 1, d)
    return out


if __name__ == "__main__":
    rng = random.Random(0)
    for c in listed() + [draw(rng) for _ in range(8)]:
        print(c.get("name", "(drawn)"), c, work(c))
