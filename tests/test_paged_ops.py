"""Serving over a paged key/value cache and the query/key norm with rotary embedding, against plain implementations in
64 bits on the CPU, through the public wrappers and the C ABI.

Tolerances count roundings: ``half(dtype)`` = finfo.eps / 2 is the most one rounding moves a value, relative to it; sums
of n fp32 terms move by at most n 2^-24 of the sum of their magnitudes.  Whole numbers are compared exactly."""
import math

import pytest
import torch

from merak_amd import mpu, ops

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def rounding(dtype, ref):
    """The most one rounding to dtype moves a value near ref.  Below the smallest normal number (2^-14 in half precision)
    values are evenly spaced by smallest_normal * eps (2^-24 there), so a rounding moves up to half of that however small
    ref is: half() * |ref| alone is no bound for those."""
    return half(dtype) * ref.abs() * 1.01 + torch.finfo(dtype).smallest_normal * half(dtype)


def gen(seed):
    return torch.Generator().manual_seed(9000 + seed)


def within(got, ref, bound):
    """|got - ref| <= bound, elementwise; NaN nowhere."""
    got, err = got.detach().double().cpu(), None
    err = (got - ref).abs()
    assert not torch.isnan(got).any()
    bad = err > bound
    assert not bad.any(), (int(bad.sum()), float((err / bound.clamp_min(1e-300)).max()))


# --------------------------------------------------------------------------- page plan
def plan_reference(lens, new, held, table, free, count, page, cap):
    table = [list(r) for r in table]
    held = list(held)
    room, cols = len(table[0]) * page if table else 0, len(table[0]) if table else 0
    count = max(0, min(count, len(free)))
    left, asked = count, 0
    slots, positions, cu, kv, granted = [-1] * cap, [-1] * cap, [0], [], []
    for r in range(len(lens)):
        n = min(max(new[r], 0), cap + 1)
        cu.append(cu[-1] + n)
        ok = lens[r] >= 0 and 0 <= held[r] <= cols and lens[r] + n <= room and cu[-1] <= cap
        need = max(0, -(-(lens[r] + n) // page) - held[r]) if ok else 0
        asked += need
        if need and asked > count:
            ok = False
        granted.append(ok)
        kv.append(lens[r] + n if ok else 0)
        if not ok:
            continue
        for _ in range(need):
            left -= 1
            table[r][held[r]] = free[left]
            held[r] += 1
        for i in range(n):
            p = lens[r] + i
            positions[cu[r] + i] = p
            slots[cu[r] + i] = table[r][p // page] * page + p % page
    return slots, positions, cu, kv, granted, held, left, table


def plan_inputs(lens, new, held, cols, n_free, seed, capacity=None):
    g = gen(seed)
    R = len(lens)
    pages = torch.randperm(sum(max(h, 0) for h in held) + n_free + 7, generator=g).tolist()
    table, at = [], 0
    for h in held:
        h = min(max(h, 0), cols)
        table.append(pages[at:at + h] + [-7] * (cols - h))
        at += h
    free = pages[at:at + n_free]
    free += [-9] * ((capacity or n_free) - n_free)
    return table, free


def run_plan(gpu, lens, new, held, table, free, count, page, cap):
    t = lambda v, dt: torch.tensor(v, dtype=dt, device=gpu)
    tab = torch.tensor(table, dtype=torch.int32, device=gpu).view(len(lens), -1)
    h, c = t(held, torch.int32), t([count], torch.int32)
    plan = ops.paged_plan(t(lens, torch.int64), t(new, torch.int64), h, tab, t(free, torch.int32), c, page, cap)
    assert h.tolist() == list(held) and c.item() == count                # the old counts are inputs only
    return (plan.slots.tolist(), plan.positions.tolist(), plan.cu.tolist(), plan.kv_lens.tolist(), plan.granted.tolist(),
            plan.held.tolist(), plan.free_count.item(), tab.tolist())


@pytest.mark.parametrize("page", [1, 16, 64])
@pytest.mark.parametrize("R,new_hi,spare", [(1, 1, 0), (3, 40, 5), (64, 1, 2), (257, 9, 0), (300, 30, 11), (1500, 3, 0)])
def test_plan_random(gpu, page, R, new_hi, spare):
    g = gen(R + page)
    lens = torch.randint(0, 200, (R,), generator=g).tolist()
    new = torch.randint(0, new_hi + 1, (R,), generator=g).tolist()
    held = [-(-a // page) + (i % 5 == 0) for i, a in enumerate(lens)]     # some hold a page more than they use
    cols = max(max(-(-(a + b) // page) for a, b in zip(lens, new)), max(held)) + 1
    need = sum(max(0, -(-(a + b) // page) - h) for a, b, h in zip(lens, new, held))
    table, free = plan_inputs(lens, new, held, cols, need + spare, R)
    cap = sum(new) + spare
    assert run_plan(gpu, lens, new, held, table, free, need + spare, page, cap) == plan_reference(
        lens, new, held, table, free, need + spare, page, cap)


def test_plan_refuses_what_does_not_fit(gpu):
    """Too few pages, a row too long, tokens behind the buffer, bad lengths and counts: each refused alone, the rest
    served; a request that needs no page is served after one that got none."""
    page, cols = 16, 6
    lens = [0, 90, 10, -3, 5, 40, 1, 12, 33, 2 ** 62, 7, 0]
    new = [17, 9, 4, 2, 20, 60, -5, 3, 40, 1, 2 ** 61, 1]
    held = [0, 6, 1, 0, 1, 3, 1, 1, 3, 0, 1, 7]
    for n_free in (0, 2, 3, 8):
        for cap in (0, 40, 90, 400):
            table, free = plan_inputs(lens, new, held, cols, n_free, 3, capacity=12)
            got = run_plan(gpu, lens, new, held, table, free, n_free, page, cap)
            want = plan_reference(lens, new, held, table, free, n_free, page, cap)
            assert got == want, (n_free, cap)
    # a count beyond the list is taken as the list's length, a negative one as empty
    for count in (-4, 99):
        table, free = plan_inputs(lens, new, held, cols, 4, 5)
        got = run_plan(gpu, lens, new, held, table, free, count, page, 300)
        assert got == plan_reference(lens, new, held, table, free, count, page, 300)


def test_plan_fills_a_table_that_lagged_behind_and_empty_batches(gpu):
    # fewer pages held than the cached tokens need: the missing ones are taken too, with or without new tokens
    lens, new, held = [50, 50, 3], [5, 0, 0], [1, 2, 0]
    table, free = plan_inputs(lens, new, held, 8, 9, 6)
    assert run_plan(gpu, lens, new, held, table, free, 9, 16, 8) == plan_reference(lens, new, held, table, free, 9, 16, 8)
    none = torch.zeros((0,), dtype=torch.int64, device=gpu)
    plan = ops.paged_plan(none, none, none.int(), torch.zeros((0, 4), dtype=torch.int32, device=gpu), none.int(),
                          torch.zeros(1, dtype=torch.int32, device=gpu), 16, 3)
    assert plan.cu.tolist() == [0] and plan.slots.tolist() == [-1] * 3 and plan.free_count.tolist() == [0]


def test_release_returns_pages_in_order(gpu):
    R, cols = 9, 5
    held = [3, 0, 5, 1, 2, 4, 5, -1, 2]
    table = torch.arange(R * cols, dtype=torch.int32).view(R, cols)
    done = torch.tensor([1, 1, 0, 1, 0, 1, 0, 1, 1], dtype=torch.bool)
    free0, count0 = torch.full((14,), -1, dtype=torch.int32), 2
    free0[:2] = torch.tensor([100, 101], dtype=torch.int32)
    want, kept = [100, 101], list(held)
    for r in range(R):
        h = max(held[r], 0)
        if done[r] and h and len(want) + h <= 14:
            want += table[r, :h].tolist()
            kept[r] = 0
    h, f, c = torch.tensor(held, dtype=torch.int32, device=gpu), free0.to(gpu), torch.tensor([count0], dtype=torch.int32, device=gpu)
    ops.paged_release(done.to(gpu), h, table.to(gpu), f, c)
    assert c.item() == len(want) and f.tolist()[:len(want)] == want and h.tolist() == kept
    # a list without room: that request and the ones behind it keep their pages
    held = [2, 3, 1]
    h, f, c = torch.tensor(held, dtype=torch.int32, device=gpu), torch.full((4,), -1, dtype=torch.int32, device=gpu), torch.tensor([0], dtype=torch.int32, device=gpu)
    ops.paged_release(torch.ones(3, dtype=torch.bool, device=gpu), h, table[:3].to(gpu), f, c)
    assert c.item() == 2 and h.tolist() == [0, 3, 1] and f.tolist() == [0, 1, -1, -1]


# --------------------------------------------------------------------------- norm + rotary
def tables(d, n, seed, equal_halves=True):
    """cos / sin of any angles; unequal halves are allowed by the definition and tested as such."""
    a = torch.rand(n, d, generator=gen(seed), dtype=torch.float64) * 50
    if equal_halves:
        a[:, d // 2:] = a[:, :d // 2]
    return a.cos(), a.sin()


def rot(x):
    h = x.shape[-1] // 2
    return torch.cat([-x[..., h:], x[..., :h]], -1)


def norm_rope64(x, w, cos, sin, eps):
    """-> value, and the sum of magnitudes of what is added up in it"""
    z = x if w is None else x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * w
    return z * cos + rot(z) * sin, (z * cos).abs() + (rot(z) * sin).abs()


def rotary_case(T, hq, hk, d, dtype, norm, seed, table_dtype=torch.float32):
    g = gen(seed)
    P = 300
    qkv = (torch.randn(T, (hq + 2 * hk) * d, generator=g) * 2).to(dtype)
    cos, sin = tables(d, P, seed, equal_halves=seed % 2 == 0)
    cos, sin = cos.to(table_dtype), sin.to(table_dtype)
    pos = torch.randint(0, P, (T,), generator=g)
    qw = kw = None
    if norm in ("both", "q"):
        qw = (torch.rand(d, generator=g) + 0.5).to(dtype)
    if norm == "both":
        kw = (torch.randn(d, generator=g)).to(dtype)
    return qkv, cos, sin, pos, qw, kw


ROTARY = [(1, 1, 1, 64), (7, 12, 12, 64), (33, 32, 8, 128), (130, 8, 1, 128), (5, 7, 7, 128), (64, 28, 4, 64)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,hq,hk,d", ROTARY)
@pytest.mark.parametrize("norm", ["both", "q", "none"])
def test_qk_norm_rope_forward(gpu, dtype, T, hq, hk, d, norm):
    table_dtype = dtype if T % 2 else torch.float32
    qkv, cos, sin, pos, qw, kw = rotary_case(T, hq, hk, d, dtype, norm, T + hq, table_dtype)
    mv = lambda t: None if t is None else t.to(gpu)
    q, k = ops.qk_norm_rope(mv(qkv), mv(cos), mv(sin), mv(pos), hq, mv(qw), mv(kw), 1e-5)
    assert q.shape == (T, hq, d) and k.shape == (T, hk, d) and q.dtype == dtype
    x = qkv.double().view(T, -1, d)
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    for got, a, w in ((q, x[:, :hq], qw), (k, x[:, hq:hq + hk], kw)):
        ref, mag = norm_rope64(a, None if w is None else w.double(), c, s, 1e-5)
        # one rounding of the result; fp32: the mean (d terms, halved by the root), root, division, three products, a sum
        within(got, ref, rounding(dtype, ref) + (d / 2 + 8) * U32 * mag)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,hq,hk,d", ROTARY + [(1200, 4, 2, 64)])
@pytest.mark.parametrize("norm", ["both", "q", "none"])
def test_qk_norm_rope_backward(gpu, dtype, T, hq, hk, d, norm):
    qkv, cos, sin, pos, qw, kw = rotary_case(T, hq, hk, d, dtype, norm, 50 + T + hq)
    g = gen(77)
    dq, dk, dv = (torch.randn(T, n, d, generator=g).to(dtype) for n in (hq, hk, hk))
    mv = lambda t: None if t is None else t.to(gpu)
    args = [mv(t) for t in (dq, dk, dv, qkv, cos, sin, pos, qw, kw)]
    dqkv, dqw, dkw = ops.qk_norm_rope_bwd(*args, 1e-5)
    again = ops.qk_norm_rope_bwd(*args, 1e-5)
    assert torch.equal(dqkv, again[0]) and all(a is None or torch.equal(a, b) for a, b in ((dqw, again[1]), (dkw, again[2])))
    got = dqkv.cpu().view(T, -1, d)
    assert torch.equal(got[:, hq + hk:], dv)                              # copied
    x = qkv.double().view(T, -1, d)
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    for gx, a, w, dy, dw in ((got[:, :hq], x[:, :hq], qw, dq, dqw), (got[:, hq:hq + hk], x[:, hq:hq + hk], kw, dk, dkw)):
        a = a.clone().requires_grad_(True)
        w64 = None if w is None else w.double().requires_grad_(True)
        norm_rope64(a, w64, c, s, 1e-5)[0].backward(dy.double())          # the formula's own derivative
        a0 = a.detach()
        mag = (dy.double() * c).abs() + (rot(dy.double() * s)).abs()      # of dz
        if w is None:
            bound = 4 * U32 * mag
        else:
            r = (a0.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
            n = a0 * r
            wz = mag * w.detach().abs().double()
            mean = (wz * n.abs()).mean(-1, keepdim=True)
            bound = (2 * d + 16) * U32 * r * (wz + n.abs() * mean)
            terms = T * gx.shape[1]
            within(dw, w64.grad, rounding(dtype, w64.grad) + (d / 2 + 16 + math.sqrt(terms) * 4) * U32 * (mag * n.abs()).sum((0, 1)))
        within(gx, a.grad, rounding(dtype, a.grad) + bound)


def test_qk_norm_rope_gradient_against_differences(gpu):
    """The module-level form in fp32: directional derivative of a scalar of the outputs against central differences."""
    T, hq, hk, d = 6, 4, 2, 64
    qkv, cos, sin, pos, qw, kw = rotary_case(T, hq, hk, d, torch.float32, "both", 8)
    g = gen(5)
    up = [torch.randn(T, n, d, generator=g) for n in (hq, hk, hk)]

    def value(a, w1, w2):
        x = a.view(T, -1, d)
        c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
        q = norm_rope64(x[:, :hq], w1, c, s, 1e-6)[0]
        k = norm_rope64(x[:, hq:hq + hk], w2, c, s, 1e-6)[0]
        return sum((o * u.double()).sum() for o, u in zip((q, k, x[:, hq + hk:]), up)).item()

    leaf = [t.to(gpu).requires_grad_(True) for t in (qkv, qw, kw)]
    out = mpu.qk_norm_rotary(leaf[0], cos.to(gpu), sin.to(gpu), pos.to(gpu), hq, leaf[1], leaf[2])
    sum((o * u.to(gpu)).sum() for o, u in zip(out, up)).backward()
    dirs = [torch.randn(t.shape, generator=g).double() for t in (qkv, qw, kw)]
    base = [t.double() for t in (qkv, qw, kw)]
    e = 1e-5
    diff = (value(*(b + e * v for b, v in zip(base, dirs))) - value(*(b - e * v for b, v in zip(base, dirs)))) / (2 * e)
    mine = sum((t.grad.double().cpu() * v).sum().item() for t, v in zip(leaf, dirs))
    scale = sum((t.grad.double().cpu() * v).abs().sum().item() for t, v in zip(leaf, dirs))
    # differences: third derivatives times e^2 and the 64-bit rounding of the value over e; gradients: a few hundred U32
    assert abs(mine - diff) < 300 * U32 * scale + 1e-6 * scale


def test_qk_norm_rope_unknown_positions_empty_and_unaligned(gpu):
    T, hq, hk, d = 9, 4, 2, 128
    qkv, cos, sin, pos, qw, kw = rotary_case(T, hq, hk, d, torch.bfloat16, "both", 4)
    pos[2], pos[5], pos[8] = -1, cos.shape[0], 2 ** 40
    bad = [2, 5, 8]
    qkv[2] = float("nan")                                                  # a padded row may hold anything
    mv = lambda t: t.to(gpu)
    q, k = ops.qk_norm_rope(mv(qkv), mv(cos), mv(sin), mv(pos), hq, mv(qw), mv(kw))
    assert not q[bad].any() and not k[bad].any() and not torch.isnan(q).any()
    dq, dk, dv = (torch.randn(T, n, d, generator=gen(1)).bfloat16().to(gpu) for n in (hq, hk, hk))
    dqkv, dqw, dkw = ops.qk_norm_rope_bwd(dq, dk, dv, mv(qkv), mv(cos), mv(sin), mv(pos), mv(qw), mv(kw))
    assert not dqkv.view(T, -1, d)[bad, :hq + hk].any() and torch.isfinite(dqw).all() and torch.isfinite(dkw).all()
    assert torch.equal(dqkv.view(T, -1, d)[:, hq + hk:], dv)
    # gradients that are not there
    some, _, _ = ops.qk_norm_rope_bwd(None, dk, None, mv(qkv), mv(cos), mv(sin), mv(pos), mv(qw), mv(kw), n_q_heads=hq)
    some = some.view(T, -1, d)
    assert not some[:, :hq].any() and not some[:, hq + hk:].any()
    assert torch.equal(some[:, hq:hq + hk], dqkv.view(T, -1, d)[:, hq:hq + hk])
    # no tokens
    q0, k0 = ops.qk_norm_rope(mv(qkv)[:0], mv(cos), mv(sin), mv(pos)[:0], hq, mv(qw), mv(kw))
    assert q0.shape == (0, hq, d) and k0.shape == (0, hk, d)
    e0 = lambda n: torch.zeros(0, n, d, dtype=torch.bfloat16, device=gpu)
    g0, w0, w1 = ops.qk_norm_rope_bwd(e0(hq), e0(hk), e0(hk), mv(qkv)[:0], mv(cos), mv(sin), mv(pos)[:0], mv(qw), mv(kw))
    assert g0.shape == (0, qkv.shape[1]) and not w0.any() and not w1.any()
    # rows of a wider tensor, and a start that is no multiple of 16 bytes: the same numbers
    wide = torch.zeros(T, qkv.shape[1] + 3, dtype=torch.bfloat16, device=gpu)
    wide[:, 3:] = mv(qkv)
    flat = torch.zeros(qkv.numel() + 1, dtype=torch.bfloat16, device=gpu)
    flat[1:] = mv(qkv).view(-1)
    for src in (wide[:, 3:], flat[1:].view(T, -1)):
        q2, k2 = ops.qk_norm_rope(src, mv(cos), mv(sin), mv(pos), hq, mv(qw), mv(kw))
        assert torch.equal(q, q2) and torch.equal(k, k2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,hq,hk,d", ROTARY)
@pytest.mark.parametrize("page", [1, 16, 64])
def test_append_writes_the_slots_and_nothing_else(gpu, dtype, T, hq, hk, d, page):
    qkv, cos, sin, pos, qw, kw = rotary_case(T, hq, hk, d, dtype, "both" if T % 2 else "none", 20 + T)
    pages = -(-T // page) + 3
    g = gen(6)
    slots = torch.randperm(pages * page, generator=g)[:T]
    if T > 4:
        slots[1], slots[2], slots[3], pos[4] = -1, pages * page, 2 ** 41, -5      # nowhere, outside, far outside, no position
    kc0, vc0 = (torch.randn(pages, hk, page, d, generator=g).to(dtype) for _ in range(2))
    kc, vc = kc0.to(gpu), vc0.to(gpu)
    mv = lambda t: None if t is None else t.to(gpu)
    q = ops.qk_norm_rope_append(mv(qkv), mv(cos), mv(sin), mv(pos), mv(slots), kc, vc, hq, mv(qw), mv(kw), 1e-5)
    q1, k1 = ops.qk_norm_rope(mv(qkv), mv(cos), mv(sin), mv(pos), hq, mv(qw), mv(kw), 1e-5)
    assert torch.equal(q, q1)                                             # the training form's numbers
    k1, v = k1.cpu(), qkv.view(T, -1, d)[:, hq + hk:]
    for t in range(T):
        sl = int(slots[t])
        if 0 <= sl < pages * page and 0 <= pos[t] < cos.shape[0]:
            kc0[sl // page, :, sl % page] = k1[t]
            vc0[sl // page, :, sl % page] = v[t]
    assert torch.equal(kc.cpu(), kc0) and torch.equal(vc.cpu(), vc0)


# --------------------------------------------------------------------------- attention
def attn_inputs(R, lens, new, hq, hk, d, page, dtype, seed, extra_pages=2):
    g = gen(seed)
    kv = [a + b for a, b in zip(lens, new)]
    rows = [-(-a // page) for a in kv]
    pages = sum(rows) + extra_pages
    ids = torch.randperm(pages, generator=g).tolist()
    table = torch.full((R, max(rows + [1]) + 1), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(rows):
        table[r, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
        at += n
    kc, vc = (torch.randn(pages, hk, page, d, generator=g).to(dtype) for _ in range(2))
    q = torch.randn(sum(new), hq, d, generator=g).to(dtype)
    cu = torch.tensor([0] + new).cumsum(0)
    return q, kc, vc, table, cu, torch.tensor(kv, dtype=torch.int64)


def attn_reference(q, kc, vc, table, cu, kv, scale):
    """-> values and bounds' ingredients (sum of p |v| / sum p, largest sum of |q k| of a row) in 64 bits"""
    T, hq, d = q.shape
    hk, page = kc.shape[1], kc.shape[2]
    out, mag = torch.zeros(T, hq, d, dtype=torch.float64), torch.zeros(T, hq, d, dtype=torch.float64)
    big = torch.zeros(T, hq, 1, dtype=torch.float64)
    for r in range(len(kv)):
        t0, t1, n_kv = int(cu[r]), int(cu[r + 1]), int(kv[r])
        if t1 == t0 or n_kv == 0:
            continue
        j = torch.arange(n_kv)
        ids = table[r].long()[j // page]
        k = kc[ids, :, j % page].double().repeat_interleave(hq // hk, 1)      # [kv, hq, d]
        v = vc[ids, :, j % page].double().repeat_interleave(hq // hk, 1)
        x = q[t0:t1].double()
        s = torch.einsum("ihd,jhd->hij", x, k) * scale
        seen = j[None, :] <= (n_kv - (t1 - t0) + torch.arange(t1 - t0))[:, None]
        s = s.masked_fill(~seen, -math.inf)
        p = (s - s.amax(-1, keepdim=True).clamp_min(-1e300)).exp()
        p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
        out[t0:t1] = torch.einsum("hij,jhd->ihd", p, v)
        mag[t0:t1] = torch.einsum("hij,jhd->ihd", p, v.abs())
        dots = torch.einsum("ihd,jhd->hij", x.abs(), k.abs()) * scale
        big[t0:t1] = dots.masked_fill(~seen, 0.0).amax(-1).transpose(0, 1)[..., None]
    return out, mag, big


def check_attn(got, case, scale=None):
    q, kc, vc, table, cu, kv = case
    d, dtype = q.shape[2], q.dtype
    scale = d ** -0.5 if scale is None else scale
    ref, mag, big = attn_reference(q, kc, vc, table, cu, kv, scale)
    # the result's rounding; each probability's rounding; scores: d products and sums, the scale, the exponent's argument
    # (a relative error of the score is an absolute one of its exponent), twice for numerator and denominator; sums of
    # the probabilities in fp32.  Half precision loses probabilities below 2^-24 of the largest.
    n = int(kv.max())
    tiny = n * 2.0 ** -25 * float(vc.abs().max()) if dtype == torch.float16 else 0.0
    bound = rounding(dtype, ref) + (half(dtype) + 2 * (d + 8) * U32 * big + 2 * n * U32 + 64 * U32) * mag * 1.02 + tiny
    within(got, ref, bound + 1e-30)


ATTN = [  # lens, new, heads, kv heads, head_dim, page
    ([0], [1], 1, 1, 64, 16),                                 # one token, nothing before it
    ([16], [1], 32, 8, 128, 16),
    ([99, 5, 64, 0, 31], [1] * 5, 32, 8, 128, 16),            # decode
    ([700, 3, 2000], [1] * 3, 8, 1, 128, 64),
    ([300, 20], [1, 1], 7, 7, 64, 32),
    ([130, 1, 515], [5, 5, 5], 32, 8, 128, 32),               # drafts: 20 rows a tile
    ([40, 333], [9, 3], 12, 2, 64, 16),                       # 54 rows: two row blocks
    ([0, 60], [11, 2], 28, 4, 128, 16),                       # 77 rows, a group that does not divide the tile
    ([0], [200], 4, 2, 128, 16),                              # a prompt
    ([70, 0, 1000], [130, 65, 1], 8, 2, 64, 64),              # mixed lengths
    ([17, 900], [33, 300], 12, 12, 64, 128),
    ([255, 256, 257], [64, 63, 65], 8, 1, 128, 16),
    ([5, 0, 9], [0, 40, 0], 4, 4, 128, 16),                   # requests without new tokens
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", range(len(ATTN)))
def test_attn_paged(gpu, dtype, case):
    lens, new, hq, hk, d, page = ATTN[case]
    inputs = attn_inputs(len(lens), lens, new, hq, hk, d, page, dtype, case)
    ws = ops.attn_paged_workspace(gpu)
    dev = [t.to(gpu) for t in inputs]
    a = ops.attn_paged(*dev, workspace=ws, max_new=max(new), len_bound=int(inputs[5].max()))
    check_attn(a, inputs)
    b = ops.attn_paged(*dev, workspace=ws, max_new=max(new), len_bound=int(inputs[5].max()))
    assert torch.equal(a, b)                                   # the same bits on every run
    assert not ws[:4096].any()                                 # counters are left as they were found
    check_attn(ops.attn_paged(*dev, workspace=ws), inputs)     # no bounds from the host: another layout of the work
    check_attn(ops.attn_paged(*dev, max_new=1), inputs)        # a bound that some requests pass


@pytest.mark.parametrize("hq,hk,d,new", [(32, 8, 128, 1), (8, 1, 128, 1), (12, 12, 64, 2), (64, 8, 128, 7), (8, 2, 128, 40)])
def test_attn_paged_is_cut_over_workgroups(gpu, hq, hk, d, new):
    """Long caches beside short ones: a long one is split over many workgroups and merged."""
    lens = [9000, 1, 0, 4100, 17]
    inputs = attn_inputs(5, lens, [new] * 5, hq, hk, d, 16, torch.bfloat16, 40 + hq)
    check_attn(ops.attn_paged(*[t.to(gpu) for t in inputs], max_new=new), inputs)


@pytest.mark.parametrize("new", [1, 3, 100])
@pytest.mark.parametrize("fill", [float("nan"), float("inf"), 3e38])
def test_attn_paged_ignores_what_lies_behind_the_length(gpu, new, fill):
    lens, hq, hk, d, page = [37, 0, 130], 8, 2, 128, 64
    inputs = attn_inputs(3, lens, [new] * 3, hq, hk, d, page, torch.bfloat16, 60)
    q, kc, vc, table, cu, kv = inputs
    used = torch.zeros(kc.shape[0], page, dtype=torch.bool)
    for r in range(3):
        j = torch.arange(int(kv[r]))
        used[table[r].long()[j // page], j % page] = True
    kc2, vc2 = kc.clone(), vc.clone()
    kc2.transpose(1, 2)[~used] = fill
    vc2.transpose(1, 2)[~used] = fill
    dev = lambda *ts: [t.to(gpu) for t in ts]
    a = ops.attn_paged(*dev(q, kc2, vc2, table, cu, kv), max_new=new)
    assert torch.equal(a, ops.attn_paged(*dev(q, kc, vc, table, cu, kv), max_new=new))
    check_attn(a, inputs)


@pytest.mark.parametrize("new", [1, 2, 90])
def test_attn_paged_rows_that_see_nothing_and_rows_of_no_request(gpu, new):
    """Lengths of zero (a refused request) and shorter than the chunk: zeros; rows in front of the first request and
    behind the last one: untouched; lengths and offsets out of range: clamped."""
    hq, hk, d, page = 8, 2, 128, 16
    q, kc, vc, table, cu, kv = attn_inputs(3, [40, 9, 70], [new] * 3, hq, hk, d, page, torch.bfloat16, 61)
    kv = torch.tensor([0, max(new - 1, 0), 70 + new])
    q = torch.cat([q[:2], q, q[:5]])
    cu = cu + 2
    out = torch.full_like(q, 7.0).to(gpu)
    dev = [t.to(gpu) for t in (q, kc, vc, table, cu, kv)]
    assert ops.attn_paged(*dev, max_new=new, out=out) is out
    got = out.cpu()
    rows = slice(2, 2 + 3 * new)
    assert (got[:2] == 7).all() and (got[2 + 3 * new:] == 7).all()
    assert not got[2:2 + new].any() and not got[2 + new].any()           # no tokens; one token less than rows
    ref, _, _ = attn_reference(q[rows], kc, vc, table, cu - 2, kv, d ** -0.5)
    inner = (q[rows], kc, vc, table, cu - 2, kv)
    check_attn(got[rows], inner)
    # a length past the table row, a negative one, offsets past the tensor and running backwards: no access outside
    wild = torch.tensor([10 ** 12, -4, 70 + new], device=gpu)
    back = torch.tensor([2 + new, 2, 10 ** 9, -5], device=gpu)
    for c, l in ((dev[4], wild), (back, dev[5]), (back, wild)):
        ops.attn_paged(*dev[:4], c, l, max_new=new)
    torch.cuda.synchronize()


def test_attn_paged_unknown_pages_read_as_zeros(gpu):
    for new in (1, 80):
        q, kc, vc, table, cu, kv = attn_inputs(1, [50], [new], 4, 2, 128, 16, torch.bfloat16, 62)
        for bad in (-1, kc.shape[0], 2 ** 30, -2 ** 31):
            t2, k2, v2 = table.clone(), torch.cat([kc, torch.zeros_like(kc[:1])]), torch.cat([vc, torch.zeros_like(vc[:1])])
            t2[0, 1] = bad
            t3 = table.clone()
            t3[0, 1] = kc.shape[0]                                       # the page of zeros
            got = ops.attn_paged(*[t.to(gpu) for t in (q, kc, vc, t2, cu, kv)], max_new=new)
            check_attn(got, (q, k2, v2, t3, cu, kv))


def test_attn_paged_softmax_ranges(gpu):
    """One key that takes all, scores of thousands, equal scores, NaN in a query: only its row."""
    for new in (1, 40):
        q, kc, vc, table, cu, kv = attn_inputs(2, [400, 33], [new] * 2, 8, 2, 128, 16, torch.bfloat16, 63)
        q = q * 30
        check_attn(ops.attn_paged(*[t.to(gpu) for t in (q, kc, vc, table, cu, kv)], max_new=new), (q, kc, vc, table, cu, kv))
        zero = torch.zeros_like(q)
        check_attn(ops.attn_paged(*[t.to(gpu) for t in (zero, kc, vc, table, cu, kv)], max_new=new), (zero, kc, vc, table, cu, kv))
        q2 = (q / 30).clone()
        q2[new, 3, 5] = float("nan")
        got = ops.attn_paged(*[t.to(gpu) for t in (q2, kc, vc, table, cu, kv)], max_new=new).cpu()
        assert torch.isnan(got[new, 3]).all()
        got[new, 3] = 0
        assert not torch.isnan(got).any()


def test_attn_paged_offsets_past_32_bits(gpu):
    """A cache of more than 4 GiB: the last pages are reached."""
    hk, page, d = 8, 64, 128
    pages = (2 ** 32) // (hk * page * d * 2) + 40
    kc = torch.zeros(pages, hk, page, d, dtype=torch.bfloat16, device=gpu)
    vc = torch.zeros_like(kc)
    ids = torch.tensor([[pages - 1, 3, pages - 7]], dtype=torch.int32)
    small_k, small_v = (torch.randn(3, hk, page, d, generator=gen(i)).bfloat16() for i in (1, 2))
    for i in range(3):
        kc[int(ids[0, i])] = small_k[i].to(gpu)
        vc[int(ids[0, i])] = small_v[i].to(gpu)
    for new in (1, 60):
        q = torch.randn(new, 16, d, generator=gen(3)).bfloat16()
        cu, kv = torch.tensor([0, new]), torch.tensor([170])
        got = ops.attn_paged(q.to(gpu), kc, vc, ids.to(gpu), cu.to(gpu), kv.to(gpu), max_new=new)
        check_attn(got, (q, small_k, small_v, torch.tensor([[0, 1, 2]], dtype=torch.int32), cu, kv))
    # the append reaches them too
    qkv, cos, sin, pos, qw, kw = rotary_case(1, 8, hk, d, torch.bfloat16, "both", 9)
    slot = torch.tensor([(pages - 2) * page + 11], device=gpu)
    ops.qk_norm_rope_append(qkv.to(gpu), cos.to(gpu), sin.to(gpu), pos.to(gpu), slot, kc, vc, 8, qw.to(gpu), kw.to(gpu))
    assert torch.equal(vc[pages - 2, :, 11].cpu(), qkv.view(-1, d)[8 + hk:])


# --------------------------------------------------------------------------- verification
def verify_reference(drafts, target, draft, u, lens=None):
    R, K = drafts.shape
    V = target.shape[2]
    clean = lambda w: torch.where((w > 0) & (w < math.inf), w, torch.zeros_like(w))
    tokens, counts = torch.full((R, K + 1), -1, dtype=torch.int64), torch.zeros(R, dtype=torch.int64)
    for r in range(R):
        have = K if lens is None else min(max(int(lens[r]), 0), K)
        n = 0
        while n < have:
            x = int(drafts[r, n])
            if not 0 <= x < V:
                break
            q = 1.0 if draft is None else float(draft[r, n, x])
            if not float(u[r, n]) * q < float(target[r, n, x]):
                break
            tokens[r, n] = x
            n += 1
        whole = clean(target[r, n].double())
        w = whole
        if n < have:
            if draft is None:
                w = whole.clone()
                if 0 <= int(drafts[r, n]) < V:
                    w[int(drafts[r, n])] = 0
            else:
                w = clean(target[r, n].double() - draft[r, n].double())
            if w.sum() <= 0:
                w = whole
        cum = w.cumsum(0)
        over = (cum > float(u[r, K]) * cum[-1]) & (w > 0)
        if over.any():
            tokens[r, n] = int(over.nonzero()[0])
        elif (w > 0).any():
            tokens[r, n] = int((w > 0).nonzero()[-1])
        counts[r] = n
    return tokens, counts


def verify_case(R, K, V, dtype, with_draft, seed):
    g = gen(seed)
    logits = torch.randn(R, K + 1, V, generator=g) * 2
    target = torch.softmax(logits, -1).to(dtype)
    guess = torch.softmax(logits[:, :K] + 0.5 * torch.randn(R, K, V, generator=g), -1).to(dtype)
    drafts = torch.multinomial(guess.float().view(-1, V), 1, generator=g).view(R, K) if K else torch.zeros(R, 0, dtype=torch.int64)
    return drafts, target, guess if with_draft else None, torch.rand(R, K + 1, generator=g)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,K,V", [(1, 1, 1), (3, 0, 77), (4, 1, 1000), (70, 4, 333), (5, 7, 50257), (2, 64, 2049), (9, 3, 131100)])
@pytest.mark.parametrize("with_draft", [True, False])
def test_verify_draft(gpu, dtype, R, K, V, with_draft):
    drafts, target, guess, u = verify_case(R, K, V, dtype, with_draft, R + K)
    lens = torch.randint(-1, K + 2, (R,), generator=gen(3)) if R % 2 else None
    mv = lambda t: None if t is None else t.to(gpu)
    tokens, n = ops.verify_draft(mv(drafts), mv(target), mv(guess), mv(u), mv(lens))
    want, count = verify_reference(drafts, target, guess, u, lens)
    assert torch.equal(n.cpu(), count) and torch.equal(tokens.cpu(), want)


def test_verify_draft_edges(gpu):
    """Rows without weight, weights that are no probabilities, drafts outside the vocabulary, uniforms of 0 and 1, all
    accepted, all rejected, target and draft alike."""
    R, K, V = 8, 2, 5000
    drafts, target, guess, u = verify_case(R, K, V, torch.float32, True, 1)
    target[0] = 0                                             # no weight anywhere: -1
    target[1, 0, 100:200] = float("nan")
    target[1, 0, 300] = float("inf")
    target[1, 0, 400:500] = -1.0
    drafts[2, 0], drafts[3, 0] = -1, V
    u[4], u[5] = 0.0, 1.0
    guess[6] = target[6, :K]
    u[6, :K] = 1.0                                            # u q = p: rejected, nothing left over: the target's row
    guess[7] = target[7, :K]
    u[7, :K] = 0.999
    mv = lambda t: None if t is None else t.to(gpu)
    for dp in (guess, None):
        tokens, n = ops.verify_draft(mv(drafts), mv(target), mv(dp), mv(u))
        want, count = verify_reference(drafts, target, dp, u)
        assert torch.equal(n.cpu(), count) and torch.equal(tokens.cpu(), want)
    assert want[0, 0] == -1
    # a single token that holds all the weight, at either end
    one = torch.zeros(2, 1, 70000)
    one[0, 0, 0] = 1e-30
    one[1, 0, 69999] = 1e-30
    none = torch.zeros(2, 0, dtype=torch.int64, device=gpu)
    tokens, _ = ops.verify_draft(none, mv(one), None, torch.full((2, 1), 0.7, device=gpu))
    assert tokens.tolist() == [[0], [69999]]


def test_verify_draft_keeps_the_targets_distribution(gpu):
    """Speculative sampling draws the target's own distribution whatever the draft's: frequencies of the first token over
    20000 requests, against 5 standard deviations of a binomial count."""
    R, V = 20000, 12
    g = gen(11)
    p, q = torch.softmax(torch.randn(V, generator=g), 0), torch.softmax(torch.randn(V, generator=g), 0)
    drafts = torch.multinomial(q.expand(R, V), 1, generator=g)
    target = p.expand(R, 2, V).contiguous()
    tokens, _ = ops.verify_draft(drafts.to(gpu), target.to(gpu), q.expand(R, 1, V).contiguous().to(gpu),
                                 torch.rand(R, 2, generator=g).to(gpu))
    count = torch.bincount(tokens[:, 0].cpu(), minlength=V).double()
    want = p.double() / p.double().sum() * R
    assert ((count - want).abs() < 5 * (want * (1 - want / R)).sqrt()).all()


# --------------------------------------------------------------------------- streams, graphs, refusals
def test_on_another_stream_and_in_a_graph(gpu):
    """A step captured once and replayed with other lengths, eager work and synchronisation between the replays."""
    R, hq, hk, d, page, pages = 4, 8, 2, 128, 16, 64
    g = gen(12)
    cos, sin = (t.float().to(gpu) for t in tables(d, 600, 2))
    w = torch.ones(d, dtype=torch.bfloat16, device=gpu)
    kc, vc = (torch.randn(pages, hk, page, d, generator=g).bfloat16().to(gpu) for _ in range(2))
    lens = torch.tensor([5, 100, 0, 33], device=gpu)
    new = torch.ones(R, dtype=torch.int64, device=gpu)
    held = ((lens + page - 1) // page).int()
    table = torch.full((R, 40), -1, dtype=torch.int32, device=gpu)
    ids = torch.randperm(pages, generator=g).int()
    at = 0
    for r, h in enumerate(held.tolist()):
        table[r, :h] = ids[at:at + h].to(gpu)
        at += h
    free = ids[at:].contiguous().to(gpu)
    count = torch.tensor([free.numel()], dtype=torch.int32, device=gpu)
    qkv = torch.zeros(R, (hq + 2 * hk) * d, dtype=torch.bfloat16, device=gpu)
    ws = ops.attn_paged_workspace(gpu)
    start = [t.clone() for t in (lens, held, table, count, kc, vc)]

    def step(workspace):
        plan = ops.paged_plan(lens, new, held, table, free, count, page, R)
        q = ops.qk_norm_rope_append(qkv, cos, sin, plan.positions, plan.slots, kc, vc, hq, w, w)
        out = ops.attn_paged(q, kc, vc, table, plan.cu, plan.kv_lens, max_new=1, workspace=workspace)
        held.copy_(plan.held)
        count.copy_(plan.free_count)
        lens.add_(new)
        return out

    rows = [torch.randn(qkv.shape, generator=g).bfloat16().to(gpu) for _ in range(20)]

    def restore():
        for t, s in zip((lens, held, table, count, kc, vc), start):
            t.copy_(s)

    eager = []
    for x in rows:
        qkv.copy_(x)
        eager.append(step(None).clone())
    final = [t.clone() for t in (lens, held, table, count, kc, vc)]
    side = torch.cuda.Stream(gpu)
    restore()
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        for x, want in zip(rows, eager):
            qkv.copy_(x)
            assert torch.equal(step(ws), want)
    torch.cuda.current_stream(gpu).wait_stream(side)
    restore()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(ws)
    restore()
    for x, want in zip(rows, eager):
        qkv.copy_(x)
        graph.replay()
        junk = torch.randn(1000, device=gpu).sum().item()                # the program's own work between replays
        assert junk == junk and torch.equal(out, want)
    for t, want in zip((lens, held, table, count, kc, vc), final):
        assert torch.equal(t, want)


def test_gradients_of_shared_heads_and_module_form(gpu):
    """bf16 module form: q, k and a view of the values come out, one gradient for the fused rows goes in; the values'
    part is exactly what arrived."""
    B, S, hq, hk, d = 2, 17, 8, 2, 128
    qkv, cos, sin, pos, qw, kw = rotary_case(B * S, hq, hk, d, torch.bfloat16, "both", 30)
    x = qkv.to(gpu).view(B, S, -1).requires_grad_(True)
    w1, w2 = (w.to(gpu).requires_grad_(True) for w in (qw, kw))
    q, k, v = mpu.qk_norm_rotary(x, cos.to(gpu), sin.to(gpu), pos.to(gpu).view(B, S), hq, w1, w2, eps=1e-5)
    assert q.shape == (B, S, hq, d) and k.shape == v.shape == (B, S, hk, d)
    up = [torch.randn(t.shape, generator=gen(2)).bfloat16().to(gpu) for t in (q, k, v)]
    torch.autograd.backward([q, k, v], up)
    flat = [u.view(B * S, -1, d) for u in up]
    want = ops.qk_norm_rope_bwd(*flat, qkv.to(gpu), cos.to(gpu), sin.to(gpu), pos.to(gpu), qw.to(gpu), kw.to(gpu), 1e-5)
    assert torch.equal(x.grad.view(B * S, -1), want[0]) and torch.equal(w1.grad, want[1]) and torch.equal(w2.grad, want[2])
    # a weight that takes no gradient, values that are not used
    x2 = qkv.to(gpu).requires_grad_(True)
    q, k, v = mpu.qk_norm_rotary(x2, cos.to(gpu), sin.to(gpu), pos.to(gpu), hq, qw.to(gpu), None, eps=1e-5)
    q.float().sum().backward()
    g2 = x2.grad.view(B * S, -1, d)
    assert g2[:, :hq].any() and not g2[:, hq:].any()


def test_refusals(gpu):
    q, kc, vc, table, cu, kv = (t.to(gpu) for t in attn_inputs(2, [20, 3], [1, 1], 4, 2, 128, 16, torch.bfloat16, 1))
    for bad in (dict(q=q.half()), dict(q=q[:, :3]), dict(cu=cu[:-1]), dict(kv_lens=kv.int()), dict(block_tables=table.long()),
                dict(k_cache=kc.transpose(0, 1)), dict(k_cache=kc[:, :1]), dict(out=torch.empty(3, 4, 128, device=gpu))):
        args = dict(q=q, k_cache=kc, v_cache=vc, block_tables=table, cu=cu, kv_lens=kv)
        args.update(bad)
        with pytest.raises(ValueError):
            ops.attn_paged(**args)
    with pytest.raises(RuntimeError, match="workspace"):
        ops.attn_paged(q, kc, vc, table, cu, kv, workspace=torch.zeros(4096, dtype=torch.uint8, device=gpu))
    with pytest.raises(RuntimeError, match="scale"):
        ops.attn_paged(q, kc, vc, table, cu, kv, scale=0.0)
    with pytest.raises(RuntimeError, match="MI355X"):
        ops.attn_paged(q.cpu(), kc, vc, table, cu, kv)
    qkv, cos, sin, pos, qw, kw = (t.to(gpu) for t in rotary_case(3, 4, 2, 128, torch.bfloat16, "both", 2))
    with pytest.raises(ValueError):
        ops.qk_norm_rope(qkv, cos, sin, pos[:2], 4, qw, kw)
    with pytest.raises(ValueError):
        ops.qk_norm_rope(qkv, cos, sin, pos, 5, qw, kw)
    with pytest.raises(ValueError):
        ops.qk_norm_rope(qkv, cos, sin, pos, 4, qw[:-1], kw)
    with pytest.raises(TypeError):
        ops.qk_norm_rope(qkv, cos.half(), sin.half(), pos, 4, qw, kw)
    with pytest.raises(ValueError):
        ops.qk_norm_rope_append(qkv, cos, sin, pos, pos.int(), kc, vc, 4, qw, kw)
    drafts, target, guess, u = (t.to(gpu) for t in verify_case(2, 3, 50, torch.float32, True, 1))
    for bad in ((drafts, target[:, :3], guess, u), (drafts, target, guess.half(), u), (drafts, target, guess, u[:, :3]),
                (drafts.int(), target, guess, u)):
        with pytest.raises(ValueError):
            ops.verify_draft(*bad)
