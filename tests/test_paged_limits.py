"""The paged-cache operators at the ends of their ranges: long flat tails of small probabilities, the largest sizes, no
tokens at all.  Against plain implementations in 64 bits; the size checks through the C ABI on a machine without a GPU."""
import math

import pytest
import torch

from merak_amd import ops

U32 = 2.0 ** -24


def gen(seed):
    return torch.Generator().manual_seed(31000 + seed)


# --------------------------------------------------------------------------- probabilities far below the largest
# f16: weights are held as 2^11 p and round below 2^-14 to multiples of 2^-24, so each is off by at most half of
# 2^-24 2^-11 = 2^-36 of the largest (the maximum that the kernel subtracts may lag: then by less), besides 2^-11 of
# itself.  Relative to the largest weight the numerator is off by sum |v| of those; the sums of n fp32 terms by
# n 2^-24 of their magnitudes; the result is rounded once.
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,hq,new", [(64, 1, 1), (128, 8, 1), (128, 12, 5), (64, 2, 80)])     # one row block, two, wide
@pytest.mark.parametrize("requests", [256, 1])                        # a tile for each workgroup; one cut over all of them
@pytest.mark.parametrize("log2p", [-18.0, math.log2(1.49) - 24, -25.1, -30.0])
def test_attn_paged_keeps_a_flat_tail(gpu, dtype, d, hq, new, requests, log2p):
    """Eight keys with score 0 and values of 0 at the start (every wave of a workgroup meets one), then 131000 keys that
    are all 2^log2p of them with values of 1 (of 1 and -1 in every second dimension): the result is the tail's share of
    the mass.  The requests share their pages."""
    n, page, top = 131072 - 7, 64, 8
    pages = -(-n // page)
    x = torch.tensor(-log2p * math.log(2.0)).to(dtype).double().item()    # the score of a tail key is -x exactly
    k = torch.zeros(pages * page, d, dtype=dtype, device=gpu)
    v = torch.ones(pages * page, d, dtype=dtype, device=gpu)
    v[1::2, 1::2] = -1.0
    k[:, 0] = -x
    k[0:32 * top:32], v[0:32 * top:32] = 0.0, 0.0
    shape = lambda t: t.view(pages, 1, page, d)
    q = torch.zeros(requests * new, hq, d, dtype=dtype, device=gpu)
    q[:, :, 0] = 1.0
    got = ops.attn_paged(q, shape(k), shape(v), torch.arange(pages, dtype=torch.int32, device=gpu).repeat(requests, 1),
                         torch.arange(requests + 1, device=gpu) * new, torch.full((requests,), n, device=gpu), scale=1.0,
                         max_new=new)
    got = got.double().cpu().view(requests, new, hq, d)
    keys = torch.arange(n - new + 1, n + 1, dtype=torch.float64)          # seen by each row
    odd = (keys / 2).floor()
    even = keys - odd - top                                               # of the tail
    tail = math.exp(-x)
    total = top + (even + odd) * tail
    mass = ((even + odd) * tail / total)[:, None, None]
    ref = torch.empty(new, 1, d, dtype=torch.float64)
    ref[..., 0::2] = mass
    ref[..., 1::2] = ((even - odd) * tail / total)[:, None, None]
    half = torch.finfo(dtype).eps / 2
    tiny = float(keys.max()) * 2.0 ** -36 / top if dtype == torch.float16 else 0.0
    step = torch.finfo(dtype).smallest_normal * half                      # of results below the smallest normal number
    # numerator and denominator share each weight's rounding, which is the same for all of the tail
    bound = half * ref.abs() * 1.01 + step + half * mass * 1.02 + 2 * tiny + (2 * n + 64 + 8 * x) * U32 * mass
    ratio = (got - ref).abs() / bound
    assert not torch.isnan(got).any() and ratio.max() <= 1, (float(ratio.max()), got[0, 0, 0, :2], ref[0, 0, :2])


# --------------------------------------------------------------------------- the most tokens of a call
def test_qk_norm_rope_token_limit():
    """2^21 rows are taken, one more is not (the null pointer is what a call of 2^21 is refused for here)."""
    from merak_amd import _lib
    lib, A = _lib.lib(), 4096
    calls = (lambda T: lib.mtp_qk_norm_rope(None, A, A, 0, A, None, None, A, A, T, 1, 1, 64, 10, 1e-6, 1, None),
             lambda T: lib.mtp_qk_norm_rope_append(None, A, A, 0, A, A, None, None, A, A, A, T, 1, 1, 64, 10, 4, 16, 1e-6, 1, None),
             lambda T: lib.mtp_qk_norm_rope_bwd(A, A, A, None, A, A, 0, A, None, None, A, None, None, None, 0, T, 1, 1, 64, 10,
                                                1e-6, 1, None))
    for call in calls:
        assert call(2 ** 21) == -1 and b"null" in lib.mtp_last_error()
        assert call(2 ** 21 + 1) == -2 and b"2^21" in lib.mtp_last_error()


@pytest.mark.gpu
def test_qk_norm_rope_of_the_most_tokens(gpu):
    """2^21 rows, forward and backward: the last rows equal those of a small call on the same data."""
    T, d, few = 2 ** 21, 64, 300
    qkv = torch.randn(few, 3 * d, generator=gen(1)).half().to(gpu)
    cos, sin = (torch.randn(50, d, generator=gen(i)).to(gpu) for i in (2, 3))
    pos = torch.randint(0, 50, (few,), generator=gen(4)).to(gpu)
    w = (torch.rand(d, generator=gen(5)) + 0.5).half().to(gpu)
    up = [torch.randn(few, 1, d, generator=gen(6 + i)).half().to(gpu) for i in range(3)]
    big = lambda t: torch.cat([torch.zeros((T - few, *t.shape[1:]), dtype=t.dtype, device=gpu), t])
    q, k = ops.qk_norm_rope(big(qkv), cos, sin, big(pos), 1, w, w)
    q1, k1 = ops.qk_norm_rope(qkv, cos, sin, pos, 1, w, w)
    assert torch.equal(q[-few:], q1) and torch.equal(k[-few:], k1) and not q[:-few].any()
    dqkv, dqw, dkw = ops.qk_norm_rope_bwd(*[big(u) for u in up], big(qkv), cos, sin, big(pos), w, w)
    d1, w1, w2 = ops.qk_norm_rope_bwd(*up, qkv, cos, sin, pos, w, w)
    assert torch.equal(dqkv[-few:], d1) and not dqkv[:-few].any()
    # the same terms, added up in another order: 2^-11 for the result's rounding on either side and the fp32 sums' own
    for a, b in ((dqw, w1), (dkw, w2)):
        assert ((a.double() - b.double()).abs() <= 2 * 2.0 ** -11 * b.double().abs() * 1.01 + 1e-3).all()


# --------------------------------------------------------------------------- sizes whose product passes 64 bits
def test_products_of_sizes_do_not_wrap():
    """page_size * max_pages and tokens * heads of 2^64: refused like every product past the limit (a wrapped one is 0)."""
    from merak_amd import _lib
    lib, A = _lib.lib(), 4096
    plan = lambda pages, page: lib.mtp_paged_plan(*(A,) * 11, A + 64, A + 64, 2, pages, page, 8, 3, None)
    attn = lambda T: lib.mtp_attn_paged(*(A,) * 8, lib.mtp_attn_paged_workspace_bytes(), T, 2, 8, 2, 128, 9, 16, 4, 1, 64, 0.1, 1,
                                        None)
    for pages, page in ((4, 2 ** 62), (2 ** 30, 2 ** 34), (2, 2 ** 62), (1, 2 ** 62), (2, 2 ** 30)):
        assert plan(pages, page) == -1 and b"power of two" in lib.mtp_last_error(), (pages, page)
    for T in (2 ** 61, 2 ** 62, 2 ** 27):
        assert attn(T) == -1 and b"T=" in lib.mtp_last_error(), T


# --------------------------------------------------------------------------- lengths next to 2^31
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,new", [(torch.bfloat16, 1), (torch.float16, 5), (torch.bfloat16, 70)])
def test_attn_paged_length_next_to_2_31(gpu, dtype, new):
    """A table row of 2^27 - 1 pages of 16 tokens of which only the last is in the cache: 2^31 - 32 tokens read as zeros
    (score 0, weight 1, value 0), 16 have scores about 22, with which their weights are of the size of that mass."""
    page, d, rows = 16, 64, 2 ** 27 - 1
    kv = page * rows
    table = torch.full((1, rows), -1, dtype=torch.int32, device=gpu)
    table[0, -1] = 0
    k = torch.zeros(1, 1, page, d, dtype=dtype)
    k[0, 0, :, 0] = 20 + torch.arange(page) * 0.125                       # exact in both types
    v = torch.randn(1, 1, page, d, generator=gen(20)).to(dtype)
    q = torch.zeros(new, 1, d, dtype=dtype)
    q[:, :, 0] = 1.0
    got = ops.attn_paged(q.to(gpu), k.to(gpu), v.to(gpu), table, torch.tensor([0, new], device=gpu),
                         torch.tensor([kv], device=gpu), scale=1.0, max_new=new).double().cpu()[:, 0]
    seen = torch.arange(kv - new + 1, kv + 1)                             # tokens of each row
    real = (seen - (kv - page)).clamp_min(0)                              # of the last page
    w = torch.exp(k[0, 0, :, 0].double()) * (torch.arange(page)[None] < real[:, None])
    total = (seen - real).double()[:, None] + w.sum(1, keepdim=True)
    ref, mag = w @ v[0, 0].double() / total, w @ v[0, 0].double().abs() / total
    half = torch.finfo(dtype).eps / 2
    # the 2^31 ones add up exactly in a lane (2^22 of them), and in fp32 over 2048 waves and their merges; the weights are
    # rounded once each, the exponent's argument is off by 3 2^-24 of 23 log2(e)
    bound = half * ref.abs() * 1.01 + torch.finfo(dtype).smallest_normal * half + (half + (2 * 2048 + 256) * U32) * 1.02 * mag
    ratio = ((got - ref).abs() / bound.clamp_min(1e-30)).max()
    assert not torch.isnan(got).any() and ratio <= 1, float(ratio)


# --------------------------------------------------------------------------- no tokens
@pytest.mark.gpu
@pytest.mark.parametrize("lead", [(0,), (0, 7), (3, 0)])
def test_qk_norm_rotary_of_no_tokens(gpu, lead):
    """An empty batch or sequence: empty heads, an empty gradient and weight gradients of zero."""
    from merak_amd import mpu
    d, hq, hk = 64, 4, 2
    x = torch.zeros(*lead, (hq + 2 * hk) * d, dtype=torch.bfloat16, device=gpu, requires_grad=True)
    w = [torch.ones(d, dtype=torch.bfloat16, device=gpu, requires_grad=True) for _ in range(2)]
    table = torch.ones(5, d, device=gpu)
    q, k, v = mpu.qk_norm_rotary(x, table, table, torch.zeros(lead, dtype=torch.int64, device=gpu), hq, *w)
    assert q.shape == (*lead, hq, d) and k.shape == v.shape == (*lead, hk, d)
    (q.sum() + k.sum() + v.sum()).backward()
    assert x.grad.shape == x.shape and all(t.grad.shape == (d,) and not t.grad.any() for t in w)


# --------------------------------------------------------------------------- memory that a call writes
@pytest.mark.gpu
def test_attn_paged_refuses_a_strided_workspace(gpu):
    """Every second byte of a buffer: as many elements as the call needs, but the bytes between are not its own."""
    need = ops.attn_paged_workspace(gpu).numel()
    k = torch.zeros(1, 1, 16, 64, dtype=torch.bfloat16, device=gpu)
    args = (torch.zeros(1, 1, 64, dtype=torch.bfloat16, device=gpu), k, k, torch.zeros(1, 1, dtype=torch.int32, device=gpu),
            torch.tensor([0, 1], device=gpu), torch.tensor([3], device=gpu))
    with pytest.raises(ValueError, match="workspace"):
        ops.attn_paged(*args, workspace=torch.zeros(2 * need, dtype=torch.uint8, device=gpu)[::2])
    ops.attn_paged(*args, workspace=torch.zeros(need + 64, dtype=torch.uint8, device=gpu)[64:])
