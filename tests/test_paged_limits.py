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
