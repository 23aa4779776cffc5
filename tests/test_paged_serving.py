"""The paged decoder as a server uses it: requests that end at the longest length, idle slots, refused requests, drafts of
different lengths, calls that fail, models from the library."""
import pytest
import torch

from merak_amd import ops
from merak_amd.inference import PagedLlamaDecoder
from test_paged_decode import D, H, NKV, NQ, V, forward_fp32, model, on, rel


def gen(seed):
    return torch.Generator().manual_seed(52000 + seed)


def decoder(m, **kw):
    args = dict(max_len=128, slots=3, page_size=16)
    args.update(kw)
    return PagedLlamaDecoder(m[0], m[1], m[2], m[3], NQ, NKV, D, **args)


@pytest.mark.gpu
@pytest.mark.parametrize("max_len,page_size", [(100, 64), (33, 32), (17, 16), (64, 16)])
def test_a_request_ends_at_max_len(gpu, max_len, page_size):
    """The last page may have room behind max_len: a token there is refused like one that finds no page, whether it comes
    alone or with others, and the request goes on with what still fits.  bf16 activations: 2e-2 norm-wise, as for the
    other tests of this decoder."""
    m = model(gpu, 5)
    text = torch.randint(0, V, (2, max_len), generator=gen(max_len))
    want = [forward_fp32(m, t) for t in text]
    dec = decoder(on(gpu, m), max_len=max_len, page_size=page_size, slots=2)
    for c in dec.k_cache + dec.v_cache:
        c.fill_(50.0)                                    # what a released request may have left
    full = max_len - 2
    out = dec.append(torch.cat([text[0, :full], text[1, :3]]).to(gpu), [full, 3])
    assert dec.granted.all() and rel(out[:full], want[0][:full]) < 2e-2
    free = dec.free_count.item()
    out = dec.append(torch.cat([text[0, :3], text[1, 3:4]]).to(gpu), [3, 1])          # one token too many
    assert dec.granted.tolist() == [False, True] and dec.lens.tolist() == [full, 4]
    assert rel(out[3:], want[1][3:4]) < 2e-2
    out = dec.append(text[0, full:].to(gpu), [2, 0])
    assert dec.granted.all() and dec.lens.tolist() == [max_len, 4] and rel(out, want[0][full:]) < 2e-2
    dec.append(torch.cat([text[0, :1], text[1, 4:5]]).to(gpu), [1, 1])
    assert dec.granted.tolist() == [False, True] and dec.lens.tolist() == [max_len, 5]
    dec.append(text[0, :1].to(gpu), [1, 0])
    assert dec.granted.tolist() == [False, True] and dec.lens.tolist() == [max_len, 5]
    assert dec.held[0].item() == -(-max_len // page_size) and dec.free_count.item() <= free
