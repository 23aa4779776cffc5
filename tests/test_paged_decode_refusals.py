"""What the paged decoder refuses before it touches a device: sizes that a step would refuse only after pages have been
handed out."""
import pytest
import torch

from merak_amd.inference import PagedLlamaDecoder
from merak_amd.inference.llama_decode import LlamaBlockWeights


def build(dtype=torch.bfloat16, heads=(4, 2), head_dim=64, weights_dim=64, norm=None, **kw):
    nq, nk = heads
    w = lambda *s: torch.zeros(*s, dtype=dtype)
    block = LlamaBlockWeights(w(128), w((4 + 2 * 2) * weights_dim, 128), w(128, 4 * weights_dim), w(128), w(512, 128), w(128, 256))
    return PagedLlamaDecoder(w(50, 128), [block], w(128), w(50, 128), nq, nk, head_dim, k_norms=None if norm is None else [norm],
                             **kw)


@pytest.mark.parametrize("page_size", [0, 1, 8, 24, 48, -16])
def test_page_sizes(page_size):
    with pytest.raises(ValueError, match="page_size"):
        build(page_size=page_size)


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=torch.float32), "head_dim"), (dict(head_dim=96), "head_dim"), (dict(heads=(4, 3)), "key heads"),
    (dict(heads=(4, 0)), "key heads"), (dict(max_len=0), "max_len"), (dict(slots=0), "slots"), (dict(slots=4097), "slots"),
    (dict(n_pages=0), "n_pages"), (dict(head_dim=128), "block 0"), (dict(heads=(8, 2)), "block 0"),
    (dict(norm=torch.ones(128, dtype=torch.bfloat16)), "head norms"), (dict(norm=torch.ones(64)), "head norms")])
def test_sizes_and_types(kw, match):
    with pytest.raises(ValueError, match=match):
        build(**kw)
