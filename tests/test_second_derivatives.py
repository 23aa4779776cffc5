"""Backward passes run kernels that autograd cannot look into: a second derivative is refused, not silently left out."""
import pytest
import torch

from merak_amd import mpu


def cases(gpu):
    g = torch.Generator().manual_seed(70)
    rnd = lambda *s: torch.randn(*s, generator=g).to(gpu)
    layer = mpu.ColumnParallelLinear(64, 96, gather_output=False).to(gpu)
    table = mpu.VocabParallelEmbedding(50, 64).to(gpu)
    ids = torch.randint(0, 50, (7,), generator=g).to(gpu)
    cos, sin, pos = rnd(9, 64), rnd(9, 64), torch.randint(0, 9, (7,), generator=g).to(gpu)
    head = rnd(50, 64).requires_grad_(True)
    leaf = lambda *s: rnd(*s).requires_grad_(True)
    x = leaf(7, 64)
    yield "linear", x, lambda: layer(x)[0].square().sum()
    yield "embedding", table.weight, lambda: table(ids).square().sum()
    y = leaf(7, 50)
    for kw in ({}, dict(materialize_softmax=True), dict(fused_backward_scale=1.0)):
        yield f"cross entropy {kw}", y, lambda kw=kw: mpu.vocab_parallel_cross_entropy(y * 1.0, ids, **kw).sum()
    yield "LM head", x, lambda: mpu.lm_head_cross_entropy(x, head, ids, loss_scale=7.0).sum()
    qkv, w = leaf(7, 3 * 64), [leaf(64), leaf(64)]
    yield "rotary", qkv, lambda: sum(t.square().sum() for t in mpu.qk_norm_rotary(qkv, cos, sin, pos, 1, *w))


@pytest.mark.gpu
def test_second_derivatives_are_refused(gpu):
    names = []
    for name, leaf, value in cases(gpu):
        (want,) = torch.autograd.grad(value(), leaf)
        (got,) = torch.autograd.grad(value(), leaf, create_graph=True)
        assert torch.equal(want, got.detach()), name
        assert got.requires_grad, name                  # not a constant
        try:
            got.square().sum().backward()
        except RuntimeError as e:
            assert "second derivative" in str(e), (name, e)
            names.append(name)
    assert len(names) == 7, names
