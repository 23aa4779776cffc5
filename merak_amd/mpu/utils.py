"""Helpers of the model-parallel layers (integers: Merak/core/mpu/utils.py:33-64,90-106)."""
from __future__ import annotations

import functools

import torch


def ensure_divisibility(numerator, denominator):
    """Assert that numerator is divisible by the denominator (utils.py:33-36)."""
    assert numerator % denominator == 0, '{} is not divisible by {}'.format(numerator, denominator)


def divide(numerator, denominator):
    """Checked integer division (utils.py:39-43)."""
    ensure_divisibility(numerator, denominator)
    return numerator // denominator


def split_tensor_along_last_dim(tensor, num_partitions, contiguous_split_chunks=False):
    """Equal views along the last dimension (utils.py:46-64)."""
    last_dim = tensor.dim() - 1
    last_dim_size = divide(tensor.size()[last_dim], num_partitions)
    tensor_list = torch.split(tensor, last_dim_size, dim=last_dim)
    if contiguous_split_chunks:
        return tuple(chunk.contiguous() for chunk in tensor_list)
    return tensor_list


class VocabUtility:
    """[first, last) vocabulary range owned by ``rank`` (utils.py:90-106)."""

    @staticmethod
    def vocab_range_from_per_partition_vocab_size(per_partition_vocab_size, rank, world_size):
        index_f = rank * per_partition_vocab_size
        index_l = index_f + per_partition_vocab_size
        return index_f, index_l

    @staticmethod
    def vocab_range_from_global_vocab_size(global_vocab_size, rank, world_size):
        per_partition_vocab_size = divide(global_vocab_size, world_size)
        return VocabUtility.vocab_range_from_per_partition_vocab_size(per_partition_vocab_size, rank, world_size)


class _NoFurtherDerivative(torch.autograd.Function):

    @staticmethod
    def forward(ctx, grad):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, grad):
        raise RuntimeError("second derivative of a function whose backward pass runs kernels autograd cannot look into")


def first_derivative_only(backward):
    """For the ``backward`` of an autograd function that calls kernels: with ``create_graph`` its results would look like
    constants to autograd and the second derivative's terms through them would be left out; they raise instead.  (torch's
    ``once_differentiable`` does so only where the incoming gradient has a graph, which that of a plain ``loss.sum()`` has
    not.)"""

    @functools.wraps(backward)
    def wrapped(ctx, *grads):
        if not torch.is_grad_enabled():      # the usual backward pass: nothing to add
            return backward(ctx, *grads)
        with torch.no_grad():
            out = backward(ctx, *grads)
        mark = lambda t: None if t is None else _NoFurtherDerivative.apply(t.detach().requires_grad_(True))
        return tuple(map(mark, out)) if isinstance(out, tuple) else mark(out)

    return wrapped
