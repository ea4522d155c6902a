"""``moe::topk_router`` and ``moe::topk_router_backward`` called as operators: they refuse what the kernels would read or write out of
range for, before anything touches a GPU, and lay out what is strided."""
import pytest
import torch

from triton_grouped_gemm_amd import ops  # registers the operators


def refused(word, call, *args):
    with pytest.raises(ValueError, match=word):
        call(*args)


def test_forward():
    call, x = torch.ops.moe.topk_router, torch.zeros(4, 16)
    refused("tokens, experts", call, x[0], 2, 0, True)
    refused("tokens, experts", call, x.double(), 2, 0, True)
    refused("tokens, experts", call, x.int(), 2, 0, True)
    refused("number of experts", call, torch.zeros(4, 1025), 2, 0, True)
    refused("number of experts", call, torch.zeros(4, 0), 1, 0, True)
    for topk in (0, -1, 17, 65, (1 << 32) + 2):  # the last one is 2 in 32 bits
        refused("topk", call, x, topk, 0, True)
    refused("topk", call, torch.zeros(4, 128), 65, 0, True)
    for scoring in (-1, 2, 1 << 32):
        refused("scoring", call, x, 2, scoring, True)
    with pytest.raises(AssertionError, match="GPU"):
        call(x, 2, 0, True)


def test_backward():
    call = torch.ops.moe.topk_router_backward
    x, probs, indices, grad = torch.zeros(4, 16), torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)
    refused("grad", call, x, probs, indices, grad[:3], 0, True)
    refused("grad", call, x, probs, indices, grad[:, :1], 0, True)
    refused("grad", call, x, probs, indices, grad.int(), 0, True)
    refused("indices", call, x, probs, indices[:3], grad, 0, True)
    refused("indices", call, x, probs, indices.long(), grad, 0, True)
    refused("probs", call, x, probs[:3], indices[:3], grad[:3], 0, True)
    refused("probs", call, x, probs.double(), indices, grad, 0, True)
    refused("probs", call, x, probs[0], indices, grad, 0, True)
    refused("topk", call, x[:, :1], probs, indices, grad, 0, True)
    refused("tokens, experts", call, x.double(), probs, indices, grad, 0, True)
    refused("scoring", call, x, probs, indices, grad, 2, True)
    with pytest.raises(AssertionError, match="GPU"):
        call(x, probs, indices, grad, 0, True)


def test_the_entry_point():
    refused("scoring must be one of", ops.topk_router, torch.zeros(4, 16), 2, "tanh")
    refused("topk", ops.topk_router, torch.zeros(4, 16), 17)
    refused("number of experts", ops.topk_router, torch.zeros(4, 1025), 2)


@pytest.mark.gpu
def test_strided_operands(dev):
    x = torch.randn(6, 40, generator=torch.Generator().manual_seed(1)).to(dev)
    grad = torch.randn(6, 3, generator=torch.Generator().manual_seed(2)).to(dev)
    flip = lambda t: t.t().contiguous().t()
    for scoring in (0, 1):
        for renormalize in (False, True):
            probs, indices = torch.ops.moe.topk_router(x, 3, scoring, renormalize)
            again = torch.ops.moe.topk_router(flip(x), 3, scoring, renormalize)
            assert torch.equal(probs, again[0]) and torch.equal(indices, again[1])
            first = torch.ops.moe.topk_router(x[:1].expand(6, 40), 3, scoring, renormalize)
            assert torch.equal(first[0], probs[:1].expand(6, 3)) and torch.equal(first[1], indices[:1].expand(6, 3))
            want = torch.ops.moe.topk_router_backward(x, probs, indices, grad, scoring, renormalize)
            got = torch.ops.moe.topk_router_backward(flip(x), flip(probs), flip(indices), flip(grad).double(), scoring, renormalize)
            assert torch.equal(got, want)
    refused("one GPU", torch.ops.moe.topk_router_backward, x, probs, indices, grad.cpu(), 0, True)
