"""CPU tests of the operators around the linear path where they meet torch: tracing, gradients, a torch build without the eager
calls' module.  Nothing is launched."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import gguf_hip

BF = torch.bfloat16


def _fake(shape, dtype=BF):
    return torch.empty(shape, dtype=dtype, device="cuda")


def test_copy_pages_of_a_fake_cache():
    """Fake tensors get the refusals of the layout and of the pairs, and nothing else happens."""
    with FakeTensorMode():
        pages = _fake((3, 9, 16, 64))
        version = pages._version
        assert gguf_hip.copy_pages(pages, [0, 0], [1, 2], dim=1) is None and pages._version > version
        gguf_hip.copy_pages(pages, [], [], dim=-3)
        gguf_hip.copy_pages(_fake((0, 9, 16)), [0], [1], dim=1)
        for src, dst in (([0], [9]), ([-1], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0], [1, 2]), ([2 ** 40], [0]), ([0.5], [1])):
            with pytest.raises(ValueError):
                gguf_hip.copy_pages(pages, src, dst, dim=1)
        for bad, dim in ((pages.transpose(2, 3), 1), (pages[:, :, :, ::2], 1), (pages[:, ::2], 2), (pages, 4)):
            with pytest.raises(ValueError):
                gguf_hip.copy_pages(bad, [0], [1], dim=dim)


def test_make_fx_traces_the_copy():
    """A traced fork holds the copy as one call, which the trace does not make."""
    from torch.fx.experimental.proxy_tensor import make_fx

    def fork(pages):
        gguf_hip.copy_pages(pages, [3, 4], [7, 8], dim=1)
        return pages[:, 7].clone()

    with FakeTensorMode():
        g = make_fx(fork)(_fake((3, 9, 16, 64)))
    calls = [n for n in g.graph.nodes if n.op == "call_function"]
    assert calls[0].target == torch.ops.gguf_hip.copy_pages.default and calls[0].args[1:] == ([3, 4], [7, 8], 1), g.code
