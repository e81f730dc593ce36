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


def _calls():
    """Of each operator: the call, its tensors that can belong to a graph, its results."""
    lo = dict(y=_fake((4, 48)), x=_fake((4, 64)), a=_fake((3, 2, 16, 64)), b=_fake((3, 48, 16)), ids=_fake((4,), torch.int32),
              scales=_fake((3,), torch.float32), n_outs=[32, 16])
    at = dict(q=_fake((3, 8, 64)), k_pages=_fake((9, 16, 2, 64)), v_pages=_fake((9, 16, 2, 64)),
              block_table=_fake((3, 4), torch.int32), lengths=_fake((3,), torch.int32), return_lse=True)
    ro = dict(q=_fake((5, 8, 64)), k=_fake((5, 2, 64)), positions=_fake((5,), torch.int64), table=_fake((100, 32), torch.float32),
              q_weight=_fake((64,)), k_weight=_fake((64,)))
    return [(gguf_hip.lora_add, lo, {"y": (0,), "x": (0,), "a": (0,), "b": (0,), "scales": (0,)}),
            (gguf_hip.paged_attention, at, {"q": (0, 1), "k_pages": (0, 1), "v_pages": (0, 1)}),
            (gguf_hip.qk_norm_rope, ro, {"q": (0,), "k": (1,), "table": (0, 1), "q_weight": (0,), "k_weight": (1,)})]


def test_gradients_are_refused_and_not_dropped():
    """A result of tensors that require gradients requires them too, and not through a gradient of its own; without a graph nothing
    changes."""
    with FakeTensorMode():
        for call, kw, marked in _calls():
            for name, which in marked.items():
                args = {**kw, name: kw[name].detach().clone().requires_grad_()}
                got = call(**args)
                got = got if isinstance(got, tuple) else (got,)
                assert [t.requires_grad for t in got] == [i in which for i in range(len(got))], (call, name)
                for i in which:
                    assert "NoBackward" in got[i].grad_fn.name()
                with torch.no_grad():
                    got = call(**args)
                assert not any(t.requires_grad for t in (got if isinstance(got, tuple) else (got,)))
            got = call(**kw)
            assert not any(t.requires_grad for t in (got if isinstance(got, tuple) else (got,)))


def test_gradients_of_results_that_are_written_into_a_tensor():
    with FakeTensorMode():
        _, kw, _ = _calls()[0]
        w = torch.nn.Parameter(_fake((4, 48)))
        y = w * 2                                            # belongs to a graph: its values are gone afterwards
        out = gguf_hip.lora_add(**{**kw, "y": y}, out=y)
        assert out is y
        assert "NoBackward" in out.grad_fn.name()
        out = _fake((4, 48))
        assert gguf_hip.lora_add(**{**kw, "x": kw["x"].detach().clone().requires_grad_()}, out=out) is out and out.requires_grad
        cache = _fake((9, 16, 2, 64))
        _, ro, _ = _calls()[2]
        gguf_hip.qk_norm_rope(**{**ro, "k": ro["k"].detach().clone().requires_grad_()}, v=_fake((5, 2, 64)), k_pages=cache,
                              v_pages=_fake((9, 16, 2, 64)), slots=_fake((5,), torch.int32))
        assert not cache.requires_grad


def test_a_torch_that_does_not_load_the_module():
    """The eager calls' module is built for one torch; without it the package is all there, with a warning."""
    import os
    import subprocess
    import sys

    code = """
import sys, warnings
sys.modules["gguf_hip._fast"] = None                         # its import raises ImportError
with warnings.catch_warnings(record=True) as seen:
    warnings.simplefilter("always")
    import gguf_hip
assert [w.category for w in seen if "_fast" in str(w.message)] == [RuntimeWarning], seen
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
with FakeTensorMode():
    e = lambda *s, dtype=torch.bfloat16: torch.empty(s, dtype=dtype, device="cuda")
    i32 = lambda *s: e(*s, dtype=torch.int32)
    assert gguf_hip.paged_attention(e(3, 8, 64), e(9, 16, 2, 64), e(9, 16, 2, 64), i32(3, 4), i32(3)).shape == (3, 8, 64)
    assert gguf_hip.lora_add(e(4, 48), e(4, 64), e(3, 1, 16, 64), e(3, 48, 16), i32(4), None, [48]).shape == (4, 48)
    assert gguf_hip.qk_norm_rope(e(5, 8, 64), None, i32(5), e(100, 32, dtype=torch.float32))[0].shape == (5, 8, 64)
    gguf_hip.copy_pages(e(3, 9, 16), [0], [1], dim=1)
print("done")
"""
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100,
                         env={**os.environ, "PYTHONPATH": os.pathsep.join(p for p in sys.path if p)})
    assert run.returncode == 0 and run.stdout.strip() == "done", run.stderr[-2000:]
