"""CPU tests of the limits of the operators of steps of several new tokens and of long caches (nothing is launched)."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import gguf_hip
from gguf_hip import _lib
from gguf_hip._lib import lib

BF, F8 = torch.bfloat16, torch.float8_e4m3fn

P = ctypes.c_void_p(4096)   # never dereferenced: the checks come first


def _c_pages(heads, dim):
    token = heads * dim
    return _lib.GqkPages(4096, 4096, 16 * token, token, dim, 16 * token, token, dim, None, None, _lib.GQK_DTYPE_BF16, 9, 16, heads, dim)


@pytest.mark.parametrize("tokens,batch,heads,group,most_tokens", [(1 << 20, 65535, 256, 1, 1 << 20), (4, 65535, 257, 1, 4), (1 << 20, 1, 128, 16, 4),
                                                                  (1 << 20, 1, 4, 1024, 1 << 20)])
def test_tree_of_more_tiles_than_a_launch_has_workgroups(tokens, batch, heads, group, most_tokens):
    """A launch has fewer than 2^24 workgroups of 256 threads."""
    pages = _c_pages(heads, 8)
    rc = lib.gqk_tree_attention(P, heads * group * 8, 8, _lib.GQK_DTYPE_BF16, tokens, batch, heads * group, ctypes.byref(pages), P, 4, 4, P, P,
                                None, 0, 64, most_tokens, 0, 0.1, P, heads * group * 8, 8, None, P, 1 << 50, None)
    assert rc == _lib.GQK_ERR_SHAPE and b"more than a launch takes" in lib.gqk_last_error()


def test_tree_splits_only_what_one_launch_joins():
    """Many places for row tiles and few tokens: no partial sums, whose join would be more workgroups than a launch has."""
    need = lib.gqk_tree_attention_workspace_bytes
    assert need(1, 65535, 130, 130, 8, 1, 1 << 20, 0) == 0 and need(1, 100, 130, 130, 8, 1, 1 << 20, 0) > _lib.GQK_CTR_BYTES


def test_eight_bit_output_beside_its_inputs():
    """An 8-bit output may lie in an input's memory where it shares no bytes with it: behind it, or beside it in each row."""
    with FakeTensorMode():
        buf, w = torch.empty((5, 300), dtype=BF, device="cuda"), torch.empty((300,), dtype=BF, device="cuda")
        x, y, own = buf[:, :64], buf[:, 96:160], torch.empty((5, 64), dtype=BF, device="cuda")
        beside, behind = buf.view(F8)[:, 128:192], buf.view(F8)[:, 536:600]
        between = buf[:4].view(F8).flatten()[600 * 3 + 128:600 * 3 + 192].expand(1, 64)     # in one row, beside its 64 values
        for kw in (dict(x=x, residual=None, out=beside), dict(x=x, residual=y, out=behind), dict(x=own, residual=x, out=beside),
                   dict(x=own, residual=own, out_residual=y, out=behind), dict(x=buf[3:4, :64], residual=None, out=between)):
            assert gguf_hip.add_rms_norm_fp8(**kw)[0] is kw["out"]
        for out in (buf.view(F8)[:, :64], buf.view(F8)[:, 64:128], buf.view(F8)[:, 127:191], buf.view(F8)[:, 1:65], buf.flatten().view(F8)[:320].view(5, 64)):
            for kw in (dict(x=x), dict(residual=x), dict(residual=own, out_residual=x)):
                with pytest.raises(ValueError, match="memory of its own"):
                    gguf_hip.add_rms_norm_fp8(**{"x": own, "residual": None, **kw, "out": out})
        one = w.view(F8)
        assert gguf_hip.add_rms_norm_fp8(torch.empty((1, 64), dtype=BF, device="cuda"), None, w[:64], out=one[None, 128:192])[0].shape == (1, 64)
        with pytest.raises(ValueError, match="memory of its own"):
            gguf_hip.add_rms_norm_fp8(torch.empty((1, 64), dtype=BF, device="cuda"), None, w[:64], out=one[None, 127:191])
