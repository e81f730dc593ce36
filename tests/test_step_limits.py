"""CPU tests of the limits of the operators of steps of several new tokens and of long caches (nothing is launched)."""
import ctypes

import pytest

from gguf_hip import _lib
from gguf_hip._lib import lib

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
