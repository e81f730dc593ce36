"""The operators around the linear path at the limits of what they accept, on the GPU: the longest sequences, very many keys of
little weight each, workspaces smaller than a call would like, batches beyond one launch.  Each against its definition in 64
bits, with bounds from the roundings that the operators are allowed: u is half a step of a type (2^-8 of a bf16 value, 2^-11 of an
fp16 one), sums and products are fp32 (2^-24 of each)."""
import pytest
import torch

import gguf_hip
from gguf_hip import _lib

pytestmark = pytest.mark.gpu

BF, F16, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
U = {BF: 2.0 ** -8, F16: 2.0 ** -11}
E32 = 2.0 ** -24


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, dtype=torch.float32):
    return torch.randn(shape, device="cuda", generator=gen).to(dtype)


def _within(got, want, tol, what):
    got, want = got.double(), want.double()
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4], want[bad][:4], (tol + 0 * want)[bad][:4])


# ---- attention -------------------------------------------------------------------------------

@pytest.mark.parametrize("length,window", [(_lib.GQK_MAX_KEYS, 0), (_lib.GQK_MAX_KEYS - 31, 0x7f000000), (2 ** 31 - 2 ** 23 + 1, 0)])
def test_attention_at_the_limit_of_keys(length, window):
    """The longest sequence, whose table names two pages again and again: keys of score 0 and value 1, and in its last page (and
    one in the middle) keys of score 10.375, together about as heavy as all others, and value 3.  A wave takes 2^16 steps: a chain of as
    many fp32 roundings in the weights' total, and in the products' sums of two a step, of up to a whole unit each."""
    page, dim = 1 << 16, 8
    k, v = (torch.zeros((2, page, 1, dim), dtype=BF, device="cuda") for _ in range(2))
    k[1, :, 0, 0], v[0], v[1] = 10.375, 1.0, 3.0
    q = torch.zeros((1, 1, dim), dtype=BF, device="cuda")
    q[0, 0, 0] = 1.0
    count = -(-length // page)
    table = torch.zeros((1, count), dtype=torch.int32, device="cuda")
    table[0, count // 2] = table[0, -1] = 1
    n = torch.tensor([length], dtype=torch.int32, device="cuda")
    out, lse = gguf_hip.paged_attention(q, k, v, table, n, scale=1.0, window=window, return_lse=True)
    first = length - window if window else 0
    heavy = torch.tensor(10.375, dtype=torch.float64).exp() * (page + length - (count - 1) * page)
    light = length - first - (page + length - (count - 1) * page)
    want = (light + 3 * heavy) / (light + heavy)
    assert 1.9 < want < 2.4                                  # of the first split alone 1; without the last one a seventh less
    chain = 2.0 ** 16 * E32
    tol = U[BF] * want + (U[BF] + 5 * chain + 2.0 ** -16) * want * (1 + U[BF])
    _within(out, want.cuda().expand(1, 1, dim), tol.cuda(), (length, window))
    want_l = (light + heavy).log()
    _within(lse, want_l.cuda().expand(1, 1), chain + 2.0 ** -16 + 4 * E32 * (want_l + 20).cuda(), "lse")
