"""The operators around the linear path at the limits of what they accept, on the GPU: the longest sequences, very many keys of
little weight each, workspaces smaller than a call would like, batches beyond one launch.  Each against its definition in 64
bits, with bounds from the roundings that the operators are allowed: u is half a step of a type (2^-8 of a bf16 value, 2^-11 of an
fp16 one), sums and products are fp32 (2^-24 of each)."""
import ctypes
import weakref

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


@pytest.mark.parametrize("qt,ct,dim", [(F16, F16, 64), (F16, F16, 128), (F16, F16, 256), (F16, F8, 128), (BF, BF, 128)])
@pytest.mark.parametrize("batch,pages", [(1, 40), (1100, 1)])
@pytest.mark.parametrize("late", [False, True])
def test_attention_flat_tail(qt, ct, dim, batch, pages, late):
    """Four heavy keys of value 0 to a page, one for each wave, first or last of it; 4092 others of 2^-25.2 of their weight each,
    which are all of the result.  A weight keeps its relative precision down there: half a step of the type."""
    page = 4096
    k, v = (torch.zeros((1, page, 1, dim), device="cuda") for _ in range(2))
    k[..., 0], v[:] = -14.0, 256.0
    heavy = torch.arange(0, 128, 32, device="cuda") + (page - 128 if late else 0)
    k[:, heavy], v[:, heavy] = 0.0, 0.0
    k, v = k.to(ct), v.to(ct)
    q = torch.zeros((batch, 2, dim), dtype=qt, device="cuda")
    q[..., 0] = 1.25                                         # scores of 0 and -17.5
    table = torch.zeros((batch, pages), dtype=torch.int32, device="cuda")
    n = torch.full((batch,), pages * page, dtype=torch.int32, device="cuda")
    out, lse = gguf_hip.paged_attention(q, k, v, table, n, scale=1.0, return_lse=True)
    light = (page - 4) * torch.tensor(-17.5, dtype=torch.float64).exp().item()
    want = 256 * light / (4 + light)
    # a score's error (one product, two factors, its exponential) and up to 2^7 steps a wave with two sums each
    e = 2.0 ** -18 + 2.0 ** 9 * E32
    _within(out, torch.full_like(out, want, dtype=torch.float64), (2 * U[qt] + 2 * e) * want + 2.0 ** -25, "out")
    want_l = torch.tensor((4 + light) * pages, dtype=torch.float64).log().item()
    _within(lse, torch.full_like(lse, want_l, dtype=torch.float64), 2 * e + 4 * E32 * (want_l + 40), "lse")


def _attend(q, k, v, table, lens, scale):
    """(out, its bound) in 64 bits, for lengths that all sequences share or not, one page to a sequence."""
    B, H, D = q.shape
    hkv = k.shape[2]
    kk, vv = (t[table[:, 0].long()].double().transpose(1, 2) for t in (k, v))           # [B, hkv, page, D]
    qq = q.double().view(B, hkv, H // hkv, D)
    live = torch.arange(k.shape[1], device="cuda")[None] < lens[:, None]
    s = (qq @ kk.transpose(2, 3).contiguous() * scale).masked_fill(~live[:, None, None], float("-inf"))
    size = (qq.abs() @ kk.abs().transpose(2, 3).contiguous() * scale).masked_fill(~live[:, None, None], 0).amax(-1, keepdim=True)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top.isinf(), 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    o, abs_o = p @ vv, p @ vv.abs()
    es = (D + 8) * E32 * size + 2.0 ** -19
    tol = U[q.dtype] * o.abs() + (1 + U[q.dtype]) * (U[q.dtype] + 2 * es + 2.0 ** -18) * abs_o + 2.0 ** -25
    return o.view(B, H, D), tol.view(B, H, D)


@pytest.mark.parametrize("batch,heads", [(1005, 64), (1020, 64), (1023, 64), (511, 128)])
def test_attention_of_many_rows_on_the_shared_workspace(batch, heads):
    """Just under as many workgroups as stay resident, of many wide heads each: two splits of all would not fit the workspace."""
    gen = _gen(batch)
    k, v = (_randn(gen, 5, 64, 1, 256, dtype=BF) for _ in range(2))
    q = _randn(gen, batch, heads, 256, dtype=BF)
    table = torch.randint(0, 5, (batch, 1), device="cuda", generator=gen).int()
    lens = torch.randint(0, 65, (batch,), device="cuda", generator=gen).int()
    wide = torch.full((batch, 128), -1, dtype=torch.int32, device="cuda")               # 8192 keys: the bound that the call goes by
    wide[:, :1] = table
    out = gguf_hip.paged_attention(q, k, v, wide, lens)
    want, tol = _attend(q, k, v, table, lens, 256 ** -0.5)
    _within(out, want, tol, batch)


@pytest.mark.parametrize("batch,heads,hkv,dim", [(1, 8, 2, 64), (3, 40, 8, 128), (2, 40, 1, 256)])
def test_attention_in_small_workspaces(batch, heads, hkv, dim):
    """A workspace that holds all, some, two or none of the splits that the call would like; its counters stay at zero, and
    nothing is written past its end."""
    gen = _gen(heads)
    k, v = (_randn(gen, 3, 4096, hkv, dim, dtype=BF) for _ in range(2))
    q = _randn(gen, batch, heads, dim, dtype=BF)
    table = torch.arange(batch, device="cuda").int()[:, None]
    lens = torch.tensor([4096, 4001, 0][:batch], device="cuda").int()
    want, tol = _attend(q, k, v, table, lens, dim ** -0.5)
    need = _lib.lib.gqk_paged_attention_workspace_bytes(batch, heads, hkv, dim, 4096, 0)
    split = batch * heads * (dim + 4) * 4
    assert need >= _lib.GQK_CTR_BYTES + 4 * split
    for size in (need, need - 4, _lib.GQK_CTR_BYTES + 3 * split, _lib.GQK_CTR_BYTES + 2 * split, _lib.GQK_CTR_BYTES + 2 * split - 4,
                 _lib.GQK_CTR_BYTES, 256):
        whole = torch.zeros(size // 4 + 1024, dtype=torch.int32, device="cuda")
        ws = whole[:size // 4]
        _within(gguf_hip.paged_attention(q, k, v, table, lens, workspace=ws), want, tol, size)
        assert not whole[size // 4:].any() and not ws[:_lib.GQK_CTR_BYTES // 4].any(), size
        _within(gguf_hip.paged_attention(q, k, v, table, lens, workspace=ws), want, tol, size)


# ---- norm, rotation, store -------------------------------------------------------------------

def test_rope_scales_that_are_negated_lazily():
    """Tensors whose memory is not their value go through the op, the pages' scales among them."""
    gen = _gen(3)
    q, k, v = (_randn(gen, 4, 2, 64, dtype=BF) for _ in range(3))
    pos, rope = torch.arange(4, device="cuda"), gguf_hip.rope_table(64, 9, device="cuda")
    ks, vs = torch.tensor([0.5, 2.0], device="cuda"), torch.tensor([0.25, 4.0], device="cuda")

    def stored(ks, vs):
        kp, vp = (torch.zeros((1, 4, 2, 64), dtype=F8, device="cuda") for _ in range(2))
        gguf_hip.qk_norm_rope(q, k, pos, rope, v=v, k_pages=kp, v_pages=vp, slots=pos, k_scale=ks, v_scale=vs)
        return kp.view(torch.uint8), vp.view(torch.uint8)

    for got, want in zip(stored(torch._neg_view(-ks), torch._neg_view(-vs)), stored(ks, vs)):
        assert torch.equal(got, want)


# ---- adapters --------------------------------------------------------------------------------

def _lora_case(gen, M, K, n_outs, rank, slots, dtype):
    y, x = _randn(gen, M, sum(n_outs), dtype=dtype), _randn(gen, M, K, dtype=dtype)
    a = (_randn(gen, slots, len(n_outs), rank, K) * K ** -0.5).to(dtype)
    b = _randn(gen, slots, sum(n_outs), rank, dtype=dtype)
    return y, x, a, b, torch.randint(-1, slots, (M,), device="cuda", generator=gen)


def _lora_exact(y, x, a, b, ids, n_outs):
    """(out, its bound) in 64 bits: h's K products in fp32, kept to 2^-16, rank products in fp32, one rounding."""
    out, tol = y.double(), torch.zeros(y.shape, dtype=torch.float64, device="cuda")
    K, rank = x.shape[1], a.shape[2]
    for i in range(a.shape[0]):
        rows = (ids == i).nonzero()[:, 0]
        X, col = x[rows].double(), 0
        for p, n in enumerate(n_outs):
            A, B = a[i, p].double(), b[i, col:col + n].double()
            h, ha = X @ A.t(), X.abs() @ A.abs().t()
            out[rows, col:col + n] += h @ B.t()
            e = (2.0 ** -16 + (rank + 4) * E32) * h.abs() + K * E32 * ha
            tol[rows, col:col + n] = e @ B.abs().t()
            col += n
    u = U[y.dtype]
    return out, (1 + u) * (tol + 2 * E32 * y.double().abs()) + u * out.abs() + 2.0 ** -25


@pytest.mark.parametrize("into", ["y", "new"])
def test_lora_turns_whose_last_is_the_smallest(into):
    """4867 rows in a workspace made for 15520 go in turns of 1217; the last, of 1216, would like more splits of K, and
    so more room, than the others.  It must not be refused once they are written."""
    K, n_outs = 17408, (24,)
    need = _lib.lib.gqk_lora_workspace_bytes
    size = need(15520, K, 1, 16)
    assert need(1217, K, 1, 16) <= size < need(1216, K, 1, 16)
    y, x, a, b, ids = _lora_case(_gen(1), 4867, K, n_outs, 16, 2, BF)
    want, tol = _lora_exact(y, x, a, b, ids, n_outs)
    ws = torch.zeros(size // 4, dtype=torch.int32, device="cuda")
    out = gguf_hip.lora_add(y, x, a, b, ids, None, n_outs, out=y if into == "y" else None, workspace=ws)
    _within(out, want, tol, into)


@pytest.mark.parametrize("rows", [8192, 4096, 2047, 300, 256, 40])
def test_lora_workspace_of_more_rows_serves_fewer(rows):
    """The C entry in a workspace sized for 16384 rows, and in the least that it takes; nothing is written past it or in the counters."""
    K, n, rank = 17408, 16, 64
    y, x, a, b, ids = _lora_case(_gen(rows), rows, K, (n,), rank, 2, BF)
    want, tol = _lora_exact(y, x, a, b, ids, (n,))
    cols = (ctypes.c_int64 * 1)(n)
    for size in (_lib.lib.gqk_lora_workspace_bytes(16384, K, 1, rank), _lib.GQK_CTR_BYTES + rows * rank * 4):
        whole = torch.zeros(size // 4 + 4096, dtype=torch.int32, device="cuda")
        out = torch.empty_like(y)
        args = [y.data_ptr(), n, x.data_ptr(), K, rows, K, a.data_ptr(), b.data_ptr(), 2, 1, cols, rank, ids.data_ptr(), 1, None,
                _lib.GQK_DTYPE_BF16, out.data_ptr(), n, whole.data_ptr(), size, torch.cuda.current_stream().cuda_stream]
        assert _lib.lib.gqk_lora_add(*args) == 0, _lib.lib.gqk_last_error()
        _within(out, want, tol, (rows, size))
        assert not whole[size // 4:].any() and not whole[:_lib.GQK_CTR_BYTES // 4].any()
    args[-2] = size - 4
    assert _lib.lib.gqk_lora_add(*args) == _lib.GQK_ERR_SHAPE


def test_lora_more_rows_than_a_launch_takes():
    """Rows beyond 65535 blocks of 64 go in turns."""
    M = 65535 * 64 + 77
    y, x, a, b, ids = _lora_case(_gen(2), M, 8, (8,), 8, 2, BF)
    want, tol = _lora_exact(y, x, a, b, ids, (8,))
    _within(gguf_hip.lora_add(y, x, a, b, ids, None, (8,)), want, tol, M)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("rows", [1, 20, 300])
@pytest.mark.parametrize("rank", [8, 32, 72, 256])
def test_lora_infinite_weights(dtype, rows, rank):
    """An infinity in B reaches its column with its sign times h's, whatever h's value rounds to: no inf - inf of h's two terms."""
    gen = _gen(rows)
    y, x, a, b, ids = _lora_case(gen, rows, 64, (40,), rank, 2, dtype)
    ids[:] = 0
    x[0] = 0
    x[0, 0] = 1.0
    a[:, :, :, 0] = 0.5                                      # row 0's h is 0.5 exactly: one term holds it
    b[0, 3, 2], b[0, 7, rank - 1] = float("inf"), float("-inf")
    out = gguf_hip.lora_add(y, x, a, b, ids, None, (40,))
    want, tol = _lora_exact(y, x, a, b, ids, (40,))
    whole = [c for c in range(40) if c not in (3, 7)]
    assert want[:, [3, 7]].isinf().all() and torch.equal(out[:, [3, 7]].double(), want[:, [3, 7]])
    _within(out[:, whole], want[:, whole], tol[:, whole], rows)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("rows", [1, 20, 300])
@pytest.mark.parametrize("rank", [8, 32, 72, 256])
def test_lora_an_infinite_rank_beside_large_ones(dtype, rows, rank):
    """One rank's h is infinite, the others' are finite and beyond fp16: they do not cancel it."""
    y, x, a, b, ids = _lora_case(_gen(rows), rows, 64, (40,), rank, 2, dtype)
    ids[:] = 0
    x, a = x * 1000, a * 1000
    a[0, 0, 3, 5] = float("inf")
    out = gguf_hip.lora_add(y, x, a, b, ids, None, (40,))
    want, _ = _lora_exact(y, x, a, b, ids, (40,))
    assert want.isinf().all() and torch.equal(out.double(), want)


# ---- page copies -----------------------------------------------------------------------------

def test_copy_pages_traced_and_watched():
    """A trace records the copy and does not make it; the recorded call, the op that a profiler sees and the eager call agree."""
    from torch.fx.experimental.proxy_tensor import make_fx

    def fork(pages):
        gguf_hip.copy_pages(pages, [3, 4], [7, 8], dim=1)
        return pages[:, 7] + 1

    pages = _randn(_gen(1), 3, 9, 16, 64, dtype=BF)
    want = pages.clone()
    want[:, [7, 8]] = want[:, [3, 4]]
    g = make_fx(fork, tracing_mode="fake")(pages)
    assert not torch.equal(pages, want)
    mine = pages.clone()
    assert torch.equal(g(mine), want[:, 7] + 1) and torch.equal(mine, want)
    mine = pages.clone()
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        gguf_hip.copy_pages(mine, [3, 4], [7, 8], dim=1)
    assert torch.equal(mine, want) and any("copy_pages" in ev.key for ev in prof.key_averages())
    version = pages._version
    gguf_hip.copy_pages(pages, [3, 4], [7, 8], dim=1)
    assert torch.equal(pages, want) and pages._version > version


# ---- the shared workspace --------------------------------------------------------------------

def test_shared_workspace_outlives_a_larger_one(monkeypatch):
    """A captured call keeps the address of the workspace that it was captured with: where a layer's plans need a larger one, the
    old one's memory is not given to others."""
    from gguf_hip import ops

    device = torch.device("cuda", 0)
    monkeypatch.setattr(ops, "_WORKSPACES", {})
    old = ops.shared_workspace(device)
    alive, size = weakref.ref(old), old.numel() * 4
    del old
    assert ops.device_workspace(device, size + 4096).numel() * 4 == size + 4096
    assert alive() is not None


# ---- gradients -------------------------------------------------------------------------------

def test_gradients_raise_and_values_stay():
    gen = _gen(1)
    y, x, a, b, ids = _lora_case(gen, 20, 64, (40,), 8, 2, BF)
    k, v = (_randn(gen, 3, 16, 2, 64, dtype=BF) for _ in range(2))
    table, lens = torch.zeros((4, 1), dtype=torch.int32, device="cuda"), torch.full((4,), 9, dtype=torch.int32, device="cuda")
    q, pos, rope = _randn(gen, 4, 8, 64, dtype=BF), torch.arange(4, device="cuda"), gguf_hip.rope_table(64, 9, device="cuda")
    for call, t in ((lambda t: gguf_hip.lora_add(y, x, t, b, ids, None, (40,)), a),
                    (lambda t: gguf_hip.lora_add(t * 1, x, a, b, ids, None, (40,)), y),
                    (lambda t: gguf_hip.paged_attention(t, k, v, table, lens), q),
                    (lambda t: gguf_hip.qk_norm_rope(q, None, pos, rope, t)[0], _randn(gen, 64, dtype=BF))):
        want = call(t)
        leaf = torch.nn.Parameter(t)
        got = call(leaf)
        assert got.requires_grad and not want.requires_grad and torch.equal(got, want)
        with pytest.raises(RuntimeError, match="no backward"):
            got.float().sum().backward()
        with torch.no_grad():
            got = call(leaf)
        assert not got.requires_grad and torch.equal(got, want)


# ---- without the eager calls' module ---------------------------------------------------------

def test_calls_without_the_eager_module(monkeypatch):
    """The same bits by way of Python."""
    from gguf_hip import adapters, attention, pages as pages_py

    gen = _gen(2)
    y, x, a, b, ids = _lora_case(gen, 20, 64, (40,), 8, 2, BF)
    k, v = (_randn(gen, 3, 16, 2, 64, dtype=BF) for _ in range(2))
    table, lens = torch.zeros((4, 1), dtype=torch.int32, device="cuda"), torch.full((4,), 9, dtype=torch.int32, device="cuda")
    q, pos, rope = _randn(gen, 4, 8, 64, dtype=BF), torch.arange(4, device="cuda"), gguf_hip.rope_table(64, 9, device="cuda")

    def calls():
        mine = k.clone()
        gguf_hip.copy_pages(mine, [0], [2])
        return (gguf_hip.lora_add(y, x, a, b, ids, None, (40,)), gguf_hip.paged_attention(q, k, v, table, lens),
                gguf_hip.qk_norm_rope(q, None, pos, rope)[0], mine)

    want = calls()
    for module in (adapters, attention, pages_py, _lib):
        monkeypatch.setattr(module, "_fast", None)
    assert all(torch.equal(g, w) for g, w in zip(calls(), want)) and torch.equal(want[3][2], k[0])
