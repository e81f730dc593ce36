"""The operators around the linear path on the GPU, each against its definition in 64 bits (plain torch on the CPU or the
GPU, written here).  Tolerances are bounds per value, from the roundings that the operators are allowed: u is half a step of
a type (2^-8 of a bf16 value, 2^-11 of an fp16 one, 2^-4 of an e4m3 one), sums and products are fp32."""
import pytest
import torch

import gguf_hip

pytestmark = pytest.mark.gpu

BF, F16, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
U = {BF: 2.0 ** -8, F16: 2.0 ** -11, F8: 2.0 ** -4}
TINY = {BF: 0.0, F16: 2.0 ** -25, F8: 2.0 ** -10}     # half of the smallest step, where a type's range ends
E32 = 2.0 ** -24


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, dtype=torch.float32):
    return torch.randn(shape, device="cuda", generator=gen).to(dtype)


def _within(got, want, tol, what):
    got, want = got.double(), want.double()
    bad = ~((got - want).abs() <= tol) & ~(got.isnan() & want.isnan()) & ~(got == want)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4], want[bad][:4], (tol + 0 * want)[bad][:4])


# ---- attention -------------------------------------------------------------------------------

def _cache(gen, lens, page, heads, dim, dtype, layout, spare=2, poison=True):
    """Pages in a random order, the table's unused entries outside of the cache, what no sequence holds NaN."""
    need = [-(-max(n, 0) // page) for n in lens]
    count, width = sum(need) + spare, max(1, max(need))
    shape = (count, heads, page, dim) if layout == "heads" else (count, page, heads, dim)
    k, v = (_randn(gen, *shape).to(dtype) for _ in range(2))
    if layout == "heads":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    order = torch.randperm(count, device="cuda", generator=gen).to(torch.int32)
    table = torch.full((len(lens), width), 2 ** 31 - 1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    if poison:
        nan = float("nan")
        as_bytes = (lambda t: t.view(torch.uint8)) if dtype == F8 else (lambda t: t)
        fill = 0x7F if dtype == F8 else nan
        for t in (k, v):
            as_bytes(t)[order[at:].long()] = fill
            for i, n in enumerate(lens):
                if n % page and n > 0:
                    as_bytes(t)[table[i, need[i] - 1].long(), n % page:] = fill
    return k, v, table


def _attend_exact(q, k, v, table, lens, scale, window, ks=None, vs=None):
    """(out, lse, bound of the error of out, of lse) in 64 bits."""
    B, H, D = q.shape
    hkv, page = k.shape[2], k.shape[1]
    out = torch.zeros((B, H, D), dtype=torch.float64, device="cuda")
    lse = torch.full((B, H), float("-inf"), dtype=torch.float64, device="cuda")
    tol, tol_l = torch.zeros_like(out), torch.zeros_like(lse)
    u = U[q.dtype]
    for b, n in enumerate(lens):
        first = max(0, n - window) if window else 0
        if n <= first:
            continue
        at = torch.arange(first, n, device="cuda")
        rows = (table[b].long()[at // page], at % page)
        kk, vv = k[rows].double(), v[rows].double()                        # [keys, heads, dim]
        if ks is not None:
            kk = kk * ks.double()[None, :, None]
        if vs is not None:
            vv = vv * vs.double()[None, :, None]
        g = H // hkv
        qq = q[b].double().reshape(hkv, g, D)
        s = torch.einsum("hgd,khd->hgk", qq, kk) * scale
        size = (torch.einsum("hgd,khd->hgk", qq.abs(), kk.abs()) * abs(scale)).amax(-1)
        top = s.amax(-1, keepdim=True)
        e = torch.exp(s - top)
        total = e.sum(-1, keepdim=True)
        o = torch.einsum("hgk,khd->hgd", e / total, vv)
        abs_o = torch.einsum("hgk,khd->hgd", e / total, vv.abs())
        # a score's error (D products and sums in fp32, its scales) and the exponential's
        es = (D + 8) * E32 * size + 2.0 ** -20 + 4 * E32 * (s - top).abs().amax(-1)
        ep = u + 2 * es + 2.0 ** -18                                       # of a probability, and of the sums in fp32
        out[b] = o.reshape(H, D)
        tol[b] = (u * o.abs() + (1 + u) * (ep[..., None] * abs_o + TINY[q.dtype] * (vv.abs().sum(0)[:, None] / total))
                  + TINY[q.dtype] + 1e-30).reshape(H, D)
        lse[b] = (top + total.log())[..., 0].reshape(H)
        tol_l[b] = (es + 2.0 ** -18 + 4 * E32 * (top[..., 0].abs() + 20)).reshape(H)
    return out, lse, tol, tol_l


def _attend_check(seed, lens, hq, hkv, dim, page, qt, ct, window=0, layout="heads", scaled=False, max_length=None, scale=None):
    gen = _gen(seed)
    k, v, table = _cache(gen, lens, page, hkv, dim, ct, layout)
    q = _randn(gen, len(lens), hq, dim, dtype=qt)
    ks = vs = None
    if scaled:
        ks, vs = (0.25 + torch.rand(hkv, device="cuda", generator=gen) for _ in range(2))
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    call = lambda: gguf_hip.paged_attention(q, k, v, table, n, scale=scale, window=window, k_scale=ks, v_scale=vs,  # noqa: E731
                                            max_length=max_length, return_lse=True)
    out, lse = call()
    want, want_l, tol, tol_l = _attend_exact(q, k, v, table, lens, dim ** -0.5 if scale is None else scale, window, ks, vs)
    _within(out, want, tol, "out")
    _within(lse, want_l, tol_l, "lse")
    again, lse2 = call()
    assert torch.equal(out, again) and torch.equal(lse, lse2)               # the same bits every time


@pytest.mark.parametrize("qt,ct", [(BF, BF), (F16, F16), (BF, F8), (F16, F8)])
@pytest.mark.parametrize("dim,hq,hkv", [(64, 8, 2), (128, 40, 8), (128, 3, 3), (256, 6, 1), (80, 5, 1), (8, 2, 1), (192, 4, 2)])
def test_attention_types_and_heads(qt, ct, dim, hq, hkv):
    _attend_check(dim + hq, [1, 0, 33, 200, 517], hq, hkv, dim, 16, qt, ct, scaled=ct == F8,
                  layout="heads" if hq % 2 else "tokens")


@pytest.mark.parametrize("hq,hkv", [(16, 1), (17, 1), (32, 2), (40, 1), (71, 1), (128, 1), (1, 1)])
def test_attention_shared_heads(hq, hkv):
    """One key head for many query heads: more than a tile's 16, and counts that do not divide by it."""
    _attend_check(hq, [130, 5, 0, 700], hq, hkv, 64, 16, BF, BF)


@pytest.mark.parametrize("qt,ct", [(BF, BF), (F16, F16), (BF, F8)])
@pytest.mark.parametrize("hq,hkv,dim", [(33, 1, 128), (96, 2, 64), (128, 1, 128), (20, 1, 256)])
def test_attention_many_heads_in_splits(qt, ct, hq, hkv, dim):
    """Many heads over one of keys, cut into few and into many splits, beside sequences that are not cut."""
    _attend_check(hq, [1500, 128, 0, 129, 1], hq, hkv, dim, 16, qt, ct, scaled=ct == F8)
    _attend_check(hq, [9000], hq, hkv, dim, 16, qt, ct, window=7777, scaled=ct == F8)
    _attend_check(hq, [40_000], hq, hkv, dim, 16, qt, ct, scaled=ct == F8)



@pytest.mark.parametrize("page", [1, 2, 7, 8, 16, 24, 33, 48, 64, 256])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
def test_attention_page_sizes(page, layout):
    """Pages that end inside a tile of keys, at its edge, or hold several."""
    _attend_check(page, [1, 31, 32, 33, 65, 300, 0], 10, 2, 128, page, BF, BF, layout=layout)


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 1000, 5000])
def test_attention_windows(window):
    """The window's start inside a page and a tile; a window longer than some or all of the lengths."""
    _attend_check(window, [0, 1, 31, 33, 64, 99, 100, 101, 1500], 8, 2, 64, 16, F16, F16, window=window)


@pytest.mark.parametrize("lens", [[1], [4095], [4096, 1], [9001], [2500, 0, 1, 1700, 64, 63, 65, 2048], [300] * 70])
def test_attention_lengths(lens):
    """One sequence split over the device, batches of many lengths, more sequences than fill it once."""
    _attend_check(len(lens) + lens[0], lens, 20, 4, 128, 16, BF, BF)


def test_attention_long():
    _attend_check(3, [70001, 5], 10, 2, 128, 64, BF, F8, scaled=True)
    _attend_check(4, [50021], 6, 1, 256, 32, F16, F16, window=33333)


def test_attention_max_length_is_only_a_bound():
    """A loose or a tight bound on the lengths: the same values up to the order of the sums; a length above it: NaN."""
    gen = _gen(5)
    lens = [700, 3, 0, 512]
    k, v, table = _cache(gen, lens, 16, 2, 64, BF, "heads")
    wide = torch.full((4, 4000), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    q = _randn(gen, 4, 8, 64, dtype=BF)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want, _, tol, _ = _attend_exact(q, k, v, table, lens, 64 ** -0.5, 0)
    for t, top in ((table, None), (table, 700), (wide, None), (wide[:, :50], 777)):
        _within(gguf_hip.paged_attention(q, k, v, t, n, max_length=top), want, tol, top)
    got = gguf_hip.paged_attention(q, k, v, table, n, max_length=600)
    assert got[0].isnan().all()
    _within(got[1:], want[1:], tol[1:], "the others")


def test_attention_bad_pages_are_not_read():
    gen = _gen(6)
    lens = [100, 600, 40, 17]
    k, v, table = _cache(gen, lens, 16, 2, 64, BF, "heads")
    q = _randn(gen, 4, 4, 64, dtype=BF)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want, _, tol, _ = _attend_exact(q, k, v, table, lens, 64 ** -0.5, 0)
    table = table.clone()
    table[1, 30], table[2, 0], table[3, 1] = k.shape[0], -1, 2 ** 30
    for _ in range(2):                                       # the second call finds the workspace as the first left it
        out, lse = gguf_hip.paged_attention(q, k, v, table, n, return_lse=True)
        assert out[1:].isnan().all() and lse[1:].isnan().all()
        _within(out[:1], want[:1], tol[:1], "the sound one")
    # outside of the window a bad page is not looked at
    out = gguf_hip.paged_attention(q, k, v, table, n, window=16)
    assert out[3].isnan().all() and not out[:3].isnan().any()


def test_attention_extreme_scores():
    """Scores far apart and far from zero, keys whose scores are -inf or +inf, and values that are not finite."""
    gen = _gen(8)
    k, v, table = _cache(gen, [90, 90, 90, 90, 90], 16, 1, 64, BF, "tokens", poison=False)
    q = _randn(gen, 5, 2, 64, dtype=BF)
    q[0] *= 200
    rows = lambda b, j: (int(table[b, j // 16]), j % 16, 0)  # noqa: E731
    q[1:, :, 0] = 1.0
    k[rows(1, 40)][0] = float("-inf")                        # score -inf: weight 0
    k[rows(2, 3)][0] = float("inf")                          # score +inf: inf - inf
    v[rows(3, 70)][5] = float("inf")
    v[rows(4, 70)][5] = float("nan")
    n = torch.full((5,), 90, dtype=torch.int32, device="cuda")
    out = gguf_hip.paged_attention(q, k, v, table, n)
    want, _, tol, _ = _attend_exact(q, k, v, table, [90] * 5, 0.125, 0)
    _within(out[0], want[0], tol[0], "far apart")
    _within(out[1], want[1], 2 * U[BF] * (1 + want[1].abs()), "-inf")
    assert out[2].isnan().all()
    assert (out[3, :, 5] == float("inf")).all() and not out[3, :, :5].isnan().any() and not out[3, :, 6:].isnan().any()
    assert out[4, :, 5].isnan().all() and not out[4, :, 6:].isnan().any()


def test_attention_strides_streams_and_outputs():
    """q as a column range of a wider tensor, an output that is one, rows of the table apart, another stream with a
    workspace of its own, shifted (unaligned) queries."""
    gen = _gen(9)
    lens = [1000, 31, 2]
    k, v, table = _cache(gen, lens, 16, 2, 128, BF, "heads")
    wide = _randn(gen, 3, 14 * 128, dtype=BF)
    q = wide.unflatten(1, (14, 128))[:, 3:13]
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want, _, tol, _ = _attend_exact(q, k, v, table, lens, 128 ** -0.5, 0)
    out = torch.zeros(3, 20, 128, dtype=BF, device="cuda")
    apart = torch.full((3, table.shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    apart[:, :table.shape[1]] = table
    got = gguf_hip.paged_attention(q, k, v, apart[:, :table.shape[1]], n, out=out[:, 5:15])
    assert got.data_ptr() == out[:, 5:15].data_ptr() and not out[:, :5].any() and not out[:, 15:].any()
    _within(out[:, 5:15], want, tol, "views")
    odd = torch.zeros(3 * 10 * 128 + 1, dtype=BF, device="cuda")[1:].view(3, 10, 128)
    odd.copy_(q)
    _within(gguf_hip.paged_attention(odd, k, v, table, n), want, tol, "unaligned")
    side, ws = torch.cuda.Stream(), torch.zeros(16 << 20, dtype=torch.int32, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = gguf_hip.paged_attention(q, k, v, table, n, workspace=ws)
    here = gguf_hip.paged_attention(q, k, v, table, n)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, here)
    with pytest.raises(ValueError):
        gguf_hip.paged_attention(q, k[..., ::2].transpose(1, 2), v, table, n)
    assert gguf_hip.paged_attention(q[:0], k, v, table[:0], n[:0]).shape == (0, 10, 128)


def test_attention_graph_replays():
    """A captured call reads lengths, table and pages anew in every replay."""
    gen = _gen(10)
    k, v, table = _cache(gen, [3000, 3000], 16, 2, 64, BF, "heads", poison=False)
    q = _randn(gen, 2, 8, 64, dtype=BF)
    n = torch.tensor([10, 20], dtype=torch.int32, device="cuda")
    gguf_hip.paged_attention(q, k, v, table, n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gguf_hip.paged_attention(q, k, v, table, n)
    for step, lens in enumerate(([10, 20], [3000, 0], [1, 2999], [1700, 64])):
        n.copy_(torch.tensor(lens, dtype=torch.int32))
        q.copy_(_randn(_gen(step), 2, 8, 64))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, gguf_hip.paged_attention(q, k, v, table, n))
        want, _, tol, _ = _attend_exact(q, k, v, table, lens, 0.125, 0)
        _within(out, want, tol, lens)


def test_attention_offsets_past_32_bits():
    """A cache of more than 2^31 elements, its last pages in use."""
    page, dim, count = 64, 128, 270_000
    k = torch.empty((count, page, 1, dim), dtype=F8, device="cuda")
    v = torch.empty((count, page, 1, dim), dtype=F8, device="cuda")
    assert k.numel() > 2 ** 31
    gen = _gen(11)
    used = torch.tensor([count - 1, 0, count - 2, 262_144, 5], dtype=torch.int32, device="cuda")
    for t in (k, v):
        t.view(torch.uint8)[used.long()] = _randn(gen, 5, page, 1, dim).to(F8).view(torch.uint8)
    q = _randn(gen, 1, 4, dim, dtype=BF)
    n = torch.tensor([300], dtype=torch.int32, device="cuda")
    out = gguf_hip.paged_attention(q, k, v, used[None], n)
    want, _, tol, _ = _attend_exact(q, k, v, used[None], [300], dim ** -0.5, 0)
    _within(out, want, tol, "far pages")


# ---- norm, rotation, store -------------------------------------------------------------------

def _rope_exact(x, w, pos, table, rot, eps, offset, interleaved):
    """(values, the sizes of what was added up for each) in 64 bits."""
    x = x.double()
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * (w.double() + (1 if offset else 0))
    out, size = x.clone(), x.abs()
    half = rot // 2
    cos, sin = (t[:, None] for t in table[pos.long()].double().split(half, 1)) if half else (None, None)
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = cos[..., i], sin[..., i]
        out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        size[..., a] = (x[..., a] * c).abs() + (x[..., b] * s).abs()
        size[..., b] = (x[..., b] * c).abs() + (x[..., a] * s).abs()
    return out, size


def _rope_tol(want, size, dtype, dim):
    """The norm's sum of dim squares, its root and four products in fp32, and one rounding to the type."""
    e = (dim / 2 + 16) * E32
    return (1 + U[dtype]) * e * size + U[dtype] * want.abs() + TINY[dtype] + 1e-30


def _rope_case(gen, tokens, hq, hkv, dim, dtype, rot, weights, most=500):
    qkv = _randn(gen, tokens, (hq + 2 * hkv) * dim, dtype=dtype) * 3
    q, k, v = (t.unflatten(1, (-1, dim)) for t in qkv.split((hq * dim, hkv * dim, hkv * dim), 1))
    table = gguf_hip.rope_table(rot, most, 1e4) if rot else torch.empty(most, 0, device="cuda")
    pos = torch.randint(0, most, (tokens,), device="cuda", generator=gen)
    wq = wk = None
    if weights is not None:
        wq, wk = (_randn(gen, dim, dtype=weights) for _ in range(2))
    return q, k, v, table, pos, wq, wk


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(64, 64), (128, 128), (128, 64), (256, 256), (256, 64), (80, 80), (80, 32), (96, 96), (8, 8),
                                     (8, 2), (128, 0), (72, 18), (136, 126), (256, 34), (192, 192)])
def test_rope_dims(dtype, interleaved, dim, rot):
    gen = _gen(dim + rot)
    q, k, v, table, pos, wq, wk = _rope_case(gen, 7, 5, 3, dim, dtype, rot, dtype)
    oq, ok = gguf_hip.qk_norm_rope(q, k, pos, table, wq, wk, interleaved=interleaved, eps=1e-5)
    for got, x, w in ((oq, q, wq), (ok, k, wk)):
        want, size = _rope_exact(x, w, pos, table, rot, 1e-5, False, interleaved)
        _within(got, want, _rope_tol(want, size, dtype, dim), (dim, rot))


@pytest.mark.parametrize("weights,offset", [(None, False), (torch.float32, False), (torch.float32, True), (BF, True)])
@pytest.mark.parametrize("tokens", [1, 2, 3, 63, 64, 65, 301])
def test_rope_weights_and_tokens(weights, offset, tokens):
    gen = _gen(tokens)
    q, k, v, table, pos, wq, wk = _rope_case(gen, tokens, 6, 2, 128, BF, 128, weights)
    oq, ok = gguf_hip.qk_norm_rope(q, k, pos.int(), table, wq, wk, unit_offset=offset)
    for got, x, w in ((oq, q, wq), (ok, k, wk)):
        want, size = _rope_exact(x, w, pos, table, 128, 1e-6, offset, False)
        _within(got, want, _rope_tol(want, size, BF, 128), tokens)
    # one of the two weights alone, and queries alone
    oq, ok = gguf_hip.qk_norm_rope(q, k, pos, table, wq, None, unit_offset=offset)
    want, size = _rope_exact(k, None, pos, table, 128, 1e-6, False, False)
    _within(ok, want, _rope_tol(want, size, BF, 128), "keys without a norm")
    alone, none = gguf_hip.qk_norm_rope(q, None, pos, table, wq, unit_offset=offset)
    assert none is None and torch.equal(alone, oq)


@pytest.mark.parametrize("dtype,ct", [(BF, BF), (F16, F16), (BF, F8), (F16, F8)])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
@pytest.mark.parametrize("dim,page", [(128, 16), (80, 7), (256, 48), (64, 1)])
def test_rope_stores(dtype, ct, layout, dim, page):
    """Keys and values land in their slots and nothing else changes; some tokens have no slot; slots of either width;
    the fp8 scales; the values that are beyond an fp8 page's range."""
    gen = _gen(page)
    tokens, hkv = 37, 3
    q, k, v, table, pos, wq, wk = _rope_case(gen, tokens, 6, hkv, dim, dtype, dim // 2 // 2 * 2, dtype)
    v[0, 0, 0], v[1, 0, 1] = 3000.0, -3000.0
    rot = table.shape[1]
    count = -(-tokens // page) + 3
    shape = (count, hkv, page, dim) if layout == "heads" else (count, page, hkv, dim)
    kp, vp = (_randn(gen, *shape).to(ct) for _ in range(2))
    if layout == "heads":
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    ks = vs = None
    if ct == F8:
        ks, vs = (0.25 + torch.rand(hkv, device="cuda", generator=gen) for _ in range(2))
    before = kp.double(), vp.double()
    slots = torch.randperm(count * page, device="cuda", generator=gen)[:tokens]
    slots[5], slots[20] = -1, -7
    slots = slots.int() if page % 2 else slots
    oq, ok = gguf_hip.qk_norm_rope(q, k, pos, table, wq, wk, v=v, k_pages=kp, v_pages=vp, slots=slots, k_scale=ks, v_scale=vs)
    assert ok is None
    kept = slots >= 0
    s = slots[kept].long()
    for pages, old, x, w, scale in ((kp, before[0], k, wk, ks), (vp, before[1], v, None, vs)):
        if x is v:
            want, size = v.double(), torch.zeros_like(v.double())
        else:
            want, size = _rope_exact(x, w, pos, table, rot, 1e-6, False, False)
        if scale is not None:
            want, size = want / scale.double()[None, :, None], size / scale.double()[None, :, None] + (want * E32).abs() * 8
        if ct == F8:
            want = want.clamp(-448, 448)
        full, tol = old.clone(), torch.zeros_like(old)
        full[s // page, s % page] = want[kept]
        exact_v = x is v and ct != F8
        tol[s // page, s % page] = torch.zeros_like(want[kept]) if exact_v else _rope_tol(want, size, ct, dim)[kept]
        _within(pages, full, tol, "values" if x is v else "keys")
    want, size = _rope_exact(q, wq, pos, table, rot, 1e-6, False, False)
    _within(oq, want, _rope_tol(want, size, dtype, dim), "queries")
    # with the keys beside the pages: the same stores, and the keys as they are without pages
    kp2, vp2 = kp.clone(), vp.clone()
    mine = torch.empty_like(k, memory_format=torch.contiguous_format)
    oq2, ok2 = gguf_hip.qk_norm_rope(q, k, pos, table, wq, wk, v=v, k_pages=kp, v_pages=vp, slots=slots, k_scale=ks, v_scale=vs,
                                     out_k=mine)
    assert ok2 is mine and torch.equal(oq, oq2)
    assert torch.equal(kp.view(torch.uint8), kp2.view(torch.uint8)) and torch.equal(vp.view(torch.uint8), vp2.view(torch.uint8))
    assert torch.equal(mine, gguf_hip.qk_norm_rope(q, k, pos, table, wq, wk)[1])


def test_rope_bad_positions_and_slots():
    gen = _gen(3)
    q, k, v, table, pos, wq, wk = _rope_case(gen, 6, 4, 2, 64, BF, 32, BF)
    kp, vp = (torch.zeros((3, 8, 2, 64), dtype=BF, device="cuda") for _ in range(2))
    good = gguf_hip.qk_norm_rope(q, k, pos, table, wq, wk)
    pos[1], pos[2] = -1, 500
    slots = torch.tensor([0, 1, 2, 24, 2 ** 40, 5], device="cuda")
    out_k = torch.empty_like(k, memory_format=torch.contiguous_format)
    oq, ok = gguf_hip.qk_norm_rope(q, k, pos, table, wq, wk, v=v, k_pages=kp, v_pages=vp, slots=slots, out_k=out_k)
    for got, want in ((oq, good[0]), (ok, good[1])):
        assert got[1:3].isnan().all() and torch.equal(got[0], want[0]) and torch.equal(got[3:], want[3:])
    flat = kp.view(24, 2, 64)
    assert torch.equal(flat[0], ok[0]) and torch.equal(flat[5], ok[5]) and flat[1:3].isnan().all()
    assert not flat[3:5].any() and not flat[6:].any() and torch.equal(vp.view(24, 2, 64)[1], v[1])


def test_rope_in_place_views_and_graph():
    gen = _gen(4)
    q, k, v, table, pos, wq, wk = _rope_case(gen, 9, 6, 2, 128, BF, 128, torch.float32)
    want = gguf_hip.qk_norm_rope(q, k, pos, table, wq, wk)
    for interleaved in (False, True):
        want = gguf_hip.qk_norm_rope(q, k, pos, table, wq, wk, interleaved=interleaved)
        q2, k2 = q.clone(), k.clone()
        oq, ok = gguf_hip.qk_norm_rope(q2, k2, pos, table, wq, wk, interleaved=interleaved, out_q=q2, out_k=k2)
        assert oq is q2 and ok is k2 and torch.equal(q2, want[0]) and torch.equal(k2, want[1])
    want = gguf_hip.qk_norm_rope(q, k, pos, table, wq, wk)
    odd = torch.zeros(9 * 6 * 128 + 3, dtype=BF, device="cuda")[3:].view(9, 6, 128)
    odd.copy_(q)
    assert torch.equal(gguf_hip.qk_norm_rope(odd, k, pos, table, wq, wk)[0], want[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gguf_hip.qk_norm_rope(q, k, pos, table, wq, wk)
    for step in range(3):
        q.copy_(_randn(_gen(step), 9, 6, 128))
        pos.copy_(torch.randint(0, 500, (9,), device="cuda", generator=_gen(step)))
        graph.replay()
        torch.cuda.synchronize()
        want = gguf_hip.qk_norm_rope(q, k, pos, table, wq, wk)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_rope_many_tokens():
    """More tokens than a grid's second dimension, against a part of them alone."""
    gen = _gen(5)
    n = 66_001
    q = _randn(gen, n, 1, 64, dtype=BF)
    k = _randn(gen, n, 1, 64, dtype=BF)
    table = gguf_hip.rope_table(64, 1000)
    pos = torch.arange(n, device="cuda") % 1000
    oq, ok = gguf_hip.qk_norm_rope(q, k, pos, table)
    for x, got in ((q, oq), (k, ok)):
        want, size = _rope_exact(x, None, pos, table, 64, 0, False, False)
        _within(got, want, _rope_tol(want, size, BF, 64), n)


# ---- adapters --------------------------------------------------------------------------------

def _lora_case(gen, M, K, n_outs, rank, slots, dtype):
    y = _randn(gen, M, sum(n_outs), dtype=dtype)
    x = _randn(gen, M, K, dtype=dtype)
    a = (_randn(gen, slots, len(n_outs), rank, K) * K ** -0.5).to(dtype)
    b = _randn(gen, slots, sum(n_outs), rank, dtype=dtype)
    return y, x, a, b, 0.25 + torch.rand(slots, device="cuda", generator=gen)


def _lora_exact(y, x, a, b, ids, scales, n_outs):
    """(out, its bound) in 64 bits: h's K products in fp32, kept to 2^-16, rank products in fp32, one rounding."""
    out, tol = y.double(), torch.zeros(y.shape, dtype=torch.float64, device="cuda")
    K, rank = x.shape[1], a.shape[2]
    for i in set(ids.tolist()):
        if i < 0:
            continue
        rows = (ids == i).nonzero()[:, 0]
        s = 1.0 if scales is None else float(scales[i])
        col = 0
        for p, n in enumerate(n_outs):
            A, B, X = a[i, p].double(), b[i, col:col + n].double(), x[rows].double()
            h, ha = X @ A.t(), X.abs() @ A.abs().t()
            out[rows, col:col + n] += s * (h @ B.t())
            e = (2.0 ** -16 + rank * E32) * h.abs() + K * E32 * ha
            tol[rows, col:col + n] = abs(s) * ((e @ B.abs().t()) + 4 * E32 * (h.abs() @ B.abs().t()))
            col += n
    u = U[y.dtype]
    return out, (1 + u) * (tol + 2 * E32 * y.double().abs()) + u * out.abs() + TINY[y.dtype] + 1e-30


def _lora_check(seed, M, K, n_outs, rank, slots, dtype, ids=None, scaled=True):
    gen = _gen(seed)
    y, x, a, b, scales = _lora_case(gen, M, K, n_outs, rank, slots, dtype)
    if ids is None:
        ids = torch.randint(-1, slots, (M,), device="cuda", generator=gen)
    scales = scales if scaled else None
    out = gguf_hip.lora_add(y, x, a, b, ids, scales, n_outs)
    want, tol = _lora_exact(y, x, a, b, ids, scales, n_outs)
    _within(out, want, tol, (M, K, n_outs, rank))
    none = ids < 0
    assert torch.equal(out[none], y[none])
    assert torch.equal(out, gguf_hip.lora_add(y, x, a, b, ids, scales, n_outs))
    return y, x, a, b, ids, scales, out


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40, 64, 128, 256])
@pytest.mark.parametrize("n_outs", [(96,), (64, 40, 24), (1, 130, 17, 3)])
def test_lora_ranks_and_parts(dtype, rank, n_outs):
    _lora_check(rank, 19, 264, n_outs, rank, 5, dtype)


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 63, 64, 65, 130, 500, 1030])
@pytest.mark.parametrize("K", [8, 40, 512, 5120])
def test_lora_rows_and_depth(M, K):
    _lora_check(M + K, M, K, (200, 56), 16, 9, BF)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("rank", [8, 24, 32, 72, 256])
@pytest.mark.parametrize("n_outs", [(264, 3), (53_000, 7_000)])
def test_lora_prompts(dtype, rank, n_outs):
    """Long batches of few and of many columns, whose rows come mixed or in runs."""
    _lora_check(rank, 300, 136, n_outs, rank, 4, dtype)
    _lora_check(rank, 300, 136, n_outs, rank, 4, dtype, torch.arange(300, device="cuda") // 90)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("rank", [8, 16, 24, 32])
@pytest.mark.parametrize("M", [7, 17, 63, 64, 65, 200])
def test_lora_many_columns(dtype, rank, M):
    """Rows that share adapters, and more columns than a row alone would take."""
    _lora_check(M, M, 520, (9000, 805), rank, 6, dtype)
    dev = "cuda"
    for ids in (torch.zeros(M, dtype=torch.int32, device=dev), torch.full((M,), -1, device=dev),
                torch.arange(M, device=dev).flip(0) % 6, torch.arange(M, device=dev) // 20 % 6):
        _lora_check(M, M, 520, (9000, 805), rank, 6, dtype, ids)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("M,K,n_outs,rank", [(1, 8192, (1000,), 16), (1, 8200, (1000,), 16), (1, 4096, (300, 7, 1), 32), (5, 504, (257,), 8),
                                             (4, 1024, (256, 1), 32), (3, 16384, (511,), 8), (120, 8, (513,), 16)])
def test_lora_few_rows(dtype, M, K, n_outs, rank):
    """Rows by themselves: K that ends inside a run, columns that end inside a workgroup, every kind of id, strides."""
    y, x, a, b, ids, scales, out = _lora_check(M + K, M, K, n_outs, rank, 3, dtype)
    N = sum(n_outs)
    wide = torch.full((M, N + 40), 7.0, dtype=dtype, device="cuda")
    wide[:, 3:N + 3] = y
    wx = torch.zeros((M, K + 16), dtype=dtype, device="cuda")
    wx[:, 8:K + 8] = x
    got = wide[:, 3:N + 3]
    gguf_hip.lora_add(got, wx[:, 8:K + 8], a, b, ids, scales, n_outs, out=got)
    assert torch.equal(got, out) and (wide[:, :3] == 7).all() and (wide[:, N + 3:] == 7).all()
    bad = gguf_hip.lora_add(y, x, a, b, torch.full((M,), 3, device="cuda"), scales, n_outs)
    assert bad.isnan().all()


@pytest.mark.parametrize("M", [1, 3, 40, 300])
def test_lora_into_its_input(M):
    """out may be y, and where the sizes allow it x."""
    y, x, a, b, ids, scales, out = _lora_check(M, M, 1024, (1000, 24), 16, 3, BF)
    want, tol = _lora_exact(y, x, a, b, ids, scales, (1000, 24))
    mine = x.clone()
    gguf_hip.lora_add(y, mine, a, b, ids, scales, (1000, 24), out=mine)
    _within(mine, want, tol, "into x")   # its sums may go in another order
    mine = y.clone()
    gguf_hip.lora_add(mine, x, a, b, ids, scales, (1000, 24), out=mine)
    assert torch.equal(mine, out)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("M,K,n_outs,rank", [(2100, 5120, (200, 56), 16), (4100, 2600, (136,), 64), (4097, 1296, (70_000,), 8),
                                             (8200, 1024, (40, 40, 8), 40)])
def test_lora_long_prompts(dtype, M, K, n_outs, rank):
    """Blocks of rows that begin with one adapter or with none and hold one or more others, cut over K in two ways."""
    _lora_check(M, M, K, n_outs, rank, 5, dtype)
    for ids in (torch.arange(M, device="cuda") // 700 % 5, torch.arange(M, device="cuda") // 31 % 6 - 1,
                (torch.arange(M, device="cuda") % 64 == 63).long() * 2 - 1):
        _lora_check(M, M, K, n_outs, rank, 5, dtype, ids)


def test_lora_batches():
    """One adapter for all rows, none for any, all rows different, runs of rows, ids of either width, no scales."""
    dev = "cuda"
    for ids in (torch.zeros(70, dtype=torch.int32, device=dev), torch.full((70,), -1, device=dev),
                torch.arange(70, device=dev).flip(0), torch.arange(70, device=dev) // 20,
                torch.arange(70, dtype=torch.int32, device=dev) % 3 - 1):
        _lora_check(1, 70, 1024, (300,), 16, 70, BF, ids)
    _lora_check(2, 33, 256, (64, 64), 32, 4, F16, scaled=False)
    long = torch.cat([torch.full((n,), i, device=dev) for i, n in ((2, 700), (-1, 5), (0, 333), (1, 1), (2, 60), (3, 400))])
    _lora_check(3, long.numel(), 640, (128, 72), 24, 4, BF, long)


def test_lora_bad_ids_and_empty():
    gen = _gen(4)
    y, x, a, b, scales = _lora_case(gen, 20, 128, (32, 16), 16, 3, BF)
    ids = torch.arange(20, device="cuda") % 3
    good = gguf_hip.lora_add(y, x, a, b, ids, scales, (32, 16))
    ids[4], ids[9], ids[13] = 3, 2 ** 40, -(2 ** 40)
    out = gguf_hip.lora_add(y, x, a, b, ids, scales, (32, 16))
    assert out[4].isnan().all() and out[9].isnan().all() and torch.equal(out[13], y[13])
    rest = [i for i in range(20) if i not in (4, 9, 13)]
    assert torch.equal(out[rest], good[rest])
    assert gguf_hip.lora_add(y[:0], x[:0], a, b, ids[:0], scales, (32, 16)).shape == (0, 48)
    none = gguf_hip.lora_add(y, x, a[:0], b[:0], torch.full((20,), -1, device="cuda"), scales[:0], (32, 16))
    assert torch.equal(none, y)


def test_lora_not_finite():
    """Infinities and NaN in a row of x, in y, and in an adapter that other rows use: they stay in their rows."""
    gen = _gen(5)
    y, x, a, b, scales = _lora_case(gen, 24, 256, (40,), 16, 3, F16)
    ids = torch.arange(24, device="cuda") % 3
    a[:, :, 0, 3] = 1.0
    good = gguf_hip.lora_add(y, x, a, b, ids, scales, (40,))
    x[4, 3], x[7, 3], y[10, 5] = float("inf"), float("nan"), float("inf")
    a[2, 0, 1, 0] = float("nan")
    out = gguf_hip.lora_add(y, x, a, b, ids, scales, (40,))
    want, _ = _lora_exact(y, x, a, b, ids, scales, (40,))
    assert torch.equal(out[4].isnan(), want[4].isnan()) and not out[4].isfinite().any() and out[7].isnan().all()
    assert out[10, 5] == float("inf") and torch.equal(out[10, :5], good[10, :5])
    assert out[2::3].isnan().all()
    keep = [i for i in range(24) if i % 3 != 2 and i not in (4, 7, 10)]
    assert torch.equal(out[keep], good[keep])


def test_lora_large_and_small_values():
    """h beyond what fp16 holds, and far below: it is kept in 32 bits."""
    gen = _gen(6)
    y, x, a, b, scales = _lora_case(gen, 20, 512, (64,), 16, 2, F16)
    ids = torch.arange(20, device="cuda") % 2
    for fx, fb in ((300.0, 2.0 ** -9), (2.0 ** -9, 1.0)):
        X, Aa, Bb = (x * fx).clamp(-6e4, 6e4), a * (fx if fx > 1 else 2.0 ** -6), b * fb
        out = gguf_hip.lora_add(y, X, Aa, Bb, ids, scales, (64,))
        want, tol = _lora_exact(y, X, Aa, Bb, ids, scales, (64,))
        big = want.abs() > 65000
        _within(out.masked_fill(big, 0), want.masked_fill(big, 0), tol, fx)


def test_lora_in_place_views_streams_and_graph():
    gen = _gen(7)
    y, x, a, b, scales = _lora_case(gen, 21, 256, (40, 24), 16, 3, BF)
    ids = torch.arange(21, device="cuda") % 4 - 1
    want = gguf_hip.lora_add(y, x, a, b, ids, scales, (40, 24))
    y2 = y.clone()
    assert gguf_hip.lora_add(y2, x, a, b, ids, scales, (40, 24), out=y2) is y2 and torch.equal(y2, want)
    wide = torch.zeros(21, 101, dtype=BF, device="cuda")                     # an odd stride and an odd first column
    wide[:, 33:97] = y
    gguf_hip.lora_add(wide[:, 33:97], x, a, b, ids, scales, (40, 24), out=wide[:, 33:97])
    assert torch.equal(wide[:, 33:97], want) and not wide[:, :33].any() and not wide[:, 97:].any()
    xs = torch.zeros(21, 512, dtype=BF, device="cuda")
    xs[:, 8:264] = x
    assert torch.equal(gguf_hip.lora_add(y, xs[:, 8:264], a, b, ids, scales, (40, 24)), want)
    assert torch.equal(gguf_hip.lora_add(y.t().contiguous().t(), x.t().contiguous().t(), a, b, ids, scales, (40, 24)), want)
    one = torch.zeros(2, 513, dtype=BF, device="cuda")
    one[:1, :256] = x[:1]
    assert torch.equal(gguf_hip.lora_add(y[:1], one[:1, :256], a, b, ids[:1] + 1, scales, (40, 24)),
                       gguf_hip.lora_add(y[:1], x[:1], a, b, ids[:1] + 1, scales, (40, 24)))
    side, ws = torch.cuda.Stream(), torch.zeros(1 << 20, dtype=torch.int32, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = gguf_hip.lora_add(y, x, a, b, ids, scales, (40, 24), workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gguf_hip.lora_add(y, x, a, b, ids, scales, (40, 24))
    for step in range(3):                                                    # other adapters in every replay
        ids.copy_(torch.randint(-1, 3, (21,), device="cuda", generator=_gen(step)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, gguf_hip.lora_add(y, x, a, b, ids, scales, (40, 24)))


def test_lora_small_workspace_goes_in_turns():
    gen = _gen(8)
    y, x, a, b, scales = _lora_case(gen, 600, 512, (64, 64), 64, 3, BF)
    ids = torch.randint(-1, 3, (600,), device="cuda", generator=gen)
    want, tol = _lora_exact(y, x, a, b, ids, scales, (64, 64))
    from gguf_hip._lib import GQK_CTR_BYTES, lib

    need = max(lib.gqk_lora_workspace_bytes(m, 512, 2, 64) for m in range(1, 65))
    assert need < lib.gqk_lora_workspace_bytes(600, 512, 2, 64) and need > GQK_CTR_BYTES
    ws = torch.zeros(need // 4, dtype=torch.int32, device="cuda")
    _within(gguf_hip.lora_add(y, x, a, b, ids, scales, (64, 64), workspace=ws), want, tol, "in turns")
    with pytest.raises(ValueError):
        gguf_hip.lora_add(y, x, a, b, ids, scales, (64, 64), workspace=ws[:1024])


# ---- page copies -----------------------------------------------------------------------------

@pytest.mark.parametrize("shape,dim,dtype", [
    ((2, 3, 40, 4, 16, 64), 2, BF), ((64, 8, 2, 80), 0, BF), ((5, 40, 1000), 1, torch.uint8), ((5, 40, 999), 1, torch.uint8),
    ((3, 30, 250), 1, torch.int32), ((1, 12, 1), 1, torch.float32), ((300, 2, 8), 1, F8), ((40, 3), 0, torch.float64),
    ((2, 20, 20000), 1, torch.int16)])
def test_copy_pages(shape, dim, dtype):
    gen = torch.Generator().manual_seed(len(shape))
    raw = torch.randint(0, 256, (*shape[:-1], shape[-1] * dtype.itemsize), dtype=torch.uint8, generator=gen)
    pages, want = raw.cuda().view(dtype), raw.clone()
    order = torch.randperm(shape[dim], generator=gen)
    n = shape[dim] // 2
    src, dst = order[:n], order[n:2 * n]
    src = src[torch.randint(0, n, (n,), generator=gen)]                      # a source may be read many times
    want.index_copy_(dim, dst, raw.index_select(dim, src))
    gguf_hip.copy_pages(pages, src, dst, dim=dim)
    assert torch.equal(pages.view(torch.uint8).cpu(), want)
    gguf_hip.copy_pages(pages, [], [], dim=dim)
    gguf_hip.copy_pages(pages, dst.tolist()[:1], src.numpy()[:1], dim=dim - len(shape))
    want.index_copy_(dim, src[:1], want.index_select(dim, dst[:1]))
    assert torch.equal(pages.view(torch.uint8).cpu(), want)


def test_copy_pages_many_pairs_and_refusals():
    """More pairs than one launch's arguments hold; nothing is copied where a pair is refused."""
    pages = torch.arange(3 * 4000, device="cuda", dtype=torch.int32).view(3, 4000, 1).expand(3, 4000, 8).contiguous()
    want = pages.clone()
    perm = torch.randperm(4000, generator=torch.Generator().manual_seed(0))
    src, dst = perm[:2000], perm[2000:]
    want[:, dst] = want[:, src]
    gguf_hip.copy_pages(pages, src, dst, dim=1)
    assert torch.equal(pages, want)
    for s, d in (([0, 1], [2, 4000]), ([-1], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 5]), ([0], [1, 2]), ([2 ** 40], [0]), ([0.5], [1])):
        with pytest.raises(ValueError):
            gguf_hip.copy_pages(pages, s, d, dim=1)
    with pytest.raises(ValueError):
        gguf_hip.copy_pages(pages, src.cuda(), dst.cuda(), dim=1)
    with pytest.raises(ValueError):
        gguf_hip.copy_pages(pages.transpose(0, 2), [0], [1], dim=1)
    with pytest.raises(ValueError):
        gguf_hip.copy_pages(pages, [0], [1], dim=3)
    assert torch.equal(pages, want)


def test_copy_pages_views_and_graph():
    store = torch.zeros(4, 10, 24, dtype=torch.int16, device="cuda")
    store.copy_(torch.arange(960).view(4, 10, 24))
    want = store.clone()
    part = store[1:, :, :16].unflatten(2, (2, 8))                            # planes apart, pages with a gap
    want[1:, 3, :16] = want[1:, 7, :16]
    gguf_hip.copy_pages(part, [7], [3], dim=1)
    assert torch.equal(store, want)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        gguf_hip.copy_pages(store, [0, 1], [8, 9], dim=1)
    for step in range(3):
        store[:, :2] = step + 1
        graph.replay()
        torch.cuda.synchronize()
        assert (store[:, 8:] == step + 1).all() and torch.equal(store[:, 2:8], want[:, 2:8])


# ---- the eager way ---------------------------------------------------------------------------

def _eager_calls():
    """Arguments of each function of the eager calls' module, as the Python functions pass them."""
    gen = _gen(1)
    k, v, table = _cache(gen, [70, 40], 16, 2, 64, BF, "heads", poison=False)
    q = _randn(gen, 2, 8, 64, dtype=BF)
    n = torch.tensor([70, 40], dtype=torch.int32, device="cuda")
    attend = [q, k, v, table, n, None, 0, None, None, None, None, True, None]
    hq, hk, hv, rt, pos, wq, wk = _rope_case(gen, 3, 4, 2, 64, BF, 64, BF)
    rope = [hq, hk, pos, rt, wq, wk, 1e-6, 0, hv, k, v, torch.tensor([0, 1, 2], device="cuda"), None, None, None, None]
    y, x, a, b, scales = _lora_case(gen, 5, 64, (16, 24), 8, 2, F16)
    lora = [y, x, a, b, torch.tensor([0, 1, -1, 0, 1], device="cuda"), scales, (16, 24), None, None]
    return {"paged_attention": attend, "qk_norm_rope": rope, "lora_add": lora, "copy_pages": [k.transpose(1, 2), [0], [1], 0]}


@pytest.mark.parametrize("name", ["paged_attention", "qk_norm_rope", "lora_add", "copy_pages"])
def test_eager_calls_are_taken_and_step_aside(name):
    """A plain call is served without the Python path; a subclass, lazy negation, autograd, a mode, a profiler or a
    functorch transform sends it there (None, and nothing written)."""
    from torch.overrides import TorchFunctionMode
    from torch.utils._python_dispatch import TorchDispatchMode

    from gguf_hip import _lib, ops

    ops.shared_workspace(torch.device("cuda", 0))
    args = _eager_calls()[name]
    call = getattr(_lib._fast, name)
    assert call(*args) is not None
    before = args[0].clone()

    class Sub(torch.Tensor):
        pass

    class Function(TorchFunctionMode):
        pass

    class Dispatch(TorchDispatchMode):
        pass

    assert call(args[0].as_subclass(Sub), *args[1:]) is None
    assert call(torch._neg_view(args[0]), *args[1:]) is None
    assert call(args[0].cpu(), *args[1:]) is None and call(None, *args[1:]) is None
    assert call(args[0].detach().requires_grad_(), *args[1:]) is None
    with torch.no_grad():
        assert call(args[0].detach().requires_grad_(), *args[1:]) is not None
    for mode in (Function(), Dispatch(), torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU])):
        with mode:
            assert call(*args) is None
    seen = []
    torch.func.vmap(lambda t: seen.append(call(*args)) or t)(torch.zeros(2, 1, device="cuda"))
    assert seen == [None]
    with torch.inference_mode():
        assert call(*args) is not None
    assert call(*args[:-1]) is None                          # another number of arguments
    assert call(*args) is not None
    if name == "copy_pages":
        assert call(args[0], [0], [0], 0) is None and call(args[0], [0, 2], [1, 1], 0) is None and call(args[0], [0], [99], 0) is None
    assert torch.equal(before, args[0])


def test_eager_calls_agree_with_the_ops():
    """The same bits through the eager module, the Python path and the registered ops; versions are bumped."""
    from gguf_hip import adapters, attention

    e = _eager_calls()
    q, k, v, table, n = e["paged_attention"][:5]
    out, lse = gguf_hip.paged_attention(q, k, v, table, n, return_lse=True)
    o2, l2 = torch.empty_like(out), torch.empty_like(lse)
    attention._attention_op(q, k, v, table, n, 0.125, 0, None, None, 80, o2, l2, None)
    assert torch.equal(out, o2) and torch.equal(lse, l2)
    o3 = torch.empty_like(out)
    version = o3._version
    gguf_hip.paged_attention(q, k, v, table, n, out=o3)
    assert o3._version > version and torch.equal(o3, out)
    y, x, a, b, ids, scales, outs = e["lora_add"][:7]
    out = gguf_hip.lora_add(y, x, a, b, ids, scales, outs)
    o2 = torch.empty_like(out)
    adapters._lora_op(y, x, a, b, ids, scales, list(outs), o2, None)
    assert torch.equal(out, o2)
    hq, hk, pos, rt, wq, wk = e["qk_norm_rope"][:6]
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        through_op = gguf_hip.qk_norm_rope(hq, hk, pos, rt, wq, wk)
    assert any("qk_norm_rope" in ev.key for ev in prof.key_averages())
    eager = gguf_hip.qk_norm_rope(hq, hk, pos, rt, wq, wk)
    assert torch.equal(eager[0], through_op[0]) and torch.equal(eager[1], through_op[1])


# ---- all together ----------------------------------------------------------------------------

def test_decode_step_example():
    """examples/decode_step.py: prompts, steps by a graph, a fork, a compaction.  Per layer a token's value is rounded at most eight
    times on its way (projection, adapter, heads, cache, probabilities, attention, projection, adapter), weights once, each at
    most 2^-8 of it: two layers stay within 18 * 2^-8."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "decode_step.py")
    spec = importlib.util.spec_from_file_location("decode_step", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    got = module.run(steps=6)
    assert sorted(got["errors"]) == ["a", "b", "c", "d"] and got["moved"] > 0
    assert max(got["errors"].values()) < 18 * 2.0 ** -8, got
