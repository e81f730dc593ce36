"""The operators of steps of several new tokens and of long caches on the GPU, each against its definition in 64 bits (plain torch on the
CPU or the GPU, written here).  Tolerances are bounds per value, from the roundings that the operators are allowed: u is half a step of a
type (2^-8 of a bf16 value, 2^-11 of an fp16 one, 2^-4 of an e4m3 one), sums and products are fp32 (2^-24 of each)."""
import pytest
import torch

import gguf_hip
from gguf_hip import _lib

pytestmark = pytest.mark.gpu

BF, F16, F32, F8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
U = {BF: 2.0 ** -8, F16: 2.0 ** -11, F8: 2.0 ** -4}
TINY = {BF: 0.0, F16: 2.0 ** -25, F8: 2.0 ** -10}     # half of the smallest step, where a type's range ends
E32 = 2.0 ** -24
NAN, INF = float("nan"), float("inf")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, dtype=torch.float32):
    return torch.randn(shape, device="cuda", generator=gen).to(dtype)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _bytes(t):
    return t.view(torch.uint8) if t.dtype == F8 else t


def _within(got, want, tol, what):
    got, want = got.double(), want.double()
    bad = ~((got - want).abs() <= tol) & ~(got.isnan() & want.isnan()) & ~(got == want)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4], want[bad][:4], (tol + 0 * want)[bad][:4])


# ---- tables of a step --------------------------------------------------------------------------

def _tables_exact(lists, requests, lengths, counts, tokens, page, parents, tree):
    """By its definition, one token after the other (the CPU's lists)."""
    n_lists, width = len(lists), len(lists[0]) if lists else 0
    words = -(-tree // 32)
    block, totals, starts = [], [], [0]
    seq, pos, slot, mask = [-1] * tokens, [0] * tokens, [-1] * tokens, [[0] * words for _ in range(tokens)]
    at = 0
    for b, (r, m, n) in enumerate(zip(requests, lengths, counts)):
        k = max(n, 0)
        sound = (0 <= r < n_lists and m >= 0 and n >= 0 and m + n <= width * page and at + k <= tokens and (tree == 0 or n <= tree))
        totals.append(0 if r < 0 and k == 0 else m + n if sound else 2 ** 31 - 1)
        pages = -(-(m + n) // page) if sound else 0
        block.append([lists[r][j] if j < pages else -1 for j in range(width)])
        seen = []
        for i in range(min(k, max(0, tokens - at))):
            t = at + i
            seq[t], pos[t] = b, -1
            if not sound:
                continue
            p = lists[r][(m + i) // page]
            slot[t], pos[t] = -1 if p < 0 else p * page + (m + i) % page, m + i
            if tree:
                up = parents[t]
                bits = None if up < -1 or up >= i or (up >= 0 and seen[up] is None) else (seen[up] if up >= 0 else 0) | 1 << i
                seen.append(bits)
                pos[t] = -1 if bits is None else m + bin(bits).count("1") - 1
                mask[t] = [((bits or 0) >> 32 * w) & 0xFFFFFFFF for w in range(words)]
        at += k
        starts.append(min(at, tokens))
    return block, totals, starts, seq, pos, slot, mask


def _tables_check(lists, requests, lengths, counts, tokens, page, parents=None, tree=0, wide=False):
    g = torch.tensor(lists, dtype=torch.int32, device="cuda").reshape(len(lists), len(lists[0]) if lists else 0)
    got = gguf_hip.step_tables(g, _i32(requests).to(torch.int64 if wide else torch.int32), _i32(lengths), _i32(counts), tokens, page,
                               parents=None if parents is None else _i32(parents), tree=tree)
    want = _tables_exact(lists, requests, lengths, counts, tokens, page, parents, tree)
    for name, w in zip(got._fields, want):
        t = getattr(got, name)
        if name == "mask" and not tree:
            assert t is None
            continue
        w = torch.tensor(w, dtype=torch.int64).reshape(t.shape)
        t = t.cpu().long() & 0xFFFFFFFF if name == "mask" else t.cpu().long()
        assert torch.equal(t, w), (name, t[t != w][:5], w[t != w][:5])
    assert got.slots.dtype == torch.int64 and all(getattr(got, n).dtype == torch.int32 for n in got._fields if n != "slots" and getattr(got, n) is not None)
    return got


def _tables_case(rng, batch, page, most, tree, pad):
    lengths = [int(rng.integers(0, 5 * page + 7)) for _ in range(batch)]
    counts = [int(rng.integers(0, most + 1)) for _ in range(batch)]
    if batch > 2:
        counts[1], lengths[0] = 0, 0
    width = max([-(-(m + n) // page) for m, n in zip(lengths, counts)] + [1]) + 2
    slots = batch + 3
    lists = rng.permutation(slots * width).reshape(slots, width).tolist()
    requests = rng.permutation(slots)[:batch].tolist()
    if batch > 4:
        requests[3], counts[3] = -1, 0
    tokens = sum(counts) + pad
    parents = None
    if tree:
        parents = [max(-1, i - 1 - int(rng.integers(0, 4))) for n in counts for i in range(n)] + [-1] * pad
    return lists, requests, lengths, counts, tokens, page, parents, tree


@pytest.mark.parametrize("batch", [1, 2, 5, 70, 300])
@pytest.mark.parametrize("page", [1, 7, 16, 64])
@pytest.mark.parametrize("most,tree", [(1, 0), (9, 0), (400, 0), (1, 1), (16, 16), (33, 64), (40, 33), (150, 150)])
def test_tables(batch, page, most, tree):
    import numpy as np

    rng = np.random.default_rng(batch * 1000 + page + most)
    for pad in (0, 77):
        _tables_check(*_tables_case(rng, batch, page, most, tree, pad), wide=bool(pad))


def test_tables_of_many_tokens_and_wide_lists():
    """More columns and tokens than one workgroup takes, a tree of the most tokens, a chain of ancestors as long."""
    import numpy as np

    rng = np.random.default_rng(1)
    lists = rng.permutation(3 * 9000).reshape(3, 9000).tolist()
    _tables_check(lists, [2, 0], [0, 140_000], [3000, 1700], 5000, 16)
    for parents in (list(range(-1, 1023)), [-1] * 1024, [max(-1, (i - 1) // 2) for i in range(1024)]):
        _tables_check(lists, [1], [100], [1024], 1030, 16, parents + [-1] * 6, 1024)


def test_tables_of_what_cannot_be():
    """A request that has no list, negative and too long lengths, negative counts, more tokens than rows or than a tree's: that sequence
    alone is given up, the others are as they would be."""
    lists = [[3, 1, 4], [15, 9, 2], [6, 5, 35]]
    for r, m, n in ((3, 4, 2), (-1, 4, 2), (2 ** 31 - 1, 0, 1), (1, -1, 2), (1, 11, 2), (1, 2 ** 31 - 1, 1), (1, 4, -3)):
        _tables_check(lists, [0, r, 2], [5, m, 0], [3, n, 4], 10, 4)
        _tables_check(lists, [0, r, 2], [5, m, 0], [3, n, 4], 10, 4, [-1, 0, 0, -1, 0, 1, 2, -1, 0, 1], 4)
    for tokens in (0, 2, 3, 6, 7, 9):
        _tables_check(lists, [0, 1, 2], [5, 2, 0], [3, 3, 3], tokens, 4)
    _tables_check(lists, [0, 1, 2], [5, 2, 0], [3, 5, 3], 11, 4, [-1, 0, 1, -1, 0, 1, 2, 3, -1, -1, 1], 4)
    _tables_check(lists, [0, 1], [0, 0], [2 ** 31 - 1, 2 ** 31 - 1], 3, 4)
    _tables_check([[3, -1, 4]], [0], [2], [8], 9, 4)                      # a page that the server has not given yet
    _tables_check([], [0], [2], [1], 2, 4)


@pytest.mark.parametrize("parents", [[-1, 0, 2, 0], [-1, 0, 3, 2], [0, 0, 1, 1], [-2, -1, 0, 1], [-1, 2 ** 31 - 1, 1, -2 ** 31], [5, 0, 1, 2]])
def test_tables_parents_that_come_after(parents):
    _tables_check([[3, 1, 4]], [0], [2], [4], 6, 4, parents + [-1, -1], 40)


def test_tables_strides_streams_and_empty_batches():
    lists = torch.arange(60, dtype=torch.int32, device="cuda").view(6, 10)[1::2, 2:7]
    want = gguf_hip.step_tables(lists.contiguous(), _i32([2, 0]), _i32([5, 9]), _i32([3, 2]), 8, 4)
    got = gguf_hip.step_tables(lists, _i32([2, 0]), _i32([5, 9]), _i32([3, 2]), 8, 4)
    assert all(torch.equal(a, b) for a, b in zip(got[:6], want[:6])) and want.block_table[0, 0] == 52
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = gguf_hip.step_tables(lists, _i32([2, 0]), _i32([5, 9]), _i32([3, 2]), 8, 4)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got[:6], want[:6]))
    none = gguf_hip.step_tables(lists, _i32([]), _i32([]), _i32([]), 3, 4)
    assert none.starts.tolist() == [0] and none.sequences.tolist() == [-1] * 3 and none.slots.tolist() == [-1] * 3
    assert none.block_table.shape == (0, 5) and none.positions.tolist() == [0] * 3


# ---- residual and norm ------------------------------------------------------------------------

def _norm_exact(x, r, w, eps, offset):
    """(s, normed, the size of its error before it is rounded): a sum of dim squares in fp32, its root, four products."""
    s = x.double() + (0 if r is None else r.double())
    y = s / (s.square().mean(1, keepdim=True) + eps).sqrt()
    if w is not None:
        y = y * (w.double() + (1 if offset else 0))
    return s, y, (x.shape[1] / 2 + 16) * E32 * y.abs()


def _norm_check(seed, rows, dim, dtype, weight, offset=False, residual=True, groups=(None, 0)):
    gen = _gen(seed)
    x, r = _randn(gen, rows, dim, dtype=dtype), _randn(gen, rows, dim, dtype=dtype) * 3
    r = r if residual else None
    w = None if weight is None else _randn(gen, dim, dtype=weight)
    s, y, e = _norm_exact(x, r, w, 1e-5, offset)
    u = U[dtype]
    for group in groups:
        if group is None:
            out, res = gguf_hip.add_rms_norm(x, r, w, eps=1e-5, unit_offset=offset)
            _within(out, y, (1 + u) * e + u * y.abs() + TINY[dtype], (rows, dim))
        else:
            out, scale, res = gguf_hip.add_rms_norm_fp8(x, r, w, eps=1e-5, unit_offset=offset, group=group)
            parts = y.unflatten(1, (-1, group or dim))
            top = parts.abs().amax(2).clamp_min(2.0 ** -100)
            ep = (dim / 2 + 20) * E32                                     # of a value, and so of the largest
            _within(scale, top / 448, (ep + 2 * E32) * top / 448, "scale")
            per = scale.double().repeat_interleave(group or dim, 1)
            want = y / per
            _within(out, want.clamp(-448, 448), (1 + U[F8]) * (e / per + 4 * E32 * want.abs()) + U[F8] * want.abs() + TINY[F8], (rows, dim, group))
            assert not out.float().isnan().any() and (parts.abs().amax(2) == 0).logical_or(
                out.float().abs().unflatten(1, (-1, group or dim)).amax(2) >= 416).all()        # the range is used
        if r is None:
            assert res is None
        else:
            _within(res, s, u * s.abs() + TINY[dtype], "residual")


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("dim", [1, 7, 8, 63, 64, 100, 511, 513, 1000, 2048, 2049, 5120, 5121, 8192, 10240, 17408, 20481, 32768])
def test_norm_dims(dtype, dim):
    _norm_check(dim, 3, dim, dtype, dtype)


@pytest.mark.parametrize("rows", [1, 2, 5, 511, 512, 700, 2047, 2049, 4099])
@pytest.mark.parametrize("dim", [40, 511, 1024, 5120])
def test_norm_rows(rows, dim):
    _norm_check(rows, rows, dim, BF, BF)


@pytest.mark.parametrize("weight,offset", [(None, False), (F32, False), (F32, True), (BF, True), (BF, False)])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,dim", [(4, 1001), (600, 5120), (2100, 264)])
def test_norm_weights(weight, offset, residual, rows, dim):
    _norm_check(dim, rows, dim, BF, weight, offset, residual)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("group", [32, 64, 128, 256, 512])
@pytest.mark.parametrize("rows,dim", [(1, 512), (3, 5120), (700, 5632), (2100, 1024), (96, 17408), (2, 32768)])
def test_norm_groups(dtype, group, rows, dim):
    _norm_check(group, rows, dim, dtype, F32, True, groups=(group,))


def test_norm_rows_of_zeros_and_of_what_is_not_finite():
    """A row of zeros is zeros with a scale that is a number; a NaN or an infinity makes its row NaN, or where only a group's scale
    is asked its whole row still; other rows are as they are."""
    for dtype in (BF, F16):
        x = _randn(_gen(1), 5, 256, dtype=dtype)
        r = torch.zeros_like(x)
        x[1], x[2, 7], x[3, 200], x[4, 3] = 0, NAN, INF, -INF
        want, _ = gguf_hip.add_rms_norm(x[:1], r[:1])
        out, res = gguf_hip.add_rms_norm(x, r)
        assert torch.equal(out[:1], want) and not out[1].any() and out[2].isnan().all() and torch.equal(res[[0, 1, 3, 4]], x[[0, 1, 3, 4]])
        # s rsqrt(inf) is 0 for what is finite, NaN for the infinity
        assert out[3, 200].isnan() and not out[3, :200].any() and out[4, 3].isnan() and not out[4, 4:].any()
        for group in (0, 32):
            out, scale, _ = gguf_hip.add_rms_norm_fp8(x, r, group=group)
            out = out.float()
            assert torch.isfinite(scale[:2]).all() and (scale[:2] > 0).all() and not out[1].any() and not out[0].isnan().any()
            assert out[2].isnan().all() and scale[2].isnan().all()
            if group == 0:
                assert out[3:].isnan().all() and scale[3:].isnan().all()
            else:
                assert out[3, 192:224].isnan().all() and scale[3].isnan().tolist() == [i == 6 for i in range(8)] and not out[3, :192].any()


def test_norm_small_and_large_values():
    """Sums that pass the 16-bit type's range are taken in 32 bits; very small rows keep their precision."""
    x = torch.full((2, 64), 60000.0, dtype=F16, device="cuda")
    out, res = gguf_hip.add_rms_norm(x, x)
    assert (out == 1).all() and res.isinf().all()            # the sum itself is beyond fp16
    x = (_randn(_gen(3), 4, 512) * 1e-15).to(BF)
    _, y, e = _norm_exact(x, x, None, 0.0, False)
    out, _ = gguf_hip.add_rms_norm(x, x, eps=0.0)
    _within(out, y, (1 + U[BF]) * e + U[BF] * y.abs(), "small")


def test_norm_in_place_strided_and_unaligned():
    gen = _gen(4)
    for rows, dim in ((5, 1000), (600, 515), (2100, 513)):
        x, r = _randn(gen, rows, dim, dtype=BF), _randn(gen, rows, dim, dtype=BF)
        w = _randn(gen, dim, dtype=BF)
        want, res = gguf_hip.add_rms_norm(x, r, w)
        a, b = x.clone(), r.clone()
        got = gguf_hip.add_rms_norm(a, b, w, out=a, out_residual=b)
        assert got[0] is a and got[1] is b and torch.equal(a, want) and torch.equal(b, res)
        a, b = x.clone(), r.clone()
        gguf_hip.add_rms_norm(a, b, w, out=b, out_residual=a)                # the other way round
        assert torch.equal(b, want) and torch.equal(a, res)
        wide = torch.zeros(rows, dim + 9, dtype=BF, device="cuda")
        wide[:, 3:dim + 3] = x
        outs = torch.full((rows, dim + 4), 7.0, dtype=BF, device="cuda")
        flat = torch.zeros(dim + 1, dtype=BF, device="cuda")
        flat[1:] = w
        got, got_r = gguf_hip.add_rms_norm(wide[:, 3:dim + 3], r, flat[1:], out=outs[:, 1:dim + 1])
        assert torch.equal(got, want) and torch.equal(got_r, res) and (outs[:, 0] == 7).all() and (outs[:, dim + 1:] == 7).all()
        got, _ = gguf_hip.add_rms_norm(x.t().contiguous().t(), r, w)         # columns apart: copied
        assert torch.equal(got, want)
        q, s, _ = gguf_hip.add_rms_norm_fp8(x, r, w)
        to = torch.zeros((rows, dim + 3), dtype=F8, device="cuda")
        q2, s2, _ = gguf_hip.add_rms_norm_fp8(x, r, w, out=to[:, 1:dim + 1])
        assert torch.equal(q2.float(), q.float()) and torch.equal(s, s2) and not to[:, 0].float().any()
    assert gguf_hip.add_rms_norm(x[:0], r[:0])[0].shape == (0, 513)
    assert gguf_hip.add_rms_norm_fp8(x[:0], None)[1].shape == (0, 1)


# ---- attention of several new tokens ----------------------------------------------------------

def _cache(gen, lens, page, heads, dim, dtype, layout, spare=2):
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
    fill = 0x7F if dtype == F8 else NAN
    for t in (k, v):
        _bytes(t)[order[at:].long()] = fill
        for i, n in enumerate(lens):
            if n % page and n > 0:
                _bytes(t)[table[i, need[i] - 1].long(), n % page:] = fill
    return k, v, table


def _rows(t, table, b, n, page, scale=None):
    at = torch.arange(n, device="cuda")
    x = t[table[b].long()[at // page], at % page].double()
    return x if scale is None else x * scale.double()[None, :, None]


def _sees(mask, t0, m, n, window):
    """Which of m + n keys each of n new tokens sees."""
    sees = torch.ones((n, m + n), dtype=torch.bool, device="cuda")
    if mask is None:
        sees[:, m:] = sees[:, m:].tril()
    else:
        j = torch.arange(n, device="cuda")
        sees[:, m:] = ((mask[t0:t0 + n].long() & 0xFFFFFFFF)[:, j // 32] >> (j % 32)) % 2 == 1
    if window:
        sees &= sees.sum(1, keepdim=True) - sees.cumsum(1) < window
    return sees


def _attend_exact(q, k, v, table, context, counts, mask, scale, window, ks=None, vs=None):
    """(out, lse, bound of the error of out, of lse) in 64 bits.  Keys that a token does not see count for nothing, whatever they hold."""
    T, H, D = q.shape
    hkv, page, u = k.shape[2], k.shape[1], U[q.dtype]
    out = torch.zeros((T, H, D), dtype=torch.float64, device="cuda")
    lse = torch.full((T, H), -INF, dtype=torch.float64, device="cuda")
    tol, tol_l = torch.zeros_like(out), torch.zeros_like(lse)
    t0 = 0
    for b, (m, n) in enumerate(zip(context, counts)):
        if n == 0:
            continue
        kk, vv = _rows(k, table, b, m + n, page, ks), _rows(v, table, b, m + n, page, vs)
        sees = _sees(mask, t0, m, n, window)
        some = sees.any(1)
        for h in range(hkv):
            for g in range(H // hkv):
                x = q[t0:t0 + n, h * (H // hkv) + g].double()
                s = (x @ kk[:, h].t() * scale).masked_fill(~sees, -INF)
                size = ((x.abs() @ kk[:, h].abs().t() * abs(scale)).masked_fill(~sees, 0)).amax(1)
                top = s.amax(1, keepdim=True)
                e = torch.exp(s - torch.where(some[:, None], top, 0.0))
                total = e.sum(1, keepdim=True).clamp_min(1e-300)
                p = e / total
                clean = vv[:, h].nan_to_num(0.0, 0.0, 0.0)
                o, abs_o = p @ clean, p @ clean.abs()
                es = (D + 8) * E32 * size + 2.0 ** -20 + 4 * E32 * (s - top).nan_to_num(0.0, 0.0, 0.0).abs().amax(1)
                ep = u + 2 * es + 2.0 ** -18
                head = h * (H // hkv) + g
                out[t0:t0 + n, head] = torch.where(some[:, None], o, 0.0)
                tol[t0:t0 + n, head] = u * o.abs() + (1 + u) * (ep[:, None] * abs_o + TINY[q.dtype] * (sees.double() @ clean.abs()) / total) + TINY[q.dtype] + 1e-30
                lse[t0:t0 + n, head] = (top + total.log())[:, 0]
                tol_l[t0:t0 + n, head] = es + 2.0 ** -18 + 4 * E32 * (top[:, 0].nan_to_num(0.0, 0.0, 0.0).abs() + 20)
        t0 += n
    return out, lse, tol, tol_l


def _masks(gen, counts, kind, words):
    """Ancestors of random trees, or any bits at all (rows without one among them; bits beyond the sequence's tokens mean nothing)."""
    rows = []
    for n in counts:
        seen = []
        for i in range(n):
            if kind == "tree":
                p = i - 1 - int(torch.randint(0, 5, (1,), generator=gen))
                seen.append((seen[p] if p >= 0 else 0) | 1 << i)
            else:
                bits = sum(int(x) << (16 * k) for k, x in enumerate(torch.randint(0, 1 << 16, (2 * words,), generator=gen)))
                seen.append(0 if i % 5 == 3 else bits)
        rows += seen
    low = [[(r >> 32 * w) & 0xFFFFFFFF for w in range(words)] for r in rows]
    return torch.tensor(low, dtype=torch.int64).reshape(len(rows), words).to(torch.int32).cuda()


def _tree_case(seed, context, counts, hq, hkv, dim, page, qt, ct, kind, layout="heads", scaled=False, words=None):
    gen = _gen(seed)
    k, v, table = _cache(gen, [m + n for m, n in zip(context, counts)], page, hkv, dim, ct, layout)
    q = _randn(gen, sum(counts), hq, dim, dtype=qt)
    ks = vs = None
    if scaled:
        ks, vs = (0.25 + torch.rand(hkv, device="cuda", generator=gen) for _ in range(2))
    words = words or max(1, -(-max(counts) // 32))
    mask = None if kind == "chain" else _masks(torch.Generator().manual_seed(seed), counts, kind, words)
    lens = _i32([m + n for m, n in zip(context, counts)])
    starts = _i32([sum(counts[:i]) for i in range(len(counts) + 1)])
    return q, k, v, table, lens, starts, mask, ks, vs


def _tree_check(seed, context, counts, hq, hkv, dim, page, qt, ct, kind="tree", window=0, layout="heads", scaled=False, scale=None,
                words=None, **bounds):
    q, k, v, table, lens, starts, mask, ks, vs = _tree_case(seed, context, counts, hq, hkv, dim, page, qt, ct, kind, layout, scaled, words)
    call = lambda: gguf_hip.tree_attention(q, k, v, table, lens, starts, mask, scale=scale, window=window, k_scale=ks,  # noqa: E731
                                           v_scale=vs, return_lse=True, **bounds)
    out, lse = call()
    want, want_l, tol, tol_l = _attend_exact(q, k, v, table, context, counts, mask, dim ** -0.5 if scale is None else scale, window, ks, vs)
    _within(out, want, tol, "out")
    _within(lse, want_l, tol_l, "lse")
    again, lse2 = call()
    assert torch.equal(out, again) and torch.equal(lse, lse2)               # the same bits every time


KINDS = ["tree", "chain", "any"]


@pytest.mark.parametrize("qt,ct", [(BF, BF), (F16, F16), (BF, F8), (F16, F8)])
@pytest.mark.parametrize("dim,hq,hkv", [(64, 8, 2), (128, 40, 8), (128, 3, 3), (256, 6, 1), (80, 5, 1), (8, 2, 1), (192, 4, 2), (24, 2, 2)])
@pytest.mark.parametrize("kind", KINDS)
def test_tree_types_and_heads(qt, ct, dim, hq, hkv, kind):
    _tree_check(dim + hq, [1, 0, 33, 200, 517], [3, 7, 0, 16, 1], hq, hkv, dim, 16, qt, ct, kind, scaled=ct == F8,
                layout="heads" if hq % 2 else "tokens")


@pytest.mark.parametrize("hq,hkv", [(16, 1), (17, 1), (32, 2), (71, 1), (130, 1), (1, 1)])
@pytest.mark.parametrize("counts", [[1, 2], [4, 0], [13, 2], [40, 3]])
def test_tree_shared_heads(hq, hkv, counts):
    """Tokens whose heads begin in one row tile and end in the next; every number of key waves."""
    _tree_check(hq, [130, 5], counts, hq, hkv, 64, 16, BF, BF)
    _tree_check(hq, [61, 300], counts, hq, hkv, 128, 16, BF, BF, "chain")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("counts", [[1], [31], [32], [33], [64], [65], [127, 1, 0, 200], [0, 0, 5], [1] * 130, [3] * 70, [300]])
def test_tree_counts(counts, kind):
    """New tokens that fill words and tiles or do not, sequences without any before, between and behind the others."""
    _tree_check(len(counts), [(37 * i) % 190 for i in range(len(counts))], counts, 5, 1, 64, 16, BF, BF, kind, layout="tokens")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("context", [0, 1, 30, 31, 32, 33, 63, 64, 65, 95, 127, 128, 129])
def test_tree_contexts(context, kind):
    """New tokens that begin anywhere in a block of keys, a step of blocks, a word of the mask; no key at all for some tokens."""
    _tree_check(context, [context, 0], [45, 2], 2, 1, 128, 16, F16, F16, kind)
    _tree_check(context, [context, 0], [7, 7], 2, 1, 64, 8, BF, BF, kind)


@pytest.mark.parametrize("page", [1, 2, 7, 8, 16, 24, 33, 48, 64, 256])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
def test_tree_page_sizes(page, layout):
    _tree_check(page, [1, 31, 32, 300, 0], [5, 1, 64, 17, 9], 10, 2, 128, page, BF, BF, layout=layout)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [1, 2, 5, 31, 32, 33, 100, 1000, 5000])
def test_tree_windows(window, kind):
    """The window's start in the cache, among the new tokens, before both; different for each token of a tile."""
    _tree_check(window, [0, 1, 31, 64, 100, 1500], [40, 33, 7, 70, 1, 12], 4, 2, 64, 16, F16, F16, kind, window=window)
    _tree_check(window, [700], [90], 6, 1, 128, 32, BF, F8, kind, window=window, scaled=True)


@pytest.mark.parametrize("kind", ["tree", "chain"])
@pytest.mark.parametrize("hq,hkv,dim,counts", [(8, 2, 128, [3]), (40, 8, 128, [16, 2]), (6, 1, 256, [1, 9]), (5, 1, 80, [30]), (8, 8, 64, [1]),
                                               (40, 8, 128, [200])])
def test_tree_long_contexts_in_splits(hq, hkv, dim, counts, kind):
    context = [20_011, 777][:len(counts)]
    _tree_check(dim, context, counts, hq, hkv, dim, 16, BF, BF, kind)
    _tree_check(dim, context, counts, hq, hkv, dim, 64, F16, F8, kind, window=7777, scaled=True, max_tokens=max(counts))


def test_tree_of_a_long_prompt():
    """A chunk of a prompt behind another, its first tokens and its last."""
    _tree_check(1, [700], [1500], 10, 2, 128, 16, BF, BF, "chain", max_length=2200, max_tokens=1500)
    _tree_check(2, [0, 513], [1100, 300], 3, 1, 256, 16, F16, F16, "chain")
    _tree_check(3, [100], [1024], 2, 1, 64, 16, BF, BF, "tree")


def test_tree_of_one_token_is_paged_attention():
    gen = _gen(5)
    lens = [700, 3, 0, 512, 64]
    k, v, table = _cache(gen, lens, 16, 2, 128, BF, "heads")
    q = _randn(gen, 5, 8, 128, dtype=BF)
    n = _i32(lens)
    want, _, tol, _ = _attend_exact(q, k, v, table, [699, 2, -1, 511, 63], [1, 1, 0, 1, 1], None, 128 ** -0.5, 0)
    starts = _i32([0, 1, 2, 2, 3, 4])
    got = gguf_hip.tree_attention(q[[0, 1, 3, 4]], k, v, table, n, starts)
    one = gguf_hip.paged_attention(q, k, v, table, n)[[0, 1, 3, 4]]
    _within(got, one, 4 * U[BF] * (one.abs() + 0.1), "single tokens")       # two results within a few roundings of the same


def test_tree_bounds_are_only_bounds():
    """Loose and tight bounds on lengths and tokens: the same values up to the order of the sums; below: NaN for the sequence."""
    context, counts = [600, 3, 512], [9, 2, 30]
    q, k, v, table, lens, starts, mask, _, _ = _tree_case(6, context, counts, 8, 2, 64, 16, BF, BF, "tree")
    want, _, tol, _ = _attend_exact(q, k, v, table, context, counts, mask, 64 ** -0.5, 0)
    wide = torch.full((3, 4000), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    for t, kw in ((table, {}), (table, {"max_length": 609}), (wide, {}), (wide[:, :50], {"max_length": 777, "max_tokens": 30}),
                  (table, {"max_tokens": 10_000})):
        _within(gguf_hip.tree_attention(q, k, v, t, lens, starts, mask, **kw), want, tol, kw)
    out, lse = gguf_hip.tree_attention(q, k, v, table, lens, starts, mask, max_length=600, return_lse=True)
    assert out[:9].isnan().all() and lse[:9].isnan().all()
    _within(out[9:], want[9:], tol[9:], "the others")
    out = gguf_hip.tree_attention(q, k, v, table, lens, starts, mask, max_tokens=29)
    assert out[11:].isnan().all()
    _within(out[:11], want[:11], tol[:11], "the others")
    out = gguf_hip.tree_attention(q, k, v, table, _i32([8, 5, 2 ** 31 - 1]), starts, mask)
    assert out[:9].isnan().all() and out[11:].isnan().all()
    _within(out[9:11], want[9:11], tol[9:11], "the other")
    narrow = torch.cat([mask, mask], 0)[:41].contiguous()                   # a mask of 32 bits for 33 tokens
    q33 = _randn(_gen(1), 33, 8, 64, dtype=BF)
    out = gguf_hip.tree_attention(q33, k, v, table[:1], lens[:1], _i32([0, 33]), narrow[:33, :1].contiguous())
    assert out.isnan().all()


def test_tree_rows_of_no_sequence_stay():
    context, counts = [40, 20, 9], [4, 3, 2]
    q, k, v, table, lens, starts, mask, _, _ = _tree_case(7, context, counts, 8, 2, 64, 16, BF, BF, "tree")
    want, _, tol, _ = _attend_exact(q, k, v, table, context, counts, mask, 64 ** -0.5, 0)
    q12 = torch.cat([torch.full((2, 8, 64), NAN, device="cuda", dtype=BF), q, q[:3]])
    m12 = torch.cat([mask[:2], mask, mask[:3]])
    out = torch.full((14, 8, 64), 7.0, dtype=BF, device="cuda")
    gguf_hip.tree_attention(q12, k, v, table, lens, starts + 2, m12, out=out)
    assert (out[:2] == 7).all() and (out[11:] == 7).all()
    _within(out[2:11], want, tol, "inside")
    # rows that are not q's: the sequence is left alone
    out.fill_(7)
    gguf_hip.tree_attention(q, k, v, table, lens, _i32([0, 4, 7, 10]), mask, out=out[:9])
    _within(out[:7], want[:7], tol[:7], "the first two")
    assert (out[7:] == 7).all()
    out.fill_(7)
    gguf_hip.tree_attention(q, k, v, table, lens, _i32([-3, 4, 2, 9]), mask, out=out[:9])
    assert (out[:2] == 7).all()
    assert gguf_hip.tree_attention(q[:0], k, v, table[:0], lens[:0], starts[:1]).shape == (0, 8, 64)
    assert gguf_hip.tree_attention(q[:0], k, v, table, lens, starts * 0).shape == (0, 8, 64)


def test_tree_bad_pages_are_not_read():
    context, counts = [100, 600, 40, 17], [4, 9, 2, 3]
    q, k, v, table, lens, starts, mask, _, _ = _tree_case(8, context, counts, 4, 2, 64, 16, BF, BF, "tree")
    want, _, tol, _ = _attend_exact(q, k, v, table, context, counts, mask, 64 ** -0.5, 0)
    table = table.clone()
    table[1, 30], table[2, 0], table[3, 1] = k.shape[0], -1, 2 ** 30
    for _ in range(2):
        out, lse = gguf_hip.tree_attention(q, k, v, table, lens, starts, mask, return_lse=True)
        assert out[4:].isnan().all() and lse[4:].isnan().all()
        _within(out[:4], want[:4], tol[:4], "the sound one")


@pytest.mark.parametrize("qt,ct", [(BF, BF), (F16, F16), (BF, F8)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kind", ["tree", "chain", "any"])
def test_tree_what_is_not_seen_does_not_matter(qt, ct, dim, kind):
    """NaN and infinite keys and values of new tokens reach those that see them, and nobody else; under a window too."""
    context, counts = [70, 3], [50, 20]
    q, k, v, table, lens, starts, mask, _, _ = _tree_case(dim, context, counts, 6, 2, dim, 16, qt, ct, kind)
    sees = [_sees(mask, 0, 70, 50, 0), _sees(mask, 50, 3, 20, 0)]
    at = lambda b, j: (int(table[b, j // 16]), j % 16, slice(None))  # noqa: E731
    k0, v0 = k.clone(), v.clone()
    touched = torch.zeros(70, dtype=torch.bool, device="cuda")
    marks = [(0, 75, "v", NAN), (0, 101, "k", NAN), (0, 110, "v", INF), (1, 11, "v", -INF), (1, 14, "k", INF)]
    for b, j, which, x in marks:
        t = k if which == "k" else v
        if t.dtype == F8:
            _bytes(t)[at(b, j)] = 0x7F                       # the type has no infinity
        else:
            t[at(b, j)] = x
        touched[50 * b:50 * b + (20 if b else 50)] |= sees[b][:, j]
    # what is marked counts for nothing where it is not seen: the clean cache's results
    want, _, tol, _ = _attend_exact(q, k0, v0, table, context, counts, mask, dim ** -0.5, 0)
    out = gguf_hip.tree_attention(q, k, v, table, lens, starts, mask)
    _within(out[~touched], want[~touched], tol[~touched], "not seen")
    assert touched.any() and not torch.isfinite(out[touched].float()).all(2).any()
    if kind == "tree" and ct != F8:   # one infinite value, seen alone by some: it is their result
        k2, v2 = k0.clone(), v0.clone()
        v2[at(0, 110)][:, 0] = INF
        out = gguf_hip.tree_attention(q, k2, v2, table, lens, starts, mask)
        seen = torch.zeros(70, dtype=torch.bool, device="cuda")
        seen[:50] = sees[0][:, 110]
        # (dim 0 of both key heads)
        assert (out[seen][:, :, 0] == INF).all() and torch.isfinite(out[~seen]).all()
        _within(out[..., 1:], want[..., 1:], tol[..., 1:], "the other dims")
    # the window's end takes keys of the cache from some rows of a tile
    v3 = v0.clone()
    _bytes(v3)[at(0, 40)] = 0x7F if ct == F8 else NAN
    sees3 = torch.cat([_sees(mask, 0, 70, 50, 45)[:, 40], torch.zeros(20, dtype=torch.bool, device="cuda")])
    want, _, tol, _ = _attend_exact(q, k0, v0, table, context, counts, mask, dim ** -0.5, 45)
    out = gguf_hip.tree_attention(q, k0, v3, table, lens, starts, mask, window=45)
    _within(out[~sees3], want[~sees3], tol[~sees3], "behind the window")
    assert out[sees3].isnan().all()


@pytest.mark.parametrize("dim", [8, 40, 72, 80, 96, 120, 136, 200, 248])
@pytest.mark.parametrize("page", [16, 7])
@pytest.mark.parametrize("qt,ct", [(BF, BF), (F16, F16), (F16, F8)])
@pytest.mark.parametrize("counts", [[3, 7, 1], [40, 9, 33]])
def test_tree_dims_that_a_tile_does_not_fill(dim, page, qt, ct, counts):
    """What an earlier call left in shared memory, infinities and NaN here, is nothing to the dims behind the last."""
    q, k, v, table, lens, starts, _, _, _ = _tree_case(1, [600, 600, 600], counts, 8, 2, 256, 16, BF, BF, "chain")
    k.fill_(INF)
    v.fill_(NAN)
    gguf_hip.tree_attention(q, k, v, table, lens, starts)
    _tree_check(dim + page, [130, 0, 61], counts, 6, 2, dim, page, qt, ct, kind="any", scaled=ct == F8)


@pytest.mark.parametrize("dim,page", [(80, 16), (80, 7), (128, 7), (200, 48), (248, 1), (256, 5)])
@pytest.mark.parametrize("qt,ct", [(BF, BF), (F16, F16), (BF, F8)])
def test_tree_not_seen_in_every_form(dim, page, qt, ct):
    """Keys and values that are not finite, at places that only some tokens see, and a page outside of the cache."""
    context, counts = [70, 3, 40], [50, 20, 4]
    q, k, v, table, lens, starts, mask, _, _ = _tree_case(dim, context, counts, 6, 2, dim, page, qt, ct, "tree")
    want, _, tol, _ = _attend_exact(q, k, v, table, context, counts, mask, dim ** -0.5, 0)
    touched = torch.zeros(74, dtype=torch.bool, device="cuda")
    for j, t in ((75, k), (99, v), (110, v)):
        _bytes(t)[int(table[0, j // page]), j % page] = 0x7F if ct == F8 else NAN
        touched[:50] |= _sees(mask, 0, 70, 50, 0)[:, j]
    table = table.clone()
    table[2, 40 // page] = k.shape[0]
    for workspace in (None, torch.zeros(65536, dtype=torch.int32, device="cuda")):
        out = gguf_hip.tree_attention(q, k, v, table, lens, starts, mask, workspace=workspace)
        assert out[70:].isnan().any(2).all()
        _within(out[:70][~touched[:70]], want[:70][~touched[:70]], tol[:70][~touched[:70]], "not seen")
        assert touched.any() and out[touched].isnan().any(2).all()


def test_tree_extreme_scores_and_scales():
    """Scores far apart, negative and zero scales, negative key scales, keys of score -inf."""
    context, counts = [150, 80], [9, 20]
    for scale in (-0.125, 0.0, 3.0):
        _tree_check(9, context, counts, 4, 2, 64, 16, BF, BF, scale=scale)
        _tree_check(9, context, counts, 4, 2, 64, 16, F16, F16, scale=scale)
    q, k, v, table, lens, starts, mask, _, _ = _tree_case(10, context, counts, 4, 2, 64, 16, BF, F8, "tree")
    ks, vs = torch.tensor([0.5, -1.5], device="cuda"), torch.tensor([-1.0, 0.75], device="cuda")
    want, _, tol, _ = _attend_exact(q, k, v, table, context, counts, mask, 0.125, 0, ks, vs)
    _within(gguf_hip.tree_attention(q, k, v, table, lens, starts, mask, k_scale=ks, v_scale=vs), want, tol, "negative scales")
    q, k, v, table, lens, starts, mask, _, _ = _tree_case(11, context, counts, 4, 2, 64, 16, BF, BF, "tree")
    q[:, :, 0] = 1.0
    k[int(table[0, 2]), 3, :, 0] = -INF                      # key 35: weight 0
    out = gguf_hip.tree_attention(q, k, v, table, lens, starts, mask)
    want, _, tol, _ = _attend_exact(q, k.nan_to_num(0, 0, -1e30), v, table, context, counts, mask, 0.125, 0)
    _within(out, want, 2 * U[BF] * (1 + want.abs()), "-inf")


@pytest.mark.parametrize("qt,ct,dim", [(F16, F16, 64), (F16, F16, 128), (F16, F16, 256), (F16, F8, 128), (BF, BF, 128)])
@pytest.mark.parametrize("counts", [[2], [200]])
def test_tree_flat_tail(qt, ct, dim, counts):
    """A few heavy keys of value 0 in each page of 4096; the others, of 2^-25.2 of their weight each, are all of the result."""
    page, pages = 4096, 6
    k, v = (torch.zeros((1, page, 1, dim), device="cuda") for _ in range(2))
    k[..., 0], v[:] = -14.0, 256.0
    heavy = torch.arange(0, 128, 32, device="cuda")
    k[:, heavy], v[:, heavy] = 0.0, 0.0
    k, v = k.to(ct), v.to(ct)
    n = counts[0]
    q = torch.zeros((n, 2, dim), dtype=qt, device="cuda")
    q[..., 0] = 1.25                                         # scores of 0 and -17.5
    table = torch.zeros((1, pages), dtype=torch.int32, device="cuda")
    mask = torch.zeros((n, -(-n // 32)), dtype=torch.int32, device="cuda")   # the cache alone
    # the new tokens' own keys lie behind the whole pages of the cache, and nobody sees them
    table = torch.zeros((1, pages + 1), dtype=torch.int32, device="cuda")
    out, lse = gguf_hip.tree_attention(q, k, v, table, _i32([pages * page + n]), _i32([0, n]), mask, scale=1.0, return_lse=True)
    light = (page - 4) * torch.tensor(-17.5, dtype=torch.float64).exp().item()
    want = 256 * light / (4 + light)
    # a score's error, and up to 2^10 steps of a wave with two roundings of the sum each
    e = 2.0 ** -18 + 2.0 ** 11 * E32
    _within(out, torch.full_like(out, want, dtype=torch.float64), (2 * U[qt] + 2 * e) * want + 2.0 ** -25, "out")
    want_l = torch.tensor((4 + light) * pages, dtype=torch.float64).log().item()
    _within(lse, torch.full_like(lse, want_l, dtype=torch.float64), 2 * e + 4 * E32 * (want_l + 40), "lse")


def test_tree_strides_streams_and_outputs():
    context, counts = [1000, 31, 2], [3, 12, 1]
    q, k, v, table, lens, starts, mask, _, _ = _tree_case(12, context, counts, 10, 2, 128, 16, BF, BF, "tree")
    want, _, tol, _ = _attend_exact(q, k, v, table, context, counts, mask, 128 ** -0.5, 0)
    wide = torch.zeros(16, 14, 128, dtype=BF, device="cuda")
    wide[:, 3:13] = q
    out = torch.zeros(16, 20, 128, dtype=BF, device="cuda")
    apart = torch.full((3, table.shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    apart[:, :table.shape[1]] = table
    got = gguf_hip.tree_attention(wide[:, 3:13], k, v, apart[:, :table.shape[1]], lens, starts, mask, out=out[:, 5:15])
    assert got.data_ptr() == out[:, 5:15].data_ptr() and not out[:, :5].any() and not out[:, 15:].any()
    _within(out[:, 5:15], want, tol, "views")
    odd = torch.zeros(16 * 10 * 128 + 1, dtype=BF, device="cuda")[1:].view(16, 10, 128)
    odd.copy_(q)
    _within(gguf_hip.tree_attention(odd, k, v, table, lens, starts, mask), want, tol, "unaligned")
    side, ws = torch.cuda.Stream(), torch.zeros(16 << 20, dtype=torch.int32, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = gguf_hip.tree_attention(q, k, v, table, lens, starts, mask, workspace=ws)
    here = gguf_hip.tree_attention(q, k, v, table, lens, starts, mask)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, here)


@pytest.mark.parametrize("counts,hq,hkv,dim", [([2], 8, 2, 64), ([9, 3, 1], 40, 8, 128), ([70], 6, 1, 256)])
def test_tree_in_small_workspaces(counts, hq, hkv, dim):
    """A workspace that holds all, some, two or none of the splits that the call would like; nothing is written past it or in the
    counters."""
    context = [4001, 3000, 0][:len(counts)]
    q, k, v, table, lens, starts, mask, _, _ = _tree_case(dim, context, counts, hq, hkv, dim, 16, BF, BF, "tree")
    want, _, tol, _ = _attend_exact(q, k, v, table, context, counts, mask, dim ** -0.5, 0)
    T = sum(counts)
    need = _lib.lib.gqk_tree_attention_workspace_bytes(T, len(counts), hq, hkv, dim, T, table.shape[1] * 16, 0)
    ctr = _lib.GQK_CTR_BYTES
    assert need > ctr
    for size in (need, need - 4, ctr + (need - ctr) // 2, ctr + (need - ctr) // 7, ctr, 256):
        size = size // 4 * 4
        whole = torch.zeros(size // 4 + 4096, dtype=torch.int32, device="cuda")
        ws = whole[:size // 4]
        _within(gguf_hip.tree_attention(q, k, v, table, lens, starts, mask, workspace=ws), want, tol, size)
        assert not whole[size // 4:].any() and not ws[:ctr // 4].any(), size


def test_tree_offsets_past_32_bits():
    """A cache of more than 2^31 elements, its last pages in use."""
    page, dim, count = 64, 128, 270_000
    k, v = (torch.empty((count, page, 1, dim), dtype=F8, device="cuda") for _ in range(2))
    assert k.numel() > 2 ** 31
    gen = _gen(11)
    used = _i32([count - 1, 0, count - 2, 262_144, 5])
    for t in (k, v):
        t.view(torch.uint8)[used.long()] = _randn(gen, 5, page, 1, dim).to(F8).view(torch.uint8)
    for n in (5, 90):
        q = _randn(gen, n, 4, dim, dtype=BF)
        out = gguf_hip.tree_attention(q, k, v, used[None], _i32([300]), _i32([0, n]))
        want, _, tol, _ = _attend_exact(q, k, v, used[None], [300 - n], [n], None, dim ** -0.5, 0)
        _within(out, want, tol, "far pages")
        bounds = torch.zeros((count, 2, 1, dim), dtype=F8, device="cuda")
        gguf_hip.page_bounds(k, used[None], _i32([300]), bounds, count=300)
        want = k[used.long()].float()
        want[4, 300 - 4 * 64:] = want[4, :1]
        assert torch.equal(bounds[used.long(), 0].float(), want.amin(1)) and torch.equal(bounds[used.long(), 1].float(), want.amax(1))


def test_tree_at_the_limit_of_keys():
    """The longest sequence, whose table names two pages again and again: keys of score 0 and value 1, and in its last page (and
    one in the middle) keys of score 10.375, together about as heavy as all others, and value 3.  Its last two tokens.  A wave takes 2^16
    steps: a chain of as many fp32 roundings in the weights' total and in the products' sums, of two a step and up to a unit each."""
    page, dim, length = 1 << 16, 8, _lib.GQK_MAX_KEYS
    k, v = (torch.zeros((2, page, 1, dim), dtype=BF, device="cuda") for _ in range(2))
    k[1, :, 0, 0], v[0], v[1] = 10.375, 1.0, 3.0
    q = torch.zeros((2, 1, dim), dtype=BF, device="cuda")
    q[:, 0, 0] = 1.0
    count = -(-length // page)
    table = torch.zeros((1, count), dtype=torch.int32, device="cuda")
    table[0, count // 2] = table[0, -1] = 1
    out = gguf_hip.tree_attention(q, k, v, table, _i32([length]), _i32([0, 2]), scale=1.0)
    for i in range(2):
        n = length - 1 + i
        heavy = torch.tensor(10.375, dtype=torch.float64).exp() * (page + n - (count - 1) * page)
        light = n - (page + n - (count - 1) * page)
        want = (light + 3 * heavy) / (light + heavy)
        chain = 2.0 ** 16 * E32
        _within(out[i], want.cuda().expand(1, dim), (U[BF] * want + (U[BF] + 5 * chain + 2.0 ** -16) * want * (1 + U[BF])).cuda(), i)


# ---- the pages that are worth reading -----------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, F16, F8])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
@pytest.mark.parametrize("dim,page,hkv", [(128, 16, 8), (80, 7, 2), (256, 48, 3), (64, 1, 1), (8, 300, 2), (200, 33, 1)])
def test_bounds(dtype, layout, dim, page, hkv):
    """The pages of the last keys alone, read anew up to the sequence's last key; the others stay as they were."""
    gen = _gen(dim + page)
    lens = [1, 0, 5 * page + 3, 2 * page, page + 1, 31]
    k, _, table = _cache(gen, lens, page, hkv, dim, dtype, layout)
    for count in (1, 2, page, 2 * page + 1, 10 ** 6, 2 ** 31 - 1):
        bounds = _randn(gen, k.shape[0], 2, hkv, dim).to(dtype)
        want = bounds.clone()
        for b, n in enumerate(lens):
            for j in range(max(0, n - count) // page, -(-n // page)):
                keys = k[int(table[b, j]), :min(page, n - j * page)].float()
                want[int(table[b, j])] = torch.stack([keys.amin(0), keys.amax(0)]).to(dtype)
        version = bounds._version
        assert gguf_hip.page_bounds(k, table, _i32(lens), bounds, count=count) is bounds and bounds._version > version
        assert torch.equal(bounds.float(), want.float()), count


def test_bounds_of_what_is_not_finite_and_out_of_range():
    k = _randn(_gen(1), 4, 8, 2, 16, dtype=BF)
    k[0, 3, 0, 5], k[1, 0, 1, 2], k[1, 1, 1, 2], k[2, 7, 0, 0] = NAN, INF, -INF, NAN
    table = _i32([[0, 1, 2], [4, 3, -1], [3, 1, 0]])
    bounds = torch.zeros((4, 2, 2, 16), dtype=BF, device="cuda")
    gguf_hip.page_bounds(k, table, _i32([23, 24, 25]), bounds, count=100)   # the last is longer than its table: nothing of it
    keys = [k[0], k[1], k[2, :7], k[3]]
    for p, x in enumerate(keys):
        want = torch.stack([x.float().amin(0), x.float().amax(0)]).to(BF)
        if p == 0:
            assert want[:, 0, 5].isnan().all()
        assert torch.equal(bounds[p].nan_to_num(123.0), want.nan_to_num(123.0)), p
    assert bounds[0, :, 0, 5].isnan().all()
    gguf_hip.page_bounds(k, table, _i32([0, -1, 2 ** 31 - 1]), bounds.fill_(5), count=3)
    assert (bounds == 5).all()


def _score(q, bounds, table, b, n, page):
    """[heads, pages] in 64 bits."""
    hkv = bounds.shape[2]
    pages = -(-n // page)
    near = bounds[table[b, :pages].long()].double() if bounds.dtype != F8 else bounds.float()[table[b, :pages].long()].double()
    x = q[b].double().view(hkv, -1, q.shape[2])
    out = []
    for h in range(hkv):
        lo, hi = near[:, 0, h], near[:, 1, h]
        out.append(torch.maximum(x[h][:, None] * lo, x[h][:, None] * hi).sum(2).amax(0))
    return torch.stack(out)


def _select_exact(q, bounds, table, lens, keep, page, sink, recent):
    hkv = bounds.shape[2]
    out = torch.full((len(lens), hkv, keep), -1, dtype=torch.int32)
    kept = []
    for b, n in enumerate(lens):
        pages = -(-n // page)
        if pages <= keep:
            out[b, :, :pages] = table[b, :pages].cpu()
            kept.append(n)
            continue
        score = _score(q, bounds, table, b, n, page).cpu()
        fixed = list(range(sink)) + list(range(pages - recent, pages))
        for h in range(hkv):
            rest = sorted((j for j in range(pages) if j not in fixed), key=lambda j: (-float(score[h, j]), j))
            out[b, h] = table[b].cpu()[sorted(fixed + rest[:keep - len(fixed)])]
        kept.append(n - (pages - keep) * page)
    return out, kept


def _long_cache(gen, lens, page, hkv, dim, dtype):
    k, v, table = _cache(gen, lens, page, hkv, dim, dtype, "heads")
    bounds = torch.zeros((k.shape[0], 2, hkv, dim), dtype=dtype, device="cuda")
    gguf_hip.page_bounds(k, table, _i32(lens), bounds, count=max(lens))
    return k, v, table, bounds


@pytest.mark.parametrize("qt,ct", [(BF, BF), (F16, F16), (BF, F8), (F16, F8)])
@pytest.mark.parametrize("dim,hq,hkv,page", [(128, 40, 8, 16), (64, 4, 4, 7), (256, 16, 1, 16), (80, 6, 2, 32), (8, 2, 1, 5)])
@pytest.mark.parametrize("keep,sink,recent", [(1, 0, 1), (4, 1, 1), (9, 2, 3), (20, 0, 1), (5, 2, 3)])
def test_select(qt, ct, dim, hq, hkv, page, keep, sink, recent):
    """The table for each key head, and the attention over it."""
    gen = _gen(dim + keep)
    lens = [50 * page + 3, 0, 1, 20 * page, 21 * page - 1, 9 * page, 33 * page + 1]
    k, v, table, bounds = _long_cache(gen, lens, page, hkv, dim, ct)
    q = _randn(gen, len(lens), hq, dim, dtype=qt)
    got, kept = gguf_hip.select_pages(q, bounds, table, _i32(lens), keep, page, sink=sink, recent=recent)
    want, want_n = _select_exact(q, bounds, table, lens, keep, page, sink, recent)
    assert torch.equal(got.cpu(), want) and kept.tolist() == want_n
    ks = vs = None
    if ct == F8:
        ks, vs = (0.25 + torch.rand(hkv, device="cuda", generator=gen) for _ in range(2))
    out, lse = gguf_hip.paged_attention(q, k, v, got, kept, k_scale=ks, v_scale=vs, return_lse=True)
    g = hq // hkv
    for h in range(hkv):
        one = lambda t: t[:, :, h:h + 1]  # noqa: E731
        s = lambda t: None if t is None else t[h:h + 1]  # noqa: E731
        rows = torch.tensor([b for b, n in enumerate(want_n) if n > 0], device="cuda")
        w, wl, tol, tol_l = _attend_exact(q[rows][:, h * g:(h + 1) * g], one(k), one(v), got[rows, h], [want_n[int(r)] - 1 for r in rows],
                                          [1] * len(rows), None, dim ** -0.5, 0, s(ks), s(vs))
        _within(out[rows][:, h * g:(h + 1) * g], w, tol, "out")
        _within(lse[rows][:, h * g:(h + 1) * g], wl, tol_l, "lse")
    assert not out[1].any() and (lse[1] == -INF).all()
    again, kept2 = gguf_hip.select_pages(q, bounds, table, _i32(lens), keep, page, sink=sink, recent=recent)
    assert torch.equal(got, again) and torch.equal(kept, kept2)


@pytest.mark.parametrize("pages,keep", [(1023, 64), (1025, 1), (1025, 1024), (5000, 300), (8192, 64), (8193, 8192), (20_000, 777)])
def test_select_of_many_pages(pages, keep):
    """More than a workgroup's threads, and than it holds in registers."""
    gen = _gen(pages)
    bounds = _randn(gen, 500, 2, 2, 8, dtype=BF).sort(dim=1).values
    table = torch.randint(0, 500, (3, pages), device="cuda", generator=gen).to(torch.int32)   # pages repeat: exact ties
    q = _randn(gen, 3, 4, 8, dtype=BF)
    lens = [pages * 4, pages * 4 - 3, (pages - 1) * 4]
    got, kept = gguf_hip.select_pages(q, bounds, table, _i32(lens), keep, 4, sink=1 if keep > 1 else 0, recent=1)
    want, want_n = _select_exact(q, bounds, table, lens, keep, 4, 1 if keep > 1 else 0, 1)
    assert torch.equal(got.cpu(), want) and kept.tolist() == want_n


def test_select_ties_take_the_first():
    """Equal scores: the first pages, in every number of them; scores of zero of either sign are equal."""
    bounds = torch.zeros((300, 2, 1, 8), dtype=BF, device="cuda")
    bounds[100:200, 0] = -0.0
    table = torch.arange(300, dtype=torch.int32, device="cuda")[None]
    q = _randn(_gen(1), 1, 3, 8, dtype=BF)
    for keep in (2, 3, 64, 65, 255, 256, 257, 299):
        got, kept = gguf_hip.select_pages(q, bounds, table, _i32([300 * 16]), keep, 16, sink=0, recent=1)
        assert got[0, 0].tolist() == list(range(keep - 1)) + [299] and kept.item() == keep * 16
    bounds[7] = 1.0
    bounds[7, :, 0, 1::2] = 0
    bounds[250] = bounds[7]
    got, _ = gguf_hip.select_pages(q.abs(), bounds, table, _i32([300 * 16]), 5, 16, sink=0, recent=1)
    assert got[0, 0].tolist() == [0, 1, 7, 250, 299]


def test_select_near_scores_are_told_apart():
    """Scores whose difference is lost in 32 bits: sums of large products that cancel, and a small one."""
    bounds = torch.zeros((64, 2, 1, 64), dtype=BF, device="cuda")
    order = torch.randperm(64, device="cuda", generator=_gen(2))
    bounds[:, :, 0, 0], bounds[:, :, 0, 1] = 2.0 ** 30, 2.0 ** 30
    bounds[:, :, 0, 2] = order.to(BF)[:, None] * 2.0 ** -4
    q = torch.zeros((1, 1, 64), dtype=BF, device="cuda")
    q[0, 0, :3] = torch.tensor([1.0, -1.0, 2.0 ** -6])
    table = torch.arange(64, dtype=torch.int32, device="cuda")[None]
    got, _ = gguf_hip.select_pages(q, bounds, table, _i32([64 * 8]), 17, 8, sink=0, recent=1)
    score = order.cpu().tolist()
    want = sorted(sorted(range(63), key=lambda j: -score[j])[:16] + [63])
    assert got[0, 0].tolist() == want


def test_select_bad_lengths_pages_and_scores():
    gen = _gen(3)
    lens = [40 * 8, 40 * 8, 30 * 8, 5, -4]
    k, v, table, bounds = _long_cache(gen, [max(n, 0) for n in lens], 8, 2, 64, BF)
    q = _randn(gen, 5, 4, 64, dtype=BF)
    want, want_n = _select_exact(q, bounds, table, [max(n, 0) for n in lens], 6, 8, 1, 1)
    got, kept = gguf_hip.select_pages(q, bounds, table, _i32(lens), 6, 8, max_length=300)
    assert kept.tolist() == [2 ** 31 - 1] * 2 + want_n[2:] and (got[:2] == -1).all() and torch.equal(got[2:].cpu(), want[2:])
    assert gguf_hip.paged_attention(q, k, v, got, kept)[:2].isnan().all()
    bad = table.clone()
    bad[0, 17], bad[1, 3] = k.shape[0], -5
    got, kept = gguf_hip.select_pages(q, bounds, bad, _i32(lens), 6, 8)
    assert (got[0] == k.shape[0]).any(1).all() and (got[1] == -5).any(1).all() and torch.equal(got[2:].cpu(), want[2:])
    out = gguf_hip.paged_attention(q, k, v, got, kept)
    assert out[:2].isnan().all() and not out[2:].isnan().any()
    bounds[table[0, 9].long(), :, 1, 7] = NAN                # a score that is no number: the page is taken
    got, _ = gguf_hip.select_pages(q, bounds, table, _i32(lens), 3, 8)
    assert (got[0, 1] == table[0, 9]).any()


def test_select_in_turns_and_views():
    """A workspace of one sequence's scores, of two, of all: the same; queries and tables as views."""
    gen = _gen(4)
    lens = [40 * 8, 3, 37 * 8 + 1, 39 * 8]
    k, v, table, bounds = _long_cache(gen, lens, 8, 2, 64, BF)
    q = _randn(gen, 4, 8, 64, dtype=BF)
    n = _i32(lens)
    want, kept = gguf_hip.select_pages(q, bounds, table, n, 6, 8)
    need = _lib.lib.gqk_select_pages_workspace_bytes(4, 2, 8, 40 * 8)
    one = (need - _lib.GQK_CTR_BYTES) // 4
    for size in (need, _lib.GQK_CTR_BYTES + 2 * one, _lib.GQK_CTR_BYTES + one):
        whole = torch.zeros(size // 4 + 1024, dtype=torch.int32, device="cuda")
        got, kept2 = gguf_hip.select_pages(q, bounds, table, n, 6, 8, workspace=whole[:size // 4])
        assert torch.equal(got, want) and torch.equal(kept, kept2)
        assert not whole[size // 4:].any() and not whole[:_lib.GQK_CTR_BYTES // 4].any()
    with pytest.raises(ValueError, match="workspace"):
        gguf_hip.select_pages(q, bounds, table, n, 6, 8, workspace=whole[:(_lib.GQK_CTR_BYTES + one) // 4 - 2])
    wide = torch.zeros(4, 11, 64, dtype=BF, device="cuda")
    wide[:, 2:10] = q
    apart = torch.full((4, table.shape[1] + 3), -1, dtype=torch.int32, device="cuda")
    apart[:, :table.shape[1]] = table
    got, _ = gguf_hip.select_pages(wide[:, 2:10], bounds, apart[:, :table.shape[1]], n, 6, 8)
    assert torch.equal(got, want)
    got, kept2 = gguf_hip.select_pages(q[:0], bounds, table[:0], n[:0], 6, 8)
    assert got.shape == (0, 2, 6) and kept2.shape == (0,)
    # tables of heads whose rows lie apart
    far = torch.full((4, 3, 9), -1, dtype=torch.int32, device="cuda")
    far[:, :2, :6] = want
    assert torch.equal(gguf_hip.paged_attention(q, k, v, far[:, :2, :6], kept), gguf_hip.paged_attention(q, k, v, want, kept))


# ---- graphs, tracing, the two ways of a call ----------------------------------------------------

def _calls(seed=1):
    """Each operator's call on fixed tensors, and those tensors."""
    gen = _gen(seed)
    context, counts = [300, 45, 0], [5, 16, 3]
    q, k, v, table, lens, starts, mask, _, _ = _tree_case(seed, context, counts, 8, 2, 64, 16, BF, BF, "tree")
    lists = torch.cat([table, table], 0).contiguous()
    req, old, new = _i32([4, 0, 2]), _i32(context), _i32(counts)
    parents = _i32([-1, 0, 0, 1, 2] + [max(-1, i - 2) for i in range(16)] + [-1, 0, 1] + [-1] * 8)
    x, r, w = _randn(gen, 24, 640, dtype=BF), _randn(gen, 24, 640, dtype=BF), _randn(gen, 640, dtype=BF)
    bounds = torch.zeros((k.shape[0], 2, 2, 64), dtype=BF, device="cuda")
    q1 = q[:3].contiguous()

    def sparse():
        gguf_hip.page_bounds(k, table, lens, bounds, count=320)
        t, n = gguf_hip.select_pages(q1, bounds, table, lens, 4, 16)
        return t, n, gguf_hip.paged_attention(q1, k, v, t, n), bounds

    return {"step_tables": (lambda: tuple(gguf_hip.step_tables(lists, req, old, new, 32, 16, parents=parents, tree=16)), (old, new)),
            "add_rms_norm": (lambda: gguf_hip.add_rms_norm(x, r, w), (x, r)),
            "add_rms_norm_fp8": (lambda: gguf_hip.add_rms_norm_fp8(x, r, w, group=128), (x, r)),
            "tree_attention": (lambda: gguf_hip.tree_attention(q, k, v, table, lens, starts, mask, return_lse=True), (q,)),
            "select_pages": (sparse, (q1,))}


def _same(a, b):
    return all(torch.equal(_bytes(x), _bytes(y)) for x, y in zip(a, b))


@pytest.mark.parametrize("name", ["step_tables", "add_rms_norm", "add_rms_norm_fp8", "tree_attention", "select_pages"])
def test_graph_replays(name):
    """A captured call reads its tensors anew in every replay, with eager work and synchronizations between."""
    call, inputs = _calls()[name]
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for step in range(4):
        for t in inputs:
            if t.dtype == torch.int32:
                t.copy_(torch.randint(0, 5, t.shape, dtype=torch.int32, device="cuda", generator=_gen(step)))
            else:
                t.copy_(_randn(_gen(step), *t.shape))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out if x is not None]
        assert _same(got, [x for x in call() if x is not None]), step
        torch.cuda.synchronize()


@pytest.mark.parametrize("name", ["step_tables", "add_rms_norm", "add_rms_norm_fp8", "tree_attention", "select_pages"])
def test_eager_calls_and_ops_agree(name, monkeypatch):
    """The eager module, the Python path and the op that a profiler sees: the same bits."""
    from gguf_hip import attention, norm, sparse, steps

    call, _ = _calls()[name]
    want = [x.clone() for x in call() if x is not None]
    if _lib._fast is not None:
        taken = []
        for module, names in ((attention, ("tree_attention", "paged_attention")), (norm, ("add_rms_norm",)),
                              (sparse, ("page_bounds", "select_pages")), (steps, ("step_tables",))):
            class Seen:
                def __getattr__(self, n):
                    def through(*a):
                        got = getattr(_lib._fast, n)(*a)
                        taken.append((n, got is not None))
                        return got
                    return through
            monkeypatch.setattr(module, "_fast", Seen())
        assert _same([x for x in call() if x is not None], want) and taken and all(ok for _, ok in taken), taken
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        assert _same([x for x in call() if x is not None], want)
    assert any(("gguf_hip::" + name.replace("_fp8", "")) in ev.key for ev in prof.key_averages())
    for module in (attention, norm, sparse, steps):
        monkeypatch.setattr(module, "_fast", None)
    assert _same([x for x in call() if x is not None], want)
    with torch.inference_mode():
        assert _same([x for x in call() if x is not None], want)


def test_gradients_raise_and_values_stay():
    context, counts = [30], [4]
    q, k, v, table, lens, starts, mask, _, _ = _tree_case(2, context, counts, 4, 2, 64, 16, BF, BF, "tree")
    x, r, w = _randn(_gen(1), 4, 256, dtype=BF), _randn(_gen(2), 4, 256, dtype=BF), _randn(_gen(3), 256, dtype=BF)
    for call, t in ((lambda t: gguf_hip.tree_attention(t, k, v, table, lens, starts, mask), q),
                    (lambda t: gguf_hip.tree_attention(q, k, t, table, lens, starts, mask), v),
                    (lambda t: gguf_hip.add_rms_norm(t, r, w)[0], x), (lambda t: gguf_hip.add_rms_norm(t * 1, r, w)[1], x),
                    (lambda t: gguf_hip.add_rms_norm(x, t, w)[1], r), (lambda t: gguf_hip.add_rms_norm(x, r, t)[0], w),
                    (lambda t: gguf_hip.add_rms_norm_fp8(x, r, t)[1], w)):
        want = call(t)
        leaf = torch.nn.Parameter(t)
        got = call(leaf)
        assert got.requires_grad and not want.requires_grad and torch.equal(got, want)
        with pytest.raises(RuntimeError, match="no backward"):
            got.float().sum().backward()
        with torch.no_grad():
            got = call(leaf)
        assert not got.requires_grad and torch.equal(got, want)
    y = torch.nn.Parameter(x) * 2                            # in place of a tensor that belongs to a graph
    out, res = gguf_hip.add_rms_norm(y, r, w, out=y)
    assert out is y and "NoBackward" in out.grad_fn.name() and "NoBackward" in res.grad_fn.name()
    assert torch.equal(out, gguf_hip.add_rms_norm(x * 2, r, w)[0])


def test_lazily_negated_tensors():
    """Tensors whose memory is not their value go through the op."""
    x, r, w = _randn(_gen(1), 4, 256, dtype=BF), _randn(_gen(2), 4, 256, dtype=BF), _randn(_gen(3), 256, dtype=BF)
    want = gguf_hip.add_rms_norm(x, r, w)
    got = gguf_hip.add_rms_norm(torch._neg_view(-x), torch._neg_view(-r), torch._neg_view(-w))
    assert _same(got, want)
    q, k, v, table, lens, starts, mask, _, _ = _tree_case(2, [30], [4], 4, 2, 64, 16, BF, BF, "tree")
    assert torch.equal(gguf_hip.tree_attention(torch._neg_view(-q), k, v, table, lens, starts, mask),
                       gguf_hip.tree_attention(q, k, v, table, lens, starts, mask))


def test_eight_bit_output_of_shared_memory_is_refused():
    x = _randn(_gen(1), 4, 256, dtype=BF)
    with pytest.raises(ValueError, match="memory of its own"):
        gguf_hip.add_rms_norm_fp8(x, None, out=x.view(F8)[:, :256])


def test_norm_outputs_that_share_memory():
    """An output may be an input, lie between its rows, or reach over other rows of it; the outputs share nothing with each other."""
    gen, dim = _gen(7), 192
    buf, r, w = _randn(gen, 65, 2 * dim, dtype=BF), _randn(gen, 64, dim, dtype=BF), _randn(gen, dim, dtype=BF)
    start = buf.clone()

    def views(t):
        return {"rows before": (t[1:, :dim], t[:-1, :dim]), "rows behind": (t[:-1, :dim], t[1:, :dim]), "columns": (t[1:, :dim], t[1:, dim:]),
                "columns across": (t[:-1, dim // 2:dim // 2 + dim], t[:-1, :dim]), "the same": (t[:-1, :dim], t[:-1, :dim])}

    for name in views(buf):
        for as_residual in (False, True):
            for to_residual in (False, True):
                buf.copy_(start)
                x, out = views(buf)[name]
                a, b = (r, x) if as_residual else (x, r)
                want, want_s = gguf_hip.add_rms_norm(a.clone(), b.clone(), w)
                got = gguf_hip.add_rms_norm(a, b, w, **{"out_residual" if to_residual else "out": out})
                assert _same(got, (want, want_s)), (name, as_residual, to_residual)
                assert got[to_residual].data_ptr() == out.data_ptr()
    for o, p in ((buf[1:, :dim], buf[1:, :dim]), (buf[1:, :dim], buf[:-1, :dim]), (buf[:-1, dim - 8:2 * dim - 8], buf[:-1, :dim])):
        with pytest.raises(ValueError, match="share memory"):
            gguf_hip.add_rms_norm(r, r, w, out=o, out_residual=p)
    for o in (torch.empty_like(r), r):   # one tensor for both
        with pytest.raises(ValueError, match="share memory"):
            gguf_hip.add_rms_norm(r, r, w, out=o, out_residual=o)
    want = gguf_hip.add_rms_norm(r, r, w)
    got = gguf_hip.add_rms_norm(r, r, w, out=buf[1:, :dim], out_residual=buf[1:, dim:])   # side by side
    assert _same(got, want)
    rows = r.clone()
    want = gguf_hip.add_rms_norm(rows, r, rows[3].clone())
    assert _same(gguf_hip.add_rms_norm(rows, r, rows[3], out=rows), want)


def test_tree_out_over_q():
    """Into q itself, and into rows and heads of it that other tokens' q lie in."""
    for counts in ([30, 1, 9], [3, 0, 2]):
        q, k, v, table, lens, starts, mask, _, _ = _tree_case(3, [40, 9, 0], counts, 8, 2, 64, 16, BF, BF, "tree")
        n = sum(counts)
        buf = torch.zeros((n + 1, 16, 64), dtype=BF, device="cuda")
        few = torch.zeros(64, dtype=torch.int32, device="cuda")   # holds no partial sums: one split
        want = gguf_hip.tree_attention(q, k, v, table, lens, starts, mask, workspace=few)
        for at, to in ((buf[:n, :8], buf[:n, :8]), (buf[:n, :8], buf[1:, :8]), (buf[1:, :8], buf[:n, :8]), (buf[:n, :8], buf[:n, 4:12])):
            at.copy_(q)
            got = gguf_hip.tree_attention(at, k, v, table, lens, starts, mask, out=to, workspace=few)
            assert got is to and torch.equal(got, want)


def test_bounds_of_more_pages_than_a_grid_has_rows():
    gen = _gen(8)
    k = _randn(gen, 70, 1, 2, 64, dtype=BF)
    table = torch.randint(0, 70, (2, 70_000), dtype=torch.int32, device="cuda", generator=gen)
    bounds = torch.zeros((70, 2, 2, 64), dtype=BF, device="cuda")
    gguf_hip.page_bounds(k, table, _i32([70_000, 3]), bounds, count=70_000)
    assert torch.equal(bounds, k.expand(70, 2, 2, 64))


def test_as_many_sequences_as_a_batch_holds():
    """65535 sequences of a token each: tables, attention in both forms, and the choice of pages."""
    gen, n = _gen(9), 65535
    k, v = (_randn(gen, 40, 8, 1, 64, dtype=BF) for _ in range(2))
    lists = torch.randint(0, 40, (50, 3), dtype=torch.int32, device="cuda", generator=gen)
    request = torch.randint(0, 50, (n,), dtype=torch.int32, device="cuda", generator=gen)
    old = torch.randint(0, 23, (n,), dtype=torch.int32, device="cuda", generator=gen)
    t = gguf_hip.step_tables(lists, request, old, torch.ones_like(old), n, 8)
    assert torch.equal(t.lengths, old + 1) and torch.equal(t.starts, torch.arange(n + 1, device="cuda", dtype=torch.int32))
    assert torch.equal(t.sequences, t.starts[:-1]) and torch.equal(t.positions, old)
    q = _randn(gen, n, 2, 64, dtype=BF)
    one = gguf_hip.paged_attention(q, k, v, t.block_table, t.lengths)
    many = gguf_hip.tree_attention(q, k, v, t.block_table, t.lengths, t.starts, max_tokens=1)
    assert (one.float() - many.float()).abs().max() <= 2 * 2.0 ** -7 * v.abs().max()   # two roundings of weights and outputs each
    bounds = gguf_hip.page_bounds(k, t.block_table, t.lengths, torch.zeros((40, 2, 1, 64), dtype=BF, device="cuda"), count=24)
    table, lengths = gguf_hip.select_pages(q, bounds, t.block_table, t.lengths, 2, 8)
    pages = (old + 8) // 8
    assert torch.equal(table[:, 0, 0], t.block_table[:, 0])
    assert torch.equal(lengths, torch.where(pages > 2, old + 1 - 8, old + 1))


# ---- all together ----------------------------------------------------------------------------

def test_draft_step_example():
    """examples/draft_step.py: chunks of prompts, trees and sparse steps by graphs over a padded batch.  Per layer a token's value is
    rounded at most ten times on its way (norm, projection, adapter, heads, cache, probabilities, attention, projection, adapter, residual),
    weights once, each at most 2^-8 of it, and once by the last norm: two layers stay within 23 * 2^-8."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "draft_step.py")
    spec = importlib.util.spec_from_file_location("draft_step", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    got = module.run(steps=5)
    assert sorted(got["errors"]) == ["a", "b", "c"] and got["outputs"] > 150 and got["pages"] > got["keep"]
    assert max(got["errors"].values()) < 23 * 2.0 ** -8, got
