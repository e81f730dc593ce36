"""The operators of steps of several new tokens and of long caches where a mask, a window, a table or a size ends, on the GPU: what a row sees reaches it
whatever it holds, what no row sees is not looked at, no page outside of the cache is read.  Definitions in 64 bits and tolerances per value are
those of test_gpu_step_ops.py."""
import pytest
import torch

import gguf_hip
from test_gpu_step_ops import BF, F8, F16, INF, NAN, _attend_exact, _bytes, _i32, _sees, _select_exact, _tree_case, _within

pytestmark = pytest.mark.gpu

# rows of a sequence and key head that one tile of 64 rows holds, whose keys two waves share, and that tiles of 128 rows hold
FEW, MANY = [4, 9, 5], [50, 21, 30]


def _behind_a_page(t, fill):
    """The cache with another page in front of its first, in the same layout."""
    first = torch.zeros_like(t[:1])
    _bytes(first)[:] = fill
    heads = t.stride(1) < t.stride(2)     # a head's tokens lie together
    parts = [x.transpose(1, 2) if heads else x for x in (first, t)]
    got = torch.cat([_bytes(x.contiguous()) for x in parts])
    got = got.view(F8) if t.dtype == F8 else got
    return got.transpose(1, 2) if heads else got


@pytest.mark.parametrize("qt,ct", [(BF, BF), (F16, F16), (BF, F8)])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (128, 7), (80, 16), (256, 48)])
@pytest.mark.parametrize("counts", [FEW, MANY])
@pytest.mark.parametrize("kind", ["tree", "chain"])
def test_tree_bad_pages_where_the_first_page_is_not_finite(qt, ct, dim, page, counts, kind):
    """A page outside of the cache gives NaN to those that see its keys and is not read, among the new tokens' keys, the last of the cache
    and far from both, whatever the cache's first page holds (as one that was never written may)."""
    context = [100, 230, 45]
    q, k, v, table, lens, starts, mask, _, _ = _tree_case(dim + page, context, counts, 6, 2, dim, page, qt, ct, kind)
    want, _, tol, _ = _attend_exact(q, k, v, table, context, counts, mask, dim ** -0.5, 0)
    k, v = (_behind_a_page(t, 0x7F if ct == F8 else NAN) for t in (k, v))
    assert _bytes(v[:1]).float().isnan().all() or ct == F8
    sound = table + 1                                   # (the entries that no sequence uses become -2^31)
    ends = [0, counts[0], counts[0] + counts[1], sum(counts)]
    out = gguf_hip.tree_attention(q, k, v, sound, lens, starts, mask)
    _within(out, want, tol, "sound")
    for bad in (-1, 2 ** 30, 2 ** 31 - 1, k.shape[0], -2 ** 31):
        for where in (3, context[1] - 1, context[1]):   # keys of the second sequence
            table = sound.clone()
            table[1, where // page] = bad
            for window in (0, 200):
                out = gguf_hip.tree_attention(q, k, v, table, lens, starts, mask, window=window)
                sees = _sees(mask, ends[1], context[1], counts[1], window)
                hit = sees[:, where // page * page:(where // page + 1) * page].any(1)
                assert window or hit.any()
                assert out[ends[1]:ends[2]][hit].isnan().all(), (bad, where, window)
                if not window:
                    for lo, hi in ((ends[0], ends[1]), (ends[2], ends[3])):
                        _within(out[lo:hi], want[lo:hi], tol[lo:hi], "the sound ones")


@pytest.mark.parametrize("qt,ct,x", [(BF, BF, NAN), (F16, F16, INF), (BF, BF, -INF), (BF, F8, NAN), (F16, F8, NAN)])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (128, 7), (256, 16), (80, 32)])
@pytest.mark.parametrize("counts", [FEW, MANY])
@pytest.mark.parametrize("kind", ["tree", "chain", "any"])
@pytest.mark.parametrize("window", [0, 90])
def test_tree_what_is_seen_counts_whatever_it_holds(qt, ct, x, dim, page, counts, kind, window):
    """One value that is not finite makes that dim of its head not finite for every token that sees its key, and changes nothing else: keys of the
    cache's last steps in either half of them, at the window's edge in either half, and the new tokens' own."""
    context = [40, 185, 64]                             # 40 of 64, 57 of 64 and 0 of 64 keys in the step where the new ones begin
    q, k, v, table, lens, starts, mask, _, _ = _tree_case(dim, context, counts, 6, 2, dim, page, qt, ct, kind)
    want, _, tol, _ = _attend_exact(q, k, v, table, context, counts, mask, dim ** -0.5, window)
    t0 = 0
    for b, (m, n) in enumerate(zip(context, counts)):
        sees = _sees(mask, t0, m, n, window)
        for j in sorted({0, 5, 31, 32, 39, *range(m - window - 20, m - window + 45, 7), *range(m - 65, m + n, 9), m, m + n - 1}):
            if not 0 <= j < m + n:
                continue
            h, d, at = j % 2, j * 5 % dim, int(table[b, j // page])
            bad = v.clone()
            if ct == F8:
                _bytes(bad)[at, j % page, h, d] = 0x7F
            else:
                bad[at, j % page, h, d] = x
            out = gguf_hip.tree_attention(q, k, bad, table, lens, starts, mask, window=window)
            hit = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
            hit[t0:t0 + n, 3 * h:3 * h + 3, d] = sees[:, j, None]
            assert not torch.isfinite(out[hit].float()).any(), (b, j)
            _within(out[~hit], want[~hit], tol[~hit], (b, j))
        t0 += n


@pytest.mark.parametrize("qt,ct", [(BF, BF), (BF, F8)])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 1), (128, 7), (128, 16), (80, 8), (80, 16), (256, 48), (64, 64), (256, 20)])
@pytest.mark.parametrize("counts", [FEW, MANY])
@pytest.mark.parametrize("kind", ["tree", "chain", "any"])
def test_tree_pages_behind_the_window_may_be_given_up(qt, ct, dim, page, counts, kind):
    """What no token of a sequence sees under the window is not looked up: entries outside of the cache there change nothing, in one split and in many.
    The first page that a token does see is looked up: such an entry in its place gives it NaN."""
    context = [700, 90, 1301]
    q, k, v, table, lens, starts, mask, _, _ = _tree_case(dim + page, context, counts, 6, 2, dim, page, qt, ct, kind)
    few = torch.zeros(64, dtype=torch.int32, device="cuda")   # holds no partial sums: one split
    for window in (1, 2, 17, 33, 64, 200, 641):
        want, _, tol, _ = _attend_exact(q, k, v, table, context, counts, mask, dim ** -0.5, window)
        given_up, t0, ends = table.clone(), 0, []
        for b, (m, n) in enumerate(zip(context, counts)):
            sees = _sees(mask, t0, m, n, window)
            first = int(sees.any(0).nonzero()[0])
            given_up[b, :first // page] = torch.tensor([-1, 2 ** 30, k.shape[0]], device="cuda").to(torch.int32).repeat(first // page)[:first // page]
            ends.append((t0, b, first // page, sees[:, :(first // page + 1) * page].any(1)))
            t0 += n
        for workspace in (None, few):
            out = gguf_hip.tree_attention(q, k, v, given_up, lens, starts, mask, window=window, workspace=workspace)
            _within(out, want, tol, window)
            again = gguf_hip.tree_attention(q, k, v, table, lens, starts, mask, window=window, workspace=workspace)
            assert torch.equal(out, again)
        t0, b, at, hit = ends[2]
        given_up[b, at] = -1
        out = gguf_hip.tree_attention(q, k, v, given_up, lens, starts, mask, window=window)
        assert out[t0:][hit].isnan().all() and hit.any()
        _within(out[:t0], want[:t0], tol[:t0], "the other sequences")


def test_norm_of_more_rows_than_a_launch_has_workgroups():
    """2^24 and more rows, in 16 bits and in 8: the first, those about the limit and the last are their own batch's."""
    rows, dim = (1 << 24) + 77, 8
    gen = torch.Generator(device="cuda").manual_seed(5)
    x, r = (torch.randint(-99, 100, (rows, dim), device="cuda", generator=gen, dtype=torch.int8).to(BF) for _ in range(2))
    out, res = gguf_hip.add_rms_norm(x, r)
    out8, scale, _ = gguf_hip.add_rms_norm_fp8(x, r)
    for lo, hi in ((0, 500), ((1 << 24) - 300, (1 << 24) + 60), (rows - 20, rows), (5_000_000, 5_000_100)):
        want, want_r = gguf_hip.add_rms_norm(x[lo:hi], r[lo:hi])
        want8, want_s, _ = gguf_hip.add_rms_norm_fp8(x[lo:hi], r[lo:hi])
        assert torch.equal(out[lo:hi], want) and torch.equal(res[lo:hi], want_r) and want.any()
        assert torch.equal(_bytes(out8[lo:hi]), _bytes(want8)) and torch.equal(scale[lo:hi], want_s)


def test_bounds_of_more_pages_than_a_launch_has_workgroups():
    """A sequence of 2^24 and more pages of one token: the first and the last of them too."""
    n = (1 << 24) + 1000
    k = torch.randn((90, 1, 1, 8), device="cuda", generator=torch.Generator(device="cuda").manual_seed(6)).to(BF)
    table = torch.full((1, n), 7, dtype=torch.int32, device="cuda")
    table[0, :10], table[0, -10:], table[0, (1 << 24) - 20:(1 << 24) + 20] = _i32(list(range(10, 20))), _i32(list(range(20, 30))), _i32(list(range(30, 70)))
    bounds = torch.zeros((90, 2, 1, 8), dtype=BF, device="cuda")
    gguf_hip.page_bounds(k, table, _i32([n]), bounds, count=n)
    used = torch.tensor([7, *range(10, 70)], device="cuda")
    assert torch.equal(bounds[used], k.expand(90, 2, 1, 8)[used])
    bounds[used] = 0
    assert not bounds.any()


@pytest.mark.parametrize("size", [2.0 ** 70, 2.0 ** -80])
def test_select_scores_beyond_32_bits(size):
    """Products that a 32-bit number cannot hold are told apart in 64 bits: of bounds and queries of a size whose square is above or below its range."""
    pages, keep = 200, 12
    gen = torch.Generator(device="cuda").manual_seed(7)
    k = (torch.randn((pages, 4, 2, 16), device="cuda", generator=gen) * size).to(BF)
    q = (torch.randn((1, 4, 16), device="cuda", generator=gen) * size).to(BF)
    table = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)[None]
    bounds = gguf_hip.page_bounds(k, table, _i32([4 * pages]), torch.zeros((pages, 2, 2, 16), dtype=BF, device="cuda"), count=4 * pages)
    got, kept = gguf_hip.select_pages(q, bounds, table, _i32([4 * pages]), keep, 4)
    want, want_n = _select_exact(q, bounds, table, [4 * pages], keep, 4, 1, 1)
    assert torch.equal(got.cpu(), want) and kept.tolist() == want_n


def test_eight_bit_output_beside_its_inputs():
    """In the bytes behind each row of the input, and of the residual."""
    buf = torch.randn((300, 200), device="cuda", generator=torch.Generator(device="cuda").manual_seed(8)).to(BF)
    for lo in (0, 1):
        x, out = buf[:, 64 * lo:64 * lo + 64], buf.view(F8)[:, 256:320]
        before = buf.clone()
        for kw in (dict(x=x, residual=None), dict(x=x, residual=buf[:, 160:200].repeat(1, 2)[:, :64]), dict(x=buf[:, :64].clone(), residual=x, out_residual=x)):
            copies = {n: None if t is None else t.clone() for n, t in kw.items() if n != "out_residual"}
            want, scale, res = gguf_hip.add_rms_norm_fp8(**copies)
            got, scale2, res2 = gguf_hip.add_rms_norm_fp8(**kw, out=out)
            assert got is out and torch.equal(_bytes(out), _bytes(want)) and torch.equal(scale, scale2)
            assert res is None and res2 is None or torch.equal(res, res2)
        assert torch.equal(buf[:, 160:], before[:, 160:]) and torch.equal(buf[:, 64 * (1 - lo):64 * (1 - lo) + 64], before[:, 64 * (1 - lo):64 * (1 - lo) + 64])


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 4), (256, 7)])
@pytest.mark.parametrize("counts", [[20], [90]])
def test_tree_rows_that_see_nothing_hold_no_page(dim, page, counts):
    """Without a cache a row whose mask is empty sees no key, and under the window the others see the last ones: the pages before them are not
    looked up for its sake."""
    n, window = counts[0], 3
    q, k, v, table, lens, starts, mask, _, _ = _tree_case(dim, [0], counts, 6, 2, dim, page, BF, BF, "tree")
    j = torch.arange(n, device="cuda")
    mask[:] = 0
    for i in range(n):                                   # the last three of the sequence, or nothing
        if i % 3:
            for bit in range(n - 3, n):
                mask[i, bit // 32] |= 1 << bit % 32 if bit % 32 < 31 else -2 ** 31
    want, _, tol, _ = _attend_exact(q, k, v, table, [0], counts, mask, dim ** -0.5, window)
    table[0, :(n - 3) // page] = -1
    assert (table[0] == -1).any()
    out = gguf_hip.tree_attention(q, k, v, table, lens, starts, mask, window=window)
    _within(out, want, tol, "out")
    assert not out[j % 3 == 0].any() and out[j % 3 > 0].any()
