"""CPU tests of the operators of steps of several new tokens and of long caches: shapes under fake tensors, the refusals of every entry
point (Python's and the C ABI's; nothing is launched), gradients and tracing."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import gguf_hip
from gguf_hip import _lib
from gguf_hip._lib import lib

BF, F16, F32, F8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
I32, I64 = torch.int32, torch.int64


def _fake(shape, dtype=BF):
    return torch.empty(shape, dtype=dtype, device="cuda")


def _i32(*shape):
    return _fake(shape, I32)


def _tables_args(**over):
    return {**dict(page_lists=_i32(6, 9), requests=_i32(3), lengths=_i32(3), counts=_i32(3), tokens=20, page_size=16), **over}


def _norm_args(**over):
    return {**dict(x=_fake((5, 64)), residual=_fake((5, 64)), weight=_fake((64,))), **over}


def _tree_args(**over):
    return {**dict(q=_fake((12, 8, 64)), k_pages=_fake((9, 16, 2, 64)), v_pages=_fake((9, 16, 2, 64)), block_table=_i32(3, 4),
                   lengths=_i32(3), starts=_i32(4), mask=_i32(12, 1)), **over}


def _select_args(**over):
    return {**dict(q=_fake((3, 8, 64)), bounds=_fake((9, 2, 2, 64)), block_table=_i32(3, 7), lengths=_i32(3), keep=4, page_size=16), **over}


def _bounds_args(**over):
    return {**dict(k_pages=_fake((9, 16, 2, 64)), block_table=_i32(3, 4), lengths=_i32(3), bounds=_fake((9, 2, 2, 64))), **over}


def test_cpu_tensors_are_refused():
    z = lambda *s, dtype=BF: torch.zeros(s, dtype=dtype)  # noqa: E731
    i = lambda *s: z(*s, dtype=I32)  # noqa: E731
    for call in (lambda: gguf_hip.step_tables(i(6, 9), i(3), i(3), i(3), 20, 16), lambda: gguf_hip.add_rms_norm(z(5, 64), None),
                 lambda: gguf_hip.add_rms_norm_fp8(z(5, 64), None),
                 lambda: gguf_hip.tree_attention(z(12, 8, 64), z(9, 16, 2, 64), z(9, 16, 2, 64), i(3, 4), i(3), i(4)),
                 lambda: gguf_hip.page_bounds(z(9, 16, 2, 64), i(3, 4), i(3), z(9, 2, 2, 64)),
                 lambda: gguf_hip.select_pages(z(3, 8, 64), z(9, 2, 2, 64), i(3, 7), i(3), 4, 16)):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_step_tables_shapes_and_refusals():
    with FakeTensorMode():
        t = gguf_hip.step_tables(**_tables_args())
        assert t.block_table.shape == (3, 9) and t.starts.shape == (4,) and t.lengths.shape == (3,) and t.mask is None
        assert t.slots.dtype == I64 and t.slots.shape == t.positions.shape == t.sequences.shape == (20,)
        t = gguf_hip.step_tables(**_tables_args(requests=_fake((3,), I64), parents=_i32(20), tree=33))
        assert t.mask.shape == (20, 2) and t.mask.dtype == I32
        assert gguf_hip.step_tables(**_tables_args(requests=_i32(0), lengths=_i32(0), counts=_i32(0))).starts.shape == (1,)
        assert gguf_hip.step_tables(**_tables_args(page_lists=_i32(12, 20)[::2, 3:12], tokens=0)).slots.shape == (0,)
        for bad in (dict(page_lists=_fake((6, 9), I64)), dict(page_lists=_i32(9)), dict(page_lists=_i32(9, 6).t()),
                    dict(page_lists=_i32(1, 9).expand(6, 9)), dict(requests=_fake((3,), F32)), dict(requests=_i32(3, 1)), dict(requests=_i32(6)[::2]),
                    dict(lengths=_i32(4)), dict(lengths=_fake((3,), I64)), dict(counts=_i32(2)), dict(counts=_i32(6)[::2]),
                    dict(tokens=-1), dict(tokens=2 ** 31), dict(page_size=0), dict(parents=_i32(20)), dict(tree=4),
                    dict(parents=_i32(19), tree=4), dict(parents=_fake((20,), I64), tree=4), dict(parents=_i32(20), tree=1025),
                    dict(parents=_i32(20), tree=-1), dict(requests=_i32(65536), lengths=_i32(65536), counts=_i32(65536))):
            with pytest.raises(ValueError):
                gguf_hip.step_tables(**_tables_args(**bad))


def test_norm_shapes_and_refusals():
    with FakeTensorMode():
        out, res = gguf_hip.add_rms_norm(**_norm_args())
        assert out.shape == res.shape == (5, 64) and out.dtype == res.dtype == BF
        assert gguf_hip.add_rms_norm(_fake((5, 64)), None)[1] is None
        x, r = _fake((5, 64)), _fake((5, 64))
        got = gguf_hip.add_rms_norm(x, r, out=x, out_residual=r)
        assert got[0] is x and got[1] is r
        out, scale, res = gguf_hip.add_rms_norm_fp8(**_norm_args())
        assert out.dtype == F8 and scale.shape == (5, 1) and scale.dtype == F32 and res.dtype == BF
        assert gguf_hip.add_rms_norm_fp8(**_norm_args(weight=_fake((64,), F32), group=32, unit_offset=True))[1].shape == (5, 2)
        both = (dict(x=_fake((5, 64), F32)), dict(x=_fake((64,))), dict(x=_fake((5, 0)), residual=None, weight=None), dict(residual=_fake((5, 63))),
                dict(residual=_fake((5, 64), F16)), dict(residual=_fake((4, 64))), dict(weight=_fake((63,))), dict(weight=_fake((64,), F16)),
                dict(weight=_fake((128,))[::2]), dict(weight=None, unit_offset=True), dict(residual=None, out_residual=_fake((5, 64))),
                dict(out_residual=_fake((5, 64), F16)), dict(out_residual=_fake((64, 5)).t()), dict(out_residual=_fake((1, 64)).expand(5, 64)),
                dict(out=_fake((5, 63))), dict(out=_fake((5, 64), F32)),
                dict(x=_fake((2, 32769)), residual=None, weight=None))
        for bad in both:
            for call in (gguf_hip.add_rms_norm, gguf_hip.add_rms_norm_fp8):
                with pytest.raises(ValueError):
                    call(**_norm_args(**bad))
        for bad in (dict(out=_fake((5, 64), F8)), dict(out=_fake((64, 5)).t())):
            with pytest.raises(ValueError):
                gguf_hip.add_rms_norm(**_norm_args(**bad))
        for bad in (dict(out=_fake((5, 64))), dict(group=16), dict(group=48), dict(group=128), dict(group=1024), dict(group=-32)):
            with pytest.raises(ValueError):
                gguf_hip.add_rms_norm_fp8(**_norm_args(**bad))


def test_tree_attention_shapes_and_refusals():
    with FakeTensorMode():
        assert gguf_hip.tree_attention(**_tree_args()).shape == (12, 8, 64)
        out, lse = gguf_hip.tree_attention(**_tree_args(mask=None), return_lse=True, max_tokens=100)
        assert out.dtype == BF and lse.shape == (12, 8) and lse.dtype == F32
        f8 = _fake((9, 16, 2, 64), F8)
        assert gguf_hip.tree_attention(**_tree_args(k_pages=f8, v_pages=f8), k_scale=_fake((2,), F32)).dtype == BF
        assert gguf_hip.tree_attention(**_tree_args(q=_fake((0, 8, 64)), mask=None)).shape == (0, 8, 64)
        for bad in (dict(q=_fake((12, 8, 64), F32)), dict(q=_fake((12, 512))), dict(q=_fake((12, 7, 64))), dict(q=_fake((12, 8, 64), F16)),
                    dict(q=_fake((12, 8, 32))), dict(q=_fake((12, 2050, 64))), dict(v_pages=_fake((9, 16, 2, 32))),
                    dict(block_table=_fake((3, 4), I64)), dict(block_table=_i32(2, 4)), dict(block_table=_i32(3, 2, 4)),
                    dict(block_table=_i32(4, 3).t()), dict(lengths=_fake((3,), I64)), dict(lengths=_i32(4)), dict(starts=_i32(3)),
                    dict(starts=_fake((4,), I64)), dict(starts=_i32(8)[::2]), dict(mask=_i32(11, 1)), dict(mask=_i32(12)), dict(mask=_i32(12, 0)),
                    dict(mask=_fake((12, 1), I64)), dict(mask=_i32(12, 4)[:, ::2]), dict(max_length=65), dict(max_length=-1),
                    dict(max_tokens=-1), dict(window=-1), dict(k_scale=_fake((3,), F32)), dict(out=_fake((12, 8, 64), F16)),
                    dict(out=_fake((12, 8, 32))), dict(workspace=_fake((1 << 20, 2), I32)[:, 0]), dict(mask=torch.empty((12, 1), dtype=I32))):
            with pytest.raises(ValueError):
                gguf_hip.tree_attention(**_tree_args(**bad))


def test_sparse_shapes_and_refusals():
    with FakeTensorMode():
        args = _bounds_args()
        assert gguf_hip.page_bounds(**args, count=5) is args["bounds"]
        for bad in (dict(k_pages=_fake((9, 16, 64))), dict(k_pages=_fake((9, 16, 2, 64), F32)), dict(k_pages=_fake((9, 16, 2, 128))[..., ::2]),
                    dict(bounds=_fake((8, 2, 2, 64))), dict(bounds=_fake((9, 2, 2, 64), F16)), dict(bounds=_fake((9, 2, 64, 2)).transpose(2, 3)),
                    dict(block_table=_fake((3, 4), I64)), dict(block_table=_i32(4, 4)), dict(lengths=_fake((3,), I64)), dict(count=-1),
                    dict(count=2 ** 31)):
            with pytest.raises(ValueError):
                gguf_hip.page_bounds(**_bounds_args(**bad))
        table, kept = gguf_hip.select_pages(**_select_args())
        assert table.shape == (3, 2, 4) and table.dtype == I32 and kept.shape == (3,)
        pages = _fake((9, 16, 2, 64))
        assert gguf_hip.paged_attention(_fake((3, 8, 64)), pages, pages, table, kept).shape == (3, 8, 64)
        for bad in (dict(q=_fake((3, 8, 64), F32)), dict(q=_fake((3, 7, 64))), dict(q=_fake((3, 8, 32))), dict(q=_fake((4, 8, 64))), dict(q=_fake((3, 512))),
                    dict(bounds=_fake((9, 2, 2, 64), F16)), dict(bounds=_fake((9, 3, 2, 64))), dict(bounds=_fake((0, 2, 2, 64))),
                    dict(bounds=_fake((9, 2, 64, 2)).transpose(2, 3)), dict(block_table=_i32(3, 2, 7)), dict(block_table=_fake((3, 7), I64)),
                    dict(lengths=_i32(2)), dict(keep=0), dict(keep=2 ** 31), dict(page_size=0), dict(sink=-1), dict(recent=0), dict(sink=4),
                    dict(sink=2, recent=3), dict(max_length=113), dict(max_length=-1), dict(workspace=torch.empty(9, dtype=I32))):
            with pytest.raises(ValueError):
                gguf_hip.select_pages(**_select_args(**bad))
        for bad in (_i32(3, 3, 4), _i32(2, 2, 4), _i32(3, 4, 2).transpose(1, 2), _i32(3, 2, 4, 1)):
            with pytest.raises(ValueError):
                gguf_hip.paged_attention(_fake((3, 8, 64)), pages, pages, bad, kept)


P = ctypes.c_void_p(4096)   # never dereferenced: the checks come first
ODD = ctypes.c_void_p(4097)


def _c_pages(**over):
    f = dict(k=4096, v=4096, k_page=2048, k_token=128, k_head=64, v_page=2048, v_token=128, v_head=64, k_scale=None,
             v_scale=None, dtype=1, pages=9, page_size=16, heads=2, dim=64)
    f.update(over)
    return _lib.GqkPages(*f.values())


def test_c_tables_refusals():
    def call(lists=P, row=9, n=6, width=9, requests=P, lengths=P, counts=P, batch=3, tokens=20, page=16, parents=None, tree=0, table=P, totals=P,
             starts=P, sequences=P, positions=P, slots=P, mask=None):
        return lib.gqk_step_tables(lists, row, n, width, requests, 0, lengths, counts, batch, tokens, page, parents, tree, table, totals, starts,
                                   sequences, positions, slots, mask, None)

    for bad in (dict(n=-1), dict(width=-1), dict(batch=-1), dict(batch=65536), dict(tokens=-1), dict(page=0), dict(parents=P), dict(tree=4),
                dict(parents=P, tree=1025, mask=P), dict(row=8), dict(tree=-1)):
        assert call(**bad) == _lib.GQK_ERR_SHAPE, bad
    for bad in (dict(lists=None), dict(requests=None), dict(lengths=None), dict(counts=None), dict(table=None), dict(totals=None), dict(starts=None),
                dict(sequences=None), dict(positions=None), dict(slots=None), dict(parents=P, tree=4)):
        assert call(**bad) == _lib.GQK_ERR_ARG, bad


def test_c_norm_refusals():
    def call(x=P, x_row=64, r=P, r_row=64, dtype=1, rows=5, dim=64, w=P, wt=1, flags=0, out=P, out_row=64, ot=1, scale=None, group=0, res=P,
             res_row=64):
        return lib.gqk_add_rms_norm(x, x_row, r, r_row, dtype, rows, dim, w, wt, 1e-6, flags, out, out_row, ot, scale, group, res, res_row, None)

    assert call(rows=0) == 0
    for bad in (dict(dtype=0), dict(dtype=3), dict(ot=2), dict(ot=0), dict(wt=2), dict(w=None, flags=1), dict(x=None), dict(out=None),
                dict(ot=3, scale=None), dict(r=None)):
        assert call(**bad) == _lib.GQK_ERR_ARG, bad
    for bad in (dict(rows=-1), dict(rows=2 ** 31), dict(dim=0), dict(dim=32769), dict(group=32), dict(ot=3, scale=P, group=16),
                dict(ot=3, scale=P, group=48), dict(ot=3, scale=P, group=128), dict(x_row=63), dict(out_row=63), dict(r_row=0), dict(res_row=1),
                dict(x=ODD), dict(out=ODD), dict(r=ODD), dict(w=ODD), dict(wt=0, w=ctypes.c_void_p(4098)), dict(ot=3, scale=ctypes.c_void_p(4098))):
        assert call(**bad) == _lib.GQK_ERR_SHAPE, bad


def test_c_tree_refusals():
    def call(pages=None, q=P, q_row=512, q_head=64, dtype=1, tokens=12, batch=3, heads=8, table=P, width=4, lengths=P, starts=P, mask=P, words=1,
             most=64, most_tokens=12, window=0, out=P, ws=P, ws_bytes=1 << 40):
        pages = _c_pages() if pages is None else pages
        return lib.gqk_tree_attention(q, q_row, q_head, dtype, tokens, batch, heads, ctypes.byref(pages) if pages else None, table, width, width,
                                      lengths, starts, mask, words, most, most_tokens, window, 0.1, out, 512, 64, None, ws, ws_bytes, None)

    assert call(tokens=0) == 0 and call(batch=0) == 0
    for bad in (dict(dtype=0), dict(dtype=3), dict(dtype=2), dict(pages=_c_pages(dtype=0)), dict(pages=_c_pages(k=None)), dict(q=None),
                dict(out=None), dict(lengths=None), dict(starts=None), dict(table=None)):
        assert call(**bad) == _lib.GQK_ERR_ARG, bad
    for bad in (dict(tokens=-1), dict(tokens=(1 << 20) + 1), dict(batch=-1), dict(batch=65536), dict(heads=7), dict(heads=0), dict(heads=2050),
                dict(most=65), dict(most=-1), dict(most_tokens=-1), dict(window=-1), dict(words=0), dict(q_row=513), dict(q=ctypes.c_void_p(4098)),
                dict(pages=_c_pages(dim=60)), dict(pages=_c_pages(k_token=100)), dict(pages=_c_pages(page_size=0)), dict(ws=ctypes.c_void_p(4096 + 16))):
        assert call(**bad) == _lib.GQK_ERR_SHAPE, bad
    need = lib.gqk_tree_attention_workspace_bytes
    assert need(12, 3, 7, 2, 64, 12, 64, 0) == need(-1, 3, 8, 2, 64, 12, 64, 0) == need(12, 3, 8, 2, 64, 12, -1, 0) == _lib.GQK_ERR_SHAPE
    assert need(0, 3, 8, 2, 64, 12, 64, 0) == 0 and need(12, 1, 8, 2, 64, 12, 1 << 20, 0) > _lib.GQK_CTR_BYTES


def test_c_sparse_refusals():
    def bounds(pages=None, table=P, width=4, lengths=P, batch=3, count=1, out=P):
        pages = _c_pages() if pages is None else pages
        return lib.gqk_page_bounds(ctypes.byref(pages) if pages else None, table, width, width, lengths, batch, count, out, None)

    assert bounds(batch=0) == bounds(count=0) == bounds(width=0) == 0
    for bad in (dict(pages=False), dict(pages=_c_pages(k=None)), dict(pages=_c_pages(dtype=0)), dict(table=None), dict(lengths=None), dict(out=None)):
        assert bounds(**bad) == _lib.GQK_ERR_ARG, bad
    for bad in (dict(pages=_c_pages(dim=60)), dict(pages=_c_pages(k_page=4)), dict(pages=_c_pages(k=4104)), dict(pages=_c_pages(heads=0)),
                dict(out=ctypes.c_void_p(4104)), dict(batch=-1), dict(batch=65536), dict(count=-1)):
        assert bounds(**bad) == _lib.GQK_ERR_SHAPE, bad

    def select(q=P, q_row=512, q_head=64, dtype=1, batch=3, heads=8, near=P, near_dtype=1, pages=9, hkv=2, dim=64, table=P, width=7, lengths=P,
               most=112, page=16, keep=4, sink=1, recent=1, out=P, kept=P, ws=P, ws_bytes=1 << 30):
        return lib.gqk_select_pages(q, q_row, q_head, dtype, batch, heads, near, near_dtype, pages, hkv, dim, table, width, width, lengths, most,
                                    page, keep, sink, recent, out, kept, ws, ws_bytes, None)

    assert select(batch=0) == 0
    for bad in (dict(dtype=0), dict(dtype=3), dict(near_dtype=0), dict(near_dtype=2), dict(q=None), dict(near=None), dict(table=None),
                dict(lengths=None), dict(out=None), dict(kept=None)):
        assert select(**bad) == _lib.GQK_ERR_ARG, bad
    for bad in (dict(batch=-1), dict(heads=7), dict(hkv=0), dict(dim=60), dict(dim=264), dict(pages=0), dict(page=0), dict(most=113), dict(most=-1),
                dict(keep=0), dict(sink=-1), dict(recent=0), dict(sink=4), dict(q_row=513), dict(q=ctypes.c_void_p(4104)),
                dict(near=ctypes.c_void_p(4104)), dict(ws=None), dict(ws_bytes=_lib.GQK_CTR_BYTES + 100), dict(ws=ctypes.c_void_p(4096 + 16))):
        assert select(**bad) == _lib.GQK_ERR_SHAPE, bad
    need = lib.gqk_select_pages_workspace_bytes
    assert need(3, 2, 16, 113) == _lib.GQK_CTR_BYTES + 3 * 2 * 8 * 8
    assert need(-1, 2, 16, 112) == need(3, 0, 16, 112) == need(3, 2, 0, 112) == need(3, 2, 16, -1) == _lib.GQK_ERR_SHAPE


def test_gradients_are_refused_and_not_dropped():
    """A result of tensors that require gradients requires them too, and not through a gradient of its own."""
    with FakeTensorMode():
        for call, args, marked in ((gguf_hip.add_rms_norm, _norm_args(), {"x": (0, 1), "residual": (0, 1), "weight": (0,)}),
                                   (gguf_hip.add_rms_norm_fp8, _norm_args(), {"x": (0, 1, 2), "residual": (0, 1, 2), "weight": (0, 1)}),
                                   (gguf_hip.tree_attention, _tree_args(return_lse=True), {"q": (0, 1), "k_pages": (0, 1), "v_pages": (0, 1)})):
            for name, which in marked.items():
                kw = {**args, name: args[name].detach().clone().requires_grad_()}
                got = call(**kw)
                assert [t.requires_grad for t in got] == [i in which for i in range(len(got))], (call, name)
                for i in which:
                    assert "NoBackward" in got[i].grad_fn.name()
                with torch.no_grad():
                    assert not any(t.requires_grad for t in call(**kw))
            assert not any(t.requires_grad for t in call(**args))


def test_make_fx_traces_the_ops():
    """A traced step holds each operator as one opaque call, and no view or copy of the caches."""
    from torch.fx.experimental.proxy_tensor import make_fx

    def step(lists, requests, old, counts, parents, x, residual, weight, q, k_pages, v_pages, bounds):
        t = gguf_hip.step_tables(lists, requests, old, counts, 12, 16, parents=parents, tree=8)
        h, residual = gguf_hip.add_rms_norm(x, residual, weight)
        h8, scale, residual = gguf_hip.add_rms_norm_fp8(h, residual, weight, group=32)
        o = gguf_hip.tree_attention(q, k_pages, v_pages, t.block_table, t.lengths, t.starts, t.mask)
        gguf_hip.page_bounds(k_pages, t.block_table, t.lengths, bounds, count=8)
        table, kept = gguf_hip.select_pages(o[:3], bounds, t.block_table, t.lengths, 4, 16)
        return h8, scale, residual, gguf_hip.paged_attention(o[:3], k_pages, v_pages, table, kept)

    with FakeTensorMode():
        g = make_fx(step)(_i32(6, 9), _i32(3), _i32(3), _i32(3), _i32(12), _fake((12, 64)), _fake((12, 64)), _fake((64,)), _fake((12, 8, 64)),
                          _fake((9, 16, 2, 64)), _fake((9, 16, 2, 64)), _fake((9, 2, 2, 64)))
    ops = torch.ops.gguf_hip
    calls = [n.target for n in g.graph.nodes if n.op == "call_function"]
    ours = [c for c in calls if str(c).startswith("gguf_hip")]
    assert ours == [ops.step_tables.default, ops.add_rms_norm.default, ops.add_rms_norm.default, ops.tree_attention.default,
                    ops.page_bounds.default, ops.select_pages.default, ops.paged_attention.default], calls
    assert all(c in ours or "empty" in str(c) or "slice" in str(c) for c in calls), calls
