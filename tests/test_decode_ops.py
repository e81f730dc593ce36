"""CPU tests of what surrounds the linear path in a decode step: the page pool's bookkeeping, the rotation's table
against its formula, the refusals of every entry point (Python's and the C ABI's; nothing is launched), and the custom ops
under tracing."""
import ctypes
import math
import random

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import gguf_hip
from gguf_hip import _lib
from gguf_hip._lib import lib

BF, F16, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


# ---- the page pool ---------------------------------------------------------------------------

def test_pool_fork_own_free():
    pool = gguf_hip.PagePool(6)
    a = pool.allocate(3)
    assert a == [0, 1, 2] and pool.free_pages == 3
    b = pool.fork(a)
    assert pool.own(b, 2) == ([2], [3]) and b == [0, 1, 3] and a == [0, 1, 2]
    assert pool.own(b, 2) == ([], [])                       # its own already
    pool.free(a)
    assert pool.uses == [1, 1, 0, 1, 0, 0]                  # the shared pages stay with b
    with pytest.raises(ValueError):
        pool.free([2])
    with pytest.raises(ValueError):
        pool.fork([5])
    with pytest.raises(ValueError):
        pool.free([0, 0])
    assert pool.uses == [1, 1, 0, 1, 0, 0]
    with pytest.raises(MemoryError):
        pool.allocate(4)
    assert pool.free_pages == 3 and pool.allocate(0) == []


def test_pool_compacts_and_renumbers():
    """Random sequences of the pool's steps against a model that keeps every sequence's tokens by value."""
    rng = random.Random(7)
    pool, store = gguf_hip.PagePool(40), [None] * 40
    tables, values, fresh = [], [], iter(range(10 ** 6))
    for step in range(600):
        kind = rng.choice(("new", "fork", "write", "free", "compact"))
        if kind == "new" and pool.free_pages >= 4:
            t = pool.allocate(rng.randint(1, 4))
            vals = [next(fresh) for _ in t]
            for p, v in zip(t, vals):
                store[p] = v
            tables.append(t), values.append(vals)
        elif kind == "fork" and tables:
            i = rng.randrange(len(tables))
            tables.append(pool.fork(tables[i])), values.append(list(values[i]))
        elif kind == "write" and tables and pool.free_pages:
            i = rng.randrange(len(tables))
            j = rng.randrange(len(tables[i]))
            src, dst = pool.own(tables[i], j)
            for s, d in zip(src, dst):
                store[d] = store[s]
            store[tables[i][j]] = values[i][j] = next(fresh)
        elif kind == "free" and tables:
            i = rng.randrange(len(tables))
            pool.free(tables.pop(i)), values.pop(i)
        elif kind == "compact":
            src, dst = pool.compact(tables)
            assert not set(src) & set(dst) and len(set(dst)) == len(dst)
            old = list(store)
            for s, d in zip(src, dst):
                store[d] = old[s]
            live = sum(1 for u in pool.uses if u)
            assert all(pool.uses[:live]) and not any(pool.uses[live:])
        assert [[store[p] for p in t] for t in tables] == values
        assert pool.free_pages == sum(1 for u in pool.uses if u == 0)
    for t in tables:
        pool.free(t)
    assert pool.free_pages == 40 and pool.compact([]) == ([], [])
    pool.allocate(1)
    with pytest.raises(ValueError):
        pool.compact([])                                    # a live page that no table names


# ---- the rotation's table --------------------------------------------------------------------

def test_rope_table_formulas():
    rot, n, base = 64, 50, 5e5
    f = [base ** (-2 * i / rot) for i in range(rot // 2)]

    def rows(freq, amp=1.0):
        a = np.arange(n)[:, None] * np.array(freq)
        return np.concatenate([np.cos(a) * amp, np.sin(a) * amp], 1)

    def near(table, want):
        assert table.dtype == torch.float32 and table.shape == (n, rot)
        # one rounding to fp32, and the last bits of numpy's and torch's 64-bit functions
        assert np.abs(table.double().numpy() - want).max() <= 2 ** -24 * np.abs(want).max() * 1.01

    make = lambda **s: gguf_hip.rope_table(rot, n, base, s or None, device="cpu")  # noqa: E731
    near(make(), rows(f))
    near(make(type="linear", factor=4), rows([x / 4 for x in f]))
    near(make(type="ntk", factor=8), rows([(base * 8 ** (rot / (rot - 2))) ** (-2 * i / rot) for i in range(rot // 2)]))
    # the slowest pair of the ntk table is slowed by exactly the factor
    assert math.isclose((base * 8 ** (rot / (rot - 2))) ** (-(rot - 2) / rot), f[-1] / 8, rel_tol=1e-12)
    orig, factor = 4096, 16
    lo = math.floor(rot * math.log(orig / (32 * 2 * math.pi)) / (2 * math.log(base)))
    hi = math.ceil(rot * math.log(orig / (1 * 2 * math.pi)) / (2 * math.log(base)))
    keep = [1 - min(max((i - lo) / (hi - lo), 0), 1) for i in range(rot // 2)]
    assert 0 < lo < hi < rot // 2
    near(make(type="yarn", factor=factor, original_length=orig),
         rows([x * k + x / factor * (1 - k) for x, k in zip(f, keep)], 0.1 * math.log(factor) + 1))
    turns = [orig * x / (2 * math.pi) for x in f]
    keep = [min(max((t - 1) / 3, 0), 1) for t in turns]
    assert any(0 < k < 1 for k in keep)
    near(make(type="bands", factor=8, original_length=orig), rows([x * k + x / 8 * (1 - k) for x, k in zip(f, keep)]))
    for bad in ({"type": "other"}, {"type": "linear", "factor": 0}, {"type": "linear", "factor": 2, "extra": 1},
                {"type": "bands", "factor": 2, "original_length": 10, "low": 4, "high": 4}):
        with pytest.raises(ValueError):
            make(**bad)
    with pytest.raises(ValueError):
        gguf_hip.rope_table(63, 4, device="cpu")


# ---- refusals --------------------------------------------------------------------------------

def test_cpu_tensors_are_refused():
    z = torch.zeros
    with pytest.raises(ValueError, match="GPU"):
        gguf_hip.paged_attention(z(1, 8, 64, dtype=BF), z(4, 16, 2, 64, dtype=BF), z(4, 16, 2, 64, dtype=BF),
                                 z(1, 2, dtype=torch.int32), z(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="GPU"):
        gguf_hip.qk_norm_rope(z(1, 8, 64, dtype=BF), None, z(1, dtype=torch.int32), z(8, 64))
    with pytest.raises(ValueError, match="GPU"):
        gguf_hip.lora_add(z(1, 8, dtype=BF), z(1, 64, dtype=BF), z(1, 1, 8, 64, dtype=BF), z(1, 8, 8, dtype=BF),
                          z(1, dtype=torch.int32), None, [8])
    with pytest.raises(ValueError, match="GPU"):
        gguf_hip.copy_pages(z(4, 16), [0], [1])


def _fake(shape, dtype=BF):
    return torch.empty(shape, dtype=dtype, device="cuda")


def _attend_args(**over):
    a = dict(q=_fake((3, 8, 64)), k_pages=_fake((9, 16, 2, 64)), v_pages=_fake((9, 16, 2, 64)),
             block_table=_fake((3, 4), torch.int32), lengths=_fake((3,), torch.int32))
    a.update(over)
    return a


def test_paged_attention_shapes_and_refusals():
    with FakeTensorMode():
        assert gguf_hip.paged_attention(**_attend_args()).shape == (3, 8, 64)
        out, lse = gguf_hip.paged_attention(**_attend_args(), return_lse=True)
        assert out.dtype == BF and lse.shape == (3, 8) and lse.dtype == torch.float32
        f8 = _fake((9, 16, 2, 64), F8)
        assert gguf_hip.paged_attention(**_attend_args(k_pages=f8, v_pages=f8), k_scale=_fake((2,), torch.float32)).dtype == BF
        assert gguf_hip.paged_attention(**_attend_args(q=_fake((0, 8, 64)), block_table=_fake((0, 4), torch.int32),
                                                       lengths=_fake((0,), torch.int32))).shape == (0, 8, 64)
        for bad in (dict(q=_fake((3, 8, 64), torch.float32)), dict(q=_fake((3, 512))), dict(q=_fake((3, 7, 64))),
                    dict(q=_fake((3, 8, 64), F16)), dict(q=_fake((3, 8, 32))), dict(k_pages=_fake((9, 16, 2, 64), F16)),
                    dict(v_pages=_fake((9, 16, 2, 32))), dict(v_pages=_fake((9, 8, 2, 64))),
                    dict(block_table=_fake((3, 4), torch.int64)), dict(block_table=_fake((2, 4), torch.int32)),
                    dict(block_table=_fake((4, 3), torch.int32).t()), dict(lengths=_fake((3,), torch.int64)),
                    dict(lengths=_fake((4,), torch.int32)), dict(max_length=65), dict(max_length=-1), dict(window=-1),
                    dict(k_scale=_fake((3,), torch.float32)), dict(k_scale=_fake((2,), BF)),
                    dict(out=_fake((3, 8, 64), F16)), dict(out=_fake((3, 8, 32))), dict(out=_fake((3, 64, 8)).transpose(1, 2))):
            with pytest.raises(ValueError):
                gguf_hip.paged_attention(**_attend_args(**bad))


def _rope_args(**over):
    a = dict(q=_fake((5, 8, 64)), k=_fake((5, 2, 64)), positions=_fake((5,), torch.int64), table=_fake((100, 32), torch.float32),
             q_weight=_fake((64,)), k_weight=_fake((64,)))
    a.update(over)
    return a


def test_qk_norm_rope_shapes_and_refusals():
    with FakeTensorMode():
        q, k = gguf_hip.qk_norm_rope(**_rope_args())
        assert q.shape == (5, 8, 64) and k.shape == (5, 2, 64)
        q, k = gguf_hip.qk_norm_rope(**_rope_args(k=None, k_weight=None))
        assert q.shape == (5, 8, 64) and k is None
        pages = dict(v=_fake((5, 2, 64)), k_pages=_fake((4, 8, 2, 64)), v_pages=_fake((4, 8, 2, 64)),
                     slots=_fake((5,), torch.int32))
        q, k = gguf_hip.qk_norm_rope(**_rope_args(**pages))
        assert k is None                                     # stored only
        for bad in (dict(q=_fake((5, 8, 64), torch.float32)), dict(q=_fake((5, 512))), dict(k=_fake((4, 2, 64))),
                    dict(k=_fake((5, 2, 32))), dict(k=_fake((5, 2, 64), F16)), dict(k=None), dict(q_weight=_fake((32,))),
                    dict(q_weight=_fake((64,), torch.float32)), dict(positions=_fake((5,), torch.float32)),
                    dict(positions=_fake((4,), torch.int64)), dict(table=_fake((100, 66), torch.float32)),
                    dict(table=_fake((100, 31), torch.float32)), dict(table=_fake((100, 32))),
                    dict(out_q=_fake((5, 8, 32))), dict(out_k=_fake((5, 8, 64))), dict(slots=_fake((5,), torch.int32)),
                    {**pages, "slots": None}, {**pages, "v": None}, {**pages, "v_pages": None}, {**pages, "v": _fake((5, 1, 64))},
                    {**pages, "k_pages": _fake((4, 8, 4, 64)), "v_pages": _fake((4, 8, 4, 64))},
                    {**pages, "slots": _fake((6,), torch.int32)}, {**pages, "v_scale": _fake((1,), torch.float32)}):
            with pytest.raises(ValueError):
                gguf_hip.qk_norm_rope(**_rope_args(**bad))


def _lora_args(**over):
    a = dict(y=_fake((4, 48)), x=_fake((4, 64)), a=_fake((3, 2, 16, 64)), b=_fake((3, 48, 16)), ids=_fake((4,), torch.int32),
             scales=_fake((3,), torch.float32), n_outs=[32, 16])
    a.update(over)
    return a


def test_lora_add_shapes_and_refusals():
    with FakeTensorMode():
        assert gguf_hip.lora_add(**_lora_args()).shape == (4, 48)
        y = _fake((4, 48))
        assert gguf_hip.lora_add(**_lora_args(y=y), out=y) is y
        assert gguf_hip.lora_add(**_lora_args(scales=None, ids=_fake((4,), torch.int64))).dtype == BF
        for bad in (dict(x=_fake((4, 64), torch.float32)), dict(x=_fake((64,))), dict(y=_fake((4, 47))), dict(y=_fake((4, 48), F16)),
                    dict(a=_fake((3, 1, 16, 64))), dict(a=_fake((3, 2, 16, 72))), dict(b=_fake((3, 47, 16))),
                    dict(b=_fake((2, 48, 16))), dict(a=_fake((3, 2, 12, 64)), b=_fake((3, 48, 12))),
                    dict(a=_fake((3, 2, 264, 64)), b=_fake((3, 48, 264))), dict(a=_fake((3, 2, 64, 16)).transpose(2, 3)),
                    dict(a=_fake((3, 2, 16, 64), F16)), dict(ids=_fake((4,), torch.float32)), dict(ids=_fake((3,), torch.int32)),
                    dict(scales=_fake((3,))), dict(scales=_fake((2,), torch.float32)), dict(n_outs=[48]), dict(n_outs=[]),
                    dict(n_outs=[48, 0]), dict(n_outs=[6] * 8), dict(out=_fake((4, 49))), dict(out=_fake((48, 4)).t())):
            with pytest.raises(ValueError):
                gguf_hip.lora_add(**_lora_args(**bad))


def test_workspaces_that_are_refused():
    with FakeTensorMode():
        apart = _fake((1 << 20, 2), torch.int32)[:, 0]
        spread = _fake((1,), torch.int32).expand(1 << 24)
        for ws in (apart, spread, torch.empty(1 << 24, dtype=torch.int32)):
            with pytest.raises(ValueError, match="workspace"):
                gguf_hip.paged_attention(**_attend_args(), workspace=ws)
            with pytest.raises(ValueError, match="workspace"):
                gguf_hip.lora_add(**_lora_args(), workspace=ws)


def test_make_fx_traces_the_ops():
    """A traced decode step holds each operator as one opaque call, and no view or copy of the caches."""
    from torch.fx.experimental.proxy_tensor import make_fx

    def step(q, k, v, positions, table, k_pages, v_pages, slots, block_table, lengths, y, x, a, b, ids):
        q, _ = gguf_hip.qk_norm_rope(q, k, positions, table, v=v, k_pages=k_pages, v_pages=v_pages, slots=slots)
        o = gguf_hip.paged_attention(q, k_pages, v_pages, block_table, lengths)
        return o, gguf_hip.lora_add(y, x, a, b, ids, None, [32, 16]), gguf_hip.lora_add(y, x, a, b, ids, None, [32, 16], out=y)

    with FakeTensorMode():
        heads, pages, i32 = _fake((3, 2, 64)), _fake((9, 16, 2, 64)), _fake((3,), torch.int32)
        lo = _lora_args()
        g = make_fx(step)(_fake((3, 8, 64)), heads, _fake((3, 2, 64)), i32, _fake((100, 64), torch.float32), pages,
                          _fake((9, 16, 2, 64)), _fake((3,), torch.int32), _fake((3, 4), torch.int32), _fake((3,), torch.int32),
                          lo["y"], lo["x"], lo["a"], lo["b"], lo["ids"])
    ops = torch.ops.gguf_hip
    calls = [n.target for n in g.graph.nodes if n.op == "call_function"]
    ours = [c for c in calls if str(c).startswith("gguf_hip")]
    assert ours == [ops.qk_norm_rope.default, ops.paged_attention.default, ops.lora_add.default, ops.lora_add_.default], calls
    assert all(c in ours or "empty" in str(c) for c in calls), calls


def test_pack_adapters():
    g = torch.Generator().manual_seed(1)
    A, B = torch.randn(5, 32, generator=g), torch.randn(12, 5, generator=g)
    a, b, s = gguf_hip.pack_adapters([None, ([A, None], [B, None], 0.5)], [12, 4], 32, dtype=torch.float32, device="cpu")
    assert a.shape == (2, 2, 8, 32) and b.shape == (2, 16, 8) and s.tolist() == [0.0, 0.5]
    assert torch.equal(a[1, 0, :5], A) and not a[1, 0, 5:].any() and not a[1, 1].any() and not a[0].any()
    assert torch.equal(b[1, :12, :5], B) and not b[1, 12:].any() and not b[1, :, 5:].any()
    for bad in (dict(rank=4), dict(rank=12), dict(rank=512)):
        with pytest.raises(ValueError):
            gguf_hip.pack_adapters([([A, None], [B, None], 1.0)], [12, 4], 32, device="cpu", **bad)
    for ad in (([A], [B], 1.0), ([A, A], [B, None], 1.0), ([A[:, :8], None], [B, None], 1.0), ([A, None], [B[:4], None], 1.0)):
        with pytest.raises(ValueError):
            gguf_hip.pack_adapters([ad], [12, 4], 32, device="cpu")


P = ctypes.c_void_p(4096)   # never dereferenced: the checks come first


def _c_pages(**over):
    f = dict(k=4096, v=4096, k_page=2048, k_token=128, k_head=64, v_page=2048, v_token=128, v_head=64, k_scale=None,
             v_scale=None, dtype=1, pages=9, page_size=16, heads=2, dim=64)
    f.update(over)
    return _lib.GqkPages(*f.values())


def _c_attend(pages=None, q=P, q_row=512, q_head=64, dtype=1, batch=3, heads=8, table=P, width=4, lengths=P, most=64, window=0,
              out=P, lse=None, ws=P, ws_bytes=1 << 40):
    pages = _c_pages() if pages is None else pages
    return lib.gqk_paged_attention(q, q_row, q_head, dtype, batch, heads, ctypes.byref(pages) if pages else None, table, width,
                                   width, lengths, most, window, 0.1, out, 512, 64, lse, ws, ws_bytes, None)


def test_c_attention_refusals():
    assert _c_attend(batch=0) == 0
    for bad in (dict(dtype=0), dict(dtype=3), dict(dtype=2), dict(pages=_c_pages(dtype=0)), dict(pages=_c_pages(k=None)),
                dict(q=None), dict(out=None), dict(lengths=None), dict(table=None)):
        assert _c_attend(**bad) == _lib.GQK_ERR_ARG, bad
    for bad in (dict(batch=-1), dict(heads=7), dict(heads=0), dict(most=65), dict(most=-1), dict(window=-1), dict(q_row=513),
                dict(q=ctypes.c_void_p(4098)), dict(pages=_c_pages(dim=60)), dict(pages=_c_pages(dim=264)),
                dict(pages=_c_pages(k_token=100)), dict(pages=_c_pages(k_page=-8)), dict(pages=_c_pages(v=4100)),
                dict(pages=_c_pages(page_size=0)), dict(pages=_c_pages(heads=0)), dict(pages=_c_pages(k_scale=4098))):
        assert _c_attend(**bad) == _lib.GQK_ERR_SHAPE, bad
    assert lib.gqk_paged_attention_workspace_bytes(3, 7, 2, 64, 64, 0) == _lib.GQK_ERR_SHAPE
    assert lib.gqk_paged_attention_workspace_bytes(1, 8, 2, 64, -1, 0) == _lib.GQK_ERR_SHAPE


def test_c_rope_refusals():
    H = lambda heads, data=4096, row=512, head=64: _lib.GqkHeads(data, row, head, heads)  # noqa: E731

    def call(q=H(8), k=H(2), v=None, dtype=1, tokens=5, dim=64, positions=P, table=P, rows=100, rot=64, qw=P, kw=P, wt=1,
             out_q=H(8), out_k=H(2), pages=None, slots=None):
        r = lambda x: None if x is None else ctypes.byref(x)  # noqa: E731
        return lib.gqk_qk_norm_rope(r(q), r(k), r(v), dtype, tokens, dim, positions, 1, table, rows, rot, qw, kw, wt, 1e-6, 0,
                                    r(out_q), r(out_k), r(pages), slots, 1, None)

    assert call(tokens=0) == 0
    for bad in (dict(dtype=0), dict(q=None), dict(out_q=None), dict(wt=2), dict(positions=None), dict(table=None),
                dict(out_k=None), dict(v=H(2)), dict(slots=P), dict(q=H(8, None)), dict(q=H(0), out_q=H(0))):
        assert call(**bad) == _lib.GQK_ERR_ARG, bad
    stored = dict(v=H(2), pages=_c_pages(), slots=P)
    for bad in (dict(dim=60), dict(dim=264), dict(rot=66), dict(rot=63), dict(tokens=-1), dict(rows=-1), dict(out_q=H(4)),
                dict(out_k=H(4)), dict(q=H(8, 4098)), dict(k=H(2, 4096, 511)), dict(table=ctypes.c_void_p(4098)),
                {**stored, "v": None}, {**stored, "slots": None}, {**stored, "v": H(4)}, {**stored, "pages": _c_pages(heads=4)},
                {**stored, "pages": _c_pages(dim=32)}):
        assert call(**bad) == _lib.GQK_ERR_SHAPE, bad


def test_c_lora_refusals():
    def call(y=P, y_row=48, x=P, x_row=64, M=4, K=64, a=P, b=P, slots=3, n=(32, 16), rank=16, ids=P, dtype=1, out=P, out_row=48,
             ws=P, ws_bytes=1 << 40):
        outs = None if n is None else (ctypes.c_int64 * len(n))(*n)
        return lib.gqk_lora_add(y, y_row, x, x_row, M, K, a, b, slots, 2 if n is None else len(n), outs, rank, ids, 0, None, dtype,
                                out, out_row, ws, ws_bytes, None)

    assert call(M=0) == 0
    for bad in (dict(dtype=0), dict(dtype=3), dict(y=None), dict(x=None), dict(a=None), dict(b=None), dict(ids=None), dict(out=None)):
        assert call(**bad) == _lib.GQK_ERR_ARG, bad
    for bad in (dict(M=-1), dict(K=60), dict(K=-8), dict(n=()), dict(n=(1,) * 9), dict(n=(32, 0)), dict(n=None), dict(rank=4),
                dict(rank=12), dict(rank=264), dict(slots=-1), dict(y_row=47), dict(out_row=47), dict(x_row=56), dict(x_row=68),
                dict(x=ctypes.c_void_p(4104)), dict(a=ctypes.c_void_p(4104)), dict(ws=None), dict(ws_bytes=1 << 18),
                dict(ws=ctypes.c_void_p(4096 + 16)), dict(n=(1 << 30, 1 << 30))):
        assert call(**bad) == _lib.GQK_ERR_SHAPE, bad
    assert lib.gqk_lora_workspace_bytes(4, 64, 2, 16) > _lib.GQK_CTR_BYTES
    assert "rank" in (lib.gqk_lora_workspace_bytes(4, 64, 2, 9), lib.gqk_last_error().decode())[1]


def test_c_copy_refusals():
    def call(src, dst, base=P, planes=2, plane=4096, pages=8, page=512, size=512):
        n = len(src)
        return lib.gqk_copy_pages(base, planes, plane, pages, page, size, (ctypes.c_int32 * max(n, 1))(*src),
                                  (ctypes.c_int32 * max(n, 1))(*dst), n, None)

    assert call([], []) == 0 and call([0], [1], planes=0) == 0 and call([0], [1], size=0) == 0
    for src, dst in (([0], [8]), ([8], [0]), ([-1], [0]), ([0], [-1])):
        assert call(src, dst) == _lib.GQK_ERR_SHAPE
    for src, dst in (([0, 1], [2, 2]), ([0], [0]), ([0, 1], [1, 2]), ([1, 0], [2, 1])):
        assert call(src, dst) == _lib.GQK_ERR_ARG
    assert call([0], [1], size=513) == _lib.GQK_ERR_SHAPE and call([0], [1], planes=-1) == _lib.GQK_ERR_SHAPE
    assert call([0], [1], base=None) == _lib.GQK_ERR_ARG
    assert lib.gqk_copy_pages(P, 1, 0, 4, 8, 8, None, None, 1, None) == _lib.GQK_ERR_ARG
    assert lib.gqk_copy_pages(P, 1, 0, 4, 8, 8, None, None, -1, None) == _lib.GQK_ERR_SHAPE
