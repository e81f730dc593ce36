"""Attention around the linear path: the heads that qkv's output holds, normalized, rotated and stored into
the pages of a key-value cache (``qk_norm_rope``), and the attention of each new token over those pages
(``paged_attention``).  Both run on the current stream (one launch; a second where a
sequence's keys are cut into more than 16 splits, or heads that share one of keys are many), allocate their outputs alone, do not synchronise the host
and can be captured in a HIP graph; under tracing they are custom ops with fakes.

Layouts: heads are [tokens, heads, dim] views with any strides (column ranges of qkv's output as they are);
pages are [pages, page_size, heads, dim] with any strides, so a cache may keep a token's heads or a head's tokens
together (the latter reads faster: a head's page is then one run of memory)."""
from __future__ import annotations

import math

import torch

from . import _lib, ops
from ._lib import GqkHeads, GqkPages, _fast, check, lib
from .eager import direct as _direct, no_backward, stream as _stream, unwatched as _unwatched

_TYPES = {torch.bfloat16: _lib.GQK_DTYPE_BF16, torch.float16: _lib.GQK_DTYPE_F16}
_PAGE_TYPES = {**_TYPES, torch.float8_e4m3fn: _lib.GQK_DTYPE_FP8}


def _strides(t: torch.Tensor) -> tuple[int, int]:
    """The token and head strides of [tokens, heads, dim] (0 where there is one alone: its stride means nothing)."""
    s = t.stride()
    return (s[0] if t.shape[0] > 1 else 0), (s[1] if t.shape[1] > 1 else 0)


def _readable(t: torch.Tensor) -> bool:
    row, head = _strides(t)
    return t.stride(2) == 1 and not (row | head) & 7 and ops._addr_aligned(t, 16)


def _heads_view(t: torch.Tensor, what: str) -> torch.Tensor:
    """t as the kernels read heads: dims side by side, strides multiples of 8, 16-byte aligned (copied if not)."""
    if t.dim() != 3:
        raise ValueError(f"{what}: expected [tokens, heads, dim], got {tuple(t.shape)}")
    return t if t.numel() == 0 or _readable(t) else t.clone(memory_format=torch.contiguous_format)


def _out_heads(t: torch.Tensor, like: torch.Tensor, what: str) -> None:
    if t.shape != like.shape or t.dtype != like.dtype or t.device != like.device or (t.numel() and not _readable(t)):
        raise ValueError(f"{what}: an output is {like.dtype} {tuple(like.shape)} on {like.device}, its dims side by side, "
                         f"strides multiples of 8, 16-byte aligned; got {t.dtype} {tuple(t.shape)} {t.stride()} on {t.device}")


def _check_pages(k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None, v_scale: torch.Tensor | None,
                 like: torch.Tensor, what: str) -> None:
    if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in _PAGE_TYPES:
        raise ValueError(f"{what}: pages are [pages, page_size, heads, dim] of one type, got {k.dtype} {tuple(k.shape)} and "
                         f"{v.dtype} {tuple(v.shape)}")
    if k.dtype != like.dtype and k.dtype != torch.float8_e4m3fn:
        raise ValueError(f"{what}: {k.dtype} pages with {like.dtype} heads")
    if k.device != like.device or v.device != like.device:
        raise ValueError(f"{what}: pages on {k.device} and {v.device}, heads on {like.device}")
    if k.shape[3] != like.shape[2]:
        raise ValueError(f"{what}: heads of {like.shape[2]} dims, pages of {k.shape[3]}")
    if k.stride(3) != 1 or v.stride(3) != 1:
        raise ValueError(f"{what}: a page's dims must lie side by side")
    for s in (k_scale, v_scale):
        if s is not None and (s.dtype != torch.float32 or s.shape != (k.shape[2],) or s.device != like.device
                              or not s.is_contiguous()):
            raise ValueError(f"{what}: a scale is contiguous fp32 [{k.shape[2]}] on {like.device}")


def _c_pages(k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None, v_scale: torch.Tensor | None) -> GqkPages:
    n, page, heads, dim = k.shape
    ks, vs = ([0 if m == 1 else st for m, st in zip(k.shape, x.stride())] for x in (k, v))
    return GqkPages(k.data_ptr(), v.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
                    None if k_scale is None else k_scale.data_ptr(), None if v_scale is None else v_scale.data_ptr(),
                    _PAGE_TYPES[k.dtype], n, page, heads, dim)


def _c_heads(t: torch.Tensor | None):
    if t is None:
        return None
    return GqkHeads(t.data_ptr(), *_strides(t), t.shape[1])


def _index(t: torch.Tensor, n: int, device: torch.device, what: str) -> None:
    if t.dtype not in (torch.int32, torch.int64) or t.shape != (n,) or t.device != device or not t.is_contiguous():
        raise ValueError(f"{what}: expected contiguous int32 or int64 [{n}] on {device}, got {t.dtype} {tuple(t.shape)} on "
                         f"{t.device}")


# ---- attention -------------------------------------------------------------------------------

def _attention_into(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                    lengths: torch.Tensor, scale: float, window: int, k_scale: torch.Tensor | None,
                    v_scale: torch.Tensor | None, max_length: int, out: torch.Tensor, lse: torch.Tensor | None,
                    workspace: torch.Tensor | None) -> None:
    batch, heads, dim = q.shape
    if batch == 0:
        return
    device = q.device
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _attention_into(q, k_pages, v_pages, block_table, lengths, scale, window, k_scale, v_scale, max_length,
                                   out, lse, workspace)
    ws = ops.shared_workspace(device) if workspace is None else workspace
    qs, os = _strides(q), _strides(out)
    check(lib.gqk_paged_attention(q.data_ptr(), qs[0], qs[1], _TYPES[q.dtype], batch, heads,
                                  _lib.byref(_c_pages(k_pages, v_pages, k_scale, v_scale)), block_table.data_ptr(),
                                  block_table.stride(0), block_table.shape[1], lengths.data_ptr(), max_length, window, scale,
                                  out.data_ptr(), os[0], os[1], None if lse is None else lse.data_ptr(), ws.data_ptr(),
                                  ws.numel() * ws.element_size(), _stream(device)), "paged_attention")


@torch.library.custom_op("gguf_hip::paged_attention", mutates_args=("out", "lse", "workspace"))
def _attention_op(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                  lengths: torch.Tensor, scale: float, window: int, k_scale: torch.Tensor | None,
                  v_scale: torch.Tensor | None, max_length: int, out: torch.Tensor, lse: torch.Tensor | None,
                  workspace: torch.Tensor | None) -> None:
    _attention_into(q, k_pages, v_pages, block_table, lengths, scale, window, k_scale, v_scale, max_length, out, lse, workspace)


@_attention_op.register_fake
def _(q, k_pages, v_pages, block_table, lengths, scale, window, k_scale, v_scale, max_length, out, lse, workspace):
    return None


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                    lengths: torch.Tensor, *, scale: float | None = None, window: int = 0,
                    k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                    max_length: int | None = None, out: torch.Tensor | None = None, return_lse: bool = False,
                    workspace: torch.Tensor | None = None):
    """Attention of one new token per sequence over its pages: q [batch, query heads, dim] (bf16 or fp16), pages
    [pages, page_size, heads, dim] of q's type or float8_e4m3fn (times ``k_scale`` / ``v_scale`` fp32 [heads]), query
    heads a multiple of the pages' heads, dim a multiple of 8 up to 256.  Key j of sequence b lies in page
    block_table[b, j // page_size] (int32); lengths int32 [batch] counts the keys, the new token's among them;
    ``window`` > 0 keeps the last ``window`` of them.  A sequence without a key gets zeros.  ``scale``: dim ** -0.5
    by default.  ``max_length``: an upper bound on lengths known to the host (default: what the table holds); the work
    is split by it, so a tight one is faster.  A sequence above it, or with a page outside of the cache, gets NaN.
    Returns out [batch, query heads, dim], with ``return_lse`` also the log-sum-exp of its scores (fp32 [batch,
    query heads], -inf without a key), which joins attention over separate caches.  ``workspace``: as
    mul_mat_grouped's (its own for calls on concurrent streams).  No backward pass."""
    if _fast is not None and _unwatched():
        got = _fast.paged_attention(q, k_pages, v_pages, block_table, lengths, scale, window, k_scale, v_scale, max_length, out,
                                    return_lse, workspace)
        if got is not None:
            return got
    ops._require_gpu(q, "paged_attention")
    if q.dtype not in _TYPES:
        raise ValueError(f"paged_attention: q is bf16 or fp16, not {q.dtype}")
    q = _heads_view(q, "paged_attention")
    _check_pages(k_pages, v_pages, k_scale, v_scale, q, "paged_attention")
    batch, heads, dim = q.shape
    if heads == 0 or heads % k_pages.shape[2]:
        raise ValueError(f"paged_attention: {heads} query heads over {k_pages.shape[2]}")
    if (block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != batch
            or block_table.device != q.device or (block_table.shape[1] > 1 and block_table.stride(1) != 1)):
        raise ValueError(f"paged_attention: block_table is int32 [{batch}, pages] on {q.device}, its columns side by side")
    if (lengths.dtype != torch.int32 or lengths.shape != (batch,) or lengths.device != q.device
            or not lengths.is_contiguous()):
        raise ValueError(f"paged_attention: lengths is contiguous int32 [{batch}] on {q.device}")
    ops.check_workspace(workspace, q.device, "paged_attention")
    room = min(block_table.shape[1] * k_pages.shape[1], _lib.GQK_MAX_KEYS)
    max_length = room if max_length is None else int(max_length)
    if not 0 <= max_length <= room or window < 0:
        raise ValueError(f"paged_attention: max_length {max_length} (the table holds {room} keys), window {window}")
    if out is None:
        out = torch.empty((batch, heads, dim), dtype=q.dtype, device=q.device)
    else:
        _out_heads(out, q, "paged_attention")
    lse = torch.empty((batch, heads), dtype=torch.float32, device=q.device) if return_lse else None
    args = (q, k_pages, v_pages, block_table, lengths, dim ** -0.5 if scale is None else float(scale), int(window), k_scale,
            v_scale, max_length, out, lse, workspace)
    if _direct(q, k_pages, v_pages, block_table, lengths, k_scale, v_scale, out, workspace):
        _attention_into(*args)
        torch.autograd.graph.increment_version(out)
    else:
        _attention_op(*args)
    for t in (out, lse):
        no_backward("paged_attention", t, q, k_pages, v_pages, k_scale, v_scale)
    return (out, lse) if return_lse else out


# ---- norm, rotation, store -------------------------------------------------------------------

def rope_table(rot: int, length: int, base: float = 10000.0, scaling: dict | None = None,
               device: torch.device | str = "cuda") -> torch.Tensor:
    """The rotation's table for positions 0 .. length - 1: fp32 [length, rot], cos | sin of angle
    position * f_i, f_i = base ** (-2 i / rot), computed in 64 bits (a product in 32 bits is off by
    0.06 rad at a million tokens).  ``scaling`` lengthens the context:

    * {"type": "linear", "factor"}: f_i / factor;
    * {"type": "ntk", "factor"}: base * factor ** (rot / (rot - 2)), so that the slowest pair is slowed
      by factor and the fastest not at all;
    * {"type": "yarn", "factor", "original_length", "beta_fast": 32, "beta_slow": 1, "attention_factor":
      0.1 ln factor + 1}: pairs that turn more than beta_fast times over the original length keep f_i, those
      below beta_slow turns get f_i / factor, a linear ramp over i between; cos and sin times attention_factor;
    * {"type": "bands", "factor", "original_length", "low": 1, "high": 4}: the same idea with a ramp over the
      number of turns: above ``high`` f_i, below ``low`` f_i / factor, linear in the turns between."""
    if rot < 2 or rot % 2 or length < 0:
        raise ValueError(f"rope_table: {rot} rotated dims (even), {length} positions")
    i = torch.arange(0, rot, 2, dtype=torch.float64, device=device)
    scaling = dict(scaling or {"type": None})
    kind, factor, amp = scaling.pop("type", None), float(scaling.pop("factor", 1.0)), 1.0
    if factor <= 0:
        raise ValueError(f"rope_table: factor {factor}")
    if kind == "ntk":
        if rot < 4:
            raise ValueError("rope_table: ntk scaling needs two pairs")
        base = base * factor ** (rot / (rot - 2))
    freq = base ** (-i / rot)
    if kind == "linear":
        freq = freq / factor
    elif kind in ("yarn", "bands"):
        original = float(scaling.pop("original_length"))
        if kind == "yarn":
            fast, slow = float(scaling.pop("beta_fast", 32.0)), float(scaling.pop("beta_slow", 1.0))
            amp = float(scaling.pop("attention_factor", 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0))
            at = lambda turns: rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
            lo, hi = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), rot - 1)
            keep = 1 - ((i / 2 - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        else:
            low, high = float(scaling.pop("low", 1.0)), float(scaling.pop("high", 4.0))
            if high <= low:
                raise ValueError(f"rope_table: bands from {low} to {high} turns")
            keep = ((original * freq / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        freq = freq * keep + freq / factor * (1 - keep)
    elif kind not in (None, "ntk"):
        raise ValueError(f"rope_table: unknown scaling {kind!r}")
    if scaling:
        raise ValueError(f"rope_table: unknown scaling keys {sorted(scaling)}")
    angle = torch.arange(length, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cat([angle.cos() * amp, angle.sin() * amp], 1).float()


def _rope_into(q: torch.Tensor, k: torch.Tensor | None, v: torch.Tensor | None, positions: torch.Tensor,
               table: torch.Tensor, q_weight: torch.Tensor | None, k_weight: torch.Tensor | None, eps: float, flags: int,
               slots: torch.Tensor | None, k_scale: torch.Tensor | None, v_scale: torch.Tensor | None,
               out_q: torch.Tensor, out_k: torch.Tensor | None, k_pages: torch.Tensor | None,
               v_pages: torch.Tensor | None) -> None:
    tokens, _, dim = q.shape
    if tokens == 0:
        return
    device = q.device
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _rope_into(q, k, v, positions, table, q_weight, k_weight, eps, flags, slots, k_scale, v_scale, out_q, out_k,
                              k_pages, v_pages)
    weight = q_weight if q_weight is not None else k_weight
    dtype = _TYPES[q.dtype]
    check(lib.gqk_qk_norm_rope(_ref(_c_heads(q)), _ref(_c_heads(k)), _ref(_c_heads(v)), dtype, tokens, dim,
                               positions.data_ptr(), positions.dtype == torch.int64, table.data_ptr(), table.shape[0],
                               table.shape[1], None if q_weight is None else q_weight.data_ptr(),
                               None if k_weight is None else k_weight.data_ptr(),
                               dtype if weight is None or weight.dtype == q.dtype else _lib.GQK_DTYPE_F32, eps, flags,
                               _ref(_c_heads(out_q)), _ref(_c_heads(out_k)),
                               None if k_pages is None else _lib.byref(_c_pages(k_pages, v_pages, k_scale, v_scale)),
                               None if slots is None else slots.data_ptr(),
                               slots is not None and slots.dtype == torch.int64, _stream(device)), "qk_norm_rope")


def _ref(c):
    return None if c is None else _lib.byref(c)


@torch.library.custom_op("gguf_hip::qk_norm_rope", mutates_args=("out_q", "out_k", "k_pages", "v_pages"))
def _rope_op(q: torch.Tensor, k: torch.Tensor | None, v: torch.Tensor | None, positions: torch.Tensor, table: torch.Tensor,
             q_weight: torch.Tensor | None, k_weight: torch.Tensor | None, eps: float, flags: int,
             slots: torch.Tensor | None, k_scale: torch.Tensor | None, v_scale: torch.Tensor | None, out_q: torch.Tensor,
             out_k: torch.Tensor | None, k_pages: torch.Tensor | None, v_pages: torch.Tensor | None) -> None:
    _rope_into(q, k, v, positions, table, q_weight, k_weight, eps, flags, slots, k_scale, v_scale, out_q, out_k, k_pages, v_pages)


@_rope_op.register_fake
def _(q, k, v, positions, table, q_weight, k_weight, eps, flags, slots, k_scale, v_scale, out_q, out_k, k_pages, v_pages):
    return None


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, table: torch.Tensor,
                 q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, *, eps: float = 1e-6,
                 unit_offset: bool = False, interleaved: bool = False, v: torch.Tensor | None = None,
                 k_pages: torch.Tensor | None = None, v_pages: torch.Tensor | None = None,
                 slots: torch.Tensor | None = None, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None, out_q: torch.Tensor | None = None,
                 out_k: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """The heads of q [tokens, query heads, dim] and k [tokens, heads, dim] (bf16 or fp16, dim a multiple of 8 up to
    256), each normalized (RMS over the head, then its weight [dim], of the heads' type or fp32; ``unit_offset``: 1 +
    weight; None: no norm) and its first table.shape[1] dims rotated by the token's position (``table`` as rope_table
    makes it; pairs (i, i + rot / 2), or (2 i, 2 i + 1) with ``interleaved``).  With pages, token t's keys and its
    values v [tokens, heads, dim] are also stored at slots[t] = page * page_size + place (negative: not stored; the
    slots of one call must differ), in float8_e4m3fn pages divided by ``k_scale`` / ``v_scale`` (fp32 [heads]) and
    held to +-448.  positions and slots: int32 or int64 [tokens]; a position outside of the table gives NaN.
    Returns (queries, keys): new tensors, or out_q / out_k, which may be q and k themselves; with pages the keys are
    returned (and written beside the pages) only into an out_k that is given.  No backward pass, and what is stored in pages is
    cut from any graph."""
    what = "qk_norm_rope"
    flags = (_lib.GQK_ROPE_UNIT_OFFSET if unit_offset else 0) | (_lib.GQK_ROPE_INTERLEAVED if interleaved else 0)
    if _fast is not None and _unwatched():
        got = _fast.qk_norm_rope(q, k, positions, table, q_weight, k_weight, eps, flags, v, k_pages, v_pages, slots, k_scale,
                                 v_scale, out_q, out_k)
        if got is not None:
            return got
    ops._require_gpu(q, what)
    if q.dtype not in _TYPES:
        raise ValueError(f"{what}: heads are bf16 or fp16, not {q.dtype}")
    if q.dim() != 3 or q.shape[1] == 0:
        raise ValueError(f"{what}: expected [tokens, heads, dim], got {tuple(q.shape)}")
    tokens, _, dim = q.shape
    for t in (k, v):
        if t is not None and (t.dim() != 3 or t.shape[0] != tokens or t.shape[1] == 0 or t.shape[2] != dim
                              or t.dtype != q.dtype or t.device != q.device):
            raise ValueError(f"{what}: keys and values are {q.dtype} [{tokens}, heads, {dim}] on {q.device}, got {t.dtype} "
                             f"{tuple(t.shape)} on {t.device}")
    if k is None and k_weight is not None or k is None and out_k is not None:
        raise ValueError(f"{what}: a key weight or output without keys")
    for w in (q_weight, k_weight):
        if w is not None and (w.shape != (dim,) or w.dtype not in (q.dtype, torch.float32) or w.device != q.device
                              or not w.is_contiguous()):
            raise ValueError(f"{what}: weights are contiguous {q.dtype} or fp32 [{dim}] on {q.device}")
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise ValueError(f"{what}: weights of two types")
    _index(positions, tokens, q.device, what)
    if (table.dtype != torch.float32 or table.dim() != 2 or table.shape[1] % 2 or table.shape[1] > dim
            or table.device != q.device or not table.is_contiguous()):
        raise ValueError(f"{what}: table is contiguous fp32 [positions, rotated dims (even, at most {dim})] on {q.device}")
    if k_pages is not None:
        if v_pages is None or k is None or v is None or slots is None:
            raise ValueError(f"{what}: pages need keys, values and slots")
        _check_pages(k_pages, v_pages, k_scale, v_scale, k, what)
        if k.shape[1] != k_pages.shape[2] or v.shape[1] != k_pages.shape[2]:
            raise ValueError(f"{what}: {k.shape[1]} key and {v.shape[1]} value heads, pages of {k_pages.shape[2]}")
        _index(slots, tokens, q.device, what)
    elif v is not None or v_pages is not None or slots is not None or k_scale is not None or v_scale is not None:
        raise ValueError(f"{what}: values, slots and scales without pages")
    if out_q is None:
        out_q = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        _out_heads(out_q, q, what)
    if out_k is not None:
        _out_heads(out_k, k, what)
    elif k is not None and k_pages is None:
        out_k = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    args = (_heads_view(q, what), None if k is None else _heads_view(k, what), None if v is None else _heads_view(v, what),
            positions, table, q_weight, k_weight, float(eps), flags, slots, k_scale, v_scale, out_q, out_k, k_pages, v_pages)
    if _direct(q, k, v, positions, table, q_weight, k_weight, slots, k_scale, v_scale, out_q, out_k, k_pages, v_pages):
        _rope_into(*args)
        for t in (out_q, out_k, k_pages, v_pages):
            if t is not None:
                torch.autograd.graph.increment_version(t)
    else:
        _rope_op(*args)
    no_backward(what, out_q, q, q_weight, table)
    no_backward(what, out_k, k, k_weight, table)
    return out_q, out_k
