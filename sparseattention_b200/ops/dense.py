"""Dense attention: queries of one sequence over the rows of another, and one new token over a paged cache.

`cross_attention` is the operator behind `HierarchicalAttention.forward` when it is given no parents or when the lengths of
query and key differ (hierarchical_attention/modules/attention.py:237-270 of the reference, which builds the
[B, H, Lq, Lk] weight matrix); `paged_attention_decode` is the dense counterpart of `span_attention_decode` for serving.
Softmax statistics and sums are float32; the backward is deterministic (one writer per gradient row).
"""
from __future__ import annotations

import ctypes
import functools
import math
from ctypes import c_void_p
from typing import NamedTuple, Optional, Tuple

import torch
from torch._compile import _disable_dynamo
from torch.autograd import forward_ad

from .. import _lib


# The kernels write through raw pointers: of a call, a tracer or a transform would see the allocation of the result and nothing that
# fills it, and a forward-mode tangent would end there.
_INFRA_MODES = (torch._C._TorchDispatchModeKey.PROXY, torch._C._TorchDispatchModeKey.FAKE, torch._C._TorchDispatchModeKey.FUNCTIONAL)
_modes, _tracing, _transform = torch._C._len_torch_dispatch_stack, torch._C._is_tracing, torch._C._functorch.peek_interpreter_stack


def transforms_active() -> bool:
    """Whether torch is tracing, compiling, transforming or watching operations, or computes forward-mode derivatives."""
    return torch.compiler.is_compiling() or _modes() > 0 or _tracing() or forward_ad._current_level >= 0 or _transform() is not None


def _refuse_transforms(who: str, *tensors: Optional[torch.Tensor]) -> None:
    if not (_modes() > 0 or _tracing() or forward_ad._current_level >= 0 or _transform() is not None):
        return
    if _tracing() or any(torch._C._get_dispatch_mode(m) is not None for m in _INFRA_MODES):
        raise _lib.HsaError(f"{who} cannot be traced: the graph would hold the allocation of its result and not the kernel")
    for t in tensors:
        if t is None:
            continue
        if torch._C._functorch.is_functorch_wrapped_tensor(t) or torch._is_functional_tensor(t):
            raise _lib.HsaError(f"{who} has no rule for torch.func transforms")
        if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
            raise _lib.HsaError(f"{who} has no forward-mode derivative; its inputs must not carry tangents")


@_disable_dynamo
def _outside_the_graph(op, *args):
    return op(*args)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """`t` [B, rows, heads, D] itself when its rows are packed, separate and aligned for vector loads, else a copy."""
    B, rows, heads, D = t.shape
    vec = 16 // t.element_size()
    if t.is_contiguous():
        ok = t.data_ptr() % 16 == 0 or D % vec != 0
    else:
        bs, rs = t.stride()[:2]
        ok = _lib.inner_contiguous(t) and (rows == 1 or rs >= heads * D) and (B == 1 or bs >= (rows - 1) * rs + heads * D)
        if ok and D % vec == 0:
            ok = t.data_ptr() % 16 == 0 and (rows == 1 or rs % vec == 0) and (B == 1 or bs % vec == 0)
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _view(t: torch.Tensor) -> _lib.HsaView:
    strides = t.stride()
    return _lib.HsaView(t.data_ptr(), strides[0], strides[1])


class _Packed(NamedTuple):
    """A mask in the bit form of hsa_dense_mask_pack: the bytes, and how many batches, heads and rows it tells apart."""
    data: torch.Tensor
    sizes: Tuple[int, int, int]


def _mask_bytes(mask: torch.Tensor, B: int, H: int, Lq: int, Lk: int, dev: torch.device) -> torch.Tensor:
    """The checked mask as a [B or 1, H or 1, Lq or 1, Lk or 1] tensor of bytes, nonzero = attend."""
    if mask.dtype.is_floating_point or mask.dtype.is_complex:
        raise _lib.HsaError(f"the mask is boolean or integer (nonzero = attend), not {mask.dtype}; additive masks are not taken")
    if mask.device != dev:
        raise _lib.HsaError("all tensors of one call must live on the same device")
    assert mask.dim() in (2, 4), "the mask is [Lq, Lk] or [B, H, Lq, Lk] (dimensions of size 1 are broadcast)"
    if mask.dim() == 2:
        mask = mask.unsqueeze(0).unsqueeze(0)
    assert all(m in (1, w) for m, w in zip(mask.shape, (B, H, Lq, Lk))), \
        f"mask shape {tuple(mask.shape)} does not broadcast to {(B, H, Lq, Lk)}"
    if mask.element_size() > 1:
        mask = mask != 0
    return mask.view(torch.uint8)


def _pack_mask(mask: torch.Tensor, dev: torch.device, Lk: int) -> _Packed:
    lib = _lib.load()
    shape, strides = mask.shape, mask.stride()
    sizes = tuple(1 if st == 0 else sz for sz, st in zip(shape[:3], strides[:3]))       # an expanded dimension is packed once
    strides = [0 if sz == 1 else st for sz, st in zip(shape, strides)]
    nbytes = lib.hsa_dense_mask_bytes(*sizes, Lk)
    data = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    rc = lib.hsa_dense_mask_pack(c_void_p(mask.data_ptr()), *strides, *sizes, Lk, c_void_p(data.data_ptr()), nbytes, _lib.stream_ptr(dev))
    _lib.check(rc, "hsa_dense_mask_pack")
    return _Packed(data, sizes)


def _mask_args(packed: Optional[_Packed]):
    return (None, 0, 0, 0) if packed is None else (c_void_p(packed.data.data_ptr()), *packed.sizes)


def _check_inputs(q, k, v):
    dev = _lib.require_cuda(q, k, v)
    _lib.dtype_code(q)
    assert q.dim() == 4 and k.dim() == 4 and v.dim() == 4, "q is [B, Lq, H, D]; k and v are [B, Lk, Hkv, D]"
    B, _, H, D = q.shape
    Bk, _, Hkv, Dk = k.shape
    assert k.shape == v.shape and Bk == B and Dk == D, \
        f"shapes disagree: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}"
    assert k.dtype == q.dtype and v.dtype == q.dtype, "dtype mismatch"
    assert Hkv >= 1 and H >= 1 and H % Hkv == 0, f"{H} query heads are not a multiple of {Hkv} key/value heads"
    assert 1 <= D <= 256, f"head dim {D} outside 1..256"
    return dev


@functools.lru_cache(maxsize=1024)
def _fwd_workspace(*sizes) -> int:
    return int(_lib.load().hsa_dense_attn_fwd_workspace_bytes(*sizes[:-1]))          # the last one is the device


@functools.lru_cache(maxsize=1024)
def _bwd_workspace(*sizes) -> int:
    return int(_lib.load().hsa_dense_attn_bwd_workspace_bytes(*sizes[:-1]))


@functools.lru_cache(maxsize=1024)
def _paged_plan(B, H, Hkv, D, page_size, max_pages, splits, device):
    lib = _lib.load()
    if splits is None:
        splits = lib.hsa_paged_attn_choose_splits(B, H, Hkv, page_size, max_pages)
    return splits, int(lib.hsa_paged_attn_workspace_bytes(B, H, D, splits))


def _lengths32(lengths, B: int, top: int, dev, name: str):
    if lengths.dtype not in (torch.int32, torch.int64):
        raise _lib.HsaError(f"{name} must be int32 or int64")
    if lengths.device != dev:
        raise _lib.HsaError("all tensors of one call must live on the same device")
    assert lengths.shape == (B,), f"{name} must have shape ({B},)"
    if lengths.dtype == torch.int64:
        lengths = lengths.clamp(-1, top + 1).to(torch.int32)
    return lengths if lengths.is_contiguous() else lengths.contiguous()


def dense_aborts() -> int:
    """Thread blocks of the tensor-core kernels that gave up a bounded wait (0 in a healthy run); synchronises."""
    count = ctypes.c_uint(0)
    _lib.check(_lib.load().hsa_dense_attn_aborts(ctypes.byref(count)), "hsa_dense_attn_aborts")
    return int(count.value)


_aborts_seen = {}


def _debug_check(what: str) -> None:
    """With HSA_B200_DEBUG=1: synchronise and raise if a thread block of the call gave up waiting."""
    if torch.cuda.is_current_stream_capturing():
        return
    dev, now = torch.cuda.current_device(), dense_aborts()
    if now != _aborts_seen.get(dev, 0):
        before, _aborts_seen[dev] = _aborts_seen.get(dev, 0), now
        raise _lib.HsaError(f"{what}: {now - before} thread block(s) gave up waiting; their rows hold NaN")


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else c_void_p(t.data_ptr())


def dense_attention_forward(q, k, v, key_lengths=None, packed_mask=None, scale: float = 1.0, empty_value: float = 0.0,
                            need_lse: bool = True, algo: int = _lib.ALGO_AUTO):
    """Raw forward on checked inputs with the device current: returns (out, rest, lse), the last two None unless need_lse.  `rest` is
    what rounding took from a 16-bit output, for the backward's row sums.  No autograd."""
    lib = _lib.load()
    dev = q.device
    B, Lq, H, D = q.shape
    Lk, Hkv = k.shape[1:3]
    out = torch.empty((B, Lq, H, D), dtype=q.dtype, device=dev)
    lse = torch.empty((B, Lq, H), dtype=torch.float32, device=dev) if need_lse else None
    rest = torch.empty((B, Lq, H, D), dtype=q.dtype, device=dev) if need_lse and q.dtype != torch.float32 else None
    dt = _lib.dtype_code(q)
    need = _fwd_workspace(B, Lq, Lk, H, Hkv, D, dt, algo, dev.index)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    rs = H * D
    rc = lib.hsa_dense_attn_fwd(_view(q), _view(k), _view(v), _lib.HsaView(out.data_ptr(), Lq * rs, rs), _ptr(rest), _ptr(lse),
                                _ptr(key_lengths),
                                *_mask_args(packed_mask), _ptr(ws), need, B, Lq, Lk, H, Hkv, D, scale, empty_value, dt, algo,
                                _lib.stream_ptr(dev))
    if rc:
        _lib.check(rc, "hsa_dense_attn_fwd")
    if _lib.DEBUG:
        _debug_check("hsa_dense_attn_fwd")
    return out, rest, lse


_NO_VIEW = _lib.HsaView(None, 0, 0)


def dense_attention_backward(q, k, v, out, rest, lse, dout, key_lengths=None, packed_mask=None, scale: float = 1.0,
                             algo: int = _lib.ALGO_AUTO, need_q: bool = True, need_kv: bool = True):
    """Raw backward with the device current: returns (dq, dk, dv), None for a side that is not asked for (one at least is)."""
    lib = _lib.load()
    dev = q.device
    B, Lq, H, D = q.shape
    Lk, Hkv = k.shape[1:3]
    dq = torch.empty((B, Lq, H, D), dtype=q.dtype, device=dev) if need_q else None
    dk = torch.empty((B, Lk, Hkv, D), dtype=q.dtype, device=dev) if need_kv else None
    dv = torch.empty((B, Lk, Hkv, D), dtype=q.dtype, device=dev) if need_kv else None
    dt = _lib.dtype_code(q)
    need = _bwd_workspace(B, Lq, Lk, H, Hkv, D, dt, algo, dev.index)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    rs, ks = H * D, Hkv * D
    view = _lib.HsaView
    rc = lib.hsa_dense_attn_bwd(_view(q), _view(k), _view(v), view(out.data_ptr(), Lq * rs, rs), _ptr(rest), _ptr(lse), _view(dout),
                                *(_NO_VIEW if t is None else view(t.data_ptr(), n * row, row) for t, n, row in ((dq, Lq, rs), (dk, Lk, ks), (dv, Lk, ks))),
                                _ptr(key_lengths), *_mask_args(packed_mask), _ptr(ws), need, B, Lq, Lk, H, Hkv, D, scale,
                                dt, algo, _lib.stream_ptr(dev))
    if rc:
        _lib.check(rc, "hsa_dense_attn_bwd")
    if _lib.DEBUG:
        _debug_check("hsa_dense_attn_bwd")
    return dq, dk, dv


class _Once(torch.autograd.Function):
    """Gradients as they are; differentiating them again is refused."""

    @staticmethod
    def forward(ctx, *grads):
        return tuple(t.view_as(t) for t in grads)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("cross_attention is differentiable once")


def _once(grads):
    # gradient mode is on inside a backward only when its result is to be differentiated (create_graph)
    if not torch.is_grad_enabled():
        return grads
    there = iter(_Once.apply(*(t.requires_grad_(True) for t in grads if t is not None)))
    return tuple(None if t is None else next(there) for t in grads)


def _unpack_mask(packed: _Packed, Lk: int) -> torch.Tensor:
    """The truth values [batches, heads, rows, Lk] of a packed mask (its first array: bit k of a row's words = key k)."""
    words = (Lk + 127) // 128 * 4
    count = math.prod(packed.sizes) * words
    bits = packed.data[:4 * count].view(torch.int32).view(*packed.sizes, words, 1) >> torch.arange(32, device=packed.data.device, dtype=torch.int32)
    return (bits & 1).bool().flatten(3)[..., :Lk]


def _elementary_gradients(q, k, v, dout, packed: Optional[_Packed], scale: float):
    """(dq, dk, dv) in torch operations, which can be differentiated again.  Heads are not shared, no lengths, no rows to fill."""
    q, k, v, dout = (t.transpose(1, 2) for t in (q, k, v, dout))
    s = (q @ k.transpose(-1, -2)) * scale
    if packed is not None:
        s = s.masked_fill(~_unpack_mask(packed, k.size(2)), -math.inf)
    p = s.softmax(dim=-1)
    dp = dout @ v.transpose(-1, -2)
    ds = p * (dp - (dp * p).sum(dim=-1, keepdim=True)) * scale
    return tuple(t.transpose(1, 2) for t in (ds @ k, ds.transpose(-1, -2) @ q, p.transpose(-1, -2) @ dout))


class _CrossAttention(torch.autograd.Function):
    """twice: gradients of gradients are wanted where the engine records them (create_graph); otherwise they are refused."""

    @staticmethod
    def forward(ctx, q, k, v, key_lengths, packed_mask, scale, empty_value, algo, twice):
        out, rest, lse = dense_attention_forward(q, k, v, key_lengths, packed_mask, scale, empty_value, True, algo)
        if packed_mask is None:
            ctx.save_for_backward(q, k, v, out, rest, lse, key_lengths)
            ctx.meta = (None, scale, algo, twice)
        else:
            ctx.save_for_backward(q, k, v, out, rest, lse, key_lengths, packed_mask.data)
            ctx.meta = (packed_mask.sizes, scale, algo, twice)
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out, rest, lse, key_lengths, *packed = ctx.saved_tensors
        sizes, scale, algo, twice = ctx.meta
        packed = _Packed(packed[0], sizes) if packed else None
        if twice and torch.is_grad_enabled():
            return (*_elementary_gradients(q, k, v, dout, packed, scale), None, None, None, None, None, None)
        with _lib.on_device(q.device):
            dout = _rows(dout if dout.dtype == q.dtype else dout.to(q.dtype))
            grads = dense_attention_backward(q, k, v, out, rest, lse, dout, key_lengths, packed, scale, algo, ctx.needs_input_grad[0],
                                             ctx.needs_input_grad[1] or ctx.needs_input_grad[2])
        return (*_once(grads), None, None, None, None, None, None)


class _NoRows(torch.autograd.Function):
    """No query, or no key for any of them: nothing to launch, and gradients of zero."""

    @staticmethod
    def forward(ctx, q, k, v, empty_value):
        ctx.save_for_backward(q, k, v)
        return torch.full(q.shape, empty_value, dtype=q.dtype, device=q.device)

    @staticmethod
    def backward(ctx, dout):
        return (*_once(tuple(torch.zeros_like(t) if need else None for t, need in zip(ctx.saved_tensors, ctx.needs_input_grad))), None)


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, key_lengths: Optional[torch.Tensor] = None,
                    mask: Optional[torch.Tensor] = None, scale: Optional[float] = None, empty_value: float = 0.0,
                    algo: int = _lib.ALGO_AUTO) -> torch.Tensor:
    """softmax(scale q k^T) v of every query over another sequence's rows.

    q [B, Lq, H, D]; k, v [B, Lk, Hkv, D] with H a multiple of Hkv (query head h reads key/value head h // (H // Hkv));
    float32, bfloat16 or float16, head dim up to 256; returns [B, Lq, H, D] of q's type.  Strided rows are read in place when
    they are packed and aligned, and copied first otherwise.
    key_lengths [B] (int32 or int64, on the device): only keys below a batch entry's length are there; values outside [0, Lk]
        mean the nearer end.
    mask: boolean or integer, nonzero = may attend, [Lq, Lk] or [B, H, Lq, Lk] with dimensions of size 1 broadcast.
    scale: positive; 1 / sqrt(D) if not given.
    A query that may look at no key gives a row of `empty_value` and passes no gradient on.  What k and v hold behind a
    length, or in keys that a mask hides from all queries, may be anything; everything else has to be finite.
    Differentiable once with respect to q, k and v.  In bfloat16 and float16 the weights and the gradients of the scores are
    rounded to that type between the products (in float16's backward moved into the middle of its range first); sums are 32-bit.
    A mask is packed into bits by every call; keys that only a length hides are cheaper given as key_lengths.  With a mask of more
        than 98304 keys, or in the backward one with a row per query where H // Hkv * ceil(Lq / 128) > 768 (say 8 query heads per
        key/value head from 12289 queries on), bfloat16 and float16 run the 32-bit kernels too, at a small part of the speed;
        algo=2 refuses there instead.
    torch.compile breaks its graph here; tracing, torch.func transforms and forward-mode tangents are refused.
    """
    if torch.compiler.is_compiling():
        return _outside_the_graph(_cross_attention, q, k, v, key_lengths, mask, scale, empty_value, algo)
    return _cross_attention(q, k, v, key_lengths, mask, scale, empty_value, algo)


def twice_differentiable_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """cross_attention for HierarchicalAttention: as many key/value heads as query heads, rows that see nothing are NaN, and gradients
    taken with create_graph come from elementary operations (with the [B, H, Lq, Lk] weights), to be differentiated again."""
    return _cross_attention(q, k, v, None, mask, None, math.nan, _lib.ALGO_AUTO, True)


def _cross_attention(q, k, v, key_lengths, mask, scale, empty_value, algo, twice=False):
    _refuse_transforms("cross_attention", q, k, v, key_lengths, mask)
    dev = _check_inputs(q, k, v)
    B, Lq, H, D = q.shape
    Lk = k.size(1)
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise _lib.HsaError("the scale must be positive and finite")
    if key_lengths is not None:
        key_lengths = _lengths32(key_lengths, B, Lk, dev, "key_lengths")
    if mask is not None:
        mask = _mask_bytes(mask, B, H, Lq, Lk, dev)
    if B * Lq * Lk == 0:
        return _NoRows.apply(q, k, v, float(empty_value))
    with _lib.on_device(dev):
        packed = None if mask is None else _pack_mask(mask, dev, Lk)
        if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
            return _CrossAttention.apply(_rows(q), _rows(k), _rows(v), key_lengths, packed, scale, float(empty_value), algo, twice)
        return dense_attention_forward(_rows(q), _rows(k), _rows(v), key_lengths, packed, scale, float(empty_value), False, algo)[0]


def paged_attention_decode(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                           lengths: torch.Tensor, scale: Optional[float] = None, splits: Optional[int] = None,
                           algo: int = _lib.ALGO_AUTO) -> torch.Tensor:
    """Attention of the single new token of every sequence over its cached keys and values, which live in pages.

    q [B, H, D]; k_pages, v_pages [num_pages, page_size, Hkv, D] (pages and slots may be strided; a slot's [Hkv, D] is packed);
    page_table [B, max_pages] int32 and lengths [B] int32 on the device: key j of sequence b is slot j % page_size of page
    page_table[b, j // page_size], for j < lengths[b].  The new token's own key and value are in the cache if it is to see them.
    Returns [B, H, D] of q's type; zeros for a length of 0.  A page number outside the pages that the length reaches, or a length the
    table cannot hold, makes that sequence's output NaN; table entries behind the length are not read.
    splits: ranges a sequence's keys are cut into (None: chosen from the sizes).  No autograd.
    torch.compile breaks its graph here; tracing, torch.func transforms and forward-mode tangents are refused.
    """
    if torch.compiler.is_compiling():
        return _outside_the_graph(_paged_attention_decode, q, k_pages, v_pages, page_table, lengths, scale, splits, algo)
    return _paged_attention_decode(q, k_pages, v_pages, page_table, lengths, scale, splits, algo)


def _paged_attention_decode(q, k_pages, v_pages, page_table, lengths, scale, splits, algo):
    _refuse_transforms("paged_attention_decode", q, k_pages, v_pages, page_table, lengths)
    lib = _lib.load()
    dev = _lib.require_cuda(q, k_pages, v_pages, page_table, lengths)
    dt = _lib.dtype_code(q)
    assert q.dim() == 3 and k_pages.dim() == 4, "q is [B, H, D]; the pages are [num_pages, page_size, Hkv, D]"
    B, H, D = q.shape
    num_pages, page_size, Hkv, Dk = k_pages.shape
    assert v_pages.shape == k_pages.shape and Dk == D, \
        f"shapes disagree: q {tuple(q.shape)}, k_pages {tuple(k_pages.shape)}, v_pages {tuple(v_pages.shape)}"
    assert k_pages.dtype == q.dtype and v_pages.dtype == q.dtype, "dtype mismatch"
    assert H >= 1 and Hkv >= 1 and H % Hkv == 0, f"{H} query heads are not a multiple of {Hkv} key/value heads"
    assert 1 <= D <= 256, f"head dim {D} outside 1..256"
    assert page_table.dtype == torch.int32 and lengths.dtype == torch.int32, "page_table and lengths are int32"
    assert page_table.dim() == 2 and page_table.size(0) == B and lengths.shape == (B,), \
        f"page_table is [{B}, max_pages] and lengths [{B}]"
    if not ((k_pages.is_contiguous() or _lib.inner_contiguous(k_pages)) and (v_pages.is_contiguous() or _lib.inner_contiguous(v_pages))):
        raise _lib.HsaError("a slot's [Hkv, D] block must be packed (the cache is not copied)")
    if scale is None:
        scale = D ** -0.5
    if not 0.0 < scale < math.inf:
        raise _lib.HsaError("the scale must be positive and finite")
    max_pages = page_table.size(1)
    out = torch.empty((B, H, D), dtype=q.dtype, device=dev)
    if B == 0:
        return out
    if max_pages == 0 or num_pages == 0 or page_size == 0:
        # no cache: every length has to be 0 (a table without room for a longer one gives NaN, as below)
        return out.copy_(torch.where(lengths.view(B, 1, 1) == 0, 0.0, math.nan).expand(B, H, D))
    if not q.is_contiguous():
        q = q.contiguous()
    if page_table.stride(1) != 1 and max_pages > 1:
        page_table = page_table.contiguous()
    if not lengths.is_contiguous():
        lengths = lengths.contiguous()
    with _lib.on_device(dev):
        splits, need = _paged_plan(B, H, Hkv, D, page_size, max_pages, splits, dev.index)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        rc = lib.hsa_paged_attn_decode(_lib.HsaView(q.data_ptr(), H * D, H * D), _lib.rows_view(k_pages), _lib.rows_view(v_pages),
                                       _lib.HsaView(out.data_ptr(), H * D, H * D), c_void_p(page_table.data_ptr()),
                                       page_table.stride(0), c_void_p(lengths.data_ptr()), _ptr(ws), need, B, H, Hkv, D,
                                       page_size, num_pages, max_pages, float(scale), dt, splits, algo, _lib.stream_ptr(dev))
    if rc:
        _lib.check(rc, "hsa_paged_attn_decode")
    return out
