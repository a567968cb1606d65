"""The operators between the two norms of a transformer block, on one rank's heads.

``qk_norm_rope`` (and its backward) norms the query and key heads and turns them by
their positions; ``qk_norm_rope_write`` does so and puts keys and values into a
``PagedKVCache``, which holds them in q's type or as e4m3 codes; ``paged_attention``
is the attention of one new token of each sequence over that cache. Its output is
the input ``a`` of ``FusedTPLinearRMSNorm``. Heads are split over a tensor-parallel
group as the projection's columns are, so none of these exchanges anything. No
counterpart in the reference. As in ``api``: ``AssertionError`` for the contract's
checks, ``RMSNormTPError`` for what the library refuses, no fallback.
"""
from __future__ import annotations

import ctypes
import functools
import struct
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import LIB, check
from .api import _DTYPES, _stream_of, dtype_code

# layouts of rmsnorm_qk_rope_args, rmsnorm_qk_rope_backward_args, rmsnorm_kv_cache and
# rmsnorm_paged_attention_args (include/rmsnorm_tp_b200.h)
_ROPE_ARGS = struct.Struct("@9Q10q2q2Q6ifi")
_BACK_ARGS = struct.Struct("@13Qq8q2q6ifi")
_CACHE = struct.Struct("@4Qq4i")
_ATTN_ARGS = struct.Struct("@7Qq3q2q2ifi")

_CACHE_DTYPES = {**_DTYPES, torch.float8_e4m3fn: _lib.KV_E4M3}


def rope_table(max_positions: int, rotary_dim: int, base: float = 10000.0,
               device=None) -> torch.Tensor:
    """fp32 [max_positions, rotary_dim]: the cosines, then the sines, of position *
    base^(-2i / rotary_dim). The angles are computed in 64 bits; any other table of
    this layout (scaled frequencies, say) serves as well."""
    if max_positions < 1 or rotary_dim < 2 or rotary_dim % 2:
        raise AssertionError(f"max_positions {max_positions} must be positive and rotary_dim "
                             f"{rotary_dim} even and positive")
    freq = float(base) ** (-torch.arange(0, rotary_dim, 2, device=device, dtype=torch.float64) / rotary_dim)
    angle = torch.arange(max_positions, device=device, dtype=torch.float64)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).to(torch.float32)


_F32, _I32, _I64 = torch.float32, torch.int32, torch.int64


# A call's tensors are looked at attribute by attribute once, in one condition (a few
# microseconds of host time are most of a decode-sized call); only where it fails does
# _explain_* look again for the words.

def _rows_fit(t: torch.Tensor, tokens: int, heads: int, d: int, dtype: torch.dtype, device: int) -> bool:
    return t.dtype is dtype and t.get_device() == device and t.shape == (tokens, heads, d) and t.stride(2) == 1


def _index_fits(t: torch.Tensor, n: int, dtype: torch.dtype, device: int) -> bool:
    return t.dtype is dtype and t.get_device() == device and t.shape == (n,) and t.is_contiguous()


def _weight_fits(t: torch.Tensor, d: int, dtype: torch.dtype, device: int) -> bool:
    return t.dtype is dtype and t.get_device() == device and t.shape == (d,) and t.is_contiguous()


def _contiguous_like(t: torch.Tensor) -> torch.Tensor:
    """A fresh contiguous tensor (empty_like, the faster call, keeps the order of strides)."""
    out = torch.empty_like(t)
    return out if out.is_contiguous() else t.new_empty(t.shape)


def _turn_sizes(q, k, q_weight, k_weight, rope, positions):
    """(device, dtype, tokens, q heads, kv heads, head_dim, table rows, rotary_dim) of
    operands that fit together; AssertionError for others."""
    qs, ks, rs = q.shape, k.shape, rope.shape
    if len(qs) == 3 and len(ks) == 3 and len(rs) == 2:
        (tokens, hq, d), (tokens_k, hk, dk), (most, r) = qs, ks, rs
        device, dtype = q.get_device(), q.dtype
        if (device >= 0 and dtype in _DTYPES and q.stride(2) == 1 and tokens_k == tokens and dk == d
                and k.dtype is dtype and k.get_device() == device and k.stride(2) == 1
                and rope.dtype is _F32 and rope.get_device() == device and rope.is_contiguous()
                and positions.dtype is _I64 and positions.get_device() == device and positions.shape == (tokens,)
                and positions.is_contiguous()
                and (q_weight is None and k_weight is None
                     or q_weight is not None and k_weight is not None
                     and _weight_fits(q_weight, d, dtype, device) and _weight_fits(k_weight, d, dtype, device))):
            return device, dtype, tokens, hq, hk, d, most, r
    _explain_turn(q, k, q_weight, k_weight, rope, positions)


def _explain_rows(name: str, t: torch.Tensor, q: torch.Tensor, heads: int) -> None:
    if t.dtype != q.dtype or t.device != q.device:
        raise AssertionError(f"{name} must have q's dtype and device, got {t.dtype} on {t.device}")
    raise AssertionError(f"{name} must be [tokens={q.shape[0]}, {heads or 'heads'}, head_dim={q.shape[2]}] with "
                         f"stride 1 in the last dimension, got {tuple(t.shape)} with strides {t.stride()}")


def _explain_index(name: str, n: int, dtype: torch.dtype) -> None:
    raise AssertionError(f"{name} must be contiguous {dtype} [{n}] on q's device")


def _explain_turn(q, k, q_weight, k_weight, rope, positions) -> None:
    if not q.is_cuda:
        raise AssertionError("q must be a CUDA tensor")
    if q.dtype not in _DTYPES:
        raise AssertionError(f"unsupported dtype {q.dtype}; expected float32, bfloat16 or float16")
    if q.dim() != 3 or q.stride(2) != 1:
        raise AssertionError("q must be [tokens, q_heads, head_dim] with stride 1 in the last "
                             f"dimension, got {tuple(q.shape)} with strides {q.stride()}")
    tokens, _, d = q.shape
    device = q.get_device()
    if k.dim() != 3 or not _rows_fit(k, tokens, k.shape[1], d, q.dtype, device):
        _explain_rows("k", k, q, 0)
    if (q_weight is None) != (k_weight is None):
        raise AssertionError("give both q_weight and k_weight, or neither (rotation without norm)")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and not _weight_fits(w, d, q.dtype, device):
            raise AssertionError(f"{name} must be contiguous [{d}] with q's dtype and device")
    if not _index_fits(positions, tokens, _I64, device):
        _explain_index("positions", tokens, _I64)
    raise AssertionError("rope must be a contiguous float32 [max_positions, rotary_dim] on q's device")


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor],
                 k_weight: Optional[torch.Tensor], rope: torch.Tensor, positions: torch.Tensor,
                 eps: float = 1e-6, interleaved: bool = False, q_out: Optional[torch.Tensor] = None,
                 k_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMSNorm of every query and key head, then the rotation by the token's position.

    ``q`` [tokens, q_heads, head_dim] and ``k`` [tokens, kv_heads, head_dim] may be views
    (column blocks of the projection's output); the weights are [head_dim], shared by the
    heads, or both None (rotation alone). ``rope``: see ``rope_table``; its width is the
    rotary_dim, and elements behind it are not turned. Pairs are (i, i + rotary_dim / 2),
    or with ``interleaved`` (2i, 2i + 1). ``positions`` int64 [tokens]; one outside the
    table makes the token's turned elements NaN. ``q_out`` / ``k_out`` receive the results
    instead of fresh tensors and may be q / k themselves. fp32 inside, rounded once. Not
    recorded for autograd: see ``qk_norm_rope_with_grad``."""
    device, dtype, tokens, hq, hk, d, most, r = _turn_sizes(q, k, q_weight, k_weight, rope, positions)
    if q_out is None:
        q_out = torch.empty_like(q)
    elif not _rows_fit(q_out, tokens, hq, d, dtype, device):
        _explain_rows("q_out", q_out, q, hq)
    if k_out is None:
        k_out = torch.empty_like(k)
    elif not _rows_fit(k_out, tokens, hk, d, dtype, device):
        _explain_rows("k_out", k_out, q, hk)
    a, b, _ = q.stride()
    c, e, _ = k.stride()
    f, g, _ = q_out.stride()
    h, i, _ = k_out.stride()
    args = _ROPE_ARGS.pack(
        q.data_ptr(), k.data_ptr(), 0, q_out.data_ptr(), k_out.data_ptr(),
        0 if q_weight is None else q_weight.data_ptr(), 0 if k_weight is None else k_weight.data_ptr(),
        rope.data_ptr(), positions.data_ptr(), a, b, c, e, 0, 0, f, g, h, i, tokens, most, 0, 0, hq, hk, d, r,
        _DTYPES[dtype], bool(interleaved), eps, device)
    check(LIB.rmsnorm_qk_rope_forward(args, _stream_of(device)), "rmsnorm_qk_rope_forward")
    return q_out, k_out


def qk_norm_rope_backward(dq_out: torch.Tensor, dk_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                          q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                          rope: torch.Tensor, positions: torch.Tensor, eps: float = 1e-6,
                          interleaved: bool = False):
    """Gradients ``(dq, dk, dq_weight, dk_weight)`` of ``qk_norm_rope`` for the output
    gradients (the last two None without weights). The weights' gradients are sums over
    tokens and heads in a fixed order; over a tensor-parallel group they are this rank's
    heads' share. Capturable in a CUDA graph."""
    device, dtype, tokens, hq, hk, d, most, r = _turn_sizes(q, k, q_weight, k_weight, rope, positions)
    if not _rows_fit(dq_out, tokens, hq, d, dtype, device):
        _explain_rows("dq_out", dq_out, q, hq)
    if not _rows_fit(dk_out, tokens, hk, d, dtype, device):
        _explain_rows("dk_out", dk_out, q, hk)
    dq, dk = _contiguous_like(q), _contiguous_like(k)
    if q_weight is None:
        dqw = dkw = None
        weights = (0, 0, 0, 0)
        ws_ptr = nbytes = 0
    else:
        dqw, dkw = torch.empty_like(q_weight), torch.empty_like(k_weight)
        weights = (dqw.data_ptr(), dkw.data_ptr(), q_weight.data_ptr(), k_weight.data_ptr())
        nbytes = _backward_workspace(tokens, hq, hk, d, r, _DTYPES[dtype])
        ws = rope.new_empty(nbytes // 4) if nbytes else None
        ws_ptr = ws.data_ptr() if nbytes else 0
    a, b, _ = dq_out.stride()
    c, e, _ = dk_out.stride()
    f, g, _ = q.stride()
    h, i, _ = k.stride()
    args = _BACK_ARGS.pack(
        dq_out.data_ptr(), dk_out.data_ptr(), q.data_ptr(), k.data_ptr(), dq.data_ptr(), dk.data_ptr(), *weights,
        rope.data_ptr(), positions.data_ptr(), ws_ptr, nbytes, a, b, c, e, f, g, h, i, tokens, most, hq, hk, d, r,
        _DTYPES[dtype], bool(interleaved), eps, device)
    check(LIB.rmsnorm_qk_rope_backward(args, _stream_of(device)), "rmsnorm_qk_rope_backward")
    return dq, dk, dqw, dkw


@functools.lru_cache(maxsize=4096)
def _backward_workspace(*sizes: int) -> int:
    """Bytes of the workspace (a function of the sizes alone); 0 where none is used, and for
    what the call itself will refuse."""
    return LIB.rmsnorm_qk_rope_backward_workspace_bytes(*sizes)


class _QkNormRopeFunction(torch.autograd.Function):
    """Autograd around qk_norm_rope: forward kernel, backward kernel."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, rope, positions, eps, interleaved):
        ctx.save_for_backward(q, k, q_weight, k_weight, rope, positions)
        ctx.eps, ctx.interleaved = eps, interleaved
        return qk_norm_rope(q, k, q_weight, k_weight, rope, positions, eps, interleaved)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight, rope, positions = ctx.saved_tensors
        dq_out = dq_out if dq_out.stride(2) == 1 else dq_out.contiguous()
        dk_out = dk_out if dk_out.stride(2) == 1 else dk_out.contiguous()
        return (*qk_norm_rope_backward(dq_out, dk_out, q, k, q_weight, k_weight, rope, positions, ctx.eps,
                                       ctx.interleaved), None, None, None, None)


def qk_norm_rope_with_grad(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor],
                           k_weight: Optional[torch.Tensor], rope: torch.Tensor, positions: torch.Tensor,
                           eps: float = 1e-6, interleaved: bool = False):
    """``qk_norm_rope`` recorded for autograd; its backward runs the backward kernel (once:
    it is not differentiable itself). q, k and the weights get gradients; a table that wants
    one is refused."""
    if rope.requires_grad and torch.is_grad_enabled():
        raise AssertionError("rope gets no gradient: give a table that does not require one")
    return _QkNormRopeFunction.apply(q, k, q_weight, k_weight, rope, positions, eps, interleaved)


def _held(i: int, doc: str) -> property:
    """A tensor whose address the native handle holds: changed in place only."""

    def put(self, value):
        if value is not self._tensors[i]:    # (`cache.k *= 2` puts back what it got)
            raise AttributeError("a PagedKVCache keeps its tensors; change them in place")

    return property(lambda self: self._tensors[i], put, doc=doc)


class PagedKVCache:
    """Keys and values of many sequences in pages of ``page_size`` tokens.

    ``k`` and ``v`` are [num_pages, kv_heads, page_size, head_dim], so a head's rows of a
    page lie in one piece; ``dtype`` float32, bfloat16, float16 or float8_e4m3fn. The last
    holds codes, with a scale for each (token, head) in ``k_scale`` and ``v_scale``
    [num_pages, kv_heads, page_size] fp32: scale = max(amax, 2^-100) / 448 of the row, code =
    e4m3(x / scale), and a row stands for code * scale. A row with an infinity reads back
    as NaN; a NaN stays where it is (the maximum is the others'). The token at ``offset`` of ``page`` has slot page * page_size + offset; which
    pages belong to which sequence is the caller's ``page_table``. head_dim is a multiple
    of 16, at most 256. A fresh cache holds zeros."""

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device=None):
        device = torch.device("cuda") if device is None else torch.device(device)
        if min(num_pages, page_size, num_kv_heads) < 1:
            raise AssertionError("num_pages, page_size and num_kv_heads must be positive")
        if dtype not in _CACHE_DTYPES:
            raise AssertionError(f"unsupported cache dtype {dtype}")
        shape = (num_pages, num_kv_heads, page_size)
        k, v = (torch.zeros(*shape, head_dim, dtype=dtype, device=device) for _ in range(2))
        scales = (None, None)
        if dtype == torch.float8_e4m3fn:
            scales = tuple(torch.zeros(shape, dtype=torch.float32, device=device) for _ in range(2))
        self._adopt(k, v, *scales)

    @classmethod
    def from_tensors(cls, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                     v_scale: Optional[torch.Tensor] = None) -> "PagedKVCache":
        """A cache over tensors that the caller holds (no copy)."""
        cache = cls.__new__(cls)
        cache._adopt(k, v, k_scale, v_scale)
        return cache

    def _adopt(self, k, v, k_scale, v_scale) -> None:
        if k.dtype not in _CACHE_DTYPES:
            raise AssertionError(f"unsupported cache dtype {k.dtype}")
        if not k.is_cuda or k.dim() != 4:
            raise AssertionError("k must be a CUDA tensor [num_pages, kv_heads, page_size, head_dim]")
        if k.shape[1] < 1 or k.shape[2] < 1:
            raise AssertionError(f"kv_heads and page_size must be positive, got {tuple(k.shape)}")
        for name, t in (("k", k), ("v", v)):
            if t.shape != k.shape or t.dtype != k.dtype or t.device != k.device or not t.is_contiguous():
                raise AssertionError(f"{name} must be contiguous with k's shape, dtype and device")
        e4m3 = k.dtype == torch.float8_e4m3fn
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if (t is not None) != e4m3:
                raise AssertionError(f"{name} belongs to a float8_e4m3fn cache, and only to one")
            if e4m3 and (t.shape != k.shape[:3] or t.dtype != torch.float32 or t.device != k.device
                         or not t.is_contiguous()):
                raise AssertionError(f"{name} must be contiguous float32 {tuple(k.shape[:3])} on k's device")
        self.num_pages, self.num_kv_heads, self.page_size, self.head_dim = k.shape
        if self.head_dim % 16 or not 16 <= self.head_dim <= 256:
            raise AssertionError(f"head_dim {self.head_dim} must be a multiple of 16, at most 256")
        self._tensors = k, v, k_scale, v_scale
        # a cache whose keys are its values (one tensor for both) can be read, not written
        ends = sorted((t.data_ptr(), t.data_ptr() + t.nbytes) for t in (k, v, k_scale, v_scale) if t is not None)
        self._apart = all(a[1] <= b[0] for a, b in zip(ends, ends[1:]))
        self.dtype, self.device, self._index = k.dtype, k.device, k.get_device()
        self._code = _CACHE_DTYPES[k.dtype]
        self._struct = ctypes.create_string_buffer(_CACHE.pack(
            k.data_ptr(), v.data_ptr(), k_scale.data_ptr() if e4m3 else 0,
            v_scale.data_ptr() if e4m3 else 0, self.num_pages, self.page_size, self.num_kv_heads,
            self.head_dim, self._code))
        self._address = ctypes.addressof(self._struct)

    # deepcopy and pickle make other tensors (copy.copy the same): the native structure is
    # made anew over them, or the copy would go on reading and writing this cache's
    def __getstate__(self):
        return {n: v for n, v in self.__dict__.items() if n not in ("_struct", "_address")}

    def __setstate__(self, state) -> None:
        self.__dict__.update(state)
        self._adopt(*state["_tensors"])

    k = _held(0, "keys, or their codes")
    v = _held(1, "values, or their codes")
    k_scale = _held(2, "scales of the keys' codes, or None")
    v_scale = _held(3, "scales of the values' codes, or None")

    def read(self, slots: torch.Tensor, dtype: Optional[torch.dtype] = None):
        """(k, v) [count, kv_heads, head_dim] of ``dtype``: the rows at ``slots`` (int64
        [count]), an e4m3 row as code * scale rounded once. A slot outside the cache gives
        zeros. ``dtype`` is the cache's own unless given (bfloat16 for an e4m3 cache)."""
        if dtype is None:
            dtype = torch.bfloat16 if self.dtype == torch.float8_e4m3fn else self.dtype
        code, device = dtype_code(dtype), self._index
        if slots.dtype is not _I64 or slots.get_device() != device or slots.dim() != 1 or \
                not slots.is_contiguous():
            raise AssertionError("slots must be contiguous int64 [count] on the cache's device")
        count = slots.shape[0]
        k = torch.empty(count, self.num_kv_heads, self.head_dim, dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        check(LIB.rmsnorm_kv_read(self._address, k.data_ptr(), v.data_ptr(), slots.data_ptr(), count, code,
                                  device, _stream_of(device)), "rmsnorm_kv_read")
        return k, v


def qk_norm_rope_write(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_weight: Optional[torch.Tensor],
                       k_weight: Optional[torch.Tensor], rope: torch.Tensor, positions: torch.Tensor,
                       cache: PagedKVCache, slots: torch.Tensor, eps: float = 1e-6,
                       interleaved: bool = False, q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``qk_norm_rope`` whose keys go into ``cache`` with ``v`` beside them; returns the
    queries. ``slots`` int64 [tokens] are distinct within a call; a token whose slot lies
    outside the cache (-1: padding) leaves the cache as it is. The cache has q's dtype, or
    float8_e4m3fn (quantised from the fp32 values); its tensors share no memory with q, k, v,
    ``q_out`` or one another (cached keys turned where they lie: ``qk_norm_rope`` on a view of
    their pages, with ``k_out`` that view)."""
    device, dtype, tokens, hq, hk, d, most, r = _turn_sizes(q, k, q_weight, k_weight, rope, positions)
    if not _rows_fit(v, tokens, hk, d, dtype, device):
        _explain_rows("v", v, q, hk)
    if not _index_fits(slots, tokens, _I64, device):
        _explain_index("slots", tokens, _I64)
    if cache._index != device or cache.num_kv_heads != hk or cache.head_dim != d:
        raise AssertionError(f"the cache holds {cache.num_kv_heads} heads of {cache.head_dim} on "
                             f"{cache.device}, the call has {hk} of {d} on {q.device}")
    if cache.dtype is not dtype and cache._code != _lib.KV_E4M3:
        raise AssertionError(f"a {cache.dtype} cache does not take {dtype}")
    if not cache._apart:
        raise AssertionError("the cache's tensors share memory: it can be read, not written")
    if q_out is None:
        q_out = torch.empty_like(q)
    elif not _rows_fit(q_out, tokens, hq, d, dtype, device):
        _explain_rows("q_out", q_out, q, hq)
    a, b, _ = q.stride()
    c, e, _ = k.stride()
    f, g, _ = v.stride()
    h, i, _ = q_out.stride()
    args = _ROPE_ARGS.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), q_out.data_ptr(), 0,
        0 if q_weight is None else q_weight.data_ptr(), 0 if k_weight is None else k_weight.data_ptr(),
        rope.data_ptr(), positions.data_ptr(), a, b, c, e, f, g, h, i, 0, 0, tokens, most, cache._address,
        slots.data_ptr(), hq, hk, d, r, _DTYPES[dtype], bool(interleaved), eps, device)
    check(LIB.rmsnorm_qk_rope_write(args, _stream_of(device)), "rmsnorm_qk_rope_write")
    return q_out


def _attention_args(q, out, lse, page_table, seq_lens, ws, ws_bytes, cache_address, strides, table_stride,
                    batch, max_pages, q_heads, dtype, scale, device) -> bytes:
    return _ATTN_ARGS.pack(cache_address, q, out, lse, page_table, seq_lens, ws, ws_bytes, *strides,
                           table_stride, batch, max_pages, q_heads, dtype, scale, device)


@functools.lru_cache(maxsize=4096)
def _attention_workspace(num_pages, page_size, kv_heads, head_dim, cache_dtype, batch, max_pages, q_heads,
                         dtype, device) -> int:
    """Bytes for a call of these sizes (a function of sizes alone); 0 where none is used,
    and for what the call itself will refuse."""
    some = 256   # an address that the size check takes and never follows
    cache = ctypes.create_string_buffer(_CACHE.pack(some, some, some, some, num_pages, page_size, kv_heads,
                                                    head_dim, cache_dtype))
    return LIB.rmsnorm_paged_attention_workspace_bytes(_attention_args(
        some, some, 0, some, some, 0, 0, ctypes.addressof(cache), (0, 0), 0, batch, max_pages, q_heads,
        dtype, 1.0, device))


def paged_attention(q: torch.Tensor, cache: PagedKVCache, page_table: torch.Tensor, seq_lens: torch.Tensor,
                    scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                    return_lse: bool = False):
    """Attention of one new token of each sequence over its cached tokens (that token's
    own key among them: write it first).

    ``q`` [batch, q_heads, head_dim], q_heads a multiple of the cache's heads, of the
    cache's dtype or any for an e4m3 cache; ``page_table`` int32 [batch, max_pages];
    ``seq_lens`` int32 [batch], on the device: the work is divided as they say when the
    kernel runs, so a captured call follows them. Returns ``out`` [batch, q_heads,
    head_dim], with ``return_lse`` also the fp32 logarithm of each head's sum of
    exponentials [batch, q_heads]. A sequence without tokens gives zeros and -inf; pages
    outside the cache are left out, lengths cut to max_pages * page_size. ``scale`` is
    head_dim^-0.5 unless given. A serving operator: not recorded for autograd.

    Fast for 16-bit queries and head_dim 64, 96, 128, 192 or 256, best with at most 16 query
    heads a kv head. fp32 queries and the other multiples of 16 take a plain kernel that reads
    the cache once for each query head, some 40 times slower on a long sequence."""
    qs, device, q_dtype = q.shape, q.get_device(), q.dtype
    if device < 0 or len(qs) != 3 or q.stride(2) != 1:
        raise AssertionError("q must be a CUDA tensor [batch, q_heads, head_dim] with stride 1 in the last "
                             f"dimension, got {tuple(qs)}")
    if q_dtype not in _DTYPES:
        raise AssertionError(f"unsupported dtype {q_dtype}; expected float32, bfloat16 or float16")
    batch, heads, d = qs
    if cache._index != device or d != cache.head_dim or heads % cache.num_kv_heads:
        raise AssertionError(f"q has {heads} heads of {d} on {q.device}, the cache {cache.num_kv_heads} of "
                             f"{cache.head_dim} on {cache.device}")
    if cache.dtype is not q_dtype and cache._code != _lib.KV_E4M3:
        raise AssertionError(f"a {cache.dtype} cache does not serve {q_dtype} queries")
    ts, tst = page_table.shape, page_table.stride()
    if page_table.dtype is not _I32 or page_table.get_device() != device or len(ts) != 2 or ts[0] != batch or \
            (ts[1] > 1 and tst[1] != 1):
        raise AssertionError(f"page_table must be int32 [{batch}, max_pages] on q's device, rows in one piece")
    if not _index_fits(seq_lens, batch, _I32, device):
        _explain_index("seq_lens", batch, _I32)
    if out is None:
        out = _contiguous_like(q)
    elif out.shape != qs or out.dtype is not q_dtype or out.get_device() != device or not out.is_contiguous():
        raise AssertionError("out must be contiguous with q's shape, dtype and device")
    lse = torch.empty(batch, heads, dtype=_F32, device=q.device) if return_lse else None
    dtype = _DTYPES[q_dtype]
    nbytes = _attention_workspace(cache.num_pages, cache.page_size, cache.num_kv_heads, d, cache._code, batch,
                                  ts[1], heads, dtype, device)
    ws = q.new_empty(nbytes // 2) if nbytes else None    # 16-bit or wider elements: at least nbytes
    a, b, _ = q.stride()
    args = _ATTN_ARGS.pack(cache._address, q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0,
                           page_table.data_ptr(), seq_lens.data_ptr(), ws.data_ptr() if nbytes else 0, nbytes, a, b, tst[0],
                           batch, ts[1], heads, dtype, d ** -0.5 if scale is None else scale, device)
    check(LIB.rmsnorm_paged_attention(args, _stream_of(device)), "rmsnorm_paged_attention")
    return (out, lse) if return_lse else out
