"""The 8-bit serving operators on device buffers (include/evelyn.h, "8-bit serving operators").

    quantize_rows(x, codes, scales)                       activation rows in 8 bits
    matmul(x, x_scales, w, w_scales, y, add=None)         8-bit product, scales per token and channel
    cache = Kv8Cache(k, v, k_scales, v_scales)            a paged KV cache in 8 bits
    batch = Kv8Batch(page_table, cu, lens, max_new, max_len)
    kv8_append(cache, batch, k, v, q=..., q_out=..., rope=...)
    kv8_attention(cache, batch, q, out, workspace=...)

A layer of a decode or prompt step runs them one after the other: quantise, the q / k / v
product, append, attention, quantise, the output product with the residual added.

Arguments are tensors in device memory, those of a call on one device: any object with
``data_ptr()``, ``dtype``, ``shape``, ``stride()`` and, to have that checked, ``device``
(PyTorch's, for one). Outputs are written into the tensors given. ``stream`` is a
CUDA stream handle (an integer; 0 is the device's default stream): a caller working on another
stream passes that one. Calls are asynchronous and allocate nothing, so they can be captured into
a graph. Arguments that do not fit raise EvelynError (InvalidInput, Unsupported); ``err``, an int32
tensor of one element that the caller has cleared, receives 3 where the device-side lists
name a position or page outside what was described.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

from . import runtime
from .runtime import EvelynError, _check, _Kv8Batch, _Kv8Cache, _Kv8Prep

# element types by name, as the C ABI numbers them
_TYPES = {"float32": 0, "float16": 1, "bfloat16": 30}
_kinds: dict = {}


def _kind(t) -> int:
    """The C ABI's number of an activation tensor's type."""
    try:
        return _kinds[t.dtype]
    except KeyError:
        name = str(t.dtype).rpartition(".")[2]
        if name not in _TYPES:
            raise EvelynError(4, f"activations are float32, float16 or bfloat16, not {name}") from None
        return _kinds.setdefault(t.dtype, _TYPES[name])


# What the checks of a call found, by the types, shapes, strides and devices of its tensors
# (never by their addresses): a call whose tensors are laid out like an earlier one's is not checked again.
_plans: dict = {}
_MOST_PLANS = 4096
_MOST_TOTALS = 64  # descriptors that a batch keeps


def _layout(*tensors) -> tuple:
    return tuple([None if t is None else (t.dtype, t.shape, t.stride(), getattr(t, "device", None)) for t in tensors])


def _planned(key: tuple, plan):
    if len(_plans) >= _MOST_PLANS:
        _plans.clear()
    _plans[key] = plan
    return plan


def _need(ok: bool, msg: str):
    if not ok:
        raise EvelynError(1, msg)


def _u32(what: str, *sizes: int):
    """The C ABI's counts have 32 bits; a larger one must not arrive there as another."""
    _need(all(n < 1 << 32 for n in sizes), f"{what} must be below 2^32")


def _device_of(*tensors, known=()):
    """The device that all of them are on (None for objects that name none)."""
    found = {d for d in known if d is not None}
    found.update(t.device for t in tensors if getattr(t, "device", None) is not None)
    _need(len(found) <= 1, f"the tensors of a call must be on one device, not on {sorted(map(str, found))}")
    return found.pop() if found else None


def _named(t, name: str, what: str):
    _need(str(t.dtype).rpartition(".")[2] == name, f"{what} must be {name}")


def _rows(t, what: str, dims: int = 2) -> int:
    """Stride between the rows of a tensor whose later dimensions are contiguous."""
    shape, stride = t.shape, t.stride()
    _need(len(shape) == dims, f"{what} must have {dims} dimensions")
    want = 1
    for n, s in zip(reversed(shape[1:]), reversed(stride[1:])):
        _need(s == want or n <= 1, f"{what}: only the first dimension may be strided")
        want *= n
    return max(stride[0], want) if shape[0] <= 1 else stride[0]


def _flat(t, n: int, name: str, what: str):
    _named(t, name, what)
    _need(len(t.shape) == 1 and t.shape[0] == n and (n <= 1 or t.stride()[0] == 1),
          f"{what} must hold {n} contiguous values")


def _ptr(t) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _check_err(err):
    if err is not None:
        _named(err, "int32", "err")
        _need(err.numel() >= 1, "err must hold one value")


def quantize_rows(x, codes, scales, stream: int = 0) -> None:
    """Rows of x [rows][cols] to codes [rows][cols] int8 and scales [rows] float32:
    scale = max|x| / 127, code = x * (1 / scale) rounded to nearest even (evl_i8_quantize_rows)."""
    key = ("rows", _layout(x, codes, scales))
    plan = _plans.get(key)
    if plan is None:
        _device_of(x, codes, scales)
        kind, xs, cs = _kind(x), _rows(x, "x"), _rows(codes, "codes")
        rows, cols = x.shape
        _u32("rows and cols", rows, cols)
        _named(codes, "int8", "codes")
        _need(tuple(codes.shape) == (rows, cols), "codes must have the shape of x")
        _flat(scales, rows, "float32", "scales")
        plan = _planned(key, (kind, xs, rows, cols, cs))
    kind, xs, rows, cols, cs = plan
    _check(runtime.lib().evl_i8_quantize_rows(kind, x.data_ptr(), xs, rows, cols, codes.data_ptr(), cs,
                                              scales.data_ptr(), stream))


def matmul(x, x_scales, w, w_scales, y, add=None, err=None, stream: int = 0) -> None:
    """y [rows][out] = (x [rows][cols] @ w [out][cols]^T) * x_scales[:, None] * w_scales (+ add),
    x and w int8 with rows on 16-byte boundaries, int32 sums (evl_i8_matmul)."""
    key = ("matmul", _layout(x, x_scales, w, w_scales, y, add, err))
    plan = _plans.get(key)
    if plan is None:
        _device_of(x, x_scales, w, w_scales, y, add, err)
        _check_err(err)
        kind, xst, wst, yst = _kind(y), _rows(x, "x"), _rows(w, "w"), _rows(y, "y")
        rows, cols = x.shape
        out = w.shape[0]
        _u32("rows, out and cols", rows, out, cols)
        _named(x, "int8", "x")
        _named(w, "int8", "w")
        _need(w.shape[1] == cols, "x and w must have the same number of columns")
        _need(tuple(y.shape) == (rows, out), "y must be [rows of x][rows of w]")
        _flat(x_scales, rows, "float32", "x_scales")
        _flat(w_scales, out, "float32", "w_scales")
        ast = 0
        if add is not None:
            ast = _rows(add, "add")
            _need(tuple(add.shape) == (rows, out) and add.dtype == y.dtype, "add must have the shape and type of y")
        # (a single row has no stride; the operand's next 16-byte boundary stands in)
        xst, wst = (-(-s // 16) * 16 if n <= 1 else s for s, n in ((xst, rows), (wst, out)))
        plan = _planned(key, (kind, xst, wst, yst, ast, rows, out, cols))
    kind, xst, wst, yst, ast, rows, out, cols = plan
    _check(runtime.lib().evl_i8_matmul(x.data_ptr(), xst, x_scales.data_ptr(), rows, w.data_ptr(), wst,
                                       w_scales.data_ptr(), out, cols, kind, _ptr(add), ast, y.data_ptr(), yst,
                                       _ptr(err), stream))


class Kv8Cache:
    """Pages of an 8-bit KV cache (evl_kv8_cache): codes k, v [pages][kv heads][page size][head dim]
    int8 and k_scales, v_scales [pages][kv heads][page size / 16] float32. Keeps the tensors."""

    def __init__(self, k, v, k_scales, v_scales):
        stride, sstride = _rows(k, "k", 4), _rows(k_scales, "k_scales", 3)
        pages, heads, page, dim = k.shape
        _u32("the cache's dimensions", pages, heads, page, dim)
        _need(tuple(v.shape) == tuple(k.shape) and _rows(v, "v", 4) == stride, "k and v must have one layout")
        _need(tuple(k_scales.shape) == (pages, heads, page // 16) and tuple(v_scales.shape) == tuple(k_scales.shape)
              and _rows(v_scales, "v_scales", 3) == sstride, "scales must be [pages][kv heads][page size / 16]")
        for t, name, what in ((k, "int8", "k"), (v, "int8", "v"), (k_scales, "float32", "k_scales"),
                              (v_scales, "float32", "v_scales")):
            _named(t, name, what)
        self.kv_heads, self.head_dim, self.page_size, self.n_pages = heads, dim, page, pages
        self._tensors = (k, v, k_scales, v_scales)
        self._device = _device_of(*self._tensors)
        self._c = _Kv8Cache(C.sizeof(_Kv8Cache), heads, dim, page, pages, 0, k.data_ptr(), v.data_ptr(),
                            k_scales.data_ptr(), v_scales.data_ptr(), stride, sstride)
        self._ref = C.byref(self._c)


class Kv8Batch:
    """The sequences of a call (evl_kv8_batch): page_table [n][pages per sequence], cu [n + 1]
    (first new token of each sequence, then their number) and lens [n] (positions once the new
    tokens are appended), int32 on the device, read when the kernels run; max_new and max_len
    bound the new tokens and the length of a sequence. Keeps the tensors."""

    def __init__(self, page_table, cu, lens, max_new: int, max_len: int):
        n = page_table.shape[0]
        tstride = _rows(page_table, "page_table")
        _named(page_table, "int32", "page_table")
        _flat(cu, n + 1, "int32", "cu")
        _flat(lens, n, "int32", "lens")
        _need(max_new >= 0 and max_len >= 0, "max_new and max_len must not be negative")
        _u32("sequences, max_new, max_len and the page table's stride", n, max_new, max_len, tstride)
        # a table row holds as many entries as its shape says, whatever the stride
        _need(page_table.shape[1] == tstride or n <= 1 or page_table.shape[1] <= tstride, "page_table rows overlap")
        self.n_seqs, self.max_new, self.max_len = n, int(max_new), int(max_len)
        self._width = page_table.shape[1]
        self._tensors = (page_table, cu, lens)
        self._device = _device_of(*self._tensors)
        self._fields = (self.max_new, self.max_len, tstride, page_table.data_ptr(), cu.data_ptr(), lens.data_ptr())
        self._by_total: dict = {}  # number of tokens -> the C descriptor of such a call

    def _of(self, total: int, page_size: int):
        _need(self.max_len <= self._width * page_size, "max_len passes the page table's rows")
        ref = self._by_total.get(total)
        if ref is None:
            if len(self._by_total) >= _MOST_TOTALS:
                self._by_total.clear()
            ref = C.byref(_Kv8Batch(C.sizeof(_Kv8Batch), self.n_seqs, total, *self._fields))
            self._by_total[total] = ref
        return ref


def _heads(t, total: int, dim: int, what: str) -> tuple[int, int]:
    stride = _rows(t, what, 3)
    _need(t.shape[0] == total and t.shape[2] == dim, f"{what} must be [{total}][heads][{dim}]")
    _u32(f"{what}'s tokens and heads", total, t.shape[1])
    return t.shape[1], stride


def kv8_append(cache: Kv8Cache, batch: Kv8Batch, k, v, q=None, q_out=None, rope=None, interleaved: bool = False,
               q_norm=None, k_norm=None, eps: float = 1e-6, err=None, stream: int = 0) -> None:
    """Appends k, v [tokens][kv heads][head dim] to the cache and makes q [tokens][heads][head dim]
    ready into q_out (evl_kv8_append): an RMS norm per head with q_norm / k_norm [head dim]
    float32, then the rotation by rope [positions][rope dim / 2][2] float32 (cos, sin)."""
    key = ("append", cache.kv_heads, cache.head_dim, cache._device, batch._device,
           _layout(k, v, q, q_out, rope, q_norm, k_norm, err))
    plan = _plans.get(key)
    if plan is None:
        _device_of(k, v, q, q_out, rope, q_norm, k_norm, err, known=(cache._device, batch._device))
        _check_err(err)
        plan = _planned(key, _append_plan(cache, k, v, q, q_out, rope, q_norm, k_norm))
    total, kind, kst, vst, qst, ost, heads, rl, rd = plan
    prep = None
    if rope is not None or q_norm is not None or k_norm is not None:
        prep = C.byref(_Kv8Prep(_PREP_BYTES, rd, int(interleaved), rl, _ptr(rope), _ptr(q_norm), _ptr(k_norm), eps, 0))
    _check(runtime.lib().evl_kv8_append(cache._ref, batch._of(total, cache.page_size), prep, kind, k.data_ptr(), kst,
                                        v.data_ptr(), vst, _ptr(q), qst, heads, _ptr(q_out), ost, _ptr(err), stream))


_PREP_BYTES = C.sizeof(_Kv8Prep)


def _append_plan(cache, k, v, q, q_out, rope, q_norm, k_norm):
    total, dim, kind = k.shape[0], cache.head_dim, _kind(k)
    hk, kst = _heads(k, total, dim, "k")
    hv, vst = _heads(v, total, dim, "v")
    _need(hk == cache.kv_heads and hv == hk and v.dtype == k.dtype, "k and v must have the cache's heads and one type")
    heads = qst = ost = rd = rl = 0
    if q is not None or q_out is not None:
        _need(q is not None and q_out is not None, "q and q_out go together")
        heads, qst = _heads(q, total, dim, "q")
        oh, ost = _heads(q_out, total, dim, "q_out")
        _need(oh == heads and q.dtype == k.dtype and q_out.dtype == k.dtype, "q and q_out must have one shape and k's type")
    if rope is not None:
        _named(rope, "float32", "rope")
        _need(len(rope.shape) == 3 and rope.shape[2] == 2 and rope.shape[0] > 0,
              "rope must be [positions][rope dim / 2][2]")
        rl, rd = rope.shape[0], 2 * rope.shape[1]
        _u32("rope's dimensions", rl, rd)
        _need(_rows(rope, "rope", 3) == rd, "rope must be contiguous")
    for t, what in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        if t is not None:
            _flat(t, dim, "float32", what)
    return total, kind, kst, vst, qst, ost, heads, rl, rd


def kv8_attention_workspace(cache: Kv8Cache, batch: Kv8Batch, q) -> int:
    """Bytes of workspace that kv8_attention needs for queries of q's shape (may be 0)."""
    n = C.c_size_t()
    _u32("q's tokens and heads", q.shape[0], q.shape[1])
    _check(runtime.lib().evl_kv8_attention_workspace_bytes(cache._ref, batch._of(q.shape[0], cache.page_size),
                                                           _kind(q), q.shape[1], C.byref(n)))
    return int(n.value)


def kv8_attention(cache: Kv8Cache, batch: Kv8Batch, q, out, scale: float = 0.0, workspace=None, err=None,
                  stream: int = 0) -> None:
    """out [tokens][heads][head dim] = attention of q over the cache, each token up to its own
    position (evl_kv8_attention); scale 0 is 1 / sqrt(head dim). workspace: a device buffer of
    kv8_attention_workspace bytes, 256-byte aligned."""
    _need(scale == 0 or abs(scale) > 2.0 ** -150, "scale must be finite and 0 or a number that f32 holds")
    key = ("attention", cache.head_dim, cache._device, batch._device, _layout(q, out, workspace, err))
    plan = _plans.get(key)
    if plan is None:
        _device_of(q, out, workspace, err, known=(cache._device, batch._device))
        _check_err(err)
        total, kind = q.shape[0], _kind(q)
        heads, qst = _heads(q, total, cache.head_dim, "q")
        oh, ost = _heads(out, total, cache.head_dim, "out")
        _need(oh == heads and out.dtype == q.dtype, "out must have the shape and type of q")
        size = 0
        if workspace is not None:
            _need(len(workspace.shape) == 1 and (workspace.shape[0] <= 1 or workspace.stride()[0] == 1),
                  "workspace must be one contiguous dimension")
            size = workspace.numel() * workspace.element_size()
        plan = _planned(key, (total, kind, heads, qst, ost, size))
    total, kind, heads, qst, ost, size = plan
    _check(runtime.lib().evl_kv8_attention(cache._ref, batch._of(total, cache.page_size), kind, q.data_ptr(), qst, heads,
                                           scale, out.data_ptr(), ost, workspace.data_ptr() if size else None, size,
                                           _ptr(err), stream))
