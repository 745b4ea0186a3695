"""Refusals of the 8-bit serving operators: every bad argument is an error before anything is
launched (no GPU needed: the checks come first)."""
import ctypes as C

import numpy as np
import pytest

import evelyn_b200 as evl
from evelyn_b200 import int8, runtime
from tests import int8_util as ref


class Fake:
    """A tensor's description, at an address that is never read."""

    def __init__(self, shape, dtype="float32", stride=None, at=1 << 20):
        self.shape, self.dtype, self._at = tuple(shape), dtype, at
        self._stride = stride or tuple(int(np.prod(shape[i + 1:])) for i in range(len(shape)))

    def stride(self):
        return tuple(self._stride)

    def data_ptr(self):
        return self._at

    def numel(self):
        return int(np.prod(self.shape))

    def element_size(self):
        return {"float32": 4, "float16": 2, "bfloat16": 2, "int8": 1, "uint8": 1, "int32": 4, "float64": 8}[self.dtype]


def refused(kind, word, fn, *a, **k):
    with pytest.raises(evl.EvelynError) as e:
        fn(*a, **k)
    assert e.value.kind == kind and word in str(e.value), str(e.value)


def test_quantize_rows_refusals():
    x, c, s = Fake((2, 32)), Fake((2, 32), "int8"), Fake((2,))
    bad = lambda kind, word, *a: refused(kind, word, int8.quantize_rows, *a)  # noqa: E731
    bad("Unsupported", "float64", Fake((2, 32), "float64"), c, s)
    bad("InvalidInput", "int8", x, Fake((2, 32), "uint8"), s)
    bad("InvalidInput", "shape", x, Fake((2, 31), "int8"), s)
    bad("InvalidInput", "scales", x, c, Fake((3,)))
    bad("InvalidInput", "float32", x, c, Fake((2,), "float16"))
    bad("InvalidInput", "strided", Fake((2, 32), stride=(64, 2)), c, s)
    bad("InvalidInput", "dimensions", Fake((2, 4, 8)), c, s)
    bad("InvalidInput", "strides", Fake((2, 32), stride=(16, 1)), c, s)
    bad("InvalidInput", "aligned", Fake((2, 32), at=(1 << 20) + 2), c, s)
    bad("InvalidInput", "cols", Fake((2, 0)), Fake((2, 0), "int8"), s)
    bad("InvalidInput", "null", Fake((2, 32), at=0), c, s)


def test_matmul_refusals():
    def call(x=(2, 32), w=(8, 32), y=(2, 8), xs=(2,), ws=(8,), xk={}, wk={}, yk={}, **k):
        int8.matmul(Fake(x, "int8", **xk), Fake(xs), Fake(w, "int8", **wk), Fake(ws), Fake(y, **yk), **k)

    bad = lambda kind, word, **k: refused(kind, word, call, **k)  # noqa: E731
    bad("InvalidInput", "columns", w=(8, 48))
    bad("InvalidInput", "y must be", y=(2, 9))
    bad("InvalidInput", "x_scales", xs=(3,))
    bad("InvalidInput", "w_scales", ws=(9,))
    bad("InvalidInput", "multiples of 16", x=(2, 30), w=(8, 30), wk=dict(stride=(32, 1)))
    bad("InvalidInput", "aligned", xk=dict(at=(1 << 20) + 8))
    bad("InvalidInput", "aligned", yk=dict(at=(1 << 20) + 2))
    bad("InvalidInput", "add must", add=Fake((2, 7)))
    bad("InvalidInput", "add must", add=Fake((2, 8), "float16"))
    bad("InvalidInput", "stride of y", add=Fake((2, 8), stride=(16, 1)))
    bad("InvalidInput", "strides", yk=dict(stride=(4, 1)))
    bad("InvalidInput", "131071", x=(1, 131072), w=(8, 131072), y=(1, 8), xs=(1,))
    bad("InvalidInput", "int32", err=Fake((1,)))
    refused("Unsupported", "activations", int8.matmul, Fake((1, 16), "int8"), Fake((1,)), Fake((1, 16), "int8"), Fake((1,)),
            Fake((1, 1), "int32"))


def _kv(dim=64, page=16, heads=2, pages=4, **k):
    return int8.Kv8Cache(Fake((pages, heads, page, dim), "int8", **k), Fake((pages, heads, page, dim), "int8", **k),
                         Fake((pages, heads, page // 16)), Fake((pages, heads, page // 16)))


def _batch(n=2, width=4, max_new=2, max_len=64):
    return int8.Kv8Batch(Fake((n, width), "int32"), Fake((n + 1,), "int32"), Fake((n,), "int32"), max_new, max_len)


def _rows(heads=2, dim=64, kind="float32", **k):
    return Fake((3, heads, dim), kind, **k)


def test_cache_and_batch_refusals():
    refused("InvalidInput", "scales", int8.Kv8Cache, Fake((4, 2, 32, 64), "int8"), Fake((4, 2, 32, 64), "int8"),
            Fake((4, 2, 1)), Fake((4, 2, 1)))
    refused("InvalidInput", "layout", int8.Kv8Cache, Fake((4, 2, 16, 64), "int8"), Fake((4, 2, 16, 128), "int8"),
            Fake((4, 2, 1)), Fake((4, 2, 1)))
    refused("InvalidInput", "int8", int8.Kv8Cache, Fake((4, 2, 16, 64), "uint8"), Fake((4, 2, 16, 64), "int8"),
            Fake((4, 2, 1)), Fake((4, 2, 1)))
    refused("InvalidInput", "cu", int8.Kv8Batch, Fake((2, 4), "int32"), Fake((2,), "int32"), Fake((2,), "int32"), 1, 8)
    refused("InvalidInput", "int32", int8.Kv8Batch, Fake((2, 4)), Fake((3,), "int32"), Fake((2,), "int32"), 1, 8)
    for k, word in ((dict(dim=96), "head_dim"), (dict(page=48), "page_size")):
        refused("InvalidInput", word, int8.kv8_append, _kv(**k), _batch(), _rows(dim=k.get("dim", 64)), _rows(dim=k.get("dim", 64)))
    refused("InvalidInput", "16-byte", int8.kv8_append, _kv(at=(1 << 20) + 4), _batch(), _rows(), _rows())
    refused("InvalidInput", "page table", int8.kv8_append, _kv(), _batch(max_len=65), _rows(), _rows())
    refused("InvalidInput", "max_new", int8.kv8_append, _kv(), _batch(max_new=0), _rows(), _rows())


def test_append_refusals():
    bad = lambda word, *a, **k: refused("InvalidInput", word, int8.kv8_append, _kv(), _batch(), *a, **k)  # noqa: E731
    bad("heads", _rows(heads=3), _rows(heads=3))
    bad("type", _rows(), _rows(kind="float16"))
    bad("v must be", _rows(), Fake((2, 2, 64)))
    bad("go together", _rows(), _rows(), q=_rows(heads=4))
    bad("one shape", _rows(), _rows(), q=_rows(heads=4), q_out=_rows(heads=2))
    bad("one stride", _rows(), _rows(), q=_rows(heads=4), q_out=_rows(heads=4, stride=(512, 64, 1)))
    bad("16-byte", _rows(at=(1 << 20) + 4), _rows())
    bad("16-byte", _rows(stride=(130, 64, 1)), _rows())
    bad("rope", _rows(), _rows(), rope=Fake((9, 32)))
    bad("rope_dim", _rows(), _rows(), rope=Fake((9, 33, 2)))
    bad("rope_dim", _rows(), _rows(), rope=Fake((9, 64, 2)))
    bad("q_norm", _rows(), _rows(), q_norm=Fake((65,)))
    bad("eps", _rows(), _rows(), k_norm=Fake((64,)), eps=float("nan"))
    refused("Unsupported", "float64", int8.kv8_append, _kv(), _batch(), _rows(kind="float64"), _rows(kind="float64"))


def test_attention_refusals():
    bad = lambda word, *a, **k: refused("InvalidInput", word, int8.kv8_attention, _kv(), _batch(), *a, **k)  # noqa: E731
    bad("multiple of kv_heads", _rows(heads=3), _rows(heads=3))
    bad("shape and type", _rows(heads=4), _rows(heads=2))
    bad("shape and type", _rows(heads=4), _rows(heads=4, kind="float16"))
    bad("16-byte", _rows(heads=4, at=(1 << 20) + 8), _rows(heads=4))
    bad("finite", _rows(heads=4), _rows(heads=4), scale=float("inf"))
    bad("out must", _rows(heads=4), Fake((2, 4, 64)))


def test_struct_sizes_are_checked():
    lib = runtime.lib()
    c, b = runtime._Kv8Cache(), runtime._Kv8Batch()
    n = C.c_size_t()
    assert lib.evl_kv8_attention_workspace_bytes(C.byref(c), C.byref(b), 0, 2, C.byref(n)) == 1
    assert b"struct_size" in lib.evl_last_error()
    assert lib.evl_kv8_attention_workspace_bytes(None, C.byref(b), 0, 2, C.byref(n)) == 1
    assert lib.evl_kv8_append(None, None, None, 0, None, 0, None, 0, None, 0, 0, None, 0, None, None) == 1


def test_host_pointers_are_refused_or_no_device():
    """A pointer that is not device memory (or, here, no device at all) ends as an error."""
    x = np.zeros((2, 32), np.float32)
    c = np.zeros((2, 32), np.int8)
    s = np.zeros(2, np.float32)
    rc = runtime.lib().evl_i8_quantize_rows(0, x.ctypes.data, 32, 2, 32, c.ctypes.data, 32, s.ctypes.data, None)
    assert rc in (1, 6)


def test_plain_forms_agree_with_their_definition():
    """The plain forms that the GPU tests compare with, against the definition in float64."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((5, 300)).astype(np.float32) * 3
    c, s = ref.quantize_rows(x)
    # half a step, plus the rounding of the scale, its reciprocal and the product (3 x 2^-24 of 127 steps)
    assert np.all(np.abs(c * s[:, None].astype(np.float64) - x) <= s[:, None] * (0.5 + 127 * 3 * 2.0 ** -24))
    assert np.all(np.abs(c).max(1) == 127)
    rope = ref.rope_table(50, 32)
    y = ref.make_ready(x[:, None, :64], np.arange(5), rope=rope)
    assert np.allclose((y.astype(np.float64) ** 2).sum(-1), (x[:, None, :64].astype(np.float64) ** 2).sum(-1), rtol=1e-6)
    codes, scales = np.zeros((4, 1, 16, 64), np.int8), np.full((4, 1, 1), np.nan, np.float32)
    rows = rng.standard_normal((40, 1, 64)).astype(np.float32)
    ref.append(codes, scales, np.array([[2, 0, 3]]), [40], [40], rows)
    got = ref.values(codes, scales, np.array([2, 0, 3]), 40)
    assert np.abs(got - rows).max() <= 0.5001 * np.abs(rows).max() / 127


class On(Fake):
    """The same with a device."""

    def __init__(self, shape, device, dtype="float32", **k):
        super().__init__(shape, dtype, **k)
        self.device = device


def test_tensors_of_one_call_are_on_one_device():
    a, b = "cuda:0", "cuda:1"

    def cache(scales=a):
        return int8.Kv8Cache(On((4, 2, 16, 64), a, "int8"), On((4, 2, 16, 64), a, "int8"), On((4, 2, 1), scales), On((4, 2, 1), scales))

    def batch(lens=a, all=a):
        return int8.Kv8Batch(On((2, 4), all, "int32"), On((3,), all, "int32"), On((2,), lens, "int32"), 2, 64)

    bad = lambda fn, *x, **k: refused("InvalidInput", "one device", fn, *x, **k)  # noqa: E731
    bad(int8.quantize_rows, On((2, 32), a), On((2, 32), "cpu", "int8"), On((2,), a))
    bad(int8.matmul, On((2, 32), a, "int8"), On((2,), a), On((8, 32), b, "int8"), On((8,), a), On((2, 8), a))
    bad(int8.matmul, On((2, 32), a, "int8"), On((2,), a), On((8, 32), a, "int8"), On((8,), a), On((2, 8), a),
        err=On((1,), "cpu", "int32"))
    bad(cache, scales="cpu")
    bad(batch, lens=b)
    rows = On((3, 2, 64), a)
    bad(int8.kv8_append, cache(), batch(), rows, On((3, 2, 64), b))
    bad(int8.kv8_append, cache(), batch(b, b), rows, rows)
    bad(int8.kv8_append, cache(), batch(), rows, rows, rope=On((64, 32, 2), "cpu"))
    bad(int8.kv8_attention, cache(), batch(), rows, On((3, 2, 64), "cpu"))
    bad(int8.kv8_attention, cache(), batch(b, b), rows, rows)
    bad(int8.kv8_attention, cache(), batch(), rows, rows, workspace=On((512,), b, "uint8"))


def test_workspace_is_one_run_of_memory():
    for shape, stride in (((8, 64), (128, 1)), ((512,), (2,))):
        refused("InvalidInput", "workspace", int8.kv8_attention, _kv(), _batch(), _rows(heads=4), _rows(heads=4),
                workspace=Fake(shape, "uint8", stride=stride))


def test_a_batch_keeps_few_descriptors():
    b = _batch()
    for total in range(1, 1000):
        b._of(total, 16)
    assert len(b._by_total) <= 64
