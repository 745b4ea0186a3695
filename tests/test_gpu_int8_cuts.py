"""The 8-bit product bit for bit in each of its cuts: CTA pairs, and tiles of 16 to 256 tokens with K whole or
split over a cluster. A cost rule chooses the cut, so a second test sees that the shapes here still reach them all."""
import ctypes as C

import pytest

from evelyn_b200 import int8, runtime
from tests import gpu_util as gu
from tests.test_gpu_int8 import KINDS, dtype, host, same

pytestmark = pytest.mark.gpu

# (tokens of a tile (0: pairs), CTAs that share its K) -> rows, outputs, columns: ragged last tiles everywhere
CUTS = {
    (0, 1): [(2000, 8200, 1000),   # more than three tiles per pair; the second CTA's last rows are all past the end
             (520, 5130, 2000), (300, 8300, 1000), (1024, 4096, 4096)],
    (16, 1): [(5, 24577, 200), (33, 24577, 300)],
    (16, 2): [(2, 300, 1000)],
    (16, 4): [(8, 8203, 4090)],
    (16, 5): [(33, 2050, 4090)],
    (16, 6): [(3, 4101, 4090)],
    (16, 8): [(1, 300, 4090)],
    (32, 1): [(17, 24577, 200)],
    (32, 2): [(33, 8203, 1000)],
    (32, 4): [(17, 8203, 4090)],
    (32, 6): [(17, 4101, 4090)],
    (32, 8): [(65, 1027, 4090)],
    (64, 2): [(33, 8203, 4090)],
    (64, 3): [(33, 5121, 4090)],
    (64, 4): [(60, 4101, 4090)],
    (64, 5): [(129, 1000, 8192)],
    (64, 6): [(33, 2050, 8192)],
    (64, 8): [(33, 100, 25600)],
    (128, 1): [(2049, 8321, 300), (250, 5121, 1000), (257, 24577, 500)],
    (128, 2): [(65, 8201, 1000)],
    (128, 3): [(65, 5120, 4090)],
    (128, 4): [(65, 4100, 4090)],
    (128, 5): [(257, 1000, 4090)],
    (128, 6): [(100, 2050, 4090)],
    (128, 8): [(520, 300, 4090)],
    (256, 1): [(4096, 1025, 1000)],
    (256, 4): [(200, 4100, 8192)],
    (256, 5): [(520, 1000, 25600)],
    (256, 8): [(1030, 300, 25600)],
}
SHAPES = [s for v in CUTS.values() for s in v]


def _operands(rows, out, cols):
    t = gu.torch()
    g = t.Generator("cuda:0").manual_seed(rows + out * 3 + cols * 7)

    def codes(n):
        wide = -(-cols // 16) * 16 + 16  # what lies between the rows is full of large codes
        return t.randint(-128, 128, (n, wide), generator=g, device="cuda:0", dtype=t.int8)[:, :cols]

    def scales(n):
        return t.rand(n, generator=g, device="cuda:0") * 0.1 + 0.001

    return codes(rows), scales(rows), codes(out), scales(out), g


def _want(x, xs, w, ws, add):
    """The sums in 64 bits (exact: below 2^53), then the operator's own f32 operations."""
    t = gu.torch()
    y = (x.to(t.float64) @ w.to(t.float64).T).float() * xs[:, None] * ws
    return y if add is None else y + add.float()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("add", ["none", "other", "in place"])
@pytest.mark.parametrize("rows,out,cols", SHAPES)
def test_matmul_in_every_cut(kind, add, rows, out, cols):
    t = gu.torch()
    x, xs, w, ws, g = _operands(rows, out, cols)
    y = t.full((rows, out + 5), -7.0, dtype=dtype(kind), device="cuda:0")
    err = t.zeros(1, dtype=t.int32, device="cuda:0")
    a = None
    if add != "none":
        a = t.randn((rows, out), generator=g, device="cuda:0").to(dtype(kind))
    want = _want(x, xs, w, ws, a).to(dtype(kind))
    if add == "in place":
        y[:, :out] = a
        a = y[:, :out]
    for _ in range(1 if add == "in place" else 2):
        int8.matmul(x, xs, w, ws, y[:, :out], add=a, err=err)
        assert bool(t.equal(y[:, :out], want))
    assert bool((y[:, out:] == -7.0).all()) and int(err) == 0


def test_the_shapes_reach_every_cut():
    """What the library says of the shapes above, for f32 without an addition (its cost moves some of them)."""
    gu.torch().cuda.init()
    lib = runtime.lib()
    for want, shapes in CUTS.items():
        for rows, out, cols in shapes:
            tokens, split = C.c_uint32(), C.c_uint32()
            assert lib.evl_internal_i8_cut(rows, out, cols, 0, 0, C.byref(tokens), C.byref(split)) == 0
            assert (tokens.value, split.value) == want, (rows, out, cols)
