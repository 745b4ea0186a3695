"""The 8-bit serving operators (include/evelyn.h) against plain implementations: rows, product
and cache contents bit for bit (both sides do the same f32 operations, each rounded once), the
attention against float64 within a bound derived beside its reference (tests/int8_util.py)."""
import numpy as np
import pytest

import evelyn_b200 as evl
from evelyn_b200 import int8
from tests import gpu_util as gu
from tests import int8_util as ref

pytestmark = pytest.mark.gpu

KINDS = ["f32", "f16", "bf16"]


def dtype(kind):
    t = gu.torch()
    return {"f32": t.float32, "f16": t.float16, "bf16": t.bfloat16}[kind]


def dev(a, kind=None):
    x = gu.to_dev(np.ascontiguousarray(a))
    return x if kind is None else x.to(dtype(kind))


def host(t):
    return t.float().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def bits(a):
    return np.ascontiguousarray(a, np.float32).view(np.uint32)


def same(a, b):
    """Equal bit for bit, any NaN for any NaN."""
    a, b = np.asarray(a, np.float32), np.asarray(b, np.float32)
    return a.shape == b.shape and bool(np.all((bits(a) == bits(b)) | (np.isnan(a) & np.isnan(b))))


# ------------------------------------------------------------------ rows
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (1, 4096, 0), (3, 17, 0), (5, 64, 8), (2, 1000, 24), (33, 5003, 5),
                                           (400, 4096, 0), (301, 8200, 8), (2, 16384, 0), (2, 40000, 0), (1, 12288, 0), (9, 7, 0), (40, 23, 2),
                                           (16, 1023, 0), (3, 110001, 0), (17, 8, 1), (8, 2047, 4)])
def test_quantize_rows(kind, rows, cols, pad):
    t = gu.torch()
    rng = np.random.default_rng(rows * 31 + cols)
    x = rng.standard_normal((rows, cols + pad)).astype(np.float32) * np.exp(rng.standard_normal((rows, 1)) * 4)
    dx = dev(x.astype(np.float32), kind)[:, :cols]
    codes = t.full((rows, cols + pad), 99, dtype=t.int8, device="cuda:0")
    scales = gu.empty_f32(rows)
    int8.quantize_rows(dx, codes[:, :cols], scales)
    want, ws = ref.quantize_rows(host(dx))
    assert same(host(scales), ws)
    assert np.array_equal(host(codes)[:, :cols], want)
    assert np.all(host(codes)[:, cols:] == 99)  # what lies between the rows is left alone


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("at", range(9))
@pytest.mark.parametrize("cols", [1, 5, 8, 16, 41, 300])
def test_quantize_rows_at_every_offset(kind, at, cols):
    """Views that start anywhere in a 16-byte granule, full of larger values around them."""
    t = gu.torch()
    rng = np.random.default_rng(at * 7 + cols)
    x = np.full((5, cols + 24), 1e4, np.float32)
    x[:, at:at + cols] = rng.standard_normal((5, cols))
    dx = dev(x, kind)[:, at:at + cols]
    codes = t.full((5, cols + 5), 99, dtype=t.int8, device="cuda:0")
    scales = gu.empty_f32(5)
    int8.quantize_rows(dx, codes[:, at % 4:at % 4 + cols], scales)
    want, ws = ref.quantize_rows(host(dx))
    assert same(host(scales), ws) and np.array_equal(host(codes)[:, at % 4:at % 4 + cols], want)
    assert np.all(host(codes)[:, :at % 4] == 99) and np.all(host(codes)[:, at % 4 + cols:] == 99)


@pytest.mark.parametrize("cols", [64, 333, 40000, 110000])
def test_quantize_rows_special_values(cols):
    x = np.random.default_rng(1).standard_normal((9, cols)).astype(np.float32)
    x[0] = 0
    x[1] *= np.float32(1e-38)         # below 2^-100: zeros
    x[2, :] = np.float32(2.0 ** -100)  # the smallest group that is kept
    x[3] *= np.float32(1e38 / 8)
    x[4, cols // 2] = np.inf
    x[5, 0] = np.nan
    x[6, -1] = -np.inf
    x[7] = np.float32(-1.0)
    x[8, :] = np.float32(3.4e38)
    t = gu.torch()
    codes, scales = t.empty((9, cols), dtype=t.int8, device="cuda:0"), gu.empty_f32(9)
    int8.quantize_rows(dev(x), codes, scales)
    want, ws = ref.quantize_rows(x)
    assert same(host(scales), ws) and np.array_equal(host(codes), want)
    assert ws[0] == 0 and ws[1] == 0 and ws[2] > 0 and np.isnan(ws[4:7]).all()
    assert not host(codes)[[0, 1, 4, 5, 6]].any()


# ------------------------------------------------------------------ product
def _codes(rng, rows, cols, full=False):
    c = rng.integers(-128, 128, (rows, cols)) if full else np.clip(np.rint(rng.standard_normal((rows, cols)) * 36), -127, 127)
    return c.astype(np.int8)


def _wide(a):
    """int8 rows on 16-byte boundaries, what lies between them full of large codes."""
    t = gu.torch()
    rows, cols = a.shape
    buf = t.full((rows, -(-cols // 16) * 16 + 16), 127, dtype=t.int8, device="cuda:0")
    buf[:, :cols] = dev(a)
    return buf[:, :cols]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("rows,out,cols", [(1, 1, 1), (1, 128, 128), (1, 1000, 4096), (2, 77, 31), (16, 130, 1000),
                                           (17, 256, 512), (33, 300, 2049), (64, 65, 130), (100, 513, 777),
                                           (129, 128, 256), (300, 260, 1040), (513, 1025, 640)])
def test_matmul(kind, add, rows, out, cols):
    t = gu.torch()
    rng = np.random.default_rng(rows + out * 3 + cols * 7)
    x, w = _codes(rng, rows, cols), _codes(rng, out, cols, full=True)
    xs, ws = rng.uniform(0.01, 0.1, rows).astype(np.float32), rng.uniform(0.001, 0.01, out).astype(np.float32)
    a = dev(rng.standard_normal((rows, out)).astype(np.float32), kind) if add else None
    y = t.full((rows, out + 3), -7.0, dtype=dtype(kind), device="cuda:0")
    int8.matmul(_wide(x), dev(xs), _wide(w), dev(ws), y[:, :out], add=a)
    want = ref.matmul(x, xs, w, ws, host(a) if add else None)
    assert same(host(y[:, :out]), host(dev(want, kind)))
    assert np.all(host(y[:, out:]) == -7.0)


@pytest.mark.parametrize("rows,out,cols", [(1, 64, 131071), (300, 129, 20000)])
def test_matmul_largest_sums(rows, out, cols):
    """Codes of -128 (a caller's own) at the longest row: the int32 sum reaches 2^31 - 2^14."""
    t = gu.torch()
    x, w = np.full((rows, cols), -128, np.int8), np.full((out, cols), -128, np.int8)
    one = np.ones(max(rows, out), np.float32)
    y = gu.empty_f32(rows * out).reshape(rows, out)
    int8.matmul(_wide(x), dev(one[:rows]), _wide(w), dev(one[:out]), y)
    assert np.all(host(y) == np.float32(128 * 128 * cols))
    w[:] = 127
    int8.matmul(_wide(x), dev(one[:rows]), _wide(w), dev(one[:out]), y)
    assert np.all(host(y) == np.float32(-128 * 127 * cols))


def test_matmul_residual_in_place_and_tall():
    """The residual added in place, over more tiles than CTAs (both accumulators take turns)."""
    rng = np.random.default_rng(3)
    rows, out, cols = 2000, 3300, 300
    x, w = _codes(rng, rows, cols), _codes(rng, out, cols)
    xs, ws = rng.uniform(0.01, 0.1, rows).astype(np.float32), rng.uniform(0.001, 0.01, out).astype(np.float32)
    y = dev(rng.standard_normal((rows, out)).astype(np.float32), "bf16")
    want = ref.matmul(x, xs, w, ws, host(y))
    int8.matmul(_wide(x), dev(xs), _wide(w), dev(ws), y, add=y)
    assert same(host(y), host(dev(want, "bf16")))


# ------------------------------------------------------------------ the cache
# Sequences without positions or tokens that every batch gets besides, so that its size lets few
# rows take the prompt kernel too.
_EMPTY = [0]


@pytest.fixture(params=[0, 1800], ids=["alone", "wide"])
def width(request):
    _EMPTY[0] = request.param
    yield
    _EMPTY[0] = 0


def _with_empty(table, cu, lens):
    n = _EMPTY[0]
    return (np.concatenate([table, np.full((n, table.shape[1]), -5, np.int32)]),
            np.concatenate([cu, np.full(n, cu[-1], np.int32)]), np.concatenate([lens, np.zeros(n, np.int32)]))


class Kv:
    """A cache with its host mirror, and sequences of given lengths in scattered pages."""

    def __init__(self, rng, kv_heads, dim, page, max_lens, spare=2, fill=True):
        t = gu.torch()
        need = [-(-n // page) for n in max_lens]
        pages = sum(need) + spare
        order = rng.permutation(pages).astype(np.int32)
        self.table = np.full((len(max_lens), max(1, max(need))), -5, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.free = order[at:]
        shape = (pages, kv_heads, page, dim)
        self.k, self.v = (rng.integers(-127, 128, shape).astype(np.int8) for _ in range(2))
        self.ks, self.vs = (np.exp(rng.standard_normal(shape[:2] + (page // 16,)) * 0.5).astype(np.float32) / 100
                            for _ in range(2))
        if not fill:  # pages as they come from an allocator
            self.ks[:], self.vs[:] = np.nan, np.nan
        self.dk, self.dv, self.dks, self.dvs = (dev(a) for a in (self.k, self.v, self.ks, self.vs))
        self.cache = int8.Kv8Cache(self.dk, self.dv, self.dks, self.dvs)
        self.err = t.zeros(1, dtype=t.int32, device="cuda:0")

    def batch(self, lens, new, slack=0):
        cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        table, cu, at = _with_empty(self.table, cu, np.asarray(lens, np.int32))
        return int8.Kv8Batch(dev(table), dev(cu), dev(at), max(1, max(new)) + slack,
                             max(lens) + min(slack, self.table.shape[1] * self.k.shape[2] - max(lens)))

    def same(self):
        return (np.array_equal(host(self.dk), self.k) and np.array_equal(host(self.dv), self.v)
                and same(host(self.dks), self.ks) and same(host(self.dvs), self.vs))


def _append_ref(kv, lens, new, k, v, pos, **prep):
    ref.append(kv.k, kv.ks, kv.table, lens, new, ref.make_ready(k, pos, **prep))
    ref.append(kv.v, kv.vs, kv.table, lens, new, np.asarray(v, np.float32))


def _positions(lens, new):
    return np.concatenate([np.arange(n - m, n) for n, m in zip(lens, new)]).astype(np.int64)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("lens,new", [([1], [1]), ([16, 17, 40], [1, 1, 1]), ([33, 5, 100, 16], [33, 0, 70, 3]),
                                      ([300], [300]), ([70, 3, 64], [9, 2, 48])])
def test_append(kind, dim, page, lens, new):
    rng = np.random.default_rng(dim + page + sum(lens))
    hk, heads = 2, 6
    kv = Kv(rng, hk, dim, page, lens)
    n = sum(new)
    k, v, q = (dev(rng.standard_normal((n + 2, h, dim)).astype(np.float32) * 2, kind) for h in (hk, hk, heads))
    qo = gu.torch().full((n + 2, heads, dim), 5.0, dtype=dtype(kind), device="cuda:0")
    rd = dim // 2 if page == 32 else dim
    inter = page == 64
    rope = ref.rope_table(max(lens) + 3, rd)
    qn, kn = (rng.uniform(0.5, 1.5, dim).astype(np.float32) for _ in range(2)) if page != 16 else (None, None)
    # (two tokens behind the last sequence's: nobody's)
    int8.kv8_append(kv.cache, kv.batch(lens, new, slack=3), k, v, q=q, q_out=qo, rope=dev(rope), interleaved=inter,
                    q_norm=None if qn is None else dev(qn), k_norm=None if kn is None else dev(kn), eps=1e-5, err=kv.err)
    pos = _positions(lens, new)
    prep = dict(eps=1e-5, rope=rope, interleaved=inter)
    _append_ref(kv, lens, new, host(k)[:n], host(v)[:n], pos, norm=kn, **prep)
    assert kv.same()
    want = ref.make_ready(host(q)[:n], pos, norm=qn, **prep)
    assert same(host(qo)[:n], host(dev(want, kind)))
    assert np.all(host(qo)[n:] == 5.0)
    assert int(kv.err) == 0


def test_append_token_by_token_rescales():
    """40 single tokens, each larger than the last: every append raises the scale and moves the
    block's codes; the values stay within one rounding per raise of what was appended."""
    rng = np.random.default_rng(9)
    kv = Kv(rng, 3, 64, 16, [40], fill=False)
    x = rng.standard_normal((40, 3, 64)).astype(np.float32) * np.linspace(1, 8, 40)[:, None, None].astype(np.float32)
    for i in range(40):
        int8.kv8_append(kv.cache, kv.batch([i + 1], [1]), dev(x[i:i + 1]), dev(-x[i:i + 1]), err=kv.err)
        _append_ref(kv, [i + 1], [1], x[i:i + 1], -x[i:i + 1], np.array([i]))
        assert kv.same(), i
    got = ref.values(kv.k, kv.ks, kv.table[0], 40)
    step = np.repeat(kv.ks[kv.table[0][:3]], 16, 2).transpose(0, 2, 1).reshape(-1, 3)[:40]
    assert np.all(np.abs(got - x) <= (0.5 * 16 + 0.01) * step[..., None])


def test_append_again_and_rewound():
    """The same call twice changes nothing; a rewound sequence's block keeps its scale, and starts
    afresh when its first position is written again."""
    rng = np.random.default_rng(10)
    kv = Kv(rng, 2, 128, 32, [64])
    x = rng.standard_normal((50, 2, 128)).astype(np.float32)
    for lens, new, a in (([50], [50], x), ([50], [50], x), ([45], [3], x[:3] * 0.1), ([45], [3], x[:3] * 9), ([40], [8], x[:8] * 0.01)):
        int8.kv8_append(kv.cache, kv.batch(lens, new), dev(a), dev(a), err=kv.err)
        _append_ref(kv, lens, new, a, a, _positions(lens, new))
        assert kv.same()
    assert int(kv.err) == 0


def test_append_values_that_are_not_finite():
    """A block that meets an infinity or a NaN becomes NaN with codes 0 and stays so until its first
    position is written again; other heads and blocks are untouched."""
    rng = np.random.default_rng(11)
    kv = Kv(rng, 2, 64, 16, [48])
    x = rng.standard_normal((48, 2, 64)).astype(np.float32)
    x[20, 0, 3], x[35, 1, 63] = np.inf, np.nan
    x[:16, 1] = 0
    for lens, new, a in (([48], [48], x), ([25], [2], x[:2]), ([17], [1], x[:1]), ([16], [16], x[:16] * 1e-38)):
        int8.kv8_append(kv.cache, kv.batch(lens, new), dev(a), dev(a), err=kv.err)
        _append_ref(kv, lens, new, a, a, _positions(lens, new))
        assert kv.same()


def test_append_skips_what_is_out_of_range():
    """Page ids, lengths and token ranges that do not fit are recorded and skipped; the rest is done."""
    rng = np.random.default_rng(12)
    kv = Kv(rng, 1, 64, 16, [40, 40, 40, 40])
    x = rng.standard_normal((40, 1, 64)).astype(np.float32)
    b = kv.batch([20, 20, 20, 20], [10, 10, 10, 10])
    kv.table[1, 0] = kv.k.shape[0]   # past the pool: the first block is skipped, the second written
    kv.table[2, 1] = -1
    b = int8.Kv8Batch(dev(kv.table), dev(np.array([0, 10, 20, 30, 40], np.int32)),
                      dev(np.array([20, 20, 20, 41], np.int32)), 10, 40)  # the last one: longer than max_len
    int8.kv8_append(kv.cache, b, dev(x), dev(x), err=kv.err)
    assert int(kv.err) == 3
    for a, s in ((kv.k, kv.ks), (kv.v, kv.vs)):
        ref.append(a, s, kv.table[[0]], [20], [10], x[:10])
        ref.append(a, s, kv.table[[1]], [20], [4], x[16:20])
        ref.append(a, s, kv.table[[2]], [16], [6], x[20:26])
    assert kv.same()


# ------------------------------------------------------------------ attention
def _attend(kv, lens, new, q, kind, scale=0.0, out=None, slack=0, stream=0):
    t = gu.torch()
    b = kv.batch(lens, new, slack)
    out = t.full(q.shape, 7.0, dtype=dtype(kind), device="cuda:0") if out is None else out
    n = int8.kv8_attention_workspace(kv.cache, b, q)
    ws = t.full((max(n, 1),), 255, dtype=t.uint8, device="cuda:0")
    int8.kv8_attention(kv.cache, b, q, out, scale=scale, workspace=ws, err=kv.err, stream=stream)
    return out


def _check(kv, lens, new, q, out, kind, scale=None):
    dim, at = q.shape[-1], 0
    scale = scale or 1 / np.sqrt(dim)
    eps = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[kind]
    # the weights of 16-bit types are held in one f16 part (half a step: 2^-11)
    weight_eps = 2.0 ** -11 if kind != "f32" else 0.0
    hq, ho = host(q), host(out).astype(np.float64)
    for s, (n, m) in enumerate(zip(lens, new)):
        k, v = (ref.values(a, b, kv.table[s], n) for a, b in ((kv.k, kv.ks), (kv.v, kv.vs)))
        want, tol = ref.attention(hq[at:at + m], k, v, n - m, scale, weight_eps)
        # the output's own rounding (f16 also has a smallest step, 2^-25 off at most)
        lim = tol[..., None] + eps * np.abs(want) + (2.0 ** -25 if kind == "f16" else 0)
        bad = np.abs(ho[at:at + m] - want) > lim
        assert not bad.any(), (s, n, m, np.abs(ho[at:at + m] - want).max(), tol.max())
        at += m
    return at


@pytest.mark.usefixtures("width")
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 32), (256, 64)])
@pytest.mark.parametrize("heads,hk", [(1, 1), (6, 2), (8, 1), (20, 1), (4, 4)])
@pytest.mark.parametrize("lens,new", [([1], [1]), ([16, 17, 3], [1, 1, 1]), ([150, 0, 700], [1, 0, 1])])
def test_attention_tokens(kind, dim, page, heads, hk, lens, new):
    rng = np.random.default_rng(dim + heads + sum(lens))
    kv = Kv(rng, hk, dim, page, [max(n, 1) for n in lens])
    q = dev(rng.standard_normal((sum(new) + 1, heads, dim)).astype(np.float32) * 2, kind)
    out = _attend(kv, lens, new, q, kind)
    n = _check(kv, lens, new, q, out, kind)
    assert np.all(host(out)[n:] == 7.0) and int(kv.err) == 0


@pytest.mark.usefixtures("width")
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,page", [(64, 32), (128, 16), (256, 32)])
@pytest.mark.parametrize("heads,hk,lens,new", [(4, 2, [5], [5]), (2, 2, [40, 33, 300], [3, 33, 2]), (8, 1, [200], [70]),
                                               (3, 1, [140, 17], [129, 17]), (4, 1, [1000, 64], [40, 1])])
def test_attention_many_tokens(kind, dim, page, heads, hk, lens, new):
    """Drafted tokens and prompts: each token up to its own position."""
    rng = np.random.default_rng(dim + heads * 5 + sum(lens))
    kv = Kv(rng, hk, dim, page, lens)
    q = dev(rng.standard_normal((sum(new), heads, dim)).astype(np.float32) * 2, kind)
    _check(kv, lens, new, q, _attend(kv, lens, new, q, kind, slack=2), kind)
    assert int(kv.err) == 0


@pytest.mark.usefixtures("width")
@pytest.mark.parametrize("lens,new", [([20001, 9], [1, 1]), ([2100, 70], [50, 64])])
@pytest.mark.parametrize("scale", [0.3, -0.2])
def test_attention_long_and_scaled(lens, new, scale):
    rng = np.random.default_rng(5)
    kv = Kv(rng, 2, 128, 64, lens)
    q = dev(rng.standard_normal((sum(new), 8, 128)).astype(np.float32))
    _check(kv, lens, new, q, _attend(kv, lens, new, q, "f32", scale=scale), "f32", scale=np.float32(scale))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,new", [(8, [30, 4]), (16, [40, 1])])
def test_attention_drafts_over_many_positions(kind, dim, heads, new):
    """Positions split over CTAs of the prompt kernel, one row tile and two."""
    rng = np.random.default_rng(dim + heads)
    lens = [3001, 500]
    kv = Kv(rng, 2, dim, 32, lens)
    q = dev(rng.standard_normal((sum(new), heads, dim)).astype(np.float32) * 2, kind)
    _check(kv, lens, new, q, _attend(kv, lens, new, q, kind), kind)
    assert int(kv.err) == 0


@pytest.mark.usefixtures("width")
def test_attention_strided_views():
    """q and out inside larger rows, pages inside a pool that holds other layers."""
    t = gu.torch()
    rng = np.random.default_rng(6)
    kv = Kv(rng, 2, 64, 16, [77])
    pool = t.full((kv.k.shape[0], 3, 2, 2, 16, 64), 1, dtype=t.int8, device="cuda:0")  # [page][layer][K|V][...]
    spool = t.full((kv.k.shape[0], 3, 2, 2, 1), 9.0, device="cuda:0")
    pool[:, 1, 0], pool[:, 1, 1], spool[:, 1, 0], spool[:, 1, 1] = kv.dk, kv.dv, kv.dks, kv.dvs
    kv.cache = int8.Kv8Cache(pool[:, 1, 0], pool[:, 1, 1], spool[:, 1, 0], spool[:, 1, 1])
    qkv = dev(rng.standard_normal((3, 8, 64)).astype(np.float32))
    out = t.zeros((3, 10, 64), device="cuda:0")
    q = qkv[:, 2:6]
    _attend(kv, [77], [3], q, "f32", out=out[:, 4:8])
    _check(kv, [77], [3], q, out[:, 4:8], "f32")
    assert not host(out[:, :4]).any() and not host(out[:, 8:]).any()


@pytest.mark.usefixtures("width")
@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("new", [4, 13])
def test_attention_scales_of_any_size(kind, new):
    """Blocks of zeros (scale 0), huge and tiny value scales side by side, keys of scale 0."""
    rng = np.random.default_rng(7)
    kv = Kv(rng, 1, 128, 16, [160])
    pg = kv.table[0]
    kv.vs[pg[0]], kv.v[pg[0]] = 0, 0
    # (f16 outputs hold up to 65504)
    kv.vs[pg[1]], kv.vs[pg[2]], kv.vs[pg[3]] = (1e-30, 1e20, 1e19) if kind == "f32" else (1e-30, 100, 1e-3)
    kv.ks[pg[4]], kv.k[pg[4]] = 0, 0
    kv.vs[pg[5]] = 0  # codes of any value under a scale of 0 stand for 0
    kv.dv.copy_(dev(kv.v)), kv.dk.copy_(dev(kv.k)), kv.dks.copy_(dev(kv.ks)), kv.dvs.copy_(dev(kv.vs))
    q = dev(rng.standard_normal((new, 4, 128)).astype(np.float32), kind)
    for n in (160, 16, 30, 96):
        _check(kv, [n], [new], q, _attend(kv, [n], [new], q, kind), kind)


@pytest.mark.usefixtures("width")
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n", [40, 90])
def test_attention_ignores_what_it_does_not_see(kind, n):
    """Codes and scales past the length, other pages and hidden blocks may hold anything."""
    rng = np.random.default_rng(8)
    kv = Kv(rng, 2, 64, 32, [100])
    kv.k[kv.free], kv.v[kv.free] = 127, -128
    last = kv.table[0][3]  # positions 96..127: 4 of them seen
    kv.k[last][:, 4:], kv.v[last][:, 4:] = -128, 127
    kv.ks[last, :, 1], kv.vs[last, :, 1] = np.nan, np.nan
    kv.ks[kv.free], kv.vs[kv.free] = np.nan, np.inf
    for d, a in ((kv.dk, kv.k), (kv.dv, kv.v), (kv.dks, kv.ks), (kv.dvs, kv.vs)):
        d.copy_(dev(a))
    q = dev(rng.standard_normal((n, 2, 64)).astype(np.float32), kind)
    _check(kv, [100], [n], q, _attend(kv, [100], [n], q, kind), kind)
    # a block that is not finite reaches the tokens that see it, and no other
    blk = kv.table[0][2]  # positions 64..95
    for s in (kv.dks, kv.dvs):
        keep = s.clone()
        s[int(blk), 0, 0] = float("nan")  # positions 64..79 of kv head 0
        got = host(_attend(kv, [100], [n], q, kind))
        s.copy_(keep)
        see = n - 36  # the tokens before it stand at positions up to 63
        assert np.isnan(got[see:, 0]).all() and np.isfinite(got[:see]).all() and np.isfinite(got[:, 1]).all()


@pytest.mark.usefixtures("width")
@pytest.mark.parametrize("n", [3, 30])
def test_attention_queries_that_are_not_finite(n):
    rng = np.random.default_rng(13)
    kv = Kv(rng, 1, 128, 16, [50])
    q = rng.standard_normal((n, 2, 128)).astype(np.float32)
    q[0, 1, 5], q[2, 0, 100] = np.nan, np.inf
    q[1, 1] = 0
    dq = dev(q)
    got = host(_attend(kv, [50], [n], dq, "f32"))
    assert np.isnan(got[0, 1]).all() and np.isnan(got[2, 0]).all()
    q[0, 1], q[2, 0] = 0, 0
    fine = np.isfinite(got).all(-1)
    assert fine.sum() == 2 * n - 2
    want = host(_attend(kv, [50], [n], dev(q), "f32"))
    assert same(got[fine], want[fine])


@pytest.mark.usefixtures("width")
@pytest.mark.parametrize("many", [False, True])
def test_attention_skips_what_is_out_of_range(many):
    """(many: max_new large enough for the prompt kernel)"""
    rng = np.random.default_rng(14)
    kv = Kv(rng, 1, 64, 16, [64, 64, 64])
    kv.table[1, 2] = kv.k.shape[0] + 7
    t = gu.torch()
    q = dev(rng.standard_normal((3, 2, 64)).astype(np.float32))
    lists = _with_empty(kv.table, np.arange(4, dtype=np.int32), np.array([64, 64, 65], np.int32))
    b = int8.Kv8Batch(*map(dev, lists), 1, 64)
    if many:  # three sequences of one token in a launch for up to 60
        q = dev(rng.standard_normal((60, 2, 64)).astype(np.float32))
        b = int8.Kv8Batch(*map(dev, lists), 60, 64)
    out = t.full(q.shape, 7.0, device="cuda:0")
    ws = t.empty(int8.kv8_attention_workspace(kv.cache, b, q) + 256, dtype=t.uint8, device="cuda:0")
    int8.kv8_attention(kv.cache, b, q, out, workspace=ws, err=kv.err)
    assert int(kv.err) == 3
    got = host(out)
    assert np.all(got[2] == 7.0)  # longer than max_len: left as it was
    kv.err.zero_()
    _check(kv, [64], [1], q[:1], out[:1], "f32")
    k, v = (ref.values(a, b, kv.table[1][[0, 1, 3]], 48) for a, b in ((kv.k, kv.ks), (kv.v, kv.vs)))
    want, tol = ref.attention(host(q)[1:2], k, v, 47, 1 / 8)
    assert np.all(np.abs(got[1:2] - want) <= tol[..., None] + 2.0 ** -24 * np.abs(want))


# ------------------------------------------------------------------ together
class Layer:
    """Attention half of a layer with 8-bit weights: quantise, q / k / v product, append, attention,
    quantise, output product with the residual."""

    def __init__(self, rng, hidden=512, heads=8, hk=2, dim=64, n_seqs=3, max_len=200):
        t = gu.torch()
        self.heads, self.hk, self.dim, self.hidden = heads, hk, dim, hidden
        self.kv = Kv(rng, hk, dim, 16, [max_len] * n_seqs, fill=False)
        self.w1, self.w2 = _codes(rng, (heads + 2 * hk) * dim, hidden), _codes(rng, hidden, heads * dim)
        self.s1 = rng.uniform(0.5, 1, len(self.w1)).astype(np.float32) * 1e-3
        self.s2 = rng.uniform(0.5, 1, len(self.w2)).astype(np.float32) * 1e-3
        self.rope = ref.rope_table(max_len, dim)
        self.norm = rng.uniform(0.5, 1.5, dim).astype(np.float32)
        self.dw1, self.dw2, self.ds1, self.ds2 = dev(self.w1), dev(self.w2), dev(self.s1), dev(self.s2)
        self.drope, self.dnorm = dev(self.rope), dev(self.norm)
        self.n, self.max_len = n_seqs, max_len

    def buffers(self, total):
        t = gu.torch()
        f = lambda *s: t.empty(s, device="cuda:0")  # noqa: E731
        i = lambda *s: t.empty(s, dtype=t.int8, device="cuda:0")  # noqa: E731
        hd = self.heads * self.dim
        return dict(c1=i(total, self.hidden), s1=f(total), qkv=f(total, hd + 2 * self.hk * self.dim),
                    q=f(total, self.heads, self.dim), o=f(total, self.heads, self.dim), c2=i(total, hd), s2=f(total))

    def run(self, x, b, buf, ws, stream=0):
        hd, kd = self.heads * self.dim, self.hk * self.dim
        int8.quantize_rows(x, buf["c1"], buf["s1"], stream=stream)
        int8.matmul(buf["c1"], buf["s1"], self.dw1, self.ds1, buf["qkv"], stream=stream)
        q, k, v = (buf["qkv"][:, a:e].unflatten(1, (-1, self.dim)) for a, e in ((0, hd), (hd, hd + kd), (hd + kd, hd + 2 * kd)))
        int8.kv8_append(self.kv.cache, b, k, v, q=q, q_out=buf["q"], rope=self.drope, q_norm=self.dnorm,
                        k_norm=self.dnorm, eps=1e-6, err=self.kv.err, stream=stream)
        int8.kv8_attention(self.kv.cache, b, buf["q"], buf["o"], workspace=ws, err=self.kv.err, stream=stream)
        int8.quantize_rows(buf["o"].flatten(1), buf["c2"], buf["s2"], stream=stream)
        int8.matmul(buf["c2"], buf["s2"], self.dw2, self.ds2, x, add=x, stream=stream)

    def check(self, x0, buf, x, lens, new):
        """Each stage against its reference on the stage's own inputs."""
        kv, pos = self.kv, _positions(lens, new)
        c1, s1 = ref.quantize_rows(x0)
        assert np.array_equal(host(buf["c1"]), c1) and same(host(buf["s1"]), s1)
        qkv = ref.matmul(c1, s1, self.w1, self.s1)
        assert same(host(buf["qkv"]), qkv)
        hd, kd = self.heads * self.dim, self.hk * self.dim
        q, k, v = (qkv[:, a:e].reshape(len(qkv), -1, self.dim) for a, e in ((0, hd), (hd, hd + kd), (hd + kd, hd + 2 * kd)))
        prep = dict(norm=self.norm, eps=1e-6, rope=self.rope)
        _append_ref(kv, lens, new, k, v, pos, **prep)
        assert kv.same()
        assert same(host(buf["q"]), ref.make_ready(q, pos, **prep))
        _check(kv, lens, new, buf["q"], buf["o"], "f32")
        c2, s2 = ref.quantize_rows(host(buf["o"]).reshape(len(x0), -1))
        assert np.array_equal(host(buf["c2"]), c2) and same(host(buf["s2"]), s2)
        assert same(host(x), ref.matmul(c2, s2, self.w2, self.s2, x0))
        assert int(kv.err) == 0


@pytest.mark.usefixtures("width")
def test_layer_prompt_then_steps():
    """A ragged prompt, then decode steps, through all operators, every stage checked."""
    t = gu.torch()
    rng = np.random.default_rng(20)
    L = Layer(rng)
    lens = [37, 5, 120]
    new = list(lens)
    for step in range(4):
        x0 = rng.standard_normal((sum(new), L.hidden)).astype(np.float32)
        x, b, buf = dev(x0), L.kv.batch(lens, new), L.buffers(sum(new))
        ws = t.empty(int8.kv8_attention_workspace(L.kv.cache, b, buf["q"]) + 1, dtype=t.uint8, device="cuda:0")
        L.run(x, b, buf, ws)
        L.check(x0, buf, x, lens, new)
        new = [1, 1, 1] if step != 1 else [2, 0, 3]
        lens = [n + m for n, m in zip(lens, new)]


@pytest.mark.usefixtures("width")
def test_layer_captured_and_replayed_on_another_stream():
    """One decode step captured into a graph; the lengths, the tokens and the pages' contents move
    on between replays through the same buffers."""
    t = gu.torch()
    rng = np.random.default_rng(21)
    L = Layer(rng, n_seqs=2, max_len=64)
    lens = [15, 30]
    x0 = rng.standard_normal((45, L.hidden)).astype(np.float32)
    x, b, buf = dev(x0), L.kv.batch(lens, lens), L.buffers(45)
    ws = t.empty(int8.kv8_attention_workspace(L.kv.cache, b, buf["q"]) + 1, dtype=t.uint8, device="cuda:0")
    L.run(x, b, buf, ws)
    L.check(x0, buf, x, lens, lens)
    dlens, cu = dev(np.array([16, 31], np.int32)), dev(np.array([0, 1, 2], np.int32))
    b = int8.Kv8Batch(dev(L.kv.table), cu, dlens, 1, 64)
    x, buf = t.zeros((2, L.hidden), device="cuda:0"), L.buffers(2)
    ws = t.empty(int8.kv8_attention_workspace(L.kv.cache, b, buf["q"]) + 1, dtype=t.uint8, device="cuda:0")
    side = t.cuda.Stream()
    t.cuda.synchronize()
    g = t.cuda.CUDAGraph()
    with t.cuda.graph(g, stream=side):
        L.run(x, b, buf, ws, stream=side.cuda_stream)
    for step in range(5):
        lens = [16 + step, 31 + step]
        x0 = rng.standard_normal((2, L.hidden)).astype(np.float32)
        x.copy_(dev(x0))
        dlens.copy_(dev(np.array(lens, np.int32)))
        g.replay()
        gu.sync()
        L.check(x0, buf, x, lens, [1, 1])


def test_outputs_do_not_depend_on_the_batch_they_run_in():
    """A sequence's cache contents are the same whichever way its tokens were split over calls
    that start at block boundaries, and whoever else was in the call."""
    rng = np.random.default_rng(22)
    x = rng.standard_normal((80, 2, 64)).astype(np.float32)
    whole, parts = (Kv(np.random.default_rng(1), 2, 64, 16, [80, 80]) for _ in range(2))
    int8.kv8_append(whole.cache, whole.batch([80, 80], [80, 0]), dev(x), dev(x))
    for a, e in ((0, 32), (32, 48), (48, 80)):
        y = np.concatenate([x[a:e], x[:7]])
        int8.kv8_append(parts.cache, parts.batch([e, 7], [e - a, 7]), dev(y), dev(y))
    rows = whole.table[0]
    for d in ("dk", "dv", "dks", "dvs"):
        assert np.array_equal(host(getattr(whole, d))[rows], host(getattr(parts, d))[rows])


@pytest.mark.usefixtures("width")
def test_calls_on_several_streams_at_once():
    """Prompts of few steps on four streams, each with its own output and workspace: nothing waits in vain
    for a product that has already ended, and the results are those of a call alone."""
    t = gu.torch()
    rng = np.random.default_rng(15)
    lens, new = [200, 90, 130], [30, 90, 12]
    kv = Kv(rng, 2, 128, 32, lens)
    q = t.randn(sum(new), 8, 128, generator=t.Generator("cuda:0").manual_seed(3), device="cuda:0").to(t.bfloat16)
    want = host(_attend(kv, lens, new, q, "bf16"))
    b = kv.batch(lens, new)
    streams = [t.cuda.Stream() for _ in range(4)]
    outs = [t.full(q.shape, 7.0, dtype=q.dtype, device="cuda:0") for _ in streams]
    spaces = [t.empty(max(1, int8.kv8_attention_workspace(kv.cache, b, q)), dtype=t.uint8, device="cuda:0") for _ in streams]
    t.cuda.synchronize()
    for _ in range(100):
        for s, o, w in zip(streams, outs, spaces):
            int8.kv8_attention(kv.cache, b, q, o, workspace=w, err=kv.err, stream=s.cuda_stream)
    t.cuda.synchronize()
    assert int(kv.err) == 0
    assert all(same(host(o), want) for o in outs)


@pytest.mark.usefixtures("width")
def test_cache_offsets_past_32_bits():
    """The same sequences in a small cache and at the end of one of 4.6 GB for K and for V: append and attention
    give the same bits."""
    t = gu.torch()
    rng = np.random.default_rng(16)
    lens, new, pages = [100, 70], [40, 1], 70000
    kv = Kv(rng, 8, 128, 64, lens, spare=0)
    n = kv.k.shape[0]
    big = [t.empty((pages, 8, 64, 128), dtype=t.int8, device="cuda:0") for _ in range(2)]
    bigs = [t.empty((pages, 8, 4), device="cuda:0") for _ in range(2)]
    for a, b in zip(big + bigs, (kv.dk, kv.dv, kv.dks, kv.dvs)):
        a[pages - n:] = b
    total = sum(new)
    k, v, q = (dev(rng.standard_normal((total, h, 128)).astype(np.float32), "bf16") for h in (8, 8, 16))
    got = []
    for cache, shift in ((kv.cache, 0), (int8.Kv8Cache(*big, *bigs), pages - n)):
        table, cu, at = _with_empty(kv.table + shift, np.array([0, 40, 41], np.int32), np.array(lens, np.int32))
        b = int8.Kv8Batch(dev(table), dev(cu), dev(at), 40, 100)
        int8.kv8_append(cache, b, k, v, err=kv.err)
        out = t.zeros_like(q)
        ws = t.empty(int8.kv8_attention_workspace(cache, b, q) + 1, dtype=t.uint8, device="cuda:0")
        int8.kv8_attention(cache, b, q, out, workspace=ws, err=kv.err)
        got.append(host(out))
    assert int(kv.err) == 0 and same(got[0], got[1])
    for a, b in zip(big + bigs, (kv.dk, kv.dv, kv.dks, kv.dvs)):
        assert same(host(a[pages - n:]), host(b))


def test_rows_more_than_32_bits_apart():
    t = gu.torch()
    rng = np.random.default_rng(17)
    far = (1 << 32) + 64
    pool = t.empty(2 * far + 4096, dtype=t.int8, device="cuda:0")
    x = rng.standard_normal((3, 300)).astype(np.float32)
    dx = t.as_strided(pool.view(t.float32), (3, 300), (far // 4, 1))
    codes = t.as_strided(pool, (3, 300), (far, 1), 2048)
    y = t.as_strided(pool.view(t.float32), (3, 20), (far // 4, 1), 800)
    dx.copy_(dev(x))
    scales = t.empty(3, device="cuda:0")
    int8.quantize_rows(dx, codes, scales)
    want, ws = ref.quantize_rows(x)
    assert same(host(codes.contiguous()), want) and same(host(scales), ws)
    w, s = _codes(rng, 20, 300), rng.uniform(0.5, 1, 20).astype(np.float32)
    int8.matmul(codes, scales, _wide(w), dev(s), y)
    z = t.empty((3, 20), device="cuda:0")
    int8.matmul(_wide(want), dev(ws), _wide(w), dev(s), z)
    assert same(host(y.contiguous()), host(z))


@pytest.mark.usefixtures("width")
def test_attention_shared_pages():
    """Sequences that share a prefix's pages, and a page that stands twice in one sequence."""
    rng = np.random.default_rng(18)
    kv = Kv(rng, 2, 64, 16, [90, 90, 90])
    kv.table[1, :3] = kv.table[0, :3]
    kv.table[2, 4] = kv.table[2, 1]
    lens, new = [90, 75, 90], [1, 20, 30]
    q = dev(rng.standard_normal((51, 4, 64)).astype(np.float32))
    _check(kv, lens, new, q, _attend(kv, lens, new, q, "f32"), "f32")
    assert int(kv.err) == 0


@pytest.mark.parametrize("captured", [False, True])
def test_calls_see_what_the_stream_wrote_before(captured):
    """Calls between other kernels of the stream that write their inputs, read their outputs and write those inputs
    again: each sees its own round's values (launches begin early, their reads and writes do not)."""
    t = gu.torch()
    rng = np.random.default_rng(19)
    base = dev(rng.integers(-5, 6, (64, 2048)).astype(np.float32))
    w, s = dev(_codes(rng, 512, 2048)), t.ones(512, device="cuda:0")
    x, y, acc = t.empty_like(base), t.empty((64, 512), device="cuda:0"), t.zeros((64, 512), device="cuda:0")
    codes, scales = t.empty((64, 2048), dtype=t.int8, device="cuda:0"), t.empty(64, device="cuda:0")
    n = 24

    def rounds(stream):
        for i in range(n):
            t.mul(base, float(1 + i % 5), out=x)
            int8.quantize_rows(x, codes, scales, stream=stream)
            int8.matmul(codes, scales, w, s, y, stream=stream)
            acc.add_(y)

    stream = t.cuda.Stream()
    if captured:
        rounds(0)  # (kernels loaded before the capture)
        t.cuda.synchronize()
        g = t.cuda.CUDAGraph()
        with t.cuda.graph(g, stream=stream):
            rounds(stream.cuda_stream)
        acc.zero_()
        g.replay()
    else:
        with t.cuda.stream(stream):
            rounds(stream.cuda_stream)
    t.cuda.synchronize()
    want = t.zeros_like(acc)
    for i in range(n):
        c, z = ref.quantize_rows(host(base) * np.float32(1 + i % 5))
        p = c.astype(np.int64) @ host(w).astype(np.int64).T
        want += dev((p.astype(np.float32) * z[:, None]).astype(np.float32))
    assert same(host(acc), host(want))


def test_calls_of_no_tokens():
    t = gu.torch()
    kv = Kv(np.random.default_rng(2), 1, 64, 16, [16])
    none = t.empty((0, 1, 64), device="cuda:0")
    b = kv.batch([16], [0])
    int8.kv8_append(kv.cache, b, none, none, err=kv.err)
    int8.kv8_attention(kv.cache, b, none, none)
    int8.quantize_rows(t.empty((0, 8), device="cuda:0"), t.empty((0, 8), dtype=t.int8, device="cuda:0"), gu.empty_f32(0))
    int8.matmul(t.empty((0, 16), dtype=t.int8, device="cuda:0"), gu.empty_f32(0),
                t.zeros((4, 16), dtype=t.int8, device="cuda:0"), gu.empty_f32(4), t.empty((0, 4), device="cuda:0"))
    gu.sync()
    assert kv.same() and int(kv.err) == 0
