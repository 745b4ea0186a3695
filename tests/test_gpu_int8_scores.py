"""Attention over the 8-bit cache where scores are far apart or large: heads whose weight lies almost
whole on one position, scores of any size, and blocks that are not finite beside such positions. Both
attention kernels, against float64 within bounds that have no term in the number of positions."""
import numpy as np
import pytest

from evelyn_b200 import int8
from tests import gpu_util as gu
from tests import int8_util as ref
from tests.test_gpu_int8 import KINDS, Kv, _attend, dev, host, width  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu

# (tokens of a sequence: one takes the token kernel, 16 beside many empty sequences the prompt kernel)
KERNELS = pytest.mark.parametrize("tokens", [1, 16])


def _wide(tokens):
    """Sequences without tokens besides, so that few rows take the prompt kernel."""
    import tests.test_gpu_int8 as t
    t._EMPTY[0] = 1800 if tokens > 1 else 0


@pytest.fixture(autouse=True)
def _alone():
    yield
    _wide(1)


def _put(kv, codes_k, codes_v, ks, vs):
    """One sequence's positions into the cache and its host mirror: codes [n][dim], scales [n / 16]."""
    n, page = len(codes_k), kv.k.shape[2]
    for p in range(-(-n // page)):
        at, rows = kv.table[0][p], min(page, n - p * page)
        kv.k[at, 0, :rows], kv.v[at, 0, :rows] = codes_k[p * page:p * page + rows], codes_v[p * page:p * page + rows]
        for b in range(page // 16):
            i = p * page // 16 + b
            if i < len(ks):
                kv.ks[at, 0, b], kv.vs[at, 0, b] = ks[i], vs[i]
    for d, a in ((kv.dk, kv.k), (kv.dv, kv.v), (kv.dks, kv.ks), (kv.dvs, kv.vs)):
        d.copy_(dev(a))


def _bound(q, k, v, first, scale, kind):
    """The attention and how far an implementation that holds its sums in f32 may be from it."""
    q = q.astype(np.float64)
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    half = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[kind]
    for i in range(q.shape[0]):
        n = max(0, first + i + 1)
        for h in range(q.shape[1]):
            x = k[:n] @ q[i, h] * scale
            w = np.exp(x - x.max())
            w /= w.sum()
            out[i, h] = w @ v[:n]
            # scores: q in fixed point (half a step of 2^-21 of the row's largest), or its f16 products summed in f32
            # with a cut of at most 2^-23 of the terms' sizes after every 16 dims; seven roundings of the score
            terms = (np.abs(k[:n]) @ np.abs(q[i, h])).max() * abs(scale)
            dx = np.abs(q[i, h]).max() * 2.0 ** -22 * np.abs(k[:n]).sum(1).max() * abs(scale) + 7 * 2.0 ** -24 * np.abs(x).max()
            if kind != "f32":
                dx += (q.shape[2] / 16 + 1) * 2.0 ** -23 * terms
            # weights: exp2 2^-22, the value scale 2^-22, and for the 16-bit types 16 bits (2^-15); sums of the
            # tensor cores: cut off at most 2^-23 each, at most 128 in a row (f32) or 2048 (16 bits) before they are
            # added rounded to nearest (unbiased: 2^-19 is four times what 30000 of them reach)
            dw = 2.0 ** -21 + 2.0 ** -19 + (2.0 ** -16 if kind == "f32" else 2.0 ** -15 + 2.0 ** -12)
            tol[i, h] = (2 * dx + dw) * (w @ np.abs(v[:n])) + 1e-30 + half * np.abs(out[i, h])
            if kind == "f16":
                tol[i, h] += 2.0 ** -25
    return out, tol


def _compare(kv, n, tokens, q, kind, scale=0.0):
    got = host(_attend(kv, [n], [tokens], q, kind, scale=scale)).astype(np.float64)
    k, v = (ref.values(a, b, kv.table[0], n)[:, 0] for a, b in ((kv.k, kv.ks), (kv.v, kv.vs)))
    want, tol = _bound(host(q), k, v, n - tokens, scale or 1 / np.sqrt(q.shape[-1]), kind)
    assert int(kv.err) == 0
    assert np.isfinite(got).all()
    off = np.abs(got - want) / tol
    assert off.max() <= 1, (off.max(), np.abs(got - want).max(), np.abs(want).max())


# ------------------------------------------------------------------ large scores
@KERNELS
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("top", [40, 60, 140, 210, 300, 1e4])
def test_attention_large_scores(tokens, kind, dim, zeros, top):
    """Scores up to `top` (in nats), a few nats apart, under ordinary value scales, a block of zeros beside them, either
    sign of the scale."""
    _wide(tokens)
    rng = np.random.default_rng(int(top) + dim)
    n = 100
    kv = Kv(rng, 1, dim, 16, [n])
    sign = rng.choice([-1, 1], dim)
    level = np.full(n, 100)
    level[rng.permutation(n)[:20]] = 126
    level[rng.permutation(n)[:8]] = 127
    v = rng.integers(-127, 128, (n, dim))
    vs = np.full(7, 1 / 40, np.float32)
    if zeros:
        v[32:48], vs[2] = 0, 0
        level[40] = 127
    _put(kv, level[:, None] * sign, v, np.full(7, 1 / 40, np.float32), vs)
    for scale in (0.25, -0.25):
        x = sign * (top / (127 / 40) / dim / scale)  # q . k of level 127 is `top`
        q = dev(np.tile(x, (tokens, 4, 1)).astype(np.float32), kind)
        _compare(kv, n, tokens, q, kind, scale=scale)


# ------------------------------------------------------------------ one position dominates
def _levels(rng, n, dim, nats, low, high):
    """Keys whose scores lie `nats` under the largest, at level 127, and a query for them (scale 1 / sqrt(dim))."""
    sign = rng.choice([-1, 1], dim)
    top = 2.0 * nats
    x = sign * (top / (127 / 40) / np.sqrt(dim))
    return sign, rng.integers(low, high, n), x


@KERNELS
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,n", [(64, 200), (128, 333), (256, 200), (64, 16384)])
@pytest.mark.parametrize("nats", [8, 12, 16, 20, 25, 40])
def test_attention_one_position_dominates(tokens, kind, dim, n, nats):
    """Nearly all weight on one position whose value is zero: the output is made of the others, whose weights are
    e^-nats of it."""
    _wide(tokens)
    rng = np.random.default_rng(nats * 7 + n + dim)
    kv = Kv(rng, 1, dim, 32, [n])
    sign, level, x = _levels(rng, n, dim, nats, 60, 67)
    sink = 5
    level[sink] = 127
    v = rng.integers(-127, 128, (n, dim))
    v[sink] = 0
    blocks = -(-n // 16)
    _put(kv, level[:, None] * sign, v, np.full(blocks, 1 / 40, np.float32), rng.uniform(0.5, 1.5, blocks).astype(np.float32) / 40)
    q = dev(np.tile(x, (tokens, 4, 1)).astype(np.float32), kind)
    _compare(kv, n, tokens, q, kind)


@KERNELS
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("v_scale,others", [(1e-25, 1e-25), (1e30, 1e30), (1e-30, 1.0), (1e30, 1e-25), (1e36, 1e36), (1e-30, 1e-30)])
def test_attention_value_scales_at_the_ends(tokens, kind, dim, v_scale, others):
    """The same with values near the ends of f32's range, alone and beside ordinary ones."""
    if kind == "f16" and max(v_scale, others) > 100:
        return  # (f16 outputs end at 65504)
    _wide(tokens)
    rng = np.random.default_rng(int(abs(np.log10(v_scale))) + dim)
    n = 128
    kv = Kv(rng, 1, dim, 16, [n])
    sign, level, x = _levels(rng, n, dim, 6, 50, 100)
    v = rng.integers(-127, 128, (n, dim))
    vs = np.full(8, others, np.float32)
    vs[3] = vs[6] = v_scale
    _put(kv, level[:, None] * sign, v, np.full(8, 1 / 40, np.float32), vs)
    q = dev(np.tile(x, (tokens, 4, 1)).astype(np.float32), kind)
    _compare(kv, n, tokens, q, kind)


@KERNELS
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("loud", [30, 1000])
def test_attention_loud_channel_in_q(tokens, kind, dim, loud):
    """One channel of q many times larger than the others, against keys that are small there."""
    _wide(tokens)
    rng = np.random.default_rng(loud + dim)
    n = 300
    kv = Kv(rng, 1, dim, 32, [n])
    k, v = rng.integers(-127, 128, (n, dim)), rng.integers(-127, 128, (n, dim))
    k[:, 7] = rng.integers(-1, 2, n)
    _put(kv, k, v, np.full(19, 1 / 60, np.float32), np.full(19, 1 / 40, np.float32))
    q = rng.standard_normal((tokens, 4, dim)).astype(np.float32)
    q[..., 7] *= loud
    _compare(kv, n, tokens, dev(q, kind), kind)


@KERNELS
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("value", [np.nan, np.inf])
@pytest.mark.parametrize("nats", [5, 60, 120])
def test_attention_block_that_is_not_finite_far_below_the_maximum(tokens, kind, dim, value, nats):
    """A value scale that is not finite reaches every token that sees its block, however small the weights there, and
    no token that does not."""
    _wide(tokens)
    rng = np.random.default_rng(nats + dim)
    n = max(60, 48 + tokens)  # all tokens see the block
    kv = Kv(rng, 1, dim, 16, [n])
    sign, level, x = _levels(rng, n, dim, nats, 60, 67)
    level[2] = 127
    vs = np.full(4, 1 / 40, np.float32)
    vs[3] = value  # positions 48 and on
    _put(kv, level[:, None] * sign, rng.integers(-127, 128, (n, dim)), np.full(4, 1 / 40, np.float32), vs)
    q = dev(np.tile(x, (tokens, 4, 1)).astype(np.float32), kind)
    assert not np.isfinite(host(_attend(kv, [n], [tokens], q, kind))).any()
    for last in (48, 48 + tokens // 2):  # the last token's length: half of the tokens see the block
        got = host(_attend(kv, [last], [tokens], q, kind))
        see = last - 48
        assert np.isfinite(got[:tokens - see]).all() and not np.isfinite(got[tokens - see:]).any()


# ------------------------------------------------------------------ long sums
@KERNELS
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,n", [(64, 30001), (128, 30001), (256, 30001), (128, 5000), (64, 70001)])
def test_attention_values_of_one_sign_over_many_positions(tokens, kind, dim, n):
    """Sums that only grow: a cut instead of a rounding at each addition would show as a bias with the length."""
    import tests.test_gpu_int8 as t
    t._EMPTY[0] = 1800  # (many sequences: one chunk of positions per row)
    rng = np.random.default_rng(dim)
    kv = Kv(rng, 1, dim, 64, [n])
    sign, level, x = _levels(rng, n, dim, 1, 90, 128)
    v = rng.integers(64, 128, (n, dim))
    blocks = -(-n // 16)
    _put(kv, level[:, None] * sign, v, np.full(blocks, 1 / 40, np.float32), np.full(blocks, 1 / 40, np.float32))
    q = dev(np.tile(x, (tokens, 4, 1)).astype(np.float32), kind)
    _compare(kv, n, tokens, q, kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("sign", [1, -1])
def test_attention_long_chunks_joined_captured_and_replayed(kind, dim, sign):
    """Forty sequences over the same pages: chunks so long that their sums leave tensor memory, several of them joined.
    Eager, captured and replayed twice over a workspace full of NaN: the same bits for all sequences."""
    t = gu.torch()
    rng = np.random.default_rng(dim)
    n, tokens, seqs = 32773, 16, 40
    kv = Kv(rng, 1, dim, 64, [n])
    signs, level, x = _levels(rng, n, dim, 3, 60, 128)
    v = rng.integers(32, 128, (n, dim)) * sign
    blocks = -(-n // 16)
    _put(kv, level[:, None] * signs, v, np.full(blocks, 1 / 40, np.float32), rng.uniform(0.5, 1.5, blocks).astype(np.float32) / 40)
    one = np.tile(x, (tokens, 4, 1)) * rng.uniform(0.3, 1, (tokens, 4, 1))
    q = dev(np.tile(one, (seqs, 1, 1)).astype(np.float32), kind)
    b = int8.Kv8Batch(dev(np.tile(kv.table, (seqs, 1))), dev(np.arange(seqs + 1, dtype=np.int32) * tokens),
                      dev(np.full(seqs, n, np.int32)), tokens, n)
    out = t.full(q.shape, 7.0, dtype=q.dtype, device="cuda:0")
    ws = t.full((int8.kv8_attention_workspace(kv.cache, b, q),), 255, dtype=t.uint8, device="cuda:0")
    int8.kv8_attention(kv.cache, b, q, out, workspace=ws, err=kv.err)
    got = host(out)
    k, w = (ref.values(a, s, kv.table[0], n)[:, 0] for a, s in ((kv.k, kv.ks), (kv.v, kv.vs)))
    want, tol = _bound(host(q)[:tokens], k, w, n - tokens, 1 / np.sqrt(dim), kind)
    assert int(kv.err) == 0 and (np.abs(got[:tokens] - want) / tol).max() <= 1
    got = got.reshape(seqs, tokens, 4, dim)
    assert np.array_equal(got, np.broadcast_to(got[:1], got.shape))
    side, g = t.cuda.Stream(), t.cuda.CUDAGraph()
    t.cuda.synchronize()
    with t.cuda.graph(g, stream=side):
        int8.kv8_attention(kv.cache, b, q, out, workspace=ws, err=kv.err, stream=side.cuda_stream)
    for _ in range(2):
        out.fill_(7.0)
        ws.fill_(255)
        g.replay()
        gu.sync()
        assert np.array_equal(host(out).reshape(got.shape), got)


@KERNELS
@pytest.mark.parametrize("kind", KINDS)
def test_attention_scales_of_minus_zero(tokens, kind):
    """A value scale of -0 is a scale of 0: its positions count in the weights and add nothing, here nearly all of them."""
    _wide(tokens)
    rng = np.random.default_rng(3)
    n, dim = 100, 128
    kv = Kv(rng, 1, dim, 16, [n])
    sign, level, x = _levels(rng, n, dim, 60, 60, 67)
    level[20] = 127
    vs = np.full(7, 1 / 40, np.float32)
    vs[1] = -0.0
    _put(kv, level[:, None] * sign, rng.integers(-127, 128, (n, dim)), np.full(7, 1 / 40, np.float32), vs)
    q = dev(np.tile(x, (tokens, 4, 1)).astype(np.float32), kind)
    _compare(kv, n, tokens, q, kind)
