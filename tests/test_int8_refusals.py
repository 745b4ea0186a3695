"""More calls of the 8-bit serving operators that are refused before anything is launched (no GPU needed)."""
import pytest

from evelyn_b200 import EvelynError, int8
from tests.test_int8_args import Fake, _batch, _kv, _rows, refused

FAR = 1 << 32


def test_sizes_that_do_not_fit_32_bits():
    """The C ABI takes them in 32 bits: cut to those they would pass every check as small sizes."""
    bad = lambda fn, *a, **k: refused("InvalidInput", "2^32", fn, *a, **k)  # noqa: E731
    bad(int8.quantize_rows, Fake((1, FAR + 64)), Fake((1, FAR + 64), "int8"), Fake((1,)))
    bad(int8.quantize_rows, Fake((FAR + 1, 32)), Fake((FAR + 1, 32), "int8"), Fake((FAR + 1,)))
    bad(int8.matmul, Fake((2, 32), "int8"), Fake((2,)), Fake((FAR + 8, 32), "int8"), Fake((FAR + 8,)), Fake((2, FAR + 8)))
    bad(int8.matmul, Fake((FAR + 2, 32), "int8"), Fake((FAR + 2,)), Fake((8, 32), "int8"), Fake((8,)), Fake((FAR + 2, 8)))
    bad(int8.matmul, Fake((2, FAR + 32), "int8"), Fake((2,)), Fake((8, FAR + 32), "int8"), Fake((8,)), Fake((2, 8)))
    bad(_kv, pages=FAR + 4)
    bad(_kv, heads=FAR + 2)
    bad(_batch, max_new=FAR + 1)
    bad(_batch, width=FAR + 4, max_len=FAR + 1)
    bad(int8.Kv8Batch, Fake((2, 4), "int32", stride=(FAR + 4, 1)), Fake((3,), "int32"), Fake((2,), "int32"), 2, 64)
    bad(int8.kv8_append, _kv(), _batch(), _rows(), _rows(), q=_rows(heads=FAR + 2), q_out=_rows(heads=FAR + 2))
    bad(int8.kv8_append, _kv(), _batch(), _rows(), _rows(), rope=Fake((FAR + 64, 32, 2)))
    bad(int8.kv8_attention, _kv(), _batch(), _rows(heads=FAR + 2), _rows(heads=FAR + 2))
    bad(int8.kv8_attention_workspace, _kv(), _batch(), _rows(heads=FAR + 2))


def test_a_rope_table_without_positions():
    """Its address is null, which the C ABI takes for no rotation at all."""
    refused("InvalidInput", "rope", int8.kv8_append, _kv(), _batch(), _rows(), _rows(), rope=Fake((0, 32, 2), at=0))


@pytest.mark.parametrize("scale", [1e-60, -1e-60, 2.0 ** -150, float("nan")])
def test_a_scale_that_f32_does_not_hold(scale):
    """Rounded to 0 it would stand for 1 / sqrt(head dim)."""
    refused("InvalidInput", "scale", int8.kv8_attention, _kv(), _batch(), _rows(heads=4), _rows(heads=4), scale=scale)


def test_the_smallest_scales_that_f32_holds_are_taken():
    """(up to the device: the arguments themselves are fine)"""
    for scale in (1e-40, -1.4e-45):
        with pytest.raises(EvelynError) as e:
            int8.kv8_attention(_kv(), _batch(), _rows(heads=4), _rows(heads=4), scale=scale)
        assert "scale" not in str(e.value)


def _product(add_at, y_at=1 << 20, rows=4, out=8, add_stride=24, y_stride=24, kind="float32"):
    int8.matmul(Fake((rows, 32), "int8"), Fake((rows,)), Fake((out, 32), "int8"), Fake((out,)),
                Fake((rows, out), kind, stride=(y_stride, 1), at=y_at),
                add=Fake((rows, out), kind, stride=(add_stride, 1), at=add_at))


@pytest.mark.parametrize("off", [-7, -1, 1, 7, 17, 23, 24, 25, -24, 72, 79, -72, -79])
def test_additions_that_overlap_other_outputs(off):
    refused("InvalidInput", "overlap", _product, (1 << 20) + 4 * off)


def test_an_addition_that_overlaps_a_single_row():
    refused("InvalidInput", "overlap", _product, (1 << 20) + 28, rows=1, add_stride=400)


@pytest.mark.parametrize("off", [8, 12, 16, -8, -16, 80, 100, -80, 32, 88])
def test_additions_beside_the_outputs_are_taken(off):
    """(up to the device) other columns of the same buffer, or memory apart"""
    with pytest.raises(EvelynError) as e:
        _product((1 << 20) + 4 * off)
    assert "overlap" not in str(e.value)


@pytest.mark.parametrize("off", [-16, 16, 64, 512, -512])
def test_queries_made_ready_over_other_queries(off):
    """d_q_out may be d_q itself; shifted by less than a row, one warp would write what another has yet to read."""
    q, o = (_rows(heads=4, stride=(512, 64, 1), at=at) for at in (1 << 20, (1 << 20) + 4 * off))
    refused("InvalidInput", "overlap", int8.kv8_append, _kv(), _batch(), _rows(), _rows(), q=q, q_out=o)


def test_queries_made_ready_beside_the_others_are_taken():
    with pytest.raises(EvelynError) as e:
        q, o = (_rows(heads=4, stride=(512, 64, 1), at=at) for at in (1 << 20, (1 << 20) + 4 * 256))
        int8.kv8_append(_kv(), _batch(), _rows(), _rows(), q=q, q_out=o)
    assert "overlap" not in str(e.value)
