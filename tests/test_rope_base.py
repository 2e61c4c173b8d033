"""The bases that rotary positions take: any whose angles are f64 numbers at
every position.  Checked ahead of the handles, so this runs anywhere."""
import pytest

from dragonwing_edge_rs_amd import HipError, ops


class NoBackend:
    handle = None


def message(base, rotary=128, sections=(64,), freq=0):
    with pytest.raises(HipError) as e:
        ops.rope_axes(NoBackend(), ops.DTYPE_F32, None, 128, 0, None, 128, 0, None, 3, 1, 128, rotary, sections, freq=freq,
                      base=base)
    return str(e.value)


@pytest.mark.parametrize("base", [5e-324, 1e-320, 1e-308, 1e-306])
def test_bases_whose_angles_are_infinite_are_refused(base):
    assert "base is so small" in message(base)
    assert "base is so small" in message(base, sections=(1, 63), freq=1)  # on the longer axis


@pytest.mark.parametrize("base", [1e-290, 1e-30, 0.5, 1.0, 10000.0, 1.7e308])
def test_other_bases_are_taken(base):
    assert "null backend" in message(base)


def test_the_pairs_decide():
    # a head of one pair has the frequency 1 whatever the base
    assert "null backend" in message(5e-324, rotary=2, sections=(1,))
