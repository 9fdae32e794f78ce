"""The axes of rotary pairs, on the host. CPU only."""
import pytest

import qw_amd
from qw_amd.paged import _axes


def test_sections_of_whole_floats():
    """Sections that are whole numbers count as such, whatever their type; others are refused."""
    _axes.cache_clear()
    for sections in ((2.0, 0.0, 1.0), (2, 0, 1)):
        assert _axes(sections, False) == bytes([0, 0, 2])
        assert _axes(sections, True) == bytes([0, 0, 2])
    for sections in ((1.5, 1), (2, -1), (), (0, 0), (300,)):
        with pytest.raises(qw_amd.QwError):
            _axes(sections, False)
