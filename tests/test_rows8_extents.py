"""Extents at which a descriptor's checks could go wrong themselves."""
import ctypes

import pytest

from pto_einsum import abi, runtime

INVALID, BOUNDS, UNSUPPORTED = -1, -2, -3


def desc(**kw):
    return abi.RowsDesc(**{**dict(rows0=2, rows1=3, D=0, groups=1, q_ms=0, eps=1e-5, scale=1.0), **kw})


@pytest.mark.parametrize("kw", [dict(rows0=1 << 62, rows1=1 << 62, groups=1 << 40), dict(rows0=1 << 62, rows1=1 << 62, groups=1 << 4),
                                dict(rows0=1 << 62, rows1=4, groups=1 << 62), dict(rows0=1, rows1=1, groups=1 << 62)])
def test_products_of_extents_past_128_bits(kw):
    """Rows without elements are any number of groups: their count with the rows'
    must not pass for a small one."""
    rc = abi.bind().pe_gated_norm(ctypes.byref(desc(**kw)), None, None, None, 64, None, None, None)
    assert rc == UNSUPPORTED, runtime.last_error()


def test_no_rows_of_any_number_of_groups():
    assert abi.bind().pe_gated_norm(ctypes.byref(desc(rows0=0, groups=1 << 62)), None, None, None, 64, None, None, None) == 0


def test_gates_of_rows_without_elements():
    """A gate for each row is read although the row has no elements."""
    d = desc(gate_row=1, g_s0=3, g_s1=1, g_numel=5)
    args = (None, None, None, None, 64, None, None, 64, 64, None)
    assert abi.bind().pe_residual_norm(ctypes.byref(d), *args) == BOUNDS
