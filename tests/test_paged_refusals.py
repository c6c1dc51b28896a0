"""CPU: what the paged cache's C entries and Python calls refuse, beside tests/test_paged_host.py."""
import ctypes as C


from bitgpu_amd import _lib


def message():
    return _lib.lib().bg_last_error_message().decode()


def test_units_of_no_batch():
    units = (C.c_int64 * 4)()
    assert _lib.lib().bg_paged_batch_units(None, units) == _lib.BG_E_INVALID
    assert "NULL" in message()
