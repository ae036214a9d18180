"""libcmol_b200.fp8 above the library (no GPU needed): what it passes on, with a
stand-in for the library where a call would need a GPU."""
import ctypes as C

import pytest

import libcmol_b200 as pkg
from libcmol_b200 import fp8


class _Word:
    """A library whose fault word holds `code`."""

    def __init__(self, code):
        self.code, self.asked = code, []

    def cmolcu_fault_status(self, device, out, clear):
        self.asked.append((device, clear))
        C.cast(out, C.POINTER(C.c_uint))[0] = self.code
        if clear:
            self.code = 0
        return 0


def test_a_wait_that_ran_out_is_seen(monkeypatch):
    word = _Word(2)
    monkeypatch.setattr(fp8, "lib", lambda: word)
    assert fp8.fault() == 2 and fp8.fault(3) == 2
    assert fp8.fault(3, clear=True) == 2 and fp8.fault(3) == 0
    assert word.asked == [(0, 0), (3, 0), (3, 1), (3, 0)]


def test_no_word_is_an_error():
    with pytest.raises(pkg.CmolError, match="fp8.fault: cmolcu_fault_status: no fault word for device 99"):
        fp8.fault(99)
