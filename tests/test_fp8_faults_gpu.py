"""The fault word of the kernels behind cmolcu.h, as a caller reads it."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def test_a_device_without_a_word_is_refused_and_leaves_no_error(gpu):
    """A device number that no GPU has: no word is made for it elsewhere, and the
    program's next look at the runtime's last error finds none."""
    from libcmol_b200 import last_error, lib
    code = C.c_uint(7)
    missing = torch.cuda.device_count()
    for device in (missing, 63, 64, -1):
        assert lib().cmolcu_fault_status(device, C.byref(code), 0) == -1
        assert last_error() == f"cmolcu_fault_status: no fault word for device {device}"
    x = torch.zeros(16, device="cuda")
    assert (x + 1 == 1).all() and torch.cuda.current_device() == 0 and code.value == 7
    assert lib().cmolcu_fault_status(0, C.byref(code), 0) == 0 and code.value == 0


def test_the_word_through_the_module(gpu):
    """Products leave it at zero; the module reads and clears it."""
    from libcmol_b200 import CmolError, fp8
    W = fp8.Fp8Weight.quantize(torch.ones(300, 640, device="cuda"))
    for n in (1, 12, 40, 300):
        W.matmul(*fp8.quantize(torch.ones(n, 640, device="cuda")))
    torch.cuda.synchronize()
    assert fp8.fault() == 0 and fp8.fault(0, clear=True) == 0
    with pytest.raises(CmolError, match="fp8.fault: cmolcu_fault_status: no fault word for device 77"):
        fp8.fault(77)
