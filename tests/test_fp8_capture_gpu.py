"""8-bit weights whose last reference goes away while a stream is captured."""
import gc
import threading

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device(gpu):
    pass


def _weight(rows=512, k=1024):
    from libcmol_b200 import fp8
    return fp8.Fp8Weight.quantize(torch.randn(rows, k, device="cuda"))


@pytest.mark.parametrize("how", ["collected", "freed", "freed by another thread"])
def test_a_weight_goes_while_a_stream_is_captured(how):
    """The capture lives on, its replay is right, and the memory is given back."""
    from libcmol_b200 import fp8
    keep, gone = _weight(), [_weight(1 << 16, 1 << 13)]              # 0.5 GB
    q, s = fp8.quantize(torch.randn(40, 1024, device="cuda"))
    want = keep.matmul(q, s)
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    g = torch.cuda.CUDAGraph()
    y = torch.zeros_like(want)
    with torch.cuda.graph(g):
        if how == "collected":
            gone.clear()
            gc.collect()
        elif how == "freed":
            gone[0].free()
        else:
            t = threading.Thread(target=gone[0].free)
            t.start()
            t.join()
        keep.matmul(q, s, y=y)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)
    gone.clear()
    assert torch.cuda.mem_get_info()[0] - free > 400 << 20
