"""GPU: the words in which the units of kernels count bounded waits that ran out, as
pkcu_wait_timeouts() and the synchronous calls sum them: every unit's counts, read
without clearing and cleared. The counts are written here by the host."""
import ctypes as C

import numpy as np
import pytest

from gpuhelp import _DeviceView

pytestmark = pytest.mark.gpu

UNITS = ("softmax", "conv", "tc", "q8", "rms")


def words(cuda):
    import torch
    L = cuda.lib()
    out = []
    for u in UNITS:
        p = C.c_void_p()
        assert getattr(L, f"pk_{u}_wait_word")(C.byref(p)) == 0
        out.append(torch.as_tensor(_DeviceView(p.value, 1, np.int32), device="cuda"))
    return out


def read(cuda, reset):
    n = C.c_uint(77)
    cuda.call("pkcu_wait_timeouts", C.byref(n), reset)
    return n.value


def test_sum_read_and_reset(cuda):
    import torch
    ws = words(cuda)
    assert len({w.data_ptr() for w in ws}) == len(UNITS) and read(cuda, 1) == 0
    for i, w in enumerate(ws):
        w.fill_(1 << i)
    torch.cuda.synchronize()
    assert read(cuda, 0) == 31 and read(cuda, 0) == 31 and read(cuda, 1) == 31 and read(cuda, 0) == 0
    assert all(int(w) == 0 for w in ws)


@pytest.mark.parametrize("unit", range(len(UNITS)))
def test_a_synchronous_call_reports_and_clears(cuda, unit):
    import torch
    words(cuda)[unit].fill_(3)
    torch.cuda.synchronize()
    L = cuda.lib()
    x, o = np.ones((2, 1024), np.float32), np.zeros((2, 1024), np.float32)
    g, b = np.ones(1024, np.float32), np.zeros(1024, np.float32)
    p = lambda a: a.ctypes.data_as(C.POINTER(C.c_float))
    L.pk_layer_norm_rows(p(x), p(g), p(b), p(o), 2, 1024)
    assert "3 bounded device wait(s) ran out" in L.pkcu_last_error().decode()
    assert read(cuda, 0) == 0


def test_two_threads(cuda):
    """Calls from several host threads at once: no count is lost or told twice."""
    import threading
    import torch
    ws = words(cuda)
    for i, w in enumerate(ws):
        w.fill_(1 << i)
    torch.cuda.synchronize()
    seen, lock = [], threading.Lock()

    def run():
        torch.cuda.set_device(0)
        for _ in range(50):
            n = read(cuda, 1)
            with lock:
                seen.append(n)
    threads = [threading.Thread(target=run) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert sorted(seen)[-1] == 31 and sum(seen) == 31
