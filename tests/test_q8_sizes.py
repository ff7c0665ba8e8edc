"""CPU: the Python wrappers of the 8-bit operators refuse sizes that do not fit the
C interface's int, which ctypes would pass on cut to their low 32 bits (2^32 + 5 rows
as 5). Tensors are stand-ins: nothing is allocated, no call goes out."""
import types

import pytest

import pkcuda

torch = pytest.importorskip("torch")


class Tensor:
    """As much of a CUDA tensor as the checks look at."""

    def __init__(self, shape, dtype):
        self.shape, self.dtype, self.is_cuda = torch.Size(shape), dtype, True

    def get_device(self):
        return 0

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()

    def is_contiguous(self):
        return True

    def stride(self):
        return (self.shape[1], 1) if len(self.shape) == 2 else (1,)

    def data_ptr(self):
        return 4096


@pytest.fixture
def sent(monkeypatch):
    calls = []
    pkcuda._load_torch()
    monkeypatch.setattr(pkcuda, "_on", lambda dev, stream, name, *args: calls.append((name, args)))
    return calls


f32, i8 = torch.float32, torch.int8


@pytest.mark.parametrize("rows,D", [(2 ** 31, 4), (2 ** 32 + 5, 4), (2, 2 ** 32 + 8)])
def test_norm(sent, rows, D):
    def call(rows, D):
        x = Tensor((rows, D), f32)
        pkcuda.residual_rms_norm_q8(x, x, None, 1.0, Tensor((D,), f32), 1e-5, x, Tensor((rows, D), i8), Tensor((rows,), f32))
    with pytest.raises(ValueError, match="32-bit"):
        call(rows, D)
    assert not sent
    call(2 ** 31 - 1, 4)
    assert sent[0][0] == "pkcu_residual_rms_norm_q8"


@pytest.mark.parametrize("M", [2 ** 31, 2 ** 32 + 5])
def test_product(sent, M):
    w = types.SimpleNamespace(N=4, K=16, handle=1, dtype=i8)
    call = lambda M: pkcuda.wmatmul_q8(Tensor((M, 16), i8), Tensor((M,), f32), w, Tensor((M, 4), f32))
    with pytest.raises(ValueError, match="32-bit"):
        call(M)
    assert not sent
    call(7)
    assert sent[0][0] == "pkcu_wmatmul_q8"


@pytest.mark.parametrize("K,N", [(1, 2 ** 32 + 64), (2 ** 32 + 16, 1)])
def test_weight(monkeypatch, K, N):
    monkeypatch.setattr(pkcuda, "call", lambda *a: pytest.fail("a call went out"))
    with pytest.raises(ValueError, match="32-bit"):
        pkcuda.WeightQ8(types.SimpleNamespace(shape=(K, N), dtype=i8, is_cuda=True, dim=lambda: 2,
                                              is_contiguous=lambda: True), 1.0)


@pytest.mark.parametrize("V", [2 ** 31, 2 ** 32 + 5])
def test_sampling(sent, V):
    call = lambda rows, V: pkcuda.sample_rows(Tensor((rows, V), f32), Tensor((rows,), f32), Tensor((rows,), torch.int32))
    with pytest.raises(ValueError, match="32-bit"):
        call(2, V)
    assert not sent
    call(2 ** 33, 4)   # the number of rows is 64 bits wide
    assert sent[0][0] == "pkcu_sample_rows"
