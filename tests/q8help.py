"""Plain 64-bit forms and inputs shared by the tests of the 8-bit operators."""
import numpy as np

from gpuhelp import ALIVE

HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def torch_dtype(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "i8": torch.int8,
            "e4m3": torch.float8_e4m3fn}[name]


def cu(a, dtype=None, offset=0):
    """A device tensor of dtype with the values of a; offset: elements by which
    its start is moved off an allocation's (256-byte aligned) start."""
    import torch
    t = torch.as_tensor(a)
    t = t.to(torch_dtype(dtype)) if dtype else t
    flat = torch.empty(t.numel() + offset, dtype=t.dtype, device="cuda")
    flat[offset:].copy_(t.reshape(-1))
    ALIVE.append(flat)
    return flat[offset:].view(t.shape)


def f64(t):
    """Host float64 values of a tensor of any type."""
    import torch
    torch.cuda.synchronize()
    return t.detach().cpu().to(torch.float64).numpy()


def rms_q8(x_stored, gamma, eps, Q):
    """(scales, values before rounding) of the norm of stored rows, in 64 bits."""
    x = x_stored.astype(np.float64)
    t = x * gamma.astype(np.float64)
    r = 1.0 / np.sqrt((x * x).mean(axis=1) + np.float64(np.float32(eps)))
    amax = np.abs(t).max(axis=1)
    v = t * (Q / np.where(amax == 0, 1, amax))[:, None]
    return amax * r / Q, v
