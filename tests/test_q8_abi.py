"""CPU: the 8-bit operators refuse bad arguments before any CUDA call."""
import ctypes as C
import os

import pytest

import pkcuda

ERR_ARG = 1


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(pkcuda.LIB_PATH):
        pkcuda.build()
    return pkcuda.lib()


P = 4096   # stands for a device address: never read


@pytest.mark.parametrize("change,word", [
    (dict(n_rows=-1), "rows"), (dict(D=0), "rows"), (dict(D=(1 << 24) + 1), "rows"), (dict(dtype=1), "type"), (dict(dtype=5), "type"),
    (dict(dtype=9), "type"), (dict(qtype=0), "output"), (dict(qtype=3), "output"), (dict(ldq=1023), "ldq"),
    (dict(eps=0.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(x=None), "NULL"),
    (dict(gamma=None), "NULL"), (dict(q=None), "NULL"), (dict(scales=None), "NULL"), (dict(x_out=None), "NULL"),
    (dict(y=None), "bias"), (dict(x=P + 2), "aligned"), (dict(gamma=P + 1), "aligned"),
    (dict(scales=P + 2), "aligned"), (dict(dtype=3, y=P + 1), "aligned")])
def test_rms_norm_refusals(L, change, word):
    a = dict(x=P, y=P, bias=P, alpha=1.0, gamma=P, eps=1e-5, dtype=0, x_out=P, q=P, qtype=1, ldq=1024, scales=P,
             n_rows=4, D=1024)
    a.update(change)
    assert L.pkcu_residual_rms_norm_q8(*a.values(), None) == ERR_ARG
    msg = L.pkcu_last_error().decode()
    assert "pkcu_residual_rms_norm_q8" in msg and word in msg, msg


@pytest.mark.parametrize("change,word", [
    (dict(dtype=0), "type"), (dict(dtype=3), "type"), (dict(K=0), "K 0"), (dict(K=131072), "K"), (dict(N=0), "N 0"),
    (dict(n_scales=2), "scales"), (dict(n_scales=0), "scales"), (dict(data=None), "NULL"),
    (dict(scales=None), "NULL"), (dict(scales=P + 2), "aligned")])
def test_weight_q8_refusals(L, change, word):
    h = C.c_void_p(7)
    a = dict(data=P, dtype=1, scales=P, n_scales=64, K=64, N=64)
    a.update(change)
    assert L.pkcu_weight_q8_create(*a.values(), None, C.byref(h)) == ERR_ARG
    msg = L.pkcu_last_error().decode()
    assert "pkcu_weight_q8_create" in msg and word in msg and not h.value, msg
    assert L.pkcu_weight_q8_create(*a.values(), None, None) == ERR_ARG
    L.pkcu_weight_q8_destroy(None)


def test_product_needs_a_weight(L):
    assert L.pkcu_wmatmul_q8(P, 64, P, None, None, 2, None, 0, 1.0, P, 64, 0, 4, None) == ERR_ARG
    assert b"NULL weight" in L.pkcu_last_error()


@pytest.mark.parametrize("change,word", [
    (dict(n_rows=-1), "rows"), (dict(V=0), "rows"), (dict(V=262145), "rows"), (dict(dtype=1), "type"),
    (dict(dtype=5), "type"), (dict(logits=None), "NULL"), (dict(u=None), "NULL"), (dict(tokens=None), "NULL"),
    (dict(ld=1024), "ld"), (dict(logits=P + 2), "aligned"), (dict(top_k=P + 1), "aligned"),
    (dict(logprobs=P + 2), "aligned")])
def test_sample_refusals(L, change, word):
    a = dict(logits=P, dtype=0, ld=1025, temperature=None, top_k=P, top_p=P, min_p=None, u=P, tokens=P, logprobs=P,
             n_rows=3, V=1025)
    a.update(change)
    assert L.pkcu_sample_rows(*a.values(), None) == ERR_ARG
    msg = L.pkcu_last_error().decode()
    assert "pkcu_sample_rows" in msg and word in msg, msg


def test_no_rows(L):
    assert L.pkcu_sample_rows(None, 0, 10, None, None, None, None, None, None, None, 0, 10, None) == 0
    assert L.pkcu_residual_rms_norm_q8(None, None, None, 1.0, None, 1e-5, 0, None, None, 1, 10, None, 0, 10, None) == 0
