"""CPU-only: arguments that the 8-bit floating point, mixture and sampling entry points refuse before anything is launched."""
import ctypes as C

import pytest

F8, BF16 = 64, 30
P = 1 << 12          # stands for a pointer; nothing reads it


@pytest.fixture(scope="module")
def L():
    from pipeinfer_b200 import lib as pib
    return pib.load().L


def refused(L, rc, text):
    return rc in (-2, -4) and text in L.pib_last_error().decode()


def test_weights(L):
    assert not L.pib_weight_upload(F8, P, 128, 128) and b"pib_weight_upload_f8" in L.pib_last_error()
    assert not L.pib_weight_from_device(F8, P, 128, 128)
    for args in ((None, P, 4, 4), (P, None, 4, 4), (P, P, 0, 4), (P, P, 4, 0), (P, P, -1, 4)):
        assert not L.pib_weight_upload_f8(*args) and not L.pib_weight_from_device_f8(*args)


def test_quantiser(L):
    for x, b, K, act in ((None, 1, 128, P), (P, 0, 128, P), (P, 1, 0, P), (P, 65537, 128, P), (P, 1, 128, None)):
        assert refused(L, L.pib_quantize_act_rows(F8, x, b, K, act, None), "act quantise")
        assert refused(L, L.pib_quantize_act(F8, x, b, K, act, None), "act quantise")
    assert refused(L, L.pib_norm_quantize_act(F8, 2, P, P, 1e-5, 1, 128, P, None, None), "RMSNorm")
    assert refused(L, L.pib_norm_quantize_act(F8, 1, P, None, 1e-5, 1, 128, P, None, None), "bad arguments")


def test_activation_bytes(L):
    # e4m3 rows of whole blocks, scales of 4-token groups, both rounded up to 256 bytes
    assert L.pib_act_bytes(F8, 1, 1) == 256 + 256
    assert L.pib_act_bytes(F8, 128, 3) == 512 + 256
    assert L.pib_act_bytes(F8, 129, 5) == 1280 + 256
    assert L.pib_act_bytes(F8, 8192, 1999) == 1999 * 8192 + 64 * 2000 * 4


def shape(**kw):
    from pipeinfer_b200 import lib as pib
    d = dict(type=F8, experts=8, shared=1, top=2, score=0, renorm=1, scale=1.0, width=256, ff=128)
    d.update(kw)
    return pib.MoeShape(*[d[n] for n, _ in pib.MoeShape._fields_])


@pytest.mark.parametrize("kw", [dict(type=12), dict(experts=0), dict(experts=513), dict(top=0), dict(top=9), dict(shared=-1), dict(shared=15), dict(score=2), dict(width=0), dict(ff=0), dict(width=1 << 21),
                                dict(shared=0x7fffffff)])
def test_mixture_shapes(L, kw):
    assert not L.pib_moe_from_device(C.byref(shape(**kw)), P, None, P, P, P, P, P, P)
    assert b"bad arguments" in L.pib_last_error()


def test_mixture_pointers(L):
    for i in (0, 2, 3, 4, 5, 6, 7):
        args = [P, None, P, P, P, P, P, P]
        args[i] = None
        assert not L.pib_moe_from_device(C.byref(shape()), *args)
    assert not L.pib_moe_from_device(None, P, None, P, P, P, P, P, P)
    assert L.pib_moe_scratch_bytes(None, 1) == 0
    assert refused(L, L.pib_moe_forward(None, P, 256, 1, None, 0, P, 256, P, None), "bad arguments")


def test_sampling(L):
    ok = dict(type=0, logits=P, ld=100, rows=2, V=100, params=P, u=P, ids=P)

    def call(**kw):
        a = dict(ok, **kw)
        return L.pib_sample(a["type"], a["logits"], a["ld"], a["rows"], a["V"], a["params"], a["u"], a["ids"], None, None, None)
    for kw in (dict(type=2), dict(logits=None), dict(ld=99), dict(rows=-1), dict(V=0), dict(V=262145, ld=300000), dict(params=None), dict(u=None), dict(ids=None)):
        assert refused(L, call(**kw), "pib_sample"), kw
    assert call(rows=0) == 0


def test_products_without_a_weight(L):
    assert refused(L, L.pib_gemv(None, P, 1, P, 0, None), "pib_gemv")
    assert refused(L, L.pib_gemm(None, P, 1, P, P, None), "pib_gemm")


def test_alignment(L):
    """pointers that no load of their type could read"""
    assert refused(L, L.pib_quantize_act_rows(F8, P + 2, 1, 128, P, None), "act quantise")
    assert refused(L, L.pib_quantize_act_rows(F8, P, 1, 128, P + 8, None), "act quantise")
    for i, off in ((0, 2), (1, 1), (3, 2), (5, 1), (7, 3)):
        args = [P] * 8
        args[i] += off
        assert not L.pib_moe_from_device(C.byref(shape()), *args) and b"bad arguments" in L.pib_last_error()
    for i in range(6):
        ptr = [P] * 6
        ptr[i] += 2
        assert refused(L, L.pib_sample(0, ptr[0], 100, 2, 100, ptr[1], ptr[2], ptr[3], ptr[4], ptr[5], None), "pib_sample")
    assert refused(L, L.pib_sample(30, P + 1, 100, 2, 100, P, P, P, None, None, None), "pib_sample")
