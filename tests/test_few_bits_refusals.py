"""CPU-only: arguments that the entry points of 8-bit integer weights and of the 4-bit key / value cache refuse before anything is launched."""
import ctypes as C

import pytest

I8, F32, BF16 = 65, 0, 30
P = 1 << 12          # stands for a pointer; nothing reads it


@pytest.fixture(scope="module")
def L():
    from pipeinfer_b200 import lib as pib
    return pib.load().L


def refused(L, rc, text):
    return rc in (-2, -4) and text in L.pib_last_error().decode()


def test_weights(L):
    assert not L.pib_weight_upload(I8, P, 128, 128) and b"pib_weight_upload_i8" in L.pib_last_error()
    assert not L.pib_weight_from_device(I8, P, 128, 128)
    for args in ((None, P, 4, 4), (P, None, 4, 4), (P, P, 0, 4), (P, P, 4, 0), (P, P, -1, 4), (P, P, 4, 131073)):
        assert not L.pib_weight_upload_i8(*args) and not L.pib_weight_from_device_i8(*args)
    assert not L.pib_weight_from_device_i8(P, P + 2, 4, 4)


def test_quantiser(L):
    for x, b, K, act in ((None, 1, 128, P), (P, 0, 128, P), (P, 1, 0, P), (P, 65537, 128, P), (P, 1, 128, None), (P, 1, 131073, P), (P + 2, 1, 128, P), (P, 1, 128, P + 8)):
        assert refused(L, L.pib_quantize_act_rows(I8, x, b, K, act, None), "act quantise")
        assert refused(L, L.pib_quantize_act(I8, x, b, K, act, None), "act quantise")
    assert refused(L, L.pib_norm_quantize_act(I8, 2, P, P, 1e-5, 1, 128, P, None, None), "RMSNorm")
    assert refused(L, L.pib_norm_quantize_act(I8, 1, P, None, 1e-5, 1, 128, P, None, None), "bad arguments")
    # rows of whole 128 bytes, a scale a token, both rounded up to 256 bytes
    assert L.pib_act_bytes(I8, 1, 1) == 256 + 256 and L.pib_act_bytes(I8, 129, 5) == 1280 + 256 and L.pib_act_bytes(I8, 8192, 1999) == 1999 * 8192 + 8192


def test_caches(L):
    for args in ((0, 1, 64), (-1, 1, 64), (1 << 25, 1, 64), (1, 0, 64), (1, 1025, 64), (1, 1, 32), (1, 1, 96), (1, 1, 256)):
        assert not L.pib_kv4_new(*args) and b"pib_kv4_new" in L.pib_last_error()
    assert L.pib_kv4_bytes(None) == 0
    L.pib_kv4_free(None)
    assert refused(L, L.pib_kv4_write(None, F32, P, 64, P, 64, P, 1, None), "no cache")
    assert refused(L, L.pib_kv4_read(None, F32, P, 1, P, 64, P, 64, None), "no cache")


def test_attention_without_a_cache(L):
    from pipeinfer_b200 import lib as pib
    b = pib.Kv4Batch(F32, 8, 1, 1, 1, 1, 0, 1.0)
    assert refused(L, L.pib_kv4_attn(None, C.byref(b), P, 512, P, P, P, P, 512, P, None), "no cache")
    assert L.pib_kv4_attn_scratch_bytes(None, C.byref(b)) == 0
