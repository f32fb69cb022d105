"""ctypes mirror of include/pipeinfer_b200.h (operator level).  Fails loudly when the CUDA library is missing."""
import ctypes as C
import os

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
SO_PATH = os.path.join(HERE, "libpipeinfer_b200.so")

TYPE_Q4_0, TYPE_Q8_0, TYPE_Q4_K = 2, 8, 12
TYPE_Q3_K = 11        # matmul + embedding rows (Q3_K_M files); activations as Q4_K
TYPE_Q5_K = 13
TYPE_Q6_K = 14        # matmul only; multiplies with the same activations as Q4_K
TYPE_F32, TYPE_BF16 = 0, 30
TYPE_F8 = 64          # e4m3 with a scale per 128 x 128 block
TYPES = {"q4_0": TYPE_Q4_0, "q8_0": TYPE_Q8_0, "q4_k": TYPE_Q4_K}
BLOCK = {TYPE_Q4_0: (32, 18), TYPE_Q8_0: (32, 34), TYPE_Q4_K: (256, 144), TYPE_Q5_K: (256, 176), TYPE_Q6_K: (256, 210), TYPE_Q3_K: (256, 110)}
ACT_BLOCK = {TYPE_Q4_0: (32, 34), TYPE_Q8_0: (32, 34), TYPE_Q4_K: (256, 292)}


class MoeShape(C.Structure):
    _fields_ = [("type", C.c_int32), ("experts", C.c_int32), ("shared", C.c_int32), ("top", C.c_int32), ("score", C.c_int32), ("renorm", C.c_int32), ("scale", C.c_float),
                ("width", C.c_int64), ("ff", C.c_int64)]


class SampleParams(C.Structure):
    _fields_ = [("temp", C.c_float), ("top_k", C.c_int32), ("top_p", C.c_float), ("min_p", C.c_float)]


class LibraryMissing(RuntimeError):
    pass


class PibError(RuntimeError):
    pass


def _p(a):
    return a.ctypes.data_as(C.c_void_p)


class Lib:
    TYPE_F32, TYPE_BF16, TYPE_F8 = TYPE_F32, TYPE_BF16, TYPE_F8

    def __init__(self, path=SO_PATH):
        if not os.path.exists(path):
            raise LibraryMissing("%s not built: run `python __graft_entry__.py build` (needs nvcc); "
                                 "there is no CPU fallback" % path)
        L = self.L = C.CDLL(path)
        L.pib_last_error.restype = C.c_char_p
        L.pib_init.argtypes = [C.c_int]
        L.pib_dev_alloc.restype = C.c_void_p
        L.pib_dev_alloc.argtypes = [C.c_size_t]
        L.pib_dev_free.argtypes = [C.c_void_p]
        L.pib_memcpy_h2d.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_void_p]
        L.pib_memcpy_d2h.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_void_p]
        L.pib_stream_sync.argtypes = [C.c_void_p]
        L.pib_weight_upload.restype = C.c_void_p
        L.pib_weight_upload.argtypes = [C.c_int, C.c_void_p, C.c_int64, C.c_int64]
        L.pib_weight_from_device.restype = C.c_void_p
        L.pib_weight_from_device.argtypes = [C.c_int, C.c_void_p, C.c_int64, C.c_int64]
        L.pib_weight_free.argtypes = [C.c_void_p]
        L.pib_weight_bytes.restype = C.c_size_t
        L.pib_weight_bytes.argtypes = [C.c_void_p]
        L.pib_weight_row_blocks.argtypes = [C.c_void_p, C.c_int64, C.c_void_p]
        L.pib_act_bytes.restype = C.c_size_t
        L.pib_act_bytes.argtypes = [C.c_int, C.c_int64, C.c_int]
        L.pib_quantize_act.argtypes = [C.c_int, C.c_void_p, C.c_int, C.c_int64, C.c_void_p, C.c_void_p]
        L.pib_norm_quantize_act.argtypes = [C.c_int, C.c_int, C.c_void_p, C.c_void_p, C.c_float, C.c_int, C.c_int64,
                                            C.c_void_p, C.c_void_p, C.c_void_p]
        L.pib_act_to_blocks.argtypes = [C.c_int, C.c_void_p, C.c_int, C.c_int64, C.c_void_p]
        L.pib_gemv.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_int, C.c_void_p]
        L.pib_gemv_q4k_noalloc.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p]
        L.pib_mul_mat_host.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_int]
        L.pib_get_rows.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p]
        for name in ("pib_weight_upload_f8", "pib_weight_from_device_f8"):
            getattr(L, name).restype, getattr(L, name).argtypes = C.c_void_p, [C.c_void_p, C.c_void_p, C.c_int64, C.c_int64]
        L.pib_quantize_act_rows.argtypes = [C.c_int, C.c_void_p, C.c_int, C.c_int64, C.c_void_p, C.c_void_p]
        L.pib_gemv_fused.argtypes = [C.c_void_p, C.c_int] + [C.c_void_p] * 4 + [C.c_int64, C.c_float, C.c_int, C.c_void_p, C.c_void_p]
        L.pib_gemm.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p]
        L.pib_gemm_host.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p]
        L.pib_gemm_check.argtypes = [C.c_void_p]
        L.pib_moe_from_device.restype, L.pib_moe_from_device.argtypes = C.c_void_p, [C.POINTER(MoeShape)] + [C.c_void_p] * 8
        L.pib_moe_free.argtypes = [C.c_void_p]
        L.pib_moe_scratch_bytes.restype, L.pib_moe_scratch_bytes.argtypes = C.c_size_t, [C.c_void_p, C.c_int]
        L.pib_moe_forward.argtypes = [C.c_void_p, C.c_void_p, C.c_int64, C.c_int, C.c_void_p, C.c_int64, C.c_void_p, C.c_int64, C.c_void_p, C.c_void_p]
        L.pib_sample.argtypes = [C.c_int, C.c_void_p, C.c_int64, C.c_int, C.c_int] + [C.c_void_p] * 6

    def check(self, rc):
        if rc != 0:
            raise PibError("libpipeinfer_b200 error %d: %s" % (rc, self.L.pib_last_error().decode()))

    def init(self, device=0):
        self.check(self.L.pib_init(device))

    # ---- device buffers ----
    def to_device(self, arr):
        arr = np.ascontiguousarray(arr)
        d = self.L.pib_dev_alloc(arr.nbytes)
        if not d:
            raise PibError(self.L.pib_last_error().decode())
        self.check(self.L.pib_memcpy_h2d(d, _p(arr), arr.nbytes, None))
        self.check(self.L.pib_stream_sync(None))
        return d

    def alloc(self, nbytes):
        d = self.L.pib_dev_alloc(nbytes)
        if not d:
            raise PibError(self.L.pib_last_error().decode())
        return d

    def to_host(self, dev, shape, dtype):
        out = np.empty(shape, dtype=dtype)
        self.check(self.L.pib_memcpy_d2h(_p(out), dev, out.nbytes, None))
        self.check(self.L.pib_stream_sync(None))
        return out

    def free(self, dev):
        self.L.pib_dev_free(dev)

    # ---- operators on numpy arrays (host in, host out) ----
    def weight_upload(self, wtype, blocks, K):
        blocks = np.ascontiguousarray(blocks)
        N = blocks.shape[0]
        w = self.L.pib_weight_upload(wtype, _p(blocks), N, K)
        if not w:
            raise PibError(self.L.pib_last_error().decode())
        return w

    def weight_rows(self, w, wtype, N, K):
        be, bb = BLOCK[wtype]
        out = np.zeros((N, K // be * bb), dtype=np.uint8)
        for r in range(N):
            self.check(self.L.pib_weight_row_blocks(w, r, _p(out[r])))
        return out

    def quantize_act(self, wtype, x, norm_w=None, eps=0.0):
        x = np.ascontiguousarray(x, dtype=np.float32)
        b, K = x.shape
        xd = self.to_device(x)
        act = self.alloc(self.L.pib_act_bytes(wtype, K, b))
        if norm_w is None:
            self.check(self.L.pib_quantize_act(wtype, xd, b, K, act, None))
        else:
            wd = self.to_device(np.ascontiguousarray(norm_w, dtype=np.float32))
            self.check(self.L.pib_norm_quantize_act(wtype, 1, xd, wd, eps, b, K, act, None, None))
            self.free(wd)
        be, bb = ACT_BLOCK[wtype]
        out = np.zeros((b, K // be * bb), dtype=np.uint8)
        self.check(self.L.pib_act_to_blocks(wtype, act, b, K, _p(out)))
        self.free(xd)
        self.free(act)
        return out

    def mul_mat(self, w, x, N, variant=0):
        x = np.ascontiguousarray(x, dtype=np.float32)
        b = x.shape[0]
        y = np.empty((b, N), dtype=np.float32)
        self.check(self.L.pib_mul_mat_host(w, _p(x), b, _p(y), variant))
        return y

    def get_rows(self, w, ids, K):
        ids = np.ascontiguousarray(ids, dtype=np.int32)
        idd = self.to_device(ids)
        out = self.alloc(len(ids) * K * 4)
        self.check(self.L.pib_get_rows(w, idd, len(ids), out, None))
        res = self.to_host(out, (len(ids), K), np.float32)
        self.free(idd)
        self.free(out)
        return res

    # ---- operators on device pointers (integers), in the order of `stream` (a cudaStream_t as an integer, 0 or None: the legacy default stream) ----
    def act_bytes(self, wtype, K, b):
        return self.L.pib_act_bytes(wtype, K, b)

    def quantize_act_dev(self, wtype, x, b, K, act, stream=None):
        self.check(self.L.pib_quantize_act(wtype, x, b, K, act, stream))

    def quantize_act_rows(self, wtype, x, b, K, act, stream=None):
        self.check(self.L.pib_quantize_act_rows(wtype, x, b, K, act, stream))

    def gemv(self, w, act, b, y, stream=None, variant=0):
        self.check(self.L.pib_gemv(getattr(w, "h", w), act, b, y, variant, stream))

    def gemv_fused(self, w, x, b, y, stream=None, prologue=0, x2=None, addend=None, sum_out=None, xstride=0, eps=0.0):
        self.check(self.L.pib_gemv_fused(getattr(w, "h", w), prologue, x, x2, addend, sum_out, xstride, eps, b, y, stream))

    def gemm(self, w, act, b, y, scratch, stream=None):
        self.check(self.L.pib_gemm(getattr(w, "h", w), act, b, y, scratch, stream))

    def gemm_check(self, stream=None):
        self.check(self.L.pib_gemm_check(stream))

    def sample(self, type_, logits, ld, rows, n_vocab, params, u, ids, p=None, kept=None, stream=None):
        """params: an array of SampleParams in device memory, one per row"""
        self.check(self.L.pib_sample(type_, logits, ld, rows, n_vocab, params, u, ids, p, kept, stream))


class F8Weight:
    """e4m3 rows [N][K] with fp32 scales [ceil(N/128)][ceil(K/128)], from device pointers; stands for the handle in Lib.gemv, gemv_fused and gemm"""

    def __init__(self, lib, q, scales, N, K):
        self.lib, self.N, self.K = lib, N, K
        self.h = lib.L.pib_weight_from_device_f8(q, scales, N, K)
        if not self.h:
            raise PibError(lib.L.pib_last_error().decode())

    def __del__(self):
        if getattr(self, "h", None):
            self.lib.L.pib_weight_free(self.h)
            self.h = None


class Moe:
    """a mixture layer for up to 16 tokens (pib_moe_from_device); weights as device pointers"""

    def __init__(self, lib, type_, experts, shared, top, width, ff, router, gate, up, down, correction=None, gate_scales=None, up_scales=None, down_scales=None, score="softmax", renorm=False,
                 scale=1.0):
        self.lib = lib
        self.shape = MoeShape(type_, experts, shared, top, {"softmax": 0, "sigmoid": 1}[score], 1 if renorm else 0, scale, width, ff)
        self.h = lib.L.pib_moe_from_device(C.byref(self.shape), router, correction, gate, gate_scales, up, up_scales, down, down_scales)
        if not self.h:
            raise PibError(lib.L.pib_last_error().decode())

    def scratch_bytes(self, b):
        return self.lib.L.pib_moe_scratch_bytes(self.h, b)

    def forward(self, x, ldx, b, residual, ldr, y, ldy, scratch, stream=None):
        self.lib.check(self.lib.L.pib_moe_forward(self.h, x, ldx, b, residual, ldr, y, ldy, scratch, stream))

    def __del__(self):
        if getattr(self, "h", None):
            self.lib.L.pib_moe_free(self.h)
            self.h = None


_lib = None


def load():
    global _lib
    if _lib is None:
        _lib = Lib()
    return _lib
