"""8-bit floating point weights with a scale per 128 x 128 block (csrc/f8_quant.cu, f8_gemv.cu, f8_gemm.cu) against float64: sizes that fill no block, no tile and no share, every number of
tokens where another kernel or tile begins, zero and tiny blocks, infinities and numbers that are none in one token, fused prologues, captured calls, other streams."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
F8 = 64


@pytest.fixture(scope="module")
def pib():
    from pipeinfer_b200 import lib as pib
    pib.load().init(0)
    return pib


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


def blocks(n):
    return (n + 127) // 128


def matrix(torch, N, K, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = (torch.randn(N, K, device="cuda", generator=g) * 96).clamp(-448, 448).to(torch.float8_e4m3fn)
    s = (torch.rand(blocks(N), blocks(K), device="cuda", generator=g) + 0.5) / 96
    return q, s, g


def rows(torch, b, K, g):
    x = torch.randn(b, K, device="cuda", generator=g)
    x[:, ::37] *= 20
    return x


def quantised(torch, x):
    """e4m3 values and scales, by their definition"""
    b, K = x.shape
    p = torch.zeros(b, blocks(K) * 128, device="cuda")
    p[:, :K] = x
    v = p.reshape(b, -1, 128)
    d = v.abs().amax(-1).clamp(min=2.0 ** -100) * float(np.float32(1) / np.float32(448))
    return (v / d.unsqueeze(-1)).to(torch.float8_e4m3fn).reshape(b, -1), d


def dense(torch, q, s):
    N, K = q.shape
    return q.double() * s.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]


def want(torch, q, s, x):
    """float64 outputs and the bound of an output's error: a block's 128 products are added in four steps of the tensor core, which may cut instead of round (2^-22 each), the blocks
    by KB fused multiply-adds with a factor of one rounding (2^-24 each)"""
    a, d = quantised(torch, x)
    K = x.shape[1]
    X = (a.double() * d.double().repeat_interleave(128, 1))[:, :K]
    W = dense(torch, q, s)
    return X @ W.T, (X.abs() @ W.abs().T) * (4 * 2.0 ** -22 + (blocks(K) + 3) * 2.0 ** -24) + 1e-36


def product(torch, pib, w, x, how, stream=0):
    lib, (b, K) = pib.load(), x.shape
    y = torch.full((b, w.N), float("nan"), device="cuda")
    if how == "fused":
        lib.gemv_fused(w, x.data_ptr(), b, y.data_ptr(), stream)
        return y
    act = torch.empty(lib.act_bytes(F8, K, b), dtype=torch.uint8, device="cuda")
    (lib.quantize_act_dev if how == "gemv" else lib.quantize_act_rows)(F8, x.data_ptr(), b, K, act.data_ptr(), stream)
    if how == "gemv":
        lib.gemv(w, act.data_ptr(), b, y.data_ptr(), stream)
    else:
        lib.gemm(w, act.data_ptr(), b, y.data_ptr(), None, stream)
        lib.gemm_check(stream)
    return y


@pytest.mark.parametrize("b,K", [(1, 1), (1, 128), (3, 127), (5, 129), (16, 1000), (17, 4096), (300, 260)])
def test_quantiser(torch, pib, b, K):
    """bytes and scales as defined; blocks of zeros, of values whose quotients with 448 are no normal numbers, of the largest floats"""
    lib = pib.load()
    g = torch.Generator(device="cuda").manual_seed(b * 7 + K)
    x = rows(torch, b, K, g)
    if b >= 3:
        x[1, :128] = 0
        x[2, :128] *= 1e-38
        x[0, :128] = x[0, :128].clamp(-2, 2) * 1.5e38
    act = torch.empty(lib.act_bytes(F8, K, b), dtype=torch.uint8, device="cuda")
    lib.quantize_act_rows(F8, x.data_ptr(), b, K, act.data_ptr())
    out = np.zeros((b, blocks(K), 132), np.uint8)
    lib.check(lib.L.pib_act_to_blocks(F8, act.data_ptr(), b, K, out.ctypes.data))
    a, d = quantised(torch, x)
    assert np.array_equal(out[:, :, :4].copy().view(np.float32)[..., 0], d.cpu().numpy())
    got = torch.from_numpy(out[:, :, 4:].copy()).view(torch.float8_e4m3fn).float()
    assert torch.equal(got, a.float().cpu().reshape(b, -1, 128))      # as values: the two zeros are one


@pytest.mark.parametrize("b,K", [(1, 128), (4, 1000), (16, 5632)])
def test_quantiser_behind_a_norm(torch, pib, b, K):
    lib = pib.load()
    g = torch.Generator(device="cuda").manual_seed(K)
    x, w = rows(torch, b, K, g), torch.rand(K, device="cuda", generator=g) + 0.5
    act, xn = torch.empty(lib.act_bytes(F8, K, b), dtype=torch.uint8, device="cuda"), torch.empty(b, K, device="cuda")
    lib.check(lib.L.pib_norm_quantize_act(F8, 1, x.data_ptr(), w.data_ptr(), 1e-5, b, K, act.data_ptr(), xn.data_ptr(), None))
    torch.cuda.synchronize()
    ref = x.double() / (x.double().pow(2).mean(1, keepdim=True) + 1e-5).sqrt() * w.double()
    # the mean's sum of K / 256 + 8 fp32 additions in a thread's chain, halved by the root; three roundings behind it
    assert ((xn.double() - ref).abs() <= ref.abs() * ((K / 256 + 16) / 2 + 6) * 2.0 ** -24).all()
    out = np.zeros((b, blocks(K), 132), np.uint8)
    lib.check(lib.L.pib_act_to_blocks(F8, act.data_ptr(), b, K, out.ctypes.data))
    a, d = quantised(torch, xn)
    assert np.array_equal(out[:, :, 4:].copy().reshape(b, -1) & 127, a.view(torch.uint8).cpu().numpy() & 127)
    assert np.array_equal(out[:, :, :4].copy().view(np.float32)[..., 0], d.cpu().numpy())


SIZES = [(1, 1), (16, 128), (17, 129), (127, 1000), (128, 256), (129, 2048), (1000, 5700), (2560, 2048), (10000, 640)]


@pytest.mark.parametrize("N,K", SIZES)
@pytest.mark.parametrize("b", [1, 2, 7, 8, 9, 13, 16])
def test_decode_batches(torch, pib, N, K, b):
    q, s, g = matrix(torch, N, K, N + K)
    x = rows(torch, b, K, g)
    w = pib.F8Weight(pib.load(), q.data_ptr(), s.data_ptr(), N, K)
    y, lim = want(torch, q, s, x)
    for how in ["gemv"] + (["fused"] if b <= 8 else []):
        err = (product(torch, pib, w, x, how).double() - y).abs()
        assert (err <= lim).all(), (how, float((err / lim).max()))


@pytest.mark.parametrize("N,K,b", [(1, 1, 1), (16, 128, 20), (130, 129, 33), (128, 256, 16), (257, 1000, 65), (300, 5700, 100), (2560, 2048, 129), (1000, 640, 256), (640, 1300, 257), (384, 8192, 40),
                                   (1100, 2000, 700), (20000, 256, 31), (19000, 128, 300), (5000, 3000, 513)])
def test_prompts(torch, pib, N, K, b):
    q, s, g = matrix(torch, N, K, N + K)
    x = rows(torch, b, K, g)
    w = pib.F8Weight(pib.load(), q.data_ptr(), s.data_ptr(), N, K)
    y, lim = want(torch, q, s, x)
    got = product(torch, pib, w, x, "gemm")
    err = (got.double() - y).abs()
    assert (err <= lim).all(), float((err / lim).max())
    for _ in range(3):
        assert torch.equal(product(torch, pib, w, x, "gemm"), got)


@pytest.mark.parametrize("how,b", [("fused", 3), ("gemv", 11), ("gemm", 50)])
@pytest.mark.parametrize("bad", [float("inf"), float("nan"), 0.0])
def test_one_bad_token(torch, pib, how, b, bad):
    """an infinity or a number that is none spoils its own token alone; a token of zeros gives zeros"""
    q, s, g = matrix(torch, 200, 700, 5)
    x = rows(torch, b, 700, g)
    if bad == 0.0:
        x[1] = 0
    else:
        x[1, 333] = bad
    w = pib.F8Weight(pib.load(), q.data_ptr(), s.data_ptr(), 200, 700)
    got = product(torch, pib, w, x, how)
    y, lim = want(torch, q, s, x)
    others = [t for t in range(b) if t != 1]
    assert ((got[others].double() - y[others]).abs() <= lim[others]).all()
    assert (got[1] == 0).all() if bad == 0.0 else torch.isnan(got[1]).all()


@pytest.mark.parametrize("K,xstride", [(1024, 0), (1000, 1003), (2048, 4096)])
def test_fused_prologues(torch, pib, K, xstride):
    lib, b, N = pib.load(), 4, 300
    q, s, g = matrix(torch, N, K, K)
    ld = xstride or K
    x, x2 = torch.randn(b, ld, device="cuda", generator=g), torch.randn(b, ld, device="cuda", generator=g)
    add, nw = torch.randn(b, K, device="cuda", generator=g), torch.rand(K, device="cuda", generator=g) + 0.5
    w = pib.F8Weight(lib, q.data_ptr(), s.data_ptr(), N, K)
    y, out = torch.empty(b, N, device="cuda"), torch.empty(b, K, device="cuda")

    def close(ref_in):
        # the prologue's own roundings move a value across an e4m3 border now and then: one step (2^-4 of the value, half of it either way from the border) of one element at a time
        ref, lim = want(torch, q, s, ref_in.float().contiguous())
        step = (ref_in.abs().amax(1, keepdim=True) / 448 * 32) * dense(torch, q, s).abs().amax()
        assert ((y.double() - ref).abs() <= lim + 2 * step).all()
        assert ((y.double() - ref).abs() <= lim).double().mean() > 0.5

    lib.gemv_fused(w, x.data_ptr(), b, y.data_ptr(), prologue=1, x2=nw.data_ptr(), addend=add.data_ptr(), sum_out=out.data_ptr(), xstride=xstride, eps=1e-6)
    sm = x[:, :K] + add
    torch.cuda.synchronize()
    assert torch.equal(out, sm)
    close(sm.double() / (sm.double().pow(2).mean(1, keepdim=True) + 1e-6).sqrt() * nw.double())
    lib.gemv_fused(w, x.data_ptr(), b, y.data_ptr(), prologue=2, x2=x2.data_ptr(), xstride=xstride)
    close((x.double() / (1 + torch.exp(-x.double())) * x2.double())[:, :K])
    lib.gemv_fused(w, x.data_ptr(), b, y.data_ptr(), xstride=xstride)
    ref, lim = want(torch, q, s, x[:, :K].contiguous())
    torch.cuda.synchronize()
    assert ((y.double() - ref).abs() <= lim).all()


def test_rows_and_host_forms(torch, pib):
    lib, N, K = pib.load(), 300, 1001
    q, s, g = matrix(torch, N, K, 9)
    W = dense(torch, q, s)
    qh, sh = q.view(torch.uint8).cpu().numpy(), s.cpu().numpy()
    h = lib.L.pib_weight_upload_f8(qh.ctypes.data, sh.ctypes.data, N, K)
    assert h and lib.L.pib_weight_bytes(h) == N * K + 4 * sh.size
    for r in (0, 127, 128, 299):
        raw = np.zeros(K + 4 * blocks(K), np.uint8)
        lib.check(lib.L.pib_weight_row_blocks(h, r, raw.ctypes.data))
        assert np.array_equal(raw[:K], qh[r]) and np.array_equal(raw[K:].copy().view(np.float32), sh[r // 128])
    ids = [0, 299, 128, 5, 5]
    assert np.array_equal(lib.get_rows(h, ids, K), W[ids].float().cpu().numpy())
    for b, fn in ((5, lambda x, y: lib.L.pib_mul_mat_host(h, x.ctypes.data, x.shape[0], y.ctypes.data, 0)), (40, lambda x, y: lib.L.pib_gemm_host(h, x.ctypes.data, x.shape[0], y.ctypes.data))):
        x = rows(torch, b, K, g)
        y = np.zeros((b, N), np.float32)
        lib.check(fn(x.cpu().numpy(), y))
        ref, lim = want(torch, q, s, x)
        assert (np.abs(y - ref.cpu().numpy()) <= lim.cpu().numpy()).all()
    lib.L.pib_weight_free(h)


@pytest.mark.parametrize("how,b", [("fused", 2), ("gemv", 9), ("gemm", 70)])
def test_captured_and_on_another_stream(torch, pib, how, b):
    """the first call on a stream may be a captured one; replays follow new inputs; a call on a stream is ordered with what is on it"""
    lib, N, K = pib.load(), 520, 900
    q, s, g = matrix(torch, N, K, 3)
    w = pib.F8Weight(lib, q.data_ptr(), s.data_ptr(), N, K)
    x, y = rows(torch, b, K, g), torch.zeros(b, N, device="cuda")
    act = torch.empty(lib.act_bytes(F8, K, b), dtype=torch.uint8, device="cuda")

    def call(stream):
        if how == "fused":
            return lib.gemv_fused(w, x.data_ptr(), b, y.data_ptr(), stream)
        lib.quantize_act_rows(F8, x.data_ptr(), b, K, act.data_ptr(), stream)
        lib.gemv(w, act.data_ptr(), b, y.data_ptr(), stream) if how == "gemv" else lib.gemm(w, act.data_ptr(), b, y.data_ptr(), None, stream)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        call(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        x.copy_(rows(torch, b, K, g))
        graph.replay()
        torch.cuda.synchronize()
        ref, lim = want(torch, q, s, x)
        assert ((y.double() - ref).abs() <= lim).all()
    with torch.cuda.stream(torch.cuda.Stream()):
        x.mul_(0.5)
        y.zero_()
        call(torch.cuda.current_stream().cuda_stream)
        z = y * 2
    torch.cuda.synchronize()
    assert ((z.double() - ref).abs() <= lim).all()


def test_rows_that_are_not_there(torch, pib):
    lib, N, K = pib.load(), 300, 260
    q, s, g = matrix(torch, N, K, 11)
    w = pib.F8Weight(lib, q.data_ptr(), s.data_ptr(), N, K)
    ids = torch.tensor([-1, 0, N, 299, 0x7fffffff, -0x80000000], dtype=torch.int32, device="cuda")
    out = torch.full((6, K), float("nan"), device="cuda")
    lib.check(lib.L.pib_get_rows(w.h, ids.data_ptr(), 6, out.data_ptr(), None))
    torch.cuda.synchronize()
    W = dense(torch, q, s)
    assert torch.equal(out[[1, 3]], W[[0, 299]].float()) and not out[[0, 2, 4, 5]].any()


# outputs that fill the last CTA's, the last tile's or the last run's rows by one, and few rows in many shares
@pytest.mark.parametrize("N,K,b", [(148 * 32 + 1, 300, 9), (148 * 96 - 31, 257, 16), (148 * 160 + 5, 130, 17), (19000, 129, 32), (148 * 128 + 1, 260, 33), (148 * 128 - 127, 128, 48), (20001, 385, 49), (31, 4100, 96),
                                     (33, 2049, 97), (9500, 1100, 128)])
def test_divided_rows(torch, pib, N, K, b):
    q, s, g = matrix(torch, N, K, N + b)
    x = rows(torch, b, K, g)
    w = pib.F8Weight(pib.load(), q.data_ptr(), s.data_ptr(), N, K)
    ref, lim = want(torch, q, s, x)
    y = product(torch, pib, w, x, "gemm")
    torch.cuda.synchronize()
    assert ((y.double() - ref).abs() <= lim).all()
    assert torch.equal(product(torch, pib, w, x, "gemm"), y)


def test_more_than_four_gigabytes(torch, pib):
    """offsets of rows, and of outputs, that 32 bits do not hold"""
    lib, N, K = pib.load(), 530000, 8192
    g = torch.Generator(device="cuda").manual_seed(5)
    q = torch.randint(0, 120, (N, K), device="cuda", generator=g, dtype=torch.uint8).view(torch.float8_e4m3fn)
    s = (torch.rand(blocks(N), blocks(K), device="cuda", generator=g) + 0.5) / 96
    w = pib.F8Weight(lib, q.data_ptr(), s.data_ptr(), N, K)
    for how, b in (("fused", 1), ("gemv", 3), ("gemm", 20), ("gemm", 70), ("gemm", 200)):
        x = rows(torch, b, K, g)
        y = product(torch, pib, w, x, how)
        torch.cuda.synchronize()
        for r0 in (0, 262144 - 128, N // 128 * 128 - 256):        # whole blocks of rows
            r1 = min(N, r0 + 512)
            ref, lim = want(torch, q[r0:r1], s[r0 // 128:blocks(r1)], x)
            assert ((y[:, r0:r1].double() - ref).abs() <= lim).all(), (how, b, r0)
    ids = torch.tensor([N - 1, 262144, 524289], dtype=torch.int32, device="cuda")
    out = torch.empty(3, K, device="cuda")
    lib.check(lib.L.pib_get_rows(w.h, ids.data_ptr(), 3, out.data_ptr(), None))
    torch.cuda.synchronize()
    for i, r in enumerate(ids.tolist()):
        assert torch.equal(out[i], dense(torch, q[r:r + 1], s[r // 128:r // 128 + 1])[0].float())


@pytest.mark.parametrize("b", [3, 12])
def test_host_forms_report_a_wait_that_ran_out(torch, pib, b):
    """the error word of the stream is written here in a kernel's place"""
    import subprocess
    lib = pib.load()
    names = subprocess.run(["nm", "-D", "--defined-only", pib.SO_PATH], capture_output=True, text=True, check=True).stdout.split()
    word = getattr(lib.L, next(n for n in names if "pib_tc_error_word" in n))
    word.restype, word.argtypes = C.c_void_p, [C.c_void_p]
    q, s, g = matrix(torch, 300, 260, 5)
    w = pib.F8Weight(lib, q.data_ptr(), s.data_ptr(), 300, 260)
    x, y, seven = np.ones((b, 260), np.float32), np.zeros((b, 300), np.float32), np.array([7], np.int32)
    for fn in (lambda: lib.L.pib_mul_mat_host(w.h, x.ctypes.data, b, y.ctypes.data, 0), lambda: lib.L.pib_gemm_host(w.h, x.ctypes.data, b, y.ctypes.data)):
        assert fn() == 0
        lib.check(lib.L.pib_memcpy_h2d(word(None), seven.ctypes.data, 4, None))
        assert fn() == -1 and b"block 6" in lib.L.pib_last_error()
        assert fn() == 0


def test_fused_outputs_over_inputs_are_refused(torch, pib):
    lib, N, K, b = pib.load(), 256, 256, 3
    q, s, g = matrix(torch, N, K, 9)
    w = pib.F8Weight(lib, q.data_ptr(), s.data_ptr(), N, K)
    buf = torch.randn(8, b, 400, device="cuda", generator=g)
    x, x2, add, out, y = (buf[i].data_ptr() for i in range(5))
    call = lambda pro, x, x2, add, out, y, xs=400: lib.L.pib_gemv_fused(w.h, pro, x, x2, add, out, xs, 1e-5, b, y, None)
    for args in ((0, x, None, None, None, x), (0, x, None, None, None, x + 255 * 4), (0, x, None, None, None, x + 801 * 4), (0, x + 800 * 4, None, None, None, x + 33 * 4), (1, x, x2, add, out, x2 + 1020),
                 (1, x, x2, add, out, add), (1, x, x2, add, x + 4, y), (1, x, x2, add, add, y), (1, x, x2, add, x2, y), (2, x, x2, None, None, x2 + 1200 * 4 - 600), (0, x, None, None, None, y, -400)):
        assert call(*args) == -2 and b"pib_gemv_fused" in lib.L.pib_last_error(), args
    for args in ((0, x, None, None, None, x + 1200 * 4), (1, x, x2, add, out, y), (2, x, x2, None, None, y), (0, x, None, None, None, x + 256 * 4, 1100)):          # the last one between two rows of x
        assert call(*args) == 0, args
    torch.cuda.synchronize()


@pytest.mark.parametrize("N,K,b", [(50, 28672, 4), (300, 28672, 8), (2500, 13000, 8), (33, 26000, 5), (129, 66000, 1), (40, 66000, 2), (17, 66001, 8), (5000, 14336, 7), (60, 28672, 13), (60, 28672, 150)])
def test_many_columns(torch, pib, N, K, b):
    """decode batches whose activations do not fit beside the ring and come with the weights; more than 32 steps of a tile, whose scales are asked for again; the same columns for more tokens"""
    q, s, g = matrix(torch, N, K, N + K)
    x = rows(torch, b, K, g)
    w = pib.F8Weight(pib.load(), q.data_ptr(), s.data_ptr(), N, K)
    y, lim = want(torch, q, s, x)
    how = "gemv" if b <= 16 else "gemm"
    got = product(torch, pib, w, x, how)
    err = (got.double() - y).abs()
    assert (err <= lim).all(), float((err / lim).max())
    for _ in range(3):
        assert torch.equal(product(torch, pib, w, x, how), got)


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_one_bad_token_of_many_columns(torch, pib, bad):
    q, s, g = matrix(torch, 70, 28672, 6)
    x = rows(torch, 6, 28672, g)
    x[2, 20000] = bad
    w = pib.F8Weight(pib.load(), q.data_ptr(), s.data_ptr(), 70, 28672)
    got = product(torch, pib, w, x, "gemv")
    y, lim = want(torch, q, s, x)
    others = [0, 1, 3, 4, 5]
    assert ((got[others].double() - y[others]).abs() <= lim[others]).all() and torch.isnan(got[2]).all()
