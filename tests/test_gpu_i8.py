"""8-bit integer weights with a scale per output (csrc/i8_quant.cu, i8_gemv.cu, i8_gemm.cu) against whole-number sums: sizes that fill no tile and no share, every number of tokens where another
kernel or tile begins, the largest sums, infinities and numbers that are none in one token, fused prologues, captured calls, other streams.  An output is fp32(sum) * fp32(d * s), each rounded once:
all bits are compared."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
I8 = 65


@pytest.fixture(scope="module")
def pib():
    from pipeinfer_b200 import lib as pib
    pib.load().init(0)
    return pib


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


def matrix(torch, N, K, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(-128, 128, (N, K), device="cuda", generator=g, dtype=torch.int8)
    return q, (torch.rand(N, device="cuda", generator=g) + 0.5) / 64, g


def rows(torch, b, K, g):
    x = torch.randn(b, K, device="cuda", generator=g)
    x[:, ::37] *= 20
    return x


def rounded(torch, x):
    """whole numbers and scales, by their definition"""
    d = x.abs().amax(1).clamp(min=2.0 ** -100) * float(np.float32(1) / np.float32(127))
    return torch.round(x / d.unsqueeze(1)).clamp(-127, 127), d


def want(torch, q, s, x):
    a, d = rounded(torch, x)
    total = a.double() @ q.double().T                    # whole numbers below 2^53
    return total.float() * (d.unsqueeze(1) * s)


def product(torch, pib, w, x, how, stream=0, y=None):
    lib, (b, K) = pib.load(), x.shape
    if y is None:
        y = torch.full((b, w.N), float("nan"), device="cuda")
    if how == "fused":
        lib.gemv_fused(w, x.data_ptr(), b, y.data_ptr(), stream)
        return y
    act = torch.empty(lib.act_bytes(I8, K, b), dtype=torch.uint8, device="cuda")
    (lib.quantize_act_dev if how == "gemv" else lib.quantize_act_rows)(I8, x.data_ptr(), b, K, act.data_ptr(), stream)
    if how == "gemv":
        lib.gemv(w, act.data_ptr(), b, y.data_ptr(), stream)
    else:
        lib.gemm(w, act.data_ptr(), b, y.data_ptr(), None, stream)
    lib.gemm_check(stream)
    return y


def handle(pib, q, s):
    return pib.I8Weight(pib.load(), q.data_ptr(), s.data_ptr(), *q.shape)


def blocks(torch, pib, act, b, K):
    Kp = (K + 127) // 128 * 128
    out = np.zeros((b, 4 + Kp), np.uint8)
    pib.load().check(pib.load().L.pib_act_to_blocks(I8, act.data_ptr(), b, K, out.ctypes.data))
    return out[:, 4:].view(np.int8), out[:, :4].copy().view(np.float32)[:, 0]


@pytest.mark.parametrize("b,K", [(1, 1), (1, 128), (3, 127), (5, 129), (16, 1000), (17, 4096), (300, 260), (2, 8193), (3, 20000), (1, 131072)])
def test_quantiser(torch, pib, b, K):
    """bytes and scales as defined; rows of zeros, of values far below and near the end of fp32"""
    lib = pib.load()
    g = torch.Generator(device="cuda").manual_seed(b * 7 + K)
    x = rows(torch, b, K, g)
    if b >= 3:
        x[1] = 0
        x[2] *= 1e-36
        x[0] = x[0].clamp(-2, 2) * 1.5e38
    act = torch.empty(lib.act_bytes(I8, K, b), dtype=torch.uint8, device="cuda")
    lib.quantize_act_rows(I8, x.data_ptr(), b, K, act.data_ptr())
    a, d = rounded(torch, x)
    got, scale = blocks(torch, pib, act, b, K)
    assert np.array_equal(scale, d.cpu().numpy())
    assert np.array_equal(got[:, :K], a.to(torch.int8).cpu().numpy()) and not got[:, K:].any()


@pytest.mark.parametrize("b,K", [(1, 128), (4, 1000), (16, 5632), (2, 9000)])
def test_quantiser_behind_a_norm(torch, pib, b, K):
    lib = pib.load()
    g = torch.Generator(device="cuda").manual_seed(K)
    x, w = rows(torch, b, K, g), torch.rand(K, device="cuda", generator=g) + 0.5
    act, xn = torch.empty(lib.act_bytes(I8, K, b), dtype=torch.uint8, device="cuda"), torch.empty(b, K, device="cuda")
    lib.check(lib.L.pib_norm_quantize_act(I8, 1, x.data_ptr(), w.data_ptr(), 1e-5, b, K, act.data_ptr(), xn.data_ptr(), None))
    torch.cuda.synchronize()
    ref = x.double() / (x.double().pow(2).mean(1, keepdim=True) + 1e-5).sqrt() * w.double()
    # the mean's sum of K / 256 + 8 fp32 additions in a thread's chain, halved by the root; three roundings behind it
    assert ((xn.double() - ref).abs() <= ref.abs() * ((K / 256 + 16) / 2 + 6) * 2.0 ** -24).all()
    a, d = rounded(torch, xn)
    got, scale = blocks(torch, pib, act, b, K)
    assert np.array_equal(got[:, :K], a.to(torch.int8).cpu().numpy()) and np.array_equal(scale, d.cpu().numpy())


SIZES = [(1, 1), (16, 128), (17, 129), (127, 1000), (128, 256), (129, 2048), (1000, 5700), (2560, 2048), (10000, 640), (40, 20000)]


@pytest.mark.parametrize("N,K", SIZES)
@pytest.mark.parametrize("b", [1, 2, 3, 7, 8, 9, 13, 16])
def test_decode_batches(torch, pib, N, K, b):
    q, s, g = matrix(torch, N, K, N + K)
    x = rows(torch, b, K, g)
    w = handle(pib, q, s)
    y = want(torch, q, s, x)
    for how in ["gemv", "gemm"] + (["fused"] if b <= 8 and K <= 8192 else []):
        assert torch.equal(product(torch, pib, w, x, how), y), how


@pytest.mark.parametrize("N,K,b", [(1, 1, 1), (16, 128, 20), (130, 129, 33), (128, 256, 16), (257, 1000, 65), (300, 5700, 100), (2560, 2048, 129), (1000, 640, 256), (640, 1300, 257), (384, 8192, 40),
                                   (1100, 2000, 700), (20000, 256, 31), (19000, 128, 300), (5000, 3000, 513), (2048, 4096, 49), (600, 20000, 70), (22000, 384, 97)])
def test_prompts(torch, pib, N, K, b):
    q, s, g = matrix(torch, N, K, N + K)
    x = rows(torch, b, K, g)
    assert torch.equal(product(torch, pib, handle(pib, q, s), x, "gemm"), want(torch, q, s, x))


@pytest.mark.parametrize("b", [1, 12, 100, 300])
def test_largest_sums(torch, pib, b):
    """every product 128 * 127 in the longest rows that there are: nearly 2^31"""
    K = 131072
    q, s = torch.full((5, K), -128, dtype=torch.int8, device="cuda"), torch.ones(5, device="cuda")
    x = torch.full((b, K), -3.0, device="cuda")
    y = product(torch, pib, handle(pib, q, s), x, "gemv" if b <= 16 else "gemm")
    assert torch.equal(y, want(torch, q, s, x)) and float(y[0, 0]) > 0


@pytest.mark.parametrize("b", [1, 5, 12, 40, 130])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_rows_that_are_no_numbers(torch, pib, b, bad):
    q, s, g = matrix(torch, 300, 1000, b)
    x = rows(torch, b, 1000, g)
    y = want(torch, q, s, x)
    x[b // 2, 997] = bad
    y[b // 2] = float("nan")
    w = handle(pib, q, s)
    for how in (["gemv"] if b <= 16 else []) + ["gemm"] + (["fused"] if b <= 8 else []):
        got = product(torch, pib, w, x, how)
        assert torch.equal(got.isnan(), y.isnan()) and torch.equal(got.nan_to_num(0), y.nan_to_num(0)), how


@pytest.mark.parametrize("N,K,b", [(100, 1000, 1), (2560, 2048, 4), (257, 8192, 8)])
def test_fused_prologues(torch, pib, N, K, b):
    """the same outputs, up to one step of a rounded activation, as the prologue's result through the quantiser"""
    lib = pib.load()
    q, s, g = matrix(torch, N, K, N)
    w, dense = handle(pib, q, s), q.double().abs()
    x, x2, add = rows(torch, b, K, g), torch.rand(K, device="cuda", generator=g) + 0.5, rows(torch, b, K, g)
    y, total = torch.empty(b, N, device="cuda"), torch.empty(b, K, device="cuda")
    lib.gemv_fused(w, x.data_ptr(), b, y.data_ptr(), prologue=1, x2=x2.data_ptr(), addend=add.data_ptr(), sum_out=total.data_ptr(), eps=1e-5)
    torch.cuda.synchronize()
    assert torch.equal(total, x + add)
    cases = [(y.clone(), (total.double() / (total.double().pow(2).mean(1, keepdim=True) + 1e-5).sqrt() * x2.double()).float())]
    gu = torch.randn(b, 2 * K, device="cuda", generator=g)
    lib.gemv_fused(w, gu.data_ptr(), b, y.data_ptr(), prologue=2, x2=gu[:, K:].data_ptr(), xstride=2 * K)
    torch.cuda.synchronize()
    cases.append((y, (gu[:, :K].double() * torch.sigmoid(gu[:, :K].double()) * gu[:, K:].double()).float()))
    for got, v in cases:
        # a value that the prologue forms with another rounding (2^-19 of it: sums of 16 values a thread, root, product) moves a whole number by one where its quotient lies within that of a half
        a, d = rounded(torch, v)
        edge = ((v / d.unsqueeze(1)).abs() % 1 - 0.5).abs() < 127 * 2.0 ** -18
        lim = (edge.double() @ dense.T) * d.double().unsqueeze(1) * s.double() + want(torch, q, s, v).double().abs() * 2.0 ** -18 + 1e-30
        assert ((got.double() - want(torch, q, s, v).double()).abs() <= lim).all()


def test_rows_and_weights(torch, pib):
    lib = pib.load()
    q, s, _ = matrix(torch, 300, 1000, 3)
    w = handle(pib, q, s)
    ids = torch.tensor([0, 299, 7, -1, 300, 128], dtype=torch.int32, device="cuda")
    out = torch.full((6, 1000), float("nan"), device="cuda")
    lib.check(lib.L.pib_get_rows(w.h, ids.data_ptr(), 6, out.data_ptr(), None))
    torch.cuda.synchronize()
    ref = q.float() * s.unsqueeze(1)
    assert torch.equal(out[[0, 1, 2, 5]], ref[[0, 299, 7, 128]]) and not out[3:5].any()
    row = np.zeros(1004, np.uint8)
    lib.check(lib.L.pib_weight_row_blocks(w.h, 131, row.ctypes.data))
    assert np.array_equal(row[:1000].view(np.int8), q[131].cpu().numpy()) and row[1000:].copy().view(np.float32)[0] == float(s[131])
    assert lib.L.pib_weight_bytes(w.h) == 300 * 1000 + 4 * 300
    qh, sh, x = q.cpu().numpy(), s.cpu().numpy(), torch.randn(40, 1000)          # (they live as long as the calls that read them)
    h, xh = lib.L.pib_weight_upload_i8(qh.ctypes.data, sh.ctypes.data, 300, 1000), x.numpy()
    y, z = np.zeros((9, 300), np.float32), np.zeros((40, 300), np.float32)
    lib.check(lib.L.pib_mul_mat_host(h, xh.ctypes.data, 9, y.ctypes.data, 0))
    lib.check(lib.L.pib_gemm_host(h, xh.ctypes.data, 40, z.ctypes.data))
    lib.L.pib_weight_free(h)
    ref = want(torch, q, s, x.cuda()).cpu().numpy()
    assert np.array_equal(y, ref[:9]) and np.array_equal(z, ref)


@pytest.mark.parametrize("b", [1, 9, 33, 200])
def test_captured_and_on_another_stream(torch, pib, b):
    q, s, g = matrix(torch, 1000, 1100, b)
    w, x = handle(pib, q, s), rows(torch, b, 1100, g)
    lib, y = pib.load(), torch.empty(b, 1000, device="cuda")
    act = torch.empty(lib.act_bytes(I8, 1100, b), dtype=torch.uint8, device="cuda")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())

    def call():
        lib.quantize_act_rows(I8, x.data_ptr(), b, 1100, act.data_ptr(), st.cuda_stream)
        lib.gemm(w, act.data_ptr(), b, y.data_ptr(), None, st.cuda_stream)
    with torch.cuda.stream(st):
        call()
    st.synchronize()
    assert torch.equal(y, want(torch, q, s, x))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        call()
    for i in range(3):
        x.copy_(rows(torch, b, 1100, g))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want(torch, q, s, x))
    lib.gemm_check(st.cuda_stream)


def test_offsets_past_32_bits(torch, pib):
    """a matrix of more than 2^32 bytes: its last rows"""
    N, K = 70000, 65536
    q = torch.empty(N, K, dtype=torch.int8, device="cuda")
    q[:-200] = 1
    q[-200:] = torch.randint(-128, 128, (200, K), device="cuda", dtype=torch.int8)
    s = torch.rand(N, device="cuda") + 0.5
    w = handle(pib, q, s)
    for b in (2, 20, 150):
        x = torch.randn(b, K, device="cuda")
        y = product(torch, pib, w, x, "gemv" if b <= 16 else "gemm")
        assert torch.equal(y[:, -200:], want(torch, q[-200:], s[-200:], x)) and torch.equal(y[:, :10], want(torch, q[:10], s[:10], x))
