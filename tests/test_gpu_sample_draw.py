"""Tokens drawn on the device (csrc/sample_draw.cu) against numpy in 64 bits: every truncation alone and together, rows divided over 1 to 8 blocks, equal logits at every border, thresholds inside
bins of thousands of tokens, rows in which nothing or almost nothing takes part, infinities, given numbers at both ends, strides, captured calls; the frequencies of many draws."""
import ctypes as C
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pib():
    from pipeinfer_b200 import lib as pib
    pib.load().init(0)
    return pib


def draw(pib, x, params, u, bf16=False, ld=None):
    lib = pib.load()
    rows, V = x.shape
    ld = ld or V
    buf = np.full((rows, ld), 1e30, np.float32)
    buf[:, :V] = x
    if bf16:
        buf = (np.ascontiguousarray(buf).view(np.uint32) >> 16).astype(np.uint16)
    p = np.zeros(rows, np.dtype([("temp", "f4"), ("top_k", "i4"), ("top_p", "f4"), ("min_p", "f4")]))
    for i in range(rows):
        p[i] = params[i]
    d, dp, du = lib.to_device(buf), lib.to_device(p), lib.to_device(np.asarray(u, np.float32))
    out = [lib.to_device(np.full(rows + 1, 77, t)) for t in (np.int32, np.float32, np.int32)]
    lib.sample(lib.TYPE_BF16 if bf16 else lib.TYPE_F32, d, ld, rows, V, dp, du, *out)
    res = [lib.to_host(o, rows + 1, t) for o, t in zip(out, (np.int32, np.float32, np.int32))]
    assert all(r[rows] == 77 for r in res)
    for q in [d, dp, du] + out:
        lib.free(q)
    return [r[:rows] for r in res]


def want(row, params, u):
    """id, share and number of kept tokens, from the definition"""
    T, k, P, m = (float(np.float32(params[0])), int(params[1]), float(np.float32(params[2])), float(np.float32(params[3])))
    row = row.astype(np.float64)
    row = np.where(np.isnan(row), -np.inf, row)
    mx = row.max()
    if mx == -np.inf:
        return -1, 0.0, 0
    if mx == np.inf:
        row = np.where(row == np.inf, 0.0, -np.inf)
    order = np.lexsort((np.arange(len(row)), -row))
    order = order[row[order] > -np.inf]
    if k > 0:
        order = order[:k]
    w = np.exp(row[order] - row[order[0]])
    if P < 1:
        c = np.cumsum(w)
        order = order[:max(1, 1 + int(np.searchsorted(c, P * c[-1], side="left")))]
    if m > 0:
        ok = np.exp(row[order] - row[order[0]]) >= m
        ok[0] = True
        order = order[ok]
    if not T > 0:
        order = order[:1]
    n = len(order)
    order = np.sort(order)
    w = np.exp((row[order] - row[order].max()) / (T if T > 0 else 1.0))
    c = np.cumsum(w)
    i = min(int(np.searchsorted(c, float(np.float32(u)) * c[-1], side="right")), n - 1)
    return int(order[i]), w[i] / c[-1], n


def compare(pib, x, params, u, **kw):
    ids, p, kept = draw(pib, x, params, u, **kw)
    for r in range(x.shape[0]):
        i, share, n = want(x[r], params[r], u[r])
        assert (ids[r], kept[r]) == (i, n), (r, params[r], u[r], ids[r], i, kept[r], n)
        assert abs(p[r] - share) <= 2.0 ** -23 * share + 1e-9, (r, p[r], share)      # one rounding to fp32, weights to 2^-45 of the largest


PARAMS = [(1.0, 0, 1.0, 0.0), (0.7, 40, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.1), (0.8, 40, 0.95, 0.05), (0.0, 0, 0.9, 0.0), (1.0, 1, 0.5, 0.0), (2.0, 1000, 0.5, 0.001), (0.05, 0, 0.999, 0.0),
          (1.0, 3, 0.999999, 0.0), (5.0, 100000, 0.3, 0.0), (1.0, 0, 0.0, 0.0), (-1.0, 7, 0.2, 0.2), (1.0, 0, 1.0, 1.0)]


@pytest.mark.parametrize("rows,V", [(1, 1), (2, 2), (3, 31), (1, 513), (5, 2048), (14, 4097), (1, 32000), (28, 32000), (1, 128256), (9, 151000), (70, 65000), (300, 1500), (1, 262144), (150, 20001)])
@pytest.mark.parametrize("kind", ["normal", "ties", "bf16"])
def test_against_numpy(pib, rows, V, kind):
    rng = np.random.default_rng(rows * 1000 + V)
    x = (rng.standard_normal((rows, V)) * 2.5).astype(np.float32)
    if kind == "ties":
        x = np.round(x)
    if kind == "bf16":
        x = (x.view(np.uint32) & np.uint32(0xffff0000)).view(np.float32)
    x[:, rng.integers(0, V, max(1, V // 50))] = -np.inf
    params = [PARAMS[(r + V) % len(PARAMS)] for r in range(rows)]
    compare(pib, x, params, rng.random(rows, np.float32), bf16=kind == "bf16")


@pytest.mark.parametrize("V", [3000, 40000, 262144])
def test_equal_logits(pib, V):
    """all equal, two values, and a bin of the histogram that holds nearly everything: borders inside runs of equal tokens go by the id"""
    rng = np.random.default_rng(V)
    x = np.zeros((8, V), np.float32)
    x[2:4] = rng.integers(0, 2, (2, V)) * -0.5
    x[4:6] = rng.integers(0, 1000, (2, V)) * np.float32(1e-6)
    x[6] = -0.0
    x[6, ::2] = 0.0
    x[7] = (rng.random(V) * 1e-3).astype(np.float32)
    params = [(1.0, V // 2 + 1, 1.0, 0.0), (0.5, 0, 0.3, 0.0), (1.0, V // 3, 0.5, 0.0), (1.0, 0, 0.9, 0.0), (1.0, 777, 0.37, 0.0), (1.0, 0, 0.5001, 0.0), (1.0, V - 1, 0.25, 0.0), (1.0, 2500, 0.99, 0.0)]
    compare(pib, x, params, rng.random(8, np.float32))


def test_little_takes_part(pib):
    V = 9000
    x = np.full((12, V), -np.inf, np.float32)
    x[1, 5000] = -3.0
    x[2, [7, 8999]] = [1.0, 1.0]
    x[3] = np.nan
    x[4, [3, 4]] = [np.nan, -1e30]
    x[5, [10, 20]] = [np.inf, np.inf]; x[5, 30] = 5.0
    x[6, [10, 20]] = [3.0e38, -3.0e38]
    x[7, :] = -3.4e38
    x[8, 1] = np.inf; x[8, 2] = np.nan
    x[9, [1, 2, 3]] = [0.0, -31.0, -40.0]
    x[10, [1, 2, 3]] = [0.0, -31.0, -40.0]
    x[11, [100, 200]] = [1e-40, 0.0]
    params = [(1.0, 5, 0.9, 0.0)] * 8 + [(1.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.0), (40.0, 0, 1.0, 0.0), (1.0, 0, 0.5, 0.0)]
    for u in (0.0, 0.3, 0.5, 0.9999999):
        compare(pib, x, params, [u] * 12)
    compare(pib, x, [(1.0, 0, 1.0, 0.0)] * 12, [0.7] * 12)


def test_given_numbers_at_the_ends(pib):
    rng = np.random.default_rng(4)
    x = rng.standard_normal((6, 5000)).astype(np.float32)
    top = np.float32(1) - np.float32(2) ** -24
    compare(pib, x, [(1.0, 0, 1.0, 0.0), (1.0, 50, 0.9, 0.0)] * 3, [0.0, 0.0, top, top, 0.5, 0.25])
    ids, p, kept = draw(pib, x, [(1.0, 10, 1.0, 0.0)] * 6, [1.0, 7.0, -1.0, np.nan, np.inf, -np.inf])      # outside 0 <= u < 1: the last or the first kept token
    for r, last in enumerate([True, True, False, False, True, False]):
        best = np.sort(np.argsort(-x[r], kind="stable")[:10])
        assert ids[r] == best[-1 if last else 0]


def test_settings_that_are_no_numbers(pib):
    x = np.random.default_rng(5).standard_normal((4, 3000)).astype(np.float32)
    nan = float("nan")
    ids, p, kept = draw(pib, x, [(nan, 0, 1.0, 0.0), (1.0, 0, nan, 0.0), (1.0, 0, 1.0, nan), (float("inf"), 0, 1.0, 0.0)], [0.5] * 4)
    assert ids[0] == x[0].argmax() and kept[0] == 1
    assert kept[1] == kept[2] == kept[3] == 3000
    assert ids[3] == 1500 and abs(p[3] - 1 / 3000) < 1e-9


@pytest.mark.parametrize("bf16", [False, True])
def test_rows_apart(pib, bf16):
    rng = np.random.default_rng(6)
    x = rng.standard_normal((5, 1001)).astype(np.float32) * 3
    x = (x.view(np.uint32) & np.uint32(0xffff0000)).view(np.float32)
    compare(pib, x, [PARAMS[r] for r in range(5)], rng.random(5, np.float32), bf16=bf16, ld=1037)


def test_frequencies(pib):
    """draws with numbers spread evenly over 0 .. 1: each token comes as often as its share says, to one draw"""
    rng = np.random.default_rng(8)
    row, n = (rng.standard_normal(600) * 2).astype(np.float32), 20000
    ids, _, _ = draw(pib, np.tile(row, (n, 1)), [(0.9, 100, 0.95, 0.0)] * n, (np.arange(n) + 0.5) / n)
    order = np.argsort(-row, kind="stable")[:100]
    w = np.exp(row[order].astype(np.float64) - row.max())
    order = order[:1 + int(np.searchsorted(np.cumsum(w), np.float32(0.95) * w.sum()))]
    share = np.exp((row[order].astype(np.float64) - row.max()) / np.float32(0.9))
    share /= share.sum()
    got = np.bincount(ids, minlength=600)
    assert got.sum() == n and (np.abs(got[order] - share * n) <= 1.01).all()


def test_captured_and_on_another_stream(pib):
    torch = pytest.importorskip("torch")
    lib, rows, V = pib.load(), 5, 33000
    x = torch.randn(rows, V, device="cuda") * 3
    params = torch.tensor([[0.8, 0.0, 0.9, 0.0]] * rows, device="cuda")
    u = torch.rand(rows, device="cuda")
    ids, p, kept = (torch.zeros(rows, dtype=d, device="cuda") for d in (torch.int32, torch.float32, torch.int32))
    torch.cuda.synchronize()
    graph, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=st):
        lib.sample(lib.TYPE_F32, x.data_ptr(), V, rows, V, params.data_ptr(), u.data_ptr(), ids.data_ptr(), p.data_ptr(), kept.data_ptr(), torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        x.copy_(torch.randn(rows, V, device="cuda") * 3)
        u.copy_(torch.rand(rows, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        for r in range(rows):
            i, share, n = want(x[r].cpu().numpy(), (0.8, 0, 0.9, 0.0), float(u[r]))
            assert (int(ids[r]), int(kept[r])) == (i, n)
    with torch.cuda.stream(torch.cuda.Stream()):
        x.neg_()
        lib.sample(lib.TYPE_F32, x.data_ptr(), V, rows, V, params.data_ptr(), u.data_ptr(), ids.data_ptr(), None, None, torch.cuda.current_stream().cuda_stream)
        got = ids.clone()
    torch.cuda.synchronize()
    assert [int(v) for v in got] == [want(x[r].cpu().numpy(), (0.8, 0, 0.9, 0.0), float(u[r]))[0] for r in range(rows)]


def test_rows_far_apart(pib):
    """rows whose distance passes 32 bits, against the same rows side by side"""
    torch = pytest.importorskip("torch")
    lib, rows, V, ld = pib.load(), 4, 40001, 1500000001
    g = torch.Generator(device="cuda").manual_seed(1)
    x = (torch.randn(rows, V, device="cuda", generator=g) * 3).bfloat16()
    far = torch.empty((rows - 1) * ld + V, dtype=torch.bfloat16, device="cuda")
    for r in range(rows):
        far[r * ld:r * ld + V] = x[r]
    p = np.array([(0.8, 40, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.1), (1.0, 0, 1.0, 0.0)], [("temp", "f4"), ("top_k", "i4"), ("top_p", "f4"), ("min_p", "f4")])
    p = torch.from_numpy(p.view(np.uint8).copy()).cuda()
    u = torch.rand(rows, device="cuda", generator=g)
    out = []
    for t, d in ((x, V), (far, ld)):
        ids, pr, kept = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        lib.sample(lib.TYPE_BF16, t.data_ptr(), d, rows, V, p.data_ptr(), u.data_ptr(), ids.data_ptr(), pr.data_ptr(), kept.data_ptr(), 0)
        torch.cuda.synchronize()
        out.append((ids.tolist(), pr.tolist(), kept.tolist()))
    assert out[0] == out[1] and min(out[0][0]) >= 0


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("V", [1000, 20000, 70000])
def test_borders_beside_zero(pib, V, bf16):
    """thresholds in the bins above and below logit 0 behind a positive maximum, where 10^8 floats have the same difference to it: equal zeros, denormal numbers, some ulps and whole bins either side"""
    rng = np.random.default_rng(V)
    n = 900                                                      # tokens beside 0, as far apart as they go; the rest weighs nothing
    around = [np.zeros(n), rng.integers(-3, 4, n) * 1e-40, rng.integers(-2000, 2000, n) * 2.0 ** -24, (rng.random(n) - 0.5) / 64, rng.integers(-1, 2, n) / 256.0]
    x, params = [], []
    for mx, top_p in ((0.5, 0.5), (3.0, 0.5), (8.0, 0.9), (12.25, 0.998), (20.0, 0.999999)):
        for a in around:
            row = np.full(V, -1000.0)
            at = rng.permutation(V)[:n + 1]
            row[at[:n]], row[at[n]] = a, mx
            for p in ((1.0, 0, top_p, 0.0), (0.7, 600, 1.0, 0.0), (1.0, 700, top_p, 1e-9)):
                x.append(row)
                params.append(p)
    x = np.array(x, np.float32)
    if bf16:
        x = (x.view(np.uint32) & np.uint32(0xffff0000)).view(np.float32)
    u = rng.random(len(params), np.float32)
    for r in range(0, len(params), 25):                          # few rows at a time, so that long ones are divided
        compare(pib, x[r:r + 25], params[r:r + 25], u[r:r + 25], bf16=bf16)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("V", [700, 33000])
def test_min_p_beside_zero(pib, V, bf16):
    """min_p 1 and just below behind a maximum of 0 (shifted logits, a row of zeros, some infinities) and next to it, and borders at 0 behind a positive maximum"""
    rng = np.random.default_rng(V + 1)
    x = np.full((9, V), -7.0, np.float32)
    x[:, 5::7] = rng.random((9, len(range(5, V, 7)))) * -1e-3
    x[0, [3, 40, 600]] = 0.0
    x[1] = 0.0
    x[2, [9, 99, 350]] = np.inf
    x[3, 50] = 1e-38; x[3, 60] = -1e-38; x[3, 61] = 0.0
    x[4] = -0.0; x[4, ::3] = 0.0
    x[5, 11] = 0.0; x[5, 12:40] = -1e-17; x[5, 40:60] = -1e-45
    x[6, 7] = 1.0; x[6, 20:40] = 0.0
    x[7, 7] = 0.6931472; x[7, 20:40] = 0.0
    x[8, 7] = 2.0 ** -24; x[8, 20:40] = 0.0
    if bf16:
        x = (x.view(np.uint32) & np.uint32(0xffff0000)).view(np.float32)
    u = rng.random(9, np.float32)
    for m in (1.0, 0.99999994, 0.3678, 0.36788, 0.4999):
        for k, p in ((0, 1.0), (300, 1.0), (0, 0.7), (500, 0.8)):
            compare(pib, x, [(0.9, k, p, m)] * 9, u, bf16=bf16)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("V", [777, 5000, 70000])
@pytest.mark.filterwarnings("ignore:invalid value")
def test_no_numbers_among_the_logits(pib, V, bf16):
    """NaN of either sign and any payload takes no part: every truncation alone, thousands of equal logits, many NaN and few, at the borders of chunks"""
    rng = np.random.default_rng(V)
    x = (rng.standard_normal((6, V)) * 2).astype(np.float32)
    x[2:4] = np.round(x[2:4])
    x[4:] = 1.5
    x = (x.view(np.uint32) & np.uint32(0xffff0000)).view(np.float32)
    nans = np.array([0x7fc00000, 0xffc00000, 0x7f810000, 0xff810000, 0x7fff0000, 0xffff0000], np.uint32)
    for r in range(6):
        at = rng.permutation(V)[:V // 3] if r % 2 else [0, 7, 8, 255, 256, V - 1]
        x.view(np.uint32)[r, at] = nans[rng.integers(0, 6, len(at))]
    u = rng.random(6, np.float32)
    for p in ((1.0, 0, 0.9, 0.0), (0.7, 0, 0.6, 0.0), (1.0, 0, 1.0, 0.0), (1.0, 40, 1.0, 0.0), (0.8, 600, 0.9, 0.0), (1.2, 0, 1.0, 0.05), (1.0, 0, 0.99, 0.2), (0.0, 0, 0.5, 0.0)):
        compare(pib, x, [p] * 6, u, bf16=bf16)
