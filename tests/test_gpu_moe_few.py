"""A whole mixture layer for 1..16 tokens (csrc/moe_few.cu) against float64: both weight types, both scores, corrections, shared experts, sizes that fill no block or tile, one expert and many,
all tokens at one expert, strides, tokens that are no numbers, captured calls and calls at the same time."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu
F8, BF16 = 64, 30
EPS = 2.0 ** -24


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


class Layer:
    def __init__(self, torch, pib, typ, E, shared, top, D, F, score="softmax", renorm=True, scale=1.0, correction=False, seed=0):
        self.t, self.E, self.shared, self.top, self.D, self.F, self.score, self.renorm, self.scale, self.f8 = torch, E, shared, top, D, F, score, renorm, scale, typ == F8
        g = self.g = torch.Generator(device="cuda").manual_seed(seed + E * 31 + D + F)
        n, w = E + shared, {}
        for name, r, k in (("gate", F, D), ("up", F, D), ("down", D, F)):
            v = torch.randn(n, r, k, device="cuda", generator=g) / k ** 0.5
            if self.f8:
                w[name] = (v * k ** 0.5 * 96).clamp(-448, 448).to(torch.float8_e4m3fn)
                w[name + "_scales"] = (torch.rand(n, blocks(r), blocks(k), device="cuda", generator=g) + 0.5) / (96 * k ** 0.5)
            else:
                w[name] = v.bfloat16()
        w["router"] = torch.randn(E, D, device="cuda", generator=g) / D ** 0.5
        w["correction"] = torch.randn(E, device="cuda", generator=g) * 0.3 if correction else None
        self.w = w
        self.moe = pib.Moe(pib.load(), typ, E, shared, top, D, F, score=score, renorm=renorm, scale=scale, **{k: (v.data_ptr() if v is not None else None) for k, v in w.items()})

    def matrices(self, e):
        out = []
        for name, r, k in (("gate", self.F, self.D), ("up", self.F, self.D), ("down", self.D, self.F)):
            m = self.w[name][e].double()
            if self.f8:
                m = m * self.w[name + "_scales"][e].double().repeat_interleave(128, 0)[:r].repeat_interleave(128, 1)[:, :k]
            out.append(m)
        return out

    def want(self, x, res):
        """float64 outputs and the bound of an output's error.  A product of K terms: activations of 23 bits (2^-23), 16 steps of the tensor core per line that may cut (2^-22 each), the lines and
        warps added in fp32 (K / 512 + 16 steps of 2^-24 at most)."""
        t = self.t
        x, R = x.double(), self.w["router"].double()
        z = x @ R.T
        score = t.softmax(z, 1) if self.score == "softmax" else t.sigmoid(z)
        choice = score + (self.w["correction"].double() if self.w["correction"] is not None else 0)
        ids = t.sort(choice, dim=1, descending=True, stable=True)[1][:, :self.top]
        wt = t.gather(score, 1, ids)
        if self.renorm:
            wt = wt / (wt.sum(1, keepdim=True) + 1e-20)
        wt = wt * self.scale
        dz = ((x.abs() @ R.abs().T) * (self.D / 256 + 16) * EPS).amax(1)           # error of a logit; the scores move by at most twice that, and by the exponential's few roundings
        prod = lambda K: (66 + K / 512 + 16) * EPS
        y, lim = res.double().clone(), res.double().abs() * EPS
        for e in range(self.E + self.shared):
            f = t.where(ids == e, wt, 0).sum(1) if e < self.E else t.ones(x.shape[0], dtype=t.float64, device="cuda")
            if not (f != 0).any():
                continue
            G, U, Dn = self.matrices(e)
            g, u = x @ G.T, x @ U.T
            h = g * t.sigmoid(g) * u
            dh = prod(self.D) * (1.1 * u.abs() * (x.abs() @ G.abs().T) + (g * t.sigmoid(g)).abs() * (x.abs() @ U.abs().T)) + 6 * EPS * h.abs()
            o = h @ Dn.T
            y += f.unsqueeze(1) * o
            rel = (2 * dz + 30 * EPS if e < self.E else t.zeros_like(dz)).unsqueeze(1)
            lim += f.abs().unsqueeze(1) * (dh @ Dn.abs().T + prod(self.F) * (h.abs() @ Dn.abs().T) + (rel + 20 * EPS) * o.abs())
        return y, lim + 1e-30

    def run(self, x, res, ldx=None, ldy=None, stream=0, scratch=None, y=None):
        t, b = self.t, x.shape[0]
        sc = t.empty(self.moe.scratch_bytes(b), dtype=t.uint8, device="cuda").fill_(0xa5) if scratch is None else scratch
        y = t.full((b, self.D), float("nan"), device="cuda") if y is None else y
        self.moe.forward(x.data_ptr(), x.stride(0), b, None if res is None else res.data_ptr(), 0 if res is None else res.stride(0), y.data_ptr(), y.stride(0), sc.data_ptr(), stream)
        return y


def check(L, x, res, got):
    y, lim = L.want(x, res)
    err = (got.double() - y).abs()
    assert (err <= lim).all(), float((err / lim).max())
    return float((err / lim).max())


CASES = [(F8, 8, 0, 2, 256, 128, {}), (F8, 5, 1, 3, 1000, 700, dict(score="sigmoid", correction=True)), (F8, 1, 0, 1, 128, 16, {}), (F8, 64, 2, 6, 512, 384, dict(renorm=False, scale=2.5)),
         (F8, 130, 1, 8, 300, 130, dict(correction=True, renorm=False)), (F8, 3, 0, 3, 1, 1, {}), (F8, 512, 0, 16, 129, 33, {}), (F8, 4, 4, 4, 2048, 1408, dict(score="sigmoid")),
         (BF16, 8, 0, 2, 256, 128, {}), (BF16, 6, 1, 2, 1001, 333, dict(correction=True)), (BF16, 16, 1, 2, 2048, 1024, {}), (BF16, 40, 2, 5, 65, 700, dict(score="sigmoid", renorm=False)),
         (BF16, 2, 0, 1, 3, 17, {}), (F8, 16, 0, 4, 4100, 260, {})]


@pytest.mark.parametrize("b", [1, 3, 8, 9, 16])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v) for v in c[:6]))
def test_against_float64(torch, pib, case, b):
    typ, E, shared, top, D, F, kw = case
    L = Layer(torch, pib, typ, E, shared, top, D, F, **kw)
    x, res = torch.randn(b, D, device="cuda", generator=L.g), torch.randn(b, D, device="cuda", generator=L.g)
    got = L.run(x, res)
    torch.cuda.synchronize()
    pib.load().gemm_check(0)
    print("worst error %.2g of the bound" % check(L, x, res, got))
    for _ in range(3):
        assert torch.equal(L.run(x, res), got)


def test_large_and_small_activations(torch, pib):
    L = Layer(torch, pib, F8, 8, 1, 2, 512, 256)
    for f in (1e-12, 1e-3, 300.0):
        x = torch.randn(5, 512, device="cuda", generator=L.g) * f
        x[:, 7] *= 1000
        res = torch.zeros(5, 512, device="cuda")
        check(L, x, res, L.run(x, res))


def test_all_tokens_at_the_same_experts(torch, pib):
    L = Layer(torch, pib, F8, 32, 0, 4, 640, 512, correction=True)
    L.w["correction"].copy_(torch.where(torch.arange(32, device="cuda") % 8 == 3, 50.0, 0.0))
    L.moe = pib.Moe(pib.load(), F8, 32, 0, 4, 640, 512, renorm=True, **{k: v.data_ptr() for k, v in L.w.items()})
    x = torch.randn(16, 640, device="cuda", generator=L.g)
    res = torch.randn(16, 640, device="cuda", generator=L.g)
    check(L, x, res, L.run(x, res))


def test_equal_scores_go_to_the_lower_index(torch, pib):
    L = Layer(torch, pib, BF16, 40, 0, 3, 64, 32)
    L.w["router"][:] = L.w["router"][0]
    L.moe = pib.Moe(pib.load(), BF16, 40, 0, 3, 64, 32, renorm=True, **{k: (v.data_ptr() if v is not None else None) for k, v in L.w.items()})
    x = torch.randn(4, 64, device="cuda", generator=L.g)
    y = torch.zeros(4, 64, dtype=torch.float64, device="cuda")
    for e in range(3):
        G, U, Dn = L.matrices(e)
        g = x.double() @ G.T
        y += (g * torch.sigmoid(g) * (x.double() @ U.T)) @ Dn.T / 3
    got = L.run(x, None)
    assert (got.double() - y).abs().max() < 1e-5


@pytest.mark.parametrize("typ", [F8, BF16])
def test_strides_residual_in_place_and_without(torch, pib, typ):
    L = Layer(torch, pib, typ, 8, 1, 2, 300, 200)
    xs, rs = torch.randn(7, 333, device="cuda", generator=L.g), torch.randn(7, 400, device="cuda", generator=L.g)
    x, res = xs[:, 5:305], rs[:, 3:303]
    y, lim = L.want(x, res)
    keep = rs.clone()
    L.run(x, res, y=res)
    torch.cuda.synchronize()
    assert ((res.double() - y).abs() <= lim).all()
    assert torch.equal(rs[:, :3], keep[:, :3]) and torch.equal(rs[:, 303:], keep[:, 303:])
    zero = torch.zeros(7, 300, device="cuda")
    check(L, x, zero, L.run(x, None))


@pytest.mark.parametrize("typ", [F8, BF16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_one_bad_token(torch, pib, typ, bad):
    L = Layer(torch, pib, typ, 12, 1, 3, 260, 140)
    x, res = torch.randn(9, 260, device="cuda", generator=L.g), torch.randn(9, 260, device="cuda", generator=L.g)
    x[4, 17] = bad
    got = L.run(x, res)
    torch.cuda.synchronize()
    pib.load().gemm_check(0)
    others = [0, 1, 2, 3, 5, 6, 7, 8]
    check(L, x[others], res[others], got[others])
    assert not torch.isfinite(got[4]).any()


def test_refused(torch, pib):
    L = Layer(torch, pib, F8, 8, 0, 2, 256, 128)
    x, sc = torch.randn(17, 256, device="cuda"), torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    y = torch.empty_like(x)
    fwd = pib.load().L.pib_moe_forward
    ok = [L.moe.h, x.data_ptr(), 256, 4, None, 0, y.data_ptr(), 256, sc.data_ptr(), None]
    assert fwd(*ok) == 0
    for i, v in ((1, None), (3, 0), (3, 17), (6, None), (6, x.data_ptr()), (8, None), (8, sc.data_ptr() + 16), (2, 255), (7, 255)):
        bad = list(ok)
        bad[i] = v
        assert fwd(*bad) == -2, (i, v)
    assert fwd(*(ok[:4] + [x.data_ptr(), 200] + ok[6:])) == -2 and fwd(*(ok[:4] + [y.data_ptr(), 300] + ok[6:])) == -2
    assert L.moe.scratch_bytes(0) == 0 and L.moe.scratch_bytes(17) == 0


def test_captured_and_at_the_same_time(torch, pib):
    """two graphs of the same layer, each with its own scratch, replayed on two streams at once, beside eager calls on a third"""
    L = Layer(torch, pib, F8, 32, 1, 4, 512, 256)
    b = 6
    xs, rs, ys, sc, graphs, streams = [], [], [], [], [], []
    torch.cuda.synchronize()
    for i in range(2):
        xs.append(torch.randn(b, 512, device="cuda", generator=L.g)); rs.append(torch.randn(b, 512, device="cuda", generator=L.g)); ys.append(torch.zeros(b, 512, device="cuda"))
        sc.append(torch.empty(L.moe.scratch_bytes(b), dtype=torch.uint8, device="cuda"))
        torch.cuda.synchronize()
        streams.append(torch.cuda.Stream())
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i], stream=streams[i]):
            L.run(xs[i], rs[i], stream=torch.cuda.current_stream().cuda_stream, scratch=sc[i], y=ys[i])
    third, s3 = torch.cuda.Stream(), torch.empty(L.moe.scratch_bytes(b), dtype=torch.uint8, device="cuda")
    y3 = torch.zeros(b, 512, device="cuda")
    for rep in range(5):
        for i in range(2):
            xs[i].copy_(torch.randn(b, 512, device="cuda", generator=L.g))
        torch.cuda.synchronize()
        for _ in range(4):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay()
            L.run(xs[0], rs[1], stream=third.cuda_stream, scratch=s3, y=y3)
        torch.cuda.synchronize()
        for i in range(2):
            check(L, xs[i], rs[i], ys[i])
        check(L, xs[0], rs[1], y3)
    pib.load().gemm_check(third.cuda_stream)


def test_more_than_four_gigabytes(torch, pib):
    """experts whose weights lie beyond what 32 bits address"""
    L = Layer(torch, pib, F8, 256, 1, 3, 4096, 2048, correction=True)
    L.w["correction"].copy_(torch.where(torch.arange(256, device="cuda") % 83 == 5, 50.0, 0.0))          # 5, 88, 171, 254
    L.moe = pib.Moe(pib.load(), F8, 256, 1, 3, 4096, 2048, renorm=True, **{k: v.data_ptr() for k, v in L.w.items()})
    x = torch.randn(5, 4096, device="cuda", generator=L.g)
    res = torch.randn(5, 4096, device="cuda", generator=L.g)
    check(L, x, res, L.run(x, res))


def layer_of(torch, pib, gate, up, down, gs, us, ds, shared=0):
    """a layer of the given e4m3 values and block scales whose one chosen expert has the weight 1"""
    n, F, D = gate.shape
    L = Layer(torch, pib, F8, 1, n - 1, 1, D, F, renorm=False)
    for k, v in dict(gate=gate, up=up, down=down, gate_scales=gs, up_scales=us, down_scales=ds).items():
        assert L.w[k].shape == v.shape
        L.w[k] = v.contiguous()
    L.moe = pib.Moe(pib.load(), F8, 1, n - 1, 1, D, F, renorm=False, **{k: (v.data_ptr() if v is not None else None) for k, v in L.w.items()})
    return L


@pytest.mark.parametrize("b", [1, 4, 7, 16])
def test_single_products(torch, pib, b):
    """tokens with one value and rows of the down matrix with one weight: every output is one product of an h that is one product each of gate and up, so nothing but the operands' own roundings
    shows.  Experts whose rows differ by 2^9 within a block and by 2^12 between blocks, gates that close, outputs that bring small h back to the size of large ones."""
    t, F, D = torch, 700, 300
    g = t.Generator(device="cuda").manual_seed(b)
    e4 = lambda v: v.clamp(-448, 448).to(t.float8_e4m3fn)
    sign = lambda *s: t.randint(0, 2, s, device="cuda", generator=g) * 2.0 - 1
    gate = e4(sign(1, F, D) * 2.0 ** t.randint(-3, 9, (1, F, D), device="cuda", generator=g) * (1 + t.randint(0, 8, (1, F, D), device="cuda", generator=g) / 8))
    up = e4(sign(1, F, D) * 2.0 ** t.randint(-3, 9, (1, F, D), device="cuda", generator=g))
    j = t.randint(0, F, (D,), device="cuda", generator=g)                          # the h of each output
    down = t.zeros(1, D, F, device="cuda")
    down[0, t.arange(D, device="cuda"), j] = sign(D) * t.randint(1, 16, (D,), device="cuda", generator=g)
    down = e4(down)
    up_f = 2.0 ** t.randint(-6, 7, (blocks(F),), device="cuda", generator=g)       # of 128 rows of gate (up); of as many columns of down its inverse
    us = up_f.view(1, -1, 1).expand(1, blocks(F), blocks(D)).contiguous()
    ds = (1 / up_f).view(1, 1, -1).expand(1, blocks(D), blocks(F)).contiguous()
    gs = t.full((1, blocks(F), blocks(D)), 2.0 ** -4, device="cuda")
    L = layer_of(t, pib, gate, up, down, gs, us, ds)
    x = t.zeros(b, D, device="cuda")
    k = t.randint(0, D, (b,), device="cuda", generator=g)
    x[t.arange(b, device="cuda"), k] = t.randn(b, device="cuda", generator=g)
    got = L.run(x, None)
    t.cuda.synchronize()
    pib.load().gemm_check(0)
    G, U, Dn = L.matrices(0)
    gt, u = x.double() @ G.T, x.double() @ U.T
    h = gt * t.sigmoid(gt) * u
    y = h @ Dn.T
    # x enters with 2^-22 of itself (two roundings to fp16), g and u with that and a step or two of fp32 (2^-24 each, three each); silu moves by at most (1 + |g|) times as much where the gate
    # closes, and by the exponential's, the sum's and the quotient's roundings (2^-22 together); h's product; h enters with 2^-22, or with 2^-39 of its tile's largest; three steps of fp32 behind it
    eps = (4 + 3) * EPS
    dh = h.abs() * ((2 + gt.abs()) * eps + 4 * EPS + EPS)
    p = t.nn.functional.pad(h.abs(), (0, (16 - F % 16) % 16)).view(b, -1, 16)
    dh = dh + 4 * EPS * h.abs() + (p.amax(2, keepdim=True) * 2.0 ** -39).expand_as(p).reshape(b, -1)[:, :F]
    lim = dh @ Dn.abs().T + 3 * EPS * y.abs() + 1e-35
    err = (got.double() - y).abs()
    assert (err <= lim).all(), float((err / lim).max())


@pytest.mark.parametrize("down_too", [False, True])
@pytest.mark.parametrize("c", [1.0, 10.0, 100.0, 300.0, 10000.0])
def test_rows_of_unlike_size(torch, pib, c, down_too):
    """one block of gate rows and one of up rows larger by c, and the columns of down that read them smaller by as much: the root mean square error over all outputs.  A sum's partial sums are no
    larger than some three times their end; products of gate and up run through 4 steps of the tensor core that may cut (2^-22 each) and 20 fp32 steps at most, the same behind h:
    2 * 3 * (4 * 2^-22 + 20 * 2^-24) and the operands' 2^-22 twice are below 2^-16.4, were all of one sign; they are not, so 2^-17"""
    t, F, D = torch, 1408, 2048
    L0 = Layer(t, pib, F8, 1, 0, 1, D, F)
    w = {k: v.clone() for k, v in L0.w.items() if v is not None}
    w["gate_scales"][:, 2] *= c
    w["up_scales"][:, 5] *= c
    if down_too:
        w["down_scales"][:, :, 2] /= c
        w["down_scales"][:, :, 5] /= c
    L = layer_of(t, pib, w["gate"], w["up"], w["down"], w["gate_scales"], w["up_scales"], w["down_scales"])
    x = t.randn(4, D, device="cuda", generator=L.g)
    got = L.run(x, None)
    G, U, Dn = L.matrices(0)
    g = x.double() @ G.T
    y = (g * t.sigmoid(g) * (x.double() @ U.T)) @ Dn.T
    err = ((got.double() - y).pow(2).mean().sqrt() / y.pow(2).mean().sqrt()).item()
    print("c %g: 2^%.2f" % (c, __import__("math").log2(err)))
    assert err <= 2.0 ** -17
    check(L, x, t.zeros_like(x), got)
