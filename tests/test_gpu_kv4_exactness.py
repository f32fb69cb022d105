"""Attention over a 4-bit cache (csrc/kv4_attn.cu, kv4_prompt.cu) where few bits inside would show: scores far from zero whose difference decides, queries far below a row's largest."""
import pytest

from .test_gpu_kv4 import BF16, F32, Case, dtype, write

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pib():
    from pipeinfer_b200 import lib as pib
    pib.load().init(0)
    return pib


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,rep", [(1, 1), (4, 4), (120, 1)])
@pytest.mark.parametrize("scale", [1.0, -1.0])
@pytest.mark.parametrize("t,spread", [(F32, 0), (F32, 2.0 ** 15), (BF16, 0), (BF16, 2.0 ** 20)])
def test_scores_of_the_queries_as_they_are(torch, pib, dim, n, rep, t, spread, scale):
    """Two keys, one in each half of the channels, and queries that differ by 2^-7 between the halves: scores of some 200, the difference of which is the answer.  Queries that are rounded to 11 bits on
    their way leave outputs off by 0.05 to 0.09 there, ten times the bound of Case.want.  `spread`: a channel in which all keys are zero and the queries as many times larger."""
    seqs = 64 if n < 100 else 2
    c = Case(torch, pib, t, 1, rep, dim, [n] * seqs, [n + 2] * seqs)
    k, v = torch.zeros(n + 2, 1, dim, device="cuda"), torch.zeros(n + 2, 1, dim, device="cuda")
    k[0, :, :dim // 2], k[1, :, dim // 2:] = 30, 30          # (a step of 2: zeros stay zeros)
    k[:, :, 0] = k[:, :, dim // 2] = 0
    v[0], v[1] = 1, -1
    if scale < 0:
        k = -k
    for i in range(seqs):
        write(torch, c.kv, F32, k, v, c.cells(i, n + 2).contiguous())
    c.batch.scale *= scale
    m = 1 + torch.randint(0, 127, c.q.shape[:2] + (1,), device="cuda", generator=c.g) / 128
    c.q[..., :dim // 2] = m.to(c.q.dtype)
    c.q[..., dim // 2:] = (m + 2.0 ** -7).to(c.q.dtype)
    if t == F32:                                          # (bits behind bfloat16's)
        c.q *= 1 + torch.rand(c.q.shape, device="cuda", generator=c.g) * 2.0 ** -8
    if spread:
        c.q[..., 0] = spread
    got = c.run()
    c.q *= scale                                          # what `want` takes times |scale|
    c.check(got)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rep,portions,lens", [(8, [1] * 40, [3 + 5 * i for i in range(40)]), (4, [4] * 30, [5 + 7 * i for i in range(30)]), (8, [150, 40], [150, 600]), (1, [300], [300])])
def test_bfloat16_outputs_are_rounded_once(torch, pib, dim, rep, portions, lens):
    """Weights beside bfloat16 rows have the bits that they have beside fp32 ones: outputs lie half a step of bfloat16 from the exact ones, and the bound of fp32 rows.  (Queries a tenth as large: scores of
    about 1, so that this bound is a few 10^-6; weights of 11 bits are 2^-12 off.)"""
    c = Case(torch, pib, BF16, 2, rep, dim, portions, lens)
    c.q *= 0.1
    got = c.run()[:c.rows].double()
    c.t = F32
    ref, lim = c.want()
    half = torch.ldexp(torch.ones_like(ref), torch.frexp(ref.abs() + lim)[1] - 9)          # |o| in [2^(e - 1), 2^e): steps of 2^(e - 8)
    assert ((got - ref).abs() <= half + lim).all(), float((((got - ref).abs() - half) / lim).max())
