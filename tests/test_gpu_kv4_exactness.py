"""Attention over a 4-bit cache (csrc/kv4_attn.cu, kv4_prompt.cu) where few bits inside would show: scores far from zero whose difference decides, queries far below a row's largest,
sums over many keys that one warp or block takes alone, weights far below a row's largest."""
import math

import pytest

from .test_gpu_kv4 import BF16, F32, PAGE, Case, dtype, read, write

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


class Long:
    """`seqs` sequences of the same `l` keys on the same pages, with as many items as the GPU has warps (single rows) or SMs (portions) and more, so that most of them lie whole in one run.  All have the same
    queries, `n` tokens of `rep` heads: one sequence's exact rows are those of all."""

    def __init__(self, torch, pib, t, n, rep, l, keys, values, window=0):
        self.torch, self.t, self.n, self.rep, self.l, self.dim, self.kvh, self.window = torch, t, n, rep, l, 128, 8, window
        sms = torch.cuda.get_device_properties(0).multi_processor_count
        self.seqs = sms * (8 if n * rep <= 32 else 1) // self.kvh * 5 // 4 + 1
        pages = (l + PAGE - 1) // PAGE
        self.kv = pib.Kv4(pib.load(), pages, self.kvh, self.dim)
        for i in range(0, l, 8192):
            m = min(8192, l - i)
            cells = torch.arange(i, i + m, dtype=torch.int32, device="cuda")
            write(torch, self.kv, F32, keys(i, m), values(i, m), cells)
        self.table = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(self.seqs, 1)
        self.starts = torch.arange(self.seqs + 1, dtype=torch.int32, device="cuda") * n
        self.lens = torch.full((self.seqs,), l, dtype=torch.int32, device="cuda")
        self.batch = pib.Kv4Batch(t, self.kvh * rep, n * self.seqs, self.seqs, n, pages, window, self.dim ** -0.5)
        self.scratch = torch.empty(self.kv.scratch_bytes(self.batch), dtype=torch.uint8, device="cuda")

    def run(self, q):
        """q [n, heads, dim] -> [seqs, n, heads, dim]"""
        torch, w = self.torch, self.kvh * self.rep * self.dim
        q = q.to(dtype(torch, self.t)).repeat(self.seqs, 1, 1, 1)
        out = torch.full_like(q, 3.0)
        self.kv.attention(self.batch, q.data_ptr(), w, self.starts.data_ptr(), self.lens.data_ptr(), self.table.data_ptr(), out.data_ptr(), w, self.scratch.data_ptr())
        self.kv.lib.gemm_check(0)
        return out

    def want(self, q, heads):
        """float64 rows of some query heads"""
        torch, out = self.torch, []
        K, V = (x.double() for x in read(torch, self.kv, F32, torch.arange(self.l, dtype=torch.int32, device="cuda"), self.kvh, self.dim))
        gap = torch.arange(self.l - self.n, self.l, device="cuda").unsqueeze(1) - torch.arange(self.l, device="cuda")
        hidden = (gap < 0) | (gap >= (self.window or self.l))
        for h in heads:
            s = (q[:, h].to(dtype(torch, self.t)).double() @ K[:, h // self.rep].T * self.dim ** -0.5).masked_fill(hidden, -math.inf)
            out.append(torch.softmax(s, 1) @ V[:, h // self.rep])
        return torch.stack(out, 1)


def normal(torch, seed, scale):
    def some(i, m):
        g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + i)
        return torch.randn(m, 8, 128, device="cuda", generator=g) * scale
    return some


def ones(torch):
    return lambda i, m: torch.ones(m, 8, 128, device="cuda")


# a token of eight heads a group, one head a group, two tokens, a portion of many rows
@pytest.mark.parametrize("n,rep", [(1, 8), (1, 1), (2, 8), (8, 8)])
@pytest.mark.parametrize("l", [64000, 262144, 1 << 20])
def test_weights_add_up_to_one(torch, pib, n, rep, l):
    """fp32, all values one, scores of 1.2: outputs are the sum of the weights in the products over their sum in the denominator.

    An addition to a sum of one sign is off by at most 2^-24 of it, by 2^-24 / sqrt(3) in the mean square, and a chain of N of them by 2^-24 sqrt(N) / 3; one in a million passes five times that.  Chains of
    64: 8e-7, for numerator and denominator 1.1e-6 (those of 256 inside 4,096 keys are many, and their errors' mean is less).  Inside 256 keys tensor cores add 32 times and cut up to 2^-23 of what the sum has grown to, half of that on average, half of the way up: 1e-6.
    Exponentials and parts, 2^-22 each, are another for each key and the same above and below.  2.4e-6 with the output's own rounding; one chain through 64,000 keys may be off by 7e-6, and is."""
    c = Long(torch, pib, F32, n, rep, l, normal(torch, 1, 1.0), ones(torch))
    q = torch.randn(n, 8 * rep, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) * 1.2
    got = c.run(q)
    off = float((got - 1).abs().max())
    assert off < 2.4e-6
    c.scratch.fill_(255)
    assert torch.equal(c.run(q), got)                     # whatever the scratch holds


@pytest.mark.parametrize("n,rep", [(1, 8), (1, 1), (2, 8), (4, 8), (8, 8)])
def test_bfloat16_sums_over_many_keys(torch, pib, n, rep):
    """Values of one sign, 131,072 keys an item, outputs next to the middle between two numbers of bfloat16: sums that are low by a part in a thousand end on the wrong side.  Between two additions in fp32
    lie 4,096 keys, 512 products; each cuts less than 2^-23 of what the sum has grown to, and the sum is halfway up on average: 512 * 2^-24 = 3.05e-5 of the output beside its rounding, and 1e-6 for what fp32
    adds (chains of 32)."""
    l = 131072

    def values(i, m):
        step = (torch.arange(i, i + m, device="cuda") * 7919 % 128).view(-1, 1) < torch.arange(128, device="cuda")
        return (1 + 2.0 ** -8 + 2.0 ** -10 * step).unsqueeze(1).repeat(1, 8, 1)
    c = Long(torch, pib, BF16, n, rep, l, normal(torch, 1, 1.0), values)
    q = torch.randn(n, 8 * rep, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) * 1.2
    got, heads = c.run(q), [0, rep, 7 * rep, 8 * rep - 1]
    ref = c.want(q, heads)
    off = float((got[:, :, heads].double() - ref).abs().max())
    assert off <= 2.0 ** -8 + 3.2e-5


@pytest.mark.parametrize("n,rep", [(1, 8), (1, 1), (2, 8), (8, 8)])
@pytest.mark.parametrize("l", [64000, 262144])
def test_weights_far_below_the_largest_count(torch, pib, n, rep, l):
    """fp32, all values one, the first key 2^32.6 ahead of all others: those are 9.5e-6 of the sum behind 64,000 keys, 3.9e-5 behind 262,144.  A weight is held to 2^-39 of the largest, so l 2^-39 at most is
    missing from the outputs; and up to 4,096 keys' weights, 6.1e-7, are added to the largest a few at a time, each less than half of its last bit (the sums of
    4,096 keys are added with what that rounds away).  The rest as in test_weights_add_up_to_one."""
    def keys(i, m):
        k = torch.zeros(m, 8, 128, device="cuda")
        if i == 0:
            k[0] = 2
        return k
    c = Long(torch, pib, F32, n, rep, l, keys, ones(torch))
    off = float((c.run(torch.ones(n, 8 * rep, 128, device="cuda")) - 1).abs().max())
    assert off < 2.4e-6 + l * 2.0 ** -39


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("n,rep,dim", [(1, 8, 128), (1, 1, 64), (4, 4, 64), (120, 1, 128)])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_all_magnitudes(torch, pib, t, n, rep, dim, sign):
    """Scores about 2^k for k from 0 to 60, most of them too far apart for a softmax: where the largest leads by more than 64 times what scores are known to, the output is its key's value, and elsewhere it lies
    between the values' ends.  `sign`: all of them positive, or negative."""
    seqs = 122 // n + 1
    c = Case(torch, pib, t, 1, rep, dim, [n] * seqs, [n + 300] * seqs)
    k = [torch.rand(n + 300, 1, dim, device="cuda", generator=c.g) + 0.5 for _ in range(seqs)]
    v = [torch.randn(n + 300, 1, dim, device="cuda", generator=c.g) for _ in range(seqs)]
    for i in range(seqs):
        write(torch, c.kv, F32, k[i], v[i], c.cells(i, n + 300).contiguous())
    c.q = (c.q.abs() * sign * 2.0 ** (torch.arange(c.rows, device="cuda") % 61 - 2 - dim // 64).view(-1, 1, 1)).to(dtype(torch, t))
    got = c.run().double()
    assert got.isfinite().all()
    for i in range(seqs):
        K, V = (x.double() for x in read(torch, c.kv, F32, c.cells(i, n + 300), 1, dim))
        q, o = c.q[i * n:(i + 1) * n].double(), got[i * n:(i + 1) * n]
        s = torch.einsum("thd,kd->thk", q, K[:, 0]) * dim ** -0.5
        s.masked_fill_((torch.arange(n + 300, device="cuda") > torch.arange(300, n + 300, device="cuda").view(-1, 1)).unsqueeze(1), -math.inf)
        top, at = s.topk(2, -1)
        E = s[..., 0].abs() * 2 * ((dim / 8) * 2.0 ** -22 + 2.0 ** -21)          # as in Case.want
        clear = top[..., 0] - top[..., 1] > 64 * E + 64
        assert ((o - V[:, 0][at[..., 0]]).abs()[clear] <= V.abs().max() * (2.0 ** -20 if t == F32 else 2.0 ** -8)).all()
        assert (o <= V.max() * 1.01).all() and (o >= V.min() * 1.01).all()


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("n,rep", [(1, 8), (2, 8), (4, 8), (8, 8)])
def test_long_items_with_a_window_and_values_that_are_none(torch, pib, t, n, rep):
    """sums that have left registers and tensor memory, first pages that a window cuts, and a last key whose values are none in one group: the last token's rows are none there, and no other bit changes.
    Scores of 1.2 as before, E of Case.want 3e-5 with S = 7: 4 E, and half a step of bfloat16"""
    l, window = 64000, 30001
    c = Long(torch, pib, t, n, rep, l, normal(torch, 1, 1.0), normal(torch, 2, 1.0), window)
    q = torch.randn(n, 8 * rep, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) * 1.2
    got, heads = c.run(q), [0, rep, 7 * rep, 8 * rep - 1]
    ref = c.want(q, heads)
    off = float((got[:, :, heads].double() - ref).abs().max())
    assert off <= 1.2e-4 + (0 if t == F32 else float(ref.abs().max()) * 2.0 ** -8)
    K, V = read(torch, c.kv, F32, torch.tensor([l - 1], dtype=torch.int32, device="cuda"), 8, 128)
    V[:, 0, 32:64] = math.nan
    write(torch, c.kv, F32, K, V, torch.tensor([l - 1], dtype=torch.int32, device="cuda"))
    none = c.run(q)
    assert none[:, n - 1, :rep, 32:64].isnan().all()
    none[:, n - 1, :rep, 32:64] = got[:, n - 1, :rep, 32:64]
    assert torch.equal(none, got)
