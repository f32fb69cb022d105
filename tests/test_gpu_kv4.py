"""Keys and values in 4 bits (csrc/kv4_cache.cu) and attention over them (csrc/kv4_attn.cu) against their definitions in float64."""
import ctypes as C
import math

import pytest

pytestmark = pytest.mark.gpu
F32, BF16 = 0, 30
PAGE, GROUP = 64, 32


@pytest.fixture(scope="module")
def pib():
    from pipeinfer_b200 import lib as pib
    pib.load().init(0)
    return pib


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


def dtype(torch, t):
    return torch.float32 if t == F32 else torch.bfloat16


def held(torch, x):
    """the values that cells hold of x [.., dim], fp16 numbers in float64; groups with something that is no finite number are nan"""
    v = x.float().unflatten(-1, (-1, GROUP))
    bad = ~v.isfinite().all(-1, keepdim=True)
    v = v.nan_to_num(0, 60000, -60000).clamp(-60000, 60000)
    m = v.amin(-1, keepdim=True).half()
    d = ((v.amax(-1, keepdim=True) - m.float()).clamp(min=0) / torch.full_like(v[..., :1], 15)).half()
    n = torch.where(d > 0, torch.round((v - m.float()) / torch.where(d > 0, d.float(), 1)), 0).clamp(0, 15)
    e = m.double() + d.double() * n.double()
    step = ((torch.frexp(e)[1].long() - 11).clamp(min=-24) + 1023 << 52).view(torch.float64)
    return torch.where(bad, math.nan, torch.round(e / step) * step).flatten(-2)


def write(torch, kv, t, k, v, cells, stream=0):
    n, w = len(cells), k.shape[1] * k.shape[2]
    kv.write(t, k.data_ptr(), w, v.data_ptr(), w, cells.data_ptr(), n, stream)


def read(torch, kv, t, cells, heads, dim):
    k, v = (torch.full((len(cells), heads, dim), 7.0, dtype=dtype(torch, t), device="cuda") for _ in range(2))
    kv.read(t, cells.data_ptr(), len(cells), k.data_ptr(), heads * dim, v.data_ptr(), heads * dim)
    torch.cuda.synchronize()
    return k, v


def same(torch, a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0), b.nan_to_num(0))


# ---- the cache ------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("heads,dim", [(1, 64), (3, 64), (8, 64), (1, 128), (5, 128), (8, 128), (33, 128)])
@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("n", [1, 2, 65, 1000])
def test_cells(torch, pib, heads, dim, t, n):
    g = torch.Generator(device="cuda").manual_seed(n + heads)
    kv = pib.Kv4(pib.load(), 40, heads, dim)
    assert kv.bytes() == 40 * heads * 80 * dim
    k, v = ((torch.randn(n, heads, dim, device="cuda", generator=g) * 10.0 ** torch.randint(-9, 5, (n, 1, 1), device="cuda", generator=g)).to(dtype(torch, t)) for _ in range(2))
    k[0, 0, :32] = 0.25                                   # one value: no step
    if n > 1:
        k[1, 0, :32] = -0.0
        v[1, 0, 3] = 3e38
        v[1, 0, 4] = -3e38
        k[1, -1, 40] = math.inf
        v[1, -1, 33] = math.nan
    cells = torch.randperm(40 * PAGE, device="cuda", generator=g)[:n].int()
    write(torch, kv, t, k, v, cells)
    K, V = read(torch, kv, F32, cells, heads, dim)
    assert same(torch, K.double(), held(torch, k)) and same(torch, V.double(), held(torch, v))
    Kb, Vb = read(torch, kv, BF16, cells, heads, dim)
    assert same(torch, Kb, K.bfloat16()) and same(torch, Vb, V.bfloat16())


def test_how_far_values_are_off(torch, pib):
    """half a step, the step's own rounding (15 steps of 2^-11 of one, or 2^-24), that of the lowest value and that of the result (2^-11 of them each)"""
    kv = pib.Kv4(pib.load(), 20, 4, 128)
    g = torch.Generator(device="cuda").manual_seed(5)
    k = torch.randn(1200, 4, 128, device="cuda", generator=g) + 3 * torch.randn(4, 128, device="cuda", generator=g)
    cells = torch.arange(1200, dtype=torch.int32, device="cuda")
    write(torch, kv, F32, k, -k, cells)
    K, V = read(torch, kv, F32, cells, 4, 128)
    x = k.unflatten(-1, (-1, GROUP))
    span, top = x.amax(-1, keepdim=True) - x.amin(-1, keepdim=True), x.abs().amax(-1, keepdim=True)
    lim = span / 30 * (1 + 32 * 2.0 ** -11) + 3 * top * 2.0 ** -11
    assert ((K - k).unflatten(-1, (-1, GROUP)).abs() <= lim).all() and ((V + k).unflatten(-1, (-1, GROUP)).abs() <= lim).all()


def test_cells_that_are_not_there_and_the_same_cell_twice(torch, pib):
    heads, dim, n = 2, 64, 900
    kv = pib.Kv4(pib.load(), 2, heads, dim)
    g = torch.Generator(device="cuda").manual_seed(9)
    k, v = (torch.randn(n, heads, dim, device="cuda", generator=g) for _ in range(2))
    cells = torch.randint(-40, 2 * PAGE + 40, (n,), device="cuda", generator=g).int()
    cells[5], cells[6] = -2 ** 31, 2 ** 31 - 1
    write(torch, kv, F32, k, v, cells)
    K, V = read(torch, kv, F32, torch.arange(-3, 2 * PAGE + 3, dtype=torch.int32, device="cuda"), heads, dim)
    last = {c: i for i, c in enumerate(cells.tolist())}
    for r, c in enumerate(range(-3, 2 * PAGE + 3)):
        for got, x in ((K, k), (V, v)):
            ref = held(torch, x[last[c]]) if 0 <= c < 2 * PAGE and c in last else torch.zeros(heads, dim, dtype=torch.float64, device="cuda")
            assert torch.equal(got[r].double(), ref), c


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("off,ld", [(0, 300), (1, 301), (8, 384)])
def test_rows_apart(torch, pib, t, off, ld):
    heads, dim, n = 2, 128, 70
    kv = pib.Kv4(pib.load(), 3, heads, dim)
    buf = torch.randn(2 * n * ld + 16, device="cuda").to(dtype(torch, t))
    k, v = (buf[off + i * n * ld:].as_strided((n, heads, dim), (ld, dim, 1)) for i in range(2))
    cells = torch.randperm(3 * PAGE, device="cuda")[:n].int()
    kv.write(t, k.data_ptr(), ld, v.data_ptr(), ld, cells.data_ptr(), n)
    K, V = read(torch, kv, F32, cells, heads, dim)
    assert torch.equal(K.double(), held(torch, k)) and torch.equal(V.double(), held(torch, v))
    out = torch.full((2 * n * ld + 16,), 5.0, device="cuda").to(dtype(torch, t))
    a, b = (out[off + i * n * ld:].as_strided((n, heads, dim), (ld, dim, 1)) for i in range(2))
    kv.read(t, cells.data_ptr(), n, a.data_ptr(), ld, b.data_ptr(), ld)
    torch.cuda.synchronize()
    assert torch.equal(a, K.to(a.dtype)) and torch.equal(b, V.to(b.dtype))
    a.fill_(5), b.fill_(5)
    assert (out == 5).all()                               # nothing between the rows
    kv.read(t, cells.data_ptr(), n, None, 0, b.data_ptr(), ld)
    torch.cuda.synchronize()
    assert (a == 5).all() and torch.equal(b, V.to(b.dtype))


# ---- attention ------------------------------------------------------------------------------------------------------------------------
class Case:
    """sequences with keys of their own on shuffled pages; `portions` new tokens and `lens` keys each"""

    def __init__(self, torch, pib, t, kvh, rep, dim, portions, lens, window=0, seed=0, extra_rows=0, spare=0):
        g = self.g = torch.Generator(device="cuda").manual_seed(seed * 1000 + sum(lens) + kvh)
        self.torch, self.t, self.kvh, self.rep, self.dim, self.window, self.portions, self.lens = torch, t, kvh, rep, dim, window, portions, lens
        n = [(l + PAGE - 1) // PAGE for l in lens]
        self.kv = pib.Kv4(pib.load(), sum(n) + 1 + spare, kvh, dim)
        order = torch.randperm(sum(n) + spare, device="cuda", generator=g).int() + 1
        self.pages = torch.zeros(len(lens), max(max(n), 1) + 1, dtype=torch.int32, device="cuda")
        for i in range(len(lens)):
            self.pages[i, :n[i]] = order[sum(n[:i]):sum(n[:i + 1])]
        cells = torch.cat([self.cells(i, l) for i, l in enumerate(lens)])
        k, v = (torch.randn(len(cells), kvh, dim, device="cuda", generator=g) for _ in range(2))
        for i in range(0, len(cells), 16384):
            write(torch, self.kv, F32, k[i:i + 16384].contiguous(), v[i:i + 16384].contiguous(), cells[i:i + 16384].contiguous())
        self.rows = sum(portions)
        self.q = (torch.randn(self.rows + extra_rows, kvh * rep, dim, device="cuda", generator=g) * 1.5).to(dtype(torch, t))
        self.starts = torch.tensor([sum(portions[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")
        self.lens_dev = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.batch = pib.Kv4Batch(t, kvh * rep, len(self.q), len(lens), max(portions + [0]), self.pages.shape[1], window, dim ** -0.5)
        self.out = torch.full_like(self.q, 3.0)
        self.scratch = torch.full((self.kv.scratch_bytes(self.batch),), 255, dtype=torch.uint8, device="cuda")

    def cells(self, i, n):
        t = self.torch
        return (self.pages[i].unsqueeze(1) * PAGE + t.arange(PAGE, dtype=t.int32, device="cuda")).flatten()[:n]

    def run(self, stream=0):
        w = self.kvh * self.rep * self.dim
        self.kv.attention(self.batch, self.q.data_ptr(), w, self.starts.data_ptr(), self.lens_dev.data_ptr(), self.pages.data_ptr(), self.out.data_ptr(), w, self.scratch.data_ptr(), stream)
        self.kv.lib.gemm_check(stream)
        return self.out

    def want(self, seen=None):
        """float64 rows and the bound of their errors.  `seen`: which keys of a sequence's table are there.

        A score is off by E: 22 bits of the queries (fp16 parts scaled by the row's power of two), D / 16 sums of the tensor core with two parts each, which may cut instead of round (2^-22), its
        scaling and the exponent's argument (2^-23 of the score each), all of S = scale * sum |q k|.  A weight e^s is then off by 2 E (its own score and the maximum's), the exponential's 2^-22 and
        its rounding to two parts (2^-21; bfloat16 rows: one fp16 number, 2^-11).  Numerator and denominator: twice that, and their sums over L / 16 steps of 2^-22.  bfloat16 rows end with half a step of
        their type."""
        torch = self.torch
        out, lim = torch.zeros(self.q.shape, dtype=torch.float64, device="cuda"), torch.zeros(self.q.shape, dtype=torch.float64, device="cuda")
        for i, (n, l) in enumerate(zip(self.portions, self.lens)):
            if not n or not l or (seen is not None and not seen[i][:l].any()):
                continue
            k, v = (x.double() for x in read(torch, self.kv, F32, self.cells(i, l), self.kvh, self.dim))
            there = torch.ones(l, dtype=torch.bool, device="cuda") if seen is None else seen[i][:l]
            k, v, pos, key = k[there], v[there], torch.arange(l - n, l, device="cuda").unsqueeze(1), torch.arange(l, device="cuda")[there]
            mask = (key <= pos) & (key > pos - (self.window or 1 << 30))
            at, some = int(self.starts[i]), mask.any(1).view(-1, 1, 1)
            for h in range(self.kvh * self.rep):
                q, K, V = self.q[at:at + n, h].double(), k[:, h // self.rep], v[:, h // self.rep]
                s = torch.where(mask, (q @ K.T) * self.dim ** -0.5, -math.inf)
                p = torch.softmax(torch.where(some[:, 0], s, 0), 1)
                o, S = p @ V.nan_to_num(0), float((q.abs() @ K.nan_to_num(0).abs().T).max()) * self.dim ** -0.5
                E = S * ((self.dim / 8) * 2.0 ** -22 + 2.0 ** -21)
                eps = 2 * (2 * E + 2.0 ** -22 + (2.0 ** -21 if self.t == F32 else 2.0 ** -11)) + l / 8 * 2.0 ** -22 + 2.0 ** -20
                out[at:at + n, h] = torch.where(some[:, 0], o, 0)
                lim[at:at + n, h] = torch.where(some[:, 0], (p @ V.nan_to_num(0).abs()) * eps + (0 if self.t == F32 else o.abs() * 2.0 ** -8), 0)
        return out[:self.rows], lim[:self.rows]

    def check(self, got=None, seen=None):
        ref, lim = self.want(seen)
        got = (self.run() if got is None else got)[:self.rows].double()
        assert got.isfinite().all()
        err = (got - ref).abs()
        assert (err <= lim).all(), float((err / lim.clamp(min=1e-30)).max())


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("kvh,rep,dim", [(1, 1, 64), (4, 8, 64), (2, 7, 64), (1, 1, 128), (5, 3, 128), (8, 8, 128), (2, 16, 128), (1, 33, 128)])
def test_one_token(torch, pib, t, kvh, rep, dim):
    for l in (1, 2, 63, 64, 65, 127, 300, 1000):
        Case(torch, pib, t, kvh, rep, dim, [1], [l]).check()


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rep", [1, 5, 8])
@pytest.mark.parametrize("window", [0, 1, 64, 100])
def test_ragged_decode(torch, pib, t, dim, rep, window):
    """sequences with no keys and no tokens among them"""
    Case(torch, pib, t, 2, rep, dim, [1, 0, 1, 2, 1, 1, 4, 0, 1, 3], [500, 70, 1, 2, 64, 0, 129, 0, 3000, 1], window).check()


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("portions,lens,window", [([17], [17], 0), ([64, 3], [64, 200], 0), ([300], [1000], 0), ([129, 1, 65], [129, 700, 66], 37), ([260, 500], [2000, 500], 0), ([513], [513], 200)])
@pytest.mark.parametrize("kvh,rep", [(1, 1), (2, 4), (1, 7)])
def test_prompts(torch, pib, t, dim, portions, lens, window, kvh, rep):
    Case(torch, pib, t, kvh, rep, dim, portions, lens, window).check()


@pytest.mark.parametrize("t", [F32, BF16])
def test_many_items_a_block(torch, pib, t):
    """more blocks of rows than the GPU has SMs, the last one of each portion less than half full"""
    Case(torch, pib, t, 16, 8, 128, [100, 33, 110, 100, 64], [150, 40, 300, 1000, 64]).check()
    Case(torch, pib, t, 16, 7, 64, [100, 40, 37, 100, 19], [100, 140, 300, 500, 640], 90).check()


@pytest.mark.parametrize("t", [F32, BF16])
def test_long(torch, pib, t):
    Case(torch, pib, t, 2, 8, 128, [1], [70001]).check()
    Case(torch, pib, t, 1, 8, 128, [2, 1, 1], [40000, 9, 20001], 30000).check()


@pytest.mark.parametrize("kvh,rep,n,lens", [(2, 4, 40, [64000]), (2, 4, 1, [64000]), (16, 8, 1, [20000] * 6)])
def test_sums_over_many_keys_stay_whole(torch, pib, kvh, rep, n, lens):
    """Tensor cores cut what they add: 2^-24 of a sum on average and each time, always towards zero, on the way up to the sum half of that.  Scores: 16 products in D = 128, times |s|, whose mean here is
    scale * 1.5 * sqrt(128) * 0.8 = 1.2; outputs: 32 products until fp32 takes over.  (16 * 1.2 + 32) * 2^-25 = 1.5e-6, and
    2^-22 each for the exponential and the rest of the parts: 2e-6.  Sums that stayed in the tensor core are off by 3.3e-6 here."""
    c = Case(torch, pib, F32, kvh, rep, 128, [n] * len(lens), lens)
    ref, _ = c.want()
    assert float((c.run().double() - ref).norm() / ref.norm()) < 2e-6


def test_many_sequences(torch, pib):
    lens = [(i * 37) % 200 for i in range(1024)]
    Case(torch, pib, BF16, 2, 4, 64, [1] * 1024, lens).check()


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("portions", [[1, 2, 5], [100, 40, 200]])
def test_rows_that_see_nothing(torch, pib, t, portions):
    """more new tokens than keys: the first ones stand in front of position 0; rows behind the last sequence are left as they were"""
    lens = [0, 1, 3] if portions[0] == 1 else [50, 0, 200]
    c = Case(torch, pib, t, 2, 4, 64, portions, lens, extra_rows=9)
    out = c.run()
    c.check(out)
    assert (out[c.rows:] == 3).all()
    for i, (n, l) in enumerate(zip(portions, lens)):
        assert not out[int(c.starts[i]):int(c.starts[i]) + max(0, n - l)].any()


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("n", [1, 4, 150])
def test_pages_that_are_not_there(torch, pib, t, n):
    """page numbers outside the cache, keys behind the table's row"""
    c = Case(torch, pib, t, 2, 4, 128, [n, n, n], [400, 400, 400])
    c.pages[0, 1], c.pages[0, 3], c.pages[1, :] = -1, 2 ** 31 - 1, -2 ** 31
    seen = [torch.ones(2000, dtype=torch.bool, device="cuda") for _ in range(3)]
    seen[0][64:128] = seen[0][192:256] = False
    seen[1][:] = False
    c.pages = c.pages.clone()
    keep, c.pages = c.pages, c.pages.clamp(min=0, max=1)   # what `cells` reads for keys that are there
    c.pages[0] = torch.where((keep[0] >= 0) & (keep[0] < 100), keep[0], 0)
    c.pages[2] = keep[2]
    ref, lim = c.want(seen)
    c.pages = keep
    got = c.run()[:c.rows].double()
    assert ((got - ref).abs() <= lim).all()
    assert not got[n:2 * n].any()
    c = Case(torch, pib, t, 1, 2, 64, [n], [300])
    c.lens_dev += 500                                      # 800 keys, a table of 6 pages: what lies behind it is not seen
    c.lens = [800]
    c.batch.max_pages = 4
    c.pages = c.pages[:, :4].contiguous()
    seen = [torch.arange(800, device="cuda") < 256]
    c.pages, short = torch.nn.functional.pad(c.pages, (0, 10)), c.pages
    ref, lim = c.want(seen)
    c.pages = short
    assert ((c.run()[:n].double() - ref).abs() <= lim).all()


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("n", [1, 3, 90])
@pytest.mark.parametrize("dim", [64, 128])
def test_what_is_no_number_in_places_that_are_not_seen(torch, pib, t, n, dim):
    """keys and values behind the sequence's end, behind a token's own position and in front of its window"""
    c = Case(torch, pib, t, 2, 4, dim, [n], [200 + n], window=100)
    ref = c.run().clone()
    cells = torch.cat([c.cells(0, 100), (c.pages[0, (200 + n) // PAGE] * PAGE + torch.arange((200 + n) % PAGE, PAGE, device="cuda")).int()])
    bad = torch.full((len(cells), 2, dim), math.nan, device="cuda")
    bad[::2] = math.inf
    write(torch, c.kv, F32, bad, bad, cells)
    assert torch.equal(c.run(), ref)
    # the last key: only the last token sees it
    one = c.cells(0, 200 + n)[-1:].clone()
    write(torch, c.kv, F32, bad[:1], bad[:1], one)
    got = c.run()
    assert torch.equal(got[:n - 1], ref[:n - 1]) and got[n - 1].isnan().all()


@pytest.mark.parametrize("t", [F32, BF16])
def test_large_and_small_numbers(torch, pib, t):
    """queries whose scores reach far beyond fp16 and fp32's exponentials, and queries of zeros and far below fp16"""
    c = Case(torch, pib, t, 2, 4, 64, [2, 1, 1, 90], [300, 300, 300, 300])
    c.q[0] *= 1e6
    c.q[1] *= 1e30
    c.q[2] = 0
    c.q[3] *= 1e-30
    c.q[4:40] *= 1e5
    ref, lim = c.want()
    got = c.run()[:c.rows].double()
    assert got.isfinite().all()
    small = [2, 3] + list(range(40, c.rows))
    assert ((got - ref).abs() <= lim)[small].all()
    # a score of 10^6 is not known to better than 2^-22 of it: the outputs lie between the values' ends
    v = torch.cat([read(torch, c.kv, F32, c.cells(i, 300), 2, 64)[1] for i in range(4)]).double()
    assert (got <= v.max() * 1.01).all() and (got >= v.min() * 1.01).all()


def test_shared_pages_and_another_order(torch, pib):
    """four drafted continuations of one prefix: the prefix' pages stand in all tables"""
    c = Case(torch, pib, BF16, 2, 8, 128, [3, 3, 3, 3], [200, 210, 220, 256])
    c.pages[1:, :3] = c.pages[0, :3]
    c.check()


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("n", [1, 120])
def test_rows_apart_in_attention(torch, pib, t, n):
    """queries inside rows of a fused projection, outputs beside them, odd distances"""
    c = Case(torch, pib, t, 2, 4, 64, [n, n], [n, 150 + n])
    w, ref = 512, c.run().clone()
    for ldq, ldo, oq, oo in ((768, 512, 0, 0), (513, 515, 1, 3), (1040, 1024, 8, 16)):
        q, o = torch.zeros(2 * n * ldq + 8, dtype=c.q.dtype, device="cuda"), torch.full((2 * n * ldo + 16,), 9.0, dtype=c.q.dtype, device="cuda")
        q[oq:].as_strided((2 * n, w), (ldq, 1)).copy_(c.q.reshape(2 * n, w))
        view = o[oo:].as_strided((2 * n, w), (ldo, 1))
        c.kv.attention(c.batch, q[oq:].data_ptr(), ldq, c.starts.data_ptr(), c.lens_dev.data_ptr(), c.pages.data_ptr(), view.data_ptr(), ldo, c.scratch.data_ptr())
        torch.cuda.synchronize()
        assert torch.equal(view.reshape(ref.shape), ref)
        view.fill_(9)
        assert (o == 9).all()


@pytest.mark.parametrize("n,hint", [(1, 0), (1, 500), (200, 1), (200, 0)])
def test_the_hint_changes_no_result(torch, pib, n, hint):
    c = Case(torch, pib, F32, 2, 4, 128, [n, 3], [n + 100, 300])
    c.batch.max_tokens = hint
    c.scratch = torch.full((c.kv.scratch_bytes(c.batch),), 255, dtype=torch.uint8, device="cuda")
    c.check()


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("n", [1, 100])
def test_same_bits_every_time_captured_and_on_other_streams(torch, pib, t, n):
    c = Case(torch, pib, t, 2, 8, 128, [n, 1, n], [900, 300, n], spare=3)
    ref = c.run().clone()
    for _ in range(3):
        c.out.fill_(0)
        c.scratch.random_(0, 255)
        assert torch.equal(c.run(), ref)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        w = 16 * 128
        c.kv.attention(c.batch, c.q.data_ptr(), w, c.starts.data_ptr(), c.lens_dev.data_ptr(), c.pages.data_ptr(), c.out.data_ptr(), w, c.scratch.data_ptr(), st.cuda_stream)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(c.out, ref)
    # the tables are read anew: fewer keys, another page order
    c.lens_dev.copy_(torch.tensor([850, 10, n], dtype=torch.int32))
    c.lens = [850, 10, n]
    graph.replay()
    torch.cuda.synchronize()
    c.check(c.out)


def test_two_calls_at_once(torch, pib):
    cases = [Case(torch, pib, F32, 4, 8, 128, [1] * 16, [3000 + 10 * i] * 16, seed=i) for i in range(2)]
    want = [c.run().clone() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(20):
        for c, st in zip(cases, streams):
            w = 32 * 128
            c.kv.attention(c.batch, c.q.data_ptr(), w, c.starts.data_ptr(), c.lens_dev.data_ptr(), c.pages.data_ptr(), c.out.data_ptr(), w, c.scratch.data_ptr(), st.cuda_stream)
    torch.cuda.synchronize()
    for c, w in zip(cases, want):
        assert torch.equal(c.out, w)


def test_offsets_past_32_bits(torch, pib):
    """a cache of 5 GB: keys on its last pages"""
    heads, dim, pages = 8, 128, 65000
    kv = pib.Kv4(pib.load(), pages, heads, dim)
    l = 200
    table = torch.arange(pages - 4, pages, dtype=torch.int32, device="cuda").view(1, 4)
    cells = (table.view(-1, 1) * PAGE + torch.arange(PAGE, dtype=torch.int32, device="cuda")).flatten()[:l].contiguous()
    k, v = (torch.randn(l, heads, dim, device="cuda") for _ in range(2))
    write(torch, kv, F32, k, v, cells)
    K, V = read(torch, kv, F32, cells, heads, dim)
    assert torch.equal(K.double(), held(torch, k)) and torch.equal(V.double(), held(torch, v))
    for n in (1, 150):
        q = torch.randn(n, heads, dim, device="cuda")
        b = pib.Kv4Batch(F32, heads, n, 1, n, 4, 0, dim ** -0.5)
        out, starts, lens = torch.empty_like(q), torch.tensor([0, n], dtype=torch.int32, device="cuda"), torch.tensor([l], dtype=torch.int32, device="cuda")
        scratch = torch.empty(kv.scratch_bytes(b), dtype=torch.uint8, device="cuda")
        kv.attention(b, q.data_ptr(), heads * dim, starts.data_ptr(), lens.data_ptr(), table.data_ptr(), out.data_ptr(), heads * dim, scratch.data_ptr())
        torch.cuda.synchronize()
        s = torch.einsum("thd,khd->htk", q.double(), K.double()) * dim ** -0.5
        s.masked_fill_(torch.arange(l, device="cuda") > torch.arange(l - n, l, device="cuda").unsqueeze(1), -math.inf)
        ref = torch.einsum("htk,khd->thd", torch.softmax(s, 2), V.double())
        assert float((out.double() - ref).abs().max()) < 1e-4


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("dim", [64, 128])
def test_scratch_of_a_larger_batch_serves_a_smaller(torch, pib, t, dim):
    kv = pib.Kv4(pib.load(), 4, 2, dim)
    for rep in (1, 7, 16):
        sizes = [kv.scratch_bytes(pib.Kv4Batch(t, 2 * rep, n, 3, 0, 5, 0, 1.0)) for n in (1, 2, 4, 5, 9, 17, 33, 64, 300, 65536)]
        assert sizes == sorted(sizes) and sizes[0] > 0
        hints = [kv.scratch_bytes(pib.Kv4Batch(t, 2 * rep, 300, 3, n, 5, 0, 1.0)) for n in (1, 2, 4, 9, 33, 64, 300, 0)]
        assert hints == sorted(hints)


def test_refusals_of_a_cache_that_is_there(torch, pib):
    lib = pib.load()
    kv = pib.Kv4(lib, 2, 2, 64)
    P, L = 1 << 12, lib.L

    def refused(rc, text):
        return rc == -2 and text in L.pib_last_error().decode()
    for kw in (dict(type=2), dict(k=None), dict(v=None), dict(ldk=127), dict(ldv=127), dict(cells=None), dict(n=-1), dict(n=16385), dict(k=P + 2), dict(cells=P + 2)):
        a = dict(dict(type=F32, k=P, ldk=128, v=P, ldv=128, cells=P, n=1), **kw)
        assert refused(L.pib_kv4_write(kv.h, a["type"], a["k"], a["ldk"], a["v"], a["ldv"], a["cells"], a["n"], None), "pib_kv4_write"), kw
        if "k" not in kw and "v" not in kw and kw != dict(n=16385):
            assert refused(L.pib_kv4_read(kv.h, a["type"], a["cells"], a["n"], a["k"], a["ldk"], a["v"], a["ldv"], None), "pib_kv4_read"), kw
    assert L.pib_kv4_write(kv.h, F32, None, 0, None, 0, None, 0, None) == 0 and L.pib_kv4_read(kv.h, BF16, None, 0, None, 0, None, 0, None) == 0
    ok = dict(type=F32, heads=4, tokens=3, seqs=1, max_tokens=3, max_pages=2, window=0, scale=1.0)
    for kw in (dict(type=12), dict(heads=0), dict(heads=3), dict(heads=1026), dict(tokens=-1), dict(tokens=65537), dict(seqs=-1), dict(seqs=1025), dict(max_tokens=-1), dict(max_pages=-1), dict(window=-1),
               dict(scale=math.nan), dict(scale=math.inf)):
        b = pib.Kv4Batch(**dict(ok, **kw))
        assert refused(L.pib_kv4_attn(kv.h, C.byref(b), P, 256, P, P, P, 1 << 20, 256, P, None), "pib_kv4_attn"), kw
        assert L.pib_kv4_attn_scratch_bytes(kv.h, C.byref(b)) == 0
    b = pib.Kv4Batch(**ok)
    for kw in (dict(q=None), dict(out=None), dict(starts=None), dict(lens=None), dict(pages=None), dict(scratch=None), dict(scratch=P + 128), dict(ldq=255), dict(ldo=255), dict(q=P + 2), dict(pages=P + 1),
               dict(out=P), dict(out=P + 1024), dict(out=P + 2 * 1024 + 1020)):
        a = dict(dict(q=P, ldq=256, starts=P, lens=P, pages=P, out=1 << 20, ldo=256, scratch=P), **kw)
        assert refused(L.pib_kv4_attn(kv.h, C.byref(b), a["q"], a["ldq"], a["starts"], a["lens"], a["pages"], a["out"], a["ldo"], a["scratch"], None), "pib_kv4_attn"), kw
    assert L.pib_kv4_attn(kv.h, C.byref(pib.Kv4Batch(**dict(ok, tokens=0))), None, 0, None, None, None, None, 0, None, None) == 0
