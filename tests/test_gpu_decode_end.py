"""The end of a decode step in one go: two mixture layers of 8-bit experts (csrc/moe_few.cu), the norm with the F8 product of the output rows (csrc/f8_gemv.cu, f8_gemm.cu), a token drawn from the
logits (csrc/sample_draw.cu); on the device throughout, eager and captured.  Each stage is held against float64 on what the device's stage in front of it gave."""
import numpy as np
import pytest

from tests import test_gpu_f8 as f8
from tests import test_gpu_moe_few as few
from tests import test_gpu_sample_draw as sd

pytestmark = pytest.mark.gpu
SETTINGS = [(0.8, 40, 0.95, 0.05), (0.0, 0, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.2, 5, 1.0, 0.0)]


class Step:
    def __init__(self, torch, pib, b, D, V):
        self.t, self.pib, self.lib, self.b, self.D, self.V = torch, pib, pib.load(), b, D, V
        self.layers = [few.Layer(torch, pib, few.F8, E, 1, 3, D, 320, seed=E) for E in (24, 9)]
        self.q, self.s, self.g = f8.matrix(torch, V, D, 7)
        self.s /= D ** 0.5
        self.head = pib.F8Weight(self.lib, self.q.data_ptr(), self.s.data_ptr(), V, D)
        self.nw = torch.rand(D, device="cuda", generator=self.g) + 0.5
        new = lambda *s, **k: torch.zeros(*s, device="cuda", **k)
        self.x, self.y, self.z, self.xn, self.logits, self.u = new(b, D), new(b, D), new(b, D), new(b, D), new(b, V), new(b)
        self.act = new(self.lib.act_bytes(f8.F8, D, b), dtype=torch.uint8)
        self.scratch = new(max(l.moe.scratch_bytes(b) for l in self.layers), dtype=torch.uint8)
        self.ids, self.p, self.kept = new(b, dtype=torch.int32), new(b), new(b, dtype=torch.int32)
        self.settings = [SETTINGS[i % len(SETTINGS)] for i in range(b)]
        rec = np.array(self.settings, [("temp", "f4"), ("top_k", "i4"), ("top_p", "f4"), ("min_p", "f4")])
        self.params = torch.from_numpy(rec.view(np.uint8).copy()).cuda()
        torch.cuda.synchronize()

    def fill(self):
        self.x.copy_(self.t.randn(self.b, self.D, device="cuda", generator=self.g))
        self.u.copy_(self.t.rand(self.b, device="cuda", generator=self.g))
        for o in (self.y, self.z, self.logits, self.p):
            o.fill_(float("nan"))
        self.ids.fill_(-7)

    def run(self, stream):
        lib, b, D = self.lib, self.b, self.D
        for l, i, o in zip(self.layers, (self.x, self.y), (self.y, self.z)):
            l.moe.forward(i.data_ptr(), D, b, i.data_ptr(), D, o.data_ptr(), D, self.scratch.data_ptr(), stream)
        lib.check(lib.L.pib_norm_quantize_act(f8.F8, 1, self.z.data_ptr(), self.nw.data_ptr(), 1e-5, b, D, self.act.data_ptr(), self.xn.data_ptr(), stream))
        (lib.gemm if b > 8 else lib.gemv)(self.head, self.act.data_ptr(), b, self.logits.data_ptr(), *((None, stream) if b > 8 else (stream,)))
        lib.sample(lib.TYPE_F32, self.logits.data_ptr(), self.V, b, self.V, self.params.data_ptr(), self.u.data_ptr(), self.ids.data_ptr(), self.p.data_ptr(), self.kept.data_ptr(), stream)

    def check(self):
        self.t.cuda.synchronize()
        few.check(self.layers[0], self.x, self.x, self.y)
        few.check(self.layers[1], self.y, self.y, self.z)
        z = self.z.double()
        ref = z / (z.pow(2).mean(1, keepdim=True) + 1e-5).sqrt() * self.nw.double()
        # the chain of a thread's fp32 additions, halved by the root; three roundings behind it
        assert ((self.xn.double() - ref).abs() <= ref.abs() * ((self.D / 256 + 16) / 2 + 6) * 2.0 ** -24).all()
        ref, lim = f8.want(self.t, self.q, self.s, self.xn)
        assert ((self.logits.double() - ref).abs() <= lim).all()
        rows, u = self.logits.cpu().numpy(), self.u.cpu().numpy()
        for r in range(self.b):
            i, share, n = sd.want(rows[r], self.settings[r], u[r])
            assert (int(self.ids[r]), int(self.kept[r])) == (i, n), r
            assert abs(float(self.p[r]) - share) <= 2.0 ** -23 * share + 1e-9


@pytest.fixture(scope="module")
def pib():
    from pipeinfer_b200 import lib as pib
    pib.load().init(0)
    return pib


@pytest.mark.parametrize("b,D,V", [(1, 512, 4001), (4, 640, 9000), (8, 500, 2000), (13, 512, 32000), (16, 384, 513)])
def test_a_step(pib, b, D, V):
    torch = pytest.importorskip("torch")
    s = Step(torch, pib, b, D, V)
    for _ in range(2):
        s.fill()
        s.run(torch.cuda.current_stream().cuda_stream)
        s.check()


@pytest.mark.parametrize("b", [1, 6, 16])
def test_captured_steps_on_two_streams(pib, b):
    """two captured steps with their own buffers, replayed at once"""
    torch = pytest.importorskip("torch")
    steps, streams, graphs = [Step(torch, pib, b, 512, 5000) for _ in range(2)], [torch.cuda.Stream() for _ in range(2)], []
    for s, st in zip(steps, streams):
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=st):
            s.run(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        for s in steps:
            s.fill()
        torch.cuda.synchronize()
        for _ in range(3):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        for s in steps:
            s.check()
