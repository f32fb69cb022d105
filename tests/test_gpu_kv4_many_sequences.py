"""Attention over a 4-bit cache with so many sequences that their tables take the place of records under way: beyond 287 a block of prompts has two instead of three, and the warps of decode batches fewer; of
1,024 sequences a thread counts the units of several."""
import pytest

from .test_gpu_kv4 import BF16, F32, Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pib():
    from pipeinfer_b200 import lib as pib
    pib.load().init(0)
    return pib


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("seqs", [287, 288, 1024])
def test_portions_of_prompts(torch, pib, t, dim, seqs):
    """up to nine tokens of eight heads: more rows than the decode kernels take.  Portions of nothing and sequences of nothing among them"""
    portions = [(i * 7) % 10 for i in range(seqs)]
    lens = [0 if i % 41 == 40 else n + (i * 37) % 300 for i, n in enumerate(portions)]
    Case(torch, pib, t, 1, 8, dim, portions, lens).check()


@pytest.mark.parametrize("seqs,t,rep", [(288, F32, 8), (288, F32, 16), (288, BF16, 8), (288, BF16, 16), (288, BF16, 32), (1024, F32, 1), (1024, F32, 9), (1024, BF16, 1), (1024, BF16, 9)])
@pytest.mark.parametrize("dim", [64, 128])
def test_single_tokens(torch, pib, seqs, t, rep, dim):
    """one, two and four tiles of eight rows"""
    lens = [(i * 53) % 400 for i in range(seqs)]
    Case(torch, pib, t, 1, rep, dim, [1] * seqs, lens, window=0 if dim == 64 else 200).check()
