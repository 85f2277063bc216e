"""Attention with a relative position bias where tiles of pairs, magnitudes and exponents change the kernels' way: against the definition in 64 bits, and by
identities that hold for any weights P as long as every kernel uses the same ones."""
import pytest
import torch

from ofb_amd import RelPosBuckets, ops
from tests import relpos_util as U
from tests.test_gpu_relpos import DT, PLANS, make, step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('Nq,Nk,H,d', [(1, 300, 2, 64), (5, 300, 2, 64), (33, 300, 1, 64), (70, 300, 2, 40), (97, 400, 1, 64), (100, 1000, 1, 64), (129, 400, 1, 64),
                                       (5, 300, 2, 128), (70, 300, 1, 128), (5, 300, 260, 72)])
def test_every_pair_reaches_the_table(Nq, Nk, H, d, dtype):
    """queries that do not fill their tile, keys far behind (and before) the last one: a tile of pairs is either summed as a whole or put into bins, whatever part
    of its queries exists.  Heads of 72 in 260 workgroups are the other variant of the wide kernels."""
    for reach in (16, 37, 40, 50, 63, 70, 100):
        plan = RelPosBuckets.clipped(reach)
        q, k, v, table, dout = make(Nq + reach, 1, Nq, Nk, H, d, DT[dtype], plan)
        for off in (0, Nk - Nq):
            U.check(step(q, k, v, table, plan, dout, q_offset=off), U.reference(q, k, v, table, plan, q_offset=off, dout=dout))


def windows():
    """plans and the bucket of theirs that a mask's bias takes: before the window, behind it, both ends of one border"""
    return (RelPosBuckets.clipped(5), 0), (RelPosBuckets.clipped(5), -1), (RelPosBuckets([0, 1], 0), 1), (RelPosBuckets([0, 1], 0), 0)


def rounding(q):
    """half a step of what is rounded on the way (P, dS) and in the result"""
    return 2.0 ** -22 if q.dtype == torch.float32 else torch.finfo(q.dtype).eps / 2


BIASES = [-1e4, -1e8, -1e9, -1e20, 1e5, 1e7, 1e8, 1e20]


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('size', [1.0, 6.0])
@pytest.mark.parametrize('bias', BIASES)
def test_finite_mask_biases(bias, size, dtype):
    """buckets beyond an end carry a bias that swallows the scores: whole tiles of it before and behind the keys that a row sees, rows of nothing else, the only ones that
    count.  A row with a key inside is exact (a masked key's weight is 0 in 32 bits); of any other the values' ends are the result's (P sums to 1: u for its rounding, u for the
    result's, n 2^-24 for the sums)."""
    for plan, masked in windows():
        for Nq, Nk, d in ((70, 300, 64), (1, 700, 64), (70, 300, 128), (33, 200, 16)):
            q, k, v, table, dout = make(Nq + int(size), 2, Nq, Nk, 2, d, DT[dtype], plan)
            q *= size
            table[masked] = bias
            for off in (0, Nk // 2, Nk - Nq, 2000, -2000):
                for causal in (False, True):
                    with torch.no_grad():
                        out = ops.relpos_attention(q, k, v, table, plan, q_offset=off, causal=causal)
                    U.check({'out': out}, U.reference(q, k, v, table, plan, q_offset=off, causal=causal))
                    assert float(out.abs().max()) <= float(v.abs().max()) * (1 + 2 * rounding(q) + (Nk + d) * 2.0 ** -24)


def one_key_each(dtype, Nq, Nk, size, plan, off, causal):
    """inputs whose scores are so large that a row has one key, and the rows where the next best is far beyond 32 bits' rounding of the scores behind it"""
    q, k, v, table, dout = make(Nq, 2, Nq, Nk, 2, 64, DT[dtype], plan)
    q, k = q * size, k * size
    s = torch.einsum('bihd,bjhd->bhij', q.cpu().double(), k.cpu().double()) / 8
    s = s + table.cpu().double()[U.bucket_matrix(plan, Nq, Nk, off)].permute(2, 0, 1)
    if causal:
        s = s.masked_fill(torch.arange(Nk) > torch.arange(Nq)[:, None] + off, -float('inf'))
    two = s.topk(2, -1)
    far = 64 * 2.0 ** -20 * float(q.abs().max()) * float(k.abs().max()) + 200
    return (q, k, v, table, dout), two.indices[..., 0], two.values[..., 0] - two.values[..., 1] > far


LARGE = [(70, 300, 0, False), (150, 150, 0, True), (1, 700, 3, False), (40, 600, 560, True)]


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('size', [300.0, 3000.0, 1e4])
def test_large_scores(size, dtype):
    """one key a row: its value is the output, to the rounding of the value's planes (f32)"""
    for name in ('clip0', 'log8', 'step'):
        plan = PLANS[name]()
        for Nq, Nk, off, causal in LARGE:
            (q, k, v, table, _), best, clear = one_key_each(dtype, Nq, Nk, size, plan, off, causal)
            assert float(clear.double().mean()) > 0.8
            with torch.no_grad():
                out = ops.relpos_attention(q, k, v, table, plan, q_offset=off, causal=causal)
            want = v.cpu().double().transpose(1, 2).gather(2, best[..., None].expand(-1, -1, -1, 64))
            err = (out.cpu().double().transpose(1, 2) - want).abs()[clear]
            assert torch.isfinite(out).all()
            assert bool((err <= 2 * rounding(q) * want.abs()[clear] + 2.0 ** -38 * float(v.abs().max())).all()), float(err.max())
