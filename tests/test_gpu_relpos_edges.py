"""Attention with a relative position bias where tiles of pairs, magnitudes and exponents change the kernels' way: against the definition in 64 bits, and by
identities that hold for any weights P as long as every kernel uses the same ones."""
import pytest
import torch

from ofb_amd import RelPosBuckets
from tests import relpos_util as U
from tests.test_gpu_relpos import DT, make, step

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
