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


def consistent(q, k, v, dout, scale, got):
    """What holds for any weights P whose rows sum to 1, if forward and backward use the same ones: |dv| <= sum of |dout|; sum v dv = sum dout out (both are
    sum P dout v); sum q dq = sum k dk (both are scale sum dS q k); the table's gradients sum to nothing (as a row of dS does).

    Tolerances: P, dS, D (bf16, f16: of an output whose P was rounded) and the results are off by u of the sums of their absolute terms each, and n terms in f32 by n 2^-24; the rows of P sum
    to 1, so a head's sums of |P dout v| and |dS q k| are at most Nq d max|dout| max|v| and Nq (2 d max|dout| max|v|) d max|q| max|k| scale.  Two sides: twice that."""
    B, Nq, H, d = q.shape
    off = 4 * rounding(q) + (k.shape[1] + Nq + d + 64) * 2.0 ** -24
    x = {n: t.detach().cpu().double().transpose(1, 2) for n, t in (('q', q), ('k', k), ('v', v), ('do', dout), *((m, got[m]) for m in ('out', 'dq', 'dk', 'dv')))}
    big = {n: float(t.abs().amax()) for n, t in x.items()}
    assert all(bool(torch.isfinite(t).all()) for t in got.values())
    assert big['dv'] <= Nq * big['do'] * (1 + off)
    apart = (x['v'] * x['dv']).sum((2, 3)) - (x['do'] * x['out']).sum((2, 3))
    assert float(apart.abs().max()) <= 2 * off * Nq * d * big['v'] * big['do'], apart
    top = 2 * d * big['do'] * big['v']
    apart = (x['q'] * x['dq']).sum((2, 3)) - (x['k'] * x['dk']).sum((2, 3))
    assert float(apart.abs().max()) <= 2 * off * Nq * top * scale * d * big['q'] * big['k'], apart
    assert float(got['dtable'].double().sum(0).abs().max()) <= B * off * Nq * top


def check_with_floors(q, k, v, dout, got, want):
    """... and what is small in absolute terms: f32 holds P to 2^-39 (half a subnormal step of f16 over the 2^14 of its scale) in dv; a pair is rounded down to a bin's unit, 2^-(55 - bits of Nk) of a
    power of two up to twice the largest |dS| <= 2 d max|dout| max|v|"""
    B, Nq, H, d = q.shape
    Nk = k.shape[1]
    U.check({n: x for n, x in got.items() if n != 'dtable'}, want, tiny=Nq * 2.0 ** -39 * float(dout.abs().max()))
    unit = 2.0 ** (2 - 55 + Nk.bit_length()) * 2 * d * float(dout.abs().max()) * float(v.abs().max())
    U.check({'dtable': got['dtable']}, want, tiny=B * Nq * Nk * unit)


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('size', [1.0, 6.0])
@pytest.mark.parametrize('bias', BIASES)
def test_gradients_of_finite_mask_biases(bias, size, dtype):
    """element by element where every row's maximum lies beside the mask, or the bias leaves its score 32-bit digits: the bounds count a score's rounding, 2^-24 of it, to first order, which is no
    bound from 2^24 on.  The identities hold everywhere."""
    for plan, masked in windows():
        for Nq, Nk, d in ((70, 300, 64), (1, 700, 64), (70, 300, 128), (33, 200, 16)):
            q, k, v, table, dout = make(Nq + int(size), 2, Nq, Nk, 2, d, DT[dtype], plan)
            q *= size
            table[masked] = bias
            for off in (0, Nk // 2, Nk - Nq, 2000, -2000):
                kw = dict(q_offset=off, causal=off == Nk // 2)
                got = step(q, k, v, table, plan, dout, **kw)
                consistent(q, k, v, dout, d ** -0.5, got)
                sees = torch.ones(Nq, Nk, dtype=torch.bool) if not kw['causal'] else torch.arange(Nk) <= torch.arange(Nq)[:, None] + off
                of_mask = sees & (U.bucket_matrix(plan, Nq, Nk, off) == masked % plan.num_buckets)
                blurred = of_mask.any(1) if bias > 0 else of_mask.any(1) & ~(sees & ~of_mask).any(1)
                if abs(bias) < 1e6 or not bool(blurred.any()):
                    check_with_floors(q, k, v, dout, got, U.reference(q, k, v, table, plan, dout=dout, **kw))


def check_one_key(q, k, v, dout, best, clear, got, scale=0.125):
    """each row has one key: P is 1 there and 0 elsewhere, so dv is the sum of those rows' dout (u for the result, 2^-24 a term); the scores' rounding must not show.  (Rows
    whose best key is not clear add their dout to some keys: those are left out.)"""
    consistent(q, k, v, dout, scale, got)
    do, dv = dout.cpu().double().transpose(1, 2), got['dv'].cpu().double().transpose(1, 2)
    Nk = k.shape[1]
    hit = torch.zeros(*best.shape[:2], Nk, dtype=torch.bool)
    want = torch.zeros_like(dv)
    for b in range(best.shape[0]):
        for h in range(best.shape[1]):
            want[b, h].index_add_(0, best[b, h], do[b, h])
            hit[b, h, best[b, h][clear[b, h]]] = True
            hit[b, h, best[b, h][~clear[b, h]]] = False
    err = (dv - want).abs()[hit]
    tol = 2 * rounding(q) * want.abs()[hit] + best.shape[2] * (rounding(q) + 2.0 ** -24) * float(do.abs().max()) * (~clear).any() + 8 * 2.0 ** -24 * float(do.abs().max())
    assert bool((err <= tol).all()), float(err.max())


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('size', [300.0, 3000.0, 1e4])
def test_gradients_of_large_scores(size, dtype):
    for name in ('clip0', 'log8', 'step'):
        plan = PLANS[name]()
        for Nq, Nk, off, causal in LARGE:
            (q, k, v, table, dout), best, clear = one_key_each(dtype, Nq, Nk, size, plan, off, causal)
            got = step(q, k, v, table, plan, dout, q_offset=off, causal=causal)
            check_one_key(q, k, v, dout, best, clear, got)


# sizes of q, k, v, dout; what f32 arithmetic forms (scores, dP, dS) fits f32 in all of them
WIDE = [(1.0, 1.0, 1e25, 1.0), (1.0, 1.0, 1.0, 1e25), (1e25, 1e-25, 1.0, 1.0), (1e-30, 1e30, 1e10, 1e-10), (1.0, 1.0, 5e36, 1e-36), (1.0, 1.0, 1e-36, 5e36), (1e-4, 1e4, 7e22, 1.0),
        (1.0, 1.0, 1e23, 1e-20), (1.0, 1.0, 1e-30, 1.0), (1.0, 1.0, 1.0, 1e-30), (1.0, 1.0, 1e-22, 1e-8), (1e-30, 1e30, 1.0, 1e-28), (1e-28, 1.0, 1.0, 1.0), (1.0, 1e-28, 1.0, 1.0), (1e-20, 1e-20, 1e20, 1e10)]


@pytest.mark.parametrize('sizes', WIDE, ids=lambda s: '-'.join(f'{x:g}' for x in s))
def test_float32_of_any_size(sizes):
    """the bounds of ordinary sizes, relative to the tensors' maxima.  (In absolute terms: planes whose exponent ends at 2^112 hold their tensor to 2^-137, of which 600 products with
    factors up to 5 are below 1e-38.)"""
    plan = PLANS['clip']()
    for Nq, Nk in ((70, 70), (1, 1500), (200, 600)):
        q, k, v, table, dout = make(33, 1, Nq, Nk, 1, 64, torch.float32, plan)
        q, k, v, dout = (x * s for x, s in zip((q, k, v, dout), sizes))
        got = step(q, k, v, table, plan, dout)
        U.check(got, U.reference(q, k, v, table, plan, dout=dout), tiny=1e-38)
        assert bool(got['out'].any()) and bool(got['dv'].any())


@pytest.mark.parametrize('largest', [3e38, torch.finfo(torch.float32).max])
def test_the_largest_float32(largest):
    """one value at the end of f32, alone in its column and met by some rows; then all values there, whose mean is (in one range of keys and joined from several).  The rows that do not meet it are held to
    2^-39 of it, like all of a head."""
    plan = PLANS['clip']()
    for Nq, Nk, off, causal in ((70, 70, 0, True), (1, 1500, 1499, False), (150, 600, 450, True)):
        q, k, v, table, dout = make(34, 1, Nq, Nk, 1, 64, torch.float32, plan)
        v[:, -3], v[:, -3, :, 2] = 0.0, largest
        kw = dict(q_offset=off, causal=causal)
        with torch.no_grad():
            U.check({'out': ops.relpos_attention(q, k, v, table, plan, **kw)}, U.reference(q, k, v, table, plan, **kw))
        v[:] = 3e38
        with torch.no_grad():
            U.check({'out': ops.relpos_attention(q, k, v, table, plan, **kw)}, U.reference(q, k, v, table, plan, **kw))


def test_forward_mode_is_refused():
    """a tangent is never dropped in silence: dual tensors need not require a gradient, with and without gradients enabled"""
    from torch.autograd import forward_ad
    plan = PLANS['clip']()
    q, k, v, table, dout = make(35, 1, 5, 5, 1, 64, torch.float32, plan)
    qkv = torch.stack([q, k, v], 2)
    with forward_ad.dual_level():
        plain = ops.relpos_attention(q, k, v, table, plan)
        for enabled in (True, False):
            with torch.set_grad_enabled(enabled):
                for at in range(4):
                    ins = [q, k, v, table]
                    ins[at] = forward_ad.make_dual(ins[at], torch.ones_like(ins[at]))
                    with pytest.raises(RuntimeError):
                        ops.relpos_attention(*ins, plan)
                for ins in ((forward_ad.make_dual(qkv, qkv), table), (qkv, forward_ad.make_dual(table, table))):
                    with pytest.raises(RuntimeError):
                        ops.relpos_attention_qkv(*ins, plan)
    assert torch.equal(plain, ops.relpos_attention(q, k, v, table, plan))


def test_a_plan_that_is_dropped_while_another_stream_reads_it():
    """its memory is not handed out before that stream is done.  (What asks for memory meanwhile writes zeros: buckets like any other.)"""
    side = torch.cuda.Stream()
    q, k, v, table, dout = make(7, 2, 60, 60, 2, 64, torch.bfloat16, RelPosBuckets.clipped(30))
    want = ops.relpos_attention(q, k, v, table, RelPosBuckets.clipped(30))
    for _ in range(3):
        plan = RelPosBuckets.clipped(30).to('cuda')
        words = sum(t.numel() for t in plan.on('cuda') if t is not None)
        ops.relpos_attention(q, k, v, table, plan)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
            got = ops.relpos_attention(q, k, v, table, plan)
        del plan
        taken = [torch.zeros(words, dtype=torch.int32, device='cuda') for _ in range(64)]
        side.synchronize()
        assert torch.equal(got, want)
        del taken
