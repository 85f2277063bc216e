"""A teacher's top logits and the distillation loss against them (value and gradient) against their definitions in 64 bits."""
import math

import pytest
import torch

from ofb_amd import ops
from tests import distill_util as U

pytestmark = pytest.mark.gpu
DT = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


def make(seed, R, V, K, dtype, short=False):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(R, V, generator=g) * 2
    idx = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(R)]).to(torch.int32)
    values = torch.randn(R, K, generator=g) * 1.5 + math.log(V)
    z.scatter_add_(1, idx.long(), 0.5 * values)
    if short:
        idx[torch.rand(R, K, generator=g) < 0.4] = -1
    return z.to(dtype).cuda(), values.to(dtype).cuda(), idx.cuda(), (torch.randn(R, generator=g) * 0.3 + math.log(V)).cuda()


def run(z, values, idx, rest, tau, up, reduction='none'):
    z = z.detach().requires_grad_(True)
    loss = ops.distill_top_logits(z, values, idx, rest, temperature=tau, reduction=reduction)
    return loss.detach(), torch.autograd.grad(loss, z, up)[0]


def check(got, want):
    for x, (ref, bound) in zip(got, want):
        x = x.cpu().double()
        assert torch.isfinite(x).all()
        ratio = float(((x - ref).abs() / (bound + 1e-30)).max())
        assert ratio <= 1.0, (ratio, float((x - ref).abs().max()))


CASES = [(1, 1, 1), (3, 2, 1), (5, 7, 7), (4, 10, 3), (9, 63, 9), (6, 1000, 10), (3, 1001, 300), (2, 5003, 64), (7, 2048, 1024), (2, 40007, 33), (1, 140001, 100)]


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('with_rest', [False, True])
@pytest.mark.parametrize('R,V,K', CASES)
def test_loss_and_gradient(R, V, K, with_rest, dtype):
    z, values, idx, rest = make(R + V + K, R, V, K, DT[dtype])
    rest = rest if with_rest else None
    for tau in (1.0, 2.5):
        up = torch.linspace(0.5, 2.0, R).cuda() * (64 if dtype == 'f16' else 1)
        check(run(z, values, idx, rest, tau, up), U.reference(z, values, idx, rest, tau, up))


@pytest.mark.parametrize('dtype', list(DT))
def test_lists_with_gaps_repeats_and_nothing(dtype):
    R, V, K = 8, 300, 12
    z, values, idx, rest = make(7, R, V, K, DT[dtype], short=True)
    idx[0] = -1                                               # nothing stored
    idx[1] = V                                                # classes there are not
    values[2] = -math.inf                                     # no probability at all
    idx[3] = idx[3, 0].clamp(min=0)                           # one class twelve times
    idx[4, 1::2] = idx[4, 0::2]
    values[5, 3:] = -math.inf
    idx[6, :] = torch.arange(K, device='cuda').int() - 5
    z[0] = math.nan                                           # a row that says nothing is not looked at
    up = torch.ones(R, device='cuda')
    for r in (rest, None):
        got = run(z, values, idx, r, 2.0, up)
        check(got, U.reference(z, values, idx, r, 2.0, up))
        assert not got[0][:3].any() and not got[1][:3].any()
        wide = run(z, values, idx.long(), r, 2.0, up)
        assert torch.equal(got[0], wide[0]) and torch.equal(got[1], wide[1])


def test_all_classes_stored_is_the_whole_divergence():
    """K = V: rest is not used, and the loss is tau^2 KL(softmax(t / tau) | softmax(z / tau))"""
    z, values, idx, rest = make(3, 6, 50, 50, torch.float32)
    up = torch.ones(6, device='cuda')
    a, b = run(z, values, idx, rest, 2.0, up), run(z, values, idx, None, 2.0, up)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    t = torch.empty(6, 50, dtype=torch.float64).scatter_(1, idx.cpu().long(), values.cpu().double()) / 2
    zz = z.cpu().double().requires_grad_(True)
    kl = (torch.softmax(t, 1) * (torch.log_softmax(t, 1) - torch.log_softmax(zz / 2, 1))).sum(1) * 4
    kl.sum().backward()
    assert torch.allclose(a[0].cpu().double(), kl.detach(), rtol=1e-5, atol=1e-5) and torch.allclose(a[1].cpu().double(), zz.grad, rtol=1e-5, atol=1e-6)


def test_reductions_and_upstream():
    z, values, idx, rest = make(5, 37, 200, 8, torch.float32)
    rows, g = run(z, values, idx, rest, 1.5, torch.ones(37, device='cuda'))
    total, gs = run(z, values, idx, rest, 1.5, torch.tensor(3.0, device='cuda'), 'sum')
    mean, gm = run(z, values, idx, rest, 1.5, torch.tensor(3.0, device='cuda'), 'mean')
    assert abs(float(total) - float(rows.double().sum())) <= 2.0 ** -22 * float(rows.double().abs().sum())
    assert abs(float(mean) - float(rows.double().mean())) <= 2.0 ** -22 * float(rows.double().abs().mean())
    assert torch.allclose(gs, 3 * g, rtol=1e-6, atol=0) and torch.allclose(gm, 3 * g / 37, rtol=1e-6, atol=0)


def test_against_differences():
    """the slope along a random direction: a step of 1e-2 leaves 1e-4 of curvature"""
    z, values, idx, rest = make(8, 5, 60, 9, torch.float32)
    x = torch.randn(z.shape, generator=torch.Generator().manual_seed(0)).cuda()
    _, g = run(z, values, idx, rest, 2.0, torch.ones(5, device='cuda'))
    f = lambda s: ops.distill_top_logits(z + s * x, values, idx, rest, temperature=2.0, reduction='none').double()
    slope, along = (f(1e-2) - f(-1e-2)) / 2e-2, (g.double() * x.double()).sum(1)
    assert bool(((slope - along).abs() <= 1e-3 * (g * x).abs().sum(1).double() + 1e-3).all())


@pytest.mark.parametrize('dtype', list(DT))
def test_extreme_logits(dtype):
    """a student that is certain: the classes that were not stored carry e^-60 of its probability and still get their gradient; -inf logits are no classes"""
    R, V, K = 4, 500, 3
    z, values, idx, rest = make(2, R, V, K, DT[dtype])
    z.scatter_(1, idx.long(), 60.0)
    z[1].masked_fill_(torch.arange(V, device='cuda') % 2 == 0, -math.inf)
    z[1, idx[1].long()] = 3.0
    up = torch.ones(R, device='cuda')
    check(run(z, values, idx, rest, 1.0, up), U.reference(z, values, idx, rest, 1.0, up))


def test_layouts_streams_graph():
    for dtype in DT.values():
        z, values, idx, rest = make(4, 9, 1003, 20, dtype)
        up = torch.ones(9, device='cuda')
        want = run(z, values, idx, rest, 2.0, up)
        wide = torch.empty(9, 1004, dtype=dtype, device='cuda')[:, 1:].copy_(z)
        got = run(wide, values.t().contiguous().t(), idx.t().contiguous().t(), rest, 2.0, up)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        tw, iw, rw = ops.top_logits(z, 20, 2.0)
        tg, ig, rg = ops.top_logits(wide, 20, 2.0)
        assert torch.equal(tw, tg) and torch.equal(iw, ig) and torch.equal(rw, rg)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            def both():
                t, i, r = ops.top_logits(z, 20, 2.0)
                return (t, i, r, *run(z.flip(0), t, i, r, 2.0, torch.ones((), device='cuda'), 'mean'))
            both()
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = both()
            for turn in range(3):
                z.copy_(make(40 + turn, 9, 1003, 20, dtype)[0])
                graph.replay()
                stream.synchronize()
                for a, b in zip(out, both()):
                    assert torch.equal(a, b), turn
        torch.cuda.current_stream().wait_stream(stream)


def same(a, b):
    """equal bits of values, NaN equal to NaN"""
    return torch.equal(torch.nan_to_num(a.float(), nan=-7e30), torch.nan_to_num(b.float(), nan=-7e30))


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('R,V,K', [(1, 1, 1), (5, 9, 9), (3, 10, 4), (4, 1000, 10), (2, 1001, 700), (3, 8193, 128), (2, 9001, 1000), (2, 30011, 64), (1, 70001, 300)])
def test_top_logits(R, V, K, dtype):
    """bf16 logits of a large row are full of ties"""
    z = make(R * V + K, R, V, 1, DT[dtype])[0]
    for tau in (1.0, 3.0):
        values, indices, rest = ops.top_logits(z, K, tau)
        v, i, r = U.top(z.cpu(), K, tau)
        assert torch.equal(indices.cpu(), i) and same(values.cpu(), v)
        if K < V:
            assert bool(((rest.cpu().double() - r).abs() <= 1e-5 * (1 + r.abs())).all())
        else:
            assert bool((rest == -math.inf).all())


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('K', [1, 7, 300, 1000])
def test_top_logits_of_rows_that_are_hard_to_cut(K, dtype):
    """equal rows, two values, sorted runs, NaN, infinities, zeros of both signs: more candidates than are ranked at once"""
    V = 20011
    x = torch.arange(V, dtype=torch.float32)
    rows = [torch.full((V,), 2.5), (x % 2), x / V, -x / V, torch.where(x % 3 == 0, math.nan, x / V), torch.where(x % 5 == 0, -math.inf, 1.0), torch.where(x % 7 == 0, -0.0, 0.0),
            torch.full((V,), -math.inf), torch.where(x < 5, math.inf, -x / V)]
    z = torch.stack(rows).to(DT[dtype])
    values, indices, rest = ops.top_logits(z.cuda(), K)
    v, i, r = U.top(z, K, 1.0)
    assert torch.equal(indices.cpu(), i) and same(values.cpu(), v)
    fine = torch.isfinite(r)
    assert bool(((rest.cpu().double() - r).abs() <= 1e-5 * (1 + r.abs()))[fine].all()) and torch.equal(torch.isnan(rest.cpu()[3:4]), torch.isnan(r[3:4]))
    assert float(rest[7]) == -math.inf


def test_rows_beyond_32_bits():
    """2^31 + classes in all: the last rows' addresses pass 32 bits"""
    V, R, K = 1 << 20, 2100, 5
    z = torch.zeros(R, V, dtype=torch.bfloat16, device='cuda')
    at = torch.arange(K, device='cuda') * 7 + 11
    z[:, at] = torch.tensor([5.0, 4.0, 3.0, 2.0, 1.0], dtype=torch.bfloat16, device='cuda')
    z[-1, V - 1] = 9.0
    values, indices, rest = ops.top_logits(z[2000:], K)
    whole = ops.top_logits(z, K)
    assert torch.equal(values, whole[0][2000:]) and torch.equal(indices, whole[1][2000:])
    # fewer rows are cut into more segments: the same sum in another order, each of at most V / 1024 + 32 terms a thread, so its logarithm is off by that times 2^-24
    assert float((rest - whole[2][2000:]).abs().max()) <= 2 * (V / 1024 + 32) * 2.0 ** -24 + 2.0 ** -20
    assert indices[0].tolist() == at.tolist() and indices[-1].tolist() == [V - 1] + at.tolist()[:4]
    loss, g = run(z, whole[0], whole[1], whole[2], 1.0, torch.ones(R, device='cuda'))
    part, gp = run(z[2000:], values, indices, rest, 1.0, torch.ones(100, device='cuda'))
    assert float(loss.abs().max()) <= 1e-4 and float((loss[2000:] - part).abs().max()) <= 1e-5
    assert float((g[2000:].float() - gp.float()).abs().max()) <= 1e-5


def test_no_rows():
    z = torch.zeros(0, 5, device='cuda', requires_grad=True)
    values, indices, rest = ops.top_logits(z, 2)
    assert values.shape == (0, 2) and indices.shape == (0, 2) and rest.shape == (0,)
    assert ops.distill_top_logits(z, values, indices, rest, reduction='none').shape == (0,)
    loss = ops.distill_top_logits(z, values, indices, reduction='sum')
    loss.backward()
    assert float(loss) == 0 and z.grad.shape == (0, 5)


def test_as_many_rows_as_there_can_be():
    R = (1 << 22) - 1
    z = torch.randn(R, 3, generator=torch.Generator().manual_seed(3)).cuda()
    values, indices, rest = ops.top_logits(z, 2)
    v, i = z.sort(dim=1, descending=True, stable=True)              # (a few of the rows have ties: the lowest class first)
    assert torch.equal(values, v[:, :2]) and torch.equal(indices.long(), i[:, :2]) and torch.allclose(rest, v[:, 2], rtol=0, atol=1e-5)
    loss, g = run(z.flip(0), values.flip(0), indices.flip(0), rest.flip(0), 1.0, torch.ones((), device='cuda'), 'sum')
    assert float(loss) <= R * 1e-6 and float(g.abs().max()) <= 1e-5


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('V', [300, 20001])
def test_classes_masked_with_the_lowest_value(V, dtype):
    """a padded vocabulary: the last classes and some others hold the type's lowest value, a stored one among them"""
    R, K = 5, 12
    z, values, idx, rest = make(6, R, V, K, DT[dtype])
    low = torch.finfo(DT[dtype]).min
    z[:, -V // 5:] = low
    z[:, ::7] = low
    z.scatter_(1, idx[:, 1:].long(), 1.5)
    idx[:, 0] = 7
    z[:, 7] = low
    values[:, 0] = values.min() - 4                           # the teacher gives a masked class next to nothing
    values[2:, 0] = -math.inf                                 # or nothing at all
    up = torch.ones(R, device='cuda')
    for r in (rest, None):
        got = run(z[2:], values[2:], idx[2:], None if r is None else r[2:], 2.0, up[2:])
        check(got, U.reference(z[2:], values[2:], idx[2:], None if r is None else r[2:], 2.0, up[2:]))
        loss, g = run(z, values, idx, r, 2.0, up)
        if dtype == 'f16':                                    # (f16's lowest value is a logit like any other)
            check((loss, g), U.reference(z, values, idx, r, 2.0, up))
        else:
            assert bool((loss[:2] > 1e30).all()) and torch.isfinite(g).all()      # probability where the student has none: beyond any loss
    t, i, left = ops.top_logits(z, K, 2.0)
    v, j, w = U.top(z.cpu(), K, 2.0)
    assert torch.equal(i.cpu(), j) and same(t.cpu(), v) and bool(((left.cpu().double() - w).abs() <= 1e-5 * (1 + w.abs())).all())


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('low', ['lowest', -1e4])
def test_rows_of_one_value(low, dtype):
    """every logit the type's lowest value, or another one, student and teacher: even rows"""
    R, V, K = 3, 5003, 10
    low = torch.finfo(DT[dtype]).min if low == 'lowest' else low
    z = torch.full((R, V), low, dtype=DT[dtype], device='cuda')
    for tau in (1.0, 2.0, 3.0):
        t, i, left = ops.top_logits(z, K, tau)
        assert torch.equal(i.cpu(), torch.arange(K, dtype=torch.int32).expand(R, K)) and bool((t == z[:, :K]).all()) and torch.isfinite(left).all()
        even = torch.full((R,), math.log(V - K), device='cuda')
        loss, g = run(z, torch.zeros_like(t), i, even, tau, torch.ones(R, device='cuda'))      # a teacher that is even
        assert float(loss.abs().max()) <= 1e-5 * tau * tau and float(g.abs().max()) <= 1e-6
        loss, g = run(z, t, i, None, tau, torch.ones(R, device='cuda'))                        # and one that is even over the ten alone
        want = torch.full((R, V), 1 / V, dtype=torch.float64)
        want[:, :K] -= 1 / K
        assert float((loss.double().cpu() - tau * tau * math.log(V / K)).abs().max()) <= 1e-5 * tau * tau
        assert bool(((g.double().cpu() - tau * want).abs() <= (torch.finfo(DT[dtype]).eps + 1e-5) * tau * want.abs() + 2.0 ** -24).all())
