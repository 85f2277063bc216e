"""Attention with a learned relative position bias (forward, backward) against its definition in 64 bits, element by element within derived bounds."""
import math

import pytest
import torch

from ofb_amd import RelPosBuckets, ops
from tests import relpos_util as U

pytestmark = pytest.mark.gpu
DT = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
PLANS = {
    'log': lambda: RelPosBuckets.log_spaced(32, 128),
    'log8': lambda: RelPosBuckets.log_spaced(8, 20),
    'causal': lambda: RelPosBuckets.log_spaced(16, 64, bidirectional=False),
    'clip': lambda: RelPosBuckets.clipped(7),
    'clip0': lambda: RelPosBuckets.clipped(0),
    'wide': lambda: RelPosBuckets.clipped(2000),
    'step': lambda: RelPosBuckets([0, 1], 0),
}


def make(seed, B, Nq, Nk, H, d, dtype, plan, packed=False):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    if packed:
        q, k, v = r(B, Nq, 3, H, d).to(dtype).cuda().unbind(2)
    else:
        q, k, v = r(B, Nq, H, d).to(dtype).cuda(), r(B, Nk, H, d).to(dtype).cuda(), r(B, Nk, H, d).to(dtype).cuda()
    return q, k, v, r(plan.num_buckets, H).cuda(), r(B, Nq, H, d).to(dtype).cuda()


def step(q, k, v, table, plan, dout, **kw):
    q, k, v, table = (t.detach().requires_grad_(True) for t in (q, k, v, table))
    out = ops.relpos_attention(q, k, v, table, plan, **kw)
    return dict(zip(('out', 'dq', 'dk', 'dv', 'dtable'), (out.detach(), *torch.autograd.grad(out, (q, k, v, table), dout))))


# B, Nq, Nk, H, d, plan, causal, q_offset
CASES = [
    (1, 1, 1, 1, 8, 'clip', False, 0), (2, 17, 17, 3, 16, 'log', False, 0), (1, 33, 70, 2, 40, 'log8', False, 37), (2, 128, 128, 1, 64, 'clip', True, 0),
    (1, 129, 257, 2, 64, 'log', False, 128), (3, 65, 65, 2, 72, 'causal', True, 0), (1, 200, 31, 1, 128, 'log', False, -5), (1, 31, 200, 2, 128, 'causal', True, 169),
    (2, 90, 40, 2, 24, 'log', True, -50), (1, 300, 300, 1, 32, 'wide', False, 0), (1, 64, 600, 1, 64, 'clip0', False, 11), (2, 50, 50, 2, 64, 'step', False, 3),
    (1, 1, 1500, 2, 64, 'causal', True, 1499), (2, 5, 1025, 1, 128, 'log', False, 0), (1, 700, 700, 2, 96, 'log', False, 0),
]


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('case', CASES, ids=lambda c: '-'.join(map(str, c)))
def test_against_the_definition(case, dtype):
    B, Nq, Nk, H, d, plan, causal, off = case
    plan = PLANS[plan]()
    q, k, v, table, dout = make(Nq * 7 + Nk + d, B, Nq, Nk, H, d, DT[dtype], plan)
    want = U.reference(q, k, v, table, plan, causal=causal, q_offset=off, dout=dout)
    got = step(q, k, v, table, plan, dout, causal=causal, q_offset=off)
    worst = U.check(got, want)
    with torch.no_grad():
        alone = ops.relpos_attention(q, k, v, table, plan, causal=causal, q_offset=off)
    assert torch.equal(alone, got['out'])
    print(case, dtype, {n: f'{x:.2g}' for n, x in worst.items()})


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('gh,gw,cls,H,d', [(14, 14, True, 2, 64), (1, 1, True, 1, 16), (5, 9, False, 2, 40), (24, 3, True, 1, 128)])
def test_patch_grid(gh, gw, cls, H, d, dtype):
    plan = RelPosBuckets.grid(gh, gw, cls_token=cls)
    N = gh * gw + cls
    q, k, v, table, dout = make(gh + gw, 3, N, N, H, d, DT[dtype], plan, packed=True)
    U.check(step(q, k, v, table, plan, dout), U.reference(q, k, v, table, plan, dout=dout))


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('causal', [False, True])
def test_lengths_and_what_lies_behind_them(dtype, causal):
    """lengths of 0, 1, one tile, past the end and below zero; NaN and infinities behind them change nothing and get no gradient"""
    plan = PLANS['log']()
    B, N, H, d = 7, 150, 2, 64
    q, k, v, table, dout = make(5, B, N, N, H, d, DT[dtype], plan)
    lens = torch.tensor([0, 1, 64, 65, 150, 4000, -3], dtype=torch.int32, device='cuda')
    want = U.reference(q, k, v, table, plan, causal=causal, key_lens=lens, dout=dout)
    clean = step(q, k, v, table, plan, dout, causal=causal, key_lens=lens)
    U.check(clean, want)
    for b, n in enumerate(lens.clamp(0, N).tolist()):
        k[b, n:], v[b, n:] = math.nan, math.inf
        assert not clean['dk'][b, n:].any() and not clean['dv'][b, n:].any()
    assert not clean['out'][0].any() and not clean['dq'][0].any()
    dirty = step(q, k, v, table, plan, dout, causal=causal, key_lens=lens)
    for n in clean:
        assert torch.equal(clean[n], dirty[n]), n


@pytest.mark.parametrize('dtype', list(DT))
def test_a_bias_of_the_lowest_value_masks_and_a_row_of_it_is_even(dtype):
    plan = RelPosBuckets([0, 1, 2], -1)                       # before, itself, after
    q, k, v, table, dout = make(9, 2, 70, 70, 2, 32, DT[dtype], plan)
    low = torch.finfo(torch.float32).min
    table[2] = low                                            # no query sees what comes after it
    want = U.reference(q, k, v, table, plan, dout=dout)
    got = step(q, k, v, table, plan, dout)
    for n in ('out', 'dq', 'dk', 'dv'):
        U.check({n: got[n]}, want)
    table[:] = low                                            # every score is the lowest value: all keys alike
    got = step(q, k, v, table, plan, dout)
    even = v.float().mean(1, keepdim=True).expand(2, 70, 2, 32)
    tol = 2 * torch.finfo(DT[dtype]).eps * v.float().abs().mean(1, keepdim=True) + 1e-6
    assert bool(((got['out'].float() - even).abs() <= tol).all())
    for plan, masked in ((RelPosBuckets([0, 1], 0), 1), (RelPosBuckets.clipped(3), 0)):
        # a long run of masked keys beside visible ones, and rows that are masked throughout: even, with the gradients of an even row
        q, k, v, table, dout = make(10, 1, 70, 300, 2, 64, DT[dtype], plan)
        table[masked] = low
        for off in (0, 2000, -2000):
            U.check(step(q, k, v, table, plan, dout, q_offset=off), U.reference(q, k, v, table, plan, q_offset=off, dout=dout))
    plan = RelPosBuckets([0, 1, 2], -1)
    q, k, v, table, dout = make(9, 2, 70, 70, 2, 32, DT[dtype], plan)
    table[:] = -math.inf                                      # nothing is seen
    got = step(q, k, v, table, plan, dout)
    assert not got['out'].any() and not got['dq'].any() and not got['dv'].any()


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('scale', [-0.3, 0.0, 1.0])
def test_scales(scale, dtype):
    """a scale of any sign: beyond the ends too"""
    for name, off in (('clip', 0), ('log8', 100), ('causal', -5)):
        plan = PLANS[name]()
        q, k, v, table, dout = make(14, 2, 70, 200, 1, 32, DT[dtype], plan)
        got, want = step(q, k, v, table, plan, dout, scale=scale, q_offset=off), U.reference(q, k, v, table, plan, scale=scale, q_offset=off, dout=dout)
        U.check(got, want)


@pytest.mark.parametrize('dtype', list(DT))
def test_layouts(dtype):
    """heads before tokens, channels not contiguous, rows off 16 bytes, a key tensor broadcast over the batch: the same bits as contiguous copies"""
    plan = PLANS['log8']()
    B, N, H, d = 3, 75, 2, 40
    q, k, v, table, dout = make(3, B, N, N, H, d, DT[dtype], plan)
    want = step(q, k, v, table, plan, dout)
    odd = torch.empty(B, N, H, d + 1, dtype=DT[dtype], device='cuda')[..., 1:].copy_(k)
    last = v.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2)
    heads = q.transpose(1, 2).contiguous().transpose(1, 2)
    got = step(heads, odd, last, table.t().contiguous().t(), plan, dout.transpose(1, 2).contiguous().transpose(1, 2))
    for n in want:
        assert torch.equal(want[n], got[n]), n
    one = k[:1].expand(B, N, H, d)
    a, b = step(q, one, v, table, plan, dout), step(q, one.contiguous(), v, table, plan, dout)
    for n in a:
        assert torch.equal(a[n], b[n]), n
    leaf = k[:1].detach().requires_grad_(True)
    out = ops.relpos_attention(q, leaf.expand(B, N, H, d), v, table, plan)
    (g,) = torch.autograd.grad(out, leaf, dout)
    assert torch.equal(g, b['dk'].sum(0, keepdim=True))


def test_packed_and_bound():
    plan = RelPosBuckets.grid(6, 7)
    g = torch.Generator().manual_seed(2)
    for dtype in DT.values():
        qkv = torch.randn(4, 43, 3, 2, 64, generator=g).to(dtype).cuda()
        table, dout = torch.randn(plan.num_buckets, 2, generator=g).cuda(), torch.randn(4, 43, 2, 64, generator=g).to(dtype).cuda()
        want = step(*qkv.unbind(2), table, plan, dout)
        x, t = qkv.clone().requires_grad_(True), table.clone().requires_grad_(True)
        out = ops.relpos_attention_qkv(x, t, plan)
        dx, dt = torch.autograd.grad(out, (x, t), dout)
        assert torch.equal(out, want['out']) and torch.equal(dt, want['dtable'])
        for i, n in enumerate(('dq', 'dk', 'dv')):
            assert torch.equal(dx[:, :, i], want[n]), n
    # f32 with a bound of the producer's: a looser exponent, the same accuracy
    qkv = torch.randn(2, 43, 3, 2, 64, generator=g).cuda()
    x, t, dout = qkv.clone().requires_grad_(True), table.clone().requires_grad_(True), torch.randn(2, 43, 2, 64, generator=g).cuda()
    out = ops.relpos_attention_qkv(x, t, plan, bound=torch.full((1,), 37.0, device='cuda'))
    dx, dt = torch.autograd.grad(out, (x, t), dout)
    q, k, v = qkv.unbind(2)
    dq, dk, dv = dx.unbind(2)
    U.check({'out': out, 'dq': dq, 'dk': dk, 'dv': dv, 'dtable': dt}, U.reference(q, k, v, t, plan, dout=dout))


def test_gradients_against_differences():
    """f32: the directional derivative along a random direction of all four inputs; the function is smooth, a step of 1e-3 leaves 1e-6 of curvature and about
    1e-7 / 1e-3 of rounding"""
    plan = PLANS['log8']()
    q, k, v, table, dout = make(21, 2, 40, 55, 2, 32, torch.float32, plan)
    lens = torch.tensor([55, 30], dtype=torch.int32, device='cuda')
    g = torch.Generator().manual_seed(1)
    dirs = [torch.randn(t.shape, generator=g).cuda() for t in (q, k, v, table)]
    got = step(q, k, v, table, plan, dout, key_lens=lens, q_offset=15, causal=True)
    h = 1e-3
    f = lambda s: float((ops.relpos_attention(*(t + s * x for t, x in zip((q, k, v, table), dirs)), plan, key_lens=lens, q_offset=15, causal=True).double() * dout.double()).sum())
    slope = (f(h) - f(-h)) / (2 * h)
    along = sum(float((got[n].double() * x.double()).sum()) for n, x in zip(('dq', 'dk', 'dv', 'dtable'), dirs))
    size = sum(float((got[n].double() * x.double()).abs().sum()) for n, x in zip(('dq', 'dk', 'dv', 'dtable'), dirs))
    assert abs(slope - along) <= 1e-3 * math.sqrt(size) + 1e-4 * abs(along), (slope, along)


@pytest.mark.parametrize('dtype', list(DT))
def test_f32_range_and_small_values(dtype):
    """values far from 1: the planes' exponents follow the tensors"""
    plan = PLANS['clip']()
    q, k, v, table, dout = make(4, 2, 70, 70, 2, 64, torch.float32, plan)
    big, small = (300.0, 1e-3) if dtype == 'f16' else (1e6, 1e-6)
    q, k, v, dout = (q * small).to(DT[dtype]), (k / small * 0.1).clamp(-3e4, 3e4).to(DT[dtype]), (v * big).to(DT[dtype]), (dout * small).to(DT[dtype])
    got, want = step(q, k, v, table, plan, dout), U.reference(q, k, v, table, plan, dout=dout)
    U.check(got, want)


def test_same_bits_on_every_run_and_on_another_stream():
    plan = PLANS['log']().to('cuda')
    for dtype in DT.values():
        q, k, v, table, dout = make(6, 4, 333, 333, 3, 64, dtype, plan)
        want = step(q, k, v, table, plan, dout)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            others = [step(q, k, v, table, plan, dout) for _ in range(2)]
        mine = step(q, k, v, table, plan, dout)
        torch.cuda.current_stream().wait_stream(side)
        for got in others + [mine]:
            for n in want:
                assert torch.equal(want[n], got[n]), n


def test_captured_step_replays():
    plan = PLANS['log']().to('cuda')
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ins = {}
        for dtype in DT.values():
            ins[dtype] = make(8, 2, 100, 100, 2, 64, dtype, plan)
            step(*ins[dtype][:4], plan, ins[dtype][4])
        one = make(8, 2, 1, 900, 2, 64, torch.bfloat16, plan)
        ops.relpos_attention(*one[:4], plan)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs = {t: step(*x[:4], plan, x[4]) for t, x in ins.items()}
            single = ops.relpos_attention(*one[:4], plan)
        for turn in range(4):
            for t in ins:
                for x in ins[t]:
                    x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(turn)).to(x.dtype))
            graph.replay()
            stream.synchronize()
            for t, x in ins.items():
                want = step(*x[:4], plan, x[4])
                for n in want:
                    assert torch.equal(want[n], outs[t][n]), (turn, t, n)
            assert torch.equal(single, ops.relpos_attention(*one[:4], plan))


def test_nothing_to_do():
    plan = PLANS['log']()
    for B, Nq, Nk in ((0, 4, 4), (2, 0, 4), (2, 4, 0)):
        q, k, v, table, dout = make(1, B, Nq, Nk, 2, 16, torch.bfloat16, plan)
        got = step(q, k, v, table, plan, dout)
        assert not any(bool(x.any()) for x in got.values())
        assert got['dk'].shape == k.shape and got['dtable'].shape == table.shape


def test_only_some_gradients_and_twice_through_one_graph():
    plan = PLANS['log']()
    q, k, v, table, dout = make(11, 2, 60, 60, 2, 64, torch.float32, plan)
    want = step(q, k, v, table, plan, dout)
    kk = k.clone().requires_grad_(True)
    out = ops.relpos_attention(q, kk, v, table, plan)
    a = torch.autograd.grad(out, kk, dout, retain_graph=True)[0]
    b = torch.autograd.grad(out, kk, 2 * dout)[0]
    assert torch.equal(a, want['dk']) and torch.equal(b, 2 * want['dk'])
    t = table.clone().requires_grad_(True)
    out = ops.relpos_attention(q, k, v, t, plan)
    g = torch.autograd.grad(out.sum(), t, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize('dtype', list(DT))
def test_positions_with_lengths_and_other_orders(dtype):
    """given positions in any order, more keys than queries, lengths, and one query over many keys"""
    g = torch.Generator().manual_seed(12)
    for Nq, Nk, d in ((70, 200, 64), (1, 1400, 40), (130, 33, 128)):
        plan = RelPosBuckets(range(41), -20, positions=(torch.randint(-30, 30, (Nq,), generator=g), torch.randint(-30, 30, (Nk,), generator=g)))
        q, k, v, table, dout = make(13 + Nq, 3, Nq, Nk, 2, d, DT[dtype], plan)
        lens = torch.tensor([Nk, 0, Nk // 2 + 1], dtype=torch.int32, device='cuda')
        U.check(step(q, k, v, table, plan, dout, key_lens=lens), U.reference(q, k, v, table, plan, key_lens=lens, dout=dout))


@pytest.mark.parametrize('dtype', list(DT))
def test_the_widest_plan(dtype):
    """4095 differences and heads of 128: the most LDS that a call can ask for"""
    plan = RelPosBuckets.clipped(2047)
    q, k, v, table, dout = make(31, 1, 150, 2300, 2, 128, DT[dtype], plan)
    for off in (0, 2200):
        U.check(step(q, k, v, table, plan, dout, q_offset=off), U.reference(q, k, v, table, plan, q_offset=off, dout=dout))


@pytest.mark.parametrize('dtype', list(DT))
def test_zeros(dtype):
    plan = PLANS['clip']()
    q, k, v, table, dout = make(1, 2, 40, 40, 1, 32, DT[dtype], plan)
    for zero in (q, k, v, dout):
        ins = [torch.zeros_like(x) if x is zero else x for x in (q, k, v)]
        do = torch.zeros_like(dout) if zero is dout else dout
        U.check(step(*ins, table, plan, do), U.reference(*ins, table, plan, dout=do))
    ins = [torch.zeros_like(x) for x in (q, k, v)]
    got = step(*ins, torch.zeros_like(table), plan, torch.zeros_like(dout))
    assert not any(bool(x.any()) for x in got.values())


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('value', [math.inf, -math.inf, math.nan])
def test_what_is_not_finite_stays_where_it_is(value, dtype):
    """in one batch item: the others are as without it, the rows that meet it are NaN, and the table's gradient is"""
    plan = PLANS['clip']()
    q, k, v, table, dout = make(15, 3, 70, 70, 2, 64, DT[dtype], plan)
    want = U.reference(q, k, v, table, plan, dout=dout)
    for at in range(4):
        ins = [q.clone(), k.clone(), v.clone(), dout.clone()]
        ins[at][1, 20, 0, 5] = value
        got = step(*ins[:3], table, plan, ins[3])
        others = {n: got[n][[0, 2]] for n in ('out', 'dq', 'dk', 'dv')}
        U.check(others, {n: tuple(x[[0, 2]] for x in want[n]) for n in others})
        U.check({n: x[:, :, 1] for n, x in ((n, got[n][1:2]) for n in others)}, {n: tuple(x[1:2, :, 1] for x in want[n]) for n in others})      # the other head
        if at < 3:
            assert bool((~torch.isfinite(got['out'][1, :, 0])).any())
        assert not bool(torch.isfinite(got['dq'][1, :, 0]).all()) and not bool(torch.isfinite(got['dtable'][:, 0]).all())
        assert torch.isfinite(got['dtable'][:, 1]).all()


@pytest.mark.parametrize('dtype', list(DT))
def test_strides_beyond_32_bits(dtype):
    """batch, token and head strides whose offsets pass 2^32 bytes and 2^31 elements: the bits of contiguous copies"""
    plan = PLANS['log8']()
    room = torch.empty(5_000_000_000, dtype=DT[dtype], device='cuda')
    for shape, stride in (((3, 70, 2, 64), (2_200_000_000, 128, 64, 1)), ((1, 300, 2, 64), (0, 16_000_000, 64, 1)), ((2, 70, 2, 64), (128, 256, 4_400_000_000, 1))):
        q, k, v, table, dout = make(17, *shape[:2], *shape[1:], DT[dtype], plan)
        want = step(q, k, v, table, plan, dout)
        for i, x in enumerate((q, k, v, dout)):
            far = room.as_strided(shape, stride)
            far.copy_(x)
            ins = [q, k, v, dout]
            ins[i] = far
            got = step(*ins[:3], table, plan, ins[3])
            for n in want:
                assert torch.equal(want[n], got[n]), (shape, i, n)


def test_gradients_beyond_32_bits():
    """2^31 + key elements of a long cache, of which eight queries at its end see the last ones: those and their gradients as in the slice alone, none for the others"""
    N, H, d, last = 530_000, 32, 128, 1024
    plan = RelPosBuckets.clipped(100)
    g = torch.Generator(device='cuda').manual_seed(3)
    k, v = (torch.randn(1, N, H, d, generator=g, device='cuda', dtype=torch.bfloat16) for _ in range(2))
    q, dout = (torch.randn(1, 8, H, d, generator=g, device='cuda', dtype=torch.bfloat16) for _ in range(2))
    table = torch.randn(201, H, generator=g, device='cuda')
    table[0] = -math.inf                                      # nothing from 100 tokens back on
    got = step(q, k, v, table, plan, dout, q_offset=N - 8)
    ks, vs = k[:, -last:].clone(), v[:, -last:].clone()
    want = U.reference(q, ks, vs, table, plan, q_offset=last - 8, dout=dout)
    want.pop('dtable')
    U.check({n: got[n][:, -last:] if n in ('dk', 'dv') else got[n] for n in want}, want)
    assert not got['dk'][:, :-last].any() and not got['dv'][:, :-last].any()


def test_queries_beyond_32_bits():
    """2^31 + query elements over few keys: the last rows' output and gradient are those of the rows alone"""
    N, H, d = 530_000, 32, 128
    plan = RelPosBuckets.clipped(20)
    g = torch.Generator(device='cuda').manual_seed(4)
    q = torch.randn(1, N, H, d, generator=g, device='cuda', dtype=torch.bfloat16)
    k, v = (torch.randn(1, 16, H, d, generator=g, device='cuda', dtype=torch.bfloat16) for _ in range(2))
    table = torch.randn(41, H, generator=g, device='cuda')
    got = step(q, k, v, table, plan, q)
    rows = slice(N - 80, N)
    part = q[:, rows].clone()
    alone = step(part, k, v, table, plan, part, q_offset=N - 80)
    for n in ('out', 'dq'):
        assert torch.equal(got[n][:, rows], alone[n]), n
    for n in ('dk', 'dv', 'dtable'):
        assert torch.isfinite(got[n]).all() and bool(got[n].any())


@pytest.mark.parametrize('dtype', ['bf16', 'f16'])
@pytest.mark.parametrize('d', [72, 128])
def test_wide_heads_in_many_workgroups(d, dtype):
    """more workgroups than the chip has CUs: causal or not, with given positions, and lengths"""
    B, H = 5, 84
    lens = torch.tensor([70, 1, 0, 33, 64], dtype=torch.int32, device='cuda')
    g = torch.Generator().manual_seed(2)
    plan = RelPosBuckets(range(21), -10, positions=(torch.randint(-15, 15, (40,), generator=g), torch.randint(-15, 15, (70,), generator=g)))
    for plan, kw in ((PLANS['log8'](), dict(q_offset=30)), (PLANS['clip'](), dict(q_offset=25, causal=True)), (plan, {})):
        q, k, v, table, dout = make(41 + d, B, 40, 70, H, d, DT[dtype], plan)
        for n in (None, lens):
            U.check(step(q, k, v, table, plan, dout, key_lens=n, **kw), U.reference(q, k, v, table, plan, key_lens=n, dout=dout, **kw))


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('N', [40, 100, 600])
def test_large_values_that_nobody_meets(dtype, N):
    """causal: queries before the first key may be far larger than the others, and keys after the last query hold anything (unused places of a cache)"""
    plan = PLANS['causal']()
    big = 6e4 if dtype == 'f16' else 1e30
    q, k, v, table, dout = make(19, 2, 70, N, 2, 64, DT[dtype], plan)
    want = U.reference(q, k, v, table, plan, causal=True, q_offset=-30, dout=dout)      # queries 0 .. 29 see nothing, keys from 40 on are not seen
    base = step(q, k, v, table, plan, dout, causal=True, q_offset=-30)
    U.check(base, want)
    far_k, far_v = k.clone(), v.clone()
    for x in (big, math.nan):
        far_k[:, 40:], far_v[:, 40:] = x, -x
        got = step(q, far_k, far_v, table, plan, dout, causal=True, q_offset=-30)
        U.check(got, want)
        assert not got['dk'][:, 40:].any() and not got['dv'][:, 40:].any()
    far_q, far_do = q.clone(), dout.clone()
    far_q[:, :30], far_do[:, :30] = 1e4, -1e4
    got = step(far_q, k, v, table, plan, far_do, causal=True, q_offset=-30)
    U.check(got, U.reference(far_q, k, v, table, plan, causal=True, q_offset=-30, dout=far_do))


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('Nq', [1, 70, 161])
def test_biases_beyond_the_exponential(dtype, Nq):
    """buckets of +150, -200 and +1000: their exponentials are infinite or 0, the softmax is not (nor are the rows behind the last query, where such a bias meets no
    score)"""
    for name, causal in (('clip', False), ('log8', False), ('causal', True)):
        plan = PLANS[name]()
        for big, low in ((150.0, -200.0), (1000.0, 0.0)):
            q, k, v, table, dout = make(23, 2, Nq, 170, 2, 64, DT[dtype], plan)
            table[-1], table[1], table[2] = big, low, big - 3.0
            kw = dict(q_offset=170 - Nq if causal else 3, causal=causal)
            U.check(step(q, k, v, table, plan, dout, **kw), U.reference(q, k, v, table, plan, dout=dout, **kw))


@pytest.mark.parametrize('v_size,do_size', [(1e-22, 1e-25), (1e-30, 1e-30), (0.0, 1e-30), (1.0, 1e-30), (1e12, 1e12)])
def test_gradients_whose_scale_leaves_f32(v_size, do_size):
    """the product of the maxima of v and dout underflows, or is large.  Exponents of the planes end at 2^60: an operand whose maximum is below 2^-45 is held to 2^-85, half a
    subnormal step of f16, so out and dv are off by N 2^-85 at most and dq, dk, dtable by the N |q| or N |k| <= 600 x 5 roundings of dS that they sum: 1e-22 in all"""
    plan = PLANS['clip']()
    for N in (70, 600):
        q, k, v, table, dout = make(27, 1, N, N, 1, 64, torch.float32, plan)
        v, dout = v * v_size, dout * do_size
        U.check(step(q, k, v, table, plan, dout), U.reference(q, k, v, table, plan, dout=dout), tiny=1e-22)
