"""The definition of attention with a relative position bias in 64 bits on the CPU, with element-wise error bounds for the kernels' arithmetic.

Bounds.  u = eps / 2 of the tensors' type.  The first products are exact in f32 up to the order of their sums (bf16, f16: d additions, d 2^-24 of the sum of
the absolute terms; f32: two f16 planes, 2^-21 a product more), exp2's argument and result are rounded once each: a probability is off by at most
e_P = e (1 + scale sum |q||k| + |bias| + |S - max|) relative, e = (d + 16) 2^-24, counted at the row's largest, and twice (the row's sum).  P and dS are rounded to the type
once more (u; f32: 2^-22), sums over n terms add n 2^-24.  f16 and f32 planes have an absolute floor of 2^-39 of their bound (half a subnormal step),
one plane of f16 of 2^-25 of the row's largest P in the forward (half a step of 2^-24 below 2^-14),
2^-39 for P in the backward (the same over the 2^14 of its scale) and 2^-39 of the bound for dS.  A bias beyond 1e30 swallows the score exactly.  Rounding the result to f16
is off by u of the value where it is a normal number and by half the subnormal step, 2^-25, below 2^-14: both are counted."""
import math

import torch


def bucket_matrix(plan, Nq, Nk, q_offset):
    pq = torch.tensor(plan.positions[0]) if plan.positions else torch.arange(Nq) + q_offset
    pk = torch.tensor(plan.positions[1]) if plan.positions else torch.arange(Nk)
    return torch.tensor(plan.lut)[(pk[None, :] - pq[:, None] - plan.lo).clamp(0, plan.width - 1)]


def reference(q, k, v, table, plan, scale=None, causal=False, key_lens=None, q_offset=0, dout=None):
    """{name: (value, bound)} in float64 for out and, with dout, dq, dk, dv, dtable"""
    dtype = q.dtype
    u = torch.finfo(dtype).eps / 2
    r = 2.0 ** -22 if dtype == torch.float32 else u
    q, k, v = (t.detach().cpu().double().transpose(1, 2) for t in (q, k, v))
    table = table.detach().cpu().double()
    B, H, Nq, d = q.shape
    Nk = k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    at = bucket_matrix(plan, Nq, Nk, q_offset)
    bias = table[at].permute(2, 0, 1)
    seen = torch.ones(B, 1, Nq, Nk, dtype=torch.bool)
    if causal:
        seen = seen & (torch.arange(Nk)[None, :] <= torch.arange(Nq)[:, None] + q_offset)
    if key_lens is not None:
        live = torch.arange(Nk)[None, :] < key_lens.cpu().long().clamp(0, Nk)[:, None]
        seen = seen & live[:, None, None, :]
        k, v = (torch.where(live[:, None, :, None], t, 0.0) for t in (k, v))      # what lies behind a length is not read
    s = (scale * (q @ k.transpose(2, 3)) + bias).masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    e = torch.exp(s - top)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total > 0, total, 1.0)
    o = p @ v
    c = 2.0 ** -24
    sub = 2.0 ** -25 if dtype == torch.float16 else 0.0
    size = abs(scale)
    near = seen & (s - top > -200)                           # beyond, P is 0 in f32 whatever the score's rounding
    spread = size * (q.abs() @ k.abs().transpose(2, 3)) + torch.where(bias.abs() < 1e30, bias.abs(), 0.0) + torch.where(near, (s - top).abs(), 0.0).clamp(max=100)
    e_p = 2 * (d + 16) * c * (1 + (spread * near).amax(-1, keepdim=True)) + 8 * c
    floor_p = 2.0 ** -39 if dtype == torch.float16 else 0.0
    floor_x = 2.0 ** -39 if dtype == torch.float32 else 0.0
    pv = p @ v.abs()
    floor_f = 2.0 ** -25 * p.amax(-1, keepdim=True) if dtype == torch.float16 else 0.0
    e_o = (e_p + r + (Nk + 8) * c) * pv + floor_f * v.abs().sum(2, keepdim=True) + floor_x * v.abs().amax()
    got = {'out': (o.transpose(1, 2), (e_o + u * (o.abs() + e_o) + sub).transpose(1, 2))}
    if dout is None:
        return got
    do = dout.detach().cpu().double().transpose(1, 2)
    D = (do * o).sum(-1, keepdim=True)
    dp = do @ v.transpose(2, 3)
    ds = p * (dp - D)
    e32 = (e_p + (Nk + 8) * c) * pv + floor_x * v.abs().amax()                      # the unrounded output; for bf16 / f16 P's rounding is in it too
    e_D = (do.abs() * (e32 + r * pv + floor_f * v.abs().sum(2, keepdim=True))).sum(-1, keepdim=True) + (d + 8) * c * (do.abs() * pv).sum(-1, keepdim=True)
    e_dp = (d + 16) * c * (do.abs() @ v.abs().transpose(2, 3)) + floor_x * d * do.abs().amax() * v.abs().amax()
    e_ds = e_p * ds.abs() + p * (1 + e_p) * (e_dp + e_D) + 4 * c * ds.abs()
    top_ds = 2 * d * do.abs().amax() * v.abs().amax()
    floor_ds = top_ds * (2.0 ** -39 if dtype != torch.bfloat16 else 0.0)
    def second(a, e_a, b, n, fl):
        """bound of a^T-like product already laid out: a (.., i, j), b (.., j, ch)"""
        return (e_a + r * a.abs() + n * c * a.abs()) @ b.abs() + fl * b.abs().sum(-2, keepdim=True) + floor_x * a.abs().sum(-1, keepdim=True) * b.abs().amax()
    dq, e_dq = scale * (ds @ k), size * second(ds, e_ds, k, Nk + 8, floor_ds)
    dk, e_dk = scale * (ds.transpose(2, 3) @ q), size * second(ds.transpose(2, 3), e_ds.transpose(2, 3), q, Nq + 8, floor_ds)
    dv, e_dv = p.transpose(2, 3) @ do, second(p.transpose(2, 3), (e_p * p).transpose(2, 3), do, Nq + 8, floor_p)
    for name, x, ex in (('dq', dq, e_dq), ('dk', dk, e_dk), ('dv', dv, e_dv)):
        got[name] = (x.transpose(1, 2), (ex + u * (x.abs() + ex) + sub).transpose(1, 2))
    flat = at.reshape(-1)
    def by_bucket(x):
        return torch.zeros(plan.num_buckets, H, dtype=torch.float64).index_add_(0, flat, x.sum(0).permute(1, 2, 0).reshape(-1, H))
    sums = by_bucket(ds)
    # sums over the batch and, beyond the ends, over a query's keys run in f32
    got['dtable'] = (sums, by_bucket(e_ds + (B + Nk + 32) * c * ds.abs()) + 2.0 ** -23 * sums.abs())
    return got


def check(got, want, tiny=1e-30):
    worst = {}
    for name, x in got.items():
        ref, bound = want[name]
        x = x.detach().cpu().double()
        assert x.shape == ref.shape, (name, tuple(x.shape), tuple(ref.shape))
        assert torch.isfinite(x).all(), name
        off = (x - ref).abs()
        ratio = float((off / (bound + tiny)).max()) if off.numel() else 0.0
        worst[name] = ratio
        assert ratio <= 1.0, f'{name}: {ratio:.3g} of its bound, worst error {float(off.max()):.3g} at {float(ref.abs().max()):.3g}'
    return worst
