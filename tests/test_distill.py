"""Refusals of ops.top_logits and ops.distill_top_logits (no GPU)."""
import pytest
import torch

from ofb_amd import hip, ops


def test_refusals():
    t = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    good = dict(logits=t(4, 9), values=t(4, 3), indices=i32(4, 3), rest=t(4))
    bad = [dict(logits=t(9)), dict(logits=t(4, 9, dtype=torch.float64), values=t(4, 3, dtype=torch.float64)), dict(values=t(4, 2)), dict(values=t(3, 3), indices=i32(3, 3)),
           dict(values=t(4, 3, dtype=torch.bfloat16)), dict(indices=t(4, 3)), dict(rest=t(3)), dict(rest=t(4, dtype=torch.float64)), dict(temperature=0.0), dict(temperature=float('inf')),
           dict(temperature=float('nan')), dict(reduction='batchmean'), dict(values=t(4, 10), indices=i32(4, 10)), dict(values=t(4, 0), indices=i32(4, 0)), dict(values=None),
           dict(logits=t(0, 9), values=t(0, 3), indices=i32(0, 3), rest=None),
           dict()]                                            # CPU tensors: there is no fallback
    for change in bad:
        with pytest.raises(hip.OfbError):
            ops.distill_top_logits(**dict(good, **change))
    for a in ((t(9), 1), (t(4, 9), 0), (t(4, 9), 10), (t(4, 2000), 1025), (t(4, 9, dtype=torch.float64), 1), (t(4, 9), 1, -1.0), (t(4, 9), 1)):
        with pytest.raises(hip.OfbError):
            ops.top_logits(*a)


def test_entries_refuse_what_the_kernels_cannot_take():
    import ctypes as C
    lib = hip.lib()
    p, i, L, f = C.c_void_p, C.c_int32, C.c_int64, C.c_float
    def fwd(z=16, R=4, V=9, K=3, tau=1.0, dtype=0, stats=16, part=None, rows=16):
        return lib.ofb_distill_fwd(p(z), p(16), p(16), i(0), None, L(R), i(V), i(K), f(tau), i(dtype), p(stats), p(part), p(rows), C.c_double(1), None, None)
    assert [fwd(**k) for k in (dict(z=None), dict(z=8), dict(R=0), dict(V=0), dict(K=0), dict(tau=0.0), dict(dtype=5), dict(stats=None), dict(rows=None), dict(V=1 << 20))] == [-1] * 10
    assert [fwd(**k) for k in (dict(K=10), dict(V=5000, K=1025), dict(V=(1 << 30) + 1), dict(R=(1 << 24) + 1))] == [-2] * 4
    bwd = lambda up, dz: lib.ofb_distill_bwd(p(16), p(16), p(16), i(0), L(4), i(9), i(3), f(1.0), i(0), p(16), p(up), i(0), f(1.0), p(dz), None)
    assert bwd(None, 16) == -1 and bwd(16, None) == -1 and bwd(16, 8) == -1
    top = lambda rest, V: lib.ofb_top_logits(p(16), L(1), i(V), i(3), f(1.0), i(0), p(16), p(16), p(rest), None, None, None)
    assert top(None, 9) == -1 and top(16, 1 << 20) == -1
    assert lib.ofb_distill_segments(L(0), i(5)) == 0 and lib.ofb_top_logits_segments(L(5), i(5), i(0)) == 0


def test_too_many_rows():
    z = torch.zeros(1, 1).expand(1 << 22, 1)
    with pytest.raises(hip.OfbError, match='2.22'):
        ops.top_logits(z, 1)
    with pytest.raises(hip.OfbError, match='2.22'):
        ops.distill_top_logits(z, z, z.int())
