"""Buckets of relative positions and the refusals of ops.relpos_attention (no GPU)."""
import copy
import math
import pickle

import pytest
import torch

from ofb_amd import RelPosBuckets, hip, ops


def by_logarithm(delta, buckets, reach, bidirectional):
    n, rows, base = max(0, -delta), buckets, 0
    if bidirectional:
        rows //= 2
        n, base = abs(delta), rows if delta > 0 else 0
    exact = rows // 2
    if n < exact:
        return base + n
    if n >= reach:
        return base + rows - 1
    # the guard is far above the logarithm's error and far below the next whole distance's step
    return base + min(rows - 1, exact + int(math.floor(math.log(n / exact) / math.log(reach / exact) * (rows - exact) + 1e-9)))


@pytest.mark.parametrize('buckets,reach,two', [(32, 128, True), (32, 128, False), (16, 64, False), (8, 20, True), (4, 9, True), (64, 1000, True), (12, 7, True)])
def test_log_spaced(buckets, reach, two):
    p = RelPosBuckets.log_spaced(buckets, reach, bidirectional=two)
    assert p.num_buckets == buckets
    for delta in range(-2 * reach - 3, 2 * reach + 4):
        assert p.lut[min(max(delta - p.lo, 0), p.width - 1)] == by_logarithm(delta, buckets, reach, two), delta


@pytest.mark.parametrize('h,w,cls', [(14, 14, True), (3, 5, True), (5, 2, False), (1, 1, True), (1, 1, False)])
def test_grid(h, w, cls):
    p = RelPosBuckets.grid(h, w, cls_token=cls)
    at = ([None] if cls else []) + [divmod(c, w) for c in range(h * w)]
    rows = (2 * h - 1) * (2 * w - 1)
    assert p.num_buckets == rows + 3 * cls
    for i, a in enumerate(at):
        for j, b in enumerate(at):
            got = p.lut[min(max(p.positions[1][j] - p.positions[0][i] - p.lo, 0), p.width - 1)]
            want = rows + 2 if a is None and b is None else rows if a is None else rows + 1 if b is None else (b[0] - a[0] + h - 1) * (2 * w - 1) + b[1] - a[1] + w - 1
            assert got == want, (a, b)


def test_clipped_trimming_and_copies():
    p = RelPosBuckets.clipped(3)
    assert (p.lut, p.lo, p.num_buckets) == (list(range(7)), -3, 7)
    p = RelPosBuckets([2, 2, 2, 0, 1, 1], -4, num_buckets=5)
    assert (p.lut, p.lo, p.num_buckets) == ([2, 0, 1], -2, 5)
    assert RelPosBuckets([4, 4, 4], 9).lut == [4]
    lut, start, order, pq, pk = p.on('cpu')
    assert lut.tolist() == [2, 0, 1] and start.tolist() == [0, 1, 2, 3, 3, 3] and order.tolist() == [1, 2, 0] and pq is None and pk is None
    assert copy.deepcopy(p) is p
    q = pickle.loads(pickle.dumps(p))
    assert (q.lut, q.lo, q.num_buckets, q.positions) == (p.lut, p.lo, p.num_buckets, p.positions)


@pytest.mark.parametrize('make', [
    lambda: RelPosBuckets([], 0), lambda: RelPosBuckets([0, -1], 0), lambda: RelPosBuckets([0, 3], 0, num_buckets=3), lambda: RelPosBuckets(range(4097), 0),
    lambda: RelPosBuckets([0], 1 << 30), lambda: RelPosBuckets([0], 0, num_buckets=1 << 21), lambda: RelPosBuckets([0], 0, positions=([1 << 30], [0])), lambda: RelPosBuckets.log_spaced(7, 20), lambda: RelPosBuckets.log_spaced(0, 20),
    lambda: RelPosBuckets.log_spaced(32, 8), lambda: RelPosBuckets.clipped(-1), lambda: RelPosBuckets.clipped(2048), lambda: RelPosBuckets.grid(0, 3), lambda: RelPosBuckets.grid(40, 40),
    lambda: RelPosBuckets.log_spaced(1000, 100000)])
def test_plans_that_are_refused(make):
    with pytest.raises(hip.OfbError):
        make()


def test_refusals():
    plan = RelPosBuckets.log_spaced(8, 20)
    t = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype)
    q, k, table = t(2, 5, 3, 16), t(2, 7, 3, 16), t(8, 3)
    grid = RelPosBuckets.grid(2, 2)
    bad = [
        dict(q=t(2, 5, 48)), dict(q=t(2, 5, 3, 16, dtype=torch.float64)), dict(k=t(2, 7, 3, 16, dtype=torch.bfloat16)), dict(k=t(2, 7, 1, 16), v=t(2, 7, 1, 16)),
        dict(v=t(2, 6, 3, 16)), dict(k=t(1, 7, 3, 16), v=t(1, 7, 3, 16)), dict(q=t(2, 5, 3, 12), k=t(2, 7, 3, 12), v=t(2, 7, 3, 12)),
        dict(q=t(2, 5, 3, 136), k=t(2, 7, 3, 136), v=t(2, 7, 3, 136)), dict(table=t(7, 3)), dict(table=t(8, 3, dtype=torch.bfloat16)), dict(key_lens=torch.zeros(2, dtype=torch.int64)),
        dict(key_lens=torch.zeros(3, dtype=torch.int32)), dict(buckets=[0, 1]), dict(table=None), dict(q_offset=1 << 30), dict(buckets=grid, table=t(12, 3)), dict(q=t(2, 5, 0, 16), k=t(2, 7, 0, 16), v=t(2, 7, 0, 16), table=t(8, 0)),
        dict(buckets=grid, table=t(12, 3), k=t(2, 5, 3, 16), v=t(2, 5, 3, 16), causal=True), dict(buckets=grid, table=t(12, 3), k=t(2, 5, 3, 16), v=t(2, 5, 3, 16), q_offset=1),
        dict(),                                                # CPU tensors: there is no fallback
    ]
    for change in bad:
        a = dict(dict(q=q, k=k, v=k, table=table, buckets=plan), **change)
        with pytest.raises(hip.OfbError):
            ops.relpos_attention(**a)
    for qkv, kw in ((t(2, 5, 2, 3, 16), {}), (t(2, 5, 3, 3, 16), dict(bound=torch.zeros(2)))):
        with pytest.raises(hip.OfbError):
            ops.relpos_attention_qkv(qkv, table, plan, **kw)


def test_entry_refuses_what_the_kernels_cannot_take():
    """the C entry's own checks: no launch is made"""
    import ctypes as C
    lib = hip.lib()
    base = dict(q=16, k=16, v=16, table=16, lut=16, out=16, width=3, n_buckets=3, lo=-1, B=2, H=3, Nq=5, Nk=7, d=16, scale=1.0, dtype=1)
    strides = {f'{n}_{s}': x for n in ('q', 'k', 'v', 'o') for s, x in (('sb', 240), ('st', 48), ('sh', 16))}
    def run(**kw):
        a = hip.RelposArgs()
        for n, x in {**base, **strides, **kw}.items():
            setattr(a, n, x)
        return lib.ofb_relpos_fwd(C.byref(a), None)
    bad = [dict(q=None), dict(q=8), dict(d=12), dict(d=0), dict(B=0), dict(Nq=0), dict(dtype=3), dict(width=0), dict(q_st=44), dict(v_sb=-8), dict(o_st=2), dict(pos_q=16),
           dict(pos_q=16, pos_k=16, causal=1), dict(out=8), dict(dtype=0, n_bound=1), dict(dtype=0, Nk=5000), dict(dtype=0, bound_k=16), dict(n_bound=257), dict(n_bound=-1)]
    assert [run(**b) for b in bad] == [-1] * len(bad)
    limit = [dict(d=136), dict(width=4097), dict(n_buckets=1 << 21), dict(q_offset=1 << 30), dict(B=1 << 20, H=1 << 10, Nk=1 << 12)]
    assert [run(**b) for b in limit] == [-2] * len(limit)
    assert lib.ofb_relpos_fwd(None, None) == -1 and lib.ofb_relpos_bwd(None, None) == -1 and lib.ofb_relpos_sizes(None, None) == -1 and lib.ofb_relpos_amax(None, 0, 1, None) == -1


def test_entries_refuse_launches_that_are_too_large():
    """threads of a launch count in 32 bits; strides that the loads of 16 bytes cannot take"""
    import ctypes as C
    lib = hip.lib()
    def args(**kw):
        a = hip.RelposArgs()
        for n, x in {**dict(q=16, k=16, v=16, table=16, lut=16, out=16, width=3, n_buckets=3, lo=-1, B=2, H=3, Nq=5, Nk=7, d=16, scale=1.0, dtype=1), **kw}.items():
            setattr(a, n, x)
        return C.byref(a)
    assert lib.ofb_relpos_fwd(args(B=1 << 14, H=1 << 10, Nk=1), None) == -2
    grads = dict(dout=16, out32=16, stats=16, delta=16, dq=16, dk=16, dv=16, dtable=16)
    assert lib.ofb_relpos_bwd(args(B=1, H=1 << 10, n_buckets=1 << 14, **grads), None) == -2
    assert lib.ofb_relpos_bwd(args(**grads), None) == -1      # no room for the table's parts
    bounds = dict(bound_q=16, bound_k=16, bound_v=16)
    assert lib.ofb_relpos_amax(args(q_st=12, **bounds), 0, 1, None) == -1 and lib.ofb_relpos_amax(args(v_sb=-8, **bounds), 0, 3, None) == -1


def test_what_a_plan_uploads():
    for plan in (RelPosBuckets.grid(3, 2), RelPosBuckets([5, 0, 5, 2], -1, 9), RelPosBuckets.grid(1, 1), RelPosBuckets([0], 0, positions=([], []))):
        lut, start, order, pq, pk = plan.on('cpu')
        assert lut.tolist() == plan.lut and order.tolist() == sorted(range(plan.width), key=lambda i: (plan.lut[i], i))
        assert start.tolist() == [sum(x < c for x in plan.lut) for c in range(plan.num_buckets + 1)]
        assert all(t.dtype == torch.int32 for t in (lut, start, order))
        assert (pq.tolist(), pk.tolist()) == tuple(plan.positions) if plan.positions else pq is None and pk is None


def test_bias_tables_are_not_decayed():
    import ofb_amd
    from ofb_amd.lr_decay import param_groups_lrd
    m = ofb_amd.VisionTransformer(img_size=32, patch_size=8, embed_dim=32, depth=2, num_heads=2, num_classes=5, rel_pos_bias=True)
    tables = [f'blocks.{i}.attn.relative_position_bias_table' for i in range(2)]
    assert m.no_weight_decay() == ['pos_embed', 'cls_token', 'dist_token'] + tables
    plain = ofb_amd.VisionTransformer(img_size=32, patch_size=8, embed_dim=32, depth=2, num_heads=2, num_classes=5)
    assert plain.no_weight_decay() == ['pos_embed', 'cls_token', 'dist_token']
    by_id = {id(p): n for n, p in m.named_parameters()}
    kept = {by_id[id(p)] for g in param_groups_lrd(m, no_weight_decay_list=m.no_weight_decay()) if g['weight_decay'] == 0 for p in g['params']}
    assert set(tables) <= kept


def test_a_plan_is_kept_for_the_streams_that_read_it(monkeypatch):
    """every stream that a call of the plan runs on is made known to the allocator once, for the memory of all its parts"""
    from ofb_amd import relpos
    device, current, known, syncs = torch.device('cuda', 0), [7], [], []

    class Stream:
        synchronize = staticmethod(lambda: syncs.append(current[0]))

    monkeypatch.setattr(relpos, 'raw_stream', lambda d: current[0])
    monkeypatch.setattr(torch.cuda, 'current_stream', lambda d=None: Stream)
    monkeypatch.setattr(torch.Tensor, 'to', lambda self, d: self)
    monkeypatch.setattr(torch.Tensor, 'record_stream', lambda self, s: known.append((current[0], self.untyped_storage().data_ptr())))
    for plan in (RelPosBuckets.grid(2, 3), RelPosBuckets.clipped(4)):
        known.clear(), syncs.clear()
        parts = plan.on(device)
        memory = {t.untyped_storage().data_ptr() for t in parts if t is not None}
        assert syncs == [7] and not known and len(memory) == 1
        for current[0] in (7, 8, 8, 9, 7, 8):
            assert plan.on(device) is parts
        assert known == [(8, *memory), (9, *memory)] and syncs == [7]
        current[0] = 7
