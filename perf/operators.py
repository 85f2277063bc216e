"""What a fine-tuning step with a learned relative position bias and a teacher's stored top logits asks of the GPU, operator by operator:

  attention    softmax(scale q k^T + table[bucket(position of key - position of query)]) v over (B, tokens, heads, d) tensors, alone or with the
               gradients of q, k, v and the table; causal and padded batches, one query against a long run of keys
  distill      the loss against the K stored logits of a teacher (with or without the mass of the classes that were not stored) and its gradient
  top_logits   what a teacher stores: the K largest logits of a row, their classes, and the log-sum-exp of the others

`run` computes them in elementary torch operations, or through the package's public entry points where `own` is true."""
import math

import torch

own = False

DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
SIZEOF = {'f32': 4, 'bf16': 2, 'f16': 2}


def attention(name, rule, B, Nq, Nk, H, d, dtype, train, buckets=32, distance=128, grid_h=0, grid_w=0, causal=False, lens=False):
    case = dict(op='attention', rule=rule, B=B, Nq=Nq, Nk=Nk, H=H, d=d, dtype=dtype, train=train, buckets=buckets, distance=distance,
                grid_h=grid_h, grid_w=grid_w, causal=causal, lens=lens)
    return dict(case, name=name) if name else case


def distill(name, R, V, K, dtype, tau, rest, short):
    case = dict(op='distill', R=R, V=V, K=K, dtype=dtype, tau=tau, rest=rest, short=short)
    return dict(case, name=name) if name else case


def top_logits(name, R, V, K, dtype, tau):
    case = dict(op='top_logits', R=R, V=V, K=K, dtype=dtype, tau=tau)
    return dict(case, name=name) if name else case


def listed():
    return [
        # fine-tuning: the block of the small model (6 heads of 64, 14 x 14 patches and a class token) at the batch of the search step
        attention('patch grid train', 'grid', 128, 197, 197, 6, 64, 'f32', True, grid_h=14, grid_w=14),
        # evaluation of a pruned subnet: ragged head width, larger batch
        attention('patch grid eval, pruned', 'grid', 256, 197, 197, 4, 40, 'f32', False, grid_h=14, grid_w=14),
        # the smallest step (tests, debugging runs): launch latency
        attention('tiny train', 'grid', 2, 17, 17, 3, 16, 'f32', True, grid_h=4, grid_w=4),
        # a text encoder's step on padded sequences, log-spaced buckets
        attention('padded encoder train', 'log', 16, 512, 512, 12, 64, 'bf16', True, lens=True),
        # a long document, no padding, odd length
        attention('long encoder train', 'log', 1, 6007, 6007, 16, 64, 'bf16', True),
        # a decoder's step: causal, one-sided buckets, wide heads
        attention('causal decoder train', 'log_causal', 4, 1025, 1025, 8, 128, 'f16', True, causal=True),
        # one new token of each of 24 sequences against what came before it
        attention('single token', 'log_causal', 24, 1, 4999, 16, 64, 'bf16', False, causal=True, lens=True),
        # distilling the classifier: 1000 classes, ten stored
        distill('classes', 1024, 1000, 10, 'f32', 2.0, True, False),
        # distilling a language model's step: a vocabulary, 64 stored of each token, some lists shorter
        distill('vocabulary', 2048, 100003, 64, 'bf16', 1.0, True, True),
        # a handful of tokens of a very large vocabulary, the stored logits renormalised
        distill('few rows', 7, 250002, 100, 'f16', 1.5, False, False),
        # the teacher's side of the two sizes
        top_logits('classes stored', 1024, 1000, 10, 'f32', 2.0),
        top_logits('vocabulary stored', 1024, 100003, 64, 'bf16', 1.0),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(['attention', 'attention', 'attention', 'distill', 'top_logits'])
    dtype = rng.choice(['f32', 'bf16', 'f16'])
    if op == 'attention':
        rule = rng.choice(['grid', 'log', 'log_causal', 'clip'])
        d = 8 * rng.randint(1, 16)
        H = rng.randint(1, 16)
        train = rng.random() < 0.6
        if rule == 'grid':
            gh, gw = rng.randint(2, 24), rng.randint(2, 24)
            n = gh * gw + 1
            B = max(1, min(_log_int(rng, 1, 256), 40_000_000 // (n * n * H)))
            return attention(None, rule, B, n, n, H, d, dtype, train, grid_h=gh, grid_w=gw, lens=rng.random() < 0.2)
        # a step trains on the whole sequence, or on its last part; a forward may meet a single token
        nk = _log_int(rng, 8 if train else 1, 6000)
        nq = nk if rng.random() < 0.6 else 1 if rng.random() < 0.5 and not train else _log_int(rng, max(1, nk // 4), nk) if train else _log_int(rng, 1, nk)
        B = max(1, min(_log_int(rng, 1, 64), 150_000_000 // (nq * nk * H), 60_000_000 // (nk * H * d)))
        buckets = 2 * rng.randint(2, 32)
        return attention(None, rule, B, nq, nk, H, d, dtype, train, buckets=buckets, distance=buckets * rng.randint(1, 12),
                         causal=rule == 'log_causal' or rng.random() < 0.3, lens=rng.random() < 0.4)
    V = _log_int(rng, 10, 260_000)
    R = max(1, min(_log_int(rng, 1, 4096), 100_000_000 // V))
    tau = rng.choice([0.5, 1.0, 2.0, 4.0])
    if op == 'distill':
        return distill(None, R, V, min(V // 2, _log_int(rng, 4, 256)), dtype, tau, rng.random() < 0.6, rng.random() < 0.4)
    return top_logits(None, R, V, min(V, _log_int(rng, 1, 256)), dtype, tau)


# ---------------------------------------------------------------------------------------------------------------------------------
# what a program has in hand
# ---------------------------------------------------------------------------------------------------------------------------------
def _thresholds(buckets, distance):
    """the smallest distance of each log-spaced bucket behind the first half: n^m first^k >= distance^k first^m, in whole numbers"""
    first = buckets // 2
    m = buckets - first
    found, n = [], first
    for k in range(1, m):
        while n ** m * first ** k < distance ** k * first ** m:
            n += 1
        found.append(n)
    return first, found


def _log_buckets(n, buckets, distance):
    """bucket of each distance n >= 0: one each below buckets / 2, log-spaced from there, the last from `distance` on"""
    first, thr = _thresholds(buckets, distance)
    far = first + (n[:, None] >= torch.tensor(thr, device=n.device, dtype=n.dtype)).sum(1) if thr else torch.full_like(n, first)
    return torch.where(n < first, n, far)


def _lut(case, device):
    """bucket by clamped distance -reach .. reach (1-D rules)"""
    reach = case['distance']
    delta = torch.arange(-reach, reach + 1, device=device)
    if case['rule'] == 'log':
        half = case['buckets'] // 2
        return _log_buckets(delta.abs(), half, reach) + half * (delta > 0)
    if case['rule'] == 'log_causal':
        return _log_buckets((-delta).clamp(min=0), case['buckets'], reach)
    return delta + reach                                                    # clip


def _table_rows(case):
    if case['rule'] == 'grid':
        return (2 * case['grid_h'] - 1) * (2 * case['grid_w'] - 1) + 3
    return 2 * case['distance'] + 1 if case['rule'] == 'clip' else case['buckets']


def _plan(case, device):
    from ofb_amd import RelPosBuckets
    if case['rule'] == 'grid':
        plan = RelPosBuckets.grid(case['grid_h'], case['grid_w'], cls_token=True)
    elif case['rule'] == 'clip':
        plan = RelPosBuckets.clipped(case['distance'])
    else:
        plan = RelPosBuckets.log_spaced(case['buckets'], case['distance'], bidirectional=case['rule'] == 'log')
    return plan.to(device)


def prepare(case, seed):
    dev = torch.device('cuda')
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=dev).to(dtype)

    dtype, state = DTYPES[case['dtype']], dict(case=case)
    if case['op'] == 'attention':
        B, Nq, Nk, H, d = (case[k] for k in ('B', 'Nq', 'Nk', 'H', 'd'))
        if Nq == Nk:                                                        # as a qkv projection leaves them: three views of one tensor
            q, k, v = normal(B, Nq, 3, H, d, dtype=dtype).unbind(2)
        else:
            q = normal(B, Nq, H, d, dtype=dtype)
            k, v = normal(B, Nk, 2, H, d, dtype=dtype).unbind(2)
        state.update(q=q.detach(), k=k.detach(), v=v.detach(), table=normal(_table_rows(case), H))
        if case['lens']:
            state['lens'] = torch.randint(Nk // 2, Nk + 1, (B,), generator=g, device=dev, dtype=torch.int32)
        if case['train']:
            for name in ('q', 'k', 'v', 'table'):
                state[name].requires_grad_(True)
            state['dout'] = normal(B, Nq, H, d, dtype=dtype)
        if own:
            state['plan'] = _plan(case, dev)
        elif case['rule'] != 'grid':
            state['lut'] = _lut(case, dev)
        return state
    R, V, K = case['R'], case['V'], case['K']
    z = normal(R, V) * 2.0
    if case['op'] == 'distill':
        tau = case['tau']
        # K different classes of each row: every (V // K)-th from a start of its own; a student that knows something of its teacher
        start = torch.randint(0, V, (R, 1), generator=g, device=dev)
        idx = (start + torch.arange(K, device=dev) * max(1, V // K)) % V
        # stored and other classes share the teacher's mass: logits around tau log(V / K), the others' sum around log V
        values = (tau * (normal(R, K) * 1.5 + math.log(V / K) + 1.0)).sort(1, descending=True).values
        z.scatter_add_(1, idx, 0.7 * values)
        if case['short']:                                                   # lists of fewer than K: the class of what is missing is -1
            have = torch.randint(K // 2, K + 1, (R, 1), generator=g, device=dev)
            idx = torch.where(torch.arange(K, device=dev) < have, idx, -1)
        state.update(z=z.to(dtype).requires_grad_(True), values=values.to(dtype), indices=idx.to(torch.int32))
        state['up'] = torch.full((), 4096.0 if case['dtype'] == 'f16' else 1.0, device=dev)     # f16 gradients: a loss scale, as scalers use
        state['rest'] = normal(R) * 0.3 + math.log(V) if case['rest'] else None
    else:
        state['z'] = z.to(dtype)
    return state


# ---------------------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------------------
def _bucket_matrix(case, state):
    """bucket of every (query, key) pair, by the positions of the two"""
    dev = state['q'].device
    if case['rule'] == 'grid':
        gh, gw = case['grid_h'], case['grid_w']
        cell = torch.arange(gh * gw, device=dev)
        y, x = cell // gw, cell % gw
        near = (y[None, :] - y[:, None] + gh - 1) * (2 * gw - 1) + (x[None, :] - x[:, None] + gw - 1)
        rows, n = _table_rows(case), gh * gw + 1
        out = torch.empty(n, n, device=dev, dtype=torch.int64)
        out[1:, 1:] = near
        out[0, 1:], out[1:, 0], out[0, 0] = rows - 3, rows - 2, rows - 1
        return out
    i = torch.arange(case['Nq'], device=dev) + (case['Nk'] - case['Nq'])
    j = torch.arange(case['Nk'], device=dev)
    reach = case['distance']
    return state['lut'][(j[None, :] - i[:, None]).clamp(-reach, reach) + reach]


def _plain_attention(state, bias):
    case = state['case']
    q, k, v = (state[n].float().transpose(1, 2) for n in ('q', 'k', 'v'))     # (B, H, tokens, d)
    Nq, Nk = case['Nq'], case['Nk']
    s = torch.matmul(q, k.transpose(2, 3)) * case['d'] ** -0.5
    s = s + bias
    if case['causal'] or case['lens']:
        j = torch.arange(Nk, device=q.device)
        seen = torch.ones(1, 1, 1, Nk, dtype=torch.bool, device=q.device)
        if case['causal']:
            seen = seen & (j[None, :] <= torch.arange(Nq, device=q.device)[:, None] + (Nk - Nq))
        if case['lens']:
            seen = seen & (j < state['lens'][:, None, None, None])
        s = s.masked_fill(~seen, -math.inf)
    top = s.detach().amax(-1, keepdim=True).clamp(min=-3e38)                  # a row that sees nothing: exp(-inf) = 0 everywhere
    e = torch.exp(s - top)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total > 0, total, 1.0)
    return torch.matmul(p, v).transpose(1, 2).to(state['q'].dtype).contiguous()


def _plain_table_grad(state, bucket, dbias):
    """the table's gradient from the bias's (H, Nq, Nk); the long sums in 64 bits"""
    case = state['case']
    Nq, Nk, H = case['Nq'], case['Nk'], case['H']
    out = torch.zeros(_table_rows(case), H, device=dbias.device, dtype=torch.float64)
    if case['rule'] == 'grid':
        return out.index_add_(0, bucket.reshape(-1), dbias.permute(1, 2, 0).reshape(-1, H).double()).float()
    # a pair's bucket goes by its distance: the last query first, each row one place further right, and the columns are the diagonals
    skew = torch.nn.functional.pad(dbias.flip(1), (0, Nq)).reshape(H, -1)[:, :Nq * (Nk + Nq - 1)].reshape(H, Nq, Nk + Nq - 1)
    at = torch.cat([bucket[:, 0].flip(0), bucket[0, 1:]])
    return out.index_add_(0, at, skew.sum(1, dtype=torch.float64).t().contiguous()).float()


def _plain_distill(state):
    tau, idx = state['case']['tau'], state['indices'].long()
    z = state['z'].float() / tau
    t = state['values'].float() / tau
    stored = idx >= 0
    t = t.masked_fill(~stored, -math.inf)
    at = idx.clamp(min=0)
    total = torch.logsumexp(t, 1)
    if state['rest'] is not None:
        total = torch.logaddexp(total, state['rest'])
    top = z.detach().amax(1, keepdim=True)
    e = torch.exp(z - top)
    log_all = torch.log(e.sum(1)) + top[:, 0]
    p = torch.exp(t - total[:, None])
    log_q = torch.gather(z, 1, at) - log_all[:, None]
    loss = (p * (torch.where(stored, t, 0.0) - total[:, None] - log_q) * stored).sum(1)
    if state['rest'] is not None:
        others = torch.ones_like(e, dtype=torch.bool)
        rows = torch.arange(z.shape[0], device=z.device)[:, None].expand_as(idx)
        others[rows[stored], idx[stored]] = False
        log_others = torch.log((e * others).sum(1)) + top[:, 0] - log_all
        log_p = state['rest'] - total
        loss = loss + torch.exp(log_p) * (log_p - log_others)
    return loss.mean() * tau * tau


def _plain_top_logits(state):
    z, K, tau = state['z'], state['case']['K'], state['case']['tau']
    ordered, at = torch.sort(z.float(), dim=1, descending=True, stable=True)   # ties: the lowest class first
    values, indices = ordered[:, :K].to(z.dtype), at[:, :K].to(torch.int32)
    others = ordered[:, K:] / tau
    if not others.shape[1]:
        return values, indices, torch.full((z.shape[0],), -math.inf, device=z.device)
    return values, indices, torch.log(torch.exp(others - others[:, :1]).sum(1)) + others[:, 0]


def run(state):
    case = state['case']
    if case['op'] == 'attention':
        bucket, bias = None, state['table']
        if own:
            from ofb_amd import ops
            out = ops.relpos_attention(state['q'], state['k'], state['v'], bias, state['plan'], causal=case['causal'],
                                       key_lens=state.get('lens'), q_offset=case['Nk'] - case['Nq'])
        else:
            bucket = _bucket_matrix(case, state)
            bias = bias.detach()[bucket].permute(2, 0, 1).contiguous().requires_grad_(case['train'])
            out = _plain_attention(state, bias)
        if not case['train']:
            return {'out': out}
        dq, dk, dv, db = torch.autograd.grad(out, [state['q'], state['k'], state['v'], bias], state['dout'])
        return {'out': out.detach(), 'dq': dq, 'dk': dk, 'dv': dv, 'dtable': db if own else _plain_table_grad(state, bucket, db)}
    if case['op'] == 'distill':
        if own:
            from ofb_amd import ops
            loss = ops.distill_top_logits(state['z'], state['values'], state['indices'], state['rest'], temperature=case['tau'])
        else:
            loss = _plain_distill(state)
        (dz,) = torch.autograd.grad(loss, [state['z']], state['up'])
        return {'loss': loss.detach(), 'dz': dz}
    if own:
        from ofb_amd import ops
        values, indices, rest = ops.top_logits(state['z'], case['K'], temperature=case['tau'])
    else:
        values, indices, rest = _plain_top_logits(state)
    return {'values': values, 'indices': indices, 'rest': rest}


def work(case):
    size = SIZEOF[case['dtype']]
    if case['op'] == 'attention':
        B, Nq, Nk, H, d = (case[k] for k in ('B', 'Nq', 'Nk', 'H', 'd'))
        pairs = Nq * Nk if not case['causal'] else sum(min(Nk, i + Nk - Nq + 1) for i in range(Nq))
        pairs *= 0.75 if case['lens'] else 1                                 # lengths are drawn between a half and the whole
        table = _table_rows(case) * H * 4
        moved = (2 * Nq + 2 * Nk) * B * H * d * size + table
        flops = 4 * B * H * pairs * d
        if case['train']:                                                    # reads q k v out dout again, writes dq dk dv and the table's
            moved += (4 * Nq + 4 * Nk) * B * H * d * size + 2 * table
            flops *= 3.5
        return {'bytes': moved, 'flops': flops}
    R, V, K = case['R'], case['V'], case['K']
    if case['op'] == 'distill':
        # the logits are read by the forward and again by the backward, which writes their gradient
        return {'bytes': R * V * size * 3 + R * K * (size + 4) + 4 * R, 'flops': 8 * R * V}
    return {'bytes': R * V * size + R * K * (size + 4) + 4 * R, 'flops': 4 * R * V}


# ---------------------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------------------
def _exact_bucket(case, delta):
    """bucket of one signed distance, from the logarithm (the guard is far above its error and far below the next whole distance)"""
    if case['rule'] == 'clip':
        return max(-case['distance'], min(case['distance'], delta)) + case['distance']
    n, rows, base = max(0, -delta), case['buckets'], 0
    if case['rule'] == 'log':
        rows //= 2
        n, base = abs(delta), rows if delta > 0 else 0
    first = rows // 2
    if n < first:
        return base + n
    if rows - first == 1 or case['distance'] <= first:
        return base + (rows - 1 if n >= case['distance'] or rows - first == 1 else first)
    return base + min(rows - 1, first + int(math.floor(math.log(n / first) / math.log(case['distance'] / first) * (rows - first) + 1e-9)))


def _exact_bias_rows(case, device):
    Nq, Nk = case['Nq'], case['Nk']
    if case['rule'] == 'grid':
        gh, gw, rows = case['grid_h'], case['grid_w'], _table_rows(case)
        at = [None] + [(c // gw, c % gw) for c in range(gh * gw)]
        table = [[rows - 1 if a is None and b is None else rows - 3 if a is None else rows - 2 if b is None else
                  (b[0] - a[0] + gh - 1) * (2 * gw - 1) + b[1] - a[1] + gw - 1 for b in at] for a in at]
        return torch.tensor(table, device=device)
    by_distance = torch.tensor([_exact_bucket(case, t) for t in range(-(Nk - 1), Nq + abs(Nk - Nq) + 1)], device=device)
    i = torch.arange(Nq, device=device).view(-1, 1)
    return by_distance[torch.arange(Nk, device=device).view(1, -1) - i - (Nk - Nq) + Nk - 1]


def _exact_attention(case, state):
    B, Nq, Nk, H, d = (case[k] for k in ('B', 'Nq', 'Nk', 'H', 'd'))
    dev, scale = state['q'].device, 1.0 / math.sqrt(d)
    rows = _exact_bias_rows(case, dev)
    hidden = torch.zeros(B, Nq, Nk, dtype=torch.bool, device=dev)
    if case['causal']:
        hidden |= torch.ones(Nq, Nk, dtype=torch.bool, device=dev).triu(1 + Nk - Nq)
    if case['lens']:
        for b, n in enumerate(state['lens'].tolist()):
            hidden[b, :, n:] = True
    got = {k: [] for k in ('out', 'dq', 'dk', 'dv', 'dtable')}
    for h in range(H):
        q, k, v = (state[n].detach()[:, :, h].double() for n in ('q', 'k', 'v'))
        s = torch.baddbmm(state['table'].detach()[:, h].double()[rows].expand(B, Nq, Nk), q, k.transpose(1, 2).contiguous(), alpha=scale)
        s[hidden] = -math.inf
        p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
        del s
        o = torch.bmm(p, v)
        got['out'].append(o)
        if not case['train']:
            continue
        do = state['dout'][:, :, h].double()
        got['dv'].append(torch.bmm(p.transpose(1, 2).contiguous(), do))
        ds = p * (torch.bmm(do, v.transpose(1, 2).contiguous()) - (do * o).sum(-1, keepdim=True))
        del p
        got['dq'].append(torch.bmm(ds, k) * scale)
        got['dk'].append(torch.bmm(ds.transpose(1, 2).contiguous(), q) * scale)
        got['dtable'].append(torch.zeros(_table_rows(case), device=dev, dtype=torch.float64).index_add_(0, rows.reshape(-1), ds.sum(0).reshape(-1)))
    if not case['train']:
        return {'out': torch.stack(got['out'], 2)}
    return {k: torch.stack(x, 1 if k == 'dtable' else 2) for k, x in got.items()}


def _exact_distill(case, state):
    R, V, tau = case['R'], case['V'], case['tau']
    losses, grads = [], []
    for r in range(0, R, 64):
        z = state['z'].detach()[r:r + 64].double() / tau
        n = z.shape[0]
        idx, t = state['indices'][r:r + 64].long(), state['values'][r:r + 64].double() / tau
        # the stored logits on the axis of all classes and one place behind it, which takes what was not stored and the rest
        target = torch.full((n, V + 1), -math.inf, device=z.device, dtype=torch.float64)
        target.scatter_(1, torch.where(idx < 0, V, idx), t)
        target[:, V] = state['rest'][r:r + 64].double() if state['rest'] is not None else -math.inf
        p = torch.softmax(target, 1)
        kept = torch.isfinite(target[:, :V])
        log_q = torch.log_softmax(z, 1)
        q = log_q.exp()
        mass = (q * ~kept).sum(1)
        log_rest = torch.logsumexp(log_q.masked_fill(kept, -math.inf), 1)
        loss = (torch.xlogy(p[:, :V], p[:, :V]) - p[:, :V] * log_q).sum(1)
        spread = torch.zeros(n, device=z.device, dtype=torch.float64)
        if state['rest'] is not None:
            loss = loss + torch.xlogy(p[:, V], p[:, V]) - p[:, V] * log_rest
            spread = p[:, V] / mass
        losses.append(loss)
        grads.append((q * torch.where(kept, 1.0, (1.0 - spread)[:, None]) - p[:, :V]) * (state['up'].double() * tau / R))
    return {'loss': torch.cat(losses).mean() * tau * tau, 'dz': torch.cat(grads)}


def exact(case, seed):
    state = prepare(case, seed)
    if case['op'] == 'attention':
        return _exact_attention(case, state)
    if case['op'] == 'distill':
        return _exact_distill(case, state)
    z, K = state['z'].double(), case['K']
    values = torch.topk(z, K, dim=1).values
    hold = torch.topk(z, K, dim=1).indices
    rest = torch.logsumexp(z.scatter(1, hold, -math.inf) / case['tau'], 1) if K < case['V'] else torch.full((case['R'],), -math.inf).double()
    return {'values': values, 'indices': None, 'rest': rest}
