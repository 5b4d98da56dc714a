"""The operators of a verification round whose requests are tenants of one
model: a prompt that many of them share, low-rank adapters of their own beside
the shared q/k/v projection, and sampling rules of their own on the logits.

A case is a dict of plain values.  Request lengths are drawn from its
`lengths` number, tensor values from the seed given to prepare, so one case
has the same sizes under every seed.  The geometry is the package's: 16 query
heads, 8 KV heads, head dim 128, hidden 1024; vocabulary 151,936 unless a case
says otherwise.
"""
import math
import random

import torch

own = False

DEV = 'cuda'
HQ, HKV, D, HIDDEN, VOCAB = 16, 8, 128, 1024, 151936
HEADS = HQ + 2 * HKV
SCALE = D ** -0.5
EPS, THETA = 1e-6, 1e6
NEG = float('-inf')


def listed():
    return [
        # Two users answer one token each after a short system prompt: latency.
        dict(name='prefix_2', kind='prefix', requests=2, groups=1, q_min=1, q_max=1, prefix=500, own_min=0, own_max=40,
             lengths=1),
        # A mid-sized batch verifies 7 tokens each over a prompt of 2,000 that it shares.
        dict(name='prefix_16', kind='prefix', requests=16, groups=1, q_min=7, q_max=7, prefix=2000, own_min=20,
             own_max=300, lengths=2),
        # A full batch, ragged proposals, a long document asked about by all.
        dict(name='prefix_64_long', kind='prefix', requests=64, groups=1, q_min=1, q_max=8, prefix=8192, own_min=64,
             own_max=1024, lengths=3),
        # Twelve users' first prompts after one of two long system prompts (prefill).
        dict(name='prefix_prompts', kind='prefix', requests=12, groups=2, q_min=100, q_max=400, prefix=6000, own_min=0,
             own_max=0, lengths=4),
        # One user, one token, a small adapter: latency.
        dict(name='adapters_1', kind='adapters', requests=1, q_min=1, q_max=1, adapters=1, rank=8, bare=False,
             lengths=5),
        # A full verification batch over two dozen adapters, some requests without one.
        dict(name='adapters_64', kind='adapters', requests=64, q_min=7, q_max=7, adapters=24, rank=16, bare=True,
             lengths=6),
        # A decode batch whose every request has an adapter of its own, of a high rank.
        dict(name='adapters_32_r64', kind='adapters', requests=32, q_min=1, q_max=1, adapters=32, rank=64, bare=False,
             lengths=7),
        # New prompts of four adapters.
        dict(name='adapters_prompts', kind='adapters', requests=6, q_min=200, q_max=1500, adapters=4, rank=32,
             bare=False, lengths=8),
        # One user samples one token with penalties: latency.
        dict(name='controls_1', kind='controls', requests=1, n_min=0, n_max=0, vocab=VOCAB, dtype='bfloat16',
             history=300, bias=0, mask=False, lengths=9),
        # A full verification round under grammars, each row with its own mask.
        dict(name='controls_64', kind='controls', requests=64, n_min=7, n_max=7, vocab=VOCAB, dtype='bfloat16',
             history=2000, bias=20, mask=True, lengths=10),
        # A decode batch of long conversations with many biases, FP32 logits.
        dict(name='controls_32_fp32', kind='controls', requests=32, n_min=0, n_max=0, vocab=VOCAB, dtype='float32',
             history=30000, bias=300, mask=False, lengths=11),
        # A small vocabulary of odd size (rows are not aligned), ragged proposals, masks.
        dict(name='controls_odd', kind='controls', requests=16, n_min=0, n_max=5, vocab=32003, dtype='bfloat16',
             history=700, bias=5, mask=True, lengths=12),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(max(lo, 1)), math.log(hi + 1))))))


def _cost(case):
    w = work(case)
    return max(w['bytes'], w['flops'] / 50)


def draw(rng):
    kind = rng.choice(('prefix', 'adapters', 'controls'))
    most = max(_cost(c) for c in listed() if c['kind'] == kind)
    while True:
        case = dict(kind=kind, lengths=rng.randrange(1 << 30))
        if kind == 'prefix':
            prompts = rng.random() < 0.3
            q_max = _log_int(rng, 9, 400) if prompts else rng.randint(1, 8)
            own_max = 0 if rng.random() < 0.2 else _log_int(rng, 1, 1500)
            case.update(requests=_log_int(rng, 2, 64), groups=rng.randint(1, 3), q_min=rng.randint(1, q_max),
                        q_max=q_max, prefix=_log_int(rng, 64, 16384), own_min=0, own_max=own_max)
        elif kind == 'adapters':
            q_max = _log_int(rng, 9, 1500) if rng.random() < 0.3 else rng.randint(1, 8)
            n = _log_int(rng, 1, 64)
            case.update(requests=n, q_min=rng.randint(1, q_max), q_max=q_max, adapters=rng.randint(1, min(n, 48)),
                        rank=rng.choice((4, 8, 16, 24, 32, 64)), bare=rng.random() < 0.3)
        else:
            n_max = rng.choice((0, 0, 5, 7, 12))
            case.update(requests=_log_int(rng, 1, 64), n_min=rng.randint(0, n_max), n_max=n_max,
                        vocab=rng.choice((VOCAB, _log_int(rng, 1000, 200000))),
                        dtype=rng.choice(('bfloat16', 'float32')), history=_log_int(rng, 1, 30000),
                        bias=rng.choice((0, 3, 300)), mask=rng.random() < 0.5)
        if _cost(case) <= most:
            return case


def _sizes(case):
    """The case's request lengths (and what else it draws per request)."""
    rng = random.Random(case['lengths'])
    n = case['requests']
    if case['kind'] == 'prefix':
        group = [r % case['groups'] for r in range(n)]            # members of a prompt are not neighbours
        prefix = [max(1, case['prefix'] - rng.randint(0, case['prefix'] // 4) * (g > 0)) for g in range(case['groups'])]
        return dict(group=group, prefix=prefix, q=[rng.randint(case['q_min'], case['q_max']) for _ in range(n)],
                    own=[rng.randint(case['own_min'], case['own_max']) for _ in range(n)])
    if case['kind'] == 'adapters':
        ids = [r % case['adapters'] for r in range(n)]
        rng.shuffle(ids)
        if case['bare']:
            ids = [-1 if rng.random() < 0.15 else a for a in ids]
        return dict(q=[rng.randint(case['q_min'], case['q_max']) for _ in range(n)], ids=ids)
    length = [rng.randint(min(1, case['history']), case['history']) for _ in range(n)]
    return dict(n=[rng.randint(case['n_min'], case['n_max']) for _ in range(n)], length=length,
                prompt=[rng.randint(0, x) for x in length],
                repetition=[rng.choice((1.0, 1.1, 1.3)) for _ in range(n)],
                presence=[rng.choice((0.0, 0.4, 1.5)) for _ in range(n)],
                frequency=[rng.choice((0.0, 0.05, 0.2)) for _ in range(n)])


def _starts(lengths):
    out = [0]
    for x in lengths:
        out.append(out[-1] + x)
    return out


def prepare(case, seed):
    s = _sizes(case)
    gen = torch.Generator(device=DEV).manual_seed(seed * 1000003 + case['lengths'] % 999983)
    state = {'prefix': _prepare_prefix, 'adapters': _prepare_adapters, 'controls': _prepare_controls}[case['kind']](
        case, s, gen, random.Random(seed * 7919 + case['lengths']))
    state['kind'] = case['kind']
    if own:
        state['call'] = {'prefix': _own_prefix, 'adapters': _own_adapters, 'controls': _own_controls}[case['kind']](
            case, s, state)
    return state


def run(state):
    if own:
        return state['call']()
    return {'prefix': _plain_prefix, 'adapters': _plain_adapters, 'controls': _plain_controls}[state['kind']](state)


def work(case):
    s = _sizes(case)
    if case['kind'] == 'prefix':
        t = sum(s['q'])
        keys = sum(s['prefix']) + sum(s['own']) + t
        pairs = sum(q * (s['prefix'][g] + o) + q * (q + 1) // 2 for q, o, g in zip(s['q'], s['own'], s['group']))
        return {'bytes': 2 * HKV * D * 2 * keys + 2 * HQ * D * 2 * t, 'flops': 4 * HQ * D * pairs}
    if case['kind'] == 'adapters':
        t, r = sum(s['q']), case['rank']
        with_one = sum(q for q, a in zip(s['q'], s['ids']) if a >= 0)
        used = len({a for a in s['ids'] if a >= 0})
        side = 3 * HIDDEN + HEADS * D
        return {'bytes': 2 * (HEADS * D * HIDDEN + t * HIDDEN + used * r * side + t * HEADS * D) + 4 * D * t,
                'flops': 2 * t * HEADS * D * HIDDEN + 2 * with_one * r * side}
    rows = sum(s['n']) + len(s['n'])
    elem = 2 if case['dtype'] == 'bfloat16' else 4
    mask = rows * ((case['vocab'] + 31) // 32) * 4 if case['mask'] else 0
    return {'bytes': 2 * rows * case['vocab'] * elem + mask + 8 * (sum(s['length']) + sum(s['n'])),
            'flops': rows * case['vocab']}


def exact(case, seed):
    return {'prefix': _exact_prefix, 'adapters': _exact_adapters, 'controls': _exact_controls}[case['kind']](
        case, _sizes(case), prepare(case, seed))


def _index(lists, fill=0):
    """Ragged index lists as a padded [rows, longest] device tensor."""
    longest = max(len(x) for x in lists)
    return torch.tensor([list(x) + [fill] * (longest - len(x)) for x in lists], device=DEV)


# -- attention of a batch that shares long prompts ------------------------------
def _prepare_prefix(case, s, gen, rng):
    def rnd(*shape, scale=1.0):
        return (scale * torch.randn(*shape, generator=gen, device=DEV)).to(torch.bfloat16)

    t, n = sum(s['q']), case['requests']
    at, own_at = _starts(s['q']), _starts(s['own'])
    state = dict(q=rnd(t, HQ, D, scale=1.5), new_k=rnd(t, HKV, D), new_v=rnd(t, HKV, D),
                 own_k=rnd(own_at[-1], HKV, D), own_v=rnd(own_at[-1], HKV, D),
                 prefix_k=rnd(case['groups'], max(s['prefix']), HKV, D),
                 prefix_v=rnd(case['groups'], max(s['prefix']), HKV, D))
    # where each request's rows are: what a program that packs its batch knows
    members = [[r for r in range(n) if s['group'][r] == g] for g in range(case['groups'])]
    tokens = [[i for r in m for i in range(at[r], at[r + 1])] for m in members]
    slot = {i: (g, j) for g, x in enumerate(tokens) for j, i in enumerate(x)}
    spot = [(r, i - at[r]) for r in range(n) for i in range(at[r], at[r + 1])]
    state.update(
        group_tokens=_index(tokens), prefix_len=torch.tensor(s['prefix'], device=DEV),
        token_group=torch.tensor([slot[i] for i in range(t)], device=DEV),
        request_tokens=_index([range(at[r], at[r + 1]) for r in range(n)]),
        request_keys=_index([[*range(own_at[r], own_at[r + 1]), *range(own_at[-1] + at[r], own_at[-1] + at[r + 1])]
                             for r in range(n)]),
        own_len=torch.tensor(s['own'], device=DEV), token_request=torch.tensor(spot, device=DEV))
    return state


def _plain_part(q, k, v, visible):
    """Softmax sums of queries [B, n, 16, 128] over keys [B, m, 8, 128]; visible
    [B, n or 1, m].  Returns (max, sum, weighted values) per [B, n, 8, 2]."""
    b, n = q.shape[:2]
    x = q.float().view(b, n, HKV, 2, D).permute(0, 2, 1, 3, 4).reshape(b, HKV, 2 * n, D)
    y = k.float().permute(0, 2, 3, 1).contiguous()
    seen = visible.expand(b, n, -1).repeat_interleave(2, 1).unsqueeze(1)
    scores = (torch.matmul(x, y) * SCALE).masked_fill(~seen, NEG)
    top = scores.amax(-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(scores - top)
    o = torch.matmul(p, v.float().permute(0, 2, 1, 3).contiguous())

    def back(z):
        return z.view(b, HKV, n, 2, -1).permute(0, 2, 1, 3, 4)
    return back(top), back(p.sum(-1, keepdim=True)), back(o)


def _plain_prefix(state):
    prefix_k = state['prefix_k']
    keys = torch.arange(prefix_k.shape[1], device=DEV)
    one = _plain_part(state['q'][state['group_tokens']], prefix_k, state['prefix_v'],
                      (keys < state['prefix_len'][:, None])[:, None])
    k = torch.cat((state['own_k'], state['new_k']))[state['request_keys']]
    v = torch.cat((state['own_v'], state['new_v']))[state['request_keys']]
    last = state['own_len'][:, None] + torch.arange(state['request_tokens'].shape[1], device=DEV)
    two = _plain_part(state['q'][state['request_tokens']], k, v,
                      torch.arange(k.shape[1], device=DEV) <= last[:, :, None])
    g, r = state['token_group'].unbind(1), state['token_request'].unbind(1)
    m1, l1, o1 = (z[g[0], g[1]] for z in one)
    m2, l2, o2 = (z[r[0], r[1]] for z in two)
    m = torch.maximum(m1, m2)
    w1, w2 = torch.exp(m1 - m), torch.exp(m2 - m)
    out = (w1 * o1 + w2 * o2) / (w1 * l1 + w2 * l2)
    return out.reshape(-1, HQ, D).to(torch.bfloat16)


def _own_prefix(case, s, state):
    """The store with the prompts shared, the requests' own rows committed and
    the transaction of the round open, its new rows staged."""
    from qwen3_dspark_amd.persistent_kv import Bucket, PersistentTargetKV
    n, at, own_at = case['requests'], _starts(s['q']), _starts(s['own'])
    held = [r for r in range(n) if s['own'][r]]
    ceiling = max(s['prefix']) + max(s['own'])
    store = PersistentTargetKV(layers=1, slots=n + case['groups'], context_capacity=ceiling + max(*s['q'], *s['own'], 1),
                               max_query_tokens=max(at[-1], own_at[-1]), heads=HKV, dim=D, device=DEV,
                               shared_prefixes=True)
    handles = []
    prompts = [store.add_request(f'prompt {g}') for g in range(case['groups'])]
    for g, h in enumerate(prompts):
        length = s['prefix'][g]
        store.load_prefix(h, state['prefix_k'][g:g + 1, :length].contiguous(),
                          state['prefix_v'][g:g + 1, :length].contiguous())
    for r in range(n):
        h = store.add_request(f'request {r}')
        store.share_prefix(prompts[s['group'][r]], h, s['prefix'][s['group'][r]])
        handles.append(h)
    if held:
        bucket = Bucket(tuple(s['own'][r] for r in held), tuple(s['prefix'][s['group'][r]] for r in held), 'own rows')
        store.register_bucket(bucket)
        tx = store.begin([handles[r] for r in held], bucket)
        store.stage_layer(tx, 0, state['own_k'], state['own_v'])
        store.commit(tx, {handles[r]: s['own'][r] for r in held})
    bucket = Bucket(tuple(s['q']), tuple(s['prefix'][g] + o for g, o in zip(s['group'], s['own'])), 'round')
    store.register_bucket(bucket)
    tx = store.begin(handles, bucket)
    store.stage_layer(tx, 0, state['new_k'], state['new_v'])
    return lambda: store.attend(tx, 0, state['q'])


def _exact_prefix(case, s, state):
    at, own_at = _starts(s['q']), _starts(s['own'])
    out = torch.empty(at[-1], HQ, D, dtype=torch.float64, device=DEV)
    for r in range(case['requests']):
        g, q = s['group'][r], s['q'][r]
        k, v = (torch.cat((state['prefix_' + x][g, :s['prefix'][g]], state['own_' + x][own_at[r]:own_at[r + 1]],
                           state['new_' + x][at[r]:at[r + 1]])).double() for x in 'kv')
        hidden = torch.ones(q, k.shape[0], dtype=torch.bool, device=DEV).triu(k.shape[0] - q + 1)
        for h in range(HQ):
            p = (state['q'][at[r]:at[r + 1], h].double() @ k[:, h // 2].T.contiguous() * SCALE).masked_fill(hidden, NEG)
            out[at[r]:at[r + 1], h] = torch.softmax(p, -1) @ v[:, h // 2].contiguous()
    return out


# -- low-rank adapters beside the q/k/v projection --------------------------------
def _prepare_adapters(case, s, gen, rng):
    def rnd(*shape, scale):
        return (scale * torch.randn(*shape, generator=gen, device=DEV)).to(torch.bfloat16)

    t, n, r = sum(s['q']), case['adapters'], case['rank']
    positions = torch.tensor([p + i for q in s['q'] for p in [rng.randint(0, 8000)] for i in range(q)], device=DEV)
    angle = positions.double()[:, None] * THETA ** (torch.arange(0, D, 2, device=DEV).double() / -D)
    out = HIDDEN ** -0.5
    return dict(x=rnd(t, HIDDEN, scale=1.0), positions=positions, rope=torch.cat((angle.cos(), angle.sin()), 1).float(),
                w={p: rnd(h * D, HIDDEN, scale=out) for p, h in (('q', HQ), ('k', HKV), ('v', HKV))},
                norm={p: 1 + rnd(D, scale=0.2) for p in 'qk'},
                a={p: rnd(n, r, HIDDEN, scale=out) for p in 'qkv'},
                b={p: rnd(n, h * D, r, scale=r ** -0.5) for p, h in (('q', HQ), ('k', HKV), ('v', HKV))},
                scaling=[rng.choice((0.25, 0.5, 1.0)) for _ in range(n)],
                ids=torch.tensor([a for a, q in zip(s['ids'], s['q']) for _ in range(q)], device=DEV))


def _norm_rope(y, weight, rope):
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * weight
    c, s = rope[:, None, :D // 2], rope[:, None, D // 2:]
    lo, hi = y[..., :D // 2], y[..., D // 2:]
    return torch.cat((lo * c - hi * s, hi * c + lo * s), -1)


def _plain_adapters(state):
    x, ids = state['x'].float(), state['ids']
    n, r = state['a']['q'].shape[:2]
    keep = torch.tensor(state['scaling'], device=DEV) * (ids[:, None] == torch.arange(n, device=DEV))

    def project(p):
        u = torch.matmul(x, state['a'][p].float().view(n * r, HIDDEN).T) * keep.repeat_interleave(r, 1)
        y = torch.matmul(x, state['w'][p].float().T)
        y = y + torch.matmul(u, state['b'][p].float().transpose(1, 2).reshape(n * r, -1))
        return y.view(len(ids), -1, D)
    q, k, v = (_norm_rope(project(p), state['norm'][p].float(), state['rope']) if p in 'qk' else project(p)
               for p in 'qkv')
    return tuple(z.to(torch.bfloat16) for z in (q, k, v))


def _own_adapters(case, s, state):
    from qwen3_dspark_amd.adapters import AdapterBatch, QKVAdapters
    from qwen3_dspark_amd.prologue import QKVPrologue
    prologue = QKVPrologue(state['w']['q'], state['w']['k'], state['w']['v'], state['norm']['q'], state['norm']['k'],
                           eps=EPS, theta=THETA)
    adapters = QKVAdapters(*(state[m][p] for p in 'qkv' for m in 'ab'), scaling=state['scaling'])
    batch = AdapterBatch(DEV, s['q'], s['ids'])
    return lambda: prologue(state['x'], state['positions'], rope=state['rope'], adapters=adapters, batch=batch)


def _exact_adapters(case, s, state):
    outs, at = [], _starts(s['q'])
    for p, heads in (('q', HQ), ('k', HKV), ('v', HKV)):
        y = state['x'].double() @ state['w'][p].double().T.contiguous()
        for r, a in enumerate(s['ids']):
            rows = slice(at[r], at[r + 1])
            if a >= 0:
                low = state['a'][p][a].double() @ state['x'][rows].double().T.contiguous()
                y[rows] += state['scaling'][a] * (state['b'][p][a].double() @ low).T
        y = y.view(-1, heads, D)
        if p != 'v':
            y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / D + EPS) * state['norm'][p].double()
            turn = torch.complex(state['rope'][:, :D // 2].double(), state['rope'][:, D // 2:].double())[:, None]
            z = torch.complex(y[..., :D // 2], y[..., D // 2:]) * turn
            y = torch.cat((z.real, z.imag), -1)
        outs.append(y)
    return tuple(outs)


# -- penalties, biases and grammar masks on logits ----------------------------------
def _prepare_controls(case, s, gen, rng):
    v, n, rows = case['vocab'], case['requests'], sum(s['n']) + case['requests']
    words = (v + 31) // 32

    def tokens(*shape):                         # a few thousand tokens make up most of a text
        u = torch.rand(*shape, generator=gen, device=DEV)
        return (v * u ** 3).long().clamp_max(v - 1)
    state = dict(logits=(3 * torch.randn(rows, v, generator=gen, device=DEV)).to(getattr(torch, case['dtype'])),
                 history=tokens(n, max(s['length'])), proposed=tokens(sum(s['n'])),
                 bias=[{rng.randrange(v): rng.choice((-4.0, -0.5, 1.0, 3.5)) for _ in range(case['bias'])} or None
                       for _ in range(n)], allowed=None)
    if case['mask']:
        bits = torch.randint(0, 1 << 32, (rows, words), generator=gen, device=DEV)
        strict = torch.rand(rows, 1, generator=gen, device=DEV) < 0.3         # few tokens follow a bracket
        few = torch.rand(rows, words, generator=gen, device=DEV) < 0.02
        bits = torch.where(strict & ~few, torch.zeros_like(bits), bits)
        bits[:, 0] |= 2                                                       # every row allows one at least
        state['allowed'] = (bits - ((bits >> 31) << 32)).to(torch.int32)      # unsigned words held in int32
    # the batch's layout, as a program that packs it knows it
    at = _starts(s['n'])
    state.update(row_request=torch.tensor([r for r in range(n) for _ in range(s['n'][r] + 1)], device=DEV),
                 length=torch.tensor(s['length'], device=DEV), prompt=torch.tensor(s['prompt'], device=DEV))
    pairs = [(at[r] + r + j, at[r] + i) for r in range(n) for j in range(s['n'][r] + 1) for i in range(j)]
    state['pairs'] = torch.tensor(pairs, dtype=torch.long, device=DEV).view(-1, 2)   # (row, proposed token before it)
    for k in ('repetition', 'presence', 'frequency'):
        state[k] = torch.tensor(s[k], device=DEV)
    flat = [(r, t, b) for r, d in enumerate(state['bias']) if d for t, b in d.items()]
    state['bias_at'] = torch.tensor([x[:2] for x in flat], dtype=torch.long, device=DEV).view(-1, 2)
    state['bias_value'] = torch.tensor([x[2] for x in flat], device=DEV)
    return state


def _plain_controls(state):
    logits, history, row = state['logits'], state['history'], state['row_request']
    n, v = history.shape[0], logits.shape[1]
    place = torch.arange(history.shape[1], device=DEV)
    held = place < state['length'][:, None]
    answer = (held & (place >= state['prompt'][:, None])).float()
    counts = torch.zeros(n, v, device=DEV).scatter_add_(1, history, answer)
    seen = torch.zeros(n, v, device=DEV).scatter_add_(1, history, held.float())
    counts, seen = counts[row], seen[row]
    pair = state['pairs'][:, 0], state['proposed'][state['pairs'][:, 1]]
    counts.index_put_(pair, torch.ones(len(pair[0]), device=DEV), accumulate=True)
    seen.index_put_(pair, torch.ones(len(pair[0]), device=DEV), accumulate=True)
    x = logits.float()
    rep = state['repetition'][row][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - counts * state['frequency'][row][:, None] - (counts > 0) * state['presence'][row][:, None]
    bias = torch.zeros(n, v, device=DEV)
    bias[state['bias_at'][:, 0], state['bias_at'][:, 1]] = state['bias_value']
    x = x + bias[row]
    if state['allowed'] is not None:
        bit = torch.arange(32, device=DEV, dtype=torch.int32)
        keep = ((state['allowed'][:, :, None] >> bit) & 1).view(len(row), -1)[:, :v]
        x = x.masked_fill(keep == 0, NEG)
    return x.to(logits.dtype)


def _own_controls(case, s, state):
    from qwen3_dspark_amd.sampling import LogitControls
    controls = LogitControls(DEV, case['vocab'], repetition=s['repetition'], presence=s['presence'],
                             frequency=s['frequency'], bias=state['bias'], masked=NEG)
    return lambda: controls(state['logits'], state['history'], lengths=s['length'], prompt_lengths=s['prompt'],
                            counts=s['n'], tokens=state['proposed'], allowed=state['allowed'])


def _exact_controls(case, s, state):
    v, rows, at = case['vocab'], [], _starts(s['n'])
    place = torch.arange(v, device=DEV)
    for r in range(case['requests']):
        text, prompt = state['history'][r, :s['length'][r]], s['prompt'][r]
        whole, answer = torch.bincount(text, minlength=v), torch.bincount(text[prompt:], minlength=v)
        for j in range(s['n'][r] + 1):
            before = torch.bincount(state['proposed'][at[r]:at[r] + j], minlength=v)
            i = len(rows)
            x = state['logits'][i].double()
            rep = torch.full_like(x, s['repetition'][r])
            x = torch.where(whole + before > 0, x * torch.where(x > 0, 1 / rep, rep), x)
            count = (answer + before).double()
            x = x - s['frequency'][r] * count - s['presence'][r] * (count > 0)
            if state['bias'][r]:
                x[list(state['bias'][r])] += torch.tensor(list(state['bias'][r].values()), dtype=x.dtype, device=DEV)
            if state['allowed'] is not None:
                x[(state['allowed'][i][place // 32] >> (place % 32)) & 1 == 0] = NEG
            rows.append(x)
    return torch.stack(rows)
