"""Lineages, groups and plans of requests that share committed rows (CPU): every plan
covers each request's keys exactly once, its partial tiles are disjoint and within the
capacity, and its regions hold what the kernels read."""
import ctypes
import random

import pytest
import torch

from kv_fake import store
from qwen3_dspark_amd import _native, shared_prefix
from qwen3_dspark_amd.schedule import REQ_INTS, WORK_INTS
from qwen3_dspark_amd.shared_prefix import (PREFIX_TILE, common_rows, inherited, mixed_part_ints, shared_capacity,
                                            shared_groups, shared_ints, shared_plan)


def test_lineages():
    a = ((1, None),)
    b = inherited(a, 1000, 2)
    d = inherited(b, 1500, 4)
    assert b == ((1, 1000), (2, None)) and d == ((1, 1000), (2, 1500), (4, None))
    assert inherited(b, 1000, 5) == ((1, 1000), (5, None)) and inherited(b, 700, 5) == ((1, 700), (5, None))
    assert inherited(a, 0, 6) == ((6, None),)
    assert [common_rows(*x) for x in ((a, b), (b, d), (a, d), (d, inherited(a, 300, 7)), (a, ((9, None),)))] == \
        [1000, 1500, 1000, 300, 0]
    assert common_rows(a, a) is None


@pytest.fixture(autouse=True)
def groups_of_any_size(monkeypatch):
    monkeypatch.setattr(shared_prefix, 'MIN_SAVED', 0)
    monkeypatch.setattr(shared_prefix, 'MIN_LONG_ROWS', 0)


def rows_of(lineage, length):
    """Who wrote each row."""
    out = []
    for origin, end in lineage:
        out += [origin] * ((length if end is None else min(end, length)) - len(out))
    return out


def family(rng, n):
    """Random requests: fresh ones, and ones that share rows of an earlier one."""
    lineages, lengths = [], []
    for r in range(n):
        if lineages and rng.random() < 0.7:
            s = rng.randrange(len(lineages))
            rows = rng.randint(0, lengths[s])
            lineages.append(inherited(lineages[s], rows, r))
            lengths.append(rows + rng.choice((0, rng.randint(0, 900))))
        else:
            lineages.append(((r, None),))
            lengths.append(rng.choice((0, rng.randint(0, 70), rng.randint(0, 5000))))
    return lineages, lengths


def check_plan(queries, keys, slots, groups, n_cu=256):
    c = shared_capacity(len(queries), sum(queries), max(queries), n_cu)
    out = shared_plan(queries, keys, slots, groups, n_cu, c).tolist()
    assert len(out) == shared_ints(c) and mixed_part_ints(c) % 8 == 0
    n_work = c.run_records + c.prompt_records
    at = WORK_INTS * n_work
    ranges = out[at:at + c.runs + 1]
    requests = [out[at + c.runs + 1 + REQ_INTS * r:][:REQ_INTS] for r in range(c.requests)]
    columns = out[at + c.runs + 1 + REQ_INTS * c.requests:][:2 * c.columns]
    base = mixed_part_ints(c)
    items = [out[base + 8 + 8 * i:][:8] for i in range(out[base])]
    tokens = [out[base + 8 + 8 * c.items + 4 * i:][:4] for i in range(c.tokens)]
    q0 = [sum(queries[:r]) for r in range(len(queries))]
    width = [-(-q // 8) for q in queries]
    covered = [[] for _ in queries]
    tiles = [[] for _ in queries]

    def own(rec, decode):
        r, k0, k1, slot, row, q, k, start = rec
        assert (row, q, k, start) == (q0[r], queries[r], keys[r], slots[r]) and (q <= 8) == decode
        covered[r].append((k0, k1))
        if slot >= 0:
            tiles[r] += range(slot, slot + width[r])
        else:
            assert requests[r][1] == 1

    assert ranges[0] == 0 and ranges == sorted(ranges) and ranges[-1] <= c.run_records
    for i in range(ranges[-1]):
        own(out[8 * i:8 * i + 8], True)
    seen = set()
    for i in range(0, len(columns), 2):
        record, t = columns[i] - 1, columns[i + 1]
        if record < 0:
            continue
        rec = out[8 * record:8 * record + 8]
        assert 32 * t < rec[5] and (record, t) not in seen
        seen.add((record, t))
        if t == 0:
            own(rec, False)
    for record, _ in seen:
        assert {t for x, t in seen if x == record} == set(range(-(-out[8 * record + 5] // 32)))
    by_token = {}
    for slot, k0, k1, seg, first, n, _, _ in items:
        assert k0 % PREFIX_TILE == 0 and k1 % PREFIX_TILE == 0 and k0 < k1 and 1 <= n <= 32
        for row, tile, sub, step in tokens[first:first + n]:
            by_token.setdefault(row, []).append((k0, k1, tile + seg * step, sub, slot))
    for r, q in enumerate(queries):
        prefix = {tuple(sorted((k0, k1, slot) for k0, k1, _, _, slot in by_token.get(q0[r] + t, []))) for t in range(q)}
        assert len(prefix) == 1
        prefix = prefix.pop()
        group = [g for g in groups if r in g.members]
        if group:
            assert prefix and {s for _, _, s in prefix} == {group[0].slot} and prefix[-1][1] == group[0].length
        else:
            assert not prefix
        for t in range(q):
            for _, _, tile, sub, _ in by_token.get(q0[r] + t, []):
                assert sub == t % 8
                if t % 8 == 0:
                    tiles[r].append(tile)
                else:
                    assert tile in tiles[r]
        spans = sorted([(a, b) for a, b, _ in prefix] + covered[r])
        assert spans[0][0] == 0 and spans[-1][1] == keys[r] and all(x[1] == y[0] for x, y in zip(spans, spans[1:]))
        first, count, row, rows = requests[r]
        assert (row, rows) == (q0[r], q) and count == len(spans)
        assert sorted(tiles[r]) == (list(range(first, first + count * width[r])) if count > 1 else [])
    every = sorted(x for t in tiles for x in t)
    assert len(set(every)) == len(every) and (not every or every[-1] < c.tiles)
    return items


@pytest.mark.parametrize('seed', range(40))
def test_random_plans(seed):
    rng = random.Random(seed)
    n = rng.choice((1, 2, 3, 7, 20, 64))
    lineages, contexts = family(rng, n)
    longest = rng.choice((1, 8, 8, 40, 300))
    queries = [rng.randint(1, longest) for _ in range(n)]
    slots = rng.sample(range(100), n)
    groups = shared_groups(lineages, contexts, slots)
    members = [r for g in groups for r in g.members]
    assert len(set(members)) == len(members)
    for g in groups:
        assert len(g.members) > 1 and g.length % PREFIX_TILE == 0 and 0 < g.length <= min(contexts[r] for r in g.members)
        assert g.slot in [slots[r] for r in g.members]
        assert len({tuple(rows_of(lineages[r], contexts[r])[:g.length]) for r in g.members}) == 1
    check_plan(queries, [c + q for c, q in zip(contexts, queries)], slots, groups, rng.choice((256, 64, 304)))


@pytest.mark.parametrize('n,q,rows,own', [(64, 1, 16384, 0), (64, 8, 100000, 5), (2, 1, 64, 0), (12, 400, 6000, 0),
                                          (256, 7, 2048, 30), (2, 2000, 30000, 100), (1024, 2, 640, 1), (3, 9, 64, 0)])
def test_large_and_small_plans(n, q, rows, own):
    a = ((0, None),)
    lineages = [inherited(a, rows, 1 + r) for r in range(n)]
    groups = shared_groups(lineages, [rows + own] * n, list(range(n)))
    assert [(len(g.members), g.length) for g in groups] == [(n, rows // 64 * 64)]
    check_plan([q] * n, [rows + own + q] * n, list(range(n)), groups)


def test_requests_with_few_keys_of_their_own_have_runs():
    """64 requests of one token right behind the prefix: a run each, not 8 a run."""
    groups = [shared_prefix.Group(list(range(64)), 512, 5)]
    c = shared_capacity(64, 64, 1, 256)
    out = shared_plan([1] * 64, [513] * 64, list(range(64)), groups, 256, c).tolist()
    ranges = out[WORK_INTS * c.run_records:WORK_INTS * c.run_records + c.runs + 1]
    assert max(b - a for a, b in zip(ranges, ranges[1:])) <= 2 and ranges[-1] <= 80


def test_columns_where_the_cus_are_no_whole_rounds():
    """38 CUs per KV head: prompts are cut for 76 workgroups, of which runs take 72."""
    check_plan([206, 300, 300, 300, 51, 300, 153, 1], [207, 302, 300, 3605, 51, 656, 153, 1], list(range(8)), [], 304)


def test_members_that_would_shorten_a_group_stay_out():
    a = ((0, None),)
    lineages = [a, inherited(a, 4000, 1), inherited(a, 4000, 2), inherited(a, 100, 3), inherited(a, 120, 4)]
    groups = shared_groups(lineages, [5000, 4000, 4100, 100, 400], [4, 3, 2, 1, 0])
    assert [(g.members, g.length, g.slot) for g in groups] == [([0, 1, 2], 3968, 4), ([3, 4], 64, 1)]
    assert shared_groups(lineages[3:], [63, 400], [1, 0]) == []
    assert shared_groups([a], [5000], [0]) == []


def test_forks_below_forks():
    """64 rows of a system prompt, on which one request puts a document that two others take
    over; then the same with more requests on the system prompt alone."""
    system, doc = ((0, None),), inherited(((0, None),), 64, 1)
    lineages = [doc, inherited(doc, 8000, 2), inherited(doc, 8100, 3)]
    groups = shared_groups(lineages, [8500, 8000, 8100], [7, 8, 9])
    assert [tuple(g) for g in groups] == [([0, 1, 2], 8000, 7)]
    lineages += [inherited(system, 64, 4), inherited(system, 60, 5), system]
    groups = shared_groups(lineages, [8500, 8000, 8100, 70, 60, 70], [7, 8, 9, 1, 2, 3])
    assert sorted(map(tuple, groups)) == [([0, 1, 2], 8000, 7), ([3, 5], 64, 1)]
    # 40 share 1,024 rows of the system prompt, 3 of which 1,088 in all: those stay
    doc = inherited(system, 1024, 1)
    lineages = [doc, inherited(doc, 1088, 2), inherited(doc, 1088, 3), *(inherited(system, 1024, 10 + r) for r in range(37))]
    groups = shared_groups(lineages, [1100] * 40, list(range(40)))
    assert [(len(g.members), g.length) for g in groups] == [(40, 1024)]


def test_long_chains_of_forks():
    chain = [((0, None),)]
    for r in range(1, 1500):
        chain.append(inherited(chain[-1], 64 * r, r))          # each has 64 rows of its own
    n = len(chain)
    groups = shared_groups(chain, [64 * (r + 1) for r in range(n)], list(range(n)))
    held = [r for g in groups for r in g.members]
    assert len(held) == len(set(held)) and all(g.length <= 64 * (min(g.members) + 1) for g in groups)
    groups = shared_groups([chain[-1], chain[-1][:-1] + ((9999, None),)], [64 * n] * 2, [0, 1])
    assert [tuple(g) for g in groups] == [([0, 1], 64 * (n - 1), 0)]


def test_groups_that_would_save_little_are_none(monkeypatch):
    monkeypatch.undo()
    a = ((0, None),)
    lineages = [a, *(inherited(a, 2048, r) for r in range(1, 4))]
    assert shared_groups(lineages[:2], [2048] * 2, [0, 1]) == []
    assert [g.length for g in shared_groups(lineages[:3], [2048] * 3, [0, 1, 2])] == [2048]
    assert [g.length for g in shared_groups(lineages, [2048, 1500, 1500, 1500], [0, 1, 2, 3])] == [1472]
    # prompts: by the rows they share
    assert [g.length for g in shared_groups(lineages[:2], [2048] * 2, [0, 1], [33, 33])] == [2048]
    assert [g.length for g in shared_groups(lineages[:2], [800] * 2, [0, 1], [1, 64])] == [768]
    assert shared_groups(lineages, [767] * 4, [0, 1, 2, 3], [400] * 4) == []
    assert shared_groups(lineages[:2], [2048] * 2, [0, 1], [32, 32]) == []


def test_share_prefix_in_the_store():
    pool = store(slots=4, context_capacity=24)
    a, b, c, d = (pool.add_request(x) for x in 'abcd')
    x = torch.randn(pool.layers, 9, pool.heads, pool.dim)
    pool.load_prefix(a, x, x + 1)
    pool.share_prefix(a, b, 7)
    pool.share_prefix(b, c, 5)
    assert [pool.length(h) for h in (a, b, c, d)] == [9, 7, 5, 0]
    assert torch.equal(pool.request_kv(c)[0], x[:, :5]) and torch.equal(pool.request_kv(b)[1], x[:, :7] + 1)
    assert common_rows(pool._ledger.lineage(a.index), pool._ledger.lineage(c.index)) == 5
    for args in ((a, b, 3), (a, a, 0), (a, d, 10), (a, d, -1), (a, d, 2.0), (a, d, True), (d, d, 0)):
        with pytest.raises(ValueError, match='empty slot'):
            pool.share_prefix(*args)
    pool.share_prefix(a, d, 0)
    assert pool.length(d) == 0
    pool.remove_request(a)
    assert torch.equal(pool.request_kv(b)[0], x[:, :7])
    with pytest.raises(ValueError, match='incarnation'):
        pool.share_prefix(a, d, 1)
    e = pool.add_request('e')
    assert e.index == a.index and common_rows(pool._ledger.lineage(e.index), pool._ledger.lineage(b.index)) == 0
    pool.kv_device.fail = 'write_prefix'
    with pytest.raises(RuntimeError, match='injected'):
        pool.share_prefix(b, d, 1)
    assert pool.failed


def test_constructor_refusals():
    from kv_fake import CpuKVDevice
    from qwen3_dspark_amd.persistent_kv import PersistentTargetKV
    dims = dict(layers=1, slots=1, context_capacity=8, max_query_tokens=4, heads=8, dim=128)
    for kw in (dict(split='request'), dict(kv_device=CpuKVDevice(**dims))):
        with pytest.raises(ValueError, match='Shared prefixes need balanced'):
            PersistentTargetKV(**dims, shared_prefixes=True, **kw)
    with pytest.raises(ValueError, match='True or False'):
        PersistentTargetKV(**dims, shared_prefixes=1)
    with pytest.raises(RuntimeError, match='gfx950'):
        PersistentTargetKV(**dims, shared_prefixes=True, device='cpu')


def test_entry_point_checks():
    lib = _native.load()
    fake = ctypes.c_void_p(1 << 20)                # never dereferenced

    def call(**kw):
        args = dict(q=fake, q_rows=8, k_res=fake, v_res=fake, k_new=fake, v_new=fake, k_scr=fake, v_scr=fake, n_req=1,
                    slot_stride=8 * 128 * 64, tok_stride=128, head_stride=128 * 64, max_q=8, scale=0.1, work=fake, n_work=1,
                    n_groups=8, n_columns=0, prefixes=fake, max_items=1, max_tokens=8, members=8, turn=8, part_tiles=1,
                    out=fake, workspace=fake, workspace_bytes=1 << 20, stream=None)
        args.update(kw)
        return lib.dspark_shared_attn_fwd(*args.values()), lib.dspark_last_error().decode()
    odd = ctypes.c_void_p((1 << 20) + 8)
    for kw, match in (*((dict.fromkeys((x,)), 'null') for x in ('q', 'k_res', 'v_res', 'k_new', 'v_new', 'work', 'prefixes',
                                                                'out', 'workspace')),
                      (dict(k_scr=None), 'together'), (dict(v_scr=None), 'together'),
                      *((dict.fromkeys((x,), odd), 'aligned') for x in ('q', 'v_res', 'k_new', 'v_scr', 'prefixes', 'out',
                                                                        'workspace')),
                      (dict(slot_stride=-8), 'strides'), (dict(tok_stride=64), 'strides'), (dict(tok_stride=132), 'strides'),
                      (dict(head_stride=4), 'strides'), (dict(tok_stride=(1 << 28) + 8), 'token stride'),
                      (dict(q_rows=0), 'q_rows'), (dict(q_rows=2 ** 31), 'q_rows'), (dict(max_q=0), 'max_q'),
                      (dict(n_work=0), 'n_work'), (dict(n_groups=12), 'n_groups'), (dict(n_groups=0), 'n_groups'),
                      (dict(n_columns=-1), 'n_columns'), (dict(max_items=0), 'max_items'), (dict(max_tokens=0), 'max_tokens'),
                      (dict(members=0), 'members'), (dict(turn=0), 'turn'), (dict(turn=65537), 'turn'),
                      (dict(n_req=0), 'n_req'), (dict(scale=float('nan')), 'scale'), (dict(part_tiles=0), 'part_tiles'),
                      (dict(workspace_bytes=100), 'workspace too small')):
        rc, message = call(**kw)
        assert rc == -1 and match in message, (kw, message)
