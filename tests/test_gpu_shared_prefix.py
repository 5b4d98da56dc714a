"""Attention of transactions whose requests share committed rows, against the formula
in float64, with every row behind a context and every foreign slot NaN; eager, staged by
the launch, through families, captured and replayed, and in a full round with adapters and
logit controls."""
import numpy as np
import pytest
import torch

from helpers import SCALE, SEED, randn_bf16

pytestmark = pytest.mark.gpu
DEV = torch.device('cuda:0')


@pytest.fixture(autouse=True)
def groups_of_any_size(monkeypatch):
    from qwen3_dspark_amd import shared_prefix
    monkeypatch.setattr(shared_prefix, 'MIN_SAVED', 0)
    monkeypatch.setattr(shared_prefix, 'MIN_LONG_ROWS', 0)


def build(families, *, layers=1, capacity=6144, rows=512, seed=0, extra=0, shared=True, shuffle=True):
    """A store and its requests: families [(prefix rows, [own rows, ..])]; the first of a family
    is the one that the others copy."""
    from qwen3_dspark_amd.persistent_kv import Bucket, PersistentTargetKV
    gen = torch.Generator().manual_seed(SEED + seed)
    total = sum(len(own) for _, own in families)
    store = PersistentTargetKV(layers=layers, slots=total + extra, context_capacity=capacity, max_query_tokens=rows, heads=8,
                               dim=128, device=DEV, shared_prefixes=shared)
    store.keys.fill_(float('nan'))
    store.values.fill_(float('nan'))
    for i in range(extra):
        store.add_request(f'idle {i}')
    handles, want = [], []
    for f, (prefix, own) in enumerate(families):
        for i, n in enumerate(own):
            h = store.add_request(f'f{f} r{i}')
            if i == 0:
                if prefix:
                    kv = randn_bf16(gen, 2, layers, prefix, 8, 128).to(DEV)
                    store.load_prefix(h, kv[0], kv[1])
                first = h
            else:
                store.share_prefix(first, h, prefix)
            handles.append(h)
            want.append(n)
    grow(store, handles, want, gen, rows)
    if shuffle:
        order = np.random.default_rng(seed).permutation(total).tolist()
        handles = [handles[i] for i in order]
    return store, handles, gen


def grow(store, handles, counts, gen, rows):
    """Commit counts[i] new rows to each request, a transaction at a time."""
    from qwen3_dspark_amd.persistent_kv import Bucket
    left = dict(zip(handles, counts))
    while any(left.values()):
        part, room = [], rows
        for h in handles:
            n = min(left[h], room)
            if n:
                part.append((h, n))
                room -= n
                left[h] -= n
        bucket = Bucket(tuple(n for _, n in part), (store.context_capacity - rows,) * len(part), f'grow {len(store.registered())}')
        store.register_bucket(bucket)
        tx = store.begin([h for h, _ in part], bucket)
        kv = randn_bf16(gen, 2, store.layers, rows - room, 8, 128).to(DEV)
        for layer in range(store.layers):
            store.stage_layer(tx, layer, kv[0, layer], kv[1, layer])
        store.commit(tx, dict(part))


def expected(store, handles, queries, q, nk, nv, layer=0):
    """float64 attention and, per output, sum p |v| / sum p."""
    out, size, at = [], [], 0
    for h, n in zip(handles, queries):
        c = store.length(h)
        k = torch.cat((store.keys[layer, h.index, :c], nk[at:at + n])).double().repeat_interleave(2, 1).permute(1, 0, 2)
        v = torch.cat((store.values[layer, h.index, :c], nv[at:at + n])).double().repeat_interleave(2, 1).permute(1, 0, 2)
        s = q[at:at + n].double().permute(1, 0, 2) @ k.transpose(1, 2).contiguous() * SCALE
        s.masked_fill_(torch.ones(n, c + n, dtype=torch.bool, device=DEV).triu(c + 1), float('-inf'))
        p = torch.softmax(s, -1)
        out.append((p @ v.contiguous()).permute(1, 0, 2))
        size.append((p @ v.abs().contiguous()).permute(1, 0, 2))
        at += n
    return torch.cat(out), torch.cat(size)


def check(got, want):
    """Half a bf16 step of the output, and of every probability (which enters PV in
    bf16) against the values' magnitudes; FP32 sums add 1e-4 of those."""
    ref, size = want
    assert torch.isfinite(got).all()
    off = (got.double() - ref).abs() - 2 ** -8 * ref.abs() - (2 ** -8 + 1e-4) * size
    assert (off <= 0).all(), float(off.max())
    # rounding errors are independent: all but few outputs are within half of that
    near = (got.double() - ref).square().mean().sqrt() / ref.square().mean().sqrt()
    assert near <= 2 ** -8, float(near)


FAMILIES = [
    [(64, [0, 0])], [(63, [1, 5])], [(500, [0, 31])], [(2000, [300, 20, 1, 0, 129])], [(5000, [7] * 20)],
    [(640, [0] * 64)], [(1000, [40, 900, 3]), (3000, [0, 0])], [(4000, [100] * 9), (0, [800, 30]), (130, [0, 600, 64])],
    [(256, [3, 4]), (320, [3, 4]), (384, [0, 0]), (448, [1, 1])]]


@pytest.mark.parametrize('longest', [1, 8])
@pytest.mark.parametrize('families', FAMILIES)
def test_decoding(families, longest):
    from qwen3_dspark_amd.persistent_kv import Bucket
    store, handles, gen = build(families, seed=longest)
    rng = np.random.default_rng(SEED)
    queries = [int(x) for x in rng.integers(1, longest + 1, len(handles))]
    bucket = Bucket(tuple(queries), (5900,) * len(handles), 'round')
    store.register_bucket(bucket)
    q, nk, nv = (randn_bf16(gen, sum(queries), h, 128).to(DEV) for h in (16, 8, 8))
    want = expected(store, handles, queries, q, nk, nv)
    tx = store.begin(handles, bucket)
    store.scratch_keys.fill_(0)
    out = store.attend(tx, 0, q, keys=nk, values=nv)
    check(out, want)
    assert torch.equal(store.scratch_keys[0, :sum(queries)], nk) and torch.equal(store.scratch_values[0, :sum(queries)], nv)
    store.abort(tx)
    tx = store.begin(handles, bucket)
    store.stage_layer(tx, 0, nk, nv)
    buf = torch.full((sum(queries) + 3, 16, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    store.attend(tx, 0, q, out=buf[:sum(queries)])
    assert torch.equal(buf[:sum(queries)], out) and (buf[sum(queries):] == 7).all()


@pytest.mark.parametrize('families,queries', [
    ([(64, [0, 0])], [9, 33]), ([(1500, [0, 0, 0])], [100, 17, 64]), ([(3000, [0, 200, 1])], [8, 300, 9]),
    ([(700, [10] * 4), (2000, [0, 0])], [1, 40, 7, 12, 160, 5]), ([(5000, [0, 50])], [16, 16]), ([(0, [900, 40])], [70, 7])])
def test_prompts(families, queries):
    from qwen3_dspark_amd.persistent_kv import Bucket
    store, handles, gen = build(families, seed=3)
    bucket = Bucket(tuple(queries), (5600,) * len(handles), 'prompts')
    store.register_bucket(bucket)
    q, nk, nv = (randn_bf16(gen, sum(queries), h, 128).to(DEV) for h in (16, 8, 8))
    want = expected(store, handles, queries, q, nk, nv)
    tx = store.begin(handles, bucket)
    out = store.attend(tx, 0, q, keys=nk, values=nv)
    check(out, want)
    assert torch.equal(store.scratch_keys[0, :sum(queries)], nk) and torch.equal(store.scratch_values[0, :sum(queries)], nv)


def test_infinite_and_nan_rows_reach_the_requests_that_see_them():
    """A NaN key in one request's own rows stays with it, though its queries share a
    workgroup with the others'."""
    from qwen3_dspark_amd.persistent_kv import Bucket
    store, handles, gen = build([(1000, [30, 30, 30])], shuffle=False)
    bucket = Bucket((7, 7, 7), (2000,) * 3, 'round')
    store.register_bucket(bucket)
    q, nk, nv = (randn_bf16(gen, 21, h, 128).to(DEV) for h in (16, 8, 8))
    tx = store.begin(handles, bucket)
    want = store.attend(tx, 0, q, keys=nk, values=nv)
    store.abort(tx)
    store.keys[0, handles[1].index, 1010] = float('nan')
    q[14:] = float('nan')
    tx = store.begin(handles, bucket)
    got = store.attend(tx, 0, q, keys=nk, values=nv)
    assert torch.equal(got[:7], want[:7]) and torch.isnan(got[7:]).all()


def test_sharing_through_steps_and_departures():
    """a -> b -> d, and c from a; then a leaves and another request takes its slot."""
    from qwen3_dspark_amd.persistent_kv import Bucket, PersistentTargetKV
    gen = torch.Generator().manual_seed(SEED)
    store = PersistentTargetKV(layers=2, slots=5, context_capacity=2048, max_query_tokens=512, heads=8, dim=128, device=DEV,
                               shared_prefixes=True)
    a, b, c, d = (store.add_request(x) for x in 'abcd')
    kv = randn_bf16(gen, 2, 2, 700, 8, 128).to(DEV)
    store.load_prefix(a, kv[0], kv[1])
    store.share_prefix(a, b, 640)
    grow(store, [a, b], [100, 300], gen, 512)
    store.share_prefix(b, d, 900)
    store.share_prefix(a, c, 200)
    bucket = Bucket((5, 8, 1, 3), (1500,) * 4, 'round')
    store.register_bucket(bucket)
    q, nk, nv = (randn_bf16(gen, 2, 17, h, 128).to(DEV) for h in (16, 8, 8))

    def round_(handles):
        tx = store.begin(handles, bucket)
        for layer in range(2):
            want = expected(store, handles, (5, 8, 1, 3), q[layer], nk[layer], nv[layer], layer)
            check(store.attend(tx, layer, q[layer], keys=nk[layer], values=nv[layer]), want)
        store.commit(tx, dict(zip(handles, (2, 8, 0, 1))))
    round_([d, a, c, b])
    round_([a, b, c, d])
    store.remove_request(a)
    e = store.add_request('e')
    kv = randn_bf16(gen, 2, 2, 800, 8, 128).to(DEV)
    store.load_prefix(e, kv[0], kv[1])
    round_([e, b, c, d])


def test_small_groups_are_attended_request_by_request(monkeypatch):
    from qwen3_dspark_amd.persistent_kv import Bucket
    monkeypatch.undo()
    store, handles, gen = build([(1000, [3, 40])])
    bucket = Bucket((7, 2), (2000,) * 2, 'round')
    store.register_bucket(bucket)
    q, nk, nv = (randn_bf16(gen, 9, h, 128).to(DEV) for h in (16, 8, 8))
    want = expected(store, handles, (7, 2), q, nk, nv)
    tx = store.begin(handles, bucket)
    check(store.attend(tx, 0, q, keys=nk, values=nv), want)


def test_counters_and_workspace():
    from qwen3_dspark_amd.persistent_kv import Bucket
    store, handles, gen = build([(1000, [3, 40, 0]), (0, [70])])
    bucket = Bucket((7, 2, 1, 40), (2000,) * 4, 'round')
    store.register_bucket(bucket)
    assert store.workspace_bytes(bucket) == store.workspace(bucket).nbytes()
    work = store.work(store.begin(handles, bucket))
    assert work['logical_active_key_tokens'] == 3 * 1000 + 3 + 40 + 70 + 50
    assert work['fused_attention_key_rows_per_layer'] == work['logical_active_key_tokens'] - 2 * 960


def test_far_slots():
    """Elements past 2^31: 48 slots of 65,536 rows; the group is the last four."""
    from qwen3_dspark_amd.persistent_kv import Bucket
    store, handles, gen = build([(1024, [5, 0, 70, 1])], capacity=65536, extra=44)
    assert min(h.index for h in handles) * 8 * 65536 * 128 > 2 ** 31
    bucket = Bucket((7,) * 4, (2000,) * 4, 'far')
    store.register_bucket(bucket)
    q, nk, nv = (randn_bf16(gen, 28, h, 128).to(DEV) for h in (16, 8, 8))
    want = expected(store, handles, (7,) * 4, q, nk, nv)
    tx = store.begin(handles, bucket)
    check(store.attend(tx, 0, q, keys=nk, values=nv), want)


def test_families_of_one_arena():
    from qwen3_dspark_amd.persistent_kv import QueryFamily
    store, handles, gen = build([(2000, [10, 0, 300]), (0, [40])])
    families = (QueryFamily(4, 12, 8, 9000, 6000, 'decode'), QueryFamily(4, 300, 280, 9000, 6000, 'prompts'),
                QueryFamily(2, 6, 5, 9000, 6000, 'two'))
    store.register_families(families)
    for family, n, queries in ((families[0], 4, (1, 7, 3, 1)), (families[1], 4, (8, 270, 9, 13)), (families[2], 2, (1, 5)),
                               (families[0], 4, (3, 3, 3, 3))):
        q, nk, nv = (randn_bf16(gen, sum(queries), h, 128).to(DEV) for h in (16, 8, 8))
        want = expected(store, handles[:n], queries, q, nk, nv)
        tx = store.begin(handles[:n], family, query_lengths=queries)
        check(store.attend(tx, 0, q, keys=nk, values=nv), want)
        store.abort(tx)
    assert store.workspace_bytes(store._arena[0]) == store._arena[1].nbytes()


def test_captured_rounds_over_changing_groups():
    """One capture; rounds with groups of other members, lengths and splits, and with none,
    each equal to the eager launches bit for bit."""
    from qwen3_dspark_amd.graph import VerificationGraph
    from qwen3_dspark_amd.persistent_kv import Bucket
    store, handles, gen = build([(3000, [5, 60, 0]), (700, [0, 9, 300]), (0, [50, 0, 20])], layers=2, shuffle=False)
    bucket = Bucket((7, 7, 7, 7), (5000,) * 4, 'captured')
    store.register_bucket(bucket)
    graph = VerificationGraph(store, bucket).capture()
    for chosen in ((0, 1, 2, 8), (3, 0, 5, 1), (6, 7, 8, 0), (4, 3, 5, 2), (2, 1, 0, 4)):
        some = [handles[i] for i in chosen]
        q, nk, nv = (randn_bf16(gen, 2, 28, h, 128).to(DEV) for h in (16, 8, 8))
        tx = store.begin(some, bucket)
        eager = [store.attend(tx, l, q[l], keys=nk[l], values=nv[l]) for l in range(2)]
        store.abort(tx)
        torch.cuda.synchronize()
        tx = store.begin(some, bucket)
        for dst, src in ((graph.query, q), (graph.keys, nk), (graph.values, nv)):
            dst.copy_(src)
        out = graph.wait(graph.submit(tx))
        for l in range(2):
            assert torch.equal(out[l], eager[l])
            check(out[l], expected(store, some, (7,) * 4, q[l], nk[l], nv[l], l))
        store.commit(tx, {h: n for h, n in zip(some, (7, 0, 3, 1))})


def test_a_store_without_sharing_gives_what_it_gave():
    """share_prefix in a plain store copies; its attention is that of loaded rows, bit for bit."""
    from qwen3_dspark_amd.persistent_kv import Bucket
    outs = []
    for copies in (False, True):
        store, handles, gen = build([(900, [20, 20])], shared=False, shuffle=False)
        if not copies:
            from qwen3_dspark_amd.persistent_kv import PersistentTargetKV
            kv = [store.request_kv(h) for h in handles]
            other = PersistentTargetKV(layers=1, slots=2, context_capacity=6144, max_query_tokens=512, heads=8, dim=128,
                                       device=DEV)
            handles = [other.add_request(f'r{i}') for i in range(2)]
            for h, (k, v) in zip(handles, kv):
                other.load_prefix(h, k, v)
            store = other
        bucket = Bucket((7, 3), (2000,) * 2, 'round')
        store.register_bucket(bucket)
        q, nk, nv = (randn_bf16(torch.Generator().manual_seed(1), 10, h, 128).to(DEV) for h in (16, 8, 8))
        outs.append(store.attend(store.begin(handles, bucket), 0, q, keys=nk, values=nv))
    assert torch.equal(*outs)


def test_a_round_of_tenants():
    """Requests that share a prompt, with adapters and sampling rules of their own: the
    adapted projections staged, attention over the shared rows, the head, the rules and the
    verification, two rounds with a commit between them."""
    from qwen3_dspark_amd.adapters import AdapterBatch, QKVAdapters
    from qwen3_dspark_amd.persistent_kv import Bucket
    from qwen3_dspark_amd.prologue import QKVPrologue
    from qwen3_dspark_amd.sampling import LogitControls, TargetHead, verify_proposals
    store, handles, gen = build([(1200, [4, 0, 33]), (0, [75])], layers=2, shuffle=False)

    def rnd(*shape, scale=0.03):
        return (scale * torch.randn(*shape, generator=gen)).to(torch.bfloat16).to(DEV)
    vocab, n = 2003, 3
    prologues = [QKVPrologue(rnd(2048, 1024), rnd(1024, 1024), rnd(1024, 1024), 1 + rnd(128), 1 + rnd(128)) for _ in range(2)]
    adapters = [QKVAdapters(*(x for h in (2048, 1024, 1024) for x in (rnd(2, 8, 1024), rnd(2, h, 8, scale=0.3)))) for _ in range(2)]
    head = TargetHead(rnd(vocab, 1024))
    bucket = Bucket((n + 1,) * 4, (5000,) * 4, 'tenants')
    store.register_bucket(bucket)
    batch = AdapterBatch(DEV, [n + 1] * 4, [0, 0, 0, 1])
    controls = LogitControls(DEV, vocab, repetition=[1.2, 1.0, 1.5, 1.0], presence=[0.0, 0.3, 0.0, 0.0],
                             bias=[None, {5: 4.0}, None, {1: -9.0}])
    history = torch.zeros(4, 64, dtype=torch.long, device=DEV)
    lengths = [0] * 4
    for rnd_no in range(2):
        proposed = torch.randint(0, 50, (4 * n,), generator=gen).to(DEV)
        hidden = rnd(4 * (n + 1), 1024, scale=1.0)
        tx = store.begin(handles, bucket)
        for layer in range(2):
            q = store.stage_projected(tx, layer, hidden, prologues[layer], adapters=adapters[layer], batch=batch)
            o = store.attend(tx, layer, q)
            rows = slice(0, 4 * (n + 1))
            check(o, expected(store, handles, (n + 1,) * 4, q, store.scratch_keys[layer, rows], store.scratch_values[layer, rows], layer))
            hidden = (hidden + o.reshape(len(o), -1)[:, :1024]).contiguous()
        allowed = torch.full((16, 63), -1, dtype=torch.int32, device=DEV)
        allowed[:, 2:] = 0                              # the first 64 tokens
        logits = controls(head(hidden), history, lengths=lengths, counts=[n] * 4, tokens=proposed, allowed=allowed)
        law = torch.zeros(4 * n, vocab, dtype=torch.float64, device=DEV)
        law[:, :50] = 0.02
        u = torch.rand(16, dtype=torch.float64, generator=gen).to(DEV)
        done = verify_proposals(logits, proposed, law, u, counts=[n] * 4, temperature=1.0, max_new_tokens=[9] * 4)
        for r, x in enumerate(done):
            assert 1 <= len(x.tokens) <= n + 1 and int(x.tokens.max()) < 64
            history[r, lengths[r]:lengths[r] + len(x.tokens)] = x.tokens
            lengths[r] += len(x.tokens)
        before = [store.length(h) for h in handles]
        store.commit(tx, {h: len(x.tokens) for h, x in zip(handles, done)})
        assert [store.length(h) - b for h, b in zip(handles, before)] == [len(x.tokens) for x in done]


def test_the_persistent_target():
    """Requests of a PersistentQwenTarget that share a prompt: hidden states and logits of the rest of
    each prompt and of later rounds are those of requests that computed all of theirs."""
    from qwen3_dspark_amd.persistent_kv import Bucket
    from test_gpu_hf_hooks import close, tiny_qwen3
    from test_gpu_persistent_target import ids, make_target
    rng = np.random.default_rng(7)
    prompt, rests = rng.integers(0, 512, 130).tolist(), [rng.integers(0, 512, n).tolist() for n in (3, 20, 9)]
    rounds = [[rng.integers(0, 512, 7).tolist() for _ in range(3)] for _ in range(2)]
    names, logits = ['a', 'b', 'c'], []
    for shared in (False, True):
        target = make_target(tiny_qwen3()[1], slots=4, context_capacity=512, max_query_tokens=512, graph_backend=None,
                             max_graph_buckets=0, graph_byte_budget=0, shared_prefixes=shared)
        for n in names:
            target.add_request(n)
        lengths = tuple(len(r) + (0 if shared else 130) for r in rests)
        first = Bucket(lengths, (130,) * 3, 'rest')
        step = Bucket((7,) * 3, (230,) * 3, 'round')
        for b in (first, step):
            target.register_bucket(b)
        if shared:
            target.add_request('prompt')
            alone = Bucket((130,), (0,), 'prompt')
            target.register_bucket(alone)
            target.release_features(target.prefill({'prompt': ids(prompt)}, bucket=alone))
            for n in names:
                target.share_prefix('prompt', n, 130)
            target.remove_request('prompt')
            assert target.lengths == dict.fromkeys(names, 130)
        got = []
        f = target.verify({n: ids(r if shared else prompt + r) for n, r in zip(names, rests)}, bucket=first)
        got += [target.predict(f)[n][0, -len(r):].float() for n, r in zip(names, rests)]
        target.commit(f, {n: x for n, x in zip(names, lengths)})
        target.release_features(f)
        for new in rounds:
            f = target.verify({n: ids(x) for n, x in zip(names, new)}, bucket=step)
            got += [x[0].float() for x in target.predict(f).values()]
            target.commit(f, dict(zip(names, (7, 2, 5))))
            target.release_features(f)
        logits.append(got)
        target.close()
    for x, y in zip(*logits):
        close(y.cpu(), x.cpu(), 'logits')        # the gate of one such model against a float32 one


def test_refusals():
    store, handles, gen = build([(100, [0, 0])])
    from qwen3_dspark_amd.persistent_kv import Bucket
    fresh = Bucket((1, 1), (200, 200), 'round')
    store.register_bucket(fresh)
    store.begin(handles, fresh)
    with pytest.raises(RuntimeError, match='Outstanding'):
        store.share_prefix(handles[0], handles[1], 10)
