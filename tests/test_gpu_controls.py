"""Logit controls (penalties, biases, masks) against the float64 oracle, at the
kernel's edges: 4,096-token chunks, 32-token mask words, 16-byte groups of rows
that start anywhere, 0 to 255 proposed tokens, rows that allow nothing."""
import numpy as np
import pytest
import torch

from helpers import SEED
from oracle import controls as oracle
from oracle import sampling as law

pytestmark = pytest.mark.gpu
DEV = torch.device('cuda:0')
LOWEST = {d: torch.finfo(d).min for d in (torch.bfloat16, torch.float32)}


def pack(allowed, words, junk=True):
    """bool [rows, V] -> int32 words, the bits behind the vocabulary set."""
    rows, v = allowed.shape
    bits = np.full((rows, 32 * words), junk)
    bits[:, :v] = allowed
    return torch.from_numpy(np.packbits(bits, axis=1, bitorder='little').view(np.int32).copy()).to(DEV)


class Batch:
    def __init__(self, vocab, counts, history, dtype, seed=0, hist_dtype=torch.long, mask=True, pad=0, masked=None,
                 out=None):
        rng = np.random.default_rng(SEED + seed)
        n, rows = len(counts), sum(counts) + len(counts)
        self.counts, self.vocab, self.dtype = counts, vocab, dtype
        gen = torch.Generator().manual_seed(SEED + seed)
        wide = (3 * torch.randn(rows, vocab + pad, generator=gen)).to(dtype)
        self.logits = wide.to(DEV)[:, pad // 2:pad // 2 + vocab]
        self.lengths = [int(x) for x in rng.integers(0, history + 1, n)]
        self.lengths[-1] = history
        self.prompts = [int(rng.integers(0, x + 1)) for x in self.lengths]
        text = rng.integers(-2, max(2, int(vocab * 1.2)), (n, history + 3))     # some are no tokens
        text[:, ::3] = rng.integers(0, min(vocab, 7), text[:, ::3].shape)       # some come often
        self.history = torch.from_numpy(text).to(hist_dtype).to(DEV)
        self.proposed = torch.from_numpy(rng.integers(0, min(vocab, 40), sum(counts))).to(DEV)
        self.rules = dict(repetition=[float(x) for x in rng.choice([1.0, 1.3, 0.7], n)],
                          presence=[float(x) for x in rng.choice([0.0, 0.6, -0.4], n)],
                          frequency=[float(x) for x in rng.choice([0.0, 0.25], n)],
                          bias=[None if r % 3 == 1 else {int(t): float(b) for t, b in
                                                         zip(rng.integers(0, vocab, 9), rng.normal(size=9))}
                                for r in range(n)])
        self.masked = masked
        self.allowed = rng.random((rows, vocab)) < 0.5 if mask else None
        if mask:
            self.allowed[rng.random(rows) < 0.3] &= rng.random(vocab) < 0.02
            self.allowed[:, rng.integers(0, vocab)] = True
        self.out_dtype = out or dtype

    def controls(self):
        from qwen3_dspark_amd.sampling import LogitControls
        return LogitControls(DEV, self.vocab, masked=self.masked, **self.rules)

    def call(self, controls=None, **kw):
        words = (self.vocab + 31) // 32
        return (controls or self.controls())(
            self.logits, self.history, lengths=self.lengths, prompt_lengths=self.prompts, counts=self.counts,
            tokens=self.proposed, allowed=None if self.allowed is None else pack(self.allowed, words), **kw)

    def expected(self, **kw):
        low = LOWEST[self.out_dtype]
        return oracle.control_rows(self.logits.double().cpu().numpy(), self.history.cpu().numpy(), self.lengths,
                                   self.prompts, self.counts, self.proposed.cpu().numpy(), allowed=self.allowed,
                                   fill=low if self.masked is None else self.masked, lowest=low, **self.rules, **kw)


def check(got, want, dtype):
    """One rounding to the output's type behind a rounding to fp32."""
    assert got.dtype == dtype
    g = got.double().cpu().numpy()
    same = (g == want) | (np.isnan(g) & np.isnan(want))
    step = torch.finfo(dtype).eps / 2 * 1.0001 + 2 ** -24
    with np.errstate(invalid='ignore'):
        near = np.abs(g - want) <= step * np.abs(want) + 1e-37
    bad = ~(same | near)
    assert not bad.any(), (np.argwhere(bad)[:5], g[bad][:5], want[bad][:5])


@pytest.mark.parametrize('dtype,out', [(torch.bfloat16, None), (torch.bfloat16, torch.float32), (torch.float32, None)])
@pytest.mark.parametrize('vocab', [1, 31, 33, 4095, 4096, 4097, 8200, 20011])
def test_sizes(vocab, dtype, out):
    b = Batch(vocab, [0, 3, 7], 300, dtype, seed=vocab, out=out)
    o = None if out is None else torch.empty(b.logits.shape, dtype=out, device=DEV)
    check(b.call(out=o), b.expected(), b.out_dtype)


@pytest.mark.parametrize('masked', [None, float('-inf'), -1e4])
@pytest.mark.parametrize('pad', [2, 5, 8, 16])
def test_strided_rows_and_fills(pad, masked):
    b = Batch(5003, [2, 0], 50, torch.bfloat16, seed=pad, pad=pad, masked=masked)
    if masked == -1e4:
        b.masked = float(torch.tensor(masked, dtype=torch.bfloat16))
    check(b.call(), b.expected(), torch.bfloat16)
    buf = torch.full((b.logits.shape[0], 5003 + 12), 7.0, dtype=torch.bfloat16, device=DEV)
    check(b.call(out=buf[:, 3:5006]), b.expected(), torch.bfloat16)
    assert (buf[:, :3] == 7).all() and (buf[:, 5006:] == 7).all()


@pytest.mark.parametrize('counts,history', [([0], 0), ([255, 0, 1], 5), ([0] * 70, 900), ([12], 20000)])
def test_proposals_and_texts(counts, history):
    b = Batch(9001, counts, history, torch.float32, seed=history, hist_dtype=torch.int32, mask=len(counts) < 4)
    check(b.call(), b.expected(), torch.float32)


@pytest.mark.parametrize('dtype,out', [(torch.bfloat16, None), (torch.bfloat16, torch.float32), (torch.float32, None)])
@pytest.mark.parametrize('mask', [False, True])
@pytest.mark.parametrize('vocab,pad', [(700, 3), (8192, 0), (17001, 5)])
def test_texts_that_are_long_for_their_rows(vocab, pad, mask, dtype, out):
    b = Batch(vocab, [0, 1], 12000, dtype, seed=pad, pad=pad, mask=mask, out=out,
              hist_dtype=torch.int32 if mask else torch.long)
    assert sum(b.lengths) > 2048 * 3
    if mask:
        b.allowed[1] = False
    o = None if out is None else torch.empty(b.logits.shape, dtype=out, device=DEV)
    check(b.call(out=o), b.expected(), b.out_dtype)


def test_far_rows():
    """Rows of logits, output, text and masks behind 2^31 elements."""
    b = Batch(700, [1, 0], 40, torch.bfloat16, seed=11)
    words, step = 22, 2 ** 30 + 8

    def far(x):
        out = torch.empty(2 * step + x.shape[1], dtype=x.dtype, device=DEV).as_strided(x.shape, (step, 1))
        return out.copy_(x)
    b.history = torch.cat((b.history, b.history[:1]))             # the third row is the second request's text
    kw = dict(lengths=b.lengths, prompt_lengths=b.prompts, counts=b.counts, tokens=b.proposed, slots=[0, 2])
    b.lengths[1] = kw['lengths'][1] = b.lengths[0]
    b.prompts[1] = kw['prompt_lengths'][1] = b.prompts[0]
    got = b.controls()(far(b.logits), far(b.history), allowed=far(pack(b.allowed, words)), out=far(b.logits), **kw)
    check(got, b.expected(slots=[0, 2]), torch.bfloat16)
    del got
    torch.cuda.empty_cache()


def test_many_requests():
    """More than a launch's arguments hold: the layout is uploaded."""
    b = Batch(300, [1] * 129 + [0, 3], 20, torch.float32, seed=9)
    check(b.call(), b.expected(), torch.float32)


def test_in_place_gives_the_same_bits():
    b = Batch(8200, [3, 0, 5], 400, torch.bfloat16)
    want = b.call()
    got = b.call(out=b.logits)
    assert got.data_ptr() == b.logits.data_ptr() and torch.equal(got, want)
    c = Batch(8200, [3], 400, torch.float32, mask=False, pad=3)
    want = c.call()
    assert torch.equal(c.call(out=c.logits), want)


def test_rows_that_allow_nothing_and_values_that_are_none():
    b = Batch(4500, [1, 1], 60, torch.bfloat16)
    b.allowed[0] = False
    b.allowed[2] = False
    b.allowed[2, 4499] = True                 # one token, in the last chunk
    b.logits[1, ::5] = float('nan')
    b.logits[2, ::7] = float('inf')
    b.logits[3, ::3] = LOWEST[torch.bfloat16]
    b.logits[3, 1::3] = -LOWEST[torch.bfloat16]
    b.logits[3, 2::3] = float('-inf')
    b.rules.update(repetition=[1.3, 4.0], presence=[0.5, 3e38], bias=[{0: 1.0}, {4499: 3e38, 3: -3e38}])
    got = b.call()
    check(got, b.expected(), torch.bfloat16)
    assert torch.isinf(got[0]).all() and (got[0] < 0).all()
    assert float(got[2, 4498]) == LOWEST[torch.bfloat16]
    x = Batch(4500, [1, 1], 60, torch.bfloat16, mask=False)
    x.logits[3] = b.logits[3]
    x.rules = b.rules
    check(x.call(), x.expected(), torch.bfloat16)


def test_shared_texts_and_single_rules():
    from qwen3_dspark_amd.sampling import LogitControls
    b = Batch(700, [0, 2, 0], 40, torch.float32, mask=False)
    c = LogitControls(DEV, 700, repetition=1.2, requests=3)
    b.rules = dict(repetition=[1.2] * 3, presence=[0.0] * 3, frequency=[0.0] * 3, bias=[None] * 3)
    b.lengths, b.prompts = [40, 7, 0], [0, 0, 0]
    got = c(b.logits, b.history, lengths=b.lengths, counts=b.counts, tokens=b.proposed, slots=[2, 2, 0])
    check(got, b.expected(slots=[2, 2, 0]), torch.float32)
    one = b.history[1:2].expand(3, -1)
    got = c(b.logits, one, lengths=b.lengths, counts=b.counts, tokens=b.proposed)
    check(got, b.expected(slots=[1, 1, 1]), torch.float32)


def test_two_streams_and_two_calls_at_once():
    b, d = Batch(20011, [4] * 9, 500, torch.bfloat16, seed=1), Batch(20011, [2] * 5, 90, torch.bfloat16, seed=2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    cb, cd = b.controls(), d.controls()
    with torch.cuda.stream(side):
        first = b.call(cb)
    second = d.call(cd)
    torch.cuda.synchronize()
    check(first, b.expected(), torch.bfloat16)
    check(second, d.expected(), torch.bfloat16)


def test_rules_prepared_on_a_busy_stream():
    b = Batch(20011, [4] * 9, 500, torch.bfloat16, seed=6)
    work = torch.randn(4096, 4096, device=DEV)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(8):
            work = work @ work * 1e-2
        controls = b.controls()
    got = b.call(controls)
    del controls
    torch.cuda.synchronize()
    check(got, b.expected(), torch.bfloat16)


@pytest.mark.parametrize('masked', [-1.0039e4, 2.99e-3, 3.4e38])
@pytest.mark.parametrize('dtype,out', [(torch.bfloat16, None), (torch.bfloat16, torch.float32), (torch.float32, None)])
def test_fills_are_rounded_to_the_output(masked, dtype, out):
    """To nearest, like every value, and alike in whole groups and in the odd ends of rows."""
    b = Batch(5003, [2, 0], 50, dtype, seed=8, pad=5, masked=masked, out=out)
    got = b.call(out=None if out is None else torch.empty(b.logits.shape, dtype=out, device=DEV))
    fill = torch.tensor(masked, dtype=torch.float32).to(b.out_dtype).to(DEV)
    assert (got[torch.from_numpy(~b.allowed).to(DEV)] == fill).all()


def test_the_law_behind_controls():
    """Masked tokens have no probability, a row that allows nothing is refused, and a
    verification of ruled logits is the oracle's."""
    from qwen3_dspark_amd.sampling import logits_to_probabilities, verify_proposals
    b = Batch(3001, [3, 0, 6], 200, torch.float32, seed=5)
    for r in range(len(b.logits)):
        b.allowed[r, :40] = True              # what may be proposed
    got = b.call()
    probs = logits_to_probabilities(got, 0.9).cpu().numpy()
    assert (probs[~b.allowed] == 0).all()
    np.testing.assert_allclose(probs, law.logits_to_probabilities(got.double().cpu().numpy(), 0.9), rtol=1e-12,
                               atol=1e-300)
    q = torch.full((9, 3001), 0.0, dtype=torch.float64, device=DEV)
    q[:, :40] = 1 / 40
    u = torch.rand(12, dtype=torch.float64, device=DEV, generator=torch.Generator(device=DEV).manual_seed(3))
    res = verify_proposals(got, b.proposed, q, u, counts=b.counts, temperature=0.9, max_new_tokens=[10] * 3)
    assert [len(r.tokens) >= 1 for r in res] == [True] * 3
    at = 0
    for r, n in zip(res, b.counts):
        for j, t in enumerate(r.tokens.tolist()):
            assert b.allowed[at + j, t]
        at += n + 1
    b.allowed[1] = False
    with pytest.raises(ValueError, match='finite floating logits'):
        logits_to_probabilities(b.call(), 0.9)


def test_refusals(monkeypatch):
    from qwen3_dspark_amd import sampling
    from qwen3_dspark_amd.sampling import LogitControls
    b = Batch(700, [1, 2], 40, torch.bfloat16, mask=False)
    c = b.controls()
    good = dict(lengths=b.lengths, prompt_lengths=b.prompts, counts=b.counts, tokens=b.proposed)
    for change, match in (
            (dict(lengths=[1]), 'rule 2 requests'), (dict(lengths=[1.0, 2]), 'integers'),
            (dict(counts=[1, 2 ** 40]), 'integers'), (dict(slots=5), 'integers'), (dict(lengths=[41, 44]), 'within history'),
            (dict(prompt_lengths=[41, 0]), 'within history'), (dict(prompt_lengths=[0]), 'per request'),
            (dict(counts=[1, 1]), 'a row for each'), (dict(counts=[-1, 4]), 'a row for each'),
            (dict(slots=[0, 2]), 'within history'), (dict(tokens=b.proposed.int()), 'int64'),
            (dict(tokens=b.proposed[:2]), 'int64'), (dict(tokens=None), 'int64'),
            (dict(allowed=torch.zeros(5, 21, dtype=torch.int32, device=DEV)), 'ceil'),
            (dict(allowed=torch.zeros(5, 22, dtype=torch.int64, device=DEV)), 'ceil'),
            (dict(out=torch.empty(5, 700, dtype=torch.float16, device=DEV)), 'type or fp32'),
            (dict(out=torch.empty(5, 701, dtype=torch.bfloat16, device=DEV)), 'type or fp32')):
        with pytest.raises(ValueError, match=match):
            c(b.logits, b.history, **{**good, **change})
    for logits, history, match in ((b.logits[:, :699], b.history, '700'), (b.logits.half(), b.history, 'bf16 or fp32'),
                                   (b.logits, b.history[0], 'contiguous rows'),
                                   (b.logits, b.history.float(), 'contiguous rows'),
                                   (b.logits, b.history.T, 'contiguous rows')):
        with pytest.raises(ValueError, match=match):
            c(logits, history, **good)
    wide = torch.zeros(6, 700, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match='not overlap'):
        c(wide[:5], b.history, **good, out=wide[1:])
    many = LogitControls(DEV, 700)
    with pytest.raises(ValueError, match='255'):
        many(torch.zeros(257, 700, device=DEV), b.history, lengths=[1], counts=[256],
             tokens=torch.zeros(256, dtype=torch.long, device=DEV))
    monkeypatch.setattr(sampling, '_MAX_TEXT', 39)
    with pytest.raises(ValueError, match='per text'):
        b.call(c)
    monkeypatch.undo()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(ValueError, match='captured graph'):
        with torch.cuda.graph(graph):
            b.call(c)
