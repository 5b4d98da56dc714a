"""Refusals of the logit controls that need no GPU: rules that are none, and the
C entry's argument checks."""
import ctypes

import pytest

from qwen3_dspark_amd import _native
from qwen3_dspark_amd.sampling import LogitControls


@pytest.mark.parametrize('kw,match', [
    (dict(repetition=0.0), 'positive'), (dict(repetition=-1.0), 'positive'), (dict(repetition=float('nan')), 'finite'),
    (dict(presence=float('inf')), 'finite'), (dict(frequency=[0.1, 1e39]), 'finite'), (dict(presence=True), 'finite'),
    (dict(repetition=[1.0, 1.1], presence=[0.0]), 'same number'), (dict(repetition=[]), 'same number'),
    (dict(repetition=[1.0], requests=2), 'same number'), (dict(requests=0), 'same number'),
    (dict(bias=[{100: 1.0}]), 'vocabulary'), (dict(bias=[{-1: 1.0}]), 'vocabulary'), (dict(bias=[{1.5: 1.0}]), 'vocabulary'),
    (dict(bias=[{1: float('-inf')}]), 'finite'), (dict(bias=[{i: 1.0 for i in range(65536)}]), '65,535'), (dict(masked=float('nan')), 'masked'), (dict(masked='low'), 'masked'), (dict(masked=1e39), 'masked'), (dict(masked=-10 ** 400), 'masked')])
def test_rules_are_checked_before_the_device(kw, match):
    with pytest.raises(ValueError, match=match):
        LogitControls('cpu', 100, **kw)


def test_vocabulary_and_device():
    for vocab in (0, -1, 2 ** 30 + 1, 1.5, True):
        with pytest.raises(ValueError, match='vocab'):
            LogitControls('cpu', vocab)
    with pytest.raises(RuntimeError, match='gfx950'):
        LogitControls('cpu', 100, bias=[{3: 1.0}, None])


def test_entry_point_checks():
    lib = _native.load()
    fake = ctypes.c_void_p(1 << 20)                # never dereferenced

    def call(**kw):
        args = dict(logits=fake, dtype=0, row_stride=100, vocab=100, layout=fake, host_layout=0, n_req=1, rows=1, text_tokens=0, history=fake,
                    history_bytes=8, history_stride=4, tokens=fake, penalties=fake, bias_start=fake, bias_token=fake,
                    bias_value=fake, allowed=fake, allowed_stride=4, fill=0.0, out=ctypes.c_void_p(1 << 21), out_dtype=0,
                    out_stride=100, stream=None)
        args.update(kw)
        return lib.dspark_logit_controls(*args.values()), lib.dspark_last_error().decode()
    for kw, match in ((dict(logits=None), 'null'), (dict(history=None), 'null'), (dict(n_req=0), 'n_req'),
                      (dict(n_req=65536), 'n_req'), (dict(layout=None), 'null'), (dict(rows=0), 'rows'), (dict(text_tokens=-1), 'rows'),
                      (dict(host_layout=1, n_req=129), 'host memory'), (dict(vocab=0), 'vocab'), (dict(vocab=2 ** 30 + 1, row_stride=2 ** 31, out_stride=2 ** 31), 'vocab'), (dict(row_stride=99), 'vocab'),
                      (dict(out_stride=99), 'vocab'), (dict(dtype=2), 'dtype'), (dict(dtype=1), 'out_dtype'),
                      (dict(history_bytes=2), 'history'), (dict(history_stride=-1), 'mask row'),
                      (dict(allowed_stride=3), 'mask row'), (dict(out=fake, out_stride=104), 'in place'),
                      (dict(out=fake, out_dtype=1), 'in place')):
        rc, message = call(**kw)
        assert rc == -1 and match in message, (kw, message)
