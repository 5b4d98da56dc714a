"""Refusals of the low-rank adapters that need no GPU."""
import ctypes

import pytest
import torch

from qwen3_dspark_amd import _native
from qwen3_dspark_amd.adapters import AdapterBatch, QKVAdapters


@pytest.mark.parametrize('lengths,ids', [([], []), ([1], []), ([0], [0]), ([2, -1], [0, 0]), ([1], [-2]), ([1.5], [0]),
                                         ([1], [None]), ([True], [0]), ([1], [2 ** 31])])
def test_batches_are_checked_before_the_device(lengths, ids):
    with pytest.raises(ValueError, match='One positive length'):
        AdapterBatch('cpu', lengths, ids)


def test_no_cpu_path():
    with pytest.raises(RuntimeError, match='gfx950'):
        AdapterBatch('cpu', [3, 4], [0, -1])
    a = torch.zeros(2, 8, 128, dtype=torch.bfloat16)
    q, kv = (torch.zeros(2, n, 8, dtype=torch.bfloat16) for n in (2048, 1024))
    with pytest.raises(RuntimeError, match='gfx950'):
        QKVAdapters(a, q, a, kv, a, kv)
    with pytest.raises(ValueError, match='rank'):
        QKVAdapters(a, kv, a, kv, a, kv)
    with pytest.raises(ValueError, match='hidden'):
        QKVAdapters(*(x[:, :, :100] if x is a else x for x in (a, q, a, kv, a, kv)))


def test_entry_point_checks():
    lib = _native.load()
    fake = ctypes.c_void_p(1 << 20)                # never dereferenced

    def project(**kw):
        args = dict(x=fake, wq=fake, wk=fake, wv=fake, qn=fake, kn=fake, inv=fake, pos=fake, rope=None, tokens=4,
                    hidden=1024, eps=1e-6, a=fake, b=fake, scaling=fake, adapters=2, rank=16, own_rank=8, token=fake,
                    tiles=fake, n_tiles=1, tile_tokens=16, u=fake, q=fake, k=fake, v=fake, stride=1024, stream=None)
        args.update(kw)
        return lib.dspark_qkv_prologue_adapted(*args.values()), lib.dspark_last_error().decode()
    off = ctypes.c_void_p(1 << 20 | 8)
    for kw, match in ((dict(x=None), 'null'), (dict(token=None), 'null'), (dict(u=None), 'null'), (dict(tiles=None), 'null'),
                      (dict(scaling=None), 'null'), (dict(adapters=0), 'adapters'), (dict(rank=24), 'rank'),
                      (dict(rank=48), 'rank'), (dict(rank=320), 'rank'), (dict(own_rank=17), 'own_rank'),
                      (dict(own_rank=0), 'own_rank'), (dict(n_tiles=0), 'n_tiles'), (dict(tile_tokens=24), 'tile_tokens'), (dict(tokens=0), 'tokens'),
                      (dict(hidden=64), 'hidden'), (dict(hidden=1000), 'hidden'), (dict(stride=1000), 'kv_row_stride'),
                      (dict(b=off), 'aligned'), (dict(u=off), 'aligned'), (dict(a=off), 'aligned'), (dict(x=off), 'aligned')):
        rc, message = project(**kw)
        assert rc == -1 and match in message, (kw, message)
