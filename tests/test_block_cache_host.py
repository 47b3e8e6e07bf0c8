"""CPU checks of the block cache, the rotary and the logits entry points:
what the library refuses before any launch, and BlockKVCache's bookkeeping
over recorded calls."""
import ctypes
from types import SimpleNamespace

import pytest
import torch

from specfit_amd import _native, ops
from specfit_amd.runtime import BlockKVCache, Eagle3DraftTree, LogitRules
from specfit_amd.runtime import block_kv_cache

FAKE = 4096  # never dereferenced: every call below fails, or has no work, before a launch


def _struct(**kwargs):
    fields = dict(k8=FAKE, v8=FAKE, k_scale=FAKE, v_scale=FAKE, flags=FAKE, k_tail=FAKE,
                  v_tail=FAKE, tail_flags=FAKE, heads=4, head_dim=128, held=0, capacity_blocks=10,
                  ring_blocks=3, folded_blocks=2)
    return _native.KVCacheStruct(**{**fields, **kwargs})


def _append(c, start, tokens, kv_heads=4, k=FAKE):
    return _native.lib().sf_kv_append(ctypes.addressof(c), kv_heads, k, 8, 8, 8, FAKE, 8, 8, 8,
                                      start, tokens, None)


def test_cache_calls_refused_on_the_host():
    lib = _native.lib()
    for bad, code in ((dict(head_dim=96), 2), (dict(heads=0), 1), (dict(heads=70000), 2),
                      (dict(held=2), 1), (dict(capacity_blocks=0), 1), (dict(ring_blocks=0), 1),
                      (dict(folded_blocks=11), 1), (dict(folded_blocks=-1), 1), (dict(k8=None), 1),
                      (dict(tail_flags=None), 1), (dict(v_tail=FAKE + 8), 3)):
        c = _struct(**bad)
        assert _append(c, 128, 1) == code, bad
        assert lib.sf_kv_fold(ctypes.addressof(c), 1, None) == code
        assert lib.sf_kv_read(ctypes.addressof(c), 0, 1, FAKE, FAKE, None) == code
        assert lib.sf_kv_compact(ctypes.addressof(c), 128, 0, FAKE, 1, 200, None) == code
    assert lib.sf_kv_fold(None, 1, None) == 1
    c = _struct()
    assert _append(c, 128, 0) == 0                # nothing to do
    assert _append(c, 127, 1) == 1                # a folded block
    assert _append(c, 128, 3 * 64 + 1) == 1       # more than the ring
    assert _append(c, 600, 41) == 1               # past the capacity
    assert _append(c, 1 << 62, 5) == 1
    assert _append(c, 128, 1, kv_heads=3) == 1
    assert _append(c, 128, 1, k=None) == 1
    assert _append(c, 128, -1) == 1
    assert lib.sf_kv_fold(ctypes.addressof(c), 4, None) == 1      # more than the ring
    assert lib.sf_kv_fold(ctypes.addressof(_struct(folded_blocks=9)), 2, None) == 1
    assert lib.sf_kv_fold(ctypes.addressof(c), 0, None) == 0
    assert lib.sf_kv_read(ctypes.addressof(c), 0, 5 * 64 + 1, FAKE, FAKE, None) == 1
    assert lib.sf_kv_read(ctypes.addressof(c), 0, 5, FAKE + 2, FAKE, None) == 3
    assert lib.sf_kv_read(ctypes.addressof(c), -1, 5, FAKE, FAKE, None) == 1
    assert lib.sf_kv_read(ctypes.addressof(c), 0, 0, None, None, None) == 0

    def compact(positions, first=0, base=128, end=300):
        n = len(positions)
        return lib.sf_kv_compact(ctypes.addressof(c), base, first, (ctypes.c_int32 * n)(*positions),
                                 n, end, None)
    assert compact([]) == 0
    assert compact([3, 3]) == 1 and compact([4, 3]) == 1
    assert compact([0], first=1) == 1             # moves up
    assert compact([172]) == 1                    # behind the last row
    assert compact([1], base=100) == 1            # a folded block
    assert compact([1], end=400) == 1             # more than the ring
    assert compact(list(range(1, 258))) == 1      # more than one call takes


def test_attention_calls_refused_on_the_host():
    lib = _native.lib()
    c = _struct()

    def attend(batch=1, kv_heads=4, keys=200, q=FAKE, strides=(8, 8, 8), queries=1, q_heads=32,
               mask=None, mask_keys=0, out=FAKE, work=None, nbytes=0, cache=c):
        return lib.sf_block_attention(ctypes.addressof(cache), batch, kv_heads, keys, q, *strides,
                                      queries, q_heads, mask, 0, 0, mask_keys, 1.0, out, work, nbytes,
                                      None)
    assert attend(batch=2) == 1 and attend(batch=0) == 1 and attend(kv_heads=2) == 1
    assert attend(keys=0) == 1 and attend(queries=0) == 1
    assert attend(keys=5 * 64 + 1) == 1           # more than the ring
    assert attend(keys=641) == 1                  # more than the capacity
    assert attend(q_heads=30) == 2 and attend(q_heads=0) == 2
    assert attend(q=None) == 1 and attend(out=None) == 1
    assert attend(q=FAKE + 8) == 3 and attend(strides=(8, 4, 8)) == 3 and attend(out=FAKE + 8) == 3
    assert attend(mask=FAKE, mask_keys=201) == 1 and attend(mask=FAKE, mask_keys=-1) == 1
    assert attend(queries=1 << 22) == 2           # more rows than fit the indexes
    big = _struct(capacity_blocks=1 << 25, ring_blocks=1 << 25, folded_blocks=0)
    assert attend(keys=(1 << 30) + 1, cache=big) == 2
    work = lib.sf_block_attention_workspace
    assert work(1, 1, 64, 32, 4, 128) == 0 and work(1, 1, 0, 32, 4, 128) == 0
    assert work(1, 1, 4096, 30, 4, 128) == 0 and work(1, 1, 4096, 32, 4, 96) == 0
    assert work(0, 1, 4096, 32, 4, 128) == 0 and work(1, 4096, 4096, 32, 4, 128) == 0
    assert work(1, 1, (1 << 30) + 1, 32, 4, 128) == 0
    for batch, queries, keys, q_heads, kv_heads, dim in (
            (1, 1, 4097, 32, 4, 128), (1, 128, 32905, 64, 4, 128), (3, 1, 1 << 30, 8, 8, 64),
            (2, 5, 9000, 14, 2, 64)):
        each = batch * queries * q_heads * (dim + 2) * 4
        splits, rest = divmod(work(batch, queries, keys, q_heads, kv_heads, dim), each)
        assert rest == 0 and 2 <= splits <= 128


def test_rotary_and_logit_calls_refused_on_the_host():
    lib = _native.lib()

    def rotary(dtype=0, q=FAKE, q_heads=2, k_heads=1, positions=FAKE, batch=1, tokens=3, dim=64,
               rot=64):
        return lib.sf_rotary(dtype, q, 8, 8, 8, q_heads, FAKE, 8, 8, 8, k_heads, positions, 0, FAKE,
                             1.0, batch, tokens, dim, rot, 0, FAKE, FAKE, None)
    assert rotary(dtype=3) == 1 and rotary(tokens=-1) == 1 and rotary(q=None) == 1
    assert rotary(positions=None) == 1
    assert rotary(rot=63) == 2 and rotary(rot=66) == 2 and rotary(rot=0) == 2
    assert rotary(dim=1026, rot=64) == 2
    assert rotary(tokens=0) == 0 and rotary(q_heads=0, k_heads=0) == 0
    assert rotary(batch=1 << 16, tokens=1 << 15) == 2

    def rules(dtype=2, logits=FAKE, rows=2, vocab=100, rep=1.0, out=FAKE, tokens=None, work=None,
              nbytes=0, path=0):
        return lib.sf_logit_rules(dtype, logits, 100, rows, vocab, None, None, path, rep, 0.0, 0.0,
                                  None, 0, None, 0, out, 100, tokens, work, nbytes, None)
    assert rules(dtype=5) == 1 and rules(rows=-1) == 1 and rules(vocab=0) == 1
    assert rules(rep=0.0) == 1 and rules(rep=float("nan")) == 1 and rules(path=-1) == 1
    assert rules(logits=None) == 1 and rules(vocab=(1 << 30) + 1) == 2
    assert rules(tokens=FAKE) == 1 and rules(tokens=FAKE, work=FAKE, nbytes=8) == 1
    assert rules(tokens=FAKE, work=FAKE + 4, nbytes=1 << 20) == 3
    assert rules(rows=0) == 0 and rules(out=None) == 0
    assert lib.sf_logit_rules_workspace(0, 100) == 0
    assert lib.sf_logit_rules_workspace(3, 151936) == 3 * 75 * 4 * 8


class _Calls(list):
    """Stands in for the device side of a cache."""

    def install(self, monkeypatch):
        def blocks(**kwargs):
            return SimpleNamespace(folded=0, **{k: v for k, v in kwargs.items()})

        def fold(b, count):
            self.append(("fold", count))
            b.folded += count
        fake = SimpleNamespace(
            KV_BLOCK=64, KVBlocks=blocks, kv_fold=fold,
            kv_append=lambda b, l, k, v, start: self.append(("append", l, start, k.shape[2])),
            kv_compact=lambda b, base, p, end: self.append(("compact", base, tuple(p), end)),
            kv_read=lambda b, l, start, stop: (start, stop),
            block_attention=lambda b, l, q, keys, m, s: (keys, s))
        monkeypatch.setattr(block_kv_cache, "ops", fake)
        return self


def _rows(n):
    return torch.empty((1, 2, n, 64))


def test_lengths_and_folds(monkeypatch):
    calls = _Calls().install(monkeypatch)
    cache = BlockKVCache(2, 2, 64, 300, tail_tokens=100)
    assert cache.blocks.capacity_blocks == 5 and cache.blocks.ring_blocks == 3
    assert cache.get_seq_length() == 0 and cache.get_mask_sizes(7, 0) == (7, 0)
    cache.append(0, _rows(150), _rows(150))
    cache.commit()                                 # the other layer has nothing yet
    with pytest.raises(RuntimeError, match="differ"):
        cache.compact(0, ())
    assert cache.update(_rows(150), _rows(150), 1) == (0, 150)
    assert cache.get_seq_length(1) == 150 and cache.get_query_offset(0) == 150
    cache.commit()
    assert cache.folded_tokens == 128
    assert cache.attend(0, None) == (150, 0.125)
    for l in (0, 1):
        cache.append(l, _rows(61), _rows(61))
    cache.compact(150, (0, 2, 40))
    assert [cache.get_seq_length(l) for l in (0, 1)] == [153, 153]
    cache.commit()                                 # 153 tokens complete no further block
    assert calls == [("append", 0, 0, 150), ("append", 1, 0, 150), ("fold", 2),
                     ("append", 0, 150, 61), ("append", 1, 150, 61),
                     ("compact", 150, (0, 2, 40), 211)]
    short = BlockKVCache(1, 2, 64, 300, tail_tokens=60)
    short.append(0, _rows(100), _rows(100))
    with pytest.raises(ValueError, match="tail"):
        short.append(0, _rows(40), _rows(40))
    short.commit()
    short.append(0, _rows(40), _rows(40))
    del calls[-3:]
    with pytest.raises(ValueError, match="holds"):
        cache.append(0, _rows(148), _rows(148))
    cache.crop(-20)
    assert cache.get_seq_length() == 133
    with pytest.raises(ValueError, match="folded"):
        cache.crop(127)
    cache.crop(1000)
    assert cache.get_seq_length() == 133
    with pytest.raises(ValueError):
        cache.read(0, 10, 134)
    cache.compact(0, tuple(range(130)))            # keeps what is folded where it is
    assert cache.get_seq_length() == 130
    with pytest.raises(ValueError, match="dropped"):
        cache.compact(0, tuple(range(120)))
    with pytest.raises(ValueError, match="moved"):
        cache.compact(100, tuple(range(1, 30)))
    cache.reset()
    assert cache.get_seq_length() == 0 and cache.folded_tokens == 0


def test_storage_needs_a_device():
    with pytest.raises(ValueError, match="HIP device"):
        ops.KVBlocks(layers=1, batch=1, kv_heads=1, head_dim=64, capacity_blocks=1, ring_blocks=1,
                     held="int8", device="cpu")
    for bad in (dict(capacity=0), dict(tail_tokens=0)):
        with pytest.raises(ValueError, match="positive"):
            BlockKVCache(**{**dict(layers=1, kv_heads=1, head_dim=64, capacity=64), **bad})


def test_path_indices_of_a_tree():
    import math
    p = 0.5
    tree = Eagle3DraftTree((5, 6, 7, 8), (0, 0, 1, 3), (1, 1, 2, 3), (p,) * 4,
                           tuple(math.log(p) * d for d in (1, 1, 2, 3)))
    assert tree.path_indices().tolist() == [[0, -1, -1, -1], [0, 1, -1, -1], [0, 2, -1, -1],
                                            [0, 1, 3, -1], [0, 1, 3, 4]]


def test_starts_past_the_capacity_are_refused():
    lib, c = _native.lib(), _struct()
    far = 2 ** 63 - 1
    for start in (641, far - 5, far):
        assert _append(c, start, 10) != 0
        assert lib.sf_kv_read(ctypes.addressof(c), start, 10, FAKE, FAKE, None) != 0
        assert lib.sf_kv_compact(ctypes.addressof(c), start, 0, (ctypes.c_int32 * 1)(3), 1, far,
                                 None) != 0


def test_tokens_outside_the_vocabulary_are_not_counted():
    rules = LogitRules.for_vocab(5, "cpu")
    rules.count(torch.tensor([[0, 4, -1], [5, 4, -7]]))
    rules.count(torch.empty(0, dtype=torch.int64))
    assert rules.counts.tolist() == [1, 0, 0, 0, 2]


def test_rotary_positions_of_too_many_tokens_are_refused():
    lib = _native.lib()
    for batch, tokens in ((1, 2 ** 27), (2 ** 14, 2 ** 14), (2 ** 31 - 1, 2 ** 31 - 1)):
        assert lib.sf_rotary(0, FAKE, 8, 8, 8, 1, FAKE, 8, 8, 8, 1, FAKE, 0, FAKE, 1.0, batch,
                             tokens, 2, 2, 0, FAKE, FAKE, None) == 2
