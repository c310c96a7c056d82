"""The 8-bit cache, its attention and the verification of drafts as far as they go without a GPU: what the entry points refuse
before they launch anything (the pointers that these calls are given lead nowhere), and the sizes of their scratch."""
import copy
import ctypes
import math
import pickle

import pytest
import torch

from lrqk_amd import _lib, ops

P = 1 << 20   # a pointer, 16-byte aligned
EINVAL, ELIMIT = -1, -3

APPEND = dict(k_new=P, v_new=P, strides=(ctypes.c_int64 * 6)(*([64] * 6)), t=5, most=5, lengths=P, counts=None, path=None, path_b=0,
              new_lengths=P, k=P, v=P, ks=P, vs=P, kt=P, vt=P, blocks=4, b=1, h=2, d=64, kind=0, dtype=1, stream=None)
ATTENTION = dict(q=P, k=P, v=P, ks=P, vs=P, kt=P, vt=P, blocks=4, lengths=P, k_new=P, v_new=P, mask=P, mask_b=0, out=P, lse=None, b=1,
                 hq=4, hc=2, hn=2, t=3, d=64, scale=0.1, kind=1, ws=P, ws_bytes=1 << 40, dtype=1, stream=None)
VERIFY = dict(tokens=P, parents=P, target=P, tb=30, tr=10, draft=P, db=30, dr=10, uniforms=P, path=P, counts=P, next=P, b=1, s=3, vocab=10,
              ws=P, ws_bytes=1 << 40, dtype=0, stream=None)


def _call(fn, good, **changed):
    return getattr(_lib.load(), fn)(*dict(good, **changed).values())


@pytest.mark.parametrize("fn,good,code,changed", [
    *(("lrqk_byte_append", APPEND, EINVAL, c) for c in (
        *({x: None} for x in ("k_new", "v_new", "strides", "lengths", "new_lengths", "k", "v", "ks", "vs", "kt", "vt")),
        *({x: 0} for x in ("t", "most", "blocks", "b", "h", "d")), dict(kind=2), dict(dtype=2), dict(most=6), dict(k_new=P + 8), dict(kt=P + 4),
        dict(strides=(ctypes.c_int64 * 6)(64, 64, 68, 64, 64, 64)))),
    *(("lrqk_byte_append", APPEND, ELIMIT, c) for c in (dict(d=60), dict(d=264), dict(blocks=(1 << 24) + 1), dict(b=40000))),
    *(("lrqk_byte_attention", ATTENTION, EINVAL, c) for c in (
        *({x: None} for x in ("q", "k", "v", "ks", "vs", "kt", "vt", "lengths", "out", "ws", "k_new", "v_new", "mask")),
        *({x: 0} for x in ("blocks", "b", "hq", "hc", "hn", "t", "d", "ws_bytes")), dict(hq=5), dict(hn=3), dict(kind=-1), dict(dtype=9),
        dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(q=P + 2), dict(v=P + 8), dict(k_new=P + 4))),
    *(("lrqk_byte_attention", ATTENTION, ELIMIT, c) for c in (
        dict(d=60), dict(d=264), dict(t=1025), dict(blocks=(1 << 24) + 1), dict(b=20000), dict(b=200, blocks=1 << 24))),
    *(("lrqk_verify_drafts", VERIFY, EINVAL, c) for c in (
        *({x: None} for x in ("tokens", "target", "uniforms", "path", "counts", "next", "ws")), *({x: 0} for x in ("b", "s", "vocab", "ws_bytes")),
        dict(dtype=3), dict(ws=P + 8))),
    *(("lrqk_verify_drafts", VERIFY, ELIMIT, c) for c in (dict(s=1025), dict(b=65536), dict(vocab=(1 << 30) + 1)))],
    ids=lambda x: x if isinstance(x, str) else ",".join(f"{k}={v}" for k, v in x.items()) if isinstance(x, dict) and len(x) < 9 else "")
def test_entry_points_refuse(fn, good, code, changed):
    assert _call(fn, good, **changed) == code
    assert _lib.load().lrqk_last_error()


def test_scratch_sizes():
    lib = _lib.load()
    small, large = (lib.lrqk_byte_attention_workspace(1, 32, 8, t, 2048, 128, 1) for t in (1, 64))
    assert 0 < small <= large < 1 << 30
    # what is not in a complete block is a part of its own: of a token over one block, of 2 heads, 16 queries' outputs and sums each
    assert lib.lrqk_byte_attention_workspace(1, 2, 2, 1, 1, 64, 1) >= 2 * 2 * 16 * (64 + 3) * 4
    assert lib.lrqk_verify_drafts_workspace(2, 9, 128256) >= 2 * (2 * 9 + 63 + 2) * 8
    for fn, args in (("lrqk_byte_attention_workspace", (0, 32, 8, 1, 10, 128, 1)), ("lrqk_byte_attention_workspace", (1, 32, 7, 1, 10, 128, 1)),
                     ("lrqk_verify_drafts_workspace", (1, 0, 10))):
        assert getattr(lib, fn)(*args) == EINVAL
    assert lib.lrqk_verify_drafts_workspace(1, 2000, 10) == ELIMIT


def test_the_cache_refuses():
    for bad in (dict(kind="int4"), dict(dtype=torch.float16), dict(batch=0), dict(heads=0), dict(capacity=0), dict(head_dim=0), dict(head_dim=60),
                dict(head_dim=264), dict(head_dim=66, dtype=torch.float32), dict(capacity=2 ** 30 + 1)):
        with pytest.raises(ValueError):
            ops.ByteCache(**{**dict(batch=1, heads=1, capacity=64, head_dim=64, device="meta"), **bad})


@pytest.mark.parametrize("kind,codes", [("int8", torch.int8), ("fp8", torch.float8_e4m3fn)])
@pytest.mark.parametrize("d,w", [(8, 64), (64, 64), (72, 128), (128, 128), (136, 256), (256, 256)])
def test_the_caches_buffers(kind, codes, d, w):
    cache = ops.ByteCache(2, 3, 65, d, torch.float32, kind, "cpu")
    assert cache.capacity == 128 and cache.head_dim == d
    assert cache.k.shape == (2, 3, 2, 64, w) and cache.v.shape == (2, 3, 2, w, 64) and cache.k.dtype == cache.v.dtype == codes
    assert cache.k_scale.shape == cache.v_scale.shape == (2, 3, 2) and cache.k_scale.dtype == torch.float32
    assert cache.k_tail.shape == cache.v_tail.shape == (2, 3, 128, d) and cache.k_tail.dtype == torch.float32


def test_tensors_off_the_gpu_are_refused():
    cache = ops.ByteCache(1, 2, 64, 64, device="cpu")
    t, n, i = torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32), torch.zeros((1, 3), dtype=torch.int32)
    for call in (lambda: ops.byte_append(cache, t, t, n), lambda: ops.byte_attention(t, cache, n),
                 lambda: ops.verify_drafts(i, torch.zeros(1, 3, 9), torch.zeros(1, 3))):
        with pytest.raises(ValueError):
            call()


FAR = (1 << 32) + 3


@pytest.mark.parametrize("call", [
    lambda x, c: ops.byte_append(c, *[x(1, 1, FAR, 64).bfloat16()] * 2, x(1).int()),
    lambda x, c: ops.byte_append(c, *[x(1, 1, 5, 64).bfloat16()] * 2, x(1).int(), path=x(1, FAR).int()),
    lambda x, c: ops.byte_attention(x(1, 1, FAR, 64).bfloat16(), c, x(1).int()),
    lambda x, c: ops.byte_attention(x(1, FAR, 1, 64).bfloat16(), c, x(1).int()),
    lambda x, c: ops.verify_drafts(x(1, FAR).int(), x(1, FAR, 2), x(1, FAR)),
    lambda x, c: ops.verify_drafts(x(1, 2).int(), x(1, 2, FAR), x(1, 2)),
    lambda x, c: ops.verify_drafts(x(FAR, 1).int(), x(FAR, 1, 2), x(FAR, 1))])
def test_sizes_beyond_32_bits_do_not_reach_the_library_as_others(monkeypatch, call):
    """(Tensors without memory: the call is refused before anything looks at what they hold.)"""
    monkeypatch.setattr(ops, "_on_one_gpu", lambda *ts: 0)
    monkeypatch.setattr(ops.ByteCache, "_on", lambda self, dev: self._sizes)
    monkeypatch.setattr(ops, "_launch", lambda *args: pytest.fail("reached the library"))
    cache = ops.ByteCache(1, 1, 64, 64, device="cpu")
    with pytest.raises(ValueError, match="beyond 32 bits"):
        call(lambda *shape: torch.empty(shape, device="meta"), cache)


@pytest.mark.parametrize("ngram", [1, 2, 3])
def test_drafts_are_what_followed_the_last_time(ngram):
    from lrqk_amd.decoder import LookedUp
    g = torch.Generator().manual_seed(ngram)
    row = LookedUp(torch.randint(0, 4, (5,), generator=g).tolist(), ngram)
    for _ in range(60):
        t, want = row.tokens, [-1] * 4
        for at in range(len(t) - ngram):
            if t[at:at + ngram] == t[-ngram:]:
                want = (t[at + ngram:] + [-1] * 4)[:4]
        assert row.drafts(4) == want
        row.tokens += torch.randint(0, 4, (int(torch.randint(1, 4, (), generator=g)),), generator=g).tolist()
    assert LookedUp([1], 2).drafts(2) == [-1, -1]


def test_copies_of_a_cache_are_given_their_own_buffers():
    one = ops.ByteCache(1, 2, 100, 16, torch.float32, "int8", "cpu")
    for other in (copy.deepcopy(one), pickle.loads(pickle.dumps(one))):
        assert other._places == tuple(x.data_ptr() for x in other._buffers) and not set(other._places) & set(one._places)
        assert [lo for lo, _ in other._ranges] == list(other._places)
    assert copy.copy(one)._places == one._places
