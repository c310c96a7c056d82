"""A cache held in 8 bits, the attention that reads it, and the verification of drafted tokens, against plain implementations in
64 bits.

Codes, scales, paths and tokens have to be equal.  The attention's tolerances count roundings: an output's own (half a step:
2^-8 of a bf16 value, 2^-24 of an fp32 one), those of probabilities and queries in fp16 (2^-11, or 2^-22 as two numbers), and
those of the arithmetic, in units of U = 2^-23 (an fp32 addition on the matrix cores need not round to nearest)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -23
BF, FP = torch.bfloat16, torch.float32
HALF = {BF: 2.0 ** -8, FP: 2.0 ** -24}
NAN, INF = float("nan"), float("inf")
KINDS = ["int8", "fp8"]


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from lrqk_amd import ops as o
    return o


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(g, *shape, dtype=FP, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _within(got, exact, tol, what=""):
    """got against exact (fp64) elementwise; where exact is not finite the same value is wanted."""
    got = got.double()
    fine = torch.isfinite(exact)
    assert torch.equal(torch.isnan(got), torch.isnan(exact)), what
    assert torch.equal(got[~fine & ~torch.isnan(exact)], exact[~fine & ~torch.isnan(exact)]), what
    off = ((got - exact).abs() / tol.clamp(min=1e-300))[fine]
    off = torch.where((got - exact).abs()[fine] == 0, torch.zeros_like(off), off)
    assert off.numel() == 0 or float(off.max()) <= 1.0, (what, float(off.max()))


# ------------------------------------------------------------------------------------------------------- append

NAMES = ("k", "v", "k_scale", "v_scale", "k_tail", "v_tail")


def _held(cache):
    return {n: getattr(cache, n).clone() for n in NAMES}


def _power(e):
    """2^e, exactly (a library's pow need not be)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _code64(rows, kind):
    """(codes fp64, scales fp32) of blocks [..., 64, d]."""
    x = rows.double()
    top = torch.where(torch.isfinite(x), x.abs(), 0.0).amax((-1, -2))
    x = torch.nan_to_num(x, 0.0)
    x = torch.where(torch.isnan(rows.double()), 0.0, x)
    if kind == "int8":
        s = torch.clamp((top / 127.0).float(), min=2.0 ** -100)   # (torch divides fp32 by a number with its reciprocal)
        c = torch.round(x / s.double()[..., None, None]).clamp(-127, 127)
        return torch.where(torch.isinf(rows), 127 * rows.sign().double(), c), s
    e = torch.frexp(top / 448.0)   # (1 / 448 is no power of two, but a quotient that is one comes out as it)
    s = _power(torch.where(top == 0, -100, torch.where(e.mantissa == 0.5, e.exponent - 1, e.exponent)).clamp(min=-100)).float()
    y = (x / s.double()[..., None, None]).clamp(-448, 448)
    step = _power(torch.frexp(y.abs().clamp(min=2.0 ** -6)).exponent - 4)
    return torch.where(torch.isinf(rows), 448 * rows.sign().double(), torch.round(y / step) * step), s


def _append64(held, kind, k, v, lengths, counts=None, path=None):
    """What an append makes of the buffers, and the new lengths."""
    held = {n: x.clone() for n, x in held.items()}
    b, h, t, d = k.shape
    blocks = held["k"].shape[2]
    new = lengths.clone()
    for i in range(b):
        n = min(max(int(lengths[i]), 0), 64 * blocks)
        take = list(range(t)) if path is None else [min(max(x, 0), t - 1) for x in path[i].tolist()]
        m = len(take) if counts is None else min(max(int(counts[i]), 0), len(take))
        m = min(m, 64 * blocks - n)
        new[i] = n + m
        for x, name in ((k, "k"), (v, "v")):
            tail = held[name + "_tail"][i]
            begin = n // 64 * 64
            rows = torch.cat((tail[:, [p % 128 for p in range(begin, n)]], x[i][:, take[:m]]), 1)
            whole = (n + m) // 64 - begin // 64
            if whole > 0:
                c, s = _code64(rows[:, :64 * whole].reshape(h, whole, 64, d), kind)
                at = slice(begin // 64, begin // 64 + whole)
                held[name + "_scale"][i, :, at] = s
                if name == "k":
                    held["k"][i, :, at, :, :d] = c.to(held["k"].dtype)
                else:
                    held["v"][i, :, at, :d] = c.transpose(-1, -2).to(held["v"].dtype)
            for p in range(max(n, n + m - 128), n + m):
                tail[:, p % 128] = x[i][:, take[p - n]]
    return held, new


def _same(cache, want, what=""):
    for n in NAMES:
        got = getattr(cache, n)
        a, z = (x.float() if x.element_size() == 1 else x for x in (got, want[n]))
        off = torch.nonzero((a != z) & ~(torch.isnan(a) & torch.isnan(z)))
        if len(off):
            pytest.fail(f"{what}: {n}: {len(off)} of {a.numel()} differ, {a[tuple(off[0])]} for {z[tuple(off[0])]} at {off[0].tolist()}")


def _check_append(ops, cache, k, v, lengths, counts=None, path=None, what=""):
    want, new = _append64(_held(cache), cache.kind, k, v, lengths, counts, path)
    was = lengths.clone()
    got = ops.byte_append(cache, k, v, lengths, counts, path)
    assert torch.equal(got, new) and torch.equal(lengths, was), what
    _same(cache, want, what)
    return got


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("t", [1, 2, 63, 64, 65, 127, 128, 129, 200, 333])
def test_append_prompts(ops, dtype, kind, t):
    print("append", dtype, kind, t, flush=True)
    g = _gen(t)
    for b, h, d in ((1, 2, 128), (3, 1, 64)):
        cache = ops.ByteCache(b, h, 400, d, dtype, kind, DEV)
        k, v = (_randn(g, b, t, h, d, dtype=dtype, scale=3.0).transpose(1, 2) for _ in range(2))
        _check_append(ops, cache, k, v, torch.zeros(b, dtype=torch.int32, device=DEV), what=(b, h, d))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [4, 8, 16, 24, 40, 64, 72, 80, 96, 128, 136, 200, 256])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_append_head_widths(ops, dtype, d, kind):
    print("append width", dtype, d, kind, flush=True)
    if dtype == BF and d % 8:
        with pytest.raises(ValueError):
            ops.ByteCache(1, 1, 64, d, dtype, kind, DEV)
        return
    g = _gen(d)
    cache = ops.ByteCache(2, 3, 192, d, dtype, kind, DEV)
    lengths = torch.zeros(2, dtype=torch.int32, device=DEV)
    for t in (70, 60, 5):
        k, v = (_randn(g, 2, 3, t, d, dtype=dtype) for _ in range(2))
        lengths = _check_append(ops, cache, k, v, lengths, what=t)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF, FP])
def test_append_paths_and_ragged_lengths(ops, dtype, kind):
    """Paths of different lengths behind sequences of different lengths, ids and counts beyond the ends, a full cache; again from
    the same lengths the same again."""
    print("append paths", dtype, kind, flush=True)
    g = _gen(5)
    b, h, d = 5, 2, 64
    cache = ops.ByteCache(b, h, 320, d, dtype, kind, DEV)
    k, v = (_randn(g, b, h, 310, d, dtype=dtype) for _ in range(2))
    lengths = _check_append(ops, cache, k, v, torch.zeros(b, dtype=torch.int32, device=DEV), _i32(0, 63, 64, 127, 310))
    for step in range(8):
        k, v = (_randn(g, b, h, 9, d, dtype=dtype) for _ in range(2))
        path = torch.randint(-2, 12, (b, 11), generator=g, dtype=torch.int32).to(DEV)
        counts = torch.randint(-1, 14, (b,), generator=g, dtype=torch.int32).to(DEV)
        new = _check_append(ops, cache, k, v, lengths, counts, path[:, 1:], what=step)
        held = _held(cache)
        assert torch.equal(ops.byte_append(cache, k, v, lengths, counts, path[:, 1:]), new)
        _same(cache, held, step)
        lengths = new
    assert int(lengths[4]) == 320
    held = _held(cache)
    # lengths that are none are cut to the cache
    _check_append(ops, cache, k, v, _i32(-5, 10 ** 9, 320, 0, 319))
    # nothing to write
    held, lengths = _held(cache), _i32(1, 2, 3, 4, 5)
    assert torch.equal(ops.byte_append(cache, k[:, :, :0], v[:, :, :0], lengths), lengths)
    assert torch.equal(ops.byte_append(cache, k, v, lengths, path=path[:, :0]), lengths)
    assert torch.equal(ops.byte_append(cache, k, v, lengths, torch.zeros_like(lengths)), lengths)
    _same(cache, held)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF, FP])
def test_token_by_token_is_as_at_once(ops, dtype, kind):
    """A block's codes depend on its rows alone: a prompt at once, in pieces, and token by token leave the same."""
    print("append pieces", dtype, kind, flush=True)
    g = _gen(6)
    k, v = (_randn(g, 1, 2, 300, 128, dtype=dtype) for _ in range(2))
    one = ops.ByteCache(1, 2, 320, 128, dtype, kind, DEV)
    ops.byte_append(one, k, v, _i32(0))
    for piece in (1, 7, 64, 100, 130):
        cache = ops.ByteCache(1, 2, 320, 128, dtype, kind, DEV)
        lengths = _i32(0)
        for i in range(0, 300, piece):
            lengths = ops.byte_append(cache, k[:, :, i:i + piece], v[:, :, i:i + piece], lengths)
        assert int(lengths) == 300
        _same(cache, _held(one), piece)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF, FP])
def test_sequences_made_shorter(ops, dtype, kind):
    """To whole blocks, to where the tail has the block that they end in, and again from the same lengths: what is appended then and
    what is read is that of the shorter ones."""
    print("byte shorter", dtype, kind, flush=True)
    g = _gen(21)
    b, d = 4, 64
    for n in (300, 320, 383):
        cache = ops.ByteCache(b, 2, 500, d, dtype, kind, DEV)
        k, v = (_randn(g, b, 2, n, d, dtype=dtype) for _ in range(2))
        ops.byte_append(cache, k, v, torch.zeros(b, dtype=torch.int32, device=DEV))
        lengths = _i32(n // 64 * 64 - 64, 64, (n - 128 + 63) // 64 * 64 + 5, 0)
        for t in (1, 64, 40):
            q, kn, vn, mask = _drafts(g, b, 4, 2, t, d, dtype)
            _check_attention(ops, q, cache, lengths, kn, vn, mask, what=(n, t))
            for _ in range(2):
                _check_append(ops, cache, kn, vn, lengths, what=(n, t))
        lengths = ops.byte_append(cache, kn, vn, lengths)
        _check_attention(ops, q, cache, lengths, what=n)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF, FP])
def test_append_odd_values(ops, dtype, kind):
    """Elements next to and on the border between two codes, of all sizes, blocks of zeros, infinities and NaN."""
    print("append values", dtype, kind, flush=True)
    g = _gen(7)
    top = 127.0 if kind == "int8" else 448.0
    x = _randn(g, 1, 1, 64 * 14, 128)
    blocks = x.view(14, 64, 128)
    blocks[0] = torch.randint(-254, 255, (64, 128), generator=g).to(DEV) / 2 * (top / 127)   # halves of a step of 1
    blocks[1] = torch.randint(-254, 255, (64, 128), generator=g).to(DEV) * (0.3 / 254)       # near halves of another
    blocks[2] = torch.exp(_randn(g, 64, 128) * 6) * _randn(g, 64, 128).sign()
    blocks[3] = 0.0
    blocks[4] = _randn(g, 64, 128) * 1e-36
    blocks[5] = _randn(g, 64, 128) * 3e37
    blocks[5, 0, 0] = 3.3e38
    blocks[6] = 0.0
    blocks[6, 3, 5] = 1e-40
    blocks[7] = torch.nextafter(blocks[0], torch.full_like(blocks[0], INF))
    blocks[8] = torch.nextafter(blocks[0], torch.full_like(blocks[0], -INF))
    blocks[9, 5, 7], blocks[9, 6, 8], blocks[9, 7, 9] = INF, -INF, NAN
    blocks[10] = NAN
    blocks[11] = INF
    blocks[12, :, ::2] = -INF
    blocks[13, 0, 0], blocks[13, 0, 1] = 3.38e38, INF
    k = x.to(dtype)
    v = k.flip(2).contiguous()
    cache = ops.ByteCache(1, 1, 64 * 15, 128, dtype, kind, DEV)
    _check_append(ops, cache, k, v, _i32(0))
    # and from the tail
    cache = ops.ByteCache(1, 1, 64 * 15, 128, dtype, kind, DEV)
    lengths = _i32(0)
    for i in range(0, 64 * 14, 48):
        lengths = _check_append(ops, cache, k[:, :, i:i + 48], v[:, :, i:i + 48], lengths, what=i)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_append_rounds_every_element_once(ops, dtype):
    """Millions of elements against quotients in 64 bits."""
    print("append many", dtype, flush=True)
    g = torch.Generator(device=DEV).manual_seed(8)
    for kind in KINDS:
        k, v = (torch.randn((1, 4, 8192, 128), generator=g, device=DEV).to(dtype) for _ in range(2))
        cache = ops.ByteCache(1, 4, 8192, 128, dtype, kind, DEV)
        _check_append(ops, cache, k, v, _i32(0))


def test_append_places_and_strides(ops):
    """A fused projection, rows between two 16-byte pieces, expanded heads, lengths and paths out of larger tensors."""
    print("append places", flush=True)
    g = _gen(9)
    for dtype in (BF, FP):
        qkv = _randn(g, 2, 70, 8, 64, dtype=dtype)
        cache = ops.ByteCache(2, 2, 128, 64, dtype, "int8", DEV)
        k, v = qkv[:, :, 4:6].transpose(1, 2), qkv[:, :, 6:].transpose(1, 2)
        _check_append(ops, cache, k, v, _i32(3, 0))
        flat = _randn(g, 2 * 2 * 70 * 64 + 1, dtype=dtype)[1:].view(2, 2, 70, 64)
        _check_append(ops, cache, flat, v, _i32(50, 1))
        _check_append(ops, cache, k[:, :1].expand(2, 2, 70, 64), v, _i32(0, 1))
        _check_append(ops, cache, k[:, :, ::3], v[:, :, ::3], _i32(0, 1))


def test_a_copy_of_a_cache_is_written_for_itself(ops):
    import copy
    g = _gen(3)
    cache, lengths = _cache(ops, g, 2, 2, 70, 64, BF, "int8")
    before = _held(cache)
    twin = copy.deepcopy(cache)
    k, v = (_randn(g, 2, 2, 60, 64, dtype=BF) for _ in range(2))
    _check_append(ops, twin, k, v, lengths)
    _same(cache, before)


def test_append_refuses_rows_of_the_cache(ops):
    cache = ops.ByteCache(2, 2, 128, 64, BF, "int8", DEV)
    n, k = _i32(0, 0), torch.zeros((2, 2, 3, 64), dtype=BF, device=DEV)
    for x in (cache.k_tail[:, :, 3:6], cache.v_tail[:, :, ::50], cache.k.view(BF).view(-1)[:2 * 2 * 3 * 64].view(2, 2, 3, 64)):
        for bad in ((x, k), (k, x)):
            with pytest.raises(ValueError, match="overlaps"):
                ops.byte_append(cache, *bad, n)


def test_append_refusals(ops):
    cache = ops.ByteCache(2, 2, 128, 64, BF, "int8", DEV)
    k = torch.zeros((2, 2, 3, 64), dtype=BF, device=DEV)
    n = _i32(0, 0)
    for bad in (lambda: ops.byte_append(cache, k.float(), k.float(), n), lambda: ops.byte_append(cache, k[:1], k[:1], n),
                lambda: ops.byte_append(cache, k, k[:, :, :2], n), lambda: ops.byte_append(cache, k[..., :32], k[..., :32], n),
                lambda: ops.byte_append(cache, k, k, n.long()), lambda: ops.byte_append(cache, k, k, n[:1]), lambda: ops.byte_append(cache, k, k, n.cpu()),
                lambda: ops.byte_append(cache, k.cpu(), k, n), lambda: ops.byte_append(cache, k, k, n, counts=n.float()),
                lambda: ops.byte_append(cache, k, k, n, path=n), lambda: ops.byte_append(cache, k, k, n, path=n[:, None].long()),
                lambda: ops.byte_append(cache, k.transpose(2, 3).contiguous().transpose(2, 3), k, n),
                lambda: ops.ByteCache(1, 1, 64, 64, torch.float16), lambda: ops.ByteCache(1, 1, 64, 64, BF, "int4"),
                lambda: ops.ByteCache(1, 1, 0, 64), lambda: ops.ByteCache(1, 1, 64, 264), lambda: ops.ByteCache(0, 1, 64, 64),
                lambda: ops.ByteCache(1, 1, 2 ** 30 + 1, 64, device="meta")):
        with pytest.raises(ValueError):
            bad()
    for name in NAMES:
        with pytest.raises(AttributeError):
            setattr(cache, name, getattr(cache, name).clone())


# --------------------------------------------------------------------------------------------------------- attention

def _rows64(cache, i, h, n):
    """(keys, values) fp64 [n,d] of a head."""
    d, whole = cache.head_dim, n // 64
    late = [p % 128 for p in range(64 * whole, n)]
    k = cache.k[i, h, :whole, :, :d].float().double() * cache.k_scale[i, h, :whole, None, None].double()
    v = cache.v[i, h, :whole, :d].float().double().transpose(1, 2) * cache.v_scale[i, h, :whole, None, None].double()
    return (torch.cat((x.reshape(-1, d), tail[i, h][late].double())) for x, tail in ((k, cache.k_tail), (v, cache.v_tail)))


def _attention64(q, cache, lengths, kn, vn, mask, scale, only=None):
    """(out, lse, tolerance of out, of lse) in fp64 (of the sequences `only`, if that is given).  Where a masked token holds
    something that is not finite, it is not met."""
    b, hq, t, d = q.shape
    hc = cache.k.shape[1]
    out = torch.zeros((b, hq, t, d), dtype=torch.float64, device=DEV)
    lse = torch.full((b, hq, t), -INF, dtype=torch.float64, device=DEV)
    tol, tol_l = torch.zeros_like(out), torch.zeros_like(lse)
    for i in range(b) if only is None else only:
        m = min(max(int(lengths[i]), 0), cache.capacity)
        sees = torch.ones((t, m), dtype=torch.bool, device=DEV)
        if mask is not None:
            sees = torch.cat((sees, mask.bool().expand(b, t, t)[i]), 1)
        for h in range(hq):
            k, v = _rows64(cache, i, h * hc // hq, m)
            if mask is not None:
                hn = kn.shape[1]
                k, v = torch.cat((k, kn[i, h * hn // hq].double())), torch.cat((v, vn[i, h * hn // hq].double()))
            x = q[i, h].double()
            s = torch.where(sees, x @ k.T * scale, -INF)
            # products of d elements summed in fp32, fp32 queries off by 2^-22 as two fp16 numbers, scales and their factors
            # rounded, the exponent rounded, the exponential 2 units
            ds = U * ((d + 12) * scale * torch.where(sees, x.abs() @ k.abs().nan_to_num(0, 0, 0).T, 0).amax(-1, keepdim=True) + 4)[:, 0] if k.shape[0] else torch.zeros(t, dtype=torch.float64, device=DEV)
            top = s.amax(-1, keepdim=True) if s.shape[1] else torch.full((t, 1), -INF, dtype=torch.float64, device=DEV)
            top = torch.where(top == -INF, 0.0, top)
            p = torch.exp(s - top)
            l = p.sum(-1, keepdim=True)
            some = l[:, 0] != 0
            w = torch.where(l > 0, p / l, torch.where(l == 0, 0.0, NAN))
            odd = ~torch.isfinite(v)
            clean = torch.where(odd, 0.0, v)
            o = w @ clean
            for j in torch.nonzero(odd.any(-1))[:, 0].tolist():   # (0 times infinity is not met where it is not seen)
                o = o + torch.where(sees[:, j:j + 1] & odd[j], v[j], 0.0)
            out[i, h] = o
            lse[i, h] = torch.where(some, (top + torch.log(l))[:, 0], -INF)
            # the exponents, the sums of numerator and denominator, a probability's bits: half a step of 2^-10 in fp16, the
            # square of that as two fp16 numbers (2^-22 covers it and the 2^-24 below), 2^-16 of the dense rows'; and what
            # fp16 loses of the smallest, 2^-25 of probabilities formed 2^8 too large
            each = 2 * ds + U * (m + t + 64) * 2 + (2.0 ** -21 if q.dtype == FP else 2.0 ** -11)
            tol[i, h] = each[:, None] * (w.nan_to_num(0) @ clean.abs()) + HALF[q.dtype] * o.nan_to_num(0, 0, 0).abs()
            if clean.shape[0]:
                tol[i, h] += 2.0 ** -33 * clean.abs().sum(0)
            tol_l[i, h] = ds + U * (m + t + 64) + 4 * U * lse[i, h].nan_to_num(0, 0, 0).abs()
    return out, lse, tol, tol_l


def _check_attention(ops, q, cache, lengths, kn=None, vn=None, mask=None, scale=None, what=""):
    out, lse = ops.byte_attention(q, cache, lengths, kn, vn, mask, scale, return_lse=True)
    e, el, tol, tol_l = _attention64(q, cache, lengths, kn, vn, mask, q.shape[-1] ** -0.5 if scale is None else scale)
    _within(out, e, tol, what)
    _within(lse, el, tol_l, what)
    return out, lse


def _cache(ops, g, b, h, n, d, dtype, kind, spread=0.5):
    """A cache with n tokens a sequence, some elements of which are larger than others; the lengths."""
    cache = ops.ByteCache(b, h, n + 8, d, dtype, kind, DEV)
    by = torch.exp(spread * _randn(g, h, 1, d))
    k, v = ((_randn(g, b, h, n, d) * by).to(dtype) for _ in range(2))
    return cache, ops.byte_append(cache, k, v, torch.zeros(b, dtype=torch.int32, device=DEV))


def _drafts(g, b, hq, hn, t, d, dtype, density=0.5):
    q = _randn(g, b, hq, t, d, dtype=dtype, scale=2.0)
    kn, vn = (_randn(g, b, hn, t, d, dtype=dtype) for _ in range(2))
    return q, kn, vn, (torch.rand((b, t, t), generator=g) < density).to(DEV)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("t,hq,hc,hn", [(1, 1, 1, 1), (1, 32, 8, 8), (3, 8, 8, 2), (7, 28, 4, 4), (16, 8, 2, 1), (33, 6, 2, 2), (64, 8, 2, 2),
                                        (100, 7, 1, 1)])
def test_attention_rows(ops, dtype, kind, t, hq, hc, hn):
    """One query to hundreds a head; lengths that end in every part of a block."""
    print("byte attention", dtype, kind, t, hq, hc, hn, flush=True)
    for n in (1, 63, 64, 65, 130, 700):
        g = _gen(n + t)
        cache, _ = _cache(ops, g, 2, hc, n, 128, dtype, kind)
        q, kn, vn, mask = _drafts(g, 2, hq, hn, t, 128, dtype)
        lengths = _i32(n, n if n > 128 else n // 2)
        _check_attention(ops, q, cache, lengths, kn, vn, mask, what=n)
        _check_attention(ops, q, cache, lengths, what=(n, "cached alone"))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [4, 8, 16, 24, 40, 64, 72, 80, 96, 128, 136, 200, 256])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_attention_head_widths(ops, dtype, d, kind):
    print("byte width", dtype, d, kind, flush=True)
    if dtype == BF and d % 8:
        return
    for t, hq in ((1, 2), (5, 8), (20, 4)):
        g = _gen(d + t)
        cache, lengths = _cache(ops, g, 2, 2, 333, d, dtype, kind)
        q, kn, vn, mask = _drafts(g, 2, hq, 2, t, d, dtype)
        _check_attention(ops, q, cache, lengths, kn, vn, mask[0], what=t)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF, FP])
def test_attention_long_caches_and_splits(ops, dtype, kind):
    print("byte long", dtype, kind, flush=True)
    for b, hq, hc, t, n in ((1, 8, 2, 1, 20000), (3, 4, 4, 5, 5000), (1, 4, 1, 40, 12345)):
        g = _gen(n)
        cache, _ = _cache(ops, g, b, hc, n, 64, dtype, kind)
        q, kn, vn, mask = _drafts(g, b, hq, hc, t, 64, dtype)
        lengths = _i32(*([n] + [n // 3] * (b - 1)))
        _check_attention(ops, q, cache, lengths, kn, vn, mask, what=(b, n))


@pytest.mark.parametrize("dtype", [BF, FP])
def test_attention_of_the_most_drafts(ops, dtype):
    """1024 drafted tokens, over nothing and over a few blocks; one more is refused."""
    print("byte most drafts", dtype, flush=True)
    g = _gen(1024)
    cache, lengths = _cache(ops, g, 2, 1, 200, 64, dtype, "int8")
    q, kn, vn, mask = _drafts(g, 2, 2, 1, 1025, 64, dtype, 0.02)
    first = [x[:, :, :1024] for x in (q, kn, vn)] + [mask[:, :1024, :1024]]
    _check_attention(ops, first[0], cache, _i32(0, 200), *first[1:])
    with pytest.raises(Exception, match="1024"):
        ops.byte_attention(q, cache, lengths, kn, vn, mask)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_attention_masks(ops, dtype):
    """Queries that see no drafted token, caches without tokens, both: zeros and -inf."""
    print("byte masks", dtype, flush=True)
    for t, hq in ((1, 2), (6, 4), (40, 4)):
        g = _gen(t)
        cache, _ = _cache(ops, g, 4, 2, 200, 64, dtype, "int8")
        q, kn, vn, mask = _drafts(g, 4, hq, 2, t, 64, dtype)
        mask[0], mask[1], mask[2] = False, torch.eye(t, dtype=torch.bool, device=DEV), True
        for lengths in (_i32(0, 0, 0, 0), _i32(200, 0, 128, -3), _i32(0, 1, 64, 10 ** 9)):
            _check_attention(ops, q, cache, lengths, kn, vn, mask, what=(t, lengths.tolist()))
            _check_attention(ops, q, cache, lengths, what=(t, lengths.tolist()))


@pytest.mark.parametrize("dtype", [BF, FP])
def test_attention_does_not_meet_what_is_masked(ops, dtype):
    """Masked drafted tokens, rows of the tail behind the length and blocks behind it that hold infinities and NaN."""
    print("byte odd values", dtype, flush=True)
    for t, hq in ((2, 2), (9, 4), (40, 2)):
        g = _gen(t)
        cache, _ = _cache(ops, g, 2, 2, 130, 64, dtype, "int8")
        q, kn, vn, mask = _drafts(g, 2, hq, 2, t, 64, dtype)
        lengths = _i32(130, 70)
        cache.k_tail[:, :, 10:64], cache.v_tail[:, :, 10:64] = NAN, INF          # (tokens 138 .. and older than a block)
        cache.k_tail[1, :, 70:], cache.v_tail[1, :, 70:] = INF, NAN
        cache.k_scale[1, :, 1:], cache.v_scale[0, :, 2:] = NAN, INF
        mask[:, :, 1] = False
        mask[0, 0, 1] = True
        kn[:, :, 1], vn[1, :, 1] = NAN, INF
        kn[0, :, 1] = 0.25
        vn[0, :, 1, ::3], vn[0, :, 1, 1::3] = INF, NAN
        _check_attention(ops, q, cache, lengths, kn, vn, mask, what=t)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("t,hq", [(3, 2), (40, 1), (70, 2)])
def test_scores_that_rise_and_fall(ops, dtype, kind, t, hq):
    """Along the cache scores rise in steps and fall again, and scales of blocks differ by orders of magnitude."""
    print("byte rising", dtype, kind, t, hq, flush=True)
    g = _gen(t)
    n = 64 * 40 + 17
    at = torch.arange(n, device=DEV, dtype=torch.float32)
    k = _randn(g, 1, 1, n, 64) * 0.05 + (torch.where(at < n / 2, at, n - at) / n * 8)[:, None] * 0.5
    v = _randn(g, 1, 1, n, 64) * torch.exp(6 * torch.sin(at / 300))[:, None]
    cache = ops.ByteCache(1, 1, n, 64, dtype, kind, DEV)
    lengths = ops.byte_append(cache, k.to(dtype), v.to(dtype), _i32(0))
    q, kn, vn, mask = _drafts(g, 1, hq, 1, t, 64, dtype)
    _check_attention(ops, q.abs(), cache, lengths, kn, vn, mask)
    _check_attention(ops, -q.abs(), cache, lengths, kn, vn, mask)
    _check_attention(ops, q * 1e-30, cache, lengths, kn, vn, mask, what="tiny")
    _check_attention(ops, q * 0, cache, lengths, kn, vn, mask, what="zero")
    wide = q.clone()
    wide[..., 0] *= 1e4   # elements of one query far apart
    wide[..., 1] *= 1e-4
    _check_attention(ops, wide, cache, lengths, kn, vn, mask, scale=1e-4, what="wide")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype,b,hq,hc,t,n,d", [
    (BF, 1, 32, 16, 10, 9000, 128), (BF, 2, 16, 8, 32, 9000, 64), (BF, 1, 16, 16, 64, 9000, 128),   # 32 queries a wave, each its blocks
    (BF, 1, 8, 2, 17, 1000, 128), (BF, 1, 8, 2, 24, 1000, 64),                                      # shared blocks
    (BF, 1, 4, 2, 16, 1000, 256), (BF, 1, 4, 2, 17, 1000, 256), (BF, 1, 4, 1, 33, 1000, 136),       # wide heads, alone and sharing
    (FP, 1, 4, 1, 8, 3000, 128), (FP, 1, 4, 1, 10, 33000, 128), (FP, 1, 4, 1, 17, 1000, 64), (FP, 1, 4, 1, 9, 1000, 256)])
def test_attention_of_every_kernel(ops, dtype, kind, b, hq, hc, t, n, d):
    """Each way that a call may take, over blocks whose values differ by orders of magnitude."""
    print("byte kernels", dtype, kind, b, hq, hc, t, n, d, flush=True)
    g = _gen(t + n)
    cache = ops.ByteCache(b, hc, n, d, dtype, kind, DEV)
    size = torch.exp2(torch.randint(-14, 15, ((n + 63) // 64,), generator=g).float()).to(DEV).repeat_interleave(64)[:n, None]
    for spread in (torch.ones_like(size), size):
        k, v = _randn(g, b, hc, n, d, dtype=dtype), (_randn(g, b, hc, n, d) * spread).to(dtype)
        lengths = ops.byte_append(cache, k, v, torch.zeros(b, dtype=torch.int32, device=DEV))
        q, kn, vn, mask = _drafts(g, b, hq, hc, t, d, dtype)
        _check_attention(ops, q, cache, lengths, kn, vn, mask)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("b,t,hq,d", [(16, 1, 2, 128), (17, 6, 8, 64), (70, 3, 2, 64), (16, 20, 4, 128), (16, 5, 2, 256)])
def test_attention_of_many_sequences(ops, dtype, kind, b, t, hq, d):
    """Sequences of none to many blocks, one split each and several, with drafted tokens that nobody sees and that hold infinities."""
    print("byte many sequences", dtype, kind, b, t, hq, d, flush=True)
    g = _gen(b + t)
    n = 64 * 30 + 8
    cache, full = _cache(ops, g, b, 2, n, d, dtype, kind)
    q, kn, vn, mask = _drafts(g, b, hq, 2, t, d, dtype)
    mask[1::3] = False
    some = torch.tensor([0, 1, 63, 64, 65, 127, 64 * 8, 64 * 8 + 1, 64 * 30, n], dtype=torch.int32, device=DEV)
    mixed = some[torch.randint(0, 10, (b,), generator=g).to(DEV)]
    # (a tail has a sequence's last 128 tokens: those of shorter lengths are other ones, finite all the same)
    for lengths in (full, mixed, mixed.flip(0), some[torch.arange(b, device=DEV) % 3], torch.zeros_like(full)):
        _check_attention(ops, q, cache, lengths, kn, vn, mask, what=lengths.tolist())
        _check_attention(ops, q, cache, lengths, what=lengths.tolist())
    vn[:, :, 0, ::3], vn[:, :, 0, 1::3] = INF, NAN
    _check_attention(ops, q, cache, mixed, kn, vn, mask, what="odd")


@pytest.mark.parametrize("b,t", [(700, 1), (400, 33), (400, 70)])
def test_attention_of_heads_that_fill_the_gpu(ops, b, t):
    """Sequences of several long splits each: sums over no more than 256 blocks."""
    print("byte many heads", b, t, flush=True)
    n, d = 17000, 64
    g = torch.Generator(device=DEV).manual_seed(b)
    cache = ops.ByteCache(b, 1, n, d, BF, "int8", DEV)
    k, v = (torch.randn((b, 1, n, d), generator=g, device=DEV).to(BF) for _ in range(2))
    lengths = ops.byte_append(cache, k, v, torch.zeros(b, dtype=torch.int32, device=DEV))
    lengths[1::3] -= 64 * 40 + 5
    lengths[1::3] = lengths[1::3] // 64 * 64
    q, kn, vn = (torch.randn((b, 1, t, d), generator=g, device=DEV).to(BF) for _ in range(3))
    mask = torch.ones((t, t), dtype=torch.bool, device=DEV).tril()
    out, lse = ops.byte_attention(q, cache, lengths, kn, vn, mask, return_lse=True)
    only = [0, 1, b // 2, b - 1]
    e, el, tol, tol_l = _attention64(q, cache, lengths, kn, vn, mask, d ** -0.5, only)
    _within(out[only], e[only], tol[only])
    _within(lse[only], el[only], tol_l[only])


@pytest.mark.parametrize("dtype", [BF, FP])
def test_scales_from_end_to_end(ops, dtype):
    """Blocks of tiny and of huge elements beside each other."""
    print("byte scales", dtype, flush=True)
    g = _gen(11)
    for kind in KINDS:
        n = 64 * 6
        size = torch.tensor([1e-30, 1e25, 1.0, 1e-12, 0.0, 1e10], device=DEV).repeat_interleave(64)[:, None]
        k, v = _randn(g, 1, 1, n, 64, dtype=dtype), (_randn(g, 1, 1, n, 64) * size).to(dtype)
        cache = ops.ByteCache(1, 1, n, 64, dtype, kind, DEV)
        lengths = ops.byte_append(cache, k, v, _i32(0))
        q, kn, vn, mask = _drafts(g, 1, 2, 1, 3, 64, dtype)
        _check_attention(ops, q, cache, lengths, kn, vn, mask, what=kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("t,hq", [(65, 1), (50, 2)])
@pytest.mark.parametrize("d", [64, 128])
def test_blocks_of_small_values_in_front_of_larger_ones(ops, kind, d, t, hq):
    """Every fourth block, the first of a split where blocks are shared, has values of (almost) nothing beside the others'; scores
    are equal, rise behind such a block, or leave the larger blocks without weight."""
    print("byte small and large", kind, d, t, hq, flush=True)
    n = 64 * 9 + 17
    small = (torch.arange(n, device=DEV) // 64 % 4 == 0)[:, None] & (torch.arange(n, device=DEV) < 64 * 9)[:, None]
    for seed, (little, size) in enumerate((x, y) for x in (0.0, 1e-30) for y in (1.0, 100.0, 1e10, 1e25)):
        g = _gen(seed)
        v = ((0.5 + torch.rand((1, 1, n, d), generator=g).to(DEV)) * torch.where(small, little, size)).to(BF)
        q, kn, vn, mask = _drafts(g, 1, hq, 1, t, d, BF, 0.1)
        q[..., 0], vn = 2.0, (vn.float().abs() * size).to(BF)
        for nats in (0.0, 5.0, -200.0):
            k = _randn(g, 1, 1, n, d, dtype=BF, scale=0.0 if nats == 0.0 else 0.02)
            k[..., 0] = torch.where(small[:, 0], 0.0, nats / 2).to(BF)
            drafts = (kn, vn, mask) if nats >= 0.0 else (None, None, None)
            cache = ops.ByteCache(1, 1, n, d, BF, kind, DEV)
            lengths = ops.byte_append(cache, k, v, _i32(0))
            _check_attention(ops, q, cache, lengths, *drafts, scale=1.0, what=(little, size, nats))
            out, _ = _check_attention(ops, q, cache, lengths // 64 * 64, scale=1.0, what=(little, size, nats, "blocks alone"))
            if nats < 0.0 and little:
                # the small values alone: an output's and a probability's rounding, 2^-12 of the scores' arithmetic (products of 128
                # elements that add up to 5, and 4 more units), V of one sign (the larger blocks' weight is e^-195 / 200)
                want = _attention64(q, cache, lengths // 64 * 64, None, None, None, 1.0)[0]
                _within(out, want, (2.0 ** -8 + 2.0 ** -11 + 2.0 ** -12) * want.abs(), (little, size, "small alone"))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 128])
def test_blocks_of_all_sizes_in_turn(ops, kind, d):
    """Shared blocks whose values lie up to 2^90 apart, as they come, in order and in turn; a second call gives the same bits."""
    print("byte all sizes", kind, d, flush=True)
    blocks, t = 70, 80
    n = 64 * blocks
    g = _gen(51)
    falling = torch.linspace(45, -45, blocks)
    sizes = (torch.randint(-45, 46, (blocks,), generator=g).float(), falling, falling.flip(0), torch.where(torch.arange(blocks) % 2 == 0, 0.0, -55.0),
             torch.where(torch.arange(blocks) % 5 == 2, 12.0, 0.0))
    for i, size in enumerate(sizes):
        v = _randn(g, 1, 1, n, d) * torch.exp2(size).to(DEV).repeat_interleave(64)[:, None]
        for back in (0.0, 1.0):   # (scores that make up for the sizes: all blocks count)
            k = _randn(g, 1, 1, n, d, scale=0.3)
            k[..., 0] = back * -math.log(2) * size.to(DEV).repeat_interleave(64)
            q, kn, vn, mask = _drafts(g, 1, 1, 1, t, d, BF)
            q[..., 0] = 1.0
            cache = ops.ByteCache(1, 1, n, d, BF, kind, DEV)
            lengths = ops.byte_append(cache, k.to(BF), v.to(BF), _i32(0))
            out, lse = _check_attention(ops, q, cache, lengths, kn, vn, mask, scale=1.0, what=(i, back))
            again = ops.byte_attention(q, cache, lengths, kn, vn, mask, 1.0, return_lse=True)
            assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


@pytest.mark.parametrize("kind", KINDS)
def test_blocks_of_smaller_values_keep_small_probabilities(ops, kind):
    """One element is large, in every fourth block alone; the others are there in the other blocks alone, 2^-order as large, with
    probabilities that end near what fp16 holds."""
    print("byte smaller values", kind, flush=True)
    n, d, t = 64 * 12, 64, 70
    g = _gen(31)
    large = (torch.arange(n, device=DEV) // 64 % 4 == 0)[:, None]
    q = torch.zeros((1, 1, t, d), dtype=BF, device=DEV)
    q[..., 0] = 1.0
    for order in (2, 5, 7, 9.5):
        for nats in (4.0, 8.0, 12.0, 18.0):
            v = torch.where(large, 0.0, _randn(g, 1, 1, n, d) * 2.0 ** -order)
            v[..., :1] = torch.where(large, 3.0, 0.0)
            k = torch.zeros((1, 1, n, d), device=DEV)
            k[..., 0] = torch.where(large[:, 0], 0.0, -nats) + 0.01 * _randn(g, 1, 1, n)
            cache = ops.ByteCache(1, 1, n, d, BF, kind, DEV)
            lengths = ops.byte_append(cache, k.to(BF), v.to(BF), _i32(0))
            out, lse = ops.byte_attention(q, cache, lengths, scale=1.0, return_lse=True)
            e, el, tol, tol_l = _attention64(q, cache, lengths, None, None, None, 1.0)
            if order < 8:   # (what is multiplied in units of the larger scale: 2^-9 of the room that probabilities have)
                V = list(_rows64(cache, 0, 0, n))[1]
                tol += (2.0 ** -24 - 2.0 ** -33) * torch.where(large, 0.0, V.abs()).sum(0)
            _within(out, e, tol, (order, nats))
            _within(lse, el, tol_l, (order, nats))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("t", [3, 70])
def test_values_near_the_largest(ops, dtype, t):
    """As large as 2^15 times a long cache's values may be, cached, in the tail and drafted; also where scores rise behind the first
    block by almost what probabilities have room for."""
    print("byte large values", dtype, t, flush=True)
    n, d = 64 * 300 + 20, 64
    g = _gen(41)
    q, kn, _, mask = _drafts(g, 1, 1, 1, t, d, dtype)
    q[..., 0] = 1.0
    most = 2.0 ** (127 - 15 - math.log2(n + t))
    v = most * (0.5 + 0.5 * torch.rand((1, 1, n + t, d), generator=g).to(DEV))
    for nats in (0.0, 4.8):
        k = torch.zeros((1, 1, n, d), device=DEV)
        k[:, :, 64:, 0] = nats
        cache = ops.ByteCache(1, 1, n, d, dtype, "int8", DEV)
        lengths = ops.byte_append(cache, k.to(dtype), v[:, :, :n].to(dtype), _i32(0))
        _check_attention(ops, q, cache, lengths, kn, v[:, :, n:].to(dtype), mask, scale=1.0, what=nats)


def test_queries_that_are_not_finite(ops):
    """They spoil their own outputs alone."""
    print("byte odd queries", flush=True)
    for dtype in (BF, FP):
        g = _gen(12)
        cache, lengths = _cache(ops, g, 1, 1, 200, 64, dtype, "int8")
        q, kn, vn, mask = _drafts(g, 1, 2, 1, 5, 64, dtype)
        want = ops.byte_attention(q, cache, lengths, kn, vn, mask)
        q[0, 0, 2, 3], q[0, 1, 4, 5] = NAN, INF
        got = ops.byte_attention(q, cache, lengths, kn, vn, mask)
        same = torch.ones((1, 2, 5), dtype=torch.bool, device=DEV)
        same[0, 0, 2] = same[0, 1, 4] = False
        assert torch.equal(got[same], want[same])
        assert not torch.isfinite(got[~same]).any()


def test_attention_places_and_strides(ops):
    """Queries out of a projection, drafted rows between two pieces, one mask for all, bytes as a mask; many sequences."""
    print("byte places", flush=True)
    g = _gen(13)
    for dtype in (BF, FP):
        cache, lengths = _cache(ops, g, 2, 2, 200, 64, dtype, "fp8")
        qkv = _randn(g, 2, 6, 8, 64, dtype=dtype)
        q, kn, vn = qkv[:, :, :4].transpose(1, 2), qkv[:, :, 4:6].transpose(1, 2), qkv[:, :, 6:].transpose(1, 2)
        mask = torch.ones((6, 6), dtype=torch.uint8, device=DEV).tril() * 3
        _check_attention(ops, q, cache, lengths, kn, vn, mask)
        flat = _randn(g, 2 * 2 * 6 * 64 + 1, dtype=dtype)[1:].view(2, 2, 6, 64)
        _check_attention(ops, q, cache, lengths, flat, vn, mask.bool())
        for b in (65, 150):
            print(b, flush=True)
            cache, _ = _cache(ops, g, b, 1, 300, 64, dtype, "int8")
            q, kn, vn, mask = _drafts(g, b, 2, 1, 3, 64, dtype)
            some = torch.tensor([64 * (i % 5) for i in range(b)], dtype=torch.int32, device=DEV)
            some[0] = 300
            _check_attention(ops, q, cache, some, kn, vn, mask, what=b)
    assert ops.byte_attention(q[:, :, :0], cache, some).shape == (150, 2, 0, 64)


def test_attention_refusals(ops):
    from lrqk_amd import _lib
    g = _gen(14)
    cache, n = _cache(ops, g, 1, 2, 70, 64, BF, "int8")
    q, kn, vn, mask = _drafts(g, 1, 4, 2, 3, 64, BF)
    for bad in (lambda: ops.byte_attention(q.float(), cache, n), lambda: ops.byte_attention(q[:, :3], cache, n), lambda: ops.byte_attention(q.cpu(), cache, n),
                lambda: ops.byte_attention(q[..., :32], cache, n), lambda: ops.byte_attention(q, cache, n.long()), lambda: ops.byte_attention(q, cache, n.cpu()),
                lambda: ops.byte_attention(q, cache, _i32(1, 2)), lambda: ops.byte_attention(q, cache, n, kn), lambda: ops.byte_attention(q, cache, n, kn, vn),
                lambda: ops.byte_attention(q, cache, n, mask=mask), lambda: ops.byte_attention(q, cache, n, kn, vn, mask[:, :2]),
                lambda: ops.byte_attention(q, cache, n, kn, vn, mask.float()), lambda: ops.byte_attention(q, cache, n, kn[:, :, :2], vn, mask),
                lambda: ops.byte_attention(q, cache, n, kn.float(), vn, mask), lambda: ops.byte_attention(q, cache, n, *[kn[:, :1].expand(1, 3, 3, 64)] * 2, mask),
                lambda: ops.byte_attention(q, cache, n, scale=0.0), lambda: ops.byte_attention(q, cache, n, scale=NAN)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(_lib.LrqkError):
        ops.byte_attention(torch.zeros((1, 2, 1025, 64), dtype=BF, device=DEV), cache, n)


# ------------------------------------------------------------------------------------------------------ verification

def _verify64(tokens, target, uniforms, draft=None, parents=None):
    """One node after the other, in fp64."""
    b, s, vocab = target.shape
    path, counts, following = torch.full((b, s), -1, dtype=torch.int32), [], []
    for i in range(b):
        x = tokens[i].tolist()
        up = list(range(-1, s - 1)) if parents is None else parents[i].tolist()
        u = uniforms[i].double().tolist()
        q = torch.nan_to_num(target[i].double().cpu(), 0.0, 0.0, 0.0).clamp(min=0)
        p = None if draft is None else torch.nan_to_num(draft[i].double().cpu(), 0.0, 0.0, 0.0).clamp(min=0)
        node, n = 0, 0
        while True:
            path[i, n] = node
            n += 1
            left, mass, taken = q[node].clone(), 1.0, None
            for c in range(node + 1, s):
                if up[c] != node:
                    continue
                known = 0 <= x[c] < vocab
                pc = 1.0 if p is None else float(p[node, x[c]]) if known else 0.0
                if known and u[c] * pc * mass < float(left[x[c]]):
                    taken = c
                    break
                if p is None:
                    if known:
                        mass -= float(left[x[c]])
                        left[x[c]] = 0.0
                else:
                    left = (left - mass * p[node]).clamp(min=0)
                    mass = float(left.sum())
            if taken is None:
                break
            node = taken
        counts.append(n)
        if not float(left.sum()) > 0:
            left = q[node]
        sums = left.cumsum(0)
        above = torch.nonzero((sums > u[0] * float(sums[-1])) & (left > 0))
        some = torch.nonzero(left)
        following.append(int(above[0] if len(above) else some[-1]) if len(some) else -1)
    return path.to(DEV), _i32(*counts), _i32(*following)


def _tree(g, b, s, children):
    up = [[-1] * s for _ in range(b)]
    for row in up:
        for i in range(1, s):
            free = [j for j in range(i) if sum(x == j for x in row[1:i]) < children]
            row[i] = free[int(torch.randint(0, len(free), (1,), generator=g))]
    return torch.tensor(up, dtype=torch.int32, device=DEV)


def _probabilities(g, b, s, vocab, dtype, near=0.6):
    x = torch.randn((b, s, vocab), generator=g) * 2
    y = x + near * torch.randn((b, s, vocab), generator=g)
    return torch.softmax(x, -1).to(dtype).to(DEV), torch.softmax(y, -1).to(dtype).to(DEV)


def _tokens(g, q, parents):
    b, s, vocab = q.shape
    up = torch.arange(-1, s - 1).expand(b, s) if parents is None else parents.cpu().long()
    rows = q.float().cpu().gather(1, up.clamp(min=0)[..., None].expand(-1, -1, vocab)).flatten(0, 1)
    return torch.multinomial(rows + 1e-9, 1, generator=g).view(b, s).to(torch.int32).to(DEV)


def _check_verify(ops, tokens, target, uniforms, draft=None, parents=None, what=""):
    got = ops.verify_drafts(tokens, target, uniforms, draft, parents)
    for a, z, name in zip(got, _verify64(tokens, target, uniforms, draft, parents), ("path", "counts", "next")):
        assert a.dtype == torch.int32 and torch.equal(a, z), (what, name, a.tolist(), z.tolist())
    return got


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("vocab", [1, 2, 7, 255, 2048, 2049, 5000, 32001])
def test_verify_chains_and_trees(ops, dtype, vocab):
    print("verify", dtype, vocab, flush=True)
    g = _gen(vocab)
    for b, s, children in ((1, 1, 1), (3, 2, 1), (4, 9, 1), (4, 2, 2), (4, 14, 3), (2, 40, 5)):
        target, draft = _probabilities(g, b, s, vocab, dtype)
        uniforms = torch.rand((b, s), generator=g).to(DEV)
        parents = _tree(g, b, s, children)
        for up in ((None, parents) if children == 1 else (parents,)):
            if children == 1:
                parents = (torch.arange(s, device=DEV) - 1).to(torch.int32).repeat(b, 1)
                up = None if up is None else parents
            tokens = _tokens(g, draft, up)
            a = _check_verify(ops, tokens, target, uniforms, draft, up, what=(b, s, children))
            if s > 1:   # the last node's row is not wanted
                z = ops.verify_drafts(tokens, target, uniforms, draft[:, :s - 1], up)
                assert all(torch.equal(x, y) for x, y in zip(a, z))
            _check_verify(ops, tokens, target, uniforms, None, up, what=(b, s, children, "no draft"))


def test_verify_of_a_single_node_with_a_row_of_the_drafting_model(ops):
    """The library's entry may be given one (the Python call leaves it out): it is not looked at."""
    from lrqk_amd import _lib
    lib, b, vocab = _lib.load(), 5, 5000
    g = _gen(6)
    target, draft = (_probabilities(g, b, 1, vocab, FP)[i].to(DEV) for i in range(2))
    tokens, u = torch.zeros((b, 1), dtype=torch.int32, device=DEV), torch.rand((b, 1), generator=g).to(DEV)
    want = ops.verify_drafts(tokens, target, u)
    need = lib.lrqk_verify_drafts_workspace(b, 1, vocab)
    for parents in (None, tokens):
        ws = torch.full((need // 4,), -1, dtype=torch.int32, device=DEV)
        path, counts, token = torch.empty_like(tokens), tokens.new_empty(b), tokens.new_empty(b)
        assert lib.lrqk_verify_drafts(tokens.data_ptr(), None if parents is None else parents.data_ptr(), target.data_ptr(), vocab, vocab,
                                      draft.data_ptr(), vocab, vocab, u.data_ptr(), path.data_ptr(), counts.data_ptr(), token.data_ptr(), b, 1,
                                      vocab, ws.data_ptr(), need, _lib.F32, torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip((path, counts, token), want))


def test_verify_accepts_all_or_nothing(ops):
    """uniforms of 0 accept what has any probability; drafts equal to the target are always accepted; tokens of probability 0 never."""
    print("verify ends", flush=True)
    g = _gen(20)
    b, s, vocab = 3, 12, 700
    target, draft = _probabilities(g, b, s, vocab, FP)
    tokens = _tokens(g, draft, None)
    zero = torch.zeros((b, s), device=DEV)
    path, counts, token = _check_verify(ops, tokens, target, zero, draft)
    assert counts.tolist() == [s] * b and token.tolist() == [0] * b
    most = torch.full((b, s), 1 - 2.0 ** -24, device=DEV)
    _, counts, _ = _check_verify(ops, tokens, target, most, target)
    assert counts.tolist() == [s] * b
    target.scatter_(2, tokens.roll(-1, 1)[..., None].long(), 0.0)
    _, counts, token = _check_verify(ops, tokens, target, zero, draft)
    assert counts.tolist() == [1] * b
    one = torch.zeros_like(target).scatter_(2, (tokens.roll(-1, 1)[..., None].long() + 1) % vocab, 1.0)   # greedy: one token each
    _, counts, token = _check_verify(ops, tokens, one, most)
    assert counts.tolist() == [1] * b and torch.equal(token, (tokens[:, 1] + 1) % vocab)


def test_verify_odd_inputs(ops):
    """Parents that are none, tokens outside the vocabulary, equal siblings, rows of zeros, NaN and negative numbers, uniforms at and
    beyond the ends."""
    print("verify odd", flush=True)
    g = _gen(21)
    b, s, vocab = 6, 15, 333
    for kind in range(6):
        target, draft = _probabilities(g, b, s, vocab, FP)
        parents = _tree(g, b, s, 4)
        tokens = _tokens(g, draft, parents)
        uniforms = torch.rand((b, s), generator=g).to(DEV)
        if kind == 0:
            parents[:, 3], parents[:, 5], parents[:, 7], parents[:, 0] = 3, -1, 40, 2
            tokens[:, 2], tokens[:, 4] = -1, vocab
        elif kind == 1:
            tokens[:, 1:] = tokens[:, 1:2]
        elif kind == 2:
            target[:, :, 40:] = 0.0
            target[1], target[2] = 0.0, NAN
        elif kind == 3:
            target[:, :, ::2] = NAN
            draft[:, :, 1::2] = -1.0
            target[:, :, 5] = -3.0
        elif kind == 4:
            uniforms[:, 0] = torch.tensor([0.0, 1.0, 1 - 2.0 ** -24, 2.0, -1.0, 0.5], device=DEV)
        else:
            draft = target * 4    # nothing is left behind a refused one
            uniforms = 1 - uniforms * 1e-3
        for d in (draft, None):
            if kind == 1 or d is None or kind != 3:
                _check_verify(ops, tokens, target, uniforms, d, parents, what=(kind, d is None))
            else:
                _check_verify(ops, tokens, target, uniforms, d, parents, what=kind)


def test_verify_looked_up_drafts_of_rows_that_do_not_add_up_to_one(ops):
    """Without probabilities of the drafts, Z is 1 less those of the refused tokens, whatever a row adds up to; with them it is the
    sum of what is left."""
    print("verify unequal sums", flush=True)
    target = torch.zeros((1, 3, 8), device=DEV)
    target[..., 0], target[..., 1] = 0.3, 0.2
    tokens, parents = _i32(5, 0, 1)[None], _i32(-1, 0, 0)[None]
    draft = torch.full_like(target, 0.125)
    for u, looked_up, drawn in ((0.28, True, True), (0.29, False, True), (0.999, False, True)):
        uniforms = torch.tensor([[0.5, 0.9, u]], device=DEV)   # 0.9 > 0.3: refused; then u 0.7 < 0.2, if the sum counted u 0.2 < 0.2
        _, counts, _ = _check_verify(ops, tokens, target, uniforms, None, parents, what=u)
        assert counts.tolist() == [1 + looked_up]
        # (0.9 / 8 < 0.3 would be accepted: 0.9 of a target of 0.1.  Left are then 0.075 of token 1, and Z is that)
        less = target.clone()
        less[..., 0] = 0.1
        _, counts, _ = _check_verify(ops, tokens, less, uniforms, draft, parents, what=u)
        assert counts.tolist() == [1 + drawn]


def test_verify_places_and_the_largest_trees(ops):
    print("verify places", flush=True)
    g = _gen(22)
    big = torch.softmax(torch.randn((3, 20, 2, 600), generator=g), -1).to(DEV)
    target, draft = big[:, :9, 0, 3:503], big[:, 9:18, 1, :500]   # rows apart and between two pieces
    uniforms = torch.rand((3, 9), generator=g).to(DEV)
    _check_verify(ops, _tokens(g, draft, None), target, uniforms, draft)
    for b, s, vocab in ((2, 1024, 50), (1, 300, 9)):
        target, draft = _probabilities(g, b, s, vocab, FP, near=0.02)
        uniforms = torch.rand((b, s), generator=g).to(DEV)
        _check_verify(ops, _tokens(g, draft, None), target, uniforms, draft)
        parents = _tree(g, b, min(s, 300), 300) if s <= 300 else ((torch.arange(s, device=DEV) - 1) // 2).clamp(min=0).to(torch.int32).repeat(b, 1)
        _check_verify(ops, _tokens(g, draft, parents), target, uniforms, draft, parents)
        _check_verify(ops, _tokens(g, target, parents), target, uniforms, None, parents)
    empty = ops.verify_drafts(*[torch.zeros((0, 3), dtype=d, device=DEV) for d in (torch.int32,)], torch.zeros((0, 3, 5), device=DEV), torch.zeros((0, 3), device=DEV))
    assert [x.shape for x in empty] == [(0, 3), (0,), (0,)]


def test_verify_vocabularies_of_many_chunks(ops):
    """More tokens than one look finds a place among, and rows of them that nothing is left of."""
    print("verify large", flush=True)
    g = torch.Generator(device=DEV).manual_seed(24)
    for vocab in (2048 * 2048 + 7, 3 * 2048 * 2048 - 1):
        target = torch.rand((2, 3, vocab), generator=g, device=DEV)
        target /= target.sum(-1, keepdim=True)
        draft = torch.rand((2, 3, vocab), generator=g, device=DEV)
        draft /= draft.sum(-1, keepdim=True)
        tokens = torch.randint(0, vocab, (2, 3), generator=g, device=DEV, dtype=torch.int32)
        parents = _i32(-1, 0, 0).repeat(2, 1)
        for u in (0.0, 0.3, 0.99999):
            uniforms = torch.full((2, 3), 1 - 2.0 ** -24, device=DEV)
            uniforms[:, 0] = u
            _check_verify(ops, tokens, target, uniforms, draft, parents, what=(vocab, u))
            _check_verify(ops, tokens, target, uniforms, 3 * target, parents, what=(vocab, u, "nothing left"))


def test_verify_of_the_last_token_in_front_of_zeros(ops):
    """More chunks than are looked through at once, the border at the sum itself: the last token that has anything, whatever zeros
    follow it in its run of chunks, in its chunk and behind both."""
    print("verify zeros behind", flush=True)
    vocab = 2048 * 2048 * 2 + 4096 + 5
    target = torch.zeros((4, 1, vocab), device=DEV)
    for i, last in enumerate((5, 2048 * 2 * 9 + 3, 2048 * 2 * 9 + 2048 + 2047, vocab - 1)):
        target[i, 0, 1], target[i, 0, last] = 0.5, 0.25
    uniforms = torch.ones((4, 1), device=DEV)
    tokens = torch.zeros((4, 1), dtype=torch.int32, device=DEV)
    for dtype in (FP, BF):
        _check_verify(ops, tokens, target.to(dtype), uniforms)
        _check_verify(ops, tokens, target.to(dtype), uniforms * 0.6)
        _check_verify(ops, tokens, target.to(dtype), uniforms * 0.7)


@pytest.mark.parametrize("children", [1, 3])
@pytest.mark.parametrize("drafted", [True, False])
def test_what_is_accepted_or_drawn_has_the_targets_distribution(ops, drafted, children):
    """The first token behind the root, of 60000 sequences with one distribution: frequencies within 5 standard deviations."""
    print("verify law", drafted, children, flush=True)
    g = _gen(23)
    n, s, vocab = 60000, 1 + children, 11
    q, p = torch.softmax(torch.randn(vocab, generator=g), 0), torch.softmax(torch.randn(vocab, generator=g), 0)
    parents = torch.zeros((n, s), dtype=torch.int32, device=DEV)
    parents[:, 0] = -1
    tokens = torch.multinomial(p, n * s, replacement=True, generator=g).view(n, s).to(torch.int32).to(DEV)
    uniforms = torch.rand((n, s), generator=g).to(DEV)
    target, draft = (x.to(DEV).expand(n, s, vocab) for x in (q, p))
    path, counts, token = ops.verify_drafts(tokens, target, uniforms, draft if drafted else None, parents)
    first = torch.where(counts > 1, tokens.gather(1, path[:, 1:2].clamp(min=0).long())[:, 0], token)
    seen = torch.bincount(first.long(), minlength=vocab).cpu().double() / n
    assert float(((seen - q).abs() / (q * (1 - q) / n).sqrt()).max()) < 5


def test_verify_refusals(ops):
    from lrqk_amd import _lib
    target = torch.ones((2, 3, 10), device=DEV) / 10
    tokens, uniforms = torch.zeros((2, 3), dtype=torch.int32, device=DEV), torch.zeros((2, 3), device=DEV)
    for bad in (lambda: ops.verify_drafts(tokens.long(), target, uniforms), lambda: ops.verify_drafts(tokens[:, :2], target, uniforms),
                lambda: ops.verify_drafts(tokens, target.half(), uniforms), lambda: ops.verify_drafts(tokens, target, uniforms.double()),
                lambda: ops.verify_drafts(tokens, target, uniforms, target[:, :1]), lambda: ops.verify_drafts(tokens, target, uniforms, target.bfloat16()),
                lambda: ops.verify_drafts(tokens, target, uniforms, target[..., :9]), lambda: ops.verify_drafts(tokens, target, uniforms, target, tokens[:1]),
                lambda: ops.verify_drafts(tokens.cpu(), target, uniforms), lambda: ops.verify_drafts(tokens, target.cpu(), uniforms.cpu()),
                lambda: ops.verify_drafts(tokens, target.transpose(1, 2).contiguous().transpose(1, 2), uniforms),
                lambda: ops.verify_drafts(tokens[:, :0], target[:, :0], uniforms[:, :0]), lambda: ops.verify_drafts(tokens, target[..., :0], uniforms)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(_lib.LrqkError):
        ops.verify_drafts(torch.zeros((1, 1025), dtype=torch.int32, device=DEV), torch.zeros((1, 1025, 4), device=DEV), torch.zeros((1, 1025), device=DEV))


def test_offsets_beyond_32_bits(ops):
    """Codes behind the first 4 GB, rows of new tokens and of probabilities that far apart."""
    print("far", flush=True)
    g = torch.Generator(device=DEV).manual_seed(40)
    heads, n, d = 68, 2 ** 20, 64
    k, v = (torch.randn((1, 1, n, d), generator=g, device=DEV).to(BF) for _ in range(2))
    cache = ops.ByteCache(1, heads, n, d, BF, "fp8", DEV)
    assert cache.k.numel() > 2 ** 32
    lengths = ops.byte_append(cache, k.expand(1, heads, n, d), v.expand(1, heads, n, d), _i32(0), counts=_i32(n - 30))
    for t in (2, 70):
        q = torch.randn((1, 1, t, d), generator=g, device=DEV).to(BF)
        out, lse = ops.byte_attention(q.expand(1, heads, t, d).contiguous(), cache, lengths, return_lse=True)
        assert all(torch.equal(out[0, 0], out[0, h]) and torch.equal(lse[0, 0], lse[0, h]) for h in (1, 62, 63, 64, 66, 67))
        one = ops.ByteCache(1, 1, n, d, BF, "fp8", DEV)
        for name in NAMES:
            getattr(one, name).copy_(getattr(cache, name)[:, heads - 1:])
        e, el, tol, tol_l = _attention64(q, one, lengths, None, None, None, d ** -0.5)
        _within(out[:, -1:], e, tol, t)
        _within(lse[:, -1:], el, tol_l, t)
    del cache, one, k, v
    flat = torch.empty(2 * 2 ** 30 + 1000, device=DEV)
    target = flat.as_strided((1, 3, 900), (1, 2 ** 30, 1))
    target.copy_(torch.softmax(torch.randn((1, 3, 900), generator=g, device=DEV), -1))
    draft = target.flip(-1).contiguous()
    tokens = torch.tensor([[0, 5, 600]], dtype=torch.int32, device=DEV)
    for u in (0.0, 0.5, 0.999):
        uniforms = torch.full((1, 3), u, device=DEV)
        _check_verify(ops, tokens, target, uniforms, draft)
        _check_verify(ops, tokens, target, uniforms)
    rows = flat.view(BF).as_strided((1, 1, 3, 64), (8, 8, 2 ** 31, 1))
    rows.copy_(torch.randn((1, 1, 3, 64), generator=g, device=DEV))
    _check_append(ops, ops.ByteCache(1, 1, 128, 64, BF, "int8", DEV), rows, rows.contiguous(), _i32(62))


# ---------------------------------------------------------------------------------------------------------- together

def _seen(parents):
    """bool [b,s,s]: a node sees itself and those between it and the root."""
    b, s = parents.shape
    sees = torch.eye(s, dtype=torch.bool, device=DEV).repeat(b, 1, 1)
    for i in range(1, s):
        sees[:, i] |= sees.gather(1, parents[:, i:i + 1, None].long().expand(-1, -1, s))[:, 0]
    return sees


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF, FP])
def test_rounds_of_drafts_over_a_cache_in_8_bits(ops, dtype, kind):
    """Positions, attention, verification and the accepted rows into the cache, round after round, every call held to its formula;
    in the end the cache is what one append of all accepted rows makes of them."""
    print("rounds", dtype, kind, flush=True)
    g = _gen(31)
    b, hq, hc, d, s, vocab = 3, 6, 2, 64, 10, 500
    plan = ops.RotaryPlan(d, 1e4, device=DEV)
    cache = ops.ByteCache(b, hc, 512, d, dtype, kind, DEV)
    k, v = (_randn(g, b, hc, 150, d, dtype=dtype) for _ in range(2))
    counts = _i32(150, 63, 1)
    kept = [[(k[i, :, :c], v[i, :, :c])] for i, c in enumerate(counts.tolist())]
    lengths = _check_append(ops, cache, k, v, torch.zeros(b, dtype=torch.int32, device=DEV), counts)
    for turn in range(12):
        parents = _tree(g, b, s, 3)
        mask = _seen(parents)
        positions = lengths[:, None] + (mask.sum(-1) - 1).to(torch.int32)
        q, k = ops.rotary(plan, _randn(g, b, hq, s, d, dtype=dtype, scale=2.0), _randn(g, b, hc, s, d, dtype=dtype), positions)
        v = _randn(g, b, hc, s, d, dtype=dtype)
        out, _ = _check_attention(ops, q, cache, lengths, k, v, mask, what=turn)
        target, draft = _probabilities(g, b, s, vocab, dtype, near=0.3)
        path, counts, token = _check_verify(ops, _tokens(g, draft, parents), target, torch.rand((b, s), generator=g).to(DEV), draft, parents)
        for i in range(b):
            nodes = path[i, :int(counts[i])].long()
            kept[i].append((k[i][:, nodes], v[i][:, nodes]))
        lengths = _check_append(ops, cache, k, v, lengths, counts, path, what=turn)
    for i in range(b):
        rows = [torch.cat(x, 1)[None] for x in zip(*kept[i])]
        assert int(lengths[i]) == rows[0].shape[2]
        one = ops.ByteCache(1, hc, 512, d, dtype, kind, DEV)
        ops.byte_append(one, *rows, _i32(0))
        for name in NAMES:
            assert torch.equal(getattr(one, name)[0].float(), getattr(cache, name)[i].float()), (i, name)


def _round(ops, cache, lengths, q, k, v, mask, tokens, target, draft, parents, uniforms):
    out = ops.byte_attention(q, cache, lengths, k, v, mask)
    path, counts, token = ops.verify_drafts(tokens, target, uniforms, draft, parents)
    lengths.copy_(ops.byte_append(cache, k, v, lengths, counts, path))
    return out, path, counts, token


def _round_inputs(g, dtype, b, hq, s, children):
    q, k, v, _ = _drafts(g, b, hq, 2, s, 64, dtype)
    parents = _tree(g, b, s, children)
    target, draft = _probabilities(g, b, s, 3000, FP, near=0.3)
    return [q, k, v, _seen(parents), _tokens(g, draft, parents), target, draft, parents, torch.rand((b, s), generator=g).to(DEV)]


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("s,hq", [(1, 2), (6, 8), (40, 8)])
def test_rounds_replayed_from_graphs(ops, dtype, s, hq):
    """Two captured rounds, replayed in turn with the lengths growing, an eager round of a third cache between the replays: the
    same bits as eager rounds."""
    print("graphs", dtype, s, hq, flush=True)
    g = _gen(s)
    b = 2

    def start():
        return _cache(ops, g, b, 2, 230, 64, dtype, "int8")[0], _i32(230, 192)
    fixed = [_round_inputs(g, dtype, b, hq, s, 2) for _ in range(2)]
    sides = [start() for _ in range(2)]
    third, scrap = start(), start()
    eager = []
    for cache, lengths in sides:
        twin = ops.ByteCache(b, 2, 238, 64, dtype, "int8", DEV)
        for n in NAMES:
            getattr(twin, n).copy_(getattr(cache, n))
        eager.append((twin, lengths.clone()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _round(ops, *scrap, *fixed[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for x, (cache, lengths) in zip(fixed, sides):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_round(ops, cache, lengths, *x))
        graphs.append(graph)
    for _ in range(5):
        for x, mine, (cache, lengths), graph, out in zip(fixed, eager, sides, graphs, outs):
            new = _round_inputs(g, dtype, b, hq, s, 2)
            for a, z in zip(x, new):
                a.copy_(z)
            graph.replay()
            _round(ops, *third, *_round_inputs(g, dtype, b, hq, s, 3))
            torch.cuda.synchronize()
            want = _round(ops, *mine, *new)
            assert all(torch.equal(a, z) for a, z in zip(out, want)) and torch.equal(lengths, mine[1])
            assert all(torch.equal(getattr(cache, n).float(), getattr(mine[0], n).float()) for n in NAMES)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("b,t,hq", [(1, 1, 4), (20, 1, 4), (20, 7, 8), (3, 40, 4)])
def test_graphs_of_one_pool_over_changing_lengths(ops, dtype, b, t, hq):
    """Two captured attentions that share the memory that they allocate, replayed in turn over lengths that change, eager calls
    between: the same bits as eager calls."""
    print("pool", dtype, b, t, hq, flush=True)
    g = _gen(b + t)
    cache, full = _cache(ops, g, b, 2, 900, 64, dtype, "int8")
    inputs = [_drafts(g, b, hq, 2, t, 64, dtype) for _ in range(2)]
    lengths = full.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.byte_attention(inputs[0][0], cache, lengths, *inputs[0][1:], return_lse=True)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs, pool = [], [], torch.cuda.graph_pool_handle()
    for q, kn, vn, mask in inputs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append([x.clone() for x in ops.byte_attention(q, cache, lengths, kn, vn, mask, return_lse=True)])
        graphs.append(graph)
    for _ in range(6):
        lengths.copy_(torch.randint(0, 901, (b,), generator=g).to(torch.int32))
        for graph, out, (q, kn, vn, mask) in zip(graphs, outs, inputs):
            want = ops.byte_attention(q, cache, lengths, kn, vn, mask, return_lse=True)
            graph.replay()
            assert all(torch.equal(x, y) for x, y in zip(out, want))
            torch.cuda.synchronize()


def test_two_streams_at_once(ops):
    """The same calls on two streams at once and on one after the other have the same bits."""
    print("streams", flush=True)
    g = _gen(33)
    x = [_round_inputs(g, BF, 2, 8, 12, 3) for _ in range(2)]
    sides = [_cache(ops, g, 2, 2, 600, 64, BF, "fp8") for _ in range(2)]
    alone = []
    for cache, lengths in sides:
        twin = ops.ByteCache(2, 2, 608, 64, BF, "fp8", DEV)
        for n in NAMES:
            getattr(twin, n).copy_(getattr(cache, n))
        alone.append((twin, lengths.clone()))
    want = [[_round(ops, *alone[i], *x[i]) for _ in range(6)] for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(_round(ops, *sides[i], *x[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, z) for r, w in zip(got[i], want[i]) for a, z in zip(r, w))
        assert all(torch.equal(getattr(sides[i][0], n).float(), getattr(alone[i][0], n).float()) for n in NAMES)


# ---------------------------------------------------------------------------------------------------------- a decoder

def _model(dtype, d=16, **kw):
    from lrqk_amd import decoder
    cfg = decoder.DecoderConfig(layers=2, hidden=64, heads=4, kv_heads=2, head_dim=d, intermediate=128, vocab=97, rope_theta=1e4, **kw)
    return decoder.LlamaShapeDecoder(cfg, dtype, DEV, seed=3)


@pytest.mark.parametrize("kind", KINDS)
def test_a_decoder_over_byte_caches(ops, kind):
    """While no block is complete every token is read as it came: the tokens of the dense cache.  Beyond that it runs."""
    print("decoder", kind, flush=True)
    m = _model(FP)
    ids = torch.randint(0, 97, (2, 24), generator=_gen(0)).to(DEV)
    dense, *_ = m.generate(ids, 20, None)
    caches = m.new_byte_caches(2, 200, kind)
    got, *_ = m.generate(ids, 20, caches)
    assert torch.equal(got, dense) and caches.lengths.tolist() == [43, 43]
    caches = m.new_byte_caches(2, 200, kind)
    m.generate(ids, 5, caches)   # (a prompt begins anew)
    long, *_ = m.generate(torch.cat((ids, dense, ids, ids), 1), 90, caches)
    assert long.shape == (2, 90) and caches.lengths.tolist() == [24 * 3 + 20 + 89] * 2 and int(long.min()) >= 0 and int(long.max()) < 97
    with pytest.raises(ValueError, match="room"):
        m.generate(ids, 300, caches)


@pytest.mark.parametrize("kind", KINDS)
def test_drafted_generation_is_greedy_generation(ops, kind):
    """Neighbouring pairs are turned by the library in both: the same tokens in fewer rounds."""
    print("drafted", kind, flush=True)
    m = _model(FP, rope_interleaved=True)
    ids = torch.randint(0, 97, (3, 20), generator=_gen(1)).to(DEV)
    ids = torch.cat((ids, ids, ids), 1)
    want, *_ = m.generate(ids, 80, m.new_byte_caches(3, 200, kind))
    caches = m.new_byte_caches(3, 200, kind)
    got, rounds = m.generate_drafted(ids, 80, caches, drafts=5)
    assert torch.equal(got, want) and rounds < 79, rounds
    # what is cached are the tokens but the last, and those behind the wanted ones that came with them
    assert all(60 + 79 <= n <= 60 + 79 + 6 for n in caches.lengths.tolist())
    drawn, _ = m.generate_drafted(ids, 30, m.new_byte_caches(3, 200, kind), drafts=5, temperature=1.0,
                                  generator=torch.Generator(device=DEV).manual_seed(0))
    assert drawn.shape == (3, 30) and int(drawn.min()) >= 0 and int(drawn.max()) < 97
    for bad in (dict(drafts=0), dict(new_tokens=0), dict(ngram=0), dict(temperature=-1.0), dict(new_tokens=190)):
        with pytest.raises(ValueError):
            m.generate_drafted(**{**dict(ids=ids, new_tokens=5, caches=caches), **bad})


def test_drafted_generation_of_short_prompts(ops):
    """Prompts of one token, fewer than are looked up with, and a cache that is full at the end."""
    print("drafted short", flush=True)
    m = _model(FP, rope_interleaved=True)
    for b, l, new in ((1, 1, 1), (2, 1, 40), (1, 3, 57)):
        ids = torch.randint(0, 97, (b, l), generator=_gen(l)).to(DEV)
        want, *_ = m.generate(ids, new, m.new_byte_caches(b, 64))
        got, _ = m.generate_drafted(ids, new, m.new_byte_caches(b, 64), drafts=4, ngram=3)
        assert torch.equal(got, want), (b, l, new)


def _turned64(x, positions, theta):
    """x [b,H,s,d] turned to positions [b,s] by halves, in fp64."""
    half = x.shape[-1] // 2
    freq = theta ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
    angle = positions.double()[:, None, :, None] * freq
    a, z = x[..., :half].double(), x[..., half:].double()
    return torch.cat((a * torch.cos(angle) - z * torch.sin(angle), z * torch.cos(angle) + a * torch.sin(angle)), -1)


def test_positions_of_prompts_tokens_and_drafts(ops):
    """Keys of a prompt, of single tokens and of drafts are turned to the same far positions alike, also where sequences have
    different lengths."""
    print("decoder positions", flush=True)
    from lrqk_amd.decoder import _rms
    m, far = _model(FP), 100000

    def keys(ids):   # of the first layer, as they are before they are turned
        return (_rms(m.embed[ids], m.layers[0]["n1"], m.cfg.rms_eps) @ m.layers[0]["wk"]).view(*ids.shape, 2, 16).transpose(1, 2)

    def check(got, ids, positions, what):
        # two products, and a sine and a cosine of 2 units each; the sums of 64 products come in another order for another count
        x = keys(ids)
        pair = torch.cat([torch.hypot(x[..., :8], x[..., 8:])] * 2, -1).double()
        sums = _rms(m.embed[ids], m.layers[0]["n1"], m.cfg.rms_eps).abs() @ m.layers[0]["wk"].abs()
        tol = 6 * U * pair + 64 * U * sums.view(*ids.shape, 2, 16).transpose(1, 2).double().amax(-1, keepdim=True)
        _within(got, _turned64(x, positions, m.cfg.rope_theta), tol, what)

    ids = torch.randint(0, 97, (2, 3000), generator=_gen(0)).to(DEV)
    caches = m.new_byte_caches(2, far + 100)
    m.forward(ids, 0, caches)
    last = torch.arange(3000 - 128, 3000, device=DEV)
    check(caches.layers[0].k_tail[:, :, last % 128], ids[:, last], last.expand(2, -1), "prompt")
    for lengths in (_i32(far, far), _i32(far, far - 70)):
        caches.lengths = lengths
        m.forward(ids[:, :1], far, caches)
        got = torch.stack([caches.layers[0].k_tail[i, :, n % 128] for i, n in enumerate(lengths.tolist())])[:, :, None]
        check(got, ids[:, :1], lengths[:, None], ("token", lengths.tolist()))
        steps = torch.arange(4, dtype=torch.int32, device=DEV)
        _, rows = m._draft_logits(ids[:, :4], torch.ones((4, 4), dtype=torch.bool, device=DEV).tril(), lengths[:, None] + steps, caches)
        check(rows[0][0], ids[:, :4], lengths[:, None] + steps, ("drafts", lengths.tolist()))


@pytest.mark.parametrize("dtype", [BF, FP])
def test_drafted_generation_of_the_default_layout(ops, dtype):
    """Halves, turned by the library in both.  While no block is complete every token is read as it came, and fp32 tokens are the
    same (beyond, a token that completes a block sees it in 8 bits, a round as it came)."""
    print("drafted halves", dtype, flush=True)
    m = _model(dtype)
    ids = torch.randint(0, 97, (2, 20), generator=_gen(5)).to(DEV).repeat(1, 3)
    got, _ = m.generate_drafted(ids, 60, m.new_byte_caches(2, 200), drafts=5)
    assert got.shape == (2, 60) and int(got.min()) >= 0 and int(got.max()) < 97
    got, _ = m.generate_drafted(ids[:, :20], 38, m.new_byte_caches(2, 64), drafts=5)
    assert got.shape == (2, 38)
    if dtype == FP:
        want, *_ = m.generate(ids[:, :20], 38, m.new_byte_caches(2, 64))
        assert torch.equal(got, want)


def _model64(m, ids, positions, keys, dtype=torch.float64):
    """The decoder's logits [b,s,vocab] by torch in `dtype`.  keys(layer, sequence, head, k, v) -> what the s tokens attend to,
    whose own rows [s,d] are k and v, in `dtype`: (keys [n,d], values [n,d], bool [s,n])."""
    c = m.cfg
    (b, s), d = ids.shape, c.head_dim

    def rms(x):
        return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + c.rms_eps)

    def heads(x, w):
        return (x @ w.to(dtype)).view(b, s, -1, d).transpose(1, 2)
    x = m.embed[ids].to(dtype)
    for li, L in enumerate(m.layers):
        y = rms(x)
        q, k = (_turned64(heads(y, L[w]), positions, c.rope_theta).to(dtype) for w in ("wq", "wk"))
        v, o = heads(y, L["wv"]), torch.zeros_like(q)
        for i in range(b):
            for h in range(c.heads):
                g = h * c.kv_heads // c.heads
                K, V, sees = keys(li, i, g, k[i, g], v[i, g])
                o[i, h] = torch.softmax((q[i, h] @ K.T * d ** -0.5).masked_fill(~sees, -INF), -1) @ V
        x = x + o.transpose(1, 2).reshape(b, s, -1) @ L["wo"].to(dtype)
        y = rms(x)
        x = x + (torch.nn.functional.silu(y @ L["wg"].to(dtype)) * (y @ L["wu"].to(dtype))) @ L["wd"].to(dtype)
    return rms(x) @ m.lm_head.to(dtype)


@pytest.mark.parametrize("kind", KINDS)
def test_logits_over_a_cache_in_8_bits(ops, kind):
    """Tokens and rounds of drafts beyond the first block: the logits are those of the rows that the cache holds by then, in 64 bits.
    Off by 16 times what the same sums in fp32 by torch are off by (queries and probabilities have 22 bits where those have 24,
    codes are scaled behind the sums)."""
    print("decoder logits", kind, flush=True)
    m = _model(FP)
    g = _gen(9)
    ids = torch.randint(0, 97, (2, 400), generator=g).to(DEV)
    caches = m.new_byte_caches(2, 400, kind)
    m.forward(ids[:, :100], 0, caches)

    def near(got, new, positions, keys):
        want, rough = (_model64(m, new, positions, lambda *a: keys(dt, *a), dt) for dt in (torch.float64, FP))
        _within(got, want, torch.full_like(want, 16 * float((rough - want).abs().max())))

    for n in range(100, 134):   # (the token at 127 is the last one of a block, and sees itself in 8 bits)
        got = m.forward(ids[:, n:n + 1], n, caches)

        def held(dt, li, i, h, k, v):
            K, V = (x.to(dt) for x in _rows64(caches.layers[li], i, h, n + 1))
            return K, V, torch.ones((1, n + 1), dtype=torch.bool, device=DEV)
        near(got[:, None], ids[:, n:n + 1], torch.full((2, 1), n, device=DEV), held)
    s, at = 6, torch.arange(2, device=DEV)[:, None]
    steps, mask = torch.arange(s, dtype=torch.int32, device=DEV), torch.ones((s, s), dtype=torch.bool, device=DEV).tril()
    for _ in range(12):   # rounds of which the sequences keep different numbers
        lengths = caches.lengths
        new = ids[at, lengths[:, None] + steps]
        got, rows = m._draft_logits(new, mask, lengths[:, None] + steps, caches)

        def both(dt, li, i, h, k, v):
            n = int(lengths[i])
            K, V = (torch.cat((x.to(dt), y)) for x, y in zip(_rows64(caches.layers[li], i, h, n), (k, v)))
            return K, V, torch.cat((torch.ones((s, n), dtype=torch.bool, device=DEV), mask), 1)
        near(got, new, lengths[:, None] + steps, both)
        counts = torch.randint(1, s + 1, (2,), generator=g, dtype=torch.int32).to(DEV)
        for layer, (k, v) in zip(caches.layers, rows):
            seen = ops.byte_append(layer, k, v, lengths, counts)
        caches.lengths = seen
    # and a token where the sequences have different lengths
    lengths = caches.lengths
    assert lengths[0] != lengths[1]
    new = ids[at, lengths[:, None]]
    got = m.forward(new, int(lengths.max()), caches)

    def ragged(dt, li, i, h, k, v):
        n = int(lengths[i]) + 1
        K, V = (x.to(dt) for x in _rows64(caches.layers[li], i, h, n))
        return K, V, torch.ones((1, n), dtype=torch.bool, device=DEV)
    near(got[:, None], new, lengths[:, None], ragged)
