"""The operators around a drafted, budgeted cache against plain implementations in 64 bits: rotary positions, attention of a
tree of drafted tokens, the attention that cached tokens got, and eviction by it.

Tolerances count roundings: an output's own (half a step: 2^-8 of a bf16 value, 2^-24 of an fp32 one) and those of the
arithmetic, in units of U = 2^-23 (an fp32 addition on the matrix cores need not round to nearest, so a whole step each)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -23
BF, FP = torch.bfloat16, torch.float32
HALF = {BF: 2.0 ** -8, FP: 2.0 ** -24}
NAN, INF = float("nan"), float("inf")


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


def _within(got, exact, tol, what=""):
    """got against exact (fp64) elementwise; where exact is not finite the same value is wanted."""
    got = got.double()
    fine = torch.isfinite(exact)
    assert torch.equal(torch.isnan(got), torch.isnan(exact)), what
    assert torch.equal(got[~fine & ~torch.isnan(exact)], exact[~fine & ~torch.isnan(exact)]), what
    off = ((got - exact).abs() / tol.clamp(min=1e-300))[fine]
    off = torch.where((got - exact).abs()[fine] == 0, torch.zeros_like(off), off)
    assert off.numel() == 0 or float(off.max()) <= 1.0, (what, float(off.max()))


# ------------------------------------------------------------------------------------------------------------- rotary

SCALINGS = [None, {"type": "linear", "factor": 4.0}, {"type": "ntk", "factor": 2.5},
            {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_context": 8192},
            {"type": "yarn", "factor": 4.0, "original_context": 4096}]


def _pairs(dim, interleaved):
    i = torch.arange(dim // 2, device=DEV)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + dim // 2)


def _rotary64(plan, x, pos, transpose=False):
    """(turned, bound of the fp32 arithmetic's error)"""
    y = x.double().clone(memory_format=torch.contiguous_format)
    a = pos.double()[..., None] * plan.inv_freq
    a = a[:, None] if pos.dim() == 2 else a
    c, s = torch.cos(a) * plan.factor, torch.sin(a) * plan.factor * (-1 if transpose else 1)
    i, j = _pairs(plan.rotary_dim, plan.interleaved)
    u, v = y[..., i], y[..., j]
    y[..., i], y[..., j] = u * c - v * s, v * c + u * s
    # the reduced angle (up to pi) rounded to 2^-24, sine and cosine to 2 of their units, factor, product and sum
    tol = torch.zeros_like(y)
    tol[..., i] = tol[..., j] = 8 * 2.0 ** -24 * plan.factor * (u.abs() + v.abs())
    return y, tol


def _check_rotary(plan, x, y, pos, transpose=False, what=""):
    exact, tol = _rotary64(plan, x, pos, transpose)
    _within(y, exact, tol + HALF[x.dtype] * exact.abs(), what)
    assert torch.equal(y[..., plan.rotary_dim:], x[..., plan.rotary_dim:])


@pytest.mark.parametrize("scaling", SCALINGS, ids=lambda s: s["type"] if s else "plain")
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_rotary_turns_as_in_64_bits(ops, dtype, interleaved, scaling):
    print("rotary", dtype, interleaved, scaling, flush=True)
    g = _gen(1)
    plan = ops.RotaryPlan(128, 5e5, interleaved, scaling, DEV)
    q, k = (_randn(g, 2, 37, h, 128, dtype=dtype).transpose(1, 2) for h in (8, 2))
    pos = torch.randint(0, 131072, (2, 37), generator=g, dtype=torch.int32).to(DEV)
    a, b = ops.rotary(plan, q, k, pos)
    assert a.is_contiguous() and b.is_contiguous()
    _check_rotary(plan, q, a, pos)
    _check_rotary(plan, k, b, pos)
    a, b = ops.rotary(plan, q, k, pos, transpose=True)
    _check_rotary(plan, q, a, pos, True)
    _check_rotary(plan, k, b, pos, True)


@pytest.mark.parametrize("d,rd", [(2, 2), (8, 4), (64, 64), (64, 32), (80, 80), (96, 64), (100, 36), (128, 96), (256, 256), (320, 256)])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_rotary_head_widths(ops, dtype, d, rd):
    print("rotary width", dtype, d, rd, flush=True)
    g = _gen(d + rd)
    for interleaved in (False, True):
        plan = ops.RotaryPlan(rd, 1e4, interleaved, None, DEV)
        for b, h, s in ((1, 1, 1), (3, 5, 17), (1, 40, 33)):
            q = _randn(g, b, h, s, d, dtype=dtype)
            pos = torch.arange(1000, 1000 + s, dtype=torch.int32, device=DEV)
            y = ops.rotary(plan, q, None, pos)
            _check_rotary(plan, q, y, pos, what=(b, h, s, interleaved))
            assert torch.equal(y, ops.rotary(plan, q, None, 1000))


def test_rotary_places_and_strides(ops):
    """In place, into a view of a cache, from a fused projection, rows that are not 16-byte aligned, positions shared and
    far, and nothing at all."""
    print("rotary places", flush=True)
    g = _gen(3)
    plan = ops.RotaryPlan(64, 1e4, False, None, DEV)
    for dtype in (BF, FP):
        qkv = _randn(g, 2, 9, 6 + 2 + 2, 64, dtype=dtype)
        q, k = qkv[:, :, :6].transpose(1, 2), qkv[:, :, 6:8].transpose(1, 2)
        pos = torch.tensor([0, 1, 2, 7, -5, 2 ** 31 - 1, 4, -2 ** 31, 100], dtype=torch.int32, device=DEV)
        wide = _randn(g, 2, 2, 20, 64, dtype=dtype)
        kept = wide.clone()
        a, b = ops.rotary(plan, q, k, pos)
        _check_rotary(plan, q, a, pos)
        c, into = ops.rotary(plan, q, k, pos, out=(torch.empty_like(a), wide[:, :, 5:14]))
        assert torch.equal(c, a) and torch.equal(into, b)
        assert torch.equal(wide[:, :, 5:14], b)
        wide[:, :, 5:14] = kept[:, :, 5:14]
        assert torch.equal(wide, kept)          # nothing beside the view was written
        before = qkv.clone()
        ops.rotary(plan, q, k, pos, out=(q, k))  # in place
        assert torch.equal(q, a) and torch.equal(k, b) and torch.equal(qkv[:, :, 8:], before[:, :, 8:])
        # rows that begin two or four bytes into a piece
        odd = _randn(g, 2 * 3 * 5 * 65 + 1, dtype=dtype)[1:].view(2, 3, 5, 65)[..., :64]
        y = ops.rotary(plan, odd, None, torch.arange(5, dtype=torch.int32, device=DEV))
        _check_rotary(plan, odd, y, torch.arange(5, dtype=torch.int32, device=DEV))
        same = pos[None].expand(2, 9)            # one row for all sequences
        assert torch.equal(ops.rotary(plan, q, None, same), ops.rotary(plan, q, None, pos))
        assert ops.rotary(plan, q[:, :, :0], None, 5).shape == (2, 6, 0, 64)
    # a turn and its transpose give back f^2 x
    plan = ops.RotaryPlan(64, 1e4, True, {"type": "yarn", "factor": 8.0, "original_context": 100, "attention_factor": 0.5}, DEV)
    x = _randn(g, 1, 3, 50, 64)
    back = ops.rotary(plan, ops.rotary(plan, x, None, 77), None, 77, transpose=True)
    # (each turn within 8 units of |u| + |v| <= 2 max|x|)
    assert float((back.double() - 0.25 * x.double()).abs().max()) <= 2 * 0.25 * 16 * 2.0 ** -24 * 2 * float(x.abs().max())


def test_rotary_transpose_is_the_gradient(ops):
    """<turn(x), w> = <x, turn^T(w)>, against the formula and against differences of it (the turn is linear, so a
    difference over any step is the derivative)."""
    print("rotary gradient", flush=True)
    g = _gen(4)
    for interleaved in (False, True):
        plan = ops.RotaryPlan(32, 1e4, interleaved, {"type": "yarn", "factor": 4.0, "original_context": 64}, DEV)
        x, w = _randn(g, 1, 2, 7, 48), _randn(g, 1, 2, 7, 48)
        grad = ops.rotary(plan, w, None, 90, transpose=True)
        y = x.double().requires_grad_()
        a = (90 + torch.arange(7, device=DEV)).double()[:, None] * plan.inv_freq
        i, j = _pairs(32, interleaved)
        u, v = y[..., i], y[..., j]
        c, s = torch.cos(a) * plan.factor, torch.sin(a) * plan.factor
        value = ((u * c - v * s) * w.double()[..., i]).sum() + ((v * c + u * s) * w.double()[..., j]).sum() + (y * w.double())[..., 32:].sum()
        value.backward()
        bound = 8 * 2.0 ** -24 * plan.factor * 2 * float(w.abs().max()) + 2.0 ** -24 * float(y.grad.abs().max())
        assert float((grad.double() - y.grad).abs().max()) <= bound
        step = torch.zeros_like(x)
        step[0, 1, 3, 5] = 1.0
        moved = ((ops.rotary(plan, x + step, None, 90).double() - ops.rotary(plan, x, None, 90).double()) * w.double()).sum()
        # x + step and both turns are rounded: three times 8 units of two elements around 4, times w
        assert abs(float(moved - grad.double()[0, 1, 3, 5])) <= 3 * 8 * 2.0 ** -24 * 2 * 10 * plan.factor * float(w.abs().max())


def test_rotary_refusals(ops):
    plan = ops.RotaryPlan(64, 1e4, False, None, DEV)
    q, k = torch.zeros(2, 4, 3, 64, device=DEV), torch.zeros(2, 2, 3, 64, device=DEV)
    pos = torch.zeros(3, dtype=torch.int32, device=DEV)
    for bad in (lambda: ops.rotary(plan, q.half(), None, pos), lambda: ops.rotary(plan, q.cpu(), None, pos),
                lambda: ops.rotary(plan, q, k.bfloat16(), pos), lambda: ops.rotary(plan, q, k[:, :, :2], pos),
                lambda: ops.rotary(plan, q[..., :32], None, pos), lambda: ops.rotary(plan, q, k, pos.long()),
                lambda: ops.rotary(plan, q, k, pos[:2]), lambda: ops.rotary(plan, q, k, 2 ** 31 - 2),
                lambda: ops.rotary(plan, q.transpose(2, 3).contiguous().transpose(2, 3), None, pos),
                lambda: ops.rotary(plan, q, k, pos, out=(q,)), lambda: ops.rotary(plan, q, k, pos, out=(q, k.bfloat16())),
                lambda: ops.rotary(plan, q[:, 1:], None, pos, out=q[:, :3]),
                lambda: ops.rotary(plan, q, None, pos, out=torch.zeros(1, 1, 1, 64, device=DEV).expand(2, 4, 3, 64)),
                lambda: ops.rotary(plan, q, k, torch.zeros(6, dtype=torch.int32, device=DEV)[::2])):
        with pytest.raises(ValueError):
            bad()


# --------------------------------------------------------------------------------------------------- tree attention

def _tree64(q, kc, vc, kn, vn, mask, lengths, scale):
    """(out, lse, tolerance of out, of lse) in fp64.  Where a masked token or one behind the length holds something that is
    not finite, it is not met."""
    b, hq, t, d = q.shape
    hc, hn = kc.shape[1], kn.shape[1]
    out = torch.zeros((b, hq, t, d), dtype=torch.float64, device=q.device)
    lse = torch.full((b, hq, t), -INF, dtype=torch.float64, device=q.device)
    tol, tol_l = torch.zeros_like(out), torch.zeros_like(lse)
    mask = mask.bool().expand(b, t, t)
    for i in range(b):
        m = kc.shape[2] if lengths is None else min(max(int(lengths[i]), 0), kc.shape[2])
        sees = torch.cat((torch.ones((t, m), dtype=torch.bool, device=q.device), mask[i]), 1)
        for h in range(hq):
            k = torch.cat((kc[i, h * hc // hq, :m], kn[i, h * hn // hq])).double()
            v = torch.cat((vc[i, h * hc // hq, :m], vn[i, h * hn // hq])).double()
            x = q[i, h].double()
            s = torch.where(sees, x @ k.T * scale, -INF)
            s = torch.where(sees, s, -INF)
            # products of d elements summed in fp32, the exponent rounded, the exponential 2 units
            ds = U * ((d + 4) * scale * torch.where(sees, x.abs() @ k.abs().nan_to_num(0, 0, 0).T, 0).amax(-1) + 4)
            top = s.amax(-1, keepdim=True)
            top = torch.where(top == -INF, 0.0, top)
            p = torch.exp(s - top)
            l = p.sum(-1, keepdim=True)
            some = l[:, 0] != 0
            w = torch.where(l > 0, p / l, torch.where(l == 0, 0.0, NAN))
            odd = ~torch.isfinite(v)
            o = w @ torch.where(odd, 0.0, v)
            for j in torch.nonzero(odd.any(-1))[:, 0].tolist():   # (0 times infinity is not met where it is not seen)
                o = o + torch.where(sees[:, j:j + 1] & odd[j], v[j], 0.0)
            out[i, h] = o
            lse[i, h] = torch.where(some, (top + torch.log(l))[:, 0], -INF)
            # numerator and denominator: the exponents, the sums (m + t addends, joined over waves and splits), and a bf16
            # probability's 16 bits, or 8 (half a step of the numerator's and of the denominator's) beyond 128 queries a head
            few = hq // hc * t <= 128
            each = 2 * ds + U * (m + t + 64) * 2 + (0.0 if q.dtype == FP else 2.0 ** -16 if few else 2 * HALF[BF])
            mag = w.nan_to_num(0) @ torch.where(odd, 0.0, v.abs())
            tol[i, h] = each[:, None] * mag + HALF[q.dtype] * o.nan_to_num(0, 0, 0).abs()
            tol_l[i, h] = ds + U * (m + t + 64) + 4 * U * lse[i, h].nan_to_num(0, 0, 0).abs()
    return out, lse, tol, tol_l


def _tree_inputs(seed, dtype, b, hq, hc, hn, t, n, d, density=0.5):
    g = _gen(seed)
    q = _randn(g, b, hq, t, d, dtype=dtype, scale=2.5)
    kc, vc = (_randn(g, b, hc, n, d, dtype=dtype) for _ in range(2))
    kn, vn = (_randn(g, b, hn, t, d, dtype=dtype) for _ in range(2))
    mask = (torch.rand((b, t, t), generator=g) < density).to(DEV)
    return q, kc, vc, kn, vn, mask


def _check_tree(ops, q, kc, vc, kn, vn, mask, lengths=None, scale=None, what=""):
    out, lse = ops.tree_attention(q, kc, vc, kn, vn, mask, lengths, scale, return_lse=True)
    e, el, tol, tol_l = _tree64(q, kc, vc, kn, vn, mask, lengths, q.shape[-1] ** -0.5 if scale is None else scale)
    _within(out, e, tol, what)
    _within(lse, el, tol_l, what)
    return out, lse


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("t,hq,hc,hn", [(1, 1, 1, 1), (1, 32, 8, 8), (3, 8, 8, 2), (7, 28, 4, 4), (16, 8, 2, 1), (33, 6, 2, 2), (64, 8, 2, 2),
                                        (100, 7, 1, 1)])
def test_tree_attention_rows(ops, dtype, t, hq, hc, hn):
    """One query to hundreds a head, dense caches and one per query head; lengths that end in every part of a tile."""
    print("tree rows", dtype, t, hq, hc, hn, flush=True)
    for n in (1, 31, 32, 33, 100, 700):
        q, kc, vc, kn, vn, mask = _tree_inputs(n + t, dtype, 2, hq, hc, hn, t, n, 128)
        lengths = torch.tensor([n, n // 2], dtype=torch.int32, device=DEV)
        _check_tree(ops, q, kc, vc, kn, vn, mask, lengths, what=n)


@pytest.mark.parametrize("d", [4, 8, 16, 24, 32, 40, 64, 80, 96, 128, 136, 200, 256])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_tree_attention_head_widths(ops, dtype, d):
    print("tree width", dtype, d, flush=True)
    from lrqk_amd import _lib
    for t, n in ((1, 65), (5, 300), (40, 77)):
        args = _tree_inputs(d + t, dtype, 1, 4, 2, 2, t, n, d)
        if d * dtype.itemsize % 16:
            with pytest.raises(_lib.LrqkError):
                ops.tree_attention(*args)
            continue
        _check_tree(ops, *args, what=(t, n))


def test_tree_attention_long_cache_and_splits(ops):
    print("tree long", flush=True)
    for dtype, b, hq, hc, t, n in ((BF, 1, 8, 2, 1, 20000), (BF, 3, 4, 1, 25, 9001), (FP, 1, 8, 2, 9, 5003), (BF, 2, 16, 16, 4, 2112)):
        q, kc, vc, kn, vn, mask = _tree_inputs(t, dtype, b, hq, hc, 1, t, n, 128)
        lengths = torch.tensor([n, 1, n - 33][:b], dtype=torch.int32, device=DEV)
        a = _check_tree(ops, q, kc, vc, kn, vn, mask, lengths, what=(n, t))
        z = ops.tree_attention(q, kc, vc, kn, vn, mask, lengths, return_lse=True)
        assert torch.equal(a[0], z[0]) and torch.equal(a[1], z[1])   # the same bits every time


@pytest.mark.parametrize("dtype", [BF, FP])
def test_tree_attention_masks(ops, dtype):
    """Masks of a tree, of nothing, shared by all sequences, of bytes; empty caches; rows that see nothing at all."""
    print("tree masks", dtype, flush=True)
    q, kc, vc, kn, vn, _ = _tree_inputs(5, dtype, 3, 4, 2, 2, 13, 50, 64)
    tree = torch.tril(torch.ones((13, 13), dtype=torch.bool, device=DEV))
    none = torch.zeros((13, 13), dtype=torch.bool, device=DEV)
    for lengths in (None, torch.tensor([50, 0, 7], dtype=torch.int32, device=DEV), torch.tensor([0, 0, 0], dtype=torch.int32, device=DEV),
                    torch.tensor([-3, 1000, 50], dtype=torch.int32, device=DEV)):   # (lengths are cut to the cache)
        for mask in (tree, none, torch.eye(13, dtype=torch.bool, device=DEV), torch.stack((tree, none, ~tree)),
                     tree.to(torch.uint8) * 255, tree.T):
            _check_tree(ops, q, kc, vc, kn, vn, mask, lengths)
    out, lse = ops.tree_attention(q, kc, vc, kn, vn, none, torch.zeros(3, dtype=torch.int32, device=DEV), return_lse=True)
    assert not out.any() and bool((lse == -INF).all())
    _check_tree(ops, q, kc[:, :, :0], vc[:, :, :0], kn, vn, tree)      # no cache at all
    assert ops.tree_attention(q, kc, vc, kn, vn, tree, scale=0.3).shape == q.shape
    _check_tree(ops, q, kc, vc, kn, vn, tree, scale=0.3)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_tree_attention_does_not_meet_what_is_masked(ops, dtype):
    """Infinities and NaN in drafted tokens that a query does not see, and behind the lengths; where it sees them they are
    in its result."""
    print("tree poison", dtype, flush=True)
    for t, hq, hc, d in ((9, 4, 2, 128), (40, 4, 1, 64), (9, 4, 4, 32), (9, 2, 1, 256)):
        q, kc, vc, kn, vn, _ = _tree_inputs(t, dtype, 2, hq, hc, 1, t, 70, d)
        lengths = torch.tensor([70, 37], dtype=torch.int32, device=DEV)
        kc[1, :, 37:], vc[1, :, 37:] = NAN, INF
        mask = torch.tril(torch.ones((t, t), dtype=torch.bool, device=DEV)).repeat(2, 1, 1)
        mask[:, :, 3] = False
        kn[:, :, 3], vn[:, :, 3] = NAN, NAN
        kn[1, :, 5], mask[1, :, 5] = INF, False
        out, _ = _check_tree(ops, q, kc, vc, kn, vn, mask, lengths)
        assert bool(torch.isfinite(out).all())
        # V of token 6 is seen by the tokens from 6 on
        vn[0, :, 6, 0], vn[0, :, 6, 1], vn[0, :, 6, 2], vn[0, :, 7, 2], vn[1, :, 6, d - 1] = INF, -INF, INF, -INF, NAN
        out, _ = _check_tree(ops, q, kc, vc, kn, vn, mask, lengths)
        assert bool(torch.isfinite(out[:, :, :6]).all()) and bool((out[0, :, 6:, 0] == INF).all())
        assert bool((out[0, :, 6:, 1] == -INF).all()) and bool(torch.isnan(out[0, :, 7:, 2]).all())
        assert bool(torch.isnan(out[1, :, 6:, d - 1]).all())


def test_tree_attention_places_and_strides(ops):
    """A cache that is a part of a wider one, the [K|V] store's rows, heads behind each other's rows, a transposed query,
    and sums that pass 32 bits of elements."""
    print("tree strides", flush=True)
    g = _gen(8)
    q, kc, vc, kn, vn, mask = _tree_inputs(8, BF, 2, 8, 2, 2, 6, 90, 128)
    ref = ops.tree_attention(q, kc, vc, kn, vn, mask)
    wide_k, wide_v = (torch.full((2, 2, 200, 128), NAN, dtype=BF, device=DEV) for _ in range(2))
    wide_k[:, :, 40:130], wide_v[:, :, 40:130] = kc, vc
    assert torch.equal(ops.tree_attention(q, wide_k[:, :, 40:130], wide_v[:, :, 40:130], kn, vn, mask), ref)
    store = torch.cat((kc, vc), -1)
    assert torch.equal(ops.tree_attention(q, store[..., :128], store[..., 128:], kn, vn, mask), ref)
    by_token = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, kc, vc, kn, vn)]
    assert torch.equal(ops.tree_attention(*by_token, mask), ref)
    assert torch.equal(ops.tree_attention(q, kc[:1].expand(2, -1, -1, -1), vc[:1].expand(2, -1, -1, -1), kn, vn, mask)[0], ref[0])
    # head 1 of a cache begins beyond 2^31 elements, 2^32 bytes
    big = torch.empty((1, 2, 2 ** 31 // 128 + 8, 128), dtype=BF, device=DEV)
    big[:, :, -90:] = kc[:1]
    tail = big[:, :, -90:]
    out = ops.tree_attention(q[:1], tail, tail, kn[:1], vn[:1], mask[:1])
    assert torch.equal(out, ops.tree_attention(q[:1], kc[:1], kc[:1], kn[:1], vn[:1], mask[:1]))
    del big, tail
    assert ops.tree_attention(q[:, :, :0], kc, vc, kn[:, :, :0], vn[:, :, :0], mask[:, :0, :0]).shape == (2, 8, 0, 128)
    _randn(g, 1)


def test_tree_attention_refusals(ops):
    from lrqk_amd import _lib
    q, kc, vc, kn, vn, mask = _tree_inputs(1, BF, 1, 4, 2, 2, 3, 40, 64)
    for bad in (lambda: ops.tree_attention(q.half(), kc, vc, kn, vn, mask), lambda: ops.tree_attention(q, kc.float(), vc, kn, vn, mask),
                lambda: ops.tree_attention(q.cpu(), kc, vc, kn, vn, mask), lambda: ops.tree_attention(q, kc, vc, kn, vn, mask.cpu()),
                lambda: ops.tree_attention(q, kc, vc, kn, vn, mask.float()), lambda: ops.tree_attention(q, kc, vc, kn, vn, mask[:, :2]),
                lambda: ops.tree_attention(q[:, :3], kc, vc, kn, vn, mask), lambda: ops.tree_attention(q, kc, vc[:, :, :39], kn, vn, mask),
                lambda: ops.tree_attention(q, kc, vc, kn, vn, mask, scale=0.0), lambda: ops.tree_attention(q, kc, vc, kn, vn, mask, scale=-1.0),
                lambda: ops.tree_attention(q, kc, vc, kn, vn, mask, scale=NAN), lambda: ops.tree_attention(q, kc, vc, kn[..., :32], vn, mask),
                lambda: ops.tree_attention(q, kc, vc, kn, vn, mask, torch.zeros(1, device=DEV)),
                lambda: ops.tree_attention(q, kc, vc, kn, vn, mask, torch.zeros(2, dtype=torch.int32, device=DEV)),
                lambda: ops.tree_attention(q, kc, vc.transpose(1, 2).contiguous().transpose(1, 2), kn, vn, mask),
                lambda: ops.tree_attention(q, kc.transpose(2, 3).contiguous().transpose(2, 3), vc, kn, vn, mask),
                lambda: ops.tree_attention(q, torch.zeros(2 * 40 * 64 + 1, dtype=BF, device=DEV)[1:].view(1, 2, 40, 64), vc, kn, vn, mask)):
        with pytest.raises(ValueError):
            bad()
    z = torch.zeros((1, 1, 1025, 64), dtype=BF, device=DEV)
    with pytest.raises(_lib.LrqkError):
        ops.tree_attention(z, z, z, z, z, torch.zeros((1025, 1025), dtype=torch.bool, device=DEV))
    z = torch.zeros((1, 1, 2, 264), dtype=BF, device=DEV)
    with pytest.raises(_lib.LrqkError):
        ops.tree_attention(z, z, z, z, z, torch.zeros((2, 2), dtype=torch.bool, device=DEV))


# ------------------------------------------------------------------------------------------------ attention weights

def _weights64(q, k, lengths, lse, scale, weights):
    """(sums, tolerance) in fp64"""
    b, hq, t, d = q.shape
    hc, n = k.shape[1], k.shape[2]
    out = torch.zeros((b, hc, n), dtype=torch.float64, device=q.device) if weights is None else weights.double()
    tol = 2.0 ** -24 * out.abs()
    for i in range(b):
        m = n if lengths is None else min(max(int(lengths[i]), 0), n)
        sees = torch.arange(m, device=q.device) <= m - t + torch.arange(t, device=q.device)[:, None]
        for h in range(hq):
            x, y = q[i, h].double(), k[i, h * hc // hq, :m].double()
            s = torch.where(sees, x @ y.T * scale, -INF)
            ds = U * ((d + 4) * scale * (torch.where(sees, x.abs() @ y.abs().T, 0).amax(-1) if m else 0.0) + 4)
            own = torch.logsumexp(s, -1) if m else torch.full((t,), -INF, device=q.device, dtype=torch.float64)
            at = own if lse is None else lse[i, h].double()
            p = torch.where(sees & (at != -INF)[:, None], torch.exp(s - torch.where(at == -INF, 0.0, at)[:, None]), 0.0)
            out[i, h * hc // hq, :m] += p.sum(0)
            # the exponent (scores, and their lse of as many addends where it is formed here), rounded at its magnitude, and the sum
            big = torch.where(at == -INF, 0.0, at).abs()
            each = ds + (ds + U * (m + 64) if lse is None else 0.0) + 4 * U * (1 + big)
            tol[i, h * hc // hq, :m] += (p * each[:, None]).sum(0) + U * (64 + t // 64) * p.sum(0)
            # fp32 has no normal number below 2^-126: each of the t exponentials below it is off by that at most, being 0 instead
            tol[i, h * hc // hq, :m] += t * 2.0 ** -126
    return out, tol + 2.0 ** -24 * out.abs()


def _check_weights(ops, q, k, lengths=None, lse=None, scale=None, weights=None, what=""):
    w0 = None if weights is None else weights.clone()
    got = ops.attention_weights(q, k, lengths, lse, scale, weights, out=None if weights is None else torch.empty_like(weights))
    exact, tol = _weights64(q, k, lengths, lse, q.shape[-1] ** -0.5 if scale is None else scale, w0)
    _within(got, exact, tol, what)
    if weights is not None:
        assert torch.equal(weights, w0)
        same = ops.attention_weights(q, k, lengths, lse, scale, w0)
        assert same is w0 and torch.equal(w0, got)     # in place, and the same bits
    return got


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("t,n", [(1, 1), (1, 70), (2, 2), (15, 40), (16, 64), (17, 17), (33, 500), (100, 100), (257, 257), (300, 900)])
def test_attention_weights_sizes(ops, dtype, t, n):
    """Whole prompts and last tokens, with the logarithms of the sums given and formed."""
    print("weights", dtype, t, n, flush=True)
    g = _gen(t + n)
    for hq, hc in ((4, 4), (8, 2), (7, 1)):
        q, k = _randn(g, 2, hq, t, 128, dtype=dtype, scale=2.0), _randn(g, 2, hc, n, 128, dtype=dtype)
        total = _check_weights(ops, q, k)
        # a query's attention adds up to one
        assert float((total.double().sum((1, 2)) - hq * t).abs().max()) <= hq * t * 1e-3
        lengths = torch.tensor([n, max(1, n // 2)], dtype=torch.int32, device=DEV)   # (shorter than t: its first queries see nothing)
        _check_weights(ops, q, k, lengths)
        lse = _randn(g, 2, hq, t) + 6.0
        lse[0, 0, 0] = -INF
        w = torch.rand((2, hc, n), generator=g).to(DEV)
        _check_weights(ops, q, k, lengths, lse, weights=w)
        _check_weights(ops, q, k, None, None, 0.2, w)


@pytest.mark.parametrize("d", [8, 16, 32, 48, 64, 96, 128, 200, 256])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_attention_weights_head_widths(ops, dtype, d):
    print("weights width", dtype, d, flush=True)
    g = _gen(d)
    for t, n in ((3, 90), (70, 70)):
        _check_weights(ops, _randn(g, 1, 4, t, d, dtype=dtype), _randn(g, 1, 2, n, d, dtype=dtype), what=(t, n))


def test_attention_weights_long_and_strided(ops):
    print("weights long", flush=True)
    g = _gen(9)
    for dtype, t, n in ((BF, 5, 20001), (BF, 1500, 1500), (FP, 40, 4100), (BF, 1, 9000)):
        _check_weights(ops, _randn(g, 1, 4, t, 128, dtype=dtype, scale=2.0), _randn(g, 1, 2, n, 128, dtype=dtype), what=(t, n))
    q, store = _randn(g, 2, 4, 6, 64, dtype=BF), _randn(g, 2, 2, 100, 128, dtype=BF)
    store[:, :, 80:] = NAN     # behind the lengths
    lengths = torch.tensor([80, 0], dtype=torch.int32, device=DEV)
    got = ops.attention_weights(q, store[..., :64], lengths)
    assert torch.equal(got, ops.attention_weights(q, store[..., :64].contiguous(), lengths))
    assert not got[1].any() and not got[0, :, 80:].any() and bool(torch.isfinite(got).all())
    # a key that later queries alone see does not spoil the earlier ones' sums
    q, k = _randn(g, 1, 2, 40, 64), _randn(g, 1, 1, 40, 64)
    k[:, :, 39] = NAN
    lse = torch.full((1, 2, 40), 5.0, device=DEV)
    got = ops.attention_weights(q, k, lse=lse)
    assert bool(torch.isfinite(got[..., :39]).all()) and bool(torch.isnan(got[..., 39]).all())


def test_attention_weights_take_the_attention_lse(ops):
    """What tree_attention leaves makes the same sums as they are formed here."""
    print("weights lse", flush=True)
    q, kc, vc, kn, vn, _ = _tree_inputs(3, BF, 2, 8, 2, 2, 6, 400, 128)
    tree = torch.tril(torch.ones((6, 6), dtype=torch.bool, device=DEV))
    lse = ops.tree_attention(q, kc, vc, kn, vn, tree, return_lse=True)[1]
    k = torch.cat((kc, kn), 2)
    _check_weights(ops, q, k, None, lse)
    a, b = ops.attention_weights(q, k), ops.attention_weights(q, k, lse=lse)
    _, tol = _weights64(q, k, None, None, 128 ** -0.5, None)
    _within(a, b.double(), 2 * tol)


def test_attention_weights_refusals(ops):
    from lrqk_amd import _lib
    q, k = torch.zeros(1, 4, 3, 64, device=DEV), torch.zeros(1, 2, 9, 64, device=DEV)
    w = torch.zeros(1, 2, 9, device=DEV)
    for bad in (lambda: ops.attention_weights(q.half(), k.half()), lambda: ops.attention_weights(q, k.bfloat16()),
                lambda: ops.attention_weights(q[:, :3], k), lambda: ops.attention_weights(q, k.cpu()),
                lambda: ops.attention_weights(q, k, lse=torch.zeros(1, 4, 2, device=DEV)), lambda: ops.attention_weights(q, k, scale=0.0),
                lambda: ops.attention_weights(q, k, weights=w[..., :8]), lambda: ops.attention_weights(q, k, weights=w.double()),
                lambda: ops.attention_weights(q, k, out=torch.zeros(1, 2, 18, device=DEV)[..., ::2]),
                lambda: ops.attention_weights(q, k, weights=torch.zeros(19, device=DEV)[:18].view(1, 2, 9),
                                              out=torch.zeros(19, device=DEV)[1:].view(1, 2, 9)[..., :8])):
        with pytest.raises(ValueError):
            bad()
    base = torch.zeros(19, device=DEV)
    with pytest.raises(ValueError):
        ops.attention_weights(q, k, weights=base[:18].view(1, 2, 9), out=base[1:].view(1, 2, 9))
    with pytest.raises(_lib.LrqkError):
        ops.attention_weights(q[..., :3].contiguous(), k[..., :3].contiguous())


# ----------------------------------------------------------------------------------------------------------- eviction

def _evict64(weights, ids, lengths, budget, recent):
    """(lengths, per head the slots whose tokens the first slots get) on the CPU"""
    b, h, n = weights.shape
    src, new = {}, []
    for i in range(b):
        m = n if lengths is None else min(max(int(lengths[i]), 0), n)
        keep = min(m, budget)
        new.append(keep)
        for j in range(h):
            w, c = weights[i, j, :m].double().tolist(), ids[i, j, :m].tolist()
            last = max(c, default=0)
            new_one = [c[s] > last - recent for s in range(m)]   # (ids that repeat may make them more than the budget: lowest slots)
            rank = [(0, 0, 0.0, s) if new_one[s] else (1, 0, 0.0, s) if w[s] != w[s] else (2, -w[s], 0.0, s) for s in range(m)]
            stay = {r[3] for r in sorted(rank)[:keep]}
            late = iter(sorted(s for s in stay if s >= keep))
            src[i, j] = [s if s in stay else next(late) for s in range(keep)]
    return new, src


def _check_evict(ops, weights, ids, k, v, lengths, budget, recent, what=""):
    held = (weights, ids, k, v)
    new, src = _evict64(weights.cpu(), ids.cpu(), None if lengths is None else lengths.cpu(), budget, recent)
    want = [x.clone() for x in held]
    room = min(budget, k.shape[2]) + 3
    out = [torch.full((*x.shape[:2], room, *x.shape[3:]), 7, dtype=x.dtype, device=DEV) for x in held]
    want_out = [x.clone() for x in out]
    for (i, j), s in src.items():
        s = torch.tensor(s, dtype=torch.int64, device=DEV)
        for x, y, z in zip(held, want, want_out):
            y[i, j, :len(s)] = x[i, j][s]
            z[i, j, :len(s)] = x[i, j][s]

    def same(xs, ys):
        return all(torch.equal(x.view(torch.int32) if x.dtype == FP else x.view(torch.int16) if x.dtype == BF else x,
                               y.view(torch.int32) if y.dtype == FP else y.view(torch.int16) if y.dtype == BF else y) for x, y in zip(xs, ys))
    before = [x.clone() for x in held]
    got = ops.evict(*held, lengths, budget, recent, out=tuple(out))
    assert got.dtype == torch.int32 and got.tolist() == new, what
    assert same(out, want_out), what
    assert same(held, before), what
    got = ops.evict(*held, lengths, budget, recent)
    assert got.tolist() == new and same(held, want), what


def _cache(g, b, h, n, d, dtype):
    return (torch.rand((b, h, n), generator=g).to(DEV), torch.arange(n, dtype=torch.int32).repeat(b, h, 1).to(DEV),
            _randn(g, b, h, n, d, dtype=dtype), _randn(g, b, h, n, d, dtype=dtype))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("n,budget,recent", [(1, 1, 0), (1, 1, 1), (2, 1, 1), (5, 8, 2), (64, 64, 8), (65, 64, 8), (100, 10, 10), (300, 1, 0),
                                             (1000, 999, 0), (1025, 512, 32), (5000, 4096, 64), (9000, 100, 16), (70000, 3000, 7)])
def test_evict_sizes(ops, dtype, n, budget, recent):
    print("evict", dtype, n, budget, recent, flush=True)
    g = _gen(n)
    for d in (16, 128):
        _check_evict(ops, *_cache(g, 2, 2, n, d, dtype), torch.tensor([n, max(0, n - n // 3)], dtype=torch.int32, device=DEV), budget, recent)
    _check_evict(ops, *_cache(g, 1, 3, n, 24, dtype), None, budget, recent)


def test_evict_ties_and_odd_values(ops):
    """Equal weights everywhere, weights of a few values, NaN, infinities, zeros of both signs, negative ones; ids in any
    order, ids that repeat, all of them new."""
    print("evict ties", flush=True)
    g = _gen(2)
    n = 6000
    w, ids, k, v = _cache(g, 1, 4, n, 8, BF)
    lengths = torch.tensor([n - 5], dtype=torch.int32, device=DEV)
    _check_evict(ops, torch.zeros_like(w), ids, k, v, lengths, 777, 0)
    _check_evict(ops, torch.ones_like(w), ids, k, v, lengths, 777, 50)
    _check_evict(ops, (w * 4).floor(), ids, k, v, lengths, 3000, 5)
    odd = torch.randn((1, 4, n), generator=g).to(DEV)
    odd[..., ::7], odd[..., 1::7], odd[..., 2::7] = 0.0, -0.0, NAN
    odd[..., 3::70], odd[..., 4::70] = INF, -INF
    odd[0, 0, 5::7] = torch.tensor(-NAN)
    for budget in (100, 860, 2000, 5000):
        _check_evict(ops, odd.clone(), ids.clone(), k.clone(), v.clone(), lengths, budget, 40, what=budget)
    mixed = ids.gather(2, torch.rand((1, 4, n), generator=g).argsort(-1).to(DEV)) * 5 - 9000
    _check_evict(ops, w.clone(), mixed, k.clone(), v.clone(), lengths, 1000, 400)
    _check_evict(ops, w.clone(), torch.zeros_like(ids), k.clone(), v.clone(), lengths, 1000, 1)
    _check_evict(ops, w.clone(), torch.full_like(ids, -2 ** 31), k.clone(), v.clone(), lengths, 1000, 1)
    _check_evict(ops, w.clone(), torch.full_like(ids, 2 ** 31 - 1), k.clone(), v.clone(), lengths, 1000, 0)
    for odd_length in (0, -4, n + 10, 777, 778):
        _check_evict(ops, w.clone(), ids.clone(), k.clone(), v.clone(), torch.tensor([odd_length], dtype=torch.int32, device=DEV), 777, 7)
    _check_evict(ops, w, ids, k, v, lengths, 2 ** 31 - 1, 2 ** 31 - 1)


def test_evict_refusals(ops):
    from lrqk_amd import _lib
    w, ids, k, v = _cache(_gen(0), 1, 2, 20, 64, BF)
    n = torch.tensor([20], dtype=torch.int32, device=DEV)
    out = (torch.zeros(1, 2, 9, device=DEV), torch.zeros(1, 2, 9, dtype=torch.int32, device=DEV), k[:, :, :9].clone(), v[:, :, :9].clone())
    for bad in (lambda: ops.evict(w, ids, k, v, n, 0, 0), lambda: ops.evict(w, ids, k, v, n, 5, 6), lambda: ops.evict(w, ids, k, v, n, 5, -1),
                lambda: ops.evict(w.double(), ids, k, v, n, 5, 1), lambda: ops.evict(w, ids.long(), k, v, n, 5, 1),
                lambda: ops.evict(w, ids, k, v.float(), n, 5, 1), lambda: ops.evict(w, ids, k[:, :, ::2], v[:, :, ::2], n, 5, 1),
                lambda: ops.evict(w, ids, k.cpu(), v, n, 5, 1), lambda: ops.evict(w, ids, k, v, n.float(), 5, 1),
                lambda: ops.evict(w, ids, k, v, n, 10, 1, out=out), lambda: ops.evict(w, ids, k, v, n, 9, 1, out=(w, ids, k, v)),
                lambda: ops.evict(w, ids, k, v, n, 9, 1, out=out[:3]), lambda: ops.evict(w, ids, k.half(), v.half(), n, 5, 1)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(_lib.LrqkError):
        ops.evict(w, ids, k[..., :5].contiguous(), v[..., :5].contiguous(), n, 5, 1)


# ----------------------------------------------------------------------------------------------------------- more sizes

@pytest.mark.parametrize("b", [65, 150])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_tree_attention_many_sequences(ops, dtype, b):
    """More sequences than a wave has lanes, lengths of every kind: the splits' places are counted over all of them."""
    print("tree many", dtype, b, flush=True)
    lengths = torch.randint(0, 600, (b,), generator=_gen(b), dtype=torch.int32)
    lengths[::7], lengths[3::11] = 0, 600
    lengths = lengths.to(DEV)
    for t, hq in ((2, 2), (20, 2)):
        q, kc, vc, kn, vn, mask = _tree_inputs(b, dtype, b, hq, 1, 1, t, 600, 32)
        _check_tree(ops, q, kc, vc, kn, vn, mask, lengths, what=t)
    _check_tree(ops, q, kc, vc, kn, vn, mask, None)


@pytest.mark.parametrize("t,hq", [(16, 1), (17, 1), (8, 4), (11, 3), (32, 2), (13, 5), (32, 4), (43, 3)])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_tree_attention_at_the_kernels_borders(ops, dtype, t, hq):
    """16 and 17, 32 and 33, 64 and 65, 128 and 129 queries a cache head."""
    print("tree borders", dtype, t, hq, flush=True)
    for d in (64, 256):
        q, kc, vc, kn, vn, mask = _tree_inputs(t, dtype, 2, hq, 1, 1, t, 333, d)
        _check_tree(ops, q, kc, vc, kn, vn, mask, torch.tensor([333, 160], dtype=torch.int32, device=DEV), what=d)


def test_tree_attention_refuses_rows_too_far_apart(ops):
    from lrqk_amd import _lib
    q, _, _, kn, vn, mask = _tree_inputs(1, BF, 1, 1, 1, 1, 2, 1, 8)
    far = torch.empty(2 ** 24 + 16, dtype=BF, device=DEV).as_strided((1, 1, 2, 8), (0, 0, 2 ** 24 + 8, 1))
    with pytest.raises(_lib.LrqkError):
        ops.tree_attention(q, far, far, kn, vn, mask)


@pytest.mark.parametrize("t,hq", [(16, 1), (17, 1), (16, 2), (11, 3), (16, 4), (13, 5), (40, 4)])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_attention_weights_at_the_kernels_borders(ops, dtype, t, hq):
    """16 and 17, 32 and 33, 64 and 65 queries a cache head, with the sums of the attention and without."""
    print("weights borders", dtype, t, hq, flush=True)
    g = _gen(t)
    for d in (32, 64, 128, 256):
        q, k = _randn(g, 2, 2 * hq, t, d, dtype=dtype, scale=2.0), _randn(g, 2, 2, 300, d, dtype=dtype)
        lengths = torch.tensor([300, 20], dtype=torch.int32, device=DEV)
        _check_weights(ops, q, k, lengths, what=d)
        _check_weights(ops, q, k, lengths, lse=_randn(g, 2, 2 * hq, t) + 3.0, weights=torch.rand((2, 2, 300), generator=g).to(DEV), what=d)


def test_attention_weights_far_rows(ops):
    """Rows and heads whose distances pass 32 bits of elements."""
    print("weights far", flush=True)
    g = _gen(11)
    step, n = 2 ** 24 + 64, 150
    place = torch.empty(step * n + 2 ** 32 + 128, dtype=BF, device=DEV)
    for strides in ((0, 64, step, 1), (0, 2 ** 32 + 64, 64, 1)):
        k = place.as_strided((1, 2, n, 64), strides)
        k.copy_(_randn(g, 1, 2, n, 64, dtype=BF))
        for t in (3, 40):
            q = _randn(g, 1, 4, t, 64, dtype=BF, scale=2.0)
            assert torch.equal(ops.attention_weights(q, k), ops.attention_weights(q, k.contiguous()))
            _check_weights(ops, q, k)


@pytest.mark.parametrize("n", [4095, 4096, 4097, 12288, 12289, 32768, 32769])
def test_evict_lengths_around_the_kernels_borders(ops, n):
    print("evict borders", n, flush=True)
    g = _gen(n)
    for over in (127, 128, 129, n // 2):
        _check_evict(ops, *_cache(g, 1, 2, n, 8, BF), None, n - over, 30, what=over)
    _check_evict(ops, *_cache(g, 2, 1, n, 16, FP), torch.tensor([n, n - 100], dtype=torch.int32, device=DEV), n - 128, 0)


def test_evict_writes_the_lengths_in_place(ops):
    """The library's own entry with the new lengths in the place of the old ones, many tokens over the budget and few."""
    from lrqk_amd import _lib
    print("evict aliased", flush=True)
    lib, g = _lib.load(), _gen(4)
    for n, budget in ((1000, 900), (1000, 300)):
        held = _cache(g, 3, 2, n, 16, BF)
        lengths = torch.tensor([n, 500, budget - 1], dtype=torch.int32, device=DEV)
        want = [x.clone() for x in held]
        new = ops.evict(*want, lengths, budget, 9)
        need = lib.lrqk_evict_workspace(3, 2, n, budget)
        ws = torch.empty(need, dtype=torch.uint8, device=DEV)
        rc = lib.lrqk_evict(*(x.data_ptr() for x in held), lengths.data_ptr(), n, None, None, None, None, n, lengths.data_ptr(), 3, 2, 16,
                            budget, 9, ws.data_ptr(), need, _lib.BF16, torch.cuda.current_stream().cuda_stream)
        assert rc == 0 and torch.equal(lengths, new)
        assert all(torch.equal(x, y) for x, y in zip(held, want))


def test_evict_far_rows(ops):
    """A head of more than 2^31 elements: tokens that move from behind them, one by one and many."""
    print("evict far", flush=True)
    n, d = 2 ** 23 + 200, 256
    g = _gen(6)
    order = torch.randperm(n, generator=g)
    weights = order.float().to(DEV).view(1, 1, n)                  # (distinct, and exact in fp32)
    ids = torch.arange(n, dtype=torch.int32, device=DEV).view(1, 1, n)
    k = torch.empty((1, 1, n, d), dtype=BF, device=DEV)
    marks = (torch.arange(n, device=DEV) % 251).to(BF)
    k.copy_(marks[None, None, :, None].expand(1, 1, n, d))
    v = -k
    for budget, in_place in ((1000, False), (n - 100, True)):
        slots = torch.arange(n)
        top = torch.where(slots >= n - 8, n + slots, order)        # the 8 newest come first
        stay = torch.zeros(n, dtype=torch.bool)
        stay[top.topk(budget).indices] = True
        source = slots[:budget].clone()
        source[~stay[:budget]] = slots[budget:][stay[budget:]]
        source = source.to(DEV)
        want = weights[0, 0, source], ids[0, 0, source], marks[source]
        if in_place:
            out = weights, ids, k, v
            assert ops.evict(*out, None, budget, 8).tolist() == [budget]
        else:
            out = tuple(torch.empty((1, 1, budget, *x.shape[3:]), dtype=x.dtype, device=DEV) for x in (weights, ids, k, v))
            assert ops.evict(weights, ids, k, v, None, budget, 8, out=out).tolist() == [budget]
        assert torch.equal(out[0][0, 0, :budget], want[0]) and torch.equal(out[1][0, 0, :budget], want[1])
        for i in (0, 127, d - 1):
            assert torch.equal(out[2][0, 0, :budget, i], want[2]) and torch.equal(out[3][0, 0, :budget, i], -want[2])


# ------------------------------------------------------------------------------------------------------- all of them

def _tree_of(parents):
    """(depths, mask) of a tree whose token i follows token parents[i] (-1: the cache)"""
    t = len(parents)
    depth, mask = [0] * t, torch.eye(t, dtype=torch.bool)
    for i, p in enumerate(parents):
        if p >= 0:
            depth[i] = depth[p] + 1
            mask[i] |= mask[p]
    return torch.tensor(depth, dtype=torch.int32), mask


class _Budgeted:
    """One layer's cache as a decoder of drafted tokens holds it."""

    def __init__(self, b, hc, room, d, dtype):
        self.k, self.v = (torch.zeros((b, hc, room, d), dtype=dtype, device=DEV) for _ in range(2))
        self.weights = torch.zeros((b, hc, room), device=DEV)
        self.ids = torch.zeros((b, hc, room), dtype=torch.int32, device=DEV)
        self.lengths = torch.zeros(b, dtype=torch.int32, device=DEV)     # tokens that are held
        self.seen = torch.zeros(b, dtype=torch.int32, device=DEV)        # tokens that there were

    def append(self, paths, k_new, v_new):
        """The drafted tokens ``paths[i]`` of sequence i, in order."""
        for i, p in enumerate(paths):
            n, s, m = int(self.lengths[i]), int(self.seen[i]), len(p)
            self.k[i, :, n:n + m], self.v[i, :, n:n + m] = k_new[i][:, p], v_new[i][:, p]
            self.ids[i, :, n:n + m] = torch.arange(s, s + m, dtype=torch.int32, device=DEV)
            self.weights[i, :, n:n + m] = 0.0
            self.lengths[i] += m
            self.seen[i] += m


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("hq,hc,d,rd", [(8, 2, 128, 128), (6, 6, 64, 32), (4, 1, 96, 96)])
def test_a_decoder_of_drafts_over_a_budget(ops, dtype, hq, hc, d, rd):
    """Prompt, then rounds of: turn the drafts, attend, accept a path of each sequence, add its attention up, evict.  Every
    call is held to its formula in 64 bits on what it was given."""
    print("together", dtype, hq, hc, d, flush=True)
    b, budget, recent, prompt = 3, 60, 10, 75
    g = _gen(d)
    plan = ops.RotaryPlan(rd, 1e4, False, {"type": "yarn", "factor": 4.0, "original_context": 64}, DEV)
    cache = _Budgeted(b, hc, 100, d, dtype)

    def heads(t):
        return [_randn(g, b, t, h, d, dtype=dtype, scale=s).transpose(1, 2) for h, s in ((hq, 2.0), (hc, 1.0), (hc, 1.0))]

    # the prompt is a tree without branches over an empty cache; its keys are turned into their slots
    q, k, v = heads(prompt)
    q1, k1 = ops.rotary(plan, q, k, 0, out=(torch.empty((b, hq, prompt, d), dtype=dtype, device=DEV), cache.k[:, :, :prompt]))
    for x, y in ((q, q1), (k, k1)):
        _check_rotary(plan, x, y, torch.arange(prompt, dtype=torch.int32, device=DEV))
    chain = torch.ones((prompt, prompt), dtype=torch.bool, device=DEV).tril()
    out, lse = _check_tree(ops, q1, cache.k, cache.v, k1, v, chain, cache.lengths)
    cache.append([list(range(prompt))] * b, k1, v)
    cache.weights = _check_weights(ops, q1, cache.k, cache.lengths, lse, weights=cache.weights)
    # what a column of the attention matrix adds up to in all is the number of rows
    assert torch.allclose(cache.weights.sum(-1), torch.full((b, hc), float(prompt * hq // hc), device=DEV), rtol=1e-4)
    held = cache.weights, cache.ids, cache.k, cache.v
    _check_evict(ops, *held, cache.lengths, budget, recent)                       # (ends in place)
    cache.lengths = torch.full((b,), budget, dtype=torch.int32, device=DEV)
    for step, (parents, paths) in enumerate((([-1, 0, 0, 1, 1, 2, -1, 6], ([0, 1, 4], [6], [0, 2, 5])), ([-1], ([0], [0], [0])),
                                             ([-1, -1, 1, 2, 3, 4], ([0], [1, 2, 3, 4, 5], [1])),
                                             ([-1, 0, 1, 2, 0, 4, 4, -1, 7, 8, 9, 10], ([0, 1, 2, 3], [7, 8, 9, 10, 11], [0, 4, 6])))):
        t = len(parents)
        depth, mask = _tree_of(parents)
        q, k, v = heads(t)
        pos = cache.seen[:, None] + depth.to(DEV)
        q1, k1 = ops.rotary(plan, q, k, pos)
        _check_rotary(plan, q, q1, pos)
        _check_rotary(plan, k, k1, pos)
        out, lse = _check_tree(ops, q1, cache.k, cache.v, k1, v, mask.to(DEV), cache.lengths, what=step)
        cache.append(paths, k1, v)
        # the accepted queries are the sequences' last tokens: shorter paths lie right in a block of the longest, and what is
        # in front of them has sums of -inf and adds nothing
        most = max(map(len, paths))
        q_last, lse_last = torch.full((b, hq, most, d), NAN, dtype=dtype, device=DEV), torch.full((b, hq, most), -INF, device=DEV)
        for i, p in enumerate(paths):
            q_last[i, :, most - len(p):], lse_last[i, :, most - len(p):] = q1[i][:, p], lse[i][:, p]
        q_clean = q_last.nan_to_num(0)
        got = _check_weights(ops, q_clean, cache.k, cache.lengths, lse_last, weights=cache.weights.clone())
        before = cache.weights.sum(-1)
        assert ops.attention_weights(q_last, cache.k, cache.lengths, lse_last, weights=cache.weights) is cache.weights
        assert torch.equal(cache.weights, got)
        gained = torch.tensor([[len(p) * hq / hc] for p in paths], device=DEV)
        assert torch.allclose(cache.weights.sum(-1) - before, gained.expand(b, hc), rtol=1e-3)
        held = cache.weights, cache.ids, cache.k, cache.v
        old = cache.lengths
        _check_evict(ops, *held, old, budget, recent)
        cache.lengths = old.clamp(max=budget)


def test_accepted_drafts_attend_as_a_whole_sequence(ops):
    """Chains of drafts, accepted one after another, have what causal attention over the whole sequence gives, and their
    tokens' sums are its columns'; all from the unturned inputs in 64 bits."""
    print("whole sequence", flush=True)
    b, hq, hc, d, total = 1, 4, 2, 64, 60
    g = _gen(12)
    plan = ops.RotaryPlan(64, 1e4, True, None, DEV)
    q, k, v = (_randn(g, b, h, total, d) for h in (hq, hc, hc))
    cache = _Budgeted(b, hc, total, d, FP)
    outs, lses, at = [], [], 0
    for m in (30, 1, 7, 1, 16, 5):
        part = slice(at, at + m)
        q1, k1 = ops.rotary(plan, q[:, :, part], k[:, :, part], at)
        tree = torch.ones((m, m), dtype=torch.bool, device=DEV).tril()
        out, lse = ops.tree_attention(q1, cache.k, cache.v, k1, v[:, :, part].contiguous(), tree, cache.lengths, return_lse=True)
        cache.append([list(range(m))], k1, v[:, :, part])
        ops.attention_weights(q1, cache.k, cache.lengths, lse, weights=cache.weights)
        outs.append(out)
        lses.append(lse)
        at += m
    pos = torch.arange(total, dtype=torch.int32, device=DEV)
    (q64, eq), (k64, ek) = _rotary64(plan, q, pos), _rotary64(plan, k, pos)
    # the turned rows' roundings reach the scores, and the exponents, through the products with the other side
    eq, ek = eq + HALF[FP] * q64.abs(), ek + HALF[FP] * k64.abs()
    causal = torch.ones((total, total), dtype=torch.bool, device=DEV).tril()
    for h in range(hq):
        x, y, z = q64[0, h], k64[0, h * hc // hq], v[0, h * hc // hq].double()
        s = torch.where(causal, x @ y.T * d ** -0.5, -INF)
        ds = d ** -0.5 * (eq[0, h] @ y.abs().T + x.abs() @ ek[0, h * hc // hq].T + U * (d + 4) * (x.abs() @ y.abs().T)).amax(-1) + 4 * U
        p = torch.softmax(s, -1)
        tol = (2 * ds + U * 2 * (total + 64))[:, None] * (p @ z.abs()) + HALF[FP] * (p @ z).abs()
        _within(torch.cat(outs, 2)[0, h], p @ z, tol, h)
        lse = torch.logsumexp(s, -1)
        _within(torch.cat(lses, 2)[0, h], lse, ds + U * (total + 64) + 4 * U * lse.abs(), h)
    for hh in range(hc):
        exact, tol = 0.0, 0.0
        for h in range(hh * hq // hc, (hh + 1) * hq // hc):
            x, y = q64[0, h], k64[0, hh]
            s = torch.where(causal, x @ y.T * d ** -0.5, -INF)
            ds = d ** -0.5 * (eq[0, h] @ y.abs().T + x.abs() @ ek[0, hh].T + U * (d + 4) * (x.abs() @ y.abs().T)).amax(-1) + 4 * U
            p, lse = torch.softmax(s, -1), torch.logsumexp(s, -1)
            exact = exact + p.sum(0)
            tol = tol + (p * (2 * ds + U * (total + 64) + 8 * U * (1 + lse.abs()))[:, None]).sum(0) + U * 80 * p.sum(0)
        _within(cache.weights[0, hh], exact, tol, hh)


def _round(ops, plan, q, k, v, mask, cache):
    """A round on fixed buffers, as it is captured: all drafts are accepted, and the cache goes to other buffers."""
    t = q.shape[2]
    pos = cache["seen"][:, None] + torch.arange(t, dtype=torch.int32, device=DEV)
    q1, k1 = ops.rotary(plan, q, k, pos)
    out, lse = ops.tree_attention(q1, cache["k"], cache["v"], k1, v, mask, cache["lengths"], return_lse=True)
    at = (cache["lengths"][:, None] + torch.arange(t, device=DEV))[:, None]
    rows = at[..., None].expand(-1, k.shape[1], -1, k.shape[3]).long()
    cache["k"].scatter_(2, rows, k1)
    cache["v"].scatter_(2, rows, v)
    cache["ids"].scatter_(2, rows[..., 0], pos[:, None].expand(-1, k.shape[1], -1))
    cache["weights"].scatter_(2, rows[..., 0], torch.zeros_like(rows[..., 0], dtype=torch.float32))
    cache["lengths"] += t
    cache["seen"] += t
    ops.attention_weights(q1, cache["k"], cache["lengths"], lse, weights=cache["weights"])
    cache["lengths"].copy_(ops.evict(cache["weights"], cache["ids"], cache["k"], cache["v"], cache["lengths"], 900, 16))
    return out


def _start(g, dtype, b=2, hc=2, room=1024, d=64):
    weights, ids, k, v = _cache(g, b, hc, room, d, dtype)
    return {"weights": weights, "ids": ids, "k": k, "v": v, "lengths": torch.tensor([890, 300], dtype=torch.int32, device=DEV),
            "seen": torch.tensor([890, 300], dtype=torch.int32, device=DEV)}


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("t,hq", [(1, 2), (5, 8), (40, 8)])
def test_rounds_replayed_from_graphs(ops, dtype, t, hq):
    """Two captured rounds, replayed in turn with the lengths growing, an eager round of a third cache between the replays:
    the same bits as eager rounds."""
    print("graphs", dtype, t, hq, flush=True)
    g = _gen(t)
    plan = ops.RotaryPlan(64, 1e4, False, None, DEV)
    mask = torch.ones((t, t), dtype=torch.bool, device=DEV).tril()

    def inputs():
        return [_randn(g, 2, h, t, 64, dtype=dtype) for h in (hq, 2, 2)]
    caches = [_start(g, dtype) for _ in range(2)]
    eager = [{n: x.clone() for n, x in c.items()} for c in caches]
    third = _start(g, dtype)
    fixed = [inputs() for _ in range(2)]
    scrap = _start(g, dtype)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _round(ops, plan, *fixed[0], mask, scrap)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for x, c in zip(fixed, caches):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_round(ops, plan, *x, mask, c))
        graphs.append(graph)
    for _ in range(5):
        for x, e, c, graph, out in zip(fixed, eager, caches, graphs, outs):
            new = inputs()
            for a, z in zip(x, new):
                a.copy_(z)
            graph.replay()
            _round(ops, plan, *inputs(), mask, third)
            torch.cuda.synchronize()
            want = _round(ops, plan, *new, mask, e)
            assert torch.equal(out, want)
            assert all(torch.equal(c[n], e[n]) for n in c)


def test_two_streams_at_once(ops):
    """The same calls on two streams at once and on one after the other have the same bits."""
    print("streams", flush=True)
    g = _gen(30)
    plan = ops.RotaryPlan(64, 1e4, False, None, DEV)
    t = 12
    mask = torch.ones((t, t), dtype=torch.bool, device=DEV).tril()
    x = [[_randn(g, 2, h, t, 64, dtype=BF) for h in (8, 2, 2)] for _ in range(2)]
    caches = [_start(g, BF) for _ in range(2)]
    alone = [{n: y.clone() for n, y in c.items()} for c in caches]
    want = [[_round(ops, plan, *x[i], mask, alone[i]) for _ in range(6)] for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(_round(ops, plan, *x[i], mask, caches[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(got[i], want[i]))
        assert all(torch.equal(caches[i][n], alone[i][n]) for n in alone[i])


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("t", [4, 16, 64, 200])
def test_attention_weights_of_queries_that_saw_nothing(ops, dtype, t):
    """Sums of -inf beside ordinary ones: such queries add nothing, NaN and infinities in them included."""
    print("weights none", dtype, t, flush=True)
    g = _gen(t)
    q, k = _randn(g, 2, 4, t, 64, dtype=dtype, scale=2.0), _randn(g, 2, 2, 500, 64, dtype=dtype)
    lse = _randn(g, 2, 4, t) + 3.0
    none = (torch.rand((2, 4, t), generator=g) < 0.2).to(DEV)
    none[1] = True
    lse = torch.where(none, -INF, lse)
    lengths = torch.tensor([500, 440], dtype=torch.int32, device=DEV)
    want = _check_weights(ops, q, k, lengths, lse)
    assert not want[1].any()
    for odd in (NAN, INF):
        assert torch.equal(ops.attention_weights(torch.where(none[..., None], torch.tensor(odd, dtype=dtype, device=DEV), q), k, lengths, lse), want)
    k[1] = NAN
    assert torch.equal(ops.attention_weights(q, k, lengths, lse), want)


def test_rotary_refuses_one_place_for_both(ops):
    plan = ops.RotaryPlan(64, 1e4, False, None, DEV)
    q, y = torch.zeros(1, 2, 3, 64, device=DEV), torch.zeros(1, 2, 3, 64, device=DEV)
    with pytest.raises(ValueError):
        ops.rotary(plan, q, q, 0, out=(q, q))
    with pytest.raises(ValueError):
        ops.rotary(plan, q, q.clone(), 0, out=(y, y))


@pytest.mark.parametrize("n", [32769, 36864, 36865, 100000])
def test_evict_longer_than_a_workgroup(ops, n):
    """Heads that several workgroups look through: ties over all of them, sequences of every length beside each other, the
    newest tokens anywhere."""
    print("evict wide", n, flush=True)
    g = _gen(n)
    w, ids, k, v = _cache(g, 3, 2, n, 8, BF)
    lengths = torch.tensor([n, 0, n - 4097], dtype=torch.int32, device=DEV)
    ids = ids.gather(2, torch.rand((3, 2, n), generator=g).argsort(-1).to(DEV))
    for budget, recent in ((1, 0), (2112, 64), (n // 2, 5000), (n - 1, 1), (n + 5, 3)):
        for x in (w, (w * 3).floor(), torch.zeros_like(w)):
            held = [y.clone() for y in (x, ids, k, v)]
            _check_evict(ops, *held, lengths, budget, recent, what=(budget, recent))
    odd = w.clone()
    odd[:, :, ::3], odd[:, :, 1::3] = NAN, -INF
    _check_evict(ops, odd, ids, k, v, None, n // 2, 100)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("t,hq", [(3, 2), (40, 1), (70, 2)])
def test_scores_that_rise_and_fall(ops, dtype, t, hq):
    """Scores that rise from tile to tile, fall, lie far below zero or jump once: the running maximum is found wherever it
    is looked for, by both operators."""
    print("scores", dtype, t, hq, flush=True)
    n, d = 1200, 64
    q, kc, vc, kn, vn, mask = _tree_inputs(9, dtype, 1, hq, 1, 1, t, n, d)
    q[..., 0] = 1.0
    for name, ramp in (("rise", torch.linspace(-300, 300, n)), ("fall", torch.linspace(300, -300, n)), ("low", torch.full((n,), -5000.0)),
                       ("high", torch.full((n,), 5000.0)), ("jump", torch.where(torch.arange(n) == 777, 900.0, -900.0))):
        k = kc.clone()
        k[..., 0] = ramp.to(DEV).to(dtype)
        for scale in (1.0, 0.125):
            out, _ = _check_tree(ops, q, k, vc, kn, vn, mask, scale=scale, what=(name, scale))
            assert bool(torch.isfinite(out).all())
            _check_weights(ops, q, k, scale=scale, what=(name, scale))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("b,hq,hk,s,d,rd", [(1, 1, 0, 300, 16, 16), (2, 3, 1, 130, 64, 48), (1, 70, 2, 9, 256, 256), (1, 8, 8, 257, 256, 256),
                                            (2, 300, 20, 5, 128, 128), (1, 2, 2, 4097, 8, 8)])
def test_rotary_over_many_tiles(ops, dtype, b, hq, hk, s, d, rd):
    """Tiles of one token to 64, the last one not whole."""
    print("rotary tiles", dtype, b, hq, hk, s, d, flush=True)
    g = _gen(s)
    for interleaved in (False, True):
        plan = ops.RotaryPlan(rd, 1e4, interleaved, None, DEV)
        q, k = _randn(g, b, s, hq, d, dtype=dtype).transpose(1, 2), _randn(g, b, hk, s, d, dtype=dtype) if hk else None
        pos = torch.randint(0, 100000, (b, s), generator=g, dtype=torch.int32).to(DEV)
        y = ops.rotary(plan, q, k, pos)
        for x, z in zip((q, k), y) if hk else ((q, y),):
            _check_rotary(plan, x, z, pos, what=interleaved)


@pytest.mark.parametrize("dtype,d", [(BF, 128), (BF, 64), (BF, 24), (FP, 64), (FP, 128)])
def test_attention_weights_of_many_products(ops, dtype, d):
    """Where a wave takes 64 keys at a time: many tokens over a long cache."""
    print("weights many", dtype, d, flush=True)
    g = _gen(d)
    q, k = _randn(g, 1, 32, 2050, d, dtype=dtype, scale=2.0), _randn(g, 1, 8, 10007, d, dtype=dtype)
    lengths = torch.tensor([10001], dtype=torch.int32, device=DEV)
    for lse in (None, _randn(g, 1, 32, 2050) + 6.0):
        _check_weights(ops, q, k, lengths, lse, weights=torch.rand((1, 8, 10007), generator=g).to(DEV))


@pytest.mark.parametrize("d", [8, 32, 48, 64, 128, 200, 256])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_tree_attention_of_every_kernel_and_width(ops, dtype, d):
    """10, 30, 60, 120 and 150 queries a cache head at every width, lengths that end in a tile."""
    print("tree all", dtype, d, flush=True)
    for t, hq in ((5, 2), (15, 2), (30, 2), (60, 2), (50, 3)):
        q, kc, vc, kn, vn, mask = _tree_inputs(d + t, dtype, 2, hq, 1, 1, t, 470, d)
        _check_tree(ops, q, kc, vc, kn, vn, mask, torch.tensor([467, 75], dtype=torch.int32, device=DEV), what=t)


@pytest.mark.parametrize("t", [1, 3, 4, 5, 7, 8, 9, 12, 31, 32, 33, 63, 65, 127, 257])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_tree_masks_of_odd_lengths(ops, dtype, t):
    """A row of the mask begins anywhere and ends in the middle of a quad's keys: every byte of it counts at its place."""
    print("tree odd masks", dtype, t, flush=True)
    for hq in (1, 6):
        for density in (0.05, 0.9):
            q, kc, vc, kn, vn, mask = _tree_inputs(t, dtype, 2, hq, 1, 1, t, 20, 32, density)
            _check_tree(ops, q, kc, vc, kn, vn, mask, torch.tensor([0, 13], dtype=torch.int32, device=DEV), what=(hq, density))
            _check_tree(ops, q, kc, vc, kn, vn, mask[1], None, what=(hq, density))


def test_strides_of_one_sequence_or_head_do_not_count(ops):
    """K and V of one sequence out of batches of different sizes, of one head out of different ones, of one token."""
    print("tree single strides", flush=True)
    q, kc, vc, kn, vn, mask = _tree_inputs(2, BF, 1, 4, 2, 2, 3, 40, 32)
    ref = ops.tree_attention(q, kc, vc, kn, vn, mask)
    wide = torch.zeros((40, 2, 80, 32), dtype=BF, device=DEV)
    wide = wide.as_strided((1, 2, 40, 32), (8, kc.stride(1), 32, 1))
    wide.copy_(vc)
    assert torch.equal(ops.tree_attention(q, kc, wide, kn, vn, mask), ref)
    one = torch.zeros((1, 3, 40, 32), dtype=BF, device=DEV)[:, 1:2].copy_(vc[:, :1])
    assert torch.equal(ops.tree_attention(q[:, :2], kc[:, :1], one, kn[:, :1], vn[:, :1], mask), ref[:, :2])
    with pytest.raises(ValueError):
        ops.tree_attention(q, kc, torch.cat((vc, vc), 3)[..., :32], kn, vn, mask)


def test_evict_refuses_one_place_for_k_and_v(ops):
    w, ids, k, v = _cache(_gen(0), 1, 1, 20, 16, BF)
    out = [x[:, :, :8].clone() for x in (w, ids, k)]
    with pytest.raises(ValueError):
        ops.evict(w, ids, k, v, None, 8, 2, out=(*out, out[2]))


def test_the_long_forms_replayed_from_a_graph(ops):
    """A prompt's weights, wide drafts and the eviction of a long head, captured together and replayed with other inputs and
    lengths, eager work between the replays."""
    print("graph, long forms", flush=True)
    g = _gen(77)
    n, t = 40000, 200
    mask = torch.ones((t, t), dtype=torch.bool, device=DEV).tril()
    q, k, v = _randn(g, 2, 4, t, 64, dtype=BF), _randn(g, 2, 2, t, 64, dtype=BF), _randn(g, 2, 2, t, 64, dtype=BF)
    w, ids, kc, vc = _cache(g, 2, 2, n, 64, BF)
    lengths = torch.tensor([n, n - 3000], dtype=torch.int32, device=DEV)
    out = [torch.zeros((2, 2, 2112, *x.shape[3:]), dtype=x.dtype, device=DEV) for x in (w, ids, kc, vc)]

    def work():
        a, lse = ops.tree_attention(q, kc, vc, k, v, mask, lengths, return_lse=True)
        prompt = ops.attention_weights(q, k)
        ops.attention_weights(q, kc, lengths, lse, weights=w)
        new = ops.evict(w, ids, kc, vc, lengths, 2112, 64, out=tuple(out))
        return a, lse, prompt, new
    kept = w.clone()
    work()
    w.copy_(kept)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    for i in range(4):
        q.copy_(_randn(g, 2, 4, t, 64, dtype=BF))
        lengths.copy_(torch.tensor([n - 1000 * i, 2000 + 9000 * i], dtype=torch.int32))
        w.copy_(kept)
        graph.replay()
        torch.cuda.synchronize()
        replayed = [x.clone() for x in (*got, w, *out)]
        w.copy_(kept)
        eager = (*work(), w, *out)
        torch.cuda.synchronize()
        keep = [min(int(m), 2112) for m in lengths]
        for x, y in zip(replayed[:5], eager[:5]):
            assert torch.equal(x, y)
        for x, y in zip(replayed[5:], eager[5:]):
            assert all(torch.equal(x[b, :, :keep[b]], y[b, :, :keep[b]]) for b in range(2))


def test_rotary_refuses_outputs_that_overlap(ops):
    """An input turned in place while the other one is read from the same memory, outputs shifted into each other, an output
    over the positions."""
    plan = ops.RotaryPlan(64, 1e4, False, None, DEV)
    q, k = torch.zeros(1, 2, 3, 64, device=DEV), torch.zeros(1, 2, 3, 64, device=DEV)
    flat, fresh = torch.zeros(2 * 384, device=DEV), torch.zeros(1, 2, 3, 64, device=DEV)
    low, high = flat[:384].view(1, 2, 3, 64), flat[4:388].view(1, 2, 3, 64)
    pos = flat[:3].view(torch.int32)
    for bad in (lambda: ops.rotary(plan, q, q, 0, out=(q, fresh)), lambda: ops.rotary(plan, q, q, 0, out=(fresh, q)),
                lambda: ops.rotary(plan, q, q[:, 1:], 0, out=(q, fresh[:, 1:])), lambda: ops.rotary(plan, q, k, 0, out=(low, high)),
                lambda: ops.rotary(plan, low, k, 0, out=(low, high)), lambda: ops.rotary(plan, q, k, 0, out=(high, low)),
                lambda: ops.rotary(plan, q, None, pos, out=low),
                lambda: ops.rotary(plan, q, None, 0, out=flat.as_strided((1, 2, 3, 64), (384, 64, 32, 1)))):
        with pytest.raises(ValueError):
            bad()


def test_rotary_of_one_projection_in_place(ops):
    """q and k between each other in memory, however the projection lays them out, in place and into each other's kind."""
    print("rotary in one buffer", flush=True)
    g = _gen(31)
    plan = ops.RotaryPlan(64, 1e4, False, None, DEV)
    for layout in ((0, 2, 1, 3), (0, 1, 2, 3), (2, 0, 1, 3)):   # of [b, heads, s, d] in memory
        back = [layout.index(i) for i in range(4)]
        for dtype in (BF, FP):
            x = _randn(g, 2, 7, 9, 64, dtype=dtype).permute(layout).contiguous().permute(back)
            y = torch.zeros_like(x, memory_format=torch.preserve_format)
            a, b = ops.rotary(plan, x[:, :4], x[:, 4:6], 11)
            ops.rotary(plan, x[:, :4], x[:, 4:6], 11, out=(y[:, :4], y[:, 4:6]))
            assert torch.equal(y[:, :4], a) and torch.equal(y[:, 4:6], b) and not y[:, 6].any()
            kept = x[:, 6].clone()
            ops.rotary(plan, x[:, :4], x[:, 4:6], 11, out=(x[:, :4], x[:, 4:6]))
            assert torch.equal(x[:, :4], a) and torch.equal(x[:, 4:6], b) and torch.equal(x[:, 6], kept)


def test_attention_weights_refuse_a_place_that_is_read(ops):
    """The sums over what the kernels still read: queries, keys, lse, lengths; as out and as weights."""
    flat = torch.zeros(4096, device=DEV)
    q, k, lse = flat[:1536].view(1, 4, 6, 64), flat[1536:2688].view(1, 2, 9, 64), flat[2688:2712].view(1, 4, 6)
    lengths = flat[2712:2713].view(torch.int32)
    for at in (0, 1530, 1536, 2680, 2688, 2700, 2712):
        place = flat[at:at + 18].view(1, 2, 9)
        for where in (dict(out=place), dict(weights=place), dict(weights=torch.zeros_like(place), out=place)):
            with pytest.raises(ValueError):
                ops.attention_weights(q, k, lengths, lse, **where)
    free = flat[3000:3018].view(1, 2, 9)
    ops.attention_weights(q, k, lengths, lse, weights=free)
    assert not free.any()   # (no tokens)


def test_evict_refuses_outputs_that_overlap(ops):
    """Outputs shifted into each other, the weights' over the ids', one over the lengths, and in place caches over each other;
    one tensor as keys and values is none of these."""
    print("evict overlaps", flush=True)
    g = _gen(5)
    w, ids, k, v = _cache(g, 1, 2, 20, 64, BF)
    n = torch.tensor([20], dtype=torch.int32, device=DEV)
    flat, rows = torch.zeros(64, device=DEV), torch.zeros(4096, dtype=BF, device=DEV)
    ok = (torch.zeros(1, 2, 9, device=DEV), torch.zeros(1, 2, 9, dtype=torch.int32, device=DEV), k[:, :, :9].clone(), v[:, :, :9].clone())
    low, high = rows[:1152].view(1, 2, 9, 64), rows[64:1216].view(1, 2, 9, 64)
    numbers = flat[9:27].view(torch.int32).view(1, 2, 9)
    for out in ((*ok[:2], low, high), (*ok[:2], high, low), (flat[:18].view(1, 2, 9), numbers, *ok[2:]),
                (flat[18:36].view(1, 2, 9), numbers, *ok[2:]), (rows[:36].view(torch.float32).view(1, 2, 9), ok[1], low, ok[3]),
                (w.view(-1)[3:21].view(1, 2, 9), *ok[1:]), (ok[0], ok[1], k.view(-1)[64:1216].view(1, 2, 9, 64), ok[3])):
        with pytest.raises(ValueError):
            ops.evict(w, ids, k, v, n, 9, 1, out=out)
    with pytest.raises(ValueError):
        ops.evict(w, ids, k, v, numbers.view(-1)[4:5], 9, 1, out=(ok[0], numbers, *ok[2:]))
    both = torch.zeros(2560 + 64, dtype=BF, device=DEV)
    for held in ((w, ids, both[:2560].view(1, 2, 20, 64), both[64:].view(1, 2, 20, 64)), (w, w.view(torch.int32), k, v)):
        with pytest.raises(ValueError):
            ops.evict(*held, n, 9, 1)
    with pytest.raises(ValueError):
        ops.evict(w, ids, k, v, ids.view(-1)[7:8], 9, 1)
    one, apart = [x.clone() for x in (w, ids, k, k)], [x.clone() for x in (w, ids, k, k)]
    one[3] = one[2]
    ops.evict(*one, n, 9, 1)
    ops.evict(*apart, n, 9, 1)
    assert all(torch.equal(x[:, :, :9], y[:, :, :9]) for x, y in zip(one, apart))


@pytest.mark.parametrize("dtype", [BF, FP])
def test_odd_strides_of_a_single_sequence_head_or_token(ops, dtype):
    """A stride that leads to nothing may be anything: no multiple of 16 bytes, or more than rows may be apart."""
    print("single strides", dtype, flush=True)
    for b, h, n in ((1, 2, 40), (2, 1, 40), (2, 2, 1), (1, 1, 40), (1, 2, 1), (1, 1, 1)):
        q, kc, vc, kn, vn, mask = _tree_inputs(b + 2 * h + n, dtype, b, 2 * h, h, h, 3, n, 64)
        odd = tuple(s if m > 1 else far for m, s, far in zip(kc.shape, kc.stride(), (13, 7, (1 << 25) + 1, 1)))
        k, v = kc.as_strided(kc.shape, odd), vc.as_strided(vc.shape, odd)
        assert torch.equal(ops.tree_attention(q, k, v, kn, vn, mask), ops.tree_attention(q, kc, vc, kn, vn, mask))
        lse = torch.full((b, 2 * h, 3), 4.0, device=DEV)
        for given in (None, lse):
            assert torch.equal(ops.attention_weights(q, k, lse=given), ops.attention_weights(q, kc, lse=given))
        plan = ops.RotaryPlan(64, 1e4, False, None, DEV)
        y = torch.empty_like(kc)
        ops.rotary(plan, k, None, 5, out=y.as_strided(y.shape, odd))
        assert torch.equal(y, ops.rotary(plan, kc, None, 5))


@pytest.mark.parametrize("dtype", [BF, FP])
def test_new_rows_that_begin_between_two_pieces(ops, dtype):
    """Queries, keys and values of the new tokens anywhere in a larger buffer."""
    print("odd places", dtype, flush=True)
    q, kc, vc, kn, vn, mask = _tree_inputs(8, dtype, 2, 4, 2, 2, 3, 50, 64)

    def odd(x):
        y = torch.zeros(x.numel() + 1, dtype=x.dtype, device=DEV)[1:].view(x.shape).copy_(x)
        assert y.is_contiguous() and y.data_ptr() % 16
        return y
    for a, b in zip(ops.tree_attention(odd(q), kc, vc, odd(kn), odd(vn), odd(mask), return_lse=True),
                    ops.tree_attention(q, kc, vc, kn, vn, mask, return_lse=True)):
        assert torch.equal(a, b)
    assert torch.equal(ops.attention_weights(odd(q), kc), ops.attention_weights(q, kc))


@pytest.mark.parametrize("b,t", [(2112, 1), (513, 1024)])
def test_attention_weights_of_thousands_of_tiles_in_one_part(ops, b, t):
    """So many heads that each walks over all its keys in one part, 4096 tiles that all add the same number to a lane's sum:
    every addition then rounds the same way, and the error may not grow with the tiles."""
    print("weights, one part", b, t, flush=True)
    n = 131072
    a = torch.linspace(0.02, 1.5, b, dtype=torch.float64).to(BF).to(DEV)   # logit of the first tile; of the others 0
    q, k = torch.zeros((b, 1, t, 8), dtype=BF, device=DEV), torch.zeros((1, 1, n, 8), dtype=BF, device=DEV)
    q[..., 0] = a[:, None, None]
    k[:, :, :32, 0] = 1.0
    got = ops.attention_weights(q, k.expand(b, 1, n, 8), scale=1.0)
    e = a.double().exp()
    seen = torch.arange(n - t + 1, n + 1, dtype=torch.float64, device=DEV)
    each = 1.0 / (32 * e[:, None] + seen - 32)                           # [b,t]: of a key of the later tiles
    # sums of 17 (in units of 2: 2^-19): of base 2 the logarithm 2 units, its sum with the maximum and the exponent half of one;
    # the exponential 2 units of 2^-23.  Additions, half of 2^-23 each: 8 exponentials of a tile, 32 tiles, and 16 of the parts,
    # those of the maximum's change and the waves' lanes; of the columns 8 a tile and as many of the parts.
    tol = math.log(2) * 3 * 2.0 ** -19 + 2 * 2.0 ** -23 + (8 + 32 + 16 + 48) * 2.0 ** -24
    for first in range(0, b, 64):
        w = each[first:first + 64]
        exact = torch.empty((w.shape[0], n), dtype=torch.float64, device=DEV)
        exact[:, :n - t + 1] = w.sum(1, keepdim=True)
        exact[:, n - t:] = w.flip(1).cumsum(1).flip(1)
        exact[:, :32] *= e[first:first + 64, None]
        off = ((got[first:first + 64, 0].double() - exact) / exact).abs().max()
        assert float(off) <= tol, (first, float(off), tol)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("b,t", [(2112, 1), (1030, 33), (1030, 65), (1030, 130)])
def test_tree_attention_of_heads_that_fill_the_gpu(ops, dtype, b, t):
    """So many heads that each could walk over its keys in one part, whose exponentials are all the same number: every addition
    then rounds the same way (the matrix cores cut off), and the error may not grow with the cache."""
    print("tree, one part", dtype, b, t, flush=True)
    n, g = 131072, _gen(t)
    a = torch.linspace(0.02, 1.5, b, dtype=torch.float64).to(BF).to(DEV)   # logit of the first 32 keys; of the others 0
    q, kn = torch.zeros((b, 1, t, 8), dtype=dtype, device=DEV), torch.zeros((b, 1, t, 8), dtype=dtype, device=DEV)
    k, v = torch.zeros((1, 1, n, 8), dtype=dtype, device=DEV), torch.rand((1, 1, n, 8), generator=g).to(dtype).to(DEV)
    q[..., 0], k[:, :, :32, 0], v[..., 0] = a[:, None, None].to(dtype), 1.0, 1.0
    mask = torch.zeros((t, t), dtype=torch.bool, device=DEV)
    out, lse = ops.tree_attention(q, k.expand(b, 1, n, 8), v.expand(b, 1, n, 8), kn, kn, mask, scale=1.0, return_lse=True)
    e = a.double().exp()[:, None]
    total = 32 * e + (n - 32)
    exact = (e * v[0, 0, :32].double().sum(0) + v[0, 0, 32:].double().sum(0)) / total
    # a split has 512 tiles for each 128 queries: a lane adds up so many numbers to one that grows, so that half of them count,
    # half of 2^-23 each, and 8 of a tile, 16 and 64 of the joins
    tiles = 512 * (2 if t > 128 else 1)
    of_sum = (tiles / 2 + 8 + 16 + 64) * 2.0 ** -24
    # log of base 2 (17: a unit is 2^-19), 2 units, its sum with the maximum half of one, times ln 2; the product's rounding
    assert float((lse.double() - total.log()[..., None]).abs().max()) <= of_sum + math.log(2) * 2.5 * 2.0 ** -19 + 2.0 ** -21
    # the product with V: a split's keys, 4 (fp32) or 32 (bf16) a step, each step up to a unit of a sum that grows; bf16 values
    # times two numbers, and the output's rounding
    steps = tiles * (16 / 4 if dtype == FP else 2)
    tol = of_sum + (steps / 2 + 64) * U + (2.0 ** -15 if dtype == BF else 0.0) + (2.0 ** -8 if dtype == BF and t > 128 else 0.0) + HALF[dtype]
    assert float(((out[:, 0].double() - exact[:, None]) / exact[:, None]).abs().max()) <= tol


def test_rotary_in_place_is_held_to_every_rule(ops):
    """Both in place: keys that lie in several heads' or tokens' place, the positions under either, queries and keys shifted."""
    plan = ops.RotaryPlan(64, 1e4, False, None, DEV)
    flat = torch.zeros(2048, device=DEV)
    q, k = flat[:384].view(1, 2, 3, 64), flat[384:768].view(1, 2, 3, 64)
    pos = torch.zeros(3, dtype=torch.int32, device=DEV)
    a, b = ops.rotary(plan, q, k, pos, out=(q, k))
    assert a is q and b is k
    one = flat[1024:1088].view(1, 1, 1, 64).expand(1, 2, 3, 64)
    shifted = flat[380:764].view(1, 2, 3, 64)
    for x, y, p in ((q, one, pos), (one, k, pos), (q, k, flat[382:385].view(torch.int32)), (q, k, flat[3:6].view(torch.int32)), (q, shifted, pos),
                    (shifted, q, pos), (q, q, pos)):
        with pytest.raises(ValueError):
            ops.rotary(plan, x, y, p, out=(x, y))
