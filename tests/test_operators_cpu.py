"""The operators around a drafted, budgeted cache as far as they go without a GPU: the angles of rotary positions, the sizes of
the scratch memory, and every argument that an entry point refuses before it launches anything (the pointers that these
calls are given lead nowhere)."""
import ctypes
import math

import pytest
import torch

from lrqk_amd import _lib, ops

P = 1 << 20   # a pointer, 16-byte aligned
EINVAL, ELIMIT = -1, -3


def _freq(dim, theta, scaling):
    """Angles per position by the definitions, one pair at a time."""
    out = []
    for i in range(dim // 2):
        f = theta ** (-2 * i / dim)
        kind = scaling and scaling["type"]
        if kind == "linear":
            f /= scaling["factor"]
        elif kind == "ntk":
            f = (theta * scaling["factor"] ** (dim / (dim - 2))) ** (-2 * i / dim)
        elif kind == "llama3":
            wave, s = 2 * math.pi / f, scaling["factor"]
            low, high = scaling["original_context"] / scaling["low_freq_factor"], scaling["original_context"] / scaling["high_freq_factor"]
            if wave > low:
                f = f / s
            elif wave > high:
                smooth = (scaling["original_context"] / wave - scaling["low_freq_factor"]) / (
                    scaling["high_freq_factor"] - scaling["low_freq_factor"])
                f = (1 - smooth) * f / s + smooth * f
        elif kind == "yarn":
            def pair(turns):   # the (fractional) pair that turns so often over the original context
                return dim * math.log(scaling["original_context"] / (turns * 2 * math.pi)) / (2 * math.log(theta))
            low, high = max(math.floor(pair(scaling.get("beta_fast", 32.0))), 0), min(math.ceil(pair(scaling.get("beta_slow", 1.0))), dim - 1)
            ramp = min(1.0, max(0.0, (i - low) / max(high - low, 0.001)))
            f = f / scaling["factor"] * ramp + f * (1 - ramp)
        out.append(f)
    return torch.tensor(out, dtype=torch.float64)


@pytest.mark.parametrize("dim,theta", [(128, 5e5), (64, 1e4), (96, 1e6), (4, 1e4), (256, 2.0)])
@pytest.mark.parametrize("scaling", [
    None, {"type": "linear", "factor": 4.0}, {"type": "ntk", "factor": 2.0},
    {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_context": 8192},
    {"type": "yarn", "factor": 4.0, "original_context": 32768},
    {"type": "yarn", "factor": 16.0, "original_context": 4096, "beta_fast": 40.0, "beta_slow": 2.0}])
def test_rotary_frequencies(dim, theta, scaling):
    plan = ops.RotaryPlan(dim, theta, scaling=scaling, device="cpu")
    want = _freq(dim, theta, scaling)
    assert plan.inv_freq.dtype == torch.float64 and plan.inv_freq.shape == (dim // 2,)
    # powers and quotients of 64-bit numbers: some units of 2^-53, times the exponent's magnitude
    assert float(((plan.inv_freq - want) / want).abs().max()) <= 64 * 2.0 ** -53
    factor = 0.1 * math.log(scaling["factor"]) + 1 if scaling and scaling["type"] == "yarn" else 1.0
    assert plan.factor == pytest.approx(factor, abs=1e-15)


def test_rotary_plan_takes_a_given_factor_and_refuses_what_it_does_not_know():
    assert ops.RotaryPlan(64, scaling={"type": "yarn", "factor": 4.0, "original_context": 99, "attention_factor": 1.5}, device="cpu").factor == 1.5
    for bad in (dict(rotary_dim=63), dict(rotary_dim=0), dict(rotary_dim=-2), dict(rotary_dim=258), dict(rotary_dim=64, theta=1.0),
                dict(rotary_dim=64, theta=math.inf), dict(rotary_dim=64, theta=math.nan), dict(rotary_dim=64, scaling={"factor": 2.0}),
                dict(rotary_dim=64, scaling={"type": "dynamic", "factor": 2.0}), dict(rotary_dim=64, scaling={"type": "linear"}),
                dict(rotary_dim=64, scaling={"type": "linear", "factor": 0.5}), dict(rotary_dim=64, scaling={"type": "linear", "factor": math.nan}),
                dict(rotary_dim=64, scaling={"type": "linear", "factor": 2.0, "low": 1}), dict(rotary_dim=2, scaling={"type": "ntk", "factor": 2.0}),
                dict(rotary_dim=64, scaling={"type": "yarn", "factor": 2.0}),
                dict(rotary_dim=64, scaling={"type": "yarn", "factor": 2.0, "original_context": 99, "beta_fast": 1.0, "beta_slow": 2.0}),
                dict(rotary_dim=64, scaling={"type": "yarn", "factor": 2.0, "original_context": 0}),
                dict(rotary_dim=64, scaling={"type": "llama3", "factor": 2.0, "original_context": 99, "low_freq_factor": 4.0, "high_freq_factor": 1.0})):
        with pytest.raises(ValueError):
            ops.RotaryPlan(device="cpu", **bad)


def _call(fn, good, **changed):
    args = dict(good, **changed)
    return getattr(_lib.load(), fn)(*args.values())


ROTARY = dict(q=P, k=P, q_out=P, k_out=P, strides=(ctypes.c_int64 * 12)(*([64] * 12)), positions=P, pos_stride=0, first=0, freq=P,
              factor=1.0, b=1, hq=4, hk=2, s=3, d=64, rotary_dim=64, interleaved=0, transpose=0, dtype=1, stream=None)
TREE = dict(q=P, k_cache=P, v_cache=P, kb=4096, kh=2048, kr=64, n=32, lengths=None, k_new=P, v_new=P, mask=P, mask_b=0, out=P, lse=None,
            b=1, hq=4, hc=2, hn=2, t=3, d=64, scale=0.1, ws=P, ws_bytes=1 << 40, dtype=1, stream=None)
WEIGHTS = dict(q=P, k=P, kb=4096, kh=2048, kr=64, n=32, lengths=None, lse=None, weights=None, out=P, b=1, hq=4, hc=2, t=3, d=64, scale=0.1,
               ws=P, ws_bytes=1 << 40, dtype=1, stream=None)
EVICT = dict(weights=P, ids=P, k=P, v=P, lengths=None, cap=32, weights_out=None, ids_out=None, k_out=None, v_out=None, cap_out=0,
             new_lengths=P, b=1, heads=2, d=64, budget=8, recent=2, ws=P, ws_bytes=1 << 40, dtype=1, stream=None)


@pytest.mark.parametrize("fn,good,code,changed", [
    *(("lrqk_rotary", ROTARY, EINVAL, c) for c in (
        dict(q=None), dict(k=None), dict(q_out=None), dict(k_out=None), dict(strides=None), dict(freq=None), dict(dtype=2), dict(b=0),
        dict(hq=0), dict(hk=-1), dict(s=-1), dict(d=0), dict(rotary_dim=63), dict(rotary_dim=66), dict(rotary_dim=0), dict(b=65536))),
    *(("lrqk_rotary", ROTARY, ELIMIT, c) for c in (dict(hq=70000), dict(s=1 << 31))),
    *(("lrqk_tree_attention", TREE, EINVAL, c) for c in (
        dict(q=None), dict(k_cache=None), dict(v_cache=None), dict(k_new=None), dict(v_new=None), dict(mask=None), dict(out=None),
        dict(ws=None), dict(ws_bytes=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(dtype=5),
        dict(b=0), dict(hq=5), dict(hn=3), dict(hc=0), dict(hn=0), dict(t=0), dict(n=-1), dict(q=P + 2), dict(k_cache=P + 8), dict(v_new=P + 4),
        dict(kr=68), dict(kh=2050), dict(kb=4100), dict(ws=P + 8))),
    *(("lrqk_tree_attention", TREE, ELIMIT, c) for c in (dict(d=60), dict(d=264), dict(t=1025), dict(n=(1 << 30) + 1), dict(b=20000))),
    *(("lrqk_attention_weights", WEIGHTS, EINVAL, c) for c in (
        dict(q=None), dict(k=None), dict(out=None), dict(ws=None), dict(ws_bytes=0), dict(scale=0.0), dict(scale=math.nan), dict(dtype=-1),
        dict(b=0), dict(hq=5), dict(t=0), dict(n=0), dict(q=P + 2), dict(k=P + 8), dict(kr=68))),
    *(("lrqk_attention_weights", WEIGHTS, ELIMIT, c) for c in (dict(d=60), dict(d=264), dict(n=(1 << 30) + 1), dict(b=20000), dict(t=1 << 30))),
    *(("lrqk_evict", EVICT, EINVAL, c) for c in (
        dict(weights=None), dict(ids=None), dict(k=None), dict(v=None), dict(new_lengths=None), dict(ws=None), dict(ws_bytes=0),
        dict(dtype=7), dict(b=0), dict(heads=0), dict(d=0), dict(cap=0), dict(budget=0), dict(recent=9), dict(recent=-1), dict(k=P + 8),
        dict(weights_out=2 * P), dict(weights_out=P, ids_out=2 * P, k_out=2 * P, v_out=2 * P, cap_out=8),
        dict(weights_out=2 * P, ids_out=2 * P, k_out=2 * P, v_out=2 * P, cap_out=7))),
    *(("lrqk_evict", EVICT, ELIMIT, c) for c in (dict(d=60), dict(b=40000), dict(cap=(1 << 30) + 1)))],
    ids=lambda x: x if isinstance(x, str) else ",".join(f"{k}={v}" for k, v in x.items()) if isinstance(x, dict) and len(x) < 9 else "")
def test_entry_points_refuse(fn, good, code, changed):
    assert _call(fn, good, **changed) == code
    assert _lib.load().lrqk_last_error()


def test_scratch_sizes():
    lib = _lib.load()
    assert lib.lrqk_attention_weights_workspace(1, 32, 8, 5, 65536, 128, 1, 1) == 0        # with lse given: none
    assert lib.lrqk_attention_weights_workspace(1, 32, 8, 64, 64, 128, 0, 1) >= 32 * 64 * 4
    assert lib.lrqk_evict_workspace(2, 8, 5000, 100) == 2 * 8 * 100 * 12
    assert lib.lrqk_evict_workspace(2, 8, 100, 5000) == 2 * 8 * 100 * 12
    small, large = (lib.lrqk_tree_attention_workspace(1, 32, 8, t, 131072, 128, 1, 1) for t in (1, 64))
    assert 0 < small <= large < 1 << 30
    for fn, args in (("lrqk_tree_attention_workspace", (0, 32, 8, 1, 10, 128, 1, 1)), ("lrqk_attention_weights_workspace", (1, 32, 7, 1, 10, 128, 1, 1)),
                     ("lrqk_evict_workspace", (1, 1, 0, 1))):
        assert getattr(lib, fn)(*args) == EINVAL


def test_tensors_off_the_gpu_are_refused():
    t = torch.zeros(1, 2, 3, 64)
    plan = ops.RotaryPlan(64, device="cpu")
    for call in (lambda: ops.rotary(plan, t, None, 0), lambda: ops.tree_attention(t, t, t, t, t, torch.ones(3, 3, dtype=torch.bool)),
                 lambda: ops.attention_weights(t, t), lambda: ops.evict(t[..., 0], t[..., 0].int(), t, t, None, 2, 1)):
        with pytest.raises(ValueError):
            call()


def _places(x):
    """Byte addresses of a view's elements."""
    at = torch.zeros((), dtype=torch.int64)
    for n, s in zip(x.shape, x.stride()):
        at = at[..., None] + torch.arange(n) * s
    return set((x.data_ptr() + at.flatten() * x.element_size()).tolist())


def _meet(x, y):
    return ops._views_meet(y.data_ptr() - x.data_ptr(), x.element_size(), x.shape, x.stride()[:3], y.shape, y.stride()[:3])


def test_views_that_meet():
    """Two views have memory in common exactly if an element of one is an element of the other, for all ways of cutting one
    buffer that a caller has; views across each other may count as meeting though they do not."""
    flat = torch.zeros(4096)
    qkv = flat[:2 * 5 * 7 * 4].view(2, 5, 7, 4)                                 # [b, s, heads, d]
    q, k, v = qkv[:, :, :4].transpose(1, 2), qkv[:, :, 4:6].transpose(1, 2), qkv[:, :, 6:].transpose(1, 2)
    heads = flat[:2 * 7 * 5 * 4].view(2, 7, 5, 4)                               # [b, heads, s, d]
    time = flat[:5 * 2 * 7 * 4].view(5, 2, 7, 4).permute(1, 2, 0, 3)            # [s, b, heads, d]
    pair = flat[:2 * 5 * 3 * 2 * 4].view(2, 5, 3, 2, 4)                         # k and v of a head side by side
    views = [q, k, v, heads[:, :4], heads[:, 4:6], heads[:, 6:], time[:, :4], time[:, 4:6], pair[..., 0, :].transpose(1, 2),
             pair[..., 1, :].transpose(1, 2), pair[:, :, :2, 1].transpose(1, 2), qkv[:, :3, :4].transpose(1, 2), qkv[:, 3:, :4].transpose(1, 2),
             q[:1], q[1:], q[:, :, ::2], q[:, :, 1::2], q[..., :2], q[..., 2:], q[..., 1:3], flat[1:281].view(2, 5, 7, 4)[:, :, :4].transpose(1, 2)]
    exact = 0
    for x in views:
        for y in views:
            common = bool(_places(x) & _places(y))
            assert _meet(x, y) >= common
            exact += _meet(x, y) == common
    assert exact >= 0.9 * len(views) ** 2
    for x, y in ((q, k), (k, v), (q, v), (heads[:, :4], heads[:, 4:6]), (time[:, :4], time[:, 4:6]), (views[8], views[9]), (views[9], views[8]),
                 (views[8], views[10]), (views[11], views[12]), (q[..., :2], q[..., 2:]), (q[:, :, ::2], q[:, :, 1::2])):
        assert not _meet(x, y) and not _meet(y, x)
    first = (2, 4, 5, 4), (80, 20, 4)
    for shift in range(-700, 700, 2):   # (in bytes, also into the middle of an element; 160 of them)
        assert ops._views_meet(shift, 4, *first, *first) is (-640 < shift < 640)


def test_views_whose_elements_have_a_place_each():
    x = torch.zeros(3, 4, 5, 6)
    once = lambda y: ops._once(y.shape, y.stride()[:3])  # noqa: E731
    assert all(once(y) for y in (x, x.transpose(1, 2), x[:, 1:3, ::2], x[..., 2:4], x[:, :1].expand(3, 1, 5, 6), x.permute(2, 0, 1, 3), x[:0]))
    assert not any(once(y) for y in (x[:, :1].expand(3, 4, 5, 6), x.as_strided((1, 3, 4, 6), (0, 13, 6, 1)), x.as_strided((1, 2, 3, 6), (0, 6, 3, 1))))


def test_what_is_written_meets_nothing_else():
    """Against all pairs: a written range and any other one with a byte in common."""
    import random
    rng = random.Random(0)
    for _ in range(3000):
        ranges = [(rng.randrange(40), rng.choice((0, 1, 3, 8)), rng.random() < 0.5) for _ in range(rng.randrange(1, 7))]
        meets = any(max(x[0], y[0]) < min(x[0] + x[1], y[0] + y[1]) and (x[2] or y[2])
                    for i, x in enumerate(ranges) for y in ranges[:i])
        assert ops._undisturbed(ranges) is not meets, ranges


@pytest.mark.parametrize("fn,good,changed", [
    ("lrqk_rotary", ROTARY, dict(s=(1 << 31) - 1)), ("lrqk_rotary", ROTARY, dict(s=(1 << 31) - 1, d=2, rotary_dim=2, hq=1, hk=0)),
    ("lrqk_attention_weights", WEIGHTS, dict(hq=32, hc=32, t=100, n=1 << 30, lse=P)),       # the columns' launch
    ("lrqk_attention_weights", WEIGHTS, dict(b=1023, hq=64, hc=64, t=1 << 20, n=1024))])    # that of the rows
def test_more_workgroups_than_a_launch_has_are_refused(fn, good, changed):
    """2^32 threads along an axis are too many, which the limits of the single sizes allow."""
    assert _call(fn, good, **changed) == ELIMIT
    assert b"places" in _lib.load().lrqk_last_error()


FAR = (1 << 32) + 3


@pytest.mark.parametrize("call", [
    lambda x: ops.rotary(ops.RotaryPlan(2, device="cpu"), x(FAR, 1, 1, 2), None, 0), lambda x: ops.rotary(ops.RotaryPlan(2, device="cpu"), x(1, FAR, 1, 2), None, 0),
    lambda x: ops.rotary(ops.RotaryPlan(2, device="cpu"), x(1, 1, 1, FAR), None, 0),
    lambda x: ops.rotary(ops.RotaryPlan(2, device="cpu"), x(1, 1, 1, 2), x(1, FAR, 1, 2), 0),
    lambda x: ops.tree_attention(x(1, 1, FAR, 8), *[x(1, 1, 5, 8)] * 2, *[x(1, 1, FAR, 8)] * 2, x(3, 3).bool()),
    lambda x: ops.tree_attention(x(FAR, 1, 3, 8), *[x(FAR, 1, 5, 8)] * 2, *[x(FAR, 1, 3, 8)] * 2, x(3, 3).bool()),
    lambda x: ops.attention_weights(x(1, 1, FAR, 8), x(1, 1, 5, 8)), lambda x: ops.attention_weights(x(1, FAR, 2, 8), x(1, 1, 5, 8)),
    lambda x: ops.attention_weights(x(1, FAR, 2, 8), x(1, FAR, 5, 8)),
    lambda x: ops.evict(x(1, 1, FAR), x(1, 1, FAR).int(), *[x(1, 1, FAR, 8)] * 2, None, 9, 1),
    lambda x: ops.evict(x(1, 1, 20), x(1, 1, 20).int(), *[x(1, 1, 20, 8)] * 2, None, 9, 1,
                        out=(x(1, 1, FAR), x(1, 1, FAR).int(), *[x(1, 1, FAR, 8)] * 2))])
def test_sizes_beyond_32_bits_do_not_reach_the_library_as_others(monkeypatch, call):
    """(Tensors without memory: the call is refused before anything looks at what they hold.)"""
    monkeypatch.setattr(ops, "_on_one_gpu", lambda *ts: 0)
    monkeypatch.setattr(ops, "_launch", lambda *args: pytest.fail("reached the library"))
    with pytest.raises(ValueError, match="beyond 32 bits"):
        call(lambda *shape: torch.empty(shape, device="meta"))


def test_scratch_of_more_than_an_eviction_takes():
    """The sizes that lrqk_evict refuses, for which the scratch's were formed beyond the integers' ends."""
    lib = _lib.load()
    for sizes in ((1, 1, (1 << 31) - 1, 10), (1, 1, (1 << 30) + 1, 10), (40000, 2, 100, 10), ((1 << 31) - 1, (1 << 31) - 1, 1 << 30, 9)):
        assert lib.lrqk_evict_workspace(*sizes) == ELIMIT
    assert lib.lrqk_evict_workspace(1, 1, 1 << 30, (1 << 31) - 1) >= 12 << 30
