"""Tensor-level wrappers over the C ABI.  torch is used only for device memory and the
current stream; every computation below happens in liblrqk_hip.so."""
from __future__ import annotations

import ctypes
import functools
import struct
import threading
from typing import Optional, Tuple

import torch

from . import _lib

_interrupted = {}   # by thread: what ended an allocator callback of the library call under way


def check(rc: int) -> int:
    """The library call's result, or the exception that it stands for.  An interrupt that ended an allocator callback is
    raised here: the library may have done without the block."""
    if rc >= 0 and not _interrupted:   # (a prompt makes some thirty calls)
        return rc
    raised = _interrupted.pop(threading.get_ident(), None)
    if raised is None:
        return _lib.check(rc)
    try:
        _lib.check(rc)
    except (_lib.LrqkError, ValueError) as e:
        raise e from raised
    raise raised


def _dt(t: torch.Tensor) -> int:
    if t.dtype == torch.float32:
        return _lib.F32
    if t.dtype == torch.bfloat16:
        return _lib.BF16
    raise ValueError(f"unsupported dtype {t.dtype}: the kernels store float32 or bfloat16")


def _stream(t: torch.Tensor) -> int:
    if t.is_cuda:   # (without the Stream object: 0.2 instead of 2 us, and a step of a short context waits for the host)
        return torch._C._cuda_getCurrentRawStream(t.get_device())
    return torch.cuda.current_stream(t.device).cuda_stream


def _need_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("tensor must live on the GPU")


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


# A ctx takes its device memory from torch's caching allocator, for the stream of the call that needs it: a cache
# object per prompt then reuses the blocks of the one before (nothing waits for the device), torch sees the memory in
# its statistics and gives it back when it runs short.
@_lib.ALLOC_FN
def _torch_alloc(nbytes, stream, user):
    try:
        return torch.cuda.caching_allocator_alloc(nbytes, stream=stream or 0)
    except BaseException as e:  # nothing may pass through the C frames, an interrupt included: a callback that is left by an
        if user and not isinstance(e, Exception):   # exception hands C an address that nobody wrote.  The library reports
            _interrupted[threading.get_ident()] = e  # the size it did not get, or does without it.
        return None


@_lib.RELEASE_FN
def _torch_release(block, user):
    try:
        torch.cuda.caching_allocator_delete(block)
    except BaseException:  # the interpreter is shutting down
        pass


class Workspace:
    """Owns one lrqk_ctx (device scratch).  Not thread safe; one per engine."""

    def __init__(self):
        self._h = ctypes.c_void_p()
        lib = _lib.load()
        check(lib.lrqk_ctx_create(ctypes.byref(self._h)))
        self._allocator = (_torch_alloc, _torch_release)  # alive as long as the ctx may call them
        check(lib.lrqk_ctx_set_allocator(self._h, *self._allocator, self._h))

    @property
    def handle(self):
        return self._h

    def reserve(self, bh, max_tokens, topk, n_active, r, d):
        """Memory for the calls to come, which are made on the stream that is current now."""
        check(_lib.load().lrqk_ctx_reserve_on(self._h, bh, max_tokens, topk, n_active, r, d,
                                              torch.cuda.current_stream().cuda_stream if torch.cuda.is_available() else None))

    def set_fetch_mode(self, mode: str, host_threads: int = 0):
        """'direct': the fetch kernel reads the pinned store itself (default); 'staged': host gather +
        hipMemcpyAsync on a side stream, as the reference stages its misses."""
        check(_lib.load().lrqk_ctx_set_fetch_mode(self.handle, {"direct": 0, "staged": 1}[mode], int(host_threads)))

    def score_index(self, enable: bool):
        """Switch the 8-bit score index of the scan on or off; either way what was indexed is dropped."""
        check(_lib.load().lrqk_ctx_score_index(self.handle, 1 if enable else 0))

    def victim_cache(self, rows_per_head: int):
        """Size (and empty) the victim cache of the fused decode step; 0 switches it off."""
        check(_lib.load().lrqk_ctx_victim_cache(self.handle, int(rows_per_head)))

    def factor_state(self, enable: bool = True):
        """Switch the kept state of the decode step's factor update on or off; either way what is kept is
        dropped (call it after changing B_Q, B_K, the active ids or rows behind the library's back)."""
        check(_lib.load().lrqk_ctx_factor_state(self.handle, 1 if enable else 0))

    def last_iterates(self, token: Optional[int] = None) -> Optional[torch.Tensor]:
        """fp64 [bh, max_iter, 2, r]: (q_hat, k_hat) of every iteration of the last decode step that ran from
        kept state, before any rounding; None if no such step ran (with ``token``: if that token's step did not)."""
        bh, it, r, tok = ctypes.c_int(), ctypes.c_int(), ctypes.c_int(), ctypes.c_int64()
        lib = _lib.load()
        check(lib.lrqk_last_iterates(self.handle, None, 0, ctypes.byref(bh), ctypes.byref(it), ctypes.byref(r),
                                     ctypes.byref(tok)))
        if bh.value * it.value * r.value == 0 or (token is not None and tok.value != token):
            return None
        out = torch.empty((bh.value, it.value, 2, r.value), dtype=torch.float64)
        check(lib.lrqk_last_iterates(self.handle, out.data_ptr(), out.numel(), ctypes.byref(bh), ctypes.byref(it),
                                     ctypes.byref(r), ctypes.byref(tok)))
        return out

    def victim_stats(self, reset: bool = True) -> int:
        """Rows the fused decode step fetched over the host link since the last reset."""
        n = ctypes.c_int64()
        check(_lib.load().lrqk_victim_stats(self.handle, ctypes.byref(n), 1 if reset else 0))
        return n.value

    def timing_enable(self, max_launches: int, every: int = 1):
        """Bracket (every `every`-th of) the next proxy-score launches with HIP events, at most max_launches."""
        check(_lib.load().lrqk_timing_enable(self._h, max_launches))
        check(_lib.load().lrqk_timing_stride(self._h, every))

    def timing_read(self):
        """(summed proxy-score kernel time in ms, launches) since the last read."""
        ms, n = ctypes.c_double(), ctypes.c_int()
        check(_lib.load().lrqk_timing_read(self._h, ctypes.byref(ms), ctypes.byref(n)))
        return ms.value, n.value

    def select_stats(self, reset: bool = True):
        """(heads served from the candidate list, heads that rescanned) since the last reset."""
        a, b = ctypes.c_int(), ctypes.c_int()
        check(_lib.load().lrqk_select_stats(self._h, ctypes.byref(a), ctypes.byref(b), 1 if reset else 0))
        return a.value, b.value

    def scan_stats(self):
        """(rows covered, rows rescored exactly) by the last scan through the score index; (0, 0) otherwise."""
        a, b = ctypes.c_int64(), ctypes.c_int64()
        check(_lib.load().lrqk_scan_stats(self._h, ctypes.byref(a), ctypes.byref(b)))
        return a.value, b.value

    def select_stats_detail(self):
        """(lists too short, lists overflowed) among the rescans of the last select_stats()."""
        a, b = ctypes.c_int(), ctypes.c_int()
        check(_lib.load().lrqk_select_stats_detail(self._h, ctypes.byref(a), ctypes.byref(b)))
        return a.value, b.value

    def close(self):
        if self._h:
            _lib.load().lrqk_ctx_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


_default_ws: Optional[Workspace] = None


def default_workspace() -> Workspace:
    global _default_ws
    if _default_ws is None:
        _default_ws = Workspace()
    return _default_ws


# --------------------------------------------------------------------------- selection

def proxy_scores(a_k: torch.Tensor, q_hat: torch.Tensor, m: Optional[int] = None,
                 round_to_storage: bool = True) -> torch.Tensor:
    """a_k [b,H,cap,r] (contiguous), q_hat [b,H,1,r] -> fp32 [b,H,m]."""
    _need_cuda(a_k, q_hat)
    b, H, cap, r = a_k.shape
    m = cap if m is None else m
    assert a_k.is_contiguous() and 0 <= m <= cap
    qh = q_hat.reshape(b * H, r).contiguous()
    out = torch.empty((b, H, m), dtype=torch.float32, device=a_k.device)
    check(_lib.load().lrqk_proxy_scores(a_k.data_ptr(), cap * r, qh.data_ptr(), b * H, m, r, _dt(a_k),
                                        1 if (round_to_storage and a_k.dtype == torch.bfloat16) else 0,
                                        out.data_ptr(), _stream(a_k)))
    return out


def score_select(ws: Workspace, a_k: torch.Tensor, q_hat: torch.Tensor, m: int, topk: int,
                 round_to_storage: bool = True, out: Optional[torch.Tensor] = None,
                 head_rows: Optional[int] = None, list_next: bool = False) -> torch.Tensor:
    """Top-k token ids (ascending) of q_hat . a_k[:m]^T per head: int32 [b,H,min(topk,m)].
    a_k is [b,H,cap,r] contiguous, or (with head_rows) a view whose heads start head_rows rows
    apart and whose rows are contiguous.  list_next: ``victim_fill`` follows."""
    _need_cuda(a_k, q_hat)
    b, H, cap, r = a_k.shape
    if head_rows is None:
        assert a_k.is_contiguous()
    else:
        cap = head_rows
    assert 0 <= m <= cap
    qh = q_hat.reshape(b * H, r).contiguous()
    kk = min(topk, m)
    if out is None:
        out = torch.empty((b, H, kk), dtype=torch.int32, device=a_k.device)
    assert out.dtype == torch.int32 and out.is_contiguous() and out.shape[-1] >= kk
    lib = _lib.load()
    select = lib.lrqk_score_select_next if list_next else lib.lrqk_score_select
    check(select(ws.handle, a_k.data_ptr(), cap * r, qh.data_ptr(), b * H, m, r, topk, _dt(a_k),
                 1 if (round_to_storage and a_k.dtype == torch.bfloat16) else 0, out.data_ptr(), out.shape[-1], _stream(a_k)))
    return out


def score_select_diff(ws: Workspace, a_k: torch.Tensor, q_hat: torch.Tensor, m: int, topk: int, hit: torch.Tensor,
                      round_to_storage: bool = True, want_new: bool = True):
    """score_select + diff in one pass (m >= topk).  hit int32 [b,H,>=topk] is updated in place.
    Returns (new_idx int32 [b,H,topk], evict u8 [b,H,topk], miss_slots int32 [b,H,topk], miss_count int32 [b,H]).
    want_new=False: only what changes is produced (new_idx is None), as inside the decode step."""
    _need_cuda(a_k, q_hat, hit)
    b, H, cap, r = a_k.shape
    assert a_k.is_contiguous() and hit.is_contiguous() and hit.dtype == torch.int32 and topk <= m <= cap
    qh = q_hat.reshape(b * H, r).contiguous()
    dev = a_k.device
    new = torch.empty((b, H, topk), dtype=torch.int32, device=dev) if want_new else None
    evict = torch.empty((b, H, topk), dtype=torch.uint8, device=dev)
    miss_slots = torch.empty((b, H, topk), dtype=torch.int32, device=dev)
    miss_count = torch.empty((b, H), dtype=torch.int32, device=dev)
    check(_lib.load().lrqk_score_select_diff(ws.handle, a_k.data_ptr(), cap * r, qh.data_ptr(), b * H, m, r, topk,
                                             _dt(a_k), 1 if (round_to_storage and a_k.dtype == torch.bfloat16) else 0,
                                             _ptr(new), hit.data_ptr(), hit.shape[-1], evict.data_ptr(),
                                             miss_slots.data_ptr(), miss_count.data_ptr(), _stream(a_k)))
    return new, evict, miss_slots, miss_count


def select_from_scores(ws: Workspace, scores: torch.Tensor, topk: int) -> torch.Tensor:
    """scores fp32 [b,H,m] -> int32 [b,H,min(topk,m)] ascending."""
    _need_cuda(scores)
    b, H, m = scores.shape
    sc = scores.contiguous().float()
    kk = min(topk, m)
    out = torch.empty((b, H, kk), dtype=torch.int32, device=scores.device)
    check(_lib.load().lrqk_select_from_scores(ws.handle, sc.data_ptr(), b * H, m, topk, out.data_ptr(), kk,
                                              _stream(scores)))
    return out


def diff(new_idx: torch.Tensor, hit: torch.Tensor, k: Optional[int] = None, replace_all: bool = False):
    """In-place hit/miss diff.  new_idx int32 [b,H,>=k] ascending; hit int32 [b,H,stride] (first k
    entries are the resident set; may be a wider buffer).  Returns (evict u8 [b,H,k], miss_slots
    int32 [b,H,k], miss_count int32 [b,H])."""
    _need_cuda(new_idx, hit)
    b, H = hit.shape[:2]
    k = hit.shape[2] if k is None else k
    assert new_idx.dtype == torch.int32 and hit.dtype == torch.int32
    assert new_idx.is_contiguous() and hit.is_contiguous()
    dev = hit.device
    evict = torch.empty((b, H, k), dtype=torch.uint8, device=dev)
    miss_slots = torch.empty((b, H, k), dtype=torch.int32, device=dev)
    miss_count = torch.empty((b, H), dtype=torch.int32, device=dev)
    fn = _lib.load().lrqk_replace_all if replace_all else _lib.load().lrqk_diff
    check(fn(new_idx.data_ptr(), new_idx.shape[2], hit.data_ptr(), hit.shape[2], b * H, k, evict.data_ptr(),
             miss_slots.data_ptr(), miss_count.data_ptr(), _stream(hit)))
    return evict, miss_slots, miss_count


def fetch_rows(kv_store: torch.Tensor, k_act: torch.Tensor, v_act: torch.Tensor, hit: torch.Tensor,
               miss_slots: torch.Tensor, miss_count: torch.Tensor, k: int):
    """kv_store [b,Hkv,cap,2d] (pinned host or device), k_act/v_act [b,Hq,n,d]."""
    _need_cuda(k_act, v_act, hit, miss_slots, miss_count)
    b, hkv, cap, d2 = kv_store.shape
    _, hq, n, d = k_act.shape
    assert d2 == 2 * d and kv_store.is_contiguous() and k_act.is_contiguous() and v_act.is_contiguous()
    assert kv_store.dtype == k_act.dtype == v_act.dtype
    if not kv_store.is_cuda and not kv_store.is_pinned():
        raise ValueError("the host [K|V] store must be pinned memory")
    check(_lib.load().lrqk_fetch_rows(kv_store.data_ptr(), cap, k_act.data_ptr(), v_act.data_ptr(), n, hit.data_ptr(),
                                      hit.shape[2], miss_slots.data_ptr(), miss_count.data_ptr(), b, hq, hkv, d, k,
                                      _dt(k_act), _stream(k_act)))


def fetch_rows_staged(ws: Workspace, kv_store: torch.Tensor, k_act: torch.Tensor, v_act: torch.Tensor,
                      hit: torch.Tensor, miss_slots: torch.Tensor, miss_count: torch.Tensor, k: int):
    """Same result as fetch_rows, through host gather + hipMemcpyAsync on the workspace's side stream
    (kv_store must be pinned host memory; waits for the stream once)."""
    _need_cuda(k_act, v_act, hit, miss_slots, miss_count)
    b, hkv, cap, d2 = kv_store.shape
    _, hq, n, d = k_act.shape
    assert d2 == 2 * d and kv_store.is_contiguous() and k_act.is_contiguous() and v_act.is_contiguous()
    assert kv_store.dtype == k_act.dtype == v_act.dtype
    if kv_store.is_cuda or not kv_store.is_pinned():
        raise ValueError("the staged fetch needs the [K|V] store in pinned host memory")
    check(_lib.load().lrqk_fetch_rows_staged(ws.handle, kv_store.data_ptr(), cap, k_act.data_ptr(), v_act.data_ptr(), n,
                                             hit.data_ptr(), hit.shape[2], miss_slots.data_ptr(),
                                             miss_count.data_ptr(), b, hq, hkv, d, k, _dt(k_act), _stream(k_act)))


def gather_rows(src: torch.Tensor, idx: torch.Tensor, dst: torch.Tensor, count: int):
    """dst[b,h,j,:] = src[b,h//g,idx[b,h,j],:] for j < count; slots whose id is negative keep their
    contents.  src [b,Hkv,l,d] on the GPU or in pinned host memory, dst [b,Hq,n,d]."""
    _need_cuda(idx, dst)
    if not src.is_cuda and not src.is_pinned():
        raise ValueError("a host source must be pinned memory")
    b, hkv, l, d = src.shape
    _, hq, n, _ = dst.shape
    # the kernel takes the row width and the element type from src alone: a source whose rows are wider than
    # the destination's (the [K|V] store, 2d wide) would be written past the end of dst
    if src.shape[-1] != dst.shape[-1] or src.dtype != dst.dtype or src.shape[0] != dst.shape[0]:
        raise ValueError(f"source rows {tuple(src.shape)} {src.dtype} do not match the destination "
                         f"{tuple(dst.shape)} {dst.dtype}: pass a K or a V source whose rows are as wide as dst")
    if hq % hkv != 0 or tuple(idx.shape[:2]) != (b, hq) or not 0 <= count <= min(idx.shape[2], n):
        raise ValueError("idx must be [b,Hq,>=count] with count slots inside dst")
    assert src.is_contiguous() and dst.is_contiguous() and idx.is_contiguous() and idx.dtype == torch.int32
    check(_lib.load().lrqk_gather_rows(src.data_ptr(), l, idx.data_ptr(), idx.shape[2], count, dst.data_ptr(), n, b, hq,
                                       hkv, d, _dt(src), _stream(dst)))


def fill_active(k: torch.Tensor, v: torch.Tensor, active_idx: torch.Tensor, k_act: torch.Tensor, v_act: torch.Tensor,
                topk: int):
    """The active set of a prompt: slots 0 .. topk-1 of k_act, v_act [b,Hq,topk+lite,d] take the rows of k, v
    [b,Hkv,l,d] that active_idx int32 [b,Hq,topk+lite] names there, the other slots the last tokens' (ids included)."""
    _need_cuda(k, v, active_idx, k_act, v_act)
    b, hkv, l, d = k.shape
    _, hq, n, _ = k_act.shape
    assert k.is_contiguous() and v.is_contiguous() and v.shape == k.shape and k_act.is_contiguous() and v_act.is_contiguous()
    assert k.dtype == v.dtype == k_act.dtype == v_act.dtype and k_act.shape == v_act.shape == (b, hq, n, d)
    assert active_idx.is_contiguous() and active_idx.dtype == torch.int32 and active_idx.shape == (b, hq, n)
    check(_lib.load().lrqk_fill_active(k.data_ptr(), v.data_ptr(), l, active_idx.data_ptr(), k_act.data_ptr(),
                                       v_act.data_ptr(), topk, n - topk, b, hq, hkv, d, _dt(k), _stream(k)))


def victim_fill(ws: Workspace, k: torch.Tensor, v: torch.Tensor, hq: int, capacity: int):
    """The rows of k, v [b,Hkv,l,d] of the tokens that the last ``score_select`` of ``ws``, called with ``list_next``, left
    out by the least go into its empty victim cache; ``capacity``: rows of the host store of the steps to come."""
    _need_cuda(k, v)
    b, hkv, l, d = k.shape
    assert k.is_contiguous() and v.is_contiguous() and v.shape == k.shape and k.dtype == v.dtype
    check(_lib.load().lrqk_victim_fill(ws.handle, k.data_ptr(), v.data_ptr(), l, capacity, b, hq, hkv, d, _dt(k), _stream(k)))


def append_token(k_new, v_new, k_act, v_act, slot: int, active_idx: Optional[torch.Tensor], token: int):
    _need_cuda(k_new, v_new, k_act, v_act)
    b, hkv = k_new.shape[:2]
    _, hq, n, d = k_act.shape
    kn, vn = k_new.reshape(b, hkv, d).contiguous(), v_new.reshape(b, hkv, d).contiguous()
    check(_lib.load().lrqk_append_token(kn.data_ptr(), vn.data_ptr(), k_act.data_ptr(), v_act.data_ptr(), n, slot,
                                        _ptr(active_idx), 0 if active_idx is None else active_idx.shape[2], token, b,
                                        hq, hkv, d, _dt(k_act), _stream(k_act)))


def flush_ring(k_act, v_act, slot0: int, count: int, kv_store: torch.Tensor, row0: int, hkv: int):
    _need_cuda(k_act, v_act)
    b, hq, n, d = k_act.shape
    cap = kv_store.shape[2]
    check(_lib.load().lrqk_flush_ring(k_act.data_ptr(), v_act.data_ptr(), n, slot0, count, kv_store.data_ptr(), cap,
                                      row0, b, hq, hkv, d, _dt(k_act), _stream(k_act)))


def interleave_kv(k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """k, v [b,Hkv,l,d] contiguous -> [b,Hkv,l,2d] on the device, each token's K row followed by its V row."""
    _need_cuda(k, v)
    b, hkv, l, d = k.shape
    assert k.is_contiguous() and v.is_contiguous() and v.shape == k.shape and v.dtype == k.dtype
    out = torch.empty((b, hkv, l, 2 * d), dtype=k.dtype, device=k.device)
    check(_lib.load().lrqk_interleave_kv(k.data_ptr(), v.data_ptr(), out.data_ptr(), b * hkv, l, d, _dt(k), _stream(k)))
    return out


def store_rows(rows: torch.Tensor, kv_store: torch.Tensor, row0: int, stream: torch.cuda.Stream):
    """rows [b,Hkv,l,2d] on the device -> rows row0 .. row0 + l of the pinned host store [b,Hkv,cap,2d], by a DMA
    engine on ``stream``.  The caller orders the stream and keeps ``rows`` until the copy is done."""
    _need_cuda(rows)
    b, hkv, l, d2 = rows.shape
    assert rows.is_contiguous() and kv_store.is_contiguous() and kv_store.is_pinned() and kv_store.dtype == rows.dtype
    assert tuple(kv_store.shape[:2]) == (b, hkv) and kv_store.shape[3] == d2
    check(_lib.load().lrqk_store_rows(rows.data_ptr(), kv_store.data_ptr(), kv_store.shape[2], row0, b * hkv, l, d2 // 2,
                                      _dt(rows), stream.cuda_stream))


def attention(ws: Workspace, q: torch.Tensor, k_act: torch.Tensor, v_act: torch.Tensor,
              n_valid: Optional[int] = None) -> torch.Tensor:
    """q [b,H,1,d]; k_act,v_act [b,H,n,d] contiguous -> [b,H,1,d]."""
    _need_cuda(q, k_act, v_act)
    b, H, n, d = k_act.shape
    n_valid = n if n_valid is None else n_valid
    assert k_act.is_contiguous() and v_act.is_contiguous() and q.dtype == k_act.dtype == v_act.dtype
    qq = q.reshape(b * H, d).contiguous()
    out = torch.empty((b, H, 1, d), dtype=q.dtype, device=q.device)
    check(_lib.load().lrqk_attention(ws.handle, qq.data_ptr(), k_act.data_ptr(), v_act.data_ptr(), n, n_valid,
                                     out.data_ptr(), b * H, d, _dt(q), _stream(q)))
    return out


def attention_static(q: torch.Tensor, k_act: torch.Tensor, v_act: torch.Tensor, out: torch.Tensor,
                     n_valid: Optional[int] = None) -> torch.Tensor:
    """The same attention through the entry point that allocates nothing: no workspace, the caller
    passes ``out`` [b,H,1,d] and a contiguous q; partial results go to a fixed block inside the library."""
    _need_cuda(q, k_act, v_act, out)
    b, H, n, d = k_act.shape
    n_valid = n if n_valid is None else n_valid
    assert k_act.is_contiguous() and v_act.is_contiguous() and q.is_contiguous() and out.is_contiguous()
    assert q.dtype == k_act.dtype == v_act.dtype == out.dtype and out.numel() == b * H * d
    check(_lib.load().lrqk_attention_static(q.data_ptr(), k_act.data_ptr(), v_act.data_ptr(), n, n_valid,
                                            out.data_ptr(), b * H, d, _dt(q), _stream(q)))
    return out


def als_decode(ws: Workspace, b_q, b_k, a_k, active_idx: Optional[torch.Tensor], k_prev, n: int, q, k_new,
               max_iter: int, tol: float, append_row: int = -1) -> Tuple[torch.Tensor, torch.Tensor]:
    """In-place factor update.  b_q,b_k [b,H,r,d]; a_k [b,H,cap,r]; active_idx int32 [b,H,>=n] or None;
    k_prev [b,H,slots,d]; q [b,H,1,d]; k_new [b,Hkv,1,d].  Returns (q_hat, k_hat) [b,H,1,r]."""
    _need_cuda(b_q, b_k, a_k, k_prev, q, k_new)
    b, H, r, d = b_q.shape
    hkv = k_new.shape[1]
    cap = a_k.shape[2]
    assert b_q.is_contiguous() and b_k.is_contiguous() and a_k.is_contiguous() and k_prev.is_contiguous()
    assert b_q.dtype == b_k.dtype == a_k.dtype == k_prev.dtype == q.dtype == k_new.dtype
    qq = q.reshape(b * H, d).contiguous()
    kn = k_new.reshape(b * hkv, d).contiguous()
    q_hat = torch.empty((b, H, 1, r), dtype=b_q.dtype, device=b_q.device)
    k_hat = torch.empty((b, H, 1, r), dtype=b_q.dtype, device=b_q.device)
    check(_lib.load().lrqk_als_decode(ws.handle, b_q.data_ptr(), b_k.data_ptr(), a_k.data_ptr(), cap * r,
                                      _ptr(active_idx), 0 if active_idx is None else active_idx.shape[2],
                                      k_prev.data_ptr(), k_prev.shape[2], n, qq.data_ptr(), kn.data_ptr(), b, H, hkv, r,
                                      d, int(max_iter), float(tol), q_hat.data_ptr(), k_hat.data_ptr(), append_row,
                                      _dt(b_q), _stream(b_q)))
    return q_hat, k_hat


def als_prefill(ws: Workspace, q: torch.Tensor, k: torch.Tensor, a_q0: torch.Tensor, a_k0: torch.Tensor,
                max_iter: int, tol: float):
    """q [b,Hq,l,d], k [b,Hkv,l,d] storage dtype; a_q0,a_k0 fp32 [b,Hq,l,r] initial factors (consumed:
    they are updated in place).  Returns fp32 (A_Q, B_Q, A_K, B_K)."""
    _need_cuda(q, k, a_q0, a_k0)
    b, hq, l, d = q.shape
    hkv = k.shape[1]
    r = a_q0.shape[-1]
    assert q.is_contiguous() and k.is_contiguous() and q.dtype == k.dtype
    assert a_q0.dtype == torch.float32 and a_k0.dtype == torch.float32 and a_q0.is_contiguous() and a_k0.is_contiguous()
    assert a_q0.shape == (b, hq, l, r) and a_k0.shape == (b, hq, l, r)
    b_q = torch.empty((b, hq, r, d), dtype=torch.float32, device=q.device)
    b_k = torch.empty((b, hq, r, d), dtype=torch.float32, device=q.device)
    check(_lib.load().lrqk_als_prefill(ws.handle, q.data_ptr(), k.data_ptr(), a_q0.data_ptr(), a_k0.data_ptr(),
                                       b_q.data_ptr(), b_k.data_ptr(), b, hq, hkv, l, r, d, int(max_iter), float(tol),
                                       _dt(q), _stream(q)))
    return a_q0, b_q, a_k0, b_k


def als_prefill_store(ws: Workspace, q: torch.Tensor, k: torch.Tensor, a_q0: torch.Tensor, a_k0: torch.Tensor,
                      max_iter: int, tol: float, a_k: Optional[torch.Tensor] = None, row0: int = 0,
                      last_query_row: bool = False):
    """The fit of als_prefill with its results in the inputs' type: (A_Q, B_Q, A_K, B_K).  A_K [b,Hq,l,r] goes to rows
    row0 .. row0 + l of ``a_k`` [b,Hq,cap,r] if that is given (and A_K is then a view of it); with ``last_query_row``
    A_Q is [b,Hq,1,r], its last row.  a_q0, a_k0 (fp32 [b,Hq,l,r]) are consumed."""
    _need_cuda(q, k, a_q0, a_k0, a_k)
    b, hq, l, d = q.shape
    hkv = k.shape[1]
    r = a_q0.shape[-1]
    assert q.is_contiguous() and k.is_contiguous() and q.dtype == k.dtype
    assert a_q0.dtype == torch.float32 and a_k0.dtype == torch.float32 and a_q0.is_contiguous() and a_k0.is_contiguous()
    assert a_q0.shape == (b, hq, l, r) and a_k0.shape == (b, hq, l, r)
    if a_k is None:
        a_k, row0 = torch.empty((b, hq, l, r), dtype=q.dtype, device=q.device), 0
    assert a_k.is_contiguous() and a_k.dtype == q.dtype and a_k.shape[:2] == (b, hq) and a_k.shape[3] == r
    out = a_k.narrow(2, row0, l)
    a_q = torch.empty((b, hq, 1 if last_query_row else l, r), dtype=q.dtype, device=q.device)
    b_q = torch.empty((b, hq, r, d), dtype=q.dtype, device=q.device)
    b_k = torch.empty((b, hq, r, d), dtype=q.dtype, device=q.device)
    check(_lib.load().lrqk_als_prefill_store(ws.handle, q.data_ptr(), k.data_ptr(), a_q0.data_ptr(), a_k0.data_ptr(),
                                             a_q.data_ptr(), a_q.shape[2], out.data_ptr(), a_k.shape[2] * r, b_q.data_ptr(),
                                             b_k.data_ptr(), b, hq, hkv, l, r, d, int(max_iter), float(tol), _dt(q),
                                             _stream(q)))
    return a_q, b_q, out, b_k


def _rows(t: torch.Tensor, n: int, d: int) -> torch.Tensor:
    """n contiguous rows of d elements: t itself where it holds them (a reshape is 1 us of host time, three of them a step)."""
    if t.is_contiguous() and t.numel() == n * d:
        return t
    t = t.reshape(n, d)
    assert t.is_contiguous()
    return t


def decode_step(ws: Workspace, b_q, b_k, a_k, active_idx, k_act, v_act, kv_store, q, k_new, v_new, *, topk: int,
                lite: int, ring_slot: int, token: int, m: int, flush_row0: int, max_iter: int, tol: float,
                round_scores: bool, no_hit_miss: bool, q_hat, k_hat, attn_out=None, evict=None, miss_count=None):
    b, H, r, d = b_q.shape
    hkv = k_new.shape[1]
    cap_a = a_k.shape[2]
    qq, kn, vn = _rows(q, b * H, d), _rows(k_new, b * hkv, d), _rows(v_new, b * hkv, d)
    check(_lib.load().lrqk_decode_step(
        ws.handle, b_q.data_ptr(), b_k.data_ptr(), a_k.data_ptr(), cap_a * r, active_idx.data_ptr(), k_act.data_ptr(),
        v_act.data_ptr(), kv_store.data_ptr(), kv_store.shape[2], qq.data_ptr(), kn.data_ptr(), vn.data_ptr(), b, H, hkv,
        r, d, topk, lite, ring_slot, token, m, flush_row0, int(max_iter), float(tol),
        1 if (round_scores and b_q.dtype == torch.bfloat16) else 0, 1 if no_hit_miss else 0, q_hat.data_ptr(),
        k_hat.data_ptr(), _ptr(attn_out), _ptr(evict), _ptr(miss_count), _dt(b_q), _stream(b_q)))


# --------------------------------------------------------------------------- drafted tokens and budgets
# These calls take no workspace object: their scratch comes from torch for the call's stream, so that several streams and
# captured graphs need not share any.

# (A call of a few tokens is bound by its host time, so sizes, types and devices are compared as they are: no device objects,
# no tuples, and the scratch sizes of a set of sizes are asked for once.)

def _launch(dev: int, fn, *args) -> int:
    """The library call on device ``dev`` and its current stream."""
    if torch.cuda.current_device() == dev:
        return check(fn(*args, torch._C._cuda_getCurrentRawStream(dev)))
    with torch.cuda.device(dev):
        return check(fn(*args, torch._C._cuda_getCurrentRawStream(dev)))


def _on_one_gpu(first: torch.Tensor, *ts) -> int:
    dev = first.get_device()
    if dev < 0:
        raise ValueError("tensor must live on the GPU")
    for t in ts:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"tensors on {first.device} and {t.device}")
    return dev


def _expect(name: str, t: torch.Tensor, shape, dtype, contiguous: bool = True):
    if t.shape != shape or t.dtype != dtype:
        raise ValueError(f"{name} is {tuple(t.shape)} {t.dtype}: {tuple(shape)} {dtype} is wanted")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _too_large(*sizes: int):
    """The library takes sizes as 32-bit numbers: a larger one would reach it as another."""
    raise ValueError(f"a size of {max(sizes)} is beyond 32 bits")


def _row_strides(name: str, t: torch.Tensor, b: int, h: int, n: int, d: int):
    """Strides of sequences, heads and rows of a tensor of these sizes whose rows are contiguous; 0 where there is one of a kind,
    whose stride leads to nothing and may be anything."""
    s = t.stride()
    if s[3] != 1 and d > 1:
        raise ValueError(f"the rows of {name} must be contiguous")
    if b == 1 or h == 1 or n == 1:
        return s[0] if b > 1 else 0, s[1] if h > 1 else 0, s[2] if n > 1 else 0
    return s[:3]


def _rows16(x: torch.Tensor) -> torch.Tensor:
    """x, or a copy of it where its rows do not follow each other or begin between two 16-byte pieces."""
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _lengths(lengths: Optional[torch.Tensor], b: int):
    if lengths is not None:
        _expect("lengths", lengths, (b,), torch.int32)


@functools.lru_cache(maxsize=1024)
def _scratch_bytes(entry: str, *sizes: int) -> int:
    return check(getattr(_lib.load(), entry)(*sizes))


def _scratch(nbytes: int, like: torch.Tensor) -> torch.Tensor:
    return torch.empty(nbytes, dtype=torch.uint8, device=like.device)


class RotaryPlan:
    """The angles per position of rotary embeddings over the first ``rotary_dim`` elements of a head, on ``device``.

    ``scaling``: None, or a dict for contexts longer than the trained one, with ``type`` and ``factor``:
      linear   angles divided by the factor
      ntk      theta stretched by factor ** (rotary_dim / (rotary_dim - 2))
      llama3   by their turns over ``original_context``: divided below ``low_freq_factor``, kept above ``high_freq_factor``
      yarn     kept for the pairs that turn more than ``beta_fast`` times over ``original_context``, divided for those that
               turn less than ``beta_slow`` times, a ramp in between; the results are multiplied by ``attention_factor``
               (0.1 ln(factor) + 1 if it is not given)
    ``interleaved``: pairs are elements 2 i and 2 i + 1, else i and i + rotary_dim / 2.  ``inv_freq``: fp64 on the device."""

    _KEYS = {"linear": (), "ntk": (), "llama3": ("low_freq_factor", "high_freq_factor", "original_context"),
             "yarn": ("beta_fast", "beta_slow", "original_context")}

    def __init__(self, rotary_dim: int, theta: float = 10000.0, interleaved: bool = False, scaling: Optional[dict] = None,
                 device="cuda:0"):
        kind, s = "plain", dict(scaling or {})
        if scaling is not None:
            kind = s.pop("type", None)
            if kind not in self._KEYS:
                raise ValueError(f"unknown scaling {kind!r}: one of {sorted(self._KEYS)}")
        attention_factor = s.pop("attention_factor", None) if kind == "yarn" else None
        if kind == "yarn":
            s = {"beta_fast": 32.0, "beta_slow": 1.0, **s}
        wanted = ("factor",) + self._KEYS[kind] if kind != "plain" else ()
        if set(s) != set(wanted):
            raise ValueError(f"scaling {kind!r} takes {sorted(wanted)}, got {sorted(s)}")
        p0, p1 = (float(s[k]) for k in self._KEYS[kind][:2]) if len(wanted) > 1 else (0.0, 0.0)
        freq = torch.empty(max(rotary_dim // 2, 1), dtype=torch.float64)
        result = ctypes.c_double()
        check(_lib.load().lrqk_rotary_frequencies(rotary_dim, float(theta), _lib.ROPE[kind], float(s.get("factor", 1.0)), p0, p1,
                                                  float(s.get("original_context", 0.0)), freq.data_ptr(), ctypes.byref(result)))
        self.rotary_dim = rotary_dim
        self.interleaved = bool(interleaved)
        self.factor = result.value if attention_factor is None else float(attention_factor)
        self.inv_freq = freq.to(device)


# Whether views share memory is asked of their layouts (b, heads, tokens, elements, and their strides but the last, which is 1)
# and of how far apart they begin.

@functools.lru_cache(maxsize=1024)
def _once(shape, strides) -> bool:
    """Whether every element of a view has a place of its own (a view that cannot be made by slicing and permuting counts as one
    that has not)."""
    inner = 1
    for stride, n in sorted((s, n) for s, n in zip((*strides, 1), shape) if n > 1):
        if stride < inner:
            return False
        inner += (n - 1) * stride
    return True


def _blocks_meet(shift: int, x: int, y: int, dims) -> bool:
    """Whether a block of x elements and one of y, ``shift`` behind it, meet.  dims: what both consist of, (elements between
    slabs, slabs of x, slabs of y), longest first; without any a block is whole."""
    if shift >= x or -shift >= y:
        return False
    if not dims:
        return True
    step, nx, ny = dims[0]
    x, y = x - (nx - 1) * step, y - (ny - 1) * step
    # a slab of y lies j steps from one of x: those j at which they reach each other, as far as whole slabs go
    first, last = max(1 - nx, (-y - shift) // step + 1), min(ny - 1, -((shift - x) // step) - 1)
    return last - first > 3 or any(_blocks_meet(shift + j * step, x, y, dims[1:]) for j in range(first, last + 1))


@functools.lru_cache(maxsize=1024)
def _common(shape_x, strides_x, shape_y, strides_y):
    """Elements from the first of a view to behind the last, of two views, and the dimensions that have the same stride in both as
    _blocks_meet takes them."""
    dims = []
    for nx, ny, sx, sy in zip(shape_x, shape_y, (*strides_x, 1), (*strides_y, 1)):
        step = sx if nx > 1 else sy
        if max(nx, ny) > 1 and step > 0 and (sx == sy or min(nx, ny) == 1):
            dims.append((step, nx, ny))
    reach = [1 + sum((n - 1) * s for n, s in zip(shape, (*strides, 1))) for shape, strides in ((shape_x, strides_x), (shape_y, strides_y))]
    return (*reach, sorted(dims, reverse=True))


def _views_meet(shift: int, e: int, shape_x, strides_x, shape_y, strides_y) -> bool:
    """Whether two views of elements of e bytes, the second of which begins ``shift`` bytes behind the first, have memory in
    common.  Views that lie between each other, as the parts of one projection do, are told apart where their dimensions
    have the same strides; otherwise views whose ranges meet count as meeting."""
    x, y, dims = _common(shape_x, strides_x, shape_y, strides_y)
    if shift % e == 0:
        return _blocks_meet(shift // e, x, y, dims)
    # (views that begin within each other's elements: what an element covers reaches into the next one)
    return _blocks_meet(shift // e, x, y, dims) or _blocks_meet(shift // e + 1, x, y, dims)


def _refuse_overlaps(e: int, b: int, s: int, d: int, views, heads, strides, pos, pos_stride: int, freq):
    """q, q', k, k' of a turn, with three strides each: an output is its input or meets none, and not the other output."""
    places = []   # where a view begins and ends; its layout
    for i, (x, h) in enumerate(zip(views, heads)):
        if x is None or h == 0:
            places.append(None)
            continue
        sb, sh, ss = st = strides[3 * i:3 * i + 3]
        at = x.data_ptr()
        places.append((at, at + e * ((b - 1) * sb + (h - 1) * sh + (s - 1) * ss + d), (b, h, s, d), st))

    def meet(x, y):
        return x is not None and y is not None and x[0] < y[1] and y[0] < x[1] and _views_meet(y[0] - x[0], e, *x[2:], *y[2:])
    q, q_out, k, k_out = places
    f_at, p_at = freq.data_ptr(), 0 if pos is None else pos.data_ptr()
    f_end, p_end = f_at + freq.nbytes, 0 if pos is None else p_at + 4 * ((b - 1) * pos_stride + s)
    for y in (q_out, k_out):
        if y is None:
            continue
        if not _once(*y[2:]):
            raise ValueError("out has several elements in one place")
        if f_at < y[1] and y[0] < f_end or p_at < y[1] and y[0] < p_end:
            raise ValueError("out overlaps the positions or the plan")
    in_place = q == q_out and k == k_out   # (then one pair is left)
    if (q != q_out and meet(q, q_out)) or (k != k_out and meet(k, k_out)) or meet(k, q_out) or (
            not in_place and meet(q, k_out)):
        raise ValueError("out overlaps an input and is not the view that is turned")
    if not in_place and meet(q_out, k_out):
        raise ValueError("out of q and out of k overlap")


def _undisturbed(ranges) -> bool:
    """Of (begin, bytes, written): whether what is written meets nothing else."""
    reach = wrote = 0   # ends of what begins further in front
    for begin, size, written in sorted(ranges):
        if size and begin < (reach if written else wrote):
            return False
        reach = max(reach, begin + size)
        if written:
            wrote = max(wrote, begin + size)
    return True


def rotary(plan: RotaryPlan, q: torch.Tensor, k: Optional[torch.Tensor], positions, transpose: bool = False, out=None):
    """q [b,Hq,s,d] and k [b,Hk,s,d] (or None) turned to ``positions``: int32 [s] or [b,s] on the GPU, or the first one of
    s that follow each other.  Any strides, rows contiguous.  ``out``: (q', k') to write to, each of them its input or a view
    that has no element in common with an input, and none with the other (parts of one projection may lie between each other);
    else new contiguous tensors.  ``transpose`` turns back: the gradient of the turn.  Returns (q', k'), or q' without a k."""
    pos = positions if isinstance(positions, torch.Tensor) else None
    dev = _on_one_gpu(q, k, pos, plan.inv_freq)
    b, hq, s, d = q.shape
    hk = 0
    if k is not None:
        hk = k.shape[1]
        if k.shape != (b, hk, s, d) or k.dtype != q.dtype:
            raise ValueError(f"k is {tuple(k.shape)} {k.dtype} beside q {tuple(q.shape)} {q.dtype}")
    if (b | hq | hk | d) >> 31:
        _too_large(b, hq, hk, d)
    if plan.rotary_dim > d:
        raise ValueError(f"a plan of {plan.rotary_dim} elements for heads of {d}")
    dt = _dt(q)
    pos_stride, first = 0, 0
    if pos is None:
        first = int(positions)
        if not -2 ** 31 <= first <= first + max(s - 1, 0) < 2 ** 31:
            raise ValueError(f"positions {first} .. beyond 32 bits")
    else:
        _expect("positions", pos, (b, s) if pos.dim() == 2 else (s,), torch.int32, contiguous=False)
        if s > 1 and pos.stride(-1) != 1:
            raise ValueError("positions of a sequence must be contiguous")
        if pos.dim() == 2:
            pos_stride = pos.stride(0)
    if out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        k_out = None if k is None else torch.empty_like(k, memory_format=torch.contiguous_format)
    else:
        ys = tuple(out)[:1 if k is None else 2] if isinstance(out, (tuple, list)) else (out,)
        if len(ys) != (1 if k is None else 2) or any(y is None for y in ys):
            raise ValueError("out holds one tensor for q, and one for k if there is a k")
        _on_one_gpu(q, *ys)
        q_out, k_out = ys if k is not None else (ys[0], None)
        if q_out is not q:
            _expect("out", q_out, q.shape, q.dtype, contiguous=False)
        if k_out is not k:
            _expect("out", k_out, k.shape, k.dtype, contiguous=False)
    strides = (*_row_strides("q", q, b, hq, s, d), *_row_strides("out", q_out, b, hq, s, d))
    if k is not None:
        strides += (*_row_strides("k", k, b, hk, s, d), *_row_strides("out", k_out, b, hk, s, d))
    if out is not None and b * s * d > 0:
        _refuse_overlaps(q.element_size(), b, s, d, (q, q_out, k, k_out), (hq, hq, hk, hk), strides, pos, pos_stride, plan.inv_freq)
    if b * s > 0:
        _launch(dev, _lib.load().lrqk_rotary, q.data_ptr(), _ptr(k), q_out.data_ptr(), _ptr(k_out),
                struct.pack(f"{len(strides)}q", *strides), _ptr(pos), pos_stride, first, plan.inv_freq.data_ptr(), plan.factor,
                b, hq, hk, s, d, plan.rotary_dim, plan.interleaved, transpose, dt)
    return q_out if k is None else (q_out, k_out)


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
                   mask: torch.Tensor, lengths: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                   return_lse: bool = False):
    """Attention of t drafted tokens over the cached ones and over each other.

    q [b,Hq,t,d]; k_cache, v_cache [b,Hc,n,d], of which sequence i has ``lengths[i]`` tokens (int32 [b] on the GPU; all n if
    None), any strides that both share, rows contiguous; k_new, v_new [b,Hn,t,d] of the drafted tokens; mask bool or uint8
    [t,t] or [b,t,t]: drafted token i sees j.  Hc = Hn for a dense cache, Hc = Hq for an active set (``engine.Kgpu``).
    ``scale`` (1 / sqrt(d) if None) is positive.  Probabilities meet bf16 values as two bf16 numbers each, and beyond 128
    queries a cache head (Hq / Hc * t) as one: an output then moves by up to 2^-8 of the mean of |v - out| (pass float32
    tensors where that is too much), lse not at all.  -> [b,Hq,t,d], zeros for a token that sees nothing; with ``return_lse``
    also fp32 [b,Hq,t], the logarithm of the sum of the exponentials (-inf for such a token)."""
    dev = _on_one_gpu(q, k_cache, v_cache, k_new, v_new, mask, lengths)
    b, hq, t, d = q.shape
    _, hc, n, _ = k_cache.shape
    hn = k_new.shape[1]
    if (b | hq | hc | hn | t | d) >> 31:
        _too_large(b, hq, hc, hn, t, d)
    dt, dtype = _dt(q), q.dtype
    _expect("k_cache", k_cache, (b, hc, n, d), dtype, contiguous=False)
    _expect("v_cache", v_cache, (b, hc, n, d), dtype, contiguous=False)
    _expect("k_new", k_new, (b, hn, t, d), dtype, contiguous=False)
    _expect("v_new", v_new, (b, hn, t, d), dtype, contiguous=False)
    if hc == 0 or hn == 0 or hq % hc or hc % hn:
        raise ValueError(f"{hq} query heads, {hc} heads of the cache, {hn} of the drafted tokens: each a multiple of the next")
    if mask.shape not in ((b, t, t), (t, t)) or mask.dtype not in (torch.bool, torch.uint8):
        raise ValueError(f"mask is {tuple(mask.shape)} {mask.dtype}: bool or uint8 [t,t] or [b,t,t] is wanted")
    _lengths(lengths, b)
    st, sv = _row_strides("k_cache", k_cache, b, hc, n, d), _row_strides("v_cache", v_cache, b, hc, n, d)
    if sv != st and n > 0:
        raise ValueError("k_cache and v_cache must have the same strides")
    q = _rows16(q)
    out = torch.empty_like(q)
    lse = torch.empty((b, hq, t), dtype=torch.float32, device=q.device) if return_lse else None
    if b * hq * t:
        k_new, v_new, mask = _rows16(k_new), _rows16(v_new), mask.contiguous()
        need = _scratch_bytes("lrqk_tree_attention_workspace", b, hq, hc, t, n, d, lengths is not None, dt)
        ws = _scratch(need, q)
        _launch(dev, _lib.load().lrqk_tree_attention, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), *st, n, _ptr(lengths),
                k_new.data_ptr(), v_new.data_ptr(), mask.data_ptr(), t * t if mask.dim() == 3 else 0, out.data_ptr(), _ptr(lse), b,
                hq, hc, hn, t, d, d ** -0.5 if scale is None else float(scale), ws.data_ptr(), need, dt)
    return (out, lse) if return_lse else out


def attention_weights(q: torch.Tensor, k: torch.Tensor, lengths: Optional[torch.Tensor] = None,
                      lse: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                      weights: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """What attention every cached token got from the last t tokens of its sequence, added to ``weights``.

    q [b,Hq,t,d] of those tokens; k [b,Hc,n,d], of which sequence i has ``lengths[i]`` tokens (n if None), any strides, rows
    contiguous; a token sees those up to itself.  lse fp32 [b,Hq,t]: the logarithms of its sums that the attention left
    (``tree_attention(return_lse=True)``; a query of -inf adds nothing); without it they are formed here.  -> fp32 [b,Hc,n]:
    ``weights`` (0 if None) plus the sums over the query heads of each head and over the tokens, in ``out`` if that is given,
    else in place if there are weights.  That place may be the weights' own, and is apart from the other inputs."""
    dev = _on_one_gpu(q, k, lengths, lse, weights, out)
    b, hq, t, d = q.shape
    hc, n = k.shape[1], k.shape[2]
    if (b | hq | hc | t | d) >> 31:
        _too_large(b, hq, hc, t, d)
    dt = _dt(q)
    _expect("k", k, (b, hc, n, d), q.dtype, contiguous=False)
    if hc == 0 or hq % hc:
        raise ValueError(f"{hq} query heads over {hc} heads of the cache")
    _lengths(lengths, b)
    if lse is not None:
        _expect("lse", lse, (b, hq, t), torch.float32)
    if weights is not None:
        _expect("weights", weights, (b, hc, n), torch.float32)
    fresh = out is None and weights is None
    if out is not None:
        _expect("out", out, (b, hc, n), torch.float32)
    else:
        out = torch.empty((b, hc, n), dtype=torch.float32, device=q.device) if fresh else weights
    w_at, out_at = _ptr(weights), out.data_ptr()
    if w_at is not None and 0 < abs(w_at - out_at) < 4 * b * hc * n:
        raise ValueError("out overlaps weights")
    if b * n == 0:
        return out
    if t == 0:
        return out.copy_(weights) if weights is not None else out.zero_()
    q, strides = _rows16(q), _row_strides("k", k, b, hc, n, d)
    q_at, k_at, l_at, lse_at = q.data_ptr(), k.data_ptr(), _ptr(lengths), _ptr(lse)
    if not fresh:   # (all contiguous but k)
        e, end = q.element_size(), out_at + 4 * b * hc * n
        k_end = k_at + e * ((b - 1) * strides[0] + (hc - 1) * strides[1] + (n - 1) * strides[2] + d)
        if (q_at < end and out_at < q_at + e * b * hq * t * d or k_at < end and out_at < k_end or
                l_at is not None and l_at < end and out_at < l_at + 4 * b or
                lse_at is not None and lse_at < end and out_at < lse_at + 4 * b * hq * t):
            raise ValueError("the place of the sums overlaps an input")
    need = _scratch_bytes("lrqk_attention_weights_workspace", b, hq, hc, t, n, d, lse is not None, dt)
    ws = _scratch(need, q) if need else None
    _launch(dev, _lib.load().lrqk_attention_weights, q_at, k_at, *strides, n, l_at, lse_at, w_at, out_at, b, hq,
            hc, t, d, d ** -0.5 if scale is None else float(scale), _ptr(ws), need, dt)
    return out


def evict(weights: torch.Tensor, ids: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lengths: Optional[torch.Tensor],
          budget: int, recent: int, out=None) -> torch.Tensor:
    """Brings a cache down to ``budget`` tokens a head by what attention they got.

    weights fp32 and ids int32 [b,H,n] (the position of every slot's token), k, v [b,H,n,d], of which sequence i has
    ``lengths[i]`` tokens (int32 [b]; n if None).  The tokens whose ids are within ``recent`` of their head's largest one
    stay, and of the others those with the largest weights (equal ones: of the lowest slots).  A token that stays keeps its
    slot if that is one of the first ``budget``; the others move, in order, into the slots that became free.  In place, or
    into ``out`` = (weights, ids, k, v), buffers of at least min(budget, n) slots that are apart from the inputs and from each
    other; slots behind the tokens that stay are left as they were.  -> the new lengths, int32 [b]."""
    dev = _on_one_gpu(weights, ids, k, v, lengths, *(out or ()))
    b, h, n, d = k.shape
    if (b | h | n | d) >> 31:
        _too_large(b, h, n, d)
    dt = _dt(k)
    _expect("weights", weights, (b, h, n), torch.float32)
    _expect("ids", ids, (b, h, n), torch.int32)
    if not k.is_contiguous():
        raise ValueError("k must be contiguous")
    _expect("v", v, (b, h, n, d), k.dtype)
    _lengths(lengths, b)
    budget, recent, cap_out = int(budget), int(recent), n
    if budget < 1 or not 0 <= recent <= budget:
        raise ValueError(f"budget={budget}, recent={recent}: 0 <= recent <= budget and at least one token are wanted")
    ptrs = (None,) * 4
    if out is not None:
        if len(out) != 4 or out[2].dim() != 4:
            raise ValueError("out holds weights, ids, k and v")
        cap_out = out[2].shape[2]
        if cap_out >> 31:
            _too_large(cap_out)
        for name, y, shape, dtype in zip(("weights", "ids", "k", "v"), out, ((b, h, cap_out),) * 2 + ((b, h, cap_out, d),) * 2,
                                         (torch.float32, torch.int32, k.dtype, k.dtype)):
            _expect("out " + name, y, shape, dtype)
        if cap_out < min(budget, n):
            raise ValueError(f"out has {cap_out} slots for min(budget={budget}, {n}) tokens")
        ptrs = tuple(y.data_ptr() for y in out)
    new = torch.empty_like(lengths) if lengths is not None else torch.empty((b,), dtype=torch.int32, device=k.device)
    slots = b * h * n
    if slots == 0:
        return new.zero_()
    # (all are contiguous, so that ranges say it: asked for tensor by tensor this took longer than the kernels)
    held = w_at, i_at, k_at, v_at = weights.data_ptr(), ids.data_ptr(), k.data_ptr(), v.data_ptr()
    l_at, l_bytes = (0, 0) if lengths is None else (lengths.data_ptr(), 4 * b)
    row = d * k.element_size()
    word, rows = 4 * slots, row * slots
    if out is None:   # (one tensor as keys and values: every row is moved to one place)
        apart = (abs(w_at - i_at) >= word and (k_at == v_at or abs(k_at - v_at) >= rows) and
                 not -word < w_at - k_at < rows and not -word < w_at - v_at < rows and
                 not -word < i_at - k_at < rows and not -word < i_at - v_at < rows and
                 not -l_bytes < l_at - w_at < word and not -l_bytes < l_at - i_at < word and
                 not -l_bytes < l_at - k_at < rows and not -l_bytes < l_at - v_at < rows)
    else:
        ranges = [(w_at, word, False), (i_at, word, False), (k_at, rows, False), (v_at, rows, False), (l_at, l_bytes, False)]
        apart = _undisturbed(ranges + [(p, b * h * cap_out * size, True) for p, size in zip(ptrs, (4, 4, row, row))])
    if not apart:
        raise ValueError("what is written overlaps something else (in place: leave out away)")
    budget = min(budget, 2 ** 30)
    need = _scratch_bytes("lrqk_evict_workspace", b, h, n, budget)
    ws = _scratch(need, k)
    _launch(dev, _lib.load().lrqk_evict, *held, l_at or None, n, *ptrs, cap_out, new.data_ptr(),
            b, h, d, budget, min(recent, budget), ws.data_ptr(), need, dt)
    return new


_SIX = struct.Struct("6q")


class ByteCache:
    """Keys and values of ``heads`` heads of ``batch`` sequences in 8 bits, room for ``capacity`` tokens (rounded up to whole blocks).

    A block is 64 tokens of a head and has one scale for its keys and one for its values; an element is code * scale.  ``kind``:
    "int8", whole numbers up to 127, or "fp8", e4m3 numbers up to 448 (elements of very different sizes keep their bits).
    ``k`` [b,H,blocks,64,w] and ``v`` [b,H,blocks,w,64] hold the codes (w: head_dim rounded up to 64, 128 or 256; the rest is 0),
    ``k_scale`` and ``v_scale`` fp32 [b,H,blocks]; ``k_tail`` and ``v_tail`` [b,H,128,d], in ``dtype`` (what queries and new tokens
    come in), the last 128 tokens as they came, token p in row p % 128.  A block is coded once, when its last token arrives; until
    then its tokens are read from the tail.  Lengths are the caller's (int32 [b] on the device), as of the other caches here, and
    so is the order of calls on one cache: those that write it and those that read it come one after the other."""

    BLOCK, TAIL = 64, 128
    _CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}

    def __init__(self, batch: int, heads: int, capacity: int, head_dim: int, dtype=torch.bfloat16, kind: str = "int8", device="cuda:0"):
        if kind not in self._CODES:
            raise ValueError(f"unknown kind {kind!r}: one of {sorted(self._CODES)}")
        if dtype not in (torch.bfloat16, torch.float32):
            raise ValueError(f"unsupported dtype {dtype}: the kernels store float32 or bfloat16")
        step = 8 if dtype == torch.bfloat16 else 4
        if min(batch, heads, capacity, head_dim) < 1 or head_dim > 256 or head_dim % step:
            raise ValueError(f"batch={batch}, heads={heads}, capacity={capacity}, head_dim={head_dim}: at least 1 each, and rows of whole "
                             "16-byte pieces, at most 256 elements")
        blocks, w = -(-capacity // self.BLOCK), 64 if head_dim <= 64 else 128 if head_dim <= 128 else 256
        if blocks > 2 ** 24:
            raise ValueError(f"capacity={capacity}: at most 2^30 tokens")
        self.kind, self.dtype, self.head_dim, self.capacity = kind, dtype, head_dim, blocks * self.BLOCK
        k = torch.zeros((batch, heads, blocks, self.BLOCK, w), dtype=self._CODES[kind], device=device)
        v = torch.zeros((batch, heads, blocks, w, self.BLOCK), dtype=self._CODES[kind], device=device)
        scales = (torch.ones((batch, heads, blocks), device=device) for _ in range(2))
        tails = (torch.zeros((batch, heads, self.TAIL, head_dim), dtype=dtype, device=device) for _ in range(2))
        self._sizes = (batch, heads, blocks, head_dim)
        self._code = _lib.CODES[kind]
        self._hold((k, v, *scales, *tails))

    def _hold(self, buffers):
        """What the calls are given: the places of these buffers, which never become others."""
        self._buffers = buffers
        self._dev = buffers[0].get_device()
        self._places = tuple(x.data_ptr() for x in buffers)
        self._ranges = tuple((x.data_ptr(), x.data_ptr() + x.nbytes) for x in buffers)

    def __setstate__(self, state):   # (a copy has buffers of its own)
        self.__dict__.update(state)
        self._hold(self._buffers)

    k, v, k_scale, v_scale, k_tail, v_tail = (property(lambda self, i=i: self._buffers[i]) for i in range(6))

    def _on(self, dev: int):
        if dev != self._dev:
            raise ValueError(f"the cache is on {self.k.device}, tensors on device {dev}")
        return self._sizes


def byte_append(cache: ByteCache, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor, counts: Optional[torch.Tensor] = None,
                path: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Writes tokens behind the ``lengths`` (int32 [b]) that the sequences of ``cache`` have, and returns the new lengths.

    k, v [b,H,t,d]: any strides, rows contiguous.  ``counts`` int32 [b]: how many of them (all t if None; at most what there is room
    for).  ``path`` int32 [b,m]: which rows, in order (0, 1, .. if None; counts up to m, ids outside the rows count as the nearest):
    ``verify_drafts`` gives both.  ``lengths`` is not changed: appending again from it writes the same again as long as that is at most
    64 tokens.  (A sequence may also be made shorter: to whole blocks, or to where the block that it then ends in lies in the
    tail as a whole.)  k and v are apart from the cache.  A block's codes: scale = amax / 127 (int8) or the smallest power of two with amax / scale <= 448 (fp8), of its
    finite elements and at least 2^-100, code = element / scale rounded once, half to even; infinities get the largest code, NaN 0."""
    dev = _on_one_gpu(k, v, lengths, counts, path)
    b, h, blocks, d = cache._on(dev)
    t, dtype = k.shape[2] if k.dim() == 4 else 0, cache.dtype
    if t >> 31:
        _too_large(t)
    _expect("k", k, (b, h, t, d), dtype, contiguous=False)
    _expect("v", v, (b, h, t, d), dtype, contiguous=False)
    _expect("lengths", lengths, (b,), torch.int32)
    most, path_at, path_stride = t, None, 0
    if path is not None:
        if path.dim() != 2 or path.shape[0] != b or path.dtype != torch.int32 or (path.shape[1] > 1 and path.stride(1) != 1):
            raise ValueError(f"path is {tuple(path.shape)} {path.dtype}: int32 [{b},m] with contiguous rows is wanted")
        most, path_at = path.shape[1], path.data_ptr()
        if most >> 31:
            _too_large(most)
        if b > 1:
            path_stride = path.stride(0)
    if counts is not None:
        _expect("counts", counts, (b,), torch.int32)
    if t == 0 or most == 0:
        return lengths.clone()
    k_at, v_at = k.data_ptr(), v.data_ptr()
    ks, vs = _row_strides("k", k, b, h, t, d), _row_strides("v", v, b, h, t, d)
    step = 7 if dtype == torch.bfloat16 else 3   # (elements of 16 bytes, less one)
    if (k_at | v_at) & 15 or (ks[0] | ks[1] | ks[2] | vs[0] | vs[1] | vs[2]) & step:
        k, v = _rows16(k), _rows16(v)
        k_at, v_at, ks, vs = k.data_ptr(), v.data_ptr(), _row_strides("k", k, b, h, t, d), _row_strides("v", v, b, h, t, d)
    e = 16 // (step + 1)
    k_end = k_at + e * ((b - 1) * ks[0] + (h - 1) * ks[1] + (t - 1) * ks[2] + d)
    v_end = v_at + e * ((b - 1) * vs[0] + (h - 1) * vs[1] + (t - 1) * vs[2] + d)
    for lo, hi in cache._ranges:
        if k_at < hi and lo < k_end or v_at < hi and lo < v_end:
            raise ValueError("k or v overlaps the cache")
    new = torch.empty_like(lengths)
    _launch(dev, _lib.load().lrqk_byte_append, k_at, v_at, _SIX.pack(*ks, *vs), t, most, lengths.data_ptr(),
            None if counts is None else counts.data_ptr(), path_at, path_stride, new.data_ptr(), *cache._places, blocks, b, h, d, cache._code,
            _lib.F32 if step == 3 else _lib.BF16)
    return new


def byte_attention(q: torch.Tensor, cache: ByteCache, lengths: torch.Tensor, k_new: Optional[torch.Tensor] = None,
                   v_new: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                   return_lse: bool = False):
    """``tree_attention`` over a cache held in 8 bits: q [b,Hq,t,d] attends to the first ``lengths`` (int32 [b] on the GPU) tokens of
    the sequences of ``cache``, and to the drafted tokens k_new, v_new [b,Hn,t,d] as mask (bool or uint8 [t,t] or [b,t,t]: drafted token i
    sees j) says; without these three to the cached ones alone.  Every number of heads is a multiple of the next: Hq, the
    cache's, Hn.  ``scale`` (1 / sqrt(d) if None) is positive.  Codes are multiplied as they are, with probabilities of 11 bits (bf16
    tensors) or 22 (float32); the tail's and the drafted tokens' rows with 16 or 24.  -> [b,Hq,t,d], zeros for a token that sees
    nothing; with ``return_lse`` also fp32 [b,Hq,t], the logarithm of the sum of the exponentials (-inf for such a token)."""
    dev = _on_one_gpu(q, lengths, k_new, v_new, mask)
    cb, hc, blocks, cd = cache._on(dev)
    b, hq, t, d = q.shape
    if (b | hq | t | d) >> 31:
        _too_large(b, hq, t, d)
    dtype = cache.dtype
    if b != cb or d != cd or q.dtype != dtype:
        raise ValueError(f"q is {tuple(q.shape)} {q.dtype}: [{cb},Hq,t,{cd}] {dtype} is wanted")
    if hq % hc:
        raise ValueError(f"{hq} query heads over {hc} heads of the cache")
    _expect("lengths", lengths, (b,), torch.int32)
    hn = hc
    if k_new is None or v_new is None or mask is None:
        if not (k_new is None and v_new is None and mask is None):
            raise ValueError("drafted keys, values and their mask come together")
    else:
        hn = k_new.shape[1]
        _expect("k_new", k_new, (b, hn, t, d), dtype, contiguous=False)
        _expect("v_new", v_new, (b, hn, t, d), dtype, contiguous=False)
        if hn == 0 or hc % hn:
            raise ValueError(f"{hc} heads of the cache, {hn} of the drafted tokens: a multiple")
        if mask.shape not in ((b, t, t), (t, t)) or mask.dtype not in (torch.bool, torch.uint8):
            raise ValueError(f"mask is {tuple(mask.shape)} {mask.dtype}: bool or uint8 [t,t] or [b,t,t] is wanted")
    q = _rows16(q)
    out = torch.empty_like(q)
    lse = q.new_empty((b, hq, t), dtype=torch.float32) if return_lse else None
    if b * hq * t:
        each, kn_at, vn_at, mask_at = 0, None, None, None
        if k_new is not None:
            k_new, v_new, mask = _rows16(k_new), _rows16(v_new), mask.contiguous()
            kn_at, vn_at, mask_at = k_new.data_ptr(), v_new.data_ptr(), mask.data_ptr()
            each = t * t if mask.dim() == 3 else 0
        dt = _lib.F32 if dtype == torch.float32 else _lib.BF16
        need = _scratch_bytes("lrqk_byte_attention_workspace", b, hq, hc, t, blocks, d, dt)
        ws = lengths.new_empty(need // 4)   # (of whole 4-byte words)
        _launch(dev, _lib.load().lrqk_byte_attention, q.data_ptr(), *cache._places, blocks, lengths.data_ptr(), kn_at, vn_at, mask_at, each,
                out.data_ptr(), None if lse is None else lse.data_ptr(), b, hq, hc, hn, t, d, d ** -0.5 if scale is None else float(scale),
                cache._code, ws.data_ptr(), need, dt)
    return (out, lse) if return_lse else out


def verify_drafts(tokens: torch.Tensor, target: torch.Tensor, uniforms: torch.Tensor, draft: Optional[torch.Tensor] = None,
                  parents: Optional[torch.Tensor] = None):
    """The accepted path of a tree of drafted tokens, and the token that follows it, from given random numbers: what is accepted and
    drawn has the target's distribution.

    tokens int32 [b,s] (as all whole numbers here): node 0 of a sequence's tree is certain, node i was drawn from row parents[i] of ``draft``, every child of a
    node for itself.  ``parents`` int32 [b,s]: a node in front of its children (None: a chain, i - 1; a node whose parent is not in
    front of it is never reached).  target [b,s,V], row i the probabilities behind node i; draft [b,s,V] or [b,s-1,V], or None for
    drafts without probabilities (looked up: equal ones among a node's children count once).  Both fp32 or bf16, rows contiguous.
    ``uniforms`` fp32 [b,s], in [0,1): the first for the token that follows, the others for their nodes' tests.

    At a node the children are looked at in order with what is left of its distribution, r of mass Z (first: its row of target,
    1): token x is accepted if u draft[x] Z < r[x] (without draft: u Z < r[x]), else r becomes max(r - Z draft, 0) and Z
    its sum (without draft: r without x and Z less r[x], that is 1 less what the refused tokens had, whatever the row adds up
    to).  The token that follows is the lowest x with r[0] + .. + r[x] > u sum(r) at the last accepted node (of its row of target
    if nothing is left, -1 if that has nothing).  In fp64; what is not a positive number counts as 0, a token outside the
    vocabulary as one of probability 0.
    -> path int32 [b,s] (accepted nodes, 0 first, -1 behind them), counts int32 [b], the token that follows int32 [b]:
    ``byte_append`` takes the first two as they are."""
    dev = _on_one_gpu(target, tokens, uniforms, draft, parents)
    b, s, vocab = target.shape
    if (b | s | vocab) >> 31:
        _too_large(b, s, vocab)
    dt = _dt(target)
    _expect("tokens", tokens, (b, s), torch.int32)
    _expect("uniforms", uniforms, (b, s), torch.float32)
    if parents is not None:
        _expect("parents", parents, (b, s), torch.int32)
    if vocab > 1 and target.stride(2) != 1:
        raise ValueError("the rows of target must be contiguous")
    draft_strides = (0, 0)
    if draft is not None:
        if draft.shape != (b, s, vocab) and draft.shape != (b, max(s - 1, 0), vocab) or draft.dtype != target.dtype:
            raise ValueError(f"draft is {tuple(draft.shape)} {draft.dtype}: {(b, s, vocab)} or a row less, {target.dtype} is wanted")
        if vocab > 1 and draft.stride(2) != 1:
            raise ValueError("the rows of draft must be contiguous")
        draft_strides = draft.stride()[:2]
    path, counts, token = torch.empty_like(tokens), tokens.new_empty(b), tokens.new_empty(b)
    if b == 0:
        return path, counts, token
    if s == 0 or vocab == 0:
        raise ValueError(f"{s} nodes over a vocabulary of {vocab}: at least 1 each")
    need = _scratch_bytes("lrqk_verify_drafts_workspace", b, s, vocab)
    ws = tokens.new_empty(need // 4)   # (of whole 8-byte words)
    st = target.stride()
    _launch(dev, _lib.load().lrqk_verify_drafts, tokens.data_ptr(), _ptr(parents), target.data_ptr(), st[0], st[1],
            draft.data_ptr() if draft is not None and s > 1 else None, *draft_strides, uniforms.data_ptr(), path.data_ptr(),
            counts.data_ptr(), token.data_ptr(), b, s, vocab, ws.data_ptr(), need, dt)
    return path, counts, token


def probe_bandwidth(nbytes: int, reps: int = 10, device="cuda:0"):
    """(read GB/s, copy GB/s of bytes read + bytes written) of plain streaming kernels over ``nbytes``."""
    src = torch.empty(nbytes, dtype=torch.uint8, device=device).fill_(1)
    dst = torch.empty_like(src)
    r_ms, c_ms = ctypes.c_double(), ctypes.c_double()
    check(_lib.load().lrqk_probe_bandwidth(src.data_ptr(), dst.data_ptr(), nbytes, reps, ctypes.byref(r_ms),
                                           ctypes.byref(c_ms), _stream(src)))
    return nbytes / (r_ms.value * 1e-3) / 1e9, 2 * nbytes / (c_ms.value * 1e-3) / 1e9


def probe_read_sweep(nbytes: int, reps: int = 5, device="cuda:0", slice_bytes: int = 0):
    """The plain read over ``nbytes`` in every variant (4 / 8 / 16 vectors in flight, plain / non-temporal loads,
    1 .. 8 workgroups per CU): ({(in_flight, nontemporal, grid_per_cu): GB/s}, best GB/s).  With ``slice_bytes`` a
    launch reads one slice of the buffer and the launches take the slices in turn: the rate of launches of that size."""
    src = torch.empty(nbytes, dtype=torch.uint8, device=device).fill_(1)
    sink = torch.zeros(1 << 16, dtype=torch.uint8, device=device)
    table = {}
    ms = ctypes.c_double()
    per_launch = slice_bytes or nbytes
    n = reps * (nbytes // slice_bytes) if slice_bytes else reps
    for nt in (0, 1):
        for fl in (4, 8, 16):
            for per_cu in (1, 2, 4, 8):
                check(_lib.load().lrqk_probe_read_variant(src.data_ptr(), sink.data_ptr(), nbytes, slice_bytes, min(n, 1000), fl,
                                                          nt, per_cu, ctypes.byref(ms), _stream(src)))
                table[(fl, nt, per_cu)] = per_launch / (ms.value * 1e-3) / 1e9
    return table, max(table.values())


def probe_event_pair(reps: int = 64, device="cuda:0", kernels: int = 1) -> float:
    """Microseconds that a pair of HIP events reads around ``kernels`` launches that do nothing (average of ``reps``
    pairs)."""
    us = ctypes.c_double()
    with torch.cuda.device(device):
        check(_lib.load().lrqk_probe_event_pair(reps, kernels, ctypes.byref(us),
                                                torch.cuda.current_stream().cuda_stream))
    return us.value


# --------------------------------------------------------------------------- host gathers

def d0_index_select(src: torch.Tensor, indices: torch.Tensor, threads: int = 8) -> torch.Tensor:
    """Host row gather into a new pinned tensor: out[i] = src[indices[i]].  src [N,w] CPU, indices int64 [n]."""
    if src.is_cuda or indices.is_cuda:
        raise ValueError("d0_index_select gathers host rows; tensors must be on the CPU")
    src = src.contiguous()
    idx = indices.to(torch.int64).contiguous()
    pin = torch.cuda.is_available()
    out = torch.empty((idx.shape[0], src.shape[1]), dtype=src.dtype, pin_memory=pin)
    check(_lib.load().lrqk_d0_indices_select(out.data_ptr(), src.data_ptr(), idx.data_ptr(), idx.shape[0],
                                             src.shape[1] * src.element_size(), src.shape[0], threads))
    return out


def take_along_dim_with_mask(src: torch.Tensor, indices: torch.Tensor, mask: torch.Tensor, threads: int = 8):
    """src [b,Hkv,seq,w] CPU; indices int64, mask bool [b,Hkv,g,k] CPU -> [sum(mask), w]."""
    for name, t in (("src", src), ("indices", indices), ("indices_mask", mask)):
        if t.is_cuda:
            raise RuntimeError(f"{name} must be a CPU tensor")
        if not t.is_contiguous():
            raise RuntimeError(f"{name} must be contiguous")
    if indices.dtype != torch.int64:
        raise RuntimeError("indices must be int64")
    if mask.dtype != torch.bool:
        raise RuntimeError("mask must be bool")
    if src.dim() != 4 or indices.dim() != 4:
        raise RuntimeError("src [bsz, kv_heads, seq_len, hdim]; indices [bsz, kv_heads, num_groups, k]")
    if mask.shape != indices.shape:
        raise RuntimeError("shape mask != indices")
    b, hkv, seq, w = src.shape
    _, _, g, k = indices.shape
    mk = mask.view(torch.uint8)
    lib = _lib.load()
    rb = w * src.element_size()
    total = check(lib.lrqk_take_along_dim_with_mask(None, src.data_ptr(), indices.data_ptr(), mk.data_ptr(), b, hkv, g,
                                                    k, seq, rb, threads))
    out = torch.empty((total, w), dtype=src.dtype)
    if total:
        check(lib.lrqk_take_along_dim_with_mask(out.data_ptr(), src.data_ptr(), indices.data_ptr(), mk.data_ptr(), b,
                                                hkv, g, k, seq, rb, threads))
    return out
