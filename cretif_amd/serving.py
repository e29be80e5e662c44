"""Serving a batch from a paged cache: cri_qk_norm_rope, cri_paged_append, cri_paged_attention and
cri_verify_drafts of include/cri.h over torch tensors.  No counterpart in the reference, which
decodes one sequence over a contiguous cache.

Row buffers are fp32 device tensors [rows, width] (or [rows, heads, head_dim]) whose rows may be
strided, such as the columns of a fused q/k/v product; or a tuple (address, ld) with n_rows given.
The descriptors Rotation, PagedKV and PagedBatch keep their tensors alive and are made once; what
the tensors hold is read by the kernels.  Everything must be on the current device.
"""
from __future__ import annotations

import ctypes

_vp, _i32, _i64, _f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float

PAIRS = {"adjacent": 0, "halves": 1}


class _PagedKV(ctypes.Structure):
    _fields_ = [("k", _vp), ("v", _vp), ("page_stride", _i64), ("type", _i32), ("n_pages", _i32), ("page_size", _i32),
                ("n_kv_heads", _i32), ("head_dim", _i32)]


class _PagedBatch(ctypes.Structure):
    _fields_ = [("offsets", _vp), ("lens", _vp), ("pages", _vp), ("n_seqs", _i32), ("n_rows", _i32), ("max_pages", _i32)]


class _Rotation(ctypes.Structure):
    _fields_ = [("q_norm", _vp), ("k_norm", _vp), ("eps", _f32), ("theta", _f32), ("rot_dim", _i32), ("pairs", _i32)]


SYMBOLS = {
    "cri_qk_norm_rope": ([_vp, _vp, _i32, _vp, _i32, _vp, _i32, _vp, _i32, _vp, _i32, _i32, _i32, _i32, _vp], _i32),
    "cri_paged_append": ([_vp, _vp, _vp, _vp, _i32, _vp, _i32, _i32, _vp, _i32, _vp, _i32, _vp], _i32),
    "cri_paged_attention": ([_vp, _vp, _vp, _i32, _vp, _i32, _vp, _i32, _i32, _f32, _vp, _i64, _vp], _i32),
    "cri_paged_attention_workspace_bytes": ([_vp, _vp, _i32, _i32], _i64),
    "cri_verify_drafts": ([_vp, _i64, _vp, _i64, _vp, _vp, _vp, _vp, _i32, _i32, _i32, _vp, _vp, _vp, _i64, _vp], _i32),
    "cri_verify_drafts_workspace_bytes": ([_i32, _i32], _i64),
}


def declare(L):
    for name, (args, res) in SYMBOLS.items():
        f = getattr(L, name)
        f.argtypes, f.restype = args, res


def _device():
    try:
        return torch._C._cuda_getDevice()
    except RuntimeError:  # no GPU: the buffers' own checks say so
        return None


def _on_device(t, name, dev=None):
    """The tensor's address; it must be on the current GPU."""
    d = t.get_device()
    if d < 0:
        raise ValueError("%s is on %s; the HIP kernels need device (cuda) tensors" % (name, t.device))
    if d != (_device() if dev is None else dev):
        raise ValueError("%s is on %s, not on the current device" % (name, t.device))
    return t.data_ptr()


def _all_on(dev, *descriptors):
    """What the descriptors hold must be on the device that is current at the call, too."""
    for d in descriptors:
        if d._dev is not None and d._dev != dev:
            raise ValueError("the tensors of a %s are on cuda:%d, not on the current device" % (type(d).__name__, d._dev))


def _rows(t, width, name, dev):
    """(address, floats from row to row, rows or None) of a row buffer of `width` floats a row."""
    if type(t) is tuple:
        return t[0], t[1], None
    sh, st = t.shape, t.stride()
    if len(sh) == 2:  # the usual case first
        n, w = sh
        ld, one = st
        if w == width and one == 1 and t.dtype is torch.float32 and t.get_device() == dev:
            return t.data_ptr(), ld if n > 1 else width, n  # (the stride of a single row says nothing)
    if t.dtype is not torch.float32:
        raise ValueError("%s must be float32, not %s" % (name, t.dtype))
    if len(sh) not in (2, 3):
        raise ValueError("%s must have the shape [rows, width] or [rows, heads, head_dim]" % name)
    inner, wide = sh[-1], sh[1] * (sh[2] if len(sh) == 3 else 1)
    if wide != width:
        raise ValueError("%s has rows of %d floats, not %d" % (name, wide, width))
    if (inner > 1 and st[-1] != 1) or (len(sh) == 3 and sh[1] > 1 and st[1] != inner):
        raise ValueError("%s: the elements of a row must be consecutive" % name)
    return _on_device(t, name, dev), st[0] if sh[0] > 1 else width, sh[0]


def _in_32_bits(*numbers):
    """Host numbers that C takes as int: ctypes would cut them to 32 bits without a word.  (The calls of a step ask first
    whether any has a bit from 31 on, 0.1 us; negative ones are C's to refuse.)"""
    if max(numbers) > 0x7FFFFFFF or min(numbers) < -0x80000000:
        raise ValueError("a size or a row stride does not fit 32 bits: %s" % (numbers,))


def _same_rows(n_rows, *named):
    for name, n in named:
        if n is not None and n != n_rows:
            if n_rows is not None:
                raise ValueError("%s has %d rows, not %d" % (name, n, n_rows))
            n_rows = n
    if n_rows is None:
        raise ValueError("n_rows must be given with (address, ld) buffers")
    return n_rows


def _ints(t, name, dims, dev=None):
    if t.dtype is not torch.int32 or t.dim() != dims or not t.is_contiguous():
        raise ValueError("%s must be a contiguous int32 tensor of %d dimension(s)" % (name, dims))
    if t.get_device() == dev:
        return t.data_ptr()
    return _on_device(t, name, dev)


def _room(workspace, dev):
    """(address, bytes) of a workspace."""
    if not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    return _on_device(workspace, "workspace", dev), workspace.nbytes


def _new_room(need, stream):
    if stream is not None:
        raise ValueError("give a workspace with an explicit stream (an allocated one belongs to the current stream)")
    return torch.empty(need, dtype=torch.uint8, device="cuda")


def _on(stream, dev):
    """The stream's address; the device's current stream when None (the buffers have initialised the GPU)."""
    return torch._C._cuda_getCurrentRawStream(dev) if stream is None else _stream(stream)


class Rotation:
    """Norms and rotation of query and key heads: norm weights [head_dim] (None: not normed), the
    rotation's base and its number of elements (0: no rotation), "adjacent" pairs (2 i, 2 i + 1) or
    "halves" (i, i + rot_dim / 2)."""

    def __init__(self, theta, rot_dim, pairs="adjacent", q_norm=None, k_norm=None, eps=1e-6):
        _torch()
        for w, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
            if w is not None and (w.dtype is not torch.float32 or w.dim() != 1 or not w.is_contiguous()):
                raise ValueError("%s must be a contiguous float32 tensor [head_dim]" % name)
        _in_32_bits(rot_dim)
        self.q_norm, self.k_norm = q_norm, k_norm
        self._c = _Rotation(None if q_norm is None else _on_device(q_norm, "q_norm"),
                            None if k_norm is None else _on_device(k_norm, "k_norm"), eps, theta, rot_dim, PAIRS[pairs])
        self._ref = ctypes.addressof(self._c)
        self._dev = None if q_norm is None and k_norm is None else _device()
        self._widths = {w.shape[0] for w in (q_norm, k_norm) if w is not None}

    def _fits(self, head_dim):
        if self._widths and self._widths != {head_dim}:
            raise ValueError("the norms have %s weights, not head_dim=%d" % (sorted(self._widths), head_dim))


class PagedKV:
    """A pool of pages: k and v [n_pages, page_size, n_kv_heads, head_dim], fp32, fp16 or bf16; pages
    may be strided (both pools alike), a page itself is contiguous."""

    def __init__(self, k, v):
        _torch()
        kinds = {torch.float32: 6, torch.float16: 5, torch.bfloat16: 7}
        if k.dtype not in kinds or k.dtype is not v.dtype:
            raise ValueError("k and v must both be float32, float16 or bfloat16")
        if k.dim() != 4 or k.shape != v.shape or k.stride() != v.stride():
            raise ValueError("k and v must both be [n_pages, page_size, n_kv_heads, head_dim], with the same strides")
        n, ps, h, d = k.shape
        _in_32_bits(n, ps, h, d)
        if n > 0 and not k[0].is_contiguous():
            raise ValueError("a page must be contiguous")
        self.k, self.v = k, v
        self.page_size, self.n_kv_heads, self.head_dim = ps, h, d
        stride = k.stride(0) if n > 1 else (ps * h * d + 7) // 8 * 8
        self._c = _PagedKV(_on_device(k, "k"), _on_device(v, "v"), stride, kinds[k.dtype], n, ps, h, d)
        self._ref = ctypes.addressof(self._c)
        self._dev = _device()


class PagedBatch:
    """A ragged batch: int32 offsets [n_seqs + 1], lens [n_seqs], pages [n_seqs, max_pages]."""

    def __init__(self, offsets, lens, pages):
        _torch()
        po, pl, pp = _ints(offsets, "offsets", 1), _ints(lens, "lens", 1), _ints(pages, "pages", 2)
        n = lens.shape[0]
        if offsets.shape[0] != n + 1 or pages.shape[0] != n:
            raise ValueError("offsets must have n_seqs + 1 entries, lens and pages n_seqs")
        _in_32_bits(n, pages.shape[1])
        self.offsets, self.lens, self.pages = offsets, lens, pages
        self._make = lambda rows: _PagedBatch(po, pl, pp, n, rows, pages.shape[1])
        self._by_rows = {}
        self._dev = _device()

    def _for(self, n_rows):
        """The descriptor of batches of n_rows rows, never changed.  Only the reference that the caller holds keeps it
        alive until its call is over: another thread may replace the kept one, or drop it when there are many."""
        c = self._by_rows.get(n_rows)
        if c is None:
            if len(self._by_rows) >= _KEPT:
                self._by_rows.clear()
            c = self._by_rows[n_rows] = self._make(n_rows)
        return c


_KEPT = 256  # row counts: a server's batches differ from step to step


def qk_norm_rope(rot, q, k, q_out, k_out, positions, n_heads, n_kv_heads, head_dim, n_rows=None, stream=None):
    """q_out and k_out = the heads of q and k, normed and rotated at positions [rows] (int32); q_out may
    be q and k_out k.  q (with n_heads 0) or k (with n_kv_heads 0) may be None."""
    L, dev = _torch(), _device()
    rot._fits(head_dim)
    _all_on(dev, rot)
    pq = lq = po = lo = pk = lk = px = lx = 0
    nq = no = nk = nx = None
    if q is not None:
        pq, lq, nq = _rows(q, n_heads * head_dim, "q", dev)
        po, lo, no = _rows(q_out, n_heads * head_dim, "q_out", dev)
    if k is not None:
        pk, lk, nk = _rows(k, n_kv_heads * head_dim, "k", dev)
        px, lx, nx = _rows(k_out, n_kv_heads * head_dim, "k_out", dev)
    pp = _ints(positions, "positions", 1, dev)
    n = _same_rows(n_rows, ("positions", positions.shape[0]), ("q", nq), ("k", nk), ("q_out", no), ("k_out", nx))
    if (lq | lo | lk | lx | n | n_heads | n_kv_heads | head_dim) >> 31:
        _in_32_bits(lq, lo, lk, lx, n, n_heads, n_kv_heads, head_dim)
    st = L.cri_qk_norm_rope(rot._ref, pq, lq, pk, lk, po, lo, px, lx, pp, n, n_heads, n_kv_heads, head_dim,
                            _on(stream, dev))
    if st:
        _check(st)


def paged_append(cache, batch, rot, k, v, q=None, q_out=None, n_heads=0, n_rows=None, stream=None):
    """The batch's k rows, normed and rotated, and v rows go to their pages; with q, its heads go to
    q_out, normed and rotated."""
    L, dev = _torch(), _device()
    D = cache.head_dim
    rot._fits(D)
    _all_on(dev, cache, batch, rot)
    pk, lk, nk = _rows(k, cache.n_kv_heads * D, "k", dev)
    pv, lv, nv = _rows(v, cache.n_kv_heads * D, "v", dev)
    pq = lq = po = lo = 0
    nq = no = None
    if q is not None:
        pq, lq, nq = _rows(q, n_heads * D, "q", dev)
        po, lo, no = _rows(q_out, n_heads * D, "q_out", dev)
    n = _same_rows(n_rows, ("k", nk), ("v", nv), ("q", nq), ("q_out", no))
    if (lq | lo | lk | lv | n | n_heads) >> 31:
        _in_32_bits(lq, lo, lk, lv, n, n_heads)
    st = L.cri_paged_append(cache._ref, ctypes.byref(batch._for(n)), rot._ref, pq, lq, po, lo, n_heads, pk, lk, pv, lv,
                            _on(stream, dev))
    if st:
        _check(st)


def paged_attention_workspace_bytes(cache, batch, n_rows, n_heads, prefix_len=0):
    """Workspace bytes of paged_attention for batches of these host numbers."""
    _in_32_bits(n_rows, n_heads, prefix_len)
    n = _torch().cri_paged_attention_workspace_bytes(cache._ref, ctypes.byref(batch._for(n_rows)), prefix_len, n_heads)
    if n < 0:
        _check(int(n))
    return int(n)


def paged_attention(cache, batch, q, out, n_heads, scale, prefix_pages=None, prefix_len=0, workspace=None, n_rows=None,
                    stream=None):
    """out = softmax(scale q K^T) V of every row over the positions it sees, those below prefix_len
    through prefix_pages, which all sequences share.  workspace: a device tensor of
    paged_attention_workspace_bytes (one is allocated when None)."""
    L, dev = _torch(), _device()
    width = n_heads * cache.head_dim
    _all_on(dev, cache, batch)
    pq, lq, nq = _rows(q, width, "q", dev)
    po, lo, no = _rows(out, width, "out", dev)
    n = _same_rows(n_rows, ("q", nq), ("out", no))
    if (lq | lo | n | n_heads | prefix_len) >> 31:
        _in_32_bits(lq, lo, n, n_heads, prefix_len)
    pp = 0
    if prefix_len > 0:
        if prefix_pages is None:
            raise ValueError("prefix_len without prefix_pages")
        pp = _ints(prefix_pages, "prefix_pages", 1, dev)
        if prefix_pages.shape[0] * cache.page_size < prefix_len:
            raise ValueError("prefix_pages holds %d pages, too few for prefix_len=%d" % (prefix_pages.shape[0], prefix_len))
    if workspace is None:
        workspace = _new_room(paged_attention_workspace_bytes(cache, batch, n, n_heads, prefix_len), stream)
    pw, wb = _room(workspace, dev)
    st = L.cri_paged_attention(cache._ref, ctypes.byref(batch._for(n)), pp, prefix_len, pq, lq, po, lo, n_heads, scale, pw,
                               wb, _on(stream, dev))
    if st:
        _check(st)


def verify_drafts_workspace_bytes(n_seqs, vocab):
    """Workspace bytes of verify_drafts."""
    _in_32_bits(n_seqs, vocab)
    n = _torch().cri_verify_drafts_workspace_bytes(n_seqs, vocab)
    if n < 0:
        _check(int(n))
    return int(n)


def verify_drafts(target, draft, draft_ids, uniforms, draws, offsets, out_ids, n_accepted, workspace=None, stream=None):
    """Drafted tokens accepted or replaced: target and draft (or None: sure drafts) probabilities
    [rows, vocab], draft_ids, uniforms (that decide about the drafts) and draws (independent ones,
    that draw the last token) [rows], offsets [n_seqs + 1]; out_ids [rows] gets the accepted drafts,
    the drawn token and -1 behind it, n_accepted [n_seqs] the drafts accepted."""
    L, dev = _torch(), _device()
    if target.dim() != 2:
        raise ValueError("target must have the shape [rows, vocab]")
    V = target.shape[1]
    pt, lt, n = _rows(target, V, "target", dev)
    pd = ld = 0
    if draft is not None:
        pd, ld, nd = _rows(draft, V, "draft", dev)
        if nd != n:
            raise ValueError("draft must have the shape of target")
    pi, po, pa = (_ints(draft_ids, "draft_ids", 1, dev), _ints(out_ids, "out_ids", 1, dev),
                  _ints(n_accepted, "n_accepted", 1, dev))
    pf = _ints(offsets, "offsets", 1, dev)
    B = n_accepted.shape[0]
    for x, name in ((uniforms, "uniforms"), (draws, "draws")):
        if x.dtype is not torch.float32 or x.shape != (n,) or not x.is_contiguous():
            raise ValueError("%s must be a contiguous float32 tensor [rows]" % name)
    if draft_ids.shape[0] != n or out_ids.shape[0] != n or offsets.shape[0] != B + 1:
        raise ValueError("draft_ids and out_ids must have target's rows, offsets n_seqs + 1 entries")
    if (n | B | V) >> 31:
        _in_32_bits(n, B, V)
    if workspace is None:
        workspace = _new_room(verify_drafts_workspace_bytes(B, V), stream)
    pw, wb = _room(workspace, dev)
    st = L.cri_verify_drafts(pt, lt, pd, ld, pi, _on_device(uniforms, "uniforms", dev), _on_device(draws, "draws", dev),
                             pf, B, n, V, po, pa, pw, wb, _on(stream, dev))
    if st:
        _check(st)


torch = _loaded = None


def _torch():
    """torch and the library are loaded by the first call, not by importing the package."""
    global torch, _loaded
    if _loaded is None:
        import torch as t

        torch, _loaded = t, _lib()
    return _loaded


from . import _check, _stream, lib as _lib  # noqa: E402
