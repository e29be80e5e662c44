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


def _on_device(t, name):
    """The tensor's address; it must be on the current GPU."""
    if not t.is_cuda:
        raise ValueError("%s is on %s; the HIP kernels need device (cuda) tensors" % (name, t.device))
    if t.get_device() != torch._C._cuda_getDevice():
        raise ValueError("%s is on %s, not on the current device" % (name, t.device))
    return t.data_ptr()


def _rows(t, name):
    """(address, floats from row to row, rows or None) of a row buffer."""
    if type(t) is tuple:
        return t[0], t[1], None
    if t.dtype is not torch.float32:
        raise ValueError("%s must be float32, not %s" % (name, t.dtype))
    d = t.dim()
    if d == 2:
        ld, inner = t.stride()
        tight = inner == 1 or t.shape[1] <= 1
    elif d == 3:
        ld, mid, inner = t.stride()
        tight = (inner == 1 or t.shape[2] <= 1) and (mid == t.shape[2] or t.shape[1] <= 1)
    else:
        raise ValueError("%s must have the shape [rows, width] or [rows, heads, head_dim]" % name)
    if not tight:
        raise ValueError("%s: the elements of a row must be consecutive" % name)
    n = t.shape[0]
    width = t.shape[1] if d == 2 else t.shape[1] * t.shape[2]
    if n <= 1:
        ld = max(ld, width)  # the stride of a single row says nothing
    return _on_device(t, name), ld, n


def _wide(t, name, width):
    if type(t) is not tuple and t.shape[0] and t.numel() // t.shape[0] != width:
        raise ValueError("%s has rows of %d floats, not %d" % (name, t.numel() // t.shape[0], width))


def _same_rows(n_rows, *named):
    for name, n in named:
        if n is None:
            continue
        if n_rows is None:
            n_rows = n
        elif n != n_rows:
            raise ValueError("%s has %d rows, not %d" % (name, n, n_rows))
    if n_rows is None:
        raise ValueError("n_rows must be given with (address, ld) buffers")
    return n_rows


def _ints(t, name, dims):
    if t.dtype is not torch.int32 or t.dim() != dims or not t.is_contiguous():
        raise ValueError("%s must be a contiguous int32 tensor of %d dimension(s)" % (name, dims))
    return _on_device(t, name)


def _room(workspace, need, stream):
    """(address, bytes, tensor) of the workspace, allocated on the current stream when there is none."""
    if workspace is None:
        if stream is not None and need:
            raise ValueError("give a workspace with an explicit stream (an allocated one belongs to the current stream)")
        workspace = torch.empty(need, dtype=torch.uint8, device="cuda")
    if not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    return _on_device(workspace, "workspace"), workspace.numel() * workspace.element_size(), workspace


class Rotation:
    """Norms and rotation of query and key heads: norm weights [head_dim] (None: not normed), the
    rotation's base and its number of elements (0: no rotation), "adjacent" pairs (2 i, 2 i + 1) or
    "halves" (i, i + rot_dim / 2)."""

    def __init__(self, theta, rot_dim, pairs="adjacent", q_norm=None, k_norm=None, eps=1e-6):
        _torch()
        for w, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
            if w is not None and (w.dtype is not torch.float32 or w.dim() != 1 or not w.is_contiguous()):
                raise ValueError("%s must be a contiguous float32 tensor [head_dim]" % name)
        self.q_norm, self.k_norm = q_norm, k_norm
        self._c = _Rotation(None if q_norm is None else _on_device(q_norm, "q_norm"),
                            None if k_norm is None else _on_device(k_norm, "k_norm"), eps, theta, rot_dim, PAIRS[pairs])
        self._ref = ctypes.addressof(self._c)

    def _fits(self, head_dim):
        for w, name in ((self.q_norm, "q_norm"), (self.k_norm, "k_norm")):
            if w is not None and w.shape[0] != head_dim:
                raise ValueError("%s has %d weights, not head_dim=%d" % (name, w.shape[0], head_dim))


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
        if n > 0 and not k[0].is_contiguous():
            raise ValueError("a page must be contiguous")
        self.k, self.v = k, v
        self.n_kv_heads, self.head_dim = h, d
        stride = k.stride(0) if n > 1 else (ps * h * d + 7) // 8 * 8
        self._c = _PagedKV(_on_device(k, "k"), _on_device(v, "v"), stride, kinds[k.dtype], n, ps, h, d)
        self._ref = ctypes.addressof(self._c)


class PagedBatch:
    """A ragged batch: int32 offsets [n_seqs + 1], lens [n_seqs], pages [n_seqs, max_pages]."""

    def __init__(self, offsets, lens, pages):
        _torch()
        po, pl, pp = _ints(offsets, "offsets", 1), _ints(lens, "lens", 1), _ints(pages, "pages", 2)
        n = lens.shape[0]
        if offsets.shape[0] != n + 1 or pages.shape[0] != n:
            raise ValueError("offsets must have n_seqs + 1 entries, lens and pages n_seqs")
        self.offsets, self.lens, self.pages = offsets, lens, pages
        self._make = lambda rows: _PagedBatch(po, pl, pp, n, rows, pages.shape[1])
        self._by_rows = {}

    def _for(self, n_rows):
        c = self._by_rows.get(n_rows)
        if c is None:
            c = self._by_rows[n_rows] = self._make(n_rows)
        return ctypes.addressof(c)


def qk_norm_rope(rot, q, k, q_out, k_out, positions, n_heads, n_kv_heads, head_dim, n_rows=None, stream=None):
    """q_out and k_out = the heads of q and k, normed and rotated at positions [rows] (int32); q_out may
    be q and k_out k.  q (with n_heads 0) or k (with n_kv_heads 0) may be None."""
    _torch()
    pq, lq, nq = _rows(q, "q") if q is not None else (None, 0, None)
    pk, lk, nk = _rows(k, "k") if k is not None else (None, 0, None)
    po, lo, no = _rows(q_out, "q_out") if q is not None else (None, 0, None)
    px, lx, nx = _rows(k_out, "k_out") if k is not None else (None, 0, None)
    rot._fits(head_dim)
    if q is not None:
        _wide(q, "q", n_heads * head_dim)
        _wide(q_out, "q_out", n_heads * head_dim)
    if k is not None:
        _wide(k, "k", n_kv_heads * head_dim)
        _wide(k_out, "k_out", n_kv_heads * head_dim)
    pp = _ints(positions, "positions", 1)
    n = _same_rows(n_rows, ("q", nq), ("k", nk), ("q_out", no), ("k_out", nx), ("positions", positions.shape[0]))
    _check(_lib().cri_qk_norm_rope(rot._ref, pq, lq, pk, lk, po, lo, px, lx, pp, n, n_heads, n_kv_heads, head_dim,
                                   _stream(stream)))


def paged_append(cache, batch, rot, k, v, q=None, q_out=None, n_heads=0, n_rows=None, stream=None):
    """The batch's k rows, normed and rotated, and v rows go to their pages; with q, its heads go to
    q_out, normed and rotated."""
    _torch()
    pk, lk, nk = _rows(k, "k")
    pv, lv, nv = _rows(v, "v")
    D = cache.head_dim
    _wide(k, "k", cache.n_kv_heads * D)
    _wide(v, "v", cache.n_kv_heads * D)
    rot._fits(D)
    if q is None:
        pq, lq, nq, po, lo, no = None, 0, None, None, 0, None
    else:
        pq, lq, nq = _rows(q, "q")
        po, lo, no = _rows(q_out, "q_out")
        _wide(q, "q", n_heads * D)
        _wide(q_out, "q_out", n_heads * D)
    n = _same_rows(n_rows, ("k", nk), ("v", nv), ("q", nq), ("q_out", no))
    _check(_lib().cri_paged_append(cache._ref, batch._for(n), rot._ref, pq, lq, po, lo, n_heads, pk, lk, pv, lv,
                                   _stream(stream)))


def paged_attention_workspace_bytes(cache, batch, n_rows, n_heads, prefix_len=0):
    """Workspace bytes of paged_attention for batches of these host numbers."""
    n = _lib().cri_paged_attention_workspace_bytes(cache._ref, batch._for(n_rows), prefix_len, n_heads)
    if n < 0:
        _check(int(n))
    return int(n)


def paged_attention(cache, batch, q, out, n_heads, scale, prefix_pages=None, prefix_len=0, workspace=None, n_rows=None,
                    stream=None):
    """out = softmax(scale q K^T) V of every row over the positions it sees, those below prefix_len
    through prefix_pages, which all sequences share.  workspace: a device tensor of
    paged_attention_workspace_bytes (one is allocated when None)."""
    _torch()
    pq, lq, nq = _rows(q, "q")
    po, lo, no = _rows(out, "out")
    width = n_heads * cache.head_dim
    _wide(q, "q", width)
    _wide(out, "out", width)
    n = _same_rows(n_rows, ("q", nq), ("out", no))
    pp = None
    if prefix_len > 0:
        if prefix_pages is None:
            raise ValueError("prefix_len without prefix_pages")
        pp = _ints(prefix_pages, "prefix_pages", 1)
        if prefix_pages.shape[0] * cache._c.page_size < prefix_len:
            raise ValueError("prefix_pages holds %d pages, too few for prefix_len=%d" % (prefix_pages.shape[0], prefix_len))
    b = batch._for(n)
    if workspace is None:
        need = paged_attention_workspace_bytes(cache, batch, n, n_heads, prefix_len)
        workspace = None if need == 0 else _room(None, need, stream)[2]
    pw, wb = (0, 0) if workspace is None else _room(workspace, 0, stream)[:2]
    _check(_lib().cri_paged_attention(cache._ref, b, pp, prefix_len, pq, lq, po, lo, n_heads, scale, pw, wb,
                                      _stream(stream)))


def verify_drafts_workspace_bytes(n_seqs, vocab):
    """Workspace bytes of verify_drafts."""
    n = _lib().cri_verify_drafts_workspace_bytes(n_seqs, vocab)
    if n < 0:
        _check(int(n))
    return int(n)


def verify_drafts(target, draft, draft_ids, uniforms, draws, offsets, out_ids, n_accepted, workspace=None, stream=None):
    """Drafted tokens accepted or replaced: target and draft (or None: sure drafts) probabilities
    [rows, vocab], draft_ids, uniforms (that decide about the drafts) and draws (independent ones,
    that draw the last token) [rows], offsets [n_seqs + 1]; out_ids [rows] gets the accepted drafts,
    the drawn token and -1 behind it, n_accepted [n_seqs] the drafts accepted."""
    _torch()
    pt, lt, n = _rows(target, "target")
    V = target.shape[1]
    pd, ld = None, 0
    if draft is not None:
        pd, ld, nd = _rows(draft, "draft")
        if nd != n or draft.shape[1] != V:
            raise ValueError("draft must have the shape of target")
    pi, po, pa = _ints(draft_ids, "draft_ids", 1), _ints(out_ids, "out_ids", 1), _ints(n_accepted, "n_accepted", 1)
    pf = _ints(offsets, "offsets", 1)
    B = n_accepted.shape[0]
    for x, name in ((uniforms, "uniforms"), (draws, "draws")):
        if x.dtype is not torch.float32 or x.shape != (n,) or not x.is_contiguous():
            raise ValueError("%s must be a contiguous float32 tensor [rows]" % name)
    if draft_ids.shape[0] != n or out_ids.shape[0] != n or offsets.shape[0] != B + 1:
        raise ValueError("draft_ids and out_ids must have target's rows, offsets n_seqs + 1 entries")
    if workspace is None:
        workspace = _room(None, verify_drafts_workspace_bytes(B, V), stream)[2]
    pw, wb = _room(workspace, 0, stream)[:2]
    _check(_lib().cri_verify_drafts(pt, lt, pd, ld, pi, _on_device(uniforms, "uniforms"),
                                    _on_device(draws, "draws"), pf, B, n, V, po, pa, pw, wb,
                                    _stream(stream)))


torch = None


def _torch():
    global torch
    if torch is None:
        import torch as t

        torch = t


from . import _check, _stream, lib as _lib  # noqa: E402
