"""A layer of experts: cri_expert_pack, cri_expert_route, cri_expert_group, cri_expert_matmul, cri_expert_swiglu and
cri_expert_combine of include/cri.h over torch tensors.  No counterpart in the reference, whose models
have one FFN.

Row buffers are fp32 device tensors [rows, width] whose rows may be strided.  ExpertWeights,
ExpertGroups and ExpertRouter keep their tensors alive and are made once; what the groups hold is
written by route_experts (or group_experts) and read by the products, on the device.  Everything must
be on the current device.
"""
from __future__ import annotations

import ctypes

_vp, _i32, _i64, _f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float

SCORING = {"softmax": 0, "sigmoid": 1}


class _ExpertWeights(ctypes.Structure):
    _fields_ = [("data", _vp), ("format", _i32), ("n_experts", _i32), ("N", _i32), ("K", _i32)]


class _ExpertGroups(ctypes.Structure):
    _fields_ = [("offsets", _vp), ("rows", _vp), ("slots", _vp), ("n_tokens", _i32), ("top_k", _i32), ("n_experts", _i32)]


class _ExpertRouter(ctypes.Structure):
    _fields_ = [("bias", _vp), ("scale", _f32), ("scoring", _i32), ("normalize", _i32)]


SYMBOLS = {
    "cri_expert_packed_bytes": ([_i32, _i32, _i32, _i32], _i64),
    "cri_expert_pack": ([_i32, _vp, _i32, _i32, _i32, _vp, _vp], _i32),
    "cri_expert_group_workspace_bytes": ([_vp], _i64),
    "cri_expert_route": ([_vp, _vp, _i32, _vp, _vp, _vp, _vp, _i64, _vp], _i32),
    "cri_expert_group": ([_vp, _vp, _vp, _i64, _vp], _i32),
    "cri_expert_matmul_workspace_bytes": ([_vp, _vp, _i32], _i64),
    "cri_expert_matmul": ([_vp, _vp, _vp, _i32, _i32, _vp, _i32, _vp, _i64, _vp], _i32),
    "cri_expert_swiglu_workspace_bytes": ([_vp, _vp], _i64),
    "cri_expert_swiglu": ([_vp, _vp, _vp, _vp, _i32, _vp, _i32, _vp, _i64, _vp], _i32),
    "cri_expert_combine_workspace_bytes": ([_vp, _vp], _i64),
    "cri_expert_plan": ([_vp, _vp, _i32, _vp], _i32),
    "cri_expert_combine": ([_vp, _vp, _vp, _i32, _vp, _vp, _i32, _vp, _i32, _vp, _i64, _vp], _i32),
}


def declare(L):
    for name, (args, res) in SYMBOLS.items():
        f = getattr(L, name)
        f.argtypes, f.restype = args, res


def _bytes(n):
    if n < 0:
        _check(int(n))
    return int(n)


class ExpertWeights:
    """A matrix per expert, laid out once for the products: raw, a uint8 device tensor that holds the
    GGUF blocks of [n_experts, N, K] (not needed afterwards; Q4_0 with element i in byte i / 2, as everywhere in the
    library, not in upstream GGML's order).  Runs on the current stream, to which its memory belongs."""

    def __init__(self, fmt, raw, n_experts, N, K):
        L, dev = _torch(), _device()
        _in_32_bits(n_experts, N, K)
        need = _bytes(L.cri_expert_packed_bytes(FORMAT_IDS[fmt], n_experts, N, K))
        if raw.dtype is not torch.uint8 or not raw.is_contiguous() or raw.numel() * BLOCK[fmt][0] != n_experts * N * K * BLOCK[fmt][1]:
            raise ValueError("raw must be a contiguous uint8 tensor of the %s blocks of [%d, %d, %d]" % (fmt, n_experts, N, K))
        src = _on_device(raw, "raw", dev)
        self.data = torch.empty(need, dtype=torch.uint8, device=raw.device)
        self.format, self.n_experts, self.N, self.K = fmt, n_experts, N, K
        _check(L.cri_expert_pack(FORMAT_IDS[fmt], src, n_experts, N, K, self.data.data_ptr(), _on(None, dev)))
        self._c = _ExpertWeights(self.data.data_ptr(), FORMAT_IDS[fmt], n_experts, N, K)
        self._ref = ctypes.addressof(self._c)
        self._dev = dev


class ExpertGroups:
    """The pairs (token, choice) grouped by expert: int32 offsets [n_experts + 1], rows and slots
    [n_tokens * top_k] (when None allocated and zeroed on the current stream, which another one has to wait for)."""

    def __init__(self, n_tokens, top_k, n_experts, offsets=None, rows=None, slots=None):
        _torch()
        _in_32_bits(n_tokens, top_k, n_experts)
        if min(n_tokens, top_k, n_experts) < 0:
            raise ValueError("negative dimension")
        made = []
        for t, n, name in ((offsets, n_experts + 1, "offsets"), (rows, n_tokens * top_k, "rows"), (slots, n_tokens * top_k, "slots")):
            t = torch.zeros(n, dtype=torch.int32, device="cuda") if t is None else t
            _ints(t, name, 1)
            if t.shape[0] != n:
                raise ValueError("%s must have %d entries" % (name, n))
            made.append(t)
        self.offsets, self.rows, self.slots = made
        self.n_tokens, self.top_k, self.n_experts = n_tokens, top_k, n_experts
        self.n_rows = n_tokens * top_k
        self._shape = (n_tokens, top_k)
        self._c = _ExpertGroups(*(t.data_ptr() for t in made), n_tokens, top_k, n_experts)
        self._ref = ctypes.addressof(self._c)
        self._dev = _device()


class ExpertRouter:
    """How logits become choices and weights: scoring "softmax" or "sigmoid", a bias [n_experts] for the
    choice alone (or None), weights divided by their sum with normalize, times scale."""

    def __init__(self, scoring="softmax", bias=None, normalize=True, scale=1.0):
        _torch()
        if bias is not None and (bias.dtype is not torch.float32 or bias.dim() != 1 or not bias.is_contiguous()):
            raise ValueError("bias must be a contiguous float32 tensor [n_experts]")
        self.bias = bias
        self._c = _ExpertRouter(None if bias is None else _on_device(bias, "bias"), scale, SCORING[scoring], 1 if normalize else 0)
        self._ref = ctypes.addressof(self._c)
        self._dev = None if bias is None else _device()


# A step's calls cost the host about as much as the GPU, so each check below has a short way for the usual case first.


def _on_it(dev, *descriptors):
    for d in descriptors:
        if d._dev != dev and d._dev is not None:
            raise ValueError("the tensors of a %s are on cuda:%d, not on the current device" % (type(d).__name__, d._dev))


def _floats(t, rows, width, name, dev):
    """(address, floats from row to row) of a row buffer."""
    if type(t) is not tuple and t.dtype is _f32t and t.is_contiguous() and t.shape == (rows, width) and t.get_device() == dev:
        return t.data_ptr(), width
    p, ld, n = _rows(t, width, name, dev)
    if n is not None and n != rows:
        raise ValueError("%s has %d rows, not %d" % (name, n, rows))
    if ld >> 31:
        _in_32_bits(ld)
    return p, ld


def _choices(t, kind, groups, name, dev):
    """The address of a contiguous [n_tokens, top_k] tensor."""
    if t.dtype is not kind or t.shape != groups._shape or not t.is_contiguous():
        raise ValueError("%s must be a contiguous %s tensor [n_tokens, top_k]" % (name, kind))
    return t.data_ptr() if t.get_device() == dev else _on_device(t, name, dev)


def _workspace(workspace, stream, dev, need, *args):
    """(address, bytes, the tensor); one is allocated when None and something is needed."""
    if workspace is None:
        n = _bytes(need(*args))
        if n == 0:
            return None, 0, None
        workspace = _new_room(n, stream)
    elif workspace.is_contiguous() and workspace.get_device() == dev:
        return workspace.data_ptr(), workspace.nbytes, workspace
    p, n = _room(workspace, dev)
    return p, n, workspace


def route_experts_workspace_bytes(groups):
    """Workspace bytes of route_experts and group_experts."""
    return _bytes(_torch().cri_expert_group_workspace_bytes(groups._ref))


def route_experts(router, logits, ids, weights, groups, workspace=None, stream=None):
    """Logits [n_tokens, n_experts] -> ids (int32) and weights (float32) [n_tokens, top_k], and the groups.
    workspace: a device tensor of route_experts_workspace_bytes (one is allocated when None)."""
    L, dev = _loaded or _torch(), _device()
    _on_it(dev, router, groups)
    if router.bias is not None and router.bias.shape[0] != groups.n_experts:
        raise ValueError("the bias has %d entries, not %d" % (router.bias.shape[0], groups.n_experts))
    pl, ldl = _floats(logits, groups.n_tokens, groups.n_experts, "logits", dev)
    pi = _choices(ids, torch.int32, groups, "ids", dev)
    pw = _choices(weights, torch.float32, groups, "weights", dev)
    ws, n, held = _workspace(workspace, stream, dev, L.cri_expert_group_workspace_bytes, groups._ref)
    st = L.cri_expert_route(router._ref, pl, ldl, pi, pw, groups._ref, ws, n, _on(stream, dev))
    if st:
        _check(st)


def group_experts(ids, groups, workspace=None, stream=None):
    """The groups of given ids (int32 [n_tokens, top_k]; outside [0, n_experts): no expert)."""
    L, dev = _loaded or _torch(), _device()
    _on_it(dev, groups)
    pi = _choices(ids, torch.int32, groups, "ids", dev)
    ws, n, held = _workspace(workspace, stream, dev, L.cri_expert_group_workspace_bytes, groups._ref)
    st = L.cri_expert_group(pi, groups._ref, ws, n, _on(stream, dev))
    if st:
        _check(st)


def expert_matmul_workspace_bytes(w, groups, grouped=False):
    """Workspace bytes of expert_matmul."""
    return _bytes(_torch().cri_expert_matmul_workspace_bytes(w._ref, groups._ref, 1 if grouped else 0))


def expert_matmul(w, groups, x, out, workspace=None, grouped=False, stream=None):
    """out[r] = x[token of r] W[e]^T for the grouped rows r of every expert e: x [n_tokens, K] (with grouped,
    [n_tokens * top_k, K] in grouped order), out [n_tokens * top_k, N].  workspace: a device tensor of
    expert_matmul_workspace_bytes (one is allocated when None)."""
    L, dev = _loaded or _torch(), _device()
    _on_it(dev, w, groups)
    px, ldx = _floats(x, groups.n_rows if grouped else groups.n_tokens, w.K, "x", dev)
    po, ldo = _floats(out, groups.n_rows, w.N, "out", dev)
    ws, n, held = _workspace(workspace, stream, dev, L.cri_expert_matmul_workspace_bytes, w._ref, groups._ref, 1 if grouped else 0)
    st = L.cri_expert_matmul(w._ref, groups._ref, px, ldx, 1 if grouped else 0, po, ldo, ws, n, _on(stream, dev))
    if st:
        _check(st)


def expert_swiglu_workspace_bytes(gate, groups):
    """Workspace bytes of expert_swiglu."""
    return _bytes(_torch().cri_expert_swiglu_workspace_bytes(gate._ref, groups._ref))


def expert_swiglu(gate, up, groups, x, out, workspace=None, stream=None):
    """out[r] = silu(x[token of r] gate[e]^T) * (x[token of r] up[e]^T): x [n_tokens, K], out [n_tokens * top_k, N]."""
    L, dev = _loaded or _torch(), _device()
    _on_it(dev, gate, up, groups)
    px, ldx = _floats(x, groups.n_tokens, gate.K, "x", dev)
    po, ldo = _floats(out, groups.n_rows, gate.N, "out", dev)
    ws, n, held = _workspace(workspace, stream, dev, L.cri_expert_swiglu_workspace_bytes, gate._ref, groups._ref)
    st = L.cri_expert_swiglu(gate._ref, up._ref, groups._ref, px, ldx, po, ldo, ws, n, _on(stream, dev))
    if st:
        _check(st)


def expert_combine_workspace_bytes(w, groups):
    """Workspace bytes of expert_combine."""
    return _bytes(_torch().cri_expert_combine_workspace_bytes(w._ref, groups._ref))


def expert_combine(w, groups, x, weights, out, residual=None, workspace=None, stream=None):
    """out[t] = residual[t] + the sum over t's choices of weight * (x[grouped row] W[e]^T): x [n_tokens * top_k, K] in
    grouped order, weights [n_tokens, top_k], out and residual (may be None, or out) [n_tokens, N]."""
    L, dev = _loaded or _torch(), _device()
    _on_it(dev, w, groups)
    px, ldx = _floats(x, groups.n_rows, w.K, "x", dev)
    pw = _choices(weights, torch.float32, groups, "weights", dev)
    po, ldo = _floats(out, groups.n_tokens, w.N, "out", dev)
    pr, ldr = (None, 0) if residual is None else _floats(residual, groups.n_tokens, w.N, "residual", dev)
    ws, n, held = _workspace(workspace, stream, dev, L.cri_expert_combine_workspace_bytes, w._ref, groups._ref)
    st = L.cri_expert_combine(w._ref, groups._ref, px, ldx, pw, pr, ldr, po, ldo, ws, n, _on(stream, dev))
    if st:
        _check(st)


torch = _loaded = _f32t = None


def _torch():
    """torch and the library are loaded by the first call, not by importing the package."""
    global torch, _loaded, _f32t
    if _loaded is None:
        lib = serving._torch()
        torch = serving.torch
        _f32t = torch.float32
        _loaded = lib
    return _loaded


from . import FORMAT_IDS, _check, serving  # noqa: E402
from .quant import BLOCK_BYTES, BLOCK_ELEMS  # noqa: E402
from .serving import _device, _in_32_bits, _ints, _new_room, _on, _on_device, _room, _rows  # noqa: E402

BLOCK = {f: (BLOCK_ELEMS[f], BLOCK_BYTES[f]) for f in FORMAT_IDS}
