"""Every kernel that a product of a layer of experts may take, in every format, against 64 bits: tiles of 1, 4, 8, 16, 32 and 64
rows, K in one and in several parts, and the weighted sums in one launch.  cri_expert_plan says which kernel a call's sizes mean;
the sizes below are the cheapest ones found for each, and a test without a GPU holds them to it, so that a change of the plan's
constants cannot take a kernel out of these tests unnoticed.

K ends inside a unit of 256 values where the format allows it, after 1, 2, 3 and 4 steps of 64 values.  Bars: experts_ref.py."""
import ctypes
import functools

import numpy as np
import pytest
import torch

import cretif_amd as cri
import experts_ref as ref
from cretif_amd import experts, quant

MATMUL, SWIGLU, COMBINE = range(3)

# (operator, rows of a tile, parts of K, waves): tokens, experts, choices, columns, units of 256 values
SIZES = [
    ((MATMUL, 1, 1, 1), (1, 4, 2, 40, 1)), ((MATMUL, 1, 1, 3), (1, 4, 2, 70, 3)), ((MATMUL, 1, 1, 5), (2, 16, 2, 40, 5)),
    ((MATMUL, 1, 1, 8), (1, 4, 2, 100, 9)), ((MATMUL, 4, 1, 2), (3, 1, 1, 40, 2)), ((MATMUL, 4, 1, 8), (4, 2, 2, 70, 11)),
    ((MATMUL, 8, 1, 1), (7, 2, 2, 40, 1)), ((MATMUL, 8, 1, 3), (20, 4, 2, 70, 3)), ((MATMUL, 8, 1, 4), (9, 2, 1, 40, 6)),
    ((MATMUL, 16, 1, 4), (250, 1, 1, 2050, 2)), ((MATMUL, 16, 2, 4), (200, 1, 1, 2050, 6)),
    ((MATMUL, 16, 4, 4), (100, 1, 1, 2050, 11)), ((MATMUL, 16, 8, 4), (48, 1, 1, 2050, 33)),
    ((MATMUL, 32, 1, 4), (400, 3, 2, 1030, 1)), ((MATMUL, 32, 2, 4), (800, 2, 1, 516, 9)),
    ((MATMUL, 32, 4, 4), (520, 1, 1, 516, 7)), ((MATMUL, 32, 8, 4), (300, 1, 1, 516, 13)),
    ((MATMUL, 64, 1, 4), (1500, 32, 4, 260, 1)), ((MATMUL, 64, 2, 4), (1500, 32, 4, 70, 16)),
    ((MATMUL, 64, 4, 4), (1500, 5, 2, 100, 8)), ((MATMUL, 64, 8, 4), (1500, 4, 1, 100, 13)),
    ((SWIGLU, 1, 1, 1), (1, 4, 2, 40, 1)), ((SWIGLU, 1, 1, 3), (1, 4, 2, 70, 3)), ((SWIGLU, 1, 1, 5), (2, 16, 2, 40, 5)),
    ((SWIGLU, 1, 1, 8), (1, 4, 2, 100, 9)), ((SWIGLU, 4, 1, 2), (3, 1, 1, 40, 2)), ((SWIGLU, 4, 1, 8), (4, 2, 2, 70, 11)),
    ((SWIGLU, 8, 1, 1), (7, 2, 2, 40, 1)), ((SWIGLU, 8, 1, 3), (20, 4, 2, 70, 3)), ((SWIGLU, 8, 1, 4), (9, 2, 1, 40, 6)),
    ((SWIGLU, 16, 1, 4), (250, 1, 1, 1030, 2)), ((SWIGLU, 16, 2, 4), (200, 1, 1, 1030, 6)),
    ((SWIGLU, 16, 4, 4), (100, 1, 1, 1030, 11)), ((SWIGLU, 16, 8, 4), (400, 1, 1, 100, 25)),
    ((SWIGLU, 32, 1, 4), (400, 3, 2, 516, 1)), ((SWIGLU, 32, 2, 4), (800, 2, 1, 260, 9)),
    ((SWIGLU, 32, 4, 4), (130, 2, 1, 1030, 7)), ((SWIGLU, 32, 8, 4), (130, 3, 2, 260, 13)),
    ((SWIGLU, 64, 1, 4), (300, 8, 2, 2050, 1)), ((SWIGLU, 64, 2, 4), (1500, 32, 4, 40, 18)),
    ((SWIGLU, 64, 4, 4), (1500, 5, 2, 40, 8)), ((SWIGLU, 64, 8, 4), (1500, 4, 1, 40, 33)),
    ((COMBINE, 0, 1, 16), (1, 4, 2, 40, 1)), ((COMBINE, 0, 1, 16), (20, 6, 5, 260, 7)), ((COMBINE, 1, 1, 1), (1, 1, 1, 8200, 1)),
    ((COMBINE, 1, 1, 4), (2, 4, 1, 4100, 4)), ((COMBINE, 4, 1, 3), (4, 1, 1, 2050, 3)), ((COMBINE, 4, 1, 8), (4, 1, 1, 2050, 9)),
    ((COMBINE, 8, 1, 1), (160, 1, 1, 40, 1)), ((COMBINE, 8, 1, 4), (160, 1, 1, 40, 5)),
    ((COMBINE, 16, 1, 4), (800, 2, 1, 1030, 2)), ((COMBINE, 16, 2, 4), (400, 1, 1, 1030, 4)),
    ((COMBINE, 16, 4, 4), (100, 1, 1, 2050, 4)), ((COMBINE, 16, 8, 4), (48, 1, 1, 2050, 18)),
    ((COMBINE, 32, 1, 4), (400, 3, 2, 1030, 1)), ((COMBINE, 32, 2, 4), (800, 2, 1, 516, 4)),
    ((COMBINE, 32, 4, 4), (250, 1, 1, 1030, 4)), ((COMBINE, 32, 8, 4), (130, 1, 1, 1030, 8)),
    ((COMBINE, 64, 1, 4), (1500, 32, 4, 260, 1)), ((COMBINE, 64, 2, 4), (1500, 16, 4, 70, 8)),
    ((COMBINE, 64, 4, 4), (1500, 5, 2, 100, 7)), ((COMBINE, 64, 8, 4), (1500, 4, 1, 100, 13)),
]
# another size where a format's plan differs
OTHERS = {((MATMUL, 64, 8, 4), "q8_0"): (800, 1, 1, 260, 13)}
# what is cut off the last unit: 4, 3, 2 and 1 steps of 64 remain (the last one half)
CUTS = {"q8_0": 32, "q4_0": 96, "q5_0": 160, "fp16": 224, "q4_k": 0, "q6_k": 0}
COLUMNS = [0, 1, 15, 16, 31, 32, 33, 39, 63, 64, 69, 95, 99, 127, 128, 255, 256, 259, 511, 515, 1023, 1029, 2047, 2049, 4099, 8199]
CASES = [(fmt, plan, i) for i, (plan, _) in enumerate(SIZES) for fmt in CUTS]
NAMES = ["%s-%s-%drows-%dparts-%dwaves-%d" % (fmt, ("matmul", "swiglu", "combine")[p[0]], p[1], p[2], p[3], i) for fmt, p, i in CASES]


def sizes_of(fmt, plan, i):
    M, E, k, N, units = OTHERS.get((plan, fmt), SIZES[i][1])
    return M, E, k, N, 256 * units - CUTS[fmt]


def plan_of(op, fmt, M, E, k, N, K):
    w = experts._ExpertWeights(0, cri.FORMAT_IDS[fmt], E, N, K)
    g = experts._ExpertGroups(0, 0, 0, M, k, E)
    p = (ctypes.c_int * 3)()
    assert cri.lib().cri_expert_plan(ctypes.addressof(w), ctypes.addressof(g), op, p) == 0
    return tuple(p)


@pytest.mark.parametrize("fmt", CUTS)
def test_plan(fmt):
    """The sizes take the kernels that they are listed for, and every one of those is there."""
    for i, (plan, _) in enumerate(SIZES):
        assert (plan[0],) + plan_of(plan[0], fmt, *sizes_of(fmt, plan, i)) == plan
    tiles = {(op, rows, parts) for (op, rows, parts, _), _ in SIZES}
    assert tiles >= {(op, rows, parts) for op in range(3) for rows in (16, 32, 64) for parts in (1, 2, 4, 8)}
    assert tiles >= {(op, rows, 1) for op in range(3) for rows in (1, 4, 8)} | {(COMBINE, 0, 1)}


def test_plan_refuses():
    w, g, p = experts._ExpertWeights(0, 3, 8, 64, 256), experts._ExpertGroups(0, 0, 0, 3, 2, 8), (ctypes.c_int * 3)(7, 7, 7)
    at, f = ctypes.addressof, cri.lib().cri_expert_plan
    assert f(at(w), at(g), 3, p) == -5 and f(at(w), at(g), -1, p) == -5 and f(at(w), at(g), 0, None) == -1
    assert f(None, at(g), 0, p) == -1 and f(at(w), None, 0, p) == -1
    w.K = 100
    assert f(at(w), at(g), 0, p) == -2 and tuple(p) == (7, 7, 7)
    w.K, g.n_tokens = 256, 0
    assert f(at(w), at(g), 2, p) == 0 and tuple(p) == (0, 0, 0)


# ---- on the GPU ------------------------------------------------------------------------------------------------------------

ROWS, WIDTH = 6000, 8448


@functools.lru_cache(maxsize=1)
def normal():
    return np.random.default_rng(2).standard_normal(ROWS * 1280 + WIDTH, dtype=np.float32)


def rows(n, K, seed):
    """n x K normal numbers out of one long row of them, other places for other seeds."""
    at = (7919 * seed) % (len(normal()) // 2)
    return np.resize(normal()[at:], n * K).reshape(n, K)


@functools.lru_cache(maxsize=2)
def blocks(fmt):
    """Random blocks of the format, on the host and on the device; matrices are stretches of them."""
    raw = quant.random_blocks(fmt, 2050, WIDTH, 4)
    return raw, torch.from_numpy(raw).cuda()


def matrix(fmt, E, N, K, second):
    """The laid out matrix, and the checked columns' values and magnitudes."""
    raw, draw = blocks(fmt)
    size = E * N * quant.row_bytes(fmt, K)
    at = (len(raw) - size) // quant.BLOCK_BYTES[fmt] * quant.BLOCK_BYTES[fmt] if second else 0
    w = cri.ExpertWeights(fmt, draw[at:at + size], E, N, K)
    cols = [c for c in COLUMNS if c < N]
    some = np.ascontiguousarray(raw[at:at + size].reshape(E, N, -1)[:, cols]).reshape(-1)
    return w, ref.weights(fmt, some, E, len(cols), K), cols


def group(M, E, k, seed):
    ids = np.argsort(np.random.default_rng(seed).random((M, E)), 1)[:, :k]
    if M > 1:
        ids[1] = -1  # a token without experts
    g = cri.ExpertGroups(M, k, E)
    cri.group_experts(torch.from_numpy(ids.astype(np.int32)).cuda(), g)
    return (ids, g) + ref.group(ids, E)


def around(rows, width):
    """(a buffer of 7s, a view of rows x width within it, off 16-byte alignment)"""
    whole = torch.full((rows + 1, width + 3), 7.0, device="cuda")
    return whole, whole[:rows, 1:1 + width]


def check_around(whole, rows, width):
    assert bool((whole[:, 0] == 7).all()) and bool((whole[:, 1 + width:] == 7).all()) and bool((whole[rows:] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,plan,i", CASES, ids=NAMES)
def test_products(fmt, plan, i):
    op = plan[0]
    M, E, k, N, K = sizes_of(fmt, plan, i)
    assert (op,) + plan_of(op, fmt, M, E, k, N, K) == plan
    ids, g, off, pairs, slots = group(M, E, k, i)
    w, (v, mag), cols = matrix(fmt, E, N, K, False)
    at = torch.tensor(cols, device="cuda")
    last = off[-1]
    if op == COMBINE:
        x = rows(M * k, K, i).copy()
        x[last:] = np.nan  # rows that are nobody's are not read
        weights, res = rows(M, k, i + 1), rows(M, N, i + 2)
        whole, out = around(M, N)
        cri.expert_combine(w, g, torch.from_numpy(x).cuda(), torch.from_numpy(weights.copy()).cuda(), out, torch.from_numpy(res.copy()).cuda())
        check_around(whole, M, N)
        r = ref.Product(np.zeros((M, K)), v[0], mag[0])
        r.want = res[:, cols].astype(np.float64)
        total, square = np.abs(r.want), np.zeros(r.want.shape)
        for e in range(E):
            if off[e] == off[e + 1]:
                continue
            t, j = pairs[off[e]:off[e + 1]] // k, pairs[off[e]:off[e + 1]] % k  # a token names an expert once
            p, f = ref.Product(x[off[e]:off[e + 1]], v[e], mag[e]), weights[t, j].astype(np.float64)[:, None]
            r.want[t] += f * p.want
            r.worst[t] += np.abs(f) * p.worst
            square[t] += (f * p.rms) ** 2
            total[t] += np.abs(f * p.want)
        r.worst += (k + 1) * ref.U * total
        r.rms = np.sqrt(square) + np.sqrt(k + 1) * ref.U * total
        ref.check(out[:, at], r)
        if M > 1:
            assert torch.equal(out[1].cpu(), torch.from_numpy(res[1]))
        return
    x = rows(M, K, i)
    whole, out = around(M * k, N)
    dx = torch.from_numpy(x.copy()).cuda()
    if op == SWIGLU:
        up, (uv, umag), _ = matrix(fmt, E, N, K, True)
        cri.expert_swiglu(w, up, g, dx, out)
    else:
        cri.expert_matmul(w, g, dx, out)
    check_around(whole, M * k, N)
    assert bool((out[last:] == 7).all()) and bool(torch.isfinite(out).all())
    for e in range(E):
        if off[e] < off[e + 1]:
            some = x[pairs[off[e]:off[e + 1]] // k]
            r = ref.Swiglu(some, (v[e], mag[e]), (uv[e], umag[e])) if op == SWIGLU else ref.Product(some, v[e], mag[e])
            ref.check(out[off[e]:off[e + 1]][:, at], r, "expert %d" % e)
    if op == MATMUL:  # rows in grouped order: the same bits
        xg = x[np.maximum(pairs, 0) // k].copy()
        xg[last:] = np.nan
        again = torch.full((M * k, N), 7.0, device="cuda")
        cri.expert_matmul(w, g, torch.from_numpy(xg).cuda(), again, grouped=True)
        assert torch.equal(again, out)
