"""A layer of experts at both ends of fp32's exponent range, through each kernel that products take: few rows (which need no
workspace), tiles of rows, and the weighted sums of few tokens in one launch.

Bars: those of experts_ref.py, which hold at any magnitude, and what fp32 itself loses below 2^-126, where its step is 2^-149: half
a step, 2^-150, for the product of every 256 values of K (sums of such products are exact there), times the choice's weight in a
weighted sum, and half a step for each of its additions."""
import numpy as np
import pytest
import torch

import cretif_amd as cri
import experts_ref as ref
from cretif_amd import quant

pytestmark = pytest.mark.gpu

FORMATS = ["q8_0", "q4_0", "q5_0", "q4_k", "q6_k", "fp16"]
HALF_STEP = 2.0 ** -150
# largest magnitudes of rows: below fp32's normal numbers, about their smallest, and large
SIZES = [2e-44, 2e-41, 1e-38, 1e-37, 1e-36, 1e-35, 1e-30, 1.0, 1e30, 1e36]


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def rows_of(M, K, seed):
    """Row t's values are normal numbers times SIZES[t mod 10]."""
    x = np.random.default_rng(seed).standard_normal((M, K)) * np.array(SIZES)[np.arange(M) % len(SIZES), None]
    return x.astype(np.float32)


def grouped(ids, E):
    g = cri.ExpertGroups(ids.shape[0], ids.shape[1], E)
    cri.group_experts(dev(ids.astype(np.int32)), g)
    return g, g.slots.cpu().numpy()


def within(got, want, worst):
    err = np.abs(ref.f64(got) - want)
    assert (err <= worst).all(), float((err / worst).max())


# few rows of one and of several tokens, and tiles
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K,few", [(10, 70, 768, True), (40, 40, 512, True), (400, 2100, 1280, False)])
def test_matmul(fmt, M, N, K, few):
    E = 2 if M > 10 else 10
    raw = quant.synthetic_weights(fmt, E * N, K, 5)
    v, mag = ref.weights(fmt, raw, E, N, K)
    w = cri.ExpertWeights(fmt, dev(raw), E, N, K)
    ids = np.arange(M)[:, None] % E
    g, slots = grouped(ids, E)
    assert (cri.expert_matmul_workspace_bytes(w, g) == 0) == few
    x = rows_of(M, K, M)
    out = torch.empty(M, N, device="cuda")
    cri.expert_matmul(w, g, dev(x), out)
    for e in range(E):
        p = ref.Product(x[e::E], v[e], mag[e])
        within(out[torch.from_numpy(slots[e::E]).cuda().long()], p.want, p.worst + (K // 256 + 1) * HALF_STEP)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K,token", [(10, 70, 768, True), (400, 2100, 1280, False)])
@pytest.mark.parametrize("residual", [False, True])
def test_combine(fmt, M, N, K, token, residual):
    """Weights of every size beside rows of every size (no result leaves fp32's range)."""
    E, k = 4, 2
    raw = quant.synthetic_weights(fmt, E * N, K, 6)
    v, mag = ref.weights(fmt, raw, E, N, K)
    w = cri.ExpertWeights(fmt, dev(raw), E, N, K)
    ids = np.stack([np.arange(M) % E, (np.arange(M) + 1) % E], 1)
    g, slots = grouped(ids, E)
    assert (cri.expert_combine_workspace_bytes(w, g) == 0) == token
    x = np.empty((M * k, K), np.float32)
    x[slots] = rows_of(M * k, K, M)
    rng = np.random.default_rng(3)
    weights = (rng.standard_normal((M, k)) * 0.037).astype(np.float32)
    weights[1::3] *= np.float32(1e-6)
    res = (rng.standard_normal((M, N)) * 1e-37).astype(np.float32) if residual else None
    out = torch.empty(M, N, device="cuda")
    cri.expert_combine(w, g, dev(x), dev(weights), out, None if res is None else dev(res))
    want = np.zeros((M, N)) if res is None else res.astype(np.float64)
    total, worst = np.abs(want), np.full((M, N), (k + 1) * HALF_STEP)
    units = K // 256 + 1
    for j in range(k):
        for e in range(E):
            t = np.flatnonzero(ids[:, j] == e)
            p = ref.Product(x[slots[t * k + j]], v[e], mag[e])
            f = np.abs(weights[t, j].astype(np.float64))[:, None]
            want[t] += weights[t, j].astype(np.float64)[:, None] * p.want
            # a launch adds up the products of 256 values with their weights, one rounding each
            worst[t] += f * (p.worst + units * HALF_STEP) + units * HALF_STEP
            total[t] += f * np.abs(p.want)
    within(out, want, worst + (k + 1) * ref.U * total)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", [(10, 70, 768), (400, 2100, 1280)])
def test_swiglu(fmt, M, N, K):
    """Rows whose products' product is about fp32's smallest normal number, and larger ones."""
    E = 5
    raws = [quant.synthetic_weights(fmt, E * N, K, seed) for seed in (7, 8)]
    (gv, gm), (uv, um) = (ref.weights(fmt, raw, E, N, K) for raw in raws)
    gate, up = (cri.ExpertWeights(fmt, dev(raw), E, N, K) for raw in raws)
    ids = np.arange(M)[:, None] % E
    g, slots = grouped(ids, E)
    x = np.random.default_rng(M).standard_normal((M, K)) * np.array([1e-22, 1e-19, 1e-18, 1e-3, 1e15])[np.arange(M) // E % 5, None]
    x = x.astype(np.float32)
    out = torch.empty(M, N, device="cuda")
    cri.expert_swiglu(gate, up, g, dev(x), out)
    for e in range(E):
        s = ref.Swiglu(x[e::E], (gv[e], gm[e]), (uv[e], um[e]))
        within(out[torch.from_numpy(slots[e::E]).cuda().long()], s.want, s.worst + HALF_STEP)


def test_a_large_weight_beside_large_rows_of_small_weights():
    """The factors' product leaves fp32's range, the result does not: rows of 2^123 against blocks scaled by 2^-24, weights 2^19."""
    E, N, K = 2, 40, 256
    rng = np.random.default_rng(1)
    blocks = np.zeros((E * N, K // 32, 34), np.uint8)
    blocks[..., 0] = 1  # fp16 2^-24
    blocks[..., 2:] = rng.integers(0, 256, blocks[..., 2:].shape)
    raw = blocks.reshape(-1)
    v, mag = ref.weights("q8_0", raw, E, N, K)
    w = cri.ExpertWeights("q8_0", dev(raw), E, N, K)
    g, slots = grouped(np.array([[0], [1]]), E)
    x = np.zeros((2, K), np.float32)
    x[0, 5], x[1, 200] = 2.0 ** 123, -2.0 ** 123
    weights = np.full((2, 1), 2.0 ** 19, np.float32)
    out = torch.empty(2, N, device="cuda")
    cri.expert_combine(w, g, dev(x), dev(weights), out)
    want = np.stack([x[e].astype(np.float64) @ v[e].T for e in range(E)]) * 2.0 ** 19
    assert np.abs(want).max() < 2.0 ** 127 and np.array_equal(ref.f64(out), want)  # one term each: exact


def test_values_of_the_smallest_numbers_add_up():
    """8192 values of 2e-41 against weights of 1: 1.6e-37, whatever number of rows the call has."""
    E, N, K = 2, 33, 8192
    raw = np.full(E * N * K, 0x3C00, np.uint16).view(np.uint8)
    w = cri.ExpertWeights("fp16", dev(raw), E, N, K)
    value = np.float32(2e-41)
    want = float(value) * K
    for M in (1, 6, 300):
        g, _ = grouped(np.arange(M)[:, None] % E, E)
        out = torch.empty(M, N, device="cuda")
        cri.expert_matmul(w, g, dev(np.full((M, K), value)), out)
        assert (np.abs(ref.f64(out) - want) <= 2.0 ** -22 * want + 33 * HALF_STEP).all()
        cri.expert_combine(w, g, dev(np.full((M, K), value)), dev(np.ones((M, 1), np.float32)), out)
        assert (np.abs(ref.f64(out) - want) <= 2.0 ** -22 * want + 33 * HALF_STEP).all()
