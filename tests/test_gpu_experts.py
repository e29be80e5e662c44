"""A layer of experts on the GPU (cri_expert_*) against its definitions in 64 bits (tests/experts_ref.py says how far off an
fp32 result may be and why).  Routing and grouping are whole numbers, equal; a choice's weight is computed in 64 bits and
rounded once: half a step of fp32, 2^-24, and 2^-50 for the order of 64-bit sums."""
import functools

import numpy as np
import pytest
import torch

import cretif_amd as cri
import experts_ref as ref
from cretif_amd import quant

pytestmark = pytest.mark.gpu

FORMATS = ["q8_0", "q4_0", "q5_0", "q4_k", "q6_k", "fp16"]
BLOCK = {"q4_k": 256, "q6_k": 256}


def randn(*shape, seed=0):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def ints(a):
    return dev(np.asarray(a, np.int32))


@functools.lru_cache(maxsize=8)
def matrix(fmt, E, N, K, seed=1):
    raw = quant.synthetic_weights(fmt, E * N, K, seed)
    return raw, ref.weights(fmt, raw, E, N, K)


def packed(fmt, E, N, K, seed=1):
    return cri.ExpertWeights(fmt, dev(matrix(fmt, E, N, K, seed)[0]), E, N, K)


def route_ids(M, E, k, kind, seed=0):
    """[M, k] ids: spread, all on one expert, on every third, with tokens without any, or one expert named twice."""
    rng = np.random.default_rng(seed)
    ids = np.argsort(rng.random((M, E)), 1)[:, :k]
    if kind == "one":
        ids[:, 0] = E // 2
        for t in range(M):
            rest = [e for e in ids[t, 1:] if e != E // 2]
            ids[t, 1:] = (rest + [e for e in range(E) if e != E // 2 and e not in rest])[:k - 1]
    if kind == "gaps":
        ids = ids // 3 * 3
        ids = np.where((np.arange(M) % 4 == 1)[:, None], -1, ids)
    if kind == "twice":
        ids[:, -1] = ids[:, 0]
    if kind == "away":
        ids = np.where(rng.random((M, k)) < 0.5, ids, E + 3)
    if kind == "none":
        ids[:] = -1
    return ids


def grouped(ids, E):
    g = cri.ExpertGroups(ids.shape[0], ids.shape[1], E)
    cri.group_experts(ints(ids), g)
    off, rows, slots = ref.group(ids, E)
    assert np.array_equal(g.offsets.cpu().numpy(), off)
    assert np.array_equal(g.rows.cpu().numpy(), rows)
    assert np.array_equal(g.slots.cpu().numpy(), slots)
    return g, off, rows, slots


def strided(rows, width, extra, fill=7.0):
    """(the whole buffer, a view of rows x width in wider rows, off 16-byte alignment)"""
    whole = torch.full((rows, width + extra), fill, device="cuda")
    return whole, whole[:, 1:1 + width] if extra else whole


def check_experts(got, make, off):
    for e in range(len(off) - 1):
        lo, hi = off[e], off[e + 1]
        if lo < hi:
            ref.check(got[lo:hi], make(e, lo, hi), "expert %d" % e)


# ---- grouping and routing -------------------------------------------------------------------------------------------


@pytest.mark.parametrize("M,E,k", [(1, 1, 1), (1, 128, 8), (3, 5, 5), (64, 8, 2), (65, 8, 2), (64, 1024, 64), (100, 64, 6),
                                   (4096, 32, 4), (4097, 1000, 1), (5003, 60, 8), (20000, 256, 8)])
@pytest.mark.parametrize("kind", ["spread", "one", "twice", "away"])
def test_group(M, E, k, kind):
    if kind == "one" and (k > 8 or M > 5000):
        pytest.skip("the ids take long to make")
    grouped(route_ids(M, E, k, kind, seed=M + E), E)


def test_group_of_strange_ids():
    ids = np.array([[0, -1], [2 ** 31 - 1, 3], [-2 ** 31, 4], [1, 1], [3, 3]])
    grouped(ids, 4)
    grouped(np.full((300, 3), -1), 7)


def test_no_tokens():
    g = cri.ExpertGroups(0, 2, 5)
    g.offsets.fill_(9)
    cri.group_experts(torch.zeros(0, 2, dtype=torch.int32, device="cuda"), g)
    assert (g.offsets == 0).all()
    g.offsets.fill_(9)
    empty = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    cri.route_experts(cri.ExpertRouter(), empty(0, 5), torch.zeros(0, 2, dtype=torch.int32, device="cuda"), empty(0, 2), g)
    assert (g.offsets == 0).all()
    w = packed("q8_0", 5, 32, 32)
    cri.expert_matmul(w, g, empty(0, 32), empty(0, 32))
    cri.expert_swiglu(w, w, g, empty(0, 32), empty(0, 32))
    cri.expert_combine(w, g, empty(0, 32), empty(0, 2), empty(0, 32))


def check_route(z, k, scoring, bias=None, normalize=True, scale=1.0, extra=0):
    M, E = z.shape
    whole, logits = strided(M, E, extra)
    logits.copy_(dev(z))
    g = cri.ExpertGroups(M, k, E)
    ids = torch.full((M, k), 77, dtype=torch.int32, device="cuda")
    weights = torch.full((M, k), 77.0, device="cuda")
    r = cri.ExpertRouter(scoring, None if bias is None else dev(bias), normalize, scale)
    cri.route_experts(r, logits, ids, weights, g)
    want, w = ref.route(z, k, scoring == "sigmoid", bias, normalize, np.float32(scale))
    assert np.array_equal(ids.cpu().numpy(), want)
    got = weights.cpu().double().numpy()
    assert (np.abs(got - w) <= (2.0 ** -24 + 2.0 ** -40) * np.abs(w) + 2.0 ** -149).all(), np.abs(got - w).max()
    off, rows, slots = ref.group(want, E)
    for a, b in ((g.offsets, off), (g.rows, rows), (g.slots, slots)):
        assert np.array_equal(a.cpu().numpy(), b)


@pytest.mark.parametrize("E,k", [(1, 1), (2, 1), (7, 7), (63, 3), (64, 8), (65, 8), (128, 8), (129, 5), (256, 6), (257, 64), (512, 8),
                                 (1000, 10), (1024, 8)])
@pytest.mark.parametrize("M", [1, 5, 64, 130])
def test_route(M, E, k):
    z = 2 * randn(M, E, seed=M + E)
    bias = 0.1 * randn(E, seed=3)
    check_route(z, k, "softmax")
    check_route(z, k, "softmax", None, False, 2.5, extra=3)
    check_route(z, k, "sigmoid", bias, True, 2.5, extra=1)
    check_route(z, k, "sigmoid", None, False)
    check_route(z, k, "softmax", bias, False)


@pytest.mark.parametrize("M", [1000, 4100])
def test_route_prompts(M):
    z = randn(M, 96, seed=M)
    z[M - 7:] = -np.inf
    check_route(z, 8, "sigmoid", 0.05 * randn(96, seed=1), True, 2.5)
    check_route(z, 4, "softmax", None, False)


@pytest.mark.parametrize("M", [4, 100])
def test_route_ties_and_what_is_never_chosen(M):
    z = np.round(2 * randn(M, 70, seed=5)).astype(np.float32)  # many ties
    z[0] = 0.5
    z[1] = -np.inf
    z[2, :] = np.nan
    z[3] = -np.inf
    z[3, [5, 69]] = [-3.0, 1.0]
    for scoring in ("softmax", "sigmoid"):
        check_route(z, 6, scoring)
        check_route(z, 6, scoring, None, False)
        check_route(z, 6, scoring, np.zeros(70, np.float32), True)
    bias = np.zeros(70, np.float32)
    bias[:60] = -np.inf
    bias[61] = np.nan
    check_route(z, 12, "sigmoid", bias, True)


def test_route_of_extreme_logits():
    z = np.array([[3e38, -3e38, 0, 1], [np.inf, np.inf, 5, -np.inf], [-800, -900, -1000, -750], [-100, -101, -102, -103],
                  [800, 700, 600, 750], [1e-45, 0, -1e-45, -0.0]], np.float32)
    for scoring in ("softmax", "sigmoid"):
        for normalize in (False, True):
            check_route(z, 3, scoring, None, normalize)
    check_route(z[3:], 3, "sigmoid", np.array([0, 1e-3, 2e-3, 0], np.float32), True)


# ---- products ------------------------------------------------------------------------------------------------------------

# tokens, experts, choices, columns, values: one token, few, a step, prompts; tiles of columns and of 256 values that are
# not full, experts without rows and with more than a tile of them
SIZES = [
    (1, 4, 2, 64, 256, "spread"), (1, 3, 1, 1, 32, "spread"), (2, 8, 8, 33, 96, "twice"), (5, 4, 3, 100, 288, "one"),
    (8, 16, 2, 257, 768, "gaps"), (9, 4, 4, 65, 544, "twice"), (16, 8, 2, 96, 1024, "spread"), (40, 4, 1, 31, 320, "one"),
    (70, 6, 2, 130, 512, "gaps"), (200, 3, 2, 290, 256, "one"), (333, 5, 2, 72, 608, "away"), (17, 4, 2, 64, 256, "none"),
]


def k_of(fmt, K):
    b = BLOCK.get(fmt, 32)
    return max(b, K // b * b)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,E,k,N,K,kind", SIZES)
def test_matmul(fmt, M, E, k, N, K, kind):
    K = k_of(fmt, K)
    ids = route_ids(M, E, k, kind, seed=M)
    g, off, rows, _ = grouped(ids, E)
    w = packed(fmt, E, N, K)
    v, mag = matrix(fmt, E, N, K)[1]
    x = randn(M, K, seed=M + 1)
    _, dx = strided(M, K, 3)
    dx.copy_(dev(x))
    whole, out = strided(M * k, N, 5)
    cri.expert_matmul(w, g, dx, out)
    tok = np.maximum(rows, 0) // k
    check_experts(out, lambda e, lo, hi: ref.Product(x[tok[lo:hi]], v[e], mag[e]), off)
    assert (whole[:, 0] == 7).all() and (whole[:, 1 + N:] == 7).all() and (out[off[-1]:] == 7).all()
    # rows in grouped order give the same
    xg = dev(x[tok])
    xg[off[-1]:] = float("nan")
    again = torch.full((M * k, N), 7.0, device="cuda")
    cri.expert_matmul(w, g, xg, again, grouped=True)
    assert torch.equal(again, out)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,E,k,N,K,kind", SIZES)
def test_swiglu(fmt, M, E, k, N, K, kind):
    K = k_of(fmt, K)
    ids = route_ids(M, E, k, kind, seed=M)
    g, off, rows, _ = grouped(ids, E)
    gate, up = (packed(fmt, E, N, K, seed) for seed in (1, 2))
    (gv, gm), (uv, um) = (matrix(fmt, E, N, K, seed)[1] for seed in (1, 2))
    x = 3 * randn(M, K, seed=M + 1)
    _, dx = strided(M, K, 2)
    dx.copy_(dev(x))
    whole, out = strided(M * k, N, 6)
    cri.expert_swiglu(gate, up, g, dx, out)
    tok = np.maximum(rows, 0) // k
    check_experts(out, lambda e, lo, hi: ref.Swiglu(x[tok[lo:hi]], (gv[e], gm[e]), (uv[e], um[e])), off)
    assert (whole[:, 0] == 7).all() and (whole[:, 1 + N:] == 7).all() and (out[off[-1]:] == 7).all()


def combined(x, v, mag, ids, slots, weights, residual):
    """The reference and its bars: the products' times |weight|, and k + 1 additions."""
    M, k = ids.shape
    N = v.shape[1]
    r = ref.Product(np.zeros((M, v.shape[2])), v[0], mag[0])
    r.want = np.zeros((M, N)) if residual is None else ref.f64(residual).copy()
    total = np.abs(r.want)
    square = np.zeros((M, N))
    for t in range(M):
        for j in range(k):
            s = slots[t * k + j]
            if s >= 0:
                p = ref.Product(x[s:s + 1], v[ids[t, j]], mag[ids[t, j]])
                w = float(weights[t, j])
                r.want[t] += w * p.want[0]
                r.worst[t] += abs(w) * p.worst[0]
                square[t] += (w * p.rms[0]) ** 2
                total[t] += abs(w * p.want[0])
    r.worst += (k + 1) * ref.U * total
    r.rms = np.sqrt(square) + np.sqrt(k + 1) * ref.U * total
    return r


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,E,k,N,K,kind", SIZES)
def test_combine(fmt, M, E, k, N, K, kind):
    K = k_of(fmt, K)
    ids = route_ids(M, E, k, kind, seed=M)
    g, off, rows, slots = grouped(ids, E)
    w = packed(fmt, E, N, K)
    v, mag = matrix(fmt, E, N, K)[1]
    x = randn(M * k, K, seed=M + 1)
    _, dx = strided(M * k, K, 1)
    dx.copy_(dev(x))
    dx[off[-1]:] = float("nan")  # rows behind the last are not read
    weights, res = randn(M, k, seed=M + 2), randn(M, N, seed=M + 3)
    whole, out = strided(M, N, 3)
    cri.expert_combine(w, g, dx, dev(weights), out)
    ref.check(out, combined(x, v, mag, ids, slots, weights, None))
    assert (whole[:, 0] == 7).all() and (whole[:, 1 + N:] == 7).all()
    want = combined(x, v, mag, ids, slots, weights, res)
    second = torch.empty(M, N, device="cuda")
    cri.expert_combine(w, g, dx, dev(weights), second, dev(res))
    ref.check(second, want)
    out.copy_(dev(res))
    cri.expert_combine(w, g, dx, dev(weights), out, out)  # in place
    assert torch.equal(out, second)


COLUMNS = [0, 1, 30, 31, 32, 63, 64, 255, 256, 300, 511, 512, 515, 1023, 1024, 2047, 2049, 3333, 4095, 4096, 4098, 4099]  # the checked ones


@functools.lru_cache(maxsize=8)
def wide(fmt, E, N, K, seed):
    """A matrix's blocks, and the values and magnitudes of some columns alone."""
    raw = quant.synthetic_weights(fmt, E * N, K, seed)
    some = np.asarray(raw).reshape(E, N, -1)[:, [c for c in COLUMNS if c < N]]
    return raw, ref.weights(fmt, np.ascontiguousarray(some).reshape(-1), E, some.shape[1], K)


def check_large(fmt, M, E, k, N, K):
    """All three products of a call, at some columns; a token without experts and every column finite."""
    cols = [c for c in COLUMNS if c < N]
    ids = route_ids(M, E, k, "spread", seed=M)
    ids[1] = -1
    g, off, rows, slots = grouped(ids, E)
    raws, refs = zip(*(wide(fmt, E, N, K, seed) for seed in (1, 2)))
    gate, up = (cri.ExpertWeights(fmt, dev(r), E, N, K) for r in raws)
    (gv, gm), (uv, um) = refs
    x = randn(M, K, seed=M + 1)
    tok = np.maximum(rows, 0) // k
    whole, out = strided(M * k, N, 3)
    at = torch.tensor(cols, device="cuda")
    cri.expert_matmul(gate, g, dev(x), out)
    check_experts(out[:, at], lambda e, lo, hi: ref.Product(x[tok[lo:hi]], gv[e], gm[e]), off)
    assert (out[off[-1]:] == 7).all() and torch.isfinite(out).all()
    whole.fill_(7.0)
    cri.expert_swiglu(gate, up, g, dev(x), out)
    check_experts(out[:, at], lambda e, lo, hi: ref.Swiglu(x[tok[lo:hi]], (gv[e], gm[e]), (uv[e], um[e])), off)
    assert (out[off[-1]:] == 7).all() and torch.isfinite(out).all()
    assert (whole[:, 0] == 7).all() and (whole[:, 1 + N:] == 7).all()
    h, weights, res = randn(M * k, K, seed=M + 2), randn(M, k, seed=M + 3), randn(M, N, seed=M + 4)
    h[off[-1]:] = np.nan
    whole, got = strided(M, N, 2)
    cri.expert_combine(gate, g, dev(h), dev(weights), got, dev(res))
    ref.check(got[:, at], combined(h, gv, gm, ids, slots, weights, res[:, cols]))
    assert torch.equal(got[1], dev(res)[1]) and torch.isfinite(got).all()
    assert (whole[:, 0] == 7).all() and (whole[:, 1 + N:] == 7).all()
    return gate, g


@pytest.mark.parametrize("fmt,K", [(f, K) for f in FORMATS for K in (32, 160, 416, 544, 640, 768, 1056) if K % BLOCK.get(f, 32) == 0])
@pytest.mark.parametrize("M", [24, 48, 96, 200, 400])
def test_wide_matrices(fmt, M, K):
    """Steps and prompts that take tiles of 16, 32 and 64 rows; K that ends inside 256 values after each number of 64, and
    inside 64."""
    w, g = check_large(fmt, M, 5, 2, 4100, K)
    if M >= 200:
        assert cri.expert_matmul_workspace_bytes(w, g) > 0  # the rows are split into their parts once for all tiles


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M", [40, 120, 300, 700])
def test_long_rows(fmt, M):
    """Few tiles of long rows: K is shared between workgroups, the last of them with less than the others."""
    K = 4352 if fmt in BLOCK else 4000
    w, g = check_large(fmt, M, 4, 2, 516, K)
    if M == 120:  # more than the rows' parts
        assert cri.expert_matmul_workspace_bytes(w, g) > M * (K + 255) // 256 * 256 * 4 + 2 * M * 516 * 4


@pytest.mark.parametrize("fmt", ["q4_k", "q6_k", "q8_0"])
@pytest.mark.parametrize("M", [4, 100])
def test_rows_of_any_magnitude(fmt, M):
    """Zero, tiny, huge and uneven rows keep their bars; a row that is not finite spoils its own results alone."""
    E, k, N, K = 2, 1, 40, 512
    x = randn(M, K, seed=9)
    x[0] = 0
    x[1] *= 1e-30
    x[2] *= 1e30
    x[3, 7] = 1e4
    ids = np.arange(M)[:, None] % E
    g, off, rows, _ = grouped(ids, E)
    v, mag = matrix(fmt, E, N, K)[1]
    w = packed(fmt, E, N, K)
    out = torch.empty(M, N, device="cuda")
    cri.expert_matmul(w, g, dev(x), out)
    r = g.slots.cpu().numpy()
    for t in range(M):
        ref.check(out[r[t]:r[t] + 1], ref.Product(x[t:t + 1], v[t % E], mag[t % E]), "token %d" % t)
    x[0, 3], x[2, 100] = np.inf, np.nan
    bad = torch.empty(M, N, device="cuda")
    cri.expert_matmul(w, g, dev(x), bad)
    for t in range(M):
        if t in (0, 2):
            assert not torch.isfinite(bad[r[t]]).any()
        else:
            assert torch.equal(bad[r[t]], out[r[t]])


@pytest.mark.parametrize("E,k,M", [(300, 4, 1000), (520, 2, 3000)])
def test_many_experts_of_many_rows(E, k, M):
    """More experts than a wave holds offsets of, tiles shared by many rows."""
    w, g = check_large("q4_0", M, E, k, 1028, 256)
    assert cri.expert_matmul_workspace_bytes(w, g) > 0


def test_rows_that_are_not_finite_in_a_wide_call():
    """As above, where the rows are split into their parts first and tiles are shared by many rows."""
    E, k, N, K, M = 3, 1, 4100, 768, 200
    for fmt in ("q4_k", "q5_0", "fp16"):
        w = cri.ExpertWeights(fmt, dev(wide(fmt, E, N, K, 1)[0]), E, N, K)
        g, _, _, slots = grouped(np.arange(M)[:, None] % E, E)
        x = randn(M, K, seed=8)
        x[5] *= 1e-35
        x[6] *= 1e30
        out, bad = torch.empty(M, N, device="cuda"), torch.empty(M, N, device="cuda")
        cri.expert_matmul(w, g, dev(x), out)
        assert torch.isfinite(out).all() and (out[slots[5]].abs() > 0).any()
        x[0, 3], x[70, 700], x[131, 0] = np.inf, np.nan, -np.inf
        cri.expert_matmul(w, g, dev(x), bad)
        hit = torch.tensor(slots[[0, 70, 131]], device="cuda").long()
        assert not torch.isfinite(bad[hit]).any()
        keep = torch.ones(M, dtype=torch.bool, device="cuda")
        keep[hit] = False
        assert torch.equal(bad[keep], out[keep])


@pytest.mark.parametrize("E,k,M", [(256, 8, 3), (257, 3, 5), (600, 9, 40), (1024, 64, 2), (1024, 2, 700)])
def test_many_experts(E, k, M):
    """More experts than a wave holds offsets of: every kernel's way to its rows."""
    N, K = 70, 256
    ids = route_ids(M, E, k, "spread", seed=E)
    ids[-1, 0] = E - 1
    ids[-1, 1:] = np.arange(k - 1)
    g, off, rows, slots = grouped(ids, E)
    w = packed("q4_0", E, N, K)
    v, mag = matrix("q4_0", E, N, K)[1]
    x = randn(M, K, seed=1)
    tok = np.maximum(rows, 0) // k
    out = torch.empty(M * k, N, device="cuda")
    cri.expert_matmul(w, g, dev(x), out)
    check_experts(out, lambda e, lo, hi: ref.Product(x[tok[lo:hi]], v[e], mag[e]), off)
    h, weights = randn(M * k, K, seed=2), randn(M, k, seed=3)
    got = torch.empty(M, N, device="cuda")
    cri.expert_combine(w, g, dev(h), dev(weights), got)
    ref.check(got, combined(h, v, mag, ids, slots, weights, None))


def test_any_alignment_of_the_blocks():
    """Raw blocks off every alignment (an expert's rows of 34 or 210 bytes begin anywhere)."""
    for fmt, K in (("q8_0", 96), ("q6_k", 256), ("q5_0", 32)):
        E, N = 3, 35
        raw, (v, mag) = matrix(fmt, E, N, K)
        buf = torch.empty(len(raw) + 1, dtype=torch.uint8, device="cuda")
        buf[1:].copy_(dev(raw))
        w = cri.ExpertWeights(fmt, buf[1:], E, N, K)
        x = randn(4, K, seed=2)
        g, off, rows, _ = grouped(np.array([[0], [1], [2], [1]]), E)
        out = torch.empty(4, N, device="cuda")
        cri.expert_matmul(w, g, dev(x), out)
        check_experts(out, lambda e, lo, hi: ref.Product(x[rows[lo:hi]], v[e], mag[e]), off)


@pytest.mark.parametrize("M", [2, 40])
def test_weights_past_4_gib(M):
    """Offsets that pass 32 bits: 4.8 GiB of FP16 weights, checked at the first, a middle and the last expert."""
    E, N, K = 40, 8192, 8192
    raw = torch.randn(E, N, K, device="cuda", generator=torch.Generator("cuda").manual_seed(3)).half()
    w = cri.ExpertWeights("fp16", raw.view(torch.uint8).reshape(-1), E, N, K)
    x = torch.randn(M, K, device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    ids = np.array([[0, E // 2, E - 1]] * M)
    g = cri.ExpertGroups(M, 3, E)
    cri.group_experts(ints(ids), g)
    out = torch.empty(M * 3, N, device="cuda")
    cri.expert_matmul(w, g, x, out)
    for i, e in enumerate((0, E // 2, E - 1)):
        cols = torch.tensor([0, 1, 31, 32, 4097, N - 1], device="cuda")
        v = raw[e][cols].cpu().double().numpy()
        p = ref.Product(x.cpu().numpy(), v, np.abs(v))
        ref.check(out[i * M:(i + 1) * M][:, cols], p, "expert %d" % e)


def test_groups_that_do_not_fit_stay_in_bounds():
    """Offsets out of order and numbers out of range: anything may come out, nowhere else."""
    E, N, K, M, k = 4, 40, 256, 20, 2
    w = packed("q4_k", E, N, K)
    x = dev(randn(M, K))
    rng = np.random.default_rng(0)
    for seed in range(6):
        wild = lambda n: ints(rng.choice([-2 ** 31, -5, 0, 3, 17, M * k, 2 ** 31 - 1, 1000], n))  # noqa: E731
        g = cri.ExpertGroups(M, k, E, wild(E + 1), wild(M * k), wild(M * k))
        whole = torch.full((M * k + 2, N), 7.0, device="cuda")
        cri.expert_matmul(w, g, x, whole[1:-1])
        cri.expert_swiglu(w, w, g, x, whole[1:-1])
        cri.expert_combine(w, g, dev(randn(M * k, K)), dev(randn(M, k)), whole[1:1 + M])
        few = cri.ExpertGroups(2, k, E, g.offsets, wild(2 * k), wild(2 * k))
        cri.expert_matmul(w, few, x[:2], whole[1:1 + 2 * k])
        assert (whole[0] == 7).all() and (whole[-1] == 7).all()
    N, M = 4100, 300
    w = packed("q4_k", E, N, K)
    for seed in range(3):
        wild = lambda n: ints(rng.choice([-2 ** 31, -5, 0, 3, 17, 200, M * k, 2 ** 31 - 1, 1000], n))  # noqa: E731
        g = cri.ExpertGroups(M, k, E, wild(E + 1), wild(M * k), wild(M * k))
        whole = torch.full((M * k + 2, N), 7.0, device="cuda")
        cri.expert_matmul(w, g, dev(randn(M, K)), whole[1:-1])
        cri.expert_swiglu(w, w, g, dev(randn(M, K)), whole[1:-1])
        cri.expert_combine(w, g, dev(randn(M * k, K)), dev(randn(M, k)), whole[1:1 + M])
        assert (whole[0] == 7).all() and (whole[-1] == 7).all()


# ---- together ------------------------------------------------------------------------------------------------------------


class Layer:
    """Router, gate, up and down of a layer of experts, the buffers of M tokens and a run of the operators over them."""

    def __init__(self, M, E=16, k=4, dim=256, inter=320, fmt="q8_0", down="q5_0"):
        self.M, self.E, self.k, self.dim, self.inter = M, E, k, dim, inter
        self.fmts = (fmt, fmt, down)
        self.router_w = 0.3 * randn(E, dim, seed=21)
        self.w = [packed(fmt, E, inter, dim, 1), packed(fmt, E, inter, dim, 2), packed(down, E, dim, inter, 3)]
        self.g = cri.ExpertGroups(M, k, E)
        self.router = cri.ExpertRouter("softmax", None, True, 1.0)
        f = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
        self.dr, self.logits, self.weights, self.h = dev(self.router_w), f(M, E), f(M, k), f(M * k, inter)
        self.ids = torch.zeros(M, k, dtype=torch.int32, device="cuda")
        self.x, self.out = f(M, dim), f(M, dim)
        need = max(cri.route_experts_workspace_bytes(self.g), cri.expert_swiglu_workspace_bytes(self.w[0], self.g),
                   cri.expert_combine_workspace_bytes(self.w[2], self.g))
        self.ws = torch.empty(need, dtype=torch.uint8, device="cuda")

    def run(self, stream=None):
        cri.matmul_transposed_b(self.x, self.dr, self.logits, self.M, self.E, self.dim, stream=stream)
        cri.route_experts(self.router, self.logits, self.ids, self.weights, self.g, self.ws, stream)
        cri.expert_swiglu(self.w[0], self.w[1], self.g, self.x, self.h, self.ws, stream)
        cri.expert_combine(self.w[2], self.g, self.h, self.weights, self.out, self.x, self.ws, stream)

    def check(self, x):
        """Against 64 bits from the layer's own logits (their order decides): the bars of both products, the first's
        error carried through the second."""
        ids, weights = ref.route(self.logits.cpu().numpy(), self.k, False, None, True, 1.0)
        assert np.array_equal(self.ids.cpu().numpy(), ids)
        (gv, gm), (uv, um) = (matrix(self.fmts[0], self.E, self.inter, self.dim, s)[1] for s in (1, 2))
        dv, dm = matrix(self.fmts[2], self.E, self.dim, self.inter, 3)[1]
        want, worst = x.astype(np.float64), np.zeros((self.M, self.dim))
        for t in range(self.M):
            for j, e in enumerate(ids[t]):
                h = ref.Swiglu(x[t:t + 1], (gv[e], gm[e]), (uv[e], um[e]))
                p = ref.Product(h.want, dv[e], dm[e])
                want[t] += weights[t, j] * p.want[0]
                worst[t] += weights[t, j] * (p.worst[0] + h.worst[0] @ np.abs(dv[e]).T + 2.0 ** -23 * np.abs(p.want[0]))
            worst[t] += (self.k + 1) * ref.U * np.abs(x[t]) + self.k * ref.U * np.abs(want[t])
        err = np.abs(ref.f64(self.out) - want)
        assert (err <= worst).all(), (err / worst).max()


@pytest.mark.parametrize("M", [1, 3, 24, 150])
def test_layer(M):
    layer = Layer(M)
    x = randn(M, layer.dim, seed=M)
    layer.x.copy_(dev(x))
    layer.run()
    layer.check(x)
    first = layer.out.clone()
    for _ in range(3):  # the same bits every time
        layer.out.zero_()
        layer.run()
        assert torch.equal(layer.out, first)


@pytest.mark.parametrize("M", [1, 24, 100])
def test_layer_captured(M):
    """One graph, replayed with other activations (and so other experts), eager calls of the same layer and of another one in
    between."""
    layer, other = Layer(M), Layer(7)
    s = torch.cuda.Stream()
    xs = [randn(M, layer.dim, seed=100 + i) for i in range(4)]
    layer.x.copy_(dev(xs[0]))
    with torch.cuda.stream(s):
        layer.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        layer.run()
    for x in xs + xs[:2]:
        layer.x.copy_(dev(x))
        layer.run()
        eager = layer.out.clone()
        layer.out.zero_()
        other.x.copy_(dev(randn(7, other.dim, seed=5)))
        other.run()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(layer.out, eager)
        layer.check(x)


@pytest.mark.parametrize("M,N,K", [(120, 516, 4352), (300, 516, 4352), (200, 4100, 768), (2, 516, 4352)])
def test_large_calls_captured(M, N, K):
    """Rows split into their parts, K shared between workgroups: a graph over one workspace, replayed with other activations and
    other choices, gives the eager calls' bits."""
    E, k = 4, 2
    w, up = (cri.ExpertWeights("q4_k", dev(wide("q4_k", E, N, K, seed)[0]), E, N, K) for seed in (1, 2))
    g = cri.ExpertGroups(M, k, E)
    f = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    x, h, weights, a, b, c = f(M, K), f(M * k, K), f(M, k), f(M * k, N), f(M * k, N), f(M, N)
    ids = torch.zeros(M, k, dtype=torch.int32, device="cuda")
    need = max(cri.expert_matmul_workspace_bytes(w, g), cri.expert_swiglu_workspace_bytes(w, g), cri.expert_combine_workspace_bytes(w, g),
               cri.route_experts_workspace_bytes(g), 16)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")

    def calls():
        cri.group_experts(ids, g, ws)
        cri.expert_matmul(w, g, x, a, ws)
        cri.expert_swiglu(w, up, g, x, b, ws)
        cri.expert_combine(w, g, h, weights, c, None, ws)

    def fill(seed):
        x.copy_(dev(randn(M, K, seed=seed)))
        h.copy_(dev(randn(M * k, K, seed=seed + 1)))
        weights.copy_(dev(randn(M, k, seed=seed + 2)))
        ids.copy_(ints(route_ids(M, E, k, "spread" if seed % 2 else "one", seed=seed)))

    s = torch.cuda.Stream()
    fill(0)
    with torch.cuda.stream(s):
        calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        calls()
    for seed in (1, 2, 3, 1):
        fill(seed)
        calls()
        eager = [t.clone() for t in (a, b, c)]
        for t in (a, b, c):
            t.zero_()
        ws.fill_(0xFF)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip((a, b, c), eager):
            assert torch.equal(got, want) and torch.isfinite(got).all()


def test_two_streams_at_once():
    """Two layers on two streams, each with its own workspace, against each alone."""
    layers = [Layer(24), Layer(40)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    alone = []
    for i, layer in enumerate(layers):
        layer.x.copy_(dev(randn(layer.M, layer.dim, seed=50 + i)))
        layer.run()
        alone.append(layer.out.clone())
        layer.out.zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for layer, s in zip(layers, streams):
            layer.run(s)
    torch.cuda.synchronize()
    for layer, want in zip(layers, alone):
        assert torch.equal(layer.out, want)


def test_python_refusals():
    """What the tensors say before the library is called."""
    E, N, K, M, k = 4, 32, 256, 3, 2
    w = packed("q4_k", E, N, K)
    raw = dev(matrix("q4_k", E, N, K)[0])
    g = cri.ExpertGroups(M, k, E)
    f = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    x, h, out, rows, ids, wts = f(M, K), f(M * k, K), f(M, N), f(M * k, N), i(M, k), f(M, k)
    ws = torch.empty(1 << 16, dtype=torch.uint8, device="cuda")
    with pytest.raises(KeyError):
        cri.ExpertWeights("q3_k", raw, E, N, K)
    with pytest.raises(KeyError):
        cri.ExpertRouter("relu")
    bad = [
        lambda: cri.ExpertWeights("q4_k", raw[:-1], E, N, K),
        lambda: cri.ExpertWeights("q4_k", raw.view(torch.int8), E, N, K),
        lambda: cri.ExpertWeights("q4_k", raw.cpu(), E, N, K),
        lambda: cri.ExpertWeights("q4_k", raw, E, N, 1 << 40),
        lambda: cri.ExpertGroups(M, k, E, offsets=i(E)),
        lambda: cri.ExpertGroups(M, k, E, rows=i(M * k).long()),
        lambda: cri.ExpertGroups(M, k, E, slots=i(M * k).cpu()),
        lambda: cri.ExpertGroups(-1, k, E),
        lambda: cri.ExpertRouter(bias=f(E).half()),
        lambda: cri.ExpertRouter(bias=f(2 * E)[::2]),
        lambda: cri.route_experts(cri.ExpertRouter(bias=f(E + 1)), f(M, E), ids, wts, g),
        lambda: cri.route_experts(cri.ExpertRouter(), f(M, E + 1), ids, wts, g),
        lambda: cri.route_experts(cri.ExpertRouter(), f(M, E).half(), ids, wts, g),
        lambda: cri.route_experts(cri.ExpertRouter(), f(M, E), ids.long(), wts, g),
        lambda: cri.route_experts(cri.ExpertRouter(), f(M, E), ids, f(k, M).t(), g),
        lambda: cri.group_experts(i(M, k + 1), g),
        lambda: cri.group_experts(ids.cpu(), g),
        lambda: cri.expert_matmul(w, g, h, rows),
        lambda: cri.expert_matmul(w, g, x, rows, grouped=True),
        lambda: cri.expert_matmul(w, g, x, out),
        lambda: cri.expert_matmul(w, g, x, f(M * k, N + 1)),
        lambda: cri.expert_matmul(w, g, x.cpu(), rows),
        lambda: cri.expert_matmul(w, g, x, rows, ws[::2]),
        lambda: cri.expert_swiglu(w, w, g, x.double(), rows),
        lambda: cri.expert_combine(w, g, h, wts[:-1], out),
        lambda: cri.expert_combine(w, g, h, wts, out, residual=f(M + 1, N)),
        lambda: cri.expert_combine(w, g, x, wts, out),
    ]
    for n, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail("call %d was not refused" % n)
    with pytest.raises(RuntimeError):
        cri.expert_matmul(w, cri.ExpertGroups(M, k, E + 1), x, rows)
    with pytest.raises(RuntimeError):
        cri.expert_swiglu(w, packed("q8_0", E, N, K), g, x, rows)
    with pytest.raises(RuntimeError):
        cri.expert_combine(w, g, h, wts, out, residual=f(M + 1, N)[1:].as_strided((M, N), (0, 1)))


def test_layer_of_a_padded_batch():
    """Rows of logits -infinity are nobody's: no work, weights 0, the residual alone comes out."""
    layer = Layer(40)
    x = randn(layer.M, layer.dim, seed=3)
    layer.x.copy_(dev(x))
    layer.run()
    full, slots = layer.out.clone(), layer.g.slots.clone()
    pad = torch.arange(layer.M, device="cuda") % 4 == 3
    layer.logits[pad] = float("-inf")
    cri.route_experts(layer.router, layer.logits, layer.ids, layer.weights, layer.g, layer.ws)
    assert int(layer.g.offsets[-1]) == 30 * layer.k
    layer.h.fill_(float("nan"))  # rows behind the last are neither written nor read
    cri.expert_swiglu(layer.w[0], layer.w[1], layer.g, layer.x, layer.h, layer.ws)
    assert torch.isnan(layer.h[30 * layer.k:]).all() and not torch.isnan(layer.h[:30 * layer.k]).any()
    cri.expert_combine(layer.w[2], layer.g, layer.h, layer.weights, layer.out, layer.x, layer.ws)
    assert torch.equal(layer.out[pad], layer.x[pad])
    assert torch.equal(layer.out[~pad], full[~pad])
