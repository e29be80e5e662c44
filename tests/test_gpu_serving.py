"""The batched serving operators on the GPU against their definitions in 64 bits (tests/serving_ref.py): head norms with
the rotation, the paged append, attention over pages with a shared prefix, draft verification, and a run of them together.

Bars, with u = 2^-24 half a step of fp32:
  * norm and rotation: the sum of squares is off by at most 13 u (8 fused additions, 5 levels of a tree), its square root,
    division by head_dim, eps and the reciprocal by 4 u more in the result, the two products by 2 u; sine and cosine by
    4 u (the half turn's rounding, u pi, and the function's); the rotation's products and sum by 2 u of the terms.  In all
    less than 24 u of the sum of the magnitudes that meet in an element.  Angles add the position times 2^-50.
  * rounding to the cache's type: half a step, 2^-11 (fp16), 2^-8 (bf16), and the smallest subnormal's half (fp16).
  * attention: fp32 accuracy.  A score of D terms is off by about sqrt(D) u of its terms' root sum, 1e-6 here, once more
    as much for its exponential, averaged over the positions of the row; operands taken in parts keep 2^-22 of each product.
    Bar 1e-5 of the row's largest, the bar of every fp32 path of this library.
  * verification: whole numbers, equal."""
import numpy as np
import pytest
import torch

import cretif_amd as cri
import serving_ref as ref

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"fp32": 0.0, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def randn(*shape, seed=0, scale=1.0):
    return (scale * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))).cuda()


# ---- norms and rotation -------------------------------------------------------------------------------------------


def check_rotated(got, x, w, positions, rot, halves, theta, D, eps=1e-6, extra=0.0):
    got, x = ref.f64(got).reshape(len(positions), -1, D), ref.f64(x).reshape(len(positions), -1, D)
    for t, p in enumerate(positions):
        want, mag = ref.norm_rotate(x[t], w, p, rot, halves, theta, eps)
        bar = (24 * U + abs(p) * 2.0 ** -50) * mag + extra * np.abs(want)
        assert (np.abs(got[t] - want) <= bar + 2.0 ** -25 * bool(extra)).all(), (t, p, np.abs(got[t] - want).max())


@pytest.mark.parametrize("M,H,Hkv,D,rot,halves,norm", [
    (1, 1, 1, 8, 8, True, True), (1, 32, 8, 128, 128, True, True), (3, 5, 1, 24, 16, True, False), (7, 4, 2, 80, 80, False, True),
    (2, 3, 3, 96, 48, True, True), (5, 8, 4, 64, 64, False, False), (4, 2, 1, 256, 256, True, True), (3, 2, 2, 256, 8, False, True),
    (6, 7, 7, 128, 0, True, True), (2, 1, 1, 136, 136, True, False), (1023, 3, 1, 64, 32, True, True), (1024, 3, 1, 64, 64, True, True),
    (1500, 40, 2, 16, 16, False, True),
])
def test_norm_rope(M, H, Hkv, D, rot, halves, norm):
    qkv = randn(M, (H + 2 * Hkv) * D + 3, seed=M + D)  # columns of wider rows, off 16-byte alignment
    q, k = qkv[:, 1:1 + H * D], qkv[:, 1 + H * D:1 + (H + Hkv) * D]
    wq, wk = (1 + 0.1 * randn(D, seed=1), 1 + 0.1 * randn(D, seed=2)) if norm else (None, None)
    pos = [(37 * m) % 5000 for m in range(M)]
    q_out = torch.full((M, H * D + 5), 7.0, device="cuda")
    k_out = torch.full((M, Hkv, D), 7.0, device="cuda")
    r = cri.Rotation(1e4, rot, "halves" if halves else "adjacent", wq, wk, 1e-6)
    cri.qk_norm_rope(r, q, k, q_out[:, :H * D], k_out, ints(pos), H, Hkv, D)
    check_rotated(q_out[:, :H * D], q, wq, pos, rot, halves, 1e4, D)
    check_rotated(k_out, k, wk, pos, rot, halves, 1e4, D)
    assert (q_out[:, H * D:] == 7).all()
    a, b = q.clone(), k.clone()  # in place, and each part alone: the same bits
    cri.qk_norm_rope(r, a, b, a, b, ints(pos), H, Hkv, D)
    assert torch.equal(a, q_out[:, :H * D]) and torch.equal(b, k_out.reshape(M, -1))
    c = torch.empty_like(a)
    cri.qk_norm_rope(r, q, None, c, None, ints(pos), H, 0, D)
    assert torch.equal(a, c)


@pytest.mark.parametrize("pos", [[0, 1, -1, -5000], [131071, 1 << 20, (1 << 24) + 1, (1 << 31) - 1]])
def test_far_positions(pos):
    q = randn(4, 2 * 128, seed=5)
    out = torch.empty_like(q)
    cri.qk_norm_rope(cri.Rotation(5e5, 128, "halves"), q, None, out, None, ints(pos), 2, 0, 128)
    check_rotated(out, q, None, pos, 128, True, 5e5, 128)


def test_norm_of_small_and_large_heads():
    """A head of zeros stays zeros, eps counts for tiny ones, large ones keep the bar."""
    q = randn(4, 64, seed=6)
    q[0] = 0
    q[1] *= 1e-6
    q[2] *= 1e15
    w = 1 + 0.1 * randn(64, seed=7)
    out = torch.empty_like(q)
    cri.qk_norm_rope(cri.Rotation(1e4, 64, "halves", w, None, 1e-5), q, None, out, None, ints([3, 4, 5, 6]), 1, 0, 64)
    assert (out[0] == 0).all()
    check_rotated(out, q, w, [3, 4, 5, 6], 64, True, 1e4, 64, eps=np.float32(1e-5))


# ---- pools and batches ---------------------------------------------------------------------------------------------


class Pool:
    """Pages of one type, an unwritten pattern in them, K and V interleaved page by page when `mixed`."""

    def __init__(self, n_pages, ps, Hkv, D, kind, seed=0, mixed=False):
        both = randn(n_pages, 2, ps, Hkv, D, seed=seed).to(TYPES[kind])
        if mixed:
            self.k, self.v = both[:, 0], both[:, 1]
        else:
            self.k, self.v = both[:, 0].contiguous(), both[:, 1].contiguous()
        self.kv = cri.PagedKV(self.k, self.v)


def tables(held, ps, seed=0, spare=2, shared=0):
    """Distinct pages for every sequence (the first `shared` the same for all), unused entries out of the pool."""
    need = [max(-(-h // ps), 0) for h in held]
    rng = np.random.default_rng(seed)
    total = shared + sum(max(n - shared, 0) for n in need) + spare
    order = [int(x) for x in rng.permutation(total)]
    width, rows, at = max(need + [1]) + 1, [], shared
    for n in need:
        own = max(n - shared, 0)
        rows.append((order[:shared] + order[at:at + own])[:max(n, shared)])
        at += own
        rows[-1] += [-1] * (width - len(rows[-1]))
    return total, [r[:width] for r in rows], order[:shared]


def starts(counts, first=0):
    return [first + sum(counts[:i]) for i in range(len(counts) + 1)]


# ---- append ---------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("counts,past,ps,H,Hkv,D,rot,halves,norm,mixed", [
    ([1], [0], 16, 8, 2, 64, 64, False, False, False),
    ([1] * 70, list(range(70)), 16, 4, 4, 128, 128, True, True, False),
    ([3, 0, 5, 1, 0], [10, 4, 0, 31, 0], 7, 6, 3, 80, 40, True, True, True),
    ([2, 2], [63, 64], 1, 2, 1, 24, 24, False, True, False),
    ([40, 1, 33], [5, 300, 0], 100, 5, 5, 256, 128, True, False, True),
    ([1200], [17], 32, 3, 1, 64, 64, True, True, False),
])
def test_append(kind, counts, past, ps, H, Hkv, D, rot, halves, norm, mixed):
    held = [a + b for a, b in zip(counts, past)]
    total, rows, _ = tables(held, ps)
    pool, ahead, behind = Pool(total, ps, Hkv, D, kind, mixed=mixed), 2, 3
    k0, v0 = pool.k.clone(), pool.v.clone()
    off, T = starts(counts, ahead), ahead + sum(counts) + behind
    qkv = randn(T, (H + 2 * Hkv) * D, seed=3)
    q, k, v = qkv[:, :H * D], qkv[:, H * D:(H + Hkv) * D], qkv[:, (H + Hkv) * D:]
    wq, wk = (1 + 0.1 * randn(D, seed=1), 1 + 0.1 * randn(D, seed=2)) if norm else (None, None)
    q_out = torch.full((T, H * D), 7.0, device="cuda")
    b = cri.PagedBatch(ints(off), ints(held), ints(rows))
    r = cri.Rotation(1e4, rot, "halves" if halves else "adjacent", wq, wk)
    cri.paged_append(pool.kv, b, r, k, v, q, q_out, H)
    pk, pv = pool.k.clone(), pool.v.clone()
    written = torch.zeros(total, ps, dtype=torch.bool)
    qs = []
    for t, s, p in ref.places(off, held, T):
        at = rows[s][p // ps], p % ps
        written[at] = True
        assert torch.equal(pv[at].reshape(-1), v[t].to(TYPES[kind])), (t, p)
        check_rotated(pk[at], k[t], wk, [p], rot, halves, 1e4, D, extra=HALF_STEP[kind])
        qs.append((t, p))
    check_rotated(q_out[[t for t, _ in qs]], q[[t for t, _ in qs]], wq, [p for _, p in qs], rot, halves, 1e4, D)
    keep = ~written.cuda()
    assert torch.equal(pk[keep], k0[keep]) and torch.equal(pv[keep], v0[keep])
    assert (q_out[:ahead] == 7).all() and (q_out[T - behind:] == 7).all()
    pool.k.copy_(k0)  # without queries: the same pages
    pool.v.copy_(v0)
    cri.paged_append(pool.kv, b, r, k, v)
    assert torch.equal(pool.k, pk) and torch.equal(pool.v, pv)


def test_lens_out_of_range():
    """Lengths of no meaning touch nothing: far below 0, below the rows."""
    ps, Hkv, D, H = 16, 2, 64, 4
    pool = Pool(4, ps, Hkv, D, "fp16")
    k0, v0 = pool.k.clone(), pool.v.clone()
    counts, held, rows = [1, 2, 1], [-2 ** 31, -5, -2 ** 31 + 1], [[0, 1], [2, 3], [1, 2]]
    b = cri.PagedBatch(ints(starts(counts)), ints(held), ints(rows))
    q, kv, q_out = randn(4, H * D), randn(4, Hkv * D, seed=1), torch.full((4, H * D), 7.0, device="cuda")
    cri.paged_append(pool.kv, b, cri.Rotation(1e4, 64), kv, kv, q, q_out, H)
    assert torch.equal(pool.k, k0) and torch.equal(pool.v, v0) and (q_out == 7).all()
    for P in (0, 20):
        out = torch.full((4, H * D), 7.0, device="cuda")
        cri.paged_attention(pool.kv, b, q, out, H, 0.125, ints([3, 0]), P)
        assert (out == 0).all()


def test_descriptors_of_another_device():
    """Descriptors made on one device are refused where another is current (their pointers are not that one's)."""
    pool = Pool(4, 16, 1, 64, "fp16")
    b = cri.PagedBatch(ints([0, 1]), ints([5]), ints([[0, 1]]))
    rot = cri.Rotation(1e4, 64, q_norm=randn(64))
    x, out = randn(1, 64), torch.zeros(1, 64, device="cuda")
    for thing in (pool.kv, b, rot):
        thing._dev += 1
        with pytest.raises(ValueError, match="current device"):
            cri.paged_append(pool.kv, b, rot, x, x)
        with pytest.raises(ValueError, match="current device"):
            if thing is rot:
                cri.qk_norm_rope(rot, x, None, out, None, ints([3]), 1, 0, 64)
            else:
                cri.paged_attention(pool.kv, b, x, out, 1, 0.125)
        thing._dev -= 1
    cri.paged_append(pool.kv, b, rot, x, x)
    cri.paged_attention(pool.kv, b, x, out, 1, 0.125)


def test_in_place_on_the_fused_rows():
    """q and k normed and rotated where the fused product left them; the values beside them untouched."""
    M, H, Hkv, D = 5, 4, 2, 64
    qkv = randn(M, (H + 2 * Hkv) * D, seed=8)
    src = qkv.clone()
    q, k = qkv[:, :H * D], qkv[:, H * D:(H + Hkv) * D]
    pos = [5, 900, 17, 0, 3]
    cri.qk_norm_rope(cri.Rotation(1e4, D, "halves"), q, k, q, k, ints(pos), H, Hkv, D)
    check_rotated(q, src[:, :H * D], None, pos, D, True, 1e4, D)
    check_rotated(k, src[:, H * D:(H + Hkv) * D], None, pos, D, True, 1e4, D)
    assert torch.equal(qkv[:, (H + Hkv) * D:], src[:, (H + Hkv) * D:])


def test_append_leaves_out_what_has_no_page():
    """Positions below 0 and past the table, page numbers outside the pool: those rows leave no trace."""
    ps, Hkv, D, H = 4, 1, 64, 2
    pool = Pool(5, ps, Hkv, D, "fp32")
    k0, v0 = pool.k.clone(), pool.v.clone()
    counts = [3, 2, 2, 2, 1]
    held = [1, 10, 3, 6, 2 ** 31 - 1]  # sequence 0: two rows below 0; 1: past the two pages of its table
    rows = [[0, 1], [2, 3], [-1, 4], [2 ** 31 - 1, 5], [0, 1]]
    q, k, v = randn(10, H * D), randn(10, D, seed=1), randn(10, D, seed=2)
    q_out = torch.full_like(q, 7.0)
    b = cri.PagedBatch(ints(starts(counts)), ints(held), ints(rows))
    cri.paged_append(pool.kv, b, cri.Rotation(1e4, 64), k, v, q, q_out, H)
    want_v, touched = v0.clone(), []
    for t, s, p in ref.places(starts(counts), held, 10):
        if 0 <= p < 2 * ps and 0 <= rows[s][p // ps] < 5:
            want_v[rows[s][p // ps], p % ps, 0] = v[t]
            touched.append(t)
    assert touched == [2]
    assert torch.equal(pool.v, want_v) and (pool.k != k0).any(-1).sum() == 1
    assert (q_out[[t for t in range(10) if t not in touched]] == 7).all() and (q_out[touched] != 7).all()


def test_append_offsets_past_32_bits():
    """A pool of more than 2^32 elements: the last page is written, and read by the attention."""
    ps, Hkv, D = 16, 8, 128
    n = 2 ** 32 // (ps * Hkv * D) + 3
    k = torch.zeros(n, ps, Hkv, D, dtype=torch.float16, device="cuda")
    kv = cri.PagedKV(k, k.clone())
    kk, vv = randn(3, Hkv * D, seed=1), randn(3, Hkv * D, seed=2)
    b = cri.PagedBatch(ints([0, 3]), ints([3]), ints([[n - 1]]))
    cri.paged_append(kv, b, cri.Rotation(1e4, 0), kk, vv)
    assert torch.equal(kv.v[n - 1, :3].reshape(3, -1), vv.half()) and torch.equal(kv.k[n - 1, :3].reshape(3, -1), kk.half())
    assert not kv.v[:n - 1].any() and not kv.v[n - 1, 3:].any()
    q, out = randn(3, Hkv * D, seed=3), torch.empty(3, Hkv * D, device="cuda")
    cri.paged_attention(kv, b, q, out, Hkv, D ** -0.5)
    small = cri.PagedKV(kv.k[n - 1:].clone(), kv.v[n - 1:].clone())
    want = torch.empty_like(out)
    cri.paged_attention(small, cri.PagedBatch(ints([0, 3]), ints([3]), ints([[0]])), q, want, Hkv, D ** -0.5)
    assert torch.equal(out, want)


# ---- attention ------------------------------------------------------------------------------------------------------


def attend(pool, off, held, rows, q, H, scale, prefix=None, P=0, out=None, **kw):
    out = torch.full((q.shape[0], q.shape[1]), 7.0, device="cuda") if out is None else out
    b = cri.PagedBatch(ints(off), ints(held), ints(rows))
    cri.paged_attention(pool.kv, b, q, out, H, scale, None if prefix is None else ints(prefix), P, **kw)
    return out


def check_rows(got, want, bar=1e-5):
    got = ref.f64(got)
    top = np.abs(want).max(-1, keepdims=True)
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= bar * top).all(), float((np.abs(got - want) / np.maximum(top, 1e-300)).max())


def case(kind, counts, own, P, ps, H, Hkv, D, seed=0, ahead=0, behind=0, qscale=2.0, mixed=False):
    """own: positions of each sequence behind the prefix, its rows' included."""
    held = [P + x for x in own]
    total, rows, first = tables(held, ps, seed=seed, shared=P // ps)
    prefix = first + ([total - 1] if P % ps else [])
    total += 1
    pool = Pool(total, ps, Hkv, D, kind, seed=seed + 1, mixed=mixed)
    if P % ps:
        prefix[-1] = total - 1
    off = starts(counts, ahead)
    q = randn(ahead + sum(counts) + behind, H * D, seed=seed + 2, scale=qscale)
    return pool, off, held, rows, prefix, q


SHAPES = [
    # counts, own, P, ps, H, Hkv, D
    ([1], [1], 0, 16, 1, 1, 64),                             # one position
    ([1], [33], 0, 16, 8, 2, 128),
    ([1, 1, 1], [1, 40, 700], 500, 16, 32, 8, 64),           # the prefix ends inside a page and a tile
    ([1] * 5, [3, 1, 17, 64, 31], 64, 32, 10, 5, 128),
    ([2, 5, 1, 3], [2, 9, 100, 40], 77, 64, 16, 2, 128),     # ragged drafts, eight heads to a key
    ([0, 4, 0, 1], [0, 4, 30, 1], 40, 16, 6, 2, 64),         # sequences without rows
    ([40, 7], [40, 90], 0, 16, 4, 1, 64),                    # pieces of prompts
    ([70, 1, 33], [70, 200, 64], 130, 16, 8, 2, 128),
    ([3, 2], [5, 70], 35, 7, 4, 2, 80),                      # pages and heads of other sizes
    ([2, 1, 6], [30, 64, 6], 33, 16, 3, 3, 24),
    ([1, 3], [300, 44], 100, 16, 4, 2, 256),
    ([9, 1], [50, 20], 21, 1, 7, 1, 200),
    ([1] * 70, [1 + i % 19 for i in range(70)], 96, 16, 4, 2, 64),   # more sequences than lanes
    ([1], [5], 3000, 16, 64, 1, 128),                        # one key head
    ([3] * 30, [3 + i for i in range(30)], 200, 16, 8, 1, 128),
]


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=[str(i) for i in range(len(SHAPES))])
def test_attention(kind, shape):
    counts, own, P, ps, H, Hkv, D = shape
    ahead, behind = 1, 2
    pool, off, held, rows, prefix, q = case(kind, counts, own, P, ps, H, Hkv, D, ahead=ahead, behind=behind, mixed=len(counts) % 2 == 0)
    out = attend(pool, off, held, rows, q, H, D ** -0.5, prefix, P)
    want = ref.attention(q, pool.k, pool.v, off, held, rows, prefix, P, H, D ** -0.5, torch.full(q.shape, 7.0))
    check_rows(out, want)
    assert (out[:ahead] == 7).all() and (out[len(q) - behind:] == 7).all()
    again = attend(pool, off, held, rows, q, H, D ** -0.5, prefix, P)
    assert torch.equal(out, again)  # sums in a fixed order


# many rows of a KV head on a long prefix: from 2^18 rows x positions on, with heads of 64 and 128 and pages of 16 n
# positions, the prefix is shared through LDS (else, and with other heads and pages: waves of their own)
MANY = [
    # counts, own, P, ps, H, Hkv, D
    ([1] * 33, [1 + 7 * i for i in range(33)], 256, 16, 4, 1, 64),         # a few rows, one tile, a whole number of tiles
    ([1] * 70, [1 + i % 40 for i in range(70)], 1000, 16, 8, 4, 128),      # ends inside a page and a tile
    ([3, 0, 5, 1] * 9, [3, 2, 50, 700] * 9, 481, 32, 8, 1, 128),           # 648 rows, ragged, sequences without any
    ([2] * 100, [2 + i for i in range(100)], 289, 64, 3, 3, 64),           # one position past a tile
    ([5] * 30, [5 + i for i in range(30)], 3000, 48, 10, 5, 64),           # many chunks
    ([40, 90], [40, 300], 320, 16, 4, 1, 128),                             # pieces of prompts: rows of two sequences in a tile
    ([1] * 40, [1 + i for i in range(40)], 300, 20, 8, 2, 128),            # pages of 20
    ([1] * 40, [1 + i for i in range(40)], 300, 16, 8, 2, 256),
    ([1] * 260, [1 + i % 90 for i in range(260)], 256, 16, 4, 1, 64),
    ([1] * 70, [1 + i % 40 for i in range(70)], 1000, 16, 8, 2, 128),
    ([2] * 155, [2 + i for i in range(155)], 289, 64, 3, 1, 64),
    ([1] * 9, [1 + 30 * i for i in range(9)], 8200, 32, 8, 2, 64),         # 44 rows
    ([40, 90], [40, 300], 505, 16, 4, 1, 128),
    ([1] * 70, [1 + i % 40 for i in range(70)], 1000, 20, 8, 2, 128),
    # other heads and pages, enough rows and positions that the prefix goes through LDS
    ([1] * 70, [1 + i % 40 for i in range(70)], 1001, 16, 8, 2, 80),
    ([2] * 60, [2 + i % 40 for i in range(60)], 1200, 16, 4, 2, 256),
    ([3, 0, 5, 1] * 9, [3, 2, 50, 90] * 9, 1000, 20, 8, 1, 256),
    ([1] * 70, [1 + i % 40 for i in range(70)], 1003, 1, 8, 2, 40),
    ([1] * 66, [1 + i % 40 for i in range(66)], 1070, 7, 8, 2, 200),
    ([1] * 70, [1 + i % 40 for i in range(70)], 1001, 24, 4, 1, 128),
    ([2] * 70, [2 + i % 40 for i in range(70)], 1024, 20, 4, 2, 64),
    ([5] * 30, [5 + i for i in range(30)], 3000, 50, 10, 5, 96),
    ([1] * 40, [1 + i for i in range(40)], 3301, 16, 4, 2, 8),
    ([1] * 36, [1 + i for i in range(36)], 7300, 33, 2, 2, 136),
    ([5] * 60, [5 + i for i in range(60)], 7001, 16, 4, 2, 256),
    ([4] * 40, [4 + i for i in range(40)], 6600, 33, 4, 1, 136),
]


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("shape", MANY, ids=[str(i) for i in range(len(MANY))])
def test_many_rows_on_a_prefix(kind, shape):
    counts, own, P, ps, H, Hkv, D = shape
    pool, off, held, rows, prefix, q = case(kind, counts, own, P, ps, H, Hkv, D, ahead=2, behind=3)
    bad = torch.ones(pool.k.shape[:2], dtype=torch.bool)  # what no position holds: never met, not even times zero
    for s, n in enumerate(held):
        for p in range(P, n):
            bad[rows[s][p // ps], p % ps] = False
    for p in range(P):
        bad[prefix[p // ps], p % ps] = False
    pool.k[bad.cuda()], pool.v[bad.cuda()] = float("nan"), float("inf")
    out = attend(pool, off, held, rows, q, H, D ** -0.5, prefix, P)
    want = ref.attention(q, pool.k, pool.v, off, held, rows, prefix, P, H, D ** -0.5, torch.full(q.shape, 7.0))
    check_rows(out, want)
    assert (out[:2] == 7).all() and (out[-3:] == 7).all()
    assert torch.equal(attend(pool, off, held, rows, q, H, D ** -0.5, prefix, P), out)


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("D,P,ps", [(64, 400, 16), (128, 400, 16), (64, 1000, 16), (128, 1000, 16), (256, 1000, 16),
                                    (80, 1000, 16), (128, 1000, 20), (200, 1000, 12), (256, 3900, 16),
                                    (200, 3900, 12)])
def test_many_rows_some_inside_the_prefix(kind, D, P, ps):
    """Rows that do not see the whole prefix, rows that see nothing and rows past their table, beside ordinary ones."""
    H, Hkv = 4, 1
    counts = [1] * 20 + [30, 6, 9, 1, 2, 1]
    held = [P + 5 + i for i in range(20)] + [P + 10, 3, P - 60, 1, 0, 5000]
    total, rows, _ = tables([P + 64] * len(held), ps)
    rows = [r[:(P + 64) // ps] for r in rows]
    pool = Pool(total, ps, Hkv, D, kind)
    prefix = [int(x) for x in np.random.default_rng(1).permutation(total)[:-(-P // ps)]]
    off = starts(counts)
    q = randn(sum(counts), H * D, seed=2)
    out = attend(pool, off, held, rows, q, H, D ** -0.5, prefix, P)
    pos = {t: p for t, _, p in ref.places(off, held, len(q))}
    want = ref.attention(q, pool.k, pool.v, off, held[:-1] + [len(rows[0]) * ps], rows, prefix, P, H, D ** -0.5, torch.zeros(q.shape))
    lost = [t for t in range(len(q)) if pos[t] < 0]
    assert len(lost) == 3 + 2 and (out[lost] == 0).all()
    keep = [t for t in range(len(q)) if pos[t] >= 0]
    check_rows(out[keep], want[keep])
    # a NaN at position 350 of the prefix reaches the rows that see it, no other
    pool.v[prefix[350 // ps], 350 % ps] = float("nan")
    got = attend(pool, off, held, rows, q, H, D ** -0.5, prefix, P)
    blind = [t for t in range(len(q)) if pos[t] < 350]
    assert len(blind) == 6 + (9 if P == 400 else 0) + 1 + 2 and torch.equal(got[blind], out[blind])
    assert torch.isnan(got[[t for t in range(len(q)) if pos[t] >= 350]]).all()


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("what", ["peak", "rising", "tiny_q", "huge_q", "large_v", "zero_q", "no_scale", "minus", "tiny_kv"])
@pytest.mark.parametrize("P", [700, 1500])
def test_many_rows_ranges(kind, what, P):
    H, Hkv, D, ps, scale = 8, 1, 128, 16, 128 ** -0.5
    pool, off, held, rows, prefix, q = case(kind, [2] * 12, [40 + i for i in range(12)], P, ps, H, Hkv, D)
    if what == "peak":
        pool.k[prefix[20], 3] *= 8
    elif what == "rising":
        for i, pg in enumerate(prefix):
            pool.k[pg] *= 0.05 * (1 + i)
    elif what == "tiny_q":
        q *= 2.0 ** -100
    elif what == "huge_q":
        q *= 2.0 ** 60
        scale *= 2.0 ** -60
    elif what == "large_v":
        pool.v[prefix[3]] *= 1000.0
    elif what == "zero_q":
        q[:5] = 0
    elif what == "no_scale":
        scale = 0.0
    elif what == "minus":
        scale = -scale
    else:  # subnormal fp16 numbers in the cache
        pool.k *= 2.0 ** -15
        pool.v *= 2.0 ** -15
        q *= 2.0 ** 15
    out = attend(pool, off, held, rows, q, H, scale, prefix, P)
    want = ref.attention(q, pool.k, pool.v, off, held, rows, prefix, P, H, np.float32(scale).astype(np.float64), torch.zeros(q.shape))
    check_rows(out, want)


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
def test_attention_without_a_prefix_is_the_same_mathematics(kind):
    """The prefix through the sequences' own tables gives what prefix_pages give."""
    counts, own, P, ps, H, Hkv, D = [1, 4, 2], [30, 4, 77], 96, 16, 8, 2, 128
    pool, off, held, rows, prefix, q = case(kind, counts, own, P, ps, H, Hkv, D)
    a = attend(pool, off, held, rows, q, H, D ** -0.5, prefix, P)
    b = attend(pool, off, held, rows, q, H, D ** -0.5)
    check_rows(a, ref.f64(b))


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("ps,D", [(16, 64), (16, 128), (9, 128), (16, 256)])
def test_rows_that_see_little(kind, ps, D):
    """Rows below position 0 see nothing and get zeros; rows inside the prefix see its first positions only; positions
    past the table are not seen."""
    H, Hkv, P = 4, 2, 40
    counts, held = [5, 3, 2, 1], [2, 30, 45, 4000]
    total, rows, _ = tables([100, 100, 100, 100], ps)
    rows = [r[:100 // ps] for r in rows]
    pool = Pool(total, ps, Hkv, D, kind)
    prefix = [int(x) for x in np.random.default_rng(1).permutation(total)[:-(-P // ps)]]
    off = starts(counts)
    q = randn(sum(counts), H * D, seed=2)
    out = attend(pool, off, held, rows, q, H, D ** -0.5, prefix, P)
    cap = len(rows[0]) * ps
    held_seen = held[:3] + [cap]
    want = ref.attention(q, pool.k, pool.v, off, held_seen, rows, prefix, P, H, D ** -0.5, torch.zeros(q.shape))
    check_rows(out[3:], want[3:])
    assert (out[:3] == 0).all()  # positions -3, -2, -1


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("ps,D,Hkv", [(16, 64, 2), (16, 128, 1), (10, 96, 2), (16, 256, 1)])
def test_what_lies_behind_a_row_never_reaches_it(kind, ps, D, Hkv):
    """NaN and infinities in stale pages, in pages of unused entries and in later drafts' keys and values."""
    H, P = 4 * Hkv, 24
    counts, own = [3, 1, 6], [11, 5, 6]
    pool, off, held, rows, prefix, q = case(kind, counts, own, P, ps, H, Hkv, D)
    clean = attend(pool, off, held, rows, q, H, D ** -0.5, prefix, P)
    used = torch.zeros(pool.k.shape[:2], dtype=torch.bool)
    for s, h in enumerate(held):
        for p in range(P, h):
            used[rows[s][p // ps], p % ps] = True
    for p in range(P):
        used[prefix[p // ps], p % ps] = True
    bad = ~used.cuda()
    pool.k[bad], pool.v[bad] = float("nan"), float("inf")
    assert torch.equal(attend(pool, off, held, rows, q, H, D ** -0.5, prefix, P), clean)
    # the last draft of sequence 2 goes bad: only its own row notices
    p = held[2] - 1
    pool.v[rows[2][p // ps], p % ps] = float("nan")
    got = attend(pool, off, held, rows, q, H, D ** -0.5, prefix, P)
    assert torch.equal(got[:-1], clean[:-1]) and torch.isnan(got[-1]).all()
    pool.v[rows[2][p // ps], p % ps] = float("inf")
    pool.k[rows[2][p // ps], p % ps] = float("nan")
    got = attend(pool, off, held, rows, q, H, D ** -0.5, prefix, P)
    assert torch.equal(got[:-1], clean[:-1]) and torch.isnan(got[-1]).all()


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
def test_a_nan_reaches_the_rows_that_see_it(kind):
    """A NaN key in the shared prefix, far from the first chunk: every row and head of its key head, no other."""
    H, Hkv, D, P, ps = 4, 2, 64, 1000, 16
    pool, off, held, rows, prefix, q = case(kind, [1, 2], [30, 60], P, ps, H, Hkv, D)
    pool.k[prefix[40], 3, 1] = float("nan")
    got = attend(pool, off, held, rows, q, H, D ** -0.5, prefix, P).reshape(3, H, D)
    assert torch.isnan(got[:, 2:]).all() and torch.isfinite(got[:, :2]).all()


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("many", [False, True])
def test_an_infinite_key_has_no_weight_or_shows(kind, many):
    """Keys of -infinity where the queries are positive: scores of -infinity.  A row is not finite, or as if those keys were
    not there; one that sees nothing else gets zeros or is not finite."""
    H, Hkv, D, P, ps = 8, 2, 128, 1000 if many else 40, 16
    counts = [2] * 40 if many else [2, 1, 3]
    pool, off, held, rows, prefix, q = case(kind, counts, [3 + i for i in range(len(counts))], P, ps, H, Hkv, D)
    q.abs_()
    pool.k[prefix[1], 5] = -float("inf")          # of all
    pool.k[rows[0][(held[0] - 1) // ps], (held[0] - 1) % ps] = -float("inf")  # of the last row of sequence 0
    out = attend(pool, off, held, rows, q, H, D ** -0.5, prefix, P)
    big = torch.where(pool.k.isinf(), torch.tensor(-1e4, device="cuda").to(pool.k.dtype), pool.k)
    want = ref.attention(q, big, pool.v, off, held, rows, prefix, P, H, D ** -0.5, torch.zeros(q.shape))
    bad = ~torch.isfinite(out).all(-1)
    check_rows(torch.where(bad[:, None], torch.from_numpy(want).float().cuda(), out), want)
    pool.k.fill_(-float("inf"))
    out = attend(pool, off, held, rows, q, H, D ** -0.5, prefix, P)
    assert ((out == 0) | ~torch.isfinite(out)).all()


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("what", ["peak", "rising", "tiny_q", "huge_q", "large_v", "spread_q", "zero_q", "no_scale", "minus", "tiny_kv"])
def test_attention_ranges(kind, what):
    H, Hkv, D, P, ps, scale = 8, 2, 128, 300, 16, 128 ** -0.5
    pool, off, held, rows, prefix, q = case(kind, [1, 3], [50, 700], P, ps, H, Hkv, D)
    if what == "peak":  # one position far above the others, met late
        pool.k[rows[1][-4], 1] *= 8
    elif what == "rising":  # every page raises the maximum
        for i, pg in enumerate(prefix):
            pool.k[pg] *= 0.1 * (1 + i)
    elif what == "tiny_q":
        q *= 2.0 ** -100
    elif what == "huge_q":
        q *= 2.0 ** 60
        scale *= 2.0 ** -60
    elif what == "large_v":
        pool.v *= 100.0
        pool.v[prefix[3]] *= 100.0
    elif what == "spread_q":  # dims of a query 2^12 apart
        q[:, ::2] *= 2.0 ** -12
    elif what == "zero_q":
        q[0] = 0
    elif what == "no_scale":
        scale = 0.0
    elif what == "minus":
        scale = -scale
    else:  # subnormal fp16 numbers in the cache
        pool.k *= 2.0 ** -15
        pool.v *= 2.0 ** -15
        q *= 2.0 ** 15
    out = attend(pool, off, held, rows, q, H, scale, prefix, P)
    want = ref.attention(q, pool.k, pool.v, off, held, rows, prefix, P, H, np.float32(scale).astype(np.float64), torch.zeros(q.shape))
    check_rows(out, want)


@pytest.mark.parametrize("many", [False, True])
def test_fp32_numbers_far_apart(many):
    """fp32 keys and values of any size: dims 2^20 apart that the scores all need, values 2^40 apart between heads, 2^100
    as a whole."""
    H, Hkv, D, P, ps = 8, 2, 128, 700 if many else 100, 16
    pool, off, held, rows, prefix, q = case("fp32", [2] * 60 if many else [2] * 3, [40 + i for i in range(60 if many else 3)],
                                            P, ps, H, Hkv, D)
    pool.k[..., ::2] *= 2.0 ** 20
    q[:, ::2] *= 2.0 ** -20
    pool.v[:, :, 1] *= 2.0 ** -40
    pool.v *= 2.0 ** 100
    out = attend(pool, off, held, rows, q, H, D ** -0.5, prefix, P)
    want = ref.attention(q, pool.k, pool.v, off, held, rows, prefix, P, H, D ** -0.5, torch.zeros(q.shape))
    for h in range(Hkv):  # each KV head by itself
        part = slice(h * 4 * D, (h + 1) * 4 * D)
        check_rows(out[:, part], want[:, part])


def check_heads(got, want, H, bar=1e-5):
    """Each head of a row against its own largest element."""
    check_rows(got.reshape(len(want) * H, -1), want.reshape(len(want) * H, -1), bar)


def sink(pool, place, q, H, scale, gap, spread, value, far, seed=0):
    """Keys whose scores lie `gap` below those of position place(0): queries have 4 in dim 0, where that key alone has
    something, and small numbers elsewhere; the others' scores differ by about `spread`.  The first value is `value` times the
    others', or (far) they rise from 2^-8 to 1 over the heads' dims."""
    Hkv, D = pool.k.shape[2:]
    q.mul_(0.5 * spread / (D - 1) ** 0.5 / scale).view(len(q), H, D)[:, :, 0] = 4.0
    pool.k[..., 0] = 0
    if far:
        pool.v.mul_(2.0 ** torch.linspace(-8, 0, D, device="cuda").to(pool.v.dtype))
    pg, at = place(0)
    pool.k[pg, at] = 0
    pool.k[pg, at, :, 0] = gap / scale / 4.0
    pool.v[pg, at] *= value


# One position takes almost all weight and has (next to) no value: the others, far below it, are the result.  Bars as above:
# the largest terms are the scores, up to 30 of 24 bits: 30 u in a probability's exponent.
@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("gap,spread,value", [(12, 0.0, 0.0), (15, 0.0, 0.0), (15, 1.0, 0.0), (18, 0.0, 0.0), (18, 1.0, 0.0), (21, 0.0, 0.0),
                                              (21, 1.0, 0.0), (18, 1.0, 2.0 ** -20), (18, 3.0, 2.0 ** -12), (26, 2.0, 0.0)])
@pytest.mark.parametrize("shape", [
    # counts, own, P, ps, H, Hkv, D: the position is the batch's first of the prefix, or each sequence's first
    ([1], [1024], 0, 16, 4, 1, 128),                               # one chunk or several
    ([1, 3], [31, 900], 0, 16, 8, 2, 64),
    ([2, 1], [700, 33], 0, 9, 6, 2, 80),                            # other heads and pages
    ([1, 2], [300, 500], 0, 16, 4, 1, 256),
    ([1], [20], 0, 16, 2, 1, 64),                                   # one chunk, straight to out
    ([1, 4], [30, 60], 700, 16, 8, 2, 128),                         # a prefix, waves of their own
    ([2] * 60, [2 + i % 40 for i in range(60)], 1200, 16, 8, 2, 128),   # through LDS
    ([2] * 70, [2 + i % 40 for i in range(70)], 1111, 20, 4, 2, 64),
    ([1] * 66, [1 + i % 40 for i in range(66)], 1070, 7, 8, 2, 120),
    ([2] * 40, [2 + i for i in range(40)], 8200, 16, 4, 2, 256),
    ([2] * 36, [2 + i for i in range(36)], 7400, 12, 4, 1, 200),
], ids=lambda s: "%dx%d_P%d_D%d" % (len(s[0]), s[0][0], s[2], s[6]))
def test_a_position_of_weight_without_value(kind, gap, spread, value, shape):
    counts, own, P, ps, H, Hkv, D = shape
    scale = D ** -0.5
    pool, off, held, rows, prefix, q = case(kind, counts, own, P, ps, H, Hkv, D, ahead=1, qscale=1.0)
    first = [(prefix[0], 0)] if P else [(r[0], 0) for r in rows]
    sink(pool, lambda i: first[i], q, H, scale, gap, spread, value, far=gap == 26)
    for pg, at in first[1:]:  # (every sequence's own)
        pool.k[pg, at], pool.v[pg, at] = pool.k[first[0]], pool.v[first[0]]
    out = attend(pool, off, held, rows, q, H, scale, prefix, P)
    want = ref.attention(q, pool.k, pool.v, off, held, rows, prefix, P, H, np.float64(np.float32(scale)), torch.full(q.shape, 7.0))
    check_heads(out[1:], want[1:], H)
    assert (out[0] == 7).all() and torch.equal(out, attend(pool, off, held, rows, q, H, scale, prefix, P))
    # a row is done again for itself alone: other queries beside it leave its bits
    other = q.clone()
    other[1::2] *= -1
    got = attend(pool, off, held, rows, other, H, scale, prefix, P)
    assert torch.equal(got[2::2], out[2::2])
    # what lies behind the rows still reaches none: those that are done again, too
    used = torch.zeros(pool.k.shape[:2], dtype=torch.bool)
    for s, n in enumerate(held):
        for p in range(P, n):
            used[rows[s][p // ps], p % ps] = True
    for p in range(P):
        used[prefix[p // ps], p % ps] = True
    bad = ~used.cuda()
    pool.k[bad], pool.v[bad] = float("nan"), float("inf")
    assert torch.equal(out, attend(pool, off, held, rows, q, H, scale, prefix, P))


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("steps", [0.6, 1.3, 10.4])
@pytest.mark.parametrize("shape", [
    # counts, own, P, ps, H, Hkv, D, wider: table entries behind the sequences' (chunks are long under wide tables)
    ([1] * 70, [1] * 70, 8192, 16, 8, 2, 128, 8000),  # through LDS
    ([7] * 20, [9] * 20, 2000, 5, 8, 2, 120, 6000),
    ([1], [2300], 0, 16, 8, 8, 64, 8000),
    ([1], [9], 3000, 16, 8, 8, 128, 8000),            # a prefix, waves of their own
], ids=["lds", "lds_other", "own", "prefix"])
def test_many_small_weights_beside_a_large_one(kind, steps, shape):
    """One position of weight 1 and thousands of `steps` half units in its last place: their sum counts, though each by itself
    rounds off, all of them the same way."""
    counts, own, P, ps, H, Hkv, D, wider = shape
    scale = D ** -0.5
    pool, off, held, rows, prefix, q = case(kind, counts, own, P, ps, H, Hkv, D)
    rows = [r + [-1] * wider for r in rows]
    place = (prefix[0], 0) if P else (rows[0][0], 0)
    pool.k.zero_()
    pool.k[place[0], place[1], :, 0] = 1.0
    q.zero_().view(len(q), H, D)[:, :, 0] = -np.log(steps * U) / scale
    out = attend(pool, off, held, rows, q, H, scale, prefix, P)
    t = counts[0] - 1  # the first sequence's last row
    want = ref.attention(q[t:t + 1], pool.k, pool.v, [0, 1], [P + own[0]], rows[:1], prefix, P, H, np.float64(np.float32(scale)), out[t:t + 1])
    check_heads(out[t:t + 1], want, H)


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("D,P,ps", [(64, 1000, 16), (128, 1000, 16), (256, 3900, 16), (80, 1000, 16), (128, 1000, 20), (200, 3900, 12),
                                    (128, 200, 16)])
def test_rows_inside_a_prefix_with_such_a_position(kind, D, P, ps):
    """Rows that are done again beside rows that see a part of the prefix, or nothing; a NaN behind some of them."""
    H, Hkv, scale = 4, 1, D ** -0.5
    counts = [1] * 20 + [30, 6, 9, 1, 2, 1]
    held = [P + 5 + i for i in range(20)] + [P + 10, 3, P - 60, 1, 0, 5000]
    total, rows, _ = tables([P + 64] * len(held), ps)
    rows = [r[:(P + 64) // ps] for r in rows]
    pool = Pool(total, ps, Hkv, D, kind)
    prefix = [int(x) for x in np.random.default_rng(1).permutation(total)[:-(-P // ps)]]
    off = starts(counts)
    q = randn(sum(counts), H * D, seed=2)
    sink(pool, lambda i: (prefix[0], 0), q, H, scale, 18, 1.0, 0.0, False)
    pos = np.array([p for _, _, p in ref.places(off, held, len(q))])
    want = ref.attention(q, pool.k, pool.v, off, held[:-1] + [len(rows[0]) * ps], rows, prefix, P, H, np.float64(np.float32(scale)), torch.zeros(q.shape))
    out = attend(pool, off, held, rows, q, H, scale, prefix, P)
    check_heads(out, want, H)
    assert (out[pos < 0] == 0).all() and (out[pos == 0] == 0).all() and (pos < 0).sum() == 5 and (pos == 0).sum() == 2
    pool.v[prefix[150 // ps], 150 % ps] = float("nan")
    got = attend(pool, off, held, rows, q, H, scale, prefix, P)
    assert torch.equal(got[pos < 150], out[pos < 150]) and torch.isnan(got[pos >= 150]).all() and (pos >= 150).sum() > 50


def test_strided_rows_and_a_given_workspace():
    H, Hkv, D, P, ps = 8, 2, 64, 40, 16
    pool, off, held, rows, prefix, q = case("fp16", [1, 4], [20, 100], P, ps, H, Hkv, D)
    want = attend(pool, off, held, rows, q, H, 0.125, prefix, P)
    wide = torch.full((5, H * D + 9), 3.0, device="cuda")
    wide[:, 1:1 + H * D] = q
    res = torch.full((5, H * D + 7), 7.0, device="cuda")
    b = cri.PagedBatch(ints(off), ints(held), ints(rows))
    n = cri.paged_attention_workspace_bytes(pool.kv, b, 5, H, P)
    room = torch.full((n + 64,), 255, dtype=torch.uint8, device="cuda")  # NaNs: nothing is read before it is written
    cri.paged_attention(pool.kv, b, wide[:, 1:1 + H * D], res[:, 3:3 + H * D], H, 0.125, ints(prefix), P, room[:n])
    assert torch.equal(res[:, 3:3 + H * D], want) and (res[:, :3] == 7).all() and (res[:, 3 + H * D:] == 7).all()
    assert (room[n:] == 255).all()
    with pytest.raises(ValueError, match="workspace"):
        cri.paged_attention(pool.kv, b, q, res[:, :H * D], H, 0.125, ints(prefix), P, stream=torch.cuda.Stream())
    with pytest.raises(ValueError, match="prefix_pages"):
        cri.paged_attention(pool.kv, b, q, res[:, :H * D], H, 0.125, ints(prefix[:1]), P)
    with pytest.raises(ValueError, match="rows"):
        cri.paged_attention(pool.kv, b, q[:4], res[:, :H * D], H, 0.125)


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("n,past,P,ps,H,Hkv,D,positions", [
    (1100, 0, 0, 16, 32, 8, 128, 131072),   # a prompt under a table of the longest context: the records' bound is met
    (1030, 700, 0, 16, 8, 2, 64, 1792),
    (1025, 90, 300, 20, 8, 1, 128, 1500),   # behind a shared prefix
    (2049, 0, 0, 16, 4, 4, 128, 2064),
])
def test_a_prompts_rows(kind, n, past, P, ps, H, Hkv, D, positions):
    """Many rows of one sequence (their causal limits run through all its tiles), and a workspace of no more than 1 GiB."""
    held = P + past + n
    need, first = -(-held // ps), -(-P // ps)
    order = [int(x) for x in np.random.default_rng(3).permutation(need + first)]
    rows, prefix = [order[:need] + [-1] * (-(-positions // ps) - need)], order[need:]
    pool = Pool(need + first, ps, Hkv, D, kind, seed=4)
    q = randn(n, H * D, seed=5, scale=2.0)
    b = cri.PagedBatch(ints([0, n]), ints([held]), ints(rows))
    room = cri.paged_attention_workspace_bytes(pool.kv, b, n, H, P)
    assert room <= 1 << 30
    ws = torch.full((room + 64,), 255, dtype=torch.uint8, device="cuda")  # NaNs
    out = attend(pool, [0, n], [held], rows, q, H, D ** -0.5, prefix, P, workspace=ws[:room])
    assert (ws[room:] == 255).all()
    j = np.arange(held)
    page = np.array([prefix[x // ps] if x < P else order[x // ps] for x in j])
    k, v = ref.f64(pool.k)[page, j % ps], ref.f64(pool.v)[page, j % ps]
    seen = j[None, :] <= (held - n + np.arange(n))[:, None]
    got, x = ref.f64(out).reshape(n, H, D), ref.f64(q).reshape(n, H, D)
    for h in range(0, H, 3):
        s = np.where(seen, x[:, h] @ k[:, h * Hkv // H].T * D ** -0.5, -np.inf)
        w = np.exp(s - s.max(-1, keepdims=True))
        check_rows(got[:, h], (w / w.sum(-1, keepdims=True)) @ v[:, h * Hkv // H])
    assert torch.equal(out, attend(pool, [0, n], [held], rows, q, H, D ** -0.5, prefix, P))


# ---- verification ---------------------------------------------------------------------------------------------------


def check_verify(target, draft, ids, u, draws, off, ahead=0):
    T, B = len(target), len(off) - 1
    out, acc = torch.full((T,), -7, dtype=torch.int32, device="cuda"), torch.full((B,), -7, dtype=torch.int32, device="cuda")
    cri.verify_drafts(target, draft, ints(ids), u, draws, ints(off), out, acc)
    want, wacc = ref.verify(target, draft, ids, u, draws, off, np.full(T, -7), np.full(B, -7))
    assert acc.tolist() == wacc.tolist()
    assert out.tolist() == want.tolist()
    return out, acc


def drafts(counts, V, seed, sure, near=1.0, first=0, behind=0):
    T = first + sum(counts) + behind
    logits = randn(T, V, seed=seed, scale=2.0)
    target = torch.softmax(logits, -1)
    draft = None if sure else torch.softmax(logits + near * randn(T, V, seed=seed + 1), -1)
    g = torch.Generator().manual_seed(seed + 2)
    src = target if sure else draft
    ids = torch.multinomial(src.cpu().double(), 1, generator=g).flatten().tolist()
    return target, draft, ids, torch.rand(T, generator=g).cuda(), torch.rand(T, generator=g).cuda(), starts(counts, first)


@pytest.mark.parametrize("sure", [False, True])
@pytest.mark.parametrize("counts,V", [
    ([1], 1), ([2], 2), ([1], 1000), ([5], 128256), ([3, 0, 1, 6, 2], 1023), ([4] * 9, 1024), ([9, 1, 2], 1025),
    ([70, 3], 50), ([2] * 300, 257), ([1 + i % 7 for i in range(40)], 5000),
    ([1100, 3], 40), ([2, 1, 4], 4096), ([3, 3], 4097), ([4, 2], 32767), ([3, 1, 2, 5], 32768), ([2, 4, 1], 32769),
    ([5, 3], 20000), ([1030, 2], 32800),
])
def test_verify(sure, counts, V):
    check_verify(*drafts(counts, V, seed=V + len(counts), sure=sure, first=2, behind=1))


def test_verify_strided_probabilities():
    target, draft, ids, u, d, off = drafts([3, 4], 300, seed=1, sure=False)
    a, b = torch.full((7, 333), float("nan"), device="cuda"), torch.full((7, 301), float("nan"), device="cuda")
    a[:, 5:305], b[:, 1:] = target, draft
    check_verify(a[:, 5:305], b[:, 1:], ids, u, d, off)


def test_verify_the_same_distribution_accepts_all():
    target, _, _, _, d, off = drafts([6, 6], 500, seed=2, sure=False)
    ids = target.argmax(-1).tolist()
    _, acc = check_verify(target, target, ids, torch.full((12,), 1 - 2.0 ** -24, device="cuda"), d, off)
    assert acc.tolist() == [5, 5]


@pytest.mark.parametrize("d", [0.0, 0.5, 1 - 2.0 ** -24, 1.0, 5.0, -1.0, float("nan")])
@pytest.mark.parametrize("V", [8, 2048, 5000, 40000])
def test_verify_borders(d, V):
    """Equal weights of a power of two: the running sum meets the number exactly; zeros at both ends."""
    p = torch.zeros(2, V, device="cuda")
    p[:, 2:6] = 0.25
    out, _ = check_verify(p, None, [7, 0], torch.tensor([0.5, 0.5]).cuda(), torch.tensor([d, d]).cuda(), [0, 2])
    assert out[0].item() == {0.0: 2, 0.5: 4, -1.0: 2}.get(d, 5)


@pytest.mark.parametrize("V", [1500, 33000])
def test_verify_odd_probabilities(V):
    """Invalid drafted tokens, drafts that leave nothing, rows of zeros, of NaN, of negatives."""
    t = torch.softmax(randn(12, V, seed=3), -1)
    q = torch.softmax(randn(12, V, seed=4), -1)
    q[0] = 2.0           # row 0: the draft leaves nothing of the target
    t[2] = 0             # row 2: no weight at all
    t[4] = float("nan")
    t[6, ::2] = -1.0
    t[6, 1::4] = float("nan")
    q[8] = float("nan")
    ids = [3, 0, 5, 0, 5, 0, 7, 0, 9, 0, -1, V]
    u, d = torch.full((12,), 0.999, device="cuda"), torch.rand(12, generator=torch.Generator().manual_seed(5)).cuda()
    out, _ = check_verify(t, q, ids, u, d, [0, 2, 4, 6, 8, 10, 12])
    assert out[2].item() == -1 and out[4].item() == -1
    check_verify(t, None, ids, u, d, [0, 2, 4, 6, 8, 10, 12])
    check_verify(t, q, [V] * 12, u, d, [0, 12])


@pytest.mark.parametrize("V", [3000, 50000])
def test_verify_leaves_no_trace_in_the_workspace_of_others(V):
    target, draft, ids, u, d, off = drafts([3, 4, 2], V, seed=6, sure=False)
    n = cri.verify_drafts_workspace_bytes(3, V)
    room = torch.full((n + 64,), 255, dtype=torch.uint8, device="cuda")
    out, acc = torch.zeros(9, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    cri.verify_drafts(target, draft, ints(ids), u, d, ints(off), out, acc, room[:n])
    want, wacc = ref.verify(target, draft, ids, u, d, off, np.zeros(9, int), np.zeros(3, int))
    assert out.tolist() == want.tolist() and acc.tolist() == wacc.tolist() and (room[n:] == 255).all()


# ---- together -------------------------------------------------------------------------------------------------------


class Serving:
    """A layer's worth of a serving step with drafts: append, attention, probabilities, verification."""

    H, Hkv, D, V, P, ps, N = 8, 2, 64, 300, 40, 16, 4  # N rows per sequence: the last token and three drafts

    def __init__(self, B, kind):
        self.B, T = B, B * self.N
        room = 200
        need = -(-room // self.ps)
        self.pool = Pool(B * need + 3, self.ps, self.Hkv, self.D, kind, seed=9)
        self.pages = ints([[s * need + i for i in range(need)] for s in range(B)])
        self.prefix = ints([B * need, B * need + 1, B * need + 2])
        self.offsets, self.lens = ints(starts([self.N] * B)), ints([self.P + self.N + 3 * s for s in range(B)])
        self.table = randn(self.V, (self.H + 2 * self.Hkv) * self.D, seed=10)  # a token's q, k, v
        self.head = randn(self.H * self.D, self.V, seed=11, scale=0.2)
        self.rot = cri.Rotation(1e4, self.D, "halves", 1 + 0.1 * randn(self.D, seed=12), 1 + 0.1 * randn(self.D, seed=13))
        self.batch = cri.PagedBatch(self.offsets, self.lens, self.pages)
        f = dict(device="cuda")
        self.ids = torch.randint(0, self.V, (T,), generator=torch.Generator().manual_seed(14)).int().cuda()
        self.next = torch.zeros(T, dtype=torch.int32, **f)  # row j: the draft that follows it
        self.u, self.d = torch.zeros(T, **f), torch.zeros(T, **f)
        self.q, self.out = torch.zeros(T, self.H * self.D, **f), torch.zeros(T, self.H * self.D, **f)
        self.tokens, self.accepted = torch.zeros(T, dtype=torch.int32, **f), torch.zeros(B, dtype=torch.int32, **f)
        self.ws = torch.zeros(cri.paged_attention_workspace_bytes(self.pool.kv, self.batch, T, self.H, self.P), dtype=torch.uint8, **f)
        self.vs = torch.zeros(cri.verify_drafts_workspace_bytes(B, self.V), dtype=torch.uint8, **f)
        self.probs = torch.zeros(T, self.V, **f)

    def step(self):
        qkv = self.table[self.ids.long()]
        a, b = self.H * self.D, (self.H + self.Hkv) * self.D
        cri.paged_append(self.pool.kv, self.batch, self.rot, qkv[:, a:b], qkv[:, b:], qkv[:, :a], self.q, self.H)
        cri.paged_attention(self.pool.kv, self.batch, self.q, self.out, self.H, self.D ** -0.5, self.prefix, self.P, self.ws)
        self.probs.copy_(torch.softmax(self.out @ self.head, -1))
        cri.verify_drafts(self.probs, None, self.next, self.u, self.d, self.offsets, self.tokens, self.accepted, self.vs)

    def draw(self, seed):
        g = torch.Generator().manual_seed(seed)
        T = self.B * self.N
        self.u.copy_(torch.rand(T, generator=g))
        self.d.copy_(torch.rand(T, generator=g))
        ids = self.ids.view(self.B, self.N)
        self.next.view(self.B, self.N)[:, :-1].copy_(ids[:, 1:])

    def advance(self):
        """The step's tokens become positions; the drawn token starts the next rows, drafts are looked up in the step."""
        tok, acc = self.tokens.view(self.B, self.N), self.accepted.long()
        last = tok.gather(1, acc[:, None])
        ids = self.ids.view(self.B, self.N).clone()
        ids[:, 1:] = (ids[:, :-1] * 7 + last) % self.V
        ids[:, :1] = last
        self.ids.copy_(ids.flatten())
        self.lens.add_(self.accepted + 1)


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
def test_steps_of_a_batch(kind):
    """Three steps, each operator's results against the definitions on the step's own state."""
    m = Serving(3, kind)
    for step in range(3):
        m.draw(step)
        before = m.pool.k.clone(), m.pool.v.clone()
        ids, lens, nxt = m.ids.tolist(), m.lens.tolist(), m.next.tolist()
        m.step()
        off, rows = m.offsets.tolist(), m.pages.tolist()
        qkv = m.table[m.ids.long()]
        a, b = m.H * m.D, (m.H + m.Hkv) * m.D
        for t, s, p in ref.places(off, lens, len(ids)):
            at = rows[s][p // m.ps], p % m.ps
            check_rotated(m.q[t], qkv[t, :a], m.rot.q_norm, [p], m.D, True, 1e4, m.D)
            check_rotated(m.pool.k[at], qkv[t, a:b], m.rot.k_norm, [p], m.D, True, 1e4, m.D, extra=HALF_STEP[kind])
            assert torch.equal(m.pool.v[at].flatten(), qkv[t, b:].to(TYPES[kind]))
            before[0][at], before[1][at] = m.pool.k[at], m.pool.v[at]
        assert torch.equal(before[0], m.pool.k) and torch.equal(before[1], m.pool.v)
        check_rows(m.out, ref.attention(m.q, m.pool.k, m.pool.v, off, lens, rows, m.prefix.tolist(), m.P, m.H, m.D ** -0.5, m.out))
        want, acc = ref.verify(m.probs, None, nxt, m.u, m.d, off, np.zeros(len(ids), int), np.zeros(m.B, int))
        assert m.tokens.tolist() == want.tolist() and m.accepted.tolist() == acc.tolist()
        m.advance()


def test_captured_steps_match_eager_ones():
    """A step captured once and replayed while lens, tokens and numbers change, eager work between: the eager bits.  Two
    graphs share the workspaces."""
    eager, graph = Serving(4, "fp16"), Serving(4, "fp16")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(s):
        keep = [x.clone() for x in (graph.pool.k, graph.pool.v)]
        graph.draw(0)
        graph.step()  # warm
        graph.pool.k.copy_(keep[0])
        graph.pool.v.copy_(keep[1])
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                graph.step()
            graphs.append(g)
    torch.cuda.synchronize()
    for i in range(6):
        eager.draw(i)
        eager.step()
        graph.draw(i)
        torch.cuda.synchronize()
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(eager.q, graph.q) and torch.equal(eager.out, graph.out), i
        assert torch.equal(eager.tokens, graph.tokens) and torch.equal(eager.accepted, graph.accepted), i
        assert torch.equal(eager.pool.k, graph.pool.k) and torch.equal(eager.pool.v, graph.pool.v), i
        eager.advance()
        graph.advance()


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
def test_captured_attention_of_many_rows(kind):
    """Captured once, replayed while the sequences grow, with eager work between: the eager bits."""
    H, Hkv, D, P, ps = 8, 2, 128, 1000, 16
    own = [1 + i % 40 for i in range(70)]
    pool, off, held, rows, prefix, q = case(kind, [1] * 70, [x + 60 for x in own], P, ps, H, Hkv, D)
    lens = ints([P + x for x in own])
    b = cri.PagedBatch(ints(off), lens, ints(rows))
    pp, ws = ints(prefix), torch.empty(cri.paged_attention_workspace_bytes(pool.kv, b, 70, H, P), dtype=torch.uint8, device="cuda")
    out, want = torch.zeros_like(q), torch.zeros_like(q)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        cri.paged_attention(pool.kv, b, q, out, H, D ** -0.5, pp, P, ws)
    for _ in range(5):
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        cri.paged_attention(pool.kv, b, q, want, H, D ** -0.5, pp, P, ws)
        assert torch.equal(out, want)
        lens += 11
        q.mul_(-0.9)


@pytest.mark.parametrize("P,own", [(1000, 70), (0, 400)])
def test_captured_rows_that_are_done_again(P, own):
    """fp16 rows that are multiplied again (a position of weight without value) in a captured call, replayed while queries and
    lengths change and eager calls run between: the eager bits."""
    H, Hkv, D, ps = 8, 2, 128, 16
    n = 70 if P else 5
    pool, off, held, rows, prefix, q = case("fp16", [1] * n, [own + i % 30 for i in range(n)], P, ps, H, Hkv, D)
    first = (prefix[0], 0) if P else (rows[0][0], 0)
    sink(pool, lambda i: first, q, H, D ** -0.5, 20, 1.0, 0.0, False)
    for r in rows:
        pool.k[r[0], 0], pool.v[r[0], 0] = pool.k[first], pool.v[first]
    lens, pp = ints([h - 60 for h in held]), ints(prefix) if P else None
    b = cri.PagedBatch(ints(off), lens, ints(rows))
    ws = torch.empty(cri.paged_attention_workspace_bytes(pool.kv, b, n, H, P), dtype=torch.uint8, device="cuda")
    out, want = torch.zeros_like(q), torch.zeros_like(q)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        cri.paged_attention(pool.kv, b, q, out, H, D ** -0.5, pp, P, ws)
    for i in range(5):
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        cri.paged_attention(pool.kv, b, q, want, H, D ** -0.5, pp, P, ws)
        assert torch.equal(out, want)
        check_heads(out, ref.attention(q, pool.k, pool.v, off, lens.tolist(), rows, prefix, P, H, np.float64(np.float32(D ** -0.5)), out), H)
        lens += 11
        q.mul_(0.97)


def test_a_side_stream_orders_with_torch():
    want = Serving(2, "bf16")
    want.draw(1)
    want.step()
    m = Serving(2, "bf16")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        busy = torch.ones(1 << 26, device="cuda").cumsum(0)
        m.ids.copy_(m.ids + (0 * busy[:1]).int())
        m.draw(1)
        m.step()
        tokens = m.tokens * 1
    s.synchronize()
    assert torch.equal(tokens, want.tokens) and torch.equal(m.out, want.out)
