"""The batched serving entry points refuse bad arguments before touching the GPU (so this runs without one), and
the definitions the GPU tests use agree with what they claim."""
import ctypes
import threading
import weakref

import numpy as np
import pytest

import cretif_amd as cri
import serving_ref as ref
from cretif_amd import serving

FAKE = 1 << 20  # never dereferenced: every case below fails validation first


def kv(**kw):
    c = dict(k=FAKE, v=FAKE, page_stride=16 * 2 * 64, type=5, n_pages=4, page_size=16, n_kv_heads=2, head_dim=64)
    c.update(kw)
    return serving._PagedKV(**c)


def batch(**kw):
    c = dict(offsets=FAKE, lens=FAKE, pages=FAKE, n_seqs=2, n_rows=3, max_pages=5)
    c.update(kw)
    return serving._PagedBatch(**c)


def rot(**kw):
    c = dict(q_norm=0, k_norm=0, eps=1e-6, theta=1e4, rot_dim=64, pairs=0)
    c.update(kw)
    return serving._Rotation(**c)


def ref_of(x):
    return None if x is None else ctypes.addressof(x)


def status(fn, *args):
    return getattr(cri.lib(), fn)(*args)


# rows of fake buffers are far apart
Q, K, V, O, O2, WS = (FAKE << i for i in range(2, 8))


def norm_rope(r=None, q=Q, ldq=256, k=K, ldk=128, qo=O, ldqo=256, ko=O2, ldko=128, pos=FAKE, M=3, H=4, Hkv=2, D=64):
    r = rot() if r is None else r
    return status("cri_qk_norm_rope", ref_of(r), q, ldq, k, ldk, qo, ldqo, ko, ldko, pos, M, H, Hkv, D, None)


@pytest.mark.parametrize("kw,want", [
    (dict(M=-1), -1), (dict(H=-1), -1), (dict(D=-8), -1), (dict(D=0), -5), (dict(D=60), -5), (dict(D=264), -5),
    (dict(r=rot(pairs=2)), -5), (dict(r=rot(rot_dim=12)), -2), (dict(r=rot(rot_dim=72)), -2), (dict(r=rot(rot_dim=-8)), -2),
    (dict(r=rot(theta=0.0)), -1), (dict(r=rot(theta=float("nan"))), -1), (dict(r=rot(theta=float("inf"))), -1),
    (dict(r=rot(q_norm=FAKE, eps=-1.0)), -1), (dict(r=rot(q_norm=FAKE + 2)), -3), (dict(pos=0), -1), (dict(pos=FAKE + 1), -3),
    (dict(q=0), -1), (dict(qo=0), -1), (dict(k=0), -1), (dict(ko=0), -1), (dict(q=Q + 2), -3), (dict(ldq=255), -2),
    (dict(ldk=127), -2), (dict(ldqo=8), -2), (dict(qo=Q + 16), -1), (dict(ko=Q), -1), (dict(qo=Q, ldqo=512), -1),
    (dict(ko=O + 4 * 128, ldko=256), -1), (dict(M=1 << 30, ldq=1 << 20), -2), (dict(M=(1 << 23) + 1), -2),
])
def test_norm_rope_refuses(kw, want):
    assert norm_rope(**kw) == want


def test_norm_rope_null_rotation():
    assert status("cri_qk_norm_rope", None, Q, 256, K, 128, O, 256, O2, 128, FAKE, 3, 4, 2, 64, None) == -1


def test_norm_rope_empty():
    assert norm_rope(M=0, q=0, k=0, qo=0, ko=0, pos=0) == 0
    assert norm_rope(H=0, Hkv=0, q=0, k=0, qo=0, ko=0, pos=0) == 0


def append(p=None, b=None, r=None, q=Q, ldq=256, qo=O, ldqo=256, H=4, k=K, ldk=128, v=V, ldv=128):
    p, b, r = kv() if p is None else p, batch() if b is None else b, rot() if r is None else r
    return status("cri_paged_append", ref_of(p), ref_of(b), ref_of(r), q, ldq, qo, ldqo, H, k, ldk, v, ldv, None)


POOL = [
    (dict(p=kv(type=3)), -5), (dict(p=kv(type=0)), -5), (dict(p=kv(head_dim=60)), -5), (dict(p=kv(head_dim=512)), -5),
    (dict(p=kv(n_pages=-1)), -1), (dict(p=kv(n_pages=0)), -2), (dict(p=kv(page_size=0)), -2), (dict(p=kv(n_kv_heads=0)), -2),
    (dict(p=kv(page_stride=16 * 2 * 64 - 8)), -2), (dict(p=kv(page_stride=16 * 2 * 64 + 4)), -2),
    (dict(p=kv(page_stride=-1)), -2), (dict(p=kv(page_stride=1 << 50)), -2), (dict(p=kv(k=0)), -1), (dict(p=kv(v=0)), -1),
    (dict(p=kv(k=FAKE + 8)), -3), (dict(p=kv(v=FAKE + 2)), -3), (dict(b=batch(n_seqs=-1)), -1), (dict(b=batch(n_rows=-1)), -1),
    (dict(b=batch(max_pages=-1)), -1), (dict(b=batch(max_pages=1 << 27)), -2), (dict(b=batch(offsets=0)), -1),
    (dict(b=batch(lens=0)), -1), (dict(b=batch(pages=0)), -1), (dict(b=batch(pages=FAKE + 2)), -3),
]


@pytest.mark.parametrize("kw,want", POOL + [
    (dict(r=rot(rot_dim=4)), -2), (dict(H=-1), -1), (dict(k=0), -1), (dict(v=0), -1), (dict(v=V + 1), -3), (dict(ldv=127), -2),
    (dict(qo=0), -1), (dict(ldq=255), -2), (dict(qo=K), -1), (dict(qo=V), -1), (dict(qo=Q, ldqo=257), -1),
    (dict(k=FAKE + 64), -1), (dict(v=FAKE + 64), -1), (dict(qo=FAKE + 64), -1), (dict(q=FAKE - 64), -1),
    (dict(b=batch(n_rows=(1 << 23) + 1)), -2),
])
def test_append_refuses(kw, want):
    assert append(**kw) == want


def test_append_empty():
    assert append(b=batch(n_seqs=0, offsets=0, lens=0, pages=0), k=0, v=0) == 0
    assert append(b=batch(n_rows=0), k=0, v=0, q=0, qo=0) == 0


def attend(p=None, b=None, pp=FAKE, P=20, q=Q, ldq=256, o=O, ldo=256, H=4, scale=0.125, ws=WS, wsb=1 << 40):
    p, b = kv() if p is None else p, batch() if b is None else b
    return status("cri_paged_attention", ref_of(p), ref_of(b), pp, P, q, ldq, o, ldo, H, scale, ws, wsb, None)


@pytest.mark.parametrize("kw,want", POOL + [
    (dict(H=3), -2), (dict(H=-2), -1), (dict(P=-1), -1), (dict(P=(1 << 30) + 1), -2), (dict(pp=0), -1), (dict(pp=FAKE + 2), -3),
    (dict(q=0), -1), (dict(o=0), -1), (dict(ldq=255), -2), (dict(ldo=100), -2), (dict(o=Q), -1), (dict(o=Q + 1024), -1),
    (dict(ws=0), -1), (dict(ws=WS + 8), -3), (dict(wsb=100), -2), (dict(b=batch(max_pages=0)), -2),
    (dict(b=batch(n_rows=1 << 23)), -2), (dict(o=FAKE + 64), -1), (dict(ws=FAKE + 64), -1), (dict(ws=Q + 16), -1),
    (dict(ws=O + 16), -1), (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1), (dict(scale=3e38), -1),
    (dict(b=batch(n_seqs=1 << 26)), -5),
])
def test_attention_refuses(kw, want):
    assert attend(**kw) == want


def test_attention_empty():
    assert attend(b=batch(n_seqs=0), q=0, o=0, ws=0) == 0
    assert attend(b=batch(n_rows=0), q=0, o=0, ws=0) == 0
    assert attend(H=0, q=0, o=0, ws=0) == 0
    f = cri.lib().cri_paged_attention_workspace_bytes
    assert f(ref_of(kv()), ref_of(batch(n_seqs=0)), 20, 4) == 0
    assert f(ref_of(kv()), ref_of(batch()), 20, 4) > 0
    assert f(ref_of(kv()), ref_of(batch()), 20, 3) == -2
    assert f(None, ref_of(batch()), 20, 4) == -1


@pytest.mark.parametrize("kind", [5, 6, 7])
@pytest.mark.parametrize("D,ps", [(128, 16), (64, 20), (256, 16), (8, 1)])
def test_attention_workspace_is_bounded(kind, D, ps):
    """1 GiB, or a record of the prefix and one of the sequences' positions per row and head."""
    f = cri.lib().cri_paged_attention_workspace_bytes
    cache = kv(type=kind, head_dim=D, page_size=ps, n_kv_heads=4, page_stride=ps * 4 * D)
    most = 0
    for n_rows in (1, 7, 480, 1100, 2048, 8192, 1 << 17, 1 << 19):
        for n_seqs in (1, 64, 1000):
            for held in (500, 8192, 32768, 1 << 20):
                for P in (0, 100, 8000, 32768):
                    b = batch(n_seqs=n_seqs, n_rows=n_rows, max_pages=-(-held // ps))
                    n = f(ref_of(cache), ref_of(b), P, 32)
                    record = n_rows * 32 * (D + 4) * 4
                    assert n == -5 or 0 <= n <= max(1 << 30, 2 * record if P else 0), (n_rows, n_seqs, held, P, n)
                    assert n == -5 or n % record == 0
                    most = max(most, n)
    assert most > 1 << 29


def verify(t=Q, ldt=100, d=K, ldd=100, ids=FAKE, u=V, dr=V, off=FAKE, B=2, n=5, vocab=100, out=O, acc=O2, ws=WS, wsb=1 << 40):
    return status("cri_verify_drafts", t, ldt, d, ldd, ids, u, dr, off, B, n, vocab, out, acc, ws, wsb, None)


@pytest.mark.parametrize("kw,want", [
    (dict(B=-1), -1), (dict(n=-1), -1), (dict(vocab=-1), -1), (dict(vocab=0), -2), (dict(t=0), -1), (dict(ids=0), -1),
    (dict(u=0), -1), (dict(dr=0), -1), (dict(dr=V + 2), -3), (dict(off=0), -1), (dict(out=0), -1), (dict(acc=0), -1), (dict(t=Q + 2), -3), (dict(d=K + 1), -3),
    (dict(ldt=99), -2), (dict(ldd=99), -2), (dict(ldt=1 << 50), -2), (dict(out=FAKE + 4), -1), (dict(ws=0), -1),
    (dict(ws=WS + 4), -3), (dict(wsb=16), -2), (dict(B=(1 << 20) + 1), -2), (dict(vocab=1 << 29, ldt=1 << 29, ldd=1 << 29), -2),
])
def test_verify_refuses(kw, want):
    assert verify(**kw) == want


def test_verify_empty():
    assert verify(B=0, t=0, ids=0, u=0, off=0, out=0, acc=0, ws=0) == 0
    f = cri.lib().cri_verify_drafts_workspace_bytes
    assert f(0, 100) == 0 and f(2, 100) > 0 and f(-1, 100) == -1


def test_messages_name_the_function():
    attend(H=3)
    assert cri.lib().cri_last_error_string().decode().startswith("cri_paged_attention: n_heads=3")


def test_python_refuses_host_tensors():
    torch = pytest.importorskip("torch")
    x = torch.zeros(4, 16, 2, 64)
    with pytest.raises(ValueError, match="device"):
        cri.PagedKV(x, x)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        cri.PagedKV(x.double(), x.double())
    with pytest.raises(ValueError, match="n_pages"):
        cri.PagedKV(x, x[0])
    with pytest.raises(ValueError, match="int32"):
        cri.PagedBatch(torch.zeros(3), torch.zeros(2), torch.zeros(2, 5))
    with pytest.raises(ValueError, match="q_norm"):
        cri.Rotation(1e4, 64, q_norm=torch.zeros(64, dtype=torch.float64))
    with pytest.raises(KeyError):
        cri.Rotation(1e4, 64, "sideways")
    with pytest.raises(ValueError, match="device"):
        cri.qk_norm_rope(cri.Rotation(1e4, 64), torch.zeros(2, 128), None, torch.zeros(2, 128), None,
                         torch.zeros(2, dtype=torch.int32), 2, 0, 64)
    with pytest.raises(ValueError, match="float32"):
        cri.verify_drafts(torch.zeros(2, 8).half(), None, None, None, None, None, None, None)


def test_definition_keeps_the_targets_distribution():
    """Rejection sampling as defined draws from the target whatever the draft: over a fine grid of numbers, every
    token's share of the first output is the target's (off by the grid's steps: one per accepted or drawn interval)."""
    p, q = np.array([0.5, 0.2, 0.0, 0.3]), np.array([0.1, 0.6, 0.2, 0.1])
    n = 40
    share = np.zeros(4)
    for x in range(4):  # the draft's token, with its probability
        for i in range(n):
            for j in range(n):
                u, d = [(i + 0.5) / n, 0.5], [(j + 0.5) / n, 0.5]
                out, _ = ref.verify(np.stack([p, p]), np.stack([q, q]), [x, 0], u, d, [0, 2], [0, 0], [0])
                share[out[0]] += q[x] / n / n
    assert np.abs(share - p).max() <= 1.0 / n


def paged_batch(make):
    """A PagedBatch whose descriptors `make` makes (its own need device tensors)."""
    b = serving.PagedBatch.__new__(serving.PagedBatch)
    b._make, b._by_rows, b._dev = make, {}, None
    return b


def paged_kv():
    p = serving.PagedKV.__new__(serving.PagedKV)
    p._c, p._dev = kv(), None
    p.page_size, p.n_kv_heads, p.head_dim = p._c.page_size, p._c.n_kv_heads, p._c.head_dim
    p._ref = ref_of(p._c)
    return p


def test_threads_that_share_a_batch_keep_their_descriptors(monkeypatch):
    """Two threads meet a new row count together: each one's descriptor lives as long as its call."""
    pytest.importorskip("torch")
    both, made, alive = threading.Barrier(2, timeout=30), [], []

    def make(rows):
        c = batch(n_rows=rows)
        made.append(weakref.ref(c))
        both.wait()  # neither has been stored
        return c

    class Lib:
        @staticmethod
        def cri_paged_attention_workspace_bytes(*args):
            both.wait()  # both have been stored, both calls run
            alive.append([r() is not None for r in made])
            both.wait()
            return 0

    monkeypatch.setattr(serving, "_torch", lambda: Lib)
    b, p = paged_batch(make), paged_kv()
    threads = [threading.Thread(target=cri.paged_attention_workspace_bytes, args=(p, b, 3, 4)) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert alive == [[True, True]] * 2


def test_a_batch_keeps_a_bounded_number_of_descriptors():
    pytest.importorskip("torch")
    b, p = paged_batch(lambda rows: batch(n_rows=rows)), paged_kv()
    want = [cri.paged_attention_workspace_bytes(p, b, n, 4) for n in range(1, 2000)]
    assert len(b._by_rows) <= 1000 and sorted(set(want)) == sorted(want) and want[0] > 0
    assert [cri.paged_attention_workspace_bytes(p, b, n, 4) for n in range(1, 2000)] == want


class Recorder:
    """Stands for the library: what reached it."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *args: self.calls.append((name, args)) or 0


class Array:
    """What the wrappers ask of a device tensor, with any shape and strides."""

    def __init__(self, torch, *shape, strides=None, dtype=None, at=FAKE):
        self.shape, self.dtype, self.device = torch.Size(shape), dtype or torch.int32, "cuda:0"
        self._strides, self._at, self.nbytes = strides, at, 1 << 40

    def stride(self, i=None):
        return self._strides if i is None else self._strides[i]

    def dim(self):
        return len(self.shape)

    def is_contiguous(self):
        return True

    def get_device(self):
        return 0

    def data_ptr(self):
        return self._at

    def __getitem__(self, i):
        return self


@pytest.fixture
def recorded(monkeypatch):
    torch, lib = pytest.importorskip("torch"), Recorder()
    monkeypatch.setattr(serving, "torch", torch)
    monkeypatch.setattr(serving, "_torch", lambda: lib)
    monkeypatch.setattr(serving, "_device", lambda: 0)
    monkeypatch.setattr(serving, "_on", lambda stream, dev: 0)
    return torch, lib


FAR = [2 ** 31, 2 ** 32 + 256, 2 ** 32 + 2 ** 31 + 512, 2 ** 62]


@pytest.mark.parametrize("ld", FAR)
@pytest.mark.parametrize("as_tuple", [False, True])
def test_row_strides_past_32_bits_are_refused(recorded, ld, as_tuple):
    """C takes rows' strides as int, which ctypes would fill with the lower 32 bits."""
    torch, lib = recorded

    def rows(width, far, n=3):
        if as_tuple:
            return FAKE, ld if far else width
        return Array(torch, n, width, strides=(ld if far else width, 1), dtype=torch.float32)

    b, p, r = paged_batch(lambda n: batch(n_rows=n)), paged_kv(), cri.Rotation(1e4, 64)
    pos, ws = Array(torch, 3), Array(torch, 1 << 40)
    for i in range(4):
        w = [rows(256, i == 0), rows(128, i == 1), rows(256, i == 2), rows(128, i == 3)]
        with pytest.raises(ValueError, match="32 bits"):
            cri.qk_norm_rope(r, *w, pos, 4, 2, 64)
        w = [rows(128, i == 0), rows(128, i == 1), rows(256, i == 2), rows(256, i == 3)]
        with pytest.raises(ValueError, match="32 bits"):
            cri.paged_append(p, b, r, *w, n_heads=4, n_rows=3)
        if i < 2:
            with pytest.raises(ValueError, match="32 bits"):
                cri.paged_attention(p, b, rows(256, i == 0), rows(256, i == 1), 4, 0.125, workspace=ws, n_rows=3)
    assert lib.calls == []
    if as_tuple:
        return
    # the stride of a single row says nothing, the verification's strides have 64 bits
    cri.qk_norm_rope(r, rows(256, True, 1), None, rows(256, True, 1), None, Array(torch, 1), 4, 0, 64)
    cri.paged_attention(p, b, rows(256, True, 1), rows(256, True, 1), 4, 0.125, workspace=ws)
    assert lib.calls[0][1][2] == 256 and lib.calls[0][1][6] == 256 and lib.calls[1][1][5] == 256 and lib.calls[1][1][7] == 256
    f = dict(dtype=torch.float32)
    cri.verify_drafts(rows(100, True), None, Array(torch, 3), Array(torch, 3, **f), Array(torch, 3, **f), Array(torch, 2),
                      Array(torch, 3), Array(torch, 1), ws)
    assert lib.calls[2][1][1] == ld


@pytest.mark.parametrize("far", [2 ** 31, 2 ** 32 + 64, -2 ** 32 + 64])
def test_sizes_past_32_bits_are_refused(recorded, far):
    torch, lib = recorded
    b, p, r = paged_batch(lambda n: batch(n_rows=n)), paged_kv(), cri.Rotation(1e4, 64)
    x, ws, wide = (FAKE, 256), Array(torch, 1 << 40), Array(torch, abs(far), 16, 2, 64, strides=(2048, 128, 64, 1), dtype=torch.float16)
    f = dict(dtype=torch.float32)
    calls = [
        lambda: cri.Rotation(1e4, far),
        lambda: cri.PagedKV(wide, wide),
        lambda: cri.PagedBatch(Array(torch, 3), Array(torch, 2), Array(torch, 2, abs(far))),
        lambda: cri.qk_norm_rope(r, x, None, x, None, Array(torch, 3), far, 0, 64),
        lambda: cri.qk_norm_rope(r, x, None, x, None, Array(torch, abs(far)), 4, 0, 64),
        lambda: cri.paged_append(p, b, r, x, x, n_rows=far),
        lambda: cri.paged_append(p, b, r, x, x, x, x, n_heads=far, n_rows=3),
        lambda: cri.paged_attention(p, b, x, x, far, 0.125, workspace=ws, n_rows=3),
        lambda: cri.paged_attention(p, b, x, x, 4, 0.125, workspace=ws, n_rows=far),
        lambda: cri.paged_attention(p, b, x, x, 4, 0.125, Array(torch, abs(far)), far, workspace=ws, n_rows=3),
        lambda: cri.paged_attention_workspace_bytes(p, b, far, 4),
        lambda: cri.paged_attention_workspace_bytes(p, b, 3, 4, far),
        lambda: cri.verify_drafts_workspace_bytes(2, far),
        lambda: cri.verify_drafts(Array(torch, 3, abs(far), strides=(abs(far), 1), **f), None, Array(torch, 3), Array(torch, 3, **f),
                                  Array(torch, 3, **f), Array(torch, 2), Array(torch, 3), Array(torch, 1), ws),
    ]
    for call in calls:
        with pytest.raises(ValueError, match="32 bits"):
            call()
    assert lib.calls == []


def refused(st, word):
    assert st == -1 and word in cri.lib().cri_last_error_string().decode(), (st, cri.lib().cri_last_error_string())


def test_norm_rope_outputs_apart_from_what_it_reads():
    far = rot(q_norm=WS, k_norm=WS + 256)
    refused(norm_rope(pos=O + 2 * 1024 + 1020), "positions")  # the last of q_out's third row
    refused(norm_rope(pos=O2 - 8), "positions")
    refused(norm_rope(r=far, qo=WS + 252), "norm weights")
    refused(norm_rope(r=far, ko=WS + 508), "norm weights")


@pytest.mark.parametrize("kind,e", [(6, 4), (5, 2), (7, 2)])
def test_append_refuses_pages_of_keys_that_are_pages_of_values(kind, e):
    page = 16 * 2 * 64
    arrays = batch(offsets=O + 4, lens=Q << 8, pages=Q << 8)  # (q_out meets offsets: refused behind the pages' check)

    def pool(v, stride):
        return append(p=kv(type=kind, v=FAKE + v * e, page_stride=stride), b=arrays)

    for v, stride in [(0, page), (8, page), (page - 8, page), (page, page), (3 * page, page), (-page, page), (0, 2 * page),
                      (2 * page, 2 * page), (page - 8, 2 * page), (page + 8, 2 * page), (-page + 8, 2 * page), (6 * page, 2 * page),
                      (5 * page + 8, 2 * page)]:
        refused(pool(v, stride), "pages of k and v")
    for v, stride in [(4 * page, page), (-4 * page, page), (page, 2 * page), (-page, 2 * page), (3 * page, 2 * page),
                      (5 * page, 2 * page), (7 * page, 2 * page), (7 * page + 8, 2 * page), (page + 8, 3 * page), (8 * page, 2 * page)]:
        refused(pool(v, stride), "q_out overlaps the batch")


def test_append_query_rows_apart_from_the_batch():
    p = kv(v=V << 8)
    for b in (batch(offsets=O + 4 * 767, lens=WS, pages=WS), batch(offsets=WS, lens=O - 4, pages=WS), batch(offsets=WS, lens=WS, pages=O - 36)):
        refused(append(p=p, b=b), "q_out overlaps the batch")
    refused(append(p=p, b=batch(offsets=WS, lens=WS, pages=WS), r=rot(q_norm=O - 252)), "norm weights")


def test_attention_outputs_apart_from_the_batch():
    p = kv(k=Q << 8, v=Q << 8)  # (reading one page as both is fine)
    for at in (O, WS):
        for b in (batch(offsets=at - 8, lens=V, pages=V), batch(offsets=V, lens=at + 4, pages=V), batch(offsets=V, lens=V, pages=at - 36)):
            refused(attend(p=p, b=b), "batch")
        refused(attend(p=p, b=batch(offsets=V, lens=V, pages=V), pp=at - 4), "prefix_pages")


def test_verify_outputs_apart_from_inputs_and_each_other():
    far = Q << 8
    ok = dict(t=far, d=far + (1 << 20), ids=far + (2 << 20), u=far + (3 << 20), dr=far + (3 << 20), off=far + (4 << 20))
    for at in (dict(out=O), dict(acc=O), dict(ws=O, wsb=100)):
        for name, back in (("t", 499), ("d", 499), ("ids", 4), ("u", 4), ("dr", 4), ("off", 2)):
            kw = dict(ok)
            kw[name] = O - back * 4  # its last element is the output's first
            refused(verify(**{**dict(out=O2, acc=O2 + 4096, ws=WS), **at, **kw}), "an input")
    refused(verify(**ok, out=O, acc=O + 16), "out_ids, n_accepted")
    refused(verify(**ok, out=O + 24, ws=O, wsb=100), "out_ids, n_accepted")
    refused(verify(**ok, acc=O2 + 24, ws=O2, wsb=100), "out_ids, n_accepted")
