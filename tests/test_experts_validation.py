"""The entry points of a layer of experts refuse bad arguments before touching the GPU (so this runs without one), take empty
calls, and say how much room they need."""
import ctypes

import pytest

import cretif_amd as cri
from cretif_amd import experts

FAKE = 1 << 20  # never dereferenced: every case below fails validation first, or has nothing to do
# fake buffers are far apart
X, OUT, WS, DATA, DATA2, IDS, WEIGHTS, OFFSETS, ROWS, SLOTS, BIAS, RES = (FAKE << i for i in range(4, 16))
Q4_K = cri.FORMAT_IDS["q4_k"]
OK, INVALID, SHAPE, ALIGNMENT, UNSUPPORTED = 0, -1, -2, -3, -5


def weights(**kw):
    c = dict(data=DATA, format=Q4_K, n_experts=8, N=64, K=256)
    c.update(kw)
    return experts._ExpertWeights(**c)


def groups(**kw):
    c = dict(offsets=OFFSETS, rows=ROWS, slots=SLOTS, n_tokens=3, top_k=2, n_experts=8)
    c.update(kw)
    return experts._ExpertGroups(**c)


def router(**kw):
    c = dict(bias=0, scale=1.0, scoring=0, normalize=1)
    c.update(kw)
    return experts._ExpertRouter(**c)


def ref(x):
    return None if x is None else ctypes.addressof(x)


def status(fn, *args):
    return getattr(cri.lib(), fn)(*args)


SIZES = [
    (dict(format=6), UNSUPPORTED), (dict(format=-1), UNSUPPORTED), (dict(n_experts=-1), INVALID), (dict(N=-1), INVALID),
    (dict(K=-256), INVALID), (dict(n_experts=0), SHAPE), (dict(n_experts=1025), SHAPE), (dict(K=0), SHAPE), (dict(K=128), SHAPE),
    (dict(K=288), SHAPE), (dict(format=0, K=48), SHAPE), (dict(format=5, K=16), SHAPE), (dict(N=1 << 25), SHAPE), (dict(K=1 << 25), SHAPE),
    (dict(n_experts=1024, N=1 << 24, K=1 << 20), SHAPE), (dict(N=2**31 - 1, K=2**31 - 256), SHAPE),
]


@pytest.mark.parametrize("kw,want", SIZES)
def test_sizes(kw, want):
    w = weights(**kw)
    g = groups(n_experts=w.n_experts)
    assert status("cri_expert_packed_bytes", w.format, w.n_experts, w.N, w.K) == want
    assert pack(**{k: v for k, v in kw.items()}) == want
    for name, rest in (("matmul", (0,)), ("swiglu", ()), ("combine", ())):
        assert status("cri_expert_%s_workspace_bytes" % name, ref(w), ref(g), *rest) == want
    assert matmul(w=w, g=g) == want and swiglu(w=w, up=w, g=g) == want and combine(w=w, g=g) == want


def pack(format=Q4_K, src=X, n_experts=8, N=64, K=256, packed=DATA):
    return status("cri_expert_pack", format, src, n_experts, N, K, packed, None)


@pytest.mark.parametrize("kw,want", [
    (dict(src=0), INVALID), (dict(packed=0), INVALID), (dict(packed=DATA + 8), ALIGNMENT), (dict(src=DATA), INVALID),
    (dict(src=DATA + 8 * 64 * 144), INVALID), (dict(src=DATA - 8 * 64 * 144 + 1), INVALID), (dict(N=0, src=0, packed=0), OK),
])
def test_pack(kw, want):
    assert pack(**kw) == want


@pytest.mark.parametrize("fmt,units,unit", [("q8_0", 2, 8704), ("q4_0", 2, 4608), ("q5_0", 2, 5632), ("q4_k", 2, 4736),
                                            ("q6_k", 2, 6720), ("fp16", 2, 16384)])
def test_packed_bytes(fmt, units, unit):
    """32 columns and 256 values at a time, and no others."""
    f = cri.FORMAT_IDS[fmt]
    assert status("cri_expert_packed_bytes", f, 3, 33, 256) == 3 * units * unit
    assert status("cri_expert_packed_bytes", f, 1, 32, 256) == unit
    assert status("cri_expert_packed_bytes", f, 1, 0, 256) == 0


GROUPS = [
    (None, INVALID), (groups(n_tokens=-1), INVALID), (groups(top_k=-1), INVALID), (groups(n_experts=-1), INVALID),
    (groups(n_experts=0, top_k=1), SHAPE), (groups(n_experts=1025), SHAPE), (groups(top_k=0), SHAPE), (groups(top_k=9), SHAPE),
    (groups(top_k=65, n_experts=128), SHAPE), (groups(n_tokens=(1 << 22) + 1), SHAPE),
]
GROUP_POINTERS = [
    (groups(offsets=0), INVALID), (groups(rows=0), INVALID), (groups(slots=0), INVALID), (groups(offsets=OFFSETS + 2), ALIGNMENT),
    (groups(rows=ROWS + 1), ALIGNMENT), (groups(slots=SLOTS + 2), ALIGNMENT),
]


@pytest.mark.parametrize("g,want", GROUPS)
def test_group_sizes(g, want):
    assert status("cri_expert_group_workspace_bytes", ref(g)) == want
    assert route(g=g) == want and group(g=g) == want
    w = weights()
    for name, rest in (("matmul", (0,)), ("swiglu", ()), ("combine", ())):
        assert status("cri_expert_%s_workspace_bytes" % name, ref(w), ref(g), *rest) == want
    assert matmul(g=g) == want and swiglu(g=g) == want and combine(g=g) == want


@pytest.mark.parametrize("g,want", GROUP_POINTERS)
def test_group_pointers(g, want):
    assert route(g=g) == want and group(g=g) == want and matmul(g=g) == want and swiglu(g=g) == want and combine(g=g) == want


def test_group_room():
    """One workgroup needs none; more leave their counts, at most 256 of them."""
    for n_tokens, n_experts, want in ((0, 8, 0), (64, 8, 0), (65, 8, 5 * 8 * 4), (1 << 22, 1024, 256 * 1024 * 4)):
        g = groups(n_tokens=n_tokens, n_experts=n_experts)
        assert status("cri_expert_group_workspace_bytes", ref(g)) == want


def route(r="", logits=X, ldl=8, ids=IDS, w=WEIGHTS, g="", ws=WS, n=1 << 19):
    r, g = router() if r == "" else r, groups() if g == "" else g
    return status("cri_expert_route", ref(r), logits, ldl, ids, w, ref(g), ws, n, None)


@pytest.mark.parametrize("kw,want", [
    (dict(r=None), INVALID), (dict(r=router(scoring=2)), UNSUPPORTED), (dict(r=router(scoring=-1)), UNSUPPORTED),
    (dict(r=router(scale=float("nan"))), INVALID), (dict(r=router(scale=float("inf"))), INVALID), (dict(r=router(bias=BIAS + 1)), ALIGNMENT),
    (dict(logits=0), INVALID), (dict(logits=X + 2), ALIGNMENT), (dict(ldl=7), SHAPE), (dict(ldl=-8), SHAPE), (dict(ids=0), INVALID),
    (dict(w=0), INVALID), (dict(ids=IDS + 2), ALIGNMENT), (dict(w=WEIGHTS + 1), ALIGNMENT), (dict(w=IDS), INVALID),
    (dict(w=IDS + 20), INVALID), (dict(ids=X), INVALID), (dict(w=X + 4), INVALID), (dict(ids=OFFSETS + 32), INVALID),
    (dict(w=ROWS), INVALID), (dict(g=groups(slots=ROWS)), INVALID), (dict(g=groups(offsets=SLOTS + 16)), INVALID),
    (dict(r=router(bias=BIAS), ids=BIAS + 28), INVALID), (dict(g=groups(n_tokens=65), ws=0), INVALID),
    (dict(g=groups(n_tokens=65), ws=WS + 2), ALIGNMENT), (dict(g=groups(n_tokens=65), n=5 * 8 * 4 - 1), SHAPE),
    (dict(g=groups(n_tokens=65), n=-1), SHAPE), (dict(g=groups(n_tokens=65), ws=X), INVALID), (dict(g=groups(n_tokens=65), ws=IDS), INVALID),
])
def test_route_refuses(kw, want):
    assert route(**kw) == want


def group(ids=IDS, g="", ws=WS, n=1 << 19):
    g = groups() if g == "" else g
    return status("cri_expert_group", ids, ref(g), ws, n, None)


@pytest.mark.parametrize("kw,want", [
    (dict(ids=0), INVALID), (dict(ids=IDS + 2), ALIGNMENT), (dict(ids=ROWS), INVALID), (dict(ids=OFFSETS + 32), INVALID),
    (dict(g=groups(slots=ROWS + 20)), INVALID), (dict(g=groups(n_tokens=65), ws=0), INVALID),
    (dict(g=groups(n_tokens=65), ws=WS + 1), ALIGNMENT), (dict(g=groups(n_tokens=65), n=159), SHAPE),
    (dict(g=groups(n_tokens=65), ws=IDS), INVALID), (dict(g=groups(n_tokens=65), ws=SLOTS), INVALID),
])
def test_group_refuses(kw, want):
    assert group(**kw) == want


def matmul(w="", g="", x=X, ldx=256, grouped=0, out=OUT, ldo=64, ws=WS, n=1 << 24):
    w, g = weights() if w == "" else w, groups() if g == "" else g
    return status("cri_expert_matmul", ref(w), ref(g), x, ldx, grouped, out, ldo, ws, n, None)


def swiglu(w="", up="", g="", x=X, ldx=256, out=OUT, ldo=64, ws=WS, n=1 << 24):
    w, up, g = weights() if w == "" else w, weights(data=DATA2) if up == "" else up, groups() if g == "" else g
    return status("cri_expert_swiglu", ref(w), ref(up), ref(g), x, ldx, out, ldo, ws, n, None)


def combine(w="", g="", x=X, ldx=256, weights_=WEIGHTS, res=RES, ldr=64, out=OUT, ldo=64, ws=WS, n=1 << 24):
    w, g = weights() if w == "" else w, groups() if g == "" else g
    return status("cri_expert_combine", ref(w), ref(g), x, ldx, weights_, res, ldr, out, ldo, ws, n, None)


# many tokens of long rows: the products take a workspace
WIDE = dict(N=512, K=1024)


def many(**kw):
    return dict(dict(w=weights(**WIDE), g=groups(n_tokens=600), ldx=1024, ldo=512), **kw)


PRODUCTS = [
    (dict(w=None), INVALID), (dict(g=groups(n_experts=4)), SHAPE), (dict(w=weights(data=0)), INVALID),
    (dict(w=weights(data=DATA + 8)), ALIGNMENT), (dict(x=0), INVALID), (dict(out=0), INVALID), (dict(x=X + 2), ALIGNMENT),
    (dict(out=OUT + 1), ALIGNMENT), (dict(ldx=255), SHAPE), (dict(ldo=63), SHAPE), (dict(ldx=-1), SHAPE),
    (dict(out=X), INVALID), (dict(out=X + 4 * (2 * 256 + 255)), INVALID), (dict(out=DATA), INVALID), (dict(out=OFFSETS + 32), INVALID),
    (dict(out=ROWS), INVALID), (dict(out=SLOTS), INVALID), (many(ws=0), INVALID),
    (many(ws=WS + 8), ALIGNMENT), (many(n=15), SHAPE), (many(n=-1), SHAPE),
    (many(ws=X), INVALID), (many(ws=DATA), INVALID), (many(ws=ROWS), INVALID),
    (many(ws=OUT), INVALID), (dict(g=groups(n_tokens=1 << 22), ldx=1 << 30, n=1 << 60), SHAPE),
]


@pytest.mark.parametrize("kw,want", PRODUCTS)
def test_products_refuse(kw, want):
    up = {"up": weights(data=DATA2, **WIDE)} if "w" in kw and kw["w"] is not None and kw["w"].N == 512 else {}
    assert matmul(**kw) == want
    assert swiglu(**kw, **up) == want
    assert combine(**dict(kw, ldr=max(kw.get("ldo", 64), 64))) == want


@pytest.mark.parametrize("kw,want", [
    (dict(up=None), INVALID), (dict(up=weights(data=DATA2, format=0)), SHAPE), (dict(up=weights(data=DATA2, N=32)), SHAPE),
    (dict(up=weights(data=DATA2, K=512)), SHAPE), (dict(up=weights(data=DATA2, n_experts=4)), SHAPE), (dict(up=weights(data=0)), INVALID),
    (dict(up=weights(data=DATA2 + 4)), ALIGNMENT), (dict(out=DATA2), INVALID), (many(up=weights(data=DATA2, **WIDE), ws=DATA2), INVALID),
])
def test_swiglu_refuses(kw, want):
    assert swiglu(**kw) == want


@pytest.mark.parametrize("kw,want", [
    (dict(weights_=0), INVALID), (dict(weights_=WEIGHTS + 2), ALIGNMENT), (dict(out=WEIGHTS), INVALID), (dict(ldr=63), SHAPE),
    (dict(res=RES + 2), ALIGNMENT), (dict(res=OUT, ldr=65), INVALID), (dict(res=OUT + 4), INVALID), (dict(res=OUT + 4 * 128), INVALID),
    (many(ldr=512, ws=RES), INVALID), (many(ldr=512, ws=WEIGHTS), INVALID), (dict(out=X + 4 * (5 * 256 + 255)), INVALID),
])
def test_combine_refuses(kw, want):
    assert combine(**kw) == want


def test_grouped_rows_are_as_many_as_pairs():
    """Behind the third token's row, but not behind the sixth pair's."""
    assert matmul(out=X + 4 * 4 * 256, grouped=1) == INVALID


@pytest.mark.parametrize("kw", [dict(g=groups(n_tokens=0, rows=0, slots=0)), dict(w=weights(N=0))])
def test_empty(kw):
    """No token or no column: nothing to do, whatever the pointers are."""
    rest = dict(x=0, out=0, ws=0, n=0)
    up = dict(up=kw["w"]) if "w" in kw else {}
    assert matmul(**kw, **rest) == OK and swiglu(**kw, **up, **rest) == OK and combine(**kw, weights_=0, res=0, **rest) == OK
    w, g = kw.get("w", weights()), kw.get("g", groups())
    for name, tail in (("matmul", (0,)), ("swiglu", ()), ("combine", ())):
        assert status("cri_expert_%s_workspace_bytes" % name, ref(w), ref(g), *tail) == OK


def test_room_is_bounded():
    """Room for the rows' parts and products, which k in up to 8 parts of up to 256 MB has several of."""
    for m in (1, 2, 7, 33, 600, 8192):
        w, g = weights(N=512, K=2048), groups(n_tokens=m)
        for name, tail in (("matmul", (0,)), ("matmul", (1,)), ("swiglu", ()), ("combine", ())):
            n = status("cri_expert_%s_workspace_bytes" % name, ref(w), ref(g), *tail)
            row = 4 * 2048 + 2048 // 256 * 32 + 4  # two halves a value, what 256 values of it have, its exponent
            assert 0 <= n <= 2 * m * (row + 4 * 512) + min(2 * 8 * 2 * m * 4 * 512, 1 << 28) + (1 << 16), (name, m, n)


def test_error_text_names_the_call():
    assert combine(ldo=63) == SHAPE
    text = cri.lib().cri_last_error_string().decode()
    assert "cri_expert_combine" in text and "out" in text


@pytest.mark.parametrize("call", [
    lambda: cri.ExpertRouter(scoring="softmax2"),
])
def test_python_refuses(call):
    with pytest.raises(KeyError):
        call()


def test_too_many_tiles():
    """More tiles than a launch takes are refused before anything is launched."""
    far = [i << 44 for i in range(1, 8)]
    w = weights(data=far[0], N=1 << 16)
    g = groups(offsets=far[1], rows=far[2], slots=far[3], n_tokens=1 << 20, top_k=8)
    got = status("cri_expert_matmul", ref(w), ref(g), far[4], 256, 0, far[5], 1 << 16, far[6], 1 << 42, None)
    assert got == UNSUPPORTED
    assert "tiles" in cri.lib().cri_last_error_string().decode()
