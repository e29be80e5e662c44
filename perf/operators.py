"""Operators of batched serving: inputs, plain forms, the library's calls, work and float64 results.

  qk_norm_rope     RMS norm of every query and key head and the position rotation, one pass
  paged_append     keys (normed, rotated) and values of new tokens into a paged cache, queries rotated
  paged_attention  attention of a ragged batch over the pages, a prefix that all sequences share read once
  verify_drafts    drafted tokens accepted or replaced from the target's and the draft's probabilities

`own` False computes them with elementary torch operations, True calls cretif_amd.
"""
import math
import random

import torch

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def listed():
    return [
        # one new token of one sequence, q and k of a model that norms its heads
        dict(name="norm_rope_token", op="qk_norm_rope", M=1, H=32, Hkv=8, D=128, rot=128, halves=True, norm=True,
             theta=1e6, start=4000),
        # a long prompt's q and k, read out of the fused q/k/v product
        dict(name="norm_rope_prompt", op="qk_norm_rope", M=8192, H=32, Hkv=8, D=128, rot=128, halves=True, norm=True,
             theta=1e6, start=0),
        # one decode step of a batch: adjacent pairs, no norm, as the GGUF llama layout has it
        dict(name="append_step_fp16", op="paged_append", B=64, n=1, ragged=False, ctx=900, H=24, Hkv=8, D=64, rot=64,
             halves=False, norm=False, theta=5e5, ps=16, type="fp16", pad=0),
        # a ragged batch of drafted tokens over an fp32 cache, part of each head rotated, padded rows behind it
        dict(name="append_drafts_fp32", op="paged_append", B=17, n=6, ragged=True, ctx=700, H=16, Hkv=4, D=96, rot=48,
             halves=True, norm=False, theta=1e4, ps=32, type="fp32", pad=3),
        # prompts of several sequences at once, normed heads
        dict(name="append_prompts_bf16", op="paged_append", B=7, n=1500, ragged=True, ctx=0, H=32, Hkv=8, D=128,
             rot=128, halves=True, norm=True, theta=1e6, ps=64, type="bf16", pad=0),
        # a few short conversations on the fp32 cache of the decoder
        dict(name="attention_few_fp32", op="paged_attention", B=4, n=1, ragged=False, P=500, own_len=100, H=32, Hkv=8,
             D=64, ps=16, type="fp32", pad=0),
        # a serving step: many conversations on one long system prompt
        dict(name="attention_chat_fp16", op="paged_attention", B=64, n=1, ragged=False, P=8192, own_len=1500, H=32,
             Hkv=8, D=128, ps=16, type="fp16", pad=0),
        # drafted tokens being checked: ragged rows, a prefix that ends inside a page, eight heads to a key
        dict(name="attention_drafts_bf16", op="paged_attention", B=48, n=6, ragged=True, P=4001, own_len=600, H=64,
             Hkv=8, D=128, ps=64, type="bf16", pad=5),
        # a large batch of drafts on a very long document
        dict(name="attention_document_fp16", op="paged_attention", B=96, n=5, ragged=False, P=32768, own_len=300,
             H=32, Hkv=8, D=128, ps=16, type="fp16", pad=0),
        # four drafted tokens of one sequence
        dict(name="verify_one", op="verify_drafts", B=1, n=5, ragged=False, V=128256, draft=True),
        # a batch's drafts, ragged, from a draft model's distributions
        dict(name="verify_batch", op="verify_drafts", B=64, n=6, ragged=True, V=128256, draft=True),
        # drafts looked up in the text, without a distribution of their own
        dict(name="verify_lookup", op="verify_drafts", B=200, n=8, ragged=True, V=32000, draft=False),
    ]


def _span(rng, lo, hi):
    """lo .. hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["qk_norm_rope", "paged_append", "paged_attention", "paged_attention", "verify_drafts"])
    if op == "verify_drafts":
        V = _span(rng, 1000, 160000)
        n = rng.randint(1, 9)
        return dict(op=op, B=_span(rng, 1, min(256, 40000000 // (V * n))), n=n, ragged=rng.random() < 0.6, V=V,
                    draft=rng.random() < 0.7)
    Hkv = rng.choice([1, 2, 4, 5, 8])
    H = Hkv * rng.choice([1, 2, 3, 4, 7, 8])
    if op != "paged_attention":
        D = rng.choice([64, 128, 128, 80, 96, 256])
        rot = rng.choice([D, D, D // 2])
        common = dict(H=H, Hkv=Hkv, D=D, rot=rot // 8 * 8, halves=rng.random() < 0.5, norm=rng.random() < 0.5,
                      theta=rng.choice([1e4, 5e5, 1e6]))
        most = 40000000 // ((H + 2 * Hkv) * D)  # elements of the largest listed cases
        if op == "qk_norm_rope":
            return dict(op=op, M=_span(rng, 1, min(8192, most)), start=_span(rng, 1, 1000000), **common)
        B = _span(rng, 1, 128)
        return dict(op=op, B=B, n=_span(rng, 1, max(1, min(2000, most // B))), ragged=rng.random() < 0.6,
                    ctx=_span(rng, 1, max(1, min(2000, 50000000 // (B * Hkv * D)))), ps=rng.choice([16, 16, 32, 64, 24, 256]),
                    type=rng.choice(["fp32", "fp16", "bf16"]), pad=rng.choice([0, 0, 3]), **common)
    D = rng.choice([64, 128, 128, 80, 256])
    B, n = _span(rng, 1, 128), rng.choice([1, 1, 2, 4, 7])
    P = _span(rng, 1, max(2, min(32768, 60000000000 // (B * n * H * D * 8))))
    own_len = n + _span(rng, 1, max(2, min(2000, 100000000 // (B * Hkv * D))))
    return dict(op=op, B=B, n=n, ragged=rng.random() < 0.5, P=P, own_len=own_len, H=H, Hkv=Hkv, D=D,
                ps=rng.choice([16, 16, 32, 64, 20, 256]), type=rng.choice(["fp32", "fp16", "bf16"]),
                pad=rng.choice([0, 0, 3]))


def _counts(c, rng):
    """New tokens of each sequence and the positions each holds, new ones included: the same ones for every seed,
    in another order."""
    fixed = random.Random(repr(sorted((k, v) for k, v in c.items() if k != "name")))
    seqs = []
    for _ in range(c["B"]):
        n = fixed.randint(1, c["n"]) if c["ragged"] else c["n"]
        if c["op"] == "paged_append":
            seqs.append((n, n + fixed.randint(0, c["ctx"])))
        elif c["op"] == "paged_attention":
            seqs.append((n, c["P"] + n + fixed.randint(0, max(0, c["own_len"] - n))))
        else:
            seqs.append((n, n))
    rng.shuffle(seqs)
    return [n for n, _ in seqs], [held for _, held in seqs]


def _tables(c, held, rng, shared):
    """Page tables over a shuffled pool; the first `shared` pages of every sequence are the same ones."""
    need = [-(-h // c["ps"]) for h in held]
    total = shared + sum(k - shared for k in need) + 1
    pool = list(range(total))
    rng.shuffle(pool)
    first, at, rows, width = pool[:shared], shared, [], max(need)
    for k in need:
        rows.append(first + pool[at:at + k - shared] + [0] * (width - k))
        at += k - shared
    return total, rows, (pool[at] if shared * c["ps"] < c.get("P", 0) else None), first


def prepare(case, seed):
    c = case
    rng = random.Random(seed)
    g = torch.Generator("cuda").manual_seed(seed)
    dev = dict(device="cuda")
    randn = lambda *s: torch.randn(*s, generator=g, **dev)  # noqa: E731
    ints = lambda v: torch.tensor(v, dtype=torch.int32, **dev)  # noqa: E731
    s = dict(case=c)
    if c["op"] == "verify_drafts":
        n, _ = _counts(c, rng)
        T = sum(n)
        logits = 3.0 * randn(T, c["V"])
        s["target"] = torch.softmax(logits, -1)
        if c["draft"]:  # a smaller model's distribution, near the target's
            s["draft"] = torch.softmax(logits + 1.0 * randn(T, c["V"]), -1)
            s["ids"] = torch.multinomial(s["draft"], 1, generator=g).flatten().int()
        else:
            s["draft"] = None
            s["ids"] = torch.where(torch.rand(T, generator=g, **dev) < 0.6, s["target"].argmax(-1),
                                   torch.randint(0, c["V"], (T,), generator=g, **dev)).int()
        s["u"] = torch.rand(T, generator=g, **dev)
        s["offsets"] = ints([sum(n[:i]) for i in range(len(n) + 1)])
        s["most"] = max(n)
        s["out_ids"] = torch.zeros(T, dtype=torch.int32, **dev)
        s["accepted"] = torch.zeros(c["B"], dtype=torch.int32, **dev)
        return s
    H, Hkv, D = c["H"], c["Hkv"], c["D"]
    if c["op"] == "qk_norm_rope":
        M = c["M"]
        s["positions"] = torch.arange(c["start"], c["start"] + M, dtype=torch.int32, **dev)
        s["k_out"] = torch.zeros(M, Hkv * D, **dev)
    else:
        n, held = _counts(c, rng)
        M = sum(n) + c["pad"]
        P = c.get("P", 0)
        total, rows, last, first = _tables(c, held, rng, P // c["ps"])
        s.update(real=sum(n), most=max(n), longest=max(held), offsets=ints([sum(n[:i]) for i in range(len(n) + 1)]),
                 lens=ints(held), pages=ints(rows))
        s["k_pages"] = randn(total, c["ps"], Hkv, D).to(TYPES[c["type"]])
        s["v_pages"] = randn(total, c["ps"], Hkv, D).to(TYPES[c["type"]])
    if c["op"] == "paged_attention":
        s["prefix_pages"] = ints(first + ([last] if last is not None else []))
        s["q"] = 2.0 * randn(M, H * D)
        s["out"] = torch.zeros(M, H * D, **dev)
        return s
    # q, k and v as the fused projection leaves them: columns of one row
    s["qkv"] = randn(M, (H + 2 * Hkv) * D)
    s["q_norm"] = 1 + 0.1 * randn(D) if c["norm"] else None
    s["k_norm"] = 1 + 0.1 * randn(D) if c["norm"] else None
    s["q_out"] = torch.zeros(M, H * D, **dev)
    return s


def run(state):
    if own:
        return OWN[state["case"]["op"]](state)
    return PLAIN[state["case"]["op"]](state)


# ---- the library's calls ----------------------------------------------------


def _parts(s):
    c = s["case"]
    a, b = c["H"] * c["D"], (c["H"] + c["Hkv"]) * c["D"]
    return s["qkv"][:, :a], s["qkv"][:, a:b], s["qkv"][:, b:]


def _handles(s):
    """What a program keeps beside its buffers: descriptors of the rotation, the cache and the batch, a workspace."""
    if "handles" not in s:
        import cretif_amd as cri

        c, h = s["case"], {"cri": cri}
        if "qkv" in s:
            h["rot"] = cri.Rotation(c["theta"], c["rot"], "halves" if c["halves"] else "adjacent", s["q_norm"],
                                    s["k_norm"], EPS)
            h["parts"] = _parts(s)
        if "k_pages" in s:
            h["cache"] = cri.PagedKV(s["k_pages"], s["v_pages"])
            h["batch"] = cri.PagedBatch(s["offsets"], s["lens"], s["pages"])
        if c["op"] == "paged_attention":
            need = cri.paged_attention_workspace_bytes(h["cache"], h["batch"], s["q"].shape[0], c["H"], c["P"])
            h["ws"] = torch.empty(need, dtype=torch.uint8, device="cuda")
        if c["op"] == "verify_drafts":
            need = cri.verify_drafts_workspace_bytes(c["B"], c["V"])
            h["ws"] = torch.empty(need, dtype=torch.uint8, device="cuda")
        s["handles"] = h
    return s["handles"]


def _own_norm_rope(s):
    h, c = _handles(s), s["case"]
    q, k, _ = h["parts"]
    h["cri"].qk_norm_rope(h["rot"], q, k, s["q_out"], s["k_out"], s["positions"], c["H"], c["Hkv"], c["D"])
    return s["q_out"], s["k_out"]


def _own_append(s):
    h, c = _handles(s), s["case"]
    q, k, v = h["parts"]
    h["cri"].paged_append(h["cache"], h["batch"], h["rot"], k, v, q, s["q_out"], c["H"])
    return s["q_out"], s["k_pages"], s["v_pages"]


def _own_attention(s):
    h, c = _handles(s), s["case"]
    h["cri"].paged_attention(h["cache"], h["batch"], s["q"], s["out"], c["H"], c["D"] ** -0.5, s["prefix_pages"],
                             c["P"], h["ws"])
    return s["out"]


def _own_verify(s):
    h = _handles(s)
    # one set of numbers decides and draws, as in the plain form (a sampler has independent ones)
    h["cri"].verify_drafts(s["target"], s["draft"], s["ids"], s["u"], s["u"], s["offsets"], s["out_ids"],
                           s["accepted"], h["ws"])
    return s["out_ids"], s["accepted"]


OWN = {"qk_norm_rope": _own_norm_rope, "paged_append": _own_append, "paged_attention": _own_attention,
       "verify_drafts": _own_verify}


# ---- the plain forms --------------------------------------------------------


def _norm_rotate(x, w, positions, c):
    """x [M, heads, D]: the norm in 32 bits, the angles in 64 (a far position's angle has no bits left in 32)."""
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    rot = c["rot"]
    inv = c["theta"] ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=x.device) / rot)
    angle = positions.double()[:, None] * inv
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    out = x.clone()
    if c["halves"]:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        out[..., :rot // 2], out[..., rot // 2:rot] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        out[..., 0:rot:2], out[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
    return out


def _plain_norm_rope(s):
    c = s["case"]
    q, k, _ = _parts(s)
    M = c["M"]
    s["q_out"][:] = _norm_rotate(q.reshape(M, c["H"], c["D"]), s["q_norm"], s["positions"], c).reshape(M, -1)
    s["k_out"][:] = _norm_rotate(k.reshape(M, c["Hkv"], c["D"]), s["k_norm"], s["positions"], c).reshape(M, -1)
    return s["q_out"], s["k_out"]


def _places(s):
    """Sequence, index in it and position of every token."""
    t = torch.arange(s["real"], device="cuda")
    off = s["offsets"].long()
    seq = torch.searchsorted(off[1:], t, right=True)
    i = t - off[seq]
    return seq, i, s["lens"].long()[seq] - (off[seq + 1] - off[seq]) + i


def _plain_append(s):
    c, R = s["case"], s["real"]
    seq, _, pos = _places(s)
    q, k, v = (x[:R] for x in _parts(s))
    page = s["pages"].long()[seq, pos // c["ps"]]
    s["q_out"][:R] = _norm_rotate(q.reshape(R, c["H"], c["D"]), s["q_norm"], pos, c).reshape(R, -1)
    k = _norm_rotate(k.reshape(R, c["Hkv"], c["D"]), s["k_norm"], pos, c)
    s["k_pages"][page, pos % c["ps"]] = k.to(s["k_pages"].dtype)
    s["v_pages"][page, pos % c["ps"]] = v.reshape(R, c["Hkv"], c["D"]).to(s["v_pages"].dtype)
    return s["q_out"], s["k_pages"], s["v_pages"]


def _plain_attention(s):
    c, R = s["case"], s["real"]
    H, Hkv, D, P, ps, B, N = c["H"], c["Hkv"], c["D"], c["P"], c["ps"], c["B"], s["most"]
    G, S, scale = H // Hkv, s["longest"] - c["P"], D ** -0.5
    seq, i, pos = _places(s)
    q = s["q"][:R].reshape(R, Hkv, G, D)
    # the prefix: one product for all rows
    pp = s["prefix_pages"].long()
    kp = s["k_pages"][pp].reshape(-1, Hkv, D)[:P].float().permute(1, 2, 0).contiguous()  # [Hkv, D, P]
    vp = s["v_pages"][pp].reshape(-1, Hkv, D)[:P].float().permute(1, 0, 2).contiguous()  # [Hkv, P, D]
    qp = q.permute(1, 0, 2, 3).reshape(Hkv, R * G, D)
    a = torch.matmul(qp, kp) * scale
    a = a.reshape(Hkv, R, G, P)
    # each sequence's own positions, padded to the longest
    own_pos = P + torch.arange(S, device="cuda")
    page = s["pages"].long()[:, own_pos // ps]
    ks = s["k_pages"][page, own_pos % ps].float().permute(0, 2, 3, 1).contiguous()  # [B, Hkv, D, S]
    vs = s["v_pages"][page, own_pos % ps].float().permute(0, 2, 1, 3).contiguous()
    qs = torch.zeros(B, N, Hkv, G, D, device="cuda")
    qs[seq, i] = q
    b = torch.matmul(qs.permute(0, 2, 1, 3, 4).reshape(B, Hkv, N * G, D), ks) * scale
    b = b.reshape(B, Hkv, N, G, S).permute(0, 2, 1, 3, 4)[seq, i]  # [R, Hkv, G, S]
    b = b.masked_fill(own_pos > pos[:, None, None, None], -math.inf)
    m = torch.maximum(a.amax(-1).permute(1, 0, 2), b.amax(-1))  # [R, Hkv, G]
    a = torch.exp(a - m.permute(1, 0, 2)[..., None])
    b = torch.exp(b - m[..., None])
    total = a.sum(-1).permute(1, 0, 2) + b.sum(-1)
    out = torch.matmul(a.reshape(Hkv, R * G, P), vp).reshape(Hkv, R, G, D).permute(1, 0, 2, 3)
    bs = torch.zeros(B, N, Hkv, G, S, device="cuda")
    bs[seq, i] = b
    more = torch.matmul(bs.permute(0, 2, 1, 3, 4).reshape(B, Hkv, N * G, S), vs)
    out = out + more.reshape(B, Hkv, N, G, D).permute(0, 2, 1, 3, 4)[seq, i]
    s["out"][:R] = (out / total[..., None]).reshape(R, H * D)
    return s["out"]


def _plain_verify(s):
    c, N = s["case"], s["most"]
    B, V = c["B"], c["V"]
    off = s["offsets"].long()
    n = off[1:] - off[:-1]
    j = torch.arange(N, device="cuda")
    row = torch.minimum(off[:-1, None] + j, off[1:, None] - 1)  # [B, N]
    ids = s["ids"].long()[row]
    p = s["target"][row, ids].double()
    q = s["draft"][row, ids].double() if s["draft"] is not None else torch.ones_like(p)
    ok = (s["u"][row].double() * q < p) & (j < n[:, None] - 1)
    a = ok.long().cumprod(1).sum(1)  # accepted drafts of each sequence
    at = off[:-1] + a
    rejected = a < n - 1
    t = s["target"][at].double()
    if s["draft"] is not None:
        d = s["draft"][at].double()
    else:
        d = torch.zeros_like(t)
        d[torch.arange(B, device="cuda"), s["ids"].long()[at]] = math.inf  # a sure draft: nothing of it is left
    left = torch.where(rejected[:, None], (t - d).clamp_min(0), t)
    left = torch.where(left.sum(1, keepdim=True) > 0, left, t)
    cum = left.cumsum(1)  # in 64 bits: the drawn number may fall next to a border
    token = (cum <= s["u"][at].double()[:, None] * cum[:, -1:]).sum(1)
    last = V - 1 - (left > 0).flip(1).long().argmax(1)
    token = torch.minimum(token, last)
    # accepted drafts, the drawn token, -1 behind it
    tok = torch.arange(s["ids"].numel(), device="cuda")
    seq = torch.searchsorted(off[1:], tok, right=True)
    i = tok - off[seq]
    s["out_ids"][:] = torch.where(i < a[seq], s["ids"].long(), torch.where(i == a[seq], token[seq], -1)).int()
    s["accepted"][:] = a.int()
    return s["out_ids"], s["accepted"]


PLAIN = {"qk_norm_rope": _plain_norm_rope, "paged_append": _plain_append, "paged_attention": _plain_attention,
         "verify_drafts": _plain_verify}


# ---- work and float64 results ------------------------------------------------


def _mean_rows(c):
    return c["B"] * ((c["n"] + 1) / 2 if c["ragged"] else c["n"])


def work(case):
    c = case
    if c["op"] == "verify_drafts":
        rows = c["B"] * (2 if c["draft"] else 1)
        return {"bytes": 4 * rows * c["V"] + 16 * _mean_rows(c), "flops": 3 * c["B"] * c["V"]}
    H, Hkv, D = c["H"], c["Hkv"], c["D"]
    if c["op"] == "qk_norm_rope":
        n = c["M"] * (H + Hkv) * D
        return {"bytes": 8 * n, "flops": 8 * n}
    T, e = _mean_rows(c), 4 if c["type"] == "fp32" else 2
    if c["op"] == "paged_append":
        return {"bytes": T * D * (8 * H + 2 * Hkv * (4 + e)), "flops": 8 * T * (H + Hkv) * D}
    own_len = c["own_len"] / 2 + T / c["B"] / 2
    return {"bytes": 2 * Hkv * D * e * (c["P"] + c["B"] * own_len) + 8 * T * H * D,
            "flops": 4 * T * H * D * (c["P"] + own_len)}


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c["op"] == "verify_drafts":
        return _exact_verify(s)
    f64 = lambda x: None if x is None else x.double()  # noqa: E731

    def rotated(x, w, p):
        """One pair at a time as a complex number."""
        x = x.double()
        if w is not None:
            x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / c["D"] + EPS) * f64(w)
        r = c["rot"]
        turn = torch.polar(torch.ones(r // 2, dtype=torch.float64, device="cuda").expand(len(p), -1),
                           p.double()[:, None] / torch.pow(torch.tensor(c["theta"], dtype=torch.float64, device="cuda"),
                                                           torch.arange(r // 2, device="cuda").double() * 2 / r))
        head = x[..., :r].reshape(*x.shape[:-1], *((2, r // 2) if c["halves"] else (r // 2, 2)))
        head = head.transpose(-1, -2) if c["halves"] else head
        z = torch.view_as_real(torch.view_as_complex(head.contiguous()) * turn[:, None])
        z = z.transpose(-1, -2) if c["halves"] else z
        return torch.cat([z.reshape(*x.shape[:-1], r), x[..., r:]], -1)

    if c["op"] == "qk_norm_rope":
        q, k, _ = (x.reshape(c["M"], -1, c["D"]) for x in _parts(s))
        return (rotated(q, s["q_norm"], s["positions"]).reshape(c["M"], -1),
                rotated(k, s["k_norm"], s["positions"]).reshape(c["M"], -1))
    off, held = s["offsets"].tolist(), s["lens"].tolist()
    if c["op"] == "paged_append":
        q_out, kp, vp = s["q_out"].double(), s["k_pages"].double(), s["v_pages"].double()
        for b in range(c["B"]):
            lo, hi = off[b], off[b + 1]
            p = torch.arange(held[b] - (hi - lo), held[b], device="cuda")
            q, k, v = (x[lo:hi].reshape(hi - lo, -1, c["D"]) for x in _parts(s))
            q_out[lo:hi] = rotated(q, s["q_norm"], p).reshape(hi - lo, -1)
            at = s["pages"][b].long()[p // c["ps"]], p % c["ps"]
            kp[at] = rotated(k, s["k_norm"], p)
            vp[at] = v.double()
        return q_out, kp, vp
    # attention: a sequence and a key head at a time over all its positions in a row
    out = s["out"].double()
    H, Hkv, D, P, ps = c["H"], c["Hkv"], c["D"], c["P"], c["ps"]
    G, pp = H // Hkv, s["prefix_pages"].long()
    if 4 * s["real"] * H * D * s["longest"] > 1.2e12:
        return None
    pos = torch.arange(s["longest"], device="cuda")
    for b in range(c["B"]):
        lo, hi, L = off[b], off[b + 1], held[b]
        page = s["pages"][b].long()[pos[:L] // ps]
        page[:P] = pp[pos[:P] // ps]
        k, v = s["k_pages"][page, pos[:L] % ps].double(), s["v_pages"][page, pos[:L] % ps].double()
        q = s["q"][lo:hi].double().reshape(hi - lo, Hkv, G, D)
        seen = pos[:L] <= torch.arange(L - (hi - lo), L, device="cuda")[:, None]
        for h in range(Hkv):
            x = q[:, h].reshape(-1, D) @ k[:, h].t().contiguous() / math.sqrt(D)
            x = x.reshape(hi - lo, G, L).masked_fill(~seen[:, None], -math.inf)
            w = torch.softmax(x, -1).reshape(-1, L)
            out[lo:hi, h * G * D:(h + 1) * G * D] = (w @ v[:, h].contiguous()).reshape(hi - lo, G * D)
    return out


def _exact_verify(s):
    import numpy as np

    off = s["offsets"].cpu().numpy()
    ids, u = s["ids"].cpu().numpy(), s["u"].cpu().numpy().astype(np.float64)
    out, acc = np.full(len(ids), -1, np.int32), np.zeros(len(off) - 1, np.int32)
    for b in range(len(off) - 1):
        a = 0
        for r in range(off[b], off[b + 1] - 1):
            p = float(s["target"][r, int(ids[r])])
            q = 1.0 if s["draft"] is None else float(s["draft"][r, int(ids[r])])
            if not u[r] * q < p:
                break
            out[r] = ids[r]
            a += 1
        r = off[b] + a
        p = s["target"][r].double().cpu().numpy()
        w = p
        if r < off[b + 1] - 1:
            w = p.copy()
            if s["draft"] is None:
                w[ids[r]] = 0
            else:
                w = np.maximum(w - s["draft"][r].double().cpu().numpy(), 0)
            if not w.sum() > 0:
                w = p
        cum = np.cumsum(w)
        t = int(np.searchsorted(cum, u[r] * cum[-1], side="right"))
        out[r] = min(t, int(np.flatnonzero(w > 0)[-1]))
        acc[b] = a
    return torch.from_numpy(out), torch.from_numpy(acc)
