"""Operators of a layer of experts over GGUF weights: inputs, plain forms, the library's calls, work and float64 results.

  route    the router's logits become each token's experts, their weights and the rows grouped by expert
  matmul   products grouped by expert with ragged numbers of rows
  swiglu   SiLU(x gate^T) * (x up^T) of every token's experts, rows grouped by expert
  combine  the experts' down products, weighted and added up per token onto the residual stream

`own` False computes them with elementary torch operations, True calls cretif_amd.
"""
import math
import random

import torch

own = False

# format: values and bytes of a block
BLOCK = {"q8_0": (32, 34), "q4_0": (32, 18), "q5_0": (32, 22), "q4_k": (256, 144), "q6_k": (256, 210), "fp16": (32, 64)}


def listed():
    return [
        # one new token of one sequence, many small experts
        dict(name="route_token", op="route", M=1, E=128, k=8, scoring="softmax", bias=False, normalize=True, pad=0),
        # a batch of long prompts: sigmoid scores, a bias that balances the load
        dict(name="route_prompt", op="route", M=8192, E=256, k=8, scoring="sigmoid", bias=True, normalize=True, pad=5),
        # a small model's step with few conversations
        dict(name="matmul_step_q8_0", op="matmul", M=16, E=32, k=4, N=1536, K=576, fmt="q8_0", pad=0),
        # few tokens through a few large experts
        dict(name="matmul_few_q4_k", op="matmul", M=3, E=8, k=2, N=8192, K=2048, fmt="q4_k", pad=0),
        # a prompt's piece
        dict(name="matmul_prompt_q6_k", op="matmul", M=1000, E=16, k=2, N=2048, K=2048, fmt="q6_k", pad=0),
        # one new token
        dict(name="swiglu_token_q4_k", op="swiglu", M=1, E=64, k=8, N=1024, K=2048, fmt="q4_k", pad=0),
        # a serving step of many conversations: every expert has a few rows
        dict(name="swiglu_step_q5_0", op="swiglu", M=48, E=60, k=4, N=1408, K=2048, fmt="q5_0", pad=0),
        # a small model's prompt in a padded batch
        dict(name="swiglu_padded_fp16", op="swiglu", M=777, E=8, k=2, N=1536, K=576, fmt="fp16", pad=77),
        # prompts of several sequences at once
        dict(name="swiglu_prompt_q4_k", op="swiglu", M=4096, E=64, k=8, N=1024, K=2048, fmt="q4_k", pad=0),
        # the way back of the token, the step and the prompts
        dict(name="combine_token_q6_k", op="combine", M=1, E=64, k=8, N=2048, K=1024, fmt="q6_k", pad=0),
        dict(name="combine_step_q4_0", op="combine", M=48, E=60, k=4, N=2048, K=1408, fmt="q4_0", pad=0),
        dict(name="combine_prompt_q4_k", op="combine", M=4096, E=64, k=8, N=2048, K=1024, fmt="q4_k", pad=0),
    ]


def _span(rng, lo, hi):
    """lo .. hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["route", "matmul", "swiglu", "swiglu", "combine", "combine"])
    E = rng.choice([4, 8, 16, 32, 60, 64, 128, 160, 256])
    k = rng.randint(1, min(E, rng.choice([2, 4, 8, 8, 10])))
    if op == "route":
        scoring = rng.choice(["softmax", "sigmoid"])
        return dict(op=op, M=_span(rng, 1, 8192), E=E, k=k, scoring=scoring, bias=scoring == "sigmoid" and rng.random() < 0.7,
                    normalize=rng.random() < 0.7, pad=rng.choice([0, 0, 3]))
    fmt = rng.choice(["q8_0", "q4_0", "q5_0", "q4_k", "q4_k", "q6_k", "fp16"])
    bs = BLOCK[fmt][0] if fmt != "fp16" else 32
    most = 64 * 1024 * 2048  # weights of the largest listed cases' matrix, and a layer's products
    K = max(bs, _span(rng, 256, 8192) // bs * bs)
    N = _span(rng, 64, max(65, min(8192, most // (E * K))))
    if rng.random() < 0.5:
        N = (N + 31) // 32 * 32
    M = _span(rng, 1, max(2, min(4096, 4096 * 8 * 1024 * 2048 // (k * N * K))))
    return dict(op=op, M=M, E=E, k=k, N=N, K=K, fmt=fmt, pad=rng.choice([0, 0, M // 10]))


# ---- inputs -------------------------------------------------------------------


def _halves(x):
    return x.to(torch.float16).unsqueeze(-1).contiguous().view(torch.uint8)


def _weights(g, fmt, E, N, K):
    """Blocks [E, N, K / values, bytes] of a trained matrix's size: values of about 1 / sqrt(K), centred."""
    dev = dict(device="cuda", generator=g)
    n, sigma = K // BLOCK[fmt][0], K ** -0.5
    scale = sigma * (0.7 + 0.6 * torch.rand(E, N, n, **dev))  # a block's own magnitude
    raw = lambda width: torch.randint(0, 256, (E, N, n, width), dtype=torch.uint8, **dev)  # noqa: E731
    if fmt == "fp16":
        return _halves(sigma * torch.randn(E, N, K, **dev)).reshape(E, N, n, 64)
    if fmt == "q8_0":
        return torch.cat([_halves(scale / 74), raw(32)], -1)
    if fmt == "q4_0":
        return torch.cat([_halves(scale / 4.6), raw(16)], -1)
    if fmt == "q5_0":
        return torch.cat([_halves(scale / 9.2), raw(20)], -1)
    if fmt == "q6_k":
        sc = torch.randint(48, 128, (E, N, n, 16), dtype=torch.uint8, **dev)
        sc = torch.where(torch.rand(sc.shape, **dev) < 0.5, sc, (256 - sc.int()).to(torch.uint8))  # int8, either sign
        return torch.cat([raw(192), sc, _halves(scale / (88 * 18.5))], -1)
    sc = torch.randint(24, 64, (E, N, n, 8), dtype=torch.int32, **dev)  # q4_k: each sub-block's range centred by its minimum
    mn = (sc + torch.randint(-4, 5, sc.shape, dtype=torch.int32, **dev)).clamp(0, 63)
    low = (sc[..., :4] | (sc[..., 4:] >> 4 << 6), mn[..., :4] | (mn[..., 4:] >> 4 << 6), (sc[..., 4:] & 15) | ((mn[..., 4:] & 15) << 4))
    d = scale / (44 * 4.6)
    return torch.cat([_halves(d), _halves(7.5 * d), torch.cat(low, -1).to(torch.uint8), raw(128)], -1)


def _routed(g, M, E, k, pad):
    """Distinct experts for each token, some experts more wanted than others; the last `pad` tokens have none."""
    dev = dict(device="cuda", generator=g)
    ids = (torch.randn(M, E, **dev) + 0.7 * torch.randn(E, **dev)).topk(k, -1).indices.int()
    ids[M - pad:] = -1
    weights = torch.softmax(torch.randn(M, k, **dev), -1)
    weights[M - pad:] = 0
    return ids, weights


def _grouped(ids, E):
    """offsets [E + 1], rows (the pairs of token and choice, by expert) and slots (where each pair is, or -1)."""
    flat = ids.flatten().long()
    key = torch.where((flat >= 0) & (flat < E), flat, E)
    order = torch.sort(key, stable=True).indices
    offsets = torch.searchsorted(key[order].contiguous(), torch.arange(E + 1, device=key.device))
    slots = torch.empty_like(order)
    slots[order] = torch.arange(len(order), device=key.device)
    slots = torch.where(key < E, slots, -1)
    rows = torch.where(torch.arange(len(order), device=key.device) < offsets[E], order, -1)
    return offsets.int(), rows.int(), slots.int()


def prepare(case, seed):
    c = case
    g = torch.Generator("cuda").manual_seed(seed)
    dev = dict(device="cuda", generator=g)
    s, M, E, k = dict(case=c), c["M"], c["E"], c["k"]
    if c["op"] == "route":
        s["logits"] = 1.5 * torch.randn(M, E, **dev) + 0.7 * torch.randn(E, **dev)
        if c["pad"] and M > c["pad"]:  # tokens of a padded batch choose nothing
            s["logits"][M - c["pad"]:] = -math.inf
        s["bias"] = 0.1 * torch.randn(E, **dev) if c["bias"] else None
        s["scale"] = 2.5 if c["scoring"] == "sigmoid" else 1.0
        s["ids"] = torch.zeros(M, k, dtype=torch.int32, device="cuda")
        s["weights"] = torch.zeros(M, k, device="cuda")
        s["offsets"] = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
        s["rows"], s["slots"] = (torch.zeros(M * k, dtype=torch.int32, device="cuda") for _ in range(2))
        return s
    ids, s["weights"] = _routed(g, M, E, k, c["pad"])
    s["offsets"], s["rows"], s["slots"] = _grouped(ids, E)
    s["most"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())
    channels = torch.where(torch.rand(c["K"], **dev) < 0.01, 8.0, 1.0)  # a few channels are larger than the others
    s["x"] = torch.randn(M * k if c["op"] == "combine" else M, c["K"], **dev) * channels
    s["w"] = _weights(g, c["fmt"], E, c["N"], c["K"])
    if c["op"] == "swiglu":
        s["up"] = _weights(g, c["fmt"], E, c["N"], c["K"])
    if c["op"] == "combine":
        s["residual"] = torch.randn(M, c["N"], **dev)
    s["out"] = torch.zeros(M if c["op"] == "combine" else M * k, c["N"], device="cuda")
    return s


def run(state):
    if own:
        return OWN[state["case"]["op"]](state)
    return PLAIN[state["case"]["op"]](state)


# ---- the library's calls ----------------------------------------------------


def _handles(s):
    """What a program keeps beside its buffers: the laid out weights, the groups' arrays, a workspace."""
    if "handles" not in s:
        import cretif_amd as cri

        c, h = s["case"], {"cri": cri}
        h["groups"] = cri.ExpertGroups(c["M"], c["k"], c["E"], s["offsets"], s["rows"], s["slots"])
        if c["op"] == "route":
            h["router"] = cri.ExpertRouter(c["scoring"], s["bias"], c["normalize"], s["scale"])
            need = cri.route_experts_workspace_bytes(h["groups"])
        else:
            h["w"] = cri.ExpertWeights(c["fmt"], s["w"], c["E"], c["N"], c["K"])
        if c["op"] == "matmul":
            need = cri.expert_matmul_workspace_bytes(h["w"], h["groups"])
        if c["op"] == "swiglu":
            h["up"] = cri.ExpertWeights(c["fmt"], s["up"], c["E"], c["N"], c["K"])
            need = cri.expert_swiglu_workspace_bytes(h["w"], h["groups"])
        if c["op"] == "combine":
            need = cri.expert_combine_workspace_bytes(h["w"], h["groups"])
        h["ws"] = torch.empty(need, dtype=torch.uint8, device="cuda")
        s["handles"] = h
    return s["handles"]


def _own_route(s):
    h = _handles(s)
    h["cri"].route_experts(h["router"], s["logits"], s["ids"], s["weights"], h["groups"], h["ws"])
    return s["ids"], s["weights"], s["offsets"], s["rows"], s["slots"]


def _own_matmul(s):
    h = _handles(s)
    h["cri"].expert_matmul(h["w"], h["groups"], s["x"], s["out"], h["ws"])
    return s["out"]


def _own_swiglu(s):
    h = _handles(s)
    h["cri"].expert_swiglu(h["w"], h["up"], h["groups"], s["x"], s["out"], h["ws"])
    return s["out"]


def _own_combine(s):
    h = _handles(s)
    h["cri"].expert_combine(h["w"], h["groups"], s["x"], s["weights"], s["out"], s["residual"], h["ws"])
    return s["out"]


OWN = {"route": _own_route, "matmul": _own_matmul, "swiglu": _own_swiglu, "combine": _own_combine}


# ---- the plain forms --------------------------------------------------------


def _decode(b, fmt):
    """Blocks [..., blocks, bytes] -> values [..., blocks * values], whole runs at a time."""
    half = lambda x: x.contiguous().view(torch.float16).float()  # noqa: E731
    if fmt == "fp16":
        v = half(b)
    elif fmt == "q8_0":
        v = half(b[..., :2]) * b[..., 2:].contiguous().view(torch.int8).float()
    elif fmt == "q4_0":
        q = b[..., 2:]
        v = half(b[..., :2]) * (torch.stack([q & 15, q >> 4], -1).flatten(-2).float() - 8)
    elif fmt == "q5_0":
        high = b[..., 2:6].unsqueeze(-1) >> torch.arange(8, dtype=torch.uint8, device=b.device) & 1
        q = torch.cat([b[..., 6:] & 15, b[..., 6:] >> 4], -1) | high.flatten(-2) << 4
        v = half(b[..., :2]) * (q.float() - 16)
    elif fmt == "q4_k":
        s = b[..., 4:16]
        sc = torch.cat([s[..., :4] & 63, (s[..., 8:] & 15) | s[..., :4] >> 6 << 4], -1).float()
        mn = torch.cat([s[..., 4:8] & 63, s[..., 8:] >> 4 | s[..., 4:8] >> 6 << 4], -1).float()
        q = b[..., 16:].unflatten(-1, (4, 1, 32))
        q = torch.cat([q & 15, q >> 4], -2).flatten(-3, -2).float()  # [..., 8, 32]
        v = ((half(b[..., :2]) * sc).unsqueeze(-1) * q - (half(b[..., 2:4]) * mn).unsqueeze(-1)).flatten(-2)
    else:
        low, high = b[..., :128].unflatten(-1, (2, 2, 32)), b[..., 128:192].unflatten(-1, (2, 1, 32))
        low = torch.cat([low & 15, low >> 4], -2)  # [..., 2, 4, 32]
        high = torch.cat([high & 3, high >> 2 & 3, high >> 4 & 3, high >> 6], -2)
        q = (low | high << 4).flatten(-3).unflatten(-1, (16, 16)).float() - 32
        sc = b[..., 192:208].contiguous().view(torch.int8).float()
        v = ((half(b[..., 208:]) * sc).unsqueeze(-1) * q).flatten(-2)
    return v.flatten(-2)


def _products(s, *weights):
    """The products of the grouped rows with each matrix of `weights`, [rows, N]."""
    c = s["case"]
    M, E, k, N, K = (c[x] for x in ("M", "E", "k", "N", "K"))
    off = s["offsets"].long()
    R = M * k
    if R <= E:  # each row with its own expert's matrix
        r = torch.arange(R, device="cuda")
        e = torch.searchsorted(off[1:], r, right=True).clamp_max(E - 1)
        a = s["x"] if c["op"] == "combine" else s["x"][s["rows"].long().clamp_min(0) // k]
        return [torch.matmul(_decode(w[e], c["fmt"]), a.unsqueeze(-1)).squeeze(-1) for w in weights]
    r = off[:-1, None] + torch.arange(s["most"], device="cuda")  # [E, most], padded to the fullest expert
    real = r < off[1:, None]
    r = r.clamp_max(R - 1)
    a = s["x"][r] if c["op"] == "combine" else s["x"][s["rows"].long().clamp_min(0)[r] // k]
    at = torch.where(real, r, R).flatten()
    results = []
    for w in weights:
        p = torch.matmul(a, _decode(w, c["fmt"]).transpose(1, 2)).flatten(0, 1)
        full = torch.zeros(R + 1, N, device="cuda")
        full[at] = p
        results.append(full[:R])
    return results


def _into_rows(s, v):
    real = torch.arange(len(v), device="cuda") < s["offsets"][-1]
    s["out"][:] = torch.where(real[:, None], v, s["out"])
    return s["out"]


def _plain_matmul(s):
    return _into_rows(s, _products(s, s["w"])[0])


def _plain_swiglu(s):
    gate, up = _products(s, s["w"], s["up"])
    return _into_rows(s, gate / (1 + torch.exp(-gate)) * up)


def _plain_combine(s):
    slots = s["slots"].long().reshape(s["weights"].shape)
    p = _products(s, s["w"])[0][slots.clamp_min(0)]  # [M, k, N]
    w = torch.where(slots >= 0, s["weights"], 0).unsqueeze(-1)
    s["out"][:] = s["residual"] + torch.where(w != 0, w * p, 0).sum(1)
    return s["out"]


def _plain_route(s):
    c, x = s["case"], s["logits"]
    wide = x.double()  # in 64 bits: scores next to each other
    if c["scoring"] == "softmax":
        score = torch.exp(wide - wide.amax(-1, keepdim=True).clamp_min(-1e30))
        score = score / score.sum(-1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-wide))
    choice = score + s["bias"].double() if s["bias"] is not None else wide
    choice = torch.where(x > -math.inf, choice, -math.inf)
    order = torch.sort(choice, dim=-1, descending=True, stable=True).indices[:, :c["k"]]
    w = score.gather(-1, order)
    if c["normalize"]:
        w = w / w.sum(-1, keepdim=True)
    there = x.gather(-1, order) > -math.inf
    s["ids"][:] = torch.where(there, order, -1).int()
    s["weights"][:] = torch.where(there, w * s["scale"], 0).float()
    s["offsets"][:], s["rows"][:], s["slots"][:] = _grouped(s["ids"], c["E"])
    return s["ids"], s["weights"], s["offsets"], s["rows"], s["slots"]


PLAIN = {"route": _plain_route, "matmul": _plain_matmul, "swiglu": _plain_swiglu, "combine": _plain_combine}


# ---- work and float64 results ------------------------------------------------


def work(case):
    c = case
    M, E, k = c["M"] - c["pad"], c["E"], c["k"]
    if c["op"] == "route":
        return {"bytes": 4 * c["M"] * (E + 4 * k) + 4 * E, "flops": 8 * c["M"] * E}
    N, K, R = c["N"], c["K"], M * k
    values, size = BLOCK[c["fmt"]]
    used = E * (1 - (1 - k / E) ** M)  # experts that any token has
    matrix = N * K / values * size * used * (2 if c["op"] == "swiglu" else 1)
    rows = 4 * (R * K + 2 * M * N) if c["op"] == "combine" else 4 * (M * K + R * N)
    return {"bytes": matrix + rows + 12 * R, "flops": 2 * R * N * K * (2 if c["op"] == "swiglu" else 1)}


def _element(b, fmt, dtype=torch.float64):
    """One expert's blocks [N, blocks, bytes] -> [N, K] in 64 bits, element by element: where element i's bits lie."""
    i = torch.arange(BLOCK[fmt][0], device=b.device)
    at = lambda j: b[..., j].int()  # noqa: E731
    num = lambda j: (at(j) | at(j + 1) << 8).to(torch.int16).view(torch.float16).to(dtype).unsqueeze(-1)  # noqa: E731
    signed = lambda v: (v ^ 128) - 128  # noqa: E731
    if fmt == "fp16":
        bits = at(2 * i) | at(2 * i + 1) << 8
        return bits.to(torch.int16).view(torch.float16).to(dtype).flatten(1)
    if fmt == "q8_0":
        v = num(0) * signed(at(2 + i)).to(dtype)
    elif fmt == "q4_0":
        v = num(0) * ((at(2 + i // 2) >> (4 * (i % 2)) & 15) - 8).to(dtype)
    elif fmt == "q5_0":
        v = num(0) * ((at(6 + i % 16) >> (4 * (i // 16)) & 15 | (at(2 + i // 8) >> (i % 8) & 1) << 4) - 16).to(dtype)
    elif fmt == "q4_k":
        j = i // 32
        first, up = j < 4, torch.clamp(j - 4, min=0)
        sc = torch.where(first, at(4 + j.clamp_max(3)) & 63, at(12 + up) & 15 | at(4 + up) >> 6 << 4)
        mn = torch.where(first, at(8 + j.clamp_max(3)) & 63, at(12 + up) >> 4 | at(8 + up) >> 6 << 4)
        q = at(16 + i // 64 * 32 + i % 32) >> (4 * (j % 2)) & 15
        v = num(0) * sc.to(dtype) * q.to(dtype) - num(2) * mn.to(dtype)
    else:
        chunk, quarter, l = i // 128, i % 128 // 32, i % 32
        q = (at(64 * chunk + 32 * (quarter % 2) + l) >> (4 * (quarter // 2)) & 15 | (at(128 + 32 * chunk + l) >> (2 * quarter) & 3) << 4) - 32
        v = num(208) * signed(at(192 + i // 16)).to(dtype) * q.to(dtype)
    return v.flatten(1)


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c["op"] == "route":
        return _exact_route(s)
    off, rows, k = s["offsets"].tolist(), s["rows"].long(), c["k"]
    out = s["residual"].double() if c["op"] == "combine" else s["out"].double()
    for e in range(c["E"]):
        lo, hi = off[e], off[e + 1]
        if lo == hi:
            continue
        x = (s["x"][lo:hi] if c["op"] == "combine" else s["x"][rows[lo:hi] // k]).double()
        y = x @ _element(s["w"][e], c["fmt"]).t()
        if c["op"] == "swiglu":
            y = y * torch.sigmoid(y) * (x @ _element(s["up"][e], c["fmt"]).t())
        if c["op"] == "combine":
            out.index_add_(0, rows[lo:hi] // k, s["weights"].flatten()[rows[lo:hi]].double()[:, None] * y)
        else:
            out[lo:hi] = y
    return out


def _exact_route(s):
    import numpy as np

    c = s["case"]
    x, k, E = s["logits"].double().cpu().numpy(), c["k"], c["E"]
    bias = 0.0 if s["bias"] is None else s["bias"].double().cpu().numpy()
    ids, weights = np.full((c["M"], k), -1, np.int32), np.zeros((c["M"], k))
    members = [[] for _ in range(E)]
    for t in range(c["M"]):
        some = np.flatnonzero(x[t] > -np.inf)
        if not len(some):
            continue
        v = x[t][some]
        score = np.exp(v - v.max()) / np.exp(v - v.max()).sum() if c["scoring"] == "softmax" else 1 / (1 + np.exp(-v))
        key = v if s["bias"] is None else score + bias[some]
        best = np.lexsort((some, -key))[:k]
        ids[t, :len(best)] = some[best]
        weights[t, :len(best)] = score[best] / (score[best].sum() if c["normalize"] else 1) * s["scale"]
        for j, e in enumerate(some[best]):
            members[e].append(t * k + j)
    offsets = np.cumsum([0] + [len(m) for m in members]).astype(np.int32)
    flat = [p for m in members for p in m]
    rows, slots = np.full(c["M"] * k, -1, np.int32), np.full(c["M"] * k, -1, np.int32)
    rows[:len(flat)] = flat
    slots[flat] = np.arange(len(flat))
    return tuple(torch.from_numpy(a) for a in (ids, weights, offsets, rows, slots))
