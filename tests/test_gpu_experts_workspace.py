"""Calls of a layer of experts that share a workspace and run at once, against their contract: anything may come out, nowhere
else, and the next call that has the workspace to itself is right."""
import numpy as np
import pytest
import torch

import cretif_amd as cri
import experts_ref as ref

pytestmark = pytest.mark.gpu

AROUND = 1 << 20


class Call:
    """One grouping of M tokens: arrays with room around them, choices drawn from `experts`."""

    def __init__(self, M, k, E, experts, seed):
        rng = np.random.default_rng(seed)
        self.ids = np.sort(rng.choice(experts, (M, k)), 1)
        self.dids = torch.from_numpy(self.ids.astype(np.int32)).cuda()
        self.whole = [torch.full((n + 2 * AROUND,), -7, dtype=torch.int32, device="cuda") for n in (E + 1, M * k, M * k)]
        self.g = cri.ExpertGroups(M, k, E, *(t[AROUND:-AROUND] for t in self.whole))

    def untouched(self):
        return all(bool((t[:AROUND] == -7).all()) and bool((t[-AROUND:] == -7).all()) for t in self.whole)

    def right(self):
        want = ref.group(self.ids, self.g.n_experts)
        return all(np.array_equal(t.cpu().numpy(), w) for t, w in zip((self.g.offsets, self.g.rows, self.g.slots), want))


def test_groupings_that_share_a_workspace_at_once():
    E, k = 64, 8
    # as many blocks of counts each, but far more pairs of an expert in the second's
    a, b = Call(5000, k, E, np.arange(E), 1), Call(100000, k, E, np.array([0, 63]), 2)
    need = max(cri.route_experts_workspace_bytes(c.g) for c in (a, b))
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    words = ws.view(torch.int32)
    s, t, u = (torch.cuda.Stream() for _ in range(3))
    torch.cuda.synchronize()
    for i in range(40):
        cri.group_experts(a.dids, a.g, ws, s)
        cri.group_experts(b.dids, b.g, ws, t)
        with torch.cuda.stream(u):
            words.fill_((1 << 30, -(1 << 30), 2 ** 31 - 1, 17)[i % 4])
    torch.cuda.synchronize()
    assert a.untouched() and b.untouched()
    for c in (a, b, a):
        cri.group_experts(c.dids, c.g, ws)
        assert c.right() and c.untouched()
