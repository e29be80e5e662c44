"""Grouping where every token names one expert beside others: its run of rows passes through every block's counts and every wave of
a block."""
import numpy as np
import pytest
import torch

import cretif_amd as cri
import experts_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,E,k", [(64, 1024, 64), (65, 1024, 64), (5003, 60, 8), (20000, 256, 8), (100001, 3, 2)])
@pytest.mark.parametrize("where", ["first", "last", "anywhere"])
def test_an_expert_of_every_token(M, E, k, where):
    rng = np.random.default_rng(M + E)
    order = rng.random((M, E))
    order[:, E // 2] = -1.0  # drawn first by every token
    ids = np.argsort(order, 1)[:, :k].astype(np.int32)
    if where == "last":
        ids = np.ascontiguousarray(ids[:, ::-1])
    if where == "anywhere":
        ids = np.take_along_axis(ids, np.argsort(rng.random((M, k)), 1), 1)
    g = cri.ExpertGroups(M, k, E)
    cri.group_experts(torch.from_numpy(ids).cuda(), g)
    off, rows, slots = ref.group(ids, E)
    assert off[E // 2 + 1] - off[E // 2] == M
    for got, want in ((g.offsets, off), (g.rows, rows), (g.slots, slots)):
        assert np.array_equal(got.cpu().numpy(), want)
