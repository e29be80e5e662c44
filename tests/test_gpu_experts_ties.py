"""Routing with a bias where scores plus bias are the same number in 64 bits although their logits differ: the lowest expert first,
as cri.h says.  The scores of these logits are the same number however they are rounded: a sigmoid of 40 or more is within 2^-57 of
1, and e^-49 and less are below 2^-70, which a bias of 2^-4 or more (its half step 2^-57) does not see."""
import numpy as np
import pytest
import torch

import cretif_amd as cri

pytestmark = pytest.mark.gpu


def routed(z, k, scoring, bias, normalize=True):
    M, E = z.shape
    g = cri.ExpertGroups(M, k, E)
    ids = torch.full((M, k), 77, dtype=torch.int32, device="cuda")
    weights = torch.full((M, k), 77.0, device="cuda")
    cri.route_experts(cri.ExpertRouter(scoring, torch.from_numpy(bias).cuda(), normalize, 1.0), torch.from_numpy(z).cuda(), ids, weights, g)
    return ids.cpu().numpy(), weights.cpu().double().numpy()


@pytest.mark.parametrize("E", [8, 70, 300])
@pytest.mark.parametrize("M", [1, 100])
def test_saturated_scores_tie(E, M):
    k = 4
    rng = np.random.default_rng(E + M)
    z = np.sort(rng.uniform(40, 90, (M, E)).astype(np.float32), 1)  # the larger logits come last
    ids, weights = routed(z, k, "sigmoid", np.full(E, 0.125, np.float32))
    assert (ids == np.arange(k)).all() and (weights == 1 / k).all()
    bias = np.zeros(E, np.float32)
    bias[E - 2:] = 2.0 ** -20  # a larger sum, and the tie within it
    ids, _ = routed(z, k, "sigmoid", bias)
    assert (ids == [E - 2, E - 1, 0, 1]).all()


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_scores_that_a_bias_hides(scoring):
    E, k = 16, 5
    z = np.linspace(-70, -49, E).astype(np.float32)[None].repeat(3, 0)
    z[:, 5] = 0.0  # (softmax: the others are e^-49 and less of it)
    ids, weights = routed(z, k, scoring, np.full(E, 0.0625, np.float32), normalize=False)
    assert (ids == [5, 0, 1, 2, 3]).all()
    want = 1 / (1 + np.exp(-z[0].astype(np.float64))) if scoring == "sigmoid" else np.exp(z[0].astype(np.float64))
    want = want[[5, 0, 1, 2, 3]]
    assert (np.abs(weights - want) <= (2.0 ** -24 + 2.0 ** -40) * want).all()  # the weights are the scores, all the same


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_without_a_bias_the_logits_decide(scoring):
    z = np.sort(np.random.default_rng(1).uniform(40, 90, (5, 33)).astype(np.float32), 1)
    g = cri.ExpertGroups(5, 3, 33)
    ids, weights = torch.zeros(5, 3, dtype=torch.int32, device="cuda"), torch.zeros(5, 3, device="cuda")
    cri.route_experts(cri.ExpertRouter(scoring), torch.from_numpy(z).cuda(), ids, weights, g)
    assert (ids.cpu().numpy() == [32, 31, 30]).all()
