"""The choice of experts where values meet that are near each other and values that are no numbers, against sorting in 64 bits by
(is no number, larger first, lower index): every row's indices differ, NaN comes behind -inf, and a group's worth that is no number
counts as -inf."""
import math

import pytest
import torch

from head_decay_plain import F32

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


def _plain(x, k, scores, bias, groups=1, groups_use=1, group_top=1):
    """(index, s of the chosen) for one row of floats."""
    E, bias = len(x), [float(b) for b in bias]
    if scores == "sigmoid":
        s = [v if v != v else 1.0 / (1.0 + math.exp(-v)) if v > -700 else 0.0 for v in x]
    else:
        top = max(x, key=lambda v: -INF if v != v else v)
        e = [NAN if v != v else 0.0 if v == -INF else math.exp(v - top) for v in x]
        s = [v / sum(e) if sum(e) != 0 else 0.0 for v in e]
    c = [a + b for a, b in zip(s, bias)]
    number = lambda v: -INF if v != v else v
    size = E // groups
    worth = [number(sum(sorted((number(v) for v in c[j * size:(j + 1) * size]), reverse=True)[:group_top])) for j in range(groups)]
    kept = sorted(range(groups), key=lambda j: (-worth[j], j))[:groups_use]
    order = sorted((i for i in range(E) if i // size in kept), key=lambda i: (c[i] != c[i], -number(c[i]), i))[:k]
    return order, [s[i] for i in order]


def _hold(x, k, scores, bias, **how):
    from transformer_b200.parts import choose_experts
    x = torch.as_tensor(x, dtype=torch.float32)
    bias = torch.as_tensor(bias, dtype=torch.float32)
    idx = torch.full((x.shape[0], k), -7, dtype=torch.int32, device="cuda")
    w = torch.full((x.shape[0], k), 7.0, device="cuda")
    choose_experts(x.cuda(), idx, w, scores=scores, bias=bias.cuda(), **how)
    idx, w = idx.cpu(), w.cpu().double()
    for t, row in enumerate(x.tolist()):
        order, s = _plain(row, k, scores, bias.tolist(), **how)
        assert idx[t].tolist() == order, (row, bias.tolist(), how)
        s = torch.tensor(s, dtype=torch.float64)
        assert torch.equal(w[t].isnan(), s.isnan())
        assert bool((((w[t] - s).abs() <= 64 * F32 * s.abs() + 1e-37) | s.isnan()).all())


@pytest.mark.parametrize("k", [1, 2, 3, 4])
def test_a_candidate_that_is_no_number(k):
    """Saturated scores are near each other in float, 64 bits tell them apart; the NaN is among the k + 1 that are looked at."""
    rows = [[20.0, 25.0, 0.0, NAN], [NAN, 25.0, 20.0, 0.0], [20.0, NAN, 0.0, 25.0], [25.0, 20.0, NAN, NAN], [NAN, NAN, NAN, 20.0],
            [20.0, 25.0, 60.0, NAN], [-INF, 25.0, 20.0, NAN], [20.0, 20.0, NAN, 25.0], [NAN, NAN, NAN, NAN]]
    _hold(rows, k, "sigmoid", [0.0] * 4)
    _hold(rows, k, "sigmoid", [0.0, 0.0, 0.0, NAN])
    _hold(rows, k, "sigmoid", [0.0, 0.0, -INF, 0.0])
    _hold(rows, k, "sigmoid", [1e-9, 0.0, 0.0, 1e-9])


@pytest.mark.parametrize("E,k,groups,groups_use", [(12, 5, 1, 1), (12, 8, 1, 1), (40, 9, 4, 1), (40, 10, 4, 1), (64, 6, 8, 3), (96, 24, 4, 1),
                                                   (256, 8, 8, 4), (300, 30, 1, 1), (600, 9, 6, 2)])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_rows_of_near_values_and_none(E, k, groups, groups_use, scores):
    gen = torch.Generator().manual_seed(E + k)
    pick = lambda values, share: torch.where(torch.rand(30, E, generator=gen) < share, torch.tensor(values)[torch.randint(0, len(values), (30, E), generator=gen)], 0.0)
    near = torch.full((30, E), 1.25).view(torch.int32) + torch.randint(0, 5, (30, E), generator=gen, dtype=torch.int32)
    x = near.view(torch.float32) + pick([20.0, 25.0, 60.0, -3.0] if scores == "sigmoid" else [-3.0, 0.5], 0.5)
    if scores == "sigmoid":             # one NaN of a softmax is all of its row's, which the last test looks at
        x = x + pick([NAN, -INF], 0.3)
    masks = torch.zeros(E)
    masks[torch.randperm(E, generator=gen)[: E // 4]] = -INF
    nans = masks.clone()
    nans[torch.randperm(E, generator=gen)[: E // 8 + 1]] = NAN
    for bias in (torch.zeros(E), masks, nans, torch.randint(0, 2, (E,), generator=gen) * 1e-8):
        for top in (1, 2):
            _hold(x, k, scores, bias, groups=groups, groups_use=groups_use, group_top=top)


def test_one_that_is_none_is_all_of_a_softmax():
    _hold([[1.0, NAN, 2.0, 3.0], [NAN, -INF, -INF, -INF]], 3, "softmax", [0.0, 0.0, 1.0, -INF])


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_a_worth_of_infinity_less_infinity(scores):
    """Groups of two, one of them with a bias of both infinities: no worth at all, so the others are used."""
    x = torch.randn(20, 8, generator=torch.Generator().manual_seed(3))
    for at in range(0, 8, 2):
        bias = torch.zeros(8)
        bias[at], bias[at + 1] = INF, -INF
        for use, k in ((1, 2), (2, 4), (3, 6)):
            _hold(x, k, scores, bias, groups=4, groups_use=use, group_top=2)
        bias[(at + 2) % 8], bias[(at + 3) % 8] = -INF, INF
        _hold(x, 4, scores, bias, groups=4, groups_use=2, group_top=2)


def test_logits_order_experts_of_equal_scores_however_their_groups_were_decided():
    """Without a bias experts are compared by their logits, also where 64 bits have no scores between (sigmoids of 1, softmaxes of 0): in rows
    whose groups are far apart, need no decision, or are equal and decided in 64 bits."""
    from transformer_b200.parts import choose_experts

    def chosen(row, k, scores, use):
        idx, w = torch.empty((1, k), dtype=torch.int32, device="cuda"), torch.empty((1, k), device="cuda")
        choose_experts(torch.tensor([row]).cuda(), idx, w, scores=scores, groups=2, groups_use=use, group_top=2)
        return idx[0].tolist()

    assert chosen([40.0, 41.0, -9.0, -8.0], 2, "sigmoid", 1) == [1, 0]
    assert chosen([40.0, 41.0, 50.0, 60.0], 2, "sigmoid", 1) == [1, 0]
    assert chosen([40.0, 41.0, 50.0, 60.0], 4, "sigmoid", 2) == [3, 2, 1, 0]
    assert chosen([3e38, INF, 50.0, 60.0], 2, "sigmoid", 1) == [1, 0]
    assert chosen([1.0, -900.0, -800.0, -999.0, 1.0, -950.0, -INF, NAN], 4, "sigmoid", 1) == [0, 2, 1, 3]
    assert chosen([1.0, -900.0, -800.0, -999.0, 1.0, -950.0, -980.0, -INF], 4, "softmax", 1) == [0, 2, 1, 3]


def test_the_most_tokens():
    """2^31 - 1 rows of one expert (26 GB): as many blocks as that is."""
    from transformer_b200.parts import choose_experts
    n = 2 ** 31 - 1
    x, idx, w = torch.zeros((n, 1), device="cuda"), torch.full((n, 1), 7, dtype=torch.int32, device="cuda"), torch.zeros((n, 1), device="cuda")
    choose_experts(x, idx, w)
    assert not bool(idx.any()) and bool((w == 1).all())
    del x, idx, w
    torch.cuda.empty_cache()
