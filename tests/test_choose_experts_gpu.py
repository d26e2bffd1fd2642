"""The choice of experts within groups against sorting in 64 bits: numbers of experts around a warp's shares, groups of every kind, ties,
masked experts, values closer than float can tell, NaN.  The weights are a few float operations on numbers of at most one (an
exponential of 2 ulp, a sum of at most 1,024 terms by pairs of 32, a division): 64 half steps of them."""
import pytest
import torch

from head_decay_plain import F32, choose

pytestmark = pytest.mark.gpu

CASES = [  # E, k, groups, groups_use
    (1, 1, 1, 1), (2, 1, 1, 1), (31, 4, 1, 1), (32, 8, 4, 2), (30, 30, 1, 1), (31, 30, 1, 1), (33, 30, 1, 1), (60, 4, 5, 2), (64, 6, 8, 3), (100, 10, 10, 4), (128, 8, 32, 4),
    (160, 6, 8, 3), (256, 8, 8, 4), (257, 30, 1, 1), (512, 12, 16, 8), (1000, 20, 20, 3), (1024, 30, 2, 1), (48, 3, 3, 1), (96, 5, 32, 7)]


def _run(x, k, **how):
    from transformer_b200.parts import choose_experts
    idx = torch.full((x.shape[0], k), -7, dtype=torch.int32, device="cuda")
    w = torch.full((x.shape[0], k), 7.0, device="cuda")
    bias = how.pop("bias", None)
    choose_experts(x, idx, w, bias=None if bias is None else bias.cuda(), **how)
    return idx.cpu(), w.cpu()


def _compare(x, k, **how):
    idx, w = _run(x, k, **how)
    want, ww = choose(x.double().cpu(), k, **how)
    assert torch.equal(idx.long(), want), (idx.long() != want).any(1).nonzero()[:4]
    assert bool(((w.double() - ww).abs() <= 64 * F32 * ww.abs() + 1e-37).all()), float((w.double() - ww).abs().max())


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,k,groups,groups_use", CASES)
def test_choice(E, k, groups, groups_use, scores):
    for seed, nt in enumerate((1, 9, 70)):
        gen = torch.Generator().manual_seed(seed + E)
        x = torch.randn(nt, E + 3, generator=gen) * (3.0 if seed else 0.5)
        if seed == 2:
            x = x.bfloat16().float()                # equal logits in many rows
        x = x.cuda()[:, (1 if seed == 1 else 0):][:, :E] if seed < 2 else x[:, :E].contiguous().cuda()
        for bias in (None, torch.randn(E, generator=gen) * 0.1, torch.zeros(E)):
            for group_top in (1, 2):
                _compare(x, k, scores=scores, bias=bias, groups=groups, groups_use=groups_use, group_top=group_top,
                         renorm=(seed + group_top) % 2 == 0, scale=2.5 if seed else 1.0)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("group_top", [1, 2])
def test_values_closer_than_float_can_tell(scores, group_top):
    """Logits that differ by single steps of float, and biases that nearly make up for other differences."""
    gen = torch.Generator().manual_seed(5)
    E = 64
    x = torch.full((40, E), 1.25)
    x = (x.view(torch.int32) + torch.randint(0, 6, (40, E), generator=gen, dtype=torch.int32)).view(torch.float32)
    s = torch.sigmoid(x[0].double()) if scores == "sigmoid" else torch.softmax(x[0].double(), -1)
    for bias in (None, torch.zeros(E), (0.5 - s).float(), torch.randint(0, 2, (E,), generator=gen) * 1e-8):
        _compare(x.cuda(), 6, scores=scores, bias=bias, groups=8, groups_use=3, group_top=group_top)
        _compare(x.cuda(), 6, scores=scores, bias=bias, renorm=True)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_masked_experts(scores):
    """-inf masks: a few, all but two (fewer than are chosen), all; logits of the type's lowest value; far logits."""
    gen = torch.Generator().manual_seed(6)
    E, inf = 64, float("inf")
    x = torch.randn(6, E, generator=gen)
    x[0, :20] = -inf
    x[1, 2:] = -inf
    x[2] = -inf
    x[3, 5:] = torch.finfo(torch.float32).min
    x[4] = -80.0 - torch.arange(E)
    x[5, ::2] = 60.0
    for bias in (None, torch.rand(E, generator=gen)):
        for groups, use in ((1, 1), (8, 2)):
            for renorm in (False, True):
                how = dict(scores=scores, bias=bias, groups=groups, groups_use=use, group_top=2, renorm=renorm)
                _compare(x[:4].cuda(), 6, **how)
                idx, w = _run(x[4:].cuda(), 6, **how)          # scores that 64 bits tell apart by less than a step of themselves
                assert all(len(set(r)) == 6 for r in idx.tolist()) and bool(torch.isfinite(w).all())
    idx, w = _run(x[2:3].cuda(), 6, scores=scores, renorm=True)
    assert idx.tolist() == [[0, 1, 2, 3, 4, 5]] and bool((w == 0).all())


def test_far_logits_keep_their_ratios_when_renormalized():
    x = torch.tensor([[-120.0, -121.0, -300.0, -122.0]]).cuda()
    for scores in ("softmax", "sigmoid"):
        idx, w = _run(x, 2, scores=scores, renorm=True)
        e = torch.exp(torch.tensor([0.0, -1.0], dtype=torch.float64))
        assert idx.tolist() == [[0, 1]] and bool(((w.double() - e / e.sum()).abs() <= 64 * F32).all())


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 4])
def test_indices_differ_whatever_the_logits(scores, groups):
    gen = torch.Generator().manual_seed(7)
    values = torch.tensor([float("nan"), float("inf"), float("-inf"), 0.0, 3e38, -3e38])
    x = values[torch.randint(0, 6, (200, 40), generator=gen)]
    x[0], x[1] = float("nan"), float("inf")
    for bias in (None, torch.randn(40, generator=gen)):
        for top in (1, 2):
            idx, _ = _run(x.cuda(), 9, scores=scores, bias=bias, groups=groups, groups_use=1 if groups == 4 else groups, group_top=top)
            for row in idx.tolist():
                assert len(set(row)) == 9 and min(row) >= 0 and max(row) < 40
    one = torch.randn(3, 40, generator=gen)
    one[:, 7] = float("nan")
    idx, w = _run(one.cuda(), 9, scores="sigmoid")
    assert 7 not in idx.flatten().tolist() and bool(torch.isfinite(w).all())


def test_replayed_with_other_logits():
    from transformer_b200.parts import choose_experts
    gen = torch.Generator().manual_seed(8)
    xs = [torch.randn(50, 256, generator=gen) for _ in range(2)]
    x, idx, w = xs[0].cuda(), torch.empty(50, 8, dtype=torch.int32, device="cuda"), torch.empty(50, 8, device="cuda")
    how = dict(scores="sigmoid", groups=8, groups_use=4, group_top=2, renorm=True)
    graph = torch.cuda.CUDAGraph()
    choose_experts(x, idx, w, **how)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        choose_experts(x, idx, w, **how)
    for other in (xs[1], xs[0]):
        x.copy_(other)
        graph.replay()
        torch.cuda.synchronize()
        want, _ = choose(other.double(), 8, **how)
        assert torch.equal(idx.cpu().long(), want)


def test_no_tokens():
    _run(torch.empty(0, 16).cuda(), 4)
