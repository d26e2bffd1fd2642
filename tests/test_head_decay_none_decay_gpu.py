"""A decay that is no number: it takes its head's state and the outputs from its token on, and nothing before it, of another head or of
another sequence, whichever kernels a call is given to."""
import pytest
import torch

from test_head_decay_gpu import _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim,vdim", [(128, 128), (64, 64), (17, 33)])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("at", [0, 1, 30, 31, 32, 127, 128, 150, 255, 256, 290, 399])
def test_outputs_before_it_keep_their_bits(dtype, dim, vdim, gated, at):
    from transformer_b200.parts import decay_attention
    n, outs = 400, []
    for value in (-0.3, float("nan")):
        d, more, starts = _inputs(dtype, 2, 2, dim, vdim, [n, 40], "input", gated, 1)
        d["log_decay"][at, 0] = value
        decay_attention(seq_start=starts, **d, **more)
        outs.append((d["out"][:n + 40].float().cpu(), d["state"][d["slots"].long()].cpu()))
    (good, good_S), (got, got_S) = outs
    assert bool(torch.isfinite(good).all()) and bool(torch.isfinite(good_S).all())
    assert bool(got[at:n, 0].isnan().all()) and bool(got_S[0, 0].isnan().all())
    got[at:n, 0], got_S[0, 0] = good[at:n, 0], good_S[0, 0]
    assert torch.equal(good, got) and torch.equal(good_S, got_S)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("at", [0, 7, 31, 32, 39])
def test_a_short_step(dtype, at):
    from transformer_b200.parts import decay_attention
    n, outs = 40, []
    for value in (-0.3, float("nan")):
        d, _, starts = _inputs(dtype, 2, 2, 64, 64, [n], "input", False, 1)
        d["log_decay"][at, 0] = value
        decay_attention(seq_start=starts, **d)
        outs.append((d["out"][:n].float().cpu(), d["state"][d["slots"].long()].cpu()))
    (good, good_S), (got, got_S) = outs
    assert bool(got[at:, 0].isnan().all()) and bool(got_S[0, 0].isnan().all())
    got[at:, 0], got_S[0, 0] = good[at:, 0], good_S[0, 0]
    assert torch.equal(good, got) and torch.equal(good_S, got_S)
