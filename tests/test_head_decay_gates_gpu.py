"""The linear attention's gate at the ends of its type: a gate far below zero closes its channel, in a prompt as for a single token; -inf times
the sigmoid's 0 is no number, +inf is the infinity of its sign, NaN stays NaN."""
import math

import pytest
import torch

from head_decay_plain import bounds, normed, recurrence
from test_head_decay_gpu import EPS, _inputs

pytestmark = pytest.mark.gpu
# below -80 a kernel may answer anything between z e^z and 0
NEXT_TO_NOTHING = 80.0 * math.exp(-80.0)


def _gates(shape, dtype, seed):
    lowest = torch.finfo(dtype).min
    values = torch.tensor([lowest, lowest / 2, -1e34, -1e30, -1e4, -100.0, -89.0, -81.0, -80.0, -79.5, -20.0, 0.0, 30.0, 200.0, 1e30,
                           float("inf"), float("-inf"), float("nan")])
    gen = torch.Generator().manual_seed(seed)
    special = values[torch.randint(0, len(values), shape, generator=gen)]
    return torch.where(torch.rand(shape, generator=gen) < 0.4, special, torch.randn(shape, generator=gen)).to(dtype).cuda()


def _hold(got, o, off, norm, gate, dtype):
    y, bound = normed(o, off, norm, gate, EPS, dtype)
    rms = (o.square().mean(-1, keepdim=True) + EPS).sqrt()
    bound = bound + torch.where(gate < -79.0, NEXT_TO_NOTHING * (o / rms * norm).abs(), 0.0)
    assert torch.equal(got.isnan(), y.isnan()), "what is no number"
    # an infinity has the sign of o, which an o that may be off by `off` has only where it is larger than that
    sure = y.isinf() & (o.abs() > off)
    assert bool(got[y.isinf()].isinf().all()) and torch.equal(got[sure], y[sure]) and int(sure.sum()) * 2 >= int(y.isinf().sum())
    fine = y.isfinite()
    assert bool(((got - y).abs() <= bound)[fine].all()), float(((got - y).abs() / bound)[fine].max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim,vdim", [(128, 128), (64, 64), (128, 256), (24, 40), (17, 33)])
def test_gates_at_the_ends_of_their_type(dtype, dim, vdim):
    from transformer_b200.csrc import lib
    from transformer_b200.parts import decay_attention, decay_attention_step
    f = lambda t: t.double().cpu()
    for lens in ([130, 40], [20]):
        d, more, starts = _inputs(dtype, 2, 1, dim, vdim, lens, "input", True, dim + len(lens))
        more["gate"] = _gates((d["out"].shape[0], 2, vdim), dtype, vdim)
        state0, scale = d["state"].clone(), dim ** -0.5
        decay_attention(seq_start=starts, **d, **more)
        assert not lib.gemm_tc_status()
        at = 0
        for b, n in enumerate(lens):
            rows = slice(at, at + n)
            o, _, size, _ = recurrence(f(d["q"][rows]), f(d["k"][rows]), f(d["v"][rows]), f(d["log_decay"][rows]), f(state0[int(d["slots"][b])]), scale)
            off = bounds(o, size, torch.float32, dim, n, dtype == torch.bfloat16)
            _hold(f(d["out"][rows]), o, off, f(more["norm"]), f(more["gate"][rows]), dtype)
            at += n
    # single tokens of 5 sequences
    d, more, _ = _inputs(dtype, 2, 1, dim, vdim, [1] * 5, "input", True, dim, behind=0)
    more["gate"] = _gates((5, 2, vdim), dtype, vdim + 1)
    state0 = d["state"].clone()
    decay_attention_step(**d, **more)
    for b in range(5):
        rows = slice(b, b + 1)
        o, _, size, _ = recurrence(f(d["q"][rows]), f(d["k"][rows]), f(d["v"][rows]), f(d["log_decay"][rows]), f(state0[int(d["slots"][b])]), scale)
        _hold(f(d["out"][rows]), o, bounds(o, size, torch.float32, dim, 1, False), f(more["norm"]), f(more["gate"][rows]), dtype)
