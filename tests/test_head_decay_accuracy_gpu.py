"""How far the linear attention's outputs are off their recurrence in 64 bits, as the operators' documentation has it: a rounding at the end, and in
bfloat16 prompts on the tensor cores one more of each term.

A rounding of the result alone is what 64 bits rounded to the type are off.  On the tensor cores each term of an output meets one of two more
roundings of the same relative size (its weight's, or the state's that its segment starts with).  Over terms of random signs the norm of
their errors has to that of the output the ratio that a rounding has to its value, so both together are off by the square root of two times
the rounding alone; 1.5 leaves 6 %.  Elsewhere float's 2^-24 of a few hundred terms, 2^-17 at most to bfloat16's 2^-8, adds under 1 %."""
import pytest
import torch

from head_decay_plain import normed, recurrence
from test_head_decay_gpu import EPS, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dim,vdim,lens,most", [(128, 128, [700, 300], 1.5), (64, 64, [300, 65], 1.5), (128, 256, [400], 1.5),
                                                 (64, 64, [50], 1.01), (17, 33, [300], 1.01), (128, 128, "single", 1.01)])
def test_outputs_against_a_rounding(dim, vdim, lens, most, gated):
    from transformer_b200.parts import decay_attention, decay_attention_step
    single, f = lens == "single", lambda t: t.double().cpu()
    lens = [1] * 40 if single else lens
    d, more, starts = _inputs(torch.bfloat16, 4, 2, dim, vdim, lens, "input", gated, dim + vdim, behind=0)
    state0 = d["state"].clone()
    if single:
        decay_attention_step(**d, **more)
    else:
        decay_attention(seq_start=starts, **d, **more)
    parts, at = [], 0
    for b, n in enumerate(lens):
        rows = slice(at, at + n)
        o, _, _, _ = recurrence(f(d["q"][rows]), f(d["k"][rows]), f(d["v"][rows]), f(d["log_decay"][rows]), f(state0[int(d["slots"][b])]), dim ** -0.5)
        parts.append(normed(o, torch.zeros_like(o), f(more["norm"]), f(more["gate"][rows]), EPS, torch.bfloat16)[0] if gated else o)
        at += n
    exact = torch.cat(parts)
    rounding = float((exact.bfloat16().double() - exact).norm())
    off = float((f(d["out"]) - exact).norm())
    assert off <= most * rounding, (off / rounding, rounding / float(exact.norm()))
