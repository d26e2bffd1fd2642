"""The linear attention with a norm and a gate of no tokens at all: the sequences keep their states, single tokens of no sequence are nothing."""
import pytest
import torch

from test_head_decay_gpu import _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim,vdim", [(128, 128), (64, 64), (17, 33)])
@pytest.mark.parametrize("decay", ["input", "fixed"])
def test_no_rows_of_a_gate(dtype, dim, vdim, decay):
    from transformer_b200.parts import decay_attention, decay_attention_step
    for of in (0, 4):           # tensors of no rows, and slices of tensors that have some
        d, more, starts = _inputs(dtype, 2, 1, dim, vdim, [0, 0, 0], decay, True, 1, behind=of)
        for name in ("q", "k", "v", "out") + (("log_decay",) if decay == "input" else ()):
            d[name] = d[name][:0]
        more["gate"] = more["gate"][:0]
        new = torch.full_like(d["state"], 5.0)
        decay_attention(seq_start=starts, new_state=new, **d, **more)
        for slot in range(5):
            assert torch.equal(new[slot], d["state"][slot] if slot in d["slots"].tolist() else torch.full_like(new[slot], 5.0))
        before = new.clone()
        none = dict(d, slots=d["slots"][:0])
        decay_attention(seq_start=starts[:1], new_state=new, **none, **more)
        decay_attention_step(new_state=new, **none, **more)
        assert torch.equal(new, before)
