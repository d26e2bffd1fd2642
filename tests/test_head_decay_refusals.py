"""What the linear attention with one decay for each head, the choice of experts within groups, and the parts made of them refuse, before
anything reaches a device."""
import pytest
import torch

from transformer_b200.parts import FEED_FORWARDS, MIXERS, choose_experts, decay_attention, decay_attention_step

F, B16 = torch.float32, torch.bfloat16


def _args(nt=6, H=4, G=2, dim=8, vdim=12, B=2, dtype=F):
    z = lambda *s, dt=dtype: torch.zeros(s, dtype=dt)
    return dict(q=z(nt, H, dim), k=z(nt, G, dim), v=z(nt, G, vdim), log_decay=z(nt, H, dt=F), state=z(3, H, dim, vdim, dt=F),
                slots=torch.zeros(B, dtype=torch.int32), out=z(nt, H, vdim))


BAD = [
    (dict(q=torch.zeros(6, 32)), "tokens, heads"), (dict(k=torch.zeros(6, 3, 8)), "share"), (dict(k=torch.zeros(5, 2, 8)), "k:"),
    (dict(v=torch.zeros(6, 4, 12)), "v:"), (dict(k=torch.zeros(6, 2, 8, dtype=B16)), "k:"), (dict(out=torch.zeros(6, 4, 12, dtype=B16)), "out:"),
    (dict(q=torch.zeros(6, 4, 8, dtype=torch.float16)), "float16"), (dict(q=torch.zeros(6, 8, 4).transpose(1, 2)), "q:"),
    (dict(out=torch.zeros(1, 4, 12).expand(6, 4, 12)), "out:"), (dict(log_decay=torch.zeros(6, 2)), "log_decay"),
    (dict(log_decay=torch.zeros(6, 4, dtype=torch.float64)), "log_decay"), (dict(log_decay=torch.zeros(4, 6).t()), "log_decay"),
    (dict(state=torch.zeros(3, 4, 12, 8)), "state"), (dict(state=torch.zeros(3, 4, 8, 12, dtype=B16)), "state"),
    (dict(state=torch.zeros(3, 4, 12, 8).transpose(2, 3)), "state"), (dict(state=torch.zeros(1, 4, 8, 12).expand(3, 4, 8, 12)), "state"),
    (dict(new_state=torch.zeros(2, 4, 8, 12)), "new_state"), (dict(new_state=torch.zeros(3, 4, 8, 11)), "new_state"),
    (dict(slots=torch.zeros(2, dtype=torch.int64)), "slots"), (dict(slots=torch.zeros(2, 1, dtype=torch.int32)), "slots"),
    (dict(norm=torch.ones(4, 12)), "together"), (dict(gate=torch.ones(6, 4, 12)), "together"),
    (dict(norm=torch.ones(4, 11), gate=torch.ones(6, 4, 12)), "norm"), (dict(norm=torch.ones(4, 12), gate=torch.ones(6, 4, 11)), "gate"),
    ({}, "current CUDA device"),
]


@pytest.mark.parametrize("change,what", BAD)
def test_operators_refuse(change, what):
    with pytest.raises(ValueError, match=what):
        decay_attention(seq_start=torch.zeros(3, dtype=torch.int32), **dict(_args(), **change))
    if not (change and "slots" in change):
        with pytest.raises(ValueError, match=what):
            decay_attention_step(**dict(_args(B=6), **change))


def test_wide_heads_are_refused():
    with pytest.raises(ValueError, match="256"):
        decay_attention(seq_start=torch.zeros(3, dtype=torch.int32), **_args(dim=257))
    with pytest.raises(ValueError, match="256"):
        decay_attention_step(**_args(vdim=260, B=6))


def test_more_rows_than_32_bits_count():
    """Of tensors that take no memory (on "meta")."""
    n, meta = 2 ** 31, lambda *s, dt=F: torch.empty(s, dtype=dt, device="meta")
    few = dict(q=meta(4, 1, 1), k=meta(4, 1, 1), v=meta(4, 1, 1), log_decay=meta(1), state=meta(n, 1, 1, 1), slots=meta(4, dt=torch.int32), out=meta(4, 1, 1))
    many = dict(few, q=meta(n, 1, 1), k=meta(n, 1, 1), v=meta(n, 1, 1), out=meta(n, 1, 1), state=meta(4, 1, 1, 1))
    for d in (few, many):
        with pytest.raises(ValueError, match="at most"):
            decay_attention(seq_start=meta(5, dt=torch.int32), **d)
        with pytest.raises(ValueError, match="at most"):
            decay_attention_step(**d)
    with pytest.raises(ValueError, match="at most"):
        choose_experts(meta(n, 1), meta(n, 1, dt=torch.int32), meta(n, 1))


LOGITS = dict(logits=torch.zeros(5, 16), index=torch.zeros(5, 4, dtype=torch.int32), weights=torch.zeros(5, 4))


@pytest.mark.parametrize("change,what", [
    (dict(scores="tanh"), "softmax"), (dict(groups=3), "groups"), (dict(groups=0), "groups"), (dict(groups=4, groups_use=5), "used"),
    (dict(groups=4, groups_use=0), "used"), (dict(group_top=3), "largest"), (dict(groups=8, groups_use=1), "per token"),
    (dict(logits=torch.zeros(5, 16, dtype=torch.float64)), "float32"), (dict(logits=torch.zeros(16, 5).t()), "contiguous"),
    (dict(logits=torch.zeros(1, 16).expand(5, 16)), "contiguous"), (dict(index=torch.zeros(5, 4, dtype=torch.int64)), "int32"),
    (dict(weights=torch.zeros(5, 3)), "contiguous"), (dict(index=torch.zeros(4, 5, dtype=torch.int32).t()), "contiguous"),
    (dict(bias=torch.zeros(15)), "bias"), (dict(bias=torch.zeros(16, dtype=B16)), "bias"), (dict(logits=torch.zeros(5, 2000)), "1024"),
    (dict(logits=torch.zeros(5, 990), groups=33), "groups"), ({}, "current CUDA device")])
def test_the_choice_refuses(change, what):
    with pytest.raises(ValueError, match=what):
        choose_experts(**dict(LOGITS, **change))


def test_more_choices_than_the_kernel_takes():
    with pytest.raises(ValueError, match="per token"):
        choose_experts(torch.zeros(5, 64), torch.zeros(5, 31, dtype=torch.int32), torch.zeros(5, 31))


MIXER = dict(width=32, heads=4, kv_heads=2, dim=8, vdim=12, eps=1e-6)
MOE = dict(width=32, di=16, nexp=16, nexp_use=4, scoring="grouped", groups=4, groups_use=2, group_top=2)


@pytest.mark.parametrize("change,what", [(dict(kv_heads=3), "share"), (dict(dim=300), "256"), (dict(vdim=300), "256"),
                                         (dict(decay="always"), "decay"), (dict(heads=0), "share")])
def test_the_mixer_refuses(change, what):
    with pytest.raises(ValueError, match=what):
        MIXERS.get("head_decay")(dict(MIXER, **change), F, torch.device("cpu"))


@pytest.mark.parametrize("change,what", [(dict(groups=5), "groups"), (dict(groups_use=5), "used"), (dict(scores="x"), "softmax"),
                                         (dict(nexp_use=9), "per token"), (dict(scoring="kept", correction=True), "correction")])
def test_the_experts_refuse(change, what):
    with pytest.raises(ValueError, match=what):
        FEED_FORWARDS.get("moe")(dict(MOE, **change), F, torch.device("cpu"))


def test_parameters():
    part = MIXERS.get("head_decay")(dict(MIXER, decay="input"), F, torch.device("cpu"))
    assert {n: p.shape for n, p in part.parameters().items()} == {
        "win": (4 * 8 + 2 * 8 + 2 * 12 + 4 * 12, 32), "rate": (4,), "norm": (12,), "wo": (32, 48), "wa": (4, 32), "bias": (4,)}
    assert part.state_need().shape == (4, 8, 12) and part.graph_safe and part.launches_only
    part = FEED_FORWARDS.get("moe")(dict(MOE, correction=True), F, torch.device("cpu"))
    assert part.parameters()["correction"].shape == (16,) and part.norm_tail(None, 1) is None
