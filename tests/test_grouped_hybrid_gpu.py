"""A model of layers with a linear attention (one decay a head) and experts chosen within groups, registered here and run through the
engine: ragged prompts, pieces of them and single tokens (captured and replayed) against the plain model in 64 bits, and generation."""
import dataclasses

import pytest
import torch

import transformer_b200 as tb
from head_decay_plain import choose, recurrence
from transformer_b200.architectures.generic import plan_from_spec
from transformer_b200.config.registry import Architecture, register_architecture, unregister_architecture
from transformer_b200.parts import LayerSpec, ModelSpec, PartSpec, RunEntry

pytestmark = pytest.mark.gpu
EPS = 1e-5


@dataclasses.dataclass(frozen=True)
class Config:
    width: int = 64
    vocab: int = 90
    context: int = 512
    dim: int = 64
    vdim: int = 64

    @classmethod
    def from_dict(cls, c):
        return cls(**{k: v for k, v in c.items() if k != "model_type"})

    def to_dict(self):
        return {"model_type": "toy_hybrid", **dataclasses.asdict(self)}


def _spec(c):
    norm = PartSpec.of("rmsnorm", width=c.width, eps=EPS)
    moe = dict(width=c.width, di=32, nexp=16, nexp_use=4, scoring="grouped", groups=4, groups_use=2)
    first = LayerSpec(PartSpec.of("head_decay", width=c.width, heads=4, kv_heads=2, dim=c.dim, vdim=c.vdim, decay="input", eps=EPS),
                      PartSpec.of("moe", scores="sigmoid", correction=True, group_top=2, renorm=True, weight_scale=2.0, **moe), norm, norm)
    second = LayerSpec(PartSpec.of("head_decay", width=c.width, heads=2, dim=c.dim, vdim=c.vdim, eps=EPS),
                       PartSpec.of("moe", scores="softmax", shared_di=24, **moe), norm, norm)
    return ModelSpec(width=c.width, vocab=c.vocab, max_context=c.context, layers=(first, second), order=tuple(RunEntry(i) for i in (0, 1, 0, 1)),
                     embedding=PartSpec.of("lookup", vocab=c.vocab, width=c.width), final_norm=norm,
                     head=PartSpec.of("linear", vocab=c.vocab, width=c.width, tied=True))


@pytest.fixture()
def registered():
    yield register_architecture(Architecture("toy_hybrid", Config, _spec, lambda c: plan_from_spec(_spec(c))))
    unregister_architecture("toy_hybrid")


def _plain(engine, ids):
    """Logits of every token of one sequence, in 64 bits, from the engine's weights."""
    f = lambda t: t.double().cpu()
    rms = lambda x, w: x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * f(w)
    glu = lambda x, w: (lambda z: z[:, : z.shape[1] // 2] * torch.sigmoid(z[:, : z.shape[1] // 2]) * z[:, z.shape[1] // 2:])(x @ f(w).T)
    x = f(engine.embedding)[ids]
    for entry in engine.spec.order:
        layer = engine.layers[entry.layer]
        spec = engine.spec.layers[entry.layer]
        parts = layer.parts()
        norms = [p for n, p in parts.items() if "norm" in n]
        m, e = layer.mixer, parts["feed_forward"]
        w = m.weights
        y = rms(x, next(iter(norms[0].weights.values())))
        q, k, v, gate = (y @ f(w["win"]).T).split(m.widths, dim=1)
        if spec.mixer.get().get("decay") == "input":
            g = -torch.exp(f(w["rate"])) * torch.nn.functional.softplus(y @ f(w["wa"]).T + f(w["bias"]))
        else:
            g = -torch.exp(f(w["rate"])).expand(len(ids), m.H)
        heads = lambda t, n: t.unflatten(1, (n, -1))
        o = recurrence(heads(q, m.H), heads(k, m.G), heads(v, m.G), g, torch.zeros(m.H, m.dim, m.vdim, dtype=torch.float64), m.dim ** -0.5)[0]
        o = o / (o.square().mean(-1, keepdim=True) + EPS).sqrt() * f(w["norm"]).view(m.H, m.vdim) * heads(gate * torch.sigmoid(gate), m.H)
        x = x + o.flatten(1) @ f(w["wo"]).T
        y = rms(x, next(iter(norms[1].weights.values())))
        w, how = e.weights, dict(e.choice)
        idx, weights = choose(y @ f(w["router"]).T, e.k, bias=f(w["correction"]) if "correction" in w else None, **how)
        out = torch.zeros_like(x)
        for t in range(len(ids)):
            for j in range(e.k):
                out[t] += weights[t, j] * (glu(y[t:t + 1], w["wgu"][idx[t, j]]) @ f(w["wd"][idx[t, j]]).T)[0]
        if e.shared:
            out = out + torch.sigmoid(y @ f(w["shared_gate"]).T) * (glu(y, w["shared_wgu"]) @ f(w["shared_wd"]).T)
        x = x + out
    x = rms(x, next(iter(engine.final_norm.weights.values())))
    return x @ f(engine.head).T


@pytest.mark.parametrize("dim,vdim", [(64, 64), (128, 128), (24, 40)])
def test_the_model_in_32_bits(registered, tmp_path, dim, vdim):
    """2e-4 of the largest logit: eight parts of some hundred float roundings each on activations of size one, as for the other designs."""
    folder = tb.write_random_model(str(tmp_path / "m"), Config(dim=dim, vdim=vdim).to_dict(), seed=2, std=0.2)
    engine = tb.load(folder, dtype="float32", max_tokens=1024)
    g = torch.Generator().manual_seed(0)
    seqs = [torch.randint(0, 90, (n,), generator=g).tolist() for n in (150, 71, 9)]
    want = [_plain(engine, s) for s in seqs]
    slots = [engine.open() for _ in seqs]
    cuts = ([100, 64, 1], [140, 65, 3])             # prompts, pieces, then one token each
    got, at = [[] for _ in seqs], [0, 0, 0]
    for cut in cuts:
        pieces = [s[a:b] for s, a, b in zip(seqs, at, cut)]
        out = engine.step(slots, pieces, [list(range(len(p))) for p in pieces]).cpu().split([len(p) for p in pieces])
        for i in range(3):
            got[i].append(out[i])
        at = list(cut)
    for j in range(6):
        out = engine.step(slots, [[s[a + j]] for s, a in zip(seqs, at)]).cpu().clone()
        for i in range(3):
            got[i].append(out[i:i + 1])
    assert 3 in engine._graphs, "single tokens are captured and replayed"
    for i in range(3):
        mine, ref = torch.cat(got[i]).double(), want[i][: at[i] + 6]
        assert float((mine - ref).abs().max()) <= 2e-4 * float(ref.abs().max()), i


@pytest.mark.parametrize("dim,vdim", [(64, 64), (128, 128)])
def test_the_model_in_bfloat16(registered, tmp_path, dim, vdim):
    """Whole, in pieces and token by token agree within a few bfloat16 roundings of eight parts (2^-4 of the logits' norm: the choice of an
    expert may turn with them), nothing of one sequence reaches another, and generation runs."""
    folder = tb.write_random_model(str(tmp_path / "m"), Config(dim=dim, vdim=vdim).to_dict(), seed=2, std=0.1)
    engine = tb.load(folder, dtype="bfloat16", max_tokens=2048)
    g = torch.Generator().manual_seed(0)
    a, b = (torch.randint(0, 90, (n,), generator=g).tolist() for n in (300, 130))
    s = engine.open()
    whole = engine.step([s], [a], [list(range(300))]).cpu().clone()
    engine.close(s)
    two = [engine.open(), engine.open()]
    both = engine.step(two, [a, b], [list(range(300)), [0]]).cpu()[:300].clone()
    for s in two:
        engine.close(s)
    assert float((whole - both).norm()) <= 2.0 ** -4 * float(whole.norm())
    s = engine.open()
    parts = [engine.step([s], [a[:129]], [list(range(129))]).cpu(), engine.step([s], [a[129:290]], [list(range(161))]).cpu()]
    parts += [engine.step([s], [[t]]).cpu().clone() for t in a[290:]]
    engine.close(s)
    assert float((whole - torch.cat(parts)).norm()) <= 2.0 ** -4 * float(whole.norm())
    out = tb.generate(engine, [a[:70], b[:1], b], max_steps=5, stop_tokens=()).tokens
    assert [len(t) for t in out] == [5, 5, 5]
    engine.check_kernels()
