"""The linear attention with one decay for each head against its recurrence in 64 bits: prompts around the edges of segments and tiles,
sequences of no token and of one, shared heads, odd sizes, slices of wider rows, decays from none to all, and single tokens."""
import pytest
import torch

from head_decay_plain import bounds, normed, recurrence, state_bounds

pytestmark = pytest.mark.gpu
EPS = 1e-6


def _inputs(dtype, H, G, dim, vdim, lens, decay, gated, seed, slots=None, behind=3):
    gen = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(s, generator=gen)
    B, nt = len(lens), sum(lens) + behind
    widths = [H * dim, G * dim, G * vdim, H * vdim]
    z = torch.zeros(nt, sum(widths) + 8)
    z[:, :sum(widths)] = randn(nt, sum(widths))
    z = z.to(dtype).cuda()
    q, k, v, gate = z[:, :sum(widths)].split(widths, dim=1)
    if decay == "fixed":
        g = -torch.exp2(-8.0 * torch.rand(H, generator=gen))
    elif decay == "strong":             # from no decay at all to one that forgets everything
        g = torch.tensor([0.0, -1e-4, -0.3, -20.0, -90.0, -300.0, float("-inf")])[torch.randint(0, 7, (nt, H), generator=gen)]
    else:
        g = -torch.nn.functional.softplus(randn(nt, H) * 2 - 2)
    slots = torch.randperm(B + 2, generator=gen)[:B] if slots is None else slots
    state = randn(B + 2, H, dim, vdim + 4)[..., :vdim].contiguous()
    state[slots[: B // 2]] = 0.0
    heads = lambda t, n: t.unflatten(1, (n, -1))
    d = {"q": heads(q, H), "k": heads(k, G), "v": heads(v, G), "log_decay": g.cuda(), "state": state.cuda(),
         "slots": slots.int().cuda(), "out": torch.full((nt, H, vdim), 7.0, dtype=dtype, device="cuda")}
    more = {"norm": (1.0 + 0.1 * randn(H, vdim)).cuda(), "gate": heads(gate, H), "eps": EPS} if gated else {}
    return d, more, torch.tensor([0] + list(lens)).cumsum(0).int().cuda()


def _check(d, more, lens, new_state, dtype, tensor_cores, state0, scale=None, untouched=True):
    H, dim, vdim = d["q"].shape[1], d["q"].shape[2], d["v"].shape[2]
    scale = dim ** -0.5 if scale is None else scale
    at, f = 0, lambda t: t.double().cpu()
    g = f(d["log_decay"])
    g = g if g.dim() == 2 else g.expand(d["q"].shape[0], H)
    for b, n in enumerate(lens):
        rows, slot = slice(at, at + n), int(d["slots"][b])
        o, S, size, M = recurrence(f(d["q"][rows]), f(d["k"][rows]), f(d["v"][rows]), g[rows], f(state0[slot]), scale)
        off = bounds(o, size, torch.float32 if more else dtype, dim, n, tensor_cores)
        if more:
            o, off = normed(o, off, f(more["norm"]), f(more["gate"][rows]), EPS, dtype)
        got = f(d["out"][rows])
        assert bool(((got - o).abs() <= off).all()), (b, n, float(((got - o).abs() / off).max()))
        err = (f(new_state[slot]) - S).abs()
        assert bool((err <= state_bounds(M, dim, n, tensor_cores)).all()), (b, n, float((err / state_bounds(M, dim, n, tensor_cores)).max()))
        at += n
    if not untouched:
        return
    assert bool((d["out"][at:] == 7.0).all()), "rows behind the last sequence"
    named = set(d["slots"].tolist())
    for slot in set(range(state0.shape[0])) - named:
        assert torch.equal(new_state[slot], state0[slot] if new_state is d["state"] else torch.full_like(state0[slot], 5.0))


SHAPES = [  # H, G, dim, vdim
    (2, 2, 128, 128), (4, 2, 64, 64), (3, 1, 128, 64), (2, 1, 64, 128), (2, 2, 80, 96), (1, 1, 256, 256), (3, 3, 17, 33), (1, 1, 1, 1),
    (2, 1, 128, 256), (2, 2, 96, 130), (2, 2, 8, 8), (2, 1, 16, 24), (2, 2, 72, 72), (1, 1, 40, 136)]


@pytest.mark.parametrize("decay", ["input", "fixed", "strong"])
@pytest.mark.parametrize("H,G,dim,vdim", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompts(dtype, H, G, dim, vdim, decay):
    from transformer_b200.csrc import lib
    from transformer_b200.parts import decay_attention
    for seed, lens in enumerate(([1], [64, 0, 65], [127, 1, 128, 129, 3], [300, 511, 70])):
        gated = (seed + H + dim) % 2 == 1
        d, more, starts = _inputs(dtype, H, G, dim, vdim, lens, decay, gated, seed)
        state0 = d["state"].clone()
        new = torch.full_like(d["state"], 5.0) if seed % 2 else None
        decay_attention(seq_start=starts, new_state=new, **d, **more)
        assert not lib.gemm_tc_status()
        if new is not None:
            assert torch.equal(d["state"], state0)
        _check(d, more, lens, d["state"] if new is None else new, dtype, dtype == torch.bfloat16, state0)


@pytest.mark.parametrize("H,G,dim,vdim", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_steps(dtype, H, G, dim, vdim):
    from transformer_b200.parts import decay_attention_step
    for seed, (B, decay) in enumerate(((1, "input"), (5, "fixed"), (7, "strong"))):
        gated = seed % 2 == 0
        d, more, _ = _inputs(dtype, H, G, dim, vdim, [1] * B, decay, gated, seed, behind=0)
        state0 = d["state"].clone()
        new = torch.full_like(d["state"], 5.0) if seed % 2 else None
        decay_attention_step(new_state=new, scale=0.3, **d, **more)
        _check(d, more, [1] * B, d["state"] if new is None else new, dtype, False, state0, scale=0.3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_long_sequence_in_pieces_and_whole(dtype):
    """2,500 tokens at once, in three prompts and the last few one by one: the same states and outputs, all within the bounds."""
    from transformer_b200.csrc import lib
    from transformer_b200.parts import decay_attention, decay_attention_step
    H, G, dim, vdim, n = 2, 1, 128, 128, 2500
    d, more, starts = _inputs(dtype, H, G, dim, vdim, [n], "input", False, 3, slots=torch.tensor([1]))
    state0 = d["state"].clone()
    decay_attention(seq_start=starts, **d)
    assert not lib.gemm_tc_status()
    _check(d, more, [n], d["state"], dtype, dtype == torch.bfloat16, state0)
    whole, d["state"] = d["out"].clone(), state0.clone()
    d["out"].fill_(7.0)
    cut = lambda a, b: {x: d[x][a:b] for x in ("q", "k", "v", "log_decay", "out")}
    for a, b in ((0, 1000), (1000, 1001), (1001, n - 3)):
        decay_attention(seq_start=torch.tensor([0, b - a], dtype=torch.int32, device="cuda"), state=d["state"], slots=d["slots"], **cut(a, b))
    for t in range(n - 3, n):
        decay_attention_step(state=d["state"], slots=d["slots"], **cut(t, t + 1))
    _check(d, more, [n], d["state"], dtype, dtype == torch.bfloat16, state0)
    assert float((whole[:n].float() - d["out"][:n].float()).norm()) <= 0.01 * float(whole[:n].float().norm())


def test_many_sequences_and_portions_of_heads(monkeypatch):
    """150 short sequences (their segments are found 32 guesses at a time), with scratch for one head at a time: the same bits."""
    from transformer_b200.csrc import lib
    from transformer_b200.parts import decay_attention, head_decay
    lens = [(3, 0, 70, 1, 130)[i % 5] for i in range(150)]
    for dtype in (torch.float32, torch.bfloat16):
        outs = []
        for most in (head_decay.WORK_BYTES, 1):
            monkeypatch.setattr(head_decay, "WORK_BYTES", most)
            d, more, starts = _inputs(dtype, 4, 2, 64, 64, lens, "input", True, 9)
            state0 = d["state"].clone()
            decay_attention(seq_start=starts, **d, **more)
            assert not lib.gemm_tc_status()
            outs.append((d["out"].clone(), d["state"].clone()))
        _check(d, more, lens, d["state"], dtype, dtype == torch.bfloat16, state0)
        assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


@pytest.mark.parametrize("dim,vdim", [(128, 128), (64, 128), (128, 64), (128, 256), (64, 64)])
def test_many_heads_behind_one_another(dim, vdim):
    """More heads and sequences than the GPU has places for blocks: a block goes through several heads.  One head at a time has the same
    bits; some are looked at in 64 bits."""
    from transformer_b200.csrc import lib
    from transformer_b200.parts import decay_attention
    H, G, lens = 11, 11, [(1, 130, 300, 0, 257, 128)[i % 6] for i in range(100)]
    d, more, starts = _inputs(torch.bfloat16, H, G, dim, vdim, lens, "input", True, 2)
    state0 = d["state"].clone()
    decay_attention(seq_start=starts, **d, **more)
    assert not lib.gemm_tc_status()
    out, state = d["out"].clone(), d["state"].clone()
    d["state"].copy_(state0)
    for h in range(H):
        one = {n: d[n][:, h:h + 1] for n in ("q", "k", "v", "out")}
        S = d["state"][:, h:h + 1].clone()
        decay_attention(state=S, slots=d["slots"], seq_start=starts, log_decay=d["log_decay"][:, h:h + 1].contiguous(),
                        norm=more["norm"][h:h + 1], gate=more["gate"][:, h:h + 1], eps=EPS, **one)
        assert torch.equal(S, state[:, h:h + 1])
    assert not lib.gemm_tc_status() and torch.equal(d["out"], out)
    d["out"], d["state"] = out[: sum(lens[:6])], state
    _check(d, {**more, "gate": more["gate"][: sum(lens[:6])]}, lens[:6], state, torch.bfloat16, True, state0, untouched=False)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim,vdim", [(128, 128), (64, 64), (80, 96)])
def test_what_is_no_number_stays_behind_its_token(dtype, dim, vdim, bad):
    """One value channel of one token, and later one key of another head, are no numbers: the outputs before those tokens, and of the
    other channels and heads, keep their bits."""
    from transformer_b200.parts import decay_attention
    H, n, at, channel, at_k = 2, 400, 150, 5, 290
    outs = []
    for value in (0.5, bad):
        d, _, starts = _inputs(dtype, H, H, dim, vdim, [n], "input", False, 1)
        d["state"].zero_()
        d["v"][at, 0, channel] = value
        d["k"][at_k, 1, 3] = value
        decay_attention(seq_start=starts, **d)
        outs.append((d["out"][:n].float().cpu(), d["state"][int(d["slots"][0])].cpu()))
    (good, good_S), (got, got_S) = outs
    assert bool(torch.isfinite(good).all())
    assert not bool(torch.isfinite(got[at:, 0, channel]).any()) and not bool(torch.isfinite(got[at_k:, 1]).any())
    got[at:, 0, channel], got[at_k:, 1] = good[at:, 0, channel], good[at_k:, 1]
    assert torch.equal(good, got)
    assert not bool(torch.isfinite(got_S[0, :, channel]).any()) and not bool(torch.isfinite(got_S[1, 3]).any())
    got_S[0, :, channel], got_S[1, 3] = good_S[0, :, channel], good_S[1, 3]
    assert torch.equal(good_S, got_S)


def test_what_is_no_number_in_a_gated_row():
    """With the norm a row of a head that has one is none as a whole; the rows before it and the other head keep their bits."""
    from transformer_b200.parts import decay_attention
    n, at, outs = 400, 150, []
    for value in (0.5, float("inf")):
        d, more, starts = _inputs(torch.bfloat16, 2, 2, 128, 128, [n], "input", True, 1)
        d["state"].zero_()
        d["v"][at, 0, 5] = value
        decay_attention(seq_start=starts, **d, **more)
        outs.append(d["out"][:n].float().cpu())
    good, got = outs
    assert bool(torch.isfinite(good).all()) and not bool(torch.isfinite(got[at:, 0]).any())
    got[at:, 0] = good[at:, 0]
    assert torch.equal(good, got)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim,vdim", [(128, 128), (64, 64), (17, 33)])
def test_no_tokens_and_no_sequences(dtype, dim, vdim):
    from transformer_b200.parts import decay_attention, decay_attention_step
    d, _, starts = _inputs(dtype, 2, 1, dim, vdim, [0, 0, 0], "input", False, 1, behind=0)
    new = torch.full_like(d["state"], 5.0)
    decay_attention(seq_start=starts, new_state=new, **d)
    for slot in range(5):
        assert torch.equal(new[slot], d["state"][slot] if slot in d["slots"].tolist() else torch.full_like(new[slot], 5.0))
    before = new.clone()
    none = dict(d, slots=d["slots"][:0])
    decay_attention(seq_start=starts[:1], new_state=new, **none)
    decay_attention_step(new_state=new, **none)
    assert torch.equal(new, before)


@pytest.mark.parametrize("shift,pitch", [(1, 0), (0, 3), (4, 4)])
@pytest.mark.parametrize("dim,vdim", [(128, 128), (64, 64), (24, 40)])
def test_rows_that_are_not_whole_16_byte_pieces(dim, vdim, shift, pitch):
    """bfloat16 rows that begin anywhere, an odd distance apart, and states with a slot pitch: what the TMA copies do not take."""
    from transformer_b200.parts import decay_attention, decay_attention_step
    H, lens = 2, [70, 3, 129]
    d, more, starts = _inputs(torch.bfloat16, H, H, dim, vdim, lens, "input", True, 8)
    for n in ("q", "k", "v", "out"):
        wide = torch.zeros(d[n].shape[0], H * d[n].shape[2] + 16 + pitch, dtype=torch.bfloat16, device="cuda")
        view = wide[:, shift:shift + H * d[n].shape[2]].unflatten(1, (H, -1))
        view.copy_(d[n])
        d[n] = view
    wide = torch.zeros(d["state"].shape[0], H * dim * vdim + pitch, device="cuda")
    state = wide[:, :H * dim * vdim].unflatten(1, (H, dim, vdim))
    state.copy_(d["state"])
    state0, d["state"] = d["state"], state
    decay_attention(seq_start=starts, **d, **more)
    _check(d, more, lens, d["state"], torch.bfloat16, True, state0)
    state.copy_(state0)
    d["out"].fill_(7.0)
    cut = {n: d[n][:3] for n in ("q", "k", "v", "log_decay", "out")}
    decay_attention_step(state=d["state"], slots=d["slots"], norm=more["norm"], gate=more["gate"][:3], eps=EPS, **cut)
    _check({**d, **cut}, {**more, "gate": more["gate"][:3]}, [1, 1, 1], d["state"], torch.bfloat16, False, state0)


def test_sequences_whose_numbers_are_out_of_range_are_left_alone():
    """Bounds and slots outside the tensors: nothing of those sequences is read or written, the others are done."""
    from transformer_b200.parts import decay_attention, decay_attention_step
    for dtype in (torch.float32, torch.bfloat16):
        lens = [70, 40, 30]
        d, _, starts = _inputs(dtype, 2, 2, 128, 128, lens, "input", False, 4, slots=torch.tensor([1, 0, 3]))
        state0, want = d["state"].clone(), None
        decay_attention(seq_start=starts, **d)
        want, want_S = d["out"].clone(), d["state"].clone()
        for slots, bounds_ in (([1, 99, 3], [0, 70, 110, 140]), ([1, -1, 3], [0, 70, 110, 140]), ([1, 0, 3], [0, 70, 110, 1 << 30])):
            d["state"].copy_(state0)
            d["out"].fill_(7.0)
            d["slots"] = torch.tensor(slots, dtype=torch.int32, device="cuda")
            decay_attention(seq_start=torch.tensor(bounds_, dtype=torch.int32, device="cuda"), **d)
            left = 1 if slots[1] != 0 else 2
            rows = slice(70, 110) if left == 1 else slice(110, 140)
            assert bool((d["out"][rows] == 7.0).all())
            keep = torch.ones(140, dtype=torch.bool)
            keep[rows] = False
            assert torch.equal(d["out"][:140][keep], want[:140][keep])
            S = want_S.clone()
            S[[0] if left == 1 else [3]] = state0[[0] if left == 1 else [3]]
            assert torch.equal(d["state"], S)
        d["state"].copy_(state0)
        d["slots"] = torch.tensor([1, 99, -5], dtype=torch.int32, device="cuda")
        d["out"].fill_(7.0)
        step = {x: d[x][:3] for x in ("q", "k", "v", "log_decay", "out")}
        decay_attention_step(state=d["state"], slots=d["slots"], **step)
        assert bool((d["out"][1:] == 7.0).all()) and not bool((d["out"][0] == 7.0).all())
        assert torch.equal(d["state"][[0, 2, 3, 4]], state0[[0, 2, 3, 4]])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_and_replayed_and_on_another_stream(dtype):
    """Both operators in one captured graph, replayed with other inputs, and run on a stream of their own, give the bits of eager calls."""
    from transformer_b200.parts import decay_attention, decay_attention_step
    make = lambda seed: _inputs(dtype, 4, 2, 128, 128, [130, 64, 7], "input", True, seed, slots=torch.tensor([4, 0, 2]), behind=0)
    d, more, starts = make(1)
    step = {x: d[x][:3] for x in ("q", "k", "v", "log_decay")}
    step_out, step_more = torch.zeros_like(d["out"][:3]), dict(more, gate=more["gate"][:3])

    def both():
        decay_attention(seq_start=starts, **d, **more)
        decay_attention_step(state=d["state"], slots=d["slots"], out=step_out, **step, **step_more)

    def fresh(seed):
        e, m, _ = make(seed)
        for x in d:
            d[x].copy_(e[x])
        for x in ("norm", "gate"):
            more[x].copy_(m[x])

    def result():
        torch.cuda.synchronize()
        return d["out"].clone(), step_out.clone(), d["state"].clone()

    want = []
    for seed in (1, 2):
        fresh(seed)
        both()
        want.append(result())
    side = torch.cuda.Stream()
    fresh(1)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        both()
    assert all(torch.equal(a, b) for a, b in zip(result(), want[0]))
    fresh(1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for seed in (1, 2, 1):
        fresh(seed)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(result(), want[seed - 1]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_distances_that_pass_32_bits(dtype):
    """Rows of decays, and slots, more than 2^31 floats apart: the bits of the same numbers side by side."""
    from transformer_b200.parts import decay_attention, decay_attention_step
    H, dim, vdim, far = 2, 72, 72, 2 ** 31 + 8
    d, _, starts = _inputs(dtype, H, H, dim, vdim, [1, 1], "input", False, 1)
    near = {k: v[:2] if k in ("q", "k", "v", "log_decay") else v for k, v in d.items()}
    near["slots"], near["out"] = torch.tensor([1, 0], dtype=torch.int32, device="cuda"), torch.empty((2, H, vdim), dtype=dtype, device="cuda")
    near["state"] = torch.randn((2, H, dim, vdim), device="cuda")
    room = torch.empty(2 * far, device="cuda")                  # 17 GB, of which a few kilobytes are touched
    g = room.as_strided((2, H), (far, 1), 0)
    g.copy_(near["log_decay"])
    for go in (lambda x: decay_attention(seq_start=starts, **x), lambda x: decay_attention_step(**x)):
        state = room.as_strided((2, H, dim, vdim), (far, dim * vdim, vdim, 1), 1024)
        state.copy_(near["state"])
        apart = dict(near, log_decay=g, state=state, out=torch.empty_like(near["out"]))
        here = dict(near, state=near["state"].clone())
        go(here)
        go(apart)
        assert torch.equal(here["out"], apart["out"]) and torch.equal(here["state"], apart["state"])
        assert not torch.equal(here["state"], near["state"])
