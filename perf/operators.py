"""The work that is timed: a linear attention with a decay for each head, and the choice of experts within groups.

  prompt    ``decay_attention``: the tokens of a ragged batch of sequences, each going on from a state of its own.
  step      ``decay_attention_step``: one token for each sequence of a batch.
  choose    ``choose_experts``: router logits to the experts of every token and their weights.

With ``decay`` "input" the logarithm of the decay is given for each (token, head), with "fixed" for each head.  ``gated``: the heads'
outputs are normed and pass a gate in the same call.  q, k, v and the gate are slices of one projection's rows, as a mixer has them.
"""
import math
import random

import torch

own = False

EPS = 1e-6
CHUNK = 128         # tokens that the plain form of a prompt takes together


# ---- the cases -----------------------------------------------------------------------------------------------------
def _attention(name, kind, batch, low, high, heads, kv_heads, dim, vdim, *, decay="input", gated=True, dtype="bfloat16"):
    """Lengths of the ``batch`` sequences uniform in [low, high]."""
    c = {"kind": kind, "batch": batch, "low": low, "high": high, "heads": heads, "kv_heads": kv_heads, "dim": dim,
         "vdim": vdim, "decay": decay, "gated": gated, "dtype": dtype}
    return c if name is None else dict(c, name=name)


def _choose(name, tokens, experts, k, *, groups=1, groups_use=1, group_top=1, scores="softmax", bias=False, renorm=False,
            scale=1.0):
    c = {"kind": "choose", "tokens": tokens, "experts": experts, "k": k, "groups": groups, "groups_use": groups_use,
         "group_top": group_top, "scores": scores, "bias": bias, "renorm": renorm, "scale": scale}
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # a short question to a small model: what a call costs when there is next to nothing to do
        _attention("prompt_short", "prompt", 1, 33, 33, 8, 8, 64, 64, gated=False),
        # the benchmark's prompt length; decays that are constants of the heads
        _attention("prompt_2048", "prompt", 1, 2048, 2048, 32, 32, 128, 128, decay="fixed"),
        # several users' prompts at once, from one token up, heads that share keys and values
        _attention("prompts_ragged", "prompt", 11, 1, 2048, 32, 4, 128, 128),
        # as many tokens as one step of the engine takes
        _attention("prompt_8192", "prompt", 1, 8192, 8192, 16, 16, 128, 128),
        # narrow keys and wide values, odd lengths
        _attention("prompts_narrow", "prompt", 6, 100, 1500, 16, 16, 64, 128, decay="fixed", gated=False),
        # the 32-bit path with heads of odd sizes
        _attention("prompts_float32", "prompt", 2, 200, 700, 8, 4, 96, 80, dtype="float32"),
        # one user
        _attention("step_1", "step", 1, 1, 1, 32, 32, 128, 128),
        # a busy server
        _attention("step_64", "step", 64, 1, 1, 32, 8, 128, 128),
        # the 32-bit path with heads of odd sizes
        _attention("step_float32", "step", 9, 1, 1, 12, 12, 80, 96, decay="fixed", gated=False, dtype="float32"),
        # a decode step's router
        _choose("choose_8", 8, 64, 6, groups=8, groups_use=3),
        # a full step's: many experts, scores each by itself, a bias for balance
        _choose("choose_8191", 8191, 256, 8, groups=8, groups_use=4, group_top=2, scores="sigmoid", bias=True, renorm=True,
                scale=2.5),
        # experts without groups, a number that no power of two divides by much
        _choose("choose_2039", 2039, 60, 4, renorm=True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "prompt", "step", "step", "choose", "choose"])
    if kind == "choose":
        groups = rng.choice([1, 1, 2, 4, 8, 16])
        size = rng.randint(2, 256 // groups) if groups > 1 else _log_int(rng, 4, 256)
        groups_use = rng.randint(1, groups)
        sigmoid = rng.random() < 0.5
        return _choose(None, _log_int(rng, 1, 8191), groups * size, rng.randint(1, min(16, groups_use * size)), groups=groups,
                       groups_use=groups_use, group_top=rng.randint(1, 2), scores="sigmoid" if sigmoid else "softmax",
                       bias=rng.random() < 0.5, renorm=rng.random() < 0.5, scale=rng.choice([1.0, 2.5]))
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4])
    if dtype == "float32":
        dim, vdim = rng.randint(16, 128), rng.randint(16, 128)
    else:
        dim, vdim = rng.choice([(64, 64), (64, 128), (128, 64), (128, 128), (128, 128), (128, 128), (80, 96), (128, 256)])
    more = {"decay": rng.choice(["input", "fixed"]), "gated": rng.random() < 0.5, "dtype": dtype}
    if kind == "step":
        return _attention(None, kind, _log_int(rng, 1, 64), 1, 1, heads, kv_heads, dim, vdim, **more)
    batch = _log_int(rng, 1, 8)
    most = (4096 if dtype == "bfloat16" else 1000) // batch
    low = _log_int(rng, 1, most)
    return _attention(None, kind, batch, low, _log_int(rng, low, most), heads, kv_heads, dim, vdim, **more)


def _lengths(c):
    """A case's own, whatever the seed; the shortest and the longest among them where there are two or more."""
    if c["kind"] == "step":
        return [1] * c["batch"]
    rng = random.Random(c["batch"] * 1000003 + c["low"] * 1009 + c["high"])
    lens = [rng.randint(c["low"], c["high"]) for _ in range(c["batch"])]
    if len(lens) > 1:
        lens[0], lens[-1] = c["high"], c["low"]
    return lens


# ---- what a program has in hand ------------------------------------------------------------------------------------
def prepare(case, seed):
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=gen, device="cuda")
    if case["kind"] == "choose":
        nt, E = case["tokens"], case["experts"]
        # logits as a trained router gives them: a spread of about 1.5, some experts more popular than others
        logits = randn(nt, E) * 1.5 + randn(E) * 0.5
        return {"case": case, "logits": logits, "bias": randn(E) * 0.1 if case["bias"] else None,
                "index": torch.empty((nt, case["k"]), dtype=torch.int32, device="cuda"),
                "weights": torch.empty((nt, case["k"]), device="cuda")}
    dtype = getattr(torch, case["dtype"])
    H, G, dim, vdim, B = case["heads"], case["kv_heads"], case["dim"], case["vdim"], case["batch"]
    lens = _lengths(case)
    nt = sum(lens)
    widths = [H * dim, G * dim, G * vdim, H * vdim]
    z = randn(nt, sum(widths)).to(dtype)                # one projection's rows: queries, keys, values, gate
    q, k, v, gate = z.split(widths, dim=1)
    if case["decay"] == "fixed":                        # from forgetting in three tokens to remembering hundreds
        log_decay = -torch.exp2(-8.0 * torch.arange(1, H + 1, device="cuda") / H) * (1.0 + 0.1 * torch.rand((H,), generator=gen, device="cuda"))
    else:
        log_decay = -torch.exp(randn(H) * 0.7 - 1.0) * torch.nn.functional.softplus(randn(nt, H) * 1.5 - 1.0)
    state = randn(B, H, dim, vdim)
    state[: B // 2] = 0.0                               # half of the sequences are new
    slots = torch.randperm(B, generator=host)
    return {"case": case, "lens": lens, "q": q.view(nt, H, dim), "k": k.view(nt, G, dim), "v": v.view(nt, G, vdim),
            "gate": gate.view(nt, H, vdim) if case["gated"] else None,
            "norm": 1.0 + 0.1 * randn(H, vdim) if case["gated"] else None, "log_decay": log_decay, "state": state,
            "new_state": torch.empty_like(state), "out": torch.empty((nt, H, vdim), dtype=dtype, device="cuda"),
            "seq_start": torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda(),
            "slots": slots.to(torch.int32).cuda(), "rows": slots.cuda()}


# ---- one pass --------------------------------------------------------------------------------------------------------
def run(state):
    kind = state["case"]["kind"]
    if own:
        from transformer_b200.parts import choose_experts, decay_attention, decay_attention_step
        s, c = state, state["case"]
        if kind == "choose":
            choose_experts(s["logits"], s["index"], s["weights"], scores=c["scores"], bias=s["bias"], groups=c["groups"],
                           groups_use=c["groups_use"], group_top=c["group_top"], renorm=c["renorm"], scale=c["scale"])
            return s["index"], s["weights"]
        if kind == "step":
            decay_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], s["slots"], s["out"], norm=s["norm"],
                                 gate=s["gate"], eps=EPS, new_state=s["new_state"])
        else:
            decay_attention(s["q"], s["k"], s["v"], s["log_decay"], s["state"], s["seq_start"], s["slots"], s["out"],
                            norm=s["norm"], gate=s["gate"], eps=EPS, new_state=s["new_state"])
        return s["out"], s["new_state"]
    if kind == "choose":
        return _plain_choose(state)
    return _plain_step(state) if kind == "step" else _plain_prompt(state)


# ---- the plain forms -------------------------------------------------------------------------------------------------
def _heads(s):
    """q, k, v in 32 bits with the keys and values of shared heads repeated, q scaled."""
    c = s["case"]
    times = c["heads"] // c["kv_heads"]
    return (s["q"].float() * c["dim"] ** -0.5, s["k"].float().repeat_interleave(times, 1),
            s["v"].float().repeat_interleave(times, 1))


def _plain_out(s, o):
    if s["gate"] is not None:
        g = s["gate"].float()
        o = o / (o.square().mean(-1, keepdim=True) + EPS).sqrt() * s["norm"] * (g / (1.0 + torch.exp(-g)))
    return o.to(s["q"].dtype)


def _plain_step(s):
    q, k, v = _heads(s)
    decay = torch.exp(s["log_decay"]).expand(q.shape[0], q.shape[1])
    S = s["state"][s["rows"]] * decay[:, :, None, None] + k[..., None] * v[:, :, None, :]
    new = torch.empty_like(s["state"])
    new[s["rows"]] = S
    return _plain_out(s, (q[..., None] * S).sum(2)), new


def _plain_prompt(s):
    q, k, v = _heads(s)
    g = s["log_decay"].double().expand(q.shape[0], q.shape[1])
    new, outs, at = torch.empty_like(s["state"]), [], 0
    below = torch.ones((CHUNK, CHUNK), dtype=torch.bool, device=q.device).tril()
    for b, n in enumerate(s["lens"]):
        pad = -n % CHUNK
        cut = lambda t: torch.nn.functional.pad(t[at:at + n], (0, 0) * (t.dim() - 1) + (0, pad)).unflatten(0, (-1, CHUNK))
        qc, kc, vc = (cut(t).transpose(1, 2) for t in (q, k, v))                    # [chunks, heads, CHUNK, .]
        c = cut(g).transpose(1, 2).cumsum(-1)                                       # in 64 bits
        decay = torch.exp((c[..., :, None] - c[..., None, :]).masked_fill(~below, -math.inf).float())
        last = c[..., -1:]
        o = (qc @ kc.transpose(-1, -2) * decay) @ vc
        U = (kc * torch.exp((last - c).float())[..., None]).transpose(-1, -2) @ vc
        S, starts = s["state"][s["rows"][b]], []
        whole = torch.exp(last.float())[..., None]
        for i in range(U.shape[0]):
            starts.append(S)
            S = whole[i] * S + U[i]
        o = o + (qc * torch.exp(c.float())[..., None]) @ torch.stack(starts)
        new[s["rows"][b]] = S
        outs.append(o.transpose(1, 2).flatten(0, 1)[:n])
        at += n
    return _plain_out(s, torch.cat(outs)), new


def _plain_choose(s):
    """In 64 bits: the scores of neighbouring experts may differ by less than a rounding."""
    c, x = s["case"], s["logits"].double()
    score = 1.0 / (1.0 + torch.exp(-x)) if c["scores"] == "sigmoid" else torch.exp(x - x.amax(-1, keepdim=True))
    if c["scores"] == "softmax":
        score = score / score.sum(-1, keepdim=True)
    rank = score if s["bias"] is None else score + s["bias"].double()
    if c["groups"] > 1:
        by_group = rank.unflatten(1, (c["groups"], -1))
        top = by_group.sort(dim=-1, descending=True).values[..., : c["group_top"]].sum(-1)
        kept = top.sort(dim=-1, descending=True, stable=True).indices[:, : c["groups_use"]]
        mask = torch.zeros_like(top, dtype=torch.bool).scatter_(1, kept, True)
        rank = by_group.masked_fill(~mask[..., None], -math.inf).flatten(1)
    index = rank.sort(dim=-1, descending=True, stable=True).indices[:, : c["k"]]
    w = score.gather(1, index)
    if c["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    return index.to(torch.int32), (w * c["scale"]).float()


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "choose":
        return {"bytes": 4 * c["tokens"] * c["experts"] + 8 * c["tokens"] * c["k"] + (4 * c["experts"] if c["bias"] else 0),
                "flops": 4 * c["tokens"] * c["experts"]}
    nt = sum(_lengths(c))
    H, G, dim, vdim = c["heads"], c["kv_heads"], c["dim"], c["vdim"]
    row = H * dim + G * (dim + vdim) + H * vdim * (2 if c["gated"] else 1)
    size = 2 if c["dtype"] == "bfloat16" else 4
    decays = 4 * H * (nt if c["decay"] == "input" else 1)
    return {"bytes": size * nt * row + decays + 8 * c["batch"] * H * dim * vdim + (4 * H * vdim if c["gated"] else 0),
            "flops": 4 * nt * H * dim * vdim}


# ---- the definition, in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "choose":
        return _exact_choose(case, s)
    H, G, dim, vdim, lens = case["heads"], case["kv_heads"], case["dim"], case["vdim"], s["lens"]
    B, most = len(lens), max(lens)
    # the sequences side by side, behind one another's ends nothing: a token that is not there writes and forgets nothing
    def side_by_side(t):
        rows = torch.zeros((most, B) + tuple(t.shape[1:]), dtype=torch.float64, device=t.device)
        for b, part in enumerate(t.double().split(lens)):
            rows[: lens[b], b] = part
        return rows
    group = torch.arange(H, device="cuda") // (H // G)
    q, k, v = side_by_side(s["q"]), side_by_side(s["k"]), side_by_side(s["v"])
    g = s["log_decay"].double()
    decay = side_by_side(g if g.dim() == 2 else g.repeat(sum(lens), 1)).exp()
    S = s["state"].double()[s["rows"]]
    o = torch.empty((most, B, H, vdim), dtype=torch.float64, device="cuda")
    for t in range(most):
        S *= decay[t][:, :, None, None]
        S += k[t][:, group, :, None] * v[t][:, group, None, :]
        o[t] = torch.einsum("bhd,bhdv->bhv", q[t], S)
    o = torch.cat([o[:n, b] for b, n in enumerate(lens)]) / math.sqrt(dim)
    if case["gated"]:
        g = s["gate"].double()
        o = o * torch.rsqrt((o * o).mean(-1, keepdim=True) + EPS) * s["norm"].double() * g * torch.sigmoid(g)
    new = torch.empty_like(S)
    new[s["rows"]] = S
    return o, new


def _exact_choose(case, s):
    """By counting: an expert is chosen if fewer than k others come before it."""
    x = s["logits"].double()
    score = torch.sigmoid(x) if case["scores"] == "sigmoid" else torch.softmax(x, -1)
    rank = score + (0.0 if s["bias"] is None else s["bias"].double())
    def place(r):       # how many come before each: larger ones, and equal ones of a lower index
        i = torch.arange(r.shape[1], device=r.device)
        return torch.cat([((p[:, None, :] > p[:, :, None]) | ((p[:, None, :] == p[:, :, None]) & (i[None, :] < i[:, None]))).sum(-1)
                          for p in r.split(512)])
    if case["groups"] > 1:
        by_group = rank.unflatten(1, (case["groups"], -1))
        worth = by_group.topk(min(case["group_top"], by_group.shape[-1]), dim=-1).values.sum(-1)
        rank = rank.masked_fill((place(worth) >= case["groups_use"]).repeat_interleave(by_group.shape[-1], 1), -math.inf)
    at = place(rank)
    index = torch.empty((x.shape[0], x.shape[1]), dtype=torch.int64, device="cuda").scatter_(1, at, torch.arange(x.shape[1], device="cuda").expand_as(at))
    index = index[:, : case["k"]]
    w = score.gather(1, index)
    return index.int(), (w / w.sum(-1, keepdim=True) if case["renorm"] else w) * case["scale"]
