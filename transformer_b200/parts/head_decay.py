"""A linear attention with one decay for each head: the two operators, and a mixer with per-sequence state made of them.

    S_t = e^{g_t} S_{t-1} + k_t v_t^T;    o_t = scale * S_t^T q_t          per head, S [dim, vdim]

S is float and carried from step to step; g_t <= 0 is given per (token, head) or per head.  Heads may share keys and values:
head h of H reads those of head h // (H / G).  With ``norm`` and ``gate`` the heads' outputs leave normed and gated:

    y = o / sqrt(mean(o^2) + eps) * norm * silu(gate)

Sums, norms and the states that are carried are float on both paths, and single tokens, float prompts and the bfloat16 prompts that run on
the CUDA cores (steps of up to 64 tokens with heads of up to 64, keys of more than 128 entries, sizes that are no multiples of eight, rows that are
not whole 16-byte pieces) round each output once.  The other bfloat16 prompts run on the tensor cores, which take bfloat16: there the weights of a
segment's tokens, and the copies of the states at the segments' starts that outputs are made from, are rounded to it too: 2^-8 of
each term at most, over terms of random signs outputs that are some 1.4 times as far off as their last rounding alone makes them.  The states that
are carried do not see these copies.
Kernels: csrc/head_decay.cu, csrc/head_decay_tc.cu.
"""
from __future__ import annotations

import torch

from ..csrc import lib
from .base import MIXERS, Mixer, ParamDecl, StateNeed
from .linear import matmul_nt

MOST_DIM = 256                  # entries of a head, key or value
MOST_ROWS = 2 ** 31 - 1         # tokens, sequences, slots: the kernels count them in 32 bits
USE_TC = True                   # bfloat16 prompts: the tcgen05 kernels, for the heads that they take
WORK_BYTES = 256 << 20          # scratch for the segments' states: of more heads than it holds, portions are done in turn, of one head at least
                                # (4,096 short sequences with heads of 128 x 128: 413 MB)


def _rows(t, name, nt, heads, dim, dtype):
    """The distance of the rows of ``t`` [nt, heads, dim], whose heads lie one behind the other."""
    if t.shape != (nt, heads, dim) or t.dtype is not dtype:
        raise ValueError(f"{name}: {t.dtype} {tuple(t.shape)}, expected {dtype} {(nt, heads, dim)}")
    row, head, entry = t.stride()
    if entry == 1 and head == dim and row >= heads * dim:
        return row
    # what the stride of an axis of one is does not matter
    if (entry != 1 and dim > 1) or (head != dim and heads > 1) or (row < heads * dim and nt > 1):
        raise ValueError(f"{name}: a row's heads must lie one behind the other, rows apart, got strides {t.stride()}")
    return row if nt > 1 else heads * dim


def _states(t, name, H, dim, vdim):
    """The distance of the slots of ``t`` [slots, H, dim, vdim], float, each contiguous."""
    if t.dim() != 4 or t.shape[1:] != (H, dim, vdim) or t.dtype is not torch.float32:
        raise ValueError(f"{name}: {t.dtype} {tuple(t.shape)}, expected float32 [slots, {H}, {dim}, {vdim}]")
    size = dim * vdim
    slot, head, row, entry = t.stride()
    if entry == 1 and row == vdim and head == size and slot >= H * size:
        return slot
    if t.numel() and ((entry != 1 and vdim > 1) or (row != vdim and dim > 1) or (head != size and H > 1) or
                      (slot < H * size and t.shape[0] > 1)):
        raise ValueError(f"{name}: a slot's state must be contiguous, slots apart, got strides {t.stride()}")
    return max(slot, H * size)


def _checked(q, k, v, log_decay, state, slots, out, norm, gate, new_state, seq_start=None):
    """The sizes and distances that both operators hand to their kernels."""
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("q, k and v are [tokens, heads, entries]")
    nt, H, dim = q.shape
    G, vdim, dtype = k.shape[1], v.shape[2], q.dtype
    if dtype is not torch.bfloat16 and dtype is not torch.float32:
        raise ValueError(f"kernels exist for float32 and bfloat16, not {dtype}")
    if G <= 0 or H <= 0 or H % G:
        raise ValueError(f"{H} heads cannot share the keys and values of {G}")
    if not (0 < dim <= MOST_DIM and 0 < vdim <= MOST_DIM):
        raise ValueError(f"heads have 1..{MOST_DIM} entries, got {dim} and {vdim}")
    ldq, ldk, ldv = _rows(q, "q", nt, H, dim, dtype), _rows(k, "k", nt, G, dim, dtype), _rows(v, "v", nt, G, vdim, dtype)
    ldo = _rows(out, "out", nt, H, vdim, dtype)
    each, strides = log_decay.shape == (nt, H), log_decay.stride()
    if log_decay.dtype is not torch.float32 or not (each or log_decay.shape == (H,)) or (strides[-1] != 1 and H > 1) or \
            (each and nt > 1 and strides[0] < H):
        raise ValueError(f"log_decay: float32 [{H}] or [{nt}, {H}] with contiguous rows, got {log_decay.dtype} {tuple(log_decay.shape)}")
    pitch = new_pitch = _states(state, "state", H, dim, vdim)
    n_slots = state.shape[0]
    if new_state is None:
        new_state = state
    elif new_state is not state:
        new_pitch = _states(new_state, "new_state", H, dim, vdim)
        if new_state.shape[0] != n_slots:
            raise ValueError(f"new_state has {new_state.shape[0]} slots, state {n_slots}")
    if max(nt, n_slots, slots.numel()) > MOST_ROWS:
        raise ValueError(f"{nt} tokens, {slots.numel()} sequences, {n_slots} slots: at most {MOST_ROWS} of each")
    if seq_start is not None and lib.head_decay_segments(nt, slots.numel(), dim, vdim) < 0:
        raise ValueError(f"{nt} tokens in {slots.numel()} sequences may be more than {MOST_ROWS} segments")
    if slots.dtype is not torch.int32 or slots.dim() != 1 or not slots.is_contiguous():
        raise ValueError("slots must be a contiguous int32 tensor")
    if (norm is None) != (gate is None):
        raise ValueError("a norm and a gate go together")
    ldgate = p_gate = p_norm = 0
    if gate is not None:
        ldgate, p_gate, p_norm = _rows(gate, "gate", nt, H, vdim, dtype), gate.data_ptr(), norm.data_ptr()
        if norm.dtype is not torch.float32 or norm.numel() != H * vdim or not norm.is_contiguous():
            raise ValueError(f"norm: a contiguous float32 tensor of [{H}, {vdim}], got {norm.dtype} {tuple(norm.shape)}")
        if nt == 0:                 # a tensor without rows has no address, and there is nothing to gate
            p_gate = p_norm = 0
    lib.check_device(q, k, v, log_decay, state, slots, out, norm, gate, new_state, seq_start)
    return (q.data_ptr(), k.data_ptr(), v.data_ptr(), p_gate, ldq, ldk, ldv, ldgate, log_decay.data_ptr(),
            max(strides[0], H) if each else 0, p_norm, state.data_ptr(), new_state.data_ptr(), pitch, new_pitch, out.data_ptr(),
            ldo), (H, G, dim, vdim, n_slots)


def _work(per, H, q, scratch):
    """So many heads as WORK_BYTES holds of ``per`` floats each, and the scratch for them."""
    heads = max(1, min(H, WORK_BYTES // (4 * max(per, 1))))
    if scratch is None:
        return heads, torch.empty(heads * per, dtype=torch.float32, device=q.device)
    return heads, scratch("head_decay.work", (heads * per,), torch.float32)


def decay_attention(q, k, v, log_decay, state, seq_start, slots, out, *, scale=None, norm=None, gate=None, eps=1e-6, new_state=None,
                    scratch=None) -> None:
    """The tokens of a ragged batch of sequences: sequence b's are rows seq_start[b] .. seq_start[b + 1] - 1 (int32 [B + 1],
    ascending), its state is row slots[b] (int32 [B], all different) of ``state`` [slots, H, dim, vdim], which goes on from there.

    q [nt, H, dim], k [nt, G, dim], v [nt, G, vdim], gate and out [nt, H, vdim] (bfloat16 or float32, all of one type) may be
    slices of wider rows; ``log_decay`` float [nt, H] or [H], a value above 0 counts as 0; ``norm`` float [H, vdim]; ``scale``
    defaults to dim^-1/2.  The states afterwards go to ``new_state`` (same rows; default: ``state`` itself).  Neither that nor ``out`` may
    overlap anything else that the call reads.  Rows of ``out``
    behind the last sequence, and states that no sequence names, are left alone, as is all of a sequence whose bounds or slot lie
    outside the tensors.  A sequence without tokens keeps its state.  What is no number in v stays in its channel, behind its
    token, a decay that is none in its head, from its token on; a gate far below 0 closes its channel.
    ``scratch(name, shape, dtype)``: where the workspace comes from (default: allocated by the call)."""
    B, nt = slots.shape[0], q.shape[0]
    if seq_start.dtype != torch.int32 or seq_start.shape != (B + 1,) or not seq_start.is_contiguous():
        raise ValueError(f"seq_start must be a contiguous int32 tensor of {B + 1} entries")
    head, sizes = _checked(q, k, v, log_decay, state, slots, out, norm, gate, new_state, seq_start)
    H, _, dim, vdim, _ = sizes
    more = (*sizes, dim ** -0.5 if scale is None else float(scale), float(eps))
    rows, stream = (seq_start.data_ptr(), slots.data_ptr()), lib.operator_stream()
    segments = lib.head_decay_segments(nt, B, dim, vdim)
    if segments == 0:               # few tokens, small heads: one kernel does all
        lib.call("tb_head_decay_" + lib.suffix(q.dtype), *head, *rows, 0, 0, 1, nt, B, *more, stream=stream)
        return
    per = lib.head_decay_tc_work(nt, B, dim, vdim) if q.dtype == torch.bfloat16 and USE_TC else 0
    if per:
        heads, work = _work(per, H, q, scratch)
        if lib.try_call("tb_head_decay_tc_bf16", *head, *rows, work.data_ptr(), heads, nt, B, *more, stream=stream):
            return
    heads, work = _work(segments * (dim * vdim + 1), H, q, scratch)
    lib.call("tb_head_decay_" + lib.suffix(q.dtype), *head, *rows, work.data_ptr(), segments, heads, nt, B, *more, stream=stream)


def decay_attention_step(q, k, v, log_decay, state, slots, out, *, scale=None, norm=None, gate=None, eps=1e-6, new_state=None) -> None:
    """The same for one token of each sequence: row b belongs to the state in row slots[b].  See :func:`decay_attention`."""
    head, sizes = _checked(q, k, v, log_decay, state, slots, out, norm, gate, new_state)
    if slots.shape[0] != q.shape[0]:
        raise ValueError(f"{q.shape[0]} tokens but {slots.shape[0]} slots")
    lib.call("tb_head_decay_step_" + lib.suffix(q.dtype), *head, slots.data_ptr(), slots.shape[0], *sizes,
             sizes[2] ** -0.5 if scale is None else float(scale), float(eps), stream=lib.operator_stream())


@MIXERS.register("head_decay")
class HeadDecay(Mixer):
    """params: width, heads, dim, vdim, eps; optional: kv_heads (default heads), decay ("fixed": one constant a head,
    g = -exp(rate), the default; "input": g = -exp(rate) softplus(Wa x1 + bias)), scale (default dim^-1/2).

        out = Wo (o / rms_head(o) * norm * silu(Wg x1)),   q, k, v, gate = Win x1"""
    graph_safe = True
    launches_only = True

    def __init__(self, params, dtype, device):
        super().__init__(params, dtype, device)
        g = lambda n: int(params[n])
        self.d, self.H, self.dim, self.vdim = g("width"), g("heads"), g("dim"), g("vdim")
        self.G = int(params.get("kv_heads") or self.H)
        self.eps, self.scale = float(params["eps"]), float(params.get("scale") or self.dim ** -0.5)
        self.decay = params.get("decay", "fixed")
        if min(self.H, self.G, self.dim, self.vdim) <= 0 or self.H % self.G:
            raise ValueError(f"{self.H} heads cannot share the keys and values of {self.G}")
        if max(self.dim, self.vdim) > MOST_DIM:
            raise ValueError(f"heads have up to {MOST_DIM} entries, got {self.dim} and {self.vdim}")
        if self.decay not in ("fixed", "input"):
            raise ValueError(f"the decay is 'fixed' or made from the 'input', got {self.decay!r}")
        self.widths = [self.H * self.dim, self.G * self.dim, self.G * self.vdim, self.H * self.vdim]
        self.rows_width = self.H * self.vdim
        self.in_weight, self.in_width = "win", sum(self.widths)

    def parameters(self):
        decl = {
            "win": ParamDecl((self.in_width, self.d)),             # rows: q heads, k heads, v heads, output gate
            "rate": ParamDecl((self.H,), "norm", "normal"),
            "norm": ParamDecl((self.vdim,), "norm", "ones"),
            "wo": ParamDecl((self.d, self.rows_width)),
        }
        if self.decay == "input":
            decl["wa"] = ParamDecl((self.H, self.d))
            decl["bias"] = ParamDecl((self.H,), "norm", "normal")
        return decl

    def bind(self, tensors) -> None:
        super().bind(tensors)
        self.weights["norm"] = self.weights["norm"].float().repeat(self.H).contiguous()
        if self.decay == "fixed":
            self.weights["log_decay"] = -torch.exp(self.weights["rate"].float())

    def state_need(self):
        return StateNeed((self.H, self.dim, self.vdim), torch.float32)

    def forward_rows(self, ctx, x1, rows, cache, state, z=None) -> None:
        nt, w = x1.shape[0], self.weights
        if z is None:
            z = ctx.scratch("head_decay.z", (nt, self.in_width), self.dtype)
            matmul_nt(x1, w["win"], z)
        q, k, v, gate = z.split(self.widths, dim=1)
        if self.decay == "input":
            a = ctx.scratch("head_decay.a", (nt, self.H), torch.float32)
            matmul_nt(x1, w["wa"], a)                   # float out on both paths: its error would add up along the sequence
            g = ctx.scratch("head_decay.g", (nt, self.H), torch.float32)
            lib.call("tb_head_decay_rates", lib.ptr(a), lib.ptr(w["rate"]), lib.ptr(w["bias"]), lib.ptr(g), nt, self.H)
        else:
            g = w["log_decay"]
        args = (q.unflatten(1, (self.H, self.dim)), k.unflatten(1, (self.G, self.dim)), v.unflatten(1, (self.G, self.vdim)), g, state)
        more = {"scale": self.scale, "norm": w["norm"], "gate": gate.unflatten(1, (self.H, self.vdim)), "eps": self.eps}
        y = rows.unflatten(1, (self.H, self.vdim))
        if ctx.decode:
            decay_attention_step(*args, ctx.slots, y, **more)
        else:
            decay_attention(*args, ctx.seq_start, ctx.slots, y, scratch=ctx.scratch, **more)

    def forward(self, ctx, x1, out, cache, state, z=None) -> None:
        rows = ctx.scratch("head_decay.y", (x1.shape[0], self.rows_width), self.dtype)
        self.forward_rows(ctx, x1, rows, cache, state, z)
        matmul_nt(rows, self.weights["wo"], out)
