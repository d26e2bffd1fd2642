"""The linear attention with one decay for each head and the choice of experts within groups, in 64 bits from their definitions,
with the sizes of the terms that a result is the sum of, for bounds on rounding."""
import math

import torch

F32, BF16 = torch.finfo(torch.float32).eps / 2, torch.finfo(torch.bfloat16).eps / 2     # half a step: a rounding's most


def recurrence(q, k, v, g, S, scale):
    """q [n, H, dim], k [n, G, dim], v [n, G, vdim], g [n, H], S [H, dim, vdim], float64.  (o [n, H, vdim], S afterwards, and for
    each of both the sum of its terms' sizes)."""
    H, times = q.shape[1], q.shape[1] // k.shape[1]
    S, M, outs, sizes = S.clone(), S.abs(), [], []
    for t in range(q.shape[0]):
        f = torch.exp(g[t].clamp(max=0.0))[:, None, None]
        kt, vt = k[t].repeat_interleave(times, 0), v[t].repeat_interleave(times, 0)
        add = kt[:, :, None] * vt[:, None, :]
        S = torch.where(f == 0, 0.0, f * S) + add
        M = torch.where(f == 0, 0.0, f * M) + add.abs()
        outs.append(scale * torch.einsum("hd,hdv->hv", q[t], S))
        sizes.append(abs(scale) * torch.einsum("hd,hdv->hv", q[t].abs(), M))
    stack = lambda x: torch.stack(x) if x else torch.zeros((0, H, v.shape[2]), dtype=q.dtype, device=q.device)
    return stack(outs), S, stack(sizes), M


def bounds(o, size, dtype, dim, n, tensor_cores):
    """What each output may be off: a chain of dim products and additions, a segment's additions (up to 512) and the passes over the
    segments before (a multiplication and an addition each), two exponentials (2 ulp of argument and result each: 8 halves), in float; on
    the tensor cores the weights and the states at the segments' starts are rounded to bfloat16 once each (a term meets one of
    both); and one rounding at the end."""
    chain = (2 * dim + 512 + n // 32 + 16) * F32
    return size * (chain + (BF16 if tensor_cores else 0.0)) + o.abs() * (BF16 if dtype == torch.bfloat16 else F32)


def state_bounds(M, dim, n, tensor_cores):
    """On the tensor cores a weighted key is three bfloat16s: what is left of it is 2^-8 of 2^-8 of 2^-8, and a third of the additions more."""
    return M * ((512 + n // 32 + 16) * F32 * (3 if tensor_cores else 1) + (BF16 ** 3 if tensor_cores else 0.0)) + 1e-30


def normed(o, off, norm, gate, eps, dtype):
    """(y, what it may be off) for outputs o that may be off by `off`: the division by the root mean square moves by the relative size of
    the errors' own root mean square, and everything after it is a few float roundings and the last one."""
    rms = (o.square().mean(-1, keepdim=True) + eps).sqrt()
    silu = gate * torch.sigmoid(gate)
    y = o / rms * norm * silu
    share = off.square().mean(-1, keepdim=True).sqrt() / rms
    moved = (off + o.abs() * share) / rms * (norm * silu).abs() * (1.0 + 2.0 * share)
    return y, moved + y.abs() * ((o.shape[-1] + 16) * F32 + (BF16 if dtype == torch.bfloat16 else F32))


def choose(x, k, *, scores, bias=None, groups=1, groups_use=1, group_top=1, renorm=False, scale=1.0):
    """x [nt, E] float64 -> (index, weights), by sorting in Python, which keeps the order of equals."""
    index, weights = [], []
    E = x.shape[1]
    for row in x.tolist():
        number = lambda v: -math.inf if v != v else v           # NaN ranks below all
        if scores == "sigmoid":
            s = [v if v != v else 1.0 / (1.0 + math.exp(-v)) if v > -700 else 0.0 for v in row]
        else:
            top = max((v for v in row if v == v), default=0.0)
            e = [v if v != v else math.exp(v - top) if v > -math.inf else 0.0 for v in row]
            total = sum(e)
            s = [v / total if total else 0.0 for v in e]
        c = [a + (float(bias[i]) if bias is not None else 0.0) for i, a in enumerate(s)]
        # below -inf: NaN; a masked expert keeps its place above it
        rank = [(number(row[i]) == row[i], number(c[i])) for i in range(E)]
        size = E // groups
        worth = [sum(sorted((number(v) for v in c[j * size:(j + 1) * size]), reverse=True)[:group_top]) for j in range(groups)]
        kept = set(sorted(range(groups), key=lambda j: -worth[j])[:groups_use])
        order = sorted((i for i in range(E) if i // size in kept), key=lambda i: rank[i], reverse=True)
        order = sorted(order, key=lambda i: (not rank[i][0], -rank[i][1], i))[:k]
        w = [s[i] for i in order]
        if renorm:
            total = sum(w)
            w = [v / total if total else v for v in w]
        index.append(order)
        weights.append([v * scale for v in w])
    return torch.tensor(index), torch.tensor(weights, dtype=torch.float64)
