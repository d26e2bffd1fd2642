"""The choice of experts within groups, from router logits.

    s = softmax(x) or sigmoid(x)          c = s + bias
    a group's worth = the sum of its ``group_top`` largest c;  the ``groups_use`` worthiest groups stay
    the k largest c of those are chosen, in descending order;  w = s (/ the chosen s' sum) * scale
"""
from __future__ import annotations

import functools

import torch

from ..csrc import lib

MOST_TOKENS = 2 ** 31 - 1
MOST_EXPERTS, MOST_CHOSEN, MOST_GROUPS = 1024, 30, 32       # of the kernel (csrc/router_groups.cu)
SCORES = ("softmax", "sigmoid")


@functools.lru_cache(maxsize=1024)
def check_choice(experts: int, k: int, scores="softmax", groups=1, groups_use=1, group_top=1) -> None:
    """ValueError unless ``k`` of ``experts`` can be chosen in this way."""
    if scores not in SCORES:
        raise ValueError(f"scores are {' or '.join(SCORES)}, got {scores!r}")
    if not 0 < experts <= MOST_EXPERTS:
        raise ValueError(f"the choice is among 1..{MOST_EXPERTS} experts, got {experts}")
    if not 0 < groups <= MOST_GROUPS or experts % groups:
        raise ValueError(f"{experts} experts cannot be {groups} groups of one size (at most {MOST_GROUPS})")
    if not 0 < groups_use <= groups:
        raise ValueError(f"groups used must lie in 1..{groups}, got {groups_use}")
    if group_top not in (1, 2):
        raise ValueError(f"a group's worth is the sum of its 1 or 2 largest, got {group_top}")
    if not 0 < k <= min(MOST_CHOSEN, experts // groups * groups_use):
        raise ValueError(f"experts per token must lie in 1..{min(MOST_CHOSEN, experts // groups * groups_use)}, got {k}")


def choose_experts(logits, index, weights, *, scores="softmax", bias=None, groups=1, groups_use=1, group_top=1, renorm=False,
                   scale=1.0) -> None:
    """Fill ``index`` (int32) and ``weights`` (float), both [tokens, k] and contiguous, from ``logits``, float [tokens, experts]
    with contiguous rows, by the formulas at the head of this file; ``bias``: float [experts] or None; up to 30 of 1,024 experts
    in up to 32 groups of neighbours.

    Equal c, and groups of equal worth, go to the lower index.  A logit of -inf masks an expert: its score is 0, in a row of
    nothing else too, and where the chosen scores are all 0 their weights are 0 also with ``renorm``.  NaN ranks below -inf,
    counts as -inf in a group's worth (as inf - inf does) and spreads to the weights that it enters.  A row's indices always
    differ.  Without a bias experts are compared by their logits; what is decided on sums of scores, or on scores and a bias, is
    what 64 bits decide."""
    nt, E = logits.shape
    row, entry = logits.stride()
    k = index.shape[-1]
    check_choice(E, k, scores, groups, groups_use, group_top)
    if nt > MOST_TOKENS:
        raise ValueError(f"{nt} tokens, at most {MOST_TOKENS}")
    if logits.dtype is not torch.float32 or (entry != 1 and E > 1) or (nt > 1 and row < E):
        raise ValueError("the choice reads float32 logits with contiguous rows")
    if index.shape != (nt, k) or weights.shape != (nt, k) or index.dtype is not torch.int32 or \
            weights.dtype is not torch.float32 or not index.is_contiguous() or not weights.is_contiguous():
        raise ValueError(f"index (int32) and weights (float32) must be contiguous [{nt}, {k}] tensors")
    if bias is not None and (bias.shape != (E,) or bias.dtype is not torch.float32 or not bias.is_contiguous()):
        raise ValueError(f"the bias must be a contiguous float32 tensor of {E} entries")
    lib.check_device(logits, index, weights, bias)
    lib.call("tb_router_groups", logits.data_ptr(), max(row, E), lib.ptr(bias), index.data_ptr(), weights.data_ptr(),
             nt, E, k, groups, groups_use, group_top, scores == "softmax", bool(renorm), float(scale),
             stream=lib.operator_stream())
