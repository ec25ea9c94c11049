"""Calls of the objectives over logits whose outputs share memory with another buffer are refused, before anything is launched:
the workgroups of a row read its inputs at times that nothing orders against the writes of another one."""
import itertools

import pytest

from tests.test_objectives_ref import k, refused      # noqa: F401

ROWS, COLS, TOP_K, BATCH = 6, 50001, 3, 2


class Room:
    """Addresses that no refused call touches, a megabyte and more between them."""

    def __init__(self):
        self.at = {}
        self.next = 1 << 30

    def __getitem__(self, name):
        if name not in self.at:
            self.at[name] = self.next
            self.next += 1 << 23
        return self.at[name]


def token_logprobs(k, a):
    return k.seraph_token_logprobs(a["logits"], a["targets"], a["logp"], a["lse"], a["entropy"], a["starts"], BATCH, ROWS, COLS, a["ws"], 1 << 20, None)


def policy(k, a):
    from seraph_amd._lib import PolicyOptions
    return k.seraph_policy_grad(a["logits"], a["targets"], a["advantages"], a["old"], a["ref"], a["weights"], a["grad"], a["loss"], a["logp"], a["kl"],
                                a["entropy"], PolicyOptions(0.2, 0.2, 0.1, 0.1), a["starts"], BATCH, ROWS, COLS, 4, a["ws"], 1 << 20, None)


def preference(k, a):
    from seraph_amd._lib import PreferenceOptions
    return k.seraph_preference_grad(a["logits"], a["targets"], a["ref"], a["grad"], a["loss"], a["scores"], a["logp"],
                                    PreferenceOptions(0, 0.1, 0.0, 0.0, 0), a["starts"], BATCH // 2, ROWS, COLS, a["ws"], 1 << 20, None)


def distill(k, a):
    from seraph_amd._lib import DistillOptions
    return k.seraph_distill_grad(a["logits"], a["ids"], a["teacher"], a["teacher_lse"], a["targets"], a["weights"], a["grad"], a["loss"],
                                 DistillOptions(1.0, 1.0, 0.5, 1), a["starts"], BATCH, ROWS, COLS, TOP_K, 4, a["ws"], 1 << 20, None)


ROW = 4 * ROWS
OPS = {
    token_logprobs: (dict(logits=ROW * COLS, targets=ROW, starts=4 * BATCH + 4), dict(logp=ROW, lse=ROW, entropy=ROW)),
    policy: (dict(logits=ROW * COLS, targets=ROW, advantages=ROW, old=ROW, ref=ROW, weights=ROW, starts=4 * BATCH + 4),
             dict(grad=ROW * COLS, loss=ROW, logp=ROW, kl=ROW, entropy=ROW, ws=16)),
    preference: (dict(logits=ROW * COLS, targets=ROW, ref=ROW, starts=4 * BATCH + 4), dict(grad=ROW * COLS, loss=2 * BATCH, scores=4 * BATCH, logp=ROW, ws=16)),
    distill: (dict(logits=ROW * COLS, ids=ROW * TOP_K, teacher=2 * ROWS * TOP_K, teacher_lse=ROW, targets=ROW, weights=ROW, starts=4 * BATCH + 4),
              dict(grad=ROW * COLS, loss=ROW, ws=16)),
}
CASES = [(op, out, other) for op, (ins, outs) in OPS.items() for out, other in itertools.product(outs, {**ins, **outs})
         if out != other and (out, other) not in (("grad", "logits"), ("ws", "logits"), ("ws", "grad"), ("grad", "ws"))]


@pytest.mark.parametrize("op,out,other", CASES, ids=lambda v: v if isinstance(v, str) else v.__name__)
def test_an_output_in_another_buffer(k, op, out, other):      # noqa: F811
    ins, outs = OPS[op]
    size = {**ins, **outs}
    ends = [0] if "ws" in (out, other) else [0, size[other] - 4, 4 - size[out]]      # the same, its last word, its first word
    for off in ends:
        a = Room()
        a.at[out] = a[other] + off // 4 * 4
        refused(k, op(k, a), -1, "overlap")
