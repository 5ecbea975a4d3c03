"""Outputs of beam selection that share memory with its inputs or with each other
are refused, but for scores over scores and flags over flags (CPU only)."""
import pytest

from doe_amd import ops
from test_mx4 import refused


def at(ptr, nbytes=1 << 30):
    return type("B", (), dict(nbytes=nbytes, ptr=ptr))()


# batch 2, 4 beams, the best 4: 32 bytes each, 64 apart
ROLES = ("scores", "finished", "parents", "tokens", "out_scores", "out_finished")
PLACES = {role: (1 << 40) + 64 * i for i, role in enumerate(ROLES)}


def call(**places):
    where = {role: at(p) for role, p in {**PLACES, **places}.items()}
    ops.beam_select(at(1 << 50), batch=2, beams=4, vocab=1000, select=4, end_token=3, workspace=at(1 << 45), **where)


@pytest.mark.parametrize("out,other", [(o, i) for o in ROLES[2:] for i in ROLES[:2] if (i, o) not in (("scores", "out_scores"), ("finished", "out_finished"))])
@pytest.mark.parametrize("off", [-28, 0, 4, 28])
def test_inputs_and_outputs(out, other, off):
    refused("overlap scores or finished", call, **{out: PLACES[other] + off})


@pytest.mark.parametrize("a,b", [(a, b) for i, a in enumerate(ROLES[2:]) for b in ROLES[3 + i:]])
@pytest.mark.parametrize("off", [-28, 0, 4, 28])
def test_outputs_with_each_other(a, b, off):
    refused("outputs overlap each other", call, **{a: PLACES[b] + off})


def test_one_buffer_for_scores_and_both_outputs():
    """Each allowed by itself; both together one would replace the other."""
    refused("overlap", call, out_scores=PLACES["scores"], out_finished=PLACES["scores"])
    refused("overlap", call, out_scores=PLACES["finished"], out_finished=PLACES["finished"])


@pytest.mark.parametrize("how", [{}, dict(out_scores=PLACES["scores"], out_finished=PLACES["finished"]), dict(finished=PLACES["scores"]),
                                 dict(parents=PLACES["scores"] + 32), dict(tokens=PLACES["finished"] - 32)])
def test_in_place_and_side_by_side_get_past_that(how):
    """... and are refused for want of a workspace."""
    where = {role: at(p) for role, p in {**PLACES, **how}.items()}
    refused("workspace of", ops.beam_select, at(1 << 50), batch=2, beams=4, vocab=1000, select=4, end_token=3, workspace=at(1 << 45, 16),
            **where)
