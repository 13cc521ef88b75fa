"""CPU: a model of the ring of stages that the decode GEMM's two MMA issuers share.

One producer loads k-block u into stage u % S as soon as that stage's previous use was
consumed; loads land in any order. Issuer 0 takes the even k-blocks, issuer 1 the odd ones.
An mbarrier wait by parity passes when the barrier's current phase has the other parity, so
it tells a phase from the one before it only. An issuer must never pass its wait before its
own k-block has landed in the stage. With an odd S, where a stage goes from issuer to
issuer, each notes what it found landed and waits for the other's note first (dc_issue in
gw_gemm_decode.cu).
"""

from __future__ import annotations

import random

import pytest


def passes(completed: int, parity: int) -> bool:
    """mbarrier.try_wait.parity on a barrier of which `completed` phases have completed."""
    return (completed & 1) != parity


def run(stages: int, blocks: int, notes: bool, rng: random.Random) -> bool:
    """One random schedule to its end; False if an issuer took a stage too early."""
    full, empty = [0] * stages, [0] * stages          # completed phases
    holds = [None] * stages                           # the k-block that has landed in each stage
    seen = [-1] * stages                              # the k-block that an issuer last found landed
    flying: list[int] = []
    issued, nxt = 0, [0, 1]                           # next k-block of the producer, of each issuer
    while min(nxt) < blocks:
        moves = [("land", u) for u in flying]
        if issued < blocks and (issued < stages or passes(empty[issued % stages], (issued // stages - 1) & 1)):
            moves.append(("load", issued))
        for u in nxt:
            noted = not notes or u < stages or seen[u % stages] >= u - stages
            if u < blocks and noted and passes(full[u % stages], (u // stages) & 1):
                moves.append(("take", u))
        assert moves, "the ring came to a standstill"
        what, u = rng.choice(moves)
        s = u % stages
        if what == "load":
            flying.append(u)
            issued += 1
        elif what == "land":
            flying.remove(u)
            holds[s] = u
            full[s] += 1
        else:
            if holds[s] != u:
                return False
            seen[s] = u
            empty[s] += 1
            nxt[u % 2] = u + 2
    return True


@pytest.mark.parametrize("blocks", [2, 3, 5, 6, 8, 16, 33])
@pytest.mark.parametrize("stages,notes", [(5, True), (3, True), (7, True), (4, False), (6, False), (8, False)])
def test_no_stage_is_taken_before_it_landed(stages, notes, blocks):
    rng = random.Random(blocks * 10 + stages)
    assert all(run(stages, blocks, notes, rng) for _ in range(3000))


@pytest.mark.parametrize("blocks", [6, 8, 16])
def test_an_odd_ring_needs_the_notes(blocks):
    """Without them some schedules take a stage early, from the first k-block past the ring on."""
    rng = random.Random(blocks)
    assert not all(run(5, blocks, False, rng) for _ in range(3000))
    assert all(run(5, 5, False, rng) for _ in range(1000))
