"""The protocols of the rings that rows come through, in every interleaving of
a small one, with waits that may run out at any moment: no barrier may be armed
while copies to it are in flight, and none may be in flight when a block ends.
On a GPU such a wait cannot be made to run out without a copy that never lands,
so this is a model of residual_norm_sm100.cu's and distill_topk_sm100.cu's steps.
"""
from __future__ import annotations

import pytest


def explore(start, moves, ended, cut=400_000):
    """Every state that can be reached; moves(state) yields the next ones and
    raises AssertionError at a step that is not allowed."""
    seen, todo, ends = {start}, [start], 0
    while todo:
        state = todo.pop()
        following = list(moves(state))
        if not following:
            ended(state)
            ends += 1
        for s in following:
            if s not in seen:
                seen.add(s)
                todo.append(s)
        assert len(seen) < cut
    return len(seen), ends


def put(t, i, v):
    return t[:i] + (v,) + t[i + 1:]


# A barrier: (phases completed, arrivals, copies in flight).
def land(bar, expected):
    phase, arrived, flight = bar[0], bar[1], bar[2] - 1
    return (phase + 1, 0, 0) if arrived == expected and flight == 0 else (phase, arrived, flight)


def waited(bar, use):
    """What a wait on the parity of the use-th phase sees."""
    return bar[0] & 1 != use & 1


def norm_ring(rows, stages, threads, mended):
    """Each thread: waits for a row's stage, meets the others at a barrier,
    issues its copy of the row that takes the stage next."""
    WAIT, MEET, ISSUE, DONE = range(4)

    def moves(state):
        at, bars, failed, failed_in, note = state
        for s, bar in enumerate(bars):
            if bar[2]:
                yield at, put(bars, s, land(bar, threads)), failed, failed_in, note
        if all(step == MEET for _, step in at):
            yield tuple((row, ISSUE) for row, _ in at), bars, failed, failed_in, note
        for i, (row, step) in enumerate(at):
            stage = row % stages
            if step == WAIT and row < rows:
                there = put(at, i, (row, MEET))
                if waited(bars[stage], row // stages):
                    yield there, bars, failed, failed_in, note
                else:  # it ran out, or another thread's did
                    yield there, bars, True, put(failed_in, row & 1, True), note
            elif step == ISSUE:
                there, later = put(at, i, (row + 1, WAIT)), row + stages
                if mended and failed_in[row & 1]:
                    kept = row if i == 0 and note is None else note
                    yield there, bars, failed, put(failed_in, ~row & 1, True), kept
                elif later >= rows:
                    yield there, bars, failed, failed_in, note
                else:
                    phase, arrived, flight = bars[stage]
                    assert phase == later // stages and arrived < threads, "armed while copies are in flight"
                    yield there, put(bars, stage, (phase, arrived + 1, flight + 1)), failed, failed_in, note
            elif step == WAIT:  # after the last row: thread 0 waits for the rows in flight
                if i > 0 or note is None or all(
                        bars[r % stages][0] > r // stages for r in range(note, min(note + stages, rows))):
                    yield put(at, i, (row, DONE)), bars, failed, failed_in, note

    def ended(state):
        at, bars = state[:2]
        assert all(step == DONE for _, step in at), "a thread waits for good"

    def moves_in_a_live_block(state):
        if all(step == DONE for _, step in state[0]):
            assert not any(bar[2] for bar in state[1]), "the block ended with copies in flight"
            return []
        return moves(state)

    first = tuple((0, threads, threads) if s < rows else (0, 0, 0) for s in range(stages))
    return explore((((0, WAIT),) * threads, first, False, (False, False), None), moves_in_a_live_block, ended)


@pytest.mark.parametrize("rows, stages, threads", [(1, 2, 2), (3, 1, 2), (5, 2, 2), (6, 3, 2), (4, 2, 3)])
def test_norm_ring(rows, stages, threads):
    states, ends = norm_ring(rows, stages, threads, mended=True)
    assert states > 10 and ends >= 1


def test_norm_ring_that_goes_on_issuing_is_caught():
    with pytest.raises(AssertionError, match="in flight"):
        norm_ring(5, 2, 2, mended=False)


def distill_ring(uses, stages, warps, mended):
    """A producer fills stages that all consumer warps have released; each warp
    waits for a stage and releases it."""

    def moves(state):
        made, stopped, drained, at, lost, full, empty, failed = state
        if drained and all(u == uses for u in at):
            assert not any(bar[2] for bar in full), "the block ended with copies in flight"
            return
        for s, bar in enumerate(full):
            if bar[2]:
                yield made, stopped, drained, at, lost, put(full, s, land(bar, 1)), empty, failed
        if made < uses and not stopped:
            s, round_ = made % stages, made // stages
            if waited(empty[s], round_ - 1):
                phase, arrived, flight = full[s]
                assert phase == round_ and arrived == 0, "armed while copies are in flight"
                yield made + 1, stopped, drained, at, lost, put(full, s, (phase, 1, flight + 1)), empty, failed
            elif mended:
                yield made, True, drained, at, lost, full, empty, True
            else:
                phase, arrived, flight = full[s]
                assert phase == round_ and arrived == 0, "armed while copies are in flight"
                yield made + 1, stopped, drained, at, lost, put(full, s, (phase, 1, flight + 1)), empty, True
        elif not drained:
            if not mended or all(full[u % stages][0] > u // stages for u in range(max(0, made - stages), made)):
                yield made, stopped, True, at, lost, full, empty, failed
        for w, use in enumerate(at):
            if use == uses:
                continue
            s = use % stages
            there, gave_up = put(at, w, use + 1), put(lost, w, True)
            phase, arrived, _ = empty[s]
            freed = put(empty, s, (phase + 1, 0, 0) if arrived + 1 == warps else (phase, arrived + 1, 0))
            if mended and lost[w]:
                yield made, stopped, drained, there, lost, full, empty, failed
            elif waited(full[s], use // stages):
                yield made, stopped, drained, there, lost, full, freed, failed
            else:
                yield made, stopped, drained, there, gave_up, full, empty if mended else freed, True

    def ended(state):
        assert state[2] and all(u == uses for u in state[3]), "a warp waits for good"

    idle = ((0, 0, 0),) * stages
    return explore((0, False, False, (0,) * warps, (False,) * warps, idle, idle, False), moves, ended)


@pytest.mark.parametrize("uses, stages, warps", [(1, 2, 2), (4, 1, 2), (5, 2, 2), (7, 3, 2), (5, 2, 3)])
def test_distill_ring(uses, stages, warps):
    states, ends = distill_ring(uses, stages, warps, mended=True)
    assert states > 10 and ends >= 1


def test_distill_ring_that_goes_on_issuing_is_caught():
    with pytest.raises(AssertionError, match="in flight"):
        distill_ring(5, 2, 2, mended=False)
