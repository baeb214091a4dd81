"""The barriers between the issuer of products and the softmax warps of a group of the shared-prefix
kernel (`csrc/prefix_attention.cu`), in every order of events: no GPU, and nothing that a run could be
lucky with.

The model is of one group: the issuer's thread, the tensor pipe (its products finish in the order in
which they were asked for, any time later), the arrivals of its commits (any time after the products
ahead of them have finished, in any order among themselves) and a softmax warp that may or may not move
its maximum at any tile but a piece's first.  What either of them does in which order is read from the
source.  A barrier's wait is by parity, as the hardware has it: it passes for a phase that is over, and
just as well for the one after next.
"""

from __future__ import annotations

import re
from pathlib import Path

import pytest

SOURCE = Path(__file__).resolve().parents[1] / "linnet_b200" / "csrc" / "prefix_attention.cu"


class Wrong(AssertionError):
    pass


def issuer_order(text: str) -> tuple[str, ...]:
    """What follows the sums of a tile: the commit of `summed` and the next scores."""
    part = text[text.index("umma_f16_ts(o_at"):]
    part = part[:part.index("++task, ++tile;")]
    marks = {"summed": "commit_at(summed", "scores": "issue_scores()", "result": "commit_at(result)"}
    assert all(part.count(mark) == 1 for mark in marks.values()), part
    order = tuple(sorted(marks, key=lambda name: part.index(marks[name])))
    assert order[0] == "result"
    return order[1:]


def barriers_of_sums(text: str) -> int:
    """Of a group: one, or one for each of its two buffers."""
    return 2 if re.search(r"\bsummed\[2\]\[2\]", text) else 1


def softmax_waits(text: str) -> tuple[tuple[int, ...], tuple[int, ...]]:
    """Of which tiles back the softmax waits for the sums: at every tile, and before it rescales."""
    part = text[text.index("ok = wait(&bars.scores[g][b]"):]
    part = part[:part.index("mbar_arrive(&bars.weights[g][b])")]
    read, moved, rescaled = (part.index(mark) for mark in ("tmem_ask_32(", "__any_sync(", "tmem_take_8("))
    both = barriers_of_sums(text) == 2
    form = r"wait\(&bars\.summed\[g\]\[b( \^ 1)?\], \(\(task - (\d)\) >> 1\) & 1" if both else \
        r"wait\(&bars\.summed\[g\](), \(task - (\d)\) & 1"
    every, rescale = [], []
    for m in re.finditer(form, part):
        back = int(m.group(2))
        assert not both or bool(m.group(1)) == bool(back & 1)  # the barrier is that tile's
        assert m.start() < read or moved < m.start() < rescaled
        (every if m.start() < read else rescale).append(back)
    assert len(every) + len(rescale) == part.count("bars.summed")
    return tuple(every), tuple(rescale)


def explore(pieces: list[int], order: tuple[str, ...], barriers: int, every: tuple[int, ...], rescale: tuple[int, ...]) -> int:
    """Walks every state of the model; returns how many there are.  `pieces`: tiles of each."""
    first, last = [], []
    for n in pieces:
        first += [True] + [False] * (n - 1)
        last += [False] * (n - 1) + [True]
    tiles, piece_of = len(first), [i for i, n in enumerate(pieces) for _ in range(n)]
    names = ["scores0", "scores1", "weights0", "weights1", "summed0", "summed1", "result"]
    at = {name: i for i, name in enumerate(names)}

    def sums(t):  # their barrier, and which of its phases
        return at[f"summed{t % barriers}"], t // barriers

    def scores(t):  # asked for, and committed
        return (("product", "S", t), ("commit", at[f"scores{t & 1}"]))

    def after(t, follows):
        out = [("wait", at[f"weights{t & 1}"], t >> 1), ("product", "PV", t)]
        if last[t]:
            out.append(("commit", at["result"]))
        for what in order:
            if what == "summed":
                out.append(("commit", sums(t)[0]))
            elif follows:
                out += scores(t + 2)
        return tuple(out) + (("next",),)

    def softmax(t, moves):
        out = [("wait", at[f"scores{t & 1}"], t >> 1)]
        out += [("wait", *sums(t - back)) for back in every if t >= back]
        out.append(("read", t))
        if moves:
            out += [("wait", *sums(t - back)) for back in rescale if t >= back]
            out.append(("rescale", t))
        out.append(("arrive", at[f"weights{t & 1}"]))
        if last[t]:
            out.append(("wait", at["result"], piece_of[t]))
            out.append(("rescale", t + 1))  # O of the piece is read: its sums are all there
        return tuple(out)

    # issuer: (task, scores asked for, script); pipe: (products asked for, how many have finished);
    # commits on their way: (barrier, products ahead of it); phases that are over; softmax: (tile, script)
    start = ((0, 0, ()), (), 0, (), (0,) * len(names), (0, ()))
    seen, todo = {start}, [start]

    def passes(counts, barrier, phase):
        if counts[barrier] & 1 == phase & 1:
            return False  # the phase of this parity is the one that is open
        if counts[barrier] != phase + 1:
            raise Wrong(f"a wait for phase {phase} of {names[barrier]} passed where {counts[barrier]} were over")
        return True

    def following(state):
        (task, asked, script), products, done, commits, counts, (tile, mine) = state
        if done < len(products):
            yield ((task, asked, script), products, done + 1, commits, counts, (tile, mine))
        for i, (barrier, ahead) in enumerate(commits):
            if ahead <= done:
                more = counts[:barrier] + (counts[barrier] + 1,) + counts[barrier + 1:]
                yield ((task, asked, script), products, done, commits[:i] + commits[i + 1:], more, (tile, mine))
        if script:
            head, rest = script[0], script[1:]
            if head[0] == "wait":
                if passes(counts, head[1], head[2]):
                    yield ((task, asked, rest), products, done, commits, counts, (tile, mine))
            elif head[0] == "product":
                yield ((task, asked + (head[1] == "S"), rest), products + (head[1:],), done, commits, counts, (tile, mine))
            elif head[0] == "commit":
                yield ((task, asked, rest), products, done, commits + ((head[1], len(products)),), counts, (tile, mine))
            else:
                yield ((task + 1, asked, rest), products, done, commits, counts, (tile, mine))
        elif task < tiles:
            if asked < min(task + 2, tiles):  # asked for early if its operands are there; at once if nothing can be done without
                yield ((task, asked, scores(asked)), products, done, commits, counts, (tile, mine))
            if asked > task:
                yield ((task, asked, after(task, False)), products, done, commits, counts, (tile, mine))
                if asked == task + 2 and asked < tiles:
                    yield ((task, asked, after(task, True)), products, done, commits, counts, (tile, mine))
        if mine:
            head, rest = mine[0], mine[1:]
            to = (tile, rest) if rest else (tile + 1, ())
            if head[0] == "wait":
                if passes(counts, head[1], head[2]):
                    yield ((task, asked, script), products, done, commits, counts, to)
            elif head[0] == "arrive":
                more = counts[:head[1]] + (counts[head[1]] + 1,) + counts[head[1] + 1:]
                yield ((task, asked, script), products, done, commits, more, to)
            else:
                if head[0] == "read":
                    written = [t for kind, t in products[:done] if kind == "S" and t & 1 == head[1] & 1]
                    if not written or written[-1] != head[1] or ("S", head[1] + 2) in products:
                        raise Wrong(f"the scores of tile {head[1]} are not the ones that are read")
                elif any(("PV", t) not in products[:done] for t in range(head[1])):
                    raise Wrong(f"O is rescaled at tile {head[1]} before the sums ahead of it were added")
                yield ((task, asked, script), products, done, commits, counts, to)
        elif tile < tiles:
            for moves in (False, True):
                if not (moves and first[tile]):
                    yield ((task, asked, script), products, done, commits, counts, (tile, softmax(tile, moves)))

    while todo:
        state = todo.pop()
        onward = list(following(state))
        if not onward and (state[0][0] < tiles or state[5][0] < tiles or state[3]):
            raise Wrong(f"nothing can go on: {state}")
        for to in onward:
            if to not in seen:
                seen.add(to)
                todo.append(to)
    return len(seen)


@pytest.mark.parametrize("pieces", [[1], [6], [2, 3], [1, 1, 3], [4, 2]], ids=str)
def test_a_rescale_waits_for_the_sums_ahead_of_it(pieces):
    text = SOURCE.read_text()
    every, rescale = softmax_waits(text)
    assert rescale == (1,)  # the sums of the tile before
    assert explore(pieces, issuer_order(text), barriers_of_sums(text), every, rescale) > sum(pieces)


@pytest.mark.parametrize("order,barriers,every,rescale", [
    # scores asked for ahead of the sums' commit, and phases of the sums that nobody waits for
    (("scores", "summed"), 1, (), (1,)),
    # the commit first, or two barriers: the arrivals of two commits are in no order
    (("summed", "scores"), 1, (), (1,)),
    (("summed", "scores"), 2, (), (1,)),
    # no wait before a rescale
    (("summed", "scores"), 2, (2,), ()),
    # a wait for a phase of the one barrier that may be over together with the next one
    (("summed", "scores"), 1, (2,), (1,))])
def test_the_model_finds_orders_that_are_wrong(order, barriers, every, rescale):
    with pytest.raises(Wrong):
        explore([6], order, barriers, every, rescale)
