"""The handoff of S and M in the prompt scan, in every order that its warps can take.

A model of the barriers between the warp that issues products and the warps that turn
S into M: one of those that have blocks of M, and the one that has none.  Products run
in order; a wait passes when the parity of the phase it asks for is over, as an
mbarrier's does.  Checked in each reachable state: a product only starts on operands
that are all there, nothing in use is written, and nobody is stuck."""

import pytest

CHUNKS = 4
WARPS = ("blocks", "none")


def issue_steps():
    for c in range(-1, CHUNKS):
        if c + 1 < CHUNKS:
            if c >= 0:
                yield "wait", "SEmpty", c
            yield "product", "S", c + 1
        if c >= 0:
            yield "wait", "MFull", c
            yield "product", "Y", c


def warp_steps(warp, last_m_waited):
    for c in range(CHUNKS):
        yield "wait", "SFull", c
        if warp == "blocks":
            yield "read", "S", c
        yield "arrive", "SEmpty", c
        if c > 0 and (warp == "blocks" or last_m_waited):
            yield "wait", "YFull", c - 1
        if warp == "blocks":
            yield "write", "M", c
        yield "arrive", "MFull", c


def explore(last_m_waited):
    """The first fault found, or None."""
    programs = [list(issue_steps())] + [list(warp_steps(w, last_m_waited)) for w in WARPS]
    needs = {"SEmpty": len(WARPS), "MFull": len(WARPS), "SFull": 1, "YFull": 1}
    names = sorted(needs)
    start = ((0,) * len(programs), (), tuple((0, 0) for _ in names))   # places, products, barriers
    seen, todo = {start}, [start]

    def arrived(bars, name):
        i = names.index(name)
        phase, count = bars[i]
        count += 1
        bar = (phase + 1, 0) if count == needs[name] else (phase, count)
        return bars[:i] + (bar,) + bars[i + 1:]

    def done(places, who, step):
        return step in programs[who][:places[who]]

    while todo:
        places, products, bars = todo.pop()
        following = []
        if products:                                   # the oldest product ends
            kind, c = products[0]
            if kind == "S" and c > 0 and not done(places, 1, ("read", "S", c - 1)):
                return f"S {c} over S {c - 1} that is still to be read"
            if kind == "Y" and not done(places, 1, ("write", "M", c)):
                return f"Y {c} from an M that is not there"
            following.append((places, products[1:], arrived(bars, kind + "Full")))
        for who, program in enumerate(programs):
            if places[who] == len(program):
                continue
            kind, what, c = program[places[who]]
            moved = places[:who] + (places[who] + 1,) + places[who + 1:]
            if kind == "wait":
                if bars[names.index(what)][0] & 1 != c & 1:
                    following.append((moved, products, bars))
            elif kind == "product":
                following.append((moved, products + ((what, c),), bars))
            elif kind == "arrive":
                following.append((moved, products, arrived(bars, what)))
            else:
                if kind == "write" and c > 0 and (
                        ("Y", c - 1) in products or not done(places, 0, ("product", "Y", c - 1))):
                    return f"M {c} over M {c - 1} that is in use"
                following.append((moved, products, bars))
        if not following and any(n < len(p) for n, p in zip(places, programs)):
            return f"stuck at {places}"
        for state in following:
            if state not in seen:
                seen.add(state)
                todo.append(state)
    return None


@pytest.mark.parametrize("last_m_waited", [True, False])
def test_m_is_whole_before_its_product(last_m_waited):
    """The kernel's order is sound; without the blockless warp's wait for the last chunk's
    product it was not: that warp arrived twice in one phase."""
    fault = explore(last_m_waited)
    assert (fault is None) == last_m_waited, fault
