"""CPU: the hand-over between prompt attention's load warp and its MMA thread as a small state machine, over every order of events.

Consecutive items of one key tile each, all of whose V tiles reach into another request: the case in which the load warp can run
furthest ahead.  A wait by parity passes when the phase that completed last has the awaited parity, so a waiter must never be two phases
behind."""
import os
import re

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "uniql_b200", "csrc", "prompt_attention.cu")
STAGES, ITEMS = 5, 6


def _explore(clean_bars):
    """Every reachable state; returns the states in which the MMA thread waits for a phase of `clean` that is two phases old."""
    # state: load pc, MMA pc, tiles landed (K and V of item k land as 2k, 2k + 1, in any order: a bit each), qfree committed
    # and arrived, clean arrivals.  load pc 3k: waits for the queries' place and the ring; 3k + 1: waits for V; 3k + 2: arrives.
    # MMA pc 3k: waits for K, then scores and commits qfree; 3k + 1: waits for V and the clearing; 3k + 2: values, ring places back.
    start = (0, 0, 0, 0, 0)                                       # load, mma, landed, issued tiles, qfree arrived
    seen, todo, stuck = {start}, [start], []
    while todo:
        load, mma, landed, issued, qfree = todo.pop()
        nxt = []
        k, at = divmod(load, 3)
        cleared = k                                               # arrivals so far: one per finished item
        freed = 2 * (mma // 3)                                    # ring places given back (at the end of each item)
        if k < ITEMS:
            if at == 0 and (k == 0 or qfree >= k) and issued + 2 - freed <= STAGES:
                nxt.append((load + 1, mma, landed, issued + 2, qfree))
            elif at == 1 and landed >> (2 * k + 1) & 1:
                nxt.append((load + 1, mma, landed, issued, qfree))
            elif at == 2:
                nxt.append((load + 1, mma, landed, issued, qfree))          # arrives on clean[k % clean_bars]
        for t in range(issued):
            if not landed >> t & 1:
                nxt.append((load, mma, landed | 1 << t, issued, qfree))
        j, at = divmod(mma, 3)
        if j < ITEMS:
            committed = j + (at > 0)                              # qfree commits behind the scores of items 0 .. committed - 1
            if qfree < committed:                                 # a commit arrives some time after it was made
                nxt.append((load, mma, landed, issued, qfree + 1))
            if at == 0 and landed >> (2 * j) & 1:
                nxt.append((load, mma + 1, landed, issued, qfree))
            elif at == 1 and landed >> (2 * j + 1) & 1:
                done = len([c for c in range(cleared) if c % clean_bars == j % clean_bars])
                want = j // clean_bars
                if done > want + 1:
                    stuck.append((load, mma))
                if (done & 1) != (want & 1):                      # the phase of the awaited parity is the last one completed
                    nxt.append((load, mma + 1, landed, issued, qfree))
            elif at == 2:
                nxt.append((load, mma + 1, landed, issued, qfree))
        for s in nxt:
            if s not in seen:
                seen.add(s)
                todo.append(s)
    assert any(s[1] == 3 * ITEMS for s in seen)                   # the work can end at all
    return stuck


def test_one_barrier_would_lose_a_phase():
    assert _explore(1)


def test_clearing_barriers_never_lose_a_phase():
    with open(SOURCE) as f:
        found = re.search(r"constexpr int kCleans = (\d+);", f.read())
    assert found and not _explore(int(found.group(1)))
