"""Order of the chunk weights kernel's column tables (kv4_mass_tc.cu), followed over every interleaving of two threads.

A thread's tile i: wait for both threads' arrivals for tile i - 2, write table i + 2, load the scores, arrive for tile i, read the
last part of table i.  A table may be overwritten only once nobody reads the tile that it belonged to."""
import os
import re

HERE = os.path.dirname(os.path.abspath(__file__))
TILES = 12


def _overwritten_while_read(tables):
    """Does some interleaving write a table that the other thread still has to read?"""
    steps = [(what, i) for i in range(TILES) for what in ("wait", "put", "arrive", "read")]
    arrived = [sum(1 for s in steps[:at] if s[0] == "arrive") for at in range(len(steps) + 1)]
    todo, seen = [(0, 0)], set()
    while todo:
        at = todo.pop()
        if at in seen:
            continue
        seen.add(at)
        for me in (0, 1):
            if at[me] == len(steps):
                continue
            what, i = steps[at[me]]
            other = at[1 - me]
            if what == "wait" and i >= 2 and arrived[other] < i - 1:
                continue
            if what == "put":
                # tables that the other thread has been given and not finished with: its current tile on, up to what is written
                current = other // 4
                if any(t % tables == (i + 2) % tables for t in range(current, i + 2)):
                    return True
            todo.append((at[0] + 1, at[1]) if me == 0 else (at[0], at[1] + 1))
    return False


def test_no_table_is_overwritten_while_it_is_read():
    with open(os.path.join(HERE, "..", "base-mlx_b200", "csrc", "kv4_mass_tc.cu")) as f:
        src = f.read()
    ring = re.search(r"constexpr int TABLES = (\d+);", src)
    slots = set(re.findall(r"\(i & ([^)]*\)?)\) \* 2 \* CM", src))
    assert ring and slots == {"(TABLES - 1)"}
    assert not _overwritten_while_read(int(ring.group(1)))


def test_the_model_finds_a_ring_that_is_too_short():
    assert _overwritten_while_read(4) and not _overwritten_while_read(5)
