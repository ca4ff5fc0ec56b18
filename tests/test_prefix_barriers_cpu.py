"""The barrier protocol of the prefix pass (tritiercache_b200/csrc/tt_prefix_shared.cuh), in every interleaving.

The thread that issues the products, the softmax warps of both accumulators (two warps each, one of which may lag) and
the tensor cores, whose commits arrive in order and at any time after they were issued, each run a fixed list of
arrivals and waits over the spans of one CTA.  An mbarrier wait knows no more than a phase's parity.  Every reachable
state is visited: none may be stuck, no wait may pass before its own phase has completed, and no queries may be
replaced while a product reads them.
"""
import itertools

import pytest


def programs(pair, tiles, all_arrive=True, wait_when_idle=True):
    """[(barrier, arrivals a phase)] and the agents' programs: ("a", barrier), ("w", barrier), ("c", barrier) for a
    commit, ("n", barrier) for a phase nobody of the agent looks at, ("q", commits) for new queries, which every product up
    to that many commits must have left alone."""
    look = 1 if pair else 2
    count = {"q": 4 if all_arrive or pair else 2, "s0": 1, "s1": 1, "p00": 2, "p01": 2, "p10": 2, "p11": 2}
    issue, reads = [], []

    def commits():
        return sum(op == "c" for op, _ in issue)

    for n in tiles:
        issue.append(("w", "q"))
        last_qk = 0
        for i in range(min(look, n)):
            for t in (0, 1) if pair else (i,):
                issue.append(("c", f"s{t}"))
                last_qk = commits()
        for j in range(n):
            for t in (0, 1) if pair else (j & 1,):
                issue += [("w", f"p{t}0"), ("w", f"p{t}1"), ("c", f"s{t}")]
                if j + look < n:  # the next first product goes before this commit
                    last_qk = commits()
        reads.append(last_qk)
    agents = [issue]
    for t, _ in itertools.product((0, 1), (0, 1)):
        ops = []
        for k, n in enumerate(tiles):
            mine = n if pair else (n - t + 1) // 2
            if pair or t == 0:
                ops.append(("q", reads[k - 1] if k else 0))
            if all_arrive or pair or t == 0:
                ops += [("a", "q"), ("w" if mine == 0 and wait_when_idle else "n", "q")]
            for _ in range(mine):
                ops += [("w", f"s{t}"), ("a", f"p{t}0"), ("a", f"p{t}1")]
            if mine:
                ops.append(("w", f"s{t}"))
        agents.append(ops)
    return count, agents


def explore(count, agents):
    """What goes wrong in some interleaving, or None."""
    names = list(count)
    # per agent and position: arrivals made on each barrier, waits made before (a skipped wait, "n", counts as one)
    arrived = [[{b: sum(op == "a" and x == b for op, x in ops[:i]) for b in names} for i in range(len(ops) + 1)] for ops in agents]
    waits = [[sum(op in "wn" and x == ops[i][1] for op, x in ops[:i]) if i < len(ops) else 0 for i in range(len(ops) + 1)]
             for ops in agents]
    commits = [[x for op, x in agents[0][:i] if op == "c"] for i in range(len(agents[0]) + 1)]
    start = (0,) * (len(agents) + 1)  # positions, commits that have arrived
    end = tuple(len(ops) for ops in agents) + (len(commits[-1]),)
    seen, todo = {start}, [start]
    while todo:
        at = todo.pop()
        done = at[-1]
        total = {b: sum(arrived[a][at[a]][b] for a in range(len(agents))) + sum(x == b for x in commits[-1][:done]) for b in names}
        moved = False
        for a, ops in enumerate(agents):
            if at[a] == len(ops):
                continue
            op, x = ops[at[a]]
            if op == "w":
                k = waits[a][at[a]]  # this wait is for phase k
                complete = total[x] // count[x]
                if (complete - 1) % 2 != k % 2:  # the parity of the last completed phase (phase -1 passes parity 1)
                    continue
                short = [i for i, o in enumerate(agents) if ("a", x) in o and arrived[i][at[i]][x] <= k]
                if complete <= k or short:
                    return f"agent {a} passes {x} phase {k} of {complete} without {short}"
            if op == "q" and done < x:
                return f"agent {a} replaces queries that are read"
            moved = True
            nxt = at[:a] + (at[a] + 1,) + at[a + 1:]
            if nxt not in seen:
                seen.add(nxt)
                todo.append(nxt)
        if done < len(commits[at[0]]):
            moved = True
            nxt = at[:-1] + (done + 1,)
            if nxt not in seen:
                seen.add(nxt)
                todo.append(nxt)
        if not moved and at != end:
            return f"stuck at {at}"
    assert end in seen
    return None


SPANS = [t for n in (1, 2, 3) for t in itertools.product((1, 2, 3) if n < 3 else (1, 2), repeat=n)] + [(4, 1, 3), (5, 4)]


@pytest.mark.parametrize("pair", [False, True])
def test_no_interleaving_is_stuck_or_early(pair):
    for tiles in SPANS:
        assert explore(*programs(pair, tiles)) is None, tiles


def test_the_model_sees_arrivals_that_are_missing():
    # one span is sound without accumulator 1's arrivals, a second one may overtake its late warp
    assert explore(*programs(False, (3,), all_arrive=False)) is None
    assert "stuck" in explore(*programs(False, (2, 2), all_arrive=False))
    # and a warp without a tile that does not wait arrives twice in a phase
    assert "without" in explore(*programs(False, (1, 2), wait_when_idle=False))
