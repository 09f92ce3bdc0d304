"""Work slots of the attention kernel whose CTAs take several work items, on the CPU: sequences without keys between others must not
leave its roles waiting for one another.

The issuer's own code is replayed (see test_flash_persistent_issuer_cpu.py); the other roles are played here as far as slots go.  The
loader puts item n (and behind the last one the end) where item n - 4 was once every role has given that back.  The softmax warps, the warp that clears tiles and the
issuer give an item back when they read it, the result warps too, but they read one only when the O of every item with keys before it
is final, and the softmax warps one only when they have been given all scores of those."""
import os
import random
import re
import shutil
import subprocess

import pytest

from tests.test_flash_persistent_issuer_cpu import CSRC, STUBS, _block

SLOTS = 4


@pytest.fixture(scope="module")
def replay(tmp_path_factory):
    """The issuer against the stubs of that test, the end of the work as an event too: it takes a slot like an item."""
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no host compiler")
    kernel, common = (open(os.path.join(CSRC, name)).read() for name in ("flash_fwd_persistent_sm100.cu", "flash_common.cuh"))
    constants = "\n".join(line for text in (common, kernel) for line in re.findall(r"^constexpr int \w+ = [^;]*;", text, re.M))
    structs = "\n".join(f"struct {n} " + _block(kernel, kernel.index(f"struct {n} {{")) + ";" for n in ("C", "Item"))
    issuer = _block(kernel, kernel.index("if (elect_one())", kernel.index("- MMA issuer")))
    stubs = STUBS.replace("if (at >= argc) return -1;", 'if (at >= argc) { std::printf("item %%d -1\\n", slot); return -1; }')
    assert stubs != STUBS
    d = tmp_path_factory.mktemp("slots")
    src, exe = str(d / "issuer.cpp"), str(d / "issuer")
    with open(src, "w") as f:
        f.write(stubs % dict(constants=constants, structs=structs, issuer=issuer))
    r = subprocess.run([gxx, "-std=c++17", "-O0", "-w", src, "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr

    def run(items):
        r = subprocess.run([exe] + [str(k) for k in items], capture_output=True, text=True)
        assert r.returncode == 0
        return [line.split() for line in r.stdout.splitlines()]
    return run


def _play(events, items):
    """Goes through the issuer's events; an item that it waits for has to be one that the loader can have published by then."""
    keyed = [k > 0 for k in items]
    units = [2 * -(-k // 128) for k in items]
    fetched, finals, scores, given = 0, 0, 0, [0] * len(items)

    def read_by_results(n):                # the result warps have got as far as item n
        return finals >= sum(keyed[:n])

    def read_by_softmax(n):
        return scores >= sum(units[:n])

    for e in events:
        if e[0] == "item":
            n = fetched - SLOTS
            if n >= 0:
                assert given[n], f"the issuer has not given item {n} back"
                assert read_by_results(n), f"item {fetched} waits for the results of item {n}, which wait for the issuer"
                assert read_by_softmax(n), f"item {fetched} waits for the softmax warps at item {n}, which wait for scores"
            fetched += 1
        elif e[:2] == ["commit", "o_final"] and e[2] == "1":
            finals += 1
        elif e[:2] == ["commit", "s_full"]:
            scores += 1
        elif e[:2] == ["arrive", "work_empty"]:
            # slots are given back in the items' order, each once
            n = given.index(0)
            assert n < fetched and int(e[2]) == n % SLOTS
            given[n] = 1
    assert fetched == len(items) + 1 and all(given) and finals == sum(keyed) and scores == sum(units)


RUNS = [[700] + [0] * n for n in range(1, 12)] + [[1] + [0] * 9 + [1], [0] * 9 + [300] + [0] * 9, [128] + [0] * 5 + [129] + [0] * 6 + [17],
        [2222, 0, 0, 0, 0, 1, 0, 0, 0, 0, 0, 391], [300, 300, 300] + [0] * 20 + [300, 1, 1, 1, 1, 1, 1], [0] * 30]


@pytest.mark.parametrize("items", RUNS, ids=str)
def test_runs_of_sequences_without_keys_pass(replay, items):
    _play(replay(items), items)


@pytest.mark.parametrize("seed", range(8))
def test_any_mixture_passes(replay, seed):
    rng = random.Random(seed)
    items = []
    while len(items) < 60:
        items += [rng.choice((1, 16, 100, 128, 129, 300, 391, 640))] * rng.randrange(4) + [0] * rng.randrange(12)
    _play(replay(items), items)


@pytest.mark.parametrize("items", RUNS + [[300, 0, 300], [300, 0], [1, 0, 1, 0, 0, 1, 300, 0, 0, 0, 0, 0, 128, 17]], ids=str)
def test_units_run_through_items_behind_those(replay, items):
    """The phases and the S buffers in turn, whichever way an item was come by; behind the last PV of all there is only o_final."""
    ev = replay(items)
    tiles = [-(-k // 128) for k in items if k]
    units = 2 * sum(tiles)
    waits = lambda name: [(int(e[2]), int(e[3])) for e in ev if e[:2] == ["wait", name]]
    commits = lambda name: [int(e[2]) for e in ev if e[:2] == ["commit", name]]
    turn = lambda n, size: [(i % size, (i // size) & 1) for i in range(n)]
    assert waits("kv_full") == turn(units, 8) and waits("p_lo") == waits("p_hi") == turn(units, 3)
    assert waits("q_full") == [(2 * (i % 2) + t, (i // 2) & 1) for i in range(len(tiles)) for t in range(2)]
    assert waits("o_free") == [(t, (i - 1) & 1) for i in range(1, len(tiles)) for t in range(2)]
    assert commits("s_full") == [u % 3 for u in range(units)] and commits("q_empty") == [i % 2 for i in range(len(tiles))]
    assert commits("o_final") == [0, 1] * len(tiles)
    if not units:
        return
    # (each phase of a barrier once, in its order; the very last V and the last PVs have none)
    assert commits("pv_done") == [0, 1] * (units // 2 - 1)
    assert sorted(commits("kv_empty")) == sorted(i % 8 for i in range(units - 1))
    last_mma = max(i for i, e in enumerate(ev) if e[0] in ("S", "PV"))
    assert [e[:2] for e in ev[last_mma + 1:] if e[0] == "commit"] == [["commit", "o_final"]]
    # S of a unit is behind the PV whose P lay in its buffer, and reads its own item's queries
    s_seen = pv_seen = 0
    for e in ev:
        if e[:2] == ["commit", "s_full"]:
            assert s_seen < 3 or pv_seen > s_seen - 3
            s_seen += 1
        if e[:2] == ["wait", "p_hi"]:
            pv_seen += 1
    of = [i for i, n in enumerate(tiles) for _ in range(2 * n)]
    s = [e for e in ev if e[0] == "S"]
    assert [int(e[1]) for e in s] == [u % 3 * 128 for u in range(units) for _ in range(4)]
    first = {0: 0}
    for u in range(units):
        first.setdefault(of[u], u)
        tile = 2 * (of[u] % 2) + (u - first[of[u]]) % 2
        assert int(s[4 * u][2]) == tile * (128 * 64 * 2 >> 4)
