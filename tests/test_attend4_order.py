"""The hand-overs between the roles of k_attend4, walked through in every order on the CPU.

A wait by parity cannot tell a phase from the one two further on. Here the widening, the two issuing
warps, the tensor pipe and the softmax are programs of waits and arrivals, as in the kernel's source,
with the barriers and parities that k3_attend4_order.h gives; every interleaving of them is visited.
In none may a wait pass before its phase, a barrier flip a second time under a wait, a buffer be
written while it is read, or the roles come to a stand."""
import ctypes
import os
import subprocess
import tempfile

import pytest

from conftest import PKG


@pytest.fixture(scope="module")
def order():
    """(buf, phase) as the kernel has them."""
    d = tempfile.mkdtemp()
    src, so = os.path.join(d, "o.c"), os.path.join(d, "o.so")
    open(src, "w").write('#include "k3_attend4_order.h"\n'
                         "int buf(int g) { return at4_buf(g); }\nunsigned phase(int g) { return at4_phase(g); }\n")
    subprocess.run(["gcc", "-O1", "-shared", "-fPIC", "-I", os.path.join(PKG, "csrc"), src, "-o", so], check=True)
    lib = ctypes.CDLL(so)
    lib.phase.restype = ctypes.c_uint
    return lib.buf, lib.phase


def programs(items, pieces, buf, phase, pbuf, pphase):
    """Each role as a list of steps: ("wait", barrier, phase it means, parity), ("flip", barrier), ("send",
    queue, step of the pipe), ("join", n-th meeting), ("write" / "read", what, tile), ("maybe", steps).
    items: (tiles, P is held for two tiles)."""
    def nth(g, b=buf):                    # how often tile g's barrier has flipped before tile g flips it
        return sum(b(i) == b(g) for i in range(g))

    def wait(name, g, tag=""):
        if name == "P":
            return ("wait", ("P", pbuf(g)), nth(g, pbuf), pphase(g))
        return ("wait", (name, buf(g), tag), nth(g), phase(g))

    def flip(name, g, tag=""):
        return ("flip", ("P", pbuf(g)) if name == "P" else (name, buf(g), tag))

    last = pieces - 1
    W, S, O, M = [], [], [], []
    g = 0
    for k, (tiles, two) in enumerate(items):
        for t in range(tiles):
            for h in range(pieces):
                if g >= 2:
                    W.append(wait("PV", g - 2, h))
                W += [("write", ("tile", buf(g), h), g), flip("K", g, h)]
            if g >= 2:
                S.append(wait("SF", g - 2))
            S += [wait("K", g, h) for h in range(pieces)]
            S.append(("send", "s", [("read", ("tile", buf(g), h), g) for h in range(pieces)]
                      + [("write", ("S", buf(g)), g), flip("S", g)]))
            O.append(wait("P", g))
            region = ("P", buf(g) if two else "whole")
            steps = [("read", region, g)]
            for h in range(pieces):
                steps += [("read2", ("tile", buf(g), h), g), flip("PV", g, h)]
            O.append(("send", "o", steps))
            M += [wait("K", g, last), wait("S", g), ("read", ("S", buf(g)), g), flip("SF", g)]
            before = [wait("PV", g - 1, last)] if t > 0 else []
            if not two:
                M += before
            M.append(("write", region, g))
            if two and before:
                M.append(("maybe", before))          # the accumulator is rescaled, or not
            M.append(flip("P", g))
            g += 1
        if tiles:
            M.append(wait("PV", g - 1, last))
        W.append(("join", k))
        M.append(("join", k))
    return W, S, O, M


class Fault(Exception):
    pass


def explore(items, pieces, buf, phase, pbuf=None, pphase=None):
    """Visits every state; raises Fault, else returns how many there are."""
    progs = programs(items, pieces, buf, phase, pbuf or buf, pphase or phase)
    done_at = [len(p) for p in progs]
    # every flip has one place in one program, so a state is the roles' places and how far each queue
    # of the pipe has come
    queues = {"s": [x for p in progs for x in p if x[0] == "send" and x[1] == "s"],
              "o": [x for p in progs for x in p if x[0] == "send" and x[1] == "o"]}
    flat = {q: [s for x in v for s in x[2]] for q, v in queues.items()}
    ends = {q: [sum(len(x[2]) for x in v[:i + 1]) for i in range(len(v))] for q, v in queues.items()}

    def past(pcs, qs):
        """Steps of the four programs and of the pipe that are over."""
        for p, pc in zip(progs, pcs):
            yield from p[:pc]
        yield from flat["s"][:qs[0]]
        yield from flat["o"][:qs[1]]

    cache = {}

    def flips(pcs, qs):
        key = (pcs, qs)
        if key not in cache:
            n, w, r, r2 = {}, {}, {}, {}
            for x in past(pcs, qs):
                if x[0] == "flip":
                    n[x[1]] = n.get(x[1], 0) + 1
                elif x[0] in ("write", "read", "read2"):
                    {"write": w, "read": r, "read2": r2}[x[0]].setdefault(x[1], set()).add(x[2])
            cache.clear()
            cache[key] = (n, w, r, r2)
        return cache[key]

    def check_write(x, pcs, qs):
        """What is written must have been read by everyone it was for."""
        n, w, r, r2 = flips(pcs, qs)
        what = x[1]
        over = [what] if what[0] != "P" else [("P", 0), ("P", 1), ("P", "whole")] if what[1] == "whole" else [what, ("P", "whole")]
        for o in over:
            for g in w.get(o, ()):
                if g not in r.get(o, ()) or (o[0] == "tile" and g not in r2.get(o, ())):
                    raise Fault("%s of tile %d written over before it was read" % (o, g))

    start = ((0, 0, 0, 0), (0, 0))
    seen, todo = {start}, [start]
    while todo:
        pcs, qs = todo.pop()
        n, w, r, r2 = flips(pcs, qs)
        sent = [sum(x[0] == "send" for x in progs[i][:pcs[i]]) for i in (1, 2)]
        nxt = []

        def passes(x):
            count = n.get(x[1], 0)
            ok = (count & 1) != x[3]
            if ok and count <= x[2]:
                raise Fault("a wait for phase %d of %s passes at %d" % (x[2], x[1], count))
            if count > x[2] + 1:
                raise Fault("%s flips again under the wait for phase %d" % (x[1], x[2]))
            return ok

        for i in range(4):
            if pcs[i] == done_at[i]:
                continue
            x = progs[i][pcs[i]]
            step = tuple(pc + (k == i) for k, pc in enumerate(pcs))
            if x[0] == "wait":
                if passes(x):
                    nxt.append((step, qs))
            elif x[0] == "maybe":
                nxt.append((step, qs))
                if passes(x[1][0]):
                    nxt.append((step, qs))
            elif x[0] == "join":
                if i == 0 and pcs[3] < done_at[3] and progs[3][pcs[3]] == x:
                    nxt.append(((pcs[0] + 1, pcs[1], pcs[2], pcs[3] + 1), qs))
            else:
                if x[0] == "write":
                    check_write(x, pcs, qs)
                nxt.append((step, qs))
        for k, q in enumerate("so"):
            limit = ends[q][sent[k] - 1] if sent[k] else 0
            if qs[k] < limit:
                x = flat[q][qs[k]]
                if x[0] == "write":
                    check_write(x, pcs, qs)
                nxt.append((pcs, tuple(v + (j == k) for j, v in enumerate(qs))))
        if not nxt and list(pcs) != done_at:
            raise Fault("the roles stand at %s" % [p[pc] if pc < len(p) else "end" for p, pc in zip(progs, pcs)])
        for s in nxt:
            if s not in seen:
                seen.add(s)
                todo.append(s)
    return len(seen)


CASES = [[(6, True)], [(6, False)], [(1, True), (3, False), (2, True)], [(3, False), (3, True)], [(2, True), (0, True), (3, True)],
         [(3, True), (1, False), (0, False), (2, False)]]


@pytest.mark.parametrize("pieces", [1, 2])
@pytest.mark.parametrize("items", CASES)
def test_no_order_of_the_roles_goes_wrong(order, items, pieces):
    assert explore(items, pieces, *order) > 50


def test_one_barrier_for_both_p_is_found(order):
    """The walk notices the order that a barrier shared by two P allows, and only where P is held
    for two tiles."""
    buf, phase = order
    with pytest.raises(Fault, match="flips again"):
        explore([(4, True)], 2, buf, phase, lambda g: 0, lambda g: g & 1)
    assert explore([(4, False)], 2, buf, phase, lambda g: 0, lambda g: g & 1) > 50


def test_other_mistakes_are_found(order):
    buf, phase = order
    with pytest.raises(Fault):
        explore([(5, True)], 2, buf, lambda g: g & 1)
    with pytest.raises(Fault):
        explore([(5, True)], 2, lambda g: 0, phase)
