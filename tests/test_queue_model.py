"""Model checking of where the engines' flag waits are enqueued
(csrc/hip/mesh.cc waitFlag), over every kind of sharing of hardware queues.

A GPU runs each hardware queue's packets in order, and HIP maps streams onto
few of them: a wait at a queue's head holds up whatever is behind it, of other
streams too. The schedules are those of test_doorbell_model.py, which mirror
what the engines enqueue, in the order in which a rank's host does it; here
they go through queues that streams share at random.

Ranks of one process on one GPU share its queues. There the host waits and
enqueues nothing that is not ready. A rank alone with its queues leaves the
waiting to the device.
"""
import random

import pytest

from test_doorbell_model import (enqueue_direct_run, enqueue_hd_run,
                                 enqueue_run)


class Recorder:
    """Takes the schedules' streams, and keeps each rank's ops in the order
    in which its host enqueues them."""

    def __init__(self):
        self.programs = {}

    def stream(self, key):
        rank, sid = key
        program = self.programs.setdefault(rank, [])

        class Stream:
            @staticmethod
            def append(op):
                program.append((sid, op))

        return Stream


class Deadlock(Exception):
    pass


def waits_for_peer(op):
    """Not for this rank's own events (EV, CE), nor for its streams (RB)."""
    return op[0] == "wait" and op[2][0] not in ("EV", "CE", "RB")


def execute(programs, queue_of, host_waits, rng):
    """Hosts enqueue and queues run, one step of any of them at a time."""
    flags, queues = {}, {}
    at = {r: 0 for r in programs}

    def ready(op):
        return op[0] != "wait" or flags.get((op[1], op[2]), 0) >= op[3]

    def host(r):
        if at[r] == len(programs[r]):
            return False
        sid, op = programs[r][at[r]]
        # a run ends when its streams are done: the host waits for them
        ends = op[0] == "wait" and op[2][0] == "RB"
        if (ends or host_waits and waits_for_peer(op)) and not ready(op):
            return False
        queues.setdefault(queue_of(r, sid), []).append(op)
        at[r] += 1
        return True

    def queue(q):
        if not queues[q] or not ready(queues[q][0]):
            return False
        op = queues[q].pop(0)
        if op[0] == "write":
            flags[op[1], op[2]] = max(flags.get((op[1], op[2]), 0), op[3])
        return True

    while True:
        steps = [(host, r) for r in at] + [(queue, q) for q in queues]
        rng.shuffle(steps)
        # one that can goes on for a while: ranks and queues drift apart
        for f, arg in steps:
            n = rng.choice((1, 3, 30))
            if f(arg):
                while n > 1 and f(arg):
                    n -= 1
                break
        else:
            break
    left = {q: ops[0] for q, ops in queues.items() if ops}
    if left or any(at[r] < len(programs[r]) for r in at):
        raise Deadlock(left)


def ring(P, strides, runs=2):
    rec, seq, last = Recorder(), 0, {}
    for r in range(P):
        for j in range(len(strides)):
            for par in (0, 1):
                last[r, j, par] = 0
    for i in range(runs):
        ks = enqueue_run(rec, P, strides, 4000, 4, 4096, seq, last, i)
        seq += max(ks.values())
    return rec.programs


def hd(P, runs=2):
    rec, state = Recorder(), {}
    for i in range(runs):
        enqueue_hd_run(rec, P, 3000, 4, 4096, state, i)
    return rec.programs


def direct(P, chunks, runs=2):
    rec, state = Recorder(), {}
    for i in range(runs):
        enqueue_direct_run(rec, P, chunks, state, i)
    return rec.programs


SCHEDULES = {
    "ring2": lambda: ring(2, [1]), "ring3": lambda: ring(3, [1, 2]),
    "ring4": lambda: ring(4, [1, 3]), "hd2": lambda: hd(2),
    "hd3": lambda: hd(3), "hd4": lambda: hd(4), "hd5": lambda: hd(5),
    "direct2": lambda: direct(2, 3), "direct4": lambda: direct(4, 3),
}


def mapping(programs, queues, shared, rng):
    """Streams to queues, by chance: one set of them for all ranks, or one
    for each."""
    streams = sorted({(r, sid) for r, p in programs.items()
                      for sid, _ in p})
    to = {s: rng.randrange(queues) for s in streams}
    return lambda r, sid: (0 if shared else r, to[r, sid])


@pytest.mark.parametrize("name", SCHEDULES)
def test_host_waits_go_with_any_queues(name):
    """Several ranks on one set of queues, from one queue for all streams to
    as many as there are."""
    programs = SCHEDULES[name]()
    for seed in range(30):
        rng = random.Random(seed)
        execute(programs, mapping(programs, 1 + seed % 8, True, rng), True,
                rng)


@pytest.mark.parametrize("name", SCHEDULES)
def test_device_waits_need_a_rank_alone(name):
    """One set of queues for each rank: any sharing within it will do. One
    set for several ranks deadlocks where their streams meet."""
    programs = SCHEDULES[name]()
    for seed in range(30):
        rng = random.Random(seed)
        execute(programs, mapping(programs, 1 + seed % 4, False, rng), False,
                rng)
    with pytest.raises(Deadlock):
        for seed in range(30):
            rng = random.Random(seed)
            execute(programs, mapping(programs, 2, True, rng), False, rng)


# ------------------------------------------------------------ point to point


class Pair:
    """Two ranks that post a send and a receive each, then flush. `ahead`:
    posts enqueue all their chunks, and the device waits; otherwise chunks go
    to their stream when their flag is there, in posts and flushes
    (HipP2P::enqueueReady)."""

    def __init__(self, orders, chunks, ahead, queue_of, rng):
        self.ahead, self.queue_of, self.rng = ahead, queue_of, rng
        self.flags, self.queues = {}, {}
        self.posted = [{"send": [], "recv": []} for _ in range(2)]
        self.todo = [[(kind, s) for kind in order
                      for s in range(1, chunks + 1)] for order in orders]

    def enqueue(self, r, kind, seq):
        q = self.queues.setdefault(self.queue_of(r, kind), [])
        if kind == "recv":
            q.append(("wait", (r, "DATA"), seq))
            q.append(("write", (1 - r, "ACK"), seq))
        else:
            if seq > 2:
                q.append(("wait", (r, "ACK"), seq - 2))
            q.append(("write", (1 - r, "DATA"), seq))

    def ready(self, r, kind, seq):
        flag, value = ("DATA", seq) if kind == "recv" else ("ACK", seq - 2)
        return value <= 0 or self.flags.get((r, flag), 0) >= value

    def enqueue_ready(self, r):
        moved = False
        for kind, posted in self.posted[r].items():
            while posted and (self.ahead or self.ready(r, kind, posted[0])):
                self.enqueue(r, kind, posted.pop(0))
                moved = True
        return moved

    def host(self, r):
        if self.todo[r]:  # posts do not block
            kind, seq = self.todo[r].pop(0)
            self.posted[r][kind].append(seq)
            return True
        return self.enqueue_ready(r)  # a flush of either kind

    def queue(self, q):
        ops = self.queues[q]
        if not ops or (ops[0][0] == "wait"
                       and self.flags.get(ops[0][1], 0) < ops[0][2]):
            return False
        op = ops.pop(0)
        if op[0] == "write":
            self.flags[op[1]] = max(self.flags.get(op[1], 0), op[2])
        return True

    def run(self):
        while True:
            steps = [(self.host, r) for r in (0, 1)] + [
                (self.queue, q) for q in self.queues]
            self.rng.shuffle(steps)
            if not any(f(arg) for f, arg in steps):
                break
        if (any(self.queues.values()) or any(
                v for p in self.posted for v in p.values())):
            raise Deadlock


@pytest.mark.parametrize("chunks", [1, 2, 5, 9])
def test_point_to_point(chunks):
    orders = [("send", "recv"), ("recv", "send")]
    for seed in range(200):
        rng = random.Random(seed)
        pick = [rng.choice(orders) for _ in range(2)]
        to = {(r, k): rng.randrange(1 + seed % 4) for r in (0, 1)
              for k in ("send", "recv")}
        Pair(pick, chunks, False, lambda r, k: to[r, k], rng).run()


def test_point_to_point_ahead_needs_two_queues_a_rank():
    """Where the device waits, a rank's sends and receives must not share a
    queue (they do not as long as there are queues enough)."""
    rng = random.Random(0)
    for order in ("send", "recv"), ("recv", "send"):
        Pair([order] * 2, 5, True, lambda r, k: (r, k), rng).run()
        with pytest.raises(Deadlock):
            Pair([order] * 2, 5, True, lambda r, k: r, rng).run()
