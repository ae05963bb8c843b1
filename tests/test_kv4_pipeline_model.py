"""A CPU model of the hand-offs inside the two attention kernels over the 4-bit cache (csrc/kv4_prompt.cu, csrc/kv4_attention.cu):
their roles run as coroutines under a random scheduler, copies and MMAs complete at random later times (MMAs of one warp in their
order), mbarriers count phases and are waited for by parity. The index arithmetic is the kernels'.

Every wait names the completion it means, and fails if it passes before that; every buffer knows whose content it holds, and a
read of another's fails. A wait may also give up, one chosen at random, and then whichever can no longer be met: the role goes
on without waiting, as in the kernel. Whatever gave up, nothing may be on its way when the block ends: shared memory and TMEM are
the next block's then."""

import random

import pytest

from tests.test_tmem_pipeline_model import Barrier

INFOS, RAW = 8, 4


class Fault(Exception):
    pass


class Block:
    def __init__(self, seed, give_up):
        self.rng = random.Random(seed)
        self.copies, self.queues, self.roles = [], {}, []
        self.waits, self.give_up, self.gave_up = 0, give_up, False

    def wait(self, bar, k, hardware=False):
        """Completion k (0-based) of bar, by parity; yields while it has not passed, returns whether it did. hardware: only a copy or an
        MMA is waited for, whose time is bounded; such a wait is not the one that gives up."""
        if not hardware:
            self.waits += 1
            if self.waits - 1 == self.give_up:
                self.gave_up = True
                return False
        while not bar.parity_wait_passes(k & 1):
            if (yield "blocked") == "expire":
                self.gave_up = True
                return False
        if bar.phase < k + 1 and not self.gave_up:
            raise Fault(f"a wait for completion {k} passed at phase {bar.phase}")
        return True

    def hold(self, have, want, what):
        if have != want and not self.gave_up:
            raise Fault(f"{what}: holds {have}, read as {want}")

    def engine(self):
        """One asynchronous completion, if any is on its way."""
        ready = [("copy", i) for i in range(len(self.copies))] + [("mma", q) for q in self.queues if self.queues[q]]
        if not ready:
            return False
        kind, which = self.rng.choice(ready)
        (self.copies.pop(which) if kind == "copy" else self.queues[which].pop(0))()
        return True

    def run(self):
        live, idle = [(r, None) for r in self.roles], 0
        while live:
            if self.rng.random() < 0.4 and self.engine():
                idle = 0
            i = self.rng.randrange(len(live))
            role, send = live[i]
            try:
                blocked = role.send(send) == "blocked"
                live[i] = (role, None)
                idle = idle + 1 if blocked else 0
            except StopIteration:
                live.pop(i)
                idle = 0
            if idle > 50 * len(live) and not self.engine():  # nobody can go on: a wait runs out
                if not self.gave_up:
                    raise Fault("no role can go on")
                i = self.rng.randrange(len(live))
                live[i] = (live[i][0], "expire")
                idle = 0
        if self.copies or any(self.queues.values()):
            raise Fault("the block ended with copies or MMAs on their way")


def prompt_block(steps, tiles, seed, give_up=None, drains=True):
    b = Block(seed, give_up)
    bars = lambda n, count: [Barrier(count) for _ in range(n)]  # noqa: E731
    q_ready, k_full, v_full = Barrier(2), bars(2, 2), bars(2, 2)
    s_full, p_full = [bars(2, 1) for _ in range(2)], [bars(2, 1) for _ in range(2)]
    before_last, o_full, drained = bars(2, 1), bars(2, 1), bars(2, 1)
    info, raw_full, raw_empty = bars(INFOS, 4), bars(RAW, 1), bars(RAW, 4)
    raw, k_smem, v_smem = [None] * RAW, [[None] * 2 for _ in range(2)], [[None] * 2 for _ in range(2)]
    s_buf, infos, loudest, done = [[None] * 2 for _ in range(2)], [[None] * 4 for _ in range(INFOS)], [None] * INFOS, [0, 0]
    b.queues = {0: [], 1: []}

    def copier():
        j = 0
        while j < steps:
            slot = j % RAW
            if j >= RAW and not (yield from b.wait(raw_empty[slot], j // RAW - 1)):
                break

            def land(j=j, slot=slot):
                raw[slot] = j
                raw_full[slot].arrive()

            b.copies.append(land)
            j += 1
            yield
        if drains:
            for k in range(max(0, j - RAW), j):
                yield from b.wait(raw_full[k % RAW], k // RAW, hardware=True)

    def codes(is_v, parity, w):
        alive = True
        for j in range(parity, steps, 2):
            slot, stage = j % RAW, j & 1
            alive = alive and (yield from b.wait(raw_full[slot], j // RAW))
            b.hold(raw[slot], j, "raw slot")
            if is_v and j > 0:
                alive = alive and (yield from b.wait(info[(j - 1) % INFOS], (j - 1) // INFOS))
                b.hold(loudest[(j - 1) % INFOS], j - 1, "the loudest so far")
            if is_v and w == 0:
                loudest[j % INFOS] = j
            infos[j % INFOS][2 * is_v + w] = j
            yield
            info[j % INFOS].arrive()
            after = j if is_v else j - 2
            for i in range(tiles if after >= 0 else 0):
                alive = alive and (yield from b.wait(s_full[i][after & 1], after // 2))
            b.hold(raw[slot], j, "raw slot")
            (v_smem if is_v else k_smem)[stage][w] = j
            yield
            (v_full if is_v else k_full)[stage].arrive()
            if alive:
                raw_empty[slot].arrive()

    def mma(i):
        def scores(j):
            def run():
                b.hold(k_smem[j & 1], [j, j], "K'")
                s_buf[i][j & 1] = ("S", j)

            b.queues[i] += [run, s_full[i][j & 1].arrive]

        def values(j):
            def run():
                b.hold(v_smem[j & 1], [j, j], "V'")
                b.hold(s_buf[i][j & 1], ("P", j), "P")
                done[i] = j + 1

            b.queues[i].append(run)

        ok = yield from b.wait(q_ready, 0)
        for j in range(min(steps, 2)):
            ok = ok and (yield from b.wait(k_full[j], 0))
            if ok:
                scores(j)
        for j in range(steps):
            stage, turn = j & 1, j >> 1
            ok = ok and (yield from b.wait(v_full[stage], turn))
            if ok and j + 2 < steps:
                ok = yield from b.wait(k_full[stage], turn + 1)
            ok = ok and (yield from b.wait(p_full[i][stage], turn))
            if not ok:
                break
            values(j)
            if j + 2 < steps:
                scores(j + 2)
            else:
                b.queues[i].append((before_last if j + 1 < steps else o_full)[i].arrive)
            yield
        if drains:
            b.queues[i].append(drained[i].arrive)
            yield from b.wait(drained[i], 0, hardware=True)

    def rows(i):
        alive = True
        q_ready.arrive()
        if i >= tiles:
            return
        for j in range(steps):
            alive = alive and (yield from b.wait(s_full[i][j & 1], j >> 1))
            alive = alive and (yield from b.wait(info[j % INFOS], j // INFOS))
            b.hold(infos[j % INFOS], [j] * 4, "what is said of the keys")
            b.hold(s_buf[i][j & 1], ("S", j), "S")
            yield
            b.hold(infos[j % INFOS], [j] * 4, "what is said of the keys")
            s_buf[i][j & 1] = ("P", j)
            if j > 0 and b.rng.random() < 0.5:  # the maximum moves: O must be nobody's
                bar, k = (s_full[i][(j + 1) & 1], (j + 1) >> 1) if j + 1 < steps else (before_last[i], 0)
                alive = alive and (yield from b.wait(bar, k))
                if done[i] != j and not b.gave_up:
                    raise Fault(f"O is scaled at step {j} with the values of {done[i]} steps in it")
            yield
            p_full[i][j & 1].arrive()
        if alive:
            yield from b.wait(o_full[i], 0)
            b.hold(done[i], steps, "O")

    b.roles = [copier(), rows(0), rows(1)] + [codes(v, x, w) for v in (0, 1) for x in (0, 1) for w in (0, 1)] + [mma(i) for i in range(tiles)]
    b.run()
    return b.waits


def split_block(stages, fills, seed, give_up=None, drains=True):
    """One consuming warp's ring; a warp that gave up reads on without waiting and hands nothing back, and the filler gives up on it."""
    b = Block(seed, give_up)
    full, empty = [Barrier(1) for _ in range(stages)], [Barrier(1) for _ in range(stages)]
    ring = [None] * stages

    def filler():
        n = 0
        while n < fills:
            slot = n % stages
            if n >= stages and not (yield from b.wait(empty[slot], n // stages - 1)):
                break

            def land(n=n, slot=slot):
                ring[slot] = n
                full[slot].arrive()

            b.copies.append(land)
            n += 1
            yield
        if drains:
            for k in range(max(0, n - stages), n):
                yield from b.wait(full[k % stages], k // stages, hardware=True)

    def consumer():
        alive = True
        for n in range(fills):
            alive = alive and (yield from b.wait(full[n % stages], n // stages))
            b.hold(ring[n % stages], n, "ring")
            yield
            b.hold(ring[n % stages], n, "ring")
            if alive:
                empty[n % stages].arrive()

    b.roles = [filler(), consumer()]
    b.run()
    return b.waits


@pytest.mark.parametrize("tiles", [1, 2])
@pytest.mark.parametrize("steps", [1, 2, 3, 4, 5, 9, 20, 33])
def test_prompt_block(steps, tiles):
    for seed in range(20):
        prompt_block(steps, tiles, seed)


@pytest.mark.parametrize("fills", [1, 2, 5, 6, 7, 31])
@pytest.mark.parametrize("stages", [2, 3, 6])
def test_split_block(stages, fills):
    for seed in range(20):
        split_block(stages, fills, seed)


def _ended_early(block, waits, **kw):
    out = 0
    for seed in range(150):
        try:
            block(seed=seed, give_up=random.Random(seed).randrange(waits), **kw)
        except Fault:
            out += 1
    return out


@pytest.mark.parametrize("steps,tiles", [(1, 1), (3, 2), (12, 2)])
def test_prompt_block_whose_waits_give_up(steps, tiles):
    waits = prompt_block(steps, tiles, 0)
    assert _ended_early(prompt_block, waits, steps=steps, tiles=tiles) == 0
    assert _ended_early(prompt_block, waits, steps=steps, tiles=tiles, drains=False) > 0  # what the waits at the end are for


@pytest.mark.parametrize("stages,fills", [(2, 9), (6, 20)])
def test_split_block_whose_waits_give_up(stages, fills):
    waits = split_block(stages, fills, 0)
    assert _ended_early(split_block, waits, stages=stages, fills=fills) == 0
    assert _ended_early(split_block, waits, stages=stages, fills=fills, drains=False) > 0
