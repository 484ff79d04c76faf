"""How a kernel of the 8-bit path ends after one of its bounded waits has run out, executed on the CPU.

Copies go to shared memory on their own and are counted on mbarriers; a CTA that leaves while one is under way lets it write into
whatever block comes next.  The model has the parts of the kernels in csrc/w8a8_gemm.cu and of stage 1 in csrc/decode_q8.cu: producers that start copies into a ring of
stages, an issuer that consumes full stages and whose products hand them back later, waits that may run out at any moment, and the
clean-up at the end.  They are run in many random orders that keep only what the machine guarantees.  Whatever the order: nothing may
be under way when the CTAs leave, and the clean-up's own waits must end by themselves.  With a rule of the clean-up taken away the
harness has to notice."""
import random

import pytest


class Bar:
    """An mbarrier: a phase ends once its arrivals and its expected bytes are both complete."""

    def __init__(self, count):
        self.count = self.pending = count
        self.tx = self.phase = 0

    def arrive(self, expect=0):
        assert self.pending > 0, "more arrivals than the phase takes"
        self.tx += expect
        self.pending -= 1
        self.flip()

    def complete(self, nbytes=1):
        self.tx -= nbytes
        self.flip()

    def flip(self):
        if self.pending == 0 and self.tx == 0:
            self.phase ^= 1
            self.pending = self.count

    def done(self, parity):
        return self.phase != parity


ALL = frozenset({"every end", "both CTAs", "level", "limit of its own"})


class Kernel:
    """`ctas` 1: the kernel for few tokens and decode stage 1 (copies and products of one CTA); 2: the pair kernel (each CTA copies its share, counted on
    the even CTA's barriers, whose issuer consumes both)."""

    def __init__(self, ctas, stages, steps, rules, rng):
        self.P, self.S, self.K, self.rules, self.rng = ctas, stages, steps, rules, rng
        self.full = [Bar(1) for _ in range(stages)]
        self.empty = [[Bar(1) for _ in range(stages)] for _ in range(ctas)]
        self.flight, self.products = [], []           # copies (cta, stage); committed products (stage) under way
        self.abort = [False] * ctas
        self.issued, self.broke, self.consumed = [0] * ctas, [False] * ctas, 0

    def land(self):
        self.full[self.flight.pop(self.rng.randrange(len(self.flight)))[1]].complete()

    def hand_back(self, cta):                         # a commit's arrival reaches each CTA in order, but not at one moment
        st = self.products[cta].pop(0)
        self.empty[cta][st].arrive()

    def run(self):
        rng = self.rng
        self.products = [[] for _ in range(self.P)]
        roles = [("p", c) for c in range(self.P)] + [("i", 0)] + [("e", c) for c in range(self.P)]
        give_up = rng.random() * 0.1
        stuck = 0
        while roles:
            todo = [("land", 0)] * bool(self.flight) + [("back", c) for c in range(self.P) if self.products[c]]
            ready = []
            for role, c in roles:
                if role == "p":
                    i = self.issued[c]
                    if i == self.K or i < self.S or self.empty[c][i % self.S].done((i // self.S - 1) & 1):
                        ready.append((role, c))
                elif role == "i" and (self.consumed == self.K or self.full[self.consumed % self.S].done((self.consumed // self.S) & 1)):
                    ready.append((role, c))
                elif role == "e" and self.consumed == self.K and not self.products[c]:
                    ready.append((role, c))
            waiting = [r for r in roles if r not in ready]
            if waiting and (rng.random() < give_up or not (todo or ready)):
                role, c = rng.choice(waiting)         # its wait runs out, or it sees that another's did
                self.abort[c] = True
                if role == "p":
                    self.broke[c] = True
                roles.remove((role, c))
                continue
            what, c = rng.choice(todo + ready)
            if what == "land":
                self.land()
            elif what == "back":
                self.hand_back(c)
            elif what == "p":
                i = self.issued[c]
                if i == self.K:
                    roles.remove(("p", c))
                    continue
                if c == 0:
                    self.full[i % self.S].arrive(expect=self.P)
                self.flight.append((c, i % self.S))
                self.issued[c] += 1
            elif what == "i":
                if self.consumed == self.K:
                    roles.remove(("i", 0))
                    continue
                for c2 in range(self.P):
                    self.products[c2].append(self.consumed % self.S)
                self.consumed += 1
            else:
                roles.remove(("e", c))
            stuck += 1
            assert stuck < 10000
        return self.clean_up()

    def drain(self, i):
        """The bounded wait for step i's stage; False where only its limit would end it."""
        bar, parity = self.full[i % self.S], (i // self.S) & 1
        while not bar.done(parity):
            if not self.flight or "limit of its own" not in self.rules and self.rng.random() < 0.1:
                return False
            self.land()
        return True

    def clean_up(self):
        ended = True
        if any(self.abort):
            while any(self.products):                 # the issuer's last commit
                self.hand_back(self.rng.choice([c for c in range(self.P) if self.products[c]]))
        if (any(self.abort) if "every end" in self.rules else self.broke[0]):
            peer = self.issued[-1] if "both CTAs" in self.rules else self.issued[0]
            mine, hi = self.issued[0], max(self.issued[0], peer)
            for i in range(max(hi - self.S, 0), hi):
                if "level" in self.rules:
                    if i >= mine:
                        self.full[i % self.S].arrive(expect=1)
                    elif i >= peer:
                        self.full[i % self.S].complete()
                ended = self.drain(i) and ended
        return ended, not self.flight


def outcomes(ctas, rules, n=4000):
    ended = empty = True
    for seed in range(n):
        rng = random.Random(seed)
        k = Kernel(ctas, rng.choice([2, 3, 6]), rng.randrange(1, 20), rules, rng)
        a, b = k.run()
        ended, empty = ended and a, empty and b
        if not any(k.abort):
            assert k.issued == [k.K] * ctas and k.consumed == k.K and not k.flight
    return ended, empty


def test_a_pair_leaves_nothing_under_way():
    assert outcomes(2, ALL) == (True, True)


@pytest.mark.parametrize("without", sorted(ALL))
def test_the_harness_notices_a_missing_rule(without):
    """every end: cleaned up whoever gave up, not only where the producer did; both CTAs: the odd CTA's copies too; level: a step that
    one CTA alone has started expects that CTA's bytes alone; limit of its own: a short limit of the waits does not end the clean-up's."""
    assert outcomes(2, ALL - {without}) != (True, True)


def test_a_cta_leaves_nothing_under_way():
    assert outcomes(1, ALL) == (True, True)
    for rule in ("every end", "limit of its own"):
        assert outcomes(1, ALL - {rule}) != (True, True)


def consumers(first_value_kept, rng):
    """The four consumer warps of decode stage 1 over one item: each looks whether to start, waits for its stage (and may give up, which
    sets the CTA's flag), and meets the others at a barrier.  True when all of them got past it."""
    flag, at = [False, False], ["start"] * 4                       # the flag that moves, and the one that keeps its first value
    while True:
        able = [w for w in range(4) if at[w] in ("start", "wait")]
        if not able:
            return "barrier" not in at or at.count("barrier") == 4
        w = rng.choice(able)
        if at[w] == "start":
            at[w] = "left" if flag[1 if first_value_kept else 0] else "wait"
        else:
            flag[0] = flag[0] or rng.random() < 0.3
            at[w] = "barrier"


def test_consumer_warps_all_start_or_none_does():
    rng = random.Random(1)
    assert all(consumers(True, rng) for _ in range(2000))
    assert not all(consumers(False, rng) for _ in range(2000))
