"""Model of the ring of the two-CTA products (k_product_tc with clusters of two in
sparsefold_b200/csrc/sf_product_tc.cuh), run under many random interleavings on the CPU.

Each CTA's producer waits for a free slot and loads its half of a stage; both CTAs' loads complete on the even CTA's
barrier, where its producer expects the bytes of both; the even CTA's issuer waits for that phase and issues the MMA,
which reads both shared memories; its commit frees the slot in both CTAs.

Beside the phases the model keeps what happens before what: a completed load is released into the barrier that it
completes on, a wait acquires what its phase has collected, a relaxed arrival carries nothing.  An MMA must have
acquired both halves of the stage that it reads, and a load may overwrite a slot only when the MMA that read it has run.
"""
import os
import random
import re

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sparsefold_b200", "csrc",
                      "sf_product_tc.cuh")


class Bar:
  """Phases of `arrivals` arrivals and as many landed loads as the arrivals announce."""

  def __init__(self, arrivals):
    self.arrivals, self.left, self.loads, self.done, self.carried, self.phases = arrivals, arrivals, 0, 0, set(), []

  def _settle(self):
    assert self.left >= 0
    if self.left == 0 and self.loads == 0:
      self.phases.append(frozenset(self.carried))
      self.left, self.carried, self.done = self.arrivals, set(), self.done + 1

  def arrive(self, expect=0, releases=()):
    self.left -= 1
    self.loads += expect
    self.carried |= set(releases)
    self._settle()

  def land(self, item):
    self.loads -= 1
    self.carried.add(item)
    self._settle()

  def passed(self, use):
    assert self.done in (use, use + 1), f"waiting for use {use} with {self.done} phases complete"
    return self.done == use + 1


def run(stages, steps, seed, relay=False, early=False):
  """relay plants the mistake of an odd CTA that reports its stages by a relaxed arrival of its own; early the one of a
  producer in the odd CTA that does not wait for its slot."""
  rng = random.Random(seed)
  full = [[Bar(2 if relay and c == 0 else 1) for _ in range(stages)] for c in range(2)]
  empty = [[Bar(1) for _ in range(stages)] for _ in range(2)]
  held = [[None] * stages for _ in range(2)]
  landing, mmas, ran = [], [], [0]

  def producer(cta):
    for i in range(steps):
      s = i % stages
      if i >= stages and not (early and cta == 1):
        while not empty[cta][s].passed(i // stages - 1):
          yield
      bar = full[0][s] if not relay else full[cta][s]
      if cta == 0 or relay:
        bar.arrive(expect=1 if relay else 2)
      assert i < stages or ran[0] > i - stages, "a slot is overwritten before the MMA that reads it"
      held[cta][s] = None
      landing.append((cta, s, i, bar))
      yield

  def relayer():
    for i in range(steps):
      while not full[1][i % stages].passed(i // stages):
        yield
      full[0][i % stages].arrive()          # relaxed: releases nothing
      yield

  def issuer():
    seen = set()
    for i in range(steps):
      s = i % stages
      while not full[0][s].passed(i // stages):
        yield
      seen |= full[0][s].phases[i // stages]
      assert {(0, i), (1, i)} <= seen, f"step {i}: the MMA is not ordered behind both halves"
      mmas.append((s, i))
      yield

  def engines():
    while True:
      if landing and rng.random() < 0.6:
        cta, s, i, bar = landing.pop(rng.randrange(len(landing)))
        held[cta][s] = i
        bar.land((cta, i))
      elif mmas:
        s, i = mmas.pop(0)
        assert held[0][s] == held[1][s] == i
        ran[0] = i + 1
        for c in range(2):
          empty[c][s].arrive()
      yield

  actors = [producer(0), producer(1), issuer()] + ([relayer()] if relay else [])
  hardware = engines()
  for _ in range(400 * steps):
    if ran[0] == steps and not actors:
      return
    next(hardware)
    if actors:
      a = rng.choice(actors)
      try:
        next(a)
      except StopIteration:
        actors.remove(a)
  raise AssertionError("the ring stopped")


@pytest.mark.parametrize("stages", [2, 3, 5, 8])
@pytest.mark.parametrize("steps", [1, 2, 7, 40])
def test_both_halves_are_ordered_before_the_mma(stages, steps):
  for seed in range(40):
    run(stages, steps, seed)


def test_the_model_catches_planted_mistakes():
  with pytest.raises(AssertionError, match="not ordered"):
    run(4, 20, 0, relay=True)
  caught = 0
  for seed in range(20):
    try:
      run(3, 30, seed, early=True)
    except AssertionError:
      caught += 1
  assert caught == 20


def stage(tiles, seed, committed=True):
  """One warp's output buffers over several tiles (rows of its own in a tile or none, chunks per tile): two buffers in turn,
  a wait for all but the last group before each use, a store that reads its buffer some time after its commit."""
  rng = random.Random(seed)
  groups, turn = [], 0              # committed groups in order: [buffer that is read, or None for an empty one; done]
  for tile, (rows, chunks) in enumerate(tiles):
    for _ in range(chunks):
      for g in groups[:-1]:
        g[1] = True                 # the wait: all but the last group have read their buffers
      buf, turn = turn & 1, turn + 1
      assert not any(g[0] == buf and not g[1] for g in groups), f"tile {tile}: a store still reads buffer {buf}"
      if rows or committed:
        groups.append([buf if rows else None, not rows])
      late = [g for g in groups if not g[1]]
      if late and rng.random() < 0.3:
        late[0][1] = True           # the engine reads on


def test_buffers_of_warps_without_rows():
  """The last row tile leaves some warps without a row; the tile before it may still be on its way out."""
  rng = random.Random(1)
  for seed in range(200):
    stage([(rng.random() < 0.6, rng.randint(0, 3)) for _ in range(30)], seed)
  caught = 0
  for seed in range(20):
    try:
      stage([(True, 2), (False, 2), (True, 2)] * 10, seed, committed=False)
    except AssertionError:
      caught += 1
  assert caught == 20


def test_every_use_of_a_buffer_commits_a_group():
  text = re.sub(r"//[^\n]*", "", open(SOURCE).read())
  at = [m.start() for m in re.finditer(r"bulk_commit\(\)", text)]
  assert len(at) == 2
  for a in at:      # in the branch of lane 0 alone, not in that of warps with rows
    before = text[:a]
    branch = before[before.rindex("if (lane == 0"):]
    assert branch.startswith("if (lane == 0) {") and branch.count("{") - branch.count("}") == 1


def test_the_kernel_has_no_other_report_of_a_landed_stage():
  """Arrivals of the odd CTA's threads on the even CTA's barriers: only of the epilogue, behind the tcgen05 fence."""
  text = re.sub(r"//[^\n]*", "", open(SOURCE).read())
  calls = [m.start() for m in re.finditer(r"mbar_arrive_cluster\(", text)]
  body = text[text.index("void free_acc("):]
  body = body[:body.index("\n}")]
  assert len(calls) == 1 and "tc_fence_before" in body and "mbar_arrive_cluster" in body
  assert "map_shared(full, 0)" in text and text.count("cta_group::2 [%0]") == 2
