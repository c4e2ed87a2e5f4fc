"""How the shared-prefix binding keeps its plans, on the CPU: threads that meet the same
lengths, and lists that are released. The plans are stand-ins for those of a GPU."""
import threading
from types import SimpleNamespace

import pytest


released: list = []


class Plan:
    """A plan that notes when it is released; `made` is called as it is made."""
    made = staticmethod(lambda: None)

    def __init__(self, *args, **kw):
        self.name = f"plan of {threading.current_thread().name}"
        Plan.made()

    def __del__(self):
        released.append(self.name)


class Ctx:
    device = 0


@pytest.fixture
def prefix(pkg, monkeypatch):
    p = pkg.prefix
    monkeypatch.setattr(p, "_plans", {})
    monkeypatch.setattr(p, "PrefixPlan", Plan)
    monkeypatch.setattr(p, "_capturing", lambda device: p.captures)
    monkeypatch.setattr(p, "captures", False, raising=False)
    monkeypatch.setattr(Plan, "made", staticmethod(lambda: None))
    released.clear()
    return p


def key(n):
    return ((0, n), None, 10, 16, 8, 0, 176, 432)


def test_two_threads_that_meet_the_same_lengths_share_a_plan(prefix):
    """The plan of the first thread, which a graph may hold by then, is not replaced by that of
    the second."""
    got, late_made, go = {}, threading.Event(), threading.Event()

    def late():
        late_made.set()
        go.wait(10)

    Plan.made = staticmethod(late)
    thread = threading.Thread(target=lambda: got.update(b=prefix._plan_for(Ctx, *key(5)).name),
                              name="late")
    thread.start()
    late_made.wait(10)  # it has seen no plan, and makes one
    Plan.made = staticmethod(lambda: None)
    first = prefix._plan_for(Ctx, *key(5)).name
    prefix.captures = True
    assert prefix._plan_for(Ctx, *key(5)).name == first  # a graph holds it from here on
    prefix.captures = False
    go.set()
    thread.join(10)
    for n in range(prefix.MAX_PLANS + 5):  # others push out what no graph holds
        prefix._plan_for(Ctx, *key(100 + n))
    assert first != "plan of late" and got["b"] == first
    assert released.count("plan of late") == 1
    assert prefix._plan_for(Ctx, *key(5)).name == first
    assert released.count(first) == 5  # of the others


def test_plans_are_released_outside_the_lock(prefix, monkeypatch):
    """Releasing a plan waits for the device; calls of other threads must not wait for
    that."""
    held = []

    class Watched(Plan):
        def __del__(self):
            held.append(prefix._plans_lock.locked())

    monkeypatch.setattr(prefix, "PrefixPlan", Watched)
    for n in range(prefix.MAX_PLANS + 3):
        prefix._plan_for(Ctx, *key(n))
    assert held == [False] * 3


def test_another_thread_releases_the_last_retired_plan(pkg, monkeypatch):
    """Lists retired during a capture are released by the next plan, whichever thread makes
    it."""
    prefix, done = pkg.prefix, []

    class Taken(list):
        """Another thread takes the last one between a look at the list and what follows."""

        def __bool__(self):
            some = len(self) > 0
            if len(self) == 1:
                self.clear()
            return some

    lib = SimpleNamespace(qwa_prefix_plan_create=lambda *a: 0, qwa_prefix_plan_deal=lambda *a: 0,
                          qwa_prefix_attention_workspace=lambda *a: 0,
                          qwa_prefix_plan_destroy=done.append)
    ctx = SimpleNamespace(lib=lib, handle=None, device=0)
    monkeypatch.setattr(prefix, "_capturing", lambda device: False)
    monkeypatch.setattr(prefix, "_retired", Taken([(lib, 1), (lib, 2)]))
    prefix.PrefixPlan([0, 5], 10, 16, 8, ctx=ctx)
    assert set(done) >= {2} and len(prefix._retired) == 0
