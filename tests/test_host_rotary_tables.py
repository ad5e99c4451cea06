"""A rotary plan's device tables go with the plan: retired when its last owner
lets go, destroyed with the transforms' plans, each by its own entry."""
import contextlib
import copy
import ctypes
import gc

import pytest

from kunlunxin_fft_amd import context, native, plan_rotary, rotary, runner


class FakeLib:
    def __init__(self):
        self.made, self.destroyed, self.plans = 0, [], []

    def mfft_rotary_create(self, out, *args):
        self.made += 1
        out._obj.value = self.made
        return 0

    def mfft_rotary_destroy(self, h):
        self.destroyed.append(h.value)

    def mfft_plan_destroy(self, h):
        self.plans.append(h)


@pytest.fixture
def lib(monkeypatch):
    fake = FakeLib()
    monkeypatch.setattr(native, "_lib", fake)
    monkeypatch.setattr(native, "_RETIRED", [])
    monkeypatch.setattr(rotary, "_NATIVE", {})
    monkeypatch.setattr(context, "device_context", lambda i: contextlib.nullcontext(i))
    monkeypatch.setattr(runner, "_sync_device", lambda dev: None)
    plan_rotary.cache_clear()
    yield fake
    plan_rotary.cache_clear()
    gc.collect()


def test_tables_go_with_their_plan(lib):
    plan = plan_rotary(64, base=777.0)
    one = plan.native(0)
    assert plan.native(0) is one and plan.native(1) is not one and lib.made == 2
    plan_rotary.cache_clear()  # as eviction by 256 other plans
    gc.collect()
    assert plan.native(0) is one and native.retired_count() == 0
    del plan
    gc.collect()
    assert not rotary._NATIVE
    assert native.retired_count() == 1  # `one` still has an owner here
    del one
    gc.collect()
    assert native.retired_count() == 2 and not lib.destroyed
    assert native.release_retired() == 2
    assert sorted(lib.destroyed) == [1, 2] and not lib.plans


def test_many_plans_do_not_pile_up(lib):
    for i in range(400):
        plan_rotary(64, base=1000.0 + i).native(0)
    gc.collect()
    assert len(rotary._NATIVE) <= 256
    assert len(rotary._NATIVE) + native.retired_count() + len(lib.destroyed) == 400


def test_copies_share_nothing_that_dies_twice(lib):
    plan = plan_rotary(64, base=778.0)
    plan.native(0)
    for other in (copy.copy(plan), copy.deepcopy(plan)):
        other.native(0)
    del plan, other
    plan_rotary.cache_clear()
    gc.collect()
    native.release_retired()
    assert sorted(lib.destroyed) == list(range(1, lib.made + 1))


def test_each_kind_by_its_own_entry(lib):
    h = native.RotaryHandle(5)
    native._RETIRED.extend([("plan", 0), (h, 0)])
    assert native.release_retired() == 2
    assert lib.plans == ["plan"] and lib.destroyed == [5]
    assert isinstance(h, ctypes.c_void_p)
