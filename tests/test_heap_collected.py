"""Arenas that the garbage collector finds: freeing waits for the device, and the collector runs between any two launches."""

import gc

import pytest

from tests.test_heap_host_logic import _FakeArena


class Holder:
    """An object in a reference cycle, as an exception with its traceback or a closure makes one."""

    def __init__(self, arena):
        self.arena, self.me = arena, self


@pytest.fixture
def freed():
    gc.collect()
    _FakeArena.freed = []
    yield _FakeArena.freed
    _FakeArena.freed = []


def test_nothing_waits_for_the_device_inside_a_collection(freed):
    Holder(_FakeArena(1024, 2))
    gc.collect()  # between the launches of two ranks, say
    assert freed == []
    other = _FakeArena(512, 1)  # a heap is made: memory of those that are gone first
    assert freed == [("handle", 1024)]
    del other
    assert freed == [("handle", 1024), ("handle", 512)]


def test_a_heap_that_lets_go_frees_what_was_collected(freed):
    kept = _FakeArena(256, 1).acquire()
    for size in (1024, 2048):
        Holder(_FakeArena(size, 1))
    gc.collect()
    assert freed == []
    kept.release()
    assert sorted(freed) == [("handle", 1024), ("handle", 2048)]


def test_without_a_cycle_the_memory_goes_at_once(freed):
    arena = _FakeArena(1024, 1)
    del arena
    assert freed == [("handle", 1024)]


def test_a_heap_in_a_cycle_lets_go_inside_the_collection(freed):
    from tileccl_amd.memory.symmetric_heap import SymmetricHeap

    arena = _FakeArena(4096, 2)
    Holder([SymmetricHeap(4096, r, 2, _arena=arena) for r in range(2)])
    del arena
    gc.collect()
    assert freed == []
    _FakeArena(16, 1)
    assert freed[0] == ("handle", 4096)


def test_a_program_can_free_them_itself(freed):
    from tileccl_amd.memory import free_collected

    Holder(_FakeArena(1024, 1))
    gc.collect()
    assert freed == []
    free_collected()
    free_collected()
    assert freed == [("handle", 1024)]
