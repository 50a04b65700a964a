"""Page-table calls of several host threads on one state and stream."""
from __future__ import annotations

import threading

import pytest

from test_kv_pages_gpu import clean_status, ints, make, same, status  # noqa: F401

pytestmark = pytest.mark.gpu


class Slow:
    """The library, with a call of two kernels that waits for another thread's call to begin."""

    def __init__(self, lib, call):
        self._lib, self._call = lib, call
        self.inside, self.other = threading.Event(), threading.Event()
        self.overlapped = None

    def __getattr__(self, name):
        fn = getattr(self._lib, name)

        def run(*args):
            if name == self._call:
                self.inside.set()
                self.overlapped = self.other.wait(0.5)
            elif self.inside.is_set():
                self.other.set()
            return fn(*args)
        return run


@pytest.mark.parametrize("call,other", [(c, o) for c in ("reserve", "fork", "compact")
                                        for o in ("free", "copy", "reserve") if c != o])
def test_a_call_waits_for_the_kernels_of_another_thread(call, other):
    """A free or copy that came between a call's plan and its application would act on pages
    that the plan has dealt out."""
    model, pages = make(4, 4, 12)
    model.reserve([0], [40])
    pages.reserve(ints([0]), ints([40]))
    args = {"reserve": lambda: pages.reserve(ints([1]), ints([33])),
            "fork": lambda: pages.fork(ints([0]), ints([1]), ints([20])), "compact": pages.compact,
            "free": lambda: pages.free(ints([0])), "copy": lambda: pages.copy(ints([0]), ints([11]))}
    lib = pages._lib = Slow(pages._lib, "axkv_pages_" + call)
    first = threading.Thread(target=args[call])
    first.start()
    assert lib.inside.wait(10)
    second = threading.Thread(target=args[other])
    second.start()
    first.join()
    second.join()
    assert lib.overlapped is False
    if call == "reserve":
        model.reserve([1], [33])
    elif call == "fork":
        model.fork([0], [1], [20])
    if other == "free":
        model.free([0])
    elif other == "reserve":
        model.reserve([1], [33])
    same(model, pages)
    assert status() == 0
