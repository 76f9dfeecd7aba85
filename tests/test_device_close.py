"""Device.close() gives back what its ropes and caches hold: over a library that only counts, with no GPU."""
import gc

import pytest

from apeiron_amd import chart


class Counting:
    """Hands out a handle for every create and notes, in order, what is freed."""

    def __init__(self):
        self.next, self.live, self.freed = 1, {}, []

    def _create(self, kind, out):
        out._obj.value, self.live[self.next] = self.next, kind
        self.next += 1
        return 0

    def _free(self, ctx, h):
        if not ctx:
            return 21
        assert self.live.pop(h.value, None), "freed twice"
        self.freed.append(h.value)
        return 0

    def ah_init(self, device, out):
        return self._create("ctx", out)

    def ah_rope_create(self, ctx, spec, out):
        return self._create("rope", out)

    def ah_kv4_create(self, ctx, *args):
        return self._create("cache", args[-1])

    def ah_rope_free(self, ctx, h):
        return self._free(ctx, h)

    ah_kv4_free = ah_rope_free

    def ah_destroy(self, h):
        return self._free(h, h)


@pytest.fixture
def lib(monkeypatch):
    counting = Counting()
    monkeypatch.setattr(chart._lib, "load", lambda: counting)
    return counting


def test_close_frees_ropes_and_caches_before_the_context(lib):
    dev = chart.Device(0)
    rope, caches = chart.Rope(dev, 64), [chart.KvCache4(dev, 4, 32, 1, 64) for _ in range(3)]
    caches[1].free()  # one already given back
    dev.close()
    assert not lib.live and lib.freed[-1] == 1 and len(lib.freed) == 5
    # afterwards neither free nor close again does anything
    for t in (rope, *caches, dev):
        (t.close if t is dev else t.free)()
    del rope, caches, t
    gc.collect()
    assert len(lib.freed) == 5


def test_dropped_handles_are_freed_once(lib):
    dev = chart.Device(0)
    cache = chart.KvCache4(dev, 4, 32, 1, 64)
    del cache
    gc.collect()
    assert list(lib.live.values()) == ["ctx"]
    rope = chart.Rope(dev, 64)
    del dev  # the rope keeps its device
    gc.collect()
    assert len(lib.live) == 2
    del rope
    gc.collect()
    assert not lib.live
