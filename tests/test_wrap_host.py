"""Wrapped memory without a GPU: who keeps it, and until when."""
import gc
import weakref

import numpy as np
import pytest

from rgpu_amd import gpu as G


class Owner:
    pass


class Calls(G.Gpu):
    """A Gpu whose library calls are only written down."""

    def __init__(self, fail=None):
        self._h, self._spare = 1, {}
        self._held, self._held_bytes, self._mark = [], 0, None
        self.made, self.fail = [], fail

    def _call(self, name, *args):
        self.made.append(name)
        if name == self.fail:
            raise G.RtError(6, "a label")
        if name in ("rt_wrap", "rt_zeros", "rt_empty", "rt_upload"):
            args[-1]._obj.value = 16
        return 0

    def close(self):
        self._h = None


def wrapped(gpu, shape=(4,)):
    owner = Owner()
    t = gpu.wrap(256, shape, owner=owner)
    return t, weakref.ref(owner)


@pytest.mark.parametrize("how", ["free", "del"])
@pytest.mark.parametrize("wait", ["sync", "download"])
def test_owner_of_freed_memory_lives_until_the_stream_is_waited_for(how, wait):
    gpu = Calls()
    other, _ = wrapped(gpu)
    t, alive = wrapped(gpu)
    if how == "free":
        t.free()
    del t
    gc.collect()
    assert "rt_free" in gpu.made and alive() is not None
    gpu.empty((0,))
    gpu.download(gpu.wrap(0, (0,)))  # nothing to move: the library does not wait
    assert alive() is not None
    gpu.sync() if wait == "sync" else gpu.download(other)
    gc.collect()
    assert alive() is None


def test_owner_survives_a_failed_wait_only_if_the_stream_may_still_run():
    labels = Calls(fail="rt_sync")
    t, alive = wrapped(labels)
    t.free()
    with pytest.raises(G.RtError):  # RT_ERR_LABEL: found after the wait
        labels.sync()
    gc.collect()
    assert G.STATUS[6] == "RT_ERR_LABEL" and alive() is None
    broken = Calls()
    t, alive = wrapped(broken)
    u, _ = wrapped(broken)
    t.free()
    broken._call = lambda *a: (_ for _ in ()).throw(G.RtError(7, "lost"))
    with pytest.raises(G.RtError):
        broken.download(u)
    assert alive() is not None


def test_held_owners_are_bounded():
    gpu = Calls()
    for count, shape in ((3 * G.Gpu._HELD_MAX, (4,)), (5, (G.Gpu._HELD_MAX_BYTES // 8,))):
        refs = []
        for _ in range(count):
            t, alive = wrapped(gpu, shape)
            refs.append(alive)
            t.free()
        gc.collect()
        assert sum(r() is not None for r in refs) < min(G.Gpu._HELD_MAX, count)
    assert "rt_sync" not in gpu.made  # which would take the label flag from the program


def test_tensors_of_the_library_hold_nothing():
    gpu = Calls()
    gpu.zeros((4,)).free()
    gpu.wrap(256, (4,)).free()
    assert not gpu._held and isinstance(gpu.download(gpu.zeros((2,))), np.ndarray)


def test_null_handles():
    assert G.lib().rt_order_after(None, None) == 2 and G.lib().rt_order_before(None, None) == 2


def test_operands_without_elements_are_passed_on():
    """A tensor of no elements is false, but not absent: the mask of an empty batch, the state of an empty parameter."""
    gpu, seen = Calls(), []
    make, t = gpu._call, [gpu.zeros(s) for s in ((0, 8), (0, 5), (8, 5), (0,))]
    gpu._call = lambda name, *args: seen.append(args) or make(name, *args)
    gpu.matmul_a_bt(t[1], t[2], t[0], relu_mask_from=t[0])
    gpu.matmul_at_b(t[1], t[0], t[2], colsum=t[3])
    gpu.split_k(t[1], t[0], t[2], t[3], 1, True, colsum=t[3])
    gpu.split_k_static(t[1], t[0], t[2], 1, True, colsum=t[3])
    gpu.sgd(t[3], t[3], 0.1, 0.9, t[3])
    assert seen[0][-2] == 16 and all(s[-1] == 16 for s in seen[1:4]) and seen[4][2] == 16
