"""AdamW / clip_grad_norm_ in the calls around a training loop, without a GPU: re-pointed parameters as the host walk sees them,
arguments by position, version counters."""
import ctypes as C
import inspect

import numpy as np
import pytest
import torch
import torch.nn as nn


@pytest.fixture(scope='module')
def host():
    from super_resolution_amd.build import build
    build(verbose=False)
    from super_resolution_amd import optim
    return optim._host_lib()


def _track(host, tensors):
    h = host.srt_track(tensors)
    assert h
    n = len(tensors)
    ptr, odd, nodd, moved = (C.c_uint64 * n)(), (C.c_int64 * n)(), C.c_int64(), C.c_int64()

    def walk():
        missing = host.srt_gradients(h, ptr, odd, C.byref(nodd), C.byref(moved))
        return missing, nodd.value, moved.value
    return h, walk


def test_walk_sees_another_memory_order(host):
    """Strides at the same address, and another storage at the same address; strides of dimensions of one element are no order."""
    memory = np.zeros(24, np.float32)
    ps = [nn.Parameter(torch.zeros(s)) for s in ((4, 8, 3, 3), (12, 12), (6, 4), (5, 1, 1, 7))]
    ps[2].data = torch.from_numpy(memory).view(6, 4)
    h, walk = _track(host, ps)
    assert walk() == (4, 0, 0)
    ps[1].data = ps[1].data.t()
    assert walk() == (4, 0, 1)
    ps[1].data = ps[1].data.t()
    assert walk() == (4, 0, 0)
    ps[3].data = ps[3].data.as_strided((5, 1, 1, 7), (7, 1, 99, 1))
    assert walk() == (4, 0, 0)
    ps[2].data = ps[2].data.view(4, 6)
    assert walk() == (4, 0, 0)          # every element is where it was
    ps[2].data = torch.from_numpy(memory).view(4, 6)
    assert walk() == (4, 0, 1)          # memory that was given back and taken again
    ps[0].data = ps[0].data.to(memory_format=torch.channels_last)
    assert walk() == (4, 0, 2)
    h2, walk2 = _track(host, ps[:1])
    assert walk2() == (1, 0, 0)
    ps[0].data = ps[0].data.as_strided((4, 8, 3, 3), (72, 9, 3, 1))
    assert walk2() == (1, 0, 1)
    host.srt_untrack(h2)
    host.srt_untrack(h)


def test_clip_takes_torchs_arguments_in_torchs_order():
    from super_resolution_amd import train
    theirs = list(inspect.signature(torch.nn.utils.clip_grad_norm_).parameters)[:4]
    assert list(inspect.signature(train.clip_grad_norm_).parameters)[:4] == theirs
    p = nn.Parameter(torch.zeros(4))
    for other in (1.0, 1, float('inf'), 0.0, 3.0, True):
        with pytest.raises(ValueError, match='norm_type'):
            train.clip_grad_norm_([p], 1.0, other)
    for two in (2.0, 2, '2'):
        assert float(train.clip_grad_norm_([p], 1.0, two)) == 0.0


def test_shared_elements_against_a_list_of_all_bytes():
    """Random strided views of one block of memory, float32 and bfloat16 mixed: refused exactly where two bytes' claims meet."""
    import random
    from super_resolution_amd import optim

    def claimed_twice(tensors):
        seen = set()
        for t in tensors:
            for index in np.ndindex(*t.shape):
                at = t.data_ptr() + sum(i * s for i, s in zip(index, t.stride())) * t.element_size()
                pairs = range(at, at + t.element_size(), 2)
                if any(b in seen for b in pairs):
                    return True
                seen.update(pairs)
        return False
    rng, found = random.Random(1), [0, 0]
    buf = torch.zeros(400)
    for _ in range(600):
        views = []
        for _ in range(rng.choice((1, 2, 3))):
            dims = rng.randrange(4)
            views.append(rng.choice((buf, buf.view(torch.bfloat16))).as_strided([rng.randrange(5) for _ in range(dims)],
                                                                              [rng.choice((0, 1, 1, 2, 3, 4, 6, 8, 12)) for _ in range(dims)], rng.randrange(60)))
        want = claimed_twice(views)
        found[want] += 1
        if want:
            with pytest.raises(RuntimeError, match='repeats|share'):
                optim._check_separate(list(enumerate(views)))
        else:
            optim._check_separate(list(enumerate(views)))
    assert min(found) > 100


def test_a_refused_walk_leaves_version_counters(host):
    ps = [nn.Parameter(torch.zeros(3)) for _ in range(4)]
    for p in ps[1:]:
        p.grad = torch.ones(3)
    h, walk = _track(host, ps)
    before = [p._version for p in ps]
    walk()
    assert [p._version - b for p, b in zip(ps, before)] == [0, 1, 1, 1]
    assert host.srt_not_written(h) == 0
    assert [p._version - b for p, b in zip(ps, before)] == [0, 0, 0, 0]
    host.srt_untrack(h)
    # a view and its base have one counter
    base = torch.zeros(6)
    ps = [nn.Parameter(t) for t in (base[:3].detach(), base[3:].detach())]
    for p in ps:
        p.grad = torch.ones(3)
    h, walk = _track(host, ps)
    before = [p._version for p in ps]
    walk()
    walk()
    host.srt_not_written(h)
    host.srt_not_written(h)
    assert [p._version for p in ps] == before
    host.srt_untrack(h)
