"""AdamW / clip_grad_norm_ without a GPU: refused arguments (Python and C ABI: nothing is launched on an error), the header's structs,
and the walk over torch's tensors that the step makes on the host."""
import copy
import ctypes as C
import os
import subprocess
import tempfile

import numpy as np
import pytest
import torch
import torch.nn as nn

import adamw_ref as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope='module')
def L():
    from super_resolution_amd.build import build
    build(verbose=False)
    from super_resolution_amd import _lib
    _lib.lib()
    return _lib


@pytest.fixture(scope='module')
def host(L):
    from super_resolution_amd import optim
    return optim._host_lib()


def test_structs_match_the_header(L):
    src = '#include <stdio.h>\n#include "sr_amd.h"\nint main(){printf("%zu %zu %zu %zu %d %d %d\\n", sizeof(sr_adamw_tensor), ' \
          'sizeof(sr_adamw_hyper), sizeof(sr_grad_list), sizeof(sr_grad_span), SR_ADAMW_BLOCK, SR_ADAMW_SCALARS_BYTES, SR_GRAD_MAX_LISTS);printf("%d %d %d\\n", SR_ADAMW_BY_VALUE, SR_GRAD_SPANS_BY_VALUE, SR_UPLOAD_WORDS);return 0;}\n'
    with tempfile.TemporaryDirectory() as d:
        open(os.path.join(d, 'a.c'), 'w').write(src)
        subprocess.check_call(['gcc', '-I', os.path.join(ROOT, 'include'), os.path.join(d, 'a.c'), '-o', os.path.join(d, 'a')])
        got = [int(x) for x in subprocess.check_output([os.path.join(d, 'a')]).split()]
    assert got == [C.sizeof(L.AdamWTensor), C.sizeof(L.AdamWHyper), C.sizeof(L.GradList), 16, L.ADAMW_BLOCK, L.ADAMW_SCALARS_BYTES, L.GRAD_MAX_LISTS,
                   L.ADAMW_BY_VALUE, L.GRAD_SPANS_BY_VALUE, L.UPLOAD_WORDS]


def test_c_entries_refuse_bad_arguments(L):
    """Every refusal comes before any HIP call (there is no device here)."""
    lib = L.lib()
    out = C.c_void_p()
    t = (L.AdamWTensor * 2)()
    for x in t:
        x.p, x.m, x.v, x.me, x.ve, x.ema, x.n, x.index = 4096, 4096, 4096, 4096, 4096, None, 8, 0
    ok = lambda **k: lib.sr_adamw_create(k.get('dtype', 0), k.get('bits', 32), k.get('count', 2), k.get('t', t), C.byref(out))  # noqa: E731
    ARG, WS = -1, -2
    assert ok(dtype=2) == ARG and ok(bits=16) == ARG and ok(count=0) == ARG and ok(t=None) == ARG
    assert lib.sr_adamw_create(0, 32, 2, t, None) == ARG
    for field, bad in (('n', -1), ('index', -1), ('p', None), ('m', None), ('v', None), ('p', 4098), ('m', 4097), ('v', 4098), ('ema', 4097)):
        keep = getattr(t[1], field)
        setattr(t[1], field, bad)
        assert ok() == ARG, field
        setattr(t[1], field, keep)
    t[1].me = None
    assert ok(bits=8) == ARG
    t[1].me, t[0].ema = 4096, 4096   # an average for some tensors only
    assert ok() == ARG
    t[0].ema = None
    h = L.AdamWHyper(1e-3, 0.9, 0.999, 1e-8, 0.0, 0.0, 0)
    assert lib.sr_adamw_step(None, C.byref(h), 1, None, 4096, 0, None, None) == ARG
    for bad in (dict(lr=-1.0), dict(beta1=1.0), dict(beta2=-0.1), dict(eps=-1.0), dict(weight_decay=-1.0), dict(ema_decay=1.5), dict(lr=float('nan'))):
        b = L.AdamWHyper(1e-3, 0.9, 0.999, 1e-8, 0.0, 0.0, 0)
        for k, x in bad.items():
            setattr(b, k, x)
        assert lib.sr_adamw_tick(C.byref(b), None, 4096, 4096, None) == ARG, bad
    assert lib.sr_adamw_tick(C.byref(h), None, None, 4096, None) == ARG
    assert lib.sr_adamw_moments(None, 0, 4096, 4096, None) == ARG
    assert lib.sr_adamw_set_moments(None, 4096, 4096, 0, None) == ARG
    lists = (L.GradList * 1)()
    lists[0].spans, lists[0].nspans, lists[0].dtype = 4096, 1, 0
    need = lib.sr_grad_norm_workspace_bytes(1)
    assert need > 0 and lib.sr_grad_norm_workspace_bytes(0) == 0
    assert lib.sr_grad_norm(1, lists, 1.0, 4096, 4096, need - 1, None) == WS
    assert lib.sr_grad_norm(1, lists, 1.0, 4096, None, need, None) == WS
    assert lib.sr_grad_norm(1, lists, -1.0, 4096, 4096, need, None) == ARG
    assert lib.sr_grad_norm(1, lists, 1.0, None, 4096, need, None) == ARG
    assert lib.sr_grad_norm(65, lists, 1.0, 4096, 4096, 1 << 30, None) == ARG
    lists[0].dtype = 2
    assert lib.sr_grad_norm(1, lists, 1.0, 4096, 4096, need, None) == ARG
    lists[0].dtype, lists[0].on_host, lists[0].nspans = 0, 1, L.GRAD_SPANS_BY_VALUE + 1
    assert lib.sr_grad_norm(1, lists, 1.0, 4096, 4096, need, None) == ARG
    assert lib.sr_grad_scale(2, 1, 4096, 0, 4096, None) == ARG and lib.sr_grad_scale(0, -1, 4096, 0, 4096, None) == ARG
    assert lib.sr_grad_scale(0, 1, None, 0, 4096, None) == ARG and lib.sr_grad_scale(0, 1, 4096, 0, None, None) == ARG
    assert lib.sr_grad_scale(0, L.GRAD_SPANS_BY_VALUE + 1, 4096, 1, 4096, None) == ARG
    assert lib.sr_grad_scale(0, 0, None, 0, 4096, None) == 0
    assert lib.sr_upload(4096, 4096, 6, None) == ARG and lib.sr_upload(None, 4096, 8, None) == ARG and lib.sr_upload(4096, 4098, 8, None) == ARG
    assert lib.sr_upload(None, None, 0, None) == 0
    for src, dst, n, done in ((4096, 4096, 6, 4096), (None, 4096, 8, 4096), (4096, None, 8, 4096), (4100, 4096, 8, 4096), (4096, 4100, 8, 4096),
                              (4096, 4096, 1 << 31, 4096), (4096, 4096, 0, 4096), (4096, 4096, 8, None), (4096, 4096, 8, 4100)):
        assert lib.sr_upload_pinned(src, dst, n, done, 1, None) == ARG


def test_python_refusals(L):
    from super_resolution_amd import train
    p = nn.Parameter(torch.zeros(4))
    with pytest.raises(RuntimeError, match='MI355X'):
        train.AdamW([p])
    for kw in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8), dict(weight_decay=-1.0), dict(state_bits=16),
               dict(ema_decay=1.5), dict(ema_decay=-0.1)):
        with pytest.raises(ValueError):
            train.AdamW([p], **kw)
    with pytest.raises(ValueError):
        train.AdamW([])
    with pytest.raises(ValueError):
        train.AdamW([p, p])
    with pytest.raises(ValueError):
        train.AdamW([{'params': [p]}, {'params': [p]}])
    with pytest.raises(ValueError):
        train.clip_grad_norm_([p], -1.0)
    with pytest.raises(ValueError):
        train.clip_grad_norm_([p], float('nan'))
    assert float(train.clip_grad_norm_([p], 1.0)) == 0.0    # no gradients: as torch
    assert float(train.clip_grad_norm_([], 1.0)) == 0.0
    p.grad = torch.ones(4)
    with pytest.raises(TypeError, match='tensor 0'):
        train.clip_grad_norm_(p, 1.0)
    with pytest.raises(RuntimeError, match='not a tensor'):
        train.clip_grad_norm_([3], 1.0)


def _track(host, tensors):
    h = host.srt_track(tensors)
    assert h
    n = len(tensors)
    return h, (C.c_uint64 * n)(), (C.c_int64 * n)(), C.c_int64(), C.c_int64()


def test_walk_over_gradients(host):
    ps = [nn.Parameter(torch.zeros(s)) for s in ((3,), (2, 3, 4, 5), (2, 3, 4, 5), (0,), (4, 6), (1,))]
    ps[2].data = ps[2].data.to(memory_format=torch.channels_last)
    g = [torch.ones_like(p) for p in ps]
    h, ptr, odd, nodd, moved = _track(host, ps)
    run = lambda: host.srt_gradients(h, ptr, odd, C.byref(nodd), C.byref(moved))  # noqa: E731
    assert run() == len(ps) and nodd.value == moved.value == 0 and list(ptr) == [0] * len(ps)
    for p, x in zip(ps, g):
        p.grad = x
    ps[0].grad = None
    assert run() == 1 and nodd.value == 0
    assert list(ptr)[1:3] == [g[1].data_ptr(), g[2].data_ptr()] and ptr[0] == 0
    ps[2].grad = torch.ones(2, 3, 4, 5)                 # another order of the same elements
    ps[4].grad = torch.ones(4, 1).expand(4, 6)          # repeated elements
    assert run() == 1 and sorted(odd[:nodd.value]) == [2, 4] and ptr[2] == ptr[4] == 0
    ps[4].grad = torch.ones(6, 4).t()
    assert run() == 1 and sorted(odd[:nodd.value]) == [2, 4]
    before = [p._version for p in ps]
    run()
    assert [p._version - b for p, b in zip(ps, before)] == [0, 1, 1, 1, 1, 1]   # those with a gradient are about to be written
    ps[5].data = torch.zeros(1)
    run()
    assert moved.value == 1
    ps[5].data = ps[0].data[:1]
    h2, ptr2, odd2, nodd2, moved2 = _track(host, [ps[0]])
    ps[0].data = ps[0].data[:2]        # the same place, another size
    assert host.srt_gradients(h2, ptr2, odd2, C.byref(nodd2), C.byref(moved2)) == 1 and moved2.value == 1
    host.srt_untrack(h2)
    host.srt_untrack(h)
    assert host.srt_track([1, 2]) is None and b'tensor' in host.srt_message()


def test_spans_refuse_what_is_not_on_one_gpu(host):
    dev, counts = C.c_int(-1), (C.c_int64 * 3)()
    assert host.srt_spans([torch.zeros(3)], 0, C.byref(dev), counts) == 1
    assert host.srt_spans([nn.Parameter(torch.zeros(3))], 1, C.byref(dev), counts) == 0 and list(counts) == [0, 0, 0]
    assert host.srt_spans((torch.zeros(3),), 0, C.byref(dev), counts) == -1     # not a list: a message, no crash
    assert b'list' in host.srt_message()


def test_exchange_and_world_without_a_process_group(L):
    from super_resolution_amd import optim
    assert optim._world(None) == 1
    assert optim._is_dense(torch.zeros(2, 3, 4, 5).to(memory_format=torch.channels_last)) and optim._is_dense(torch.zeros(0, 3))
    assert not optim._is_dense(torch.zeros(4, 6)[:, ::2]) and not optim._is_dense(torch.zeros(3).expand(2, 3)) and not optim._is_dense(torch.zeros(4, 6)[:, :5])
    assert optim._is_dense(torch.zeros(4, 6).t())


# ---- the test reference against its own definitions ----------------------------------------------------------------------
def test_reference_rounding_is_unbiased_and_in_range():
    """2^16 noise values, one each: the mean of the rounded values is the value, to the resolution of the noise (2^-17 of a step)."""
    noise = np.arange(1 << 16, dtype=np.uint64)
    for second in (False, True):
        for x in (1.0, 1.06, 1.9, 0.3, 1e-3, 3e-5):
            b = np.full(256, np.float32(x), np.float32)
            b[0] = 1.0 if x <= 1 else x
            vals = [R.to_8_bits(b, noise[i:i + 256], second)[1:] for i in range(0, 1 << 16, 256)]
            got = np.concatenate(vals).astype(np.float64)
            q = max(np.diff(np.unique(got)).max(initial=0.0), 0.0)
            skipped = 256 / 65536 * q            # the first element of each block is another one
            assert abs(got.mean() - float(b[1])) <= q * 2 ** -16 + skipped + 1e-12, (second, x)
    with np.errstate(invalid='ignore'):
        bad = R.to_8_bits(np.array([1.0, np.inf], np.float32), noise[:2], False)
    assert np.isnan(bad).all()


def test_reference_matches_torch_adamw():
    """float32, five steps, against torch.optim.AdamW in float64: a step's relative error is at most 12 roundings (three on p, the others
    on the update, which is at most 10 lr / |p| of it): 16 * 2^-24 per step on values of order 1."""
    rng = np.random.default_rng(3)
    p = rng.standard_normal(1000).astype(np.float32)
    hp = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
    r = R.Tensors([p], hp)
    t = nn.Parameter(torch.from_numpy(p.astype(np.float64)))
    opt = torch.optim.AdamW([t], **hp)
    for _ in range(5):
        g = rng.standard_normal(1000).astype(np.float32)
        r.step([g])
        t.grad = torch.from_numpy(g.astype(np.float64))
        opt.step()
    assert np.abs(r.p[0] - t.detach().numpy()).max() <= 5 * 16 * 2 ** -24 * max(1.0, np.abs(p).max())
    assert copy.copy(r.t) == [5]


def _exchange_worker(rank, world, port, q):
    import sys
    sys.path.insert(0, ROOT)
    os.environ.update(MASTER_ADDR='127.0.0.1', MASTER_PORT=str(port))
    import torch.distributed as dist
    dist.init_process_group('gloo', rank=rank, world_size=world)
    from super_resolution_amd import optim
    params = [nn.Parameter(torch.full((3, 2), 1.0 + rank)), nn.Parameter(torch.full((5,), 2.0 + rank)), nn.Parameter(torch.full((4,), 3.0 + rank).bfloat16())]
    with torch.no_grad():
        optim._broadcast_parameters(params, None)
    ok = all(bool((p == v).all()) for p, v in zip(params, (1.0, 2.0, 3.0))) and optim._world(None) == 2
    params[0].grad = torch.full((3, 2), 1.0 + 2 * rank)
    params[2].grad = torch.full((4,), 4.0 * rank).bfloat16()
    if rank == 0:
        params[1].grad = torch.full((5,), 6.0)       # the other rank has none: zeros
    optim._exchange_gradients(params, None, True)
    ok = ok and all(bool((p.grad == v).all()) for p, v in zip(params, (2.0, 3.0, 2.0)))
    optim._exchange_gradients(params, None, False)
    ok = ok and all(bool((p.grad == v).all()) for p, v in zip(params, (4.0, 6.0, 4.0)))
    q.put((rank, ok))
    dist.barrier()
    dist.destroy_process_group()


def test_gradients_and_parameters_over_two_ranks(L):
    import torch.multiprocessing as mp
    ctx = mp.get_context('spawn')
    q = ctx.Queue()
    port = 33500 + os.getpid() % 2000
    procs = [ctx.Process(target=_exchange_worker, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    res = sorted(q.get(timeout=120) for _ in procs)
    for p in procs:
        p.join(60)
        assert p.exitcode == 0
    assert res == [(0, True), (1, True)]
