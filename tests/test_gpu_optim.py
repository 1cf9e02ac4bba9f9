"""train.AdamW (csrc/adamw.hip) and train.clip_grad_norm_ on the MI355X.

The float32 results are compared bit for bit with the formulas evaluated one operation at a time (tests/adamw_ref.py); that
reference is held to float64 and to torch.optim.AdamW in test_cpu_optim.py and below."""
import copy
import ctypes as C

import numpy as np
import pytest
import torch
import torch.nn as nn

import adamw_ref as R

pytestmark = pytest.mark.gpu
U = 2.0 ** -24      # largest relative error of one float32 rounding


@pytest.fixture(scope='module')
def T():
    from super_resolution_amd import _lib, train
    _lib.lib()
    assert torch.cuda.is_available()
    return train


SIZES = {
    'one': [1],
    'block edges': [255, 256, 257, 1],
    'piece edges': [1023, 1024, 1025, 2048, 3, 769],
    'empty ones': [5, 0, 300, 0],
    'ragged': [7, 4099, 64, 1, 1, 10007, 513, 96],
    'many': [1 + (37 * i) % 61 for i in range(2500)],
}
HP = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)


def f32(x):
    return torch.from_numpy(x).cuda()


def inputs(sizes, seed, scale=1.0):
    rng = np.random.default_rng(seed)
    ps = [rng.standard_normal(n).astype(np.float32) for n in sizes]

    def grads():
        return [(scale * np.exp(2 * rng.standard_normal()) * rng.standard_normal(n) * (rng.random(n) > 0.05)).astype(np.float32) for n in sizes]
    return ps, grads


def to_bf16(xs):
    return [torch.from_numpy(x).bfloat16().float().numpy() for x in xs]


def views(arrays, dtype, pad):
    """Parameters as views of one buffer with `pad` elements between them (any alignment); the buffer and the places of the pads."""
    total = sum(len(a) + pad for a in arrays) + pad
    buf = torch.full((total,), 7.0, dtype=dtype, device='cuda')
    out, at = [], pad
    for a in arrays:
        buf[at:at + len(a)] = f32(a).to(dtype)
        out.append(buf[at:at + len(a)])
        at += len(a) + pad
    hole = torch.ones(total, dtype=torch.bool)
    at = pad
    for a in arrays:
        hole[at:at + len(a)] = False
        at += len(a) + pad
    return out, buf, hole


def same(got, want, what):
    got, want = got.detach().float().cpu().numpy().reshape(-1), np.asarray(want).reshape(-1)
    assert got.shape == want.shape, what
    bad = ~((got == want) | (np.isnan(got) & np.isnan(want)))
    assert not bad.any(), '%s: %d of %d differ, first %d: %r, reference %r' % (what, bad.sum(), bad.size, bad.argmax(), got[bad.argmax()], want[bad.argmax()])


@pytest.mark.parametrize('name', list(SIZES))
@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('bf16', [False, True])
@pytest.mark.parametrize('clip,ema', [(None, None), (1.0, 0.9)])
def test_steps_bit_for_bit(T, name, bits, bf16, clip, ema):
    sizes, dtype = SIZES[name], torch.bfloat16 if bf16 else torch.float32
    arrays, grads = inputs(sizes, 11)
    if bf16:
        arrays = to_bf16(arrays)
    ps, buf, hole = views(arrays, dtype, 1)
    params = [nn.Parameter(p) for p in ps]
    opt = T.AdamW(params, state_bits=bits, ema_decay=ema, seed=5, **HP)
    ref = R.Tensors(arrays, dict(HP, ema=ema), bits, bf16, seed=5)
    for step in range(3):
        gs = to_bf16(grads()) if bf16 else grads()
        gv, _, _ = views(gs, dtype, 3)
        for p, g in zip(params, gv):
            p.grad = g
        before = [p._version for p in params]
        opt.step(clip_grad_norm=clip)
        ref.step(gs, clip)
        assert all(p._version > b for p, b in zip(params, before))
        m, v = opt.moments()
        same(m, np.concatenate(ref.m), 'm, step %d' % step)
        same(v, np.concatenate(ref.v), 'v, step %d' % step)
        for i, p in enumerate(params):
            same(p, ref.p[i], 'p[%d], step %d' % (i, step))
        if ema:
            same(opt.ema, np.concatenate(ref.ema), 'ema, step %d' % step)
        if clip:
            norm = np.sqrt(sum(float(np.sum(g.astype(np.float64) ** 2)) for g in gs))
            assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm
        for a, b in zip(gv, gs):
            same(a, b, 'the gradients are left as they were')
    assert (buf[hole.cuda()] == 7.0).all(), 'memory between the parameters was written'
    if bits == 32:
        assert torch.equal(opt.exp_avg, m) and torch.equal(opt.exp_avg_sq, v)


def test_step_against_64_bits(T):
    """Bounds by counting roundings: m and v: three operations and a rounded constant each on terms of like size; p: three roundings on p,
    and on the update at most the two of m, half of the two of v, and eight more."""
    n = 50021
    (p,), grads = inputs([n], 21)
    rng = np.random.default_rng(22)
    m = rng.standard_normal(n).astype(np.float32)
    v = (rng.standard_normal(n) ** 2).astype(np.float32)
    g = grads()[0]
    par = nn.Parameter(f32(p))
    opt = T.AdamW([par], **HP)
    opt.load_state_dict({'state': {0: {'step': 9, 'exp_avg': f32(m), 'exp_avg_sq': f32(v)}}, 'param_groups': opt.state_dict()['param_groups']})
    par.grad = f32(g)
    opt.step()
    p64, m64, v64 = R.step64(p, g, m, v, HP, 10)
    b1, b2 = HP['betas']
    em = np.abs(opt.exp_avg.cpu().numpy() - m64)
    assert (em <= 3.5 * U * (np.abs(b1 * m) + np.abs((1 - b1) * g))).all()
    ev = np.abs(opt.exp_avg_sq.cpu().numpy() - v64)
    assert (ev <= 4.5 * U * v64 + 1e-45).all()
    upd = np.abs(p64 - p.astype(np.float64) * (1 - HP['lr'] * HP['weight_decay']))
    slack = HP['lr'] / (1 - b1 ** 10) * 3.5 * U * (np.abs(b1 * m) + np.abs((1 - b1) * g)) / (np.sqrt(v64 / (1 - b2 ** 10)) + HP['eps'])
    ep = np.abs(par.detach().cpu().numpy() - p64)
    assert (ep <= 3.5 * U * np.abs(p) + 12 * U * upd + slack).all()


@pytest.mark.parametrize('bits,times', [(32, 1), (8, 1), (32, 200)])
def test_missing_gradients_keep_their_own_count(T, bits, times):
    """A parameter without a gradient is skipped and its step count stays, as in torch.optim.AdamW; its average goes on."""
    sizes = [300, 5, 2000, 64] * times
    arrays, grads = inputs(sizes, 31)
    params = [nn.Parameter(f32(a)) for a in arrays]
    opt = T.AdamW(params, state_bits=bits, ema_decay=0.5, **HP)
    ref = R.Tensors(arrays, dict(HP, ema=0.5), bits)
    twin = [nn.Parameter(torch.from_numpy(a.astype(np.float64))) for a in arrays]
    topt = torch.optim.AdamW(twin, **HP)
    for have in ([1, 1, 0, 1], [0, 0, 0, 0], [1, 0, 0, 1], [1, 1, 1, 1], [1, 1, 1, 1], [0, 1, 1, 0]):
        have = have * times
        gs = [g if h else None for g, h in zip(grads(), have)]
        for p, q, g in zip(params, twin, gs):
            p.grad = None if g is None else f32(g)
            q.grad = None if g is None else torch.from_numpy(g.astype(np.float64))
        before = [p._version for p in params]
        opt.step()
        ref.step(gs)
        topt.step()
        assert [p._version > b for p, b in zip(params, before)] == [bool(h) for h in have]
    for i, p in enumerate(params):
        same(p, ref.p[i], 'p[%d]' % i)
    same(opt.ema, np.concatenate(ref.ema), 'ema')
    sd = opt.state_dict()
    assert [int(sd['state'][i]['step']) for i in range(4 * times)] == ref.t == [4, 4, 3, 4] * times
    if bits == 32:   # six steps of order 1e-2 on values of order 4: 16 roundings of 2^-24 each
        for p, q in zip(params, twin):
            assert np.abs(p.detach().cpu().numpy() - q.detach().numpy()).max() <= 6 * 16 * U * 5


def test_empty_parameters_count_their_steps(T):
    p = [nn.Parameter(torch.ones(5, device='cuda')), nn.Parameter(torch.zeros(0, device='cuda')), nn.Parameter(torch.ones(700, device='cuda'))]
    opt = T.AdamW(p, ema_decay=0.9)
    for have in ((1, 1, 1), (0, 1, 1), (1, 1, 1), (0, 0, 0), (1, 1, 0)):
        for q, h in zip(p, have):
            q.grad = torch.ones_like(q) if h else None
        opt.step()
    sd = opt.state_dict()
    assert [int(sd['state'][i]['step']) for i in range(3)] == [3, 4, 3]
    never = T.AdamW([nn.Parameter(torch.ones(5, device='cuda')), nn.Parameter(torch.ones(5, device='cuda'))], ema_decay=0.9)
    never.params[0].grad = torch.ones(5, device='cuda')
    never.step()
    assert sorted(never.state_dict()['state']) == [0]       # as torch: a parameter without a step has no state
    twin = [nn.Parameter(q.detach().clone()) for q in never.params]
    topt = torch.optim.AdamW(twin)
    topt.load_state_dict(never.state_dict())
    for q in twin:
        q.grad = torch.ones(5, device='cuda')
    topt.step()
    with pytest.raises(ValueError, match='no group'):
        never.load_state_dict({'state': {7: {}}, 'param_groups': never.state_dict()['param_groups']})


def test_layouts(T):
    """Parameters in channels_last memory, gradients in another order, expanded, or with holes."""
    torch.manual_seed(1)
    shapes = [(4, 8, 3, 3), (4, 8, 3, 3), (16, 12), (7, 5), (6,)]
    base = [torch.randn(s) for s in shapes]
    params = [nn.Parameter(b.cuda()) for b in base]
    params[0].data = params[0].data.to(memory_format=torch.channels_last)
    grads = [torch.randn(4, 8, 3, 3).cuda(), torch.randn(4, 8, 3, 3).cuda().to(memory_format=torch.channels_last), torch.randn(16, 1).cuda().expand(16, 12),
             torch.randn(7, 10).cuda()[:, ::2], torch.randn(()).cuda().expand(6)]
    opt = T.AdamW(params, ema_decay=0.9, **HP)
    for p, g in zip(params, grads):
        p.grad = g
    opt.step()
    opt.step()
    state = opt.state_dict()['state']
    for i, (b, p, g) in enumerate(zip(base, params, grads)):
        ref = R.Tensors([b.numpy().reshape(-1)], dict(HP, ema=0.9))
        for _ in range(2):
            ref.step([g.cpu().contiguous().numpy().reshape(-1)])
        same(p.contiguous(), ref.p[0], 'p[%d]' % i)
        same(state[i]['exp_avg'].contiguous(), ref.m[0], 'm[%d]' % i)
        same(opt.ema_parameters()[i].contiguous(), ref.ema[0], 'ema[%d]' % i)


# ---- moments in 8 bits ---------------------------------------------------------------------------------------------------
def _eight(T, n=3 * 256 + 40, scale=1.0, seed=41, steps=1):
    (p,), grads = inputs([n], seed, scale)
    par = nn.Parameter(f32(p))
    opt = T.AdamW([par], state_bits=8, **HP)
    for _ in range(steps):
        par.grad = f32(grads()[0])
        opt.step()
    return par, opt, grads


def equal(a, b):
    return bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


@pytest.mark.parametrize('scale', [1e-18, 1e-10, 1.0, 1e8, 1e18])
def test_8_bit_moments_survive_a_checkpoint(T, scale):
    """What the codes stand for encodes to itself, through float32 and (in range) bfloat16, and so the steps that follow are the same.
    (At 1e18 some squares are beyond float32: those blocks are NaN, before and after.)"""
    par, opt, grads = _eight(T, scale=scale, steps=3)
    sd = copy.deepcopy(opt.state_dict())
    twin = nn.Parameter(par.detach().clone())
    other = T.AdamW([twin], state_bits=8, **HP)
    other.load_state_dict(sd)
    for a, b in zip(opt.moments(), other.moments()):
        assert equal(a, b)
    m, v = opt.moments()
    mb, vb = opt.moments(torch.bfloat16)
    if scale >= 1e-10:
        assert equal(m, mb.float()) and equal(v, vb.float())
    for _ in range(2):
        g = f32(grads()[0])
        par.grad, twin.grad = g, g.clone()
        opt.step()
        other.step()
    assert equal(par, twin)
    for a, b in zip(opt.moments(), other.moments()):
        assert equal(a, b)


def test_8_bit_second_moment_follows_its_mean(T):
    """v under a constant gradient must go to g^2 although one step moves it by a thousandth, a fraction of a code's distance: 2000 steps,
    mean over 65536 elements of the same gradient.  One rounding adds at most q v / 2 of noise to an element (q = 1/8: distance of
    two codes); 1000 such steps (the memory of beta2) on 65536 elements leave 0.0625 * sqrt(1000 / 65536) = 0.8 % of v as five times
    its worst standard deviation is 4 %."""
    n = 65536
    par = nn.Parameter(torch.zeros(n, device='cuda'))
    opt = T.AdamW([par], state_bits=8, lr=0.0, betas=(0.9, 0.999), weight_decay=0.0)
    par.grad = torch.full((n,), 0.37, device='cuda')
    for _ in range(2000):
        opt.step()
    m, v = (x.double() for x in opt.moments())
    want = 0.37 ** 2 * (1 - 0.999 ** 2000)
    assert abs(float(v.mean()) / want - 1) < 0.04, float(v.mean()) / want
    assert abs(float(m.mean()) / 0.37 - 1) < 0.04
    assert float((v == 0).sum()) == 0


@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')])
def test_8_bit_nonfinite_gradients_stay_in_their_block(T, bad):
    par, opt, grads = _eight(T, n=1024, steps=1)
    g = grads()[0]
    g[300] = bad
    keep = par.detach().clone()
    par.grad = f32(g)
    opt.step()
    m, v = opt.moments()
    inside = torch.zeros(1024, dtype=torch.bool, device='cuda')
    inside[256:512] = True
    assert torch.isnan(m[inside]).all() and torch.isnan(v[inside]).all()
    assert torch.isfinite(m[~inside]).all() and torch.isfinite(v[~inside]).all() and torch.isfinite(par.detach()[~inside]).all()
    assert not torch.isfinite(par.detach()[300]) and int(torch.isfinite(par.detach()).sum()) == 1023 and not torch.equal(par, keep)


def test_8_bit_zero_and_tiny_moments(T):
    par = nn.Parameter(torch.ones(600, device='cuda'))
    opt = T.AdamW([par], state_bits=8, lr=1e-2, weight_decay=0.0)
    par.grad = torch.zeros(600, device='cuda')
    opt.step()
    assert torch.equal(par.detach(), torch.ones(600, device='cuda')) and not any(bool(x.any()) for x in opt.moments())
    g = torch.full((600,), 1e-30, device='cuda')      # squares are below float32
    g[5] = 1.0                                        # beside a large one: far below the block's smallest code
    par.grad = g
    opt.step()
    m, v = opt.moments()
    assert torch.isfinite(par.detach()).all() and float(m[5]) != 0 and float(v[5]) != 0
    assert float((par.detach() - 1).abs().max()) < 1e-1


def test_mixed_groups_one_norm(T):
    """Groups with 32 and 8 bits and their own rates, float32 and bfloat16 parameters in one group: one norm over all."""
    arrays, grads = inputs([500, 64, 3000, 129], 51)
    arrays[1], arrays[3] = to_bf16([arrays[1], arrays[3]])
    dts = [torch.float32, torch.bfloat16, torch.float32, torch.bfloat16]
    params = [nn.Parameter(f32(a).to(d)) for a, d in zip(arrays, dts)]
    opt = T.AdamW([{'params': params[:2], 'state_bits': 8}, {'params': params[2:], 'lr': 3e-3, 'weight_decay': 0.0}], ema_decay=0.9, seed=3, **HP)
    refs = [R.Tensors([a], dict(HP, ema=0.9) if i < 2 else dict(HP, ema=0.9, lr=3e-3, weight_decay=0.0), 8 if i < 2 else 32, d == torch.bfloat16, 3, at)
            for i, (a, d, at) in enumerate(zip(arrays, dts, (0, 500, 564, 3564)))]
    for _ in range(2):
        gs = [to_bf16([g])[0] if d == torch.bfloat16 else g for g, d in zip(grads(), dts)]
        norm = np.sqrt(sum(float(np.sum(g.astype(np.float64) ** 2)) for g in gs))
        for p, g, d, r in zip(params, gs, dts, refs):
            p.grad = f32(g).to(d)
            r.step([g * np.float32(min(1.0, 2.0 / (norm + 1e-6)))])   # the factor of the whole
        opt.step(clip_grad_norm=2.0)
        assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm
    for i, (p, r) in enumerate(zip(params, refs)):
        same(p, r.p[0], 'p[%d]' % i)
    m, v = opt.moments()
    same(m, np.concatenate([r.m[0] for r in refs]), 'm')
    same(v, np.concatenate([r.v[0] for r in refs]), 'v')
    with pytest.raises(RuntimeError, match='moments'):
        opt.exp_avg
    with pytest.raises(RuntimeError, match='constructor'):
        opt.add_param_group({'params': [nn.Parameter(torch.zeros(3, device='cuda'))]})


def test_checkpoints_go_between_torch_and_32_and_8_bits(T):
    arrays, grads = inputs([40, 700], 61)
    a = [nn.Parameter(f32(x)) for x in arrays]
    opt = T.AdamW(a, ema_decay=0.99, **HP)
    for _ in range(3):
        for p, g in zip(a, grads()):
            p.grad = f32(g)
        opt.step()
    sd = copy.deepcopy(opt.state_dict())
    # into torch.optim.AdamW on the CPU in float64 and on from there
    b = [nn.Parameter(p.detach().cpu().double()) for p in a]
    topt = torch.optim.AdamW(b, lr=1.0)
    topt.load_state_dict({'state': {i: {k: (x.double() if k != 'step' else x) for k, x in s.items() if k != 'ema'} for i, s in sd['state'].items()},
                          'param_groups': [dict(topt.state_dict()['param_groups'][0], **{k: sd['param_groups'][0][k] for k in ('lr', 'betas', 'eps', 'weight_decay')})]})
    # and back from torch's own dictionary into a fresh optimizer
    c = [nn.Parameter(p.detach().clone()) for p in a]
    copt = T.AdamW(c, lr=1.0)
    copt.load_state_dict(topt.state_dict())
    assert copt.param_groups[0]['lr'] == HP['lr'] and copt.param_groups[0]['state_bits'] == 32
    gs = grads()
    for ps, dt, o in ((a, torch.float32, opt), (b, torch.float64, topt), (c, torch.float32, copt)):
        for p, g in zip(ps, gs):
            p.grad = torch.from_numpy(g).to(p.device, dt)
        o.step()
    for p, q, r in zip(a, b, c):
        assert torch.equal(p, r)
        assert np.abs(p.detach().cpu().numpy() - q.detach().numpy()).max() <= 16 * U * 5
    d = [nn.Parameter(f32(x)) for x in arrays]
    dopt = T.AdamW(d, state_bits=8, ema_decay=0.99, **HP)
    dopt.load_state_dict(sd)
    m, v = dopt.moments()
    for i, at in ((0, 0), (1, 40)):
        s = sd['state'][i]
        n = s['exp_avg'].numel()
        big = max(float(x.abs().max()) for x in s['exp_avg'].split(256))
        # a value moves by less than one distance of codes: an eighth of it, or 2^-16 of the block's largest below the normal range
        assert ((m[at:at + n] - s['exp_avg']).abs() <= s['exp_avg'].abs() / 8 + big * 2 ** -16).all()
        assert ((v[at:at + n] - s['exp_avg_sq']).abs() <= s['exp_avg_sq'] / 8 + float(s['exp_avg_sq'].max()) * 2 ** -32).all()
        assert torch.equal(dopt.ema_parameters()[i], s['ema'])
    with pytest.raises(ValueError):
        dopt.load_state_dict({'state': {}, 'param_groups': [dict(sd['param_groups'][0], params=[0])]})
    with pytest.raises(ValueError):
        dopt.load_state_dict({'state': {0: {'step': 1, 'exp_avg': torch.zeros(3), 'exp_avg_sq': torch.zeros(3)}}, 'param_groups': sd['param_groups']})
    with pytest.raises(TypeError):
        copy.deepcopy(dopt)


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('scale,eps', [(1e-25, 1e-8), (1e-18, 1e-8), (1e-18, 1e-13), (1e-9, 0.0), (1.0, 0.0), (1e5, 1e-8), (2e7, 1e-8), (1e9, 1e-8), (1e15, 1e-8)])
def test_the_ends_of_the_range_bit_for_bit(T, bits, scale, eps):
    """Gradients whose squares are subnormal or vanish, moments around the bounds between which the kernel leaves out the handling of the
    range (v 2^60, m 2^20, eps 2^-40), zero gradients with eps 0 (0 / 0, as the formula has it)."""
    hp = dict(HP, eps=eps)
    arrays, grads = inputs([2000, 300], 45, scale)
    params = [nn.Parameter(f32(a)) for a in arrays]
    opt = T.AdamW(params, state_bits=bits, **hp)
    ref = R.Tensors(arrays, hp, bits)
    for step in range(3):
        gs = grads()
        for p, g in zip(params, gs):
            p.grad = f32(g)
        opt.step()
        ref.step(gs)
        m, v = opt.moments()
        same(m, np.concatenate(ref.m), 'm, step %d' % step)
        same(v, np.concatenate(ref.v), 'v, step %d' % step)
        for i, p in enumerate(params):
            same(p, ref.p[i], 'p[%d], step %d' % (i, step))


def test_only_empty_parameters_and_sparse_gradients(T):
    p = [nn.Parameter(torch.zeros(0, 3, device='cuda')) for _ in range(2)]
    opt = T.AdamW(p, state_bits=8, ema_decay=0.9)
    for q in p:
        q.grad = torch.zeros_like(q)
    opt.step(clip_grad_norm=1.0)
    assert float(opt.grad_norm) == 0.0 and opt.moments()[0].numel() == 0 and float(T.clip_grad_norm_(p, 1.0)) == 0.0
    opt.load_state_dict(opt.state_dict())
    emb = nn.Embedding(10, 4, sparse=True).cuda()
    emb(torch.tensor([1, 2], device='cuda')).sum().backward()
    before = emb.weight.detach().clone()
    with pytest.raises(RuntimeError, match='does not fit'):
        T.AdamW(emb.parameters()).step()
    with pytest.raises(TypeError):
        T.clip_grad_norm_(emb.parameters(), 1.0)
    assert torch.equal(emb.weight, before)


def test_clip_from_two_threads(T):
    import threading
    sizes = [1 + (31 * i) % 900 for i in range(700)]
    jobs, errors = [], []
    for k in range(2):
        _, grads = inputs(sizes[k:], 47 + k)
        gs = grads()
        params = [nn.Parameter(torch.zeros(len(g), device='cuda')) for g in gs]
        norm = np.sqrt(sum(float(np.sum(g.astype(np.float64) ** 2)) for g in gs))
        jobs.append((params, [f32(g) for g in gs], norm))

    def work(params, gs, norm):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    for p, g in zip(params, gs):
                        p.grad = g.clone()
                    got = float(T.clip_grad_norm_(params, 1.0))
                    assert abs(got - norm) <= 2 * U * norm, (got, norm)
        except BaseException as e:   # noqa: B902 -- reported by the main thread
            errors.append(e)
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


# ---- streams, graphs, re-pointed parameters ------------------------------------------------------------------------------
@pytest.mark.parametrize('bits,count', [(32, 5), (8, 5), (32, 2500)])
def test_captured_steps(T, bits, count):
    """forward-less step in a graph: step count and learning rate move on the device; replays between eager work equal eager steps."""
    sizes = [1 + (97 * i) % 1500 for i in range(count)]
    arrays, grads = inputs(sizes, 71)
    a, b = ([nn.Parameter(f32(x)) for x in arrays] for _ in range(2))
    lr = torch.tensor(1e-2, device='cuda')
    opt = T.AdamW(a, lr=lr, state_bits=bits, ema_decay=0.9, capturable=True, weight_decay=0.1)
    ref = T.AdamW(b, lr=float(lr), state_bits=bits, ema_decay=0.9, weight_decay=0.1)
    static = [torch.zeros_like(p) for p in a]
    for p, g in zip(a, static):
        p.grad = g

    def feed():
        gs = [f32(g) for g in grads()]
        torch._foreach_copy_(static, gs)
        for p, g in zip(b, gs):
            p.grad = g
    feed()
    opt.step(clip_grad_norm=1.0)       # eager
    ref.step(clip_grad_norm=1.0)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        opt.step(clip_grad_norm=1.0)
    for k in range(4):
        feed()
        if k == 2:
            lr.fill_(3e-3)
            ref.param_groups[0]['lr'] = float(lr)
        graph.replay()
        ref.step(clip_grad_norm=1.0)
        torch.cuda.synchronize()
        junk = torch.randn(100000, device='cuda').sum()      # eager work between the replays
        for i, (p, q) in enumerate(zip(a, b)):
            assert torch.equal(p, q), (k, i)
        assert torch.equal(opt.ema, ref.ema) and bool(torch.isfinite(junk))
        assert torch.equal(opt.grad_norm, ref.grad_norm)
    assert int(opt.state_dict()['state'][0]['step']) == 5 == int(ref.state_dict()['state'][0]['step'])
    opt.step(clip_grad_norm=1.0)       # eager again
    ref.step(clip_grad_norm=1.0)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    a[0].grad = None
    with pytest.raises(RuntimeError, match='same parameters'):
        opt.step()


def test_capture_without_capturable_is_refused(T):
    p = nn.Parameter(torch.zeros(10, device='cuda'))
    p.grad = torch.ones(10, device='cuda')
    opt = T.AdamW([p])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = torch.zeros(4, device='cuda') + 1
        with pytest.raises(RuntimeError, match='capturable'):
            opt.step()
    graph.replay()
    torch.cuda.synchronize()
    assert float(q.sum()) == 4 and float(p.detach().abs().sum()) == 0


def test_two_optimizers_on_two_streams(T):
    arrays, grads = inputs([100003, 77], 81)
    streams = [torch.cuda.Stream() for _ in range(2)]
    runs = []
    torch.cuda.synchronize()
    for s in streams:
        with torch.cuda.stream(s):
            ps = [nn.Parameter(f32(x)) for x in arrays]
            runs.append((ps, T.AdamW(ps, state_bits=8, **HP)))
    ref = R.Tensors(arrays, HP, 8)
    for _ in range(3):
        gs = grads()
        for s, (ps, opt) in zip(streams, runs):
            with torch.cuda.stream(s):
                for p, g in zip(ps, gs):
                    p.grad = f32(g)
                opt.step(clip_grad_norm=5.0)
        ref.step(gs, 5.0)
    torch.cuda.synchronize()
    for ps, _ in runs:
        for i, p in enumerate(ps):
            same(p, ref.p[i], 'p[%d]' % i)


def test_re_pointed_parameters(T):
    arrays, grads = inputs([300, 20], 91)
    ps = [nn.Parameter(f32(x)) for x in arrays]
    opt = T.AdamW(ps, **HP)
    ref = R.Tensors(arrays, HP)

    def go():
        gs = grads()
        for p, g in zip(ps, gs):
            p.grad = f32(g)
        opt.step()
        ref.step(gs)
    go()
    old = ps[0].data
    ps[0].data = old.clone()
    go()
    for i, p in enumerate(ps):
        same(p, ref.p[i], 'p[%d]' % i)
    ps[1].grad = None
    ps[1].data = ps[0].data[:20]       # into the other one
    with pytest.raises(ValueError, match='share'):
        opt.step()
    ps[1].data = torch.zeros(21, device='cuda')
    with pytest.raises(RuntimeError, match='rebuild'):
        opt.step()
    with pytest.raises(ValueError, match='share'):
        T.AdamW([nn.Parameter(old), nn.Parameter(old[5:7])])
    with pytest.raises(ValueError, match='holes'):
        T.AdamW([nn.Parameter(old[::2])])
    with pytest.raises(TypeError):
        T.AdamW([nn.Parameter(old.half())])


def test_element_numbers_beyond_32_bits(T):
    """A list whose elements are numbered across 2^32 (C ABI): the hash goes on, 8-bit moments and weights as the reference has them."""
    from super_resolution_amd import _lib as L
    n, index, hp = 5000, (1 << 32) - 1500, dict(HP, ema=0.0)
    (p,), grads = inputs([n], 101)
    p = to_bf16([p])[0]
    par = f32(p).bfloat16()
    m8, v8 = (torch.zeros(n, dtype=torch.uint8, device='cuda') for _ in range(2))
    me, ve = (torch.ones(20, dtype=torch.uint8, device='cuda') for _ in range(2))
    t = (L.AdamWTensor * 1)()
    t[0].p, t[0].m, t[0].v, t[0].me, t[0].ve, t[0].n, t[0].index = par.data_ptr(), m8.data_ptr(), v8.data_ptr(), me.data_ptr(), ve.data_ptr(), n, index
    h = C.c_void_p()
    L.check(L.lib().sr_adamw_create(1, 8, 1, t, C.byref(h)))
    ref = R.Tensors([p], hp, 8, True, seed=9, index=index)
    hyper = L.AdamWHyper(hp['lr'], *hp['betas'], hp['eps'], hp['weight_decay'], 0.0, 9)
    for step in (1, 2):
        g = to_bf16(grads())[0]
        gd = f32(g).bfloat16()
        table = torch.tensor([gd.data_ptr()], device='cuda')
        L.check(L.lib().sr_adamw_step(h, C.byref(hyper), step, None, table.data_ptr(), 0, None, L.stream_ptr(par.device)))
        torch.cuda.synchronize()
        ref.step([g])
        same(par, ref.p[0], 'p, step %d' % step)
    L.lib().sr_adamw_destroy(h)


def test_a_tensor_of_more_than_2_31_elements(T):
    """Offsets beyond 32 bits: the ends of a tensor of 2^31 + 1500 bfloat16 values, 8-bit moments."""
    n = (1 << 31) + 1500
    par = nn.Parameter(torch.full((n,), 0.5, dtype=torch.bfloat16, device='cuda'))
    grad = torch.zeros(n, dtype=torch.bfloat16, device='cuda')
    rng = np.random.default_rng(1)
    head, tail = (to_bf16([rng.standard_normal(4096).astype(np.float32)])[0] for _ in range(2))
    cut = (n - 3000) // 256 * 256          # from a block's start to the end
    tail = tail[:n - cut]
    grad[:4096] = f32(head).bfloat16()
    grad[cut:cut + len(tail)] = f32(tail).bfloat16()
    par.grad = grad
    opt = T.AdamW([par], state_bits=8, seed=2, **HP)
    opt.step(clip_grad_norm=1e9)
    norm = np.sqrt(float(np.sum(head.astype(np.float64) ** 2) + np.sum(tail.astype(np.float64) ** 2)))
    assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm
    m, v = opt.moments(torch.bfloat16)
    for at, g in ((0, head), (cut, tail)):
        ref = R.Tensors([np.full(len(g), 0.5, np.float32)], HP, 8, True, 2, at)
        ref.step([g])
        same(par[at:at + len(g)], ref.p[0], 'p at %d' % at)
        same(m[at:at + len(g)], ref.m[0], 'm at %d' % at)
        same(v[at:at + len(g)], ref.v[0], 'v at %d' % at)
    assert not bool(m[4096:1 << 20].any()) and not bool(v[4096:1 << 20].any())


# ---- clipping ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('name', list(SIZES))
@pytest.mark.parametrize('mode', ['f32', 'bf16', 'mixed'])
@pytest.mark.parametrize('max_norm', [0.5, 1e9])
def test_clip_grad_norm(T, name, mode, max_norm):
    arrays, grads = inputs(SIZES[name], 111)
    dts = [torch.bfloat16 if mode == 'bf16' or mode == 'mixed' and i % 2 else torch.float32 for i in range(len(arrays))]
    gs = [to_bf16([g])[0] if d == torch.bfloat16 else g for g, d in zip(grads(), dts)]
    params = [nn.Parameter(f32(a).to(d)) for a, d in zip(arrays, dts)]
    buf = []
    for p, g, d in zip(params, gs, dts):
        b = torch.full((len(g) + 2,), 7.0, dtype=d, device='cuda')
        b[1:1 + len(g)] = f32(g).to(d)
        p.grad = b[1:1 + len(g)]
        buf.append(b)
    norm = np.sqrt(sum(float(np.sum(g.astype(np.float64) ** 2)) for g in gs))
    before = [p.grad._version for p in params]
    got = T.clip_grad_norm_(params, max_norm)
    assert abs(float(got) - norm) <= 2 * U * norm and got.shape == ()
    f = max_norm / (norm + 1e-6)
    factor = np.float32(1.0 if f >= 1 else f)
    for i, (p, g, d, b) in enumerate(zip(params, gs, dts, buf)):
        want = g * factor
        same(p.grad, torch.from_numpy(want).to(d).float().numpy(), 'gradient %d' % i)
        assert float(b[0]) == 7.0 and float(b[-1]) == 7.0
        assert p.grad._version > before[i]


def test_clip_special_values(T):
    p = [nn.Parameter(torch.zeros(3, device='cuda')) for _ in range(3)]
    p[0].grad = torch.tensor([1e30, -1e30, 0.0], device='cuda')      # squares beyond float32
    p[1].grad = torch.zeros(3, device='cuda')
    norm = T.clip_grad_norm_(p, 1.0)                                  # p[2] has none
    assert abs(float(norm) / (2 ** 0.5 * 1e30) - 1) < 1e-6 and p[2].grad is None
    assert torch.allclose(p[0].grad, torch.tensor([2 ** -0.5, -2 ** -0.5, 0.0], device='cuda'), rtol=1e-6, atol=0)
    assert float(T.clip_grad_norm_(p[1], 1.0)) == 0.0 and not bool(p[1].grad.any())
    p[0].grad = torch.tensor([float('inf'), 1.0, 2.0], device='cuda')
    with pytest.raises(RuntimeError, match='finite'):
        T.clip_grad_norm_(p, 1.0, error_if_nonfinite=True)
    assert torch.equal(p[0].grad, torch.tensor([float('inf'), 1.0, 2.0], device='cuda'))
    assert float(T.clip_grad_norm_(p, 1.0)) == float('inf')
    assert torch.isnan(p[0].grad[0]) and not bool(p[0].grad[1:].any())   # as torch: inf * 0
    p[0].grad = torch.tensor([float('nan'), 1.0, 2.0], device='cuda')
    assert np.isnan(float(T.clip_grad_norm_(iter(p), 1.0))) and torch.isnan(p[0].grad).all()
    p[0].grad = torch.ones(3, device='cuda')
    assert abs(float(T.clip_grad_norm_(p[0], 0.0)) - 3 ** 0.5) < 1e-6 and not bool(p[0].grad.any())


def test_clip_layouts_and_shared_gradients(T):
    p = [nn.Parameter(torch.zeros(s, device='cuda')) for s in ((6, 8), (6, 8), (5,), (2, 3, 4, 4))]
    whole = torch.randn(6, 16, device='cuda')
    p[0].grad = whole[:, ::2]                                        # holes
    p[1].grad = torch.randn(8, 6, device='cuda').t()
    p[2].grad = torch.randn(5, device='cuda')
    p[3].grad = torch.randn(2, 3, 4, 4, device='cuda').to(memory_format=torch.channels_last)
    gs, rest = [q.grad.clone() for q in p], whole[:, 1::2].clone()
    norm = T.clip_grad_norm_(p, 0.25)
    want = sum(float(g.double().square().sum()) for g in gs) ** 0.5
    assert abs(float(norm) - want) <= 2 * U * want
    factor = torch.tensor(0.25 / (want + 1e-6), dtype=torch.float32, device='cuda')
    for q, g in zip(p, gs):
        assert torch.equal(q.grad, g * factor)
    assert torch.equal(whole[:, 1::2], rest)
    a, b = nn.Parameter(torch.zeros(4, device='cuda')), nn.Parameter(torch.zeros(4, device='cuda'))
    a.grad = torch.ones(4, device='cuda')
    b.grad = a.grad
    with pytest.raises(RuntimeError, match='share'):
        T.clip_grad_norm_([a, b], 1.0)
    with pytest.raises(RuntimeError, match='share'):
        T.clip_grad_norm_([a, a], 1.0)
    assert torch.equal(a.grad, torch.ones(4, device='cuda'))
    a.grad = None
    h = nn.Parameter(torch.zeros(4, dtype=torch.float16, device='cuda'))
    h.grad = torch.ones(4, dtype=torch.float16, device='cuda')
    with pytest.raises(TypeError, match='tensor 1'):
        T.clip_grad_norm_([b, h], 1.0)


@pytest.mark.parametrize('count', [4, 2500])
def test_clip_captured(T, count):
    sizes = [1 + (53 * i) % 700 for i in range(count)]
    arrays, grads = inputs(sizes, 121)
    p = [nn.Parameter(f32(a)) for a in arrays]
    for q in p:
        q.grad = torch.zeros_like(q)
    T.clip_grad_norm_(p, 1.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = T.clip_grad_norm_(p, 1.0)
    for _ in range(3):
        gs = [f32(g) for g in grads()]
        torch._foreach_copy_([q.grad for q in p], gs)
        graph.replay()
        torch.cuda.synchronize()
        twin = [nn.Parameter(torch.zeros_like(q)) for q in p]
        for q, g in zip(twin, gs):
            q.grad = g
        assert torch.equal(T.clip_grad_norm_(twin, 1.0), norm)
        assert all(torch.equal(q.grad, r.grad) for q, r in zip(p, twin))


# ---- as the framework's training uses them -------------------------------------------------------------------------------
@pytest.mark.parametrize('bits', [32, 8])
def test_train_step_with_adamw(T, bits):
    """train_step on RRDBNet-FDConv: the first step against FlatAdam's update of the same gradients (weight_decay 0: the same rule), the
    running average, a falling count of nothing left behind -- every parameter moves and the cached spectral bases follow."""
    import super_resolution_amd as sra
    torch.manual_seed(0)
    net = sra.replace_conv_with_fdconv(sra.RRDBNet(1, 1, 4, 64, 1, 32)).cuda()
    twin = copy.deepcopy(net)
    x, y = torch.rand(2, 1, 16, 16, device='cuda'), torch.rand(2, 1, 64, 64, device='cuda')
    opt = T.AdamW(net.parameters(), lr=1e-3, weight_decay=0.0, state_bits=bits, ema_decay=0.5)
    start = [p.detach().clone() for p in net.parameters()]
    loss = T.train_step(net, opt, x, y, clip_grad_norm=1.0)
    assert bool(torch.isfinite(loss)) and float(opt.grad_norm) > 0
    grads = [p.grad for p in net.parameters()]
    flat = T.FlatAdam(twin.parameters(), lr=1e-3)
    for q, g in zip(twin.parameters(), grads):
        q.grad = g.clone()
    flat.step(clip_grad_norm=1.0)
    for (n, p), q, s, e in zip(net.named_parameters(), twin.parameters(), start, opt.ema_parameters()):
        # one step is at most lr; m and v are not rounded before it: float32 roundings of p and of the update (the clip factors
        # differ by FlatAdam's float32 norm of 20000 terms, 2^-13 of the gradient, which eps alone turns into a difference)
        assert float((p - q).detach().abs().max()) <= 4 * U * float(s.abs().max()) + 1e-3 * 2 ** -12, n
        assert torch.allclose(e, 0.5 * s + 0.5 * p.detach(), rtol=4 * U, atol=4 * U * float(s.abs().max())), n
    # evaluation after the step sees the new weights (FDConv keys its cached bases on the version counters)
    net.eval()
    fresh = sra.replace_conv_with_fdconv(sra.RRDBNet(1, 1, 4, 64, 1, 32)).cuda()
    fresh.load_state_dict(net.state_dict())
    with torch.no_grad():
        assert torch.equal(net(x), fresh.eval()(x))
    T.train_step(net, opt, x, y)
    assert int(opt.state_dict()['state'][0]['step']) == 2


def test_scheduler_drives_the_rate(T):
    p = nn.Parameter(torch.ones(300, device='cuda'))
    opt = T.AdamW([p], lr=1e-2, weight_decay=0.0)
    sch = torch.optim.lr_scheduler.ReduceLROnPlateau(opt, mode='min', factor=0.5, patience=0)
    ref = R.Tensors([np.ones(300, np.float32)], dict(HP, weight_decay=0.0))
    for _ in range(4):
        g = np.random.default_rng(7).standard_normal(300).astype(np.float32)
        p.grad = f32(g)
        opt.step()
        ref.hp = dict(ref.hp, lr=opt.param_groups[0]['lr'])
        ref.step([g])
        sch.step(1.0)
    assert opt.param_groups[0]['lr'] < 1e-2
    same(p, ref.p[0], 'p')
    assert float(opt.step(closure=lambda: torch.tensor(3.0))) == 3.0


def _two_ranks(rank, port, q):
    import os
    import sys
    sys.path[:0] = [os.path.dirname(os.path.dirname(os.path.abspath(__file__))), os.path.dirname(os.path.abspath(__file__))]
    os.environ.update(MASTER_ADDR='127.0.0.1', MASTER_PORT=str(port))
    import torch.distributed as dist
    dist.init_process_group('gloo', rank=rank, world_size=2)
    from super_resolution_amd import train
    arrays, _ = inputs([700, 33], 131)
    params = [nn.Parameter(f32(a) + rank) for a in arrays]      # replicas that start apart
    opt = train.AdamW(params, state_bits=8, seed=4, **HP)
    for p, g in zip(params, _rank_gradients(rank)):
        p.grad = f32(g)
    opt.step(clip_grad_norm=1.0)
    torch.cuda.synchronize()
    q.put((rank, [p.detach().cpu().tolist() for p in params], float(opt.grad_norm)))
    dist.barrier()
    dist.destroy_process_group()


def _rank_gradients(rank):
    rng = np.random.default_rng(140 + rank)
    return [rng.standard_normal(n).astype(np.float32) for n in (700, 33)]


def test_two_ranks_average_their_gradients(T):
    """Two processes on the one card, gradients exchanged over the host: both end with rank 0's parameters stepped by the mean."""
    import os
    import torch.multiprocessing as mp
    ctx = mp.get_context('spawn')
    q = ctx.Queue()
    procs = [ctx.Process(target=_two_ranks, args=(r, 35500 + os.getpid() % 2000, q)) for r in range(2)]
    for p in procs:
        p.start()
    res = sorted(q.get(timeout=100) for _ in procs)
    for p in procs:
        p.join(60)
        assert p.exitcode == 0
    arrays, _ = inputs([700, 33], 131)
    ref = R.Tensors(arrays, HP, 8, seed=4)
    ref.step([(a + b) / np.float32(2) for a, b in zip(_rank_gradients(0), _rank_gradients(1))], 1.0)
    for _, ps, norm in res:
        for i, p in enumerate(ps):
            same(torch.tensor(p), ref.p[i], 'p[%d]' % i)
    assert res[0][2] == res[1][2]
