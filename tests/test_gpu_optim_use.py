"""train.AdamW and train.clip_grad_norm_ in the calls around a training loop: re-pointed parameters, schedulers and checkpoints, captured
steps beside evaluation, many groups, gradients that share memory.

As in test_gpu_optim.py float32 results are compared bit for bit with the formulas of tests/adamw_ref.py."""
import copy

import numpy as np
import pytest
import torch
import torch.nn as nn

import adamw_ref as R

pytestmark = pytest.mark.gpu
U = 2.0 ** -24      # largest relative error of one float32 rounding
HP = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)


@pytest.fixture(scope='module')
def T():
    from super_resolution_amd import _lib, train
    _lib.lib()
    assert torch.cuda.is_available()
    return train


def f32(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def same(got, want, what):
    """Bit for bit (NaN as NaN), in the order of the indices, whatever the strides."""
    got, want = got.detach().float().cpu().contiguous().numpy().reshape(-1), np.asarray(want).reshape(-1)
    assert got.shape == want.shape, what
    bad = ~((got == want) | (np.isnan(got) & np.isnan(want)))
    assert not bad.any(), '%s: %d of %d differ, first %d: %r, reference %r' % (what, bad.sum(), bad.size, bad.argmax(), got[bad.argmax()], want[bad.argmax()])


# ---- parameters whose memory order changes -------------------------------------------------------------------------------
ORDERS = {
    'channels_last': ((4, 8, 3, 3), lambda x: x.to(memory_format=torch.channels_last)),
    'contiguous again': ((4, 8, 3, 3), lambda x: x.contiguous()),
    'transposed memory': ((40, 60), lambda x: x.t().contiguous().t()),
    'transposed at the same address': ((24, 24), lambda x: x.t()),
}


@pytest.mark.parametrize('name', list(ORDERS))
@pytest.mark.parametrize('capturable', [False, True])
def test_another_memory_order_keeps_every_elements_moments(T, name, capturable):
    """Element (i, j, ...) keeps its moments and its average, as in torch.optim.AdamW."""
    shape, turn = ORDERS[name]
    rng = np.random.default_rng(5)
    a, b = rng.standard_normal(shape).astype(np.float32), rng.standard_normal(50).astype(np.float32)
    p, q = nn.Parameter(f32(a)), nn.Parameter(f32(b))
    if name == 'contiguous again':
        p.data = p.data.to(memory_format=torch.channels_last)
    opt = T.AdamW([q, p], ema_decay=0.9, capturable=capturable, **HP)
    ref = R.Tensors([b, a.reshape(-1)], dict(HP, ema=0.9))

    def go():
        gs = [rng.standard_normal(50).astype(np.float32), rng.standard_normal(shape).astype(np.float32)]
        q.grad, p.grad = f32(gs[0]), f32(gs[1])
        opt.step()
        ref.step([g.reshape(-1) for g in gs])

    def check(what):
        same(p, ref.p[1], 'p, ' + what)
        same(q, ref.p[0], 'q, ' + what)
        state = opt.state_dict()['state']
        for i in range(2):
            same(state[i]['exp_avg'], ref.m[i], 'm[%d], %s' % (i, what))
            same(state[i]['exp_avg_sq'], ref.v[i], 'v[%d], %s' % (i, what))
            same(state[i]['ema'], ref.ema[i], 'ema[%d], %s' % (i, what))
            same(opt.ema_parameters()[i], ref.ema[i], 'ema_parameters[%d], %s' % (i, what))
    go()
    go()
    check('before')
    p.data = turn(p.data)
    ref.p[1] = p.detach().cpu().contiguous().numpy().reshape(-1)     # (the transposed one has other values at its indices)
    check('re-pointed')
    saved = copy.deepcopy(opt.state_dict())
    go()
    go()
    check('stepped')
    opt.load_state_dict(saved)       # the dictionary goes by index, not by memory
    for i, s in opt.state_dict()['state'].items():
        assert all(torch.equal(s[k], saved['state'][i][k]) for k in ('exp_avg', 'exp_avg_sq', 'ema'))


def test_another_memory_order_with_8_bit_moments(T):
    """The moments are rounded once more on the way.  Gradients 2^(i % 5): all codes in the normal range, where one rounding moves a value
    by less than its eighth; so two of them (the way and the step with zero gradients after it) by a factor within (1 - 1/8)^2 and
    (1 + 1/8)^2.  Neighbours differ by a factor of two at least."""
    shape = (8, 16, 3, 3)
    n = int(np.prod(shape))
    g = (2.0 ** (np.arange(n) % 5)).astype(np.float32).reshape(shape)
    p, q = nn.Parameter(torch.ones(shape, device='cuda')), nn.Parameter(torch.ones(300, device='cuda'))
    opt = T.AdamW([p, q], state_bits=8, ema_decay=0.9, **HP)
    for _ in range(3):
        p.grad, q.grad = f32(g), torch.ones(300, device='cuda')
        opt.step()
    m, v = (opt.state_dict()['state'][0][k].cpu().numpy() for k in ('exp_avg', 'exp_avg_sq'))
    ema, other = opt.ema_parameters()[0].cpu().numpy(), opt.state_dict()['state'][1]['exp_avg'].clone()
    p.data = p.data.to(memory_format=torch.channels_last)
    p.grad, q.grad = torch.zeros_like(p), None
    opt.step()
    s = opt.state_dict()['state']
    lo, hi = (1 - 1 / 8) ** 2, (1 + 1 / 8) ** 2
    r = s[0]['exp_avg'].cpu().numpy() / (np.float32(0.9) * m)
    assert lo <= r.min() and r.max() <= hi, (r.min(), r.max())
    r = s[0]['exp_avg_sq'].cpu().numpy() / (np.float32(0.999) * v)
    assert lo <= r.min() and r.max() <= hi, (r.min(), r.max())
    want = ema * np.float32(0.9) + p.detach().cpu().numpy() * np.float32(1 - 0.9)
    same(opt.ema_parameters()[0], want, 'ema')
    assert torch.equal(s[1]['exp_avg'], other)


def test_another_shape_is_refused(T):
    p = nn.Parameter(torch.randn(6, 4, device='cuda'))
    opt = T.AdamW([p], **HP)
    for x in (p.data.t().contiguous(), p.data.clone().view(-1)):
        p.data = x
        p.grad = torch.zeros_like(p)
        with pytest.raises(RuntimeError, match='rebuild'):
            opt.step()


# ---- clipping ------------------------------------------------------------------------------------------------------------
def test_clip_arguments_by_position(T):
    p = nn.Parameter(torch.zeros(3, device='cuda'))
    p.grad = torch.tensor([float('inf'), 1.0, 2.0], device='cuda')
    assert float(T.clip_grad_norm_(p, 1e30, 2.0)) == float('inf')        # the norm's type, not error_if_nonfinite
    p.grad = torch.tensor([float('inf'), 1.0, 2.0], device='cuda')
    with pytest.raises(RuntimeError, match='finite'):
        T.clip_grad_norm_(p, 1.0, 2.0, True)
    p.grad = torch.tensor([3.0, 4.0, 0.0], device='cuda')
    with pytest.raises(ValueError, match='norm_type'):
        T.clip_grad_norm_(p, 1.0, float('inf'))
    assert p.grad.tolist() == [3.0, 4.0, 0.0]


@pytest.mark.parametrize('name', ['the same tensor', 'two views alike', 'columns of each other', 'a dense one over a strided one', 'one parameter twice'])
def test_clip_refuses_shared_memory_in_any_layout(T, name):
    """A gradient that would be scaled twice is refused before anything is written."""
    whole = torch.ones(6, 16, device='cuda')
    ps = [nn.Parameter(torch.zeros(s, device='cuda')) for s in ((6, 8), (6, 8), (7,))]
    ps[2].grad = torch.full((7,), 3.0, device='cuda')
    ps[0].grad = whole[:, ::2]
    if name == 'the same tensor':
        ps[1].grad = ps[0].grad
    elif name == 'two views alike':
        ps[1].grad = whole[:, ::2]
    elif name == 'columns of each other':
        ps[1].grad = whole[:, :8]
    elif name == 'a dense one over a strided one':
        ps[1].grad = whole[:3].view(6, 8)
    else:
        ps.append(ps[0])
    with pytest.raises(RuntimeError, match='share'):
        T.clip_grad_norm_(ps, 1.0)
    assert bool((whole == 1).all()) and bool((ps[2].grad == 3).all())


def test_clip_refuses_repeated_elements(T):
    """Expanded gradients, and windows that slide, cannot be scaled in place (torch raises too): refused before anything is written."""
    for g in (torch.ones(6, 1, device='cuda').expand(6, 8), torch.ones(60, device='cuda').as_strided((6, 8), (3, 1))):
        ps = [nn.Parameter(torch.zeros(s, device='cuda')) for s in ((7,), (2,), (6, 8))]
        ps[0].grad, ps[2].grad = torch.full((7,), 3.0, device='cuda'), g
        with pytest.raises(RuntimeError, match='tensor 2.*repeat'):
            T.clip_grad_norm_(ps, 1.0)
        assert bool((g == 1).all()) and bool((ps[0].grad == 3).all())


def test_clip_of_interleaved_gradients(T):
    """Views that lie between each other without sharing an element are scaled like any others."""
    whole, half = torch.ones(6, 16, device='cuda'), torch.ones(4, 6, 2, device='cuda', dtype=torch.bfloat16)
    ps = [nn.Parameter(torch.zeros(s, device='cuda', dtype=d)) for s, d in (((6, 8), torch.float32), ((6, 8), torch.float32), ((7,), torch.float32),
                                                                           ((4, 6), torch.bfloat16), ((4, 6), torch.bfloat16))]
    for p, g in zip(ps, (whole[:, ::2], whole[:, 1::2], torch.full((7,), 3.0, device='cuda'), half[..., 0], half[..., 1])):
        p.grad = g
    want = (96 + 9 * 7 + 48) ** 0.5
    assert abs(float(T.clip_grad_norm_(ps, 1.0)) - want) <= 2 * U * want
    f = np.float32(1.0 / (want + 1e-6))
    assert bool((whole == float(f)).all()) and bool((ps[2].grad == float(np.float32(3) * f)).all())
    assert bool((half == torch.tensor(f).bfloat16().cuda()).all())


def test_clip_names_the_parameter_that_does_not_fit(T):
    """Counted among the parameters, also where one has no gradient and another one is not dense."""
    ps = [nn.Parameter(torch.zeros(4, 3, device='cuda', dtype=d)) for d in (torch.float32, torch.float32, torch.float16)]
    whole = torch.ones(4, 6, device='cuda')
    ps[1].grad, ps[2].grad = whole[:, ::2], torch.ones(4, 3, device='cuda', dtype=torch.float16)
    with pytest.raises(TypeError, match='tensor 2'):
        T.clip_grad_norm_(ps, 1.0)
    assert bool((whole == 1).all())


# ---- checkpoints, schedulers ---------------------------------------------------------------------------------------------
def _one(T, **kw):
    p = nn.Parameter(torch.ones(300, device='cuda'))
    return p, T.AdamW([p], **dict(dict(lr=1e-2), **kw))


def test_a_scheduler_resumes(T):
    """What a scheduler keeps in the groups (initial_lr, max_lr, ...) comes back with the checkpoint; what belongs to the layout or to
    another optimizer's implementation does not."""
    p, opt = _one(T)
    sch = torch.optim.lr_scheduler.StepLR(opt, step_size=2, gamma=0.1)
    p.grad = torch.ones_like(p)
    for _ in range(3):
        opt.step()
        sch.step()
    saved = copy.deepcopy(opt.state_dict())
    _, again = _one(T, state_bits=8)
    again.load_state_dict(saved)
    assert again.param_groups[0]['initial_lr'] == 1e-2 and again.param_groups[0]['state_bits'] == 8
    sch2 = torch.optim.lr_scheduler.StepLR(again, step_size=2, gamma=0.1, last_epoch=sch.last_epoch - 1)   # (the constructor takes a step)
    p2 = again.params[0]
    for _ in range(2):
        p2.grad = torch.ones_like(p2)
        opt.step()
        again.step()
        sch.step()
        sch2.step()
        assert abs(opt.param_groups[0]['lr'] - again.param_groups[0]['lr']) <= 1e-12
    _, third = _one(T)
    theirs = torch.optim.AdamW([nn.Parameter(torch.ones(300))], lr=3e-4)
    third.load_state_dict(theirs.state_dict())
    assert third.param_groups[0]['lr'] == 3e-4 and 'fused' not in third.param_groups[0] and 'foreach' not in third.param_groups[0]
    with pytest.raises(ValueError, match='decay'):      # Adam's decay is not this one
        third.load_state_dict(torch.optim.Adam([nn.Parameter(torch.ones(300))], weight_decay=0.1).state_dict())
    third.load_state_dict(torch.optim.Adam([nn.Parameter(torch.ones(300))], lr=2e-4).state_dict())
    assert third.param_groups[0]['lr'] == 2e-4


def test_loading_takes_copies(T):
    p, opt = _one(T, betas=[0.9, 0.99])
    opt.param_groups[0]['note'] = {'k': [1]}
    saved = opt.state_dict()
    _, other = _one(T)
    other.load_state_dict(saved)
    other.param_groups[0]['note']['k'].append(2)
    other.param_groups[0]['betas'][1] = 0.5
    assert opt.param_groups[0]['note'] == {'k': [1]} and list(opt.param_groups[0]['betas']) == [0.9, 0.99]


def test_loading_keeps_the_rate_on_the_device(T):
    """A captured step reads the learning rate where it was: loading writes there."""
    (p, opt), (q, ref) = _one(T, lr=torch.tensor(1e-2, device='cuda'), capturable=True), _one(T)
    lr = opt.param_groups[0]['lr']
    for x in (p, q):
        x.grad = torch.linspace(-1, 1, 300, device='cuda')
    opt.step()
    ref.step()
    saved = copy.deepcopy(opt.state_dict())
    saved['param_groups'][0]['lr'] = torch.tensor(3e-3, device='cuda')
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    opt.load_state_dict(saved)
    assert opt.param_groups[0]['lr'] is lr and float(lr) == float(np.float32(3e-3))
    ref.param_groups[0]['lr'] = float(lr)
    for k in range(3):
        graph.replay()
        ref.step()
        torch.cuda.synchronize()
        junk = torch.full((1000,), 7.0, device='cuda').sum()
        assert torch.equal(p, q), k
        if k == 1:      # and the dictionary's tensor is not the optimizer's
            saved['param_groups'][0]['lr'].fill_(1.0)
    assert bool(junk == 7000)
    saved['param_groups'][0]['lr'] = 5e-4
    opt.load_state_dict(saved)
    assert opt.param_groups[0]['lr'] is lr and float(lr) == float(np.float32(5e-4))


def test_loading_where_groups_share_the_rates_tensor(T):
    def build(**kw):
        ps = [nn.Parameter(torch.ones(30, device='cuda')) for _ in range(2)]
        return ps, T.AdamW([{'params': [p]} for p in ps], lr=torch.tensor(1e-2, device='cuda'), **kw)
    ps, opt = build(capturable=True)
    lr = opt.param_groups[0]['lr']
    assert opt.param_groups[1]['lr'] is lr
    saved = opt.state_dict()
    saved['param_groups'][0]['lr'], saved['param_groups'][1]['lr'] = 0.25, 0.25
    opt.load_state_dict(saved)
    assert [g['lr'] is lr for g in opt.param_groups] == [True, True] and float(lr) == 0.25
    saved['param_groups'][1]['lr'] = 0.5
    for p in ps:
        p.grad = torch.ones_like(p)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    with pytest.raises(ValueError, match='captured'):
        opt.load_state_dict(saved)
    assert float(lr) == 0.25
    _, free = build(capturable=True)
    free.load_state_dict(saved)
    assert [float(g['lr']) for g in free.param_groups] == [0.25, 0.5]
    _, eager = build()
    saved['param_groups'][1]['lr'] = torch.tensor(0.5, device='cuda')
    eager.load_state_dict(saved)
    assert eager.param_groups[1]['lr'] == 0.5 and not torch.is_tensor(eager.param_groups[1]['lr'])


# ---- captured steps ------------------------------------------------------------------------------------------------------
def test_replayed_steps_reach_what_is_cached(T):
    """Networks keep packed weights under the parameters' version counters; replayed() moves them after replays of a captured step."""
    import super_resolution_amd as sra
    torch.manual_seed(0)
    net = sra.SRVGGNetCompact(3, 3, 64, 2, 4).cuda()
    x = torch.rand(1, 3, 16, 16, device='cuda')
    opt = T.AdamW(net.parameters(), lr=1e-2, capturable=True)
    for p in net.parameters():
        p.grad = torch.randn_like(p)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()

    def evaluate():
        net.eval()
        fresh = sra.SRVGGNetCompact(3, 3, 64, 2, 4).cuda().eval()
        fresh.load_state_dict(net.state_dict())
        with torch.no_grad():
            return net(x), fresh(x)
    a, b = evaluate()
    assert torch.equal(a, b)
    for _ in range(2):
        graph.replay()
        graph.replay()
        before = [p._version for p in net.parameters()]
        opt.replayed()
        assert all(p._version > v for p, v in zip(net.parameters(), before))
        c, d = evaluate()
        assert torch.equal(c, d) and not torch.equal(a, c)
        a = c


def test_the_average_of_parameters_without_a_step_is_saved(T):
    """Weights loaded after construction: the average of a frozen layer is on its way from the old ones to them."""
    def build():
        ps = [nn.Parameter(torch.zeros(20, 30, device='cuda')), nn.Parameter(torch.zeros(50, device='cuda')), nn.Parameter(torch.zeros(6, 4, device='cuda'))]
        ps[0].data = ps[0].data.t().contiguous().t()
        return ps, T.AdamW(ps, ema_decay=0.9)
    ps, opt = build()
    with torch.no_grad():
        for k, p in enumerate(ps):
            p.copy_(torch.arange(p.numel(), device='cuda').view(p.shape) + 1.0 + k)
    first = copy.deepcopy(opt.state_dict())              # before any step
    for _ in range(3):
        ps[1].grad = torch.ones(50, device='cuda')
        opt.step()
    saved = copy.deepcopy(opt.state_dict())
    assert sorted(saved['state']) == [1] and bool((opt.ema_parameters()[0] < ps[0]).all())
    for sd, want in ((saved, [e.clone() for e in opt.ema_parameters()]), (first, [torch.zeros_like(p) for p in ps])):
        qs, other = build()
        with torch.no_grad():
            for p, q in zip(ps, qs):
                q.copy_(p)
        other.load_state_dict(sd)
        for got, w in zip(other.ema_parameters(), want):
            assert torch.equal(got, w)
    bad = dict(saved, ema={0: torch.zeros(3)})
    with pytest.raises(ValueError, match='ema'):
        other.load_state_dict(bad)
    with pytest.raises(ValueError, match='no group'):
        other.load_state_dict(dict(saved, ema={9: torch.zeros(3)}))
    # into torch's, and a dictionary without averages
    topt = torch.optim.AdamW([nn.Parameter(p.detach().clone()) for p in ps])
    topt.load_state_dict(saved)
    other.load_state_dict({k: saved[k] for k in ('state', 'param_groups')})
    assert torch.equal(other.ema_parameters()[0], qs[0]) and torch.equal(other.ema_parameters()[1], saved['state'][1]['ema'])
    plain = T.AdamW([nn.Parameter(p.detach().clone()) for p in ps])
    plain.load_state_dict(saved)
    assert 'ema' not in plain.state_dict()


# ---- refused calls -------------------------------------------------------------------------------------------------------
def test_refused_calls_leave_version_counters(T):
    """Autograd and the networks' caches take a moved counter for a write."""
    def counters(ps):
        return [(p._version, None if p.grad is None else p.grad._version) for p in ps]
    whole = torch.ones(6, 16, device='cuda')
    ps = [nn.Parameter(torch.ones(s, device='cuda')) for s in ((5,), (6, 8), (6, 8), (300,))]
    ps[0].grad = torch.full((5,), float('inf'), device='cuda')
    ps[3].grad = torch.ones(300, device='cuda')
    before = counters(ps)
    with pytest.raises(RuntimeError, match='finite'):
        T.clip_grad_norm_(ps, 1.0, error_if_nonfinite=True)
    assert counters(ps) == before
    ps[1].grad = whole[:, ::2]
    before = counters(ps)
    with pytest.raises(RuntimeError, match='finite'):
        T.clip_grad_norm_(ps, 1.0, error_if_nonfinite=True)
    assert counters(ps) == before
    ps[2].grad = ps[1].grad
    before = counters(ps)
    with pytest.raises(RuntimeError, match='share'):
        T.clip_grad_norm_(ps, 1.0)
    assert counters(ps) == before
    ps[1].grad = ps[2].grad = torch.ones(6, 8, device='cuda')
    before = counters(ps)
    with pytest.raises(RuntimeError, match='share'):
        T.clip_grad_norm_(ps, 1.0)
    assert counters(ps) == before
    ps[1].grad = None
    half = nn.Parameter(torch.ones(3, device='cuda', dtype=torch.float16))
    half.grad = torch.ones_like(half)
    before = counters(ps + [half])
    with pytest.raises(TypeError):
        T.clip_grad_norm_(ps + [half], 1.0)
    with pytest.raises(RuntimeError, match='not a tensor'):
        T.clip_grad_norm_(ps + [3], 1.0)
    assert counters(ps + [half]) == before
    # steps: two groups, the second one refused
    opt = T.AdamW([{'params': ps[:2]}, {'params': ps[2:]}], capturable=True)
    opt.step()
    ps[3].data = torch.ones(301, device='cuda')
    ps[3].grad = None
    before = counters(ps)
    with pytest.raises(RuntimeError, match='rebuild'):
        opt.step()
    assert counters(ps) == before
    ps[3].data = torch.ones(300, device='cuda')
    ps[1].grad = torch.ones(6, 8, device='cuda')
    before = counters(ps)
    with pytest.raises(RuntimeError, match='same parameters'):
        opt.step()
    assert counters(ps) == before


@pytest.mark.parametrize('bf16', [False, True])
def test_more_groups_than_a_norm_takes_lists(T, bf16):
    """Layer-wise rates: 150 groups, with the norm of the whole, tensors without a gradient and empty ones among them."""
    rng = np.random.default_rng(9)
    sizes = [1 + (617 * i) % 3001 for i in range(150)]
    sizes[3], sizes[7], sizes[149] = 0, 70001, 5
    arrays = [rng.standard_normal(n).astype(np.float32) for n in sizes]
    dts = [torch.bfloat16 if bf16 and i % 3 == 0 else torch.float32 for i in range(150)]
    arrays = [torch.from_numpy(a).to(d).float().numpy() for a, d in zip(arrays, dts)]
    params = [nn.Parameter(f32(a).to(d)) for a, d in zip(arrays, dts)]
    starts = np.cumsum([0] + sizes)
    opt = T.AdamW([{'params': [p], 'lr': 1e-3 * (1 + i % 7)} for i, p in enumerate(params)], seed=3, **HP)
    refs = [R.Tensors([a], dict(HP, lr=1e-3 * (1 + i % 7)), 32, d == torch.bfloat16, 3, int(at)) for i, (a, d, at) in enumerate(zip(arrays, dts, starts))]
    for clip in (None, 0.5, 1e9):
        gs = [torch.from_numpy(rng.standard_normal(n).astype(np.float32)).to(d).float().numpy() for n, d in zip(sizes, dts)]
        for i in (11, 64, 149):
            gs[i] = None
        norm = np.sqrt(sum(float(np.sum(g.astype(np.float64) ** 2)) for g in gs if g is not None))
        factor = 1.0 if clip is None else min(1.0, clip / (norm + 1e-6))
        for p, g, d, r in zip(params, gs, dts, refs):
            p.grad = None if g is None else f32(g).to(d)
            r.step([None if g is None else g * np.float32(factor)])
        opt.step(clip_grad_norm=clip)
        if clip is not None:
            assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm
    for i, (p, r) in enumerate(zip(params, refs)):
        same(p, r.p[0], 'p[%d]' % i)


def test_capturable_loads_parameters_without_a_step(T):
    """One count on the device serves the parameters that have one: the others keep theirs, and may not join later."""
    def build(n=3, **kw):
        ps = [nn.Parameter(torch.ones(40 + k, device='cuda')) for k in range(n)]
        return ps, T.AdamW(ps, **dict(HP, **kw))
    ps, opt = build()
    for p in ps[:2]:
        p.grad = torch.ones_like(p)
    for _ in range(4):
        opt.step()
    saved = copy.deepcopy(opt.state_dict())
    qs, cap = build(capturable=True)
    with torch.no_grad():
        for p, q in zip(ps, qs):
            q.copy_(p)
    cap.load_state_dict(saved)
    assert sorted(cap.state_dict()['state']) == [0, 1]
    for q in qs:
        q.grad = torch.ones_like(q)
    with pytest.raises(RuntimeError, match='count'):
        cap.step()
    assert torch.equal(qs[0], ps[0])
    qs[2].grad = None
    opt.step()
    cap.step()
    assert torch.equal(qs[0], ps[0]) and torch.equal(qs[1], ps[1])
    assert {i: int(s['step']) for i, s in cap.state_dict()['state'].items()} == {0: 5, 1: 5}
    # a part of what was loaded goes on: the rest keeps its moments and its count
    rs, part = build(capturable=True)
    part.load_state_dict(saved)
    rs[0].grad = torch.ones_like(rs[0])
    part.step()
    s = part.state_dict()['state']
    assert {i: int(x['step']) for i, x in s.items()} == {0: 5, 1: 4} and torch.equal(s[1]['exp_avg'], saved['state'][1]['exp_avg'])


def test_replays_after_loading_are_counted(T):
    p, opt = _one(T, capturable=True)
    p.grad = torch.ones_like(p)
    opt.step()
    saved = copy.deepcopy(opt.state_dict())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(2):
        opt.load_state_dict(saved)
        assert int(opt.state_dict()['state'][0]['step']) == 1
        graph.replay()
        graph.replay()
        assert int(opt.state_dict()['state'][0]['step']) == 3


# ---- 8-bit moments at the ends of the range ------------------------------------------------------------------------------
@pytest.mark.parametrize('lr,eps', [(1e-18, 1e-8), (1e-19, 1e-8), (1e-22, 1e-8), (1e-27, 1e-8), (1e-36, 1e-8), (1e-2, 1e12), (1e30, 1e35), (1e30, 1e38)])
def test_rates_and_eps_at_the_ends_bit_for_bit(T, lr, eps):
    """Weights of zero show every bit of the update, also where the rate, scaled inside the kernel, would leave the normal range."""
    hp = dict(HP, lr=lr, eps=eps, weight_decay=0.0)
    rng = np.random.default_rng(4)
    p = nn.Parameter(torch.zeros(2000, device='cuda'))
    opt = T.AdamW([p], state_bits=8, **hp)
    ref = R.Tensors([np.zeros(2000, np.float32)], hp, 8)
    for step in range(3):
        g = rng.standard_normal(2000).astype(np.float32)
        p.grad = f32(g)
        opt.step()
        ref.step([g])
        same(p, ref.p[0], 'p, step %d' % step)


def test_largest_magnitude_of_a_block(T):
    """Up to 1.875 * 2^127 a value has its place; a block with a larger one becomes NaN like one with an infinity."""
    big = np.float32(1.875 * 2.0 ** 127)
    m = np.zeros(768, np.float32)
    m[3], m[300], m[600] = big, np.nextafter(big, np.float32(np.inf)), -big
    v = np.zeros(768, np.float32)
    v[5], v[301], v[700] = np.nextafter(big, np.float32(np.inf)), 1.0, big
    p = nn.Parameter(torch.zeros(768, device='cuda'))
    opt = T.AdamW([p], state_bits=8, **HP)
    opt.load_state_dict({'state': {0: {'step': 1, 'exp_avg': f32(m), 'exp_avg_sq': f32(v)}}, 'param_groups': opt.state_dict()['param_groups']})
    m[256:512] = np.nan
    v[:256] = np.nan
    a, b = opt.moments()
    same(a, m, 'm')
    same(b, v, 'v')


def test_checkpoints_beside_a_resized_parameter(T):
    """Refused by the step, a parameter of another size does not shift what is saved and loaded for the others."""
    p, q = nn.Parameter(torch.ones(5, 4, device='cuda')), nn.Parameter(torch.ones(300, device='cuda'))
    opt = T.AdamW([p, q], ema_decay=0.9)
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    opt.step()
    want = copy.deepcopy(opt.state_dict())
    p.data, p.grad = torch.ones(9, 7, device='cuda'), None
    with pytest.raises(RuntimeError, match='rebuild'):
        opt.step()
    for _ in range(2):
        got = opt.state_dict()
        for i in range(2):
            assert all(torch.equal(got['state'][i][k], want['state'][i][k]) for k in ('exp_avg', 'exp_avg_sq', 'ema'))
        opt.load_state_dict(want)
