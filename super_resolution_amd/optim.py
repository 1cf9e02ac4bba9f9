"""AdamW over many tensors, with moments in 32 or in 8 bits, and clipping by the global gradient norm, on libsr_amd.

Reference: `torch.optim.Adam(...)` / `optimizer.step()` of train/train_realESRGAN_fdconv_1.py:104,118, `clip_grad_norm_(..., 1.0)` of
train/train_realESRGAN_fdconv.py:142, and the weight average that Real-ESRGAN checkpoints carry as `params_ema`
(Real-ESRGAN-master/realesrgan/utils.py:59-63).

`train.FlatAdam` re-points the parameters into one buffer and runs torch operators on it; `AdamW` leaves them where they are:
one kernel (csrc/adamw.hip) walks all tensors of a group, reads gradients, parameters and moments once and writes them once.
"""
import contextlib
import copy
import ctypes as C
import os
import threading

import numpy as np
import torch

from . import _lib as L

_HOST_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), 'libsr_amd_torch.so')
_host = None
_BY_VALUE = 3840   # bytes of a table that go to the device as kernel arguments, in one launch; longer ones are read from pinned memory


def _host_lib():
    """libsr_amd_torch.so (csrc/torch_host.cpp): reads torch's tensor objects, with the GIL held."""
    global _host
    if _host is None:
        if not os.path.exists(_HOST_PATH):
            raise RuntimeError('%s is missing: build it with `python -m super_resolution_amd.build`; there is no fallback path' % _HOST_PATH)
        h = C.PyDLL(_HOST_PATH)
        h.srt_message.restype, h.srt_message.argtypes = C.c_char_p, []
        h.srt_track.restype, h.srt_track.argtypes = C.c_void_p, [C.py_object]
        h.srt_untrack.restype, h.srt_untrack.argtypes = None, [C.c_void_p]
        h.srt_gradients.restype, h.srt_gradients.argtypes = C.c_int64, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p]
        h.srt_spans.restype, h.srt_spans.argtypes = C.c_int64, [C.py_object, C.c_int, C.c_void_p, C.c_void_p]
        h.srt_not_written.restype, h.srt_not_written.argtypes = C.c_int64, [C.c_void_p]
        h.srt_spans_not_written.restype, h.srt_spans_not_written.argtypes = C.c_int64, [C.py_object, C.c_int]
        h.srt_take_spans.restype, h.srt_take_spans.argtypes = None, [C.c_void_p]
        _host = h
    return _host


def _host_failed(what):
    raise RuntimeError('%s: %s' % (what, _host_lib().srt_message().decode()))


def _on(dev):
    """torch.cuda.device(dev), which takes 2 us, where another device is current."""
    return contextlib.nullcontext() if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def _stream(dev):
    """The current stream of `dev` as the C ABI takes it (L.stream_ptr without the Python stream object: 2 us less a step)."""
    return torch._C._cuda_getCurrentRawStream(dev.index)


class _Pinned:
    """A block of pinned memory: words that the GPU writes when it has read the rest, and the table behind them."""

    free = []                   # blocks that were handed to a kernel; ready() tells whether it has read them
    lock = threading.Lock()

    def __init__(self, nbytes):
        self.size = 1 << max(13, (nbytes - 1).bit_length())
        self.memory = torch.zeros(8 * L.UPLOAD_WORDS + self.size, dtype=torch.uint8, pin_memory=True)
        self.done = self.memory.data_ptr()
        self.table = self.done + 8 * L.UPLOAD_WORDS
        self.ticket, self.expected = 0, bytes(8 * L.UPLOAD_WORDS)

    def next_ticket(self):
        self.ticket += 1
        self.expected = self.ticket.to_bytes(8, 'little') * L.UPLOAD_WORDS
        return self.ticket

    def ready(self):
        return C.string_at(self.done, 8 * L.UPLOAD_WORDS) == self.expected

    @classmethod
    def take(cls, nbytes):
        with cls.lock:
            for i, b in enumerate(cls.free):
                if b.size >= nbytes and b.ready():
                    return cls.free.pop(i)
        return cls(nbytes)


class _Stage:
    """Host memory at `at` for a table of nbytes, and its way to the device.  Under capture it travels by value: what a captured kernel
    or copy reads from the host is read again at every replay."""

    def __init__(self, nbytes):
        self.nbytes = nbytes
        self.by_value = nbytes <= _BY_VALUE or torch.cuda.is_current_stream_capturing()
        if self.by_value:
            self.host = (C.c_char * max(nbytes, 1))()
            self.at = C.addressof(self.host)
        else:
            self.host = _Pinned.take(nbytes)
            self.at = self.host.table

    def upload(self, dev, st):
        table = torch.empty(max(self.nbytes, 1), dtype=torch.uint8, device=dev)
        if self.by_value:
            L.check(L.lib().sr_upload(self.at, table.data_ptr(), self.nbytes, st), 'sr_upload')
        else:
            block = self.host
            L.check(L.lib().sr_upload_pinned(self.at, table.data_ptr(), self.nbytes, block.done, block.next_ticket(), st), 'sr_upload_pinned')
            with _Pinned.lock:
                _Pinned.free.append(block)
        return table


def _exchange_gradients(params, group, average):
    """Gradients summed (or averaged) over the ranks; `group`: the ProcessGroup."""
    import torch.distributed as dist
    from .train import allreduce_gradients
    grads = [p for p in params if p.requires_grad]
    if not (grads and grads[0].is_cuda and dist.get_backend(group) == 'gloo'):
        allreduce_gradients(grads, group=group, average=average)
        return
    # gloo reduces host memory (its device path stalls when ranks share one GPU)
    for dt in sorted({p.dtype for p in grads}, key=str):
        part = [p for p in grads if p.dtype == dt]
        host = torch.cat([(p.grad if p.grad is not None else torch.zeros_like(p)).reshape(-1) for p in part]).cpu()
        dist.all_reduce(host, op=dist.ReduceOp.SUM, group=group)
        if average:
            host /= dist.get_world_size(group)
        flat = host.to(part[0].device)
        for p, g in zip(part, flat.split([p.numel() for p in part])):
            p.grad = g.view(p.shape).clone() if p.grad is None else p.grad.copy_(g.view(p.shape))


def _broadcast_parameters(params, group):
    """Rank 0's values everywhere, one collective per dtype."""
    import torch.distributed as dist
    src = dist.get_global_rank(group, 0) if group is not None else 0
    for dt in sorted({p.dtype for p in params}, key=str):
        part = [p for p in params if p.dtype == dt]
        flat = torch.cat([p.reshape(-1) for p in part])
        if flat.is_cuda and dist.get_backend(group) == 'gloo':
            host = flat.cpu()
            dist.broadcast(host, src=src, group=group)
            flat.copy_(host)
        else:
            dist.broadcast(flat, src=src, group=group)
        for p, x in zip(part, flat.split([p.numel() for p in part])):
            p.copy_(x.view(p.shape))


def _world(group):
    import torch.distributed as dist
    return dist.get_world_size(group) if dist.is_available() and dist.is_initialized() else 1


# ------------------------------------------------------------------------------------------------------------------
# clipping
# ------------------------------------------------------------------------------------------------------------------
def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """torch.nn.utils.clip_grad_norm_ for the 2-norm (any other norm_type raises): scales the gradients in place by
    min(1, max_norm / (norm + 1e-6)) and returns the norm, a 0-d float32 tensor.  Squares are summed in float64, in an order that
    the shapes alone determine; nothing waits for the GPU unless error_if_nonfinite is set.  float32 and bfloat16 gradients, mixed,
    on one GPU."""
    params = [parameters] if torch.is_tensor(parameters) else list(parameters)
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError('clip_grad_norm_: max_norm must not be negative (got %r)' % max_norm)
    if isinstance(norm_type, bool) or float(norm_type) != 2:
        raise ValueError('clip_grad_norm_: norm_type is 2 (got %r)' % (norm_type,))
    host, lib = _host_lib(), L.lib()
    device, counts = C.c_int(-1), (C.c_int64 * 3)()
    rc = host.srt_spans(params, 1, C.byref(device), counts)
    odd, walked = [], (params, 1)
    if rc <= -2:   # gradients with holes: the norm reads dense copies, torch scales the originals
        grads = [(i, p.grad) for i, p in enumerate(params) if p.grad is not None]
        for i, g in grads:
            if g.layout != torch.strided or g.dtype not in (torch.float32, torch.bfloat16) or not g.is_cuda or g.device != grads[0][1].device:
                raise _unfit(i)
        _check_separate(grads)
        odd = [g for _, g in grads if not _is_dense(g)]
        dense = [g if _is_dense(g) else g.detach().contiguous() for _, g in grads]      # (alive until the norm is launched)
        device, walked = C.c_int(-1), (dense, 0)
        rc = host.srt_spans(*walked, C.byref(device), counts)
    if rc == -1:
        _host_failed('clip_grad_norm_')
    if rc > 0:
        raise _unfit(rc - 1)
    if not counts[2]:
        return torch.tensor(0.0)
    dev = torch.device('cuda', device.value)
    with _on(dev):
        st = _stream(dev)
        try:
            n32, n16 = counts[0], counts[1]
            stage = _Stage(16 * (n32 + n16))
            host.srt_take_spans(stage.at)
            on_host = int(n32 + n16 <= L.GRAD_SPANS_BY_VALUE)
            spans = stage.at if on_host else stage.upload(dev, st)
            first = spans if on_host else spans.data_ptr()
            lists = (L.GradList * (1 + (n16 > 0 and n32 > 0)))()
            for l, (at, n, code) in zip(lists, [x for x in ((first, n32, L.SR_F32), (first + 16 * n32, n16, L.SR_BF16)) if x[1]]):
                l.spans, l.nspans, l.dtype, l.on_host = at, n, code, on_host
            buf, norm = _norm(lists, max_norm, dev, st)
            if error_if_nonfinite and not bool(torch.isfinite(norm)):
                raise RuntimeError('clip_grad_norm_: the norm of the gradients is not finite')
        except BaseException:    # nothing was written
            host.srt_spans_not_written(*walked)
            raise
        for l in lists:
            if l.nspans:
                L.check(lib.sr_grad_scale(l.dtype, l.nspans, l.spans, l.on_host, buf.data_ptr() + 4 * buf.numel() - 4, st), 'sr_grad_scale')
        with torch.no_grad() if odd else contextlib.nullcontext():
            for g in odd:
                g.mul_(buf[-1])
    return norm


def _is_dense(t):
    """Whether the tensor's elements fill one run of memory, each once."""
    if t.is_contiguous():
        return True
    n = 1
    for size, stride in sorted(((s, st) for s, st in zip(t.shape, t.stride()) if s != 1), key=lambda x: x[1]):
        if stride != n:
            return False
        n *= size
    return True


def _unfit(i):
    return TypeError('clip_grad_norm_: gradients are float32 or bfloat16 on one GPU; tensor %d is not' % i)


def _extent(t):
    """The bytes between which the tensor lies: (first, behind the last)."""
    return t.data_ptr(), t.data_ptr() + ((sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size() if t.numel() else 0)


def _claimed_twice(tensors):
    """Whether tensors with overlapping extents, of any strides, have an element's memory in common, or one of them has it twice: every
    pair of bytes is marked."""
    first = min(_extent(t)[0] for t in tensors)
    mark, claims = np.zeros((max(_extent(t)[1] for t in tensors) - first) // 2, dtype=bool), 0
    for t in tensors:
        k = t.element_size() // 2
        at = (t.data_ptr() - first) // 2
        np.lib.stride_tricks.as_strided(mark[at:], tuple(t.shape) + (k,), tuple(s * k for s in t.stride()) + (1,))[...] = True
        claims += t.numel() * k
    return int(np.count_nonzero(mark)) != claims


def _check_separate(grads):
    """Refuses gradients (numbered; not all dense) that scaling in place would scale twice."""
    grads = [(i, g) for i, g in grads if g.numel()]
    for i, g in grads:
        reach = 0     # elements that the smaller strides reach: beyond them nothing repeats
        for s, n in sorted((s, n) for n, s in zip(g.shape, g.stride()) if n != 1):
            if s <= reach and _claimed_twice([g]):
                raise RuntimeError('clip_grad_norm_: the gradient of tensor %d repeats its elements: it cannot be scaled in place' % i)
            reach += (n - 1) * s
    cluster, end = [], 0
    for (lo, hi), g in sorted(((_extent(g), g) for _, g in grads), key=lambda x: x[0]) + [((float('inf'), 0), None)]:
        if lo >= end:
            if len(cluster) > 1 and _claimed_twice(cluster):
                raise RuntimeError('clip_grad_norm_: two gradients share memory')
            cluster, end = [], 0
        cluster.append(g)
        end = max(end, hi)


def _norm(lists, max_norm, dev, st):
    """(a float32 buffer on the device whose last two elements are norm and factor, the norm)."""
    lib, n = L.lib(), len(lists)
    nbytes = lib.sr_grad_norm_workspace_bytes(n)
    buf = torch.empty(nbytes // 4 + 2, dtype=torch.float32, device=dev)
    ws = buf.data_ptr()
    L.check(lib.sr_grad_norm(n, lists, max_norm, ws + nbytes, ws, nbytes, st), 'sr_grad_norm')
    return buf, buf[-2]


# ------------------------------------------------------------------------------------------------------------------
# AdamW
# ------------------------------------------------------------------------------------------------------------------
class _List:
    """The tensors of one parameter group with one dtype: the device tables, and the walk over their gradients."""

    buried = []   # handles dropped while a stream was capturing, where freeing is not allowed

    def __init__(self, opt, group, bits, members):
        self.group, self.bits, self.members = group, bits, members   # indices into opt.param_groups and opt.params
        self.params = [opt.params[i] for i in members]
        self.n = len(members)
        self.sizes = [p.numel() for p in self.params]
        self.dtype = self.params[0].dtype
        self.handle, self.tracked, self.retired = None, None, []
        self.steps = 0              # int: all tensors alike; else an int64 array
        # by-value tables are read by the launch itself: one buffer serves every step
        self.ptrs, self.stage = None, _Stage(8 * self.n) if self.n <= L.ADAMW_BY_VALUE else None
        self.odd = (C.c_int64 * self.n)()
        self.nodd, self.moved = C.c_int64(), C.c_int64()
        self.step_dev = self.scalars = None
        self.loaded = np.zeros(self.n, dtype=np.int64)      # capturable: step counts that a checkpoint brought, and the tensors that
        self.seen = self.captured = None                    # count on the device since then (of the last step, of the last captured one)
        self.rates = []             # learning rates on the device that captured steps read
        if opt.capturable:          # fixed memory: captured graphs point to it
            self.step_dev = torch.zeros((), dtype=torch.int64, device=opt.device)
            self.scalars = torch.empty(L.ADAMW_SCALARS_BYTES, dtype=torch.uint8, device=opt.device)

    def build(self, opt):
        t = np.zeros(self.n, dtype=np.dtype([(name, np.int64) for name, _ in L.AdamWTensor._fields_]))
        index, at, block = (x[self.members] for x in (opt._index, opt._at, opt._block))
        t['p'], t['n'], t['index'] = [p.data_ptr() for p in self.params], self.sizes, index
        if self.bits == 32:
            t['m'], t['v'] = opt._m32.data_ptr() + 4 * at, opt._v32.data_ptr() + 4 * at
        else:
            t['m'], t['v'] = opt._m8.data_ptr() + at, opt._v8.data_ptr() + at
            t['me'], t['ve'] = opt._me.data_ptr() + block, opt._ve.data_ptr() + block
        if opt.ema is not None:
            t['ema'] = opt.ema.data_ptr() + 4 * index
        h = C.c_void_p()
        L.check(L.lib().sr_adamw_create(L.dtype_code(self.dtype), self.bits, self.n, t.ctypes.data_as(C.POINTER(L.AdamWTensor)), C.byref(h)),
                'sr_adamw_create')
        tracked = _host_lib().srt_track(self.params)
        if not tracked:
            L.lib().sr_adamw_destroy(h)
            _host_failed('AdamW')
        while self.buried and not torch.cuda.is_current_stream_capturing():
            L.lib().sr_adamw_destroy(self.buried.pop())
        old = (self.handle, self.tracked)
        self.handle, self.tracked = h, tracked
        if opt.capturable and old[0]:
            self.retired.append(old)   # a captured graph may still read the tables
        else:
            self._free(*old)

    @classmethod
    def _free(cls, handle, tracked):
        if handle:
            if torch.cuda.is_current_stream_capturing():
                cls.buried.append(handle)
            else:
                L.lib().sr_adamw_destroy(handle)
        if tracked:
            _host_lib().srt_untrack(tracked)

    def __del__(self):
        try:
            for pair in self.retired + [(self.handle, self.tracked)]:
                self._free(*pair)
        except Exception:   # interpreter shutdown
            pass

    def gradients(self, keep, walked):
        """Fills self.ptrs; returns the number of tensors without a gradient.  keep: copies that must live until the launch; walked: the
        lists whose parameters' version counters have moved."""
        if self.n > L.ADAMW_BY_VALUE or self.ptrs is None:
            if self.n > L.ADAMW_BY_VALUE:
                self.stage = _Stage(8 * self.n)
            self.ptrs = (C.c_uint64 * self.n).from_address(self.stage.at)
        missing = _host_lib().srt_gradients(self.tracked, self.ptrs, self.odd, C.byref(self.nodd), C.byref(self.moved))
        if missing < 0:
            _host_failed('AdamW')
        walked.append(self)
        for k in range(self.nodd.value):
            p = self.params[self.odd[k]]
            g = p.grad
            if g.layout != torch.strided or g.shape != p.shape or g.dtype != p.dtype or g.device != p.device:
                raise RuntimeError('AdamW: the gradient of parameter %d (%s %s on %s) does not fit it (%s %s on %s)'
                                   % (self.members[self.odd[k]], tuple(g.shape), g.dtype, g.device, tuple(p.shape), p.dtype, p.device))
            with torch.no_grad():
                g = torch.empty_like(p).copy_(g)
            keep.append(g)
            self.ptrs[self.odd[k]] = g.data_ptr()
        # kept for what looks at them after the table has gone: its memory is given back with the upload
        self.copy = np.frombuffer(self.ptrs, dtype=np.uint64).copy() if missing or not isinstance(self.steps, int) else None
        return missing

    def table(self, dev, st, ptrs=None):
        """What the kernels read the gradients' addresses from: (address, whether on the host, what keeps it)."""
        stage = self.stage
        if ptrs is not None:
            stage = _Stage(8 * self.n)
            C.memmove(stage.at, ptrs, 8 * self.n)
        if self.n <= L.ADAMW_BY_VALUE:
            return stage.at, 1, stage
        t = stage.upload(dev, st)
        return t.data_ptr(), 0, t


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW (decoupled weight decay, no amsgrad) as one hand-written kernel per parameter group, for groups of any
    number of tensors; moments in float32 or, with `state_bits=8` (per group), in 8 bits each.

        opt = AdamW(net.parameters(), lr=1e-4, state_bits=8, ema_decay=0.999)
        ...
        loss.backward()
        opt.step(clip_grad_norm=1.0)          # or train.train_step(net, opt, ...)

    Parameters: float32 or bfloat16, dense, on one GPU; they stay where they are.  Re-pointed ones (`.data =`) of the same dtype, device and
    shape are followed, element by element where the order in memory changes.  bfloat16 parameters are rounded
    stochastically (an update of 1e-4 of a weight is below half a bfloat16 step and would be lost).  8-bit moments: 256 values share an
    exponent byte, m and v have three mantissa bits each and are rounded stochastically (rounded to nearest, v would not move under
    beta2 = 0.999); 2.01 bytes of state a parameter instead of 8.  The random bits are a hash of (seed, step, element): two runs
    give the same bits, whatever the launch.

    ema_decay: keeps `opt.ema`, a float32 average of the weights (ema = d ema + (1 - d) p after every step, in the same
    kernel); `ema_parameters()` gives it tensor by tensor, for a `params_ema` checkpoint.
    clip_grad_norm in step(): the global norm of all gradients, its factor applied as the gradients are read (they are not
    written back); `opt.grad_norm` holds the norm afterwards, on the device.  Nothing in step() waits for the GPU.
    In a process group of more than one rank step() all-reduces the gradients first (train.allreduce_gradients: a missing one
    counts as zeros), and the constructor broadcasts rank 0's parameters (`broadcast=False`: not).

    Parameters without a gradient are skipped, with their own step count, as torch does; their average goes on.
    state_dict() / load_state_dict() use torch.optim.AdamW's layout (float32 `exp_avg`, `exp_avg_sq`, `step`; plus `ema`), so a
    checkpoint moves between the two and between 32 and 8 bits; values that 8 bits hold come back as they were.
    capturable=True: the step count (and an lr given as a float32 GPU tensor) live on the device, for steps inside a captured
    graph; every step then has to bring the same gradients.  Without it a step under capture raises.  After replays call
    `replayed()`: what keeps packed weights under the parameters' version counters cannot see them otherwise."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, ema_decay=None, seed=0, capturable=False,
                 broadcast=True, group=None):
        if ema_decay is not None and not 0.0 <= ema_decay <= 1.0:
            raise ValueError('AdamW: ema_decay must lie in [0, 1] (got %r)' % (ema_decay,))
        self._built = False
        self.capturable, self.ema_decay, self.seed = bool(capturable), ema_decay, int(seed) & (1 << 64) - 1
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits))
        self.params = [p for g in self.param_groups for p in g['params']]
        if not self.params:
            raise ValueError('AdamW: no parameters')
        self.device = dev = self.params[0].device
        for g in self.param_groups:
            self._hyper(g)
        for p in self.params:
            L.require_gpu(p, 'AdamW')
            if p.dtype not in (torch.float32, torch.bfloat16) or p.device != dev:
                raise TypeError('AdamW: float32 or bfloat16 parameters on one GPU')
            if not _is_dense(p):
                raise ValueError('AdamW: a parameter with holes or repeated elements')
        self._check_overlap()
        # the shapes, and strides where not contiguous, that moments and average are kept in
        self._shape, self._stride = [tuple(p.shape) for p in self.params], {}
        for i, p in enumerate(self.params):
            if not p.is_contiguous():
                self._stride[i] = p.stride()
        # places: element number among all parameters; offset among the tensors of the same kind of moments; first block
        size = np.array([p.numel() for p in self.params], dtype=np.int64)
        bits = np.repeat([g['state_bits'] for g in self.param_groups], [len(g['params']) for g in self.param_groups])
        in_8 = np.where(bits == 8, size, 0)
        in_32, in_blocks = size - in_8, -(-in_8 // L.ADAMW_BLOCK)
        before = lambda x: np.cumsum(x) - x     # noqa: E731
        self._index, self._block = before(size), before(in_blocks)
        self._at = np.where(bits == 8, before(in_8), before(in_32))
        n, blocks = {32: int(in_32.sum()), 8: int(in_8.sum())}, int(in_blocks.sum())
        self.numel, self._sizes = int(size.sum()), size.tolist()
        with torch.cuda.device(dev), torch.no_grad():
            if broadcast and _world(group) > 1:
                _broadcast_parameters(self.params, group)
            self._m32, self._v32 = (torch.zeros(n[32], dtype=torch.float32, device=dev) for _ in range(2))
            self._m8, self._v8 = (torch.zeros(n[8], dtype=torch.uint8, device=dev) for _ in range(2))
            self._me, self._ve = (torch.ones(blocks, dtype=torch.uint8, device=dev) for _ in range(2))
            self.ema = None
            if ema_decay is not None:
                self.ema = torch.empty(self.numel, dtype=torch.float32, device=dev)
                self._reset_ema()
            self._lists, first = [], 0
            for k, g in enumerate(self.param_groups):
                for dt in (torch.float32, torch.bfloat16):
                    members = [first + i for i, p in enumerate(g['params']) if p.dtype == dt]
                    if members:
                        self._lists.append(_List(self, k, g['state_bits'], members))
                first += len(g['params'])
            for lst in self._lists:
                lst.build(self)
        self.grad_norm = None   # of the last step with clip_grad_norm: a 0-d float32 tensor on the GPU
        self._built = True

    def add_param_group(self, param_group):
        if self._built:
            raise RuntimeError('AdamW: give all parameter groups to the constructor (the moments of all tensors are laid out there)')
        bits = param_group.get('state_bits', self.defaults['state_bits'])
        if bits not in (32, 8):
            raise ValueError('AdamW: state_bits is 32 or 8 (got %r)' % (bits,))
        super().add_param_group(param_group)
        ps = self.param_groups[-1]['params']
        if len({id(p) for p in ps}) != len(ps):
            raise ValueError('AdamW: a parameter appears twice')

    def __getstate__(self):   # copy and pickle
        raise TypeError('AdamW holds device tables and cannot be copied or pickled: keep its state_dict()')

    # ---- state ---------------------------------------------------------------------------------------------------------
    def _hyper(self, g):
        lr, (b1, b2) = g['lr'], g['betas']
        if torch.is_tensor(lr):
            if lr.numel() != 1:
                raise ValueError('AdamW: lr must have one element')
            if self.capturable and lr.is_cuda:
                if lr.dtype != torch.float32 or lr.device != self.device:
                    raise TypeError("AdamW: a learning rate on the GPU is float32, on the parameters' device")
                lr = 0.0   # the kernel reads it
            else:
                lr = float(lr)
        if not (lr >= 0 and 0 <= b1 < 1 and 0 <= b2 < 1 and g['eps'] >= 0 and g['weight_decay'] >= 0):
            raise ValueError('AdamW: lr %r, betas %r, eps %r, weight_decay %r out of range' % (g['lr'], g['betas'], g['eps'], g['weight_decay']))
        return L.AdamWHyper(lr, b1, b2, g['eps'], g['weight_decay'], self.ema_decay or 0.0, self.seed)

    def _reset_ema(self):
        if self.numel:
            self.ema.copy_(self._cat(self.params))

    @staticmethod
    def _cat(tensors):
        """Dense tensors' elements in memory order, one after the other."""
        with torch.no_grad():
            if len({t.dtype for t in tensors}) == 1 and all(t.is_contiguous() for t in tensors):
                return torch._utils._flatten_dense_tensors(tensors)    # one C++ call for thousands of tensors
            return torch.cat([t.as_strided((t.numel(),), (1,)).float() for t in tensors])

    def _shaped(self, flat):
        """The parameters' parts of a flat array, with the elements at the parameters' indices."""
        parts = flat.split(self._sizes)
        return [x.as_strided(shape, self._stride[i]) if i in self._stride else x.view(shape) for i, (x, shape) in enumerate(zip(parts, self._shape))]

    @property
    def exp_avg(self):
        """The first moments of all parameters as one flat float32 buffer, in the order of the parameters (32-bit moments)."""
        if self._m8.numel():
            raise RuntimeError('AdamW: with 8-bit moments use moments()')
        return self._m32

    @property
    def exp_avg_sq(self):
        if self._v8.numel():
            raise RuntimeError('AdamW: with 8-bit moments use moments()')
        return self._v32

    def moments(self, dtype=torch.float32):
        """(exp_avg, exp_avg_sq) of all parameters as new flat tensors, in the order of the parameters; 8-bit moments as the values
        that their codes stand for (bfloat16 holds those of m and v exactly, within its range)."""
        code = L.dtype_code(dtype)
        with _on(self.device):
            m, v = (torch.empty(self.numel, dtype=dtype, device=self.device) for _ in range(2))
            for lst in self._lists:
                if self.numel:
                    L.check(L.lib().sr_adamw_moments(lst.handle, code, m.data_ptr(), v.data_ptr(), _stream(self.device)), 'sr_adamw_moments')
        return m, v

    def ema_parameters(self):
        """The average of the weights, one float32 view of `ema` per parameter."""
        if self.ema is None:
            raise RuntimeError('AdamW: built without ema_decay')
        return self._shaped(self.ema)

    # ---- step ----------------------------------------------------------------------------------------------------------
    def step(self, closure=None, group=None, average=True, clip_grad_norm=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if _world(group) > 1:
            with torch.no_grad():
                _exchange_gradients(self.params, group, average)
        if clip_grad_norm is not None and not clip_grad_norm >= 0:
            raise ValueError('AdamW: clip_grad_norm must not be negative (got %r)' % (clip_grad_norm,))
        dev = self.device
        with _on(dev):
            st = _stream(dev)
            capturing = torch.cuda.is_current_stream_capturing()
            if capturing and not self.capturable:
                raise RuntimeError('AdamW: a step under graph capture needs capturable=True (the step count would stay what it is now)')
            keep, walked, hypers, missing, seen = [], [], [], [], []
            try:
                for lst in self._lists:   # everything that can fail comes before the first launch
                    hypers.append(self._hyper(self.param_groups[lst.group]))
                    missing.append(lst.gradients(keep, walked))
                    if lst.moved.value:
                        self._follow(lst, capturing)
                    if self.capturable and missing[-1] < lst.n:
                        seen.append((lst, self._same_gradients(lst)))
                many = clip_grad_norm is not None and len(self._lists) > L.GRAD_MAX_LISTS
                if many:
                    lists = self._spans(keep, dev, st)
                tables = [lst.table(dev, st) for lst in self._lists]
                factor = None
                if clip_grad_norm is not None:
                    if not many:
                        lists = (L.GradList * len(self._lists))()
                        for l, lst, table in zip(lists, self._lists, tables):
                            l.list, l.grads, l.on_host = lst.handle, table[0], table[1]
                    buf, self.grad_norm = _norm(lists, float(clip_grad_norm), dev, st)
                    factor = buf.data_ptr() + 4 * buf.numel() - 4
            except BaseException:    # nothing was written
                for lst in walked:
                    _host_lib().srt_not_written(lst.tracked)
                raise
            for lst, have in seen:
                lst.seen = have
                if capturing:
                    lst.captured = have
            for lst, h, miss, table in zip(self._lists, hypers, missing, tables):
                self._launch(lst, h, miss, table, factor, st)
        return loss

    def _spans(self, keep, dev, st):
        """The gradients of more lists than one norm takes, as one list of spans per dtype."""
        lists = (L.GradList * 2)()
        for l, dt in zip(lists, (torch.float32, torch.bfloat16)):
            l.dtype = L.dtype_code(dt)
            part = [lst for lst in self._lists if lst.dtype == dt]
            if not part:
                continue
            at, n = np.concatenate([np.frombuffer(lst.ptrs, dtype=np.uint64) for lst in part]), np.concatenate([lst.sizes for lst in part])
            at, n = at[(at != 0) & (n > 0)], n[(at != 0) & (n > 0)]
            longest = max(4096, -(-int(n.sum()) // 8192 // 1024) * 1024)     # as clip_grad_norm_ shares long tensors out
            pieces = -(-n // longest)
            first = (np.arange(int(pieces.sum())) - np.repeat(np.cumsum(pieces) - pieces, pieces)) * longest
            spans = np.stack([np.repeat(at.astype(np.int64), pieces) + first * dt.itemsize, np.minimum(np.repeat(n, pieces) - first, longest)], axis=1)
            if len(spans):
                stage = _Stage(spans.nbytes)
                C.memmove(stage.at, np.ascontiguousarray(spans).ctypes.data, spans.nbytes)
                table = stage.upload(dev, st)
                keep.append(table)
                l.spans, l.nspans = table.data_ptr(), len(spans)
        return lists

    def replayed(self):
        """To be called after a graph that holds a step was replayed, before the parameters are used outside it: a replay writes them
        without moving their version counters, by which autograd's saved-tensor checks and the networks' packed weights tell."""
        torch.autograd.graph.increment_version([p for p in self.params if not p.is_inference()])

    def _launch(self, lst, h, missing, table, factor, st):
        lib = L.lib()

        def run(step, scalars, table):
            L.check(lib.sr_adamw_step(lst.handle, C.byref(h), step, scalars, table[0], table[1], factor, st), 'sr_adamw_step')
        if missing == lst.n:
            if self.ema is not None:
                run(1, None, table)
            return
        if self.capturable:
            lr = self.param_groups[lst.group]['lr']
            if torch.is_tensor(lr) and lr.is_cuda and torch.cuda.is_current_stream_capturing() and not any(lr is x for x in lst.rates):
                lst.rates.append(lr)
            L.check(lib.sr_adamw_tick(C.byref(h), lr.data_ptr() if torch.is_tensor(lr) and lr.is_cuda else None, lst.step_dev.data_ptr(),
                                      lst.scalars.data_ptr(), st), 'sr_adamw_tick')
            run(0, lst.scalars.data_ptr(), table)
            return
        if not missing and isinstance(lst.steps, int):
            lst.steps += 1
            run(lst.steps, None, table)
            return
        # step counts differ: one launch per count, the other tensors marked; the first one also takes those without a gradient
        # (their averages)
        ptrs = lst.copy
        have = ptrs != 0
        steps = np.full(lst.n, lst.steps, dtype=np.int64) if isinstance(lst.steps, int) else lst.steps
        lst.steps = steps = steps + have
        rest = ~have
        for t in np.unique(steps[have]):
            now = have & (steps == t) | rest
            rest = np.zeros_like(rest)
            part = np.where(now, ptrs, np.uint64(L.ADAMW_SKIP))
            run(int(t), None, lst.table(self.device, st, part.ctypes.data))
        if (steps == steps[0]).all():
            lst.steps = int(steps[0])

    def _follow(self, lst, capturing):
        """Parameters lie elsewhere (`.data =`): same dtype, device and size are followed, anything else is refused."""
        turned = []
        for i, p in zip(lst.members, lst.params):
            if p.device != self.device or p.dtype != lst.dtype or p.shape != self._shape[i] or not _is_dense(p):
                raise RuntimeError('AdamW: a parameter was moved, cast or resized after the optimizer was built -- rebuild the optimizer')
            if (None if p.is_contiguous() else p.stride()) != self._stride.get(i):
                turned.append(i)
        if capturing:
            raise RuntimeError('AdamW: a parameter was re-pointed; run one step outside the capture first')
        self._check_overlap()
        for i in turned:
            self._reorder(i, lst.bits)
        lst.build(self)

    @torch.no_grad()
    def _reorder(self, i, bits):
        """The memory order of parameter i has changed (channels_last and back): its moments and its average follow, so that every
        element keeps its own.  Blocks of 8-bit moments then hold other elements, and these are rounded once more."""
        p, n = self.params[i], self.params[i].numel()
        shape, stride = self._shape[i], self._stride.get(i)
        index, at, block = int(self._index[i]), int(self._at[i]), int(self._block[i])

        def turn(x):
            old = x.clone()
            x.as_strided(p.shape, p.stride()).copy_(old.as_strided(shape, stride) if stride else old.view(shape))
        if bits == 32:
            turn(self._m32[at:at + n])
            turn(self._v32[at:at + n])
        else:
            t, h, lib, st = (L.AdamWTensor * 1)(), C.c_void_p(), L.lib(), _stream(self.device)
            t[0].p, t[0].n = p.data_ptr(), n
            t[0].m, t[0].v = self._m8.data_ptr() + at, self._v8.data_ptr() + at
            t[0].me, t[0].ve = self._me.data_ptr() + block, self._ve.data_ptr() + block
            L.check(lib.sr_adamw_create(L.dtype_code(p.dtype), 8, 1, t, C.byref(h)), 'sr_adamw_create')
            try:
                m, v = (torch.empty(n, dtype=torch.float32, device=self.device) for _ in range(2))
                L.check(lib.sr_adamw_moments(h, L.SR_F32, m.data_ptr(), v.data_ptr(), st), 'sr_adamw_moments')
                turn(m)
                turn(v)
                L.check(lib.sr_adamw_set_moments(h, m.data_ptr(), v.data_ptr(), self.seed, st), 'sr_adamw_set_moments')
            finally:
                lib.sr_adamw_destroy(h)
        if self.ema is not None:
            turn(self.ema[index:index + n])
        if p.is_contiguous():
            del self._stride[i]
        else:
            self._stride[i] = p.stride()

    def _check_overlap(self):
        spans = np.array([(p.data_ptr(), p.numel() * p.element_size()) for p in self.params if p.numel()], dtype=np.int64).reshape(-1, 2)
        spans = spans[np.argsort(spans[:, 0])]
        if (spans[1:, 0] < spans[:-1].sum(1)).any():
            raise ValueError('AdamW: two parameters share memory')

    def _same_gradients(self, lst):
        """One step count on the device serves all tensors of a list."""
        have = np.frombuffer(lst.ptrs, dtype=np.uint64) != 0
        if lst.seen is None:
            other = lst.loaded[have] != lst.loaded.max()
            if other.any():
                raise RuntimeError('AdamW(capturable=True): one step count serves all tensors, but of those with a gradient %d have not the %d steps of the '
                                   'checkpoint' % (other.sum(), lst.loaded.max()))
        elif not np.array_equal(lst.seen, have):
            raise RuntimeError('AdamW(capturable=True): a step must bring gradients for the same parameters as the one before')
        return have

    # ---- checkpoints ---------------------------------------------------------------------------------------------------
    # group keys that belong to this optimizer's layout, or to the implementation that wrote the dictionary
    _NOT_LOADED = ('params', 'state_bits', 'amsgrad', 'maximize', 'foreach', 'capturable', 'differentiable', 'fused', 'decoupled_weight_decay')

    def _steps_of(self, lst):
        if self.capturable:
            counting = lst.seen if lst.seen is not None else lst.captured
            if counting is None:
                return lst.loaded.tolist()
            return np.where(counting & (lst.loaded == lst.loaded.max()), int(lst.step_dev.item()), lst.loaded).tolist()
        return [lst.steps] * lst.n if isinstance(lst.steps, int) else lst.steps.tolist()

    def state_dict(self):
        """torch.optim.AdamW's layout: {'state': {i: {'step', 'exp_avg', 'exp_avg_sq'[, 'ema']}}, 'param_groups': [...]}; with an average
        also 'ema': {i: ...} for the parameters that took no step (they have no state there; their average moves all the same)."""
        steps = {}
        for lst in self._lists:
            steps.update(zip(lst.members, self._steps_of(lst)))
        state, resting = {}, {}
        if any(steps.values()):
            m, v = (self._shaped(x) for x in self.moments())
            for i in (i for i in range(len(self.params)) if steps[i]):
                state[i] = {'step': torch.tensor(float(steps[i])), 'exp_avg': m[i], 'exp_avg_sq': v[i]}
        if self.ema is not None:
            for i, x in enumerate(self._shaped(self.ema.clone())):
                if steps[i]:
                    state[i]['ema'] = x
                else:
                    resting[i] = x
        groups, first = [], 0
        for g in self.param_groups:
            hp = {k: x for k, x in g.items() if k != 'params'}
            hp['params'] = list(range(first, first + len(g['params'])))
            first += len(g['params'])
            groups.append(hp)
        return {'state': state, 'param_groups': groups, **({'ema': resting} if resting else {})}

    @torch.no_grad()
    def load_state_dict(self, sd):
        groups = sd['param_groups']
        if [len(g['params']) for g in groups] != [len(g['params']) for g in self.param_groups]:
            raise ValueError('AdamW.load_state_dict: expected groups of %s parameters' % [len(g['params']) for g in self.param_groups])
        for g in groups:
            if g.get('amsgrad') or g.get('maximize'):
                raise ValueError('AdamW.load_state_dict: amsgrad and maximize are not supported')
            if g.get('decoupled_weight_decay') is False and g.get('weight_decay'):
                raise ValueError('AdamW.load_state_dict: the weight decay of torch.optim.Adam (part of the gradient) is not supported')
        place = {}
        for i, key in enumerate(k for g in groups for k in g['params']):
            place[key] = i
        resting = sd.get('ema') or {}
        if any(k not in place for k in [*sd['state'], *resting]):
            raise ValueError('AdamW.load_state_dict: a state for a parameter that no group holds')
        state = {place[k]: {'ema': x} for k, x in resting.items()}
        for k, s in sd['state'].items():
            state[place[k]] = {**state.get(place[k], {}), **s}
        for i, s in state.items():
            for name in ('exp_avg', 'exp_avg_sq', 'ema'):
                if name in s and s[name].shape != self._shape[i]:
                    raise ValueError('AdamW.load_state_dict: parameter %d has shape %s, its %s %s' % (i, self._shape[i], name, tuple(s[name].shape)))
        # the rates, and what schedulers keep beside them
        new = [{**{k: mine[k] for k in ('lr', 'betas', 'eps', 'weight_decay')}, **{k: copy.deepcopy(x) for k, x in g.items() if k not in self._NOT_LOADED}}
               for g, mine in zip(groups, self.param_groups)]
        for hp in new:
            self._hyper(hp)
        steps = [np.array([int(float(state.get(i, {}).get('step', 0))) for i in lst.members], dtype=np.int64) for lst in self._lists]
        if self.capturable and any(set(t.tolist()) - {0, int(t.max())} for t in steps):
            raise ValueError('AdamW.load_state_dict: capturable=True takes one step count')
        rates = [(mine['lr'], float(hp['lr'])) for mine, hp in zip(self.param_groups, new)]
        for (lr, value), hp in zip(rates, new):
            if torch.is_tensor(lr) and lr.is_cuda and self.capturable:
                if all(other == value for x, other in rates if x is lr):
                    hp['lr'] = lr                      # captured steps read it where it is: the value goes there
                elif any(x is lr for lst in self._lists for x in lst.rates):
                    raise ValueError('AdamW.load_state_dict: groups with different rates, but a captured step reads one tensor for them')
                else:
                    hp['lr'] = torch.full_like(lr, value)
            elif torch.is_tensor(hp['lr']) and hp['lr'].is_cuda and not self.capturable:
                hp['lr'] = value                       # (every step would wait for it)
        for mine, hp, (lr, value) in zip(self.param_groups, new, rates):
            if hp['lr'] is lr and torch.is_tensor(lr):
                lr.fill_(value)
            mine.update(hp)

        def part(name, i):
            stride, x = self._stride.get(i), state.get(i, {}).get(name, self.params[i] if name == 'ema' else None)
            if x is None:
                return torch.zeros(self._sizes[i], dtype=torch.float32, device=self.device)
            if x.dtype != torch.float32 or x.device != self.device:
                x = x.to(self.device, torch.float32)
            if stride is None:
                return x.contiguous()
            return x if x.stride() == stride else torch.empty_strided(self._shape[i], stride, dtype=torch.float32, device=self.device).copy_(x)

        def flat(name):
            return self._cat([part(name, i) for i in range(len(self.params))])
        with _on(self.device):
            if self.numel:
                m, v = flat('exp_avg'), flat('exp_avg_sq')
                for lst in self._lists:
                    L.check(L.lib().sr_adamw_set_moments(lst.handle, m.data_ptr(), v.data_ptr(), self.seed, _stream(self.device)),
                            'sr_adamw_set_moments')
            for lst, t in zip(self._lists, steps):
                if self.capturable:
                    lst.step_dev.fill_(int(t.max()))
                    lst.loaded, lst.seen = t, None
                else:
                    lst.steps = int(t[0]) if (t == t[0]).all() else t
            if self.ema is not None and self.numel:
                self.ema.copy_(flat('ema'))
