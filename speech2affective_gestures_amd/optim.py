"""Flat parameter arenas and the fused Adam step.

MI355X-first memory layout: every trainable tensor of a network is a view into ONE contiguous fp32
arena, its gradient a view into a second one.  Consequences: ``zero_grad`` is one memset, Adam is one
kernel launch per optimizer (s2ag_adam_step), and the data-parallel gradient exchange is a single RCCL
all-reduce over the arena (parallel.py) instead of one collective per tensor.
"""
import array
import ctypes as C
import itertools
import math
import operator
from typing import Iterable, List, Optional, Sequence, Union

import torch

from . import _lib as L
from .text import _on, _stream


class ParamArena:
    def __init__(self, params: Iterable[torch.nn.Parameter], first: Iterable[torch.nn.Parameter] = ()):
        """``first``: parameters placed at the front of the arena (the rest keep their order) -- the data-parallel
        exchange wants the row-sparse word embedding in front of the dense buckets (parallel.GradExchange)."""
        seen, uniq = set(), []
        params = list(params)
        front = [p for p in first if any(p is q for q in params)]
        for p in front + params:
            if id(p) not in seen and p.requires_grad:
                seen.add(id(p))
                uniq.append(p)
        if not uniq:
            raise ValueError('no trainable parameters')
        dev = uniq[0].device
        L.require_gpu_device(dev, 'ParamArena (its parameters)')
        self.params: List[torch.nn.Parameter] = uniq
        self.epoch = 0          # bumped whenever the arena's values change behind torch's back (FusedAdam.step)
        sizes = [(p.numel() + 3) // 4 * 4 for p in uniq]          # keep every view 16-byte aligned
        self.numel = sum(sizes)
        self.data = torch.zeros(self.numel, dtype=torch.float32, device=dev)
        self.grad = torch.zeros(self.numel, dtype=torch.float32, device=dev)
        off = 0
        self.offsets = []
        for p, n in zip(uniq, sizes):
            view = self.data[off:off + p.numel()].view(p.shape)
            view.copy_(p.data)
            p.data = view
            p.grad = self.grad[off:off + p.numel()].view(p.shape)
            p._s2ag_arena = self
            self.offsets.append(off)
            off += n

    def offset_of(self, p: torch.nn.Parameter) -> int:
        """Element offset of ``p``'s view inside ``data`` / ``grad``."""
        for q, off in zip(self.params, self.offsets):
            if q is p:
                return off
        raise KeyError('parameter is not in this arena')

    def zero_grad(self):
        self.grad.zero_()
        for p, off in zip(self.params, self.offsets):      # re-attach if autograd replaced a grad tensor
            if p.grad is None or p.grad.data_ptr() != self.grad.data_ptr() + 4 * off:
                p.grad = self.grad[off:off + p.numel()].view(p.shape)


class FusedAdam:
    """torch.optim.Adam(lr, betas, eps=1e-8) semantics (processor_v2.py:215-220) as one launch."""

    def __init__(self, arena: ParamArena, lr: float, betas=(0.5, 0.999), eps: float = 1e-8):
        self.arena = arena
        self.lr, self.betas, self.eps = float(lr), (float(betas[0]), float(betas[1])), float(eps)
        self.exp_avg = torch.zeros_like(arena.data)
        self.exp_avg_sq = torch.zeros_like(arena.data)
        self.step_count = torch.zeros(1, dtype=torch.int32, device=arena.data.device)
        self.param_groups = [dict(lr=self.lr, betas=self.betas, eps=self.eps, params=arena.params)]

    def zero_grad(self, set_to_none: bool = False):
        self.arena.zero_grad()

    def step(self, grad_scale: float = 1.0):
        lib = L.load()
        s = C.c_void_p(torch.cuda.current_stream().cuda_stream)
        lr = float(self.param_groups[0]['lr'])
        L.check(lib.s2ag_counter_inc(C.c_void_p(self.step_count.data_ptr()), None, s), 'counter_inc')
        a = self.arena
        L.check(lib.s2ag_adam_step(C.c_void_p(a.data.data_ptr()), C.c_void_p(a.grad.data_ptr()),
                                   C.c_void_p(self.exp_avg.data_ptr()), C.c_void_p(self.exp_avg_sq.data_ptr()),
                                   a.numel, lr, self.betas[0], self.betas[1], self.eps,
                                   C.c_void_p(self.step_count.data_ptr()), float(grad_scale), s), 'adam_step')
        a.epoch += 1            # tensors derived from these parameters (ops._DerivedGroup) are stale now

    def clip_grad_norm(self, max_norm: float, norm_type: float = 2.0) -> torch.Tensor:
        """Clips the arena's gradients in place (``clip_grads``); call it between the backward pass and ``step``.  The norm is that of
        the gradients as they stand: before ``step``'s grad_scale, which has to be allowed for in max_norm."""
        return clip_grads([self.arena.grad], max_norm, norm_type)

    def state_dict(self):
        return dict(exp_avg=self.exp_avg, exp_avg_sq=self.exp_avg_sq, step=self.step_count, lr=self.param_groups[0]['lr'])

    def load_state_dict(self, sd):
        self.exp_avg.copy_(sd['exp_avg'])
        self.exp_avg_sq.copy_(sd['exp_avg_sq'])
        self.step_count.copy_(sd['step'])
        self.param_groups[0]['lr'] = sd['lr']


_CLIP_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_CLIP_BYTES = (4, 2)
_DEVICE, _DTYPE = operator.attrgetter('device'), operator.attrgetter('dtype')


def _dense(t: torch.Tensor) -> bool:
    """Whether the elements fill one piece of memory, in whatever order of the dimensions."""
    if t.is_contiguous():
        return True
    need = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz > 1):
        if stride != need:
            return False
        need *= size
    return True


def clip_grads(grads: Sequence[torch.Tensor], max_norm: float, norm_type: float = 2.0,
               out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Scales gradients by ``min(1, max_norm / (norm + 1e-6))`` and returns their global norm, a 0-dim fp32 tensor on the device.

    norm: the root of the sum of all squares (``norm_type`` 2, summed in 64 bits) or the largest magnitude (``math.inf``).  grads:
    fp32 or bf16 tensors of one device, in any mix, each dense in memory (any order of dimensions); a tensor that is listed twice
    counts once, two that share a part of their memory are refused.  out: where the results go, shaped and strided like grads, fp32
    or bf16; None: in place (nothing is written where the factor is 1).  A norm that is not finite follows the formula: NaN
    gradients for a NaN norm, zeros for an infinite one (and NaN for the infinities themselves).  Two launches per 128 tensors, no
    synchronisation; can be captured into a graph."""
    grads = list(grads)
    inf = norm_type == math.inf
    if not inf and norm_type != 2.0:
        raise ValueError(f'clip_grads: norm_type must be 2 or inf, got {norm_type}')
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f'clip_grads: max_norm must not be negative, got {max_norm}')
    if not grads:
        raise ValueError('clip_grads: no gradients')
    results = grads
    if out is not None:
        results = list(out)
        if len(results) != len(grads):
            raise ValueError(f'clip_grads: {len(grads)} gradients and {len(results)} outputs')
    # (whole lists at a time: a call is as long as its Python code for tensors that the kernels take some us for)
    tensors = grads if out is None else grads + results
    dev = grads[0].device
    if not grads[0].is_cuda:
        raise RuntimeError('clip_grads: got a CPU tensor; the S2AG ops run on MI355X only and there is no CPU fallback')
    if len(set(map(torch.Tensor.get_device, tensors))) > 1:
        raise ValueError(f'clip_grads: tensors on {sorted(set(map(str, map(_DEVICE, tensors))))}')
    kinds = list(map(_CLIP_DTYPES.get, map(_DTYPE, tensors)))
    if None in kinds:
        raise TypeError(f'clip_grads: tensors must be float32 or bfloat16, got {tensors[kinds.index(None)].dtype}')
    contiguous = all(map(torch.Tensor.is_contiguous, tensors))
    if not contiguous:
        for t in tensors:
            if not _dense(t):
                raise ValueError(f'clip_grads: a tensor of shape {tuple(t.shape)} and strides {tuple(t.stride())} is not dense in memory')
    if out is not None:
        for g, o in zip(grads, results):
            if o.shape != g.shape or not contiguous and o.stride() != g.stride() and not (o.is_contiguous() and g.is_contiguous()):
                raise ValueError(f'clip_grads: output {tuple(o.shape)} / {tuple(o.stride())} for a gradient {tuple(g.shape)} / {tuple(g.stride())}')
    # rows of s2ag_clip_tensor: src, dst, elements, (src is bf16) + 2^32 (dst is bf16); one that is listed again has the same row
    src, counts = list(map(torch.Tensor.data_ptr, grads)), list(map(torch.Tensor.numel, grads))
    dst = src if out is None else list(map(torch.Tensor.data_ptr, results))
    rows = [r for r in dict.fromkeys(zip(src, dst, counts, (a + (b << 32) for a, b in zip(kinds, kinds[-len(grads):])))) if r[2]]
    spans = [(r[0], r[0] + r[2] * _CLIP_BYTES[r[3] & 1]) for r in rows]
    if out is not None:
        spans += [(r[1], r[1] + r[2] * _CLIP_BYTES[r[3] >> 32]) for r in rows if r[0] != r[1] or (r[3] & 1) != r[3] >> 32]
    spans.sort()
    if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
        raise ValueError('clip_grads: two of the tensors share memory, or one that is listed twice has two outputs')
    k = len(rows)
    words = array.array('q', itertools.chain.from_iterable(rows))
    table = (L.ClipTensor * k).from_buffer(words) if k else (L.ClipTensor * 1)()
    lib = L.load()
    with _on(grads[0]):
        partials = torch.empty(lib.s2ag_clip_partials(table, k), dtype=torch.float64, device=dev)
        norm = torch.empty((), dtype=torch.float32, device=dev)
        L.check(lib.s2ag_clip_grads(table, k, max_norm, inf, partials.data_ptr(), norm.data_ptr(), _stream(norm)), 'clip_grads')
    torch.autograd.graph.increment_version(results)                # written behind torch's back
    return norm


def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0) -> torch.Tensor:
    """``clip_grads`` in place over the ``.grad`` of the parameters that have one (torch.nn.utils.clip_grad_norm_'s call);
    ValueError where none has one."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    return clip_grads([p.grad for p in parameters if p.grad is not None], max_norm, norm_type)
