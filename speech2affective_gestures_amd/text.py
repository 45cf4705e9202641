"""Operators of a text model's two ends: the word embedding with a gradient by sorted ids, and the softmax cross entropy of the
output layer over a large vocabulary without its logits (kernels: csrc/text/, C ABI: include/s2ag_text.h).

Public names: ``ops.embedding_sorted`` and ``ops.linear_cross_entropy``.  Both take fp32 or bf16, run on torch's current
stream of their tensors' device, can be captured into a graph (kernels only, memory from the caching allocator), and give the same
bits for the same inputs."""
from __future__ import annotations

import contextlib
import ctypes as C
from typing import Optional

import torch

from . import _lib as L

Tensor = torch.Tensor
_DTYPES = (torch.float32, torch.bfloat16)
_IDS = (torch.int64, torch.int32)
_REDUCTIONS = {'mean': 0, 'sum': 1, 'none': 2}
MAX_ROWS = MAX_WORDS = 1 << 21         # linear_cross_entropy: rows of x, rows of weight


def _p(t: Optional[Tensor]):
    return None if t is None else t.data_ptr()


_NOTHING = contextlib.nullcontext()


def _on(t: Tensor):
    """Context in which ``t``'s device is the current one (nothing to do where it is: the usual case)."""
    dev = t.device                                                 # (torch.cuda.current_device asks first whether torch is set up)
    return _NOTHING if dev.index == torch._C._cuda_getDevice() else torch.cuda.device(dev)


def _like(t: Tensor) -> Tensor:
    return torch.empty_like(t, memory_format=torch.contiguous_format)      # (half the time of torch.empty with a shape)


def _stream(t: Tensor) -> int:
    return torch._C._cuda_getCurrentRawStream(t.device.index)      # (torch.cuda.current_stream builds an object: some us a call)


def _once(backward):
    """once_differentiable, whose bookkeeping is only wanted where a second derivative might be."""
    full = torch.autograd.function.once_differentiable(backward)
    return lambda ctx, *grads: (full if torch.is_grad_enabled() else backward)(ctx, *grads)


def _check_tensors(what: str, **ts) -> None:
    dev = None
    for name, t in ts.items():
        if not isinstance(t, Tensor):
            raise TypeError(f'{what}: {name} must be a tensor, got {type(t).__name__}')
        if not t.is_cuda:
            raise RuntimeError(f'{what}: {name} is a CPU tensor; the S2AG ops run on MI355X only and there is no CPU fallback')
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f'{what}: tensors on {dev} and {t.device}')


def _check_ids(what: str, name: str, t: Tensor) -> None:
    if t.dtype not in _IDS:
        raise TypeError(f'{what}: {name} must be int64 or int32, got {t.dtype}')


def _check_matrix(what: str, name: str, t: Tensor) -> None:
    if t.dtype not in _DTYPES:
        raise TypeError(f'{what}: {name} must be float32 or bfloat16, got {t.dtype}')
    if t.dim() != 2 or t.shape[0] == 0 or t.shape[1] == 0:
        raise ValueError(f'{what}: {name} must be a matrix with rows and columns, got shape {tuple(t.shape)}')


def _rows(t: Tensor):
    """(tensor, row pitch): ``t`` as a matrix with unit column stride; a copy only if its rows do not lie at one pitch."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.is_contiguous():
        return t, t.shape[1]
    if t.numel() and (t.stride(1) != 1 and t.shape[1] > 1 or (t.shape[0] > 1 and t.stride(0) < t.shape[1])):
        t = t.contiguous()
    return t, (t.stride(0) if t.shape[0] > 1 else t.shape[1])


def _arena_slot(p: Tensor) -> Optional[Tensor]:
    """The gradient of a parameter that lives in an optim.ParamArena: the kernels add to it in place."""
    if getattr(p, '_s2ag_arena', None) is None:
        return None
    from .ops import _grad_slot
    slot = _grad_slot(p)
    if slot is not None:
        turn = p.__dict__.setdefault('_s2ag_turn', _Turn())
        if turn.handle != _stream(slot):
            turn.pass_on(torch.cuda.current_stream(slot.device))
    return slot


class _Turn:
    """The stream that added to a parameter's gradient last.  The kernels add without atomics: another stream's pass waits for what that
    one has been given.  (A captured pass does not wait for one outside, nor the other way round: a graph is ordered where it is replayed.)"""

    def __init__(self):
        self.handle, self.stream = -1, None

    def pass_on(self, cur) -> None:
        last = self.stream
        if last is not None and _capturing(last) == _capturing(cur):
            cur.wait_stream(last)
        self.handle, self.stream = cur.cuda_stream, cur

    def __reduce__(self):                                          # (a parameter that is saved or copied starts anew)
        return _Turn, ()


def _capturing(stream) -> bool:
    with torch.cuda.stream(stream):
        return torch.cuda.is_current_stream_capturing()


# ----------------------------------------------------------------------------------------------------
# embedding
# ----------------------------------------------------------------------------------------------------
class _EmbeddingSorted(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale, padding_idx, grads):
        lib = L.load()
        with _on(table):
            ids = ids.contiguous()
            data = table.contiguous()
            n, (entries, dim) = ids.numel(), data.shape
            i32, bf16 = ids.dtype == torch.int32, data.dtype == torch.bfloat16
            out = data.new_empty(ids.shape + (dim,))
            L.check(lib.s2ag_emb_lookup(ids.data_ptr(), i32, data.data_ptr(), bf16, n, dim, entries, scale, out.data_ptr(), _stream(out)),
                    'emb_lookup')
        if grads and ctx.needs_input_grad[1]:
            ctx.save_for_backward(ids)
            # (sizes, types and the workspace's size for the backward pass, so that it has less Python code to run: 91 to 87 us a step
            # of a small embedding)
            ctx.plan = (lib, table, i32, bf16, n, dim, entries, padding_idx, scale, lib.s2ag_emb_grad_workspace_bytes(n, dim, entries))
        return out

    @staticmethod
    @_once
    def backward(ctx, dy):
        (ids,) = ctx.saved_tensors
        lib, table, i32, bf16, n, dim, entries, padding_idx, scale, ws_bytes = ctx.plan
        with _on(dy):
            dy, ld = _rows(dy)
            slot = _arena_slot(table)
            dt = _like(table) if slot is None else slot
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dy.device)
            L.check(lib.s2ag_emb_grad(ids.data_ptr(), i32, dy.data_ptr(), ld, bf16, n, dim, entries, padding_idx, scale, dt.data_ptr(),
                                      slot is not None, ws.data_ptr(), ws_bytes, _stream(dy)), 'emb_grad')
        return None, (dt if slot is None else None), None, None, None


def embedding_sorted(ids: Tensor, table: Tensor, scale: float = 1.0, padding_idx: Optional[int] = None) -> Tensor:
    """``scale * table[ids]`` in the table's type, rounded once: (*ids.shape, dim).

    ids: int64 or int32, any shape; an id outside the table reads as a row of zeros and sends no gradient.  table: (n, dim) fp32 or
    bf16.  padding_idx: a row that is looked up like any other and gets no gradient.
    The table's gradient is summed per id in fp32, in an order that the ids alone decide, and rounded once.  Where the table is a parameter of
    an optim.ParamArena, the backward pass adds to its gradient there, in the rows that were looked up, and hands autograd None: on
    the stream of the lookup, which a reader on another stream waits for; passes of these operators on several streams take turns."""
    what = 'embedding_sorted'
    _check_tensors(what, ids=ids, table=table)
    _check_ids(what, 'ids', ids)
    _check_matrix(what, 'table', table)
    n, dim = table.shape
    if ids.numel() >= (1 << 31) - 65536 or n >= (1 << 30) or dim > (1 << 24):
        raise ValueError(f'{what}: {ids.numel()} ids in a table of shape {tuple(table.shape)} is more than the kernels index')
    pad = -1
    if padding_idx is not None:
        pad = int(padding_idx) + (n if padding_idx < 0 else 0)
        if not 0 <= pad < n:
            raise ValueError(f'{what}: padding_idx {padding_idx} is not a row of a table of {n}')
    return _EmbeddingSorted.apply(ids, table, float(scale), pad, torch.is_grad_enabled())


# ----------------------------------------------------------------------------------------------------
# linear + softmax cross entropy
# ----------------------------------------------------------------------------------------------------
def _lce_workspace(lib, a, backward: bool, device) -> Tensor:
    n = lib.s2ag_lce_workspace_bytes(a, backward)
    if n < 0:
        raise RuntimeError(f'linear_cross_entropy: sizes refused ({n})')
    ws = torch.empty(n, dtype=torch.uint8, device=device)
    a.workspace, a.workspace_bytes = ws.data_ptr(), n
    return ws


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, target, ignore_index, reduction, grads):
        lib, a = L.load(), L.LceArgs()
        with _on(x):
            xr, a.ldx = _rows(x)
            w, a.ldw = _rows(weight)
            t = target.contiguous()
            a.x, a.w, a.target = xr.data_ptr(), w.data_ptr(), t.data_ptr()
            a.target_i32, a.bf16 = t.dtype == torch.int32, x.dtype == torch.bfloat16
            (a.rows, a.dim), a.vocab = xr.shape, w.shape[0]
            # (grads: grad mode at the call; in here it is off, and needs_input_grad does not know of it)
            a.ignore_index, a.reduction, a.keep = ignore_index, reduction, grads and any(ctx.needs_input_grad)
            state = torch.empty(lib.s2ag_lce_state_bytes(a), dtype=torch.uint8, device=x.device)
            loss = torch.empty(target.shape if reduction == 2 else (), dtype=torch.float32, device=x.device)
            a.state = state.data_ptr()
            a.loss = loss.data_ptr() or a.state                   # (no rows, no reduction: nothing is written)
            ws = _lce_workspace(lib, a, False, x.device)
            L.check(lib.s2ag_lce_fwd(a, _stream(ws)), 'lce_fwd')
        if a.keep:
            ctx.save_for_backward(x, weight, t, state)
            ctx.plan = (lib, a, w, weight)       # (w: the rows that a.w points at, where weight's own do not lie at one pitch)
        return loss

    @staticmethod
    @_once
    def backward(ctx, dloss):
        x, weight, t, state = ctx.saved_tensors
        lib, a, w, leaf = ctx.plan
        need_x, need_w = ctx.needs_input_grad[:2]
        with _on(x):
            slot = _arena_slot(leaf) if need_w else None
            dx = _like(x) if need_x else None
            dw = slot
            if need_w and slot is None:
                dw = _like(weight)
            if a.rows == 0:
                if dw is not None and slot is None:
                    dw.zero_()
            else:
                g = dloss.contiguous()                           # (fp32, as the loss is)
                b = L.LceArgs.from_buffer_copy(a)                # (a graph that is kept runs backward again)
                # hooks on saved tensors and checkpoints hand back others than were saved, whose memory is gone
                b.x, b.target, b.state = x.data_ptr(), t.data_ptr(), state.data_ptr()
                b.grad_out, b.dx, b.dw, b.dw_accumulate = g.data_ptr(), _p(dx), _p(dw), slot is not None
                ws = _lce_workspace(lib, b, True, x.device)
                L.check(lib.s2ag_lce_bwd(b, _stream(ws)), 'lce_bwd')
        return dx, (dw if slot is None else None), None, None, None, None


def linear_cross_entropy(x: Tensor, weight: Tensor, target: Tensor, ignore_index: int = -100, reduction: str = 'mean') -> Tensor:
    """Softmax cross entropy of the logits ``x @ weight.T`` against ``target``, in fp32; the logits are never stored.

    x: (..., dim), weight: (vocab, dim), both fp32 or both bf16; target: (...) int64 or int32.  Rows whose target is
    ``ignore_index`` have a loss and a gradient of zero and are left out of every product.  reduction: 'mean' over the other rows
    (0 if there are none), 'sum', or 'none' (target's shape).  A target outside the vocabulary that is not ``ignore_index`` makes that
    row's loss NaN, and every gradient that it enters.  So does, in fp32, an infinity in a row of x or weight.
    Sums, statistics and losses are fp32.  Of bf16 operands the gradient of the logits, softmax minus one-hot, is rounded to bf16 for the
    products that make the gradients of x and weight (2^-8 of each value at most); of fp32 ones it keeps 24 bits.
    At most 2^21 rows and 2^21 words.  Where the weight is a parameter of an optim.ParamArena, the backward pass adds to its gradient
    there and hands autograd None: on the stream of the loss, which a reader on another stream waits for; passes of these operators on
    several streams take turns."""
    what = 'linear_cross_entropy'
    _check_tensors(what, x=x, weight=weight, target=target)
    _check_ids(what, 'target', target)
    _check_matrix(what, 'weight', weight)
    if reduction not in _REDUCTIONS:
        raise ValueError(f"{what}: reduction must be 'mean', 'sum' or 'none', got {reduction!r}")
    if x.dtype != weight.dtype:
        raise TypeError(f'{what}: x is {x.dtype} and weight {weight.dtype}')
    if x.dim() < 1 or x.shape[-1] != weight.shape[1] or x.shape[:-1] != target.shape:
        raise ValueError(f'{what}: x {tuple(x.shape)}, weight {tuple(weight.shape)} and target {tuple(target.shape)} do not go together')
    ignore_index = int(ignore_index)
    if not -(1 << 63) <= ignore_index < 1 << 63:
        raise ValueError(f'{what}: ignore_index {ignore_index} is no int64')
    if target.numel() > MAX_ROWS or weight.shape[0] > MAX_WORDS or weight.shape[1] > (1 << 20):
        raise ValueError(f'{what}: at most {MAX_ROWS} rows, {MAX_WORDS} words and {1 << 20} columns')
    return _LinearCrossEntropy.apply(x, weight, target, ignore_index, _REDUCTIONS[reduction], torch.is_grad_enabled())
