"""Rows of routed experts: sorted by expert and back, the experts' own linear layers, learned codes by id.

The routed models choose an expert for each row (`model.route`) and read that expert's table (`ExpertHashQuery`).
The operators here give experts layers of their own: `sort_rows` orders the (row, choice) pairs by expert,
`dispatch` copies each row to its places, `linear` multiplies every group of consecutive rows by its expert's
matrix with bias, activation and residual in the same kernel, `combine` brings the results back as weighted sums;
`embed` looks rows of a learned table up by id.  All of them run the kernels of libodie_b200.so on the current
stream of their tensors' device, are differentiable (once) and give the same bits in every run.  `ExpertHeads`
is the MLP of `model.Head` with one set of weights per expert, built from them.

There is no CPU path: tensors that are not on a CUDA device are refused.
"""
import math
from typing import NamedTuple

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib

__all__ = ['RowOrder', 'sort_rows', 'dispatch', 'combine', 'linear', 'embed', 'ExpertHeads']

ROW_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
ACTIVATIONS = {'none': 0, 'relu': 1, 'silu': 2, 'gelu': 3}


class RowOrder(NamedTuple):
    """The (row, choice) pairs in expert order (sort_rows).

    Pair i = row * choices + choice.  order int32 [pairs]: the pair at each place; slot int32 [rows, choices]: the
    place of each pair; offsets int32 [bins + 1]: the first place of each expert, the last one the count of pairs
    that have an expert.  Dropped pairs stand behind: their order is ~pair and their slot ~place."""
    order: torch.Tensor
    slot: torch.Tensor
    offsets: torch.Tensor

    @property
    def rows(self):
        return self.slot.shape[0]

    @property
    def choices(self):
        return self.slot.shape[1]


def _stream(index):
    return torch._C._cuda_getCurrentRawStream(index)


def _call(name, device, *arguments):
    """One library call on the device's current stream (the library launches on the current device)."""
    index = device.index
    if index == torch.cuda.current_device():
        status = getattr(_lib.library(), name)(*arguments, _stream(index))
    else:
        with torch.cuda.device(device):
            status = getattr(_lib.library(), name)(*arguments, _stream(index))
    _lib.check(status, name)


def _scratch(device, count, *sizes):
    size = getattr(_lib.library(), count)(*sizes)
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


def _need(condition, message):
    if not condition:
        raise ValueError(message)


def _check_rows(x, name):
    if not (isinstance(x, torch.Tensor) and x.is_cuda and x.dtype in ROW_TYPES and x.dim() == 2 and x.shape[1] > 0):
        raise ValueError(f'{name} must be a CUDA fp16, bf16 or fp32 tensor [rows, width] with at least one column')


def _check_ids(ids, name):
    if not (isinstance(ids, torch.Tensor) and ids.is_cuda and ids.dtype in (torch.int32, torch.int64)):
        raise ValueError(f'{name} must be a CUDA int32 or int64 tensor')


def _same_device(x, **others):
    device = x.device
    for name, t in others.items():
        if t is not None and t.device != device:
            raise ValueError(f'{name} is on {t.device}, not {device}')


def _needs_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---------------------------------------------------------------- order
def sort_rows(expert, bins):
    """Order the choices of `expert` (CUDA int32 or int64, [rows] or [rows, choices]) by expert, those of one
    expert in their own order.  Values outside [0, bins) drop the choice."""
    _check_ids(expert, 'expert')
    _need(expert.dim() in (1, 2) and (expert.dim() == 1 or expert.shape[1] > 0),
          'expert must have the shape [rows] or [rows, choices]')
    bins = int(bins)
    _need(1 <= bins < 1 << 30, 'bins must be 1 to 2^30 - 1')
    rows, choices = expert.shape[0], 1 if expert.dim() == 1 else expert.shape[1]
    n, device = rows * choices, expert.device
    _need(n < 2 ** 31 - 4096, 'too many (row, choice) pairs')
    expert = expert.detach().contiguous()
    order, slot, offsets = torch.empty(2 * n + bins + 1, dtype=torch.int32, device=device).split((n, n, bins + 1))
    scratch = _scratch(device, 'odie_sort_rows_scratch', n, bins)
    _call('odie_sort_rows', device, expert.data_ptr(), expert.element_size(), n, bins, order.data_ptr(),
          slot.data_ptr(), offsets.data_ptr(), _lib.ptr(scratch))
    return RowOrder(order, slot.view(rows, choices), offsets)


def _check_order(order):
    if not isinstance(order, RowOrder):
        raise ValueError('order must be the RowOrder of sort_rows')
    order_, slot = order.order, order.slot
    if not (slot.is_cuda and slot.dtype == torch.int32 and slot.dim() == 2 and slot.is_contiguous()
            and order_.device == slot.device and order_.dtype == torch.int32 and order_.shape == (slot.numel(),)
            and order_.is_contiguous()):
        raise ValueError('order must hold contiguous CUDA int32 tensors: order [rows * choices] and slot [rows, choices]')


def _check_weights(weights, order):
    if weights is None:
        return None
    shape = tuple(order.slot.shape)
    _need(isinstance(weights, torch.Tensor) and weights.is_cuda and weights.is_floating_point(),
          'weights must be a CUDA floating-point tensor')
    _need(tuple(weights.shape) == shape or (shape[1] == 1 and tuple(weights.shape) == shape[:1]),
          f'weights must have the shape of the choices {shape}, not {tuple(weights.shape)}')
    return weights.float().reshape(shape)  # differentiable: the gradient takes the weights' own type and shape


def _dispatch(x, order, weights):
    n, choices = order.slot.shape
    out = torch.empty((n * choices, x.shape[1]), dtype=x.dtype, device=x.device)
    _call('odie_dispatch', x.device, x.data_ptr(), n, choices, x.shape[1], ROW_TYPES[x.dtype], order.order.data_ptr(),
          order.slot.data_ptr(), _lib.ptr(weights), out.data_ptr())
    return out


def _combine(rows, order, weights):
    n, choices = order.slot.shape
    out = torch.empty((n, rows.shape[1]), dtype=rows.dtype, device=rows.device)
    _call('odie_combine', rows.device, rows.data_ptr(), n, choices, rows.shape[1], ROW_TYPES[rows.dtype],
          order.slot.data_ptr(), _lib.ptr(weights), out.data_ptr())
    return out


def _combine_backward(d_out, rows, order, weights, need_rows, need_weights):
    n, choices = order.slot.shape
    width = d_out.shape[1]
    d_rows = torch.empty((n * choices, width), dtype=d_out.dtype, device=d_out.device) if need_rows else None
    d_weights = torch.empty((n, choices), dtype=torch.float32, device=d_out.device) if need_weights else None
    _call('odie_combine_backward', d_out.device, d_out.data_ptr(), _lib.ptr(rows), n, choices, width,
          ROW_TYPES[d_out.dtype], order.order.data_ptr(), order.slot.data_ptr(), _lib.ptr(weights), _lib.ptr(d_rows),
          _lib.ptr(d_weights))
    return d_rows, d_weights


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weights, order, slot):
        ctx.save_for_backward(x if ctx.needs_input_grad[1] else None, weights, order, slot)
        return _dispatch(x, RowOrder(order, slot, None), weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_rows):
        x, weights, order, slot = ctx.saved_tensors
        order, d_rows = RowOrder(order, slot, None), d_rows.contiguous()
        d_x = _combine(d_rows, order, weights) if ctx.needs_input_grad[0] else None
        # d weights[t, j] = <x[t], d_rows[slot]>: the same product as combine's, the rows' roles exchanged
        d_weights = _combine_backward(x, d_rows, order, None, False, True)[1] if ctx.needs_input_grad[1] else None
        return d_x, d_weights, None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, order, slot):
        ctx.save_for_backward(rows if ctx.needs_input_grad[1] else None, weights, order, slot)
        return _combine(rows, RowOrder(order, slot, None), weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        rows, weights, order, slot = ctx.saved_tensors
        d_rows, d_weights = _combine_backward(d_out.contiguous(), rows, RowOrder(order, slot, None), weights,
                                              ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        return d_rows, d_weights, None, None


def dispatch(x, order, weights=None):
    """Rows in expert order: [rows * choices, width] from x [rows, width] (CUDA fp16, bf16 or fp32), each times its
    weight where `weights` [rows, choices] is given; zero rows for dropped choices."""
    _check_rows(x, 'x')
    _check_order(order)
    _need(x.shape[0] == order.rows, f'x has {x.shape[0]} rows, the order {order.rows}')
    weights = _check_weights(weights, order)
    _same_device(x, order=order.slot, weights=weights)
    x = x.contiguous()
    if _needs_grad(x, weights):
        return _Dispatch.apply(x, weights, order.order, order.slot)
    return _dispatch(x, order, weights)


def combine(rows, order, weights=None):
    """Back from expert order: out [order.rows, width], row t the sum over its choices of weights[t, j] (1 without
    `weights`) times the row at slot[t, j]; dropped choices are left out.  fp32 sums in ascending j."""
    _check_rows(rows, 'rows')
    _check_order(order)
    _need(rows.shape[0] == order.rows * order.choices,
          f'rows has {rows.shape[0]} rows, the order {order.rows} x {order.choices}')
    weights = _check_weights(weights, order)
    _same_device(rows, order=order.slot, weights=weights)
    rows = rows.contiguous()
    if _needs_grad(rows, weights):
        return _Combine.apply(rows, weights, order.order, order.slot)
    return _combine(rows, order, weights)


# ---------------------------------------------------------------- linear
def _aligned(t):
    """Contiguous, starting on a 16-byte boundary (a view of an odd offset is copied)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _linear(x, weight, bias, residual, offsets, activation, training):
    rows, inputs = x.shape
    groups, outputs = (weight.shape[0] if weight.dim() == 3 else 1), weight.shape[-2]
    y = torch.empty((rows, outputs), dtype=x.dtype, device=x.device)
    slope = None
    if training and activation:
        slope = torch.empty((rows, outputs), dtype=torch.int16, device=x.device)
    scratch = _scratch(x.device, 'odie_linear_scratch', rows, inputs, outputs, groups)
    _call('odie_linear', x.device, x.data_ptr(), weight.data_ptr(), _lib.ptr(bias), _lib.ptr(residual), rows, inputs,
          outputs, groups, _lib.ptr(offsets), ROW_TYPES[x.dtype], activation, y.data_ptr(), _lib.ptr(slope),
          _lib.ptr(scratch))
    return y, slope


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, offsets, activation):
        x, weight = _aligned(x), _aligned(weight)
        bias, residual = (None if t is None else t.contiguous() for t in (bias, residual))
        need = ctx.needs_input_grad
        # a ReLU's slope is the sign of its output, unless a residual hides it
        sign = activation == ACTIVATIONS['relu'] and residual is None
        y, slope = _linear(x, weight, bias, residual, offsets, activation, any(need[:3]) and not sign)
        ctx.save_for_backward(x if need[1] else None, weight if need[0] else None, slope,
                              y if sign and any(need[:3]) else None, offsets)
        ctx.sizes = (x.shape, weight.shape)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, d_y):
        x, weight, slope, relu_y, offsets = ctx.saved_tensors
        (rows, inputs), shape = ctx.sizes
        groups, outputs = (shape[0] if len(shape) == 3 else 1), shape[-2]
        need = ctx.needs_input_grad
        d_y = _aligned(d_y)

        def empty(wanted, *size):
            return torch.empty(size, dtype=d_y.dtype, device=d_y.device) if wanted else None
        d_x, d_weight = empty(need[0], rows, inputs), empty(need[1], *shape)
        d_bias = empty(need[2], *shape[:-1])
        # without offsets every row is a group's row, and the residual's gradient is d_y itself
        d_residual = d_y if offsets is None else empty(need[3], rows, outputs)
        if any(need[:3]) or (need[3] and offsets is not None):
            scratch = _scratch(d_y.device, 'odie_linear_backward_scratch', rows, inputs, outputs, groups)
            _call('odie_linear_backward', d_y.device, d_y.data_ptr(), _lib.ptr(slope), _lib.ptr(relu_y), _lib.ptr(x),
                  _lib.ptr(weight), rows, inputs, outputs, groups, _lib.ptr(offsets), ROW_TYPES[d_y.dtype], _lib.ptr(d_x),
                  _lib.ptr(d_weight), _lib.ptr(d_bias), None if offsets is None else _lib.ptr(d_residual),
                  _lib.ptr(scratch))
        return d_x, d_weight, d_bias, d_residual if need[3] else None, None, None


def linear(x, weight, bias=None, residual=None, activation='none', offsets=None):
    """residual + act(x W^T + bias), fp32 sums rounded once; x [..., inputs] CUDA fp16 or bf16, everything of its type.

    Without offsets: weight [outputs, inputs], bias [outputs].  With offsets (CUDA int32 [experts + 1], as of
    RowOrder; non-decreasing from 0): x [rows, inputs], weight [experts, outputs, inputs], bias [experts, outputs];
    rows [offsets[e], offsets[e + 1]) take expert e's layer, rows behind the last offset give zero rows (without
    the residual).  residual: broadcastable to the result.  activation: 'none', 'relu', 'silu' or 'gelu' (erf)."""
    if not (isinstance(x, torch.Tensor) and x.is_cuda and x.dtype in (torch.float16, torch.bfloat16) and x.dim() >= 1
            and x.shape[-1] > 0):
        raise ValueError('x must be a CUDA fp16 or bf16 tensor with at least one column')
    if activation not in ACTIVATIONS:
        raise ValueError(f'activation must be one of {", ".join(ACTIVATIONS)}')
    if not (isinstance(weight, torch.Tensor) and weight.dim() == (2 if offsets is None else 3)
            and weight.shape[-1] == x.shape[-1] and weight.numel() > 0):
        raise ValueError(f'weight must be {"[outputs" if offsets is None else "[experts, outputs"}, {x.shape[-1]}]')
    if bias is not None and bias.shape != weight.shape[:-1]:
        raise ValueError(f'bias must be {tuple(weight.shape[:-1])}')
    for name, t in (('weight', weight), ('bias', bias), ('residual', residual)):
        if t is not None and t.dtype != x.dtype:
            raise ValueError(f'{name} must have the type of x, {x.dtype}')
    if offsets is not None:
        _need(x.dim() == 2, 'x must be [rows, inputs] with offsets')
        _need(weight.shape[0] <= 1024, 'at most 1024 experts')
        if not (isinstance(offsets, torch.Tensor) and offsets.is_cuda and offsets.dtype == torch.int32
                and offsets.shape == (weight.shape[0] + 1,)):
            raise ValueError(f'offsets must be CUDA int32 [{weight.shape[0] + 1}]')
        offsets = offsets.contiguous()
    _same_device(x, weight=weight, bias=bias, residual=residual, offsets=offsets)
    outputs, lead = weight.shape[-2], x.shape[:-1]
    flat = x if x.dim() == 2 else x.reshape(math.prod(lead), x.shape[-1])
    if residual is not None:
        if residual.shape != (*lead, outputs):
            residual = residual.expand(*lead, outputs)
        if residual.dim() != 2:
            residual = residual.reshape(flat.shape[0], outputs)
    if _needs_grad(flat, weight, bias, residual):
        y = _Linear.apply(flat, weight, bias, residual, offsets, ACTIVATIONS[activation])
    else:
        bias, residual = (None if t is None else t.contiguous() for t in (bias, residual))
        y, _ = _linear(_aligned(flat), _aligned(weight), bias, residual, offsets, ACTIVATIONS[activation], False)
    return y if x.dim() == 2 else y.reshape(*lead, outputs)


# ---------------------------------------------------------------- learned rows by id
def _embed(ids, table, scale):
    out = torch.empty((ids.numel(), table.shape[1]), dtype=table.dtype, device=table.device)
    _call('odie_embed', table.device, ids.data_ptr(), ids.element_size(), ids.numel(), table.data_ptr(),
          table.shape[0], table.shape[1], ROW_TYPES[table.dtype], scale, out.data_ptr())
    return out


class _Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale):
        ctx.save_for_backward(ids)
        ctx.shape, ctx.scale = table.shape, scale
        return _embed(ids, table, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        (ids,) = ctx.saved_tensors
        rows, width = ctx.shape
        d_out = d_out.contiguous()
        d_table = torch.empty((rows, width), dtype=d_out.dtype, device=d_out.device)
        scratch = _scratch(d_out.device, 'odie_embed_backward_scratch', ids.numel(), rows, width)
        _call('odie_embed_backward', d_out.device, ids.data_ptr(), ids.element_size(), ids.numel(), d_out.data_ptr(),
              rows, width, ROW_TYPES[d_out.dtype], ctx.scale, d_table.data_ptr(), _lib.ptr(scratch))
        return None, d_table, None


def embed(ids, table, scale=1.0):
    """scale * table[ids]: ids of any shape (CUDA int32 or int64), table [rows, width] CUDA fp16, bf16 or fp32, result
    [*ids.shape, width] of the table's type.  An id outside the table gives a zero row and takes no gradient."""
    _check_ids(ids, 'ids')
    _check_rows(table, 'table')
    _need(1 <= table.shape[0] < 1 << 30, 'the table must have 1 to 2^30 - 1 rows')
    _need(ids.numel() < 2 ** 31 - 4096, 'too many ids')
    _same_device(table, ids=ids)
    flat, table = ids.contiguous(), table.contiguous()
    out = _Embed.apply(flat, table, float(scale)) if _needs_grad(table) else _embed(flat, table, float(scale))
    return out if ids.dim() == 1 else out.view(*ids.shape, table.shape[1])


# ---------------------------------------------------------------- a model of them
class ExpertHeads(nn.Module):
    """The MLP of `model.Head` (ReLU hidden layers, linear output, fp16 activations, fp32 masters) with biases, one
    set of weights per expert and, with codes > 0, a learned input code for each of that many ids (the tile of a
    coordinate, say) added to the features."""

    def __init__(self, n_input, n_output, width, depth, experts, seed, codes=0, device='cuda'):
        super().__init__()
        _need(depth >= 1 and experts >= 1, 'depth and experts must be at least 1')
        self.experts = int(experts)
        shapes = [(width, n_input)] + [(width, width)] * (depth - 1) + [(n_output, width)]
        generator = torch.Generator().manual_seed(int(seed))
        weights = []
        for out_dim, in_dim in shapes:
            bound = math.sqrt(6.0 / (in_dim + out_dim))
            weights.append((torch.rand((experts, out_dim, in_dim), generator=generator) * 2 - 1) * bound)
        self.weights = nn.ParameterList([nn.Parameter(w.to(device)) for w in weights])
        self.biases = nn.ParameterList([nn.Parameter(torch.zeros(w.shape[:2], device=device)) for w in weights])
        self.codes = nn.Parameter(torch.zeros((codes, n_input), device=device)) if codes else None

    def forward(self, features, expert, weights=None, ids=None):
        """fp16 [rows, n_output]: the sum over row t's choices expert[t, j] (negative: none) of weights[t, j] times
        that expert's MLP of features[t] (plus the code of ids[t])."""
        _need((ids is None) == (self.codes is None), 'ids go with codes')
        h = features.to(torch.float16)
        if ids is not None:
            h = h + embed(ids, self.codes).to(torch.float16)
        order = sort_rows(expert, self.experts)
        h = dispatch(h, order)
        for i, (w, b) in enumerate(zip(self.weights, self.biases)):
            h = linear(h, w.to(torch.float16), b.to(torch.float16), offsets=order.offsets,
                       activation='relu' if i + 1 < len(self.weights) else 'none')
        return combine(h, order, weights)
