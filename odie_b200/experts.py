"""Rows of routed experts: sorted by expert and back, the experts' own linear layers, learned codes by id.

The routed models choose an expert for each row (`model.route`) and read that expert's table (`ExpertHashQuery`).
The operators here give experts layers of their own: `sort_rows` orders the (row, choice) pairs by expert,
`dispatch` copies each row to its places, `linear` multiplies every group of consecutive rows by its expert's
matrix with bias, activation and residual in the same kernel, `combine` brings the results back as weighted sums;
`embed` looks rows of a learned table up by id.  All of them run the kernels of libodie_b200.so on the current
stream of their tensors' device, are differentiable (once, backward; forward-mode derivatives and transforms of
torch.func are refused) and give the same bits in every run.  `ExpertHeads`
is the MLP of `model.Head` with one set of weights per expert, built from them.

There is no CPU path: tensors that are not on a CUDA device are refused.
"""
from functools import lru_cache
import math
from typing import NamedTuple

import torch
from torch import nn

from . import _lib

__all__ = ['RowOrder', 'sort_rows', 'dispatch', 'combine', 'linear', 'embed', 'check', 'ExpertHeads']

ACTIVATIONS = {'none': 0, 'relu': 1, 'silu': 2, 'gelu': 3}


@lru_cache(maxsize=1)
def _ops():
    """The torch functions over the library (csrc/torch_ops.cpp)."""
    _lib.library()
    try:
        from . import _torch_ops
    except ImportError as e:
        raise _lib.LibraryMissing(f'odie_b200/_torch_ops.so cannot be loaded ({e}): run odie_b200.build() where torch has its headers') from e
    return _torch_ops


class RowOrder(NamedTuple):
    """The (row, choice) pairs in expert order (sort_rows).

    Pair i = row * choices + choice.  order int32 [pairs]: the pair at each place; slot int32 [rows, choices]: the
    place of each pair; offsets int32 [bins + 1]: the first place of each expert, the last one the count of pairs
    that have an expert.  Dropped pairs stand behind: their order is ~pair and their slot ~place."""
    order: torch.Tensor
    slot: torch.Tensor
    offsets: torch.Tensor


def sort_rows(expert, bins):
    """Order the choices of `expert` (CUDA int32 or int64, [rows] or [rows, choices]) by expert, those of one
    expert in their own order.  Values outside [0, bins) drop the choice."""
    return RowOrder(*_ops().sort_rows(expert, bins))


def _tensors(order):
    if not isinstance(order, RowOrder):
        raise ValueError('order must be the RowOrder of sort_rows')
    return order.order, order.slot


def dispatch(x, order, weights=None):
    """Rows in expert order: [rows * choices, width] from x [rows, width] (CUDA fp16, bf16 or fp32), each times its
    weight where `weights` [rows, choices] is given; zero rows for dropped choices."""
    return _ops().dispatch(x, *_tensors(order), weights)


def combine(rows, order, weights=None):
    """Back from expert order: out [order rows, width], row t the sum over its choices of weights[t, j] (1 without
    `weights`) times the row at slot[t, j]; dropped choices are left out.  fp32 sums in ascending j."""
    return _ops().combine(rows, *_tensors(order), weights)


def linear(x, weight, bias=None, residual=None, activation='none', offsets=None):
    """residual + act(x W^T + bias), fp32 sums rounded once; x [..., inputs] CUDA fp16 or bf16, everything of its type.

    Without offsets: weight [outputs, inputs], bias [outputs].  With offsets (CUDA int32 [experts + 1], as of
    RowOrder; non-decreasing from 0): x [rows, inputs], weight [experts, outputs, inputs], bias [experts, outputs];
    rows [offsets[e], offsets[e + 1]) take expert e's layer, rows behind the last offset give zero rows (without
    the residual).  residual: broadcastable to the result.  activation: 'none', 'relu', 'silu' or 'gelu' (erf).  Up to
    2^20 inputs and outputs, 1024 experts and 2^31 - 257 rows.

    The kernels' waits are bounded (some ten seconds).  If one runs out, as on a device that has stopped answering, the
    results are incomplete, and the next `linear` or gradient of it, or `check`, raises RuntimeError."""
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f'activation must be one of {", ".join(ACTIVATIONS)}')
    return _ops().linear(x, weight, bias, residual, code, offsets)


def embed(ids, table, scale=1.0):
    """scale * table[ids]: ids of any shape (CUDA int32 or int64), table [rows, width] CUDA fp16, bf16 or fp32, result
    [*ids.shape, width] of the table's type.  An id outside the table gives a zero row and takes no gradient."""
    return _ops().embed(ids, table, scale)


def check(device=None):
    """Wait for the device (the current one) and raise RuntimeError if a wait of `linear` has run out there that no call
    has raised for yet: after the last step of a program, say, or after replaying a captured graph."""
    with torch.cuda.device(device):
        torch.cuda.synchronize()
        _lib.check(_lib.library().odie_linear_check(), 'linear')


# ---------------------------------------------------------------- a model of them
class ExpertHeads(nn.Module):
    """An MLP like `model.Head` (ReLU hidden layers, linear output, fp16 activations, fp32 masters) with biases, one
    set of weights per expert and, with codes > 0, a learned input code for each of that many ids (the tile of a
    coordinate, say) added to the features.  Weights start uniform within sqrt(6 / (inputs + outputs)) of the layer's own
    sizes (`Head` draws matrices padded to 16, so the same seed gives others there)."""

    def __init__(self, n_input, n_output, width, depth, experts, seed, codes=0, device='cuda'):
        super().__init__()
        if depth < 1 or experts < 1:
            raise ValueError('depth and experts must be at least 1')
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
        if (ids is None) != (self.codes is None):
            raise ValueError('ids go with codes')
        h = features.to(torch.float16)
        if ids is not None:
            h = h + embed(ids, self.codes).to(torch.float16)
        order = sort_rows(expert, self.experts)
        h = dispatch(h, order)
        for i, (w, b) in enumerate(zip(self.weights, self.biases)):
            h = linear(h, w.to(torch.float16), b.to(torch.float16), offsets=order.offsets,
                       activation='relu' if i + 1 < len(self.weights) else 'none')
        return combine(h, order, weights)
