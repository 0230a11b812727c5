"""Rows of routed experts: chosen, sorted by expert and back, the experts' own linear layers, learned codes by id.

The routed models choose an expert for each row (`model.route`) and read that expert's table (`ExpertHashQuery`).
The operators here give experts layers of their own: `sort_rows` orders the (row, choice) pairs by expert,
`dispatch` copies each row to its places, `linear` multiplies every group of consecutive rows by its expert's
matrix with bias, activation and residual in the same kernel, `combine` brings the results back as weighted sums;
`embed` looks rows of a learned table up by id.  `gate` chooses the experts of rows from a learned router's logits, and
`balance` says how evenly; `linear4` is `linear` for decoding, with weights that `quantize` has put into 4 bits.  All of them
run the kernels of libodie_b200.so on the current
stream of their tensors' device, are differentiable (once, backward; forward-mode derivatives and transforms of
torch.func are refused; the 4-bit ones not at all) and give the same bits in every run.  `ExpertHeads`
is the MLP of `model.Head` with one set of weights per expert, built from them, `ExpertRouter` a router to train with it.

There is no CPU path: tensors that are not on a CUDA device are refused.
"""
from functools import lru_cache
import math
from typing import NamedTuple

import torch
from torch import nn

from . import _lib

__all__ = ['RowOrder', 'sort_rows', 'dispatch', 'combine', 'linear', 'embed', 'Gating', 'gate', 'Balance', 'balance', 'Micro', 'quantize',
           'dequantize', 'linear4', 'check', 'ExpertHeads', 'MicroHeads', 'ExpertRouter']

SCORES = {'softmax': 0, 'sigmoid': 1}
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
    results are incomplete, and the next `linear`, gradient of it or `linear4`, or `check`, raises RuntimeError."""
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f'activation must be one of {", ".join(ACTIVATIONS)}')
    return _ops().linear(x, weight, bias, residual, code, offsets)


def embed(ids, table, scale=1.0):
    """scale * table[ids]: ids of any shape (CUDA int32 or int64), table [rows, width] CUDA fp16, bf16 or fp32, result
    [*ids.shape, width] of the table's type.  An id outside the table gives a zero row and takes no gradient."""
    return _ops().embed(ids, table, scale)


def _score(name):
    code = SCORES.get(name)
    if code is None:
        raise ValueError(f'score must be one of {", ".join(SCORES)}')
    return code


class Gating(NamedTuple):
    """The choices of rows (gate): expert int32 [rows, choices], -1 where none was left; weights fp32 [rows, choices]."""
    expert: torch.Tensor
    weights: torch.Tensor


def gate(logits, choices, bias=None, mask=None, score='softmax', normalize=True, scale=1.0):
    """The experts of each row, and their weights, from a router's logits [rows, experts] (CUDA fp16, bf16 or fp32).

    A row takes its `choices` (up to 64) experts of the highest logit + bias (fp32; bias [experts], not differentiated),
    ties to the lowest, among those whose mask (bool, broadcastable to the logits) is on and of which neither logit nor sum is
    -inf; a choice for which none is left is -1 with weight 0.  The bias is added to the logit, also with score 'sigmoid': a
    router that was trained with a bias on its scores, sigmoid(logit) + bias, takes other experts here.  A NaN is taken
    first, and makes its row's weights NaN (a sigmoid without normalize: its own).  weights: scale times the softmax over the
    row's open experts, or the sigmoid of the logit, with `normalize` divided by its sum over the row's choices.
    Differentiable in the logits through the weights; a closed expert's gradient is 0.  For sort_rows, dispatch and combine.
    Up to 1024 experts."""
    return Gating(*_ops().gate(logits, choices, bias, mask, _score(score), normalize, scale))


class Balance(NamedTuple):
    """How evenly rows are spread over experts (balance): loss and z, fp32 scalars, and counts int32 [experts]."""
    loss: torch.Tensor
    z: torch.Tensor
    counts: torch.Tensor


def balance(logits, expert, mask=None, score='softmax', total=None):
    """The balance loss of a router's logits [rows, experts] (CUDA fp16, bf16 or fp32) and choices `expert` (int32 or
    int64, [rows] or [rows, choices]; values outside [0, experts) are dropped): experts * sum_e f_e P_e, which is 1 for
    an even load.

    f_e is expert e's share of the choices (without gradient), from `total` [experts], where given: counts summed over
    several ranks, say.  P_e is the mean over live rows (those with an expert whose mask is on and whose logit is not -inf)
    of the softmax over open experts, or with score 'sigmoid' of the sigmoids divided by their sum.  z: the mean over live
    rows of the square of log sum exp of their logits.  counts: this call's choices of each expert.  Without rows or
    choices the loss is 0.  Differentiable in the logits through loss and z."""
    return Balance(*_ops().balance(logits, expert, mask, _score(score), total))


class Micro(NamedTuple):
    """Microscaled 4-bit rows (quantize): value = row scale x block scale x code.

    codes uint8 [..., rows, 16 ceil(width / 32)]: e2m1, two to a byte, the even one low; scales uint8 [groups,
    ceil(rows / 128), ceil(width / (4 block)), 512]: one for each block, e4m3 (block 16) or e8m0 (block 32), in tiles of
    128 rows x 4 blocks: row r, block b at byte 16 (r % 32) + 4 (r // 32) + b; row_scales fp32 [..., rows]."""
    codes: torch.Tensor
    scales: torch.Tensor
    row_scales: torch.Tensor
    width: int
    block: int

    @property
    def shape(self):
        return torch.Size((*self.codes.shape[:-1], self.width))


def quantize(x, block=16):
    """x [rows, width] or [groups, rows, width] (CUDA fp16, bf16 or fp32, up to 2^20 columns) as microscaled 4-bit rows.

    block 16: blocks of 16 values share an e4m3 scale, rows a power of two (so that the largest block's scale is near
    e4m3's largest); block 32: blocks of 32 share a power of two, the least with which nothing saturates.  All roundings
    to nearest even.  A row that holds an infinity or a NaN becomes NaN.  Not differentiable."""
    return Micro(*_ops().quantize(x, block), x.shape[-1], block)


def _micro(m):
    if not isinstance(m, Micro):
        raise ValueError('microscaled rows must be the Micro of quantize')
    return m.codes, m.scales, m.row_scales, m.width, m.block


def dequantize(micro, dtype=torch.float32):
    """The values of microscaled rows, rounded to dtype (exact in fp32, and in bf16 for its normal numbers)."""
    return _ops().dequantize(*_micro(micro), dtype)


def linear4(x, weight, bias=None, residual=None, activation='none', offsets=None):
    """`linear` in 4 bits, for decoding: residual + act(q(x) W^T + bias) with weight the Micro of quantize([outputs,
    inputs]), or of [experts, outputs, inputs] with offsets, and q(x) the rows of x (CUDA fp16 or bf16) quantised in the
    same format in the call; fp32 sums rounded once.  For layers of some 500 inputs and outputs and more: smaller ones are not
    faster than `linear`.  Everything else as for `linear`, but that there are no gradients: an
    argument that wants one is refused.  A row's result does not depend on the rows beside it, but for the order of its
    sum, which depends on how many there are."""
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f'activation must be one of {", ".join(ACTIVATIONS)}')
    return _ops().linear4(x, *_micro(weight), bias, residual, code, offsets)


def check(device=None):
    """Wait for the device (the current one) and raise RuntimeError if a wait of `linear` or `linear4` has run out there that
    no call has raised for yet: after the last step of a program, say, or after replaying a captured graph."""
    with torch.cuda.device(device):
        torch.cuda.synchronize()
        _lib.check(_lib.library().odie_linear_check(), 'linear or linear4')


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

    def microscaled(self, block=16):
        """These heads for decoding, weights in 4 bits (see quantize)."""
        return MicroHeads(self, block)


class MicroHeads(nn.Module):
    """The heads of an ExpertHeads with weights in 4 bits, as they are now: `linear4` in the place of `linear`, without
    gradients; called like ExpertHeads.  Its buffers are copies, and all that it needs: a state dict of it is loaded into the
    4-bit form, of the same block, of any heads of the same sizes.  Casts leave weights and their scales as they are.  For
    wide heads: many rows of narrow ones are not faster (2^20 of 32 -> 64 -> 64 -> 3: 610 us, ExpertHeads 302; 4096 of 1024 ->
    2048 -> 2048 -> 1024 in 64 experts: 162 and 719)."""

    def __init__(self, heads, block=16):
        super().__init__()
        self.experts, self.block = heads.experts, int(block)
        self.widths = [w.shape[-1] for w in heads.weights]
        with torch.no_grad():
            for i, (w, b) in enumerate(zip(heads.weights, heads.biases)):
                micro = quantize(w, block=block)
                self.register_buffer(f'weight{i}', micro.codes)
                self.register_buffer(f'scales{i}_{block}', micro.scales)  # named by the block: those of another do not fit
                self.register_buffer(f'row_scales{i}', micro.row_scales.view(torch.int32))  # as bits: a module's casts are for floats
                self.register_buffer(f'bias{i}', b.to(torch.float16, copy=True))
            self.register_buffer('codes', None if heads.codes is None else heads.codes.to(torch.float16, copy=True))

    @property
    def weights(self):
        """The layers' weights, a Micro each."""
        b = self._buffers
        return [Micro(b[f'weight{i}'], b[f'scales{i}_{self.block}'], b[f'row_scales{i}'].view(torch.float32), width, self.block)
                for i, width in enumerate(self.widths)]

    @property
    def biases(self):
        return [self._buffers[f'bias{i}'].to(torch.float16) for i in range(len(self.widths))]

    @torch.no_grad()
    def forward(self, features, expert, weights=None, ids=None):
        if (ids is None) != (self.codes is None):
            raise ValueError('ids go with codes')
        h = features.to(torch.float16)
        if ids is not None:
            h = h + embed(ids, self.codes).to(torch.float16)
        order = sort_rows(expert, self.experts)
        h = dispatch(h, order)
        for i, (w, b) in enumerate(zip(self.weights, self.biases)):
            h = linear4(h, w, b, offsets=order.offsets, activation='relu' if i + 1 < len(self.widths) else 'none')
        return combine(h, order, weights)


class ExpertRouter(nn.Module):
    """A learned choice of `choices` of `experts` for each row, for ExpertHeads: bf16 logits of one linear layer (fp16
    would lose the gradient of a mean over many rows; logits that round to one number are a tie, which goes to the lower
    expert), `gate` and `balance`.  `shift` [experts] is added to the logits for
    the choice alone; it has no gradient, and a program may move it against the load."""

    def __init__(self, n_input, experts, choices, seed, score='softmax', normalize=True, device='cuda'):
        super().__init__()
        if not 1 <= choices <= experts:
            raise ValueError('choices must be 1 to experts')
        _score(score)
        self.choices, self.score, self.normalize = int(choices), score, bool(normalize)
        bound = math.sqrt(6.0 / (n_input + experts))
        weight = (torch.rand((experts, n_input), generator=torch.Generator().manual_seed(int(seed))) * 2 - 1) * bound
        self.weight = nn.Parameter(weight.to(device))
        self.register_buffer('shift', torch.zeros(experts, device=device))

    def forward(self, features, mask=None):
        """(Gating, Balance) of features [rows, n_input]; mask as for gate."""
        logits = linear(features.to(torch.bfloat16), self.weight.to(torch.bfloat16))
        routing = gate(logits, self.choices, bias=self.shift, mask=mask, score=self.score, normalize=self.normalize)
        return routing, balance(logits, routing.expert, mask=mask, score=self.score)
