"""The router's operators, the experts' heads and their 4-bit form together, as a program trains and decodes with them."""
import pytest
import torch

from rows_cases import activated
from router_cases import plain_micro

pytestmark = pytest.mark.gpu


def generator(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def made(rows, experts, choices, seed, score='softmax', normalize=True):
    from odie_b200.experts import ExpertHeads, ExpertRouter
    g = generator(seed)
    router, heads = ExpertRouter(32, experts, choices, seed, score, normalize), ExpertHeads(32, 3, 64, 2, experts, seed=seed, codes=5)
    with torch.no_grad():
        heads.codes.normal_(0, 0.5, generator=g)
        for b in heads.biases:
            b.normal_(0, 0.2, generator=g)
        router.weight.mul_(4)
    features = torch.randn((rows, 32), generator=g, device='cuda').half()
    return router, heads, features, torch.randint(0, 5, (rows,), generator=g, device='cuda')


def plain_router(router, features, mask):
    """(logits as the layer rounds them, weights [rows, experts] of the choices, loss, z) in 64 bits, differentiable in the
    router's weights."""
    exact = features.bfloat16().double() @ router.weight.double().t()
    logits = exact + ((features.bfloat16().double() @ router.weight.bfloat16().double().t()).bfloat16().double() - exact).detach()
    open_ = logits if mask is None else torch.where(mask, logits, float('-inf'))
    return open_


@pytest.mark.parametrize('rows, experts, choices', [(1, 4, 2), (700, 8, 2), (900, 16, 1)])
@pytest.mark.parametrize('score, normalize', [('softmax', True), ('softmax', False), ('sigmoid', True)])
def test_router_and_heads_run_and_gradients(cuda, rows, experts, choices, score, normalize):
    """features -> router -> sort -> dispatch -> three layers -> weighted sum, with the balance terms, and back, against 64 bits.

    The heads' tolerance is that of their own test (12 and 24 halves of fp16's step and the corners of ReLU); the router's
    logits are bf16 and its gradient goes through two bf16 roundings more, 2^-8 each of terms whose sum is smaller than they:
    a share of 2^-4 covers cancellation to a sixth of their magnitude."""
    router, heads, features, ids = made(rows, experts, choices, rows + experts, score, normalize)
    mask = torch.rand((rows, 1), generator=generator(1), device='cuda') < 0.9
    mask[0] = True
    routing, load = router(features, mask=mask)
    out = heads(features, routing.expert, routing.weights, ids)
    d = torch.randn((rows, 3), generator=generator(2), device='cuda').half()
    leaves = [router.weight, *heads.parameters()]
    terms = [out, load.loss, load.z]
    scales = [d, torch.tensor(0.5, device='cuda') * rows ** 0.5, torch.tensor(0.05, device='cuda') * rows ** 0.5]
    got = torch.autograd.grad(terms, leaves, scales)

    open_ = plain_router(router, features, mask)
    chosen = routing.expert.long().clamp(min=0)
    live = routing.expert >= 0
    assert torch.equal(live, mask.expand(rows, choices))
    safe = torch.where(mask, open_, 0.0)
    share = torch.softmax(safe, 1) if score == 'softmax' else torch.sigmoid(safe)
    weights = share.gather(1, chosen) * live
    if normalize:
        weights = weights / weights.sum(1, keepdim=True).clamp(min=1e-300)
    assert (routing.weights.double() - weights).abs().max() <= 2.0 ** -7  # a product may round its logit the other way
    h0 = features.double() + heads.codes.double()[ids]
    want = torch.zeros((rows, 3), dtype=torch.float64, device='cuda')
    for j in range(choices):
        for e in range(experts):
            at = ((routing.expert[:, j] == e).nonzero()).view(-1)
            h = h0[at]
            for i, (w, b) in enumerate(zip(heads.weights, heads.biases)):
                h = h @ w[e].double().t() + b[e].double()
                h = h.clamp(min=0) if i < 2 else h
            want = want.index_add(0, at, h * weights[at, j:j + 1])
    assert (out.double() - want).norm() <= (12 * 2 ** -11 + 2 ** -7) * want.norm()
    p = share if score == 'softmax' else share / share.sum(1, keepdim=True)
    f = torch.bincount(routing.expert[live].long(), minlength=experts).double() / live.sum()
    assert torch.equal(load.counts.long(), torch.bincount(routing.expert[live].long(), minlength=experts))
    count = mask.sum()
    loss = experts * (f * (p * mask).sum(0)).sum() / count
    z = (torch.logsumexp(safe, 1).square() * mask[:, 0]).sum() / count
    assert abs(load.loss.item() - loss.item()) <= 2 ** -7 * loss.item() and abs(load.z.item() - z.item()) <= 2 ** -6 * z.item() + 2 ** -10
    plain = torch.autograd.grad([want, loss, z], leaves, [d.double(), scales[1].double(), scales[2].double()])
    for a, b in zip(got[1:], plain[1:]):
        assert torch.isfinite(a).all() and (a.double() - b).norm() <= (2 ** -4.5 + 24 * 2 ** -11 + 2 ** -7) * b.norm()
    assert torch.isfinite(got[0]).all()
    if rows > 1:
        assert (got[0].double() - plain[0]).norm() <= 2 ** -4 * plain[0].norm()


@pytest.mark.parametrize('rows, choices', [(1, 1), (3, 2), (500, 2), (3000, 1)])
@pytest.mark.parametrize('block', [16, 32])
def test_microscaled_heads(cuda, rows, choices, block):
    """The heads in 4 bits against the same quantised layers in 64 bits: from layer to layer a code next to a border may
    round the other way, by a step of 1/6 of its block's largest at most; such values are the share of about 2^-6 (a result
    half a step of fp16, 2^-11, off, over the codes' half step of 2^-3 at the least, times four for its terms), so that a
    layer's relative error stays within 2^-3 sqrt(2^-6) = 2^-6, and three layers' within 2^-4."""
    router, heads, features, ids = made(rows, 6, choices, rows)
    micro = heads.microscaled(block)
    routing, _ = router(features)
    out = micro(features, routing.expert, routing.weights, ids)
    assert out.dtype == torch.float16 and not out.requires_grad
    h0 = (features + heads.codes.half()[ids])
    want = torch.zeros((rows, 3), dtype=torch.float64, device='cuda')
    for j in range(choices):
        for e in range(6):
            at = (routing.expert[:, j] == e).nonzero().view(-1)
            if not at.numel():
                continue
            h = h0[at]
            for i, (w, b) in enumerate(zip(heads.weights, heads.biases)):
                z = plain_micro(h, block)[0] @ plain_micro(w[e].detach(), block)[0].t() + b[e].half().double()
                h = activated(z, 'relu' if i < 2 else 'none')[0].half()
            want.index_add_(0, at, h.double() * routing.weights[at, j:j + 1].detach().double())
    assert (out.double() - want).norm() <= 2 ** -4 * want.norm()
    assert torch.equal(out, micro(features, routing.expert, routing.weights, ids))
    with pytest.raises(ValueError, match='codes'):
        micro(features, routing.expert, routing.weights)


def test_a_step_beside_a_living_graph(cuda):
    """A training step of router and heads, captured while the graph of an eager one of the same leaves lives, and replayed.
    (Both on one stream: torch refuses to capture a backward pass whose leaves first had a graph on the default stream.)"""
    router, heads, features, ids = made(400, 8, 2, 3)
    leaves = [router.weight, *heads.parameters()]

    def step():
        routing, load = router(features)
        out = heads(features, routing.expert, routing.weights, ids)
        return out.float().square().mean() + 0.01 * load.loss + 0.001 * load.z
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = step()
        torch.autograd.grad(step(), leaves)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = torch.autograd.grad(step(), leaves)
    with torch.cuda.stream(side):
        want = torch.autograd.grad(alive, leaves)
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_streams_at_once(cuda):
    """Steps in flight on two streams share nothing."""
    from odie_b200.experts import linear4, quantize
    cases = [made(rows, 8, 2, rows) for rows in (2000, 3000)]
    wide = quantize(torch.randn((600, 700), device='cuda'))
    rows = [torch.randn((n, 700), device='cuda').half() for n in (2, 900)]

    def step(case, x):
        router, heads, features, ids = case
        routing, load = router(features)
        out = heads(features, routing.expert, routing.weights, ids)
        return [out.detach(), load.counts, *torch.autograd.grad(out.float().square().mean() + load.loss, [router.weight, heads.weights[0]]),
                linear4(x, wide)]
    want = [step(c, x) for c, x in zip(cases, rows)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(4):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i] = step(cases[i], rows[i])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))


def test_router_refusals(cuda):
    from odie_b200.experts import Micro, balance, dequantize, gate, linear4, quantize
    x = torch.randn((6, 8), device='cuda')
    ids = torch.zeros((6, 2), dtype=torch.int32, device='cuda')
    mask = torch.ones((6, 8), dtype=torch.bool, device='cuda')
    for call in (lambda: gate(x, 0), lambda: gate(x, 9), lambda: gate(x.double(), 2), lambda: gate(x[0], 2), lambda: gate(x[:, :0], 1),
                 lambda: gate(torch.zeros((2, 1025), device='cuda'), 1), lambda: gate(x, 2, scale=0.0), lambda: gate(x, 2, scale=float('nan')),
                 lambda: gate(x, 2, bias=x[0, :7]), lambda: gate(x, 2, bias=x[:1]), lambda: gate(x, 2, bias=x[0].cpu()),
                 lambda: gate(x, 2, bias=x[0].clone().requires_grad_()), lambda: gate(x, 2, mask=mask.int()), lambda: gate(x, 2, mask=mask[:5]),
                 lambda: gate(x, 2, mask=mask[None]), lambda: gate(x, 2, mask=mask.cpu()), lambda: gate(x, 2, mask=mask[:, :7]),
                 lambda: balance(x, ids[:5]), lambda: balance(x, ids.float()), lambda: balance(x, ids[..., None]), lambda: balance(x, ids.cpu()),
                 lambda: balance(x, ids, mask=mask[:5]), lambda: balance(x, ids, total=ids[0]), lambda: balance(x, ids, total=x[0]),
                 lambda: quantize(x.double()), lambda: quantize(x[0]), lambda: quantize(x[:, :0]), lambda: quantize(x, block=24),
                 lambda: dequantize(quantize(x), torch.float64)):
        with pytest.raises(ValueError):
            call()
    w, h = quantize(x.half()), torch.randn((3, 8), device='cuda').half()
    grouped = quantize(x.half()[None].repeat(2, 1, 1))
    offsets = torch.tensor([0, 1, 3], dtype=torch.int32, device='cuda')
    for call in (lambda: linear4(h.float(), w), lambda: linear4(h[:, :7], w), lambda: linear4(h, grouped), lambda: linear4(h, w, offsets=offsets),
                 lambda: linear4(h, grouped, offsets=offsets.long()), lambda: linear4(h, grouped, offsets=offsets[:2]), lambda: linear4(h, w, bias=h[0]),
                 lambda: linear4(h, w, bias=torch.zeros(6, device='cuda')), lambda: linear4(h, w, residual=h[:, :1].float()), lambda: linear4(h, w[:3]),
                 lambda: linear4(h, w._replace(width=7)), lambda: linear4(h, w._replace(width=40)), lambda: linear4(h, w._replace(block=24)),
                 lambda: linear4(h, w._replace(row_scales=w.row_scales[:5])), lambda: linear4(h, w._replace(scales=w.scales[..., :256])),
                 lambda: linear4(h, w._replace(codes=w.codes.t().contiguous().t())), lambda: linear4(h, w._replace(codes=w.codes.cpu())),
                 lambda: linear4(h.clone().requires_grad_(), w), lambda: linear4(h, w, bias=torch.zeros(6, device='cuda').half().requires_grad_()),
                 lambda: dequantize(Micro(*w[:3], 8, 20)), lambda: dequantize(w._replace(row_scales=w.row_scales.half()))):
        with pytest.raises(ValueError):
            call()
    with torch.no_grad():
        assert linear4(h.clone().requires_grad_(), w).shape == (3, 6)
    with pytest.raises(RuntimeError):
        linear4(h, w, residual=torch.zeros((4, 6), device='cuda').half())
