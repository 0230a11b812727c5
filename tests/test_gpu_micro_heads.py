"""MicroHeads as a module: what it holds is saved, loaded, moved and copied, and is its own."""
import copy
import io

import pytest
import torch

pytestmark = pytest.mark.gpu


def made(seed, codes=5, block=16):
    from odie_b200.experts import ExpertHeads
    g = torch.Generator(device='cuda').manual_seed(seed)
    heads = ExpertHeads(32, 3, 64, 2, 4, seed=seed, codes=codes)
    with torch.no_grad():
        for b in heads.biases:
            b.normal_(0, 0.2, generator=g)
        if codes:
            heads.codes.normal_(0, 0.5, generator=g)
    return heads


def arguments(codes=5):
    g = torch.Generator(device='cuda').manual_seed(9)
    ids = torch.randint(0, codes, (70,), generator=g, device='cuda') if codes else None
    return (torch.randn((70, 32), generator=g, device='cuda').half(), torch.randint(-1, 4, (70, 2), generator=g, device='cuda'),
            torch.rand((70, 2), generator=g, device='cuda'), ids)


@pytest.mark.parametrize('codes', [0, 5])
@pytest.mark.parametrize('block', [16, 32])
def test_saved_and_loaded(cuda, codes, block):
    """The 4-bit form goes through a file into heads of other weights, without the heads that it came from."""
    a = arguments(codes)
    micro = made(1, codes).microscaled(block)
    want = micro(*a)
    file = io.BytesIO()
    torch.save(micro.state_dict(), file)
    file.seek(0)
    other = made(2, codes).microscaled(block)
    assert not torch.equal(other(*a), want)
    other.load_state_dict(torch.load(file))
    assert torch.equal(other(*a), want)
    state = micro.state_dict()
    # 4.5 or 4.25 bits to a weight, padded to tiles; nothing of full precision
    assert sum(t.numel() for t in state.values() if t.dtype == torch.uint8) > 4 * (32 * 64 + 64 * 64 + 3 * 64) // 2
    with pytest.raises(RuntimeError):
        made(2, codes).microscaled(48 - block).load_state_dict(state)
    with pytest.raises(RuntimeError):
        other.load_state_dict({})


def test_moved_and_copied(cuda):
    a = arguments()
    micro = made(3).microscaled()
    want = micro(*a)
    assert torch.equal(copy.deepcopy(micro)(*a), want)
    assert torch.equal(micro.cpu().cuda()(*a), want)
    there = micro.to('cpu')
    assert there.state_dict() and all(not t.is_cuda for t in there.state_dict().values())
    micro.to('cuda')
    for cast in (lambda m: m.half(), lambda m: m.float()):  # fp16 is what it has; the scales of 4-bit rows are no numbers to cast
        assert torch.equal(cast(micro)(*a), want)
    assert not list(micro.parameters()) and not micro(*a).requires_grad


@pytest.mark.parametrize('half', [False, True])
def test_what_it_holds_is_its_own(cuda, half):
    """Heads that change afterwards, also fp16 ones, do not change their 4-bit form."""
    a = arguments()
    heads = made(4)
    if half:
        heads.half()
    micro = heads.microscaled()
    want = micro(*a)
    with torch.no_grad():
        for p in heads.parameters():
            p.mul_(3)
    assert torch.equal(micro(*a), want)
