"""The checks of adapters_sharp on the CPU: they take the exact outputs, rounded, and reject
what a kernel that loses a block of columns or a plane of f32 values would give."""
import pytest
import torch

import adapters_sharp as sharp

F32, BF16 = torch.float32, torch.bfloat16


def without(x, block):
    x = x.clone()
    x[:, block * sharp.BLOCK:(block + 1) * sharp.BLOCK] = 0
    return x


@pytest.mark.parametrize("T,E,R,K,N", sharp.SHAPES)
def test_checks_reject_a_lost_block(T, E, R, K, N):
    blocks = -(-K // sharp.BLOCK)
    some = sorted({0, 1, 7, 8, blocks // 2, blocks - 2, blocks - 1} & set(range(blocks)))
    for make, ok in ((sharp.whole, sharp.whole_ok), (sharp.normal, sharp.normal_ok)):
        case = make(T, E, R, K, N, F32)
        want = sharp.exact(case)
        assert ok(want.float(), case) and ok(want.to(BF16), case)
        for b in some:
            bad = sharp.exact(case, without(case[3], b))
            assert not ok(bad.float(), case), b
    case = sharp.picks(T, E, R, K, N)
    assert sharp.picks_ok(sharp.exact(case).float(), case)
    assert sharp.picks_ok(sharp.exact(case).to(BF16), case)
    used = torch.unique(sharp.picked(R, K, E)[torch.unique(case[2].clamp(min=0)).long(), :N])
    used = torch.unique(used // sharp.BLOCK).tolist()
    for b in set(some) & set(used):
        assert not sharp.picks_ok(sharp.exact(case, without(case[3], b)).float(), case), b


@pytest.mark.parametrize("T,E,R,K,N", sharp.SHAPES)
def test_picks_reject_a_lost_plane(T, E, R, K, N):
    case = sharp.picks(T, E, R, K, N)
    x = case[3]
    assert torch.equal(sharp.planes(x, 3), x)
    for n in (1, 2):
        assert not sharp.picks_ok(sharp.exact(case, sharp.planes(x, n)).float(), case), n
    # one row and one block alone lose the last plane
    cols = sharp.picked(R, K, E)[E - 1, :min(N, R)]
    lost = x.clone()
    at = cols[len(cols) // 2] // sharp.BLOCK * sharp.BLOCK
    lost[0, at:at + sharp.BLOCK] = sharp.planes(x[0, at:at + sharp.BLOCK], 1)
    assert not sharp.picks_ok(sharp.exact(case, lost).float(), case)


def test_every_block_is_picked():
    for _, E, R, K, _ in sharp.SHAPES:
        blocks = -(-K // sharp.BLOCK)
        cols = sharp.picked(R, K, E)
        assert int(cols.max()) == K - 1 and int(cols.min()) >= 0
        if E * R >= blocks:
            assert torch.unique(cols // sharp.BLOCK).numel() == blocks
