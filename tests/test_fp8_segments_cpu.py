"""Offsets that fall or leave the rows: the CPU's statement and the kernel take the same segments."""
import pytest
import torch

from shift_b200.ops import fp8

FALLING = [[-10, 90, 50, 400], [0, 200, 100, 200], [50, 20, 20, 130], [150, 0, 0, 0], [300, 300, 10, 200]]


def taken(o, limit):
    """The group of every row, -1 for none: a row belongs to the first group whose end, the largest so far, is behind it."""
    group = [-1] * limit
    for r in range(limit):
        for g in range(len(o) - 1):
            if max(max(x, 0) for x in o[:g + 1]) <= r < max(max(x, 0) for x in o[:g + 2]):
                group[r] = g
    return group


def check_rows(o, device):
    """Group g's matrix is 2^g ones: a row's sums name its group."""
    a = fp8.quantize(torch.ones(200, 64, device=device))
    b = fp8.quantize(torch.stack([torch.full((32, 64), 2.0 ** g) for g in range(3)]).to(device), tiles=True)
    out = torch.full((200, 32), -64.0, device=device)
    fp8.grouped_matmul(a, b, torch.tensor(o, dtype=torch.int32, device=device), out=out)
    want = torch.tensor([64.0 * 2.0 ** g if g >= 0 else -64.0 for g in taken(o, 200)])
    assert torch.equal(out.cpu(), want[:, None].expand(200, 32))


def check_contraction(o, device):
    """The same offsets in blocks of 128: sums count the columns of each segment."""
    a, b = fp8.quantize(torch.ones(16, 200 * 128, device=device)), fp8.quantize(torch.ones(8, 200 * 128, device=device))
    out = torch.full((3, 16, 8), -1.0, device=device)
    fp8.grouped_wgrad(a, b, torch.tensor([128 * x for x in o], dtype=torch.int32, device=device), out)
    group = taken(o, 200)
    assert out[:, 0, 0].tolist() == [128.0 * group.count(g) for g in range(3)]
    assert bool((out == out[:, :1, :1]).all())


@pytest.mark.parametrize("o", FALLING)
def test_rows(o):
    check_rows(o, "cpu")


@pytest.mark.parametrize("o", FALLING)
def test_contraction(o):
    check_contraction(o, "cpu")


def check_nothing_to_contract(o, device):
    a = fp8.quantize(torch.ones(200, 0, device=device))
    b = fp8.quantize(torch.ones(3, 32, 0, device=device), tiles=True)
    out = torch.full((200, 32), -64.0, device=device)
    fp8.grouped_matmul(a, b, torch.tensor(o, dtype=torch.int32, device=device), out=out)
    want = torch.tensor([0.0 if g >= 0 else -64.0 for g in taken(o, 200)])
    assert torch.equal(out.cpu(), want[:, None].expand(200, 32))


@pytest.mark.parametrize("o", FALLING + [[20, 30, 30, 90]])
def test_nothing_to_contract(o):
    check_nothing_to_contract(o, "cpu")
