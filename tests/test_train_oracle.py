"""The generator that dropout's tests compare with: Philox4x32-10 against the published known answers."""

from __future__ import annotations

import torch

from tests.train_helpers import factors, numbers, philox


def test_known_answers():
    ones = 0xFFFFFFFF
    assert philox((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert philox((ones,) * 4, (ones, ones)) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert philox((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0)) == [
        0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def test_numbers_are_spread_evenly():
    """Of 32768 numbers the share below a threshold is off by less than five standard deviations; rows, keys, offsets
    and sites differ, and a site is an offset."""
    n = numbers(64, 512, (3, 4))
    for p in (0.1, 0.5, 0.9):
        assert abs(float((n < 65536 * p).double().mean()) - p) < 5 * (p * (1 - p) / n.numel()) ** 0.5
    assert not torch.equal(n[0], n[1])
    assert not torch.equal(n, numbers(64, 512, (3, 5))) and not torch.equal(n, numbers(64, 512, (2, 4)))
    assert torch.equal(numbers(2, 9, (3, 4), site=1), numbers(2, 9, (3, 5)))
    assert torch.equal(numbers(2, 9, (-1, -1)), numbers(2, 9, (2 ** 64 - 1, 2 ** 64 - 1)))
    assert float(factors(3, 7, 1.0, (1, 2)).sum()) == 0.0 and torch.equal(factors(3, 7, 0.0, (1, 2)), torch.ones(3, 7).double())
