"""CPU: which pairs of row blocks share memory, against the sets of their addresses."""
import itertools

import torch

from muxi_race_b200._args import overlap


def addresses(t):
    size = t.element_size()
    return {t.data_ptr() + (r * t.stride(0) + c) * size + b for r in range(t.shape[0]) for c in range(t.shape[1])
            for b in range(size)}


def test_shared_memory_is_found_exactly_for_one_pitch():
    big = torch.zeros(7, 20, dtype=torch.float16)
    blocks = [big[r0:r0 + n, c0:c0 + c] for r0 in (0, 1, 4) for n in (1, 2, 3) for c0 in (0, 3, 8, 13) for c in (1, 4, 7)]
    # single rows are one range of memory, whatever pitch they are said to have
    for a, b in itertools.product(blocks, blocks):
        shared = bool(addresses(a) & addresses(b))
        assert overlap(a, b) >= shared
        if a.shape[0] > 1 and b.shape[0] > 1:
            assert overlap(a, b) == shared


def test_other_types_pitches_and_tensors():
    big = torch.zeros(4096, dtype=torch.uint8)
    half = big.view(torch.float16)
    wide = half[:512].view(16, 32)
    assert overlap(wide, wide) and overlap(wide[:, :8], wide[:, 4:12]) and not overlap(wide[:, :8], wide[:, 8:])
    assert overlap(wide[:4], half[:256].view(4, 64))
    assert not overlap(wide, half[512:1024].view(16, 32)) and not overlap(wide, torch.zeros(16, 32))
    assert overlap(wide[3:4], wide) and not overlap(wide[:0], wide)
    assert overlap(wide[:1].expand(16, 32), wide[:2])  # one row for all
    assert overlap(wide[:1].expand(16, 32), wide[:1].expand(4, 32))
    assert not overlap(wide[:1].expand(16, 32), wide[1:])
