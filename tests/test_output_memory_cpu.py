"""Which tensors the operators take to share memory (CPU only)."""

from __future__ import annotations

import pytest
import torch


@pytest.mark.parametrize("a,b,meet", [
    (slice(0, 10), slice(10, 20), False),
    (slice(10, 20), slice(0, 10), False),
    (slice(0, 11), slice(10, 20), True),
    (slice(0, 20), slice(5, 6), True),
    (slice(5, 5), slice(0, 20), False),
])
def test_parts_of_one_allocation(pkg, a, b, meet):
    from dflash_mlx_b200 import _runtime

    x = torch.empty(20, dtype=torch.bfloat16)
    assert _runtime.overlap(x[a], x[b]) == meet and _runtime.overlap(x[b], x[a]) == meet
    assert _runtime.overlap(x[a], None, torch.empty(20), x[b]) == meet
    bytes_ = x.view(torch.uint8)
    assert _runtime.overlap(bytes_[2 * a.start:2 * a.stop], x[b]) == meet


def test_strided_views(pkg):
    from dflash_mlx_b200 import _runtime

    wide = torch.empty((4, 30))
    assert not _runtime.overlap(wide[:2, 10:], wide[2:, :10])
    assert _runtime.overlap(wide[:, :10], wide[1:3])          # between its first and its last element
    assert not _runtime.overlap(wide[:0, :10], wide)
    assert _runtime.overlap(wide.t(), wide[3, 29:])
    assert not _runtime.overlap(wide[0, :1].expand(5), wide[0, 1:])
