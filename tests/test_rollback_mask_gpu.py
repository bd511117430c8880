"""``RecurrentRollbackCache``: an armed block with masked steps, rolled back.

The state after a rollback is the snapshot's, moved by the first ``n + 1`` steps of
the block that the mask leaves: the same replay without the masked steps bit for
bit, and the recurrence's state within the bounds of ``test_gdn_rule_gpu``.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import gdn as ogdn
from tests.test_gdn_rule_gpu import _check, _dev, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vec", [False, True])
@pytest.mark.parametrize("counts", [0, 6, [15, 3, 0], "tensor"])
def test_masked_steps_stay_out_of_the_replay(pkg, dev, counts, vec):
    b, t, hk, hv, dk, dv = 3, 16, 2, 4, 128, 128
    arrays = _inputs(71, b, t, hk, hv, dk, dv, vec=vec)
    mask = np.ones((b, t), bool)
    mask[0, :5] = False                 # padded on the left
    mask[1, ::3] = False
    mask[2, :2] = False
    held = [a.copy() for a in arrays]
    for a in held[:5]:                  # what masked steps hold does not matter
        a[~mask] = np.nan
    q, k, v, g, beta, s0 = _dev(held, dev)
    cache = pkg.RecurrentRollbackCache()
    cache[1] = s0
    cache.arm_rollback()
    y = cache.advance(q, k, v, g, beta, mask=torch.from_numpy(mask).to(dev))
    ry, rs = ogdn.gated_delta_rule(*arrays, mask=mask)
    _check(y, cache[1], ry, rs, arrays, t)
    given = torch.tensor([1, 9, 15], dtype=torch.int32, device=dev) if counts == "tensor" else counts
    cache.rollback(given)
    steps = [1 + (counts if isinstance(counts, int) else list(given)[i]) for i in range(b)]
    assert torch.isfinite(cache[1]).all()
    for i in range(b):
        n = int(steps[i])
        one = tuple(a[i:i + 1, :n] for a in arrays[:5]) + (arrays[5][i:i + 1],)
        ry, rs = ogdn.gated_delta_rule(*one, mask=mask[i:i + 1, :n])
        _check(torch.from_numpy(ry), cache[1][i:i + 1], ry, rs, one, n)
        if not mask[i, :n].any():       # nothing left to replay: the snapshot
            assert torch.equal(cache[1][i].cpu(), torch.from_numpy(arrays[5][i]))


def test_replay_in_place_takes_the_mask_of_the_replay(pkg, dev):
    b, t, hk, hv, d = 2, 9, 1, 2, 64
    arrays = _inputs(72, b, t, hk, hv, d, d)
    _, k, v, g, _, s0 = _dev(arrays, dev)
    tape = v.float()
    mask = torch.rand((b, t), generator=torch.Generator().manual_seed(3)).to(dev) < 0.5
    want = pkg.tape_replay_kernel(tape, k, g, s0, mask)
    assert torch.equal(pkg.tape_replay_(s0.clone(), tape, k, g, mask=mask), want)
    steps = torch.tensor([4, 7], dtype=torch.int32, device=dev)
    cut = mask & (torch.arange(t, device=dev)[None] < steps[:, None])
    want = pkg.tape_replay_kernel(tape, k, g, s0, cut)
    assert torch.equal(pkg.tape_replay_(s0.clone(), tape, k, g, steps, mask), want)
    with pytest.raises(ValueError):
        pkg.tape_replay_(s0.clone(), tape, k, g, steps, mask[:, :5])


def test_an_unmasked_block_forgets_the_last_mask(pkg, dev):
    arrays = _inputs(73, 1, 8, 1, 2, 64, 64)
    q, k, v, g, beta, s0 = _dev(arrays, dev)
    cache = pkg.RecurrentRollbackCache()
    cache[1] = s0
    cache.arm_rollback()
    cache.advance(q, k, v, g, beta, mask=torch.zeros((1, 8), dtype=torch.bool, device=dev))
    cache.rollback(7)
    assert torch.equal(cache[1], s0)
    cache.arm_rollback()
    cache.advance(q, k, v, g, beta)
    cache.rollback(4)
    part = tuple(a[:, :5] for a in arrays[:5]) + (arrays[5],)
    ry, rs = ogdn.gated_delta_rule(*part)
    _check(torch.from_numpy(ry), cache[1], ry, rs, part, 5)
