"""``RecurrentRollbackCache`` refuses, before it touches a device, calls that a
rollback could not take back (CPU only)."""

from __future__ import annotations

import pytest
import torch


def _armed(pkg):
    cache = pkg.RecurrentRollbackCache()
    cache[1] = torch.ones((1, 2, 32, 32))
    cache.arm_rollback()
    cache.record_tape(tape=torch.zeros((1, 3, 2, 32)), k=torch.zeros((1, 3, 1, 32)), g=torch.ones((1, 3, 2)))
    return cache


def _block(t=3):
    bf16 = torch.bfloat16
    return (torch.zeros((1, t, 1, 32), dtype=bf16), torch.zeros((1, t, 1, 32), dtype=bf16),
            torch.zeros((1, t, 2, 32), dtype=bf16), torch.ones((1, t, 2)), torch.ones((1, t, 2)))


def test_a_second_block_on_an_armed_cache_is_refused(pkg):
    """The tape holds one block, from the snapshot on: a second one would be
    replayed onto the state before the first."""
    cache = _armed(pkg)
    tape, state, snapshot = cache._tape, cache[1], cache._snapshot[1]
    with pytest.raises(RuntimeError, match="rollback"):
        cache.advance(*_block())
    assert cache._tape is tape and cache[1] is state and cache._snapshot[1] is snapshot


def test_a_new_arming_or_a_full_acceptance_opens_the_cache_again(pkg):
    for again in (lambda c: c.arm_rollback(), lambda c: c.clear_transients(),
                  lambda c: pkg.restore_after_acceptance([c], target_len=0, acceptance_length=2, drafted_tokens=2)):
        cache = _armed(pkg)
        again(cache)
        with pytest.raises(ValueError, match="CUDA"):   # the operators' own check
            cache.advance(*_block())
