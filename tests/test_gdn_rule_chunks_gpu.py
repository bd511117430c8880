"""Every block of 64 steps of ``gated_delta_rule`` by itself: y and states of
whole prompts against the recurrence in float64, where a wrong chunk or piece
must not be averaged away by the others.

Bounds, in the 2-norm.  y of a block: one rounding to bf16 moves every value by at
most 2^-8 of itself, so the block by 2^-8 of its norm; the products before it hold
16 bits or more of the state, of Delta and of the decayed Q K^T, 2^-16 of what a
value is summed from, and with |q| = 1 / sqrt(Dk) spread over the columns that is
less than 16 times the value's own size: 2^-12 together.  A step of no sequence
or a masked one is an exact 0.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import bf16 as obf16
from oracle import gdn as ogdn
from tests.test_gdn_rule_gpu import _dev, _inputs

Y_BOUND = 2.0 ** -8 + 2.0 ** -12
BLOCK = 64


def _bad_blocks(y, ry, ranges=None):
    """``(sequence, first step, error / norm)`` of the blocks whose y is off by more
    than the bound; ``ranges``: token ranges of packed sequences."""
    if ranges is None:
        rows = [(b, 0, ry.shape[1]) for b in range(ry.shape[0])]
    else:
        rows = [(0, a, e) for a, e in ranges]
    bad = []
    for n, (b, a, e) in enumerate(rows):
        for t in range(a, e, BLOCK):
            for h in range(ry.shape[2]):
                want = ry[b, t:min(e, t + BLOCK), h]
                err = np.linalg.norm(y[b, t:min(e, t + BLOCK), h] - want)
                if not err <= Y_BOUND * np.linalg.norm(want):
                    bad.append((n, t - a, h, err / max(np.linalg.norm(want), 1e-300)))
    return bad


def _host(x):
    return x.float().cpu().numpy().astype(np.float64)


@pytest.mark.gpu
@pytest.mark.parametrize("t,hk,hv,dk,dv", [(1100, 50, 150, 128, 128), (1090, 80, 160, 64, 128)])
def test_refilled_buffers_on_a_full_card(pkg, dev, t, hk, hv, dk, dv):
    """More heads than SMs and many chunks each: the shared-memory tile through
    which a chunk's y is turned is the one that later V tiles are copied to.  All
    y right in every call, and the same bits."""
    arrays = _inputs(61, 1, t, hk, hv, dk, dv, slow=True)
    ins = _dev(arrays, dev)
    y, s = pkg.gated_delta_rule(*ins)
    for _ in range(5):
        y2, s2 = pkg.gated_delta_rule(*ins)
        assert torch.equal(y, y2) and torch.equal(s, s2)
    ry, rs = ogdn.gated_delta_rule(*arrays)
    assert _bad_blocks(_host(y), ry) == []
    assert np.linalg.norm(_host(s) - rs) <= 1e-5 * np.linalg.norm(rs)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [1, 100])
def test_one_arena_for_inputs_and_outputs(pkg, dev, t):
    """``out`` and ``out_state`` beside q, k, v and the state in one allocation."""
    arrays = _inputs(62, 2, t, 2, 4, 64, 64)
    ins = _dev(arrays, dev)
    want = pkg.gated_delta_rule(*ins)
    sizes = [ins[0].nbytes, ins[1].nbytes, ins[2].nbytes, ins[2].nbytes, ins[5].nbytes, ins[5].nbytes]
    arena = torch.zeros(sum(sizes), dtype=torch.uint8, device=dev)
    q, k, v, out, state, out_state = (
        part.view(x.dtype).view_as(x)
        for part, x in zip(arena.split(sizes), (*ins[:3], ins[2], ins[5], ins[5])))
    for dst, src in zip((q, k, v, state), (*ins[:3], ins[5])):
        dst.copy_(src)
    y, s = pkg.gated_delta_rule(q, k, v, *ins[3:5], state, out=out, out_state=out_state)
    assert y is out and s is out_state
    assert torch.equal(y, want[0]) and torch.equal(s, want[1]) and torch.equal(state, ins[5])
    with pytest.raises(ValueError, match="share"):
        pkg.gated_delta_rule(q, k, v, *ins[3:5], state, out=v)


@pytest.mark.gpu
def test_outputs_over_inputs_are_refused(pkg, dev):
    """Some threads would still read what others have written over."""
    t, hk, hv, d = 64, 1, 2, 64
    ins = list(_dev(_inputs(63, 1, t, hk, hv, d, d), dev))
    q, k, v, g, beta, s0 = ins
    mask = torch.ones((1, t), dtype=torch.bool, device=dev)
    cu = torch.tensor([0, t], dtype=torch.int32, device=dev)

    def arena(*tensors):
        """The tensors again, all from the first byte of one allocation on."""
        buf = torch.zeros(max(x.nbytes for x in tensors), dtype=torch.uint8, device=dev)
        return [buf[:x.nbytes].view(x.dtype).view(x.shape) for x in tensors]

    for i in range(5):
        mine, out = arena(ins[i], v)
        with pytest.raises(ValueError, match="share"):
            pkg.gated_delta_rule(*ins[:i], mine, *ins[i + 1:], out=out)
        mine, held = arena(ins[i], s0)
        with pytest.raises(ValueError, match="share"):
            pkg.gated_delta_rule(*ins[:i], mine, *ins[i + 1:], out_state=held)
    for kw in (dict(mask=mask), dict(cu_seqlens=cu)):
        (name, x), = kw.items()
        mine, out = arena(x, v)
        with pytest.raises(ValueError, match="share"):
            pkg.gated_delta_rule(*ins, out=out, **{name: mine})
        mine, held = arena(x, s0)
        with pytest.raises(ValueError, match="share"):
            pkg.gated_delta_rule(*ins, out_state=held, **{name: mine})
    held, out = arena(s0, v)
    with pytest.raises(ValueError, match="share"):
        pkg.gated_delta_rule(*ins[:5], held, out=out)
    with pytest.raises(ValueError, match="share"):
        pkg.gated_delta_rule(*ins, out=out, out_state=held)
    # the state's own memory stays open, whole or in part
    want = pkg.gated_delta_rule(*ins)
    y, s = pkg.gated_delta_rule(*ins[:5], s0, out_state=s0)
    assert torch.equal(y, want[0]) and torch.equal(s, want[1])


def _alike(arrays, seed, cosine, norm, beta):
    """The inputs with keys of the given norm and mean cosine to one another."""
    q, k, v, g, _, s0 = arrays
    rng = np.random.default_rng(seed)
    unit = lambda x: x / np.linalg.norm(x, axis=-1, keepdims=True)  # noqa: E731
    base = unit(rng.standard_normal((1, 1, *k.shape[2:])))
    mixed = np.sqrt(cosine) * base + np.sqrt(1 - cosine) * unit(rng.standard_normal(k.shape))
    k = obf16.round_f32((norm * unit(mixed)).astype(np.float32))
    spread = rng.standard_normal(arrays[4].shape)
    b = 1 / (1 + np.exp(-spread)) if beta is None else np.full(spread.shape, beta)
    return q, k, v, g, b.astype(np.float32), s0


@pytest.mark.gpu
@pytest.mark.parametrize("cosine", [0.0, 0.3, 0.5, 0.8, 0.95])
@pytest.mark.parametrize("norm,beta", [(1.0, None), (1.0, 0.98), (0.3, None), (1.3, 1.0)])
@pytest.mark.parametrize("t,hk,hv,dk,dv", [(520, 1, 3, 128, 128), (300, 2, 2, 64, 96), (1500, 1, 2, 128, 64)])
def test_keys_that_are_alike(pkg, dev, t, hk, hv, dk, dv, cosine, norm, beta):
    """The states keep 32-bit accuracy however the keys lie to one another, as long as
    beta |k|^2 < 2 (a step does not stretch a state): 2^-19 of their 2-norm, times
    max(1, beta |k|^2)^2.

    T = (I + A)^-1 is joined twice from blocks, each time by two products of
    32-bit factors in two parts of 11 bits, 2^-22 of a factor left out: 4 x 2^-22 =
    2^-20 of entries that are at most b = beta |k|^2, from products of three blocks
    of such entries, b^2 times as large where b is above 1.  It meets R with 24 bits
    on both sides.  The same again is left for what the recurrence in 32 bits errs
    itself (sums over Dk, decays; a quarter of 2^-20 for random roundings)."""
    arrays = _alike(_inputs(64 + t, 1, t, hk, hv, dk, dv, slow=True), t, cosine, norm, beta)
    y, s = pkg.gated_delta_rule(*_dev(arrays, dev))
    ry, rs = ogdn.gated_delta_rule(*arrays)
    bound = 2.0 ** -19 * max(1.0, (beta or 1.0) * norm ** 2) ** 2
    for h in range(hv):
        assert np.linalg.norm(_host(s)[:, h] - rs[:, h]) <= bound * np.linalg.norm(rs[:, h])
    assert _bad_blocks(_host(y), ry) == []


PADDED = [
    # (b, t, hk, hv, dk, dv, decay per column)
    (1, 1, 16, 48, 128, 128, False),
    (2, 3, 1, 2, 64, 32, True),
    (1, 65, 1, 2, 256, 96, False),
    (1, 63, 1, 3, 128, 128, False),
    (3, 129, 2, 4, 64, 64, False),
    (2, 200, 1, 1, 128, 256, False),
    (1, 700, 1, 2, 128, 128, False),
    (2, 1027, 1, 3, 64, 160, False),
    (1, 1500, 1, 2, 128, 128, False),
    (1, 3000, 2, 4, 128, 32, False),
]
PACKED = [
    ([64, 1, 63, 0, 65, 130], 2, 2, 128, 128),
    ([3, 2000, 0, 700, 1], 1, 2, 128, 128),
    ([64, 2500], 1, 1, 64, 64),
]


def _ranges(lens):
    ends = np.cumsum([0] + lens)
    return list(zip(ends[:-1].tolist(), ends[1:].tolist()))


def _states_right(s, rs):
    """Every sequence's and head's state to 2^-19 of its 2-norm (keys of unit length)."""
    err = np.linalg.norm((s - rs).reshape(*rs.shape[:2], -1), axis=-1)
    return bool(np.all(err <= 2.0 ** -19 * np.linalg.norm(rs.reshape(*rs.shape[:2], -1), axis=-1)))


@pytest.mark.gpu
@pytest.mark.parametrize("slow", [False, True])
@pytest.mark.parametrize("b,t,hk,hv,dk,dv,vec", PADDED)
def test_every_block_of_a_padded_batch(pkg, dev, b, t, hk, hv, dk, dv, vec, slow):
    arrays = _inputs(81 + t, b, t, hk, hv, dk, dv, vec=vec, slow=slow)
    y, s = pkg.gated_delta_rule(*_dev(arrays, dev))
    ry, rs = ogdn.gated_delta_rule(*arrays)
    assert _bad_blocks(_host(y), ry) == [] and _states_right(_host(s), rs)


@pytest.mark.gpu
@pytest.mark.parametrize("slow", [False, True])
@pytest.mark.parametrize("lens,hk,hv,dk,dv", PACKED)
def test_every_block_of_packed_sequences(pkg, dev, lens, hk, hv, dk, dv, slow):
    arrays = _inputs(82 + len(lens), 1, sum(lens), hk, hv, dk, dv, n=len(lens), slow=slow)
    cu = torch.tensor(np.cumsum([0] + lens), dtype=torch.int32, device=dev)
    y, s = pkg.gated_delta_rule(*_dev(arrays, dev), cu_seqlens=cu)
    ry, rs = ogdn.gated_delta_rule(*arrays, lens=_ranges(lens))
    assert _bad_blocks(_host(y), ry, _ranges(lens)) == [] and _states_right(_host(s), rs)


@pytest.mark.gpu
@pytest.mark.parametrize("t,dk,dv", [(40, 128, 128), (300, 64, 64), (1100, 128, 128)])
def test_every_block_under_a_mask(pkg, dev, t, dk, dv):
    arrays = _inputs(83 + t, 2, t, 1, 2, dk, dv, slow=True)
    mask = np.random.default_rng(t).random((2, t)) < 0.6
    mask[1, : t // 2] = False
    y, s = pkg.gated_delta_rule(*_dev(arrays, dev), mask=torch.from_numpy(mask).to(dev))
    ry, rs = ogdn.gated_delta_rule(*arrays, mask=mask)
    assert _bad_blocks(_host(y), ry) == [] and _states_right(_host(s), rs)


@pytest.mark.parametrize("case", PADDED + PACKED)
@pytest.mark.parametrize("slow", [False, True])
def test_the_bounds_reject_wrong_results(case, slow):
    """On the CPU, from the oracle alone: a rounded y passes; y of zeros, scaled by 1% or
    with one block of one sequence a step late does not, nor does a state off by 1e-5."""
    if isinstance(case[0], list):
        lens, hk, hv, dk, dv = case
        arrays = _inputs(82 + len(lens), 1, sum(lens), hk, hv, dk, dv, n=len(lens), slow=slow)
        ranges, rows = _ranges(lens), [(0, a, e) for a, e in _ranges(lens) if e > a]
        ry, rs = ogdn.gated_delta_rule(*arrays, lens=ranges)
    else:
        b, t, hk, hv, dk, dv, vec = case
        arrays = _inputs(81 + t, b, t, hk, hv, dk, dv, vec=vec, slow=slow)
        ranges, rows = None, [(i, 0, t) for i in range(b)]
        ry, rs = ogdn.gated_delta_rule(*arrays)
    rounded = obf16.round_f32(ry.astype(np.float32)).astype(np.float64)
    assert _bad_blocks(rounded, ry, ranges) == [] and _states_right(rs.astype(np.float32).astype(np.float64), rs)
    blocks = sum(-(-(e - a) // BLOCK) for _, a, e in rows) * hv
    assert len(_bad_blocks(np.zeros_like(ry), ry, ranges)) == blocks
    assert len(_bad_blocks(rounded * 1.01, ry, ranges)) == blocks
    b, a, e = max(rows, key=lambda r: r[2] - r[1])
    if e - a > 1:
        last = a + (e - a - 1) // BLOCK * BLOCK        # the longest sequence's last block
        wrong = rounded.copy()
        wrong[b, last + (last == a):e] = rounded[b, last - (last > a):e - 1]
        assert _bad_blocks(wrong, ry, ranges) != []
    assert not _states_right(rs * (1 + 1e-5), rs)
