"""GPU parity of ``gated_delta_rule`` (whole sequences, no tape) with the
recurrence in float64 (``oracle.gdn.gated_delta_rule``).

Tolerances, from the arithmetic: with unit k and beta, g in [0, 1] a step's
map on a state row does not stretch, so the row error of T steps is at most
the sum of what each step adds.  A step's delta holds a Dk-term sum and a few
roundings of values up to R + V (largest row norm and value), (Dk + 8) half
steps of 2^-24 at the very most; the update adds two more.  ``_check`` bounds
every state row by T (Dk + 10) 2^-24 (R + V), and the 2-norm over all states
by 1e-5 of the states' (random roundings do not all point one way).  y adds
one rounding to bf16, 2^-8 of the value, to |q| <= 1 times the row error.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import bf16 as obf16
from oracle import gdn as ogdn

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24


def _inputs(seed, b, t, hk, hv, dk, dv, n=None, vec=False, slow=False):
    rng = np.random.default_rng(seed)
    unit = lambda x: x / np.linalg.norm(x, axis=-1, keepdims=True)  # noqa: E731
    q = obf16.round_f32((unit(rng.standard_normal((b, t, hk, dk))) / np.sqrt(dk)).astype(np.float32))
    k = obf16.round_f32(unit(rng.standard_normal((b, t, hk, dk))).astype(np.float32))
    v = obf16.round_f32(rng.standard_normal((b, t, hv, dv)).astype(np.float32))
    beta = (1 / (1 + np.exp(-rng.standard_normal((b, t, hv))))).astype(np.float32)
    rate = 0.02 if slow else 0.6
    g = np.exp(-rate * np.log1p(np.exp(rng.standard_normal((b, t, hv, dk) if vec else (b, t, hv)))))
    s0 = (rng.standard_normal((b if n is None else n, hv, dv, dk)) * 0.05).astype(np.float32)
    return q, k, v, g.astype(np.float32), beta, s0


def _dev(arrays, dev):
    q, k, v, g, beta, s0 = (torch.from_numpy(np.ascontiguousarray(a)).to(dev) for a in arrays)
    return q.bfloat16(), k.bfloat16(), v.bfloat16(), g, beta, s0


def _check(y, s, ry, rs, arrays, steps):
    q, k, v, g, beta, s0 = arrays
    y, s = y.float().cpu().numpy().astype(np.float64), s.cpu().numpy().astype(np.float64)
    dk = k.shape[-1]
    reach = max(np.linalg.norm(rs, axis=-1).max(initial=0), np.linalg.norm(s0, axis=-1).max(initial=0))
    reach += np.sqrt(steps) + np.abs(v).max(initial=0)
    row = max(steps, 1) * (dk + 10) * EPS * reach
    assert np.linalg.norm(s - rs, axis=-1).max(initial=0) <= row
    assert np.linalg.norm(s - rs) <= 1e-5 * np.linalg.norm(rs)
    qn = np.linalg.norm(q, axis=-1).max(initial=0)
    assert np.all(np.abs(y - ry) <= 2.0 ** -8 * np.abs(ry) + qn * row + 1e-30)


@pytest.mark.parametrize("b,t,hk,hv,dk,dv,vec", [
    (1, 1, 16, 48, 128, 128, False),     # a single token
    (5, 1, 2, 6, 128, 128, False),
    (1, 1, 1, 1, 32, 32, False),
    (2, 3, 1, 2, 64, 32, True),
    (1, 65, 1, 2, 256, 96, False),
    (1, 33, 2, 2, 256, 32, True),
    (2, 16, 2, 4, 32, 160, False),
    (2, 17, 2, 2, 128, 32, True),
    (1, 63, 1, 3, 128, 128, False),
    (2, 64, 2, 2, 128, 64, False),
    (1, 65, 1, 2, 128, 128, False),
    (3, 129, 2, 4, 64, 64, False),
    (2, 200, 1, 1, 128, 256, False),
    (1, 700, 1, 2, 128, 128, False),
    (1, 300, 1, 2, 64, 96, False),
    (1, 1500, 1, 2, 128, 128, False),    # few heads: cut in pieces
    (2, 1027, 1, 3, 64, 160, False),
    (1, 3000, 2, 4, 128, 32, False),
])
@pytest.mark.parametrize("slow", [False, True])
def test_padded_batch(pkg, dev, b, t, hk, hv, dk, dv, vec, slow):
    arrays = _inputs(t * 7 + dk + slow, b, t, hk, hv, dk, dv, vec=vec, slow=slow)
    y, s = pkg.gated_delta_rule(*_dev(arrays, dev))
    _check(y, s, *ogdn.gated_delta_rule(*arrays), arrays, t)


@pytest.mark.parametrize("lens,hk,hv,dk,dv", [
    ([1], 1, 1, 128, 128),
    ([1, 0, 2, 1], 1, 2, 128, 128),
    ([0, 0], 1, 2, 128, 128),
    ([64, 1, 63, 0, 65, 130], 2, 2, 128, 128),
    ([200, 7, 300], 1, 3, 64, 64),
    ([5, 131], 1, 1, 256, 64),
    ([90, 91, 300], 1, 1, 128, 160),
    ([3, 2000, 0, 700, 1], 1, 2, 128, 128),   # pieces of very unlike sequences
    ([64, 2500], 1, 1, 64, 64),
])
def test_packed_sequences(pkg, dev, lens, hk, hv, dk, dv):
    """Lengths of zero and one, ends inside a tile, rows before the first and
    behind the last sequence: left as they were in ``out``, zero in a new y."""
    lead, tail = 3, 5
    total = lead + sum(lens) + tail
    arrays = _inputs(sum(lens), 1, total, hk, hv, dk, dv, n=len(lens))
    cu = np.cumsum([lead] + lens).astype(np.int32)
    ranges = list(zip(cu[:-1].tolist(), cu[1:].tolist()))
    # what stands in rows of no sequence must not matter
    for a in arrays[:5]:
        a[0, :lead] = np.nan
        a[0, lead + sum(lens):] = np.nan
    ins = _dev(arrays, dev)
    ref = ogdn.gated_delta_rule(*arrays, lens=ranges)
    cut = slice(lead, lead + sum(lens))
    clean = tuple(a[:, cut] if i < 5 else a for i, a in enumerate(arrays))
    tcu = torch.from_numpy(cu).to(dev)
    y, s = pkg.gated_delta_rule(*ins, cu_seqlens=tcu)
    assert torch.all(y[0, :lead] == 0) and torch.all(y[0, cut.stop:] == 0)
    _check(y[:, cut], s, ref[0][:, cut], ref[1], clean, max(lens + [1]))
    out = torch.full_like(y, 7.0)
    y2, s2 = pkg.gated_delta_rule(*ins, cu_seqlens=tcu, out=out)
    assert y2 is out and torch.all(out[0, :lead] == 7) and torch.all(out[0, cut.stop:] == 7)
    assert torch.equal(out[:, cut], y[:, cut]) and torch.equal(s, s2)


@pytest.mark.parametrize("t,dk,dv", [(1, 128, 128), (40, 128, 128), (150, 128, 128), (150, 64, 64), (40, 256, 32),
                                      (1100, 128, 128)])
def test_mask(pkg, dev, t, dk, dv):
    """Masked steps change nothing, whatever they hold; one sequence is masked whole."""
    b, hk, hv = 3, 2, 4
    arrays = _inputs(t, b, t, hk, hv, dk, dv)
    rng = np.random.default_rng(5)
    mask = rng.random((b, t)) < 0.7
    mask[0, : t // 2] = False
    mask[1] = False
    ref = ogdn.gated_delta_rule(*arrays, mask=mask)
    q, k, v, g, beta, s0 = (a.copy() for a in arrays)
    for a, x in ((q, np.nan), (k, np.inf), (v, -np.inf), (g, np.nan), (beta, np.inf)):
        a[~mask] = x
    y, s = pkg.gated_delta_rule(*_dev((q, k, v, g, beta, s0), dev), mask=torch.from_numpy(mask).to(dev))
    assert torch.all(y[1] == 0) and torch.equal(s[1].cpu(), torch.from_numpy(s0[1]))
    _check(y, s, *ref, arrays, t)


@pytest.mark.parametrize("lens", [[3, 1, 5], [40, 0, 90, 64], [700, 900]])
def test_mask_over_packed_sequences(pkg, dev, lens):
    arrays = _inputs(sum(lens), 1, sum(lens), 1, 2, 128, 128, n=len(lens))
    cu = np.cumsum([0] + lens)
    mask = np.random.default_rng(8).random((1, sum(lens))) < 0.6
    ref = ogdn.gated_delta_rule(*arrays, mask=mask, lens=list(zip(cu[:-1].tolist(), cu[1:].tolist())))
    for a in arrays[:5]:
        a[~mask] = np.nan
    y, s = pkg.gated_delta_rule(*_dev(arrays, dev), mask=torch.from_numpy(mask).to(dev),
                                cu_seqlens=torch.from_numpy(cu.astype(np.int32)).to(dev))
    clean = tuple(np.nan_to_num(a) for a in arrays)
    _check(y, s, *ref, clean, max(lens))


@pytest.mark.parametrize("t", [24, 39, 40, 63, 64])
@pytest.mark.parametrize("dk,dv", [(64, 64), (64, 128), (128, 32)])
def test_many_small_heads(pkg, dev, t, dk, dv):
    """More heads than SMs, steps on both sides of where 64 are taken at a time."""
    arrays = _inputs(31 + t, 19, t, 4, 8, dk, dv)
    y, s = pkg.kernels.gated_delta_rule(*_dev(arrays, dev))
    ry, rs = ogdn.gated_delta_rule(*arrays)
    _check(y, s, ry, rs, arrays, t)


def test_no_sequences(pkg, dev):
    arrays = _inputs(4, 1, 30, 1, 2, 128, 128, n=0)
    y, s = pkg.gated_delta_rule(*_dev(arrays, dev), cu_seqlens=torch.zeros(1, dtype=torch.int32, device=dev))
    assert torch.all(y == 0) and s.shape == (0, 2, 128, 128)


def test_no_steps(pkg, dev):
    arrays = _inputs(3, 2, 0, 2, 4, 64, 32)
    y, s = pkg.gated_delta_rule(*_dev(arrays, dev))
    assert y.shape == (2, 0, 4, 32) and torch.equal(s.cpu(), torch.from_numpy(arrays[5]))


@pytest.mark.parametrize("t,dk", [(150, 128), (9, 128), (150, 64)])
def test_decay_of_zero_one_and_small_values(pkg, dev, t, dk):
    """g = 0 forgets everything before the step; 1 keeps all; tiny ones underflow."""
    arrays = _inputs(11, 2, t, 1, 3, dk, 128)
    g = arrays[3]
    g[:, :, 0] = 1.0
    g[:, t // 3, 1] = 0.0
    g[:, t - 1, 1] = 0.0
    g[:, :, 2] = 1e-30
    y, s = pkg.gated_delta_rule(*_dev(arrays, dev))
    assert torch.isfinite(y.float()).all() and torch.isfinite(s).all()
    _check(y, s, *ogdn.gated_delta_rule(*arrays), arrays, t)


def test_beta_of_zero_and_one_and_repeated_keys(pkg, dev):
    """The same key at every step with beta = 1: each value replaces the last one."""
    arrays = _inputs(12, 1, 200, 1, 2, 128, 128)
    q, k, v, g, beta, s0 = arrays
    k[:] = k[:, :1]
    g[:] = 1.0
    beta[:, :, 0] = 1.0
    beta[:, :, 1] = 0.0
    y, s = pkg.gated_delta_rule(*_dev(arrays, dev))
    _check(y, s, *ogdn.gated_delta_rule(*arrays), arrays, 200)
    assert torch.equal(s[0, 1].cpu(), torch.from_numpy(s0[0, 1]))


@pytest.mark.parametrize("t", [1, 100])
def test_views_of_a_wider_projection(pkg, dev, t):
    """q, k, v as slices of one [B, T, C] output, read in place or copied (odd offset)."""
    b, hk, hv, dk, dv = 2, 2, 4, 128, 128
    arrays = _inputs(21, b, t, hk, hv, dk, dv)
    q, k, v, g, beta, s0 = _dev(arrays, dev)
    want = pkg.gated_delta_rule(q, k, v, g, beta, s0)
    for lead in (0, 8, 3):
        c = lead + 2 * hk * dk + hv * dv
        wide = torch.full((b, t, c), float("nan"), dtype=torch.bfloat16, device=dev)
        cut = [lead, lead + hk * dk, lead + 2 * hk * dk, c]
        parts = []
        for x, a, e in zip((q, k, v), cut[:-1], cut[1:]):
            wide[:, :, a:e] = x.reshape(b, t, -1)
            parts.append(wide[:, :, a:e].unflatten(-1, x.shape[2:]))
        y, s = pkg.gated_delta_rule(*parts, g, beta, s0)
        assert torch.equal(y, want[0]) and torch.equal(s, want[1])
    # heads first in memory, and every second token of a longer tensor
    y, s = pkg.gated_delta_rule(q.transpose(1, 2).contiguous().transpose(1, 2),
                                torch.stack([k, k], 2).flatten(1, 2)[:, ::2],
                                v.transpose(2, 3).contiguous().transpose(2, 3), g, beta, s0)
    assert torch.equal(y, want[0]) and torch.equal(s, want[1])


@pytest.mark.parametrize("t", [1, 100, 1100])
def test_in_place_and_overlapping_state(pkg, dev, t):
    arrays = _inputs(22, 2, t, 2, 4, 128, 128)
    ins = _dev(arrays, dev)
    y, s = pkg.gated_delta_rule(*ins)
    assert torch.equal(ins[5].cpu(), torch.from_numpy(arrays[5]))
    held = ins[5].clone()
    y2, s2 = pkg.gated_delta_rule(*ins[:5], held, out_state=held)
    assert s2 is held and torch.equal(held, s) and torch.equal(y2, y)
    buf = torch.zeros(held.numel() + 64, device=dev)
    old, new = buf[:held.numel()].view_as(held), buf[64:].view_as(held)
    old.copy_(ins[5])
    y3, s3 = pkg.gated_delta_rule(*ins[:5], old, out_state=new)
    assert torch.equal(s3, s) and torch.equal(y3, y)


def test_same_bits_on_every_call_and_in_any_company(pkg, dev):
    """No atomics, no order of arrival: the same sequence gives the same bits
    again, alone, and beside others of its length."""
    lens = [150, 40, 150]
    arrays = _inputs(23, 1, sum(lens), 2, 4, 128, 128, n=3)
    q, k, v, g, beta, s0 = _dev(arrays, dev)
    cu = torch.tensor([0, 150, 190, 340], dtype=torch.int32, device=dev)
    y, s = pkg.gated_delta_rule(q, k, v, g, beta, s0, cu_seqlens=cu)
    y2, s2 = pkg.gated_delta_rule(q, k, v, g, beta, s0, cu_seqlens=cu)
    assert torch.equal(y, y2) and torch.equal(s, s2)
    y3, s3 = pkg.gated_delta_rule(*(x[:, 190:] for x in (q, k, v, g, beta)), s0[2:])
    assert torch.equal(y[:, 190:], y3) and torch.equal(s[2:], s3)


def test_prompt_in_pieces(pkg, dev):
    """A prompt taken whole, and in pieces that end anywhere, from one state to the next."""
    arrays = _inputs(24, 1, 333, 1, 2, 128, 128)
    ins = _dev(arrays, dev)
    ref = ogdn.gated_delta_rule(*arrays)
    state, ys, at = ins[5], [], 0
    for n in (1, 63, 64, 100, 1, 104):
        y, state = pkg.gated_delta_rule(*(x[:, at:at + n] for x in ins[:5]), state)
        ys.append(y)
        at += n
    assert at == 333
    _check(torch.cat(ys, 1), state, *ref, arrays, 333)


def test_bad_offsets_are_reported_and_stay_inside(pkg, dev):
    from dflash_mlx_b200 import _lib

    arrays = _inputs(25, 1, 90, 1, 2, 128, 128, n=3)
    ins = _dev(arrays, dev)
    assert _lib.device_error() == 0
    for bad in ([0, 95, 90, 90], [-4, 10, 20, 90], [50, 20, 60, 2**31 - 1], [-2**31, -5, 300, 400]):
        cu = torch.tensor(bad, dtype=torch.int32, device=dev)
        y, s = pkg.gated_delta_rule(*ins, cu_seqlens=cu)
        assert y.shape == (1, 90, 2, 128) and _lib.device_error() == 3
    cu = torch.tensor([0, 30, 60, 90], dtype=torch.int32, device=dev)
    pkg.gated_delta_rule(*ins, cu_seqlens=cu)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("t", [1, 150, 1100])
def test_captured_and_on_another_stream(pkg, dev, t):
    arrays = _inputs(26, 2, t, 2, 4, 128, 128)
    ins = _dev(arrays, dev)
    want = pkg.gated_delta_rule(*ins)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graphs, got = [], []
    with torch.cuda.stream(side):
        got.append(pkg.gated_delta_rule(*ins))
        side.synchronize()
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                got.append(pkg.gated_delta_rule(*ins))
            graphs.append(g)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    graphs[0].replay()
    with torch.cuda.stream(other):   # two graphs at once
        graphs[1].replay()
    torch.cuda.synchronize()
    for y, s in got:
        assert torch.equal(y, want[0]) and torch.equal(s, want[1])
    # new inputs in the same buffers
    ins[2].mul_(0.5)
    graphs[0].replay()
    torch.cuda.synchronize()
    again = pkg.gated_delta_rule(*ins)
    assert torch.equal(got[1][0], again[0]) and torch.equal(got[1][1], again[1])


@pytest.mark.parametrize("t,hk,hv", [(1800, 1, 2), (300, 2, 4), (20, 2, 4)])
def test_replayed_with_other_offsets(pkg, dev, t, hk, hv):
    """A captured packed call holds for any offsets, those that leave all but one
    sequence empty among them."""
    arrays = _inputs(41, 1, t, hk, hv, 128, 64, n=3)
    ins = _dev(arrays, dev)
    cu = torch.tensor([0, t // 3, t // 2, t], dtype=torch.int32, device=dev)
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        pkg.gated_delta_rule(*ins, cu_seqlens=cu)
        side.synchronize()
        with torch.cuda.graph(g, stream=side):
            y, s = pkg.gated_delta_rule(*ins, cu_seqlens=cu)
    for ends in ([0, t // 3, t // 2, t], [0, 0, t, t], [0, 1, 2, t - 1], [t, t, t, t]):
        cu.copy_(torch.tensor(ends, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        ry, rs = np.zeros(y.shape), np.zeros(s.shape)
        for n in range(3):
            part = [a[:, ends[n]:ends[n + 1]] for a in arrays[:5]] + [arrays[5][n:n + 1]]
            ry[:, ends[n]:ends[n + 1]], rs[n:n + 1] = ogdn.gated_delta_rule(*part)
        _check(y, s, ry, rs, arrays, t)


def test_refusals(pkg, dev):
    ins = list(_dev(_inputs(27, 2, 4, 2, 4, 64, 32), dev))

    def call(i=None, x=None, **kw):
        a = list(ins)
        if i is not None:
            a[i] = x
        return pkg.gated_delta_rule(*a, **kw)

    cu = torch.tensor([0, 2, 4], dtype=torch.int32, device=dev)
    with pytest.raises(ValueError, match="CUDA"):
        call(5, ins[5].cpu())
    with pytest.raises(ValueError, match="CUDA"):
        call(0, ins[0].cpu())
    for i in (0, 1, 2):
        with pytest.raises(NotImplementedError):
            call(i, ins[i].float())
    for i in (3, 4, 5):
        with pytest.raises(NotImplementedError):
            call(i, ins[i].double())
    with pytest.raises(ValueError):
        call(0, ins[0][:, :3])
    with pytest.raises(ValueError):
        call(2, ins[2][..., :16])
    with pytest.raises(ValueError):
        call(2, ins[2][:, :, :3])
    with pytest.raises(ValueError):
        call(4, ins[4][..., :2])
    with pytest.raises(ValueError):
        call(3, ins[3][:, :3])
    with pytest.raises(ValueError):
        call(5, ins[5][:1])
    with pytest.raises(ValueError):
        call(cu_seqlens=cu)   # B = 2 is not packed
    with pytest.raises(ValueError):
        call(mask=torch.ones(2, 5, dtype=torch.bool, device=dev))
    with pytest.raises(ValueError):
        call(mask=torch.ones(2, 4, device=dev))
    with pytest.raises(ValueError):
        call(out=torch.empty(2, 4, 4, 32, device=dev))
    with pytest.raises(ValueError):
        call(out_state=torch.empty(2, 4, 64, 32, device=dev))
    shared = torch.empty(2 * 4 * 4 * 32, dtype=torch.bfloat16, device=dev).view(2, 4, 4, 32)
    with pytest.raises(ValueError, match="share"):
        call(2, shared, out=shared)
    one = [x[:1] for x in ins[:5]]
    with pytest.raises(ValueError):
        pkg.gated_delta_rule(*one, ins[5], cu_seqlens=cu.long())
    with pytest.raises(ValueError):
        pkg.gated_delta_rule(*one, ins[5][:1], cu_seqlens=cu)


def test_cache_advance_then_rollback(pkg, dev):
    """A GDN layer's life: prompt and token without a tape, a verify block with
    one, a rollback to the accepted steps -- the states of the recurrence."""
    arrays = _inputs(28, 2, 130, 2, 4, 128, 128)
    q, k, v, g, beta, s0 = _dev(arrays, dev)
    cache = pkg.RecurrentRollbackCache()
    cache[1] = s0
    piece = lambda a, e: [x[:, a:e] for x in (q, k, v, g, beta)]  # noqa: E731
    ys = [cache.advance(*piece(0, 100)), cache.advance(*piece(100, 101))]
    cache.arm_rollback()
    cache.advance(*piece(101, 117))
    cache.rollback(4)   # the staged token and four drafts: 106 tokens in all
    ys.append(cache.advance(*piece(101, 106)) * 0)
    part = tuple(a[:, :106] for a in arrays[:5]) + (arrays[5],)
    twice = [np.concatenate([a, a[:, 101:106]], 1) for a in part[:5]]
    _, rs = ogdn.gated_delta_rule(*twice, arrays[5])
    ry, _ = ogdn.gated_delta_rule(*part)
    _check(torch.cat(ys[:2], 1), cache[1], ry[:, :101], rs, tuple(a[:, :101] for a in part[:5]) + (part[5],), 111)
    fresh = pkg.RecurrentRollbackCache()
    y = fresh.advance(*piece(0, 70))
    ry, rs = ogdn.gated_delta_rule(*(a[:, :70] for a in arrays[:5]), np.zeros_like(arrays[5]))
    _check(y, fresh[1], ry, rs, tuple(a[:, :70] for a in arrays[:5]) + (np.zeros_like(arrays[5]),), 70)
