"""GPU parity of ``route_experts`` with the definition in float64
(``oracle.moe.route_experts``), of the route table made from its ids with
``route``'s, and of the MoE layers that take a ``Router``.

Ids have to be equal (scores are 64 bits on both sides; ties are put in on
purpose).  Weights: 64-bit arithmetic and one rounding to fp32, 2^-24 of the
value, twice that allowed for the two exponentials' last bits.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import moe as omoe

pytestmark = pytest.mark.gpu


def _check(pkg, dev, lg, k, bias=None, **kw):
    w, ids = pkg.route_experts(lg.to(dev), k, bias=None if bias is None else bias.to(dev), **kw)
    rw, rids = omoe.route_experts(lg.float().numpy(), k, bias=None if bias is None else bias.numpy(), **kw)
    assert w.dtype == torch.float32 and ids.dtype == torch.int32
    np.testing.assert_array_equal(ids.cpu().numpy(), rids)
    np.testing.assert_allclose(w.cpu().numpy(), rw, rtol=2.0 ** -23, atol=1e-45)
    return w, ids


@pytest.mark.parametrize("t,e,k,groups,kept", [
    (1, 1, 1, 1, 1),
    (1, 8, 2, 1, 1),
    (16, 256, 8, 8, 4),
    (16, 256, 8, 1, 1),
    (17, 60, 6, 1, 1),
    (33, 96, 10, 3, 2),
    (5, 128, 32, 4, 2),
    (3, 33, 5, 33, 7),
    (9, 64, 1, 8, 1),
    (2, 4096, 16, 64, 9),
    (4, 1000, 9, 8, 3),
    (1025, 160, 6, 8, 3),
])
@pytest.mark.parametrize("score,with_bias", [("softmax", False), ("softmax", True), ("sigmoid", False),
                                             ("sigmoid", True)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_matches_the_definition(pkg, dev, t, e, k, groups, kept, score, with_bias, dtype):
    gen = torch.Generator().manual_seed(t + e + k)
    lg = (torch.randn((t, e), generator=gen) * 2).to(dtype)
    bias = torch.randn(e, generator=gen) * 0.1 if with_bias else None
    _check(pkg, dev, lg, k, bias, score=score, n_groups=groups, topk_groups=kept)


@pytest.mark.parametrize("kw", [
    dict(score="sigmoid", renormalize=False, scale=2.5),
    dict(score="softmax", renormalize=False),
    dict(score="softmax", n_groups=4, topk_groups=2, group_score="top2"),
    dict(score="sigmoid", n_groups=4, topk_groups=2, group_score="max", scale=16.0),
])
def test_other_weights_and_group_scores(pkg, dev, kw):
    lg = torch.randn((21, 64), generator=torch.Generator().manual_seed(2))
    _check(pkg, dev, lg, 6, **kw)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 8])
def test_ties_go_to_the_lower_id(pkg, dev, score, groups):
    lg = torch.randint(-1, 2, (40, 64), generator=torch.Generator().manual_seed(3)).float()
    lg[0] = 0.25
    bias = torch.zeros(64)
    bias[32:] = 0.125
    kw = dict(score=score, n_groups=groups, topk_groups=max(1, groups // 2))
    _check(pkg, dev, lg, 8, **kw)
    if score == "sigmoid":   # equal scores stay equal with the bias of a half
        _check(pkg, dev, lg, 8, bias, **kw)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,kept", [(1, 1), (4, 2)])
def test_experts_that_cannot_be_had(pkg, dev, score, groups, kept):
    """-inf, NaN, the type's lowest value, +inf; rows that leave nothing."""
    lg = torch.randn((12, 32), generator=torch.Generator().manual_seed(4))
    lg[0] = -torch.inf
    lg[1] = torch.nan
    lg[2, 3:] = -torch.inf
    lg[3, ::2] = torch.nan
    lg[4, 5] = torch.inf
    lg[5, [7, 20]] = torch.inf
    lg[6] = torch.finfo(torch.float32).min
    lg[7, 1:] = torch.finfo(torch.float32).min
    lg[8, :31] = -torch.inf
    lg[9] = -50.0
    lg[10] = 300.0
    w, ids = _check(pkg, dev, lg, 6, score=score, n_groups=groups, topk_groups=kept)
    assert torch.all(w[:2] == 0) and torch.isfinite(w).all()
    assert all(len(set(r)) == 6 for r in ids.tolist())
    bias = torch.zeros(32)
    bias[4] = -torch.inf
    _check(pkg, dev, lg, 6, bias, score=score, n_groups=groups, topk_groups=kept)


def test_strided_rows_no_rows_and_streams(pkg, dev):
    lg = torch.randn((16, 256), generator=torch.Generator().manual_seed(5))
    want = _check(pkg, dev, lg, 8, score="sigmoid", n_groups=8, topk_groups=4)
    wide = torch.full((16, 301), float("nan"))
    wide[:, 7:263] = lg
    kw = dict(score="sigmoid", n_groups=8, topk_groups=4)
    dwide = wide.to(dev)
    for view in (dwide[:, 7:263], lg.to(dev).t().contiguous().t(), lg.to(dev)[:1].expand(16, 256)):
        w, ids = pkg.route_experts(view, 8, **kw)
        if view.stride(0) == 0:
            assert torch.equal(ids, want[1][:1].expand(16, 8))
        else:
            assert torch.equal(w, want[0]) and torch.equal(ids, want[1])
    w, ids = pkg.route_experts(lg.to(dev)[:0], 8, **kw)
    assert w.shape == (0, 8) and ids.shape == (0, 8)
    d = lg.to(dev)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        pkg.route_experts(d, 8, **kw)
        side.synchronize()
        with torch.cuda.graph(g, stream=side):
            w, ids = pkg.route_experts(d, 8, **kw)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(w, want[0]) and torch.equal(ids, want[1])


def test_refusals(pkg, dev):
    lg = torch.randn((4, 32), device=dev)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.route_experts(lg.cpu(), 4)
    with pytest.raises(NotImplementedError):
        pkg.route_experts(lg.double(), 4)
    for args, kw in (((lg[0], 4), {}), ((lg, 0), {}), ((lg, 33), {}), ((lg, 4), dict(score="top")),
                     ((lg, 4), dict(group_score="sum")), ((lg, 4), dict(n_groups=5)),
                     ((lg, 4), dict(n_groups=4, topk_groups=5)), ((lg, 9), dict(n_groups=4, topk_groups=1)),
                     ((lg, 4), dict(n_groups=0)), ((lg, 4), dict(bias=torch.zeros(31, device=dev))),
                     ((lg, 4), dict(bias=torch.zeros(32, dtype=torch.float64, device=dev)))):
        with pytest.raises(ValueError):
            pkg.route_experts(*args, **kw)


@pytest.mark.parametrize("t,e,k", [(16, 256, 8), (1, 3, 2), (7, 31, 16), (16, 16, 16), (16, 300, 1)])
def test_route_table_from_ids_is_routes(pkg, dev, t, e, k):
    """The same table as ``route`` makes beside its ids (active problems only)."""
    from dflash_mlx_b200 import moe

    lg = torch.randn((t, e), generator=torch.Generator().manual_seed(6)).to(dev)
    table, _, ids = moe.route(lg, k)
    mine = moe.route_table(ids, e)
    a, b = table.cpu().numpy(), mine.cpu().numpy()
    n = a[0]
    assert b[0] == n
    np.testing.assert_array_equal(a[1:1 + n], b[1:1 + n])
    np.testing.assert_array_equal(a[1 + e:1 + e + n], b[1 + e:1 + e + n])
    for i in range(n):
        rows = a[1 + e + i]
        for base in (1 + 2 * e + 16 * i, 1 + 18 * e + 16 * i):
            np.testing.assert_array_equal(a[base:base + rows], b[base:base + rows])


def test_route_table_reports_bad_ids(pkg, dev):
    from dflash_mlx_b200 import _lib, moe

    assert _lib.device_error() == 0
    ids = torch.tensor([[0, 5], [-1, 2], [2, 9]], dtype=torch.int32, device=dev)
    table = moe.route_table(ids, 6)
    assert _lib.device_error() == 3
    assert table[:4].tolist() == [3, 0, 2, 5] and table[7:10].tolist() == [1, 2, 1]
    moe.route_table(torch.zeros((16, 3), dtype=torch.int32, device=dev), 6)   # one expert 48 times
    assert _lib.device_error() == 3
    with pytest.raises(ValueError):
        moe.route_table(ids.long(), 6)


def _stack(gen, dev, e, n, k):
    from dflash_mlx_b200.moe import QuantWeight

    q = torch.randint(-2**31, 2**31 - 1, (e, n, k // 8), generator=gen, dtype=torch.int64).to(torch.int32)
    s = torch.rand((e, n, k // 64), generator=gen) * 0.01 + 0.002
    b = -8 * s + torch.randn((e, n, k // 64), generator=gen) * 0.1 * s
    return QuantWeight(q.to(dev), s.bfloat16().to(dev), b.bfloat16().to(dev))


@pytest.mark.parametrize("with_shared", [False, True])
def test_layers_take_a_router(pkg, dev, with_shared):
    """moe_layer and MoEPlanLayer with a Router: the experts and weights that
    route_experts gives (the per-expert sums restated with the same entry
    points), and a softmax Router gives the layer without one."""
    from dflash_mlx_b200 import moe

    gen = torch.Generator().manual_seed(7)
    t, h, inter, e, k = 8, 256, 128, 16, 4
    experts = {"gate": _stack(gen, dev, e, inter, h), "up": _stack(gen, dev, e, inter, h),
               "down": _stack(gen, dev, e, h, inter)}
    shared = None
    if with_shared:
        one = {n: _stack(gen, dev, 1, *s) for n, s in (("gate", (inter, h)), ("up", (inter, h)),
                                                       ("down", (h, inter)))}
        shared = {n: moe.QuantWeight(w.q[0], w.s[0], w.b[0]) for n, w in one.items()}
    x = torch.randn((t, h), generator=gen).bfloat16().to(dev)
    lg = torch.randn((t, e), generator=gen).to(dev)
    bias = (torch.randn(e, generator=gen) * 0.2).to(dev)
    plain = moe.moe_layer(x, lg, experts, shared, k)
    soft = moe.moe_layer(x, lg, experts, shared, k, router=pkg.Router())
    # the weights of the two routers may differ in their last bit before the bf16 rounding
    step = 2.0 ** -7 * plain.float().abs().max()
    assert (plain.float() - soft.float()).abs().max() <= step
    router = pkg.Router(score="sigmoid", bias=bias, n_groups=4, topk_groups=2, scale=1.5)
    w, ids = router(lg, k)
    want = torch.zeros((t, h), device=dev)
    for i in range(t):
        for j in range(k):
            ex = int(ids[i, j])
            one = lambda s: moe.QuantWeight(s.q[ex], s.s[ex], s.b[ex])  # noqa: E731
            want[i] += w[i, j] * moe.dense_mlp(x[i:i + 1], *(one(experts[n]) for n in ("gate", "up", "down")))[0].float()
    if with_shared:
        want += moe.dense_mlp(x, shared["gate"], shared["up"], shared["down"]).float()
    # each expert's three roundings to bf16 (2^-8 of a value each, the middle ones
    # seen through a product of 128 terms) against a different order of sums
    tol = 2.0 ** -6 * want.abs().max()
    y = moe.moe_layer(x, lg, experts, shared, k, router=router)
    assert (y.float() - want).abs().max() <= tol
    layer = moe.MoEPlanLayer(experts, shared, t, k, router=router)
    y2 = layer(x, lg)
    assert (y2.float() - want).abs().max() <= tol
    assert torch.equal(y2, layer(x, lg))
