"""What ``MoEPlanLayer`` reports of its routing, with a ``Router`` and without."""

from __future__ import annotations

import pytest
import torch

from tests.test_route_gpu import _stack

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("score", [None, "softmax", "sigmoid"])
def test_weights_and_ids_of_the_last_call(pkg, dev, score):
    from dflash_mlx_b200 import moe

    gen = torch.Generator().manual_seed(17)
    t, h, inter, e, k = 5, 256, 128, 16, 3
    experts = {"gate": _stack(gen, dev, e, inter, h), "up": _stack(gen, dev, e, inter, h),
               "down": _stack(gen, dev, e, h, inter)}
    router = None if score is None else pkg.Router(score=score, n_groups=4, topk_groups=2, scale=1.5)
    layer = moe.MoEPlanLayer(experts, None, t, k, router=router)
    x = torch.randn((t, h), generator=gen).bfloat16().to(dev)
    for _ in range(2):
        lg = torch.randn((t, e), generator=gen).to(dev)
        layer(x, lg)
        if router is None:
            _, w, ids = moe.route(lg, k)
        else:
            w, ids = router(lg, k)
        assert torch.equal(layer.ids, ids) and torch.equal(layer.weights, w)
    # of a captured call: what its last replay routed
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            layer(x, lg)
    lg.copy_(torch.randn((t, e), generator=gen))
    graph.replay()
    torch.cuda.synchronize()
    ids = moe.route(lg, k)[2] if router is None else router(lg, k)[1]
    assert torch.equal(layer.ids, ids)
