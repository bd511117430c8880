"""One sampled step of a small gated-delta MoE target with the operators as they
are used together: prompts prefilled, a token decoded, a block of drafts run
with its tape, its rows routed by a sigmoid router through an expert layer,
the drafts verified against the logits from given uniforms, and the recurrent
state rolled back to what was accepted -- all from device to device, and each
part equal to its definition on what the part before it gave.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import gdn as ogdn
from oracle import moe as omoe
from oracle import sampled as osm
from tests.test_gdn_rule_gpu import _check, _dev, _inputs
from tests.test_route_gpu import _stack

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed,draft", [(1, True), (2, False), (3, True)])
def test_prefill_verify_route_accept_rollback(pkg, dev, seed, draft):
    from dflash_mlx_b200 import moe

    b, prompt, block, hk, hv, d, vocab = 2, 90, 8, 2, 4, 64, 515
    arrays = _inputs(seed, b, prompt + 1 + block, hk, hv, d, d)
    q, k, v, g, beta, s0 = _dev(arrays, dev)
    cut = lambda a, e: [x[:, a:e] for x in (q, k, v, g, beta)]  # noqa: E731
    cache = pkg.RecurrentRollbackCache()
    cache[1] = s0
    y = torch.cat([cache.advance(*cut(0, prompt)), cache.advance(*cut(prompt, prompt + 1))], 1)
    part = tuple(a[:, :prompt + 1] for a in arrays[:5]) + (arrays[5],)
    ry, rs = ogdn.gated_delta_rule(*part)
    _check(y, cache[1], ry, rs, part, prompt + 1)

    cache.arm_rollback()
    yb = cache.advance(*cut(prompt + 1, prompt + 1 + block))

    # the block's rows through an expert layer with its router
    gen = torch.Generator().manual_seed(seed)
    h, inter, experts = hv * d, 128, 16
    x = (yb.reshape(b * block, h).float() * 20).bfloat16()
    stacks = {"gate": _stack(gen, dev, experts, inter, h), "up": _stack(gen, dev, experts, inter, h),
              "down": _stack(gen, dev, experts, h, inter)}
    router = pkg.Router(score="sigmoid", bias=torch.randn(experts, generator=gen).to(dev) * 0.1, n_groups=4,
                        topk_groups=2)
    lg = torch.randn((b * block, experts), generator=gen).to(dev)
    w, ids = router(lg, 4)
    rw, rids = omoe.route_experts(lg.cpu().numpy(), 4, score="sigmoid", bias=router.bias.cpu().numpy(), n_groups=4,
                                  topk_groups=2)
    np.testing.assert_array_equal(ids.cpu().numpy(), rids)
    out = moe.MoEPlanLayer(stacks, None, b * block, 4, router=router)(x, lg)
    again = moe.moe_layer(x, lg, stacks, None, 4, router=router)
    assert (out.float() - again.float()).abs().max() <= 2.0 ** -6 * again.float().abs().max()

    # logits of the block, drafts, uniforms
    head = torch.randn((vocab, h), generator=gen).to(dev)
    logits = (out.float() @ head.t() / out.float().std() / h ** 0.5 * 2).bfloat16().view(b, block, vocab)
    dl = (logits[:, :-1].float() + 0.5 * torch.randn((b, block - 1, vocab), generator=gen).to(dev)).bfloat16()
    vid = torch.cat([torch.zeros((b, 1), dtype=torch.int64, device=dev), dl.float().argmax(-1)], 1).to(torch.int32)
    u, us = torch.rand((b, block - 1), generator=gen) ** 3, torch.rand(b, generator=gen)
    acc, tok, prob = pkg.verify_accept_sampled(logits, vid, u.to(dev), us.to(dev), draft_logits=dl if draft else None,
                                               temperature=0.8)
    ref = osm.verify_accept_sampled(logits.float().cpu().numpy(), vid.cpu().numpy(), u.numpy(), us.numpy(),
                                    draft=dl.float().cpu().numpy() if draft else None,
                                    temperature=np.full(b, 0.8, np.float32))
    np.testing.assert_array_equal(acc.cpu().numpy(), ref[0])
    np.testing.assert_array_equal(tok.cpu().numpy(), ref[1])
    np.testing.assert_allclose(prob.cpu().numpy(), ref[2], rtol=1e-6, atol=1.2e-38)

    # back to the staged token and the accepted drafts
    cache.rollback(acc)
    for i in range(b):
        e = prompt + 1 + int(ref[0][i]) + 1
        one = tuple(a[i:i + 1, :e] for a in arrays[:5]) + (arrays[5][i:i + 1],)
        ry, rs = ogdn.gated_delta_rule(*one)
        _check(torch.from_numpy(ry), cache[1][i:i + 1], ry, rs, one, e)
