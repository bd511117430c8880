"""GPU parity of ``verify_accept_sampled`` with the definition in float64
(``oracle.sampled``).  Accepted lengths and ids are whole numbers and have to
be equal; the uniforms are kept 1e-5 of a probability away from every border
of an acceptance (the kernel's 32-bit sums of a row are good to about 1e-6)
and 1e-9 of the total away from every border of an id (64-bit sums).
draft_prob: one 32-bit sum and one division, 1e-6 of the value (V roundings
that do not all point one way, plus the exponentials' own 2 half steps), plus
the smallest normal number.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import sampled as osm

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _case(seed, b, t, v, dtype, draft, ragged=False, suppress=False, spread=3.0, cool=()):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    ru = lambda *s: torch.rand(s, generator=gen)  # noqa: E731
    dt = TYPES[dtype]
    logits = (rn(b, t, v) * spread).to(dt)
    dl = (logits[:, :-1].float() + rn(b, t - 1, v) * 0.7).to(dt)
    temp = 0.5 + ru(b)
    for i in cool:
        temp[i] = 0.0
    noise = -torch.log(-torch.log(ru(b, t - 1, v).clamp(1e-7, 1 - 1e-7)))
    ids = torch.zeros(b, t, dtype=torch.int32)
    ids[:, 0] = 1
    pick = (dl.float() / temp.clamp(min=0.1)[:, None, None] + noise) if draft else logits[:, :-1].float()
    if t > 1:
        ids[:, 1:] = pick.argmax(-1).to(torch.int32)
    case = dict(logits=logits, ids=ids, u=ru(b, t - 1) ** (1 if draft else 3), s=ru(b),
                draft=dl if draft and t > 1 else None, temp=temp,
                lens=torch.randint(0, t, (b,), generator=gen).to(torch.int32) if ragged else None,
                sup=(ru(v) < 0.1) if suppress else None)
    return case


def _np(x):
    return None if x is None else (x.float().numpy() if x.dtype in TYPES.values() else x.numpy())


def _ref(c):
    return osm.verify_accept_sampled(_np(c["logits"]), c["ids"].numpy(), c["u"].numpy(), c["s"].numpy(),
                                     draft=_np(c["draft"]), temperature=c["temp"].numpy(),
                                     lens=_np(c["lens"]), suppressed=_np(c["sup"]))


def _run(pkg, dev, c, **kw):
    to = lambda x: None if x is None else x.to(dev)  # noqa: E731
    return pkg.verify_accept_sampled(to(c["logits"]), to(c["ids"]), to(c["u"]), to(c["s"]),
                                     draft_logits=to(c["draft"]), temperature=to(c["temp"]),
                                     draft_lens=to(c["lens"]), suppress_token_mask=to(c["sup"]), **kw)


def _off_borders(c):
    """Uniforms moved off the borders by the margins named above (inputs are made
    so before any run)."""
    b, t, v = c["logits"].shape
    lg, dl = _np(c["logits"]), _np(c["draft"])
    for i in range(b):
        z = float(c["temp"][i])
        n = t - 1 if c["lens"] is None else int(c["lens"][i])
        for r in range(n):
            x = int(c["ids"][i, r + 1])
            if not (0 <= x < v):
                continue
            p = osm.distribution(lg[i, r], z, _np(c["sup"]))[x]
            q = 1.0 if dl is None or not z > 0 else osm.distribution(dl[i, r], z)[x]
            while q > 0 and abs(float(c["u"][i, r]) * q - p) < 1e-5 * p:
                c["u"][i, r] = (float(c["u"][i, r]) + 0.377) % 1.0
    for _ in range(20):
        acc, _, _ = _ref(c)
        near = False
        for i in range(b):
            z, a = float(c["temp"][i]), int(acc[i])
            n = t - 1 if c["lens"] is None else int(c["lens"][i])
            if not z > 0:
                continue
            w = osm.distribution(lg[i, a], z, _np(c["sup"]))
            if a < n:
                x = int(c["ids"][i, a + 1])
                q = (np.arange(v) == x).astype(float) if dl is None else osm.distribution(dl[i, a], z)
                left = np.maximum(w - q, 0.0)
                w = left if left.sum() > 0 else w
            cum = np.cumsum(w)
            if cum[-1] > 0 and np.abs(cum / cum[-1] - float(c["s"][i])).min() < 1e-9:
                c["s"][i] = (float(c["s"][i]) + 0.377) % 1.0
                near = True
        if not near:
            return c
    raise AssertionError("no uniforms off the borders")


def _same(got, ref):
    acc, tok, prob = (x.cpu().numpy() for x in got)
    np.testing.assert_array_equal(acc, ref[0])
    np.testing.assert_array_equal(tok, ref[1])
    assert acc.dtype == np.int32 and tok.dtype == np.int32 and prob.dtype == np.float32
    np.testing.assert_allclose(prob, ref[2], rtol=1e-6, atol=1.2e-38)


@pytest.mark.parametrize("b,t,v,dtype,draft,ragged,suppress", [
    (1, 1, 1, "fp32", False, False, False),
    (2, 1, 7, "bf16", False, False, False),
    (3, 2, 33, "fp16", True, False, False),
    (4, 16, 1000, "bf16", True, True, False),
    (4, 16, 1001, "bf16", False, True, True),
    (3, 5, 4096, "fp32", True, False, True),
    (3, 5, 4097, "fp16", True, True, True),
    (2, 16, 8191, "fp32", False, False, False),
    (5, 9, 50257, "bf16", True, True, True),
    (1, 16, 248320, "bf16", True, False, False),
    (1, 33, 30011, "fp16", False, False, False),
    (40, 3, 1555, "fp32", True, True, True),
])
def test_matches_the_definition(pkg, dev, b, t, v, dtype, draft, ragged, suppress):
    c = _off_borders(_case(b * 31 + t + v, b, t, v, dtype, draft, ragged, suppress))
    _same(_run(pkg, dev, c), _ref(c))


def test_greedy_rows_and_sampled_rows_in_one_batch(pkg, dev):
    c = _off_borders(_case(3, 6, 8, 3001, "bf16", True, True, True, cool=(0, 2, 5)))
    c["temp"][5] = -1.0
    _same(_run(pkg, dev, c), _ref(c))


def test_temperature_zero_is_greedy_acceptance(pkg, dev):
    """As ``match_acceptance_length`` on the argmax ids, ties to the lowest."""
    c = _case(4, 4, 16, 999, "bf16", False)
    c["logits"][1, 3] = 1.0   # all equal: id 0
    c["ids"][1, 4] = 0
    c["ids"][2, 5] = 998
    dev_logits = c["logits"].to(dev)
    acc, tok, prob = pkg.verify_accept_sampled(dev_logits, c["ids"].to(dev), c["u"].to(dev), c["s"].to(dev),
                                               temperature=0.0)
    best = c["logits"].float().argmax(-1).to(torch.int32)
    best[1, 3] = 0
    want = pkg.match_acceptance_length(c["ids"][:, 1:].to(dev), best[:, :-1].to(dev))
    assert torch.equal(acc, want)
    assert torch.equal(tok.cpu(), best[torch.arange(4), acc.cpu().long()])
    assert set(prob.cpu().unique().tolist()) <= {0.0, 1.0}


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_masked_places(pkg, dev, dtype):
    """-inf, NaN and the type's lowest value; infinities and NaN under the
    suppress mask; rows that leave nothing; drafts on ids that cannot be drawn."""
    c = _case(5, 8, 4, 5003, dtype, True, suppress=True)
    lg, dl = c["logits"], c["draft"]
    low = torch.finfo(TYPES[dtype]).min
    lg[0, :, 100:] = -torch.inf
    lg[1, :, 7] = torch.nan
    dl[1, :, 9] = torch.nan
    lg[2, :, 50:] = low
    lg[3, :] = low                 # all the lowest: uniform
    lg[4, 1] = -torch.inf          # nothing left in row 1
    lg[5, :, 1000:] = torch.nan
    lg[6, 2] = torch.nan           # nothing left in row 2
    lg[7, :, 11] = torch.inf       # spread over the ids that hold +inf
    lg[7, :, 4000] = torch.inf
    c["sup"][11] = c["sup"][4000] = False
    for x in (torch.nan, torch.inf, -torch.inf):
        where = torch.nonzero(c["sup"])[:, 0]
        lg[:7, :, where[torch.randperm(len(where))[:40]]] = x
    c["ids"][4, 1:] = 5
    c["u"][4] = 0.0
    c["ids"][6, 1:] = torch.nonzero(~c["sup"])[:3, 0].to(torch.int32)
    c["u"][6] = 0.0
    c["ids"][0, 2] = 3000
    c = _off_borders(c)
    got, ref = _run(pkg, dev, c), _ref(c)
    _same(got, ref)
    assert ref[1][4] == -1 or ref[0][4] == 0
    everything = torch.ones(5003, dtype=torch.bool)
    c["sup"] = everything
    acc, tok, prob = _run(pkg, dev, c)
    assert torch.all(acc == 0) and torch.all(tok == -1) and torch.all(prob == 0)


def test_ids_outside_the_vocabulary_and_bad_lengths(pkg, dev):
    from dflash_mlx_b200 import _lib

    assert _lib.device_error() == 0
    for draft in (False, True):
        c = _case(6, 4, 5, 257, "fp32", draft)
        c["ids"][0, 1], c["ids"][1, 2], c["ids"][2, 3] = -1, 257, 2**31 - 1
        c["u"][:3] = 0.0
        c = _off_borders(c)
        _same(_run(pkg, dev, c), _ref(c))
    assert _lib.device_error() == 0
    c["lens"] = torch.tensor([-3, 99, 2, 4], dtype=torch.int32)
    got = _run(pkg, dev, c)
    assert _lib.device_error() == 3
    c["lens"] = torch.tensor([0, 4, 2, 4], dtype=torch.int32)
    _same(got, _ref(c))


def test_ids_past_32_bits_are_outside_the_vocabulary(pkg, dev):
    c = _case(16, 3, 4, 101, "fp32", False)
    c["u"][:] = 0.0
    args = [c["logits"].to(dev), c["ids"].to(dev).long(), c["u"].to(dev), c["s"].to(dev)]
    args[1][0, 1] += 2**32
    args[1][1, 2] -= 2**33
    acc, _, prob = pkg.verify_accept_sampled(*args, temperature=c["temp"].to(dev).clamp(min=0.5))
    assert acc.tolist() == [0, 1, 3]
    assert prob[0, 0] == 0 and prob[1, 1] == 0 and prob[2].min() > 0


def test_uniforms_at_the_ends(pkg, dev):
    """u = 0 accepts whatever has a probability and draws the first such id;
    1 (outside the range), the last one; NaN draws as 0 and accepts nothing."""
    c = _case(7, 4, 3, 777, "fp32", False)
    c["logits"][:, :, :5] = -torch.inf
    c["logits"][:, :, 770:] = -torch.inf
    c["u"][:] = torch.tensor([0.0, 0.0])
    c["s"] = torch.tensor([0.0, 1.0, float("nan"), 2.0])
    acc, tok, _ = _run(pkg, dev, c)
    assert torch.all(acc == 2) and tok.tolist() == [5, 769, 5, 769]
    c["u"][:] = float("nan")
    assert torch.all(_run(pkg, dev, c)[0] == 0)


def test_temperatures_at_the_ends(pkg, dev):
    """Very high: uniform over what is not masked; very low: all on the largest."""
    v = 640
    c = _case(8, 4, 2, v, "fp32", False)
    c["logits"][:, :, v // 2:] = -torch.inf
    c["temp"] = torch.tensor([1e30, torch.inf, 1e-30, 1e-45])
    c["u"][:] = 1.0
    c["s"] = torch.tensor([0.5 + 1e-4, 0.25 + 1e-4, 0.5, 0.5])
    best = c["logits"][2:, 0].argmax(-1)
    c["ids"][2:, 1] = best.to(torch.int32)
    c["u"][2:] = 0.999
    acc, tok, prob = _run(pkg, dev, c)
    assert acc.tolist() == [0, 0, 1, 1]
    # the drafted id of a row may lie among the masked ones (it was picked before they were masked)
    want = [1.0 / 320 if int(i) < 320 else 0.0 for i in c["ids"][:2, 1]]
    np.testing.assert_allclose(prob.cpu()[:2, 0], want, rtol=1e-6)
    np.testing.assert_allclose(prob.cpu()[2:, 0], 1.0)
    left = [i for i in range(320) if i != int(c["ids"][0, 1])]
    assert int(tok[0]) == left[int(float(c["s"][0]) * len(left))]


def test_nothing_left_after_the_draft_falls_back_to_the_target(pkg, dev):
    """p equal to q and a draft that q cannot give: max(p - q, 0) is empty."""
    c = _case(9, 2, 3, 500, "fp32", True)
    c["draft"] = c["logits"][:, :-1].clone()
    c["logits"][:, :, 3] = c["draft"][:, :, 3] = -torch.inf
    c["ids"][:, 1:] = 3
    c = _off_borders(c)
    ref = _ref(c)
    assert np.all(ref[0] == 0) and np.all(ref[1] >= 0)
    _same(_run(pkg, dev, c), ref)


def test_committed_tokens_follow_the_target(pkg, dev):
    """First committed token (draft or replacement) over many requests: within 5
    standard deviations of the target's probabilities for every id."""
    b, v = 20000, 12
    gen = torch.Generator(device=dev).manual_seed(1)
    one = torch.randn((1, 2, v), generator=gen, device=dev)
    dl = torch.randn((1, 1, v), generator=gen, device=dev)
    q = torch.softmax(dl[0, 0], -1)
    x = torch.multinomial(q.expand(b, v), 1, generator=gen).to(torch.int32)
    ids = torch.cat([torch.zeros_like(x), x], 1)
    acc, tok, _ = pkg.verify_accept_sampled(one.expand(b, 2, v), ids, torch.rand((b, 1), generator=gen, device=dev),
                                            torch.rand((b,), generator=gen, device=dev),
                                            draft_logits=dl.expand(b, 1, v))
    first = torch.where(acc > 0, x[:, 0], tok)
    freq = torch.bincount(first, minlength=v).double().cpu() / b
    p = torch.softmax(one[0, 0].double(), -1).cpu()
    assert torch.all((freq - p).abs() <= 5 * torch.sqrt(p * (1 - p) / b))


def test_views_streams_and_graphs(pkg, dev):
    """Rows of a larger buffer, vocabulary slices at odd offsets, a side stream,
    two captured graphs replayed at once, new inputs in the same buffers."""
    c = _off_borders(_case(10, 3, 6, 2003, "bf16", True, True, True))
    ref = _ref(c)
    want = _run(pkg, dev, c)
    _same(want, ref)
    wide = torch.full((3, 9, 2011), float("nan"), dtype=torch.bfloat16, device=dev)
    wide[:, 2:8, 3:2006] = c["logits"].to(dev)
    dwide = torch.full((3, 9, 2011), float("nan"), dtype=torch.bfloat16, device=dev)
    dwide[:, 1:6, 5:2008] = c["draft"].to(dev)
    args = [wide[:, 2:8, 3:2006], c["ids"].to(dev), c["u"].to(dev), c["s"].to(dev)]
    kw = dict(draft_logits=dwide[:, 1:6, 5:2008], temperature=c["temp"].to(dev), draft_lens=c["lens"].to(dev),
              suppress_token_mask=c["sup"].to(dev))
    _same(pkg.verify_accept_sampled(*args, **kw), ref)
    _same(pkg.verify_accept_sampled(args[0].transpose(1, 2).contiguous().transpose(1, 2), *args[1:], **kw), ref)
    torch.cuda.synchronize()
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    graphs, got = [], []
    with torch.cuda.stream(side):
        got.append(pkg.verify_accept_sampled(*args, **kw))
        side.synchronize()
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                got.append(pkg.verify_accept_sampled(*args, **kw))
            graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(3):
        graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
    torch.cuda.synchronize()
    for x in got:
        _same(x, ref)


def test_refusals(pkg, dev):
    c = _case(11, 2, 4, 100, "bf16", True, True, True)
    to = {k: (x.to(dev) if x is not None else None) for k, x in c.items()}

    def call(**kw):
        a = {**to, **kw}
        return pkg.verify_accept_sampled(a["logits"], a["ids"], a["u"], a["s"], draft_logits=a["draft"],
                                         temperature=a["temp"], draft_lens=a["lens"],
                                         suppress_token_mask=a["sup"])

    call()
    with pytest.raises(ValueError, match="CUDA"):
        call(logits=c["logits"])
    with pytest.raises(ValueError, match="CUDA"):
        call(u=c["u"])
    with pytest.raises(NotImplementedError):
        call(logits=to["logits"].double())
    for kw in (dict(logits=to["logits"][0]), dict(ids=to["ids"][:, :3]), dict(ids=to["ids"].float()),
               dict(u=to["u"][:, :2]), dict(u=to["u"].double()), dict(s=to["s"][:1]),
               dict(draft=to["draft"].float()), dict(draft=to["draft"][:, :2]), dict(temp=-0.5),
               dict(temp=float("nan")), dict(temp=to["temp"].double()), dict(temp=to["temp"][:1]),
               dict(lens=to["lens"].long()), dict(lens=to["lens"][:1]), dict(sup=to["sup"][:99]),
               dict(sup=to["sup"].float())):
        with pytest.raises(ValueError):
            call(**kw)
    empty = pkg.verify_accept_sampled(to["logits"][:0], to["ids"][:0], to["u"][:0], to["s"][:0])
    assert [tuple(x.shape) for x in empty] == [(0,), (0,), (0, 3)]
