"""Cases of the operators around the verify step, for measurement: the gated
delta rule over whole prompts and single tokens, the sampled verification of
drafted tokens, and the routing of tokens to experts.

``listed()`` and ``draw()`` give cases, ``prepare()`` their inputs, ``run()``
one pass (the plain torch form, or the framework's kernels where ``own`` is
set), ``work()`` the bytes and operations that a pass cannot do without and
``exact()`` the results from the definitions in 64 bits.
"""

import math

import torch

own = False

DEV = "cuda"


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one request's next token in a decoder layer of 48 value heads on 16 key heads
        dict(name="gdn_token_1", op="gdn", lens="1", hk=16, hv=48, dk=128, dv=128, packed=True),
        # the next token of 40 requests at once
        dict(name="gdn_tokens_40", op="gdn", lens=",".join(["1"] * 40), hk=16, hv=48, dk=128, dv=128,
             packed=True),
        # a few short prompts of odd lengths packed one after the other, one of them a single token
        dict(name="gdn_short_packed", op="gdn", lens="217,64,1,130,399", hk=16, hv=48, dk=128, dv=128,
             packed=True),
        # a left-padded batch with its mask, smaller heads
        dict(name="gdn_padded_mask", op="gdn", lens="1000,517,3", hk=8, hv=8, dk=64, dv=64, packed=False),
        # one long prompt
        dict(name="gdn_prompt_8k", op="gdn", lens="8192", hk=16, hv=48, dk=128, dv=128, packed=True),
        # prompts of several requests prefilled together
        dict(name="gdn_prompts_packed", op="gdn", lens="4096,2049,1500,777,5000,64,300,2100", hk=16, hv=48,
             dk=128, dv=128, packed=True),
        # one request's block of a staged token and 15 greedy drafts
        dict(name="verify_1", op="verify", b=1, t=16, v=248320, draft=False, dtype="bf16", ragged=False),
        # a batch of requests of several draft lengths with the draft model's logits
        dict(name="verify_draft_8", op="verify", b=8, t=16, v=248320, draft=True, dtype="bf16", ragged=True),
        # many requests with the draft model's logits
        dict(name="verify_draft_48", op="verify", b=48, t=16, v=248320, draft=True, dtype="bf16",
             ragged=False),
        # the block of one verify step, softmax scores
        dict(name="route_16", op="route", t=16, e=256, k=8, score="softmax", bias=False, groups=1,
             topk_groups=1, dtype="fp32"),
        # the same block, sigmoid scores with a balance bias, 4 of 8 groups
        dict(name="route_16_groups", op="route", t=16, e=256, k=8, score="sigmoid", bias=True, groups=8,
             topk_groups=4, dtype="fp32"),
        # a prompt's tokens
        dict(name="route_8191_groups", op="route", t=8191, e=256, k=8, score="sigmoid", bias=True, groups=8,
             topk_groups=4, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gdn", "gdn", "verify", "route"])
    if op == "gdn":
        kind = rng.choice(["tokens", "prompts", "padded"])
        dk = rng.choice([64, 128, 128])
        dv = rng.choice([64, 128, 128])
        hk = rng.choice([4, 8, 16])
        hv = hk * rng.choice([1, 2, 3])
        if kind == "tokens":
            lens = [1] * _log_int(rng, 1, 40)
        elif kind == "prompts":
            lens = [_log_int(rng, 2, 8000) for _ in range(rng.randint(1, 6))]
        else:
            lens = [_log_int(rng, 1, 2000) for _ in range(rng.randint(2, 5))]
        while sum(lens) > 15000:
            lens.pop()
        return dict(op=op, lens=",".join(map(str, lens)), hk=hk, hv=hv, dk=dk, dv=dv,
                    packed=kind != "padded")
    if op == "verify":
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        return dict(op=op, b=_log_int(rng, 1, 20 if dtype == "fp32" else 40), t=rng.randint(1, 16),
                    v=_log_int(rng, 1001, 248320), draft=rng.random() < 0.5, dtype=dtype,
                    ragged=rng.random() < 0.5)
    groups = rng.choice([1, 4, 8])
    k = rng.randint(1, 10)
    e = groups * _log_int(rng, 10, 64)
    return dict(op=op, t=_log_int(rng, 1, 8000), e=e, k=k, score=rng.choice(["softmax", "sigmoid"]),
                bias=rng.random() < 0.5, groups=groups, topk_groups=rng.randint((groups + 1) // 2, groups),
                dtype=rng.choice(["fp32", "bf16"]))


_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _lens(case):
    return [int(x) for x in case["lens"].split(",")]


# ----------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    rn = lambda *s: torch.randn(s, generator=gen, device=DEV)  # noqa: E731
    ru = lambda *s: torch.rand(s, generator=gen, device=DEV)  # noqa: E731
    st = {"case": dict(case)}
    if case["op"] == "gdn":
        lens, hk, hv, dk, dv = _lens(case), case["hk"], case["hv"], case["dk"], case["dv"]
        n = len(lens)
        b, t = (1, sum(lens)) if case["packed"] else (n, max(lens))
        unit = lambda x: x / x.norm(dim=-1, keepdim=True)  # noqa: E731
        # queries and keys of unit length (queries scaled by Dk^-0.5), values N(0, 1), a decay per head
        # from nearly none to about a half a step, states as they stand in the middle of a text
        st["q"] = (unit(rn(b, t, hk, dk)) / math.sqrt(dk)).to(torch.bfloat16)
        st["k"] = unit(rn(b, t, hk, dk)).to(torch.bfloat16)
        st["v"] = rn(b, t, hv, dv).to(torch.bfloat16)
        rate = torch.exp(ru(hv) * math.log(50.0)) * 0.02
        st["g"] = torch.exp(-rate * torch.nn.functional.softplus(rn(b, t, hv)))
        st["beta"] = torch.sigmoid(rn(b, t, hv))
        st["state"] = rn(n, hv, dv, dk) * 0.05
        st["cu"] = st["mask"] = None
        if case["packed"]:
            ends = [0]
            for x in lens:
                ends.append(ends[-1] + x)
            st["cu"] = torch.tensor(ends, dtype=torch.int32, device=DEV)
        else:
            first = torch.tensor([t - x for x in lens], device=DEV)
            st["mask"] = torch.arange(t, device=DEV)[None, :] >= first[:, None]
    elif case["op"] == "verify":
        b, t, v, dt = case["b"], case["t"], case["v"], _TYPES[case["dtype"]]
        st["logits"] = torch.empty((b, t, v), dtype=dt, device=DEV)
        st["draft_logits"] = torch.empty((b, t - 1, v), dtype=dt, device=DEV) if case["draft"] else None
        st["temperature"] = 0.6 + 0.6 * ru(b)
        ids = torch.randint(0, v, (b, t), generator=gen, device=DEV)
        for i in range(b):
            target = rn(t, v) * 3.0
            st["logits"][i] = target
            # the drafts: the draft model's own samples, or its greedy tokens
            draft = target[:-1] + rn(t - 1, v) * 0.7
            if case["draft"]:
                st["draft_logits"][i] = draft
                noise = -torch.log(-torch.log(ru(t - 1, v).clamp(1e-7, 1 - 1e-7)))
                ids[i, 1:] = (st["draft_logits"][i].float() / st["temperature"][i] + noise).argmax(-1)
            else:
                ids[i, 1:] = draft.argmax(-1)
        st["ids"] = ids.to(torch.int32)
        st["accept_u"], st["sample_u"] = ru(b, t - 1), ru(b)
        if not case["draft"]:
            st["accept_u"] = st["accept_u"] ** 6
        st["lens"] = torch.randint(0, t, (b,), generator=gen, device=DEV).to(torch.int32) if case["ragged"] else None
        # control tokens that are never to be written
        st["suppress"] = torch.arange(v, device=DEV) >= v - max(1, v // 200)
    else:
        t, e = case["t"], case["e"]
        st["logits"] = (rn(t, e) * 1.5).to(_TYPES[case["dtype"]])
        st["bias"] = rn(e) * 0.05 if case["bias"] else None
    return st


# ------------------------------------------------------------ plain forms
_CHUNK = 64


def _rows_of(st):
    """The inputs as [sequences, heads, steps, ...] in 32 bits, steps of no sequence as steps that change nothing."""
    c = st["case"]
    lens, rep = _lens(c), c["hv"] // c["hk"]
    t = max(lens)
    pad = -t % _CHUNK
    rows, keep = [], None
    if c["packed"]:
        at = torch.arange(t + pad, device=DEV)[None, :]
        ln = (st["cu"][1:] - st["cu"][:-1])[:, None]
        keep = at < ln
        idx = torch.where(keep, st["cu"][:-1, None] + at, 0).long()
        pick = lambda x: x[0][idx]  # noqa: E731
    else:
        keep = torch.nn.functional.pad(st["mask"], (0, pad))
        pick = lambda x: torch.nn.functional.pad(x, [0, 0] * (x.dim() - 2) + [0, pad])  # noqa: E731
    for name in ("q", "k", "v", "g", "beta"):
        x = pick(st[name]).float()
        x = torch.where(keep.view(*keep.shape, *[1] * (x.dim() - 2)), x, 1.0 if name == "g" else 0.0)
        if name in ("q", "k"):
            x = x.repeat_interleave(rep, dim=2)
        rows.append(x.transpose(1, 2))
    return rows, keep


def _rows_back(st, y, keep):
    """[sequences, heads, steps, Dv] as the outputs are laid out."""
    c = st["case"]
    y = y.transpose(1, 2)
    if c["packed"]:
        return y[keep][None]
    return torch.where(keep[..., None, None], y, 0.0)[:, : st["q"].shape[1]]


def _plain_gdn(st):
    (q, k, v, g, beta), keep = _rows_of(st)
    s = st["state"]
    n = q.shape[2] // _CHUNK
    cut = lambda x: x.reshape(*x.shape[:2], n, _CHUNK, *x.shape[3:])  # noqa: E731
    q, k, v, g, beta = map(cut, (q, k, v, g, beta))
    logs = torch.cumsum(torch.log(g.double()), dim=-1)
    i = torch.arange(_CHUNK, device=DEV)
    low = i[:, None] >= i[None, :]
    decay = torch.exp(torch.where(low, logs[..., :, None] - logs[..., None, :], -math.inf)).float()
    since = torch.exp(logs).float()
    until = torch.exp(logs[..., -1:] - logs).float()
    a = beta[..., None] * decay * (k @ k.transpose(-1, -2)) * (i[:, None] > i[None, :])
    eye = torch.eye(_CHUNK, device=DEV)
    p = decay * (q @ k.transpose(-1, -2))
    y = torch.empty_like(v)
    for c in range(n):
        r = beta[:, :, c, :, None] * (v[:, :, c] - since[:, :, c, :, None] * (k[:, :, c] @ s.transpose(-1, -2)))
        d = torch.linalg.solve_triangular(eye + a[:, :, c], r, upper=False, unitriangular=True)
        y[:, :, c] = since[:, :, c, :, None] * (q[:, :, c] @ s.transpose(-1, -2)) + p[:, :, c] @ d
        s = since[:, :, c, -1, None, None] * s + (until[:, :, c, :, None] * d).transpose(-1, -2) @ k[:, :, c]
    y = y.reshape(*y.shape[:2], n * _CHUNK, y.shape[-1])
    return {"y": _rows_back(st, y, keep).to(torch.bfloat16), "state": s}


def _softmax(x, temperature):
    # 64 bits: an accepted length and a sampled id turn on values next to a border
    x = x.double()
    x = torch.exp((x - x.amax(dim=-1, keepdim=True)) / temperature)
    return x / x.sum(dim=-1, keepdim=True)


def _plain_verify(st):
    c = st["case"]
    b, t = c["b"], c["t"]
    rows = torch.arange(b, device=DEV)
    temp = st["temperature"].double()
    p = torch.empty((b, t, c["v"]), dtype=torch.float64, device=DEV)
    q = None if st["draft_logits"] is None else torch.empty((b, t - 1, c["v"]), dtype=torch.float64, device=DEV)
    hidden = st["suppress"]
    for i in range(b):
        p[i] = _softmax(torch.where(hidden, -math.inf, st["logits"][i].float()), temp[i])
        if q is not None:
            q[i] = _softmax(st["draft_logits"][i], temp[i])
    ids = st["ids"][:, 1:].long()
    lens = st["lens"] if st["lens"] is not None else torch.full((b,), t - 1, device=DEV)
    px = p[:, :-1].gather(-1, ids[..., None])[..., 0]
    qx = torch.ones_like(px) if q is None else q.gather(-1, ids[..., None])[..., 0]
    inside = torch.arange(t - 1, device=DEV)[None, :] < lens[:, None]
    ok = (st["accept_u"].double() * qx < px) & inside
    n = torch.cumprod(ok.to(torch.int32), dim=1).sum(dim=1)
    left = p[rows, n]
    if t > 1:
        at = n.clamp(max=t - 2)
        if q is None:
            drawn = torch.zeros_like(left).scatter_(1, ids[rows, at][:, None], 1.0)
        else:
            drawn = q[rows, at]
        left = torch.where((n < lens)[:, None], (left - drawn).clamp(min=0.0), left)
    cdf = torch.cumsum(left, dim=-1)
    token = (cdf <= st["sample_u"].double()[:, None] * cdf[:, -1:]).sum(dim=-1)
    return {"accepted": n.to(torch.int32), "token": token.to(torch.int32),
            "draft_prob": torch.where(inside, px, 0.0).float()}


def _plain_route(st):
    c = st["case"]
    # 64 bits: which experts are kept turns on values next to a border
    x = st["logits"].double()
    s = torch.sigmoid(x) if c["score"] == "sigmoid" else _softmax(x, 1.0)
    choice = s if st["bias"] is None else s + st["bias"].double()
    if c["groups"] > 1:
        by = choice.reshape(c["t"], c["groups"], -1)
        score = by.sort(dim=-1, descending=True)[0][..., : 2 if c["score"] == "sigmoid" else 1].sum(-1)
        order = score.sort(dim=-1, descending=True, stable=True)[1][:, : c["topk_groups"]]
        kept = torch.zeros_like(score, dtype=torch.bool).scatter_(1, order, True)
        choice = torch.where(kept[..., None], by, -math.inf).reshape(c["t"], -1)
    ids = choice.sort(dim=-1, descending=True, stable=True)[1][:, : c["k"]]
    w = s.gather(1, ids)
    w = w / w.sum(dim=-1, keepdim=True)
    return {"weights": w.float(), "ids": ids.to(torch.int32)}


# ------------------------------------------------------------------- run
def run(state):
    c = state["case"]
    if own:
        import __graft_entry__

        pkg = __graft_entry__.load_package()
        if c["op"] == "gdn":
            y, s = pkg.gated_delta_rule(state["q"], state["k"], state["v"], state["g"], state["beta"],
                                        state["state"], mask=state["mask"], cu_seqlens=state["cu"])
            return {"y": y, "state": s}
        if c["op"] == "verify":
            n, token, prob = pkg.verify_accept_sampled(
                state["logits"], state["ids"], state["accept_u"], state["sample_u"],
                draft_logits=state["draft_logits"], temperature=state["temperature"],
                draft_lens=state["lens"], suppress_token_mask=state["suppress"])
            return {"accepted": n, "token": token, "draft_prob": prob}
        w, ids = pkg.route_experts(state["logits"], c["k"], score=c["score"], bias=state["bias"],
                                   n_groups=c["groups"], topk_groups=c["topk_groups"])
        return {"weights": w, "ids": ids}
    if c["op"] == "gdn":
        return _plain_gdn(state)
    if c["op"] == "verify":
        return _plain_verify(state)
    return _plain_route(state)


# ------------------------------------------------------------------ work
def work(case):
    if case["op"] == "gdn":
        lens, hk, hv, dk, dv = _lens(case), case["hk"], case["hv"], case["dk"], case["dv"]
        tokens = sum(lens)
        per = 2 * (2 * hk * dk + 2 * hv * dv) + 8 * hv
        # three products of the state's size per token and head: S k, the rank-one update, S q
        return {"bytes": tokens * per + 8 * len(lens) * hv * dv * dk, "flops": 6 * tokens * hv * dk * dv}
    if case["op"] == "verify":
        size = 4 if case["dtype"] == "fp32" else 2
        # a request of a draft length that is drawn has about half its rows
        drafts = case["b"] * (case["t"] - 1) / (2 if case["ragged"] else 1)
        rows = case["b"] + drafts * (2 if case["draft"] else 1)
        return {"bytes": int(rows * case["v"] * size) + case["v"], "flops": int(rows * case["v"] * 3)}
    size = 4 if case["dtype"] == "fp32" else 2
    return {"bytes": case["t"] * (case["e"] * size + 8 * case["k"]), "flops": case["t"] * case["e"] * 4}


# ----------------------------------------------------------------- exact
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "gdn":
        return _exact_gdn(case, st)
    if case["op"] == "verify":
        return _exact_verify(case, st)
    return _exact_route(case, st)


def _exact_gdn(case, st):
    """The recurrence, step by step, over all sequences that still have one."""
    lens, rep = _lens(case), case["hv"] // case["hk"]
    s = st["state"].double()
    y = torch.zeros(st["v"].shape, dtype=torch.float64, device=DEV)
    order = sorted(range(len(lens)), key=lambda i: -lens[i])
    starts = [sum(lens[:i]) for i in range(len(lens))] if case["packed"] else [max(lens) - x for x in lens]
    for step in range(max(lens)):
        live = [i for i in order if lens[i] > step]
        if case["packed"]:
            at = (0, torch.tensor([starts[i] + step for i in live], device=DEV))
        else:
            at = (torch.tensor(live, device=DEV), torch.tensor([starts[i] + step for i in live], device=DEV))
        pos = torch.tensor(live, device=DEV)
        cur = s[pos]
        q = st["q"][at].double().repeat_interleave(rep, dim=1)[..., None]
        k = st["k"][at].double().repeat_interleave(rep, dim=1)[..., None]
        cur = cur * st["g"][at].double()[..., None, None]
        d = st["beta"][at].double()[..., None, None] * (st["v"][at].double()[..., None] - cur @ k)
        cur = cur + d @ k.transpose(-1, -2)
        y[at] = (cur @ q)[..., 0]
        s[pos] = cur
    return {"y": y, "state": s}


def _exact_verify(case, st):
    b, t = case["b"], case["t"]
    accepted, tokens = [], []
    prob = torch.zeros((b, t - 1), dtype=torch.float64, device=DEV)
    for i in range(b):
        z = st["temperature"][i].double()
        have = t - 1 if st["lens"] is None else int(st["lens"][i])
        draw_of = None

        def target(r):
            x = st["logits"][i, r].double() / z
            x[st["suppress"]] = -math.inf
            return torch.exp(x - torch.logsumexp(x, 0))

        for r in range(have):
            prob[i, r] = target(r)[int(st["ids"][i, r + 1])]
        n = 0
        while n < have:
            x = int(st["ids"][i, n + 1])
            if st["draft_logits"] is None:
                draw_of = torch.zeros(case["v"], dtype=torch.float64, device=DEV)
                draw_of[x] = 1.0
            else:
                draw_of = st["draft_logits"][i, n].double() / z
                draw_of = torch.exp(draw_of - torch.logsumexp(draw_of, 0))
            if not float(st["accept_u"][i, n]) * float(draw_of[x]) < float(prob[i, n]):
                break
            n += 1
        rest = target(n)
        if n < have:
            rest = torch.clamp(rest - draw_of, min=0.0)
        cdf = torch.cumsum(rest, 0)
        border = float(st["sample_u"][i]) * cdf[-1]
        accepted.append(n)
        tokens.append(int(torch.nonzero(cdf > border)[0]))
    whole = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    return {"accepted": whole(accepted), "token": whole(tokens), "draft_prob": prob}


def _exact_route(case, st):
    x = st["logits"].double()
    t, e = x.shape
    if case["score"] == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-x))
    else:
        s = torch.exp(x - torch.logsumexp(x, -1, keepdim=True))
    choice = s.clone()
    if st["bias"] is not None:
        choice += st["bias"].double()
    rows = torch.arange(t, device=DEV)
    if case["groups"] > 1:
        size = e // case["groups"]
        by = choice.view(t, case["groups"], size)
        first, at = by.max(-1)
        score = first.clone()
        if case["score"] == "sigmoid" and size > 1:
            score += by.scatter(-1, at[..., None], -math.inf).max(-1)[0]
        open_ = torch.full_like(choice, -math.inf).view(t, case["groups"], size)
        for _ in range(case["topk_groups"]):
            best = score.argmax(-1)
            open_[rows, best] = by[rows, best]
            score[rows, best] = -math.inf
        choice = open_.view(t, e)
    ids = []
    for _ in range(case["k"]):
        best = choice.argmax(-1)
        ids.append(best)
        choice[rows, best] = -math.inf
    ids = torch.stack(ids, 1)
    w = s.gather(1, ids)
    return {"weights": w / w.sum(-1, keepdim=True), "ids": ids.to(torch.int32)}
