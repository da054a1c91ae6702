"""Workloads of the operators around a paged generation cache: rotary positions, per-head norms with the rotation, block
tables and slot maps, rows into the pages, and one new token's attention over them.

Every case has a ``kind``:

  rotary   ``rotary_embedding`` of one tensor, with its gradient where ``train``
  norm     ``qk_norm_rotary`` of queries and keys, with all its gradients where ``train``
  tables   ``page_tables``: pages for the new tokens of every request, and where each token goes
  update   ``paged_update``: keys, values and gates of a packed batch of tokens into the cache
  attend   ``paged_forgetting_attention``: one query per request against its pages

The plain forms below are elementary torch operations in 32 bits (angles and sums of gates in 64), rounded once.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # a decoding step of a small batch: one token each, the whole head rotated in halves, far positions
        dict(name="rotary_step_t16_h24_d64", kind="rotary", train=False, B=1, T=16, H=24, D=64, rot=64, dtype="bf16",
             interleaved=False, head_first=False, far=1000000),
        # one tensor of the long-context training shape, forward and backward
        dict(name="rotary_train_t16384_h24_d64", kind="rotary", train=True, B=2, T=16384, H=24, D=64, rot=64, dtype="bf16",
             interleaved=False, head_first=False, far=0),
        # a part of the head, neighbouring channels paired, odd length, head-first
        dict(name="rotary_train_part_t2047_fp16", kind="rotary", train=True, B=3, T=2047, H=12, D=128, rot=32, dtype="fp16",
             interleaved=True, head_first=True, far=5000),
        # a decoding step: queries and keys of 8 requests at their own positions
        dict(name="norm_step_t8_h16_d128", kind="norm", train=False, B=1, T=8, H=16, Hk=16, D=128, rot=128, dtype="bf16",
             interleaved=False, shared=False, far=1000000),
        # queries and keys of a training layer, with the gradients of both and of the norms' weights
        dict(name="norm_train_t8192_h16_d128", kind="norm", train=True, B=2, T=8192, H=16, Hk=16, D=128, rot=128,
             dtype="bf16", interleaved=False, shared=False, far=0),
        # a step's bookkeeping of a serving batch: one token for most requests, none for some
        dict(name="tables_step_r256", kind="tables", R=256, most_old=8192, most_new=1, page=16),
        # prompts of very different lengths taken into the cache together
        dict(name="tables_prompts_r500", kind="tables", R=500, most_old=512, most_new=4096, page=64),
        # a step's rows: one token for each of 61 requests
        dict(name="update_step_t61_h16_d128", kind="update", T=61, H=16, Hk=16, D=128, page=16, pages=4096, dtype="bf16",
             logits=False),
        # the rows of long prompts, from the gates' logits
        dict(name="update_prompts_t30000_h24_d64", kind="update", T=30000, H=24, Hk=24, D=64, page=64, pages=1024,
             dtype="bf16", logits=True),
        # one request of a few hundred tokens: a step here is latency
        dict(name="attend_one_n500_h12_d64", kind="attend", R=1, shortest=500, longest=500, idle=0, H=12, Hk=12, D=64, page=16,
             dtype="bf16", mu=3.0),
        # a serving batch: lengths from a few tokens to thousands, some places without a request
        dict(name="attend_ragged_r48_h16_d128", kind="attend", R=48, shortest=7, longest=8000, idle=3, H=16, Hk=16, D=128, page=32,
             dtype="bf16", mu=4.0),
        # two very long requests, queries in groups that share keys and values
        dict(name="attend_long_n65000_h32_k8_d64", kind="attend", R=2, shortest=64999, longest=65536, idle=0, H=32, Hk=8, D=64,
             page=64, dtype="fp16", mu=6.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "norm", "tables", "update", "attend", "attend"])
    D = rng.choice([64, 64, 128, 128, 32, 16])
    H = rng.choice([4, 7, 8, 12, 16, 24, 32])
    dtype = rng.choice(["bf16", "fp16"])
    page = rng.choice([16, 32, 64, 128])
    groups = rng.choice([g for g in (1, 1, 2, 4, 7, 8, 16) if H % g == 0])
    if kind in ("rotary", "norm"):
        train = rng.random() < 0.6
        B = rng.choice([1, 2, 3])
        heads = H if kind == "rotary" else H + H // groups
        T = min(_log(rng, 1, 16384), 65_000_000 // (B * heads * D))
        rot = rng.choice([D, D, D // 2, 2 * rng.randint(1, D // 2)])
        c = dict(kind=kind, train=train, B=B, T=T, H=H, D=D, rot=rot, dtype=dtype, interleaved=rng.random() < 0.5,
                 far=rng.choice([0, 5000, 1000000]))
        if kind == "rotary":
            return dict(c, head_first=rng.random() < 0.5)
        return dict(c, Hk=H // groups, shared=rng.random() < 0.5)
    if kind == "tables":
        R = _log(rng, 1, 1000)
        return dict(kind=kind, R=R, most_old=_log(rng, 1, 8192), most_new=_log(rng, 1, max(1, 400000 // R)), page=page)
    if kind == "update":
        T = _log(rng, 1, 30000)
        return dict(kind=kind, T=T, H=H, Hk=H // groups, D=D, page=page, pages=T // page + rng.randint(2, 500), dtype=dtype,
                    logits=rng.random() < 0.5)
    R = _log(rng, 1, 200)
    longest = min(_log(rng, 1, 65536), max(1, 140_000_000 // (R * max(H // groups, 2) * D)))
    shortest = rng.randint(1, longest)
    return dict(kind=kind, R=R, shortest=shortest, longest=longest, idle=rng.randint(0, R // 8), H=H, Hk=H // groups, D=D, page=page,
                dtype=dtype, mu=rng.uniform(-1.0, 6.0))


# ------------------------------------------------------------------ inputs
def _lengths(case):
    """Lengths of the requests: from the shortest to the longest by equal factors, and places without a request."""
    n = case["R"] - case["idle"]
    a, b = case["shortest"], case["longest"]
    return [int(round(a * (b / a) ** (i / max(1, n - 1)))) for i in range(n)] + [0] * case["idle"]


def _old_new(case):
    """Tokens in the cache and new tokens of every request: the old by equal steps, the new by equal factors, every ninth
    request with nothing new."""
    R = case["R"]
    old = [(i * 7919) % (case["most_old"] + 1) for i in range(R)]
    new = [0 if i % 9 == 8 else int(round(case["most_new"] ** (((i * 31) % R) / max(1, R - 1)))) for i in range(R)]
    return old, new


def _pages(n, page):
    return -(-n // page)


def _frequencies(rot, dev):
    return torch.pow(10000.0, -torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot).float()


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    def order(n):
        return torch.randperm(n, generator=g, device=dev)

    kind = case["kind"]
    s = {"case": case}
    if kind in ("rotary", "norm"):
        dt, B, T, H, D = DTYPES[case["dtype"]], case["B"], case["T"], case["H"], case["D"]
        s["inv_freq"] = _frequencies(case["rot"], dev)
        # packed requests sit at positions of their own; a training batch counts from zero
        s["positions"] = (torch.randint(0, case["far"] + 1, (T,), generator=g, device=dev, dtype=torch.int32) if case["far"]
                          else torch.arange(T, device=dev, dtype=torch.int32))
    if kind == "rotary":
        shape = (B, H, T, D) if case["head_first"] else (B, T, H, D)
        s["x"] = randn(*shape).to(dt)
        if case["train"]:
            s["x"].requires_grad_()
            s["dy"] = randn(*shape).to(dt)
    elif kind == "norm":
        # q and k as the projections leave them: slices of one row
        Hk = case["Hk"]
        qkv = randn(B, T, (H + Hk) * D).to(dt)
        s["q"] = qkv[:, :, :H * D].view(B, T, H, D)
        s["k"] = qkv[:, :, H * D:].view(B, T, Hk, D)
        s["q_weight"] = 1 + 0.3 * randn(D if case["shared"] else H * D)
        s["k_weight"] = 1 + 0.3 * randn(D if case["shared"] else Hk * D)
        if case["train"]:
            s["leaves"] = [s[n].requires_grad_() for n in ("q", "k", "q_weight", "k_weight")]
            s["dq"], s["dk"] = randn(B, T, H, D).to(dt), randn(B, T, Hk, D).to(dt)
    elif kind == "tables":
        old, new = _old_new(case)
        R, page = case["R"], case["page"]
        perm = order(R).cpu()
        old, new = torch.tensor(old)[perm], torch.tensor(new)[perm]
        have = (old + page - 1) // page
        need = (old + new + page - 1) // page - have
        width = int((have + need).max()) + 2
        total = int((have + need).sum()) + 100
        pages = order(total).int()
        s["free_pages"] = pages                                  # a stack: the last num_free of them are taken first
        s["num_free"] = torch.tensor([total - int(have.sum())], dtype=torch.int32, device=dev)
        at = torch.arange(width)[None, :] < have[:, None]
        table = torch.full((R, width), -1, dtype=torch.int32)
        table[at] = pages.cpu()[total - int(have.sum()):]
        s["block_table"] = table.to(dev)
        s["lengths"], s["new"] = old.int().to(dev), new.int().to(dev)
        s["max_tokens"] = int(new.sum()) + R                      # some room behind the last token
    elif kind == "update":
        dt, T, H, Hk, D, P, page = DTYPES[case["dtype"]], case["T"], case["H"], case["Hk"], case["D"], case["pages"], case["page"]
        s["k_pages"], s["v_pages"] = randn(P, Hk, page, D).to(dt), randn(P, Hk, page, D).to(dt)
        s["gate_pages"] = -randn(P, H, page).abs()
        s["k"], s["v"] = randn(T, Hk, D).to(dt), randn(T, Hk, D).to(dt)
        s["gates"] = (randn(T, H) + 4).to(dt) if case["logits"] else torch.nn.functional.logsigmoid(randn(T, H) + 4)
        # a page's rows in their order, pages in any; the last tokens of the batch are padding
        t = torch.arange(T, device=dev)
        s["slots"] = (order(P)[t // page] * page + t % page).int()
        s["slots"][T - T // 16:] = -1
    else:
        dt, R, H, Hk, D, page = DTYPES[case["dtype"]], case["R"], case["H"], case["Hk"], case["D"], case["page"]
        lengths = torch.tensor(_lengths(case))[order(R).cpu()]
        have = (lengths + page - 1) // page
        width = int(have.max())
        P = int(have.sum()) + 5
        table = torch.full((R, width), -1, dtype=torch.int32)
        table[torch.arange(width)[None, :] < have[:, None]] = order(P).cpu().int()[:P - 5]
        s["block_table"], s["lengths"] = table.to(dev), lengths.int().to(dev)
        s["q"] = randn(R, H, D).to(dt)
        s["k_pages"], s["v_pages"] = randn(P, Hk, page, D).to(dt), randn(P, Hk, page, D).to(dt)
        s["gate_pages"] = torch.nn.functional.logsigmoid(randn(P, H, page) + case["mu"])
    return s


# ------------------------------------------------------------------ plain forms
def _angles(s):
    a = s["positions"].double()[:, None] * s["inv_freq"].double()
    return a.cos().float(), a.sin().float()


def _rotate(x, cos, sin, rot, interleaved):
    """x (..., D) in 32 bits; cos, sin broadcast over all of its axes but the last."""
    r, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y, rest), -1)


def _plain_rotary(s):
    c = s["case"]
    cos, sin = _angles(s)
    if not c["head_first"]:
        cos, sin = cos[:, None], sin[:, None]
    x = s["x"].detach()
    y = _rotate(x.float(), cos, sin, c["rot"], c["interleaved"]).to(x.dtype)
    if not c["train"]:
        return y
    return y, _rotate(s["dy"].float(), cos, -sin, c["rot"], c["interleaved"]).to(x.dtype)


def _plain_norm(s):
    c = s["case"]
    cos, sin = [t[:, None] for t in _angles(s)]
    outs, grads, weights = [], [], []
    for x, w, dy in ((s["q"], s["q_weight"], s.get("dq")), (s["k"], s["k_weight"], s.get("dk"))):
        dt = x.dtype
        x, w = x.detach().float(), w.detach().view(-1, c["D"])
        rstd = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5)
        xhat = x * rstd
        outs.append(_rotate(xhat * w, cos, sin, c["rot"], c["interleaved"]).to(dt))
        if c["train"]:
            dn = _rotate(dy.float(), cos, -sin, c["rot"], c["interleaved"])
            dxhat = dn * w
            grads.append((rstd * (dxhat - xhat * (dxhat * xhat).mean(-1, keepdim=True))).to(dt))
            weights.append((dn * xhat).sum((0, 1, 2) if c["shared"] else (0, 1), dtype=torch.float64).float().flatten())
    return outs + grads + weights


def _plain_tables(s):
    page, table, free = s["case"]["page"], s["block_table"], s["free_pages"]
    old, new = s["lengths"].long(), s["new"].long()
    ends = new.cumsum(0)
    have = (old + page - 1) // page
    need = (old + new + page - 1) // page - have
    taken = need.cumsum(0) - need
    j = torch.arange(table.shape[1], device=table.device)
    fresh = (j >= have[:, None]) & (j < (have + need)[:, None])
    at = s["num_free"].long() - 1 - taken[:, None] - (j - have[:, None])
    table.copy_(torch.where(fresh, free[at.clamp(0, free.numel() - 1)], table))
    t = torch.arange(s["max_tokens"], device=table.device)
    valid = t < ends[-1]
    r = torch.searchsorted(ends, t, right=True).clamp(max=old.numel() - 1)
    pos = old[r] + t - (ends - new)[r]
    slot = table[r, (pos // page).clamp(max=table.shape[1] - 1)].long() * page + pos % page
    starts = torch.cat((ends.new_zeros(1), ends))
    out = (old + new, s["num_free"].long() - need.sum(), starts, torch.where(valid, r, -1), torch.where(valid, pos, 0),
           torch.where(valid, slot, -1))
    return [x.int() for x in out] + [table]


def _plain_update(s):
    slots = s["slots"].long()
    page = s["case"]["page"]
    gates = s["gates"].float()
    if s["case"]["logits"]:
        gates = torch.clamp(gates, max=0) - torch.log1p(torch.exp(-gates.abs()))
    # a row without a place goes where the first one goes, with that one's values
    keep = torch.where(slots >= 0, torch.arange(slots.numel(), device=slots.device), 0)
    slots = slots[keep]
    p, r = slots // page, slots % page
    s["k_pages"][p, :, r] = s["k"][keep]
    s["v_pages"][p, :, r] = s["v"][keep]
    s["gate_pages"][p, :, r] = gates[keep]
    return s["k_pages"], s["v_pages"], s["gate_pages"]


def _plain_attend(s):
    c = s["case"]
    R, H, Hk, D = c["R"], c["H"], c["Hk"], c["D"]
    at = s["block_table"].long().clamp(min=0)
    n = at.shape[1] * c["page"]
    k = s["k_pages"][at].transpose(1, 2).reshape(R, Hk, n, D).float()
    v = s["v_pages"][at].transpose(1, 2).reshape(R, Hk, n, D).float()
    live = torch.arange(n, device=at.device) < s["lengths"][:, None]
    v = torch.where(live[:, None, :, None], v, 0.0)
    g = torch.where(live[:, None], s["gate_pages"][at].transpose(1, 2).reshape(R, H, n).double(), 0.0)
    after = (g.flip(-1).cumsum(-1).flip(-1) - g).float()        # gates behind each key
    q = s["q"].float().view(R, Hk, H // Hk, D)
    u = (q @ k.transpose(-1, -2) / math.sqrt(D)).view(R, H, n) + after
    u = torch.where(live[:, None], u, float("-inf"))
    top = u.amax(-1, keepdim=True)
    e = torch.exp(u - torch.where(top > float("-inf"), top, 0.0))
    o = (e.view(R, Hk, H // Hk, n) @ v).view(R, H, D) / e.sum(-1, keepdim=True).clamp(min=1e-30)
    return o.to(s["q"].dtype)


# ------------------------------------------------------------------ one pass
def run(s):
    c = s["case"]
    kind = c["kind"]
    if not own:
        return {"rotary": _plain_rotary, "norm": _plain_norm, "tables": _plain_tables, "update": _plain_update,
                "attend": _plain_attend}[kind](s)
    import forgetting_transformer_b200 as fox
    if kind == "rotary":
        y = fox.rotary_embedding(s["x"], s["inv_freq"], s["positions"], head_first=c["head_first"], interleaved=c["interleaved"])
        if not c["train"]:
            return y
        return y, torch.autograd.grad(y, s["x"], s["dy"])[0]
    if kind == "norm":
        q, k = fox.qk_norm_rotary(s["q"], s["k"], s["q_weight"], s["k_weight"], s["inv_freq"], s["positions"], eps=1e-5,
                                  interleaved=c["interleaved"])
        if not c["train"]:
            return [q, k]
        return [q, k, *torch.autograd.grad((q, k), s["leaves"], (s["dq"], s["dk"]))]
    if kind == "tables":
        t = fox.page_tables(s["lengths"], s["new"], s["block_table"], s["free_pages"], s["num_free"], c["page"], s["max_tokens"])
        return [t.lengths, t.num_free, t.starts, t.requests, t.positions, t.slots, s["block_table"]]
    if kind == "update":
        fox.paged_update(s["k_pages"], s["v_pages"], s["gate_pages"], s["k"], s["v"], s["gates"], s["slots"],
                         gate_is_logit=c["logits"])
        return s["k_pages"], s["v_pages"], s["gate_pages"]
    return fox.paged_forgetting_attention(s["q"], s["k_pages"], s["v_pages"], s["gate_pages"], s["block_table"], s["lengths"])


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "rotary":
        n = case["B"] * case["T"] * case["H"] * case["D"]
        passes = 2 if case["train"] else 1
        return {"bytes": passes * 4 * n + 4 * case["T"], "flops": passes * 3 * n}
    if kind == "norm":
        n = case["B"] * case["T"] * (case["H"] + case["Hk"]) * case["D"]
        return {"bytes": (10 if case["train"] else 4) * n + 4 * case["T"], "flops": (25 if case["train"] else 8) * n}
    if kind == "tables":
        old, new = _old_new(case)
        fresh = sum(_pages(a + b, case["page"]) - _pages(a, case["page"]) for a, b in zip(old, new))
        tokens = sum(new) + case["R"]
        return {"bytes": 4 * (4 * case["R"] + 2 * fresh + 3 * tokens), "flops": 8 * tokens}
    if kind == "update":
        n = case["T"] - case["T"] // 16
        gate = 2 if case["logits"] else 4
        return {"bytes": n * (8 * case["Hk"] * case["D"] + (gate + 4) * case["H"] + 4), "flops": 4 * n * case["H"]}
    keys = sum(_lengths(case))
    return {"bytes": keys * (4 * case["Hk"] * case["D"] + 4 * case["H"]) + 4 * case["R"] * case["H"] * case["D"],
            "flops": 4 * keys * case["H"] * case["D"]}


# ------------------------------------------------------------------ 64 bits
def _turn(x, positions, inv_freq, interleaved, sign):
    """x (tokens, heads, D) in 64 bits, rotated as complex numbers."""
    half = inv_freq.numel()
    a = sign * positions.double()[:, None, None] * inv_freq.double()
    turn = torch.polar(torch.ones_like(a), a)
    y = x.clone()
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    z = torch.complex(x[..., first], x[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "rotary":
        def turned(x, sign):
            x = x.detach().double()
            rows = x.transpose(1, 2) if case["head_first"] else x
            y = torch.stack([_turn(r, s["positions"], s["inv_freq"], case["interleaved"], sign) for r in rows])
            return y.transpose(1, 2) if case["head_first"] else y
        y = turned(s["x"], 1)
        return (y, turned(s["dy"], -1)) if case["train"] else y
    if kind == "norm":
        outs = []
        for n in ("q", "k"):
            x = s[n].detach().double()
            w = s[n + "_weight"].detach().double()
            if case["train"]:
                x.requires_grad_()
                w.requires_grad_()
            y = x / (x.pow(2).sum(-1, keepdim=True) / case["D"] + 1e-5).sqrt() * w.view(-1, case["D"])
            y = torch.stack([_turn(r, s["positions"], s["inv_freq"], case["interleaved"], 1) for r in y])
            grads = torch.autograd.grad(y, (x, w), s["d" + n].double()) if case["train"] else ()
            outs.append([y.detach(), *grads])
        return [o[i] for i in range(len(outs[0])) for o in outs]
    if kind == "tables":
        page, free, n_free = case["page"], s["free_pages"].tolist(), int(s["num_free"])
        table, old, new = s["block_table"].tolist(), s["lengths"].tolist(), s["new"].tolist()
        starts, tokens = [0], []
        for r, row in enumerate(table):
            for pos in range(old[r], old[r] + new[r]):
                if pos % page == 0:
                    n_free -= 1
                    row[pos // page] = free[n_free]
                tokens.append((r, pos, row[pos // page] * page + pos % page))
            starts.append(len(tokens))
        tokens += [(-1, 0, -1)] * (s["max_tokens"] - len(tokens))
        out = ([a + b for a, b in zip(old, new)], [n_free], starts, *zip(*tokens), table)
        return [torch.tensor(x, dtype=torch.int32) for x in out]
    if kind == "update":
        p = [s[n].double() for n in ("k_pages", "v_pages", "gate_pages")]
        slots = s["slots"].tolist()
        keep = [i for i, x in enumerate(slots) if x >= 0]
        gates = s["gates"].double()
        if case["logits"]:
            gates = -torch.log1p(torch.exp(-gates))
        to = torch.tensor([slots[i] for i in keep], device=gates.device, dtype=torch.long)
        at = torch.tensor(keep, device=gates.device, dtype=torch.long)
        for pages, rows in zip(p, (s["k"].double(), s["v"].double(), gates)):
            pages.transpose(1, 2)[to // case["page"], to % case["page"]] = rows[at]
        return tuple(p)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    group = case["H"] // case["Hk"]
    for r, n in enumerate(s["lengths"].tolist()):
        if n == 0:
            continue
        pages = s["block_table"][r, :_pages(n, case["page"])].long()
        gates = torch.cat(list(s["gate_pages"][pages].double()), -1)[:, :n]
        total = torch.cumsum(gates, -1)
        bias = total[:, -1:] - total
        for h in range(case["Hk"]):
            k = s["k_pages"][pages, h].flatten(0, 1)[:n].double()
            v = s["v_pages"][pages, h].flatten(0, 1)[:n].double()
            heads = slice(h * group, (h + 1) * group)
            logits = s["q"][r, heads].double() @ k.T / case["D"] ** 0.5 + bias[heads]
            out[r, heads] = torch.softmax(logits, -1) @ v
    return out
