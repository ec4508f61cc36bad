"""Performance cases of the row-selection operators: embedding lookup and its
gradient, routing to experts with its gradient and plan, the exchange of rows
with the experts in both directions, and gradient clipping.

listed() names the cases, prepare() makes one's inputs, run() computes it (in
its plain form, or with the library's kernels where `own` is set), exact()
computes it in 64 bits, work() counts the bytes and operations it needs.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}
_context = []


def listed():
    return [
        # A serving step: sixteen sequences, one new token each.
        {"name": "lookup 16 x 1024 bf16", "op": "lookup", "tokens": 16, "rows": 100000, "width": 1024, "type": "bfloat16",
         "scale": 32.0, "padding": 0.0},
        # A packed prompt or training batch, rows scaled by sqrt(width).
        {"name": "lookup 16384 x 4096 bf16", "op": "lookup", "tokens": 16384, "rows": 131072, "width": 4096,
         "type": "bfloat16", "scale": 64.0, "padding": 0.02},
        # Ragged micro-batch added into a float32 gradient, a tenth of it padding.
        {"name": "lookup grad 5003 x 1001 f32 add", "op": "lookup_grad", "tokens": 5003, "rows": 32003, "width": 1001,
         "type": "float32", "scale": 1.0, "padding": 0.1, "accumulate": True},
        # The dense gradient of a large table from one training batch.
        {"name": "lookup grad 16384 x 4096 bf16", "op": "lookup_grad", "tokens": 16384, "rows": 131072, "width": 4096,
         "type": "bfloat16", "scale": 64.0, "padding": 0.02, "accumulate": False},
        # Serving one sequence.
        {"name": "route 1 x 64 softmax bf16", "op": "route", "tokens": 1, "experts": 64, "k": 2, "score": "softmax",
         "renormalise": True, "groups": 1, "groups_kept": 1, "group_top": 1, "bias": False, "scale": 1.0, "type": "bfloat16",
         "padding": 0.0},
        # A training batch over many experts: groups, and a bias that balances their load.
        {"name": "route 16384 x 256 sigmoid f32", "op": "route", "tokens": 16384, "experts": 256, "k": 8, "score": "sigmoid",
         "renormalise": True, "groups": 8, "groups_kept": 4, "group_top": 2, "bias": True, "scale": 2.5, "type": "float32",
         "padding": 0.02},
        # Odd sizes, weights that are not renormalised, masked padding rows.
        {"name": "route grad 4099 x 60 softmax f16", "op": "route_grad", "tokens": 4099, "experts": 60, "k": 4,
         "score": "softmax", "renormalise": False, "groups": 1, "groups_kept": 1, "group_top": 1, "bias": False, "scale": 1.0,
         "type": "float16", "padding": 0.1},
        {"name": "route grad 16384 x 256 sigmoid f32", "op": "route_grad", "tokens": 16384, "experts": 256, "k": 8,
         "score": "sigmoid", "renormalise": True, "groups": 8, "groups_kept": 4, "group_top": 2, "bias": True, "scale": 2.5,
         "type": "float32", "padding": 0.02},
        # A serving step's tokens to their experts and back.
        {"name": "exchange 32 x 8 x 2048 bf16", "op": "exchange", "tokens": 32, "experts": 64, "k": 8, "width": 2048,
         "type": "bfloat16", "backward": False, "padding": 0.0},
        # The same of a training batch, backward: rows' and weights' gradients.
        {"name": "exchange grad 4096 x 8 x 4096 bf16", "op": "exchange", "tokens": 4096, "experts": 256, "k": 8, "width": 4096,
         "type": "bfloat16", "backward": True, "padding": 0.02},
        # A small model's float32 gradients.
        {"name": "clip 26 f32", "op": "clip", "tensors": 26, "values": 180001, "type": "float32"},
        # A bucket of a large model's gradients.
        {"name": "clip 290 bf16 512M", "op": "clip", "tensors": 290, "values": 512000000, "type": "bfloat16"},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["lookup", "lookup_grad", "route", "route_grad", "exchange", "clip"])
    kind = rng.choice(sorted(TYPES))
    tokens = _log(rng, 1, 16384)
    width = _log(rng, 16, 4096 * 2 // SIZE[kind])
    if rng.random() < 0.6:
        width = max(16, width // 16 * 16)
    padding = rng.choice([0.0, 0.02, 0.1])
    if op in ("lookup", "lookup_grad"):
        case = {"op": op, "tokens": tokens, "rows": _log(rng, 1000, 131072), "width": width, "type": kind,
                "scale": rng.choice([1.0, round(math.sqrt(width), 3)]), "padding": padding}
        return case | ({"accumulate": rng.random() < 0.5} if op == "lookup_grad" else {})
    if op == "exchange":
        experts = _log(rng, 4, 256)
        k = rng.randint(1, min(8, experts))
        return {"op": op, "tokens": max(1, tokens // 4), "experts": experts, "k": k, "width": width, "type": kind,
                "backward": rng.random() < 0.5, "padding": padding}
    if op == "clip":
        return {"op": op, "tensors": _log(rng, 1, 300), "values": _log(rng, 1000, 512000000 * 2 // SIZE[kind]), "type": kind}
    groups = rng.choice([1, 1, 2, 4, 8])
    experts = groups * _log(rng, 4, 256 // groups)
    kept = rng.randint(1, groups)
    k = rng.randint(1, min(10, experts // groups * kept))
    return {"op": op, "tokens": tokens, "experts": experts, "k": k, "score": rng.choice(["softmax", "sigmoid"]),
            "renormalise": rng.random() < 0.5, "groups": groups, "groups_kept": kept, "group_top": rng.choice([1, 2]),
            "bias": rng.random() < 0.5, "scale": rng.choice([1.0, 2.5]), "type": kind, "padding": padding}


# ---- inputs -------------------------------------------------------------------

def _tokens(case, g):
    """Token ids as text has them: a few frequent ones and a long tail,
    spread over the table; -1 where a batch is padded."""
    t, rows = case["tokens"], case["rows"]
    u = torch.rand(t, generator=g, device="cuda", dtype=torch.float64)
    rank = (rows * u ** 3).long().clamp_(max=rows - 1)
    ids = (rank * 7919 + 13) % rows
    pad = torch.rand(t, generator=g, device="cuda") < case["padding"]
    return torch.where(pad, -1, ids).int()


def _logits(case, g):
    """Router logits around each expert's own mean; rows of padding masked."""
    t, e = case["tokens"], case["experts"]
    mean = torch.randn(e, generator=g, device="cuda") * 0.5
    x = torch.randn(t, e, generator=g, device="cuda") * 1.5 + mean
    pad = torch.rand(t, generator=g, device="cuda") < case["padding"]
    return torch.where(pad[:, None], float("-inf"), x).to(TYPES[case["type"]])


def _sizes(case, seed):
    """Ragged tensor sizes that add up to case["values"]."""
    n, total = case["tensors"], case["values"]
    share = np.exp(np.random.RandomState(seed % (1 << 31)).uniform(0.0, 5.0, n))
    sizes = np.maximum(1, (share / share.sum() * total).astype(np.int64))
    sizes[np.argmax(sizes)] += total - sizes.sum()
    return [int(v) for v in sizes]


def _buffers(case):
    t, k, e = case["tokens"], case["k"], case["experts"]
    return {"indices": torch.full((t, k), -1, dtype=torch.int32, device="cuda"),
            "weights": torch.zeros(t, k, device="cuda"),
            "offsets": torch.zeros(e + 1, dtype=torch.int32, device="cuda"),
            "order": torch.full((t * k,), -1, dtype=torch.int32, device="cuda"),
            "position": torch.full((t, k), -1, dtype=torch.int32, device="cuda")}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, kind = case["op"], TYPES[case["type"]]
    state = {"case": case}
    if own:
        import spmvbench_b200 as S
        if not _context:
            _context.append(S.Context(0))
        ctx = _context[0]
    if op in ("lookup", "lookup_grad"):
        t, rows, width = case["tokens"], case["rows"], case["width"]
        state["tokens"] = _tokens(case, g)
        if op == "lookup":
            state["table"] = torch.randn(rows, width, generator=g, device="cuda", dtype=kind)
            state["out"] = torch.zeros(t, width, device="cuda", dtype=kind)
        else:
            state["dout"] = torch.randn(t, width, generator=g, device="cuda", dtype=kind)
            state["dtable"] = torch.zeros(rows, width, device="cuda", dtype=kind)
        if own:
            state["embedding"] = S.Embedding(ctx, rows, width, max_tokens=t)
    elif op in ("route", "route_grad"):
        state["logits"] = _logits(case, g)
        state |= _buffers(case)
        # Balance biases move in small steps and stay near zero.
        state["bias"] = torch.randn(case["experts"], generator=g, device="cuda") * 0.05 if case["bias"] else None
        if op == "route_grad":
            state["indices"] = _choice(case, state["logits"], state["bias"])[0]
            state["dweights"] = torch.randn(case["tokens"], case["k"], generator=g, device="cuda")
            state["dlogits"] = torch.zeros_like(state["logits"])
        if own:
            state["router"] = S.Router(ctx, case["experts"], case["k"], max_tokens=case["tokens"], score=case["score"],
                                       renormalise=case["renormalise"], scale=case["scale"], groups=case["groups"],
                                       groups_kept=case["groups_kept"], group_top=case["group_top"])
    elif op == "exchange":
        t, k, e, width = case["tokens"], case["k"], case["experts"], case["width"]
        # k different experts a token, some more in demand than others.
        liked = torch.randn(e, generator=g, device="cuda")
        noise = -torch.log(-torch.log(torch.rand(t, e, generator=g, device="cuda").clamp_(1e-9, 1 - 1e-7)))
        indices = (liked + noise).topk(k, dim=1).indices.int()
        pad = torch.rand(t, generator=g, device="cuda") < case["padding"]
        indices[pad] = -1
        position = _plan(indices, e)[2]
        state["position"] = position
        state["weights"] = torch.rand(t, k, generator=g, device="cuda").softmax(1)
        if case["backward"]:
            state["y"] = torch.randn(t * k, width, generator=g, device="cuda", dtype=kind)
            state["dout"] = torch.randn(t, width, generator=g, device="cuda", dtype=kind)
            state["dxs"] = torch.randn(t * k, width, generator=g, device="cuda", dtype=kind)
            state["dy"] = torch.zeros(t * k, width, device="cuda", dtype=kind)
            state["dweights"] = torch.zeros(t, k, device="cuda")
            state["dx"] = torch.zeros(t, width, device="cuda", dtype=kind)
        else:
            state["x"] = torch.randn(t, width, generator=g, device="cuda", dtype=kind)
            state["y"] = torch.randn(t * k, width, generator=g, device="cuda", dtype=kind)
            state["xs"] = torch.zeros(t * k, width, device="cuda", dtype=kind)
            state["out"] = torch.zeros(t, width, device="cuda", dtype=kind)
        if own:
            state["router"] = S.Router(ctx, e, k, max_tokens=t)
    else:
        # Gradients as views of one bucket, as a data-parallel trainer keeps them.
        bucket = torch.randn(case["values"], generator=g, device="cuda", dtype=kind)
        state["bucket"] = bucket
        state["grads"] = list(bucket.split(_sizes(case, seed)))
        state["norm"] = torch.zeros(1, device="cuda")
        state["max_norm"] = 0.25 * math.sqrt(case["values"])
        if own:
            state["clip"] = S.GradClip(ctx, state["grads"])
    return state


# ---- plain forms ----------------------------------------------------------------

def _scores(case, logits):
    """Scores in 64 bits (a choice between experts whose scores lie close
    together hangs on the last bits), 0 for masked experts; True for the
    rows that have scores."""
    l = logits.double()
    if case["score"] == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-l)), torch.ones(l.shape[0], dtype=torch.bool, device=l.device)
    top = l.amax(dim=1, keepdim=True)
    fine = ~(torch.isnan(l).any(1) | (top[:, 0] == math.inf))
    x = torch.exp(l - torch.where(top > -math.inf, top, 0.0))
    total = x.sum(1, keepdim=True)
    return x / torch.where(total == 0, 1.0, total), fine


def _choice(case, logits, bias):
    """Chosen experts (-1: none) and their weights."""
    t, e, k = case["tokens"], case["experts"], case["k"]
    score, fine = _scores(case, logits)
    open_ = (logits > -math.inf) & fine[:, None]
    value = score if bias is None else score + bias.double()
    rank = logits.double() if bias is None else value
    open_ &= rank > -math.inf
    if case["groups"] > 1:
        inside = torch.where(open_, value, -math.inf).view(t, case["groups"], -1).sort(dim=2, descending=True).values
        first, second = inside[:, :, 0], inside[:, :, min(1, inside.shape[2] - 1)]
        both = (case["group_top"] == 2) & (second > -math.inf) & (inside.shape[2] > 1)
        if bias is None and case["group_top"] == 1:
            first = torch.where(open_, rank, -math.inf).view(t, case["groups"], -1).amax(2)
        level = torch.where(both, first + second, first)
        kept = level.sort(dim=1, descending=True, stable=True).indices[:, :case["groups_kept"]]
        held = torch.zeros(t, case["groups"], dtype=torch.bool, device=logits.device).scatter_(1, kept, True)
        open_ = open_ & held.repeat_interleave(e // case["groups"], dim=1)
    rank = torch.where(open_, rank, -math.inf)
    indices = rank.sort(dim=1, descending=True, stable=True).indices[:, :k]
    there = open_.gather(1, indices)
    chosen = torch.where(there, score.gather(1, indices), 0.0)
    if case["renormalise"]:
        total = chosen.sum(1, keepdim=True)
        chosen = chosen / torch.where(total == 0, 1.0, total)
    weights = torch.where(fine[:, None], chosen * case["scale"], math.nan)
    return torch.where(there, indices, -1).int(), weights.float()


def _plan(indices, experts, order=None):
    flat = indices.reshape(-1).long()
    key = torch.where(flat < 0, experts, flat)
    by = key.sort(stable=True).indices
    offsets = torch.bincount(key, minlength=experts + 1).cumsum(0)
    offsets = torch.cat([torch.zeros_like(offsets[:1]), offsets[:experts]])
    place = torch.arange(flat.numel(), device=flat.device)
    there = place < offsets[-1]
    position = torch.empty_like(by)
    position[by] = torch.where(there, place, -1)
    left = torch.full_like(flat, -1) if order is None else order.long()
    return offsets.int(), torch.where(there, by, left).int(), position.view(indices.shape).int()


def _route_grad(case, logits, indices, dweights):
    score, fine = _scores(case, logits)
    score = score.float()
    there = indices >= 0
    at = indices.long().clamp(min=0)
    chosen = torch.where(there, score.gather(1, at), 0.0)
    dw = torch.where(there, dweights, 0.0) * case["scale"]
    if case["renormalise"]:
        total = chosen.sum(1, keepdim=True)
        part = chosen / torch.where(total == 0, 1.0, total)
        d = part * (dw - (part * dw).sum(1, keepdim=True))
        if case["score"] == "sigmoid":
            d = d * (1.0 - chosen)
        full = torch.zeros_like(score)
    elif case["score"] == "sigmoid":
        d = chosen * (1.0 - chosen) * dw
        full = torch.zeros_like(score)
    else:
        d = chosen * dw
        full = -score * d.sum(1, keepdim=True)
    full = full.scatter_add(1, at, torch.where(there, d, 0.0))
    return torch.where(fine[:, None], full, math.nan).to(logits.dtype)


def _rows(source, position):
    """source's rows at `position`, zeros where it is -1, in 32 bits."""
    got = source[position.long().clamp(min=0)].float()
    return torch.where((position >= 0).unsqueeze(-1), got, 0.0)


def run(state):
    case = state["case"]
    op = case["op"]
    if op == "lookup":
        if own:
            state["embedding"].lookup(state["tokens"], state["table"], state["out"], scale=case["scale"])
            return state["out"]
        return (_rows(state["table"], state["tokens"]) * case["scale"]).to(state["table"].dtype)
    if op == "lookup_grad":
        if own:
            state["embedding"].lookup_grad(state["tokens"], state["dout"], state["dtable"], scale=case["scale"],
                                           accumulate=case["accumulate"])
            return state["dtable"]
        tokens, dtable = state["tokens"], state["dtable"]
        d = torch.where((tokens >= 0)[:, None], state["dout"].float(), 0.0) * case["scale"]
        total = dtable.float() if case["accumulate"] else torch.zeros(dtable.shape, device="cuda")
        state["dtable"] = total.index_add_(0, tokens.clamp(min=0), d).to(dtable.dtype)
        return state["dtable"]
    if op == "route":
        if own:
            state["router"].route(state["logits"], state["indices"], state["weights"], bias=state["bias"],
                                  offsets=state["offsets"], order=state["order"], position=state["position"])
            return [state[n] for n in ("indices", "weights", "offsets", "order", "position")]
        indices, weights = _choice(case, state["logits"], state["bias"])
        return [indices, weights, *_plan(indices, case["experts"], state["order"])]
    if op == "route_grad":
        if own:
            state["router"].route_grad(state["logits"], state["indices"], state["dweights"], state["dlogits"])
            return state["dlogits"]
        return _route_grad(case, state["logits"], state["indices"], state["dweights"])
    if op == "exchange":
        position, weights = state["position"], state["weights"]
        if own:
            router = state["router"]
            if case["backward"]:
                router.combine_grad(position, weights, state["y"], state["dout"], state["dy"], state["dweights"])
                router.dispatch_grad(position, state["dxs"], state["dx"])
                return [state["dy"], state["dweights"], state["dx"]]
            router.dispatch(position, state["x"], state["xs"])
            router.combine(position, weights, state["y"], state["out"])
            return [state["xs"], state["out"]]
        t, k = position.shape
        entry = torch.arange(t * k, device="cuda")[(position >= 0).reshape(-1)]
        to = position.reshape(-1)[entry].long()
        if case["backward"]:
            dout = state["dout"].float()
            dy = state["dy"].index_copy(0, to, (dout[entry // k] * weights.reshape(-1, 1)[entry]).to(state["dy"].dtype))
            dweights = (_rows(state["y"], position) * dout[:, None]).sum(2)
            return [dy, dweights, _rows(state["dxs"], position).sum(1).to(dy.dtype)]
        xs = state["xs"].index_copy(0, to, state["x"][entry // k])
        return [xs, (_rows(state["y"], position) * weights[:, :, None]).sum(1).to(xs.dtype)]
    if own:
        state["clip"].clip(state["max_norm"], state["norm"])
        return [state["norm"], state["bucket"]]
    norm = torch.sqrt(sum(g.double().square().sum() for g in state["grads"]))
    factor = torch.clamp(state["max_norm"] / (norm + 1e-6), max=1.0).float()
    state["bucket"].copy_(state["bucket"].float() * factor)
    return [norm.float().reshape(1), state["bucket"]]


# ---- 64 bits ----------------------------------------------------------------------

def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    op = case["op"]
    if op == "lookup":
        pad = torch.cat([s["table"], torch.zeros_like(s["table"][:1])])
        at = torch.where(s["tokens"] < 0, case["rows"], s["tokens"])
        return pad.index_select(0, at).double().mul_(case["scale"])
    if op == "lookup_grad":
        # One product with the tokens' incidence matrix over the distinct rows.
        seen, back = s["tokens"].unique(return_inverse=True)
        out = s["dtable"].double()
        for a in range(0, case["width"], 512):
            part = torch.zeros(seen.numel(), min(512, case["width"] - a), device="cuda", dtype=torch.float64)
            for b in range(0, case["tokens"], 2048):
                hit = (back[b:b + 2048] == torch.arange(seen.numel(), device="cuda")[:, None]).double()
                part += hit @ s["dout"][b:b + 2048, a:a + 512].double()
            there = seen >= 0
            out[seen[there].long(), a:a + 512] += part[there] * case["scale"]
        return out
    if op in ("route", "route_grad"):
        l = s["logits"].double()
        # Logarithms of the scores.
        if case["score"] == "sigmoid":
            log = torch.nn.functional.logsigmoid(l)
        else:
            log = l - torch.where(torch.isinf(l).all(1), 0.0, torch.logsumexp(l, 1))[:, None]
        indices = s["indices"] if op == "route_grad" else _choice(case, s["logits"], s["bias"])[0]
        there = indices >= 0
        at = torch.where(there, indices, 0).long()
        chosen = torch.where(there, log.gather(1, at), -math.inf)
        none = ~there.any(1, keepdim=True)
        if case["renormalise"]:
            share = torch.exp(chosen - torch.where(none, 0.0, torch.logsumexp(chosen, 1, keepdim=True)))
        else:
            share = torch.exp(chosen)
        if op == "route":
            return [None, share * case["scale"], None, None, None]
        # d w_i / d l_e summed over the chosen i, from the derivative of each logarithm.
        dw = s["dweights"].double() * case["scale"] * there
        dlog = share * dw
        if case["renormalise"]:
            dlog = dlog - share * dlog.sum(1, keepdim=True)
        if case["score"] == "sigmoid":
            return torch.zeros_like(l).scatter_add(1, at, dlog * torch.sigmoid(-l.gather(1, at)) * there)
        whole = torch.zeros_like(l).scatter_add(1, at, torch.where(there, dlog, 0.0))
        return whole - torch.exp(log) * whole.sum(1, keepdim=True)
    if op == "exchange":
        position = s["position"]
        t, k = position.shape
        weights = s["weights"].double()
        if case["backward"]:
            dy, dx, dw = s["dy"].double(), [], []
            for j in range(k):
                ok = position[:, j] >= 0
                dy[position[ok, j].long()] = torch.einsum("tc,t->tc", s["dout"][ok].double(), weights[ok, j])
            ybar = torch.cat([s["y"], torch.zeros_like(s["y"][:1])])
            dbar = torch.cat([s["dxs"], torch.zeros_like(s["dxs"][:1])])
            at = torch.where(position < 0, t * k, position).long()
            for a in range(0, t, 512):
                dw.append(torch.einsum("tkc,tc->tk", ybar[at[a:a + 512]].double(), s["dout"][a:a + 512].double()))
                dx.append(torch.einsum("tkc->tc", dbar[at[a:a + 512]].double()))
            return [dy, torch.cat(dw), torch.cat(dx)]
        xs = s["xs"].double()
        out = []
        for j in range(k):
            ok = position[:, j] >= 0
            xs[position[ok, j].long()] = s["x"][ok].double()
        ybar = torch.cat([s["y"], torch.zeros_like(s["y"][:1])])
        at = torch.where(position < 0, t * k, position).long()
        for a in range(0, t, 512):
            out.append(torch.einsum("tkc,tk->tc", ybar[at[a:a + 512]].double(), weights[a:a + 512]))
        return [xs, torch.cat(out)]
    total = sum(float(torch.linalg.vector_norm(g, dtype=torch.float64)) ** 2 for g in s["grads"])
    norm = math.sqrt(total)
    return [torch.tensor([norm], dtype=torch.float64), s["bucket"].double() * min(1.0, s["max_norm"] / (norm + 1e-6))]


# ---- what a pass cannot do without ----------------------------------------------

def _distinct(case):
    """Expected distinct rows among the tokens, from their distribution."""
    edge = (np.arange(case["rows"] + 1) / case["rows"]) ** (1.0 / 3.0)
    p = np.diff(edge) * (1.0 - case["padding"])
    return float(np.sum(-np.expm1(case["tokens"] * np.log1p(-np.minimum(p, 1 - 1e-12)))))


def work(case):
    op, size = case["op"], SIZE[case["type"]]
    if op in ("lookup", "lookup_grad"):
        t, row = case["tokens"], case["width"] * size
        real = t * (1.0 - case["padding"])
        if op == "lookup":
            return {"bytes": 4 * t + _distinct(case) * row + t * row, "flops": real * case["width"]}
        table = 2 * _distinct(case) * row if case["accumulate"] else case["rows"] * row
        return {"bytes": 4 * t + real * row + table, "flops": 2 * real * case["width"]}
    if op in ("route", "route_grad"):
        t, e, k = case["tokens"], case["experts"], case["k"]
        if op == "route":  # logits; indices, weights, order and position; offsets and bias
            return {"bytes": t * e * size + 16 * t * k + 4 * (e + 1) + 4 * e * case["bias"], "flops": 5 * t * e}
        # The scores of the whole row are needed where the softmax runs over it; else those of the chosen ones.
        whole = case["score"] == "softmax" and not case["renormalise"]
        return {"bytes": (t * e * size if whole else t * k * size) + t * e * size + 8 * t * k,
                "flops": (8 * t * e if whole else 8 * t * k)}
    if op == "exchange":
        t, k, w = case["tokens"], case["k"], case["width"]
        sent = t * k * (1.0 - case["padding"])
        if case["backward"]:
            return {"bytes": (3 * sent + 2 * t) * w * size + 12 * t * k, "flops": 4 * sent * w}
        return {"bytes": (2 * sent + 2 * t) * w * size + 8 * t * k, "flops": 2 * sent * w}
    return {"bytes": 2 * case["values"] * size + 4, "flops": 3 * case["values"]}
