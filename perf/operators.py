"""What the routing and the 128-block FP8 operators of this repository are judged by: one pass of a case is one call of the
public API as a program that trains or serves a Mixture-of-Experts layer makes it.

A case is a dict of plain values.  `kind` says which operator, and how it is used:

  route         `group_limited_routing` of a batch that is served: scores and experts of every token
  route_train   the same with its backward pass: scores, experts and the gradient of the logits
  quant_weight  `quantize_weight_block128`: a layer's weights in e4m3 with one scale for each 128 x 128 block
  quant_rows    `quantize_rows_block128`: activations in e4m3 with one scale for each row and 128 columns; with `swiglu`,
                of the gated activation of a projection's output
  linear        `block128_linear` with weights that were quantised once: y = x W^T by expert segments, nothing saved
  linear_train  the same from bf16 weights with its backward pass: y and the gradients of x and W
  experts       `block128_experts`: routing table in, quantised tokens, both products with the gated activation between them,
                and the weighted sum of a token's experts

A segment is the run of rows of one expert; it starts at a multiple of 128 rows, and only its first `counts[e]` rows are live.
"""
import math
import os
import sys

import torch

own = False

E4M3_MAX = 448.0
TINY = 2.0 ** -100           # the smallest maximum a group's scale is made from


def listed():
    return [
        # one decode step of a serving batch: 256 experts in 8 groups, of which a token may use 4; latency
        dict(name="route_decode_64", kind="route", T=64, E=256, K=8, groups=8, top_groups=4, group_score=2, score="sigmoid",
             bias=True, normalize=True, scale=2.5, dtype="f32"),
        # the router of a training step over the fine-grained layer's 128 experts
        dict(name="route_train_16384", kind="route_train", T=16384, E=128, K=8, groups=8, top_groups=4, group_score=2,
             score="sigmoid", bias=True, normalize=True, scale=1.0, dtype="bf16"),
        # softmax scores, groups ranked by their best expert, an odd number of tokens, experts no power of two
        dict(name="route_train_softmax_5003", kind="route_train", T=5003, E=60, K=6, groups=5, top_groups=3, group_score=1,
             score="softmax", bias=False, normalize=False, scale=16.0, dtype="f32"),
        # up-projections of 32 fine-grained experts, once per optimizer step
        dict(name="quant_weight_e32", kind="quant_weight", E=32, N=1536, K=2048),
        # the gated activation between the two products of a prompt's experts
        dict(name="quant_rows_swiglu_16384", kind="quant_rows", rows=16384, K=1536, swiglu=True),
        # tokens of a ragged batch, a last block of 80 columns
        dict(name="quant_rows_odd_3001", kind="quant_rows", rows=3001, K=720, swiglu=False),
        # one token through a dense projection: weights from HBM, latency
        dict(name="linear_1", kind="linear", E=1, N=4096, K=4096, rows=1, skew=0.0),
        # a prompt chunk through the same projection
        dict(name="linear_8192", kind="linear", E=1, N=4096, K=4096, rows=8192, skew=0.0),
        # a training step of one expert projection under a skewed router
        dict(name="linear_train_16384", kind="linear_train", E=8, N=4096, K=2048, rows=16384, skew=0.6),
        # the same for few experts of sizes that no tile divides, with empty and short segments
        dict(name="linear_train_odd_700", kind="linear_train", E=5, N=1000, K=720, rows=700, skew=1.2),
        # one decode step of 64 tokens through 128 fine-grained experts
        dict(name="experts_decode_64", kind="experts", E=128, H=2048, I=768, T=64, topk=8, skew=0.0),
        # a prompt through them
        dict(name="experts_prefill_4096", kind="experts", E=128, H=2048, I=768, T=4096, topk=8, skew=0.6),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("route", "route_train", "quant_weight", "quant_rows", "linear", "linear", "linear_train", "linear_train",
                       "experts", "experts"))
    if kind.startswith("route"):
        groups = rng.choice((1, 1, 4, 5, 8))
        E = groups * rng.choice((3, 8, 12, 16, 32)) if groups > 1 else rng.choice((8, 37, 64, 128, 160, 256))
        top_groups = rng.randint((groups + 1) // 2, groups)
        K = rng.randint(1, min(8, top_groups * (E // groups)))
        score = rng.choice(("sigmoid", "softmax"))
        return dict(kind=kind, T=_log(rng, 1, 16384), E=E, K=K, groups=groups, top_groups=top_groups,
                    group_score=rng.choice((1, 2)), score=score, bias=rng.random() < 0.6, normalize=rng.random() < 0.6,
                    scale=rng.choice((1.0, 2.5)), dtype=rng.choice(("f32", "bf16")))
    if kind == "quant_weight":
        return dict(kind=kind, E=_log(rng, 1, 32), N=8 * _log(rng, 8, 192), K=16 * _log(rng, 4, 128))
    if kind == "quant_rows":
        return dict(kind=kind, rows=_log(rng, 1, 16384), K=16 * _log(rng, 2, 128), swiglu=rng.random() < 0.5)
    if kind == "linear":
        return dict(kind=kind, E=rng.choice((1, 1, 4, 8)), N=8 * _log(rng, 16, 512), K=16 * _log(rng, 8, 256),
                    rows=_log(rng, 1, 8192), skew=rng.choice((0.0, 0.6, 1.2)))
    if kind == "linear_train":
        return dict(kind=kind, E=rng.choice((1, 3, 8)), N=8 * _log(rng, 16, 512), K=16 * _log(rng, 8, 128),
                    rows=_log(rng, 16, 16384), skew=rng.choice((0.0, 0.6, 1.2)))
    E = rng.choice((8, 37, 128))
    return dict(kind=kind, E=E, H=16 * _log(rng, 16, 128), I=16 * _log(rng, 8, 48), T=_log(rng, 1, 4096),
                topk=rng.randint(1, 8), skew=rng.choice((0.0, 0.6)))


# ------------------------------------------------------------------------------------------------ the rule of a scale
def _blocks(x, dim):
    """x with `dim` cut into blocks of 128 (the last one filled up with zeros): that dimension becomes two."""
    n = x.shape[dim]
    pad = -n % 128
    if pad:
        shape = list(x.shape)
        shape[dim] = pad
        x = torch.cat([x, x.new_zeros(shape)], dim)
    return x.unflatten(dim, ((n + pad) // 128, 128))


def _scales(amax):
    """(what the values are multiplied by, what stands in the scale) from the largest magnitude of a group."""
    amax = amax.clamp(min=TINY)
    most = torch.full_like(amax, E4M3_MAX)             # a quotient of tensors is rounded once, one with a number may not be
    return most / amax, amax / most


def _rounded(v, like):
    return v.to(torch.float8_e4m3fn) if like == torch.float32 else v.float().to(torch.float8_e4m3fn)


def _quant_rows(x, f):
    """x [rows, K] -> e4m3 [rows, K], scales [rows, K/128]; f: the type it is computed in."""
    b = _blocks(x.to(f), 1)
    inv, s = _scales(b.abs().amax(2))
    q = _rounded((b * inv[:, :, None]).flatten(1)[:, :x.shape[1]], f)
    return q, s


def _quant_weight(w, f):
    """w [E, N, K] -> e4m3 [E, N, K], scales [E, N/128, K/128]."""
    E, N, K = w.shape
    b = _blocks(_blocks(w.to(f), 1), 3)                            # [E, nb, 128, kb, 128]
    inv, s = _scales(b.abs().amax((2, 4)))
    q = _rounded((b * inv[:, :, None, :, None]).flatten(3).flatten(1, 2)[:, :N, :K], f)
    return q, s


def _quant_cols(x, f):
    """x [rows, n], rows a multiple of 128 -> e4m3 [rows, n], scales [rows/128, n]: one for each column and 128 rows."""
    b = x.to(f).unflatten(0, (x.shape[0] // 128, 128))
    inv, s = _scales(b.abs().amax(1))
    return _rounded((b * inv[:, None, :]).flatten(0, 1), f), s


def _deq_rows(q, s, f):
    return q.to(f) * s.to(f).repeat_interleave(128, 1)[:, :q.shape[1]]


def _deq_weight(q, s, f):
    return q.to(f) * s.to(f).repeat_interleave(128, 1)[:, :q.shape[1]].repeat_interleave(128, 2)[:, :, :q.shape[2]]


def _deq_cols(q, s, f):
    return q.to(f) * s.to(f).repeat_interleave(128, 0)


def _swiglu(z, f):
    g, u = z[:, 0::2].to(f), z[:, 1::2].to(f)
    return g / (1 + torch.exp(-g)) * u


# ------------------------------------------------------------------------------------------------ inputs
def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _randn(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda").mul_(scale)


def _weight(g, E, N, K):
    w = torch.empty(E, N, K, dtype=torch.bfloat16, device="cuda")
    for e in range(E):
        w[e] = _randn(g, N, K, scale=1 / math.sqrt(K))
    return w


def _shares(g, E, skew):
    """How a trained router's tokens spread over the experts: Zipf(skew) in a random order."""
    p = torch.arange(1, E + 1, dtype=torch.float64) ** -skew
    return (p / p.sum())[torch.randperm(E, generator=g)]


def _segments(case, seed):
    """Live rows of each expert, and the rows of the table that holds them, from the seed alone."""
    g = torch.Generator().manual_seed(seed)
    counts = torch.bincount(torch.multinomial(_shares(g, case["E"], case["skew"]), case["rows"], True, generator=g),
                            minlength=case["E"])
    efo = torch.zeros(case["E"] + 1, dtype=torch.int64)
    efo[1:] = ((counts + 127) // 128 * 128).cumsum(0)
    return counts, efo


def prepare(case, seed):
    kind = case["kind"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    if kind.startswith("route"):
        T, E, K = case["T"], case["E"], case["K"]
        st = dict(case=case, logits=_randn(g, T, E, scale=1.5).to(_dtype(case)),
                  bias=_randn(g, E, scale=0.05) if case["bias"] else None)
        if kind == "route_train":
            st["dscores"] = _randn(g, T, K)
            st["logits"].requires_grad_(True)
        return st
    if kind == "quant_weight":
        return dict(case=case, w=_weight(g, case["E"], case["N"], case["K"]))
    if kind == "quant_rows":
        return dict(case=case, x=_randn(g, case["rows"], case["K"]).to(torch.bfloat16))
    if kind in ("linear", "linear_train"):
        E, N, K = case["E"], case["N"], case["K"]
        st = dict(case=case, w=_weight(g, E, N, K))
        if E == 1:                                                 # one projection: every row is live
            rows, st["efo"], st["counts"], cap = case["rows"], None, None, case["rows"]
            st["place"] = torch.arange(rows, device="cuda")
            st["live"] = torch.ones(rows, dtype=torch.bool, device="cuda")
        else:
            counts, efo = _segments(case, seed)
            rows, cap = _up(case["rows"]) + 128 * E, int((counts.max() + 127) // 128 * 128)   # what the routing table is allocated
            at = torch.arange(rows)
            e = torch.searchsorted(efo[1:], at, right=True)
            inside = e < E
            e = e.clamp(max=E - 1)
            r = at - efo[e]
            st.update(efo=efo.int().cuda(), counts=counts.int().cuda(), live=(inside & (r < counts[e])).cuda(),
                      place=torch.where(inside, e * cap + r, E * cap).cuda())
        st["cap"] = cap
        st["x"] = _randn(g, rows, K).to(torch.bfloat16)
        st["x"][~st["live"]] = 0
        if kind == "linear":
            st["w_fp8"] = _quant_weight(st.pop("w"), torch.float32)
        else:
            st["dy"] = _randn(g, rows, N).to(torch.bfloat16)
            st["x"].requires_grad_(True)
            st["w"].requires_grad_(True)
        return st
    T, E, H, I, K = case["T"], case["E"], case["H"], case["I"], case["topk"]
    gc = torch.Generator().manual_seed(seed)
    logits = _randn(g, T, E) + _shares(gc, E, case["skew"]).log().float().cuda() * 1.5
    scores, idx = logits.softmax(-1).topk(K, dim=-1)
    at, cap = _places(idx, E)
    return dict(case=case, x=_randn(g, T, H).to(torch.bfloat16), idx=idx.int(), scores=scores / scores.sum(-1, keepdim=True),
                w1=_quant_weight(_weight(g, E, 2 * I, H), torch.float32), w2=_quant_weight(_weight(g, E, H, I), torch.float32),
                at=at, cap=cap)


def _places(idx, E):
    """A place in an [E, cap] table for each entry of idx, by the experts' own order of tokens."""
    flat = idx.flatten().long()
    order = flat.argsort(stable=True)
    counts = torch.bincount(flat, minlength=E)
    rank = torch.empty_like(flat)
    rank[order] = torch.arange(flat.numel(), device=flat.device) - (counts.cumsum(0) - counts)[flat[order]]
    cap = max(1, int(counts.max()))
    return flat * cap + rank, cap


# ------------------------------------------------------------------------------------------------ the plain forms
def _route(logits, bias, case):
    """Scores, experts, and what the gradient needs; in 64 bits, since a border between two experts may be as near as that."""
    T, E = logits.shape
    K, G, n = case["K"], case["groups"], case["groups"] and case["E"] // case["groups"]
    x = logits.detach().double()
    open_ = x != -math.inf
    s = torch.sigmoid(x) if case["score"] == "sigmoid" else torch.softmax(x, -1)
    c = s + bias.double() if bias is not None else s
    order = c if bias is not None else x                           # without a bias the logits say it, the scores follow them
    low = -torch.finfo(torch.float64).max
    order = torch.where(open_, torch.nan_to_num(order, nan=low, neginf=low), -math.inf)
    if G > 1:
        m = min(case["group_score"], n)
        by = torch.where(open_, torch.nan_to_num(c, nan=low, neginf=low), -math.inf) if m > 1 else order
        best = by.view(T, G, n).topk(m, dim=-1).values
        rank = torch.where(torch.isinf(best) & (best < 0), 0.0, best).sum(-1)
        rank = torch.where(open_.view(T, G, n).any(-1), rank, -math.inf)
        chosen = rank.sort(dim=-1, descending=True, stable=True).indices[:, :case["top_groups"]]
        keep = torch.zeros(T, G, dtype=torch.bool, device=x.device).scatter_(1, chosen, True)
        order = torch.where(keep[:, :, None].expand(T, G, n).reshape(T, E), order, -math.inf)
    val, idx = order.sort(dim=-1, descending=True, stable=True)
    val, idx = val[:, :K], idx[:, :K]
    real = val > -math.inf
    sk = torch.where(real, s.gather(1, idx), 0.0)
    total = sk.sum(-1, keepdim=True) + 1e-20 if case["normalize"] else torch.ones(T, 1, dtype=x.dtype, device=x.device)
    return sk / total * case["scale"], torch.where(real, idx, -1), s, sk, total, idx, real


def _route_backward(dw, case, s, sk, total, idx, real):
    dw = torch.where(real, dw.double(), 0.0)
    ds = dw * case["scale"] / total
    if case["normalize"]:
        ds = ds - (ds * sk).sum(-1, keepdim=True) / total
    full = torch.zeros_like(s).scatter_add_(1, idx, torch.where(real, ds, 0.0))
    if case["score"] == "sigmoid":
        return full * s * (1 - s)
    return s * (full - (full * s).sum(-1, keepdim=True))


def _product(x, w, place, E, cap):
    """Rows of x times the transpose of their experts' w [E, N, K]: one batched product over an [E, cap] table; the place E * cap
    is that of the rows behind the last segment."""
    y = torch.bmm(_table(x, place, E, cap), w.transpose(1, 2)).flatten(0, 1)
    return torch.cat([y, y.new_zeros(1, y.shape[1])])[place]


def _table(x, place, E, cap):
    table = x.new_zeros(E * cap + 1, x.shape[1])
    table[place] = x
    return table[:-1].view(E, cap, -1)


def _linear(st, f, train):
    case, live, place, cap = st["case"], st["live"], st["place"], st["cap"]
    E = case["E"]
    x = st["x"].detach()
    wq, ws = _quant_weight(st["w"].detach(), f) if train else st["w_fp8"]
    w = _deq_weight(wq, ws, f)
    zero = torch.zeros((), dtype=f, device=x.device)
    y = _product(_deq_rows(*_quant_rows(x, f), f), w, place, E, cap)
    y = torch.where(live[:, None], y, zero)
    if not train:
        return (y,)
    dy = torch.where(live[:, None], st["dy"].to(f), zero)
    dx = _product(_deq_rows(*_quant_rows(dy, f), f), w.transpose(1, 2), place, E, cap)
    dx = torch.where(live[:, None], dx, zero)
    dyc, xc = (_deq_cols(*_quant_cols(_whole(t, live, f), f), f) for t in (dy, x))
    at = place if E > 1 else torch.arange(dyc.shape[0], device=x.device)
    dw = torch.bmm(_table(dyc, at, E, _up(cap)).transpose(1, 2), _table(xc, at, E, _up(cap)))
    return y, dx, dw


def _up(n):
    return (n + 127) // 128 * 128


def _whole(t, live, f):
    """Live rows, the others and those up to the next multiple of 128 zero."""
    t = torch.where(live[:, None], t.to(f), torch.zeros((), dtype=f, device=t.device))
    return torch.cat([t, t.new_zeros(_up(t.shape[0]) - t.shape[0], t.shape[1])])


def _experts(st, f):
    case, at, cap = st["case"], st["at"], st["cap"]
    T, E, K = case["T"], case["E"], case["topk"]
    xq = _deq_rows(*_quant_rows(st["x"], f), f).repeat_interleave(K, 0)
    z = _product(xq, _deq_weight(*st["w1"], f), at, E, cap).to(torch.bfloat16)       # the products leave bf16
    y = _deq_rows(*_quant_rows(_swiglu(z, f), f), f)
    o = _product(y, _deq_weight(*st["w2"], f), at, E, cap).to(torch.bfloat16)
    return (o.to(f).view(T, K, -1) * st["scores"].to(f)[:, :, None]).sum(1)


def _plain(st):
    case, f = st["case"], torch.float32
    kind = case["kind"]
    if kind.startswith("route"):
        r = _route(st["logits"], st["bias"], case)
        out = [r[0].float(), r[1].int()]
        if kind == "route_train":
            out.append(_route_backward(st["dscores"], case, *r[2:]).to(st["logits"].dtype))
        return out
    if kind == "quant_weight":
        return list(_quant_weight(st["w"], f))
    if kind == "quant_rows":
        return list(_quant_rows(_swiglu(st["x"], f) if case["swiglu"] else st["x"], f))
    if kind == "linear":
        return [_linear(st, f, False)[0].to(torch.bfloat16)]
    if kind == "linear_train":
        return [t.to(torch.bfloat16) for t in _linear(st, f, True)]
    return [_experts(st, f).to(torch.bfloat16)]


def _package():
    """The framework: nothing but its own calls needs it."""
    at = os.path.join(os.getcwd(), "supersonic-moe_b200")
    if at not in sys.path:
        sys.path.insert(1, at)
    import sonicmoe
    return sonicmoe


def run(state):
    if not own:
        return _plain(state)
    sonicmoe = sys.modules.get("sonicmoe") or _package()
    case = state["case"]
    kind = case["kind"]
    if kind.startswith("route"):
        scores, idx = sonicmoe.group_limited_routing(
            state["logits"], case["K"], score=case["score"], bias=state["bias"], groups=case["groups"],
            top_groups=case["top_groups"], group_score=case["group_score"], normalize=case["normalize"], scale=case["scale"])
        if kind == "route":
            return [scores, idx]
        return [scores.detach(), idx, *torch.autograd.grad(scores, state["logits"], state["dscores"])]
    if kind == "quant_weight":
        return list(sonicmoe.quantize_weight_block128(state["w"]))
    if kind == "quant_rows":
        return list(sonicmoe.quantize_rows_block128(state["x"], swiglu=case["swiglu"]))
    if kind == "linear":
        with torch.no_grad():
            return [sonicmoe.block128_linear(state["x"], state["w_fp8"], state["efo"], state["counts"])]
    if kind == "linear_train":
        y = sonicmoe.block128_linear(state["x"], state["w"], state["efo"], state["counts"])
        return [y.detach(), *torch.autograd.grad(y, (state["x"], state["w"]), state["dy"])]
    return [sonicmoe.block128_experts(state["x"], state["idx"], state["scores"], state["w1"], state["w2"])]


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind.startswith("route"):
        T, E, K = case["T"], case["E"], case["K"]
        es = 2 if case["dtype"] == "bf16" else 4
        b, fl = T * E * es + 8 * T * K + (4 * E if case["bias"] else 0), 6 * T * E
        if kind == "route_train":
            b, fl = b + T * E * es + 4 * T * K, fl + 4 * T * E
        return {"bytes": b, "flops": fl}
    if kind == "quant_weight":
        n = case["E"] * case["N"] * case["K"]
        return {"bytes": 3 * n + 4 * case["E"] * -(-case["N"] // 128) * -(-case["K"] // 128), "flops": 2 * n}
    if kind == "quant_rows":
        rows, out = case["rows"], case["K"] // 2 if case["swiglu"] else case["K"]
        return {"bytes": rows * (2 * case["K"] + out + 4 * -(-out // 128)), "flops": 2 * rows * out}
    if kind in ("linear", "linear_train"):
        E, N, K, rows = case["E"], case["N"], case["K"], case["rows"]
        if kind == "linear":
            return {"bytes": min(E, rows) * N * K + 2 * rows * (N + K), "flops": 2 * rows * N * K}
        return {"bytes": 2 * 2 * E * N * K + 2 * rows * (2 * N + 2 * K), "flops": 6 * rows * N * K}
    E, H, I, T, K = case["E"], case["H"], case["I"], case["T"], case["topk"]
    return {"bytes": min(E, T * K) * 3 * H * I + 4 * T * H + 8 * T * K, "flops": 6 * T * K * H * I}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """The definitions with numpy-like loops over experts, apart from the plain form above: groups one at a time, products one
    expert at a time.  Quantised values are those of the definition, so they are the same numbers in any precision."""
    kind, D = case["kind"], torch.float64
    st = prepare(case, seed)

    def quotients(m):
        """A group's scale and multiplier: 32-bit numbers by definition."""
        m = m.float()
        top = torch.full_like(m, 448.0)
        return (m / top).double(), (top / m).double()

    def groups_of(v, size):
        """[(first, last, scale, multiplier)] along the last dimension of v."""
        out = []
        for a in range(0, v.shape[-1], size):
            m = v[..., a:a + size].abs().amax(-1).clamp(min=TINY)
            s, inv = quotients(m)
            out.append((a, min(a + size, v.shape[-1]), s, inv))
        return out

    def held(v):
        """What e4m3 holds of values that were multiplied in 32 bits."""
        return v.float().to(torch.float8_e4m3fn).double()

    def rows_held(v):
        """Values that a row quantiser's output stands for, its payload, its scales."""
        v, q, scales = v.double(), torch.empty_like(v, dtype=D), []
        deq = torch.empty_like(q)
        for a, b, s, inv in groups_of(v, 128):
            q[..., a:b] = held(v[..., a:b] * inv[..., None])
            deq[..., a:b] = q[..., a:b] * s[..., None]
            scales.append(s)
        return deq, q, torch.stack(scales, -1)

    def weight_held(w):
        q, s = torch.empty_like(w, dtype=D), w.new_zeros(-(-w.shape[0] // 128), -(-w.shape[1] // 128), dtype=D)
        deq = torch.empty_like(q)
        for i in range(s.shape[0]):
            for j in range(s.shape[1]):
                r, c = slice(128 * i, 128 * i + 128), slice(128 * j, 128 * j + 128)
                s[i, j], inv = quotients(w[r, c].abs().amax().float().clamp(min=TINY))
                q[r, c] = held(w[r, c].double() * inv)
                deq[r, c] = q[r, c] * s[i, j]
        return deq, q, s

    if kind.startswith("route"):
        x = st["logits"].detach().double()
        e = torch.exp(x - x.amax(-1, keepdim=True))
        s = 1 / (1 + torch.exp(-x)) if case["score"] == "sigmoid" else e / e.sum(-1, keepdim=True)
        c = s + (st["bias"].double() if st["bias"] is not None else 0)
        key = c if st["bias"] is not None else x
        T, E, G, K = case["T"], case["E"], case["groups"], case["K"]
        n = E // G
        m = min(case["group_score"], n)
        gs = torch.stack([(key if m == 1 else c)[:, a * n:(a + 1) * n].sort(-1, descending=True).values[:, :m].sum(-1)
                          for a in range(G)], 1)
        ahead = torch.stack([((gs > gs[:, a:a + 1]).sum(1) + (gs[:, :a] == gs[:, a:a + 1]).sum(1)) for a in range(G)], 1)
        key = key.masked_fill((ahead >= case["top_groups"]).repeat_interleave(n, 1), -math.inf)
        idx = torch.empty(T, K, dtype=torch.int64, device=x.device)
        for k in range(K):                                         # the best of what is left; the first of equal ones
            best = key == key.amax(-1, keepdim=True)
            idx[:, k] = best.int().argmax(-1)
            key = key.scatter(1, idx[:, k:k + 1], -math.inf)
        sk = s.gather(1, idx)
        d = sk.sum(-1, keepdim=True) + 1e-20 if case["normalize"] else torch.ones_like(sk[:, :1])
        out = [case["scale"] * sk / d, idx.int()]
        if kind == "route_train":
            dw = case["scale"] * st["dscores"].double()
            ds = (dw - (dw * sk).sum(-1, keepdim=True) / d) / d if case["normalize"] else dw
            if case["score"] == "sigmoid":
                grad = torch.zeros_like(s).scatter_(1, idx, ds * sk * (1 - sk))
            else:
                grad = (torch.zeros_like(s).scatter_(1, idx, ds * sk)) - s * (ds * sk).sum(-1, keepdim=True)
            out.append(grad)
        return out
    if kind == "quant_weight":
        if case["E"] * case["N"] * case["K"] > 2 << 26:
            return None
        parts = [weight_held(w)[1:] for w in st["w"]]
        return [torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts])]
    if kind == "quant_rows":
        x = st["x"].double()
        if case["swiglu"]:
            gate, up = x[:, ::2], x[:, 1::2]
            x = gate * up / (1 + (-gate).exp())
        return list(rows_held(x)[1:])
    if kind in ("linear", "linear_train"):
        x, live = st["x"].detach(), st["live"].cpu()
        train = kind == "linear_train"
        E = case["E"]
        starts = [0] if E == 1 else st["efo"][:-1].tolist()
        counts = [case["rows"]] if E == 1 else st["counts"].tolist()
        y = torch.zeros(x.shape[0], case["N"], dtype=D, device="cuda")
        dx, dw = torch.zeros(x.shape[0], case["K"], dtype=D, device="cuda"), []
        for e in range(E):
            r = slice(starts[e], starts[e] + counts[e])
            if train:
                w = weight_held(st["w"][e].detach())[0]
            else:
                sc = torch.kron(st["w_fp8"][1][e].double(), torch.ones(128, 128, dtype=D, device="cuda"))
                w = st["w_fp8"][0][e].double() * sc[:case["N"], :case["K"]]
            y[r] = rows_held(x[r])[0] @ w.T
            if train:
                dx[r] = rows_held(st["dy"][r])[0] @ w
                total = torch.zeros(case["N"], case["K"], dtype=D, device="cuda")
                for a in range(0, counts[e], 128):
                    t = slice(starts[e] + a, starts[e] + min(a + 128, counts[e]))
                    total += rows_held(st["dy"][t].T)[0] @ rows_held(x[t].T)[0].T
                dw.append(total)
        return [y, dx, torch.stack(dw)] if train else [y]
    x, K = rows_held(st["x"])[0], case["topk"]
    out = torch.zeros(case["T"], case["H"], dtype=D, device="cuda")
    flat = st["idx"].flatten().long()
    for e in range(case["E"]):
        hit = (flat == e).nonzero().flatten()
        if hit.numel() == 0:
            continue
        t = hit // K
        ones = torch.ones(128, 128, dtype=D, device="cuda")
        w1, w2 = (q[e].double() * torch.kron(s[e].double(), ones)[:q.shape[1], :q.shape[2]] for q, s in (st["w1"], st["w2"]))
        z = (x[t] @ w1.T).to(torch.bfloat16).double()              # the definition has bf16 between the products
        gate, up = z[:, ::2], z[:, 1::2]
        o = rows_held(gate * up / (1 + (-gate).exp()))[0] @ w2.T
        out.index_add_(0, t, o.to(torch.bfloat16).double() * st["scores"].flatten()[hit].double()[:, None])
    return [out]
