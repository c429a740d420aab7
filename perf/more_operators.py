"""What the operators around the experts of this repository are judged by: the norm in front of the layer, products grouped by
expert in bf16, and the norm and clipping of the gradients behind it.  One pass of a case is one call of the public API as a
program that trains or serves a Mixture-of-Experts layer makes it.

A case is a dict of plain values.  `kind` says which operator, and how it is used:

  norm           `rms_norm`: residual added, the sum and its norm returned
  norm_train     the same with its backward pass: also the gradients of x and of the weight
  norm_quant     `rms_norm_quantized`: the norm as the 8-bit payload and scales that the experts take, with or without the bf16
                 rows that the router takes
  grouped        `grouped_linear`: y = x W^T by segments of rows, nothing saved
  grouped_train  the same with its backward pass: y and the gradients of x and W
  grad_norm      `gradient_norm` of a list of gradients
  clip           `clip_gradients` of a list of gradients into other tensors

A segment is the run of rows of one expert.  `padded`: segments start at multiples of 128 rows, as the routing metadata leaves
them, and the rows in between are nobody's; otherwise they follow one another wherever they end.
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-6
E4M3_MAX = 448.0


def listed():
    return [
        # one decoded token in front of a layer: residual stream, router rows and MXFP8 payload; latency
        dict(name="norm_quant_1", kind="norm_quant", T=1, H=4096, residual="bf16", scales="mx", rows_too=True),
        # a prompt in front of a layer
        dict(name="norm_quant_8192", kind="norm_quant", T=8192, H=4096, residual="bf16", scales="mx", rows_too=True),
        # a ragged batch with a residual stream in 32 bits, scales per 128, a last block of 104 columns, payload alone
        dict(name="norm_quant_odd_3001", kind="norm_quant", T=3001, H=1000, residual="f32", scales="block128", rows_too=False),
        # a training step's norm in front of the fine-grained layer
        dict(name="norm_train_16384", kind="norm_train", T=16384, H=2048, x="bf16", residual="bf16", weight="bf16"),
        # 32-bit rows of an odd width, no residual
        dict(name="norm_train_odd_1003", kind="norm_train", T=1003, H=1001, x="f32", residual=None, weight="f32"),
        # one token through a dense projection: weights from HBM, latency
        dict(name="grouped_1", kind="grouped", E=1, N=4096, K=4096, rows=1, skew=0.0, padded=False),
        # one decode step of 64 tokens x 8 through 128 fine-grained experts
        dict(name="grouped_decode_512", kind="grouped", E=128, N=1536, K=2048, rows=512, skew=0.0, padded=False),
        # a training step of one expert projection under a skewed router
        dict(name="grouped_train_16384", kind="grouped_train", E=8, N=4096, K=2048, rows=16384, skew=0.6, padded=False),
        # the same for few experts of sizes that no tile divides, over the routing metadata's padded segments
        dict(name="grouped_train_odd_700", kind="grouped_train", E=5, N=1000, K=720, rows=700, skew=1.2, padded=True),
        # every weight gradient of a model of a few small layers, odd sizes, before an optimizer step
        dict(name="grad_norm_many", kind="grad_norm", shapes="small", tensors=300, types="mixed"),
        # the f32 accumulators of a layer of 128 experts, its router and norms, clipped into bf16 gradients
        dict(name="clip_experts", kind="clip", shapes="experts", tensors=8, types="f32", out="bf16", E=128, H=2048, I=768,
             max_norm=1.0),
        # the same accumulators of a small model, left in 32 bits
        dict(name="clip_small", kind="clip", shapes="small", tensors=40, types="f32", out="f32", max_norm=0.5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("norm", "norm_train", "norm_quant", "norm_quant", "grouped", "grouped", "grouped_train", "grouped_train",
                       "grad_norm", "clip"))
    if kind in ("norm", "norm_train"):
        x = rng.choice(("bf16", "bf16", "f32"))
        residual = rng.choice((None, x, "f32"))
        return dict(kind=kind, T=_log(rng, 1, 16384), H=rng.choice((1, 8, 8)) * _log(rng, 16, 768), x=x, residual=residual,
                    weight=rng.choice(("bf16", "f32")))
    if kind == "norm_quant":
        scales = rng.choice(("mx", "block128"))
        H = 32 * _log(rng, 2, 192) if scales == "mx" else 8 * _log(rng, 4, 768)
        return dict(kind=kind, T=_log(rng, 1, 16384), H=H, residual=rng.choice((None, "bf16", "f32")), scales=scales,
                    rows_too=rng.random() < 0.5)
    if kind in ("grouped", "grouped_train"):
        E = rng.choice((1, 5, 8, 37, 128))
        wide = E <= 8
        N, K = 8 * _log(rng, 8, 512 if wide else 192), 8 * _log(rng, 8, 256)
        return dict(kind=kind, E=E, N=N, K=K, rows=_log(rng, 1, 16384), skew=rng.choice((0.0, 0.6, 1.2)), padded=rng.random() < 0.3)
    case = dict(kind=kind, shapes="small", tensors=_log(rng, 1, 600), types=rng.choice(("f32", "bf16", "mixed")))
    if rng.random() < 0.3:
        case.update(shapes="experts", tensors=8, E=rng.choice((8, 32, 64)), H=64 * rng.randint(4, 32), I=64 * rng.randint(2, 12))
    if kind == "clip":
        case.update(out=rng.choice(("f32", "bf16")), max_norm=rng.choice((0.1, 1.0, 1e6)))
    return case


# ------------------------------------------------------------------------------------------------ inputs
_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _randn(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda").mul_(scale)


def _shares(case, seed):
    """How a trained router's tokens spread over the experts: Zipf(skew) in a random order."""
    g = torch.Generator().manual_seed(seed)
    p = torch.arange(1, case["E"] + 1, dtype=torch.float64) ** -case["skew"]
    return (p / p.sum())[torch.randperm(case["E"], generator=g)], g


def _segments(case, seed):
    """First rows, live rows, and the rows of the table, from the seed alone."""
    p, g = _shares(case, seed)
    counts = torch.bincount(torch.multinomial(p, case["rows"], True, generator=g), minlength=case["E"]).tolist()
    step = 128 if case["padded"] else 1
    starts, at = [], 0
    for n in counts:
        starts.append(at)
        at += -(-n // step) * step
    return starts + [at], counts, -(-case["rows"] // 128) * 128 + 128 * case["E"] if case["padded"] else at    # as allocated


def _gradient_shapes(case):
    """Shapes and types of a list of gradients: the model's, whatever its values are."""
    if case["shapes"] == "experts":
        E, H, I = case["E"], case["H"], case["I"]
        shapes = [(E, 2 * I, H), (E, H, I), (E, H), (H,), (H,), (H, H), (H,), (E,)][:case["tensors"]]
    else:
        g = torch.Generator().manual_seed(case["tensors"])
        shapes = []
        for i in range(case["tensors"]):
            n = int(torch.randint(1, 700, (1,), generator=g))
            shapes.append((n,) if i % 3 == 0 else (n, int(torch.randint(1, 900, (1,), generator=g))))
    kinds = [torch.float32, torch.bfloat16]
    return [(s, kinds[i % 2] if case["types"] == "mixed" else _TYPES[case["types"]]) for i, s in enumerate(shapes)]


def prepare(case, seed):
    kind = case["kind"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    if kind.startswith("norm"):
        T, H = case["T"], case["H"]
        tx = _TYPES[case.get("x", "bf16")]
        st = dict(case=case, x=_randn(g, T, H).to(tx),
                  weight=(1 + _randn(g, H, scale=0.2)).to(_TYPES[case.get("weight", "bf16")]),
                  residual=_randn(g, T, H, scale=3.0).to(_TYPES[case["residual"]]) if case["residual"] else None)
        if kind == "norm_train":
            st["dy"] = _randn(g, T, H).to(tx)
            st["dh"] = _randn(g, T, H).to(st["residual"].dtype) if case["residual"] else None
            st["x"].requires_grad_(True)
            st["weight"].requires_grad_(True)
        return st
    if kind.startswith("grouped"):
        E, N, K = case["E"], case["N"], case["K"]
        starts, counts, rows = _segments(case, seed)
        w = torch.empty(E, N, K, dtype=torch.bfloat16, device="cuda")
        for e in range(E):
            w[e] = _randn(g, N, K, scale=1 / math.sqrt(K))
        st = dict(case=case, w=w, x=_randn(g, rows, K).to(torch.bfloat16), starts=starts, live=counts,
                  efo=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                  counts=torch.tensor(counts, dtype=torch.int32, device="cuda") if case["padded"] else None)
        if kind == "grouped_train":
            st["dy"] = _randn(g, rows, N).to(torch.bfloat16)
            st["x"].requires_grad_(True)
            st["w"].requires_grad_(True)
        return st
    grads = [_randn(g, *s, scale=1e-2).to(t) for s, t in _gradient_shapes(case)]
    st = dict(case=case, grads=grads)
    if kind == "clip":
        st["out"] = [torch.empty(t.shape, dtype=_TYPES[case["out"]], device="cuda") for t in grads]
    return st


# ------------------------------------------------------------------------------------------------ the plain forms
def _norm(st, f):
    """h of its own type; r and y before rounding, in f."""
    x, res = st["x"].detach(), st["residual"]
    h = x if res is None else (x.to(f) + res.to(f)).to(res.dtype)
    hf = h.to(f)
    r = 1 / torch.sqrt((hf * hf).mean(-1, keepdim=True) + EPS)
    return h, r, hf * r * st["weight"].detach().to(f)


def _bf16(v):
    """The bf16 nearest to each f64, without a stop in f32 that may turn a value beside a border into one on it."""
    f = v.float()
    bits = f.view(torch.int32)
    side = (v.abs() - f.double().abs()).sign().int()
    return torch.where((bits & 0xFFFF) == 0x8000, bits + side, bits).view(torch.float32).to(torch.bfloat16)


def _norm_train(st, f):
    h, r, y = _norm(st, f)
    hf, dy = h.to(f), st["dy"].to(f)
    g = dy * st["weight"].detach().to(f)
    dx = r * (g - hf * (r * r * (g * hf).mean(-1, keepdim=True)))
    if st["dh"] is not None:
        dx = dx + st["dh"].to(f)
    return h, y, dx, (dy * hf * r).sum(0)


def _mx_exponents(amax):
    """Biased exponents of the scales of groups with these largest magnitudes, and what the values are multiplied by."""
    bits = amax.float().view(torch.int32)
    e = (bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()
    e = torch.where((bits >> 23) > 0, e.clamp(min=0), 0)
    return e.to(torch.uint8), torch.ldexp(torch.ones_like(amax, dtype=torch.float32), 127 - e)


def _payload(y, scales):
    """bf16 rows -> e4m3 rows and scales."""
    T, H = y.shape
    size = 32 if scales == "mx" else 128
    v = torch.cat([y.float(), y.new_zeros(T, -H % size, dtype=torch.float32)], 1).view(T, -1, size)
    amax = v.abs().amax(2)
    if scales == "mx":
        s, inv = _mx_exponents(amax)
    else:
        amax = amax.clamp(min=2.0 ** -100)
        most = torch.full_like(amax, E4M3_MAX)         # a quotient of tensors is rounded once, one with a number may not be
        s, inv = amax / most, most / amax
    q = (v * inv[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q.view(T, -1)[:, :H].contiguous(), s


def _grouped(st, f, train):
    case, x, w = st["case"], st["x"].detach(), st["w"].detach()
    y = torch.zeros(x.shape[0], case["N"], dtype=f, device=x.device)
    dx = torch.zeros(x.shape[0], case["K"], dtype=f, device=x.device) if train else None
    dw = torch.zeros(w.shape, dtype=f, device=x.device) if train else None
    for e, n in enumerate(st["live"]):
        if n:
            r = slice(st["starts"][e], st["starts"][e] + n)
            we = w[e].to(f)
            y[r] = x[r].to(f) @ we.T
            if train:
                dy = st["dy"][r].to(f)
                dx[r] = dy @ we
                dw[e] = dy.T @ x[r].to(f)
    return y, dx, dw


def _squares(grads):
    total = torch.zeros((), dtype=torch.float64, device="cuda")
    for t in grads:
        total = total + t.float().square().sum(dtype=torch.float64)        # a long sum
    return total


def _plain(st):
    case, f = st["case"], torch.float32
    kind = case["kind"]
    if kind == "norm":
        h, _, y = _norm(st, f)
        return [y.to(st["x"].dtype)] + ([] if st["residual"] is None else [h])
    if kind == "norm_train":
        h, y, dx, dw = _norm_train(st, f)
        out = [y.to(st["x"].dtype), dx.to(st["x"].dtype), dw.to(st["weight"].dtype)]
        return out + ([] if st["residual"] is None else [h])
    if kind == "norm_quant":
        h, _, y = _norm(st, torch.float64)                      # which side of a border between two bf16 a value lies on
        y = _bf16(y)
        return [*_payload(y, case["scales"])] + ([y] if case["rows_too"] else []) + ([] if st["residual"] is None else [h])
    if kind == "grouped":
        return [_grouped(st, f, False)[0].to(torch.bfloat16)]
    if kind == "grouped_train":
        return [t.to(torch.bfloat16) for t in _grouped(st, f, True)]
    n = _squares(st["grads"]).sqrt()
    if kind == "grad_norm":
        return [n.float()]
    c = (case["max_norm"] / (n + 1e-6)).clamp(max=1.0)
    for o, t in zip(st["out"], st["grads"]):
        o.copy_(t.float() * c.float())
    return [n.float(), *st["out"]]


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
    if kind == "norm":
        with torch.no_grad():
            out = sonicmoe.rms_norm(state["x"], state["weight"], state["residual"], eps=EPS)
        return [out] if state["residual"] is None else list(out)
    if kind == "norm_train":
        out = sonicmoe.rms_norm(state["x"], state["weight"], state["residual"], eps=EPS)
        leaves = (state["x"], state["weight"])
        if state["residual"] is None:
            return [out.detach(), *torch.autograd.grad(out, leaves, state["dy"])]
        y, h = out
        return [y.detach(), *torch.autograd.grad((y, h), leaves, (state["dy"], state["dh"])), h.detach()]
    if kind == "norm_quant":
        with torch.no_grad():
            out = sonicmoe.rms_norm_quantized(state["x"], state["weight"], state["residual"], eps=EPS, scales=case["scales"],
                                              with_output=case["rows_too"])
        return [t for t in out if t is not None]
    if kind == "grouped":
        with torch.no_grad():
            return [sonicmoe.grouped_linear(state["x"], state["w"], state["efo"], state["counts"])]
    if kind == "grouped_train":
        y = sonicmoe.grouped_linear(state["x"], state["w"], state["efo"], state["counts"])
        return [y.detach(), *torch.autograd.grad(y, (state["x"], state["w"]), state["dy"])]
    if kind == "grad_norm":
        return [sonicmoe.gradient_norm(state["grads"])]
    return [sonicmoe.clip_gradients(state["grads"], case["max_norm"], out=state["out"]), *state["out"]]


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
_BYTES = {"bf16": 2, "f32": 4, None: 0}


def work(case):
    kind = case["kind"]
    if kind.startswith("norm"):
        T, H = case["T"], case["H"]
        bx, br = _BYTES[case.get("x", "bf16")], _BYTES[case["residual"]]
        b = T * H * (bx + 2 * br) + H * _BYTES[case.get("weight", "bf16")]
        if kind == "norm_quant":
            b += T * H + (T * -(-H // 32) if case["scales"] == "mx" else 4 * T * -(-H // 128)) + (2 * T * H if case["rows_too"] else 0)
            return {"bytes": b, "flops": 6 * T * H}
        b += T * H * bx
        if kind == "norm_train":
            b += T * H * (2 * bx + br) + H * _BYTES[case["weight"]]
            return {"bytes": b, "flops": 14 * T * H}
        return {"bytes": b, "flops": 5 * T * H}
    if kind.startswith("grouped"):
        E, N, K, rows = case["E"], case["N"], case["K"], case["rows"]
        p = [(i + 1) ** -case["skew"] for i in range(E)]
        busy = sum(1 - (1 - v / sum(p)) ** rows if E > 1 else 1 for v in p)        # experts that have rows, in the mean
        if kind == "grouped":
            return {"bytes": 2 * busy * N * K + 2 * rows * (N + K), "flops": 2 * rows * N * K}
        return {"bytes": 2 * busy * N * K + 2 * E * N * K + 4 * rows * (N + K), "flops": 6 * rows * N * K}
    n = read = written = 0
    for shape, t in _gradient_shapes(case):
        m = math.prod(shape)
        n, read = n + m, read + m * (4 if t == torch.float32 else 2)
        written += m * _BYTES[case.get("out")]
    return {"bytes": read + written, "flops": 3 * n if written else 2 * n}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """The definitions, apart from the plain forms above: rows through a linear-algebra view of the norm, products one expert at
    a time, payloads by their values."""
    kind, D = case["kind"], torch.float64
    st = prepare(case, seed)
    if kind.startswith("norm"):
        x, w = st["x"].detach().double(), st["weight"].detach().double()
        h, H = x, case["H"]
        if st["residual"] is not None:
            h = (x + st["residual"].double()).to(st["residual"].dtype).double()     # the sum is held in the residual's type
        length = (torch.linalg.vector_norm(h, dim=1, keepdim=True) ** 2 / H + EPS).sqrt()
        unit = h / length
        out = [unit * w]
        if kind == "norm_train":
            g = st["dy"].double() * w
            along = torch.einsum("th,th->t", g, unit)[:, None] / H
            dh = (g - unit * along) / length
            out += [dh if st["dh"] is None else dh + st["dh"].double(), torch.einsum("th,th->h", st["dy"].double(), unit)]
        if kind == "norm_quant":
            v = out.pop()                                            # the definition quantises bf16 rows: 8 bits of v, rounded once
            step = torch.ldexp(torch.ones_like(v), torch.frexp(v).exponent.clamp(min=-125) - 8)
            y = torch.round(v / step) * step
            size = 32 if case["scales"] == "mx" else 128
            q, scales = torch.empty_like(y), []
            for a in range(0, H, size):
                part = y[:, a:a + size]
                m = part.abs().amax(1)
                if case["scales"] == "mx":
                    # the power of two at which the largest magnitude is 448 or less: 448 = 1.75 * 2^8
                    e = torch.frexp(m).exponent - 1 + 127
                    e = (e - 8 + (m > 1.75 * torch.ldexp(torch.ones_like(m), torch.frexp(m).exponent - 1)).int()).clamp(min=0)
                    e = torch.where(m > 0, e, 0)
                    scales.append(e.to(torch.uint8))
                    inv = torch.ldexp(torch.ones_like(m), 127 - e)
                else:
                    m = m.float().clamp(min=2.0 ** -100)
                    top = torch.full_like(m, 448.0)
                    scales.append((m / top).double())
                    inv = (top / m).double()
                q[:, a:a + size] = (part * inv[:, None]).float().to(torch.float8_e4m3fn).double()
            out = [q, torch.stack(scales, 1)] + ([y] if case["rows_too"] else [])
        return out + ([] if st["residual"] is None else [h])
    if kind.startswith("grouped"):
        x, w = st["x"].detach(), st["w"].detach()
        train = kind == "grouped_train"
        owner = torch.full((x.shape[0],), -1)
        for e, n in enumerate(st["live"]):
            owner[st["starts"][e]:st["starts"][e] + n] = e
        owner = owner.cuda()
        y = torch.zeros(x.shape[0], case["N"], dtype=D, device="cuda")
        dx, dw = torch.zeros(x.shape[0], case["K"], dtype=D, device="cuda"), []
        for e in range(case["E"]):
            mine = (owner == e).nonzero().flatten()
            y[mine] = torch.einsum("rk,nk->rn", x[mine].double(), w[e].double())
            if train:
                dx[mine] = torch.einsum("rn,nk->rk", st["dy"][mine].double(), w[e].double())
                dw.append(torch.einsum("rn,rk->nk", st["dy"][mine].double(), x[mine].double()))
        return [y, dx, torch.stack(dw)] if train else [y]
    n = torch.stack([torch.linalg.vector_norm(t.double()) for t in st["grads"]]).square().sum().sqrt()
    if kind == "grad_norm":
        return [n]
    c = min(1.0, case["max_norm"] / (float(n) + 1e-6))
    return [n, *(c * t.double() for t in st["grads"])]
