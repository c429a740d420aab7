"""Products with one scale per block of 128, on CPU: the quantisers' rule in f32 (its definition), products in 64 bits."""
import torch

TINY = torch.tensor(2.0 ** -100)


def _held(x, amax):
    """e4m3 payload and scale of values under a maximum that broadcasts against them."""
    a = torch.maximum(torch.nan_to_num(amax.float(), nan=0.0, posinf=float("inf")), TINY)
    top = torch.full_like(a, 448.0)                            # a quotient of tensors is rounded once, one with a number may not be
    v = (x.float() * (top / a)).clamp(-448, 448)              # saturating
    return v.to(torch.float8_e4m3fn), a / top


def _amax(x, dim):
    return torch.where(torch.isnan(x), torch.zeros((), dtype=x.dtype), x.abs()).amax(dim)


def quant_rows(x):
    rows, K = x.shape
    q, s = torch.empty(rows, K, dtype=torch.float8_e4m3fn), torch.empty(rows, -(-K // 128))
    for b in range(s.shape[1]):
        c = slice(128 * b, min(128 * b + 128, K))
        q[:, c], sc = _held(x[:, c], _amax(x[:, c], 1)[:, None])
        s[:, b] = sc[:, 0]
    return q, s


def quant_weight(w):
    E, N, K = w.shape
    q, s = torch.empty(E, N, K, dtype=torch.float8_e4m3fn), torch.empty(E, -(-N // 128), -(-K // 128))
    for e in range(E):
        for i in range(s.shape[1]):
            for j in range(s.shape[2]):
                r, c = slice(128 * i, 128 * i + 128), slice(128 * j, 128 * j + 128)
                q[e, r, c], s[e, i, j] = _held(w[e, r, c], _amax(w[e, r, c].flatten(), 0))
    return q, s


def quant_cols(x, live=None):
    """x [rows,K] -> payload [rows,K], scales [rows/128,K]; rows that are not live are zero."""
    rows, K = x.shape
    x = x if live is None else torch.where(live[:, None], x, torch.zeros((), dtype=x.dtype))
    q, s = torch.empty(rows, K, dtype=torch.float8_e4m3fn), torch.empty(-(-rows // 128), K)
    for b in range(s.shape[0]):
        r = slice(128 * b, min(128 * b + 128, rows))
        q[r], sc = _held(x[r], _amax(x[r], 0)[None])
        s[b] = sc[0]
    return q, s


def deq_rows(q, s):
    return q.double() * s.double().repeat_interleave(128, 1)[:, :q.shape[1]]


def deq_weight(q, s):
    return q.double() * s.double().repeat_interleave(128, 1)[:, :q.shape[1]].repeat_interleave(128, 2)[:, :, :q.shape[2]]


def deq_cols(q, s):
    return q.double() * s.double().repeat_interleave(128, 0)[:q.shape[0]]


def segments(efo, counts, rows):
    """(expert, first row, end of the live rows) of each segment."""
    if efo is None:
        return [(0, 0, rows)]
    return [(e, int(efo[e]), int(efo[e]) + int(counts[e]) if counts is not None else int(efo[e + 1])) for e in range(len(efo) - 1)]


def live_rows(efo, counts, rows):
    live = torch.zeros(rows, dtype=torch.bool)
    for _, a, b in segments(efo, counts, rows):
        live[a:b] = True
    return live


def rows_product(x, w, efo, counts):
    """x [rows,K], w [E,N,K] in 64 bits -> (products, sums of the magnitudes of their terms); zero where no row is live."""
    y = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(y)
    for e, a, b in segments(efo, counts, x.shape[0]):
        y[a:b], mag[a:b] = x[a:b] @ w[e].T, x[a:b].abs() @ w[e].abs().T
    return y, mag


def cols_product(a, b, efo, counts, E):
    """a [rows,M], b [rows,N] -> (products [E,M,N] of each segment's live rows, magnitudes)."""
    c = torch.zeros(E, a.shape[1], b.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(c)
    for e, i, j in segments(efo, counts, a.shape[0]):
        c[e], mag[e] = a[i:j].T @ b[i:j], a[i:j].abs().T @ b[i:j].abs()
    return c, mag


def swiglu(z):
    g, u = z[:, 0::2].double(), z[:, 1::2].double()
    return g / (1 + torch.exp(-g)) * u
