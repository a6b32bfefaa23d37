"""The language-model operators in 64 bits, and bounds on how far 32-bit arithmetic may be from them.

Every function returns (value, bound) pairs of float64 tensors.  A bound follows the operator's own recurrences with
magnitudes in place of values; U is the largest relative rounding of a 32-bit operation.  What is counted:
  a gate and its complement: exp within 3 U (reduction, table, product), 1 + e, the reciprocal, a product: 6 U; for 16-bit
  rows exp2(fl(-|z| fl(log2 e))): the product is off by U, the constant by 0.23 U of itself, which moves the power by 1.23
  U |z|, on top of the exponential's 2 U, 1 + e, a reciprocal within 2 U and a product: (6 + 1.3 |z|) U
  a product or a sum: U each; a sum of n terms in any order: n U of the sum of magnitudes
and the output's own rounding, half a unit of its type, on top.  Terms of order U^2 are covered by the slack factor 1.01.
Every rule also allows the smallest numbers of the types to be flushed (TINY)."""
import torch

U = 2.0 ** -24
GATE = 6 * U
TINY = 1e-36
SLACK = 1.01


def out_round(value, bound, dtype):
    """the bound after one rounding to `dtype`: half a unit (and half the smallest subnormal of a half)"""
    half = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else TINY
    return value, SLACK * (bound + half * (value.abs() + bound)) + tiny


def embed(table, ids, scale, dtype):
    ok = (ids >= 0) & (ids < table.shape[0])
    scale = float(torch.tensor(scale, dtype=torch.float32))
    y = torch.zeros(ids.shape[0], table.shape[1], dtype=torch.float64)
    y[ok] = table.double()[ids[ok].long()] * scale
    return out_round(y, U * y.abs(), dtype)


def sum_by_word(ids, rows, bound, vocab):
    """sum of the rows (float64 [n, dim]; each within `bound` already) by word, the rounding of the products and of the sum"""
    ok = (ids >= 0) & (ids < vocab)
    at = ids[ok].long()
    zero = torch.zeros(vocab, rows.shape[1], dtype=torch.float64)
    value, mag, err = zero.clone(), zero.clone(), zero.clone()
    value.index_add_(0, at, rows[ok])
    mag.index_add_(0, at, rows[ok].abs())
    err.index_add_(0, at, bound[ok])
    count = torch.bincount(at, minlength=vocab).double()[:, None]
    return out_round(value, err + (count + 1) * U * mag, torch.float32)


def embed_grad(dy, ids, vocab, scale):
    scale = float(torch.tensor(scale, dtype=torch.float32))
    rows = dy.double() * scale
    return sum_by_word(ids, rows, torch.zeros_like(rows), vocab)


def _gates(gate):
    """a, 1 - a and the relative rounding of either (beyond |z| = 104 both are 0 or 1)"""
    z = gate.double()
    err = torch.full_like(z, GATE) if gate.dtype == torch.float32 else (6 + 1.3 * z.abs().clamp(max=104)) * U
    return torch.sigmoid(z), torch.sigmoid(-z), torch.nan_to_num(err)


def scan(gate, x, offsets, state, dtype, fill):
    """h (rows of no sentence: `fill`), last"""
    a, b, err = _gates(gate)
    xd = x.double()
    n, dim = len(offsets) - 1, x.shape[1]
    h = fill.double().clone()
    hb = torch.zeros_like(h)
    before, before_b, before_m = torch.zeros_like(h), torch.zeros_like(h), torch.zeros_like(h)
    last = torch.zeros(n, dim, dtype=torch.float64) if state is None else state.double().clone()
    last_b = torch.zeros_like(last)
    for i in range(n):
        v, e, m = last[i].clone(), torch.zeros(dim, dtype=torch.float64), last[i].abs()
        for t in range(int(offsets[i]), int(offsets[i + 1])):
            before[t], before_b[t], before_m[t] = v, e, m
            v = a[t] * v + b[t] * xd[t]
            m = a[t] * m + b[t] * xd[t].abs()
            # the gates, the products and the sum of this row; in chunks the products of gates are rounded once more
            e = a[t] * e + (err[t] + 4 * U) * m
            h[t], hb[t] = v, e
        last[i], last_b[i] = v, e
    return out_round(h, hb, dtype), out_round(last, last_b, torch.float32), (before, before_b, before_m)


def scan_grad(gate, x, offsets, state, dh, dlast, dtype, fill):
    """dgate, dx (rows of no sentence: `fill`), dstate"""
    _, _, (before, before_b, before_m) = scan(gate, x, offsets, state, torch.float32, fill)
    a, b, err = _gates(gate)
    xd, dhd = x.double(), dh.double()
    n, dim = len(offsets) - 1, x.shape[1]
    dgate, dx = fill.double().clone(), fill.double().clone()
    dgate_b, dx_b = torch.zeros_like(dx), torch.zeros_like(dx)
    ds = torch.zeros(n, dim, dtype=torch.float64) if dlast is None else dlast.double().clone()
    ds_b = torch.zeros_like(ds)
    for i in range(n):
        v, e, m = ds[i].clone(), torch.zeros(dim, dtype=torch.float64), ds[i].abs()
        for t in reversed(range(int(offsets[i]), int(offsets[i + 1]))):
            v, m = dhd[t] + v, dhd[t].abs() + m
            e = e + 2 * U * m
            dx[t], dx_b[t] = v * b[t], b[t] * (e + (err[t] + U) * m)
            ab, diff, span = a[t] * b[t], before[t] - xd[t], before_m[t] + xd[t].abs()
            dgate[t] = v * ab * diff
            dgate_b[t] = ab * (e * diff.abs() + m * before_b[t] + (2 * err[t] + 5 * U) * m * span)
            v, m, e = v * a[t], m * a[t], a[t] * (e + (err[t] + 3 * U) * m)
        ds[i], ds_b[i] = v, e
    return out_round(dgate, dgate_b, dtype), out_round(dx, dx_b, dtype), out_round(ds, ds_b, torch.float32)


def nce_score(h, table, ids, constant):
    vocab, dim = table.shape
    ok = (ids >= 0) & (ids < vocab)
    rows = table.double()[torch.where(ok, ids, torch.zeros_like(ids)).long()] if vocab else torch.zeros(*ids.shape, dim, dtype=torch.float64)
    rows = torch.where(ok[:, :, None], rows, torch.zeros(1, dtype=torch.float64))   # (row 0 may hold anything)
    constant = float(torch.tensor(constant, dtype=torch.float32))
    prod = rows * h.double()[:, None, :]
    s, m = prod.sum(-1), prod.abs().sum(-1)
    b = (dim + 1) * U * m + U * (s - constant).abs()
    value = torch.where(ok, s - constant, torch.full_like(s, -float('inf')))
    return value, torch.where(ok, SLACK * (b + U * m) + TINY, torch.zeros_like(b)), (s, b, rows, ok)


def nce_loss(h, table, ids, log_noise, constant, weight, dtype):
    vocab, dim = table.shape
    _, _, (s, sb, rows, ok) = nce_score(h, table, ids, constant)
    ok = ok & ok[:, :1]
    constant = float(torch.tensor(constant, dtype=torch.float32))
    safe = torch.where(ok, ids, torch.zeros_like(ids)).long()
    ln = log_noise.double()[safe] if vocab else torch.zeros_like(s)
    z = s - constant - ln
    # the kernel takes constant + log_noise off in one step
    zb = sb + U * (constant + ln).abs() + 2 * U * z.abs()
    sign = torch.ones_like(z)
    sign[:, 0] = -1
    w = torch.ones(h.shape[0], dtype=torch.float64) if weight is None else weight.double()
    l = torch.nn.functional.softplus(sign * z, threshold=1e9) * ok
    sg = torch.sigmoid(sign * z) * ok
    k = ids.shape[1]
    # softplus moves by at most sigmoid(z) for a unit of z; its own arithmetic: exp, logarithm (3 U of ln 2), sums
    lb = (sg * zb + (GATE + 4 * U) * l + 3 * U * ok) * ok
    loss = l.sum(1) * w
    loss_b = (lb.sum(1) + (k + 1) * U * l.sum(1)) * w.abs()
    g = sign * sg * w[:, None]
    # sigmoid' = sigmoid (1 - sigmoid) <= sigmoid
    gb = (sg * zb + (GATE + U) * sg) * w[:, None].abs() * ok
    # the one that 16-bit rows of dh are summed with: exp2(fl(-z fl(log2 e))) within (2 + 1.23 |z|) U, 1 + e, a reciprocal
    # within 2 U
    gb_dh = gb if dtype == torch.float32 else gb + 1.3 * z.abs().clamp(max=104) * U * sg * w[:, None].abs() * ok
    live = ok[:, 0]
    hd = torch.where(live[:, None], h.double(), torch.zeros(1, dtype=torch.float64))
    # (a row that does not count may hold anything in the table's or h's place)
    rows = torch.where(ok[:, :, None], rows, torch.zeros(1, dtype=torch.float64))
    zero = torch.zeros(1, dtype=torch.float64)
    g, gb, gb_dh = torch.where(ok, g, zero), torch.where(ok, gb, zero), torch.where(ok, gb_dh, zero)
    loss, loss_b = torch.where(live, loss, zero), torch.where(live, loss_b, zero)
    dh = (g[:, :, None] * rows).sum(1)
    dh_b = (gb_dh[:, :, None] * rows.abs()).sum(1) + (k + 2) * U * (g.abs()[:, :, None] * rows.abs()).sum(1)
    entry = (g[:, :, None] * hd[:, None, :]).reshape(-1, dim)
    entry_b = (gb[:, :, None] * hd.abs()[:, None, :]).reshape(-1, dim)
    key = torch.where(ok, ids, torch.full_like(ids, -1)).reshape(-1)
    dtable = sum_by_word(key, entry, entry_b, vocab)
    return out_round(loss, loss_b, torch.float32), out_round(dh, dh_b, dtype), dtable
