"""Window attention by its definition, dense and in float64, with the bounds of a kernel's error.

``reference`` returns the output and gradients, and for each the largest error that an
implementation may show which rounds inputs, weights and their gradients once to the inputs' type
(unit u) and computes in float32 (unit e = 2^-24):

* a score is a sum of D products: absolute error at most e (D + 4) S, S = scale |q|.|k| + |bias|, so
  a weight's relative error is at most w = 2 e ((D + 4) max S + 4) + e n, n keys summed
* out: u |o| + (u + w) sum p |v|
* delta = g.o from the rounded o: error (u + e D) |g|.|o|; ds = p (g.v - delta), so
  |ds error| <= p ((w + e D) (|g|.|v| + |g|.|o|) + (u + e D) |g|.|o| + u |g.v - delta|), the last
  for its rounding to the inputs' type before the products with k and q
* dq, dk, dv: those errors through the products, and the result's own rounding
* a value below the inputs' type's least normal one rounds to a multiple of its least one: any
  rounding above has an error of half that (SPACING / 2) besides, which matters for float16
"""

import math

import torch

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SPACING = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def bucket(d, buckets, maxd, two_sided):
    half = buckets // 2 if two_sided else buckets
    e, n = half // 2, abs(d) if two_sided else max(-d, 0)
    b = n if n < e else e + sum(n ** (half - e) >= e ** (half - e - k) * maxd ** k for k in range(1, half - e))
    return b + (half if two_sided and d > 0 else 0)


def visible(T, left, right, sinks, ptr=None, mask=None):
    """[T, T] bool: query i sees key j."""
    i, j = torch.arange(T).view(T, 1), torch.arange(T)
    first, end = torch.zeros(T, dtype=torch.long), torch.zeros(T, dtype=torch.long)
    for a, b in zip(ptr[:-1], ptr[1:]) if ptr is not None else [(0, T)]:
        first[a:b], end[a:b] = a, b
    first, end = first.view(T, 1), end.view(T, 1)
    seen = (j >= first) & (j < end) & (j <= i + right) & ((j >= i - left) | (j < first + sinks))
    return seen & mask.cpu() if mask is not None else seen


def reference(q, k, v, g, seen, scale=None, table=None, maxd=128, two_sided=True):
    """({name: value}, {name: bound}) for out and, where g is given, dq, dk, dv, dbias."""
    u, e, z = UNIT[q.dtype], 2.0 ** -24, SPACING[q.dtype] / 2
    q, k, v = (x.detach().double().cpu().transpose(0, 1) for x in (q, k, v))
    H, T, D = q.shape
    Hk = k.shape[0]
    scale = 1 / math.sqrt(D) if scale is None else scale
    k, v = (x.repeat_interleave(H // Hk, 0) for x in (k, v))
    s = scale * q @ k.transpose(1, 2)
    S = scale * q.abs() @ k.abs().transpose(1, 2)
    if table is not None:
        far = torch.arange(T).view(1, T) - torch.arange(T).view(T, 1)
        lut = torch.tensor([bucket(d, table.shape[0], maxd, two_sided) for d in range(-T, T + 1)])
        b = lut[far + T]
        t = table.detach().double().cpu().t()[:, b]
        s, S = s + t, S + t.abs()
    s = s.masked_fill(~seen, -math.inf)
    p = torch.nan_to_num(s.softmax(-1), nan=0.0)
    n = seen.sum(-1).view(1, T, 1)
    w = 2 * e * ((D + 4) * S.masked_fill(~seen, 0).amax(-1, keepdim=True) + 4) + e * n
    o = p @ v
    pw = p * (u + w) + z * seen
    out, tol = {"out": o}, {"out": u * o.abs() + z + pw @ v.abs()}
    if g is not None:
        g = g.detach().double().cpu().transpose(0, 1)
        dp, delta = g @ v.transpose(1, 2), (g * o).sum(-1, keepdim=True)
        adp, adelta = g.abs() @ v.abs().transpose(1, 2), (g * o).abs().sum(-1, keepdim=True)
        ds = p * (dp - delta)
        eds = p * ((w + e * D) * (adp + adelta) + (u + e * D) * adelta)
        erd = eds + u * ds.abs() + z * seen
        out["dq"], tol["dq"] = scale * ds @ k, scale * erd @ k.abs()
        out["dk"], tol["dk"] = scale * ds.transpose(1, 2) @ q, scale * erd.transpose(1, 2) @ q.abs()
        out["dv"], tol["dv"] = p.transpose(1, 2) @ g, pw.transpose(1, 2) @ g.abs()
        # sums over up to T queries and the heads that share a key, in float32
        for x in ("dk", "dv"):
            tol[x] = tol[x] + e * T * ((ds.abs().transpose(1, 2) @ q.abs()) * scale if x == "dk" else p.transpose(1, 2) @ g.abs())
        tol["dq"] = tol["dq"] + e * n * scale * (ds.abs() @ k.abs())
        for x in ("dk", "dv"):
            out[x], tol[x] = (y[x].unflatten(0, (Hk, H // Hk)).sum(1) for y in (out, tol))
        for x in ("dq", "dk", "dv"):
            tol[x] = tol[x] + u * out[x].abs() + z
        if table is not None:
            db, tb = torch.zeros(table.shape[0], H, dtype=torch.float64), torch.zeros(table.shape[0], H, dtype=torch.float64)
            flat = b.reshape(-1)
            db.index_add_(0, flat, ds.reshape(H, -1).t().contiguous())
            tb.index_add_(0, flat, (eds + e * T * ds.abs()).reshape(H, -1).t().contiguous())
            out["dbias"], tol["dbias"] = db, tb + UNIT[table.dtype] * db.abs() + SPACING[table.dtype] / 2
    for x in ("out", "dq", "dk", "dv"):
        if x in out:
            out[x], tol[x] = out[x].transpose(0, 1), tol[x].transpose(0, 1)
    return out, tol


def assert_within(got, want, tol, what=""):
    for name, w in want.items():
        x = got[name].detach().double().cpu()
        assert x.shape == w.shape, (what, name, x.shape, w.shape)
        off = (x - w).abs() - tol[name] - 1e-37
        bad = ~(off <= 0)
        assert not bad.any(), (what, name, int(bad.sum()), x.numel(), (x - w).abs().max().item(),
                               (x - w)[bad].flatten()[:4].tolist(), tol[name][bad].flatten()[:4].tolist(), bad.nonzero()[:6].tolist())
