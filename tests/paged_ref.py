"""Paged caches by their definition: codes and values of rows, pools token by token, attention over them in
float64 with the bounds of a kernel's error.

Bounds of an implementation that rounds the weights once to a type of unit u (see below), the output once
to the inputs' type and computes in float32 (unit e = 2^-24), with S = scale |q|.|K| + |bias| and n keys:

* a score is a sum of D products, times up to three factors: absolute error at most e (D + 8) S, so a
  weight's relative error is at most w = 2 e ((D + 8) max S + 4) + e n
* out: u_out |o| + (u + w + e) sum p |V|, and half a step of float16's least numbers for each weight
* weights meet 16-bit values in their type (u = u_out), codes in parts of 8 bits: one for bfloat16 queries,
  two for float16 (2^-16), three for float32 (2^-24)
"""

import math

import torch

from attention_ref import SPACING, UNIT, bucket

MOST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def block(dtype):
    return 64 // dtype.itemsize


def quantise(x, dtype):
    """(codes, scales float32) of rows x [..., D]: round(x * fl(M / a)) of the exact product, fl(a / M)."""
    x = x.detach().cpu().double()
    a = x.abs().amax(-1, keepdim=True)
    most = torch.full_like(a, MOST[dtype])
    finite, kept = torch.isfinite(a), a >= 2.0 ** -100
    scale = torch.where(finite, torch.where(kept, (a / most).float(), 0.0), math.nan)
    y = torch.where(finite & kept, x * (most / a).float().double(), 0.0)
    if dtype is torch.int8:
        return y.round().to(torch.int8), scale.squeeze(-1)
    step = 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return ((y / step).round() * step).float().to(torch.float8_e4m3fn), scale.squeeze(-1)


def stored(x, dtype):
    """What rows x stand for in a pool of ``dtype``, float64."""
    if dtype not in MOST:
        return x.detach().cpu().double()
    codes, scale = quantise(x, dtype)
    return codes.float().double() * scale.double().unsqueeze(-1)


def bits(t):
    return t.view(torch.uint8) if t.dtype is torch.float8_e4m3fn else t


def put(cache, name, page, slot, rows):
    """Rows [Hk, D] of one token into a pool's tensors (CPU copies in a dict)."""
    pool = cache[name]
    if pool.dtype in MOST:
        rows, scale = quantise(rows, pool.dtype)
        cache[name + "_scale"][page, :, slot] = scale
    blk = block(pool.dtype)
    if name == "k":
        bits(pool)[page, :, slot] = bits(rows.cpu())
    else:
        bits(pool)[page, :, slot // blk, :, slot % blk] = bits(rows.cpu())


def get(cache, name, page, slot):
    """Values float64 [Hk, D] of one token."""
    pool, blk = cache[name], block(cache[name].dtype)
    x = bits(pool)[page, :, slot] if name == "k" else bits(pool)[page, :, slot // blk, :, slot % blk]
    x = x.contiguous().view(pool.dtype).float().double()
    return x * cache[name + "_scale"][page, :, slot].double().unsqueeze(-1) if pool.dtype in MOST else x


def copy(cache):
    """A PagedCache's tensors on the CPU."""
    out = {"k": cache.k.cpu(), "v": cache.v.cpu()}
    if cache.k_scale is not None:
        out.update(k_scale=cache.k_scale.cpu(), v_scale=cache.v_scale.cpu())
    return out


def same(cache, want):
    """Every bit of a PagedCache's tensors is as in ``want``."""
    for name, w in want.items():
        g = getattr(cache, name).cpu()
        kind = {4: torch.int32, 2: torch.int16, 1: torch.uint8}[g.element_size()]
        wrong = g.contiguous().view(kind) != w.contiguous().view(kind)
        assert not wrong.any(), (name, int(wrong.sum()), wrong.nonzero()[:5].tolist())


def attend(q, K, V, first, pool_dtype, scale=None, table=None, maxd=128, unit=None):
    """(out, bound) [m, H, D] of queries q [m, H, D] at positions first .. over K, V float64 [n, Hk, D].  unit: of the
    weights' rounding, where it is another than above."""
    dtype, (m, H, D), (n, Hk, _) = q.dtype, q.shape, K.shape
    e, u_out, z = 2.0 ** -24, UNIT[q.dtype], SPACING[q.dtype] / 2
    u = u_out if pool_dtype not in MOST else {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -16, torch.float32: e}[dtype]
    u = u if unit is None else unit
    scale = 1 / math.sqrt(D) if scale is None else scale
    q = q.detach().cpu().double().transpose(0, 1)
    K, V = (x.transpose(0, 1).repeat_interleave(H // Hk, 0) for x in (K, V))
    s, S = scale * q @ K.transpose(1, 2), abs(scale) * q.abs() @ K.abs().transpose(1, 2)
    back = first + torch.arange(m).view(m, 1) - torch.arange(n)
    if table is not None:
        lut = torch.tensor([bucket(-d, table.shape[0], maxd, False) for d in range(int(back.max()) + 1)])
        t = table.detach().cpu().double().t()[:, lut[back.clamp(min=0)]]
        s, S = s + t, S + t.abs()
    seen = back >= 0
    p = s.masked_fill(~seen, -math.inf).softmax(-1)
    w = 2 * e * ((D + 8) * S.masked_fill(~seen, 0).amax(-1, keepdim=True) + 4) + e * seen.sum(-1).view(1, m, 1)
    o = p @ V
    tol = u_out * o.abs() + z + (p * (u + w + e) + z * seen) @ V.abs()
    return o.transpose(0, 1), tol.transpose(0, 1)


def assert_near(got, want, tol, what=""):
    x = got.detach().double().cpu()
    assert x.shape == want.shape, (what, x.shape, want.shape)
    bad = ~((x - want).abs() - tol - 1e-37 <= 0)
    assert not bad.any(), (what, int(bad.sum()), x.numel(), (x - want).abs().max().item(), (x - want)[bad].flatten()[:4].tolist(),
                           tol[bad].flatten()[:4].tolist(), bad.nonzero()[:6].tolist())


def random_table(lengths, page, pages, gen, spare=1):
    """int32 [B, n]: pages of a pool of ``pages`` in random order, -1 where a stream needs none."""
    need = [-(-n // page) for n in lengths]
    assert sum(need) <= pages
    order = torch.randperm(pages, generator=gen).tolist()
    table = torch.full((len(lengths), max(need) + spare), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    return table
