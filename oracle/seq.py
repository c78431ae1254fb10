"""Plain 64-bit statements of the operators of token sequences with positions and a cache (rotary positions, attention over packed
sequences, attention over a paged cache), with the bounds that roundings of a 16- or 32-bit device run stay within.  Test infrastructure."""
import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # one rounding, relative
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}      # one step below the normal range
U32 = 2.0 ** -24
FLUSH = 2.0 ** -126          # the device's power of two gives 0 below this, its matrix instructions may take and leave 0 there


def rotate(x, pos, freqs, sections, interleaved=False, inverse=False):
    """x [T, H, D] -> the turned x in 64 bits."""
    x, n, at, ang = x.detach().double().cpu(), sum(sections), 0, []
    for a, m in enumerate(sections):
        ang.append(pos[:, a].double().cpu()[:, None] * freqs.cpu()[at:at + m])
        at += m
    ang = torch.cat(ang, 1)[:, None] * (-1 if inverse else 1)
    c, s, y = torch.cos(ang), torch.sin(ang), x.clone()
    i0 = slice(0, 2 * n, 2) if interleaved else slice(0, n)
    i1 = slice(1, 2 * n, 2) if interleaved else slice(n, 2 * n)
    y[..., i0] = x[..., i0] * c - x[..., i1] * s
    y[..., i1] = x[..., i1] * c + x[..., i0] * s
    return y


def rotate_bound(x, y, sections, interleaved, dtype):
    """|device - rotate()| is at most this: sin and cos are within 4 steps of 32 bits (the reduced angle's rounding and the polynomial's
    operations), each product and the sum round once more in 32 bits, the result once in its own format."""
    x, n = x.detach().double().abs().cpu(), sum(sections)
    b = torch.zeros_like(x)
    i0 = slice(0, 2 * n, 2) if interleaved else slice(0, n)
    i1 = slice(1, 2 * n, 2) if interleaved else slice(n, 2 * n)
    b[..., i0] = b[..., i1] = (x[..., i0] + x[..., i1]) * 6 * U32
    return b + HALF_STEP[dtype] * (y.abs() + b) + TINY[dtype]


def limit(p, frame, length):
    return length if frame == 0 else max(0, min(length, (p // frame + 1) * frame))


def attend(q, k, v, limits, scale, dtype, do=None, low=False, fine=False):
    """One head: q [n, D], k, v [L, D], limits [n] keys seen by each row; do [n, D].  -> dict of 64-bit results and of bounds.

    The bounds follow the kernels' roundings.  A score is a 32-bit sum of D products (at most D / 8 + 8 dependent additions); the exponent
    and its power of two round a few times more; so a probability is off by 2 * es relative (numerator and denominator), es the
    score's absolute error + 8 steps.  Probabilities and dS round once to a 16-bit operand (up).  A sum over n terms is off by at most
    (n / 16 + 40) steps of 32 bits of the sum of magnitudes.  delta reads the stored, rounded output.  low: a probability enters its
    product as the 16-bit operand and the rounded rest (at most up of it, so the two are off by up * up).

    Weights are powers of two of s - m, m no larger than the row's maximum, so their sum is at least 1 and a weight that is flushed to 0
    takes at most FLUSH from a probability; so does every term of a sum that lies below it.

    fine: the training pass over short sequences.  Probabilities and dS enter their products with their rests (up * up); delta reads the
    output and the rounded rest of its rounding; fp16 operands carry powers of two, so that probabilities lose 2^-40 at most and dS 2^-35
    of its column's largest (2^-33 here: one head's largest for its group's)."""
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    n, L, D = q.shape[0], k.shape[0], q.shape[1]
    u = HALF_STEP[dtype]
    up, tiny = (0.0, 0.0) if dtype == torch.float32 else (u * u if low or fine else u, TINY[dtype])
    lost = max(tiny * 0.5, FLUSH)
    seen = torch.arange(L)[None] < torch.as_tensor(limits)[:, None]
    if L == 0:
        z = torch.zeros(n, D, dtype=torch.float64)
        r = dict(out=z, out_b=z)
        if do is not None:
            r.update(dq=z, dq_b=z, dk=torch.zeros(0, D, dtype=torch.float64), dk_b=torch.zeros(0, D, dtype=torch.float64),
                     dv=torch.zeros(0, D, dtype=torch.float64), dv_b=torch.zeros(0, D, dtype=torch.float64))
        return r
    s = (q @ k.t() * scale).masked_fill(~seen, -math.inf)
    m = s.amax(1, keepdim=True).nan_to_num(neginf=0.0)
    p = torch.exp(s - m)
    p = p / p.sum(1, keepdim=True).clamp_min(1e-300)
    out = p @ v
    mag = (q.abs() @ k.abs().t() * scale).masked_fill(~seen, 0.0)
    big = mag.amax(1, keepdim=True)
    es = ((D / 8 + 8) * big + 8 * (1 + big)) * U32                       # absolute, of a natural exponent
    ep = 2 * es + (L / 16 + 40) * U32 + 2.0 ** -22                          # relative, of a probability
    ones = seen.double()
    out_b = (p * (up + ep)) @ v.abs() + lost * (ones @ v.abs()) + FLUSH * L + (L / 16 + 40) * U32 * (p @ v.abs())
    unrounded = out_b
    out_b = out_b + u * (out.abs() + out_b) + TINY[dtype]
    r = dict(out=out, out_b=out_b)
    if do is None:
        return r
    do = do.detach().double().cpu()
    dp = do @ v.t()
    delta = (do * out).sum(1, keepdim=True)
    ds = p * (dp - delta)
    lost_s = lost
    if fine:
        lost, lost_s = 2.0 ** -40, 2.0 ** -33 * ds.abs().max() + FLUSH
    pb = p * (up + ep) + lost * ones
    N = n / 16 + 40
    dv = p.t() @ do
    dv_b = pb.t() @ do.abs() + FLUSH * n + N * U32 * (p.t() @ do.abs())
    read = unrounded + up * (out.abs() + unrounded) + TINY[dtype] if fine else out_b
    delta_b = (do.abs() * (read + D * U32 * out.abs())).sum(1, keepdim=True)
    dp_b = (D / 8 + 8) * U32 * (do.abs() @ v.abs().t())
    ds_b = p * (dp_b + delta_b + 2 * U32 * (dp.abs() + delta.abs())) + (p * ep + FLUSH * ones) * (dp - delta).abs()
    ds_b = ds_b + up * (ds.abs() + ds_b) + lost_s * ones
    dq, dk = ds @ k * scale, ds.t() @ q * scale
    dq_b = (ds_b @ k.abs() + FLUSH * L + (L / 16 + 40) * U32 * (ds.abs() @ k.abs())) * scale
    dk_b = (ds_b.t() @ q.abs() + FLUSH * n + N * U32 * (ds.abs().t() @ q.abs())) * scale
    r.update(dq=dq, dk=dk, dv=dv, dq_b=dq_b + u * (dq.abs() + dq_b) + TINY[dtype], dk_b=dk_b, dv_b=dv_b)   # dk, dv: rounded after the group's sum
    return r


def packed(q, k, v, cu, frame, scale=None, do=None, fine=False):
    """Attention over packed sequences: q [T, Hq, D], k, v [T, Hk, D], cu: list of bounds -> dict of [T, H, D] results and bounds.  fine: as
    in attend()."""
    T, Hq, D = q.shape
    Hk, dt = k.shape[1], q.dtype
    g, scale = Hq // Hk, D ** -0.5 if scale is None else scale
    names = ['out'] + (['dq', 'dk', 'dv'] if do is not None else [])
    r = {}
    for nm in names:
        h = Hk if nm in ('dk', 'dv') else Hq
        r[nm], r[nm + '_b'] = torch.zeros(T, h, D, dtype=torch.float64), torch.zeros(T, h, D, dtype=torch.float64)
    for a, b in zip(cu[:-1], cu[1:]):
        limits = [limit(p, frame, b - a) for p in range(b - a)]
        for h in range(Hq):
            one = attend(q[a:b, h], k[a:b, h // g], v[a:b, h // g], limits, scale, dt, None if do is None else do[a:b, h], fine=fine)
            for nm in names:
                i = h // g if nm in ('dk', 'dv') else h
                r[nm][a:b, i] += one[nm]
                r[nm + '_b'][a:b, i] += one[nm + '_b']
    for nm in names[2:]:
        r[nm + '_b'] = r[nm + '_b'] + HALF_STEP[dt] * (r[nm].abs() + r[nm + '_b']) + TINY[dt]
    return r


def paged(q, k_cache, v_cache, table, lengths, frame, scale=None, low=False):
    """q [B, n, Hq, D] against the pages: (out, bound) [B, n, Hq, D].  A page outside the cache holds no keys.  low: as in attend()."""
    B, n, Hq, D = q.shape
    pages, page, Hk = k_cache.shape[:3]
    g, scale = Hq // Hk, D ** -0.5 if scale is None else scale
    out, bound = torch.zeros(B, n, Hq, D, dtype=torch.float64), torch.zeros(B, n, Hq, D, dtype=torch.float64)
    for b in range(B):
        length = max(0, min(int(lengths[b]), table.shape[1] * page))
        at = [(int(table[b, j // page]), j % page, j) for j in range(length)]
        at = [x for x in at if 0 <= x[0] < pages]
        pg, row = [x[0] for x in at], [x[1] for x in at]
        limits = [sum(1 for x in at if x[2] < limit(length - n + i, frame, length)) for i in range(n)]
        for h in range(Hq):
            one = attend(q[b, :, h], k_cache[pg, row, h // g], v_cache[pg, row, h // g], limits, scale, q.dtype, low=low)
            out[b, :, h], bound[b, :, h] = one['out'], one['out_b']
    return out, bound
