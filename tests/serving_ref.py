"""Plain 64-bit restatements of the serving operators, with the error that a
correct fp32 computation of each may have."""
import torch

# unit roundoff of one rounding to each type
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}


def rounding(y, dtype):
    """Largest error of rounding y to dtype (fp16's spacing below its normal range included)."""
    return UNIT[dtype] * y.abs() + TINY[dtype]


def rotate(x, positions, cos, sin, interleaved):
    """(rotated x, sum of the absolute products) in fp64; x [tokens, heads, dim]."""
    x = x.double()
    y, mag = x.clone(), x.abs()
    half = cos.shape[1]
    for t, p in enumerate(positions.tolist()):
        if p < 0:
            continue
        for i in range(half):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
            c, s = float(cos[p, i]), float(sin[p, i])
            u, w = x[t, :, a], x[t, :, b]
            y[t, :, a], y[t, :, b] = u * c - w * s, w * c + u * s
            mag[t, :, a], mag[t, :, b] = (u * c).abs() + (w * s).abs(), (w * c).abs() + (u * s).abs()
    return y, mag


def gather(pool, pages, n):
    """Rows 0..n of one sequence: [n, kv heads, dim] fp64."""
    ps = pool.shape[2]
    j = torch.arange(n)
    return pool[pages.long()[j // ps], :, j % ps].double()


def attend(q, k_pool, v_pool, table, lens, scale, window=0):
    """(out, lse, bound on out, bound on lse) in fp64 from CPU tensors.

    Bound.  Let A_j = scale sum_i |q_i k_ji|.  A score has the error of its
    products and sums: every partial sum is below A_j, at most dim + 8
    roundings or truncations of 2^-23, operands split into parts that keep 22
    bits or more (2^-21), plus 2^-23 |z| for the exponent's argument; the
    exponential adds 2^-21.  So each weight is off by a factor 1 + e_j,
    e_j <= (dim + 12) 2^-23 A_j + 2^-20.  Weights take part as two 8-bit parts
    at the least (2^-16; 16-bit queries only) and are added up in at most n
    sums of 2^-23, numerator and denominator alike.
    """
    seqs, hq, d = q.shape
    h = k_pool.shape[1]
    g = hq // h
    out = torch.zeros(seqs, hq, d, dtype=torch.float64)
    lse = torch.full((seqs, hq), float("-inf"), dtype=torch.float64)
    bound, lbound = torch.zeros_like(out), torch.zeros_like(lse)
    for s in range(seqs):
        n = int(lens[s])
        if n <= 0:
            continue
        first = max(0, n - window) if window else 0
        k, v = gather(k_pool, table[s], n)[first:], gather(v_pool, table[s], n)[first:]
        k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)  # [n, hq, d]
        x = q[s].double()
        z = torch.einsum("hd,nhd->hn", x, k) * scale
        a = torch.einsum("hd,nhd->hn", x.abs(), k.abs()) * scale
        p = torch.softmax(z, -1)
        out[s] = torch.einsum("hn,nhd->hd", p, v)
        lse[s] = torch.logsumexp(z, -1)
        e = ((d + 12) * 2.0 ** -23 * a + 2.0 ** -20).amax(-1)  # [hq]
        split = 2.0 ** -22 if q.dtype == torch.float32 else 2.0 ** -16
        sums = (n - first) * 2.0 ** -23
        mass = torch.einsum("hn,nhd->hd", p, v.abs())
        bound[s] = (2 * (e + sums) + split)[:, None] * mass + rounding(out[s], q.dtype)
        lbound[s] = e + sums + 2.0 ** -22 * lse[s].abs() + 2.0 ** -22
    return out, lse, bound, lbound


def adapters(x, ids, down, up, scales, base, dtype):
    """(y, bound): fp64 result, and its bound from K + rank sums of 2^-23 each
    plus operands that keep 21 bits or more in parts (2^-20)."""
    m, n = up[0].shape[0], x.shape[1]
    y = torch.zeros(m, n, dtype=torch.float64) if base is None else base.double().clone()
    mag = y.abs()
    terms = 4
    for t in range(n):
        a = int(ids[t])
        if a < 0 or a >= len(down):
            continue
        xd = x[:, t].double()
        y[:, t] += scales[a] * (up[a].double() @ (down[a].double() @ xd))
        mag[:, t] += abs(scales[a]) * (up[a].double().abs() @ (down[a].double().abs() @ xd.abs()))
        terms = max(terms, x.shape[0] + down[a].shape[0] + 4)
    return y, (terms * 2.0 ** -23 + 2.0 ** -20) * mag + rounding(y, dtype)
