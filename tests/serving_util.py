"""Plain 64-bit forms of the serving operators and the error bounds of their outputs.

Bounds, with u the unit roundoff of the element type (8 significant bits in
bf16: 2^-8; 11 in f16: 2^-11), e =
2^-24 and A = sum_j p_j |v_j| of an output element:
  * the output is rounded once: u |want|;
  * each weight p_j may be rounded to the element type for the second product:
    u A; an f16 weight below the normal range 2^-14 is off by at most 2^-25 of
    the row's largest: 2^-25 sum_j |v_j| over the n keys;
  * a score x_j = scale q.k_j summed in f32 in any order is off by at most
    dim e X, X = max_j scale sum_d |q_d k_jd|, plus e X for each of the few
    roundings on its way to the exponent, which itself is good to 2^-22: p_j,
    and with it each output, moves by at most 2 ((dim + 4) e X + 2^-21) A
    (numerator and denominator);
  * sums over n keys in f32: 2 n e A.
The lse moves by the scores' and the sum's error: (dim + 4) e X + 2^-21 + n e,
plus 2 e |lse| for the last operations."""

import math

U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}
E = 2.0 ** -24


def dtype_of(name):
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16}[name]


def rows(q, k, v, scale, seen):
    """q [n, d], k and v [m, d], seen [n, m] bool -> (out, A, X, lse, count, sum |v|) in f64."""
    import torch
    q, k, v = q.double(), k.double(), v.double()
    n, m = q.shape[0], k.shape[0]
    if m == 0:
        z = torch.zeros(n, v.shape[1], dtype=torch.float64, device=q.device)
        o = torch.zeros(n, dtype=torch.float64, device=q.device)
        return z, z.clone(), o, torch.full_like(o, -math.inf), o.clone(), z.clone()
    keep = seen.any(0)
    k = torch.where(keep[:, None], k, 0.0)          # what no row sees may hold anything
    v = torch.where(keep[:, None], v, 0.0)
    x = (q @ k.T) * scale
    x = torch.where(seen, x, -math.inf)
    top = x.amax(1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    e = (x - top).exp()
    s = e.sum(1, keepdim=True)
    p = e / torch.where(s == 0, 1.0, s)
    big = torch.where(seen, (q.abs() @ k.abs().T) * scale, 0.0).amax(1)
    w = seen.double()
    return p @ v, p @ v.abs(), big, (top + s.log())[:, 0], w.sum(1), w @ v.abs()


def check_rows(name, got, want, typ, dim, lse=None):
    import torch
    out, mag, big, ref_lse, count, absv = want
    score = (dim + 4) * E * big + 2.0 ** -21
    bound = U[typ] * out.abs() + (U[typ] + 2 * score[:, None] + 2 * E * count[:, None]) * mag
    if typ == "f16":
        bound = bound + 2.0 ** -25 * absv + 2.0 ** -25      # and the output's own subnormal step
    err = (got.double() - out).abs()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    assert (err <= bound).all(), f"{name}: {float((err - bound).max()):.3g} above the bound, " \
                                 f"at most {float((err / bound.clamp(min=1e-300)).max()):.3g} of it"
    if lse is not None:
        empty = ref_lse == -math.inf
        assert torch.equal(lse == -math.inf, empty), f"{name}: lse of empty rows"
        off = (lse.double() - ref_lse).abs()[~empty]
        lim = (score + E * count + 2 * E * ref_lse.abs())[~empty]
        assert (off <= lim).all(), f"{name}: lse off by {float((off / lim).max()):.3g} of the bound"


def decode(q, k_cache, v_cache, pages, lengths, scale, check):
    """check(b, h, rows(...)) for each sequence and head."""
    import torch
    group = q.shape[1] // k_cache.shape[2]
    page = k_cache.shape[1]
    for b, m in enumerate(lengths.tolist()):
        own = pages[b, :-(-m // page)].long()
        k = k_cache[own].flatten(0, 1)[:m]
        v = v_cache[own].flatten(0, 1)[:m]
        for g in range(k_cache.shape[2]):
            seen = torch.ones(group, m, dtype=torch.bool, device=q.device)
            hs = slice(g * group, (g + 1) * group)
            check(b, hs, rows(q[b, hs], k[:, g], v[:, g], scale, seen))


def prompt(q, k, v, offsets, kv_offsets, causal, scale, check):
    """check(token slice, head, rows(...)) for each sequence and head."""
    import torch
    group = q.shape[1] // k.shape[1]
    qo, ko = offsets.tolist(), kv_offsets.tolist()
    for b in range(len(qo) - 1):
        n, m = qo[b + 1] - qo[b], ko[b + 1] - ko[b]
        if not n:
            continue
        seen = torch.ones(n, m, dtype=torch.bool, device=q.device)
        if causal:
            seen = seen.tril(m - n)
        ts, ks = slice(qo[b], qo[b + 1]), slice(ko[b], ko[b + 1])
        for h in range(q.shape[1]):
            check(ts, h, rows(q[ts, h], k[ks, h // group], v[ks, h // group], scale, seen))


def rotate(x, table, positions, interleaved):
    """(rotated x in f64, bound of an f32 rotation rounded once to x's type)."""
    import torch
    rot = table.shape[1]
    half = rot // 2
    t = table.double()[positions.long()][:, None]
    c, s = t[..., :half], t[..., half:]
    y = x.double().clone()
    mag = y.abs()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, half), slice(half, rot))
    u, w = y[..., a].clone(), y[..., b].clone()
    y[..., a], y[..., b] = u * c - w * s, w * c + u * s
    mag[..., a], mag[..., b] = (u * c).abs() + (w * s).abs(), (w * c).abs() + (u * s).abs()
    unit = U["f16" if x.dtype == torch.float16 else "bf16"]
    return y, unit * y.abs() + 2 * E * mag + (2.0 ** -25 if x.dtype == torch.float16 else 0.0)
