"""Plain float64 forms of the sequence operators (tests only): rotary positions, window attention with sinks, its cache.

Each is written from the operator's definition, sequence by sequence and position by position; nothing is shared with the
kernels.  The attention forms also return what the error bounds of the tests need (see ``tolerance``)."""


import torch


def rotary(x, pos, freqs, sections, interleaved=False, inverse=False):
    """x [N, H, D] -> float64 [N, H, D]."""
    out = x.double().clone()
    pairs = sum(sections)
    i = 0
    for axis, m in enumerate(sections):
        for _ in range(m):
            t = pos[:, axis].double() * freqs[i].double()
            c, s = torch.cos(t)[:, None], torch.sin(t)[:, None] * (-1.0 if inverse else 1.0)
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
            xa, xb = x[:, :, a].double(), x[:, :, b].double()
            out[:, :, a], out[:, :, b] = xa * c - xb * s, xa * s + xb * c
            i += 1
    return out


def attend(q, k, v, seen, scale):
    """One row set: q [n, D], k / v [m, D], seen [n, m] bool -> (o [n, D], mag [n, D], reach [n], count [n]).
    mag = sum p |v| / sum p, reach = max over seen keys of scale * sum |q k| (what rounding errors of a score scale with)."""
    n, d = q.shape
    o, mag = torch.zeros(n, d, dtype=torch.float64), torch.zeros(n, d, dtype=torch.float64)
    reach, count = torch.zeros(n, dtype=torch.float64), seen.sum(1)
    for i in range(n):
        j = seen[i].nonzero(as_tuple=True)[0]
        if j.numel() == 0:
            continue
        kj, vj, qi = k[j].double(), v[j].double(), q[i].double()
        s = scale * (kj * qi).sum(1)
        p = torch.exp(s - s.max())
        p = p / p.sum()
        o[i], mag[i] = p @ vj, p @ vj.abs()
        reach[i] = float((scale * (kj * qi).abs().sum(1)).max())
    return o, mag, reach, count


def window(q, k, v, cu_q, win, sinks, cu_k=None, key_mask=None, scale=None):
    """attn_window on CPU tensors -> (o, mag, reach, count), all [Nq, Hq, ...]."""
    cu_k = cu_q if cu_k is None else cu_k
    nq, hq, d = q.shape
    g = hq // k.size(1)
    scale = d ** -0.5 if scale is None else scale
    o, mag = torch.zeros(nq, hq, d, dtype=torch.float64), torch.zeros(nq, hq, d, dtype=torch.float64)
    reach, count = torch.zeros(nq, hq, dtype=torch.float64), torch.zeros(nq, hq, dtype=torch.int64)
    for b in range(len(cu_q) - 1):
        qa, qz, ka, kz = int(cu_q[b]), int(cu_q[b + 1]), int(cu_k[b]), int(cu_k[b + 1])
        p = torch.arange(qz - qa)[:, None] + (kz - ka) - (qz - qa)
        j = torch.arange(kz - ka)[None]
        seen = (j <= p) & ((j > p - win) | (j < sinks))
        if key_mask is not None:
            seen = seen & key_mask[ka:kz][None]
        for h in range(hq):
            r = attend(q[qa:qz, h], k[ka:kz, h // g], v[ka:kz, h // g], seen, scale)
            o[qa:qz, h], mag[qa:qz, h], reach[qa:qz, h], count[qa:qz, h] = r
    return o, mag, reach, count


def append(k, v, cu, lengths, k_cache, v_cache, sinks, key_mask=None, mask_cache=None):
    """window_cache_append token by token, on CPU tensors in place."""
    win = k_cache.size(2) - sinks
    for b in range(len(cu) - 1):
        if int(lengths[b]) < 0:
            continue
        for i in range(int(cu[b]), int(cu[b + 1])):
            p = int(lengths[b]) + i - int(cu[b])
            c = p if p < sinks else sinks + (p - sinks) % win
            k_cache[b, :, c], v_cache[b, :, c] = k[i], v[i]
            if mask_cache is not None:
                mask_cache[b, c] = True if key_mask is None else key_mask[i]


def step(q, k, v, lengths, k_cache, v_cache, sinks, key_mask=None, mask_cache=None, scale=None):
    """attn_window_step on CPU tensors (caches in place) -> (o, mag, reach, count)."""
    batch, hq, d = q.shape
    g = hq // k.size(1)
    scale = d ** -0.5 if scale is None else scale
    slots = k_cache.size(2)
    append(k, v, list(range(batch + 1)), lengths, k_cache, v_cache, sinks, key_mask, mask_cache)
    o, mag = torch.zeros(batch, hq, d, dtype=torch.float64), torch.zeros(batch, hq, d, dtype=torch.float64)
    reach, count = torch.zeros(batch, hq, dtype=torch.float64), torch.zeros(batch, hq, dtype=torch.int64)
    for b in range(batch):
        if int(lengths[b]) < 0:
            continue
        n = min(int(lengths[b]) + 1, slots)
        seen = torch.ones(1, n, dtype=torch.bool) if mask_cache is None else mask_cache[b:b + 1, :n].bool()
        for h in range(hq):
            r = attend(q[b:b + 1, h], k_cache[b, h // g, :n], v_cache[b, h // g, :n], seen, scale)
            o[b, h], mag[b, h], reach[b, h], count[b, h] = r[0][0], r[1][0], r[2][0], r[3][0]
    return o, mag, reach, count


def tolerance(dtype, dim, o, mag, reach, count, v_max):
    """Bound of |kernel - o| per element, from the kernels' arithmetic.

    u = 2^-24 (half a step of fp32), h = half a step of the output type.
    * a score is an fp32 sum of `dim` products of exact (or once rounded) inputs, scaled: off by at most (dim + 3) u reach;
      the running maximum it is compared with is one of these scores, so an exponent's argument is off by twice that, plus its
      own rounding u |s - max| <= 2 u reach, plus the conversion to base 2 (the same again);  exp2 is off by 2^-22 relative;
    * so each p is off by e_p = (2 dim + 10) u reach + 2^-22 relative, and sum(p v) / sum(p) by at most 2 e_p mag, plus the
      sums' own roundings: count terms, at most 2 (count + 8) u mag (rescaling and joining of partial sums among them);
    * 16-bit types: p is rounded once to the type for the matrix product: h mag; float16's smallest steps (2^-25 absolute, p
      relative to a maximum at least 2^-8 of the largest term, so sum(p) >= 1) add count 2^-25 v_max;
    * the output is rounded once: h |o|."""
    u = 2.0 ** -24
    h = torch.finfo(dtype).eps / 2
    e_p = (2 * dim + 10) * u * reach + 2.0 ** -22
    tol = (2 * e_p + 2 * (count + 8) * u).unsqueeze(-1) * mag + h * o.abs() * 1.01
    if dtype != torch.float32:
        tol = tol + h * 1.01 * mag
    if dtype == torch.float16:
        tol = tol + (count.unsqueeze(-1) + 1) * 2.0 ** -25 * v_max
    return tol + 1e-30


def rotary_tolerance(dtype, x, want, pairs, interleaved):
    """The fraction of a turn is rounded to fp32 (angle off by at most pi 2^-24 = 1.9e-7), sincospi by 2 ulp (1.2e-7); two products and
    a sum round by u (|a| + |b|) each; the output by half a step."""
    d = x.size(-1)
    big = torch.zeros(x.shape, dtype=torch.float64)
    xa = x.double().abs()
    for i in range(pairs):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
        big[..., a] = big[..., b] = xa[..., a] + xa[..., b]
    assert 2 * pairs <= d
    return torch.finfo(dtype).eps / 2 * want.abs() * 1.01 + (1.9e-7 + 1.2e-7 + 3 * 2.0 ** -24) * big
