"""Plain 64-bit forms of the serving operators, on the CPU, and the error a
kernel's rounding points allow.

The attention kernels round three things to the element type, half a step u =
finfo.eps / 2 each: nothing of the scores (FP32 products and sums), the
probabilities P before the second product, and O at the end. With weights w_j (sum 1):
  |O - o| <= u sum_j w_j |v_j|        P rounded, l summed unrounded
          +  u |o| (1 + u)            O rounded
          +  e (sum_j w_j |v_j| + |o|)   FP32: scores off by ds change a weight by ds,
                                      up to 2^-24 * (128 + 4) sum |q k| scale for the
                                      dot product and its scaling (bounded below with
                                      the case's own sum |q k|), exp2, and the two
                                      FP32 sums over n keys, 2^-24 sqrt(n) and more
          +  tiny * sum_j |v_j|       FP16 only: a P under 2^-14 is a subnormal,
                                      2^-25 off at most, and l >= 1
The log-sum-exp, FP32, is off by ds plus 2^-24 of its size and the sums' error.
"""

import torch


def attend64(q, k, v, pos, key, window, sinks, scale):
    """q [R, 128] at positions pos [R], k and v [N, 128] at positions key [N]:
    (o, lse, sum w |v|, sum of visible |v|, max |ds| factor) in 64 bits. Only visible
    keys enter."""
    q, k, v = q.double(), k.double(), v.double()
    visible = key[None] <= pos[:, None]
    if window is not None:
        visible &= (key[None] > pos[:, None] - window) | (key[None] < sinks)
    seen = visible.any(0)
    s = torch.full(visible.shape, -float("inf"), dtype=torch.float64)
    r, c = visible.nonzero(as_tuple=True)
    reach = torch.zeros(visible.shape, dtype=torch.float64)
    if seen.any() and len(r):
        full = q @ torch.where(seen[:, None], k, 0.0).t() * scale
        s[r, c] = full[r, c]
        sizes = q.abs() @ torch.where(seen[:, None], k, 0.0).abs().t() * scale
        reach[r, c] = sizes[r, c]
    lse = torch.logsumexp(s, 1) if s.shape[1] else torch.full((len(q),), -float("inf"), dtype=torch.float64)
    w = torch.where(visible, torch.exp(s - lse[:, None]), 0.0)
    w = torch.where(lse[:, None] == -float("inf"), 0.0, w)
    o = torch.zeros(q.shape, dtype=torch.float64)
    spread = torch.zeros(q.shape, dtype=torch.float64)
    total = torch.zeros(q.shape, dtype=torch.float64)
    vz = torch.where(seen[:, None], v, 0.0)
    if torch.isfinite(vz).all():
        o, spread, total = w @ vz, w @ vz.abs(), visible.double() @ vz.abs()
    else:                                     # key by key: a hidden key never enters
        for i in range(len(q)):
            j = visible[i].nonzero().flatten()
            o[i] = w[i, j] @ v[j]
            spread[i] = w[i, j] @ v[j].abs()
            total[i] = v[j].abs().sum(0)
    return o, lse, spread, total, reach.amax(1) if s.shape[1] else reach.new_zeros(len(q))


def bounds(dtype, o, lse, spread, total, reach, keys):
    """Largest error of o and of lse (see above)."""
    u = torch.finfo(dtype).eps / 2
    # Scores and their exponents, and sums over the keys in some order (pairwise
    # or in up to `keys` / 4 steps a partial sum: the worst case).
    ds = 2.0 ** -24 * 140 * reach + 2.0 ** -22
    sums = 2.0 ** -24 * (keys / 4 + 64)
    e = (2 * ds + 2 * sums).unsqueeze(-1)
    tol = u * spread * (1 + u) + u * o.abs() * (1 + u) + e * (spread + o.abs())
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25 * total + 2.0 ** -25
    return tol, ds + sums + 2.0 ** -22 * (lse.abs() + 8)


def paged64(q, k_cache, v_cache, table, starts, lengths, window=None, sinks=0, scale=None):
    """(o, lse, tolerances of both) over the rows of all requests, in 64 bits; other
    rows NaN. Lists or tensors on the CPU."""
    scale = 128 ** -0.5 if scale is None else scale
    tokens, heads, _ = q.shape
    page, heads_kv = k_cache.shape[1:3]
    group = heads // heads_kv
    o = torch.full(q.shape, float("nan"), dtype=torch.float64)
    lse = torch.full(q.shape[:2], float("nan"), dtype=torch.float64)
    tol, tol_lse = torch.zeros_like(o), torch.zeros_like(lse)
    for b, length in enumerate(lengths):
        s0, s1 = starts[b], starts[b + 1]
        if s1 <= s0:
            continue
        key = torch.arange(length)
        pos = torch.arange(length - (s1 - s0), length)
        where = (torch.as_tensor(table[b])[key // page].long(), key % page)
        k, v = k_cache[where], v_cache[where]
        for h in range(heads):
            x = attend64(q[s0:s1, h], k[:, h // group], v[:, h // group], pos, key, window, sinks, scale)
            o[s0:s1, h], lse[s0:s1, h] = x[0], x[1]
            tol[s0:s1, h], tol_lse[s0:s1, h] = bounds(q.dtype, *x, length)
    return o, lse, tol, tol_lse


def window64(q, k, v, window, sinks=0, causal="bottom_right", scale=None):
    scale = 128 ** -0.5 if scale is None else scale
    batch, heads, nq, _ = q.shape
    group = heads // k.shape[1]
    nk = k.shape[2]
    off = nk - nq if causal == "bottom_right" else 0
    o = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.zeros(q.shape[:3], dtype=torch.float64)
    tol, tol_lse = torch.zeros_like(o), torch.zeros_like(lse)
    pos, key = torch.arange(nq) + off, torch.arange(nk)
    for b in range(batch):
        for h in range(heads):
            x = attend64(q[b, h], k[b, h // group], v[b, h // group], pos, key, window, sinks, scale)
            o[b, h], lse[b, h] = x[0], x[1]
            tol[b, h], tol_lse[b, h] = bounds(q.dtype, *x, nk)
    return o, lse, tol, tol_lse


def plan(past, new, table, pages, taken, tokens, page):
    """The page plan in plain Python: (table, starts, lengths, positions, slots, taken)."""
    table = [list(row) for row in table]
    starts, lengths, positions, slots = [0], [], [], []
    for row, p, n in zip(table, past, new):
        p, n = max(p, 0), max(n, 0)
        for column in range(-(-p // page), -(-(p + n) // page)):
            if column < len(row):
                row[column] = pages[taken] if taken < len(pages) else -1
            taken += 1
        for position in range(p, p + n):
            column = position // page
            held = row[column] if column < len(row) else -1
            positions.append(position)
            slots.append(held * page + position % page if held >= 0 else -1)
        starts.append(starts[-1] + n)
        lengths.append(p + n)
    rest = tokens - len(slots)
    return (table, starts, lengths, (positions + [0] * max(rest, 0))[:tokens],
            (slots + [-1] * max(rest, 0))[:tokens], taken)


def rotate64(x, positions, frequencies, magnitude, layout, backward=False):
    """x [T, H, 128] rotated, in 64 bits."""
    import numpy as np

    x = x.double().numpy()
    half = len(frequencies)
    angle = positions.double().numpy()[:, None] * np.asarray(frequencies)[None]
    turn = magnitude * np.exp((-1j if backward else 1j) * angle)[:, None]
    out = x.copy()
    if layout == "half":
        z = (x[..., :half] + 1j * x[..., half:2 * half]) * turn
        out[..., :half], out[..., half:2 * half] = z.real, z.imag
    else:
        z = (x[..., 0:2 * half:2] + 1j * x[..., 1:2 * half:2]) * turn
        out[..., 0:2 * half:2], out[..., 1:2 * half:2] = z.real, z.imag
    return torch.from_numpy(out)
