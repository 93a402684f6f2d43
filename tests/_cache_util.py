"""The operators around attention in 64 bits, from their definitions: what the tests of the cache, of attention over it, and
of the norm and rotation compare with.  Everything runs on the CPU or wherever its inputs are."""
import math

import torch

RANGE = {torch.float8_e4m3fn: (448.0, -64, 119), torch.int8: (127.0, -64, 121)}


def grid(x, dtype):
    """x (fp64) rounded to the payload's grid, nearest even."""
    if dtype == torch.int8:
        return torch.round(x).clamp(-127, 127)
    a = x.abs().clamp(max=448.0)
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    return torch.sign(x) * (torch.round(a / step) * step).clamp(max=448.0)


def least_exponent(amax, dtype):
    """Least e with amax <= M 2^e for one magnitude, in range."""
    m, lo, hi = RANGE[dtype]
    if amax == 0:
        return lo
    e = math.ceil(math.log2(amax / m))
    while m * 2.0 ** e < amax:
        e += 1
    while m * 2.0 ** (e - 1) >= amax:
        e -= 1
    return min(max(e, lo), hi)


def write(payload, scale, x, table, start, lengths):
    """payload [pages, H, P, w] (fp64 values of the payload), scale [pages, H] fp64, updated in place with x [B, S, H, w];
    `dtype` of the payload in payload_dtype.  Plain loops."""
    values, dtype = payload
    pages, H, P, _ = values.shape
    B, S = x.shape[:2]
    for b in range(B):
        n = S if lengths is None else min(max(int(lengths[b]), 0), S)
        rows = [(int(start[b]) + i, i) for i in range(n) if int(start[b]) + i >= 0]
        for j in sorted({p // P for p, _ in rows}):
            if j >= table.shape[1] or not 0 <= int(table[b, j]) < pages:
                continue
            page = int(table[b, j])
            here = [(p - j * P, i) for p, i in rows if p // P == j]
            first = here[0][0]
            for h in range(H):
                new = torch.stack([x[b, i, h] for _, i in here]).double()
                finite = new[torch.isfinite(new)]
                e = least_exponent(float(finite.abs().max()) if finite.numel() else 0.0, dtype)
                dead = dtype == torch.int8 and bool((~torch.isfinite(new)).any())
                if first > 0:
                    old = float(scale[page, h])
                    if math.isnan(old):
                        dead = True
                    else:
                        e = max(e, round(math.log2(old)))
                        values[page, h, :first] = grid(values[page, h, :first] * (old / 2.0 ** e), dtype)
                q = grid(torch.where(torch.isfinite(new), new, torch.zeros_like(new)) / 2.0 ** e, dtype)
                if dtype != torch.int8:
                    q[~torch.isfinite(new)] = math.nan
                values[page, h, first:first + len(here)] = q
                scale[page, h] = math.nan if dead else 2.0 ** e


def dense(values, scale, table, n):
    """[n, H, w]: positions 0 .. n - 1 of one sequence (its row of the page table), and which of them are tokens."""
    pages, H, P, w = values.shape
    out = torch.zeros(n, H, w, dtype=torch.float64)
    there = torch.zeros(n, dtype=torch.bool)
    for j in range(-(-n // P)):
        if j >= len(table) or not 0 <= int(table[j]) < pages:
            continue
        page, lo, hi = int(table[j]), j * P, min(n, (j + 1) * P)
        out[lo:hi] = (values[page] * scale[page][:, None, None]).transpose(0, 1)[:hi - lo]
        there[lo:hi] = True
    return out, there


def attention(q, k, v, there, n_rows, causal, window, scale, sink):
    """One sequence: q [S, Hq, d] fp64, k, v [len, H, *], `there` [len].  Returns out [S, Hq, dv], lse [Hq, S], and for the
    tolerances sum_j p_j |v_j| [S, Hq, dv] and the largest sum_c |q_c k_c| of a visible key [S, Hq]."""
    S, Hq, d = q.shape
    L, H = k.shape[:2]
    out = torch.zeros(S, Hq, v.shape[2], dtype=torch.float64)
    weight, reach = torch.zeros_like(out), torch.zeros(S, Hq, dtype=torch.float64)
    lse = torch.full((Hq, S), -math.inf, dtype=torch.float64)
    if sink is not None:
        lse[:] = sink.double()[:, None]
    pos = torch.arange(L)
    for i in range(n_rows):
        at = L - n_rows + i
        seen = there & ((pos <= at) if causal else torch.ones_like(there))
        if window:
            seen &= pos > at - window
        if not bool(seen.any()):
            continue
        for h in range(Hq):
            kk, vv = k[seen, h * H // Hq], v[seen, h * H // Hq]
            x = kk @ q[i, h] * scale
            reach[i, h] = (kk.abs() @ q[i, h].abs()).max() * abs(scale)
            if sink is not None:
                x = torch.cat([x, sink[h:h + 1].double()])
            lse[h, i] = torch.logsumexp(x, 0)
            p = torch.softmax(x, 0)[:kk.shape[0]]
            out[i, h] = p @ vv
            weight[i, h] = p @ vv.abs()
    return out, lse, weight, reach


def norm_rotary(x, w, cos, sin, pos, eps, interleaved):
    """y in 64 bits of x [B, S, H, d]; differentiable."""
    d, n = x.shape[-1], cos.shape[1]
    u = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    if w is not None:
        u = u * w
    c, s = cos[pos][:, :, None], sin[pos][:, :, None]
    if interleaved:
        a, b = u[..., 0:2 * n:2], u[..., 1:2 * n:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = u[..., :n], u[..., n:2 * n]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([turned, u[..., 2 * n:]], -1)
