"""The sequence operators from their definitions, in 64 bits on the CPU, with how far a kernel may be from them.

Bounds count roundings.  `u` is half a step of the tensors' type (0 where that is float32, whose steps `e` counts), `e` = 2^-24 half a step of float32, in
which every sum is held: a sum of n products is off by at most n e times the sum of their absolute values.  `low` is what a rounding to float16 may be off
where u times the value is less: below 2^-14 its steps stay 2^-24, half of that is 2^-25, whatever the value.  A weight that is rounded takes `low` times the
absolute value it multiplies, an output takes it once.  (float32's and bfloat16's range ends at 2^-126: 1e-30 stands for that.)"""
import math

import torch

E32 = 2.0 ** -24


def half_step(dtype):
    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def low_step(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 0.0


def attention(q, k, v, scale, causal, d_o=None, hidden=None):
    """One sequence and head, double: q [n, d], k and v [m, d]; hidden [n, m] (True: not seen) for forms other than causal.
    -> a dict of o, lse (with d_o: dq, dk, dv) and their bounds as functions of (u, low)."""
    n, d = q.shape
    m = k.shape[0]
    s = scale * q @ k.T
    s_abs = scale * q.abs() @ k.abs().T
    if hidden is None:
        hidden = torch.ones(n, m, dtype=torch.bool).triu(1) if causal else torch.zeros(n, m, dtype=torch.bool)
    s = s.masked_fill(hidden, -math.inf)
    lse = torch.logsumexp(s, 1) if m else torch.full((n,), -math.inf, dtype=torch.float64)
    p = torch.where(hidden | (lse == -math.inf)[:, None], 0.0, torch.exp(s - lse[:, None]))
    o = p @ v
    # a weight's exponent: the score (d products), its scaling, the maximum's, the exponential's own 2 steps: relative to the weight
    w = E32 * ((d + 4) * s_abs.masked_fill(hidden, 0).amax(1) + 4) if m else torch.zeros(n, dtype=torch.float64)
    a_o, seen = p @ v.abs(), (~hidden).double()
    r = {"o": o, "lse": lse,
         "tol_o": lambda u, low: (u + 2 * w[:, None] + (m + 8) * E32) * a_o + (u + E32) * o.abs() + low * (seen @ v.abs() + 1) + 1e-30,
         "tol_lse": lambda u, low: w + (m + 8) * E32 + 4 * E32 * lse.abs()}
    if d_o is not None:
        d_p, delta = d_o @ v.T, (d_o * o).sum(1, keepdim=True)
        d_p_abs, delta_abs = d_o.abs() @ v.abs().T, (d_o.abs() * o.abs()).sum(1, keepdim=True)
        d_s = p * (d_p - delta)
        # dS: P's exponent; dP and delta are sums of d products; delta takes o as it was rounded (u; and o's own float32 error, in a_o)
        a_s = p * (d_p_abs + delta_abs)
        o_err = (2 * w[:, None] + (m + 8) * E32) * a_o
        f32 = (2 * w[:, None] + (d + 8) * E32) * a_s + p * (d_o.abs() * o_err).sum(1, keepdim=True)

        def ds_err(u, low):     # P carries the forward's u into o (inside delta), beside o's own rounding; then dS is rounded, as scale dS
            o_low = low * (seen @ v.abs() + 1)
            return f32 + p * (u * delta_abs + (d_o.abs() * (u * a_o + o_low)).sum(1, keepdim=True)) + u * d_s.abs() + low / scale * seen
        r.update(dq=scale * d_s @ k, dk=scale * d_s.T @ q, dv=p.T @ d_o)
        r["tol_dq"] = lambda u, low: scale * ds_err(u, low) @ k.abs() + (m + 8) * E32 * scale * a_s @ k.abs() + (u + E32) * r["dq"].abs() + low + 1e-30
        r["tol_dk"] = lambda u, low: scale * ds_err(u, low).T @ q.abs() + (n + 8) * E32 * scale * a_s.T @ q.abs() + (u + E32) * r["dk"].abs() + low + 1e-30
        r["tol_dv"] = lambda u, low: ((u + 2 * w[:, None] + (n + 8) * E32) * p + low * seen).T @ d_o.abs() + (u + E32) * r["dv"].abs() + low + 1e-30
    return r


def attention_heads(q, k, v, lens, scale, causal, dtype, d_o=None):
    """Packed [T, heads, d] in double -> {name: (value, bound)}; a shared head's gradient is the sum over its group"""
    H, Hk, u, low, T = q.shape[1], k.shape[1], half_step(dtype), low_step(dtype), sum(lens)
    names = ["o", "lse"] + (["dq", "dk", "dv"] if d_o is not None else [])
    shape = {"o": q[:T], "lse": q[:T, :, 0], "dq": q[:T], "dk": k[:T], "dv": k[:T]}
    out = {x: [torch.zeros_like(shape[x]), torch.zeros_like(shape[x])] for x in names}
    at = 0
    for n in lens:
        part = slice(at, at + n)
        at += n
        for h in range(H if n else 0):
            g = h // (H // Hk)
            r = attention(q[part, h], k[part, g], v[part, g], scale, causal, None if d_o is None else d_o[part, h])
            for x in names:
                of = g if x in ("dk", "dv") else h
                # (a group's sum is rounded to the type once: the bound of each part counts it for its own size, which together is no less)
                out[x][0][part, of] += r[x]
                out[x][1][part, of] += r["tol_" + x](u, low)
    return out


def linear(q, k, v, log_decay, state, scale, d_o=None, d_last=None):
    """One sequence, all heads, double, token by token: q, k, v [n, H, d], state [H, d, d] or None.  -> (values, absolute sums), dicts of the same names.
    The absolute sums run the same recurrences on absolute values."""
    def run(scale, q, k, v, s0, d_o, d_last):
        n, H, d = q.shape
        g = torch.exp(log_decay)[:, None, None]
        s = torch.zeros(H, d, d, dtype=torch.float64) if s0 is None else s0.clone()
        o, dq, dk, dv = (torch.zeros(n, H, d, dtype=torch.float64) for _ in range(4))
        for t in range(n):
            s = g * s + k[t][:, :, None] * v[t][:, None, :]
            o[t] = scale * (q[t][:, :, None] * s).sum(1)
            if d_o is not None:
                dq[t] = scale * (s * d_o[t][:, None, :]).sum(2)
        r = {"o": o, "last": s}
        if d_o is not None:
            ds = torch.zeros(H, d, d, dtype=torch.float64) if d_last is None else d_last.clone()
            for t in reversed(range(n)):
                ds = ds + scale * q[t][:, :, None] * d_o[t][:, None, :]
                dk[t], dv[t] = (ds * v[t][:, None, :]).sum(2), (ds * k[t][:, :, None]).sum(1)
                ds = g * ds
            r.update(dq=dq, dk=dk, dv=dv, dstate=ds)
        return r

    def absolute(x):
        return None if x is None else x.abs()
    return run(scale, q, k, v, state, d_o, d_last), run(abs(scale), *(absolute(x) for x in (q, k, v, state, d_o, d_last)))


def linear_bound(name, value, total, n, d, dtype, largest=0.0):
    """Outputs: the weights of a chunk and the state are each rounded to the type for their product (u each, of parts that together make the absolute sum), the output
    once.  States: never rounded.  float32: sums over d, over a chunk's 64 tokens and over the chunks, decays whose exponent (|x| e^-|x| <= 0.4 per step, at
    most two steps each for the chunk, the segment and the whole) is off by a step.  float16: `low` for the up to 64 weights and d state elements of an
    output, times `largest`, the largest absolute value of what they multiply (the weights carry the scale when they are rounded, the state takes it afterwards)."""
    state = name in ("last", "dstate")
    u, low = (0.0, 0.0) if state else (half_step(dtype), low_step(dtype))
    f32 = E32 * (d + n + 64 + 32)
    return (2 * u + f32) * total + (u + E32) * value.abs() + low * ((64 + d) * largest + 1) + 1e-30
