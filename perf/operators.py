"""The sequence operators of taco_amd/sequence.py as measured workloads.

A policy that remembers (attention over its episode, or a decaying linear memory) is trained on whole episodes packed one behind the other
and acts one token per env step.  Five calls:

  attention              causal attention inside each packed sequence, grouped heads          (forward, or forward + gradients)
  attention_step         one new token per row over a paged key-value cache, which it joins
  linear_attention       o_t = scale * q_t S_t, S_t = exp(log_decay) S_{t-1} + k_t v_t^T        (forward, or forward + gradients)
  linear_attention_step  the same recurrence for one token per row, the state updated in place

`run` with `own` false is the plain form: padded batches, elementary torch operations in float32, rounded once at the end.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SCORES = 4.4e9      # padded scores (rows x length^2 x heads) of the plain form: 17 GB in float32


def listed():
    return [
        # a handful of short episodes in the policy's own type: every launch is latency
        {"name": "attention_few_short", "op": "attention", "train": False, "dtype": "float32", "rows": 4, "longest": 33, "spread": "ragged", "heads": 4, "kv_heads": 4, "dim": 32},
        # a batch of prompts of very different lengths, grouped heads
        {"name": "attention_ragged_prompts", "op": "attention", "train": False, "dtype": "bfloat16", "rows": 24, "longest": 2048, "spread": "ragged", "heads": 16, "kv_heads": 4, "dim": 128},
        # one long history
        {"name": "attention_one_long", "op": "attention", "train": False, "dtype": "bfloat16", "rows": 1, "longest": 16384, "spread": "equal", "heads": 16, "kv_heads": 4, "dim": 128},
        # the update on a whole rollout: 4 096 envs x 32 steps, cut where an episode ended
        {"name": "attention_train_rollout", "op": "attention", "train": True, "dtype": "float32", "rows": 4096, "longest": 32, "spread": "rollout", "heads": 4, "kv_heads": 4, "dim": 32},
        # training on long ragged sequences, grouped heads
        {"name": "attention_train_long", "op": "attention", "train": True, "dtype": "bfloat16", "rows": 6, "longest": 4096, "spread": "ragged", "heads": 16, "kv_heads": 4, "dim": 128},
        # one request, a short history: a serving step's latency
        {"name": "step_one_row", "op": "attention_step", "dtype": "float16", "rows": 1, "longest": 129, "spread": "equal", "heads": 8, "kv_heads": 2, "dim": 64, "page": 16},
        # a serving batch, histories from empty to 8 192 tokens
        {"name": "step_ragged_batch", "op": "attention_step", "dtype": "bfloat16", "rows": 64, "longest": 8192, "spread": "ragged", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16},
        # few rows, long histories: the cache's length is the only axis left to split
        {"name": "step_long_cache", "op": "attention_step", "dtype": "bfloat16", "rows": 4, "longest": 65536, "spread": "equal", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64},
        # prompts through the linear memory
        {"name": "linear_prompts", "op": "linear_attention", "train": False, "dtype": "bfloat16", "rows": 6, "longest": 8000, "spread": "ragged", "heads": 16, "dim": 128},
        # its training pass, the odd head size
        {"name": "linear_train", "op": "linear_attention", "train": True, "dtype": "float16", "rows": 32, "longest": 1000, "spread": "ragged", "heads": 8, "dim": 80},
        # one row's step: latency
        {"name": "linear_step_one_row", "op": "linear_attention_step", "dtype": "float32", "rows": 1, "heads": 4, "dim": 64},
        # a step of all 4 096 envs, some of which have just been reset
        {"name": "linear_step_envs", "op": "linear_attention_step", "dtype": "float32", "rows": 4096, "heads": 4, "dim": 64},
    ]


def draw(rng):
    def log_uniform(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["attention", "attention", "attention_step", "attention_step", "linear_attention", "linear_attention", "linear_attention_step"])
    c = {"op": op, "dtype": rng.choice(["bfloat16", "float16", "float32"])}
    if op == "linear_attention_step":
        c.update(rows=log_uniform(1, 4096), heads=rng.choice([1, 2, 4, 5]), dim=rng.choice([16, 32, 40, 64]))
        return c
    c["spread"] = rng.choice(["equal", "ragged", "ragged"])
    if op == "linear_attention":
        c.update(train=rng.choice([False, True]), heads=rng.choice([1, 2, 4, 6, 8, 16]), dim=rng.choice([16, 32, 40, 64, 80, 96, 128]))
        c["longest"] = log_uniform(1, 8000)
        c["rows"] = log_uniform(1, max(1.0, min(4096, 6 * 8000 * 16 * 128 / (2.0 * c["longest"] * c["heads"] * c["dim"]), SCORES / 2 / (c["heads"] * c["longest"] ** 2))))
        return c
    c["kv_heads"] = rng.choice([1, 2, 3, 4, 8])
    c["heads"] = c["kv_heads"] * rng.choice([1, 2, 3, 4])
    c["dim"] = rng.choice([8, 16, 32, 48, 64, 80, 96, 128])
    if op == "attention":
        c["train"] = rng.choice([False, True])
        # (a sequence of one token has no gradient but dv: nothing but such rows would compare rounding with rounding)
        c["longest"] = log_uniform(2 if c["train"] else 1, 8192 if c["heads"] <= 16 else 4096)
        c["rows"] = log_uniform(1, max(1.0, min(4096, 65536.0 / c["longest"], SCORES / (4 if c["train"] else 2) / (c["heads"] * c["longest"] ** 2))))
    else:
        c["longest"] = log_uniform(1, 65536)
        c["rows"] = log_uniform(1, max(1.0, min(4096, 4 * 65536 * 8 * 128 / (2.0 * c["longest"] * c["kv_heads"] * c["dim"]))))
        c["page"] = rng.choice([1, 8, 16, 24, 64, 256])
    return c


def lengths_of(case, seed):
    """The sequences' lengths: the case gives them, the seed their order.  A rollout's envs are cut where an episode ended."""
    n, top = case["rows"], case["longest"]
    r = np.random.RandomState((1000003 * n + top) % (1 << 31))
    if case["spread"] == "equal":
        return np.full(n, top, np.int64)
    if case["spread"] == "ragged":
        low = 0 if case["op"] == "attention_step" else 1
        lens = r.randint(low, top + 1, n)
        lens[r.randint(n)] = top
        return np.random.RandomState(seed % (1 << 31)).permutation(lens).astype(np.int64)
    done = r.rand(n, top) < 0.02        # an episode ends in one of fifty steps
    done[:, -1] = True
    ends = np.flatnonzero(np.random.RandomState(seed % (1 << 31)).permutation(done).reshape(-1)) + 1
    return np.diff(ends, prepend=0)


def offsets_of(lens):
    return np.concatenate([[0], np.cumsum(lens)])


def prepare(case, seed):
    dev, dt = torch.device("cuda", torch.cuda.current_device()), TYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    H, D, B = case["heads"], case["dim"], case["rows"]

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device=dev, dtype=dtype)

    s = {"case": case}
    if case["op"] == "linear_attention_step":
        s.update(q=normal(B, H, D), k=normal(B, H, D), v=normal(B, H, D), log_decay=decays(H, dev), state=normal(B, H, D, D, dtype=torch.float32),
                 reset=torch.rand(B, generator=g, device=dev) < 0.02)
        return s
    lens = lengths_of(case, seed)
    if case["op"] == "attention_step":
        Hk, page = case["kv_heads"], case["page"]
        need = lens // page + 1                         # the pages of a row, with room for the token that comes
        P, width = int(need.sum()), int(need.max())
        order = np.random.RandomState((seed + 1) % (1 << 31)).permutation(P)
        table = np.zeros((B, width), np.int32)
        table[np.arange(width)[None] < need[:, None]] = order
        s.update(q=normal(B, H, D), k=normal(B, Hk, D), v=normal(B, Hk, D), k_pages=normal(P, page, Hk, D), v_pages=normal(P, page, Hk, D),
                 page_table=torch.from_numpy(table).to(dev), lengths=torch.from_numpy(lens.astype(np.int32)).to(dev))
        return s
    T, top, start = int(lens.sum()), int(lens.max()), offsets_of(lens)[:-1]
    at = np.arange(top)[None] + start[:, None]
    at[np.arange(top)[None] >= lens[:, None]] = T       # the padded batch of the plain form: row T is padding
    s.update(at=torch.from_numpy(at).to(dev), lengths=torch.from_numpy(lens).to(dev))
    if own:
        from taco_amd import sequence
        s["sequences"] = sequence.Packed(lens, dev)
    Hk = case.get("kv_heads", H)
    s.update(q=normal(T, H, D), k=normal(T, Hk, D), v=normal(T, Hk, D))
    if case["op"] == "linear_attention":
        s.update(log_decay=decays(H, dev), state=normal(B, H, D, D, dtype=torch.float32))
    if case["train"]:
        s["d_out"] = normal(T, H, D)
        if case["op"] == "linear_attention":
            s["d_state"] = normal(B, H, D, D, dtype=torch.float32)
        for name in ("q", "k", "v") + (("state",) if "state" in s else ()):
            s[name].requires_grad_(own)
    return s


def decays(heads, dev):
    """log decays from a memory of some 30 tokens to one of some 1 000"""
    return torch.linspace(math.log(1 - 1 / 32), math.log(1 - 1 / 1024), heads, device=dev, dtype=torch.float32)


def run(s):
    return run_own(s) if own else run_plain(s)


def run_own(s):
    from taco_amd import sequence
    op = s["case"]["op"]
    if op == "attention_step":
        return sequence.attention_step(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["page_table"], s["lengths"]), s["k_pages"], s["v_pages"]
    if op == "linear_attention_step":
        return sequence.linear_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], reset=s["reset"]), s["state"]
    if op == "attention":
        out, lse = sequence.attention(s["q"], s["k"], s["v"], s["sequences"], return_lse=True)
        if not s["case"]["train"]:
            return out, lse
        return (out.detach(), lse) + torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["d_out"])
    out, last = sequence.linear_attention(s["q"], s["k"], s["v"], s["log_decay"], s["sequences"], state=s["state"])
    if not s["case"]["train"]:
        return out, last
    return (out.detach(), last.detach()) + torch.autograd.grad((out, last), (s["q"], s["k"], s["v"], s["state"]), (s["d_out"], s["d_state"]))


def run_plain(s):
    op = s["case"]["op"]
    if op == "attention_step":
        return plain_attention_step(s)
    if op == "linear_attention_step":
        return plain_linear_step(s)
    return plain_attention(s) if op == "attention" else plain_linear(s)


# ---- the plain forms -------------------------------------------------------------------------------------------------------------

def padded(x, at):
    """packed [T, H, D] -> float32 [rows, H, length, D]; row T of the packed tensor is padding"""
    x = torch.cat([x.float(), x.new_zeros((1,) + x.shape[1:], dtype=torch.float32)])
    return x[at].transpose(1, 2).contiguous()


def packed(x, at, T, dtype):
    """float32 [rows, H, length, ...] -> packed [T, H, ...]; the padding falls into row T, which is cut off"""
    x = x.transpose(1, 2)
    out = x.new_empty((T + 1, x.shape[2]) + x.shape[3:])
    out[at.reshape(-1)] = x.reshape((-1,) + x.shape[2:])
    return out[:T].to(dtype)


def plain_attention(s):
    q, k, v, at = s["q"], s["k"], s["v"], s["at"]
    (T, H, D), Hk, (n, L) = q.shape, k.shape[1], at.shape
    scale, dt = 1 / math.sqrt(D), q.dtype
    Q, K, V = padded(q, at).view(n, Hk, -1, D), padded(k, at), padded(v, at)       # the heads of a group are rows behind one another
    i = torch.arange(L, device=q.device)
    hidden = i[None, :] > i[:, None]
    P = (Q @ K.transpose(2, 3).contiguous()).mul_(scale).view(n, H, L, L).masked_fill_(hidden, -math.inf)
    m = P.amax(3, keepdim=True)
    P = P.sub_(m).exp_()
    z = P.sum(3, keepdim=True)
    P = P.div_(z).view(n, Hk, -1, L)
    O = P @ V
    out, lse = packed(O.view(n, H, L, D), at, T, dt), packed((m + z.log())[..., 0], at, T, torch.float32)
    if not s["case"]["train"]:
        return out, lse
    dO = padded(s["d_out"], at).view(n, Hk, -1, D)
    dV = P.transpose(2, 3).contiguous() @ dO
    dP = dO @ V.transpose(2, 3).contiguous()
    dS = dP.sub_((dO * O).sum(3, keepdim=True)).mul_(P).mul_(scale)
    dQ, dK = dS @ K, dS.transpose(2, 3).contiguous() @ Q
    return out, lse, packed(dQ.view(n, H, L, D), at, T, dt), packed(dK, at, T, dt), packed(dV, at, T, dt)


def plain_attention_step(s):
    q, k, v, kc, vc, table, n = (s[x] for x in ("q", "k", "v", "k_pages", "v_pages", "page_table", "lengths"))
    (B, H, D), Hk, page = q.shape, k.shape[1], kc.shape[1]
    n = n.long()
    own_page = table.gather(1, (n // page)[:, None])[:, 0].long()
    kc[own_page, n % page] = k                          # the new token joins the cache
    vc[own_page, n % page] = v
    K = kc[table.long()].view(B, -1, Hk, D).transpose(1, 2).float()
    V = vc[table.long()].view(B, -1, Hk, D).transpose(1, 2).float()
    S = (K @ q.float().view(B, Hk, -1, D).transpose(2, 3).contiguous()) / math.sqrt(D)      # [B, Hk, tokens, G]
    S = S.masked_fill(torch.arange(K.shape[2], device=q.device)[None, None, :, None] > n[:, None, None, None], -math.inf)
    P = (S - S.amax(2, keepdim=True)).exp()
    P = P / P.sum(2, keepdim=True)
    return (P.transpose(2, 3).contiguous() @ V).reshape(B, H, D).to(q.dtype), kc, vc


def plain_linear(s):
    """The quadratic form: o_i = scale * (sum_{j <= i} g^(i-j) (q_i . k_j) v_j + g^(i+1) q_i S_0), S_end = sum_j g^(L-1-j) k_j v_j^T + g^L S_0."""
    q, k, v, at, S0 = s["q"], s["k"], s["v"], s["at"], s["state"]
    (T, H, D), L = q.shape, at.shape[1]
    scale, dt = 1 / math.sqrt(D), q.dtype
    Q, K, V = padded(q, at), padded(k, at), padded(v, at)
    g = s["log_decay"].view(1, H, 1, 1)
    i = torch.arange(L, device=q.device, dtype=torch.float32)
    n = s["lengths"].view(-1, 1, 1, 1)
    W = torch.where(i[None, :] <= i[:, None], (g * (i[:, None] - i[None, :])).exp(), 0.0)       # [1, H, L, L]
    head = (g * (i + 1).view(1, 1, L, 1)).exp() * scale                                         # the old state's weight in o_i
    rest = (n - 1 - i.view(1, 1, L, 1)).clamp(min=0)                                            # padding has k = v = 0
    tail = (g * rest).exp()                                                                     # token j's weight in the last state
    whole = (g * n).exp()
    A = (Q @ K.transpose(2, 3).contiguous()).mul_(W)
    out = (A @ V) * scale + (Q * head) @ S0
    last = (K * tail).transpose(2, 3).contiguous() @ V + whole * S0
    res = packed(out, at, T, dt), last
    if not s["case"]["train"]:
        return res
    dO, dS = padded(s["d_out"], at), s["d_state"]
    dA = (dO @ V.transpose(2, 3).contiguous()).mul_(W)
    dQ = (dA @ K) * scale + (dO @ S0.transpose(2, 3).contiguous()) * head
    dK = (dA.transpose(2, 3).contiguous() @ Q) * scale + (V @ dS.transpose(2, 3).contiguous()) * tail
    dV = (A.transpose(2, 3).contiguous() @ dO) * scale + (K @ dS) * tail
    dS0 = (Q * head).transpose(2, 3).contiguous() @ dO + whole * dS
    return res + (packed(dQ, at, T, dt), packed(dK, at, T, dt), packed(dV, at, T, dt), dS0)


def plain_linear_step(s):
    q, k, v, S = s["q"].float(), s["k"].float(), s["v"].float(), s["state"]
    keep = torch.where(s["reset"][:, None], 0.0, s["log_decay"].exp())
    S.mul_(keep[:, :, None, None]).add_(k[..., :, None] * v[..., None, :])
    return ((q[..., :, None] * S).sum(2) / math.sqrt(q.shape[-1])).to(s["q"].dtype), S


# ---- the cost ---------------------------------------------------------------------------------------------------------------------

def work(case):
    size = TYPES[case["dtype"]].itemsize
    H, D, B = case["heads"], case["dim"], case["rows"]
    if case["op"] == "linear_attention_step":
        return {"bytes": B * H * (4 * D * size + 8 * D * D) + B, "flops": 5 * B * H * D * D}
    lens = lengths_of(case, 0).astype(np.float64)
    T = lens.sum()
    Hk = case.get("kv_heads", H)
    if case["op"] == "attention_step":
        pages = (lens // case["page"] + 1).sum()
        return {"bytes": float(2 * (T + 2 * B) * Hk * D * size + 2 * B * H * D * size + 4 * pages + 4 * B), "flops": float(4 * (T + B) * H * D)}
    if case["op"] == "attention":
        pairs = (lens * (lens + 1) / 2).sum() * H
        moved = T * (2 * H + 2 * Hk) * D * size + 4 * T * H
        if case["train"]:           # the gradient's five products; d_out read, dq, dk and dv written
            return {"bytes": float(moved + T * (2 * H + 2 * Hk) * D * size), "flops": float(14 * D * pairs)}
        return {"bytes": float(moved), "flops": float(4 * D * pairs)}
    # a token costs the cheaper of the recurrence (a rank-one update, a product with the state) and the products with those before it
    flops = (lens * np.minimum(4 * D * D, 2 * D * (lens + 1))).sum() * H
    moved = 4 * T * H * D * size + 8 * B * H * D * D
    if case["train"]:               # three more products of the same kind; d_out and d_state read, dq, dk, dv and the state's gradient written
        return {"bytes": float(2 * moved), "flops": float(4 * flops)}
    return {"bytes": float(moved), "flops": float(flops)}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    f = {k: x.detach().double() if isinstance(x, torch.Tensor) and x.is_floating_point() else x for k, x in s.items()}
    return {"attention": exact_attention, "attention_step": exact_attention_step, "linear_attention": exact_linear,
            "linear_attention_step": exact_linear_step}[case["op"]](f, case, lengths_of(case, seed) if "longest" in case else None)


def exact_attention(f, case, lens):
    """Sequences of one length together, a key-value head at a time; the gradients from autograd."""
    q, k, v = f["q"], f["k"], f["v"]
    (T, H, D), Hk, train = q.shape, k.shape[1], case["train"]
    G, start = H // Hk, offsets_of(lens)
    out, lse = torch.empty_like(q), q.new_empty(T, H)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    for L in np.unique(lens):
        of = torch.from_numpy(start[:-1][lens == L][:, None] + np.arange(L)[None]).to(q.device)
        seen = torch.ones(L, L, dtype=torch.bool, device=q.device).tril()
        for h in range(Hk):
            for part in of.split(max(1, int(2e8 / L ** 2))):
                for j in range(h * G, (h + 1) * G):
                    a, b, c = (x.requires_grad_(train) for x in (q[part, j], k[part, h], v[part, h]))
                    x = (a @ b.transpose(1, 2)) * D ** -0.5
                    x = torch.where(seen, x, -torch.inf)
                    z = torch.logsumexp(x, 2)
                    o = torch.exp(x - z[..., None]) @ c
                    out[part, j], lse[part, j] = o.detach(), z.detach()
                    if train:
                        x, y, z = torch.autograd.grad(o, (a, b, c), f["d_out"][part, j])
                        dq[part, j] = x
                        dk[part, h] = y if j == h * G else dk[part, h] + y
                        dv[part, h] = z if j == h * G else dv[part, h] + z
    return (out, lse, dq, dk, dv) if train else (out, lse)


def exact_attention_step(f, case, lens):
    """A row at a time, its cache read page by page off the table."""
    q, kc, vc, out = f["q"], f["k_pages"], f["v_pages"], torch.empty_like(f["q"])
    table, page = f["page_table"].cpu().numpy(), case["page"]
    (B, H, D), Hk = q.shape, kc.shape[2]
    for b in range(B):
        n = int(lens[b])
        kc[int(table[b, n // page]), n % page] = f["k"][b]
        vc[int(table[b, n // page]), n % page] = f["v"][b]
        pages = torch.from_numpy(table[b, :n // page + 1].astype(np.int64)).to(q.device)
        K, V = (x[pages].reshape(-1, Hk, D)[:n + 1].permute(1, 0, 2) for x in (kc, vc))
        w = torch.softmax(torch.einsum("hgd,htd->hgt", q[b].view(Hk, -1, D), K) / math.sqrt(D), -1)
        out[b] = torch.einsum("hgt,htd->hgd", w, V).reshape(H, D)
    return out, kc, vc


def exact_linear(f, case, lens):
    """The recurrence itself, a token of every sequence at a time, and its transpose from the last token to the first."""
    q, k, v, g = f["q"], f["k"], f["v"], f["log_decay"].exp()[:, None, None]
    (T, H, D), L = q.shape, int(lens.max())
    if case["rows"] * H * D * D * L > 6e11:
        return None
    at, n = f["at"], f["lengths"]
    scale = D ** -0.5
    zero = q.new_zeros(1, H, D)
    q, k, v = (torch.cat([x, zero]) for x in (q, k, v))
    out = torch.empty_like(q)
    dq, dk, dv = (torch.empty_like(q) for _ in range(3))
    S = f["state"].clone()
    dO = torch.cat([f["d_out"], zero]) if case["train"] else None
    for t in range(L):
        a = at[:, t]
        S = torch.where((t < n)[:, None, None, None], g * S + k[a][..., :, None] * v[a][..., None, :], S)
        out[a] = (q[a][..., None, :] @ S)[..., 0, :] * scale
        if case["train"]:
            dq[a] = (S @ dO[a][..., :, None])[..., 0] * scale
    if not case["train"]:
        return out[:T], S
    dS = f["d_state"].clone()                       # the gradient of the state behind token t
    for t in reversed(range(L)):
        a = at[:, t]
        new = dS + scale * q[a][..., :, None] * dO[a][..., None, :]
        dk[a] = (new @ v[a][..., :, None])[..., 0]
        dv[a] = (k[a][..., None, :] @ new)[..., 0, :]
        dS = torch.where((t < n)[:, None, None, None], g * new, dS)
    return out[:T], S, dq[:T], dk[:T], dv[:T], dS


def exact_linear_step(f, case, lens):
    S = f["state"]
    S[f["reset"]] = 0
    S = f["log_decay"].exp()[None, :, None, None] * S + torch.einsum("bhi,bhj->bhij", f["k"], f["v"])
    return torch.einsum("bhi,bhij->bhj", f["q"], S) * f["q"].shape[-1] ** -0.5, S
