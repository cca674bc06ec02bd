"""float16's range inside the sequence kernels: what they round for their matrix products (weights, their gradients, states) keeps its digits, and stays finite, wherever the
inputs and the results fit the type."""
import math

import pytest
import torch

import seq_ref as R
from test_sequence_gpu import S, near, randn

pytestmark = pytest.mark.gpu
F16 = torch.float16


def linear_case(lens, d, seed=0, heads=2, q=1.0, k=1.0, v=1.0, d_o=1.0, state=1.0, d_last=1.0, scale=None):
    """-> {name: (kernel's, definition's, absolute sums)} of linear_attention in float16, packed; and the definition's largest output"""
    T = sum(lens)
    x = [randn(T, heads, d, dtype=F16, seed=seed + i, scale=s).requires_grad_() for i, s in enumerate((q, k, v))]
    g = randn(T, heads, d, dtype=F16, seed=seed + 3, scale=d_o)
    x.append(randn(len(lens), heads, d, d, seed=seed + 4, scale=state).requires_grad_())
    gs = randn(len(lens), heads, d, d, seed=seed + 5, scale=d_last)
    decay = torch.tensor([math.log(1 - 0.5 ** (3 + h)) for h in range(heads)], dtype=torch.float32, device="cuda")
    o, last = S().linear_attention(*x[:3], decay, S().Packed(lens, "cuda:0"), state=x[3], scale=scale)
    got = dict(zip(("o", "last", "dq", "dk", "dv", "dstate"), (o, last) + torch.autograd.grad((o, last), x, (g, gs))))
    at, parts = 0, []
    for i, n in enumerate(lens):
        part = slice(at, at + n)
        at += n
        parts.append(R.linear(*(t[part].detach().double().cpu() for t in x[:3]), decay.double().cpu(), x[3][i].detach().double().cpu(), 1 / math.sqrt(d) if scale is None else scale,
                              g[part].double().cpu(), gs[i].double().cpu()))
    rows = [t.detach().abs().amax(-1) for t in x[:3] + [g]]
    out = {"n": max(lens), "spread": max(float(r.max() / r.min()) for r in rows)}
    for name, t in got.items():
        join = torch.stack if name in ("last", "dstate") else torch.cat
        out[name] = (t.detach().double().cpu(),) + tuple(join([p[j][name] for p in parts]) for j in (0, 1))
    return out


def check_linear(out, d):
    """Within the roundings that the operator states, none of which falls below the type's normal range: seq_ref's bound without what that would add (`largest` 0), and for what
    the kernels do not lift, a weight (state) of at least 2^-8 with smaller ones beside it: those are off by half of float16's smallest step, 2^-25, so 2^-17 of the
    largest, up to 64 weights and d elements of an output, times what they multiply.  The largest product of the two is at most the largest absolute sum times
    the ratio `spread` between the largest element of a tensor and the largest of any row."""
    spread, n = out.pop("spread"), out.pop("n")
    for name, (got, value, total) in out.items():
        state = name in ("last", "dstate")
        assert state or 0.01 < float(value.abs().max()) < 65504, name
        near(got, value, R.linear_bound(name, value, total, n, d, F16) + (0 if state else 2.0 ** -17 * (64 + d) * spread * float(total.max())), name)


def check_rms(got, value, times, what, beside=None):
    """root mean square errors: at most `times` that of the value rounded once, and that of `beside` (an error of the inputs), if given"""
    got, value = got.detach().double().cpu(), value.double()
    assert torch.isfinite(got).all(), what
    once = float((value.half().double() - value).square().mean().sqrt())
    err = float((got - value).square().mean().sqrt())
    more = 0.0 if beside is None else float(beside.square().mean().sqrt())
    assert err <= times * once + more, f"{what}: {err:.3g}, {err / once:.3g} x the value rounded once"


@pytest.mark.parametrize("lens", [[40, 1, 130], [600, 300]])
@pytest.mark.parametrize("d,kw", [
    (128, dict(d_last=2000.0, v=0.1, k=0.1)),                       # (d_last / scale is past 65 504)
    (64, dict(d_last=100.0, scale=1e-3)),
    (80, dict(d_last=5.0, scale=1.0 / 4096, d_o=50.0)),
    (128, dict(state=60000.0, q=0.005, d_o=0.1))])
def test_linear_attention_states_past_float16(lens, d, kw):
    """states, and state gradients over the scale, past float16's range where their products with q, k and v are not"""
    check_linear(linear_case(lens, d, **kw), d)


@pytest.mark.parametrize("lens", [[40, 1, 130], [600, 300]])
def test_linear_attention_weights_past_float16(lens):
    """weights past 65 504 whose outputs are not: large q and k with small v, and the same of d_o and v with small k and q"""
    check_linear(linear_case(lens, 64, q=160.0, k=2000.0, v=1e-3, d_o=1e-3, state=1.0, d_last=1e-3, scale=1.0), 64)
    check_linear(linear_case(lens, 64, q=0.005, k=0.005, v=60.0, d_o=8000.0, state=1.0, d_last=1.0), 64)


@pytest.mark.parametrize("kw", [dict(d_o=1e-3, v=0.02, k=30.0, q=30.0, state=0.02, d_last=1e-3), dict(v=2e-4, k=0.05, q=30.0, state=1e-5, d_last=0.01, d_o=30.0)])
def test_linear_attention_small_weights(kw):
    """Weights and states below float16's normal range with results inside it.  Three roundings of a size (a weight, a state, the output), independent: sqrt(3) times the error of
    one, and three leaves room for their being unequal."""
    lens, d = [300, 700], 64
    out = linear_case(lens, d, **kw)
    for name in ("o", "dq", "dk", "dv"):
        got, value, _ = out[name]
        assert float(value.abs().median()) > 2.0 ** -13, name
        check_rms(got, value, 3, name)


def attention_case(H, n, d, d_o, sink=0.0, seed=0):
    """one causal sequence, all gradients.  `sink`: the first key gets that much more score from every query, and its value is zero."""
    q, k, v = (randn(n, H, d, dtype=F16, seed=seed + i) for i in range(3))
    g = randn(n, H, d, dtype=F16, seed=seed + 3, scale=d_o)
    if sink:
        q[:, :, 0], k[:, :, 0], k[0, :, 0], v[0] = 4.0, 0.0, sink * math.sqrt(d) / 4, 0.0
    x = [t.requires_grad_() for t in (q, k, v)]
    o = S().attention(*x, S().Packed([n], "cuda:0"))
    got = (o,) + torch.autograd.grad(o, x, g)
    names, want, beside = ("o", "dq", "dk", "dv"), [[] for _ in got], [[], []]
    for h in range(H):
        q, k, v = (t[:, h].detach().double().cpu() for t in x)
        r = R.attention(q, k, v, 1 / math.sqrt(d), True, g[:, h].double().cpu())
        for w, name in zip(want, names):
            w.append(r[name])
        # The backward pass takes o as the forward pass returned it, rounded: d_s = P (d_p - rowsum(d_o o)) is off by P rowsum(d_o (o rounded - o)), whoever computes it.
        # Where o itself is below the normal range (its steps are 2^-24 there) and the first key is large, that is the larger part.
        p = torch.exp((q @ k.T / math.sqrt(d)).masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), -math.inf) - r["lse"][:, None])
        d_s = -p * (g[:, h].double().cpu() * (r["o"].half().double() - r["o"])).sum(1, keepdim=True) / math.sqrt(d)
        beside[0].append(d_s @ k)
        beside[1].append(d_s.T @ q)
    beside = dict(zip(("dq", "dk"), (torch.stack(b, 1) for b in beside)))
    return {name: (a, torch.stack(w, 1), beside.get(name)) for name, a, w in zip(names, got, want)}


# Roundings on the way: the weight P for o, o for delta, the weight's gradient dS, the result; independent and of a size, so twice the error of one, and three leaves
# room for their being unequal.
@pytest.mark.parametrize("H,n,d,d_o", [(2, 30, 64, 1e-4), (2, 200, 64, 1e-3), (1, 2048, 64, 1e-3), (1, 1500, 128, 1e-2), (64, 600, 128, 1e-3), (64, 600, 32, 1e-3)])
def test_attention_small_gradients(H, n, d, d_o):
    """an upstream gradient of a thousandth (a mean loss): dS, that times the weight and the scale, is far below float16's normal range, dq and dk are not"""
    for name, (got, want, _) in attention_case(H, n, d, d_o).items():
        assert float(want[1:].abs().median()) > 2.0 ** -17, name
        check_rms(got[1:], want[1:], 3, name)          # (the first query sees one key: its dq is 0)


@pytest.mark.parametrize("H,n,d", [(2, 30, 64), (2, 300, 64), (40, 700, 128)])
def test_attention_small_weights(H, n, d):
    """a first key that draws nearly all the weight and has no value (a sink): the others' weights are below float16's normal range, what they add up to is not"""
    for name, (got, want, beside) in attention_case(H, n, d, 2000.0, sink=15.0).items():
        check_rms(got[1:], want[1:], 3, name, None if beside is None else beside[1:])


@pytest.mark.parametrize("d,page,width", [(64, 16, None), (128, 16, 400)])
def test_attention_step_small_weights(d, page, width):
    from test_sequence_gpu import cache_of
    lens, H, Hk = [300, 700], 4, 2
    kp, vp, table, lengths, keys = cache_of(lens, Hk, d, page, F16, width=width)
    q, k, v = (randn(len(lens), h, d, dtype=F16, seed=50 + h) for h in (H, Hk, Hk))
    q[:, :, 0] = 4.0
    for b, (kb, vb) in enumerate(keys):
        kb[:, :, 0], kb[0, :, 0], vb[0] = 0.0, 15.0 * math.sqrt(d) / 4, 0.0
        for t in range(lens[b]):
            kp[table[b, t // page], t % page], vp[table[b, t // page], t % page] = kb[t].cuda(), vb[t].cuda()
    got = S().attention_step(q, k, v, kp, vp, table, lengths)
    want = torch.zeros(len(lens), H, d, dtype=torch.float64)
    for b in range(len(lens)):
        K, V = (torch.cat([x, y[b][None].cpu()]).double() for x, y in zip(keys[b], (k, v)))
        for h in range(H):
            want[b, h] = R.attention(q[b, h][None].double().cpu(), K[:, h // 2], V[:, h // 2], 1 / math.sqrt(d), False)["o"][0]
    check_rms(got, want, 3, "o")
