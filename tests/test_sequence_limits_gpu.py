"""The sequence operators' memory, limits and layouts on an MI355X, beside test_sequence_gpu.py's values."""
import math

import pytest
import torch

import seq_ref as R
from test_sequence_gpu import DTYPES, S, check_attention, near, randn
from taco_amd import _lib

pytestmark = pytest.mark.gpu


def test_short_grouped_sequences_need_no_sums_of_parts():
    """a rollout's update with shared heads takes memory for its gradients and statistics, not for sums that no launch makes"""
    lens, H, Hk, d = [32] * 512, 32, 4, 64
    T = sum(lens)
    x = [randn(T, h, d, dtype=torch.bfloat16, seed=h).requires_grad_() for h in (H, Hk, Hk)]
    seqs = S().Packed(lens, "cuda:0")
    o = S().attention(*x, seqs)
    g = torch.ones_like(o)
    torch.autograd.grad(o, x, g, retain_graph=True)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    grads = torch.autograd.grad(o, x, g)
    torch.cuda.synchronize()
    own = sum(t.numel() * t.element_size() for t in grads) + T * H * 4       # dq, dk, dv and delta
    assert torch.cuda.max_memory_allocated() - before <= own + (1 << 20)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [40, 128])
def test_attention_group_in_parts_beside_short_sequences(monkeypatch, dtype, d):
    """the sums lie tile by tile: short sequences before, between and behind the long ones, in launches of their own"""
    monkeypatch.setattr(S(), "_FEW_SHORT", 0)
    lens = [3, 700, 33, 64, 129, 1]
    seqs = S().Packed(lens, "cuda:0")
    assert seqs._parts(64, 32, True) > 1 and [t[0] for t in seqs._tiles(64)] == [128, 32]
    check_attention(64, 2, d, lens, dtype)


# ---- more workgroups than one launch counts (2^32 threads): each row's result by its formula, which for one token is short ----------------------

def test_linear_attention_step_of_many_rows():
    B, d = 2 ** 24 + 5, 8
    q, k, v = (torch.randn(B, 1, d, generator=torch.Generator("cuda").manual_seed(i), device="cuda") for i in range(3))
    state = torch.zeros(B, 1, d, d, device="cuda")
    o = S().linear_attention_step(q, k, v, torch.zeros(1, device="cuda"), state)
    # (sums of 8 products, each rounded in float32, in an order of its own: 16 half steps of the absolute sum)
    want, bound = (q * k).double().sum(2, keepdim=True) * v / math.sqrt(d), (q * k).abs().double().sum(2, keepdim=True) * v.abs() * (16 * R.E32)
    assert ((o - want).abs() <= bound).all()
    assert torch.equal(state, k[..., :, None] * v[..., None, :])


def test_attention_of_many_short_sequences_and_heads():
    """A sequence of one token sees itself alone: o is v, d_v is d_o, d_q and d_k are zero but for P: it is the exponential of s - lse, a difference of equal numbers that are each off
    by (d + 4) half steps of the absolute sum s_abs (a product of d, its scaling, the exponent's unit) and the exponential by 4, so d_s = P (d_p - P d_p) by as much of d_p."""
    T, H, d = 1100, 65535, 8
    x = [torch.randn(T, H, d, generator=torch.Generator("cuda").manual_seed(i), device="cuda", dtype=torch.float16).requires_grad_() for i in range(3)]
    g = torch.randn(T, H, d, generator=torch.Generator("cuda").manual_seed(9), device="cuda", dtype=torch.float16)
    o = S().attention(*x, S().Packed([1] * T, "cuda:0"))
    assert torch.equal(o, x[2])
    dq, dk, dv = torch.autograd.grad(o, x, g)
    assert torch.equal(dv, g)
    with torch.no_grad():
        scale, a = 1 / math.sqrt(d), [t.float().abs() for t in x + [g]]
        off = 2 * R.E32 * ((d + 4) * scale * (a[0] * a[1]).sum(2, keepdim=True) + 4) * scale * (a[3] * a[2]).sum(2, keepdim=True)
        assert (dq.abs() <= off * a[1] + R.low_step(dq.dtype)).all() and (dk.abs() <= off * a[0] + R.low_step(dk.dtype)).all()


def test_attention_step_of_many_rows():
    B, Hk, d = 4200, 4000, 8
    q = torch.randn(B, Hk, d, generator=torch.Generator("cuda").manual_seed(1), device="cuda", dtype=torch.float16)
    kp, vp = (torch.randn(3, 100, Hk, d, generator=torch.Generator("cuda").manual_seed(i), device="cuda", dtype=torch.float16) for i in (2, 3))
    table = torch.arange(B, device="cuda", dtype=torch.int32)[:, None] % 3
    o = S().attention_step(q, None, None, kp, vp, table, torch.ones(B, dtype=torch.int32, device="cuda"))
    assert torch.equal(o, vp[table[:, 0].long(), 0])


def test_attention_step_heads_before_rows():
    """a query whose heads lie farther apart than a descriptor reaches"""
    B, H, d = 33000, 2, 64
    q = torch.randn(H, B, d, generator=torch.Generator("cuda").manual_seed(1), device="cuda", dtype=torch.float16).transpose(0, 1)
    assert q.stride(1) > 1 << 21
    kp, vp = (torch.randn(1, 8, 1, d, generator=torch.Generator("cuda").manual_seed(i), device="cuda", dtype=torch.float16) for i in (2, 3))
    args = kp, vp, torch.zeros(B, 1, dtype=torch.int32, device="cuda"), torch.arange(B, device="cuda", dtype=torch.int32) % 9
    assert torch.equal(S().attention_step(q, None, None, *args), S().attention_step(q.contiguous(), None, None, *args))


@pytest.mark.parametrize("op", ["attention", "linear"])
def test_gradients_asked_for_with_create_graph(op):
    """the same bits, and a second derivative is refused instead of left out (a gradient penalty)"""
    leaf = [randn(50, 2, 41, seed=i).requires_grad_() for i in range(3)]       # (rows that are copied first)
    state, decay, seqs = randn(2, 2, 40, 40).requires_grad_(), torch.full((2,), -0.1, device="cuda"), S().Packed([30, 20], "cuda:0")
    x = [t[..., :40] for t in leaf]
    of = leaf + [state] if op == "linear" else leaf

    def out():
        return S().attention(*x, seqs).sum() if op == "attention" else sum(t.sum() for t in S().linear_attention(*x, decay, seqs, state=state))
    want = torch.autograd.grad(out(), of)
    for i, t in enumerate(of):
        o = out()
        g, = torch.autograd.grad(o, t, create_graph=True)
        assert torch.equal(g, want[i])
        with pytest.raises(_lib.TacoError, match="second derivative"):
            torch.autograd.grad(o + g.square().sum(), t)
    out().backward(create_graph=True)
    assert all(torch.equal(t.grad, w) for t, w in zip(of, want))
