"""The sequence kernels (taco_amd/sequence.py, include/taco_sequence.h) on an MI355X against their definitions in 64 bits (seq_ref.py)."""
import math

import pytest
import torch

import seq_ref as R
from taco_amd import _lib

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def S():
    from taco_amd import sequence
    return sequence


def randn(*shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed + 7919 * len(shape) + sum(shape))
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def near(got, value, bound, what):
    got = got.detach().double().cpu()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    err = (got - value).abs()
    both = (got == value)          # infinities
    bad = ~((err <= bound) | both)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / bound.clamp_min(1e-300))[bad].max()):.3g} x the bound"


def run_attention(q, k, v, lens, causal, scale, d_o=None):
    seqs = S().Packed(lens, "cuda:0")
    if d_o is None:
        return S().attention(q, k, v, seqs, causal=causal, scale=scale, return_lse=True)
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    o, lse = S().attention(q, k, v, seqs, causal=causal, scale=scale, return_lse=True)
    return (o, lse) + torch.autograd.grad(o, (q, k, v), d_o)


def check_attention(H, Hk, d, lens, dtype, causal=True, scale=None, seed=0, train=True):
    T = sum(lens)
    q, k, v, g = (randn(T, h, d, dtype=dtype, seed=seed + i) for i, h in enumerate((H, Hk, Hk, H)))
    got = run_attention(q, k, v, lens, causal, scale, g if train else None)
    want = R.attention_heads(*(t.double().cpu() for t in (q, k, v)), lens, 1 / math.sqrt(d) if scale is None else scale, causal, dtype, g.double().cpu() if train else None)
    for name, x in zip(("o", "lse", "dq", "dk", "dv"), got):
        near(x, *want[name], f"{name}, {dtype}, heads {H}/{Hk}, dim {d}, lengths {lens}")


# ---- attention ---------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hk,d,lens", [
    (1, 1, 8, [1]), (2, 2, 32, [1, 2, 31, 32, 33]), (4, 2, 64, [5, 64, 1, 65, 17]), (6, 2, 80, [40, 3]), (4, 2, 96, [70, 33, 20]), (8, 1, 128, [70, 1, 33]), (3, 3, 24, [0, 7, 0, 64]),
    (8, 8, 16, [128, 100])])
def test_attention_and_its_gradients(dtype, H, Hk, d, lens):
    check_attention(H, Hk, d, lens, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("few,launches", [(0, [(128, 6, 0), (32, 3, 1)]), (1024, [(128, 8, 0)])])
def test_attention_in_tiles_of_128_rows(monkeypatch, dtype, d, few, launches):
    """enough tiles that the wide form runs (256 and more, heads counted), with short sequences beside the long ones, in tiles of their own and in the same ones"""
    monkeypatch.setattr(S(), "_FEW_SHORT", few)
    lens = [129, 64, 300, 1, 128]
    check_attention(60, 20, d, lens, dtype)
    seqs = S().Packed(lens, "cuda:0")
    assert [(x[0], x[3], x[4]) for x in seqs._tiles(60)] == launches


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [24, 128])
def test_attention_group_in_parts(dtype, d):
    """one long sequence, few key-value heads: the group's heads are shared out, and their sums joined"""
    lens = [700, 129]
    seqs = S().Packed(lens, "cuda:0")
    assert seqs._parts(64, 32, True) > 1 and seqs._tiles(64)[0][0] == 128
    check_attention(64, 2, d, lens, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_not_causal(dtype):
    check_attention(4, 2, 48, [1, 33, 64, 70, 130], dtype, causal=False)
    check_attention(64, 64, 32, [129, 260, 100], dtype, causal=False, train=False)


def test_attention_scale_and_large_scores():
    """scores of some hundreds: the running maximum has to hold (a weight's exponent is off by the score's own error, which the bound counts)"""
    check_attention(2, 2, 64, [90, 150], torch.float32, scale=3.0)
    check_attention(2, 1, 64, [90, 150], torch.bfloat16, scale=1e-3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,d,lens,bad", [(2, 64, [70, 150, 33], 41), (130, 64, [70, 150, 33], 41), (130, 128, [70, 150, 33], 41), (2, 64, [9, 30, 32], 11)])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf")])
def test_hidden_tokens_have_no_influence(dtype, H, d, lens, bad, poison):
    """a token that diverges at one step of a sequence: the steps before it, and the other sequences, get the bits they get without it, forward and backward"""
    T = sum(lens)
    at = lens[0] + bad
    q, k, v, g = (randn(T, H, d, dtype=dtype, seed=i) for i in range(4))
    clean = run_attention(q, k, v, lens, True, None, g)
    x = [t.clone() for t in (q, k, v)]
    for t in x:
        t[at] = poison
    o, lse = run_attention(*x, lens, True, None)
    safe = torch.ones(T, dtype=torch.bool)
    safe[at:lens[0] + lens[1]] = False
    for a, b in ((o, clean[0]), (lse, clean[1])):
        assert torch.isfinite(a[safe]).all()
        near(a[safe], b[safe].double().cpu(), b[safe].abs().double().cpu() * 2 ** -6 + 2 ** -6, "rows that see nothing of it")
        assert torch.equal(a[safe], b[safe])
    # values alone: an infinity that is seen arrives with its sign, in the rows that see it
    y = v.clone()
    y[at, :, 3] = poison
    o = run_attention(q, k, y, lens, True, None)[0]
    assert torch.equal(o[safe], clean[0][safe])
    seen = o[at:lens[0] + lens[1], :, 3].float()
    assert torch.isnan(seen).all() if math.isnan(poison) else bool((torch.isnan(seen) | (seen == poison)).all() and (seen[0] == poison).all())
    assert torch.isfinite(o[at:lens[0] + lens[1], :, 4:]).all()
    # backward: keys behind an upstream gradient that diverged, and the other sequences, are untouched by it
    bad_g = g.clone()
    bad_g[at] = poison
    dq, dk, dv = run_attention(q, k, v, lens, True, None, bad_g)[2:]
    after = torch.ones(T, dtype=torch.bool)
    after[lens[0]:at + 1] = False
    others = torch.ones(T, dtype=torch.bool)
    others[at] = False
    assert torch.equal(dq[others], clean[2][others])
    assert torch.equal(dk[after], clean[3][after]) and torch.equal(dv[after], clean[4][after])
    assert torch.isnan(dq[at]).all()
    # a key whose row diverged makes every gradient that sees it NaN, and no other
    dq, dk, dv = run_attention(q, x[1], v, lens, True, None, g)[2:]
    assert torch.equal(dq[safe], clean[2][safe])
    own = slice(lens[0] + lens[1], None)
    assert torch.equal(dk[own], clean[3][own]) and torch.equal(dk[:lens[0]], clean[3][:lens[0]])
    # a query whose row diverged leaves the keys behind it alone
    dq, dk, dv = run_attention(x[0], k, v, lens, True, None, g)[2:]
    assert torch.equal(dk[after], clean[3][after]) and torch.equal(dv[after], clean[4][after]) and torch.equal(dq[others], clean[2][others])


def test_rows_behind_the_last_sequence():
    q, k, v = (randn(100, 2, 32, seed=i) for i in range(3))
    for t in (q, k, v):
        t[60:] = float("nan")
    seqs = S().Packed([20, 40], "cuda:0")
    out = torch.full_like(q, 7.0)
    assert S().attention(q, k, v, seqs, out=out) is out
    assert (out[60:] == 7).all() and torch.isfinite(out[:60]).all()
    assert (S().attention(q, k, v, seqs)[60:] == 0).all()
    x = [t.clone().requires_grad_() for t in (q, k, v)]
    o = S().attention(*x, seqs)
    for grad in torch.autograd.grad(o, x, torch.ones_like(o)):
        assert (grad[60:] == 0).all() and torch.isfinite(grad).all()
    decay = torch.full((2,), -0.1, device="cuda")
    o, last = S().linear_attention(*x, decay, seqs)
    assert (o[60:] == 0).all() and torch.isfinite(last).all()
    for grad in torch.autograd.grad((o, last), x, (torch.ones_like(o), torch.ones_like(last))):
        assert (grad[60:] == 0).all() and torch.isfinite(grad).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype):
    """slices of one projection, heads before tokens, rows that are no whole chunks, an offset of half a chunk, and heads that are one broadcast head"""
    H, Hk, d, lens = 4, 2, 40, [50, 20]
    T = 70
    fused = randn(T, H + 2 * Hk, d, dtype=dtype)
    q, k, v = fused.split([H, Hk, Hk], 1)
    want = run_attention(q.contiguous(), k.contiguous(), v.contiguous(), lens, True, None, randn(T, H, d, dtype=dtype, seed=9))
    g = randn(T, H, d, dtype=dtype, seed=9)

    def same(q, k, v, g):
        for a, b in zip(run_attention(q, k, v, lens, True, None, g), want):
            assert torch.equal(a, b)
    same(q, k, v, g)
    same(*(t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v, g)))
    odd = [torch.nn.functional.pad(t, (1, 2))[..., 1:1 + d] for t in (q, k, v, g)]
    assert odd[0].stride(1) == d + 3
    same(*odd)
    one = randn(T, 1, d, dtype=dtype, seed=3)
    a = run_attention(q, one.expand(T, Hk, d), one.expand(T, Hk, d), lens, True, None, g)
    b = run_attention(q, one.expand(T, Hk, d).contiguous(), one.expand(T, Hk, d).contiguous(), lens, True, None, g)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    # the gradient of a broadcast input is the sum over what it was broadcast to
    leaf = one.clone().requires_grad_()
    o = S().attention(q, leaf.expand(T, Hk, d), k, S().Packed(lens, "cuda:0"))
    whole = one.expand(T, Hk, d).contiguous().requires_grad_()
    p = S().attention(q, whole, k, S().Packed(lens, "cuda:0"))
    assert torch.equal(torch.autograd.grad(o, leaf, g)[0], torch.autograd.grad(p, whole, g)[0].sum(1, keepdim=True))
    # a gradient that arrives expanded (a sum's)
    x = [t.clone().requires_grad_() for t in (q, k, v)]
    a = torch.autograd.grad(S().attention(*x, S().Packed(lens, "cuda:0")).sum(), x)
    b = torch.autograd.grad(S().attention(*x, S().Packed(lens, "cuda:0")), x, torch.ones(T, H, d, dtype=dtype, device="cuda"))
    assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_nothing_to_do():
    s = S()
    z = torch.zeros(0, 2, 32, device="cuda")
    assert s.attention(z, z, z, s.Packed([], "cuda:0")).shape == (0, 2, 32)
    assert s.attention(z, z, z, s.Packed([0, 0], "cuda:0")).shape == (0, 2, 32)
    decay = torch.zeros(2, device="cuda")
    o, last = s.linear_attention(z, z, z, decay, s.Packed([], "cuda:0"))
    assert o.shape == z.shape and last.shape == (0, 2, 32, 32)
    state = randn(2, 2, 32, 32)
    o, last = s.linear_attention(z, z, z, decay, s.Packed([0, 0], "cuda:0"), state=state)
    assert torch.equal(last, state)
    pages = torch.zeros(1, 4, 2, 32, device="cuda")
    i0 = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert s.attention_step(z, z, z, pages, pages, i0.view(0, 1), i0).shape == (0, 2, 32)
    assert s.linear_attention_step(z, z, z, decay, torch.zeros(0, 2, 32, 32, device="cuda")).shape == (0, 2, 32)


def directional(f, x, dx, h):
    return (f([a + h * b for a, b in zip(x, dx)]) - f([a - h * b for a, b in zip(x, dx)])) / (2 * h)


@pytest.mark.parametrize("op", ["attention", "linear"])
def test_gradients_against_differences(op):
    """Differences of the float32 forward itself along a random direction.  A central difference with step h is off by c h^2, so (D(h) - D(h/2)) * 4/3 is D(h)'s own
    error up to h^4; beside it the forward's rounding, 2^-20 of the loss's absolute sum (some ten roundings), over h."""
    lens, H, d = [40, 1, 90], 2, 32
    T = sum(lens)
    seqs = S().Packed(lens, "cuda:0")
    g = randn(T, H, d, seed=5)
    x, dx = [randn(T, H, d, seed=i) for i in range(3)], [randn(T, H, d, seed=10 + i) for i in range(3)]
    decay = torch.tensor([-0.02, -0.3], device="cuda")
    if op == "linear":
        x.append(randn(3, H, d, d, seed=20))
        dx.append(randn(3, H, d, d, seed=21))

    def out(x):
        return S().attention(*x, seqs) if op == "attention" else S().linear_attention(*x[:3], decay, seqs, state=x[3])[0]

    def loss(x):
        return float((out(x).double() * g.double()).sum())
    leaf = [t.clone().requires_grad_() for t in x]
    grads = torch.autograd.grad(out(leaf), leaf, g)
    analytic = sum(float((a.double() * b.double()).sum()) for a, b in zip(grads, dx))
    h = 1 / 64
    full, half = directional(loss, x, dx, h), directional(loss, x, dx, h / 2)
    rounding = 2 ** -20 * float((out(x).double() * g.double()).abs().sum()) / (h / 2)
    assert abs(half - analytic) <= abs(full - half) * 2 / 3 + rounding, (full, half, analytic, rounding)
    assert abs(analytic) > 20 * (abs(full - half) * 2 / 3 + rounding)      # (and the comparison says something)


# ---- attention of one token over a paged cache -------------------------------------------------------------------------------------

def cache_of(lens, Hk, d, page, dtype, seed=0, spare=2, width=None, joins=True):
    """pages in a random order, NaN in every slot that holds no token (of any row)"""
    need = [n // page + 1 if joins else max(1, -(-n // page)) for n in lens]
    P = sum(need) + spare
    order = torch.randperm(P, generator=torch.Generator().manual_seed(seed)).tolist()
    width = width or max(need)
    table = torch.full((len(lens), width), -7, dtype=torch.int32)
    kp, vp = (torch.full((P, page, Hk, d), float("nan"), dtype=dtype) for _ in range(2))
    keys, at = [], 0
    for b, n in enumerate(lens):
        table[b, :need[b]] = torch.tensor(order[at:at + need[b]], dtype=torch.int32)
        at += need[b]
        k, v = (randn(max(n, 1), Hk, d, dtype=dtype, seed=seed + 31 * b + i).cpu()[:n] for i in (1, 2))
        for t in range(n):
            kp[table[b, t // page], t % page], vp[table[b, t // page], t % page] = k[t], v[t]
        keys.append((k, v))
    return kp.cuda(), vp.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), keys


def want_step(q, keys, k, v, scale):
    B, H, d = q.shape
    o, bound = torch.zeros(B, H, d, dtype=torch.float64), torch.zeros(B, H, d, dtype=torch.float64)
    u, low = R.half_step(q.dtype), R.low_step(q.dtype)
    for b in range(B):
        K, V = (torch.cat([x, y[b][None].cpu()]) if y[b] is not None else x for x, y in zip(keys[b], (k, v)))
        G = H // K.shape[1]
        for h in range(H if len(K) else 0):
            r = R.attention(q[b, h][None].double().cpu(), K[:, h // G].double(), V[:, h // G].double(), scale, False)
            o[b, h], bound[b, h] = r["o"][0], r["tol_o"](u, low)[0]
    return o, bound


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hk,d,page,lens", [
    (1, 1, 8, 1, [0]), (4, 4, 32, 8, [0, 1, 7, 8, 9, 31]), (8, 2, 64, 16, [129, 0, 63, 300]), (6, 3, 80, 24, [5, 47, 48, 200]), (6, 3, 96, 24, [5, 200]), (40, 1, 128, 16, [33, 500]),
    (16, 4, 128, 64, [1000, 3]), (5, 5, 16, 3, [2, 100])])
def test_attention_step(dtype, H, Hk, d, page, lens):
    kp, vp, table, lengths, keys = cache_of(lens, Hk, d, page, dtype)
    q, k, v = (randn(len(lens), h, d, dtype=dtype, seed=50 + h) for h in (H, Hk, Hk))
    before = [t.clone() for t in (kp, vp, table, lengths)]
    got = S().attention_step(q, k, v, kp, vp, table, lengths)
    near(got, *want_step(q, keys, k, v, 1 / math.sqrt(d)), f"step, {dtype}")
    # the token is in the cache, bit for bit, and nothing else has changed
    for b, n in enumerate(lens):
        before[0][table[b, n // page], n % page], before[1][table[b, n // page], n % page] = k[b], v[b]
    for a, b in zip((kp, vp, table, lengths), before):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    # without a new token: the cache as it is, which now holds it
    lengths += 1
    again = S().attention_step(q, None, None, kp, vp, table, lengths)
    assert torch.equal(again, got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [32, 64, 80, 128])
def test_attention_step_in_pieces(dtype, d):
    """tables wide enough that rows are split over workgroups: long rows, rows shorter than a piece, an empty one"""
    lens, page, H, Hk = [2500, 0, 255, 256, 1023, 1], 16, 4, 2
    kp, vp, table, lengths, keys = cache_of(lens, Hk, d, page, dtype, width=400)
    table[table == -7] = 2 ** 31 - 1        # entries behind a row's pages are never read as pages
    q, k, v = (randn(len(lens), h, d, dtype=dtype, seed=50 + h) for h in (H, Hk, Hk))
    got = S().attention_step(q, k, v, kp, vp, table, lengths)
    near(got, *want_step(q, keys, k, v, 1 / math.sqrt(d)), f"pieces, {dtype}")
    lengths.zero_()
    assert (S().attention_step(q, None, None, kp, vp, table, lengths) == 0).all()


def test_attention_step_rows_that_are_wrong():
    """bad pages, negative lengths and full tables give NaN in their own rows, leave the cache alone and the other rows as they are"""
    lens, page, H, Hk, d = [40, 40, 40, 40, 40, 40, 47], 16, 4, 2, 32
    kp, vp, table, lengths, keys = cache_of(lens, Hk, d, page, torch.float16)
    q, k, v = (randn(len(lens), h, d, dtype=torch.float16, seed=50 + h) for h in (H, Hk, Hk))
    want = S().attention_step(q, k, v, kp.clone(), vp.clone(), table, lengths)
    table[1, 0], table[2, 1], lengths[3], lengths[4] = -1, kp.shape[0], -1, 48
    table[5, 2] = 2 ** 31 - 1                # the page the new token goes to
    kc, vc = kp.clone(), vp.clone()
    got = S().attention_step(q, k, v, kc, vc, table, lengths)
    assert torch.isnan(got[1:6]).all()
    assert torch.equal(got[[0, 6]], want[[0, 6]])
    same = torch.ones(kp.shape[0], page, dtype=torch.bool)
    for b in (0, 1, 2, 6):
        if 0 <= int(table[b, lens[b] // page]) < kp.shape[0]:
            same[table[b, lens[b] // page], lens[b] % page] = False
    assert torch.equal(kc[same].view(torch.uint8), kp[same].view(torch.uint8)) and torch.equal(vc[same].view(torch.uint8), vp[same].view(torch.uint8))
    wide = torch.zeros(len(lens), 500, dtype=torch.int32, device="cuda")      # (the same through the form in pieces)
    wide[:, :3] = table
    got = S().attention_step(q, k, v, kp.clone(), vp.clone(), wide, lengths)
    assert torch.isnan(got[[1, 2, 3, 5]]).all()
    value, bound = want_step(q, keys, k, v, 1 / math.sqrt(d))
    near(got[[0, 6]], value[[0, 6]], bound[[0, 6]], "rows beside wrong ones, in pieces")


def test_attention_step_shared_pages_and_layouts():
    """two rows over the same prompt pages; the same cache with its heads before its tokens; a table and rows that are slices"""
    H, Hk, d, page, dtype = 4, 2, 64, 16, torch.bfloat16
    kp, vp, table, lengths, keys = cache_of([40, 32], Hk, d, page, dtype)
    table[1, :2] = table[0, :2]
    keys[1] = tuple(x[:32] for x in keys[0])
    q, k, v = (randn(2, h, d, dtype=dtype, seed=50 + h) for h in (H, Hk, Hk))
    a = S().attention_step(q, k, v, kp.clone(), vp.clone(), table, lengths)
    near(a, *want_step(q, keys, k, v, 1 / math.sqrt(d)), "shared pages")
    kt, vt = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (kp, vp))
    wide = torch.cat([table, table], 1)[:, :table.shape[1]]
    fused = torch.cat([q, k, v], 1)
    b = S().attention_step(*fused.split([H, Hk, Hk], 1), kt, vt, wide, lengths)
    assert torch.equal(a, b)
    out = torch.zeros(2, H, 2 * d, dtype=dtype, device="cuda")
    S().attention_step(q, None, None, kt, vt, wide, lengths + 1, out=out[..., :d])
    assert torch.equal(out[..., :d], a) and (out[..., d:] == 0).all()


def test_attention_step_offsets_past_32_bits():
    """a cache of 2^32 + elements: the pages in use are its last ones"""
    Hk, d, page, dtype = 2, 128, 64, torch.bfloat16
    P = 2 ** 32 // (page * Hk * d) + 8
    kp, vp = (torch.zeros(P, page, Hk, d, dtype=dtype, device="cuda") for _ in range(2))
    small = cache_of([300], Hk, d, page, dtype, spare=0)
    n = small[0].shape[0]
    kp[-n:], vp[-n:] = small[0], small[1]
    q, k, v = (randn(1, h, d, dtype=dtype, seed=50 + h) for h in (4, Hk, Hk))
    got = S().attention_step(q, k, v, kp, vp, small[2] + (P - n), small[3])
    near(got, *want_step(q, small[4], k, v, 1 / math.sqrt(d)), "far pages")
    slot = int(small[2][0, 300 // page]) + P - n
    assert torch.equal(kp[slot, 300 % page], k[0]) and torch.equal(vp[slot, 300 % page], v[0])


# ---- linear attention --------------------------------------------------------------------------------------------------------------

def check_linear(lens, H, d, dtype, with_state=True, train=True, decays=None, seed=0, scale=None):
    T = sum(lens)
    q, k, v, g = (randn(T, H, d, dtype=dtype, seed=seed + i) for i in range(4))
    decay = torch.tensor(decays if decays is not None else [math.log(1 - 0.5 ** (2 + h)) for h in range(H)], dtype=torch.float32, device="cuda")
    state = randn(len(lens), H, d, d, seed=seed + 5) if with_state else None
    d_last = randn(len(lens), H, d, d, seed=seed + 6)
    seqs = S().Packed(lens, "cuda:0")
    x = [t.requires_grad_(train) if t is not None else None for t in (q, k, v, state)]
    o, last = S().linear_attention(x[0], x[1], x[2], decay, seqs, state=x[3], scale=scale)
    got = {"o": o, "last": last}
    if train:
        grads = torch.autograd.grad((o, last), [t for t in x if t is not None], (g, d_last))
        got.update(zip(("dq", "dk", "dv", "dstate"), grads))
    sc, at = 1 / math.sqrt(d) if scale is None else scale, 0
    for i, n in enumerate(lens):
        part = slice(at, at + n)
        at += n
        val, tot = R.linear(*(t[part].detach().double().cpu() for t in (q, k, v)), decay.double().cpu(), None if state is None else state[i].detach().double().cpu(), sc,
                            g[part].double().cpu() if train else None, d_last[i].double().cpu() if train else None)
        for name, y in got.items():
            mine = y[i] if name in ("last", "dstate") else y[part]
            near(mine, val[name], R.linear_bound(name, val[name], tot[name], n, d, dtype, max(1, abs(sc)) * max(float(x.abs().max()) for x in (q, k, v, g))), f"{name}, {dtype}, length {n}, heads {H}, dim {d}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,H,d", [([1], 1, 8), ([1, 2, 31, 32, 33], 2, 32), ([63, 64, 65, 0, 130], 3, 64), ([100, 7], 2, 80), ([130, 5], 2, 96), ([129, 200], 2, 128)])
def test_linear_attention_and_its_gradients(dtype, lens, H, d):
    check_linear(lens, H, d, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_attention_in_segments(dtype):
    """a sequence of several segments, the last one of a single token, beside short ones and an empty one"""
    lens = [513, 20, 0, 256, 257]
    seqs = S().Packed(lens, "cuda:0")
    assert seqs._segments(2)[2] > len(lens)
    check_linear(lens, 2, 40, dtype)
    check_linear([300, 600], 2, 80, dtype)
    check_linear(lens, 2, 32, dtype, with_state=False)


def test_linear_attention_decays():
    """no decay at all, one that leaves nothing, -inf, and one that grows"""
    for dtype in DTYPES:
        check_linear([70, 300], 4, 32, dtype, decays=[0.0, -40.0, -math.inf, 0.01])
    check_linear([70], 2, 32, torch.float32, scale=-0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_linear_attention_later_tokens_have_no_influence(dtype, poison):
    lens, H, d, bad = [300, 100], 2, 64, 170
    q, k, v, g = (randn(400, H, d, dtype=dtype, seed=i) for i in range(4))
    decay = torch.tensor([-0.01, -0.2], device="cuda")
    seqs = S().Packed(lens, "cuda:0")
    clean = S().linear_attention(q, k, v, decay, seqs)
    x = [t.clone() for t in (q, k, v)]
    for t in x:
        t[bad] = poison
    o, last = S().linear_attention(*x, decay, seqs)
    safe = torch.ones(400, dtype=torch.bool)
    safe[bad:300] = False
    assert torch.equal(o[safe], clean[0][safe]) and torch.equal(last[1], clean[1][1])
    leaf = [t.clone().requires_grad_() for t in (q, k, v)]
    want = torch.autograd.grad(S().linear_attention(*leaf, decay, seqs)[0], leaf, g)
    g[bad] = poison
    got = torch.autograd.grad(S().linear_attention(*leaf, decay, seqs)[0], leaf, g)
    others = torch.ones(400, dtype=torch.bool)
    others[bad] = False
    after = torch.ones(400, dtype=torch.bool)
    after[:bad + 1] = False
    assert torch.equal(got[0][others], want[0][others])
    assert torch.equal(got[1][after], want[1][after]) and torch.equal(got[2][after], want[2][after])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,d", [(1, 1, 8), (3, 2, 40), (5, 3, 64), (2, 2, 128), (70, 4, 24)])
def test_linear_attention_step(dtype, B, H, d):
    q, k, v = (randn(B, H, d, dtype=dtype, seed=i) for i in range(3))
    state = randn(B, H, d, d, seed=4)
    decay = torch.linspace(-0.5, 0.0, H, device="cuda")
    reset = torch.zeros(B, dtype=torch.int64)
    reset[::3] = 256            # (any value but 0)
    state[0] = float("nan")     # a row that begins anew does not look at what it held
    s0 = state.double().cpu()
    out = S().linear_attention_step(q, k, v, decay, state, reset=reset.cuda())
    for b in range(B):
        args = [t[b][None].double().cpu() for t in (q, k, v)]
        val, tot = R.linear(*args, decay.double().cpu(), None if reset[b] else s0[b], 1 / math.sqrt(d))
        near(out[b], val["o"][0], R.linear_bound("o", val["o"][0], tot["o"][0], 1, d, dtype), "o")
        near(state[b], val["last"], R.linear_bound("last", val["last"], tot["last"], 1, d, dtype), "state")
    for kind in (torch.bool, torch.uint8, torch.int32):
        s1, s2 = randn(B, H, d, d, seed=4), randn(B, H, d, d, seed=4)
        r = (reset != 0)
        a = S().linear_attention_step(q, k, v, decay, s1, reset=r.to(kind).cuda())
        b = S().linear_attention_step(q, k, v, decay, s2, reset=reset.cuda())
        assert torch.equal(a, b) and torch.equal(s1, s2)
    assert torch.isfinite(S().linear_attention_step(q, k, v, decay, torch.zeros_like(state))).all()


# ---- together ----------------------------------------------------------------------------------------------------------------------

def test_an_episode_acted_and_trained():
    """A rollout of 6 envs x 40 steps with episodes that end on the way: every env acts token by token (paged cache, linear memory, cleared by the done flag), then the
    episodes are packed (RolloutBuffer.episodes) and run whole.  Both forms hold the same bounds against 64 bits, so they agree within twice those."""
    from taco_amd.rollout import RolloutBuffer
    N, T, H, Hk, d, page = 6, 40, 4, 2, 32, 8
    buf = RolloutBuffer(N, 26, 1, 26, 1, 4, T, 4, 0.99, 0.95, "cuda:0")
    done = (torch.rand(T, N, generator=torch.Generator().manual_seed(1)) < 0.1)
    q, k, v = (randn(T, N, h, d, seed=h + i) for i, h in enumerate((H, Hk, Hk)))
    lq, lk, lv = (randn(T, N, H, d, seed=60 + i) for i in range(3))
    decay = torch.tensor([-0.5, -0.1, -0.02, 0.0], device="cuda")
    kp, vp = (torch.full((N * (T // page), page, Hk, d), float("nan"), device="cuda") for _ in range(2))
    table = torch.randperm(N * (T // page), generator=torch.Generator().manual_seed(2)).view(N, -1).int().cuda()
    lengths = torch.zeros(N, dtype=torch.int32, device="cuda")
    state = torch.zeros(N, H, d, d, device="cuda")
    reset = torch.ones(N, dtype=torch.int64, device="cuda")
    acted, remembered = [], []
    for t in range(T):
        lengths.masked_fill_(reset.bool(), 0)
        acted.append(S().attention_step(q[t], k[t], v[t], kp, vp, table, lengths))
        remembered.append(S().linear_attention_step(lq[t], lk[t], lv[t], decay, state, reset=reset))
        lengths += 1
        buf.done_buf[t] = done[t].float().cuda().view(N, 1)
        reset = done[t].long().cuda()
        buf.step += 1
    seqs = buf.episodes()
    flat = done.clone()
    flat[-1] = True
    ends = torch.nonzero(flat.t().reshape(-1))[:, 0] + 1
    lens = torch.diff(ends, prepend=torch.zeros(1, dtype=ends.dtype)).tolist()
    assert seqs.lengths.tolist() == lens

    def packed(x):
        return x.transpose(0, 1).reshape(N * T, *x.shape[2:])
    whole = S().attention(packed(q), packed(k), packed(v), seqs)
    want = R.attention_heads(*(packed(x).double().cpu() for x in (q, k, v)), lens, 1 / math.sqrt(d), True, torch.float32)["o"]
    near(whole, *want, "whole episodes")
    near(packed(torch.stack(acted)), *want, "token by token")
    o, last = S().linear_attention(packed(lq), packed(lk), packed(lv), decay, seqs)
    at = 0
    steps = packed(torch.stack(remembered))
    for i, n in enumerate(lens):
        val, tot = R.linear(*(packed(x)[at:at + n].double().cpu() for x in (lq, lk, lv)), decay.double().cpu(), None, 1 / math.sqrt(d))
        bound = R.linear_bound("o", val["o"], tot["o"], n, d, torch.float32)
        near(o[at:at + n], val["o"], bound, "linear, whole")
        near(steps[at:at + n], val["o"], bound, "linear, token by token")
        at += n
    ended = done[-1]
    for n_env in range(N):
        i = int((torch.tensor(lens).cumsum(0) == (n_env + 1) * T).nonzero()[0])
        if not ended[n_env]:
            near(state[n_env], last[i].double().cpu(), last[i].abs().double().cpu() * 1e-5 + 1e-5, "the memory an env goes on with")


def test_graphs_and_streams():
    """The acting step captured once and replayed while its inputs and lengths change; the training pass captured with its gradients; two graphs and eager work side
    by side; a stream of its own.  Every replay is compared with the eager result, with eager work between the replays."""
    s = S()
    B, H, Hk, d, page = 3, 4, 2, 64, 16
    kp, vp, table, lengths, _ = cache_of([20, 0, 37], Hk, d, page, torch.float16, width=60, spare=180)
    free = sorted(set(range(kp.shape[0])) - set(table[table >= 0].tolist()))
    for b in range(B):
        for j in range(60):
            if int(table[b, j]) < 0:
                table[b, j] = free.pop()
    q, k, v = (randn(B, h, d, dtype=torch.float16, seed=h) for h in (H, Hk, Hk))
    state, decay, reset = randn(B, H, d, d), torch.full((H,), -0.1, device="cuda"), torch.zeros(B, dtype=torch.bool, device="cuda")
    lin = [randn(B, H, d, dtype=torch.float16, seed=70 + i) for i in range(3)]

    def step(kp, vp, lengths, state):
        a = s.attention_step(q, k, v, kp, vp, table, lengths)
        b = s.linear_attention_step(*lin, decay, state, reset=reset)
        lengths.add_(1)
        return a, b
    mine = [t.clone() for t in (kp, vp, lengths, state)]
    step(*[t.clone() for t in mine])
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*mine)
    T = 150
    lens = [100, 50]
    seqs = s.Packed(lens, "cuda:0")
    train = [randn(T, H, d, dtype=torch.bfloat16, seed=i) for i in range(4)]
    lead = [randn(T, H, d, dtype=torch.bfloat16, seed=80 + i) for i in range(3)]

    def gradients():
        x = [t.detach().requires_grad_() for t in train[:3]]
        y = [t.detach().requires_grad_() for t in lead]
        o = s.attention(*x, seqs)
        p, last = s.linear_attention(*y, decay, seqs)
        return (o.detach(), p.detach(), last.detach()) + torch.autograd.grad((o, p), x + y, (train[3], train[3]))
    gradients()
    torch.cuda.synchronize()
    with torch.cuda.graph(second):
        grads = gradients()
    theirs = [t.clone() for t in (kp, vp, lengths, state)]
    for i in range(5):
        for t in [q, k, v] + lin + train + lead:
            t.copy_(randn(*t.shape, dtype=t.dtype, seed=1000 * i + t.shape[0]))
        reset.copy_(torch.tensor([i % 2 == 0, False, i == 3]))
        graph.replay()
        want = step(*theirs)
        second.replay()
        eager = gradients()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), f"replay {i}"
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(mine, theirs)), f"replay {i}"
        assert all(torch.equal(a, b) for a, b in zip(grads, eager)), f"replay {i}"
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        there = gradients()
        fresh = s.Packed(lens, "cuda:0")
        o = s.attention(*train[:3], fresh)
    torch.cuda.current_stream().wait_stream(other)
    assert all(torch.equal(a, b) for a, b in zip(there, eager)) and torch.equal(o, eager[0])
    cold = s.Packed([10, 5], "cuda:0")
    with pytest.raises(_lib.TacoError, match="before capturing"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            s.attention(*[t[:15] for t in train[:3]], cold)
    torch.cuda.synchronize()


def test_the_same_bits_every_time():
    s = S()
    lens = [300, 513, 64, 1]
    seqs = s.Packed(lens, "cuda:0")
    x = [randn(sum(lens), h, 64, dtype=torch.bfloat16, seed=h).requires_grad_() for h in (8, 2, 2)]
    y = [randn(sum(lens), 4, 64, dtype=torch.float16, seed=40 + i).requires_grad_() for i in range(3)]
    decay = torch.full((4,), -0.05, device="cuda")

    def run():
        o = s.attention(*x, seqs)
        p, last = s.linear_attention(*y, decay, seqs)
        return (o, p, last) + torch.autograd.grad((o, p, last), x + y, (torch.ones_like(o), torch.ones_like(p), torch.ones_like(last)))
    first = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, run()))


def test_what_is_written_in_place_counts_as_changed():
    """a state, a cache or an output that a graph has saved: backward refuses instead of using what a later call wrote there"""
    s = S()
    x = [randn(8, 2, 32, seed=i).requires_grad_() for i in range(3)]
    decay, state, seqs = torch.full((2,), -0.1, device="cuda"), randn(4, 2, 32, 32), s.Packed([2, 2, 2, 2], "cuda:0")
    o, _ = s.linear_attention(*x, decay, seqs, state=state)
    tok = [randn(4, 2, 32, seed=9 + i) for i in range(3)]
    s.linear_attention_step(*tok, decay, state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()
    pages = torch.zeros(4, 4, 2, 32, device="cuda")
    w = torch.ones(1, device="cuda", requires_grad=True)
    y = (pages * w).sum()
    s.attention_step(*tok, pages, pages.clone(), torch.arange(4, dtype=torch.int32, device="cuda").view(4, 1), torch.zeros(4, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        z = [t.detach().clone() for t in tok]
        assert torch.equal(s.linear_attention_step(*z, decay, torch.zeros(4, 2, 32, 32, device="cuda")), s.linear_attention_step(*tok, decay, torch.zeros(4, 2, 32, 32, device="cuda")))


def test_attention_step_room_past_32_bits():
    """a table with room for more than 2^31 tokens (one page, named over and over): a short row reads only its own"""
    H, d, page = 2, 32, 1 << 20
    kp, vp = (torch.zeros(1, page, 1, d, dtype=torch.float16, device="cuda") for _ in range(2))
    kp[0, :40], vp[0, :40] = randn(40, 1, d, dtype=torch.float16, seed=1), randn(40, 1, d, dtype=torch.float16, seed=2)
    q = randn(1, H, d, dtype=torch.float16, seed=3)
    n = torch.tensor([40], dtype=torch.int32, device="cuda")
    wide = torch.zeros(1, 4096, dtype=torch.int32, device="cuda")
    got = S().attention_step(q, None, None, kp, vp, wide, n)
    near(got, *want_step(q, [(kp[0, :40].cpu(), vp[0, :40].cpu())], [None], [None], 1 / math.sqrt(d)), "room past 2^31")
    assert (S().attention_step(q, None, None, kp, vp, wide, torch.zeros_like(n)) == 0).all()


def test_float16_gradients_that_nearly_fill_its_range():
    """an upstream gradient of some thousands (a scaled loss): dP is past 65 504, the gradients themselves are not"""
    d, H, lens = 128, 2, [40, 20]
    T = sum(lens)
    q, k, v, g = (randn(T, H, d, dtype=torch.float16, seed=i, scale=s) for i, s in enumerate((0.25, 0.25, 1.0, 4000.0)))
    q, k, v, g = (x.half() for x in (q, k, v, g))
    assert torch.isfinite(g).all() and float((g.float()[:, 0] @ v.float()[:, 0].T).abs().max()) > 65504
    got = run_attention(q, k, v, lens, True, None, g)
    want = R.attention_heads(*(t.double().cpu() for t in (q, k, v)), lens, 1 / math.sqrt(d), True, torch.float16, g.double().cpu())
    for name, x in zip(("o", "lse", "dq", "dk", "dv"), got):
        assert float(want[name][0].abs().max()) < 65504
        near(x, *want[name], name)
