"""Constrained log-probabilities and the losses on them (fmidx.losses) against
their definitions in 64 bits on the CPU.

Tolerances, in units of u = 2^-24 (half a step of float32), from what the
kernels round.  A row's sum adds V terms, at most V / 256 + 32 of them one after
the other in one lane and the rest in trees: (V / 256 + 64) u.  A term's
exponent (z - m) log2(e) / T is off by 3 roundings of at most 30 ln-units where
the term still counts (exp(-30) of the largest): 90 u, and exp2 by 4 u.  So a
log-probability is off by E = (V / 256 + 160) u, and half a step of itself.
A gradient c (1[t = a] - p) is off by |c| (p (E + (3 x + 8) u) + 2 u [t = a]),
x the exponent's size (at most 150 before p vanishes), plus |dc|, plus half a
step of the type it is stored in (its smallest step near zero).
"""
import numpy as np
import pytest
import torch

from row_mask_oracle import NEG, constrained, mask_values, pack, random_fields

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
gpu = pytest.mark.gpu


def fm():
    import fmidx.constraint
    import fmidx.losses
    return fmidx.losses, fmidx.constraint


# ---- the definition --------------------------------------------------------------------------------

def oracle_logp(z, tokens, temperature):
    """(logp [n], log-probabilities of every token [n, V], live [n]) of constrained scores z (float64)."""
    n, vocab = z.shape
    u = z / temperature
    lse = torch.logsumexp(u, 1, keepdim=True)
    full = torch.where(u == NEG, torch.full_like(u, NEG), u - lse)
    ok = (tokens >= 0) & (tokens < vocab)
    lp = full.gather(1, tokens.clamp(0, vocab - 1)[:, None])[:, 0]
    lp = torch.where(ok, lp, torch.zeros_like(lp))
    return lp, full, ok & (lp != NEG)


def err_logp(vocab, lp):
    return (vocab / 256 + 160) * U + lp.abs() * U


def check_logp(got, want, vocab):
    got = got.cpu().double()
    assert torch.equal(torch.isfinite(got), torch.isfinite(want)), (got, want)
    fin = torch.isfinite(want)
    assert torch.equal(got[~fin], want[~fin])
    bad = (got - want).abs()[fin] > err_logp(vocab, want[fin])
    assert not bad.any(), (got[fin][bad], want[fin][bad])


def check_grad(got, full, tokens, coef, dcoef, temperature, live, dtype, tiny=False):
    """got: the scores' gradient; coef: dL/dlogp (float64), off by dcoef.  tiny: probabilities down to float32's
    subnormals; exp2 gives one of those to a smallest step s, so c p is off by |c| s before its own rounding."""
    vocab = full.shape[1]
    got = got.cpu().double()
    c = torch.where(live, coef, torch.zeros_like(coef)) / temperature
    dc = torch.where(live, dcoef, torch.zeros_like(dcoef)) / temperature
    p = full.exp()
    hot = torch.zeros_like(p)
    hot[torch.arange(len(tokens)), tokens.clamp(0, vocab - 1)] = 1
    c, dc = c[:, None], dc[:, None]
    want = torch.where(c == 0, torch.zeros_like(p), c * (hot - p))
    e = (vocab / 256 + 160) * U + (3 * full.abs().clamp(max=150) / np.log(2) + 8) * U
    tol = c.abs() * (p * e + 2 * U * hot) + dc * (p + hot)
    info = torch.finfo(dtype)
    tol = tol + want.abs() * info.eps / 2 + info.smallest_normal * info.eps
    if tiny:
        tol = tol + c.abs() * 2.0 ** -149
    bad = (got - want).abs() > tol
    assert not bad.any(), ((got - want).abs()[bad][:5], tol[bad][:5], bad.nonzero()[:5])
    assert not got[full == NEG].any(), "a token that is out has a gradient"
    assert not got[~live].any(), "a row that does not count has a gradient"


# ---- cases -----------------------------------------------------------------------------------------

def make(n, vocab, dtype, mask, seed, poison=True):
    """scores, tokens, member, fields, unigrams on the CPU.  Odd rows' out tokens hold NaN, infinities and
    the type's lowest value; some rows allow nothing, some tokens are padding or forbidden."""
    g = torch.Generator().manual_seed(seed)
    scores = (torch.randn(n, vocab, generator=g) * 3).to(dtype)
    tokens = torch.randint(0, vocab, (n,), generator=g)
    member = fields = uni = None
    if mask != "none":
        member = torch.rand(n, vocab, generator=g) < torch.rand(n, 1, generator=g) ** 3
        member[torch.arange(n), tokens] |= torch.rand(n, generator=g) < 0.9
        if n > 2:
            member[n // 2] = False
        uni = torch.rand(vocab, generator=g) < 0.5
    if mask in ("soft", "records"):
        fields = random_fields(n, g, vocab, dtype, mask == "records")
    if n > 4:
        tokens[1], tokens[4] = -100, vocab
    values = mask_values(n, vocab, member, fields, uni, eos=vocab // 3)
    if poison and mask in ("hard", "records"):
        out = values == NEG
        junk = torch.tensor([float("nan"), float("inf"), NEG, torch.finfo(dtype).min]).to(dtype)
        fill = junk[torch.randint(0, 4, (n, vocab), generator=g)]
        scores[1::2] = torch.where(out[1::2], fill[1::2], scores[1::2])
    return scores, tokens, member, fields, uni, values


def constraint_of(member, fields, uni, vocab, dev):
    if member is None:
        return None
    C = fm()[1]
    rows = None
    if fields is not None:
        rows = C.row_params(len(member), base=fields["base"], v_dist=fields["v_dist"], v_uni=fields["v_uni"],
                            v_eos=fields["v_eos"], flags=fields["flags"], special=fields["special"], device="cpu")
        rows = rows.to(dev)
    return C.Constraint(allowed=pack(member).to(dev), rows=rows, unigrams=pack(uni[None])[0].to(dev), eos=vocab // 3)


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "gpu tests need a HIP device"
    return torch.device("cuda:0")


SIZES = [(1, 1), (1, 7), (3, 8), (5, 9), (17, 33), (33, 257), (64, 1000), (6, 4099), (2, 50265)]


@gpu
@pytest.mark.parametrize("mask", ["none", "hard", "soft", "records"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,vocab", SIZES)
def test_token_logprobs(dev, n, vocab, dtype, mask):
    L, _ = fm()
    scores, tokens, member, fields, uni, values = make(n, vocab, dtype, mask, 1000 * n + vocab)
    for temperature in (1.0, 0.6):
        lp, full, live = oracle_logp(constrained(scores, values), tokens, temperature)
        leaf = scores.to(dev).requires_grad_()
        got = L.token_logprobs(leaf, tokens.to(dev), constraint=constraint_of(member, fields, uni, vocab, dev),
                               temperature=temperature)
        check_logp(got.detach(), lp, vocab)
        up = torch.randn(n, generator=torch.Generator().manual_seed(n))
        up[0] = 0
        got.backward(up.to(dev))
        check_grad(leaf.grad, full, tokens, up.double(), up.double().abs() * U, temperature, live, dtype)


@gpu
@pytest.mark.parametrize("n,vocab", [(300, 5003), (1500, 2048), (2500, 333)])
def test_many_rows(dev, n, vocab):
    """Row counts on both sides of the launch rules."""
    L, _ = fm()
    scores, tokens, member, fields, uni, values = make(n, vocab, torch.bfloat16, "soft", n)
    lp, full, live = oracle_logp(constrained(scores, values), tokens, 1.0)
    leaf = scores.to(dev).requires_grad_()
    con = constraint_of(member, fields, uni, vocab, dev)
    got = L.token_logprobs(leaf, tokens.to(dev), constraint=con)
    check_logp(got.detach(), lp, vocab)
    up = torch.randn(n, generator=torch.Generator().manual_seed(n))
    got.backward(up.to(dev))
    check_grad(leaf.grad, full, tokens, up.double(), up.double().abs() * U, 1.0, live, torch.bfloat16)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_equals_the_processors_distribution(dev, dtype):
    """z is fm_apply_boosts' output bit for bit: the log-probabilities of its output without a mask are equal."""
    from ctypes import c_void_p

    from fmidx._lib import check, lib
    from fmidx.processors import _DTYPE_CODE

    L, _ = fm()
    n, vocab = 40, 2049
    scores, tokens, member, fields, uni, _ = make(n, vocab, dtype, "soft", 5)
    con = constraint_of(member, fields, uni, vocab, dev)
    s = scores.to(dev)
    boosted = torch.empty_like(s)
    check(lib().fm_apply_boosts(_DTYPE_CODE[dtype], c_void_p(s.data_ptr()), c_void_p(boosted.data_ptr()), n, vocab,
                                vocab, vocab, c_void_p(con.allowed.data_ptr()), con.allowed.stride(0),
                                c_void_p(con.unigrams.data_ptr()), c_void_p(con.rows.data_ptr()), con.eos,
                                c_void_p(torch.cuda.current_stream().cuda_stream)))
    a = L.token_logprobs(s, tokens.to(dev), constraint=con)
    b = L.token_logprobs(boosted, tokens.to(dev))
    assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("mask", ["none", "hard", "soft", "records"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,vocab", [(5, 9), (17, 600), (300, 5003), (5, 50265), (3, 270001)])
def test_chosen_token_holds_nearly_all(dev, n, vocab, dtype, mask):
    """Log-probabilities near 0, and the gradient 1 - p of their token, keep their digits.  The other tokens'
    sum is off by E = (V / 256 + 160) u of itself, so logp = -log1p(sum) by (1 - p) E, and half a step; the token's
    gradient c (1 - p) by |c| (1 - p) (E + 16 u): the logarithm's and expm1's roundings, 16 for all."""
    L, _ = fm()
    scores, tokens, member, fields, uni, _ = make(n, vocab, dtype, mask, 77 * n + vocab, poison=False)
    rows = torch.arange(n)
    ok = (tokens >= 0) & (tokens < vocab)
    scores[rows[ok], tokens[ok]] = (torch.tensor([12.0, 20.0, 30.0, 45.0])[rows % 4]).to(dtype)[ok]
    if fields is not None:                                   # boosts that leave the token ahead
        for f in ("base", "v_dist", "v_uni", "v_eos"):
            fields[f] = torch.where(torch.isfinite(fields[f]), fields[f].clamp(-2, 2), fields[f])
    values = mask_values(n, vocab, member, fields, uni, eos=vocab // 3)
    z = constrained(scores, values)
    live = ok & (z[rows, tokens.clamp(0, vocab - 1)] != NEG)
    for temperature in (1.0, 0.6):
        u = z / temperature
        za = u[rows, tokens.clamp(0, vocab - 1)]
        others = u.clone()
        others[rows[ok], tokens[ok]] = NEG
        rest = torch.logsumexp(others, 1) - za
        lp = torch.where(live, -torch.log1p(rest.exp()), torch.where(ok, za, torch.zeros_like(za)))
        leaf = scores.to(dev).requires_grad_()
        got = L.token_logprobs(leaf, tokens.to(dev), constraint=constraint_of(member, fields, uni, vocab, dev),
                               temperature=temperature)
        e = (vocab / 256 + 160) * U
        g = got.detach().cpu().double()
        assert torch.equal(g[~live], lp[~live])
        off = (g - lp).abs()[live]
        miss = -torch.expm1(lp[live])                        # 1 - p
        assert (off <= miss * e + lp[live].abs() * U).all(), (off, lp[live])
        up = torch.randn(n, generator=torch.Generator().manual_seed(n))
        got.backward(up.to(dev))
        c = up.double()[live] / temperature
        hot = leaf.grad.cpu().double()[rows[live], tokens[live]]
        info = torch.finfo(dtype)
        tol = c.abs() * miss * (e + 18 * U) + (c * miss).abs() * info.eps / 2 + info.smallest_normal * info.eps
        assert ((hot - c * miss).abs() <= tol).all(), (hot, c * miss)
        _, full, _ = oracle_logp(z, tokens, temperature)
        check_grad(leaf.grad, full, tokens, up.double(), up.double().abs() * U, temperature, live, dtype, tiny=True)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_scores_at_the_types_limits(dev, dtype):
    """In tokens at the lowest value: a row of them is uniform; beside others they vanish."""
    L, _ = fm()
    vocab = 1003
    low = torch.finfo(dtype).min
    scores = torch.full((3, vocab), low, dtype=dtype)
    scores[1, ::2] = 1.0
    scores[2, 5] = torch.finfo(dtype).max
    tokens = torch.tensor([7, 4, 5])
    got = L.token_logprobs(scores.to(dev), tokens.to(dev)).cpu().double()
    want = torch.tensor([-np.log(vocab), -np.log((vocab + 1) // 2), 0.0], dtype=torch.float64)
    assert ((got - want).abs() <= err_logp(vocab, want)).all(), got
    # inf or NaN among the in tokens: the row is NaN, its neighbours are not
    scores = torch.zeros(3, vocab, dtype=dtype)
    scores[1, 9] = float("nan")
    scores[2, 9] = float("inf")
    leaf = scores.to(dev).requires_grad_()
    lp = L.token_logprobs(leaf, tokens.to(dev))
    lp.sum().backward()
    assert torch.isfinite(lp[0]) and torch.isnan(lp[1:]).all()
    assert torch.isfinite(leaf.grad[0]).all() and torch.isnan(leaf.grad[1]).all()


@gpu
def test_strides_and_alignments(dev):
    """Row pitches, odd offsets, 3-D slices, transposes, expanded rows: the same bits as contiguous rows."""
    L, _ = fm()
    g = torch.Generator().manual_seed(3)
    for dtype in DTYPES:
        base = (torch.randn(4, 9, 1013, generator=g) * 3).to(dtype).to(dev)
        tokens = torch.randint(0, 900, (4, 9), generator=g).to(dev)
        views = [base[:, :, :1001], base[:, 1:, 3:1000], base[:, :-1, 1:950], base[::2, ::3, 5:906],
                 base.transpose(0, 1)[:, :, 2:999], base[0, :, 7:940], base[1, 2, 1:990], base[:, :1, :901].expand(4, 9, 901),
                 base[:, :, ::1][:, :, :1013].permute(2, 0, 1)[:9, :, :].permute(1, 2, 0)]
        for v in views:
            v = v.detach()
            t = tokens[:, :].reshape(-1)[: v.numel() // v.shape[-1]].reshape(v.shape[:-1]).clamp(max=v.shape[-1] - 1)
            a, b = v.clone(memory_format=torch.contiguous_format).requires_grad_(), v.requires_grad_()
            x, y = L.token_logprobs(a, t), L.token_logprobs(b, t)
            assert torch.equal(x, y)
            up = torch.randn(x.shape, generator=g).to(dev)
            assert torch.equal(torch.autograd.grad(x, a, up)[0], torch.autograd.grad(y, b, up)[0])
    # int32 and strided tokens, wide bit rows
    s = base[0].detach()
    t = tokens[:, 0]
    assert torch.equal(L.token_logprobs(s[:4], t), L.token_logprobs(s[:4], t.to(torch.int32).contiguous()))


# ---- the losses ------------------------------------------------------------------------------------

def policy_oracle(lp, live, old, adv, w, ref, lo, hi, kl):
    x = torch.where(live, lp, torch.zeros_like(lp)).requires_grad_()
    r = torch.exp(x - old)
    each = -torch.minimum(r * adv, r.clamp(1 - lo, 1 + hi) * adv)
    scale = (r * adv).abs()
    if kl:
        d = ref - x
        each = each + kl * (torch.expm1(d) - d)
        scale = scale + kl * d.exp()
    loss = torch.where(live, w * each, torch.zeros_like(w)).sum()
    return loss, torch.autograd.grad(loss, x)[0], (w.abs() * scale).detach()


@gpu
@pytest.mark.parametrize("mask", ["none", "hard", "soft", "records"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,vocab,kl", [(1, 9, 0.0), (7, 130, 0.3), (65, 1001, 0.0), (600, 3000, 0.1), (1100, 515, 0.1)])
def test_policy_loss(dev, n, vocab, kl, dtype, mask):
    L, _ = fm()
    scores, tokens, member, fields, uni, values = make(n, vocab, dtype, mask, n + vocab)
    T = 0.8
    lp, full, live = oracle_logp(constrained(scores, values), tokens, T)
    g = torch.Generator().manual_seed(n)
    base = torch.where(live, lp, torch.full_like(lp, -2.0))
    old = (base + 0.3 * torch.randn(n, generator=g)).float()
    r = torch.exp(base - old)
    old = torch.where(((r - 0.7).abs() < 1e-3) | ((r - 1.3).abs() < 1e-3), old + 0.02, old)   # off the clip's corners
    adv = torch.randn(n, generator=g)
    w = torch.rand(n, generator=g) / n
    w[torch.rand(n, generator=g) < 0.2] = 0
    ref = (base + 0.3 * torch.randn(n, generator=g)).float()
    if n > 5:
        adv[2] = 0
        old[5] = old[5] - 3                              # far outside the clip
    loss, coef, scale = policy_oracle(lp, live, old.double(), adv.double(), w.double(), ref.double(), 0.3, 0.3, kl)
    leaf = scores.to(dev).requires_grad_()
    got = L.policy_loss(leaf, tokens.to(dev), old.to(dev), adv.to(dev), weights=w.to(dev), ref_logprobs=ref.to(dev),
                        clip_low=0.3, clip_high=0.3, kl_coef=kl,
                        constraint=constraint_of(member, fields, uni, vocab, dev), temperature=T)
    check_logp(got.logprobs, lp, vocab)
    assert not got.logprobs.requires_grad
    e = err_logp(vocab, torch.where(live, lp, torch.zeros_like(lp)))
    assert abs(got.loss.item() - loss.item()) <= (2 * scale * e)[live].sum().item() + abs(loss.item()) * U + 1e-12
    for scale_up in (1.0, 0.25):                         # a loss used as it is, and one divided up
        grad = torch.autograd.grad(got.loss * scale_up, leaf, retain_graph=True)[0]
        check_grad(grad, full, tokens, coef * scale_up, scale_up * (2 * scale * e + 2 * coef.abs() * U), T, live, dtype)
    grad2 = torch.autograd.grad(got.loss, leaf)[0]
    check_grad(grad2, full, tokens, coef, 2 * scale * e + 2 * coef.abs() * U, T, live, dtype)


@gpu
def test_policy_loss_default_weights_and_clip_sides(dev):
    """weights=None is 1 / N; a clipped position has no gradient on the side the minimum drops it."""
    L, _ = fm()
    vocab = 77
    scores = torch.zeros(4, vocab)
    tokens = torch.arange(4)
    lp = -np.log(vocab)
    old = torch.tensor([lp - 0.5, lp - 0.5, lp + 0.5, lp + 0.5])       # r = e^.5, e^.5, e^-.5, e^-.5
    adv = torch.tensor([1.0, -1.0, 1.0, -1.0])
    leaf = scores.to(dev).requires_grad_()
    got = L.policy_loss(leaf, tokens.to(dev), old.to(dev), adv.to(dev))
    r = np.exp([0.5, 0.5, -0.5, -0.5])
    want = (-1.2 + r[1] - r[2] + 0.8) / 4
    assert abs(got.loss.item() - want) <= 2000 * U
    got.loss.backward()
    live = leaf.grad.abs().sum(1).cpu() > 0
    assert live.tolist() == [False, True, True, False]
    assert abs(leaf.grad[1, 1].item() - r[1] / 4 * (1 - 1 / vocab)) <= 2000 * U


def preference_oracle(lp, live, cu, ref, w, beta, ls, margin):
    x = torch.where(live, lp, torch.zeros_like(lp)).requires_grad_()
    wx = torch.where(live, w, torch.zeros_like(w)) * x
    sums = torch.stack([wx[a:b].sum() for a, b in zip(cu[:-1], cu[1:])])
    rel = sums - ref
    D = beta * (rel[0::2] - rel[1::2]) - margin
    sp = torch.nn.functional.softplus
    loss = ((1 - ls) * sp(-D, threshold=100) + ls * sp(D, threshold=100)).mean()
    return loss, sums.detach(), torch.autograd.grad(loss, x)[0]


@gpu
@pytest.mark.parametrize("mask", ["none", "hard", "soft"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,vocab,cu,beta,ls,margin", [
    (2, 5, [0, 1, 2], 0.1, 0.0, 0.0),
    (40, 333, [0, 11, 11, 25, 38], 0.5, 0.1, 0.2),          # an empty sequence, rows behind the last one
    (33, 64, [3, 9, 30, 31, 33], 0.1, 0.0, 0.0),            # rows in front of the first
    (700, 1001, list(range(0, 701, 100))[:7], 2.0, 0.3, 0.0),
    (2100, 257, [0] + sorted(np.random.default_rng(0).choice(2099, 50, replace=False).tolist()), 0.05, 0.0, 0.5),
])
def test_preference_loss(dev, n, vocab, cu, beta, ls, margin, dtype, mask):
    L, _ = fm()
    scores, tokens, member, fields, uni, values = make(n, vocab, dtype, mask, 7 * n + vocab)
    lp, full, live = oracle_logp(constrained(scores, values), tokens, 1.0)
    g = torch.Generator().manual_seed(n)
    w = torch.rand(n, generator=g)
    w[torch.rand(n, generator=g) < 0.2] = 0
    base = torch.where(live, lp, torch.zeros_like(lp)) * w
    ref = torch.stack([base[a:b].sum() for a, b in zip(cu[:-1], cu[1:])])
    ref = (ref + torch.randn(len(ref), generator=g)).float()
    loss, sums, coef = preference_oracle(lp, live, cu, ref.double(), w.double(), beta, ls, margin)
    leaf = scores.to(dev).requires_grad_()
    cud = torch.tensor(cu).to(dev)
    got = L.preference_loss(leaf, tokens.to(dev), cud, ref_logprobs=ref.to(dev), weights=w.to(dev), beta=beta,
                            label_smoothing=ls, margin=margin, constraint=constraint_of(member, fields, uni, vocab, dev))
    e = (w * err_logp(vocab, torch.where(live, lp, torch.zeros_like(lp))))
    es = torch.stack([e[a:b].sum() for a, b in zip(cu[:-1], cu[1:])])
    assert ((got.logprobs.cpu().double() - sums).abs() <= es + sums.abs() * U).all()
    eD = beta * (es[0::2] + es[1::2])
    assert abs(got.loss.item() - loss.item()) <= eD.mean().item() + abs(loss.item()) * U + 1e-12
    # the slope sigma(D) changes by at most a quarter of D's error
    pairs = len(cu) // 2
    ec = torch.zeros(n, dtype=torch.float64)
    for q in range(2 * pairs):
        ec[cu[q]:cu[q + 1]] = beta / pairs * eD[q // 2] / 4
    dcoef = w.double() * ec + 3 * coef.abs() * U
    grad = torch.autograd.grad(got.loss, leaf, retain_graph=True)[0]
    check_grad(grad, full, tokens, coef, dcoef, 1.0, live, dtype)
    half = torch.autograd.grad(0.5 * got.loss, leaf)[0]
    check_grad(half, full, tokens, 0.5 * coef, 0.5 * dcoef, 1.0, live, dtype)


@gpu
def test_preference_bounds_are_clamped(dev):
    """cu_seqlens past the positions, or decreasing, reads nothing outside them."""
    L, _ = fm()
    scores, tokens, *_ = make(20, 50, torch.float32, "none", 1)
    args = dict(beta=0.3)
    t = tokens.to(dev)
    a = L.preference_loss(scores.to(dev), t, torch.tensor([0, 10, 99999]).to(dev), **args)
    b = L.preference_loss(scores.to(dev), t, torch.tensor([-5, 10, 20]).to(dev), **args)
    assert torch.equal(a.loss, b.loss) and torch.equal(a.logprobs, b.logprobs)
    c = L.preference_loss(scores.to(dev), t, torch.tensor([15, 3, 8]).to(dev), **args)
    assert c.logprobs[0].item() == 0 and torch.isfinite(c.loss)
    z = L.preference_loss(scores.to(dev), t, torch.tensor([4]).to(dev), **args)
    assert z.loss.item() == 0 and z.logprobs.numel() == 0


@gpu
def test_gradients_against_differences(dev):
    """A central difference of the float32 losses along a direction d, |d_t| <= 1, of step h = 2^-6.  logp's
    third derivative along d is a third cumulant, at most 8; the losses here bend by at most 16 times that:
    off by h^2 / 6 * 128, and by the losses' own rounding over 2 h."""
    L, _ = fm()
    n, vocab, h = 12, 40, 2.0 ** -6
    g = torch.Generator().manual_seed(11)
    scores = torch.randn(n, vocab, generator=g)
    tokens = torch.randint(0, vocab, (n,), generator=g).to(dev)
    d = (torch.rand(n, vocab, generator=g) * 2 - 1).to(dev)
    member = torch.rand(n, vocab, generator=g) < 0.6
    member[torch.arange(n), tokens.cpu()] = True
    con = fm()[1].Constraint(allowed=pack(member).to(dev))
    old = torch.full((n,), -3.0).to(dev)
    adv, ref = torch.ones(n).to(dev) * 0.1, torch.full((n,), -3.2).to(dev)
    cu = torch.tensor([0, 6, 12]).to(dev)
    fs = [lambda s: L.token_logprobs(s, tokens, constraint=con).mean(),
          lambda s: L.policy_loss(s, tokens, old, -adv, ref_logprobs=ref, kl_coef=0.01, clip_high=50.0,
                                  clip_low=1.0, constraint=con).loss,
          lambda s: L.preference_loss(s, tokens, cu, beta=0.1, constraint=con).loss]
    for f in fs:
        leaf = scores.to(dev).requires_grad_()
        y = f(leaf)
        y.backward()
        slope = (leaf.grad.double() * d.double()).sum().item()
        s = scores.to(dev)
        diff = (f(s + h * d).item() - f(s - h * d).item()) / (2 * h)
        assert abs(diff - slope) <= h * h / 6 * 128 + 400 * U * max(1.0, abs(y.item())) / h, (diff, slope)


@gpu
def test_results_repeat(dev):
    L, _ = fm()
    scores, tokens, member, fields, uni, _ = make(300, 5001, torch.bfloat16, "soft", 2)
    con = constraint_of(member, fields, uni, 5001, dev)
    old, adv = torch.full((300,), -4.0, device=dev), torch.randn(300, generator=torch.Generator().manual_seed(1)).to(dev)
    runs = []
    for _ in range(3):
        leaf = scores.to(dev).requires_grad_()
        out = L.policy_loss(leaf, tokens.to(dev), old, adv, constraint=con)
        runs.append((out.loss.detach(), out.logprobs, torch.autograd.grad(out.loss, leaf)[0]))
    for r in runs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(r, runs[0]))


@gpu
def test_empty_calls(dev):
    L, _ = fm()
    s = torch.empty((0, 9), device=dev, requires_grad=True)
    t = torch.empty((0,), dtype=torch.int64, device=dev)
    f = torch.empty((0,), device=dev)
    lp = L.token_logprobs(s, t)
    assert lp.shape == (0,)
    lp.sum().backward()
    assert s.grad.shape == (0, 9)
    assert L.policy_loss(s, t, f, f).loss.item() == 0
    s3 = torch.empty((2, 0, 9), device=dev)
    assert L.token_logprobs(s3, t.view(2, 0)).shape == (2, 0)


@gpu
def test_other_streams(dev):
    """Two calls at once on two side streams, each with its own workspace."""
    L, _ = fm()
    scores, tokens, *_ = make(64, 30001, torch.bfloat16, "none", 9)
    a = scores.to(dev).requires_grad_()
    b = (scores.float() * 0.5).to(torch.bfloat16).to(dev).requires_grad_()
    t = tokens.to(dev)
    want = [L.token_logprobs(a, t), L.token_logprobs(b, t)]
    wg = [torch.autograd.grad(w.sum(), x)[0] for w, x in zip(want, (a, b))]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s, x in zip(streams, (a, b)):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            y = L.token_logprobs(x, t)
            got.append((y, torch.autograd.grad(y.sum(), x)[0]))
    torch.cuda.synchronize()
    for (y, gr), w, g2 in zip(got, want, wg):
        assert torch.equal(y, w) and torch.equal(gr, g2)


@gpu
def test_saved_tensor_hooks_and_in_place_changes(dev):
    L, _ = fm()
    scores, tokens, member, _, uni, _ = make(8, 257, torch.float32, "hard", 4)
    con = constraint_of(member, None, uni, 257, dev)
    t = tokens.to(dev)
    wide = torch.zeros(8, 300, device=dev)
    wide[:, :257] = scores.to(dev)
    leaf = wide[:, :257].requires_grad_()                  # a row pitch that the saved copy will not have
    want = torch.autograd.grad(L.token_logprobs(leaf, t, constraint=con).sum(), leaf)[0]
    with torch.autograd.graph.save_on_cpu():
        y = L.token_logprobs(leaf, t, constraint=con).sum()
    assert torch.equal(torch.autograd.grad(y, leaf)[0], want)
    x = scores.to(dev).requires_grad_()
    z = x * 1.0
    y = L.token_logprobs(z, t, constraint=con).sum()
    z.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    x = scores.to(dev).requires_grad_()
    gx = torch.autograd.grad(L.token_logprobs(x, t, constraint=con).sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        gx.sum().backward()                                # differentiated once only


@gpu
@pytest.mark.parametrize("n", [5, 1200])
def test_captured_step_replays(dev, n):
    """Forward and backward captured together; every replay equals the eager step on the inputs it then holds."""
    L, _ = fm()
    vocab = 2003
    scores, tokens, member, fields, uni, _ = make(n, vocab, torch.bfloat16, "soft", 8)
    con = constraint_of(member, fields, uni, vocab, dev)
    t = tokens.to(dev)
    s, old, adv = scores.to(dev), torch.full((n,), -5.0, device=dev), torch.ones(n, device=dev)
    w = torch.full((n,), 1.0 / n, device=dev)
    cu = torch.tensor([0, n // 3, n // 2]).to(dev)

    def step(x):
        x = x.detach().requires_grad_()
        a = L.policy_loss(x, t, old, adv, weights=w, ref_logprobs=old, kl_coef=0.1, constraint=con)
        b = L.preference_loss(x, t, cu, weights=w, constraint=con)
        g1 = torch.autograd.grad(a.loss, x, retain_graph=True)[0]
        g2 = torch.autograd.grad(b.loss * 3.0, x)[0]
        return [a.loss.detach(), a.logprobs, b.loss.detach(), b.logprobs, g1, g2]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(s)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(s)
    for k in range(4):
        s.copy_((scores.float() * (1 + 0.3 * k)).to(torch.bfloat16).to(dev))
        adv.fill_(1.0 - k)
        want = step(s)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for i, (x, y) in enumerate(zip(held, want)):
            assert torch.equal(x, y), (k, i)


# ---- refusals (no GPU needed) ------------------------------------------------------------------------

def test_refusals_of_arguments():
    L, C = fm()
    s, t = torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64)
    f = torch.zeros(3)
    for bad in [lambda: L.token_logprobs(s.double(), t), lambda: L.token_logprobs(s, f),
                lambda: L.token_logprobs(s, t.bool()), lambda: L.token_logprobs(s.tolist(), t)]:
        with pytest.raises(TypeError):
            bad()
    for bad in [lambda: L.token_logprobs(s, t[:2]), lambda: L.token_logprobs(s[:, :0], t),
                lambda: L.token_logprobs(s, t),                                  # not on a GPU
                lambda: L.policy_loss(s, t, f, f, clip_low=1.5), lambda: L.policy_loss(s, t, f, f, clip_high=-0.1),
                lambda: L.policy_loss(s, t, f, f, clip_high=float("inf")),
                lambda: L.policy_loss(s, t, f, f, kl_coef=0.1),                  # no reference
                lambda: L.policy_loss(s, t, f, f, kl_coef=float("nan")),
                lambda: L.preference_loss(s, t, t, label_smoothing=1.1),
                lambda: L.preference_loss(s, t, t, beta=float("inf"))]:
        with pytest.raises(ValueError):
            bad()


def test_refusals_of_constraints():
    _, C = fm()
    cpu = torch.device("cpu")
    bits = torch.zeros(3, 2, dtype=torch.int32)
    rows = C.row_params(3, device="cpu")
    C.Constraint(allowed=bits, rows=rows, unigrams=bits[0]).checked(3, 40, cpu)
    C.Constraint(allowed=bits.view(1, 3, 2)).checked(3, 64, cpu)
    for con, n, v in [(C.Constraint(), 3, 40), (C.Constraint(allowed=bits), 3, 65), (C.Constraint(allowed=bits), 2, 40),
                      (C.Constraint(rows=rows[:2]), 3, 40), (C.Constraint(rows=rows[:, :16]), 3, 40),
                      (C.Constraint(allowed=bits, unigrams=bits[0][:1]), 3, 40),
                      (C.Constraint(allowed=bits, unigrams=bits), 3, 40)]:
        with pytest.raises(ValueError):
            con.checked(n, v, cpu)
    for con in [C.Constraint(allowed=bits.long()), C.Constraint(allowed=bits, rows=rows.view(torch.int32)),
                C.Constraint(allowed=bits.bool())]:
        with pytest.raises(TypeError):
            con.checked(3, 40, cpu)
    with pytest.raises(ValueError):
        C.Constraint(allowed=bits).checked(3, 40, torch.device("meta"))


def test_refusals_at_the_c_abi():
    """Bad structs are an error before anything is launched."""
    import ctypes
    import math

    from fmidx._lib import last_error, lib

    L, _ = fm()
    good = dict(d_scores=16, ld_scores=8, ld_outer=0, inner=3, N=3, V=8, d_tokens=16, d_bits=None, ld_bits=0,
                d_unigram_bits=None, d_rows=None, eos=-1, temperature=1.0, dtype=0, reserved=0)
    for change, text in [(dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(V=0), "V = 0"),
                         (dict(V=1 << 31), "out of range"), (dict(N=1 << 22), "out of range"),
                         (dict(temperature=0.0), "temperature"), (dict(temperature=-1.0), "temperature"),
                         (dict(temperature=math.nan), "temperature"), (dict(temperature=math.inf), "temperature"),
                         (dict(temperature=1e-40), "temperature"), (dict(inner=0), "inner"),
                         (dict(d_bits=16, ld_bits=0), "ld_bits"), (dict(d_scores=None), "null"),
                         (dict(d_tokens=None), "null"), (dict(), "workspace")]:
        rows = L._ScoreRows(**{**good, **change})
        rc = lib().fm_token_logprobs(ctypes.byref(rows), None, None, None, 0, None)
        assert rc == -1 and text in last_error(), (change, last_error())
    rows = L._ScoreRows(**good)
    assert lib().fm_token_logprobs(None, None, None, None, 0, None) == -1
    assert lib().fm_token_logprobs(ctypes.byref(rows), None, None, 8, 1 << 20, None) == -1 and "16-B" in last_error()
    assert lib().fm_token_logprobs_grad(ctypes.byref(rows), None, 16, None, 0, 16, 8, None) == -1
    assert lib().fm_token_logprobs_grad(ctypes.byref(rows), 16, 16, None, 0, 16, 7, None) == -1
    assert lib().fm_policy_loss(ctypes.byref(rows), None, None) == -1
    assert lib().fm_preference_loss(ctypes.byref(rows), None, None) == -1
    pol = L._PolicyArgs(16, None, 16, 16, 0.2, 0.2, 0.5, 16, 16, 16, 16, None, 0, 16, 1 << 20)
    assert lib().fm_policy_loss(ctypes.byref(rows), ctypes.byref(pol), None) == -1 and "reference" in last_error()
    for lo, hi in [(1.5, 0.2), (0.2, -1.0), (math.nan, 0.2)]:
        pol = L._PolicyArgs(16, None, 16, 16, lo, hi, 0.0, 16, 16, 16, 16, None, 0, 16, 1 << 20)
        assert lib().fm_policy_loss(ctypes.byref(rows), ctypes.byref(pol), None) == -1 and "clip" in last_error()
    pre = L._PreferenceArgs(16, None, None, 1, 0.1, 2.0, 0.0, 16, 16, 16, 16, 16, 1 << 20)
    assert lib().fm_preference_loss(ctypes.byref(rows), ctypes.byref(pre), None) == -1 and "smoothing" in last_error()
    assert lib().fm_score_workspace(3, 8, 0, None) == -1


def test_structs_match_the_header():
    from test_abi import _header_struct_fields

    L, _ = fm()
    for cls, name in [(L._ScoreRows, "fm_score_rows"), (L._PolicyArgs, "fm_policy_args"),
                      (L._PreferenceArgs, "fm_preference_args")]:
        assert [f[0] for f in cls._fields_] == _header_struct_fields(name)
