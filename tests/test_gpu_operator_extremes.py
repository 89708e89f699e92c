"""fmidx.losses and fmidx.head at the ends of their ranges: boosts and scores far
from 0, temperatures near 0, NaN and infinities among the tokens that count,
coefficients near the smallest floats, and results read after something else has
written what they were made from.

Expected values are 64-bit definitions on the CPU; tolerances are those of
test_gpu_losses.py unless a test derives its own.
"""
import pytest
import torch

from row_mask_oracle import NEG, constrained, mask_values, pack
from test_gpu_losses import (DTYPES, U, check_grad, check_logp, constraint_of, err_logp, oracle_logp, policy_oracle,
                             preference_oracle)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "gpu tests need a HIP device"
    return torch.device("cuda:0")


def fm():
    import fmidx.constraint
    import fmidx.head
    import fmidx.losses
    return fmidx


# ---- large finite boosts ---------------------------------------------------------------------------

def boosted(lengths, vocab, dtype, eos_rows, seed):
    """Rows that follow a passage of the given lengths: allowed tokens at 10 * 2^length, the corpus's at 5; where
    eos_rows says so the eos has that boost instead and the allowed tokens 10.  Chosen: an allowed token, not eos."""
    g = torch.Generator().manual_seed(seed)
    n, eos = len(lengths), vocab // 3
    scores = (torch.randn(n, vocab, generator=g) * 3).to(dtype)
    member = torch.rand(n, vocab, generator=g) < 0.05
    tokens = torch.randint(0, vocab, (n,), generator=g)
    tokens = torch.where(tokens == eos, tokens + 1, tokens)
    member[torch.arange(n), tokens] = True
    uni = torch.rand(vocab, generator=g) < 0.5
    # the processors round a boost to the scores' type
    large = torch.ldexp(torch.tensor(10.0), torch.tensor(lengths)).to(dtype).float()
    ten, eos_rows = torch.full((n,), 10.0), torch.tensor(eos_rows)
    fields = dict(base=torch.zeros(n), v_dist=torch.where(eos_rows, ten, large), v_uni=ten / 2,
                  v_eos=torch.where(eos_rows, large, ten), flags=torch.where(eos_rows, 7, 3).to(torch.int32),
                  special=torch.full((n,), -1))
    return scores, tokens, member, fields, uni, mask_values(n, vocab, member, fields, uni, eos)


def check_all_losses(dev, scores, tokens, con, values, dtype, T, weigh):
    """All three losses and their gradients; positions outside `weigh` weigh nothing in the last two."""
    L = fm().losses
    n, vocab = scores.shape
    z = constrained(scores, values)
    # relative to the row's maximum before the temperature: 64 bits too lose what scores of 1e30 / T differ by
    lp, full, live = oracle_logp(z - z.amax(1, keepdim=True), tokens, T)
    leaf = scores.to(dev).requires_grad_()
    t = tokens.to(dev)
    g = torch.Generator().manual_seed(n)
    up = torch.randn(n, generator=g)
    got = L.token_logprobs(leaf, t, constraint=con, temperature=T)
    check_logp(got.detach(), lp, vocab)
    if dtype == torch.float16 and T < 1e-3:
        return                                       # a gradient of 1 / T is past float16
    check_grad(torch.autograd.grad(got, leaf, up.to(dev))[0], full, tokens, up.double(), up.double().abs() * U, T, live,
               dtype)
    e = err_logp(vocab, torch.where(live & weigh, lp, torch.zeros_like(lp)))
    base = torch.where(live & weigh, lp, torch.zeros_like(lp))
    w = (weigh / weigh.sum()).float()
    old, ref, adv = (base - 0.1).float(), (base + 0.2).float(), torch.randn(n, generator=g)
    loss, coef, scale = policy_oracle(base, live & weigh, old.double(), adv.double(), w.double(), ref.double(), 0.3, 0.3,
                                      0.2)
    got = L.policy_loss(leaf, t, old.to(dev), adv.to(dev), weights=w.to(dev), ref_logprobs=ref.to(dev), kl_coef=0.2,
                        clip_low=0.3, clip_high=0.3, constraint=con, temperature=T)
    check_logp(got.logprobs, lp, vocab)
    assert abs(got.loss.item() - loss.item()) <= (2 * scale * e)[live].sum().item() + abs(loss.item()) * U + 1e-12
    check_grad(torch.autograd.grad(got.loss, leaf)[0], full, tokens, coef, 2 * scale * e + 2 * coef.abs() * U, T, live,
               dtype)
    if n < 2:
        return
    cu = [0, n // 2, n]
    loss, sums, coef = preference_oracle(base, live & weigh, cu, torch.zeros(2, dtype=torch.float64), w.double(), 0.2, 0.1,
                                         0.0)
    got = L.preference_loss(leaf, t, torch.tensor(cu).to(dev), weights=w.to(dev), beta=0.2, label_smoothing=0.1,
                            constraint=con, temperature=T)
    es = torch.stack([(w.double() * e)[a:b].sum() for a, b in zip(cu[:-1], cu[1:])])
    assert ((got.logprobs.cpu().double() - sums).abs() <= es + sums.abs() * U).all()
    eD = 0.2 * es.sum()
    assert abs(got.loss.item() - loss.item()) <= eD.item() + abs(loss.item()) * U + 1e-12
    check_grad(torch.autograd.grad(got.loss, leaf)[0], full, tokens, coef, w.double() * eD / 4 + 3 * coef.abs() * U, T,
               live, dtype)


@pytest.mark.parametrize("T", [0.7, 1.0, 1.3])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_soft_rows_of_long_passages(dev, dtype, T):
    """Boosts of 10 * 2^length for lengths 0 to 110: on allowed tokens, and on an eos that is not chosen (whose
    position has a log-probability down to -1e34, so it weighs nothing in the losses)."""
    lengths = list(range(111)) * 2
    eos_rows = [i >= 111 for i in range(222)]
    scores, tokens, member, fields, uni, values = boosted(lengths, 4099, dtype, eos_rows, 5)
    con = constraint_of(member, fields, uni, 4099, dev)
    check_all_losses(dev, scores, tokens, con, values, dtype, T, ~torch.tensor(eos_rows))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_soft_rows_of_long_passages_in_slices(dev, dtype):
    """The same past 2^18 tokens, where few rows are cut into slices."""
    vocab = 270001
    scores, tokens, member, fields, uni, values = boosted([3, 29, 40, 60, 95], vocab, dtype, [False] * 5, 6)
    con = constraint_of(member, fields, uni, vocab, dev)
    check_all_losses(dev, scores, tokens, con, values, dtype, 1.0, torch.ones(5, dtype=torch.bool))


@pytest.mark.parametrize("mask", ["none", "hard"])
@pytest.mark.parametrize("vocab", [700, 6200])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_rows_of_large_negative_scores(dev, dtype, vocab, mask):
    """Another processor's fill: whole rows of it, and rows whose first 4096 tokens are filled (whole lanes see
    nothing else for a while)."""
    fills = [-1e8, -1e9, -5e9, -1e10, -1e11, -1e20, -1e29, -1e30]
    g = torch.Generator().manual_seed(vocab)
    n = 2 * len(fills)
    scores = (torch.randn(n, vocab, generator=g) * 3).to(dtype)
    tokens = torch.randint(4096 if vocab > 4096 else 0, vocab, (n,), generator=g)
    for i, fill in enumerate(fills):
        scores[2 * i] = fill
        scores[2 * i + 1, :min(4096, vocab)] = fill
    member = None
    if mask == "hard":
        member = torch.rand(n, vocab, generator=g) < torch.where(torch.arange(n) % 4 < 2, 0.02, 0.9)[:, None]
        member[torch.arange(n), tokens] = True
    values = mask_values(n, vocab, member)
    con = None if member is None else fm().constraint.Constraint(allowed=pack(member).to(dev))
    for T in (0.3, 1.0):
        check_all_losses(dev, scores, tokens, con, values, dtype, T, torch.ones(n, dtype=torch.bool))


@pytest.mark.parametrize("T", [0.3, 1e-6, 1e-9, 1e-12, 1e-20])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_low_temperatures(dev, dtype, T):
    """Ordinary scores; the chosen token is a row's highest, one of two that share it, or another.  The last ones'
    log-probabilities go down to -1e21, so they weigh nothing in the losses."""
    n, vocab = 33, 2500
    g = torch.Generator().manual_seed(2)
    scores = (torch.randn(n, vocab, generator=g) * 3).to(dtype)
    tokens = torch.randint(0, vocab, (n,), generator=g)
    kind = torch.arange(n) % 3
    rows = torch.arange(n)
    top = scores.float().max(1).values.to(dtype)
    scores[rows[kind < 2], tokens[kind < 2]] = top[kind < 2]
    scores[rows[kind == 0], tokens[kind == 0]] = (top.float() + 1).to(dtype)[kind == 0]
    check_all_losses(dev, scores, tokens, None, torch.zeros(n, vocab), dtype, T, kind < 2)


# ---- NaN and infinities ------------------------------------------------------------------------------

@pytest.mark.parametrize("kl", [0.0, 0.1])
@pytest.mark.parametrize("vocab", [50, 270001])
@pytest.mark.parametrize("where", ["nan score", "inf score", "nan old", "nan advantage"])
def test_policy_loss_keeps_nan(dev, where, vocab, kl):
    """One bad position: the loss and that row's gradient are NaN, the other rows as without it; with weight 0 it
    changes nothing."""
    L = fm().losses
    n, bad = 6, 3
    g = torch.Generator().manual_seed(vocab)
    clean = torch.randn(n, vocab, generator=g)
    tokens = torch.randint(0, vocab, (n,), generator=g)
    old = torch.log_softmax(clean, 1)[torch.arange(n), tokens] + 0.4 * torch.randn(n, generator=g)
    for a in (1.0, -1.0, 0.0):
        adv = torch.linspace(-1.0, 1.0, n)
        adv[bad] = a
        runs = []
        for hurt, w in ((False, 1.0), (True, 1.0), (True, 0.0)):
            scores, o, av, weights = clean.clone(), old.clone(), adv.clone(), torch.full((n,), 1.0 / n)
            weights[bad] *= w
            if hurt and where.endswith("score"):
                scores[bad, (tokens[bad] + 7) % vocab] = float(where.split()[0])
            elif hurt:
                (o if where == "nan old" else av)[bad] = float("nan")
            leaf = scores.to(dev).requires_grad_()
            out = L.policy_loss(leaf, tokens.to(dev), o.to(dev), av.to(dev), weights=weights.to(dev),
                                ref_logprobs=old.to(dev) if kl else None, kl_coef=kl)
            runs.append((out.loss, torch.autograd.grad(out.loss, leaf)[0]))
        rest = torch.arange(n) != bad
        assert torch.isfinite(runs[0][0]) and torch.isnan(runs[1][0]) and torch.isfinite(runs[2][0])
        assert torch.isnan(runs[1][1][bad]).all()
        assert not runs[2][1][bad].any()
        for r in runs[1:]:
            assert torch.equal(r[1][rest], runs[0][1][rest])


def test_policy_loss_of_infinite_ratios(dev):
    """exp(logp - old) past every float: the clipped side is finite, an advantage of 0 adds nothing."""
    L = fm().losses
    scores, tokens = torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64)
    leaf = scores.to(dev).requires_grad_()
    old = torch.full((3,), -1e6)
    out = L.policy_loss(leaf, tokens.to(dev), old.to(dev), torch.tensor([1.0, 0.0, 2.0]).to(dev),
                        weights=torch.ones(3).to(dev))
    assert abs(out.loss.item() + 3.6) <= 3.6 * U
    assert not torch.autograd.grad(out.loss, leaf)[0].any()


@pytest.mark.parametrize("mask,vocab", [("hard", 700), ("records", 700), ("records", 4099), ("hard", 250007)])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_forbidden_tokens_of_nan_rows_have_no_gradient(dev, dtype, mask, vocab):
    """NaN in a row's statistics or in its coefficient, or an infinite coefficient: forbidden tokens stay at 0 in
    every form of the mask, tokens that count are NaN or infinite, other rows are untouched."""
    from test_gpu_losses import make

    L = fm().losses
    n = 32
    scores, tokens, member, fields, uni, values = make(n, vocab, dtype, mask, 3, poison=False)
    lp, _, live = oracle_logp(constrained(scores, values), tokens, 1.0)
    con = constraint_of(member, fields, uni, vocab, dev)
    rows = live.nonzero()[:, 0]
    clean = scores.to(dev).requires_grad_()
    want = torch.autograd.grad(L.token_logprobs(clean, tokens.to(dev), constraint=con), clean, torch.ones(n, device=dev))[0]
    up = torch.ones(n)
    hurt = scores.clone()
    hurt[rows[0], tokens[rows[0]]] = float("nan")
    hurt[rows[1], tokens[rows[1]]] = float("inf")
    up[rows[2]], up[rows[3]] = float("nan"), float("inf")
    leaf = hurt.to(dev).requires_grad_()
    got = torch.autograd.grad(L.token_logprobs(leaf, tokens.to(dev), constraint=con), leaf, up.to(dev))[0]
    out = (values == NEG).to(dev)
    assert not got[out].any()
    bad = torch.zeros(n, dtype=torch.bool)
    bad[rows[:4]] = True
    assert torch.equal(got[~bad.to(dev)], want[~bad.to(dev)])
    for r in rows[:4].tolist():
        assert not torch.isfinite(got[r, tokens[r]])


# ---- small coefficients ------------------------------------------------------------------------------

@pytest.mark.parametrize("mask", ["none", "hard", "soft", "records"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_gradients_of_small_coefficients(dev, dtype, mask):
    """Coefficients from 2 down to 2^-130, as many accumulated steps or a mean over many positions make them: every
    gradient that the type can hold.  f32's own smallest results are off by half of their step, 2^-150, twice."""
    from test_gpu_losses import make

    L = fm().losses
    n, vocab = 133, 67
    scores, tokens, member, fields, uni, values = make(n, vocab, dtype, mask, 17)
    lp, full, live = oracle_logp(constrained(scores, values), tokens, 1.0)
    leaf = scores.to(dev).requires_grad_()
    up = torch.ldexp(torch.tensor(1.5), 1 - torch.arange(n)).float()
    got = L.token_logprobs(leaf, tokens.to(dev), constraint=constraint_of(member, fields, uni, vocab, dev))
    check_grad(torch.autograd.grad(got, leaf, up.to(dev))[0], full, tokens, up.double(), up.double() * U + 2.0 ** -149,
               1.0, live, dtype)


def test_bf16_gradients_below_the_exponential(dev):
    """Probabilities under 2^-126, which the hardware's exponential gives up, times coefficients on both sides of
    2^-8: what bf16 can hold of them is there."""
    L = fm().losses
    vocab = 40
    ups = torch.ldexp(torch.tensor(1.25), torch.tensor([20, 3, 0, -1, -6, -7, -8, -9, -20])).float()
    scores = torch.zeros(len(ups), vocab)
    scores[:, 1:] = -torch.linspace(80.0, 100.0, vocab - 1)
    scores = scores.to(torch.bfloat16)
    tokens = torch.zeros(len(ups), dtype=torch.int64)
    lp, full, live = oracle_logp(scores.double(), tokens, 1.0)
    leaf = scores.to(dev).requires_grad_()
    got = torch.autograd.grad(L.token_logprobs(leaf, tokens.to(dev)), leaf, ups.to(dev))[0]
    assert got[0, 1:].cpu().all()
    check_grad(got, full, tokens, ups.double(), ups.double() * U, 1.0, live, torch.bfloat16)


# ---- passes that are replayed apart --------------------------------------------------------------------

def policy_inputs(n, vocab, dev):
    g = torch.Generator().manual_seed(n)
    s = torch.randn(n, vocab, generator=g).to(torch.bfloat16).to(dev)
    t = torch.randint(0, vocab, (n,), generator=g).to(dev)
    return s, t, torch.full((n,), -6.0, device=dev), torch.randn(n, generator=g).to(dev)


def test_captured_forward_with_eager_backward_passes(dev):
    """The gradients that were taken keep their values when the captured forward pass runs again."""
    L = fm().losses
    s, t, old, adv = policy_inputs(40, 1003, dev)
    x = s.clone().requires_grad_()
    L.policy_loss(x, t, old, adv)                       # warm
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = L.policy_loss(x, t, old, adv).loss
    got, want = [], []
    for k in range(3):
        adv.mul_(-1.5)
        y = s.clone().requires_grad_()
        want.append(torch.autograd.grad(L.policy_loss(y, t, old, adv).loss, y)[0])
        graph.replay()
        got.append(torch.autograd.grad(loss, x, retain_graph=True)[0])
        torch.cuda.synchronize()
    for k, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(a, b), k


def test_passes_captured_into_a_graph_each(dev):
    """A backward graph replayed twice behind one forward replay, at two scales."""
    L = fm().losses
    s, t, old, adv = policy_inputs(40, 1003, dev)
    step = torch.cuda.make_graphed_callables(lambda x: L.policy_loss(x, t, old, adv).loss, (s.clone().requires_grad_(),))
    for k in range(3):
        x = (s * (1 + k)).requires_grad_()
        y = (s * (1 + k)).requires_grad_()
        want = L.policy_loss(y, t, old, adv).loss
        loss = step(x)
        for scale in (0.5, 1.0, 0.25):
            a = torch.autograd.grad(loss * scale, x, retain_graph=True)[0].clone()
            b = torch.autograd.grad(want * scale, y, retain_graph=True)[0]
            torch.cuda.synchronize()
            assert torch.equal(a, b), (k, scale)
        assert loss.item() == want.item()


# ---- buffers that kernels write again ------------------------------------------------------------------

def test_bits_written_again_before_the_backward_pass(dev):
    """A decode step or mask call that reuses a constraint's bits, or scores written again by head_scores, before
    backward(): an error, not the gradient of something else."""
    import numpy as np

    from fmidx.index import FMIndex

    M = fm()
    rng = np.random.default_rng(3)
    docs = [rng.integers(0, 60, size=30).tolist() for _ in range(40)]
    ix = FMIndex(device=0)
    ix.initialize(docs, in_memory=True)
    n, vocab, d = 5, 64, 16
    lo = torch.zeros(n, dtype=torch.int64, device=dev)
    hi = torch.full((n,), ix.size(), dtype=torch.int64, device=dev)
    s = torch.randn(n, vocab, generator=torch.Generator().manual_seed(1)).to(dev)
    t = torch.tensor([docs[0][0]] * n, device=dev)
    h = torch.randn(n, d, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(dev)
    w = torch.randn(vocab, d, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(dev)
    for again in ("mask", "step", "head", None):
        bits = ix.allowed_mask(lo, hi, vocab, 10, packed=True)
        con = M.constraint.Constraint(allowed=bits)
        x = s.clone().requires_grad_()
        z = x * 1.0
        loss = M.losses.token_logprobs(z, t, constraint=con).sum()
        if again == "mask":
            ix.allowed_mask(lo, hi, vocab, 10, out=bits, packed=True)
        elif again == "step":
            ix.decode_step(t, lo.clone(), hi.clone(), bits, vocab, 10, packed=True)
        elif again == "head":
            with torch.no_grad():
                M.head.head_scores(h, w, out=z, out_dtype=torch.float32)
        if again:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                loss.backward()
        else:
            loss.backward()
            assert x.grad.any()
    leaf = s.clone().requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        M.head.head_scores(h, w, out=leaf, out_dtype=torch.float32)
    # buffers of inference mode have no versions
    with torch.inference_mode():
        bits = ix.allowed_mask(lo, hi, vocab, 10, packed=True)
        ix.decode_step(t, lo.clone(), hi.clone(), bits, vocab, 10, packed=True)
        out = torch.empty(n, vocab, device=dev)
        M.head.head_scores(h, w, out=out, out_dtype=torch.float32, constraint=M.constraint.Constraint(allowed=bits))


# ---- the soft cap --------------------------------------------------------------------------------------

@pytest.mark.parametrize("listed", [False, True])
def test_soft_cap_to_its_last_bits(dev, listed):
    """tanh alone (a cap of 1, products that add up exactly), f32 out.  1 - 2 / (e + 1), from x = 0.7 on: e is off by
    2 x u from its argument and 2 u of its own, e + 1 by u, the reciprocal by 2 u and the difference by u of the
    result: at 0.7 that is (0.80 * 3.4 + 3) * 0.396 / 0.604 + 1 = 4.8 u, less above.  Below 0.7 the fit, its products
    and its last add: 1.5 u.  So 5 u."""
    M = fm()
    vocab = 70001 if listed else 40001
    g = torch.Generator().manual_seed(4)
    x = torch.exp(torch.rand(vocab, generator=g) * 6.5 - 4.3) * torch.where(torch.rand(vocab, generator=g) < 0.5, 1.0, -1.0)
    hi = x.half()
    lo = ((x - hi.float()) * 2048).half()
    d = 1024 if listed else 2                        # depth for the list of needed tokens to be made
    w = torch.zeros(vocab, d, dtype=torch.float16)
    w[:, 0], w[:, 1] = hi, lo
    h = torch.zeros(1, d, dtype=torch.float16)
    h[0, 0], h[0, 1] = 1.0, 1.0 / 2048
    con, member = None, torch.ones(1, vocab, dtype=torch.bool)
    if listed:
        member = torch.rand(1, vocab, generator=g) < 0.3
        con = M.constraint.Constraint(allowed=pack(member).to(dev))
    got = M.head.head_scores(h.to(dev), w.to(dev), softcap=1.0, constraint=con, out_dtype=torch.float32).cpu().double()
    want = torch.tanh(hi.double() + lo.double() / 2048)
    off = ((got - want).abs() / want.abs())[member[0][None]]
    assert off.max().item() <= 5 * U, off.max().item() / U


def test_soft_cap_of_large_sums(dev):
    """Sums past every float give the cap, NaN stays NaN."""
    M = fm()
    h = torch.full((1, 64), 60000.0, dtype=torch.bfloat16, device=dev)
    w = torch.full((4, 64), 3e38, dtype=torch.bfloat16, device=dev)
    w[1] = -w[0]
    w[2] = float("nan")
    w[3] = 0.0
    got = M.head.head_scores(h, w, softcap=30.0, out_dtype=torch.float32)[0].tolist()
    assert got[0] == 30.0 and got[1] == -30.0 and got[2] != got[2] and got[3] == 0.0
