"""fmidx.losses and fmidx.head where offsets, vocabularies and lists are large:
element offsets past 32 bits, vocabularies past what the kernels hold in LDS or
list, and masks on either side of the product's switch between gathering weight
rows and taking all of them.

Expected values are computed in 64 bits on the GPU, for the rows that are
looked at; tolerances are those of test_gpu_losses.py and test_gpu_head.py.
"""
import pytest
import torch

from row_mask_oracle import NEG, pack
from test_gpu_head import check as check_head
from test_gpu_losses import U, check_grad, check_logp, oracle_logp

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


def test_rows_past_32_bit_offsets(dev):
    """34000 x 128256 bf16: 4.4e9 scores; the last rows lie past 2^32 elements."""
    L = fm().losses
    n, vocab = 34000, 128256
    g = torch.Generator(device=dev).manual_seed(1)
    scores = torch.empty(n, vocab, dtype=torch.bfloat16, device=dev)
    for i in range(0, n, 2000):
        scores[i:i + 2000] = torch.randn(min(2000, n - i), vocab, generator=g, device=dev) * 3
    tokens = torch.randint(0, vocab, (n,), generator=g, device=dev)
    scores.requires_grad_()
    lp = L.token_logprobs(scores, tokens)
    up = torch.randn(n, generator=g, device=dev)
    grad = torch.autograd.grad(lp, scores, up)[0]
    pol = L.policy_loss(scores, tokens, lp.detach() - 0.1, up)
    grad2 = torch.autograd.grad(pol.loss, scores)[0]
    for rows in ([0, 1], [16743, 16744], [33487, 33488, 33999]):
        z = scores.detach()[rows].cpu().double()
        t = tokens[rows].cpu()
        want, full, live = oracle_logp(z, t, 1.0)
        check_logp(lp.detach()[rows], want, vocab)
        u = up[rows].cpu().double()
        check_grad(grad[rows], full, t, u, u.abs() * U, 1.0, live, torch.bfloat16)
        r = torch.exp(want - (lp.detach()[rows] - 0.1).cpu().double())
        c = -r * u / n
        check_grad(grad2[rows], full, t, c, c.abs() * 2000 * U, 1.0, live, torch.bfloat16)
    del scores, grad, grad2
    torch.cuda.empty_cache()


@pytest.mark.parametrize("n,vocab", [(3, 300001), (260, 250007), (300, 245761), (2, 1 << 21)])
@pytest.mark.parametrize("share", [0.0005, 0.2])
def test_hard_masks_over_long_vocabularies(dev, n, vocab, share):
    """Past the words that a workgroup holds in LDS the rows take the general form."""
    M = fm()
    g = torch.Generator(device=dev).manual_seed(n)
    scores = torch.randn(n, vocab, generator=g, device=dev).to(torch.float16)
    bits = torch.zeros(n, (vocab + 31) // 32, dtype=torch.int32, device=dev)
    member = torch.rand(n, vocab, generator=g, device=dev) < share
    for i in range(n):
        bits[i] = pack(member[i:i + 1].cpu())[0].to(dev)
    tokens = member.float().argmax(1)
    tokens[-1] = vocab - 1
    con = M.constraint.Constraint(allowed=bits)
    scores.requires_grad_()
    lp = M.losses.token_logprobs(scores, tokens, constraint=con)
    up = torch.ones(n, device=dev)
    grad = torch.autograd.grad(lp, scores, up)[0]
    old = torch.full((n,), -3.0, device=dev)
    pol = M.losses.policy_loss(scores, tokens, old, up, clip_low=1.0, clip_high=1e6, constraint=con)
    grad2 = torch.autograd.grad(pol.loss, scores)[0]
    assert torch.equal(torch.nan_to_num(pol.logprobs, neginf=-1e9), torch.nan_to_num(lp.detach(), neginf=-1e9))
    rows = sorted({0, n // 2, n - 1})
    z = scores.detach()[rows].cpu().double().masked_fill(~member[rows].cpu(), NEG)
    t = tokens[rows].cpu()
    want, full, live = oracle_logp(z, t, 1.0)
    check_logp(lp.detach()[rows], want, vocab)
    one = torch.ones(len(rows), dtype=torch.float64)
    check_grad(grad[rows], full, t, one, one * U, 1.0, live, torch.float16)
    c = -torch.exp(torch.where(live, want, torch.zeros_like(want)) + 3.0) / n
    check_grad(grad2[rows], full, t, c, c.abs() * (vocab / 256 + 300) * U, 1.0, live, torch.float16)


def head_expected(h, w, member, out):
    h, w = h.double(), w.double()
    y, m = h @ w.t(), h.abs() @ w.abs().t()
    tol = (2 * h.shape[1] + 2) * U * m
    info = torch.finfo(out)
    if member is not None:
        y = y.masked_fill(~member, NEG)
    return y.cpu(), (tol + y.abs().nan_to_num(posinf=0) * info.eps / 2 + info.smallest_normal * info.eps).cpu()


def test_head_past_32_bit_offsets(dev):
    """Outputs past 2^32 elements, and weights past 2^31 elements and 2^32 bytes, gathered and not."""
    M = fm()
    g = torch.Generator(device=dev).manual_seed(2)
    h = torch.randn(34000, 64, generator=g, device=dev).to(torch.bfloat16)
    w = torch.randn(128256, 64, generator=g, device=dev).to(torch.bfloat16)
    got = M.head.head_scores(h, w)
    rows, toks = [0, 33487, 33999], slice(128000, 128256)
    y, tol = head_expected(h[rows], w[toks], None, torch.bfloat16)
    check_head(got[rows][:, toks], y, tol)
    del got
    torch.cuda.empty_cache()
    vocab, d = 600000, 4096
    w = torch.empty(vocab, d, dtype=torch.float16, device=dev)
    for i in range(0, vocab, 50000):
        w[i:i + 50000] = torch.randn(50000, d, generator=g, device=dev) * 0.05
    for n in (3, 40):
        h = torch.randn(n, d, generator=g, device=dev).to(torch.float16)
        member = torch.rand(n, vocab, generator=g, device=dev) < 0.001
        member[:, -2:] = True
        con = M.constraint.Constraint(allowed=pack(member.cpu()).to(dev))
        toks = torch.cat([torch.arange(100), torch.arange(vocab - 300, vocab)]).to(dev)
        for c in (None, con):
            got = M.head.head_scores(h, w, constraint=c, out_dtype=torch.float32)
            y, tol = head_expected(h, w[toks], member[:, toks] if c is not None else None, torch.float32)
            check_head(got[:, toks], y, tol)
    del w
    torch.cuda.empty_cache()


@pytest.mark.parametrize("n", [1, 16, 17, 64, 65, 128, 129, 300])
def test_head_lists_around_half_the_vocabulary(dev, n):
    """One more or one fewer needed token than half: gathered on one side, all of them on the other."""
    M = fm()
    g = torch.Generator(device=dev).manual_seed(n)
    for vocab in (2, 3, 4096, 6145):
        w = torch.randn(vocab, 96, generator=g, device=dev).to(torch.bfloat16)
        h = torch.randn(n, 96, generator=g, device=dev).to(torch.bfloat16)
        for k in {0, 1, vocab // 2 - 1, vocab // 2, vocab // 2 + 1, vocab}:
            if k < 0 or k > vocab:
                continue
            pick = torch.randperm(vocab, generator=g, device=dev)[:k]
            member = torch.zeros(n, vocab, dtype=torch.bool, device=dev)
            member[:, pick] = torch.rand(n, k, generator=g, device=dev) < 0.5
            member[n // 2, pick] = True                    # the union is exactly pick
            con = M.constraint.Constraint(allowed=pack(member.cpu()).to(dev))
            got = M.head.head_scores(h, w, constraint=con, out_dtype=torch.float32)
            y, tol = head_expected(h, w, member, torch.float32)
            check_head(got, y, tol)


def test_head_beyond_the_longest_list(dev):
    """Vocabularies past 2^20 tokens are never gathered."""
    M = fm()
    g = torch.Generator(device=dev).manual_seed(5)
    vocab = (1 << 20) + 9
    w = torch.randn(vocab, 40, generator=g, device=dev).to(torch.float16)
    for n in (2, 70):
        h = torch.randn(n, 40, generator=g, device=dev).to(torch.float16)
        member = torch.rand(n, vocab, generator=g, device=dev) < 0.01
        con = M.constraint.Constraint(allowed=pack(member.cpu()).to(dev))
        got = M.head.head_scores(h, w, constraint=con, out_dtype=torch.float32)
        y, tol = head_expected(h, w, member, torch.float32)
        check_head(got, y, tol)


def test_head_of_the_longest_vocabulary(dev):
    """2^30 tokens, one product each: exact in float32, rounded once."""
    M = fm()
    vocab = 1 << 30
    w = torch.randn(1 << 20, 1, generator=torch.Generator(device=dev).manual_seed(8), device=dev).to(torch.bfloat16)
    h = torch.tensor([[1.375]], dtype=torch.bfloat16, device=dev)
    want = (w.float() * 1.375).to(torch.bfloat16).view(-1)
    got = M.head.head_scores(h, w.repeat(1 << 10, 1))
    assert got.shape == (1, vocab)
    assert all(torch.equal(got[0, i << 20:i + 1 << 20], want) for i in range(1 << 10))


def test_head_of_no_depth_under_a_mask(dev):
    """d = 0: the bias alone, where the mask leaves a token in."""
    M = fm()
    vocab = 500
    bias = torch.arange(vocab, device=dev).to(torch.float16)
    for n in (1, 20, 200):
        member = torch.zeros(n, vocab, dtype=torch.bool)
        member[:, 7::50] = True
        con = M.constraint.Constraint(allowed=pack(member).to(dev))
        e = torch.empty(0, dtype=torch.float16, device=dev)
        got = M.head.head_scores(e.view(n, 0) if n else e, e.view(vocab, 0), bias=bias, constraint=con)
        want = bias.float().cpu().expand(n, vocab).masked_fill(~member, NEG)
        assert torch.equal(got.float().cpu(), want)


def test_head_workspace_is_checked(dev):
    import ctypes

    from fmidx._lib import last_error, lib
    from fmidx.head import _HeadArgs

    need = ctypes.c_uint64()
    assert lib().fm_head_workspace(2, 5000, ctypes.byref(need)) == 0 and need.value > 0
    a = _HeadArgs(d_hidden=16, d_weight=16, d_out=16, ld_hidden=8, ld_weight=8, ld_out=5000, B=2, V=5000, d=8, d_bits=16,
                  ld_bits=157, eos=-1, dtype=1, d_ws=16, ws_bytes=need.value - 1)
    assert lib().fm_head_scores(ctypes.byref(a), None) == -1 and "workspace" in last_error()
    a.d_ws, a.ws_bytes = 8, need.value
    assert lib().fm_head_scores(ctypes.byref(a), None) == -1 and "workspace" in last_error()


def test_the_same_token_and_row_many_times(dev):
    """Every position the same token of the same expanded row: gradients of each position, and their sum."""
    L = fm().losses
    vocab, n = 700, 300
    one = torch.randn(1, vocab, generator=torch.Generator().manual_seed(3)).to(dev).requires_grad_()
    rows = one.expand(n, vocab)
    t = torch.full((n,), 5, device=dev)
    lp = L.token_logprobs(rows, t)
    assert torch.equal(lp, lp[:1].expand(n))
    lp.sum().backward()
    want, full, live = oracle_logp(one.detach().cpu().double(), t[:1].cpu(), 1.0)
    hot = torch.zeros_like(full)
    hot[0, 5] = 1
    assert ((one.grad.cpu().double() - n * (hot - full.exp())).abs() <= n * 400 * U * (full.exp() + hot)).all()


def test_spare_bits_of_the_last_word(dev):
    """Bits past the vocabulary in a row's last word mean nothing, whatever they hold."""
    M = fm()
    for vocab in (33, 2049, 5001, 4097):
        for n in (3, 40, 300):
            g = torch.Generator().manual_seed(vocab + n)
            member = torch.rand(n, vocab, generator=g) < 0.02
            member[:, -1] = True
            clean = pack(member).to(dev)
            dirty = clean.clone()
            dirty[:, -1] |= -1 << (vocab % 32)
            uni = torch.full((clean.shape[1],), -1, dtype=torch.int32, device=dev)
            rows = M.constraint.row_params(n, base=NEG, v_dist=0.0, v_uni=torch.where(torch.arange(n) % 3 == 0, 0.0, 2.0),
                                           flags=torch.where(torch.arange(n) % 2 == 0, 1, 3), device="cpu").to(dev)
            s = torch.randn(n, vocab, generator=g).to(torch.bfloat16).to(dev).requires_grad_()
            t = torch.full((n,), vocab - 1, device=dev)
            h = torch.randn(n, 64, generator=g).to(torch.bfloat16).to(dev)
            w = torch.randn(vocab, 64, generator=g).to(torch.bfloat16).to(dev)
            out = []
            for bits, u in ((clean, uni), (dirty, uni)):
                for r in (None, rows):
                    con = M.constraint.Constraint(allowed=bits, rows=r, unigrams=u)
                    lp = M.losses.token_logprobs(s, t, constraint=con)
                    out.append([lp.detach(), torch.autograd.grad(lp.sum(), s)[0],
                                M.head.head_scores(h, w, constraint=con)])
            for a, b in zip(out[:2], out[2:]):
                assert all(torch.equal(x, y) for x, y in zip(a, b))
            assert torch.isfinite(out[0][0]).all()


def test_inference_mode_and_no_grad(dev):
    M = fm()
    s = torch.randn(4, 99, generator=torch.Generator().manual_seed(1)).to(dev).requires_grad_()
    t = torch.arange(4, device=dev)
    f = torch.zeros(4, device=dev)
    want = M.losses.token_logprobs(s, t).detach()
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            assert torch.equal(M.losses.token_logprobs(s, t), want)
            assert not M.losses.policy_loss(s, t, f, f).loss.requires_grad
            cu = torch.tensor([0, 2, 4], device=dev)
            assert not M.losses.preference_loss(s, t, cu).loss.requires_grad


def test_prefix_constraint_from_ranges(dev):
    """Positions after a forced prefix: its ranges as the start equal the prefix spelled out."""
    import numpy as np

    from fmidx.index import FMIndex

    M = fm()
    rng = np.random.default_rng(9)
    docs = [rng.integers(0, 60, size=30).tolist() for _ in range(40)]
    ix = FMIndex(device=0)
    ix.initialize(docs, in_memory=True)
    F = [t for doc in reversed(docs) for t in doc]
    starts = rng.integers(0, len(F) - 8, 5)
    whole = torch.tensor([F[s:s + 7] for s in starts], device=dev)
    full = M.constraint.prefix_constraint(ix, whole, 64)
    lo, hi = ix.get_range_batch([F[s:s + 2] for s in starts], 10)
    lo, hi = (torch.from_numpy(x.astype(np.int64)).to(dev) for x in (lo, hi))
    keep = lo.clone()
    tail = M.constraint.prefix_constraint(ix, whole[:, 2:].contiguous(), 64, lo=lo, hi=hi)
    assert torch.equal(tail.allowed, full.allowed[:, 2:]) and torch.equal(lo, keep)
    assert M.constraint.prefix_constraint(ix, whole[:0], 64).allowed.shape == (0, 7, 2)
    for bad in (lambda: M.constraint.prefix_constraint(ix, whole, 64, lo=lo),
                lambda: M.constraint.prefix_constraint(ix, whole, 0),
                lambda: M.constraint.prefix_constraint(ix, whole.int(), 64),
                lambda: M.constraint.prefix_constraint(ix, whole.cpu(), 64),
                lambda: M.constraint.prefix_constraint(ix, whole, 64, lo=lo[:2], hi=hi[:2])):
        with pytest.raises(ValueError):
            bad()


def test_two_graphs_and_eager_calls_between(dev):
    """Two captured training steps whose scratch the capture's pools hold, replayed in either order with eager
    calls between: each replay equals the eager step."""
    L = fm().losses
    n, vocab = 300, 20001
    g = torch.Generator(device=dev).manual_seed(8)
    s = torch.randn(n, vocab, generator=g, device=dev).to(torch.bfloat16)
    t = torch.randint(0, vocab, (n,), generator=g, device=dev)
    old, adv = torch.full((n,), -9.0, device=dev), torch.randn(n, generator=g, device=dev)

    def step(temperature):
        x = s.detach().requires_grad_()
        out = L.policy_loss(x, t, old, adv, temperature=temperature)
        return out.loss.detach(), out.logprobs, torch.autograd.grad(out.loss, x)[0]

    step(1.0)
    torch.cuda.synchronize()
    graphs, held = [], []
    for temperature in (1.0, 0.5):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(step(temperature))
        graphs.append(graph)
    for k in range(3):
        s.mul_(0.9)
        want = [step(1.0), step(0.5)]
        torch.cuda.synchronize()
        for i in ((0, 1), (1, 0))[k % 2]:
            graphs[i].replay()
        torch.cuda.synchronize()
        for h, w in zip(held, want):
            assert all(torch.equal(a, b) for a, b in zip(h, w))


@pytest.mark.parametrize("mask", ["none", "hard", "soft", "records"])
@pytest.mark.parametrize("n", [1, 5, 20])
def test_few_rows_of_long_vocabularies(dev, n, mask):
    """Rows cut into slices (few of them, past 2^18 tokens): all three losses against 64 bits."""
    from test_gpu_losses import constraint_of, err_logp, make, policy_oracle, preference_oracle
    from row_mask_oracle import constrained

    L = fm().losses
    vocab = 270001
    for dtype in (torch.float32, torch.bfloat16):
        scores, tokens, member, fields, uni, values = make(n, vocab, dtype, mask, n)
        con = constraint_of(member, fields, uni, vocab, dev)
        want, full, live = oracle_logp(constrained(scores, values), tokens, 0.9)
        t = tokens.to(dev)
        leaf = scores.to(dev).requires_grad_()
        lp = L.token_logprobs(leaf, t, constraint=con, temperature=0.9)
        check_logp(lp.detach(), want, vocab)
        up = torch.randn(n, generator=torch.Generator().manual_seed(n))
        check_grad(torch.autograd.grad(lp, leaf, up.to(dev))[0], full, tokens, up.double(), up.double().abs() * U, 0.9,
                   live, dtype)
        base = torch.where(live, want, torch.full_like(want, -2.0))
        old, ref = (base - 0.1).float(), (base + 0.2).float()
        one = torch.ones(n)
        loss, coef, scale = policy_oracle(want, live, old.double(), one.double(), one.double() / n, ref.double(), 0.3,
                                          0.3, 0.2)
        got = L.policy_loss(leaf, t, old.to(dev), one.to(dev), ref_logprobs=ref.to(dev), kl_coef=0.2, clip_low=0.3,
                            clip_high=0.3, constraint=con, temperature=0.9)
        e = err_logp(vocab, torch.where(live, want, torch.zeros_like(want)))
        check_logp(got.logprobs, want, vocab)
        assert abs(got.loss.item() - loss.item()) <= (2 * scale * e)[live].sum().item() + abs(loss.item()) * U + 1e-12
        check_grad(torch.autograd.grad(got.loss, leaf)[0], full, tokens, coef, 2 * scale * e + 2 * coef.abs() * U, 0.9,
                   live, dtype)
        if n >= 5:
            cu = [1, 3, n - 1]
            loss, sums, coef = preference_oracle(want, live, cu, torch.zeros(2, dtype=torch.float64), one.double(), 0.2,
                                                 0.1, 0.0)
            got = L.preference_loss(leaf, t, torch.tensor(cu).to(dev), beta=0.2, label_smoothing=0.1, constraint=con,
                                    temperature=0.9)
            es = torch.stack([e[a:b].sum() for a, b in zip(cu[:-1], cu[1:])])
            assert ((got.logprobs.cpu().double() - sums).abs() <= es + sums.abs() * U).all()
            eD = 0.2 * es.sum()
            assert abs(got.loss.item() - loss.item()) <= eD.item() + abs(loss.item()) * U + 1e-12
            check_grad(torch.autograd.grad(got.loss, leaf)[0], full, tokens, coef, 0.2 * eD / 4 + 3 * coef.abs() * U,
                       0.9, live, dtype)
