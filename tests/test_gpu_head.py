"""The scores product (fmidx.head.head_scores) against its formula in 64 bits on
the CPU.

Tolerance: products of 16-bit operands are exact in float32; d of them are added
in some order, each add off by at most a step (2 u, u = 2^-24) of the sum of
magnitudes M = sum |h w|: 2 d u M.  Bias, residual and mask adds are off by u of
what they give (at most u (M + |bias| + |residual| + |mask|) each), tanh by 4 u
of the cap and of its argument's size, and the store by half a step of its type.
"""
import pytest
import torch

from row_mask_oracle import NEG, mask_values, pack, random_fields

U = 2.0 ** -24
gpu = pytest.mark.gpu


def fm():
    import fmidx.constraint
    import fmidx.head
    return fmidx.head.head_scores, fmidx.constraint


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "gpu tests need a HIP device"
    return torch.device("cuda:0")


def make(n, vocab, d, dtype, out, mask, seed, share=None):
    g = torch.Generator().manual_seed(seed)
    x = dict(hidden=torch.randn(n, d, generator=g).to(dtype),
             weight=(torch.randn(vocab, d, generator=g) * 0.5).to(dtype), bias=torch.randn(vocab, generator=g).to(dtype),
             residual=torch.randn(n, vocab, generator=g).to(out))
    member = fields = uni = None
    if mask != "none":
        p = torch.rand(n, 1, generator=g) ** 3 if share is None else torch.full((n, 1), share)
        member = torch.rand(n, vocab, generator=g) < p
        member[n // 2] = False
        uni = torch.rand(vocab, generator=g) < 0.5
    if mask in ("soft", "records"):
        fields = random_fields(n, g, vocab, out, mask == "records")
        if mask == "records" and share is not None:
            fields["flags"] = fields["flags"] & ~2
    x.update(member=member, fields=fields, uni=uni,
             values=mask_values(n, vocab, member, fields, uni, eos=vocab // 3))
    return x


def constraint_of(x, vocab, dev):
    if x["member"] is None:
        return None
    C = fm()[1]
    f, rows = x["fields"], None
    if f is not None:
        rows = C.row_params(len(x["member"]), base=f["base"], v_dist=f["v_dist"], v_uni=f["v_uni"], v_eos=f["v_eos"],
                            flags=f["flags"], special=f["special"], device="cpu").to(dev)
    return C.Constraint(allowed=pack(x["member"]).to(dev), rows=rows, unigrams=pack(x["uni"][None])[0].to(dev),
                        eos=vocab // 3)


def expected(x, softcap, bias, residual, out):
    """(out, tolerance) in 64 bits."""
    h, w = x["hidden"].double(), x["weight"].double()
    y, m = h @ w.t(), h.abs() @ w.abs().t()
    tol = 2 * h.shape[1] * U * m
    if bias:
        y, m = y + x["bias"].double(), m + x["bias"].double().abs()
        tol = tol + U * m
    if softcap:
        y = softcap * torch.tanh(y / softcap)
        tol = tol + 4 * U * (softcap + m)
    if residual:
        y, m = y + x["residual"].double(), m + x["residual"].double().abs()
        tol = tol + U * m
    v = x["values"].double()
    fin = torch.where(v == NEG, torch.zeros_like(v), v)
    y = torch.where(v == NEG, v, y + fin)
    tol = tol + U * (m + fin.abs())
    info = torch.finfo(out)
    return y, tol + torch.where(v == NEG, torch.zeros_like(y), y.abs()) * info.eps / 2 + info.smallest_normal * info.eps


def check(got, y, tol):
    got = got.cpu().double()
    out = y == NEG
    assert torch.equal(got == NEG, out)
    bad = (got - y).abs()[~out] > tol[~out]
    assert not bad.any(), ((got - y).abs()[~out][bad][:5], tol[~out][bad][:5], ((got - y).abs() > tol).nonzero()[:5])


# rows on every side of a tile edge, odd depths and vocabularies
SIZES = [(1, 1, 1), (1, 33, 8), (2, 100, 7), (3, 1000, 64), (5, 257, 130), (16, 515, 96), (17, 1024, 256),
         (33, 300, 72), (64, 777, 128), (65, 513, 200), (100, 2049, 64), (128, 640, 520), (200, 1500, 77),
         (256, 1031, 128), (300, 700, 64), (520, 900, 192)]


@gpu
@pytest.mark.parametrize("mask", ["none", "hard", "soft", "records"])
@pytest.mark.parametrize("dtype,out", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                       (torch.float16, torch.float16), (torch.float16, torch.float32)], ids=str)
@pytest.mark.parametrize("n,vocab,d", SIZES)
def test_head_scores(dev, n, vocab, d, dtype, out, mask):
    head, _ = fm()
    x = make(n, vocab, d, dtype, out, mask, n + vocab + d)
    con = constraint_of(x, vocab, dev)
    for bias, softcap, residual in ((False, 0.0, False), (True, 5.0, True)):
        y, tol = expected(x, softcap, bias, residual, out)
        got = head(x["hidden"].to(dev), x["weight"].to(dev), bias=x["bias"].to(dev) if bias else None, softcap=softcap,
                   residual=x["residual"].to(dev) if residual else None, constraint=con, out_dtype=out)
        assert got.dtype == out and got.shape == (n, vocab)
        check(got, y, tol)


@gpu
@pytest.mark.parametrize("mask", ["hard", "records"])
@pytest.mark.parametrize("share", [0.0, 0.0003, 0.01, 0.9])
@pytest.mark.parametrize("n,vocab,d", [(1, 5003, 256), (7, 20011, 64), (40, 9001, 128), (256, 6007, 64), (270, 3500, 100)])
def test_hard_masks_from_nothing_to_nearly_all(dev, n, vocab, d, share, mask):
    head, _ = fm()
    x = make(n, vocab, d, torch.bfloat16, torch.float32, mask, 7 * n + vocab, share)
    y, tol = expected(x, 0.0, True, False, torch.float32)
    got = head(x["hidden"].to(dev), x["weight"].to(dev), bias=x["bias"].to(dev), constraint=constraint_of(x, vocab, dev),
               out_dtype=torch.float32)
    check(got, y, tol)


# each form of the whole vocabulary's tiles: both sides of every bound on the batch and on one tile per CU
@gpu
@pytest.mark.parametrize("mask", ["none", "hard", "soft"])
@pytest.mark.parametrize("n,vocab,d", [(n, vocab, d) for n, vocab, depths in [
    (2, 16384, (72, 245, 776)), (2, 16385, (245, 768, 769, 776)), (64, 32768, (776, 801)), (64, 32769, (72, 776, 801)),
    (65, 8192, (72, 245)), (65, 8193, (72, 245)), (128, 32769, (72, 245)), (129, 5441, (72, 245)),
    (129, 16385, (72, 245)), (200, 32769, (72, 245)), (513, 1821, (72, 245)), (513, 6600, (72, 245))] for d in depths])
def test_every_tile(dev, n, vocab, d, mask):
    head, _ = fm()
    x = make(n, vocab, d, torch.bfloat16, torch.bfloat16, mask, n + vocab, share=0.8)
    y, tol = expected(x, 0.0, True, False, torch.bfloat16)
    got = head(x["hidden"].to(dev), x["weight"].to(dev), bias=x["bias"].to(dev), constraint=constraint_of(x, vocab, dev))
    check(got, y, tol)


def on(x, dev):
    return {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in x.items()}


# products large enough that the needed tokens are listed first, on both sides of 16, 32 and 64 rows
@gpu
@pytest.mark.parametrize("mask", ["hard", "records"])
@pytest.mark.parametrize("share", [0.0, 0.0003, 0.01, 0.9])
@pytest.mark.parametrize("n,vocab,d", [(1, 5003, 4096), (7, 20011, 1024), (16, 9001, 2110), (17, 25001, 2048),
                                       (64, 50265, 1000), (65, 50265, 997), (256, 60007, 520)])
def test_large_hard_masks(dev, n, vocab, d, share, mask):
    head, _ = fm()
    x = make(n, vocab, d, torch.bfloat16, torch.float32, mask, 7 * n + vocab, share)
    con = constraint_of(x, vocab, dev)
    x = on(x, dev)
    y, tol = expected(x, 3.0, True, True, torch.float32)
    got = head(x["hidden"], x["weight"], bias=x["bias"], softcap=3.0, residual=x["residual"], constraint=con,
               out_dtype=torch.float32)
    check(got, y.cpu(), tol.cpu())


@gpu
@pytest.mark.parametrize("n", [2, 20, 70])
def test_large_lists_around_half_the_vocabulary(dev, n):
    """One more or one fewer needed token than half, NaN in the weight rows that no row needs: gathered on one side,
    all of them on the other."""
    head, C = fm()
    vocab, d = 50001, 1024
    x = on(make(n, vocab, d, torch.float16, torch.float32, "none", n), dev)
    g = torch.Generator(device=dev).manual_seed(n)
    for k in (0, 1, vocab // 2 - 1, vocab // 2, vocab // 2 + 1, vocab):
        pick = torch.randperm(vocab, generator=g, device=dev)[:k]
        member = torch.zeros(n, vocab, dtype=torch.bool, device=dev)
        member[:, pick] = torch.rand(n, k, generator=g, device=dev) < 0.5
        member[n // 2, pick] = True                    # the union is exactly pick
        x["values"] = torch.zeros(n, vocab, device=dev).masked_fill(~member, NEG)
        y, tol = expected(x, 0.0, True, False, torch.float32)
        w = torch.full_like(x["weight"], float("nan"))
        w[pick] = x["weight"][pick]
        got = head(x["hidden"], w, bias=x["bias"], constraint=C.Constraint(allowed=pack(member.cpu()).to(dev)),
                   out_dtype=torch.float32)
        check(got, y.cpu(), tol.cpu())


@gpu
@pytest.mark.parametrize("n", [3, 40])
def test_captured_lists_replay(dev, n):
    """Two captured graphs of listed products and eager calls on another stream between their replays."""
    head, C = fm()
    vocab, d = 50001, 1024
    g = torch.Generator(device=dev).manual_seed(n)
    h = torch.randn(n, d, generator=g, device=dev).to(torch.bfloat16)
    w = torch.randn(vocab, d, generator=g, device=dev).to(torch.bfloat16)
    masks = [pack(torch.rand(n, vocab, generator=torch.Generator().manual_seed(i)) < p).to(dev)
             for i, p in enumerate((0.001, 0.7, 0.004))]
    bits = masks[0].clone()
    con = C.Constraint(allowed=bits)
    head(h, w, constraint=con)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for k in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(head(h, w, constraint=con, softcap=4.0 * k))
        graphs.append(graph)
    side = torch.cuda.Stream()
    for i in range(5):
        bits.copy_(masks[i % 3])
        h.mul_(1.01)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = [head(h, w, constraint=con, softcap=4.0 * k) for k in range(2)]
        for k in (1, 0):
            graphs[k].replay()
        torch.cuda.synchronize()
        for k in range(2):
            assert torch.equal(outs[k], want[k]), (i, k)


@gpu
def test_forbidden_tokens_are_never_used(dev):
    """NaN and infinities in the weight rows, biases and residuals of forbidden tokens leave -inf and nothing else."""
    head, C = fm()
    n, vocab, d = 20, 700, 96
    x = make(n, vocab, d, torch.float16, torch.float16, "none", 3)
    allowed = torch.rand(vocab, generator=torch.Generator().manual_seed(1)) < 0.2
    for junk in (float("nan"), float("inf"), NEG):
        y = dict(x, weight=x["weight"].clone(), bias=x["bias"].clone(), residual=x["residual"].clone())
        for k in ("weight", "bias"):
            y[k][~allowed] = junk
        y["residual"][:, ~allowed] = junk
        member = allowed[None].expand(n, vocab)
        con = C.Constraint(allowed=pack(member).to(dev))
        got = head(y["hidden"].to(dev), y["weight"].to(dev), bias=y["bias"].to(dev), softcap=3.0,
                   residual=y["residual"].to(dev), constraint=con)
        x["values"] = mask_values(n, vocab, member)
        check(got, *expected(x, 3.0, True, True, torch.float16))


@gpu
def test_strides_and_out(dev):
    """Row pitches, odd offsets, 3-D batches, a residual written in place; nothing outside the rows is touched."""
    head, C = fm()
    for dtype in (torch.bfloat16, torch.float16):
        for n, vocab, d in ((6, 301, 64), (48, 515, 128), (70, 1000, 129)):
            x = make(n, vocab, d, dtype, dtype, "hard", n)
            con = constraint_of(x, vocab, dev)
            want = head(x["hidden"].to(dev), x["weight"].to(dev), residual=x["residual"].to(dev), constraint=con)
            wide = torch.zeros(n, d + 11, dtype=dtype, device=dev)
            wide[:, 3:3 + d] = x["hidden"].to(dev)
            wwide = torch.zeros(vocab, d + 5, dtype=dtype, device=dev)
            wwide[:, 1:1 + d] = x["weight"].to(dev)
            buf = torch.full((n + 2, vocab + 9), 7.0, dtype=dtype, device=dev)
            buf[1:-1, 2:2 + vocab] = x["residual"].to(dev)
            view = buf[1:-1, 2:2 + vocab]
            bits = torch.full((n, con.allowed.shape[1] + 3), -1, dtype=torch.int32, device=dev)
            bits[:, :con.allowed.shape[1]] = con.allowed
            c2 = C.Constraint(allowed=bits)
            got = head(wide[:, 3:3 + d], wwide[:, 1:1 + d], residual=view, constraint=c2, out=view)
            assert got.data_ptr() == view.data_ptr()
            assert torch.equal(got, want)
            edge = buf.clone()
            edge[1:-1, 2:2 + vocab] = 7.0
            assert (edge == 7.0).all()
            h3 = x["hidden"].to(dev).view(2, n // 2, d)
            w2 = x["weight"].to(dev).t().contiguous().t()           # columns of unit stride: copied
            c3 = C.Constraint(allowed=con.allowed.view(2, n // 2, -1))
            got = head(h3, w2, residual=x["residual"].to(dev).view(2, n // 2, vocab), constraint=c3)
            assert torch.equal(got.view(n, vocab), want)


@gpu
def test_empty_calls_and_depth_zero(dev):
    head, _ = fm()
    w = torch.zeros(9, 4, dtype=torch.bfloat16, device=dev)
    assert head(w[:0], w).shape == (0, 9)
    assert head(w, w[:0]).shape == (9, 0)
    b = torch.arange(9, device=dev).to(torch.bfloat16)
    assert torch.equal(head(w[:2, :0], w[:, :0], bias=b), b.expand(2, 9))


@gpu
def test_captured_calls_replay(dev):
    """Two captured graphs and eager calls between their replays; each replay equals the eager call."""
    head, _ = fm()
    vocab, d, n = 3001, 256, 24
    x = make(n, vocab, d, torch.bfloat16, torch.float32, "hard", 5, 0.01)
    con = constraint_of(x, vocab, dev)
    w, h = x["weight"].to(dev), x["hidden"].to(dev)
    other = pack(torch.rand(n, vocab, generator=torch.Generator().manual_seed(9)) < 0.3).to(dev)
    bits = con.allowed.clone()
    from fmidx.constraint import Constraint
    con = Constraint(allowed=bits)
    head(h, w, constraint=con, out_dtype=torch.float32)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for k in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(head(h, w, constraint=con, softcap=4.0 * k, out_dtype=torch.float32))
        graphs.append(g)
    first = bits.clone()
    for i in range(4):
        bits.copy_(other if i % 2 else first)
        h.mul_(1.01)
        want = [head(h, w, constraint=con, softcap=4.0 * k, out_dtype=torch.float32) for k in range(2)]
        torch.cuda.synchronize()
        for k in (1, 0):
            graphs[k].replay()
        torch.cuda.synchronize()
        for k in range(2):
            assert torch.equal(outs[k], want[k]), (i, k)


@gpu
def test_two_streams_at_once(dev):
    head, _ = fm()
    x = make(64, 5001, 256, torch.float16, torch.float16, "hard", 6, 0.02)
    con = constraint_of(x, 5001, dev)
    h, w = x["hidden"].to(dev), x["weight"].to(dev)
    want = [head(h, w, constraint=con), head(h * 2, w, constraint=con)]
    h2 = h * 2
    torch.cuda.synchronize()
    got = []
    for a in (h, h2):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got.append(head(a, w, constraint=con))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- together, as they are used ------------------------------------------------------------------------

@gpu
def test_a_documents_training_step_and_decode_step(dev):
    """An index; the constraint at every position of given answers; log-probabilities, a policy step and a
    preference step under it; then the decode step's scores: against the same from the CPU oracle's index."""
    import numpy as np

    from fmidx.constraint import Constraint, prefix_constraint
    from fmidx.index import FMIndex
    from fmidx.losses import policy_loss, preference_loss, token_logprobs
    from oracle.fm_oracle import OracleIndex, allowed_mask

    rng = np.random.default_rng(4)
    vocab, d = 90, 32
    docs = [rng.integers(0, 80, size=int(rng.integers(8, 40))).tolist() for _ in range(50)]
    ours, ora = FMIndex(device=0), OracleIndex()
    ours.initialize(docs, in_memory=True)
    ora.initialize(docs, in_memory=True)
    F = [t for doc in reversed(docs) for t in doc]
    B, L = 6, 7
    answers = torch.tensor([F[s:s + L] for s in rng.integers(0, len(F) - L, B)])
    answers[2, 4:] = -100                                    # padding
    answers[3, 3] = 85                                       # a token no document has
    con = prefix_constraint(ours, answers.to(dev), vocab)
    member = torch.zeros(B, L, vocab, dtype=torch.bool)
    for b in range(B):
        for pos in range(L):
            if (answers[b, :pos + 1] < 0).any():
                continue
            lo, hi = ora.get_range(answers[b, :pos].tolist())
            member[b, pos] = torch.from_numpy(allowed_mask(ora, [lo], [hi], vocab, 10)[0].astype(bool))
    assert torch.equal(con.allowed.cpu().view(B * L, -1), pack(member.view(B * L, vocab)))
    g = torch.Generator().manual_seed(0)
    scores = torch.randn(B, L, vocab, generator=g).to(dev).requires_grad_()
    lp = token_logprobs(scores, answers.to(dev), constraint=con)
    z = torch.where(member, scores.detach().cpu().double(), torch.tensor(NEG, dtype=torch.float64))
    full = z - torch.logsumexp(z, 2, keepdim=True)
    want = full.gather(2, answers.clamp(min=0)[..., None])[..., 0]
    want = torch.where(answers < 0, torch.zeros_like(want), torch.where(want.isnan(), torch.tensor(NEG).double(), want))
    assert torch.equal(torch.isinf(lp.cpu()), torch.isinf(want)) and want.isinf().sum() >= 1
    fin = torch.isfinite(want)
    assert ((lp.detach().cpu().double() - want).abs()[fin] <= 200 * U + want.abs()[fin] * U).all()
    live = (answers >= 0) & fin
    weights = (live / live.sum()).to(dev)
    old = torch.where(fin, want, torch.zeros_like(want)).float().to(dev)
    adv = torch.randn(B, L, generator=g).to(dev)
    out = policy_loss(scores, answers.to(dev), old, adv, weights=weights, ref_logprobs=old, kl_coef=0.1, constraint=con)
    # on the policy itself every ratio is 1: the loss is the weighted mean advantage, negated
    assert abs(out.loss.item() + (weights * adv).sum().item()) <= 1000 * U
    grad = torch.autograd.grad(out.loss, scores, retain_graph=True)[0]
    p = torch.where(member, full.exp(), torch.zeros_like(full))
    hot = torch.nn.functional.one_hot(answers.clamp(min=0), vocab).double()
    c = torch.where(live, -(weights * adv).cpu().double(), torch.zeros(B, L, dtype=torch.float64))[..., None]
    assert ((grad.cpu().double() - torch.where(c != 0, c * (hot - p), torch.zeros_like(p))).abs() <= 2000 * U * c.abs()
            + 1e-30).all()
    cu = (torch.arange(B + 1) * L).to(dev)
    pref = preference_loss(scores, answers.to(dev), cu, weights=weights, constraint=con)
    assert torch.isfinite(pref.loss)
    grad2 = torch.autograd.grad(pref.loss, scores)[0]
    assert not grad2[~live.to(dev)].any() and grad2[live.to(dev)].any()
    # the decode step behind the same prefixes
    hidden = torch.randn(B, d, generator=g).to(torch.bfloat16).to(dev)
    weight = torch.randn(vocab, d, generator=g).to(torch.bfloat16).to(dev)
    head, _ = fm()
    s = head(hidden, weight, constraint=Constraint(allowed=con.allowed[:, 3].contiguous()), out_dtype=torch.float32)
    plain = hidden.cpu().double() @ weight.cpu().double().t()
    m = hidden.cpu().double().abs() @ weight.cpu().double().abs().t()
    assert torch.equal(s.cpu() == NEG, ~member[:, 3])
    assert ((s.cpu().double() - plain).abs()[member[:, 3]] <= ((2 * d + 4) * U * m)[member[:, 3]]).all()


# ---- refusals (no GPU needed) ----------------------------------------------------------------------------

def test_refusals_of_arguments():
    head, _ = fm()
    h, w = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(5, 8, dtype=torch.bfloat16)
    for bad in [lambda: head(h.float(), w.float()), lambda: head(h, w.half()), lambda: head(h, w, bias=w[:, 0].float()),
                lambda: head(h, w, out_dtype=torch.float16), lambda: head(h, w, residual=torch.zeros(2, 5)),
                lambda: head(h.tolist(), w)]:
        with pytest.raises(TypeError):
            bad()
    for bad in [lambda: head(h, w[:, :7]), lambda: head(h, w[0]), lambda: head(h, w, bias=w[:4, 0]),
                lambda: head(h, w, residual=torch.zeros(2, 6, dtype=torch.bfloat16)),
                lambda: head(h, w, out=torch.zeros(1, 5, dtype=torch.bfloat16)),
                lambda: head(h, w)]:                                        # not on a GPU
        with pytest.raises(ValueError):
            bad()


def test_refusals_at_the_c_abi():
    import ctypes
    import math

    from fmidx._lib import last_error, lib
    from fmidx.head import _HeadArgs

    good = dict(d_hidden=16, d_weight=16, d_bias=None, d_residual=None, d_out=16, ld_hidden=8, ld_weight=8,
                ld_residual=0, ld_out=5, B=2, V=5, d=8, d_bits=None, ld_bits=0, d_unigram_bits=None, d_rows=None,
                eos=-1, softcap=0.0, dtype=1, out_dtype=0, d_ws=None, ws_bytes=0)
    for change, text in [(dict(dtype=0), "dtype"), (dict(dtype=3), "dtype"), (dict(out_dtype=2), "dtype"),
                         (dict(B=1 << 21), "out of range"), (dict(V=1 << 31), "out of range"),
                         (dict(d=1 << 31), "out of range"), (dict(d_out=None), "null"), (dict(d_weight=None), "null"),
                         (dict(ld_weight=7), "stride"), (dict(ld_out=4), "stride"),
                         (dict(d_residual=16, ld_residual=4), "stride"), (dict(d_bits=16, ld_bits=0), "ld_bits"),
                         (dict(softcap=-1.0), "softcap"), (dict(softcap=math.nan), "softcap"),
                         (dict(softcap=math.inf), "softcap")]:
        a = _HeadArgs(**{**good, **change})
        assert lib().fm_head_scores(ctypes.byref(a), None) == -1 and text in last_error(), (change, last_error())
    assert lib().fm_head_scores(None, None) == -1
    assert lib().fm_head_workspace(1, 1, None) == -1


def test_struct_matches_the_header():
    from fmidx.head import _HeadArgs
    from test_abi import _header_struct_fields

    assert [f[0] for f in _HeadArgs._fields_] == _header_struct_fields("fm_head_args")


@gpu
def test_gradients_are_refused(dev):
    head, _ = fm()
    w = torch.zeros(5, 8, dtype=torch.bfloat16, device=dev, requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        head(w[:2].detach(), w)
    with torch.no_grad():
        head(w[:2], w)
