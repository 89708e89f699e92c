"""Measured cases of the constrained-scores operators.

Four operators over the next-token scores of a document-constrained model: the log-probability of
chosen tokens under the constraint, the clipped policy loss and the preference loss built on it
(each with its gradient), and the scores product that writes constrained scores from hidden states.
``run`` computes them in plain torch where ``own`` is false and calls ``fmidx`` where it is true.

The constraint is the framework's: packed allowed-token bits (bit t % 32 of word t // 32) and 32-byte
row records (base, v_dist, v_uni, v_eos as float32, flags as uint32, 4 bytes unused, special as int64).
A token's mask value is base, then v_uni for the corpus's tokens (flag 2), then v_dist for the allowed
ones (flag 1) and for ``special`` (flag 8), then v_eos for eos (flag 4); a value of -inf forbids it.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
_EOS = 2                      # the reference processors' default eos token
_NEG = float("-inf")
_CHUNK = 1 << 26              # scores per step of the row-wise plain forms


# ---- cases -----------------------------------------------------------------------------------------
#
# mask: "none"; "hard": the allowed bits alone; "ended": hard rows, some of which only take eos;
#       "soft": the boosts of a soft processor (rows still thinking, restarted, following a document)
# allowed: the mean share of the vocabulary in a hard row's bits

def listed():
    return [
        # rescoring 8 beams of one request: a call that is all latency
        dict(name="logprobs_beams", op="logprobs", rows=8, vocab=151936, dtype="f32", mask="hard", allowed=0.002,
             temperature=1.0, grad=False),
        # scoring a batch of rollouts under a soft processor, no gradient
        dict(name="logprobs_soft", op="logprobs", rows=2048, vocab=128256, dtype="bf16", mask="soft", allowed=0.01,
             temperature=1.0, grad=False),
        # a loss of the caller's own on the log-probabilities; odd vocabulary, rows off any alignment
        dict(name="logprobs_train_odd", op="logprobs", rows=1031, vocab=50265, dtype="f16", mask="hard",
             allowed=0.3, temperature=0.8, grad=True),
        # one short answer
        dict(name="policy_short", op="policy", rows=24, vocab=32001, dtype="f32", mask="hard", allowed=0.01,
             temperature=1.0, kl=0.05),
        # a minibatch of document-constrained rollouts: few tokens allowed per position
        dict(name="policy_documents", op="policy", rows=4096, vocab=128256, dtype="bf16", mask="ended",
             allowed=0.003, temperature=1.0, kl=0.02),
        # the same step without a constraint: every score counts
        dict(name="policy_free", op="policy", rows=1500, vocab=151936, dtype="bf16", mask="none", allowed=1.0,
             temperature=0.7, kl=0.05),
        # two pairs of short answers over a small test vocabulary
        dict(name="preference_short", op="preference", rows=70, pairs=2, vocab=3000, dtype="f32", mask="hard",
             allowed=0.05, temperature=1.0, smoothing=0.0),
        # eight pairs, about 190 tokens an answer, soft boosts
        dict(name="preference_long", op="preference", rows=3001, pairs=8, vocab=128256, dtype="bf16", mask="soft",
             allowed=0.01, temperature=1.0, smoothing=0.1),
        # one sequence's decode step inside a document: a few hundred tokens allowed
        dict(name="head_one", op="head", rows=1, vocab=128256, dim=2048, dtype="bf16", out="f32", mask="hard",
             allowed=0.003, bias=False, softcap=0.0, residual=False),
        # the benchmark's batch, hard-masked: a few percent of the vocabulary in the union
        dict(name="head_documents", op="head", rows=256, vocab=151936, dim=1024, dtype="f16", out="f16",
             mask="ended", allowed=0.0005, bias=True, softcap=0.0, residual=True),
        # the benchmark's batch under a soft processor: every weight row is needed
        dict(name="head_soft", op="head", rows=256, vocab=128256, dim=4096, dtype="bf16", out="f32", mask="soft",
             allowed=0.01, bias=False, softcap=30.0, residual=False),
        # 512 requests of 4 beams, no constraint yet
        dict(name="head_beams", op="head", rows=2048, vocab=128256, dim=2048, dtype="bf16", out="bf16", mask="none",
             allowed=1.0, bias=True, softcap=0.0, residual=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logprobs", "policy", "preference", "head"])
    case = dict(op=op, dtype=rng.choice(["f32", "bf16", "f16"]) if op != "head" else rng.choice(["bf16", "f16"]),
                mask=rng.choice(["none", "hard", "ended", "soft"]))
    vocab = _log_int(rng, 1000, 151936)
    if rng.random() < 0.5:
        vocab = max(1000, vocab // 64 * 64)
    case["vocab"] = vocab
    case["allowed"] = 1.0 if case["mask"] == "none" else math.exp(rng.uniform(math.log(0.0005), math.log(0.5)))
    if op == "head":
        case["dim"] = _log_int(rng, 64, 4096)
        if rng.random() < 0.8:
            case["dim"] = max(64, case["dim"] // 64 * 64)
        # no more products than the largest listed case
        case["rows"] = min(_log_int(rng, 1, 2048), 2048 * 128256 * 2048 // (vocab * case["dim"]))
        case["out"] = rng.choice([case["dtype"], "f32"])
        case["bias"] = rng.random() < 0.5
        case["softcap"] = rng.choice([0.0, 30.0])
        case["residual"] = rng.random() < 0.3
        return case
    # no more scores than the largest listed case holds bytes
    rows = _log_int(rng, 1, 4096)
    case["rows"] = min(rows, 4096 * 128256 * 2 // (vocab * _BYTES[case["dtype"]]))
    case["temperature"] = rng.choice([1.0, 1.0, 0.7, 1.3])
    if op == "logprobs":
        case["grad"] = rng.random() < 0.6
    elif op == "policy":
        case["kl"] = rng.choice([0.0, 0.02, 0.1])
    else:
        case["pairs"] = max(1, min(_log_int(rng, 1, 16), case["rows"] // 2))
        case["rows"] = max(case["rows"], 2)
        case["smoothing"] = rng.choice([0.0, 0.1])
    return case


# ---- inputs ----------------------------------------------------------------------------------------

def _chunks(n, vocab):
    step = max(1, _CHUNK // vocab)
    return [(i, min(i + step, n)) for i in range(0, n, step)]


def _pack(member):
    """bool [n, V] -> int32 [n, ceil(V / 32)], bit t % 32 of word t // 32."""
    n, v = member.shape
    words = (v + 31) // 32
    wide = torch.zeros((n, words * 32), dtype=torch.int32, device=member.device)
    wide[:, :v] = member
    shift = torch.arange(32, dtype=torch.int32, device=member.device)
    return (wide.view(n, words, 32) << shift).sum(2, dtype=torch.int64).to(torch.int32)   # bit 31 wraps


def _unpack(bits, vocab):
    n, words = bits.shape
    shift = torch.arange(32, dtype=torch.int32, device=bits.device)
    return ((bits.unsqueeze(2) >> shift) & 1).bool().view(n, words * 32)[:, :vocab]


def _constraint(case, n, gen, dev, tokens):
    """Allowed bits, row records and the corpus's tokens for n rows.  tokens (or None): the chosen
    tokens, allowed in all but about one row in fifty."""
    mask, vocab = case["mask"], case["vocab"]
    con = dict(bits=None, rows=None, uni=None, fields=None)
    if mask == "none":
        return con
    share = torch.rand(n, 1, generator=gen, device=dev) * 2 * case["allowed"]     # rows differ in width
    keep = torch.rand(n, generator=gen, device=dev) > 0.02
    out = []
    for a, b in _chunks(n, vocab):
        member = torch.rand(b - a, vocab, generator=gen, device=dev) < share[a:b]
        if tokens is not None:
            at = torch.arange(b - a, device=dev)
            t = tokens[a:b].clamp(min=0)
            member[at, t] = torch.where(keep[a:b], True, member[at, t])
        out.append(_pack(member))
    con["bits"] = torch.cat(out)
    con["uni"] = _pack(torch.rand(1, vocab, generator=gen, device=dev) < 0.7)[0].contiguous()
    if mask == "hard":
        return con
    kind = torch.rand(n, generator=gen, device=dev)
    f = dict(base=torch.zeros(n, device=dev), v_dist=torch.zeros(n, device=dev), v_uni=torch.zeros(n, device=dev),
             v_eos=torch.zeros(n, device=dev), flags=torch.zeros(n, dtype=torch.int32, device=dev),
             special=torch.zeros(n, dtype=torch.int64, device=dev))
    if mask == "ended":        # finished rows take eos alone, the others their bits
        f["base"].fill_(_NEG)
        f["flags"] = torch.where(kind < 0.1, 8, 1).to(torch.int32)
        f["special"].fill_(_EOS)
    else:                      # soft: thinking, restarted, following (boost 10, or doubling with the length), ended
        length = torch.randint(0, 7, (n,), generator=gen, device=dev)
        grow = torch.rand(n, generator=gen, device=dev) < 0.25
        f["v_dist"] = torch.where(grow, 10.0 * 2.0 ** length.float(), torch.tensor(10.0, device=dev))
        f["v_uni"] = torch.where(kind < 0.3, 10.0, 5.0)
        f["flags"] = torch.where(kind < 0.15, 0, torch.where(kind < 0.3, 2, torch.where(kind < 0.95, 3, 10)))
        f["flags"] = (f["flags"] | torch.where(torch.rand(n, generator=gen, device=dev) < 0.2, 4, 0)).to(torch.int32)
        f["v_eos"] = f["v_dist"].clone()
        f["special"].fill_(_EOS)
    con["fields"] = f
    rec = torch.zeros((n, 8), dtype=torch.int32, device=dev)
    for k, name in enumerate(("base", "v_dist", "v_uni", "v_eos")):
        rec[:, k] = f[name].view(torch.int32)
    rec[:, 4] = f["flags"]
    rec[:, 6] = f["special"].to(torch.int32)
    con["rows"] = rec.view(torch.uint8)
    return con


def _inputs(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(1000003 * seed + 17)
    n, vocab, dt = case["rows"], case["vocab"], _DTYPES[case["dtype"]]
    st = dict(case=case)
    if case["op"] == "head":
        d = case["dim"]
        st["hidden"] = torch.randn(n, d, generator=gen, device=dev).to(dt)
        st["weight"] = torch.empty(vocab, d, dtype=dt, device=dev)
        for a, b in _chunks(vocab, d):
            st["weight"][a:b] = torch.randn(b - a, d, generator=gen, device=dev) * (3.0 / math.sqrt(d))
        st["bias"] = torch.randn(vocab, generator=gen, device=dev).to(dt) if case["bias"] else None
        st["residual"] = (torch.randn(n, vocab, generator=gen, device=dev).to(_DTYPES[case["out"]])
                          if case["residual"] else None)
        st["con"] = _constraint(case, n, gen, dev, None)
        return st
    st["tokens"] = torch.randint(0, vocab, (n,), generator=gen, device=dev)
    if n >= 16:                # a padded position or two
        st["tokens"][torch.randint(0, n, (max(1, n // 100),), generator=gen, device=dev)] = -100
    con = st["con"] = _constraint(case, n, gen, dev, st["tokens"])
    scores = st["scores"] = torch.empty(n, vocab, dtype=dt, device=dev)
    for a, b in _chunks(n, vocab):
        scores[a:b] = torch.randn(b - a, vocab, generator=gen, device=dev) * 2.5
    lift = torch.rand(n, generator=gen, device=dev) * 12          # a sampled token is mostly a likely one
    at = torch.arange(n, device=dev)
    t = st["tokens"].clamp(min=0)
    scores[at, t] = (scores[at, t].float() + lift).to(dt)
    if case["op"] == "logprobs":
        if case["grad"]:
            st["upstream"] = torch.randn(n, generator=gen, device=dev) / n
        return st
    logp = _plain_forward(scores, st["tokens"], con, case["temperature"])[0]
    logp = torch.where(torch.isfinite(logp), logp, torch.tensor(-1.0, dtype=logp.dtype, device=dev))
    noise = torch.randn(n, generator=gen, device=dev)
    if case["op"] == "policy":
        # no ratio within 1e-3 of a border of the clip, where 32-bit rounding would pick the branch
        old = (logp + 0.15 * noise).float()
        ratio = torch.exp(logp - old)
        near = (ratio - 1.2).abs().minimum((ratio - 0.8).abs()) < 1e-3
        st["old"] = torch.where(near, old + 0.01, old)
        st["ref"] = (logp + 0.3 * torch.randn(n, generator=gen, device=dev)).float() if case["kl"] else None
        st["advantages"] = torch.randn(n, generator=gen, device=dev)
        live = (torch.rand(n, generator=gen, device=dev) > 0.15).float()      # prompt positions weigh nothing
        st["weights"] = live / live.sum().clamp(min=1)
        return st
    p = case["pairs"]
    cut = torch.randperm(n - 1, generator=gen, device=dev)[:2 * p].sort().values + 1
    if len(cut) < 2 * p:       # two rows and one pair
        cut = torch.arange(1, 2 * p + 1, device=dev)
    st["cu"] = torch.cat([torch.zeros(1, dtype=torch.int64, device=dev), cut.to(torch.int64)])  # a tail past the end
    live = (torch.rand(n, generator=gen, device=dev) > 0.25).float()
    st["weights"] = live
    csum = torch.cat([torch.zeros(1, dtype=torch.float64, device=dev), (logp * live).cumsum(0)])
    sums = csum[st["cu"][1:]] - csum[st["cu"][:-1]]
    st["ref"] = (sums + 4 * torch.randn(2 * p, generator=gen, device=dev)).float()
    return st


def _package():
    pkg = os.path.join(os.getcwd(), "fm-index-constrained-decoding_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import fmidx.constraint
    import fmidx.head
    import fmidx.losses
    return fmidx


def prepare(case, seed):
    st = _inputs(case, seed)
    if own:
        fm = _package()
        con = st["con"]
        st["constraint"] = (None if con["bits"] is None else
                            fm.constraint.Constraint(allowed=con["bits"], rows=con["rows"], unigrams=con["uni"],
                                                     eos=_EOS))
        st["fm"] = fm
    return st


# ---- plain forms -----------------------------------------------------------------------------------

def _values(con, a, b, vocab):
    """Mask values [b - a, V] in float32 of rows a .. b, or None."""
    if con["bits"] is None:
        return None
    member = _unpack(con["bits"][a:b], vocab)
    f = con["fields"]
    if f is None:
        return torch.where(member, 0.0, _NEG)
    col = lambda k: f[k][a:b].unsqueeze(1)
    has = lambda bit: (col("flags") & bit) != 0
    ids = torch.arange(vocab, device=member.device).unsqueeze(0)
    v = torch.where(has(2) & _unpack(con["uni"].unsqueeze(0), vocab), col("v_uni"), col("base"))
    v = torch.where((has(1) & member) | (has(8) & (ids == col("special"))), col("v_dist"), v)
    return torch.where(has(4) & (ids == _EOS), col("v_eos"), v)


def _masked(scores, con, a, b):
    """The processor's scores of rows a .. b, in float32: rounded to the scores' type by the add."""
    s = scores[a:b].float()
    v = _values(con, a, b, scores.shape[1])
    if v is None:
        return s
    return torch.where(v == _NEG, _NEG, (s + v).to(scores.dtype).float())


def _plain_forward(scores, tokens, con, temperature):
    """Log-probabilities (64 bits: they are summed over sequences) and log-sums of every row."""
    n, vocab = scores.shape
    logp = torch.empty(n, dtype=torch.float64, device=scores.device)
    lse = torch.empty(n, dtype=torch.float64, device=scores.device)
    for a, b in _chunks(n, vocab):
        z = _masked(scores, con, a, b)
        top = z.max(1, keepdim=True).values.clamp(min=torch.finfo(torch.float32).min)
        lse[a:b] = (torch.exp((z - top) / temperature).sum(1).double().log()
                    + top.squeeze(1).double() / temperature)
        t = tokens[a:b]
        at = torch.arange(b - a, device=scores.device)
        za = z[at, t.clamp(min=0)].double()
        lp = torch.where(za == _NEG, za, za / temperature - lse[a:b])
        logp[a:b] = torch.where(t < 0, torch.zeros_like(lp), lp)
    return logp, lse


def _plain_backward(scores, tokens, con, temperature, lse, coef):
    """d/dscores of sum coef * logp, rows without a log-probability left out."""
    n, vocab = scores.shape
    out = torch.empty_like(scores)
    for a, b in _chunks(n, vocab):
        z = _masked(scores, con, a, b)
        c = coef[a:b].float().unsqueeze(1) / temperature
        g = -torch.exp(z / temperature - lse[a:b].float().unsqueeze(1)) * c
        t = tokens[a:b]
        at = torch.arange(b - a, device=scores.device)
        g[at, t.clamp(min=0)] += c.squeeze(1)
        out[a:b] = torch.where(c == 0, torch.zeros_like(g), g).to(scores.dtype)
    return out


def _live(logp, tokens):
    return (tokens >= 0) & torch.isfinite(logp)


def _policy_terms(st, logp):
    """Per-position loss and its derivative by the log-probability (64 bits)."""
    case = st["case"]
    live = _live(logp, st["tokens"])
    lp = torch.where(live, logp, st["old"].double())
    w, adv = st["weights"].double(), st["advantages"].double()
    r = torch.exp(lp - st["old"].double())
    free, held = r * adv, r.clamp(0.8, 1.2) * adv
    loss = -torch.minimum(free, held)
    slope = torch.where(free <= held, -free, torch.zeros_like(free))
    if case["kl"]:
        d = st["ref"].double() - lp
        loss = loss + case["kl"] * (torch.exp(d) - d - 1)
        slope = slope + case["kl"] * (1 - torch.exp(d))
    zero = torch.zeros_like(w)
    return torch.where(live, w * loss, zero).sum(), torch.where(live, w * slope, zero)


def _preference_terms(st, logp):
    case = st["case"]
    beta, ls, p = 0.1, case["smoothing"], case["pairs"]
    live = _live(logp, st["tokens"])
    w = torch.where(live, st["weights"].double(), torch.zeros_like(logp))
    lp = torch.where(live, logp, torch.zeros_like(logp))
    seq = torch.searchsorted(st["cu"], torch.arange(len(lp), device=lp.device), right=True) - 1
    inside = seq < 2 * p
    sums = torch.zeros(2 * p + 1, dtype=torch.float64, device=lp.device)
    sums.index_add_(0, torch.where(inside, seq, 2 * p), w * lp)
    sums = sums[:2 * p]
    rel = (sums - st["ref"].double()).view(p, 2)
    delta = beta * (rel[:, 0] - rel[:, 1])
    softplus = lambda x: torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))
    loss = ((1 - ls) * softplus(-delta) + ls * softplus(delta)).mean()
    slope = beta / p * (1 / (1 + torch.exp(-delta)) - 1 + ls)
    per = torch.cat([torch.stack([slope, -slope], 1).view(-1), torch.zeros(1, dtype=torch.float64, device=lp.device)])
    return loss, sums, w * per[torch.where(inside, seq, 2 * p)]


def _plain(st):
    case = st["case"]
    if case["op"] == "head":
        h = torch.matmul(st["hidden"].float(), st["weight"].float().t())
        if st["bias"] is not None:
            h = h + st["bias"].float()
        if case["softcap"]:
            h = case["softcap"] * torch.tanh(h / case["softcap"])
        if st["residual"] is not None:
            h = h + st["residual"].float()
        out = torch.empty(h.shape, dtype=_DTYPES[case["out"]], device=h.device)
        for a, b in _chunks(*h.shape):
            v = _values(st["con"], a, b, h.shape[1])
            out[a:b] = h[a:b] if v is None else torch.where(v == _NEG, _NEG, h[a:b] + v)
        return out
    scores, tokens, con, temp = st["scores"], st["tokens"], st["con"], case["temperature"]
    logp, lse = _plain_forward(scores, tokens, con, temp)
    if case["op"] == "logprobs":
        if not case["grad"]:
            return logp.float()
        coef = torch.where(_live(logp, tokens), st["upstream"].double(), torch.zeros_like(logp))
        return logp.float(), _plain_backward(scores, tokens, con, temp, lse, coef)
    if case["op"] == "policy":
        loss, coef = _policy_terms(st, logp)
        return loss.float(), logp.float(), _plain_backward(scores, tokens, con, temp, lse, coef)
    loss, sums, coef = _preference_terms(st, logp)
    return loss.float(), sums.float(), _plain_backward(scores, tokens, con, temp, lse, coef)


# ---- the framework's calls -------------------------------------------------------------------------

def _own(st):
    case, fm, con = st["case"], st["fm"], st["constraint"]
    if case["op"] == "head":
        return fm.head.head_scores(st["hidden"], st["weight"], bias=st["bias"], softcap=case["softcap"],
                                   residual=st["residual"], constraint=con, out_dtype=_DTYPES[case["out"]])
    scores, tokens, temp = st["scores"], st["tokens"], case["temperature"]
    if case["op"] == "logprobs" and not case["grad"]:
        return fm.losses.token_logprobs(scores, tokens, constraint=con, temperature=temp)
    leaf = scores.detach().requires_grad_()
    if case["op"] == "logprobs":
        logp = fm.losses.token_logprobs(leaf, tokens, constraint=con, temperature=temp)
        return logp.detach(), torch.autograd.grad(logp, leaf, st["upstream"])[0]
    if case["op"] == "policy":
        loss, logp = fm.losses.policy_loss(leaf, tokens, st["old"], st["advantages"], weights=st["weights"],
                                           ref_logprobs=st["ref"], clip_low=0.2, clip_high=0.2, kl_coef=case["kl"],
                                           constraint=con, temperature=temp)
    else:
        loss, logp = fm.losses.preference_loss(leaf, tokens, st["cu"], ref_logprobs=st["ref"], weights=st["weights"],
                                               beta=0.1, label_smoothing=case["smoothing"], constraint=con,
                                               temperature=temp)
    return loss.detach(), logp, torch.autograd.grad(loss, leaf)[0]


def run(state):
    return _own(state) if own else _plain(state)


# ---- floors ----------------------------------------------------------------------------------------

def work(case):
    n, vocab, es = case["rows"], case["vocab"], _BYTES[case["dtype"]]
    mask = case["mask"]
    hard = mask in ("hard", "ended")
    share = min(1.0, case["allowed"]) if hard else 1.0       # of the scores that count
    bits = 0 if mask == "none" else n * ((vocab + 31) // 32) * 4
    if mask in ("soft", "ended"):
        bits += 32 * n + vocab // 8
    if case["op"] == "head":
        d = case["dim"]
        # the weight rows that some batch row allows; widths are uniform up to twice the mean
        union = vocab
        if hard:
            none = 1.0 - share
            union = vocab * (1.0 - none ** n)
        out = n * vocab * _BYTES[case["out"]]
        byts = union * d * es + n * d * es + out + bits
        byts += vocab * es if case["bias"] else 0
        byts += n * vocab * share * _BYTES[case["out"]] if case["residual"] else 0
        return {"bytes": byts, "flops": 2.0 * n * vocab * share * d}
    byts = n * vocab * share * es + bits + 12 * n
    flops = 4.0 * n * vocab * share
    if case["op"] != "logprobs" or case["grad"]:
        byts += n * vocab * es + 16 * n
        flops *= 2
    return {"bytes": byts, "flops": flops}


# ---- 64-bit values from the definition ---------------------------------------------------------------

def _exact_rows(st, a, b):
    """log p over the vocabulary of rows a .. b in 64 bits, -inf where a token is out."""
    scores, con, case = st["scores"], st["con"], st["case"]
    vocab = scores.shape[1]
    s = scores[a:b]
    if con["bits"] is None:
        z = s.double()
    else:
        pos = torch.arange(vocab, device=s.device)
        word = con["bits"][a:b].long()[:, pos // 32]
        inside = ((word >> (pos % 32)) & 1) == 1
        del word
        f = con["fields"]
        if f is None:
            z = s.double().masked_fill(~inside, _NEG)
        else:
            corpus = ((con["uni"].long()[pos // 32] >> (pos % 32)) & 1) == 1
            add = f["base"][a:b, None].repeat(1, vocab)
            for i in range(b - a):
                fl = int(f["flags"][a + i])
                if fl & 2:
                    add[i, corpus] = f["v_uni"][a + i]
                if fl & 1:
                    add[i, inside[i]] = f["v_dist"][a + i]
                if fl & 8:
                    add[i, f["special"][a + i]] = f["v_dist"][a + i]
                if fl & 4:
                    add[i, _EOS] = f["v_eos"][a + i]
            # the mask is added in the scores' own type, as the processors add it
            z = (s + add.to(s.dtype)).double() if s.dtype == torch.float32 else \
                (s.float() + add).to(s.dtype).double()
            z = z.masked_fill(add == _NEG, _NEG)
    u = z / case["temperature"]
    return u - torch.logsumexp(u, 1, keepdim=True)


def exact(case, seed):
    st = _inputs(case, seed)
    if case["op"] == "head":
        n, vocab = case["rows"], case["vocab"]
        out = torch.empty((n, vocab), dtype=torch.float64, device=st["hidden"].device)
        h = st["hidden"].double()
        for a, b in _chunks(vocab, max(case["dim"], n)):
            out[:, a:b] = h @ st["weight"][a:b].double().t()
        if st["bias"] is not None:
            out += st["bias"].double()
        if case["softcap"]:
            out = torch.tanh(out / case["softcap"]) * case["softcap"]
        if st["residual"] is not None:
            out += st["residual"].double()
        for a, b in _chunks(n, vocab):
            v = _values(st["con"], a, b, vocab)
            if v is not None:
                out[a:b] = (out[a:b] + v.double()).masked_fill(v == _NEG, _NEG)
        return out
    scores, tokens = st["scores"], st["tokens"]
    n, vocab = scores.shape
    dev = scores.device
    logp = torch.zeros(n, dtype=torch.float64, device=dev)
    spans = [(i, min(i + max(1, _CHUNK // 2 // vocab), n)) for i in range(0, n, max(1, _CHUNK // 2 // vocab))]
    for a, b in spans:
        rows = _exact_rows(st, a, b)
        got = rows.gather(1, tokens[a:b].clamp(min=0)[:, None])[:, 0]
        got = torch.where(torch.isnan(got), torch.full_like(got, _NEG), got)      # nothing allowed at all
        logp[a:b] = torch.where(tokens[a:b] >= 0, got, torch.zeros_like(got))
    if case["op"] == "logprobs":
        if not case["grad"]:
            return logp
        live = (tokens >= 0) & (logp > _NEG)
        first, second = None, st["upstream"].double() * live
    else:
        # the loss by torch's own differentiation of its formula in 64 bits
        live = (tokens >= 0) & (logp > _NEG)
        x = torch.where(live, logp, torch.zeros_like(logp)).requires_grad_()
        if case["op"] == "policy":
            r = torch.exp(x - st["old"].double())
            adv = st["advantages"].double()
            each = -torch.min(r * adv, torch.clamp(r, 0.8, 1.2) * adv)
            if case["kl"]:
                gap = st["ref"].double() - x
                each = each + case["kl"] * (torch.expm1(gap) - gap)
            first = (each * st["weights"].double() * live).sum()
            extra = logp
        else:
            wx = x * st["weights"].double() * live
            cu = st["cu"].tolist()
            sums = torch.stack([wx[i:j].sum() for i, j in zip(cu[:-1], cu[1:])])
            rel = sums - st["ref"].double()
            delta = 0.1 * (rel[0::2] - rel[1::2])
            ls = case["smoothing"]
            first = -((1 - ls) * torch.nn.functional.logsigmoid(delta)
                      + ls * torch.nn.functional.logsigmoid(-delta)).mean()
            extra = sums.detach()
        second = torch.autograd.grad(first, x)[0] * live
    grad = torch.empty((n, vocab), dtype=torch.float64, device=dev)
    for a, b in spans:
        rows = torch.exp(_exact_rows(st, a, b))
        c = (second[a:b] / case["temperature"])[:, None]
        g = -rows * c
        g.scatter_add_(1, tokens[a:b].clamp(min=0)[:, None], c)
        grad[a:b] = torch.where(c == 0, torch.zeros_like(g), g)
    if case["op"] == "logprobs":
        return logp, grad
    return first.detach(), extra, grad
