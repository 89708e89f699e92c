"""Mask values and constrained scores on the CPU, from the definition: the plain
side of the tests of fmidx.losses and fmidx.head."""
import torch

NEG = float("-inf")


def pack(member):
    """bool [n, V] -> int32 [n, ceil(V / 32)], token t at bit t % 32 of word t // 32."""
    n, v = member.shape
    words = (v + 31) // 32
    wide = torch.zeros((n, words * 32), dtype=torch.int64)
    wide[:, :v] = member
    x = (wide.view(n, words, 32) << torch.arange(32)).sum(2)
    return torch.where(x >= 1 << 31, x - (1 << 32), x).to(torch.int32)


def mask_values(n, vocab, member=None, fields=None, unigrams=None, eos=-1):
    """float32 [n, vocab].  fields: per-row tensors base, v_dist, v_uni, v_eos,
    flags, special; None with member: the hard mask."""
    if fields is None:
        if member is None:
            return torch.zeros(n, vocab)
        return torch.zeros(n, vocab).masked_fill(~member, NEG)
    out = torch.empty(n, vocab)
    for i in range(n):
        row = torch.full((vocab,), float(fields["base"][i]))
        fl, sp = int(fields["flags"][i]), int(fields["special"][i])
        if fl & 2 and unigrams is not None:
            row[unigrams] = fields["v_uni"][i]
        if fl & 1 and member is not None:
            row[member[i]] = fields["v_dist"][i]
        if fl & 8 and 0 <= sp < vocab:
            row[sp] = fields["v_dist"][i]
        if fl & 4 and 0 <= eos < vocab:
            row[eos] = fields["v_eos"][i]
        out[i] = row
    return out


def constrained(scores, values):
    """(scores + values) in the scores' type as float64, -inf where a value is -inf."""
    z = (scores.float() + values).to(scores.dtype).double()
    return z.masked_fill(values == NEG, NEG)


def random_fields(n, gen, vocab, dtype, hard):
    """Row records with every flag in every combination: n should pass 16."""
    rnd = lambda: (torch.randn(n, generator=gen) * 4).to(dtype).float()
    f = dict(base=rnd(), v_dist=rnd() + 8, v_uni=rnd(), v_eos=rnd(), flags=torch.arange(n, dtype=torch.int32) % 16,
             special=torch.randint(0, vocab, (n,), generator=gen))
    f["v_dist"] = f["v_dist"].to(dtype).float()
    if hard:
        f["base"] = torch.full((n,), NEG)
        f["v_uni"][::5] = NEG
        f["v_dist"][1::3] = 0
    return f
