"""Attention in 64 bits with a per-element error bound, for the GPU tests of the decode and prefill
forms (torch, on the GPU).

A kernel rounds each weight exp(s - m) to bf16 (half a step, 2^-8 of it, in the product and in the
sum alike) and the quotient once more, and its scores carry the fp32 sum over the head dim.  With
weights p (1 + e), |e| <= E:
  |sum p (1+e) v / sum p (1+e) - o| <= E sum p |v - o| / sum p (1 - E) <= 1.01 E (sum p |v| / sum p + |o|)
and E = 2^-8 + e^ds - 1, where ds bounds the score: the sum of D products in fp32, (D + 8) 2^-24
times the largest sum |q k| scale, plus 2^-20 times the largest score that a cap or a bias formed
(a few fp32 roundings and a tanh good to 2^-22).  Then the quotient's rounding, 2^-8 |o|.
"""
import torch


def attend64(q, k, v, seen, scale, softcap=0.0, bias=None, score_err=0.0):
    """q [n, D], k / v [m, D], seen [n, m] bool, bias [n, m] (taken off) -> (o [n, D], bound [n, D]),
    float64.  A row that sees nothing is 0.  Masked keys and values may be anything.  score_err: what a
    score may be off by beside the above."""
    q, k, v = q.double(), k.double(), v.double()
    used = seen.any(0)
    kz = torch.where(used[:, None], k, 0.0)  # keys that no row sees: never read
    x = scale * (q @ kz.T)
    size = scale * (q.abs() @ kz.abs().T)
    s = softcap * torch.tanh(x / softcap) if softcap else x
    extra = s.abs() if softcap else torch.zeros_like(s)
    if bias is not None:
        s = s - bias
        extra = extra + bias.abs()
    s = torch.where(seen, s, -torch.inf)
    top = s.amax(1, keepdim=True)
    p = torch.exp(s - torch.where(top.isinf(), 0.0, top))
    total = p.sum(1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    ds = torch.where(seen, (q.shape[1] + 8) * 2.0 ** -24 * size + 2.0 ** -20 * extra, 0.0).amax(1, keepdim=True) + score_err
    vz = torch.where(used[:, None], v, 0.0)
    o = p @ vz
    e = 2.0 ** -8 + torch.expm1(2 * ds)  # a weight's score against the largest one's: both off
    return o, 1.01 * e * (p @ vz.abs() + o.abs()) + 2.0 ** -8 * o.abs() + 1e-30


def check(got, want, bound, what=""):
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} past the bound, worst "
                                 f"{float((err / bound).nan_to_num(1e9).max()):.2f} of it")
