"""Oracle (test infrastructure): distillation from a teacher's top logits in 64 bits on the CPU, from the formulas, with a bound
on what fp32 arithmetic may be off.

    p = softmax over the row's entries of t / T;  ls = log_softmax(z / T);  loss = T^2 w sum_k p_k (log p_k - ls_{idx_k})
    dz_c = g w T (exp(ls_c) - sum_{k: idx_k = c} p_k);  a row without an entry: 0
"""
import torch


def distill(z, t, index, T=1.0, w=None, g=None, bits=None, centred=False):
    """z [N, C], t / index [N, K]; g [N]: gradient of every row's loss (ones).  -> dict of loss [N], lse [N], dlogits [N, C] and,
    with the working type `bits`, '<name>_off': an elementwise worst case.  centred: of arithmetic that takes every logit
    relative to its row's maximum, so that a common offset of a row's logits costs nothing (the bounds of loss and dlogits)."""
    z, t, index = z.detach().cpu().double(), t.detach().cpu().double(), index.cpu().long()
    N, C = z.shape
    K = t.shape[1]
    w = torch.ones(N, dtype=torch.float64) if w is None else w.cpu().double()
    g = torch.ones(N, dtype=torch.float64) if g is None else g.cpu().double()
    ok = (index >= 0) & (index < C)
    at = index.clamp(0, C - 1)
    t = torch.where(ok, t / T, torch.full_like(t, -float("inf")))
    empty = (t == -float("inf")).all(1)
    top = t.amax(1, keepdim=True) if K else torch.zeros(N, 1, dtype=torch.float64)
    top = torch.where(empty[:, None], torch.zeros_like(top), top)
    e = (t - top).exp()
    lp = t - top - e.sum(1, keepdim=True).log()
    p = torch.where(empty[:, None], torch.zeros_like(lp), lp.exp())
    lse = torch.logsumexp(z / T, 1)
    ls = torch.log_softmax(z / T, 1)  # (z / T - lse loses the differences of logits of 10^9 and more in 64 bits too)
    gap = torch.where(p > 0, lp - ls.gather(1, at), torch.zeros_like(p))
    loss = torch.where(empty, torch.zeros(N, dtype=torch.float64), T * T * w * (p * gap).sum(1))
    f = (g * w * T)[:, None]
    s = ls.exp()
    per_class = torch.zeros(N, C, dtype=torch.float64).scatter_add_(1, at, p)
    grad = torch.where(empty[:, None], torch.zeros_like(s), f * (s - per_class))
    r = {"loss": loss, "lse": lse, "dlogits": grad}
    if bits is None:
        return r
    u = 2.0 ** -23  # a step of fp32, rounded either way
    last = torch.finfo(bits).eps / 2 if bits != torch.float32 else u
    chain = min(C, 128 + C // 256) + 32  # longest chain of a row's sum: a thread's share, then the tree over threads
    span = torch.where(z.isfinite(), (z / T - lse[:, None]).abs(), torch.zeros_like(z)).amax(1, keepdim=True)
    e_lse = chain * u + 4 * u * (1 + span) + 2 * u * lse.abs()[:, None]
    e_ls = e_lse + 4 * u * (ls.abs().clamp(max=200) + lse.abs()[:, None] + 1)
    if centred:
        # A term of the sum is off by 4 u (1 + |ls|) of itself, and weighs s in it.  A log-sum-exp of at most 32 powers of two (22.2)
        # that was stored in 32 bits: half a step of it, of its product with log2(e), of the logit's and of the constant's, each
        # 2^-20 or (the last) 2^-19 of a power of two: 5.5 x 2^-20 x ln 2 < 32 u.
        e_c = chain * u + (s * 4 * u * (1 + ls.abs().clamp(max=200))).sum(1, keepdim=True) + 32 * u
        e_ls = e_c + 4 * u * (ls.abs().clamp(max=200) + 1)
    tspan = torch.where(p > 0, lp.abs(), torch.zeros_like(p)).amax(1, keepdim=True) if K else torch.zeros_like(top)
    e_lp = (K + 8) * u + 8 * u * (1 + tspan)
    r["lse_off"] = e_lse[:, 0]
    off = (p * ((e_lp + e_ls.gather(1, at)) + (torch.expm1(e_lp) + (K + 8) * u) * gap.abs())).sum(1)
    r["loss_off"] = T * T * w.abs() * off + 4 * u * loss.abs()
    e_p = torch.zeros(N, C, dtype=torch.float64).scatter_add_(1, at, p * (torch.expm1(e_lp) + K * u))
    r["dlogits_off"] = f.abs() * (s * torch.expm1(e_ls) + e_p + 4 * u * (s + per_class)) + last * grad.abs() + 1e-37
    return r
