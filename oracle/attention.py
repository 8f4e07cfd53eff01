"""Oracle (test infrastructure): softmax attention and its gradients in 64 bits on the CPU, written from the formulas, with a
bound on what fp32 / bf16 arithmetic may be off.

    s = scale q.k over visible keys;  p = exp(s - lse);  out = p v
    delta = dout.out;  ds = p (dout.v - delta);  dq = scale ds k;  dk = scale ds^T q;  dv = p^T dout
A row without a visible key: out 0, lse -inf, no gradient.
"""
import math

import torch


def visible(B, Lq, Lk, lengths=None, key_mask=None, causal=False, q_start=None):
    vis = torch.ones(B, Lq, Lk, dtype=torch.bool)
    j = torch.arange(Lk)
    if lengths is not None:
        vis &= (j[None] < lengths.cpu()[:, None])[:, None]
    if key_mask is not None:
        vis &= key_mask.cpu().bool()[:, None]
    if causal:
        start = torch.full((B,), Lk - Lq) if q_start is None else q_start.cpu().long()
        vis &= j[None, None] <= (start[:, None] + torch.arange(Lq))[:, :, None]
    return vis


def attention(q, k, v, dout=None, scale=None, bits=None, **hide):
    """-> dict of out, lse and, with dout, dq, dk, dv in 64 bits.  bits: the working type (torch.float32 / bfloat16) -> also
    '<name>_off', an elementwise worst case of the error of arithmetic that multiplies and sums in fp32, rounds the
    probabilities and their gradients to `bits` as operands and the results to `bits`."""
    dt = q.dtype
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    B, Lq, Hq, D = q.shape
    Lk, Hkv = k.shape[1], k.shape[2]
    G = Hq // Hkv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    vis = visible(B, Lq, Lk, **hide)[:, None]
    seen = vis.any(2)[..., None]  # [B,1,Lk,1]: keys that any row sees
    q = q.permute(0, 2, 1, 3)
    k = torch.where(seen, k.permute(0, 2, 1, 3), torch.zeros((), dtype=torch.float64)).repeat_interleave(G, 1)
    v = torch.where(seen, v.permute(0, 2, 1, 3), torch.zeros((), dtype=torch.float64)).repeat_interleave(G, 1)
    s = scale * (q @ k.transpose(2, 3))
    s = s.masked_fill(~vis, -math.inf)
    if Lk:
        m = s.amax(-1, keepdim=True)
    else:
        m = torch.full((B, Hq, Lq, 1), -math.inf, dtype=torch.float64)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = (s - m).exp()
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, torch.ones_like(total), total)
    lse = (m + total.log())[..., 0]
    out = p @ v
    r = {"out": out.permute(0, 2, 1, 3), "lse": lse}

    def group(x):  # [B,Hq,Lk,D] -> [B,Lk,Hkv,D]: sum over the query heads that share a key/value head
        return x.reshape(B, Hkv, G, Lk, D).sum(2).permute(0, 2, 1, 3)

    if dout is not None:
        do = dout.detach().cpu().double().permute(0, 2, 1, 3)
        dp = do @ v.transpose(2, 3)
        delta = (do * out).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        r.update(dq=(scale * ds @ k).permute(0, 2, 1, 3), dk=group(scale * ds.transpose(2, 3) @ q),
                 dv=group(p.transpose(2, 3) @ do))
    if bits is None:
        return r
    u = 2.0 ** -23                                                    # a sum's step: rounded either way
    half = torch.finfo(bits).eps / 2 if bits != torch.float32 else 0  # operands of the second products
    last = torch.finfo(bits).eps / 2                                  # results
    mag = scale * (q.abs() @ k.abs().transpose(2, 3)) * vis
    es = (D + 3) * u * mag                                            # error of a score
    el = es.amax(-1, keepdim=True) if Lk else torch.zeros_like(m)
    span = torch.where(vis, s.abs(), torch.zeros_like(s)).amax(-1, keepdim=True) if Lk else torch.zeros_like(m)
    el = el + (Lk + 8) * u + 2 * u * span                             # error of the log of the sum
    rho = torch.expm1(es + el + 4 * u * (1 + span))                   # relative error of a probability
    out_off = (p * (rho + half + (Lk + 2) * u)) @ v.abs()
    r["out_off"] = (out_off + last * out.abs()).permute(0, 2, 1, 3)
    empty = lse == -math.inf
    r["lse_off"] = torch.where(empty, torch.zeros_like(lse), el[..., 0] + 2 * u * torch.where(empty, torch.zeros_like(lse), lse.abs()))
    if dout is not None:
        o_off = out_off + last * out.abs()
        e_delta = (do.abs() * o_off).sum(-1, keepdim=True) + (D + 2) * u * (do.abs() * out.abs()).sum(-1, keepdim=True)
        e_dp = (D + 2) * u * (do.abs() @ v.abs().transpose(2, 3))
        ds_off = p * ((rho + half + 2 * u) * (dp - delta).abs() + (1 + rho) * (e_dp + e_delta))
        n = Lq * G + 2
        r["dq_off"] = (scale * ((ds_off + (Lk + 2) * u * ds.abs()) @ k.abs())).permute(0, 2, 1, 3) + last * r["dq"].abs()
        r["dk_off"] = group(scale * (ds_off + n * u * ds.abs()).transpose(2, 3) @ q.abs()) + last * r["dk"].abs()
        r["dv_off"] = group((p * (rho + half + n * u)).transpose(2, 3) @ do.abs()) + last * r["dv"].abs()
    return r
