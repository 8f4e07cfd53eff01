"""The attention and distillation operators as a program uses them: inputs, one pass, its work, and their definition in 64 bits.

With `own` false, `run` computes every operator in elementary torch operations in 32 bits; with `own` true it makes the calls of
gp_nerf_amd's operators.  Three kinds of case:

  forward   softmax attention: out and the log-sum-exp of every row (one query against a cache, prompts, the rays of a chunk)
  step      attention forward and backward: out and the gradients of q, k and v
  distill   loss on a teacher's top logits and the gradient of the student's logits
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------ cases
def _attn(name, kind, dtype, B, Lq, Lk, Hq, Hkv, D, causal=False, lengths=False, mask=False):
    c = {"kind": kind, "dtype": dtype, "B": B, "Lq": Lq, "Lk": Lk, "Hq": Hq, "Hkv": Hkv, "D": D, "causal": causal,
         "lengths": lengths, "mask": mask}
    if name:
        c["name"] = name
    return c


def _dist(name, dtype, N, C, K, planes, temperature):
    c = {"kind": "distill", "dtype": dtype, "N": N, "C": C, "K": K, "planes": planes, "T": temperature}
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one new token against a short cache: nothing but latency
        _attn("forward one token", "forward", "bf16", 1, 1, 257, 8, 8, 64),
        # one new token for each of eight sequences of different lengths, shared heads: the cache is read once
        _attn("forward tokens, long cache", "forward", "bf16", 8, 1, 16384, 32, 8, 128, lengths=True),
        # the ray attention of one 4096-ray render chunk (64 samples, 4 heads of 16)
        _attn("forward rays", "forward", "fp32", 4096, 64, 64, 4, 4, 16),
        # a long prompt
        _attn("forward causal, long", "forward", "bf16", 1, 8192, 8192, 32, 8, 128, causal=True),
        # cross attention with masked keys, sizes that fit no tile
        _attn("forward masked, odd", "forward", "fp32", 3, 333, 1021, 6, 3, 80, mask=True),
        # training of a ray block: 1024 rays, samples that no view sees are masked
        _attn("step rays", "step", "fp32", 1024, 64, 64, 4, 4, 16, mask=True),
        # the same at the stress shape: 128 samples, bf16
        _attn("step rays, 128 samples", "step", "bf16", 4096, 128, 128, 4, 4, 16),
        # training on long sequences with shared heads
        _attn("step causal, long", "step", "bf16", 2, 4096, 4096, 16, 4, 128, causal=True),
        # a padded batch of odd lengths (an empty sequence among them)
        _attn("step padded, odd", "step", "bf16", 5, 777, 777, 8, 2, 64, lengths=True),
        # class logits of the semantic head (planes of a 240 x 320 image, 20 classes and the background)
        _dist("distill head", "fp32", 76800, 21, 5, True, 1.0),
        # rows of an odd number of classes: no row but the first is aligned
        _dist("distill rows, odd", "fp32", 257, 10007, 16, False, 1.5),
        # a batch of tokens over a large vocabulary
        _dist("distill vocabulary", "bf16", 4096, 48000, 64, False, 2.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["forward", "cache", "rays", "step", "step rays", "step", "distill rows", "distill planes"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if kind == "distill rows":
        N, C = _log_int(rng, 1, 8192), _log_int(rng, 2, 131072)
        N = max(1, min(N, (190_000_000 if dtype == "bf16" else 95_000_000) // C))
        return _dist(None, dtype, N, C, min(C, _log_int(rng, 1, 64)), False, rng.choice([1.0, 2.0, 4.0]))
    if kind == "distill planes":
        C = rng.randint(2, 150)
        return _dist(None, dtype, _log_int(rng, 300, 320000), C, min(C, rng.randint(1, 8)), True, rng.choice([1.0, 2.0]))
    if kind in ("rays", "step rays"):
        B, L, H = _log_int(rng, 64, 4096), rng.randint(8, 128), rng.choice([1, 2, 4])
        B = min(B, (1 << 19 if dtype == "bf16" else 1 << 18) // L)
        return _attn(None, "forward" if kind == "rays" else "step", dtype, B, L, L, H, H, 16, rng.random() < 0.3, False,
                     rng.random() < 0.5)
    Hkv, G, D = rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 2, 3, 4, 8]), rng.choice([16, 24, 32, 40, 64, 80, 96, 128])
    if kind == "cache":
        B, Lk, Lq = _log_int(rng, 1, 32), _log_int(rng, 1, 32768), rng.choice([1, 1, 1, 2, 4, 7])
        Lk = max(Lq, min(Lk, (130_000_000 if dtype == "bf16" else 65_000_000) // (B * Hkv * D)))
        return _attn(None, "forward", dtype, B, Lq, Lk, Hkv * G, Hkv, D, rng.random() < 0.5, rng.random() < 0.7, rng.random() < 0.2)
    B, Lk = _log_int(rng, 1, 16), _log_int(rng, 16, 8192)
    most = (4.5e11 if dtype == "bf16" else 4.5e10) / ((14 if kind == "step" else 4) * D * Hkv * G)  # pairs of one head
    B = max(1, min(B, int(most / Lk ** 2)))
    Lk = min(Lk, int(math.sqrt(most / B)))
    Lq = Lk if rng.random() < 0.7 else rng.randint(1, Lk)
    return _attn(None, kind, dtype, B, Lq, Lk, Hkv * G, Hkv, D, rng.random() < 0.5, rng.random() < 0.4, rng.random() < 0.3)


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(B, Lk):
    """Sequence lengths of a padded batch: spread from empty (or one, for a batch of up to four) to full."""
    first = 0 if B > 4 else 1
    return [Lk] if B == 1 else [first + (Lk - first) * b // (B - 1) for b in range(B)]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    if case["kind"] == "distill":
        N, C, K = case["N"], case["C"], case["K"]
        logits = 2.0 * normal(C, N) if case["planes"] else 2.0 * normal(N, C)
        logits = logits.to(dt)
        if case["planes"]:
            logits = logits.t()  # [N, C] view of class planes, as the head's [1, C, H, W] output gives it
        index = torch.randint(0, C, (N, K), generator=g, device=DEV)  # the same class twice now and then
        teacher = (4.0 + 2.0 * normal(N, K)).to(dt)
        return {"case": case, "logits": logits, "teacher": teacher, "index": index}
    B, Lq, Lk, Hq, Hkv, D = (case[n] for n in ("B", "Lq", "Lk", "Hq", "Hkv", "D"))
    s = {"case": case, "q": normal(B, Lq, Hq, D).to(dt), "k": normal(B, Lk, Hkv, D).to(dt),
         "v": normal(B, Lk, Hkv, D).to(dt), "lengths": None, "mask": None}
    if case["kind"] == "step":
        s["dout"] = normal(B, Lq, Hq, D).to(dt)
    if case["lengths"]:
        s["lengths"] = torch.tensor(_lengths(B, Lk), dtype=torch.int32, device=DEV)
    if case["mask"]:
        s["mask"] = torch.rand((B, Lk), generator=g, device=DEV) < 0.7
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    if case["kind"] == "distill":
        return _distill_plain(state["logits"], state["teacher"], state["index"], case["T"])
    return _attention_plain(state, case)


def _run_own(state, case):
    if case["kind"] == "distill":
        from gp_nerf_amd.semantic_branch import distill_topk_step
        loss, dlogits = distill_topk_step(state["logits"], state["teacher"], state["index"], temperature=case["T"])
        return {"loss": loss, "dlogits": dlogits}
    from gp_nerf_amd.attention import attention_backward, attention_forward
    q, k, v = state["q"], state["k"], state["v"]
    hidden = {"lengths": state["lengths"], "key_mask": state["mask"], "causal": case["causal"]}
    out, lse = attention_forward(q, k, v, **hidden)
    if case["kind"] == "forward":
        return {"out": out, "lse": lse}
    dq, dk, dv = attention_backward(state["dout"], q, k, v, out, lse, **hidden)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _visible(state, case):
    """[B or 1, 1, 1, Lq or 1, Lk] truth values, or None where every query sees every key."""
    Lq, Lk = case["Lq"], case["Lk"]
    j = torch.arange(Lk, device=DEV)
    vis = None
    if case["causal"]:
        vis = (j <= torch.arange(Lq, device=DEV)[:, None] + (Lk - Lq))[None, None, None]
    for keys in ((j < state["lengths"][:, None]) if state["lengths"] is not None else None, state["mask"]):
        if keys is not None:
            keys = keys[:, None, None, None, :]
            vis = keys if vis is None else vis & keys
    return vis


def _attention_plain(state, case):
    B, Lq, Lk, Hq, Hkv, D = (case[n] for n in ("B", "Lq", "Lk", "Hq", "Hkv", "D"))
    G, dt, scale = Hq // Hkv, state["q"].dtype, 1.0 / math.sqrt(D)
    q = state["q"].float().view(B, Lq, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * Lq, D)
    k = state["k"].float().permute(0, 2, 1, 3).contiguous()
    v = state["v"].float().permute(0, 2, 1, 3).contiguous()
    p = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(scale).view(B, Hkv, G, Lq, Lk)
    vis = _visible(state, case)
    if vis is not None:
        p.masked_fill_(~vis, -math.inf)
    m = p.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)  # a row that sees nothing
    p = p.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (m + total.log()).view(B, Hq, Lq)
    p = p.div_(torch.where(total == 0, torch.ones_like(total), total)).view(B, Hkv, G * Lq, Lk)
    o = torch.matmul(p, v)

    def rows(x):  # [B, Hkv, G * Lq, D] -> [B, Lq, Hq, D]
        return x.view(B, Hkv, G, Lq, D).permute(0, 3, 1, 2, 4).reshape(B, Lq, Hq, D).to(dt)

    out = rows(o)
    if case["kind"] == "forward":
        return {"out": out, "lse": lse}
    do = state["dout"].float().view(B, Lq, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * Lq, D)
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    ds = torch.matmul(do, v.transpose(2, 3).contiguous()).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q)
    return {"out": out, "dq": rows(dq), "dk": dk.permute(0, 2, 1, 3).to(dt).contiguous(),
            "dv": dv.permute(0, 2, 1, 3).to(dt).contiguous()}


def _distill_plain(logits, teacher, index, T):
    N, C = logits.shape
    z = logits.float() / T
    z = z - z.amax(1, keepdim=True)
    e = z.exp()
    total = e.sum(1, keepdim=True)
    log_s = z - total.log()
    t = teacher.float() / T
    t = t - t.amax(1, keepdim=True)
    log_p = t - t.exp().sum(1, keepdim=True).log()
    p = log_p.exp()
    loss = (p * (log_p - log_s.gather(1, index))).sum() * (T * T / N)
    grad = (e / total).scatter_add_(1, index, -p) * (T / N)
    if logits.stride(0) == 1 and C > 1:
        grad = grad.t().to(logits.dtype).contiguous().t()
    return {"loss": loss, "dlogits": grad.to(logits.dtype)}


# ------------------------------------------------------------------------------------------------ work
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "distill":
        N, C, K = case["N"], case["C"], case["K"]
        return {"bytes": 2 * N * C * size + N * K * (size + 8) + 4, "flops": 6 * N * C}
    B, Lq, Lk, Hq, Hkv, D = (case[n] for n in ("B", "Lq", "Lk", "Hq", "Hkv", "D"))
    lens = _lengths(B, Lk) if case["lengths"] else [Lk] * B
    pairs = sum(_pairs(Lq, Lk, n, case["causal"]) for n in lens) * Hq
    keys, rows = sum(lens) * Hkv * D, B * Lq * Hq * D
    if case["mask"]:  # seven keys of ten are looked at
        pairs, keys = 0.7 * pairs, 0.7 * keys
    if case["kind"] == "forward":
        return {"bytes": (2 * rows + 2 * keys) * size + 4 * B * Hq * Lq, "flops": 4 * D * pairs}
    full = B * Lk * Hkv * D  # gradients are written for hidden keys too
    return {"bytes": (4 * rows + 2 * keys + 2 * full) * size, "flops": 14 * D * pairs}


def _pairs(Lq, Lk, n, causal):
    """Visible (query, key) pairs of one head: query i sees the first min(n, Lk - Lq + i + 1) keys."""
    if not causal:
        return Lq * n
    a = Lk - Lq + 1
    below = max(0, min(Lq, n - a + 1))  # queries whose causal bound is at most n
    return below * a + below * (below - 1) // 2 + (Lq - below) * n


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "distill":
        T, N, C = case["T"], case["N"], case["C"]
        losses = torch.zeros((), dtype=torch.float64, device=DEV)
        like = s["logits"]
        grad = torch.empty_strided(like.shape, like.stride(), dtype=torch.float64, device=DEV)
        for a in range(0, N, 8192):
            z = like[a:a + 8192].double().requires_grad_(True)
            p = torch.softmax(s["teacher"][a:a + 8192].double() / T, dim=1)
            student = torch.log_softmax(z / T, dim=1).gather(1, s["index"][a:a + 8192])
            loss = (p * (p.log() - student)).sum() * (T * T) / N
            grad[a:a + 8192] = torch.autograd.grad(loss, z)[0]
            losses += loss.detach()
        return {"loss": losses, "dlogits": grad}
    B, Lq, Lk, Hq, Hkv, D = (case[n] for n in ("B", "Lq", "Lk", "Hq", "Hkv", "D"))
    hide = torch.zeros((B, Lq, Lk), dtype=torch.bool, device=DEV)
    at = torch.arange(Lk, device=DEV)
    if s["lengths"] is not None:
        hide |= (at >= s["lengths"][:, None])[:, None]
    if s["mask"] is not None:
        hide |= ~s["mask"][:, None]
    if case["causal"]:
        hide |= at[None] > torch.arange(Lk - Lq, Lk, device=DEV)[:, None]
    empty = hide.all(-1, keepdim=True)
    hide &= ~empty
    step = case["kind"] == "step"
    k = s["k"].double().requires_grad_(step)
    v = s["v"].double().requires_grad_(step)
    outs, lses, dqs, dk, dv = [], [], [], torch.zeros_like(k), torch.zeros_like(v)
    for h in range(Hq):
        g = h // (Hq // Hkv)
        q = s["q"][:, :, h].double().requires_grad_(step)
        score = torch.matmul(q, k[:, :, g].transpose(1, 2).contiguous()) / D ** 0.5
        score = score.masked_fill(hide, -math.inf)
        o = torch.matmul(torch.softmax(score, dim=-1), v[:, :, g].contiguous()).masked_fill(empty, 0.0)
        lses.append(torch.logsumexp(score.detach(), dim=-1).masked_fill(empty[..., 0], -math.inf))
        if step:
            dq, dkh, dvh = torch.autograd.grad(o, (q, k, v), s["dout"][:, :, h].double())
            dqs.append(dq)
            dk += dkh
            dv += dvh
        outs.append(o.detach())
        del score, o
    out = torch.stack(outs, 2)
    if not step:
        return {"out": out, "lse": torch.stack(lses, 1)}
    return {"out": out, "dq": torch.stack(dqs, 2), "dk": dk, "dv": dv}
