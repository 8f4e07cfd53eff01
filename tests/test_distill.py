"""Distillation from a teacher's top logits (gp_nerf_amd.semantic_branch.distill_topk_*) against the formulas in 64 bits.  Bounds
are worst cases of fp32 arithmetic, elementwise (oracle.distill.distill)."""
import ctypes

import pytest
import torch

from oracle import distill as oracle

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _inputs(dtype, N, C, K, seed=0, planes=False, dev="cuda", teacher=torch.float32):
    g = torch.Generator().manual_seed(seed)
    z = (3.0 * torch.randn(N, C, generator=g)).to(TYPES[dtype])
    if planes:
        z = z.t().contiguous().t()
    idx = torch.randint(0, C, (N, K), generator=g)
    t = (2.0 + 3.0 * torch.randn(N, K, generator=g)).to(teacher)
    return z.to(dev), t.to(dev), idx.to(dev)


def _near(name, got, want):
    x, y, off = got.detach().cpu().double(), want[name], want[name + "_off"]
    assert x.shape == y.shape, name
    same = (x == y) | ((x - y).abs() <= off) | (x.isnan() & y.isnan())
    assert bool(same.all()), "%s: off by %.3g where %.3g is allowed (%d of %d)" % (
        name, float((x - y).abs().nan_to_num(1e30)[~same].max()), float(off[~same].max()), int((~same).sum()), same.numel())


def _all(z, t, idx, T=1.0, w=None):
    """Every entry point and reduction on the same data."""
    from gp_nerf_amd import semantic_branch as S
    N = z.shape[0]
    want = oracle.distill(z, t, idx, T, w, bits=z.dtype)
    loss, lse = S.distill_topk_forward(z, t, idx, T, w, "none")
    _near("loss", loss, want)
    _near("lse", lse, want)
    step_loss, step = S.distill_topk_step(z, t, idx, T, w, "none")
    assert torch.equal(step_loss.nan_to_num(7.), loss.nan_to_num(7.))
    _near("dlogits", step, want)
    ones = torch.ones(N, device=z.device)
    back = S.distill_topk_backward(ones, z, t, idx, lse, T, w, "none")
    _near("dlogits", back, want)
    assert step.stride() == back.stride() and step.dtype == back.dtype == z.dtype
    g = torch.linspace(-2, 3, N, device=z.device)
    _near("dlogits", S.distill_topk_backward(g, z, t, idx, lse, T, w, "none"), oracle.distill(z, t, idx, T, w, g, bits=z.dtype))
    for red, f in (("sum", 1.0), ("mean", 1.0 / max(N, 1))):
        total = f * float(want["loss"].sum())
        slack = f * float(want["loss_off"].sum()) + 2.0 ** -22 * abs(total) + 1e-30
        for scalar in (S.distill_topk_forward(z, t, idx, T, w, red)[0], S.distill_topk_step(z, t, idx, T, w, red)[0]):
            assert scalar.shape == () and (float(scalar) == total or abs(float(scalar) - total) <= slack)
        d = S.distill_topk_step(z, t, idx, T, w, red, grad_scale=2.5)[1]
        scaled = oracle.distill(z, t, idx, T, w, torch.full((N,), 2.5 * f), bits=z.dtype)
        _near("dlogits", d, scaled)
        up = torch.tensor(2.5, device=z.device)
        _near("dlogits", S.distill_topk_backward(up, z, t, idx, lse, T, w, red), scaled)
    return loss, step


# ---------------------------------------------------------------------------------------------------- formula, refusals
def test_oracle_gradient_is_the_derivative():
    g = torch.Generator().manual_seed(2)
    z, t = torch.randn(4, 9, generator=g, dtype=torch.float64), torch.randn(4, 3, generator=g, dtype=torch.float64)
    idx = torch.tensor([[0, 5, 8], [3, 3, 1], [-1, 2, 9], [-1, -1, 99]])
    w = torch.tensor([1.0, 0.5, 2.0, 1.0], dtype=torch.float64)
    r = oracle.distill(z, t, idx, 1.7, w)
    assert float(r["loss"][3]) == 0 and not bool(r["dlogits"][3].any())
    d = torch.randn(4, 9, generator=g, dtype=torch.float64)
    f = [float(oracle.distill(z + e * d, t, idx, 1.7, w)["loss"].sum()) for e in (1e-5, -1e-5)]
    assert abs((f[0] - f[1]) / 2e-5 - float((r["dlogits"] * d).sum())) < 1e-8
    leaf = z.clone().requires_grad_(True)  # and torch's own derivative of the definition, for the rows without gaps
    kl = torch.nn.functional.kl_div(torch.log_softmax(leaf[:2] / 1.7, 1).gather(1, idx[:2]), torch.log_softmax(t[:2] / 1.7, 1),
                                    reduction="none", log_target=True).sum(1) * 1.7 ** 2 * w[:2]
    assert torch.allclose(kl, r["loss"][:2], atol=1e-12)
    assert torch.allclose(torch.autograd.grad(kl.sum(), leaf)[0][:2], r["dlogits"][:2], atol=1e-12)


def test_refuses_what_it_cannot_take():
    from gp_nerf_amd import semantic_branch as S
    z, t, idx = _inputs("fp32", 4, 6, 2, dev="cpu")
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        S.distill_topk_forward(z, t, idx)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        S.distill_topk_step(z, t, idx)
    with pytest.raises(ValueError, match="expected"):
        S.distill_topk_forward(z[0], t, idx)


def _fake(**kw):
    from gp_nerf_amd import _lib
    a = _lib.DistillArgs(0, 0, 8, 10, 3, 2, 1.0, 1.0, 4, 16, 10, 1, 16, (3, 1), 16, (3, 1))
    a.loss_rows = a.loss = a.lse = a.dloss = a.dlogits = 16
    a.drow_stride, a.dclass_stride = 10, 1
    for n, x in kw.items():
        setattr(a, n, x)
    return a


@pytest.mark.parametrize("bad,text", [
    (dict(dtype=2), "unknown dtype"), (dict(teacher_dtype=-1), "teacher dtype"), (dict(index_bytes=2), "indices"),
    (dict(N=-1), "rows"), (dict(C=0), "classes"), (dict(K=257), "K must be"), (dict(K=-1), "K must be"),
    (dict(temperature=0.0), "temperature"), (dict(temperature=float("inf")), "temperature"), (dict(reduction=3), "reduction"),
    (dict(logits=None), "null logits"), (dict(teacher=None), "null teacher"), (dict(index=None), "null teacher"),
    (dict(class_stride=2, row_stride=20), "contiguous classes or contiguous rows"), (dict(N=1 << 31), "rows"),
])
def test_c_entry_refuses(bad, text):
    from gp_nerf_amd import _lib
    L = _lib.lib()
    for fn in (L.gpn_distill_forward, L.gpn_distill_backward, L.gpn_distill_step):
        assert fn(ctypes.byref(_fake(**bad)), None) == -1
        assert text in L.gpn_last_error().decode()


@pytest.mark.parametrize("temperature", [1e-20, 1e20, -1.0, float("nan")])
def test_c_entry_refuses_temperatures_whose_square_is_lost(temperature):
    from gp_nerf_amd import _lib
    L = _lib.lib()
    for fn in (L.gpn_distill_forward, L.gpn_distill_backward, L.gpn_distill_step):
        assert fn(ctypes.byref(_fake(temperature=temperature)), None) == -1
        assert b"temperature must be between" in L.gpn_last_error()


def test_c_entry_refuses_missing_outputs():
    from gp_nerf_amd import _lib
    L = _lib.lib()
    for fn, name in ((L.gpn_distill_forward, "loss_rows"), (L.gpn_distill_forward, "lse"), (L.gpn_distill_forward, "loss"),
                     (L.gpn_distill_backward, "lse"), (L.gpn_distill_backward, "dloss"), (L.gpn_distill_backward, "dlogits"),
                     (L.gpn_distill_step, "dlogits"), (L.gpn_distill_step, "loss_rows")):
        assert fn(ctypes.byref(_fake(**{name: None})), None) == -1
        assert ("null " + name).encode() in L.gpn_last_error()
    assert L.gpn_distill_step(ctypes.byref(_fake(dclass_stride=4, drow_stride=1)), None) == -1
    assert b"must lie as the logits do" in L.gpn_last_error()
    assert L.gpn_distill_forward(None, None) == -1
    assert L.gpn_distill_backward(ctypes.byref(_fake(N=0, logits=None)), None) == 0


def test_distill_struct_layout_matches_header(tmp_path):
    import os
    import subprocess
    from gp_nerf_amd import _lib
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = [n for n, _ in _lib.DistillArgs._fields_]
    src = "#include <stdio.h>\n#include <stddef.h>\n#include \"gpnerf_hip.h\"\nint main(){printf(\"%zu\", sizeof(gpn_distill_args_t));"
    src += "".join('printf(" %%zu", offsetof(gpn_distill_args_t, %s));' % n for n in names) + "return 0;}"
    (tmp_path / "p.c").write_text(src)
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(tmp_path / "p.c"), "-o", str(tmp_path / "p")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "p")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(_lib.DistillArgs)] + [getattr(_lib.DistillArgs, n).offset for n in names]


# ------------------------------------------------------------------------------------------------------------ numerics
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("N,C,K", [(1, 1, 1), (3, 2, 2), (5, 21, 5), (2, 255, 7), (3, 1000, 64), (2, 4097, 3), (3, 9001, 65),
                                   (2, 20011, 16), (1, 50001, 256), (2, 70001, 9), (1, 131075, 4), (2, 140000, 1)])
def test_rows(dtype, N, C, K):
    """From one class to rows that are walked in several segments; odd counts leave every row differently aligned."""
    _all(*_inputs(dtype, N, C, K), T=1.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("N,C,K", [(2, 1, 1), (7, 2, 1), (300, 21, 5), (257, 32, 8), (1025, 33, 3), (90, 150, 40), (1, 40, 2)])
def test_planes(dtype, N, C, K):
    _all(*_inputs(dtype, N, C, K, planes=True), T=0.7)


@pytest.mark.gpu
@pytest.mark.parametrize("planes", [False, True])
def test_missing_repeated_and_weighted_entries(planes):
    z, t, idx = _inputs("fp32", 40, 30, 6, planes=planes, teacher=torch.bfloat16)
    idx[0] = -1                       # no entry at all
    idx[1, 1:] = 30                   # one entry, the others past the classes
    idx[2] = 4                        # one class, six times
    idx[3, 2] = 2 ** 40               # far outside
    t[4] = -float("inf")              # entries without weight
    t[5, 1] = -float("inf")
    z[0] = float("nan")               # a row that counts for nothing may hold anything
    z[4, 3] = float("inf")
    z[6, idx[6, 0]] = -float("inf")   # the student rules out a class of the teacher's: an infinite loss, a finite gradient
    z[7] = torch.finfo(torch.float32).min
    w = torch.linspace(0, 2, 40).cuda()
    loss, d = _all(z, t, idx, 2.0, w)[0:2]
    assert float(loss[0]) == 0 and float(loss[4]) == 0 and not bool(d[0].any()) and not bool(d[4].any())
    assert float(loss[6]) == float("inf") and bool(d[6].isfinite().all())
    i32 = _all(z, t, idx.clamp(-1, 30).to(torch.int32), 2.0, w)[1]
    assert torch.equal(i32.nan_to_num(5.), d.nan_to_num(5.))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_nan_and_extreme_logits(dtype):
    z, t, idx = _inputs(dtype, 6, 700, 4)
    z[0, 13] = float("nan")
    z[1] *= 1000.0
    z[2] = -float("inf")
    z[2, 5] = 1.0
    z[3, 1] = torch.finfo(TYPES[dtype]).min
    z[4] = 3e4
    from gp_nerf_amd import semantic_branch as S
    loss, d = S.distill_topk_step(z, t, idx, reduction="none")
    assert bool(loss[0].isnan()) and bool(d[0].isnan().all())
    assert bool(d[1:].isfinite().all()) and bool(loss[3:].isfinite().all())
    keep = torch.tensor([1, 3, 4, 5])
    want = oracle.distill(z[keep], t[keep], idx[keep], bits=z.dtype)
    _near("loss", loss[keep], want)
    _near("dlogits", d[keep], want)


@pytest.mark.gpu
def test_layouts():
    from gp_nerf_amd import semantic_branch as S
    z, t, idx = _inputs("bf16", 24, 50, 4)
    want_loss, want = S.distill_topk_step(z, t, idx)

    def same(zz, tt=t, ii=idx):
        loss, d = S.distill_topk_step(zz, tt, ii)
        assert torch.equal(loss, want_loss) and torch.equal(d.reshape(want.shape) if d.dim() == 2 else d, want)

    wide = torch.full((24, 61), float("nan"), dtype=z.dtype).cuda()
    wide[:, 7:57] = z
    same(wide[:, 7:57])                                            # a slice of longer rows, not aligned
    both = torch.zeros(24, 50, 2, dtype=z.dtype).cuda()
    both[..., 1] = z
    same(both[..., 1])                                             # neither stride is one: copied
    same(z, t.t().contiguous().t(), idx.t().contiguous().t())      # the teacher's planes
    # images: the head's logits with the teacher's top planes
    img, tt, ii = z.t().reshape(1, 50, 4, 6).contiguous(), t.t().reshape(1, 4, 4, 6), idx.t().reshape(1, 4, 4, 6)
    ref_loss, ref = S.distill_topk_step(z.t().contiguous().t(), t, idx)
    for x in (img, img[0], img.contiguous(memory_format=torch.channels_last)):
        loss, d = S.distill_topk_step(x, tt, ii)
        assert d.shape == x.shape
        off = oracle.distill(z, t, idx, g=torch.full((24,), 1 / 24), bits=z.dtype)
        _near("dlogits", d.reshape(50, 24).t(), off)
        assert abs(float(loss - ref_loss)) <= 1e-5 * float(ref_loss)
    # rows of one call leave what lies around them alone
    assert bool(wide[:, :7].isnan().all()) and bool(wide[:, 57:].isnan().all())


@pytest.mark.gpu
def test_nothing_to_do():
    from gp_nerf_amd import semantic_branch as S
    z, t, idx = _inputs("fp32", 0, 9, 3)
    for red in ("mean", "sum"):
        loss, d = S.distill_topk_step(z, t, idx, reduction=red)
        assert float(loss) == 0 and d.shape == (0, 9)
    z, t, idx = _inputs("fp32", 5, 9, 0)
    loss, d = S.distill_topk_step(z, t, idx, reduction="none")
    assert not bool(loss.any()) and not bool(d.any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_autograd(dtype):
    from gp_nerf_amd import semantic_branch as S
    z, t, idx = _inputs(dtype, 12, 300, 8)
    w = torch.rand(12, generator=torch.Generator().manual_seed(0)).cuda()
    for red in ("mean", "sum", "none"):
        leaf = z.clone().requires_grad_(True)
        loss = S.distill_topk_loss(leaf, t, idx, 2.0, w, red)
        up = torch.linspace(1, 2, 12).cuda() if red == "none" else torch.tensor(0.5).cuda()
        loss.backward(up)
        f, lse = S.distill_topk_forward(z, t, idx, 2.0, w, red)
        assert torch.equal(loss, f)
        assert torch.equal(leaf.grad, S.distill_topk_backward(up, z, t, idx, lse, 2.0, w, red))
    # a gradient against differences of the kernel's own loss
    z = z.float()
    d = torch.randn(z.shape, generator=torch.Generator().manual_seed(1)).cuda()
    d /= d.norm()
    e = 2.0 ** -5
    f = [float(S.distill_topk_forward(z + s * e * d, t, idx, 1.0, None, "sum")[0]) for s in (1, -1)]
    slope = float((S.distill_topk_step(z, t, idx, 1.0, None, "sum")[1].double() * d.double()).sum())
    # third derivative along a unit direction at most 1 per row: e^2 / 6 * 12 = 2e-3; rounding of the sum: 2^-23 * 100 / (2 e)
    assert abs((f[0] - f[1]) / (2 * e) - slope) < 3e-3


@pytest.mark.gpu
def test_refuses_on_device():
    from gp_nerf_amd import semantic_branch as S
    z, t, idx = _inputs("fp32", 4, 6, 2)
    bad = [
        (lambda: S.distill_topk_step(z.half(), t, idx), "float32 or bfloat16"),
        (lambda: S.distill_topk_step(z, t[:3], idx), "for each of the 4 rows"),
        (lambda: S.distill_topk_step(z, t, idx[:, :1]), "for each of the 4 rows"),
        (lambda: S.distill_topk_step(z, t, idx.float()), "int32 or int64"),
        (lambda: S.distill_topk_step(z, t, idx.cpu()), "teacher_index"),
        (lambda: S.distill_topk_step(z, t, idx, row_weight=torch.ones(3).cuda()), "row_weight"),
        (lambda: S.distill_topk_step(z, t, idx, row_weight=torch.ones(4)), "no CPU fallback"),
        (lambda: S.distill_topk_step(z, t, idx, reduction="max"), "reduction"),
        (lambda: S.distill_topk_step(z[None, None], t, idx), "logits: expected|for each"),
        (lambda: S.distill_topk_backward(torch.ones(4).cuda(), z, t, idx, torch.ones(4).cuda()), "dloss"),
        (lambda: S.distill_topk_backward(torch.tensor(1.).cuda(), z, t, idx, torch.ones(3).cuda()), "lse"),
        (lambda: S.distill_topk_step(z, t.repeat(1, 200), idx.repeat(1, 200)), "at most 256"),
    ]
    for f, text in bad:
        with pytest.raises((ValueError, RuntimeError), match=text):
            f()
    with pytest.raises(RuntimeError, match="temperature"):
        S.distill_topk_step(z, t, idx, temperature=-1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("planes", [False, True])
def test_captured_step(planes):
    from gp_nerf_amd import semantic_branch as S
    z, t, idx = _inputs("bf16", 33, 700, 5, planes=planes)
    S.distill_topk_step(z, t, idx)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        loss, d = S.distill_topk_step(z, t, idx)
    for seed in (1, 2, 3):
        new = _inputs("bf16", 33, 700, 5, seed=seed, planes=planes)
        for a, b in zip((z, t, idx), new):
            a.copy_(b)
        g.replay()
        want = S.distill_topk_step(*new)
        torch.cuda.synchronize()
        assert torch.equal(loss, want[0]) and torch.equal(d, want[1])
    leaf = z.clone().requires_grad_(True)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="cannot be captured"):
            S.distill_topk_loss(leaf, t, idx)
        z.mul_(1.0)


@pytest.mark.gpu
def test_ray_attention_under_a_distilled_head():
    """The operators as a training step uses them: ray attention of a block, mean over the samples, class logits, a teacher's top
    classes.  Loss and every gradient against 64-bit autograd of the definitions."""
    from gp_nerf_amd import semantic_branch as S
    from gp_nerf_amd.attention import attention
    g = torch.Generator().manual_seed(11)
    R, L, H, D, C, K = 50, 48, 4, 16, 21, 5
    x = torch.randn(R, L, H * D, generator=g)
    wts = [0.2 * torch.randn(64, 64, generator=g) for _ in range(3)] + [0.3 * torch.randn(C, 64, generator=g)]
    keep = torch.rand(R, L, generator=g) < 0.8
    keep[3] = False
    t, idx = (2 * torch.randn(R, C, generator=g)).topk(K, dim=1)

    def step(x, wts, attend, loss_of):
        q, k, v = (torch.nn.functional.linear(x, w).view(R, L, H, D) for w in wts[:3])
        y = (x + attend(q, k, v).reshape(R, L, H * D)).mean(1)
        return loss_of(torch.nn.functional.linear(y, wts[3]))

    def plain(q, k, v):
        q, k, v = (z.permute(0, 2, 1, 3) for z in (q, k, v))
        s = (q @ k.transpose(2, 3) / D ** 0.5).masked_fill(~keep[:, None, None], -1e300)
        return (torch.softmax(s, -1) @ v).permute(0, 2, 1, 3) * keep.any(1)[:, None, None, None]

    def plain_loss(z):
        p = torch.softmax(t.double() / 2, 1)
        return (p * (p.log() - torch.log_softmax(z / 2, 1).gather(1, idx))).sum() * 4 / R

    ref = [z.double().requires_grad_(True) for z in (x, *wts)]
    want = step(ref[0], ref[1:], plain, plain_loss)
    want.backward()
    own = [z.cuda().requires_grad_(True) for z in (x, *wts)]
    got = step(own[0], own[1:], lambda q, k, v: attention(q, k, v, key_mask=keep.cuda()),
               lambda z: S.distill_topk_loss(z, t.cuda(), idx.cuda(), 2.0))
    got.backward()
    # chains of at most 64 + 16 + 48 + 48 + 64 + 21 sums before the loss and the like behind it, 2400 rows for a weight: fewer
    # than 3200 half steps of 2^-24, on values whose magnitudes sum to at most 4 times the largest result
    tol = 4 * 3200 * 2.0 ** -24
    assert abs(float(got.detach()) - float(want.detach())) <= tol * abs(float(want.detach()))
    for a, b in zip(own, ref):
        assert float((a.grad.cpu().double() - b.grad).abs().max()) <= tol * float(b.grad.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("planes,C,K", [(False, 30, 6), (False, 1500, 6), (False, 140000, 6), (True, 30, 6), (True, 50, 6), (True, 40, 12)])
def test_rows_of_weight_zero_may_hold_anything(dtype, planes, C, K):
    """They count as rows without an entry: the others' results do not change by a bit."""
    from gp_nerf_amd import semantic_branch as S
    z, t, idx = _inputs(dtype, 10, C, K, planes=planes)
    w = torch.linspace(0.5, 2, 10).cuda()
    out = [1, 2, 4, 5, 9]
    w[out] = torch.tensor([0.0, -0.0, 0.0, 0.0, 0.0]).cuda()
    clean = z.clone(), t.clone()
    z[1] = float("nan")
    z[2, 3] = float("inf")
    z[4, idx[4, 1]] = -float("inf")   # a class of the teacher's that the student rules out
    t[5, 2] = float("nan")
    t[9] = float("inf")
    for red in ("none", "sum", "mean"):
        up = torch.full((10,) if red == "none" else (), 1.5, device="cuda")
        got, want = [], []
        for zz, tt, to in ((z, t, got), (*clean, want)):
            loss, lse = S.distill_topk_forward(zz, tt, idx, 0.9, w, red)
            to += [loss, S.distill_topk_backward(up, zz, tt, idx, lse, 0.9, w, red), *S.distill_topk_step(zz, tt, idx, 0.9, w, red)]
        for a, b in zip(got, want):
            assert bool(a.isfinite().all()) and torch.equal(a, b), red
        assert not bool(got[1][out].any()) and not bool(got[3][out].any())
        assert red != "none" or not bool(got[0][out].any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("planes", [False, True])
def test_log_sum_exp_of_the_largest_logits(dtype, planes):
    """Logits at the ends of their type have a log-sum-exp that fp32 holds."""
    from gp_nerf_amd import semantic_branch as S
    z, t, idx = _inputs(dtype, 6, 40, 4, planes=planes)
    top = torch.finfo(TYPES[dtype]).max
    z[0], z[1], z[2, 3], z[3] = -top, top, top, -0.75 * top
    for T in (1.0, 3.0):
        lse = S.distill_topk_forward(z, t, idx, T)[1]
        assert bool(lse.isfinite().all())
        _near("lse", lse, oracle.distill(z, t, idx, T, bits=z.dtype))


@pytest.mark.parametrize("offset", [-1e9, 1e16, -3e38, "cold"])
def test_oracle_does_not_depend_on_a_common_offset(offset):
    """Differences of a row's logits that 64 bits hold come back from it whatever they are added to; its bounds stay finite."""
    z, t, idx = _inputs("fp32", 5, 60, 4, dev="cpu")
    z, T = z.double().round() * 4, 1.0
    if offset == "cold":
        z, far, T = z * 1e4, z * 1e4, 1e-3
    else:
        far = z + offset if abs(offset) < 1e17 else torch.full_like(z, offset)
        z = z if abs(offset) < 1e17 else torch.zeros_like(z)
    want = torch.softmax(z / T, 1) * T - torch.zeros_like(z).scatter_add_(1, idx, torch.softmax(t.double() / T, 1)) * T
    got = oracle.distill(far, t, idx, T, bits=torch.float32, centred=True)
    assert float((got["dlogits"] - want).abs().max()) < 1e-14
    assert bool(got["dlogits_off"].isfinite().all()) and float(got["dlogits_off"].max()) < 1e-3


def _far(kind, dtype, z):
    """Logits whose common offset, or whose temperature, makes 32 bits of their log-sum-exp too few. -> logits, temperature"""
    top = torch.finfo(TYPES[dtype]).max
    if kind == "cold":
        return z * 10.0, 1e-3
    if kind == "lowest":
        return torch.full_like(z, -top), 1.0
    return (z.float() + kind).to(z.dtype), 1.0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("kind", [30.0, -1e5, 1e7, -1e9, "cold", "lowest"], ids=str)
@pytest.mark.parametrize("planes,N,C,K", [(False, 9, 60, 5), (False, 5, 1000, 5), (False, 3, 9001, 5), (False, 2, 140000, 5),
                                          (True, 60, 21, 5), (True, 61, 21, 12), (True, 60, 70, 5), (True, 31, 70, 12)])
def test_offsets_that_cancel_in_the_softmax(dtype, kind, planes, N, C, K):
    """Forward and backward apart against the formula (as exact as the step, whose logits are taken relative to the maximum)."""
    from gp_nerf_amd import semantic_branch as S
    z, t, idx = _inputs(dtype, N, C, K, planes=planes)
    far, T = _far(kind, dtype, z)
    z = torch.where(torch.arange(N, device="cuda")[:, None] % 3 == 1, z, far)   # ordinary rows beside them
    if planes:
        z = z.t().contiguous().t()
    want = oracle.distill(z, t, idx, T, bits=z.dtype, centred=True)
    assert bool(want["dlogits_off"].isfinite().all())
    loss, lse = S.distill_topk_forward(z, t, idx, T, None, "none")
    _near("lse", lse, want)
    _near("dlogits", S.distill_topk_backward(torch.ones(N, device="cuda"), z, t, idx, lse, T, None, "none"), want)
    _near("dlogits", S.distill_topk_step(z, t, idx, T, None, "none")[1], want)


@pytest.mark.parametrize("recording", [True, False])
def test_capture_is_refused_for_recorded_graphs_only(monkeypatch, recording):
    """Nothing is recorded under no_grad, whatever the logits require: the refusal there is the one of CPU tensors."""
    from gp_nerf_amd import semantic_branch as S
    z, t, idx = _inputs("fp32", 4, 6, 2, dev="cpu")
    z.requires_grad_(True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with torch.set_grad_enabled(recording), pytest.raises(RuntimeError, match="cannot be captured" if recording else "no CPU fallback"):
        S.distill_topk_loss(z, t, idx)


@pytest.mark.gpu
def test_captured_loss_without_a_graph():
    from gp_nerf_amd import semantic_branch as S
    z, t, idx = _inputs("fp32", 33, 700, 5)
    leaf = z.clone().requires_grad_(True)
    S.distill_topk_forward(z, t, idx)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g), torch.no_grad():
        loss = S.distill_topk_loss(leaf, t, idx)
    for seed in (1, 2, 3):
        new = _inputs("fp32", 33, 700, 5, seed=seed)[0]
        with torch.no_grad():
            leaf.copy_(new)
        g.replay()
        want = S.distill_topk_forward(new, t, idx)[0]
        torch.cuda.synchronize()
        assert torch.equal(loss, want)
