"""Softmax attention and its gradients (gp_nerf_amd.attention) against the formulas in 64 bits.  Bounds are worst cases of the
kernels' arithmetic, elementwise (oracle.attention.attention): no tolerance is fitted."""
import ctypes

import pytest
import torch

from oracle import attention as oracle

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _inputs(dtype, B, Lq, Lk, Hq, Hkv, D, seed=0, dev="cuda"):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(s, generator=g).to(TYPES[dtype]).to(dev)  # noqa: E731
    return mk(B, Lq, Hq, D), mk(B, Lk, Hkv, D), mk(B, Lk, Hkv, D), mk(B, Lq, Hq, D)


def _check(got, want, names):
    for n in names:
        x, y, off = got[n].detach().cpu().double(), want[n], want[n + "_off"]
        assert x.shape == y.shape, n
        same = (x == y) | ((x - y).abs() <= off + 1e-30)
        assert bool(same.all()), "%s: off by up to %.3g where %.3g is allowed (%d of %d values)" % (
            n, float((x - y).abs().nan_to_num(1e30)[~same].max()), float(off[~same].max()), int((~same).sum()), same.numel())


def _both(q, k, v, do, **kw):
    from gp_nerf_amd.attention import attention_backward, attention_forward
    out, lse = attention_forward(q, k, v, **kw)
    dq, dk, dv = attention_backward(do, q, k, v, out, lse, **kw)
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def _run(q, k, v, do, **kw):
    got = _both(q, k, v, do, **kw)
    torch.cuda.synchronize()
    _check(got, oracle.attention(q, k, v, do, bits=q.dtype, **kw), ("out", "lse", "dq", "dk", "dv"))
    return got


# ------------------------------------------------------------------------------------------------- the formula itself
def test_oracle_gradients_are_the_derivatives():
    g = torch.Generator().manual_seed(1)
    q, k, v, do = (torch.randn(2, 5, 4, 8, generator=g, dtype=torch.float64),
                   torch.randn(2, 7, 2, 8, generator=g, dtype=torch.float64),
                   torch.randn(2, 7, 2, 8, generator=g, dtype=torch.float64),
                   torch.randn(2, 5, 4, 8, generator=g, dtype=torch.float64))
    kw = dict(lengths=torch.tensor([7, 4]), causal=True, q_start=torch.tensor([1, -2]))
    r = oracle.attention(q, k, v, do, **kw)
    for name, x in (("dq", q), ("dk", k), ("dv", v)):
        d = torch.randn(x.shape, generator=g, dtype=torch.float64)
        f = []
        for e in (1e-5, -1e-5):
            y = [t + e * d if t is x else t for t in (q, k, v)]
            f.append(float((oracle.attention(*y, **kw)["out"] * do).sum()))
        # central difference: error of order e^2 and 1e-16 / e
        assert abs((f[0] - f[1]) / 2e-5 - float((r[name] * d).sum())) < 1e-8


# ------------------------------------------------------------------------------------------------------ refusals (CPU)
def test_refuses_what_it_cannot_take():
    from gp_nerf_amd import attention as A
    q, k, v, do = _inputs("fp32", 1, 2, 3, 2, 1, 16, dev="cpu")
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        A.attention_forward(q, k, v)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        A.attention(q, k, v)
    with pytest.raises(TypeError, match="torch.Tensor"):
        A.attention_forward(None, k, v)


def _fake(**kw):
    """Arguments whose pointers are never followed: every refusal comes before a launch."""
    from gp_nerf_amd import _lib
    a = _lib.AttnArgs(0, 2, 8, 8, 4, 2, 16, 0, 0.25, 16, 16, 16, (512, 64, 16), (256, 32, 16), (256, 32, 16))
    a.out = a.lse = a.dout = a.dq = a.dk = a.dv = 16
    a.dout_stride = (512, 64, 16)
    for n, x in kw.items():
        setattr(a, n, x)
    return a


@pytest.mark.parametrize("bad,text", [
    (dict(dtype=2), "unknown dtype"), (dict(B=-1), "negative size"), (dict(Lk=-1), "negative size"),
    (dict(Hq=3), "cannot share"), (dict(Hkv=0), "cannot share"), (dict(D=12), "head width"), (dict(D=136), "head width"),
    (dict(D=0), "head width"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(q=None), "null q"), (dict(k=None), "null k"), (dict(v=8), "16-byte"),
    (dict(out=None), "null out"), (dict(lse=None), "null lse"), (dict(q_stride=(512, 64, 2)), "stride"),
    (dict(k_stride=(-256, 32, 16)), "stride"), (dict(Lq=(1 << 23) + 1), "queries"), (dict(Lk=(1 << 30) + 1), "keys"),
    (dict(B=1 << 24), "batches"),
])
def test_c_entry_refuses(bad, text):
    from gp_nerf_amd import _lib
    L = _lib.lib()
    assert L.gpn_attn_forward(ctypes.byref(_fake(**bad)), None) == -1
    assert text in L.gpn_last_error().decode()
    assert L.gpn_attn_backward(ctypes.byref(_fake(**bad)), None) == -1


@pytest.mark.parametrize("scale", [1e-38, 3e38])
def test_c_entry_refuses_scales_that_overflow(scale):
    from gp_nerf_amd import _lib
    L = _lib.lib()
    for fn in (L.gpn_attn_forward, L.gpn_attn_backward):
        assert fn(ctypes.byref(_fake(scale=scale)), None) == -1
        assert b"scale must be between" in L.gpn_last_error()


def test_c_entry_refuses_missing_workspace_and_gradients():
    from gp_nerf_amd import _lib
    L = _lib.lib()
    assert L.gpn_attn_forward(None, None) == -1 and b"null arguments" in L.gpn_last_error()
    assert L.gpn_attn_workspace_bytes(ctypes.byref(_fake(Lq=300, Lk=300)), 1) >= 2 * 300 * 4 * 4
    assert L.gpn_attn_backward(ctypes.byref(_fake(Lq=300, Lk=300)), None) == -1 and b"workspace" in L.gpn_last_error()
    for n in ("dq", "dk", "dv", "dout"):
        assert L.gpn_attn_backward(ctypes.byref(_fake(**{n: None})), None) == -1
        assert ("null " + n).encode() in L.gpn_last_error()
    # few rows against many keys: the keys are divided and the parts need room
    long = _fake(B=1, Lq=1, Lk=1 << 16)
    assert L.gpn_attn_workspace_bytes(ctypes.byref(long), 0) > 0
    assert L.gpn_attn_forward(ctypes.byref(long), None) == -1 and b"workspace" in L.gpn_last_error()
    # nothing to do is a success
    assert L.gpn_attn_forward(ctypes.byref(_fake(B=0, q=None)), None) == 0
    assert L.gpn_attn_backward(ctypes.byref(_fake(B=0, q=None)), None) == 0


def test_attn_struct_layout_matches_header(tmp_path):
    import os
    import subprocess
    from gp_nerf_amd import _lib
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = [n for n, _ in _lib.AttnArgs._fields_]
    src = "#include <stdio.h>\n#include <stddef.h>\n#include \"gpnerf_hip.h\"\nint main(){printf(\"%zu\", sizeof(gpn_attn_args_t));"
    src += "".join('printf(" %%zu", offsetof(gpn_attn_args_t, %s));' % n for n in names) + "return 0;}"
    (tmp_path / "p.c").write_text(src)
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(tmp_path / "p.c"), "-o", str(tmp_path / "p")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "p")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(_lib.AttnArgs)] + [getattr(_lib.AttnArgs, n).offset for n in names]


# ------------------------------------------------------------------------------------------------------------ numerics
SHAPES = [  # B, Lq, Lk, Hq, Hkv, D
    (1, 1, 1, 1, 1, 8), (2, 1, 7, 4, 2, 16), (3, 5, 1, 2, 1, 24), (1, 64, 64, 4, 4, 16), (2, 63, 65, 4, 1, 16),
    (1, 33, 129, 2, 2, 32), (2, 100, 31, 6, 3, 40), (1, 130, 200, 2, 1, 64), (1, 17, 300, 8, 2, 80), (1, 77, 77, 3, 3, 96),
    (1, 129, 257, 2, 1, 104), (1, 200, 190, 4, 2, 128), (5, 128, 128, 4, 4, 16), (9, 3, 40, 1, 1, 128),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_matches_the_formula(dtype, shape):
    _run(*_inputs(dtype, *shape))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(2, 1, 9, 4, 2, 16), (3, 64, 64, 4, 4, 16), (2, 70, 70, 4, 2, 64), (2, 131, 67, 2, 1, 32),
                                   (1, 67, 260, 6, 2, 128), (2, 300, 300, 2, 1, 16)], ids=str)
def test_causal(dtype, shape):
    """More queries than keys among them: the first rows then see nothing."""
    _run(*_inputs(dtype, *shape), causal=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_every_kind_of_mask(dtype):
    B, Lq, Lk = 6, 75, 141
    q, k, v, do = _inputs(dtype, B, Lq, Lk, 6, 2, 48)
    g = torch.Generator().manual_seed(3)
    lengths = torch.tensor([0, 1, 64, 65, 141, 100], dtype=torch.int32).cuda()
    mask = (torch.rand(B, Lk, generator=g) < 0.6)
    mask[5] = False  # a batch whose mask leaves nothing
    mask = mask.cuda()
    start = torch.tensor([3, 0, -10, 64, 66, -80], dtype=torch.int32).cuda()
    _run(q, k, v, do, lengths=lengths)
    _run(q, k, v, do, key_mask=mask)
    _run(q, k, v, do, lengths=lengths, key_mask=mask.to(torch.uint8) * 7)
    _run(q, k, v, do, causal=True, q_start=start)
    got = _run(q, k, v, do, lengths=lengths, key_mask=mask, causal=True, q_start=start, scale=0.37)
    assert bool((got["lse"][5] == -float("inf")).all()) and not bool(got["out"][5].any()) and not bool(got["dk"][0].any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_lengths_and_starts_outside_the_keys_are_taken_in(dtype):
    q, k, v, do = _inputs(dtype, 4, 20, 50, 2, 2, 16)
    big = 2 ** 31 - 1
    a = _both(q, k, v, do, lengths=torch.tensor([-5, 51, big, -big - 1], dtype=torch.int32).cuda(), causal=True,
              q_start=torch.tensor([0, big, -big - 1, 0], dtype=torch.int32).cuda())
    b = _both(q, k, v, do, lengths=torch.tensor([0, 50, 50, 0], dtype=torch.int32).cuda(), causal=True,
              q_start=torch.tensor([0, 50, -20, 0], dtype=torch.int32).cuda())
    for n in a:
        assert torch.equal(a[n], b[n]), n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("D", [16, 64, 128])
@pytest.mark.parametrize("Lq", [1, 40])
def test_hidden_keys_may_hold_anything(dtype, D, Lq):
    B, Lk = 3, 150
    q, k, v, do = _inputs(dtype, B, Lq, Lk, 4, 2, D)
    lengths = torch.tensor([37, 150, 0], dtype=torch.int32).cuda()
    mask = torch.ones(B, Lk, dtype=torch.bool).cuda()
    mask[1, ::3] = False
    want = _both(q, k, v, do, lengths=lengths, key_mask=mask)
    hide = ~(mask & (torch.arange(Lk).cuda() < lengths[:, None]))
    for x, junk in ((k, float("nan")), (v, float("inf"))):
        x[hide] = junk
    got = _both(q, k, v, do, lengths=lengths, key_mask=mask)
    for n in want:
        assert torch.equal(want[n], got[n]), n
    assert not bool(got["dk"][hide].any()) and not bool(got["dv"][hide].any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape,kw", [((1, 1, 5000, 8, 2, 128), {}), ((2, 3, 4099, 4, 4, 64), {"causal": True}),
                                      ((1, 200, 3000, 2, 1, 32), {}), ((2, 1, 2500, 32, 1, 80), {}),
                                      ((3, 2, 1111, 3, 3, 16), {"lengths": (1111, 2, 0)})], ids=str)
def test_long_keys_and_few_rows(dtype, shape, kw):
    """The keys are divided over workgroups and joined; a part may be empty."""
    if "lengths" in kw:
        kw = {"lengths": torch.tensor(kw["lengths"], dtype=torch.int32).cuda()}
    _run(*_inputs(dtype, *shape), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_extreme_scores(dtype):
    """A score far above or below the others, and scores whose exponentials would overflow without the maximum."""
    q, k, v, do = _inputs(dtype, 2, 40, 70, 2, 1, 32)
    q[:, ::2] *= 30.0
    k[:, 3] *= 20.0
    _run(q, k, v, do)
    k[:, :] = k[:, :1]  # all scores equal
    _run(q, k, v, do)


@pytest.mark.gpu
def test_nan_reaches_its_own_row_only():
    q, k, v, do = _inputs("fp32", 1, 40, 50, 2, 2, 16)
    from gp_nerf_amd.attention import attention_forward
    want, _ = attention_forward(q, k, v)
    q[0, 7, 1, 3] = float("nan")
    out, lse = attention_forward(q, k, v)
    assert bool(out[0, 7, 1].isnan().all()) and bool(lse[0, 1, 7].isnan())
    rest = torch.ones(40, 2, dtype=torch.bool).cuda()
    rest[7, 1] = False
    assert torch.equal(out[0][rest], want[0][rest])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_strides_alignment_and_broadcast(dtype):
    B, Lq, Lk, H, D = 2, 37, 61, 2, 32
    q, k, v, do = _inputs(dtype, B, Lq, Lk, H, H, D)
    want = _both(q, k, v, do)

    def same(*x):
        got = _both(*x)
        for n in want:
            assert torch.equal(want[n], got[n]), n

    heads_first = [t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (q, k, v, do)]
    same(*heads_first)
    packed = torch.zeros(B, 80, 3, H, D, dtype=q.dtype).cuda()   # one tensor for all, rows 5 .. of a longer buffer
    packed[:, 5:5 + Lq, 0], packed[:, 5:5 + Lk, 1], packed[:, 5:5 + Lk, 2] = q, k, v
    same(packed[:, 5:5 + Lq, 0], packed[:, 5:5 + Lk, 1], packed[:, 5:5 + Lk, 2], do)
    odd = torch.zeros(q.numel() + 1, dtype=q.dtype).cuda()       # not 16-byte aligned: copied
    odd[1:] = q.flatten()
    same(odd[1:].view(q.shape), k, v, do)
    last = torch.zeros(B, Lk, H, D, 2, dtype=q.dtype).cuda()     # last dimension not contiguous
    last[..., 0] = v
    same(q, k, last[..., 0], do)
    e = _both(q, k[:1].expand(B, -1, -1, -1), v, do)             # one cache for the whole batch
    f = _both(q, k[:1].repeat(B, 1, 1, 1), v, do)
    for n in e:
        assert torch.equal(e[n], f[n]), n


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 3, 4, 2, 1, 16), (2, 0, 4, 2, 1, 16), (2, 3, 0, 2, 1, 16)], ids=str)
def test_nothing_to_do(shape):
    got = _run(*_inputs("bf16", *shape))
    assert not any(bool(t.nan_to_num(0, 0, 0).any()) for t in got.values())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_same_bits_every_time(dtype):
    for shape, kw in (((2, 150, 333, 8, 2, 64), dict(causal=True)), ((1, 1, 4000, 8, 1, 128), {})):
        x = _inputs(dtype, *shape)
        a, b = _both(*x, **kw), _both(*x, **kw)
        for n in a:
            assert torch.equal(a[n], b[n]), n


@pytest.mark.gpu
def test_gradient_against_differences():
    """Central differences of the fp32 kernel itself along random directions."""
    from gp_nerf_amd.attention import attention_forward
    q, k, v, do = _inputs("fp32", 2, 30, 50, 4, 2, 16)
    lengths = torch.tensor([50, 21], dtype=torch.int32).cuda()
    r = _both(q, k, v, do, lengths=lengths)
    g = torch.Generator().manual_seed(9)
    e = 2.0 ** -6
    for name, at in (("dq", 0), ("dk", 1), ("dv", 2)):
        x = [q, k, v]
        d = torch.randn(x[at].shape, generator=g).cuda()
        d /= d.double().norm().float()
        f = []
        for sign in (1, -1):
            y = list(x)
            y[at] = y[at] + sign * e * d
            f.append(float((attention_forward(*y, lengths=lengths)[0].double() * do.double()).sum()))
        slope = float((r[name].double() * d.double()).sum())
        # A unit step changes the loss by at most a few times |do| (60); its third derivative along it is of that order: e^2 / 6 of
        # 60 = 2.4e-3.  Rounding: 2^-24 of each of 3840 outputs times do, in all about 4e-6 of a standard deviation, over 2 e.
        assert abs((f[0] - f[1]) / (2 * e) - slope) < 5e-3, name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_autograd(dtype):
    from gp_nerf_amd.attention import attention
    q, k, v, do = _inputs(dtype, 2, 21, 30, 4, 2, 32)
    mask = (torch.rand(2, 30, generator=torch.Generator().manual_seed(1)) < 0.7).cuda()
    want = _both(q, k, v, do, key_mask=mask, causal=True)
    x = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = attention(*x, key_mask=mask, causal=True)
    out.backward(do)
    assert torch.equal(out, want["out"])
    for t, n in zip(x, ("dq", "dk", "dv")):
        assert torch.equal(t.grad, want[n]), n
    # a broadcast key/value cache: autograd sums the batches' gradients
    kk = k[:1].clone().requires_grad_(True)
    attention(q, kk.expand(2, -1, -1, -1), v).backward(do)
    full = _both(q, k[:1].repeat(2, 1, 1, 1), v, do)["dk"]
    assert torch.equal(kk.grad, full.sum(0, keepdim=True))
    with torch.no_grad():
        assert attention(q, k, v).grad_fn is None
    out = attention(*x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        x[0].data  # noqa: B018  (reading does nothing)
        with torch.no_grad():
            x[0].add_(1)
        out.backward(do)


@pytest.mark.gpu
def test_refuses_on_device():
    from gp_nerf_amd import attention as A
    q, k, v, do = _inputs("fp32", 2, 4, 6, 4, 2, 16)
    bad = [
        (lambda: A.attention_forward(q.half(), k, v), "float32 or bfloat16"),
        (lambda: A.attention_forward(q, k.bfloat16(), v), "expected torch.float32"),
        (lambda: A.attention_forward(q[0], k, v), "q must be"),
        (lambda: A.attention_forward(q, k[:1], v), "k and v must be"),
        (lambda: A.attention_forward(q, k, v[:, :3]), "k and v must be"),
        (lambda: A.attention_forward(q[..., :12], k[..., :12], v[..., :12]), "multiple of 8"),
        (lambda: A.attention_forward(q[:, :, :3], k, v), "cannot share"),
        (lambda: A.attention_forward(q, k, v, lengths=torch.tensor([1, 2]).cuda()), "lengths"),
        (lambda: A.attention_forward(q, k, v, lengths=torch.tensor([1, 2], dtype=torch.int32)), "lengths"),
        (lambda: A.attention_forward(q, k, v, key_mask=torch.ones(2, 6).cuda()), "key_mask"),
        (lambda: A.attention_forward(q, k, v, key_mask=torch.ones(2, 5, dtype=torch.bool).cuda()), "key_mask"),
        (lambda: A.attention_forward(q, k, v, q_start=torch.zeros(2, dtype=torch.int32).cuda()), "only causal"),
        (lambda: A.attention_backward(do[:, :3], q, k, v, do, do), "dout"),
        (lambda: A.attention_backward(do, q, k, v, do, do), "lse"),
        (lambda: A.attention_backward(do.cpu(), q, k, v, do, do), "no CPU fallback"),
    ]
    for f, text in bad:
        with pytest.raises((ValueError, RuntimeError), match=text):
            f()
    with pytest.raises(RuntimeError, match="scale"):
        A.attention_forward(q, k, v, scale=0.0)


@pytest.mark.gpu
def test_other_streams_and_overlapping_calls():
    """Two streams with divided keys (a workspace each) at once, and a result used on its own stream."""
    x = _inputs("bf16", 1, 2, 6000, 8, 2, 128)
    y = _inputs("bf16", 1, 2, 6000, 8, 2, 128, seed=5)
    want = [_both(*x), _both(*y)]
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        got = [None, None]
        for i, z in enumerate((x, y)):
            with torch.cuda.stream(s[i]):
                got[i] = _both(*z)
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            for n in a:
                assert torch.equal(a[n], b[n]), n


@pytest.mark.gpu
def test_captured_step():
    """Forward and backward in one graph, replayed on changing inputs with eager work between; autograd's form is refused there."""
    from gp_nerf_amd.attention import attention
    x = _inputs("bf16", 2, 1, 3000, 8, 2, 64)
    q, k, v, do = (t.clone() for t in x)
    _both(q, k, v, do)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):  # two graphs of the same call: nothing is shared between them
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_both(q, k, v, do))
        graphs.append(g)
    for seed in (1, 2, 3):
        new = _inputs("bf16", 2, 1, 3000, 8, 2, 64, seed=seed)
        for t, y in zip((q, k, v, do), new):
            t.copy_(y)
        for g in graphs:
            g.replay()
        want = _both(*new)
        torch.cuda.synchronize()
        for got in outs:
            for n in want:
                assert torch.equal(want[n], got[n]), n
    leaf = q.clone().requires_grad_(True)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="cannot be captured"):
            attention(leaf, k, v)
        do.mul_(1.0)


@pytest.mark.gpu
def test_ray_attention_of_a_block():
    """GNT's ray attention module: forward against the oracle of the renderer's, and its gradients."""
    import types
    from gp_nerf_amd import synth
    from gp_nerf_amd.transformer_network import GNT
    from oracle import gnt
    args = types.SimpleNamespace(netwidth=64, trans_depth=8, save_feature=False, semantic_model="fpn", num_classes=20)
    net = GNT(args, 32, 63, 63, ret_alpha=True)
    sd = synth.gnt_state_dict()
    net.load_state_dict(sd)
    net = net.cuda()
    attn = net.view_selftrans[2].attn
    g = torch.Generator().manual_seed(4)
    x, do = torch.randn(9, 48, 64, generator=g), torch.randn(9, 48, 64, generator=g)
    dsd = {n: t.double().requires_grad_(True) for n, t in sd.items() if n.startswith("view_selftrans.2.attn.")}
    xd = x.double().requires_grad_(True)
    want, _ = gnt.ray_attention(dsd, "view_selftrans.2.attn", xd)
    (want * do.double()).sum().backward()
    xg = x.cuda().requires_grad_(True)
    out = attn(xg)
    (out * do.cuda()).sum().backward()
    pairs = [(out, want), (xg.grad, xd.grad)] + [
        (getattr(attn, n).weight.grad, dsd["view_selftrans.2.attn.%s.weight" % n].grad) for n in ("q_fc", "k_fc", "v_fc", "out_fc")]
    for got, ref in pairs:
        # chains of at most 64 + 16 + 48 + 64 (+ 432 rows for weights) sums of fp32: 700 half steps of 2^-24, times the
        # ratio of magnitudes summed to the largest result (below 2 here: random signs add up to less, not more)
        assert float((got.detach().cpu().double() - ref.detach()).abs().max()) <= 1400 * 2.0 ** -24 * max(1.0, float(ref.detach().abs().max()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,shape,kw", [("bf16", (1, 300, 300, 4, 2, 128), dict(causal=True)), ("fp32", (2, 90, 200, 2, 2, 128), {}),
                                            ("bf16", (40, 64, 64, 4, 4, 16), {}), ("fp32", (3, 128, 128, 2, 2, 32), {})], ids=str)
def test_captured_kernels_of_every_path(dtype, shape, kw):
    """The kernels with more LDS than a launch has by default, and those of short sequences, captured and replayed."""
    x = _inputs(dtype, *shape)
    cur = [t.clone() for t in x]
    _both(*cur, **kw)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = _both(*cur, **kw)
    for seed in (1, 2, 3):
        new = _inputs(dtype, *shape, seed=seed)
        for t, y in zip(cur, new):
            t.copy_(y)
        g.replay()
        want = _both(*new, **kw)
        torch.cuda.synchronize()
        for n in want:
            assert torch.equal(want[n], got[n]), n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("Lq,D", [(1, 128), (40, 64), (300, 64)])
def test_offsets_past_32_bits(dtype, Lq, D):
    """Keys, values and queries that lie more than 2^32 elements apart: between batches, and between positions."""
    q, k, v, do = _inputs(dtype, 2, Lq, 20, 2, 1, D)
    want = oracle.attention(q, k, v, do, bits=q.dtype)  # (kernels for near rows round in another order: no equal bits to expect)
    names = ("out", "lse", "dq", "dk", "dv")
    step = 2 ** 27 + 16
    buf = torch.empty(20 * step + 2 * D + 64, dtype=q.dtype, device="cuda")  # about 5 (11) GB
    far = lambda t, off, sb, sl, sh: buf.as_strided(t.shape, (sb, sl, sh, 1), off)  # noqa: E731
    kk, vv = far(k, 0, D, step, 0), far(v, 64 + 2 * D, D, step, 0)  # positions apart
    kk.copy_(k), vv.copy_(v)
    _check(_both(q, kk, vv, do), want, names)
    qq, dd = far(q, 0, 17 * step, 2 * D, D), far(do, 2 ** 21, 18 * step, 2 * D, D)  # batches apart
    qq.copy_(q), dd.copy_(do)
    _check(_both(qq, k, v, dd), want, names)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 64, 64, 1, 1, 16), (2, 40, 120, 3, 1, 16), (3, 128, 20, 2, 2, 32), (1, 20, 128, 4, 2, 64),
                                   (2, 16, 100, 8, 1, 24), (4, 31, 33, 1, 1, 8)], ids=str)
def test_short_sequences_with_masks(dtype, shape):
    """Rows and keys that one workgroup holds: whole and partial tiles, masks, causal bounds that skip tiles."""
    B, Lq, Lk = shape[:3]
    x = _inputs(dtype, *shape)
    g = torch.Generator().manual_seed(5)
    mask = (torch.rand(B, Lk, generator=g) < 0.5).cuda()
    lengths = torch.randint(0, Lk + 1, (B,), generator=g).to(torch.int32).cuda()
    start = torch.randint(-Lq, Lk, (B,), generator=g).to(torch.int32).cuda()
    _run(*x)
    _run(*x, causal=True)
    _run(*x, key_mask=mask, lengths=lengths)
    _run(*x, key_mask=mask, lengths=lengths, causal=True, q_start=start)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("G", [1, 2, 3, 8, 24, 32])
def test_groups_of_heads(dtype, G):
    """Shared heads: groups that divide the tiles and those that do not, over several stages and parts."""
    _run(*_inputs(dtype, 1, 150, 270, G, 1, 64), causal=True)
    _run(*_inputs(dtype, 1, 37, 90, 2 * G, 2, 128))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape,causal", [((130, 140, 150, 4, 4, 128), False), ((130, 150, 150, 4, 4, 72), True),
                                          ((65, 150, 300, 8, 8, 24), True)], ids=str)
def test_many_problems(dtype, shape, causal):
    """More problems than workgroups fit the card at once."""
    _run(*_inputs(dtype, *shape), causal=causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape,causal", [((6, 200, 300, 6, 3, 64), False), ((2, 1100, 2100, 4, 4, 24), True),
                                          ((2, 1500, 2100, 4, 2, 40), True), ((4, 130, 700, 4, 2, 80), False),
                                          ((5, 700, 200, 16, 16, 96), True), ((66, 140, 200, 8, 8, 16), False),
                                          ((66, 260, 140, 4, 4, 112), False)], ids=str)
def test_every_cut_of_masked_batches(dtype, shape, causal):
    """Lengths, masks and starts with every way of cutting rows and keys: few rows, halves of tiles, whole tiles, parts."""
    B, Lq, Lk = shape[:3]
    q, k, v, do = _inputs(dtype, *shape)
    g = torch.Generator().manual_seed(5)
    lengths = torch.randint(0, Lk + 1, (B,), generator=g, dtype=torch.int32)
    lengths[0] = Lk
    lengths[-1] = 0
    mask = torch.rand(B, Lk, generator=g) < 0.8
    mask[0, :130] = False  # whole stages without a key
    kw = dict(causal=True, q_start=(Lk - Lq + torch.arange(B, dtype=torch.int32) % 5 - 2).cuda()) if causal else {}
    _run(q, k, v, do, lengths=lengths.cuda(), key_mask=mask.cuda(), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
def test_narrow_heads_over_many_stages(dtype, causal):
    """Heads of 16, whose stages of rows one wave brings alone."""
    _run(*_inputs(dtype, 33, 700, 260, 16, 8, 16), causal=causal)


@pytest.mark.parametrize("name", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("at,single", [(0, dict(B=1)), (1, dict(Lq=1)), (1, dict(Lk=1)), (2, dict(Hq=1, Hkv=1)), (2, dict(Hkv=1))], ids=str)
def test_c_entry_takes_any_stride_of_one_batch_position_or_head(name, at, single):
    """No element lies a stride away along a dimension of one.  The call then stops at its missing workspace, before a launch."""
    from gp_nerf_amd import _lib
    L = _lib.lib()
    alone = {"q": "Lq" in single or "Hq" in single, "k": "Lk" in single or "Hkv" in single}
    alone = alone["q" if name in ("q", "dout") else "k"] or at == 0
    for big in (2565, 1 << 40, -3):
        sizes = dict(dict(Lq=300, Lk=300), **single)
        strides = [512, 64, 16]
        strides[at] = big
        bad = _fake(**sizes, **{name + "_stride": tuple(strides)})
        assert L.gpn_attn_backward(ctypes.byref(bad), None) == -1
        text = L.gpn_last_error().decode()
        assert "workspace" in text if alone or (big > 0 and big % 8 == 0) else "stride" in text, text
        if name != "dout" and "Lk" not in single:
            few = _fake(**dict(sizes, Lq=1, Lk=1 << 16), **{name + "_stride": tuple(strides)})  # (keys in parts)
            assert L.gpn_attn_forward(ctypes.byref(few), None) == -1
            text = L.gpn_last_error().decode()
            one = alone or (at == 1 and name == "q")
            assert "workspace" in text if one or (big > 0 and big % 8 == 0) else "stride" in text, text


def test_strides_of_single_dimensions_do_not_choose_the_kernel():
    """Gradients of short sequences need no workspace unless rows lie far apart."""
    from gp_nerf_amd import _lib
    L = _lib.lib()
    far = (1 << 24, 1 << 24, 16)
    assert L.gpn_attn_workspace_bytes(ctypes.byref(_fake()), 1) == 0
    assert L.gpn_attn_workspace_bytes(ctypes.byref(_fake(q_stride=far)), 1) > 0
    assert L.gpn_attn_workspace_bytes(ctypes.byref(_fake(Lq=1, q_stride=far, dout_stride=far)), 1) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 5, 9, 4, 2, 64), (3, 1, 1, 2, 2, 16), (2, 40, 70, 1, 1, 32), (1, 1, 300, 8, 8, 64),
                                   (1, 200, 1, 1, 1, 128)], ids=str)
def test_single_batches_positions_and_heads_of_any_pitch(dtype, shape):
    """Dimensions of one element, as slices of larger tensors have them: their strides fit no alignment."""
    x = _inputs(dtype, *shape)
    want = _both(*x)

    def odd(t, pitch):  # the same elements; dimensions of one get an odd stride
        s = [p if n > 1 else pitch for n, p in zip(t.shape[:3], t.stride()[:3])]
        return t.as_strided(t.shape, (*s, 1))

    for pitch in (1027, 3, 2 ** 21 + 1):
        got = _both(*(odd(t, pitch) for t in x))
        for n in want:
            assert torch.equal(want[n], got[n]), n
    B, Lk, Hkv, D = x[1].shape
    cache = torch.zeros(3, Lk * Hkv * D + 3, dtype=x[1].dtype).cuda()  # one batch of a buffer with an odd pitch
    cache[0, :Lk * Hkv * D] = x[1][0].flatten()
    k = cache[:, :Lk * Hkv * D].view(3, Lk, Hkv, D)[:1]
    got = _both(x[0][:1], k, x[2][:1], x[3][:1])
    want = _both(*(t[:1].contiguous() for t in x))
    for n in want:
        assert torch.equal(want[n], got[n]), n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(2, 20, 30, 2, 2, 16), (2, 64, 64, 4, 2, 32), (2, 60, 128, 2, 1, 24), (2, 128, 100, 2, 2, 16),
                                   (2, 30, 70, 2, 1, 128), (2, 300, 200, 2, 2, 64)], ids=str)
def test_gradients_of_hidden_keys_are_zero_under_overflown_ones(dtype, shape):
    """A gradient that overflowed, or a query that is NaN, reaches no key that lengths or key_mask hide."""
    B, Lq, Lk = shape[:3]
    q, k, v, do = _inputs(dtype, *shape)
    mask = torch.ones(B, Lk, dtype=torch.bool).cuda()
    mask[:, 1::3] = False
    lengths = torch.tensor([Lk, Lk // 2], dtype=torch.int32).cuda()
    hide = ~(mask & (torch.arange(Lk).cuda() < lengths[:, None]))
    do[0, 2, 0, 3] = float("inf")
    q[1, 1, 1, 5] = float("nan")
    got = _both(q, k, v, do, lengths=lengths, key_mask=mask)
    assert not bool(got["dk"][hide].any()) and not bool(got["dv"][hide].any())


@pytest.mark.parametrize("recording", [True, False])
def test_capture_is_refused_for_recorded_graphs_only(monkeypatch, recording):
    """Nothing is recorded under no_grad, whatever the arguments require: the refusal there is the one of CPU tensors."""
    from gp_nerf_amd.attention import attention
    q, k, v, _ = _inputs("fp32", 1, 2, 3, 2, 1, 16, dev="cpu")
    k.requires_grad_(True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with torch.set_grad_enabled(recording), pytest.raises(RuntimeError, match="cannot be captured" if recording else "no CPU fallback"):
        attention(q, k, v)


@pytest.mark.gpu
def test_captured_without_a_graph():
    """The differentiable form of leaves that require gradients, captured under no_grad."""
    from gp_nerf_amd.attention import attention, attention_forward
    q, k, v, _ = _inputs("bf16", 2, 50, 70, 4, 2, 32)
    leaf = q.clone().requires_grad_(True)
    attention_forward(q, k, v)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g), torch.no_grad():
        out = attention(leaf, k, v)
    for seed in (1, 2, 3):
        new = _inputs("bf16", 2, 50, 70, 4, 2, 32, seed=seed)[0]
        with torch.no_grad():
            leaf.copy_(new)
        g.replay()
        want = attention_forward(new, k, v)[0]
        torch.cuda.synchronize()
        assert torch.equal(out, want)
