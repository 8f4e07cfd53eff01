"""Softmax attention with its gradients, on the HIP kernels of csrc/attention.hip (`gpn_attn_forward`, `gpn_attn_backward`).

The renderer's own ray attention (`gpn_ray_attn`) is one fused, inference-only launch for rays of at most 128 samples.  The
functions here are its inner product (reference gpnerf/transformer_network.py:155-178, attn_mode 'qk') for what that launch does
not cover: training, longer sequences, masks, shared key/value heads, and single queries against a cache.

    out, lse = attention_forward(q, k, v)                     no graph: inference, captured loops, hand-written steps
    dq, dk, dv = attention_backward(dout, q, k, v, out, lse)
    out = attention(q, k, v)                                  the same pair behind torch.autograd

q is [B, Lq, Hq, D]; k and v are [B, Lk, Hkv, D]; query head h reads key/value head h // (Hq // Hkv).  float32 or bfloat16, all
of one type; D a multiple of 8 up to 128; Hq at most 256 Hkv, Lq * Hq / Hkv and B * Hkv at most 2^24.  Any strides (slices of a
cache, expanded tensors); a tensor whose last dimension is not contiguous or whose rows are not 16-byte aligned is copied first.

A key is visible to a query where all of these hold:
    lengths   [B] int32: the key's position is below its batch's length
    key_mask  [B, Lk] bool or uint8: its entry is not zero
    causal    its position is at most q_start[b] + i for query i.  q_start [B] int32; without it queries are the last
              Lq of Lk positions (Lk - Lq).  For a cache that is filled to `lengths`, q_start = lengths - Lq.
A query that sees no key has out = 0, lse = -inf and no gradient.  Keys hidden by lengths or key_mask are never read: padding
may hold anything.  Keys hidden by causal alone have to be finite, and so have the padding rows of q and dout.

Sums are float32.  In bfloat16 the probabilities and their gradients are rounded to it where they enter the second products, so an
output or a gradient is off by about 0.0024 of its norm, its own rounding (0.0017) among it; float32 arguments are the way to
more bits.
"""
import math

import torch

from . import _lib

MAX_D = 128


def _rows(t):
    """(tensor the kernels can read, its strides between batches, positions and heads): 16-byte rows, contiguous along D."""
    if t.is_contiguous() and t.data_ptr() % 16 == 0:  # (D is a multiple of 8)
        return t, t.stride()[:3]
    per = 16 // t.element_size()
    for copy in (None, torch.Tensor.contiguous, torch.Tensor.clone):
        if copy is not None:
            t = copy(t)
        sb, sl, sh, sd = t.stride()
        if t.shape[0] < 2:
            sb = 0
        if t.shape[1] < 2:
            sl = 0
        if t.shape[2] < 2:
            sh = 0
        if sd == 1 and t.data_ptr() % 16 == 0 and not (sb % per or sl % per or sh % per):
            return t, (sb, sl, sh)
    raise AssertionError("unreachable: a clone is aligned")


def _index(t, name, B, dev):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or tuple(t.shape) != (B,) or t.device != dev:
        raise ValueError("%s: expected an int32 tensor of shape (%d,) on %s" % (name, B, dev))
    return t.contiguous()


def _args(q, k, v, lengths, key_mask, causal, q_start, scale):
    """Checks what both directions take -> (first part of the packed gpn_attn_args_t, up to q_start; its sizes; tensors that
    have to live until the launch)."""
    dt = _lib.dev_float(q, "q").dtype
    _lib.dev_float(k, "k", None, dt)
    _lib.dev_float(v, "v", None, dt)
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError("q must be [B, Lq, Hq, D] and k [B, Lk, Hkv, D]")
    B, Lq, Hq, D = q.shape
    Bk, Lk, Hkv, Dk = k.shape
    if Bk != B or Dk != D or v.shape != k.shape:
        raise ValueError("k and v must be [%d, Lk, Hkv, %d] (got %s and %s)" % (B, D, tuple(k.shape), tuple(v.shape)))
    if D % 8 or not 8 <= D <= MAX_D:
        raise ValueError("head width must be a multiple of 8 up to %d (got %d)" % (MAX_D, D))
    if Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise ValueError("%d query heads cannot share %d key/value heads" % (Hq, Hkv))
    dev = q.device
    if k.device != dev or v.device != dev:
        _lib.same_device(q, k=k, v=v)
    if q_start is not None and not causal:
        raise ValueError("q_start: only causal attention has positions")
    q, sq = _rows(q)
    k, sk = _rows(k)
    v, sv = _rows(v)
    if lengths is not None:
        lengths = _index(lengths, "lengths", B, dev)
    if q_start is not None:
        q_start = _index(q_start, "q_start", B, dev)
    if key_mask is not None:
        if not isinstance(key_mask, torch.Tensor) or key_mask.dtype not in (torch.bool, torch.uint8) or \
                tuple(key_mask.shape) != (B, Lk) or key_mask.device != dev:
            raise ValueError("key_mask: expected a bool or uint8 tensor of shape (%d, %d) on %s" % (B, Lk, dev))
        if Lk > 1 and key_mask.stride(1) != 1:
            key_mask = key_mask.contiguous()
    head = (_lib.DTYPES[dt], B, Lq, Lk, Hq, Hkv, D, 1 if causal else 0, 1.0 / math.sqrt(D) if scale is None else scale,
            q.data_ptr(), k.data_ptr(), v.data_ptr(), *sq, *sk, *sv, 0 if lengths is None else lengths.data_ptr(),
            0 if key_mask is None else key_mask.data_ptr(), 0 if key_mask is None else key_mask.stride(0),
            0 if q_start is None else q_start.data_ptr())
    return head, (q, k, v, lengths, q_start, key_mask)


def _call(fn, name, backward, dev, *fields):
    """Workspace and launch on the current stream of the tensors' device."""
    pack = _lib.ATTN.pack
    args = pack(*fields, 0, 0)
    need = _lib.lib().gpn_attn_workspace_bytes(args, backward)
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        args = pack(*fields, ws.data_ptr(), need)
    _lib.call_on(dev, fn, name, args)


def attention_forward(q, k, v, lengths=None, key_mask=None, causal=False, q_start=None, scale=None):
    """-> out [B, Lq, Hq, D] of q's type, lse [B, Hq, Lq] float32 (natural logarithm of the row's sum; -inf without a key).
    scale: of the scores, from 1e-30 to 1e30 (1 / sqrt(D) unless given).  No graph is recorded."""
    head, keep = _args(q, k, v, lengths, key_mask, causal, q_start, scale)
    out = q.new_empty(q.shape)
    lse = q.new_empty((head[1], head[4], head[2]), dtype=torch.float32)
    _call(_lib.lib().gpn_attn_forward, "gpn_attn_forward", 0, q.device, *head, out.data_ptr(), lse.data_ptr(), 0, 0, 0, 0, 0, 0, 0)
    return out, lse


def attention_backward(dout, q, k, v, out, lse, lengths=None, key_mask=None, causal=False, q_start=None, scale=None):
    """Gradients of sum(out * dout) -> dq, dk, dv (shapes and type of q, k, v, contiguous).  out and lse are what
    attention_forward returned for the same arguments; the probabilities are computed again from them.  No graph is recorded."""
    head, keep = _args(q, k, v, lengths, key_mask, causal, q_start, scale)
    shape, dt, dev = q.shape, q.dtype, q.device
    _lib.dev_float(dout, "dout", shape, dt)
    _lib.dev_float(out, "out", shape, dt)
    _lib.dev_float(lse, "lse", (shape[0], shape[2], shape[1]), torch.float32)
    if dout.device != dev or out.device != dev or lse.device != dev:
        _lib.same_device(q, dout=dout, out=out, lse=lse)
    dout, sdo = _rows(dout)
    if not out.is_contiguous() or out.data_ptr() % 16:
        out = out.clone(memory_format=torch.contiguous_format)
    lse = lse.contiguous()
    dq, dk, dv = q.new_empty(shape), k.new_empty(k.shape), v.new_empty(v.shape)
    _call(_lib.lib().gpn_attn_backward, "gpn_attn_backward", 1, dev, *head, out.data_ptr(), lse.data_ptr(), dout.data_ptr(), *sdo,
          dq.data_ptr(), dk.data_ptr(), dv.data_ptr())
    return dq, dk, dv


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, key_mask, causal, q_start, scale, recording):
        if recording and any(ctx.needs_input_grad):  # (which says what the arguments require, under no_grad too)
            _lib.refuse_capture("attention", "attention_forward and attention_backward")
        out, lse = attention_forward(q, k, v, lengths, key_mask, causal, q_start, scale)
        ctx.save_for_backward(q, k, v, out, lse, lengths, key_mask, q_start)
        ctx.causal, ctx.scale = causal, scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        _lib.refuse_capture("attention", "attention_forward and attention_backward")
        q, k, v, out, lse, lengths, key_mask, q_start = ctx.saved_tensors
        grads = attention_backward(dout, q, k, v, out, lse, lengths, key_mask, ctx.causal, q_start, ctx.scale)
        return (*grads, None, None, None, None, None, None)


def attention(q, k, v, lengths=None, key_mask=None, causal=False, q_start=None, scale=None):
    """attention_forward's output, differentiable in q, k and v (once; not inside a captured graph, unless under no_grad)."""
    return _Attention.apply(q, k, v, lengths, key_mask, causal, q_start, scale, torch.is_grad_enabled())
