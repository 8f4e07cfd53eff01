"""`NeRFSemSegFPNHead` -- eval branch of reference gpnerf/semantic_branch.py (ctor :13-43, forward
:89-107) with the reference's state-dict names (`scale_heads.{i}.{j}.weight`,
`scale_heads.{i}.{j}.norm.{weight,bias}`, `predictor.{weight,bias}`).

Runs once per image on the rendered [1,512,h,w] feature image (about 8 GFLOP) as a
plain torch module on the HIP device: conv / GroupNorm / bilinear resize are library ops, not part of
the per-ray hot path that the HIP kernels of this package replace.  detectron2's `Conv2d(norm=...,
activation=...)` is restated as conv -> GroupNorm(32,128) -> ReLU and fvcore's c2_msra_fill as
kaiming_normal_(fan_out, relu).  The head's own training branch (:60-88: feature
distillation, depth guidance) is out of scope and raises.  `distill_topk_loss` teaches class logits (the head's, or rows over
a vocabulary) from a teacher's top entries, with its gradient.  The reference hard-codes a 120x160 feature image (:95); here
the size is taken from the input (identical for 120x160).
"""
import ctypes as C

import numpy as np
import torch
from torch import nn
from torch.nn import functional as F

from . import _lib


def semantic_labels(logits, dtype=torch.int64):
    """Label image of the head's logits [1,C,H,W] (or [C,H,W]): what the reference obtains as
    `sems.permute(0,2,3,1).argmax(dim=-1)` (eval_gpnerf.py:201-206, loss.py:293-300), in one HIP
    kernel over the NCHW logits.  dtype int64 (reference) or uint8 (1 byte per pixel, for gathers)."""
    x = _lib.dev_f32(_lib.as_f32c(logits), "logits")
    if x.dim() == 4:
        if x.shape[0] != 1:
            raise ValueError("semantic_labels: one image at a time (batch %d)" % x.shape[0])
        x = x[0]
    if x.dim() != 3:
        raise ValueError("semantic_labels: expected [1,C,H,W] or [C,H,W]")
    Cn, H, W = x.shape
    if dtype not in (torch.int64, torch.uint8):
        raise ValueError("semantic_labels: dtype must be torch.int64 or torch.uint8")
    out = torch.empty((H, W), dtype=dtype, device=x.device)
    p64 = _lib.ptr(out) if dtype == torch.int64 else None
    p8 = _lib.ptr(out) if dtype == torch.uint8 else None
    with torch.cuda.device(x.device):
        _lib.check(_lib.lib().gpn_argmax_labels(_lib.ptr(x), Cn, H * W, p64, p8, _lib.stream()),
                   "gpn_argmax_labels")
    return out


_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}  # GPN_RED_* of include/gpnerf_hip.h
MAX_TEACHER_ENTRIES = 256


def _as_rows(x, name):
    """[N, C] as it is; an image [1, C, H, W] or [C, H, W] as the [H*W, C] view of its planes."""
    if isinstance(x, torch.Tensor):
        if x.dim() == 2:
            return x
        if x.dim() in (3, 4) and x.is_contiguous() and x.numel() and x.shape[:-3] in ((), (1,)):
            c, h, w = x.shape[-3:]
            return x.as_strided((h * w, c), (1, h * w))
        if x.dim() == 4 and x.shape[0] == 1:
            x = x[0]
        if x.dim() == 3:
            return x.flatten(1).t()
    raise ValueError("%s: expected [N, classes], [classes, H, W] or [1, classes, H, W]" % name)


def _distill_args(logits, teacher_logits, teacher_index, temperature, row_weight, reduction, grad_scale=1.0):
    """Checks -> (first part of the packed gpn_distill_args_t, up to row_weight; logits as rows; whether their rows are what is
    contiguous; tensors that have to live until the launch)."""
    z = _lib.dev_float(_as_rows(logits, "logits"), "logits")
    t = _lib.dev_float(_as_rows(teacher_logits, "teacher_logits"), "teacher_logits")
    x = _as_rows(teacher_index, "teacher_index")
    N, Cn = z.shape
    K = t.shape[1]
    if t.shape[0] != N or x.shape != t.shape:
        raise ValueError("teacher_logits and teacher_index must have a row of K entries for each of the %d rows (got %s and %s)"
                         % (N, tuple(t.shape), tuple(x.shape)))
    if x.dtype not in (torch.int32, torch.int64):
        raise ValueError("teacher_index: expected int32 or int64, got %s" % x.dtype)
    if K > MAX_TEACHER_ENTRIES:
        raise ValueError("at most %d teacher entries per row (got %d)" % (MAX_TEACHER_ENTRIES, K))
    if Cn < 1:
        raise ValueError("logits: no classes")
    if reduction not in _REDUCTIONS:
        raise ValueError("reduction must be one of %s (got %r)" % (sorted(_REDUCTIONS), reduction))
    if row_weight is not None:
        row_weight = _lib.dev_float(row_weight, "row_weight", (N,), torch.float32).contiguous()
    dev = z.device
    if t.device != dev or x.device != dev or row_weight is not None:
        _lib.same_device(z, teacher_logits=t, teacher_index=x, row_weight=row_weight)
    rs, cs = z.stride()
    planes = cs != 1 and Cn > 1
    if planes and rs != 1 and N > 1:
        z = z.contiguous()
        (rs, cs), planes = z.stride(), False
    head = (_lib.DTYPES[z.dtype], _lib.DTYPES[t.dtype], x.element_size(), Cn, K, _REDUCTIONS[reduction], temperature, grad_scale, N,
            z.data_ptr(), rs, cs, t.data_ptr(), *t.stride(), x.data_ptr(), *x.stride(),
            0 if row_weight is None else row_weight.data_ptr())
    return head, z, planes, (t, x, row_weight)


def _distill_gradient(z, planes, logits):
    """Memory for dlogits as the logits lie (class planes or rows) -> it in the logits' shape, (address, strides)."""
    N, Cn = z.shape
    if planes:
        d = z.new_empty((Cn, N))
        return d.t() if logits.dim() == 2 else d.view(logits.shape), (d.data_ptr(), 1, N)
    d = z.new_empty((N, Cn))
    return d if logits.dim() == 2 else d.t().reshape(logits.shape), (d.data_ptr(), Cn, 1)


def _distill_call(name, dev, *fields):
    _lib.call_on(dev, getattr(_lib.lib(), name), name, _lib.DISTILL.pack(*fields))


def distill_topk_forward(logits, teacher_logits, teacher_index, temperature=1.0, row_weight=None, reduction="mean"):
    """Loss of class logits against a teacher's top logits: per row T^2 * KL(softmax of the teacher's K entries at
    temperature T || softmax of all the student's classes at T).

    logits [N, C] (any strides with contiguous classes or contiguous rows, others are copied; with contiguous classes at most
    4194303 rows) or an image [1, C, H, W] as NeRFSemSegFPNHead gives it; float32 or bfloat16.  teacher_logits, teacher_index
    [N, K] (or [1, K, H, W]): what `teacher.topk(K, dim=1)` returns; int32 or int64 classes; an entry outside [0, C) (-1) is left
    out and a row without an entry counts as zero.  row_weight [N] float32: weight of each row (0 leaves it out, whatever it holds).
    reduction: 'mean' over all N rows, 'sum' or 'none'.  temperature from 1e-12 to 1e12.  -> loss (scalar, or [N]), lse [N]
    (what distill_topk_backward needs).  No graph is recorded."""
    head, z, _, keep = _distill_args(logits, teacher_logits, teacher_index, temperature, row_weight, reduction)
    N, dev = z.shape[0], z.device
    rows = torch.empty(N, device=dev)
    lse = torch.empty(N, device=dev)
    loss = rows if reduction == "none" else torch.empty((), device=dev)
    _distill_call("gpn_distill_forward", dev, *head, rows.data_ptr(), loss.data_ptr(), lse.data_ptr(), 0, 0, 0, 0)
    return loss, lse


def distill_topk_backward(dloss, logits, teacher_logits, teacher_index, lse, temperature=1.0, row_weight=None,
                          reduction="mean"):
    """Gradient of the logits for the loss's gradient `dloss` (float32; scalar, or [N] for 'none'); other arguments as given
    to distill_topk_forward, lse as it returned.  -> dlogits, of the logits' type, shape and layout."""
    head, z, planes, keep = _distill_args(logits, teacher_logits, teacher_index, temperature, row_weight, reduction)
    N = z.shape[0]
    dloss = _lib.dev_float(dloss, "dloss", (N,) if reduction == "none" else (), torch.float32).contiguous()
    lse = _lib.dev_float(lse, "lse", (N,), torch.float32).contiguous()
    _lib.same_device(z, dloss=dloss, lse=lse)
    d, at = _distill_gradient(z, planes, logits)
    _distill_call("gpn_distill_backward", z.device, *head, 0, 0, lse.data_ptr(), dloss.data_ptr(), *at)
    return d


def distill_topk_step(logits, teacher_logits, teacher_index, temperature=1.0, row_weight=None, reduction="mean",
                      grad_scale=1.0):
    """distill_topk_forward and the gradient of `grad_scale * loss` in one pass over the logits, for a training step that
    knows the loss's weight (with 'none': of the sum of the rows).  -> loss, dlogits."""
    head, z, planes, keep = _distill_args(logits, teacher_logits, teacher_index, temperature, row_weight, reduction, grad_scale)
    dev = z.device
    rows = torch.empty(z.shape[0], device=dev)
    loss = rows if reduction == "none" else torch.empty((), device=dev)
    d, at = _distill_gradient(z, planes, logits)
    _distill_call("gpn_distill_step", dev, *head, rows.data_ptr(), loss.data_ptr(), 0, 0, *at)
    return loss, d


class _DistillTopK(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher_logits, teacher_index, temperature, row_weight, reduction, recording):
        if recording and ctx.needs_input_grad[0]:  # (which says what the logits require, under no_grad too)
            _lib.refuse_capture("distill_topk_loss", "distill_topk_step")
        loss, lse = distill_topk_forward(logits, teacher_logits, teacher_index, temperature, row_weight, reduction)
        ctx.save_for_backward(logits, teacher_logits, teacher_index, row_weight, lse)
        ctx.temperature, ctx.reduction = temperature, reduction
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        _lib.refuse_capture("distill_topk_loss", "distill_topk_step")
        logits, t, x, w, lse = ctx.saved_tensors
        return (distill_topk_backward(dloss, logits, t, x, lse, ctx.temperature, w, ctx.reduction), None, None, None, None, None,
                None)


def distill_topk_loss(logits, teacher_logits, teacher_index, temperature=1.0, row_weight=None, reduction="mean"):
    """distill_topk_forward's loss, differentiable in the logits (once; not inside a captured graph, unless under no_grad).  The
    teacher and the weights take no gradient."""
    return _DistillTopK.apply(logits, teacher_logits, teacher_index, temperature, row_weight, reduction, torch.is_grad_enabled())


class _ConvGNReLU(nn.Conv2d):
    def __init__(self, cin, cout):
        super().__init__(cin, cout, kernel_size=3, stride=1, padding=1, bias=False)
        self.norm = nn.GroupNorm(32, cout)
        nn.init.kaiming_normal_(self.weight, mode="fan_out", nonlinearity="relu")

    def forward(self, x):
        return F.relu(self.norm(super().forward(x)))


class NeRFSemSegFPNHead(nn.Module):
    def __init__(self, args, feature_strides=[2, 4, 8, 16], feature_channels=[128, 128, 128, 128],
                 num_classes=20):
        super().__init__()
        self.n_p = getattr(args, "n_p", 0)
        conv_dims = 128
        self.common_stride = 2
        self.scale_heads = nn.ModuleList()
        for stride, channels in zip(feature_strides, feature_channels):
            ops = []
            head_length = max(1, int(np.log2(stride) - np.log2(self.common_stride)))
            for k in range(head_length):
                ops.append(_ConvGNReLU(channels if k == 0 else conv_dims, conv_dims))
                if stride != self.common_stride:
                    ops.append(nn.Upsample(scale_factor=2, mode="bilinear", align_corners=False))
            self.scale_heads.append(nn.Sequential(*ops))
        self.predictor = nn.Conv2d(conv_dims, num_classes + 1, kernel_size=1, stride=1, padding=0)

    @torch.no_grad()
    def forward(self, deep_feats, agg_sem_feats=None, select_inds=None):
        """deep_feats [1,512,h,w] -> logits [1,num_classes+1,2h,2w] (reference :89-107)."""
        if select_inds is not None:
            raise NotImplementedError("training branch (distillation / depth-guided losses, reference "
                                      "semantic_branch.py:60-88) is outside the rendering hot path")
        h, w = deep_feats.shape[-2:]
        flat = deep_feats.reshape(1, deep_feats.shape[1], -1).squeeze(0).permute(1, 0)
        x = None
        for i, chunk in enumerate(torch.chunk(flat, 4, dim=1)):
            chunk = chunk.reshape(h, w, chunk.shape[-1]).permute(2, 0, 1).unsqueeze(0)
            if i == 0:
                x = self.scale_heads[i](chunk)
            else:
                chunk = F.interpolate(chunk, scale_factor=1 / (2 ** i), mode="bilinear",
                                      align_corners=True, recompute_scale_factor=True)
                x = x + self.scale_heads[i](chunk)
        out = self.predictor(x)
        return F.interpolate(out, scale_factor=2, mode="bilinear", align_corners=True)

    @torch.no_grad()
    def labels(self, deep_feats, dtype=torch.int64):
        """Eval-branch logits followed by the label epilogue (`semantic_labels`): [2h, 2w] labels."""
        return semantic_labels(self.forward(deep_feats), dtype)
