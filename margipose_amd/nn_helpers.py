"""Initial values of the parameters this package owns, and layer normalisation.

The MargiPose hot path holds exactly two kinds of learnable layers -- bias-free (transposed)
convolutions and BatchNorm2d -- and the reference seeds them with the rule of its
`init_parameters` (src/margipose/nn_helpers.py:7-21): He/Kaiming normal with the fan counted on
the *leading* weight dimension (`mode='fan_out'`, so Cin*k*k for a ConvTranspose2d whose weight
is (Cin, Cout, k, k)), zero conv bias where one exists, and an identity BatchNorm or LayerNorm (gamma 1,
beta 0).  Only the columns and combiners are seeded this way (margipose_model.py:62,146); the
feature extractor keeps its own initialisation.

layer_norm / LayerNorm (csrc/norm.hip) stand beside the BatchNorm of the columns: that one normalises over the images a GPU holds
(local statistics), these over the channels of one position, whatever the batch.
"""
import math

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib


def _he_normal_leading_(weight):
    """N(0, 2 / (size(0) * receptive field)) in place -- what kaiming_normal_(w, 0, 'fan_out') draws."""
    receptive = weight[0][0].numel() if weight.dim() > 2 else 1
    std = math.sqrt(2.0 / (weight.size(0) * receptive))
    with torch.no_grad():
        return weight.normal_(0.0, std)


def init_parameters(net):
    convs = [m for m in net.modules() if isinstance(m, (nn.Conv2d, nn.ConvTranspose2d))]
    norms = [m for m in net.modules() if isinstance(m, (nn.BatchNorm2d, nn.LayerNorm))]
    for conv in convs:
        _he_normal_leading_(conv.weight)
        if conv.bias is not None:
            nn.init.zeros_(conv.bias)
    for norm in norms:
        if norm.weight is not None:
            nn.init.ones_(norm.weight)
        if norm.bias is not None:
            nn.init.zeros_(norm.bias)
    return net


def _rows(t, cols, who):
    """`t` as (tensor, rows, distance of the rows in elements): a view where its rows are evenly spaced, else a copy."""
    rows = t.numel() // cols
    if t.is_contiguous():
        return t, rows, cols
    if cols == 1 or t.stride(-1) == 1:
        try:
            v = t.view(rows, cols) if rows else t
            return v, rows, (v.stride(0) if rows > 1 else cols)
        except RuntimeError:
            pass
    if _lib.plan_recording():
        raise _lib.MposeError('layer_norm: %s must have evenly spaced rows while a launch plan is recorded' % who)
    return t.contiguous(), rows, cols


def _norm_fwd(x, weight, bias, cols, eps, statistics):
    xr, rows, ld = _rows(x, cols, 'input')
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty((2, rows), dtype=torch.float32, device=x.device) if statistics else None
    at = stats.data_ptr() if statistics else None
    wb = weight if weight is not None else bias
    _lib.check(_lib.lib().mpose_layer_norm_fwd(xr.data_ptr(), ld, weight.data_ptr() if weight is not None else None, bias.data_ptr() if bias is not None else None,
                                               y.data_ptr(), at, at + 4 * rows if statistics else None, rows, cols, eps, _lib.IO_DTYPES[x.dtype],
                                               _lib.IO_DTYPES[wb.dtype] if wb is not None else 0, _lib.stream_ptr()), 'mpose_layer_norm_fwd')
    return y, stats, xr


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, cols, eps):
        with _lib.on_device(x.device):
            y, stats, xr = _norm_fwd(x, weight, bias, cols, eps, True)
        ctx.save_for_backward(x if xr.data_ptr() == x.data_ptr() else xr, weight, stats)
        wb = weight if weight is not None else bias
        ctx.cols, ctx.w_dtype, ctx.w_shape = cols, wb.dtype if wb is not None else torch.float32, wb.shape if wb is not None else None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, stats = ctx.saved_tensors
        cols, dev = ctx.cols, x.device
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        with _lib.on_device(dev):
            xr, rows, x_ld = _rows(x, cols, 'input')
            gr, _, g_ld = _rows(grad, cols, 'gradient')
            dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
            dw = torch.empty(ctx.w_shape, dtype=ctx.w_dtype, device=dev) if need_w else None
            db = torch.empty(ctx.w_shape, dtype=ctx.w_dtype, device=dev) if need_b else None
            n = _lib.lib().mpose_layer_norm_bwd_ws_bytes(rows, cols) if need_w or need_b else 0
            ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
            at = stats.data_ptr()
            _lib.check(_lib.lib().mpose_layer_norm_bwd(gr.data_ptr(), g_ld, xr.data_ptr(), x_ld, weight.data_ptr() if weight is not None else None, at, at + 4 * rows,
                                                       dx.data_ptr() if need_x else None, dw.data_ptr() if need_w else None, db.data_ptr() if need_b else None,
                                                       rows, cols, _lib.IO_DTYPES[x.dtype], _lib.IO_DTYPES[ctx.w_dtype], ws.data_ptr() if n else None, n,
                                                       _lib.stream_ptr()), 'mpose_layer_norm_bwd')
        return dx, dw, db, None, None


def _capture_leaves(leaves):
    """Inside a graph capture: refuse leaves that an autograd graph from outside the capture still holds.  Such a graph ties the leaf's
    gradient accumulation to another stream, and a captured backward pass over it ends the process.  (A leaf's accumulation node lives
    as long as a graph holds it: a mark on the node that is still there after letting the node go says that one does.)"""
    stream = _lib.stream_ptr().value
    for t in leaves:
        node = torch.autograd.graph.get_gradient_edge(t).node
        if node.metadata.get('mpose_captured') == (stream,):
            continue                                  # held by this capture's own calls
        node.metadata['mpose_probe'] = True
        del node
        node = torch.autograd.graph.get_gradient_edge(t).node
        if node.metadata.pop('mpose_probe', False):
            raise _lib.MposeError('layer_norm: an autograd graph made outside this capture still holds one of its leaves: delete the outputs of '
                                  'earlier passes before the capture')
        del node
    return (stream,)


def layer_norm(x, normalized_shape, weight=None, bias=None, eps=1e-5):
    """torch.nn.functional.layer_norm on the device (csrc/norm.hip): (x - mean) / sqrt(var + eps) * weight + bias over the axes
    `normalized_shape`, the last ones of x.  x: float32, bfloat16 or float16, any strides (rows that are evenly spaced are read in
    place); weight and bias: float32 or x's type, contiguous, of shape `normalized_shape`.  Statistics and sums are float32; the gradients of weight and
    bias are added in a fixed order.  Differentiable once.  Inside a graph capture the call is refused while an autograd graph from outside holds
    one of its leaves."""
    shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise _lib.MposeError('layer_norm: x must be a tensor on a ROCm device: margipose_amd has no CPU path')
    if x.dtype not in _lib.IO_DTYPES:
        raise _lib.MposeError('layer_norm: x must be float32, bfloat16 or float16 (got %s)' % x.dtype)
    if not shape or tuple(x.shape[-len(shape):]) != shape or len(shape) > x.dim():
        raise _lib.MposeError('layer_norm: the last axes of x %s are not normalized_shape %s' % (tuple(x.shape), shape))
    cols = math.prod(shape)
    if not 1 <= cols < 2 ** 31:
        raise _lib.MposeError('layer_norm: normalized_shape %s holds no element (or 2^31)' % (shape,))
    for t, name in ((weight, 'weight'), (bias, 'bias')):
        if t is None:
            continue
        if t.device != x.device or t.dtype not in (torch.float32, x.dtype) or tuple(t.shape) != shape or not t.is_contiguous():
            raise _lib.MposeError('layer_norm: %s must be a contiguous tensor of shape %s on x\'s device, float32 or of x\'s type' % (name, shape))
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise _lib.MposeError('layer_norm: weight and bias must have one type')
    eps = float(eps)
    if not 0.0 <= eps < math.inf:
        raise _lib.MposeError('layer_norm: eps must be finite and not negative')
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad)):
        if not torch.cuda.is_current_stream_capturing():
            return _LayerNorm.apply(x, weight, bias, cols, eps)
        leaves = [t for t in (x, weight, bias) if t is not None and t.requires_grad and t.is_leaf]
        mark = _capture_leaves(leaves)
        y = _LayerNorm.apply(x, weight, bias, cols, eps)
        for t in leaves:
            torch.autograd.graph.get_gradient_edge(t).node.metadata['mpose_captured'] = mark
        return y
    with _lib.on_device(x.device):
        return _norm_fwd(x, weight, bias, cols, eps, False)[0]


class LayerNorm(nn.LayerNorm):
    """torch.nn.LayerNorm -- same arguments, parameters and state dict -- on layer_norm."""

    def forward(self, x):
        return layer_norm(x, self.normalized_shape, self.weight, self.bias, self.eps)
