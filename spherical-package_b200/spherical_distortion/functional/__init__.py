"""Functional interface of the mapped-operator path.

Mirrors layers/functional/mapped_convolution.py:121-148,
layers/functional/mapped_pooling.py:203-245, layers/functional/resample.py:113-219,
layers/functional/convolution.py:62-71 and the map-driven halves of
layers/functional/tangent_images.py:6-55 of the reference: the same call
signatures and assertions, on top of ``_spherical_distortion_ext``.

Beside them stand operators that a network of mapped convolutions is trained and read with and that the reference takes from
its host framework: ``rms_norm`` / ``rms_norm_quantized`` and ``token_log_probs`` (the optimizer step is in ``sphmap.optim``).
"""
from typing import NamedTuple, Optional

import torch

import _spherical_distortion_ext._C as _C
import _spherical_distortion_ext._convolution as _std_conv
import _spherical_distortion_ext._mapped_avg_pooling as _avgpool
import _spherical_distortion_ext._transposed_convolution as _std_tconv
import _spherical_distortion_ext._uv_resample as _uv
import _spherical_distortion_ext._voting_resample as _vote
import _spherical_distortion_ext._weighted_mapped_avg_pooling as _wavgpool

from ..layer_utils import InterpolationType, check_args, check_input_map_shape


def _scalars(kernel_size, interp):
    return torch.tensor(kernel_size), torch.tensor(int(interp))


class _AsFunction(torch.autograd.Function):
    """A native operator inside a Python autograd Function, for what its own node is invisible to: torch.jit traces record the
    Function as one opaque node; forward-mode differentiation and torch.func transforms refuse it, as they do any without rules
    of their own."""

    @staticmethod
    def forward(ctx, op, *args):
        wanted = [i for i in range(len(args)) if ctx.needs_input_grad[i + 1]]
        inner = [a.detach().requires_grad_(i in wanted) if isinstance(a, torch.Tensor) else a for i, a in enumerate(args)]
        with torch.set_grad_enabled(bool(wanted)):
            out = op(*inner, True)
        if out is None:
            raise AssertionError("arguments do not fit the operator")
        many = isinstance(out, (tuple, list))
        outs = out if many else (out,)
        ctx.wanted, ctx.inputs, ctx.outputs = wanted, [inner[i] for i in wanted], outs
        result = [o.detach() for o in outs]
        ctx.mark_non_differentiable(*[r for o, r in zip(outs, result) if not o.requires_grad])
        return tuple(result) if many else result[0]

    @staticmethod
    def backward(ctx, *grad_outputs):
        pairs = [(o, g) for o, g in zip(ctx.outputs, grad_outputs) if o.requires_grad and g is not None]
        grads = iter(torch.autograd.grad([o for o, _ in pairs], ctx.inputs, [g for _, g in pairs], retain_graph=True, allow_unused=True))
        return (None,) + tuple(next(grads) if i in ctx.wanted else None for i in range(len(ctx.needs_input_grad) - 1))


def _by_function(op, args, *checks):
    """The native operator returned nothing: its arguments fail the checks, whose assertions are raised here, or something
    that its autograd node is invisible to looks at the call."""
    for fn, *a in checks:
        fn(*a)
    return _AsFunction.apply(op, *args)


# The operators' autograd nodes are part of the native extension: one call per operator.
def mapped_convolution(input, weight, bias, sample_map, kernel_size, interp, interp_weights=None, activation=None):
    """`activation` (None or "relu") is an extension of this library: the ReLU runs inside the convolution kernels
    instead of as separate passes over the output and its gradient."""
    assert activation in (None, "relu"), "activation must be None or 'relu'"
    args = (input, weight, bias, sample_map, kernel_size, interp, interp_weights, activation is not None)
    out = _C.mapped_convolution_op(*args)
    if out is None:
        out = _by_function(_C.mapped_convolution_op, args,
                           (check_args, input, sample_map, interp_weights, weight.shape[1], weight.shape[2]))
    return out


def mapped_transposed_convolution(input, weight, bias, sample_map, output_height, output_width, kernel_size, interp,
                                  interp_weights=None):
    args = (input, weight, bias, sample_map, output_height, output_width, kernel_size, interp, interp_weights)
    out = _C.mapped_transposed_convolution_op(*args)
    if out is None:
        out = _by_function(_C.mapped_transposed_convolution_op, args,
                           (check_args, input, sample_map, interp_weights, weight.shape[0], weight.shape[2]),
                           (check_input_map_shape, input, sample_map))
    return out


def mapped_max_pool(input, sample_map, kernel_size, interp, interp_weights=None):
    args = (input, sample_map, kernel_size, interp, interp_weights)
    out = _C.mapped_max_pool_op(*args)
    if out is None:
        out = _by_function(_C.mapped_max_pool_op, args, (check_args, input, sample_map, interp_weights, None, kernel_size))
    return out


def _with_batch(fn, input, *args):
    assert input.dim() in (3, 4), "Input must have 3 or 4 dimensions (input.dim() == {})".format(input.dim())
    if input.dim() == 3:
        return fn(input.unsqueeze(0), *args).squeeze(0)
    return fn(input, *args)


def resample(input, sample_map, output_shape, interp, interp_weights=None):
    """Scatter forward, gather backward (layers/functional/resample.py:11-48)."""
    def run(x):
        args = (x, sample_map, interp, interp_weights, True, output_shape[0], output_shape[1])
        out = _C.resample_op(*args)
        if out is None:
            out = _by_function(_C.resample_op, args, (check_args, x, sample_map, interp_weights, None, None),
                               (check_input_map_shape, x, sample_map))
        return out
    return _with_batch(run, input)


def unresample(input, sample_map, interp, interp_weights=None):
    """Gather forward, scatter backward (layers/functional/resample.py:51-83)."""
    def run(x):
        args = (x, sample_map, interp, interp_weights, False, 0, 0)
        out = _C.resample_op(*args)
        if out is None:
            out = _by_function(_C.resample_op, args, (check_args, x, sample_map, interp_weights, None, None))
        return out
    return _with_batch(run, input)


# ---- average pooling (layers/functional/mapped_pooling.py:9-101, 203-223) ---------------------------------
class _MappedAvgPool(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, sample_map, kernel_size, interp, interp_weights):
        ctx.save_for_backward(torch.tensor([x.shape[2], x.shape[3]]), sample_map, *_scalars(kernel_size, interp), interp_weights)
        if interp_weights is None:
            return _avgpool.mapped_avg_pool(x, sample_map, kernel_size, interp)
        return _wavgpool.weighted_mapped_avg_pool(x, sample_map, interp_weights, kernel_size, interp)

    @staticmethod
    def backward(ctx, grad_output):
        in_shape, sample_map, kernel_size, interp, interp_weights = ctx.saved_tensors
        interp = InterpolationType(interp)
        if interp_weights is None:
            gx = _avgpool.mapped_avg_unpool(grad_output, sample_map, in_shape[0], in_shape[1], kernel_size, interp)
        else:
            gx = _wavgpool.weighted_mapped_avg_unpool(grad_output, sample_map, interp_weights, in_shape[0], in_shape[1],
                                                      kernel_size, interp)
        return gx, None, None, None, None


class _MappedAvgUnpool(torch.autograd.Function):
    """The adjoint used as a forward operator (an up-sampling layer); its gradient is the pooling itself."""

    @staticmethod
    def forward(ctx, x, oh, ow, sample_map, kernel_size, interp, interp_weights):
        ctx.save_for_backward(sample_map, *_scalars(kernel_size, interp), interp_weights)
        if interp_weights is None:
            return _avgpool.mapped_avg_unpool(x, sample_map, oh, ow, kernel_size, interp)
        return _wavgpool.weighted_mapped_avg_unpool(x, sample_map, interp_weights, oh, ow, kernel_size, interp)

    @staticmethod
    def backward(ctx, grad_output):
        sample_map, kernel_size, interp, interp_weights = ctx.saved_tensors
        interp = InterpolationType(interp)
        grad_output = grad_output.contiguous()
        if interp_weights is None:
            gx = _avgpool.mapped_avg_pool(grad_output, sample_map, kernel_size, interp)
        else:
            gx = _wavgpool.weighted_mapped_avg_pool(grad_output, sample_map, interp_weights, kernel_size, interp)
        return gx, None, None, None, None, None, None


def mapped_avg_pool(input, sample_map, kernel_size, interp, interp_weights=None):
    check_args(input, sample_map, interp_weights, None, kernel_size)
    return _MappedAvgPool.apply(input, sample_map, kernel_size, interp, interp_weights)


def mapped_avg_unpool(input, oh, ow, sample_map, kernel_size, interp, interp_weights=None):
    check_args(input, sample_map, interp_weights, None, kernel_size)
    check_input_map_shape(input, sample_map)
    return _MappedAvgUnpool.apply(input, oh, ow, sample_map, kernel_size, interp, interp_weights)


# ---- UV-map and voting resampling (layers/functional/resample.py:86-110, 159-219) -----------------------------
class _UVResample(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, quad_idx, tex_uv, interp):
        ctx.save_for_backward(quad_idx, tex_uv, torch.tensor(int(interp)), torch.tensor(x.shape[-3:]))
        return _uv.resample_from_uv_maps(x, quad_idx, tex_uv, interp)

    @staticmethod
    def backward(ctx, grad_output):
        quad_idx, tex_uv, interp, tex_shape = ctx.saved_tensors
        return _uv.resample_to_uv_maps(grad_output.contiguous(), quad_idx, tex_uv, tex_shape[0], tex_shape[1], tex_shape[2],
                                       InterpolationType(interp)), None, None, None


def uv_resample(input, quad_idx, tex_uv, interp):
    """input ([B,] C, textures, TH, TW) -> ([B,] C, H, W): every image pixel samples texture quad_idx[y, x] at tex_uv[y, x]."""
    assert input.dim() in (4, 5), "Input must have 4 or 5 dimensions (input.dim() == {})".format(input.dim())
    if input.dim() == 4:
        return _UVResample.apply(input.unsqueeze(0), quad_idx, tex_uv, interp).squeeze(0)
    return _UVResample.apply(input, quad_idx, tex_uv, interp)


def voting_resample(input, sample_map, interp_weights, output_shape, num_candidates):
    """Integer labels are moved through an integer (x, y) sample map; every output pixel takes the label most of the
    pixels that land on it carry (layers/functional/resample.py:159-190; `interp_weights` is accepted and, as in the
    reference, has no effect on the result)."""
    def run(x):
        check_args(x, sample_map, interp_weights, None, None)
        check_input_map_shape(x, sample_map)
        return _vote.voting_resample_to_map(x.long().contiguous(), sample_map.long().contiguous(), *output_shape, num_candidates)
    return _with_batch(run, input)


def resample_normalized(input, sample_map, output_shape, interp, interp_weights=None):
    """resample(...) divided by the resampled weight sum: scatter(x) / (scatter(1) + 1e-12), the normalisation the
    reference applies after its scatters (layers/functional/sphere_ops.py:74-80), fused into the scatter kernel.
    Forward only (no autograd node)."""
    def run(x):
        check_args(x, sample_map, interp_weights, None, None)
        check_input_map_shape(x, sample_map)
        return _C.resample_to_map_normalized(x, sample_map, interp_weights, output_shape[0], output_shape[1], interp)
    return _with_batch(run, input.detach())


# ---- tangent images (layers/functional/tangent_images.py:6-55) -------------------------------------------------
def create_tangent_images(input, sample_map, num_samples, interpolation=InterpolationType.BISPHERICAL):
    """([B,] C, H, W) equirectangular image -> ([B,] C, faces, num_samples, num_samples) tangent images through a
    (faces, num_samples*num_samples, 2) sample map.  The reference derives the map from its icosphere mesh utilities
    (layers/util/tangent_images.py), which are outside this package: pass the map in."""
    t = unresample(input, sample_map, interpolation)
    return t.view(*t.shape[:-1], num_samples, num_samples)


def tangent_images_to_equirectangular(tangent_images, quad, uv, interpolation=InterpolationType.BILINEAR):
    """([B,] C, faces, D, D) tangent images -> ([B,] C, H, W) through the (H, W) face-index / (H, W, 2) UV maps."""
    assert tangent_images.dim() in (4, 5), \
        "tangent_images must be a 4D or 5D tensor (tangent_images.dim() == {})".format(tangent_images.dim())
    return uv_resample(tangent_images, quad, uv, interpolation)


# ---- standard convolution (layers/functional/convolution.py:10-71) -------------------------------------------
class _Convolution(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, kernel_size, stride, padding, dilation):
        ctx.save_for_backward(x, weight, bias)
        ctx.geom = (tuple(kernel_size), tuple(stride), tuple(padding), tuple(dilation))
        return _std_conv.conv_forward(x, weight, bias, *kernel_size, *stride, *padding, *dilation)

    @staticmethod
    def backward(ctx, grad_output):
        x, weight, bias = ctx.saved_tensors
        k, s, p, d = ctx.geom
        gx, gw, gb = _std_conv.conv_backward(grad_output, x, weight, bias, *k, *s, *p, *d)
        return gx, gw, gb, None, None, None, None


class _TransposedConvolution(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, kernel_size, stride, padding, dilation):
        ctx.save_for_backward(x, weight, bias)
        ctx.geom = (tuple(kernel_size), tuple(stride), tuple(padding), tuple(dilation))
        return _std_tconv.transposed_conv_forward(x, weight, bias, *kernel_size, *stride, *padding, *dilation)

    @staticmethod
    def backward(ctx, grad_output):
        x, weight, bias = ctx.saved_tensors
        k, s, p, d = ctx.geom
        gx, gw, gb = _std_tconv.transposed_conv_backward(grad_output, x, weight, bias, *k, *s, *p, *d)
        return gx, gw, gb, None, None, None, None


def convolution(input, weight, bias, kernel_size, stride, padding, dilation):
    return _Convolution.apply(input, weight, bias, kernel_size, stride, padding, dilation)


def transposed_convolution(input, weight, bias, kernel_size, stride, padding, dilation):
    return _TransposedConvolution.apply(input, weight, bias, kernel_size, stride, padding, dilation)


# ---- normalisation and log probabilities (no counterpart in the reference) ---------------------------------------
def rms_norm(input, weight=None, residual=None, eps=1e-6, dim=1):
    """out = s / sqrt(mean(s^2) + eps) * weight with the mean over `dim` (default: the channels of an image batch) and
    s = residual + input, or the input alone.  Returns out, or (out, s) with a residual; both are differentiable.

    float32, bfloat16 or float16; statistics are float32.  s is rounded to that type, as it is returned, before it is
    normalised.  weight (size of dim; float32 or the input's dtype) may be None.  The input is contiguous, or its `dim` has
    stride 1 and its other dimensions are rows of one stride (a slice of wider rows, a channels-last image); the residual lies
    alike.  Squares are summed in float32: magnitudes above 1e18 overflow."""
    args = (input, weight, residual, float(eps), int(dim))
    out = _C.rms_norm_op(*args)
    if out is None:
        out = _by_function(_C.rms_norm_op, args)
    return out[0] if residual is None else tuple(out)


def rms_norm_quantized(input, weight=None, residual=None, eps=1e-6, dim=1):
    """rms_norm with its output in 8 bits: (q, scale), or (q, scale, s) with a residual, where q is float8_e4m3fn and
    q * scale.unsqueeze(dim) the output; scale (float32, the input's size without dim) is the largest magnitude of each
    normalised row / 448, and 0 over a row of zeros.  Forward only (no autograd node)."""
    args = (input, weight, residual, float(eps), int(dim))
    out = _C.rms_norm_quantized(*args)
    if out is None:
        out = _by_function(_C.rms_norm_quantized, args)
    return tuple(out)


class TokenLogProbs(NamedTuple):
    log_probs: torch.Tensor
    entropy: torch.Tensor
    top_log_probs: Optional[torch.Tensor]
    top_indices: Optional[torch.Tensor]


def token_log_probs(logits, target, dim=1, top_k=0, ignore_index=-100):
    """Log probabilities of given classes, over `dim` (default: the channels of an image batch, one label per pixel; -1 for
    rows of tokens), with the entropy of each distribution and its `top_k` most probable classes.

    logits float32, bfloat16 or float16, laid out as for `rms_norm`; target int64, their size without dim.  Results are float32:
    log_probs and entropy of target's size, top_log_probs and (int64) top_indices with top_k in the place of dim, equal
    logits in the order of their indices; None with top_k = 0.  All but the indices are differentiable.  More than 32 of the best
    of rows of more than about 1000 classes cost a pass over the row each, and more than 8 of a pixel's a pass for eight.

    A target equal to ignore_index gives log probability 0 and no gradient, any other outside the classes NaN.  Logits of
    -inf are classes out of the question; where there is no other, log probabilities are -inf, the entropy 0 and the
    gradient 0.  +inf and NaN give NaN."""
    args = (logits, target, int(dim), int(top_k), int(ignore_index))
    out = _C.token_log_probs_op(*args)
    if out is None:
        out = _by_function(_C.token_log_probs_op, args)
    return TokenLogProbs(*out) if top_k else TokenLogProbs(*out, None, None)
