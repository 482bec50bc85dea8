"""``turing_utils::*`` custom ops of the linear path.

Same op names, schemas, Python-side checks and fake (meta) implementations as
the reference (kernel/comfyui_turing_utils_kernel/ops.py:8-352), so
``torch.compile(fullgraph=True)`` treats them as leaves and the plugin's
dispatcher calls them unchanged.  The CUDA implementations run the sm_100a
kernels of libturing_b200.so through ``_C``.
"""
from __future__ import annotations

import math

import torch
import torch.autograd.forward_ad as forward_ad
from torch.utils._python_dispatch import is_in_torch_dispatch_mode

from . import _C


def _require_cuda(t: torch.Tensor, what: str) -> None:
    if t.device.type != "cuda":
        raise RuntimeError(f"{what} requires CUDA tensors")
    if torch.cuda.get_device_capability(t.device)[0] != 10:
        raise RuntimeError(f"{what} requires an sm_100 (B200) device for this build")


@torch.library.custom_op("turing_utils::w4a8_linear", mutates_args=())
def turing_w4a8_linear(
    activation: torch.Tensor,
    weight: torch.Tensor,
    activation_scale: torch.Tensor,
    weight_scale: torch.Tensor,
    bias: torch.Tensor | None = None,
) -> torch.Tensor:
    """Signed-nibble W4A8 linear (ops.py:8-26)."""
    _require_cuda(activation, "Turing W4A8")
    return _C.turing_w4a8_linear(
        activation.contiguous(), weight.contiguous(), activation_scale.contiguous(),
        weight_scale.contiguous(), None if bias is None else bias.contiguous())


@turing_w4a8_linear.register_fake
def _w4a8_fake(activation, weight, activation_scale, weight_scale, bias=None):
    return torch.empty((activation.size(0), weight.size(0)), dtype=torch.bfloat16,
                       device=activation.device)


@torch.library.custom_op("turing_utils::int4_linear", mutates_args=())
def turing_int4_linear(
    activation: torch.Tensor,
    weight: torch.Tensor,
    activation_scale: torch.Tensor,
    weight_scale: torch.Tensor,
    bias: torch.Tensor | None = None,
) -> torch.Tensor:
    """W4A4 linear on packed INT4 ConvRot activations (no counterpart in the
    reference package: the plugin calls comfy-kitchen's int4_linear there,
    comfyui_turing_utils/quantization/dispatch.py:791-804)."""
    _require_cuda(activation, "Turing W4A4")
    return _C.turing_int4_linear(
        activation.contiguous(), weight.contiguous(), activation_scale.contiguous(),
        weight_scale.contiguous(), None if bias is None else bias.contiguous())


@turing_int4_linear.register_fake
def _int4_fake(activation, weight, activation_scale, weight_scale, bias=None):
    return torch.empty((activation.size(0), weight.size(0)), dtype=torch.bfloat16,
                       device=activation.device)


@torch.library.custom_op("turing_utils::codebook_w4a8_linear", mutates_args=())
def turing_codebook_w4a8_linear(
    activation: torch.Tensor,
    weight: torch.Tensor,
    activation_scale: torch.Tensor,
    group_scale: torch.Tensor,
    channel_scale: torch.Tensor,
    codebook: torch.Tensor,
    bias: torch.Tensor | None = None,
    group_size: int = 16,
    chunk_rows: int = 0,
) -> torch.Tensor:
    """Grouped-codebook W4A8 (ops.py:38-74).  ``chunk_rows`` bounds the staged
    decode workspace (0 = production policy)."""
    _require_cuda(activation, "Turing codebook W4A8")
    if group_scale.dtype == torch.float8_e4m3fn:
        group_scale = group_scale.view(torch.uint8)
    if group_scale.dtype != torch.uint8:
        raise TypeError("group_scale must be float8_e4m3fn or its raw uint8 view")
    return _C.turing_codebook_w4a8_linear(
        activation.contiguous(), weight.contiguous(), activation_scale.contiguous(),
        group_scale.contiguous(), channel_scale.contiguous(), codebook.contiguous(),
        None if bias is None else bias.contiguous(), group_size, chunk_rows)


@turing_codebook_w4a8_linear.register_fake
def _codebook_fake(activation, weight, activation_scale, group_scale, channel_scale, codebook,
                   bias=None, group_size=16, chunk_rows=0):
    return torch.empty((activation.size(0), weight.size(0)), dtype=torch.bfloat16,
                       device=activation.device)


@torch.library.custom_op("turing_utils::int8_linear", mutates_args=())
def turing_int8_linear(
    activation: torch.Tensor,
    weight: torch.Tensor,
    activation_scale: torch.Tensor,
    weight_scale: torch.Tensor,
    bias: torch.Tensor | None = None,
) -> torch.Tensor:
    """W8A8 contraction with the fused dequant/bias/bf16 epilogue (ops.py:96-126)."""
    _require_cuda(activation, "Turing INT8 linear")
    return _C.turing_int8_linear(activation.contiguous(), weight.contiguous(),
                                 activation_scale.contiguous(), weight_scale.contiguous(),
                                 None if bias is None else bias.contiguous())


@turing_int8_linear.register_fake
def _int8_linear_fake(activation, weight, activation_scale, weight_scale, bias=None):
    return torch.empty((activation.size(0), weight.size(0)), dtype=torch.bfloat16,
                       device=activation.device)


@torch.library.custom_op("turing_utils::int8_gemm_s32", mutates_args=())
def turing_int8_gemm_s32(activation: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """Exact INT32 accumulators (feeds turing_dequantize_int8_bf16)."""
    _require_cuda(activation, "Turing INT8 GEMM")
    return _C.turing_int8_gemm_s32(activation.contiguous(), weight.contiguous())


@turing_int8_gemm_s32.register_fake
def _int8_gemm_s32_fake(activation, weight):
    return torch.empty((activation.size(0), weight.size(0)), dtype=torch.int32,
                       device=activation.device)


@torch.library.custom_op("turing_utils::dequantize_int8_bf16", mutates_args=())
def turing_dequantize_int8_bf16(
    accumulator: torch.Tensor,
    activation_scale: torch.Tensor,
    weight_scale: torch.Tensor,
    output_columns: int = -1,
) -> torch.Tensor:
    """Dequantize an INT32 GEMM workspace directly into packed BF16 stores."""
    _require_cuda(accumulator, "Turing BF16 epilogue")
    if accumulator.dtype != torch.int32 or accumulator.ndim != 2:
        raise TypeError("accumulator must be a 2D int32 tensor")
    return _C.turing_dequantize_int8_bf16(accumulator.contiguous(), activation_scale.contiguous(),
                                          weight_scale.contiguous(), output_columns)


@turing_dequantize_int8_bf16.register_fake
def _dequant_fake(accumulator, activation_scale, weight_scale, output_columns=-1):
    columns = accumulator.size(1) if output_columns < 0 else output_columns
    return torch.empty((accumulator.size(0), columns), dtype=torch.bfloat16,
                       device=accumulator.device)


def _staged_op(name, doc, width_div, int4):
    @torch.library.custom_op(f"turing_utils::{name}", mutates_args=())
    def op(x: torch.Tensor, group_size: int = 256) -> tuple[torch.Tensor, torch.Tensor]:
        _require_cuda(x, doc)
        if x.dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"{doc} input must be float16 or bfloat16")
        if x.ndim != 2:
            raise ValueError(f"{doc} input must be 2D")
        return getattr(_C, f"turing_{name}")(x.contiguous(), group_size)

    @op.register_fake
    def _fake(x, group_size=256):
        hidden = x.size(1) // width_div
        return (torch.empty((x.size(0), hidden // 2 if int4 else hidden), dtype=torch.int8,
                            device=x.device),
                torch.empty((x.size(0), 1), dtype=torch.float32, device=x.device))

    return op


turing_swiglu_int8_convrot_quantize = _staged_op(
    "swiglu_int8_convrot_quantize", "Turing SwiGLU ConvRot", 2, False)
turing_swiglu_int4_convrot_quantize = _staged_op(
    "swiglu_int4_convrot_quantize", "Turing SwiGLU INT4 ConvRot", 2, True)
turing_gelu_int8_convrot_quantize = _staged_op(
    "gelu_int8_convrot_quantize", "Turing GELU ConvRot", 1, False)
turing_gelu_int4_convrot_quantize = _staged_op(
    "gelu_int4_convrot_quantize", "Turing GELU INT4 ConvRot", 1, True)


@torch.library.custom_op("turing_utils::bf16_int8_convrot_quantize", mutates_args=())
def turing_bf16_int8_convrot_quantize(
    x: torch.Tensor,
    group_size: int = 256,
    *,
    swiglu: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Whole-row BF16 ConvRot INT8 quantization (ops.py:257-273)."""
    _require_cuda(x, "BF16 row-buffer ConvRot")
    if x.dtype != torch.bfloat16:
        raise TypeError("BF16 row-buffer ConvRot input must be bfloat16")
    if x.ndim != 2:
        raise ValueError("BF16 row-buffer ConvRot input must be 2D")
    return _C.turing_bf16_int8_convrot_quantize(x.contiguous(), group_size, swiglu)


@turing_bf16_int8_convrot_quantize.register_fake
def _bf16_int8_fake(x, group_size=256, *, swiglu=False):
    hidden = x.size(1) // 2 if swiglu else x.size(1)
    return (torch.empty((x.size(0), hidden), dtype=torch.int8, device=x.device),
            torch.empty((x.size(0), 1), dtype=torch.float32, device=x.device))


@torch.library.custom_op("turing_utils::bf16_int4_convrot_quantize", mutates_args=())
def turing_bf16_int4_convrot_quantize(
    x: torch.Tensor,
    group_size: int = 256,
    *,
    swiglu: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Whole-row BF16 ConvRot INT4 quantization (ops.py:285-301)."""
    _require_cuda(x, "BF16 row-buffer INT4 ConvRot")
    if x.dtype != torch.bfloat16:
        raise TypeError("BF16 row-buffer INT4 ConvRot input must be bfloat16")
    if x.ndim != 2:
        raise ValueError("BF16 row-buffer INT4 ConvRot input must be 2D")
    return _C.turing_bf16_int4_convrot_quantize(x.contiguous(), group_size, swiglu)


@turing_bf16_int4_convrot_quantize.register_fake
def _bf16_int4_fake(x, group_size=256, *, swiglu=False):
    hidden = x.size(1) // 2 if swiglu else x.size(1)
    return (torch.empty((x.size(0), hidden // 2), dtype=torch.int8, device=x.device),
            torch.empty((x.size(0), 1), dtype=torch.float32, device=x.device))


@torch.library.custom_op("turing_utils::bf16_gelu_int8_convrot_quantize", mutates_args=())
def turing_bf16_gelu_int8_convrot_quantize(
    x: torch.Tensor,
    group_size: int = 256,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Whole-row BF16 tanh-GELU + ConvRot INT8 quantization."""
    _require_cuda(x, "BF16 GELU ConvRot")
    if x.dtype != torch.bfloat16 or x.ndim != 2:
        raise TypeError("BF16 GELU ConvRot input must be a 2D bfloat16 tensor")
    return _C.turing_bf16_gelu_int8_convrot_quantize(x.contiguous(), group_size)


@turing_bf16_gelu_int8_convrot_quantize.register_fake
def _bf16_gelu_int8_fake(x, group_size=256):
    return (torch.empty(x.shape, dtype=torch.int8, device=x.device),
            torch.empty((x.size(0), 1), dtype=torch.float32, device=x.device))


@torch.library.custom_op("turing_utils::bf16_gelu_int4_convrot_quantize", mutates_args=())
def turing_bf16_gelu_int4_convrot_quantize(
    x: torch.Tensor,
    group_size: int = 256,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Whole-row BF16 tanh-GELU + ConvRot INT4 quantization."""
    _require_cuda(x, "BF16 GELU INT4 ConvRot")
    if x.dtype != torch.bfloat16 or x.ndim != 2:
        raise TypeError("BF16 GELU INT4 ConvRot input must be a 2D bfloat16 tensor")
    return _C.turing_bf16_gelu_int4_convrot_quantize(x.contiguous(), group_size)


@turing_bf16_gelu_int4_convrot_quantize.register_fake
def _bf16_gelu_int4_fake(x, group_size=256):
    return (torch.empty((x.size(0), x.size(1) // 2), dtype=torch.int8, device=x.device),
            torch.empty((x.size(0), 1), dtype=torch.float32, device=x.device))


@torch.library.custom_op("turing_utils::segmented_rms_adaln", mutates_args=())
def turing_segmented_rms_adaln(
    x: torch.Tensor,
    weight: torch.Tensor,
    scale: torch.Tensor,
    shift: torch.Tensor,
    segments: torch.Tensor,
    epsilon: float = 1.0e-5,
) -> torch.Tensor:
    """Fused affine RMSNorm and segmented AdaLN modulation (ops.py:355-396)."""
    if x.device.type != "cuda":
        raise RuntimeError("Segmented RMSNorm+AdaLN requires CUDA tensors")
    _require_cuda(x, "Segmented RMSNorm+AdaLN")
    if x.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise TypeError("segmented RMSNorm+AdaLN input must be float16, bfloat16, or float32")
    if x.ndim != 2:
        raise ValueError("segmented RMSNorm+AdaLN input must be 2D [M, K]")
    if weight.device != x.device or scale.device != x.device or shift.device != x.device:
        raise ValueError("weight, scale, and shift must be on the input device")
    weight = weight.to(dtype=x.dtype).contiguous()
    scale = scale.to(dtype=x.dtype)
    shift = shift.to(dtype=x.dtype)
    if scale.stride(-1) != 1:
        scale = scale.contiguous()
    if shift.stride(-1) != 1:
        shift = shift.contiguous()
    if segments.device != x.device or segments.dtype != torch.int32:
        raise ValueError("segments must be an int32 tensor on the input device")
    return _C.turing_segmented_rms_adaln(x.contiguous(), weight, scale, shift,
                                         segments.contiguous(), epsilon)


@turing_segmented_rms_adaln.register_fake
def _segmented_rms_adaln_fake(x, weight, scale, shift, segments, epsilon=1.0e-5):
    return torch.empty_like(x)


@torch.library.custom_op("turing_utils::layer_norm_adaln", mutates_args=())
def turing_layer_norm_adaln(
    x: torch.Tensor,
    scale: torch.Tensor,
    shift: torch.Tensor,
    epsilon: float = 1.0e-5,
) -> torch.Tensor:
    """Fused FP32-statistics LayerNorm and Wan AdaLN modulation (ops.py:399-418)."""
    if x.device.type != "cuda":
        raise RuntimeError("LayerNorm+AdaLN requires a CUDA tensor")
    _require_cuda(x, "LayerNorm+AdaLN")
    if x.dtype not in (torch.float16, torch.bfloat16, torch.float32) or x.ndim != 3:
        raise TypeError("LayerNorm+AdaLN input must be 3D float16, bfloat16, or float32")
    scale = scale.to(device=x.device, dtype=x.dtype).contiguous()
    shift = shift.to(device=x.device, dtype=x.dtype).contiguous()
    return _C.turing_layer_norm_adaln(x.contiguous(), scale, shift, epsilon)


@turing_layer_norm_adaln.register_fake
def _layer_norm_adaln_fake(x, scale, shift, epsilon=1.0e-5):
    return torch.empty_like(x)


# ----------------------------------------------------------- rotary positions

def turing_rope_inv_freq(
    rot_dim: int,
    theta: float = 10000.0,
    *,
    axis_pairs: list[int] | None = None,
    scaling: str = "none",
    factor: float = 1.0,
    original_length: int = 0,
    beta_fast: float = 32.0,
    beta_slow: float = 1.0,
    device: torch.device | str | None = None,
) -> tuple[torch.Tensor, float]:
    """Rotary frequencies, fp64 [rot_dim / 2], and the scale to rotate with.

    Pair i of an axis of n pairs (one axis without axis_pairs) turns by
    theta^(-i / n) per position.  For contexts `factor` times as long as trained:
      "linear"  divides every frequency by factor;
      "ntk"     raises theta to theta * factor^(n / (n - 1)), which keeps the
                fastest frequency and divides the slowest by factor;
      "yarn"    divides the frequencies that turn less than beta_slow times in
                original_length tokens, keeps those above beta_fast turns (and always
                the first), blends linearly in the pair index between, and scales by
                0.1 ln(factor) + 1.
    Otherwise the scale is 1.
    """
    if rot_dim <= 0 or rot_dim % 2:
        raise ValueError("rot_dim must be positive and even")
    if not (math.isfinite(theta) and theta > 1.0):
        raise ValueError("theta must be finite and larger than 1")
    if scaling not in {"none", "linear", "ntk", "yarn"}:
        raise ValueError(f"Unknown rotary scaling: {scaling}")
    if not (math.isfinite(factor) and factor >= 1.0):
        raise ValueError("factor must be finite and at least 1")
    if scaling == "yarn" and (original_length <= 0 or not beta_fast > beta_slow > 0.0):
        raise ValueError("yarn needs original_length > 0 and beta_fast > beta_slow > 0")
    parts = [rot_dim // 2] if axis_pairs is None else [int(n) for n in axis_pairs]
    if min(parts, default=-1) < 0 or sum(parts) != rot_dim // 2:
        raise ValueError("axis_pairs must add up to rot_dim / 2")
    freqs = []
    for n in parts:
        i = torch.arange(n, dtype=torch.float64)
        base = theta * factor ** (n / (n - 1)) if scaling == "ntk" and n > 1 else theta
        f = base ** (-i / max(n, 1))
        if scaling == "linear":
            f = f / factor
        elif scaling == "yarn":
            def pair_of(turns):  # the pair that turns this often in original_length
                return n * math.log(original_length / (turns * 2.0 * math.pi)) / math.log(theta)
            low = max(math.floor(pair_of(beta_fast)), 0)
            # Pairs are counted in 2 n channels: the ramp may end past the last one.
            high = min(math.ceil(pair_of(beta_slow)), 2 * n - 1)
            slow = ((i - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
            f = f * (1.0 - slow) + f / factor * slow
        freqs.append(f)
    scale = 0.1 * math.log(factor) + 1.0 if scaling == "yarn" else 1.0
    return torch.cat(freqs).to(device), scale


def _refuse_tangents(*tensors):
    """A registered op has no forward-mode rule and would drop the tangent."""
    if forward_ad._current_level >= 0 and any(
            forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("the registered rotary ops have no forward-mode derivative; call "
                           "turing_rope or turing_rope_qk")


@torch.library.custom_op("turing_utils::rope", mutates_args=())
def _rope_op(
    x: torch.Tensor,
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    tensor_layout: str = "HND",
    split_half: bool = False,
    axis_pairs: list[int] | None = None,
    scale: float = 1.0,
    inverse: bool = False,
) -> torch.Tensor:
    _require_cuda(x, "Rotary positions")
    _refuse_tangents(x)
    return _C.turing_rope(x, None, positions, inv_freq, tensor_layout, split_half, axis_pairs,
                          scale, inverse)[0]


@_rope_op.register_fake
def _rope_fake(x, positions, inv_freq, tensor_layout="HND", split_half=False, axis_pairs=None,
               scale=1.0, inverse=False):
    return torch.empty(x.shape, dtype=x.dtype, device=x.device)


@torch.library.custom_op("turing_utils::rope_qk", mutates_args=())
def _rope_qk_op(
    query: torch.Tensor,
    key: torch.Tensor,
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    tensor_layout: str = "HND",
    split_half: bool = False,
    axis_pairs: list[int] | None = None,
    scale: float = 1.0,
    inverse: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    _require_cuda(query, "Rotary positions")
    _refuse_tangents(query, key)
    return _C.turing_rope(query, key, positions, inv_freq, tensor_layout, split_half, axis_pairs,
                          scale, inverse)


@_rope_qk_op.register_fake
def _rope_qk_fake(query, key, positions, inv_freq, tensor_layout="HND", split_half=False,
                  axis_pairs=None, scale=1.0, inverse=False):
    return (torch.empty(query.shape, dtype=query.dtype, device=query.device),
            torch.empty(key.shape, dtype=key.dtype, device=key.device))


def _rope_setup(ctx, inputs, output):
    tensors = len(inputs) - 7
    ctx.save_for_backward(*inputs[tensors:tensors + 2])
    ctx.options = inputs[tensors + 2:]


def _rope_grad_args(ctx):
    layout, split_half, axis_pairs, scale, inverse = ctx.options
    return (*ctx.saved_tensors, layout, split_half, axis_pairs, scale, not inverse)


def _rope_backward(ctx, grad):
    return (_rope_op(grad, *_rope_grad_args(ctx)), *(None,) * 7)


def _rope_qk_backward(ctx, grad_query, grad_key):
    args = _rope_grad_args(ctx)
    need_q = ctx.needs_input_grad[0] and grad_query is not None
    need_k = ctx.needs_input_grad[1] and grad_key is not None
    if need_q and need_k:
        return (*_rope_qk_op(grad_query, grad_key, *args), *(None,) * 7)
    return (_rope_op(grad_query, *args) if need_q else None,
            _rope_op(grad_key, *args) if need_k else None, *(None,) * 7)


_rope_op.register_autograd(_rope_backward, setup_context=_rope_setup)
_rope_qk_op.register_autograd(_rope_qk_backward, setup_context=_rope_setup)


# Eager calls on plain CUDA tensors skip the custom op's dispatcher, which costs
# more than a small launch (one token: 68 us a call through it against 21, with
# its gradients 289 against 140): without gradients they reach the binding, with
# gradients by way of an autograd function.  Tracing (torch.compile, torch.jit,
# fake and subclass tensors, dispatch modes) sees the custom op.  Function
# transforms (torch.func, torch.vmap) and forward-mode differentiation, whose
# wrapped tensors have the plain type, go through _RopeTransformed.

_PLAIN = (torch.Tensor, torch.nn.Parameter)


_function_transforms_active = torch._C._are_functorch_transforms_active
_jit_tracing = torch._C._is_tracing


def _transformed() -> bool:
    return _function_transforms_active() or forward_ad._current_level >= 0


def _eager(*tensors: torch.Tensor) -> bool:
    if (torch.compiler.is_compiling() or is_in_torch_dispatch_mode() or _transformed()
            or _jit_tracing()):
        return False
    return all(type(t) in _PLAIN and t.is_cuda for t in tensors)


class _RopeFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, positions, inv_freq, options):
        ctx.save_for_backward(positions, inv_freq)
        ctx.set_materialize_grads(False)
        ctx.options = options
        query, key = _C.turing_rope(query, key, positions, inv_freq, *options)
        return query if key is None else (query, key)

    @staticmethod
    def backward(ctx, grad_query, grad_key=None):
        positions, inv_freq = ctx.saved_tensors
        options = (*ctx.options[:-1], not ctx.options[-1])
        if not ctx.needs_input_grad[0]:
            grad_query = None
        if not ctx.needs_input_grad[1]:
            grad_key = None
        if grad_query is None:
            if grad_key is not None:
                grad_key = _rope_call(grad_key, None, positions, inv_freq, options)
        elif grad_key is None:
            grad_query = _rope_call(grad_query, None, positions, inv_freq, options)
        else:
            grad_query, grad_key = _rope_call(grad_query, grad_key, positions, inv_freq, options)
        return grad_query, grad_key, None, None, None


class _Options:
    """Options of a call as one opaque argument (a tuple would be taken apart)."""

    def __init__(self, values):
        self.values = values


def _rope_registered(query, key, positions, inv_freq, options):
    if key is None:
        return _rope_op(query, positions, inv_freq, *options)
    return _rope_qk_op(query, key, positions, inv_freq, *options)


class _RopeTransformed(torch.autograd.Function):
    """The rotation under function transforms: linear in query and key, so the
    tangent is the rotated tangent; batched by the registered ops' rule."""

    generate_vmap_rule = True

    @staticmethod
    def forward(query, key, positions, inv_freq, options):
        return _rope_registered(query, key, positions, inv_freq, options.values)

    @staticmethod
    def setup_context(ctx, inputs, output):
        _, key, positions, inv_freq, options = inputs
        ctx.save_for_backward(positions, inv_freq)
        ctx.save_for_forward(positions, inv_freq)
        ctx.pair, ctx.options = key is not None, options

    @staticmethod
    def backward(ctx, grad_query, grad_key=None):
        values = ctx.options.values
        back = _Options((*values[:-1], not values[-1]))
        grads = _RopeTransformed.apply(grad_query, grad_key, *ctx.saved_tensors, back)
        return (*(grads if ctx.pair else (grads, None)), None, None, None)

    @staticmethod
    def jvp(ctx, query, key, *_):
        return _RopeTransformed.apply(query, key, *ctx.saved_tensors, ctx.options)


def _rope_call(query, key, positions, inv_freq, options):
    if _eager(query, positions, inv_freq) if key is None else _eager(query, key, positions,
                                                                     inv_freq):
        if torch.is_grad_enabled() and (query.requires_grad
                                        or (key is not None and key.requires_grad)):
            return _RopeFunction.apply(query, key, positions, inv_freq, options)
        rotated = _C.turing_rope(query, key, positions, inv_freq, *options)
        return rotated[0] if key is None else rotated
    if not torch.compiler.is_compiling() and _transformed():
        return _RopeTransformed.apply(query, key, positions, inv_freq, _Options(options))
    return _rope_registered(query, key, positions, inv_freq, options)


def _options(tensor_layout, split_half, axis_pairs, scale, inverse):
    # A list of its own: the gradients use it after the caller may have changed theirs.
    return (tensor_layout, split_half, None if axis_pairs is None else list(axis_pairs),
            float(scale), inverse)


def turing_rope(
    x: torch.Tensor,
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    *,
    tensor_layout: str = "HND",
    split_half: bool = False,
    axis_pairs: list[int] | None = None,
    scale: float = 1.0,
    inverse: bool = False,
) -> torch.Tensor:
    """Rotary positions on x [B, H, L, D] (HND) or [B, L, H, D] (NHD), float16,
    bfloat16 or float32, differentiable in x.

    The first 2 * len(inv_freq) channels of each head turn; the others are
    copied.  Pair p, channels (2p, 2p + 1) or with split_half (p, p + pairs),
    turns by position * inv_freq[p] (the angle is taken in fp64) and is
    multiplied by scale.  positions: int32, int64, float32 or float64, within 2^51
    in magnitude as their products with inv_freq, [L] or [1 or B, L]; with axis_pairs (pairs of each of 1 to 4 axes)
    [L, axes] or [1 or B, L, axes].  inverse turns the other way.  No gradients
    reach positions and inv_freq.  To capture a backward pass into a CUDA graph,
    take leaves that no live eager graph holds (torch raises an error otherwise).
    """
    return _rope_call(x, None, positions, inv_freq, _options(
        tensor_layout, split_half, axis_pairs, scale, inverse))


def turing_rope_qk(
    query: torch.Tensor,
    key: torch.Tensor,
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    *,
    tensor_layout: str = "HND",
    split_half: bool = False,
    axis_pairs: list[int] | None = None,
    scale: float = 1.0,
    inverse: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """turing_rope of query and key (same batch, length and head dimension, any
    head counts) in one launch, differentiable in both."""
    return _rope_call(query, key, positions, inv_freq, _options(
        tensor_layout, split_half, axis_pairs, scale, inverse))


@torch.library.custom_op("turing_utils::rope_freqs", mutates_args=())
def _rope_freqs_op(
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    axis_pairs: list[int] | None,
    scale: float,
    dtype: torch.dtype,
) -> torch.Tensor:
    _require_cuda(positions, "Rotary positions")
    return _C.turing_rope_freqs(positions, inv_freq, axis_pairs, scale, dtype)


@_rope_freqs_op.register_fake
def _rope_freqs_fake(positions, inv_freq, axis_pairs, scale, dtype):
    lead = positions.shape if axis_pairs is None else positions.shape[:-1]
    batch, length = (1, lead[0]) if len(lead) == 1 else lead
    return torch.empty((batch, length, 1, inv_freq.size(0), 2, 2), dtype=dtype,
                       device=positions.device)


def turing_rope_freqs(
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    *,
    axis_pairs: list[int] | None = None,
    scale: float = 1.0,
    dtype: torch.dtype = torch.bfloat16,
) -> torch.Tensor:
    """The rotations of turing_rope as matrices scale * [[cos, -sin], [sin, cos]],
    [1 or B, L, 1, len(inv_freq), 2, 2] (B up to 65535): the freqs argument of
    turing_sage.prequantize_rms_rope_qk."""
    if _eager(positions, inv_freq):
        return _C.turing_rope_freqs(positions, inv_freq, axis_pairs, float(scale), dtype)
    return _rope_freqs_op(positions, inv_freq, axis_pairs, float(scale), dtype)
