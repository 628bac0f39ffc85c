"""B200-native (sm_100a) W8A8 / FP8 linear family with the reference's
operator interface, the low-rank adapters that run beside it, and what training
them needs: their gradients, the linear's input gradient, and activations kept
in 8 bits.

The operators load libw8a8.so on first use and raise if it is missing (there
is no fallback).  Importing the package itself does not load the library, so
`imagine_b200.build` can run on a checkout that has not been built yet.
"""
_OPS = (
    "dequantize_int8_linear",
    "device_error",
    "fp8_linear",
    "int8_gemm_s32",
    "int8_gemv",
    "int8_linear",
    "int8_linear_host",
    "quantize_int8_rowwise",
    "quantize_int8_rowwise_convrot",
    "quantize_int8_rowwise_modulated",
    "int8_linear_modulated",
    "int8_linear_rms_modulated",
    "adaln_int8_linear",
    "rms_rope",
    "int8_linear_rms_rope",
    "rope_freqs_rows",
    "pack_weight_tiles",
    "TiledInt8Weight",
    "quantize_per_tensor_fp8",
    "quantize_weight",
    "row_absmax",
    "quantize_int8_rowwise_given_absmax",
    "quantize_mxfp8",
    "mxfp8_linear",
)

_ADAPTER_OPS = (
    "int8_linear_backward",
    "int8_linear_lora",
    "lora_add",
    "lora_backward",
)

_ACTIVATION_OPS = (
    "act_backward_int8",
    "act_checkpoint_int8",
    "checkpointed_activation",
)

__all__ = [*_OPS, *_ADAPTER_OPS, *_ACTIVATION_OPS]


def __getattr__(name):
    if name in _OPS:
        from . import linear as module
    elif name in _ADAPTER_OPS:
        from . import adapters as module
    elif name in _ACTIVATION_OPS:
        from . import activation as module
    else:
        raise AttributeError(name)
    value = globals()[name] = getattr(module, name)  # later look-ups skip this function
    return value
