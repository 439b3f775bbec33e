"""The reference's operator API (include/cuvit/kernels.hpp) over the C ABI.

Names, argument order and meaning follow the reference's free functions: launch_gemm,
launch_layer_norm, launch_gelu, launch_softmax, launch_extract_patches, launch_add,
launch_add_broadcast, launch_broadcast; plus launch_attention, the fused replacement of
the Q.K^T -> softmax -> .V sequence. Pointers are device addresses: an int, or any object
with data_ptr() (a torch tensor). Streams are a cudaStream_t as an int, None (the legacy
default stream) or an object with a cuda_stream attribute (torch.cuda.Stream).
"""

from __future__ import annotations

import ctypes
import dataclasses

from . import _lib
from .errors import check

LAYOUT_NO_TRANSPOSE = _lib.LAYOUT_NO_TRANSPOSE
LAYOUT_TRANSPOSED = _lib.LAYOUT_TRANSPOSED
DTYPE_F32 = _lib.DTYPE_F32
DTYPE_BF16 = _lib.DTYPE_BF16
DTYPE_TF32 = _lib.DTYPE_TF32
MATH_FP32 = _lib.MATH_FP32
MATH_TF32 = _lib.MATH_TF32
MATH_BF16 = _lib.MATH_BF16
ROTARY_HALVES = _lib.ROTARY_HALVES
ROTARY_ADJACENT = _lib.ROTARY_ADJACENT
ROTARY_LADDER_AXIS = _lib.ROTARY_LADDER_AXIS
ROTARY_LADDER_SHARED = _lib.ROTARY_LADDER_SHARED
NORM_RMS = _lib.NORM_RMS
NORM_LAYER = _lib.NORM_LAYER
ACTIVATION_NONE = _lib.ACTIVATION_NONE
ACTIVATION_GELU = _lib.ACTIVATION_GELU
ACTIVATION_GELU_TANH = _lib.ACTIVATION_GELU_TANH
ACTIVATION_SILU = _lib.ACTIVATION_SILU


def _ptr(value) -> int | None:
    """A tensor's or an integer's address; plain integers, since wrapping each in a c_void_p costs a
    launch a quarter of a microsecond."""
    if value is None:
        return None
    data_ptr = getattr(value, "data_ptr", None)
    return int(value) if data_ptr is None else data_ptr()


def _stream(stream) -> int | None:
    if stream is None:
        return None
    handle = getattr(stream, "cuda_stream", None)
    return int(stream) if handle is None else handle


@dataclasses.dataclass
class GemmBatch:
    """reference: GemmBatch, include/cuvit/kernels.hpp:46-59."""

    count: int = 1
    stride_a: int = 0
    stride_b: int = 0
    stride_c: int = 0
    inner: int = 0
    outer_stride_a: int = 0
    outer_stride_b: int = 0
    outer_stride_c: int = 0


@dataclasses.dataclass
class GemmEpilogue:
    """reference: GemmEpilogue, include/cuvit/kernels.hpp:30-36."""

    accumulate: bool = False
    gelu: bool = False


@dataclasses.dataclass
class GemmProblem:
    """reference: GemmProblem, include/cuvit/kernels.hpp:74-85."""

    m: int = 0
    n: int = 0
    k: int = 0
    layout: int = LAYOUT_NO_TRANSPOSE
    alpha: float = 1.0
    lda: int = 0
    ldb: int = 0
    ldc: int = 0
    batch: GemmBatch = dataclasses.field(default_factory=GemmBatch)
    epilogue: GemmEpilogue = dataclasses.field(default_factory=GemmEpilogue)

    def to_c(self) -> _lib.GemmProblemC:
        b = self.batch
        return _lib.GemmProblemC(
            self.m, self.n, self.k, self.layout, self.alpha, self.lda, self.ldb, self.ldc,
            _lib.GemmBatchC(b.count, b.stride_a, b.stride_b, b.stride_c, b.inner,
                            b.outer_stride_a, b.outer_stride_b, b.outer_stride_c),
            _lib.GemmEpilogueC(int(self.epilogue.accumulate), int(self.epilogue.gelu)),
        )


def gemm_problem(m: int, n: int, k: int, layout: int) -> GemmProblem:
    """reference: gemm_problem(), include/cuvit/kernels.hpp:89-96."""
    return GemmProblem(m=m, n=n, k=k, layout=layout)


def launch_gemm(a, b, bias, c, problem: GemmProblem, stream=None) -> None:
    """reference: launch_gemm (kernels.hpp:98-99). FP32 operands, process math mode."""
    p = problem.to_c()
    check(_lib.library().cuvit_gemm(_ptr(a), _ptr(b), _ptr(bias), _ptr(c), ctypes.byref(p),
                                    _stream(stream)))


def launch_gemm_ex(a, b, bias, c, problem: GemmProblem, c_dtype: int = DTYPE_F32,
                   math: int = MATH_BF16, stream=None) -> None:
    """Typed GEMM: bf16 operands for MATH_BF16, float otherwise; C in c_dtype."""
    p = problem.to_c()
    check(_lib.library().cuvit_gemm_ex(_ptr(a), _ptr(b), _ptr(bias), _ptr(c), c_dtype, math,
                                       ctypes.byref(p), _stream(stream)))


def set_math_mode(math: int) -> None:
    check(_lib.library().cuvit_set_math_mode(math))


def get_math_mode() -> int:
    return _lib.library().cuvit_get_math_mode()


def launch_layer_norm(input, gamma, beta, output, rows: int, columns: int,
                      epsilon: float = 1.0e-6, stream=None) -> None:
    """reference: launch_layer_norm (kernels.hpp:107-109)."""
    check(_lib.library().cuvit_layer_norm(_ptr(input), _ptr(gamma), _ptr(beta), _ptr(output),
                                          rows, columns, epsilon, _stream(stream)))


def launch_layer_norm_ex(input, input_row_stride: int, gamma, beta, output, out_dtype: int,
                         output_row_stride: int, rows: int, columns: int,
                         epsilon: float = 1.0e-6, stream=None) -> None:
    check(_lib.library().cuvit_layer_norm_ex(_ptr(input), input_row_stride, _ptr(gamma),
                                             _ptr(beta), _ptr(output), out_dtype,
                                             output_row_stride, rows, columns, epsilon,
                                             _stream(stream)))


def launch_gelu(input, output, count: int, stream=None) -> None:
    """reference: launch_gelu (kernels.hpp:117-118)."""
    check(_lib.library().cuvit_gelu(_ptr(input), _ptr(output), count, _stream(stream)))


def launch_softmax(input, output, rows: int, columns: int, stream=None) -> None:
    """reference: launch_softmax (kernels.hpp:122-123)."""
    check(_lib.library().cuvit_softmax(_ptr(input), _ptr(output), rows, columns,
                                       _stream(stream)))


def launch_softmax_ex(input, output, rows: int, columns: int, row_stride: int,
                      stream=None) -> None:
    check(_lib.library().cuvit_softmax_ex(_ptr(input), _ptr(output), rows, columns, row_stride,
                                          _stream(stream)))


def launch_extract_patches(images, patches, batch: int, channels: int, height: int, width: int,
                           patch: int, stream=None) -> None:
    """reference: launch_extract_patches (kernels.hpp:137-138)."""
    check(_lib.library().cuvit_extract_patches(_ptr(images), _ptr(patches), batch, channels,
                                               height, width, patch, _stream(stream)))


def launch_extract_patches_ex(images, patches, out_dtype: int, batch: int, channels: int,
                              height: int, width: int, patch: int, stream=None) -> None:
    check(_lib.library().cuvit_extract_patches_ex(_ptr(images), _ptr(patches), out_dtype, batch,
                                                  channels, height, width, patch,
                                                  _stream(stream)))


def launch_add(accumulator, addend, count: int, stream=None) -> None:
    """reference: launch_add (kernels.hpp:141-142)."""
    check(_lib.library().cuvit_add(_ptr(accumulator), _ptr(addend), count, _stream(stream)))


def launch_add_broadcast(accumulator, addend, count: int, batch: int, stream=None) -> None:
    """reference: launch_add_broadcast (kernels.hpp:147-148)."""
    check(_lib.library().cuvit_add_broadcast(_ptr(accumulator), _ptr(addend), count, batch,
                                             _stream(stream)))


def launch_broadcast(destination, source, count: int, destination_stride: int, batch: int,
                     stream=None) -> None:
    """reference: launch_broadcast (kernels.hpp:153-154)."""
    check(_lib.library().cuvit_broadcast(_ptr(destination), _ptr(source), count,
                                         destination_stride, batch, _stream(stream)))


def launch_init_tokens(tokens, class_token, position, batch: int, tokens_per_image: int,
                       embed: int, stream=None) -> None:
    check(_lib.library().cuvit_init_tokens(_ptr(tokens), _ptr(class_token), _ptr(position),
                                           batch, tokens_per_image, embed, _stream(stream)))


def launch_convert_f32_to_bf16(input, output, count: int, stream=None) -> None:
    check(_lib.library().cuvit_convert_f32_to_bf16(_ptr(input), _ptr(output), count,
                                                   _stream(stream)))


def launch_round_to_tf32(input, output, count: int, stream=None) -> None:
    check(_lib.library().cuvit_round_to_tf32(_ptr(input), _ptr(output), count,
                                             _stream(stream)))


def launch_logits_top_k(logits, indices, values, probabilities, batch: int, classes: int,
                        k: int, stream=None) -> None:
    """reference: report_top (src/main.cpp:90-114) on the device: per row the k largest
    logits (descending; equal logits by ascending class index) with their softmax
    probabilities, into int32 / float32 / float32 arrays [batch, k]."""
    check(_lib.library().cuvit_logits_top_k(_ptr(logits), batch, classes, k, _ptr(indices),
                                            _ptr(values), _ptr(probabilities),
                                            _stream(stream)))


def launch_attention(qkv, context, dtype: int, batch: int, tokens: int, heads: int,
                     head_dim: int, scale: float, stream=None) -> None:
    """Fused Q.K^T -> softmax -> .V (replaces src/model/vit.cu:198-242)."""
    check(_lib.library().cuvit_attention(_ptr(qkv), _ptr(context), dtype, batch, tokens, heads,
                                         head_dim, scale, _stream(stream)))


def launch_preprocess(pixels, tensor, batch: int, width: int, height: int, size: int = 224,
                      crop_fraction: float = 0.9, mean=(0.5, 0.5, 0.5), stddev=(0.5, 0.5, 0.5),
                      image_stride: int = 0, stream=None) -> None:
    """Device preprocessing (replaces cuvit::preprocess, src/runtime/image.cpp:90-135):
    `batch` interleaved uint8 RGB images -> planar float [batch, 3, size, size]."""
    settings = _lib.PreprocessingC(size, crop_fraction, (ctypes.c_float * 3)(*mean),
                                   (ctypes.c_float * 3)(*stddev))
    check(_lib.library().cuvit_preprocess(_ptr(pixels), batch, width, height, image_stride,
                                          ctypes.byref(settings), _ptr(tensor),
                                          _stream(stream)))


# ---- encoder blocks over packed images and videos ------------------------------------------


@dataclasses.dataclass
class QkProblem:
    """cuvit_qk_problem: queries [tokens, q_heads, head_dim] and keys [tokens, k_heads,
    head_dim], strides in elements between tokens (0 = packed)."""

    tokens: int = 0
    q_heads: int = 0
    k_heads: int = 0
    head_dim: int = 0
    dtype: int = DTYPE_BF16
    q_stride: int = 0
    k_stride: int = 0
    q_out_stride: int = 0
    k_out_stride: int = 0
    position_stride: int = 0

    def to_c(self) -> _lib.QkProblemC:
        return _lib.QkProblemC(self.tokens, self.q_heads, self.k_heads, self.head_dim, self.dtype,
                               self.q_stride, self.k_stride, self.q_out_stride,
                               self.k_out_stride, self.position_stride)


@dataclasses.dataclass
class QkNorm:
    """cuvit_qk_norm: per-head norms; gains and offsets are float32 [head_dim] device arrays
    shared by a side's heads, None for 1 and 0."""

    kind: int = NORM_RMS
    epsilon: float = 1.0e-6
    q_gamma: object = None
    q_beta: object = None
    k_gamma: object = None
    k_beta: object = None

    def to_c(self) -> _lib.QkNormC:
        return _lib.QkNormC(self.kind, self.epsilon, _ptr(self.q_gamma), _ptr(self.q_beta),
                            _ptr(self.k_gamma), _ptr(self.k_beta))


@dataclasses.dataclass
class AttentionProblem:
    """cuvit_attention_problem: packed sequences, strides in elements between rows
    (0 = packed)."""

    batch: int = 0
    q_tokens: int = 0
    kv_tokens: int = 0
    q_heads: int = 0
    kv_heads: int = 0
    head_dim: int = 0
    dtype: int = DTYPE_BF16
    causal: bool = False
    scale: float = 1.0
    q_stride: int = 0
    k_stride: int = 0
    v_stride: int = 0
    out_stride: int = 0

    def to_c(self) -> _lib.AttentionProblemC:
        return _lib.AttentionProblemC(self.batch, self.q_tokens, self.kv_tokens, self.q_heads,
                                      self.kv_heads, self.head_dim, self.dtype,
                                      int(self.causal), self.scale, self.q_stride,
                                      self.k_stride, self.v_stride, self.out_stride)


@dataclasses.dataclass
class LinearProblem:
    """cuvit_linear_problem: x [m, k], weight [n, k] (gated: [2n, k], gate rows first)."""

    m: int = 0
    n: int = 0
    k: int = 0
    math: int = MATH_BF16
    out_dtype: int = DTYPE_BF16
    activation: int = ACTIVATION_NONE
    gated: bool = False
    ldx: int = 0
    ldw: int = 0
    ldr: int = 0
    ldo: int = 0

    def to_c(self) -> _lib.LinearProblemC:
        return _lib.LinearProblemC(self.m, self.n, self.k, self.math, self.out_dtype,
                                   self.activation, int(self.gated), self.ldx, self.ldw, self.ldr,
                                   self.ldo)


def rotary_axes(sections, base: float = 10000.0, pairing: int = ROTARY_HALVES,
                ladder: int = ROTARY_LADDER_AXIS) -> _lib.RotaryC:
    """The rotation plan of position axes turning sections[a] pairs each, made once and passed
    to launch_rotary / launch_qk_norm_rotary."""
    rotary = _lib.RotaryC()
    sections = list(sections)
    check(_lib.library().cuvit_rotary_init(ctypes.byref(rotary), len(sections),
                                           (ctypes.c_int * len(sections))(*sections), base,
                                           pairing, ladder))
    return rotary


def _optional(value):
    return None if value is None else ctypes.byref(value)


def launch_rotary(q, k, q_out, k_out, positions, rotary: _lib.RotaryC, problem: QkProblem,
                  stream=None) -> None:
    """Turns query and key pairs by their positions (int32 [axes, tokens])."""
    p = problem.to_c()
    check(_lib.library().cuvit_rotary_qk(_ptr(q), _ptr(k), _ptr(q_out), _ptr(k_out),
                                         _ptr(positions), _optional(rotary), ctypes.byref(p),
                                         _stream(stream)))


def launch_qk_norm_rotary(q, k, q_out, k_out, norm: QkNorm, positions,
                          rotary: _lib.RotaryC | None, problem: QkProblem, stream=None) -> None:
    """Per-head norms of queries and keys, then (rotary not None) the rotation, in one pass."""
    p = problem.to_c()
    n = norm.to_c()
    check(_lib.library().cuvit_qk_norm_rotary(_ptr(q), _ptr(k), _ptr(q_out), _ptr(k_out),
                                              ctypes.byref(n), _ptr(positions),
                                              _optional(rotary), ctypes.byref(p),
                                              _stream(stream)))


def attention_varlen_workspace(problem: AttentionProblem) -> int:
    """Bytes of workspace with which launch_attention_varlen may split long key ranges (0: the
    problem is not split)."""
    p = problem.to_c()
    size = ctypes.c_size_t(0)
    check(_lib.library().cuvit_attention_varlen_workspace(ctypes.byref(p), ctypes.byref(size)))
    return size.value


def launch_attention_varlen(q, k, v, out, q_offsets, kv_offsets, problem: AttentionProblem,
                            workspace=None, workspace_bytes: int = 0, stream=None) -> None:
    """Attention over packed sequences given by int32 device offsets [batch + 1]; kv_offsets
    None: the queries' own."""
    p = problem.to_c()
    check(_lib.library().cuvit_attention_varlen(_ptr(q), _ptr(k), _ptr(v), _ptr(out),
                                                _ptr(q_offsets), _ptr(kv_offsets),
                                                ctypes.byref(p), _ptr(workspace),
                                                workspace_bytes, _stream(stream)))


def launch_linear(x, weight, bias, scale, residual, out, problem: LinearProblem,
                  stream=None) -> None:
    """out = residual + scale * activation(x weight^T + bias), with a gate when gated; bias,
    scale and residual may be None."""
    p = problem.to_c()
    check(_lib.library().cuvit_linear(_ptr(x), _ptr(weight), _ptr(bias), _ptr(scale),
                                      _ptr(residual), _ptr(out), ctypes.byref(p),
                                      _stream(stream)))


def device_status() -> int:
    """Synchronises the current device, returns and clears its status bits (raises on a
    device-side timeout)."""
    flags = ctypes.c_uint(0)
    check(_lib.library().cuvit_device_status(ctypes.byref(flags)))
    return flags.value


def launch_count() -> int:
    return int(_lib.library().cuvit_launch_count())
