"""The operators over packed images and videos on the CPU: what their entry points refuse, on the
host and before any launch, and what they take as a no-op; and the rotary plan's numbers."""

from __future__ import annotations

import math
import pathlib
import subprocess

import numpy as np
import pytest

from cuvit import _lib, kernels
from cuvit.errors import InvalidArgument, LengthError
from cuvit.kernels import AttentionProblem, LinearProblem, QkNorm, QkProblem

FAKE = 0x10000  # never dereferenced: validation fails first
FAR = 0x40000000


def qk(**changes):
    values = dict(tokens=4, q_heads=2, k_heads=2, head_dim=8, dtype=kernels.DTYPE_F32)
    return QkProblem(**{**values, **changes})


def attention(**changes):
    values = dict(batch=2, q_tokens=8, kv_tokens=8, q_heads=4, kv_heads=2, head_dim=8,
                  dtype=kernels.DTYPE_F32, scale=0.5)
    return AttentionProblem(**{**values, **changes})


def linear(**changes):
    values = dict(m=4, n=8, k=16, math=kernels.MATH_FP32, out_dtype=kernels.DTYPE_F32)
    return LinearProblem(**{**values, **changes})


@pytest.mark.parametrize("ladder", [kernels.ROTARY_LADDER_AXIS, kernels.ROTARY_LADDER_SHARED])
def test_rotary_rates(ladder):
    sections, base = [3, 0, 5], 10000.0
    rotary = kernels.rotary_axes(sections, base, kernels.ROTARY_ADJACENT, ladder)
    assert (rotary.axes, rotary.pairing) == (3, kernels.ROTARY_ADJACENT)
    assert list(rotary.first) == [0, 3, 3, 8, 8]
    for axis, pairs in enumerate(sections):
        for j in range(pairs):
            i = rotary.first[axis] + j
            exponent = j / pairs if ladder == kernels.ROTARY_LADDER_AXIS else i / 8
            want = base ** -exponent / (2 * math.pi)
            # The rate in turns, to a double's accuracy (pow: a few half steps of 2^-53).
            assert rotary.turns[i] / 2.0 ** 64 == pytest.approx(want, rel=1e-15)


@pytest.mark.parametrize("sections,base,pairing,ladder", [
    ([], 10000.0, 0, 0), ([1] * 5, 10000.0, 0, 0), ([0, 0], 10000.0, 0, 0), ([-1, 4], 1e4, 0, 0),
    ([129], 1e4, 0, 0), ([128, 1], 1e4, 0, 0), ([2 ** 31 - 1, 2 ** 31 - 1], 1e4, 0, 0),
    ([4], 0.5, 0, 0), ([4], float("nan"), 0, 0), ([4], float("inf"), 0, 0), ([4], 1e4, 2, 0),
    ([4], 1e4, 0, -1)])
def test_rotary_plan_refusals(sections, base, pairing, ladder):
    with pytest.raises(InvalidArgument):
        kernels.rotary_axes(sections, base, pairing, ladder)


def test_rotary_no_ops():
    rotary = kernels.rotary_axes([4])
    kernels.launch_rotary(None, None, None, None, None, rotary, qk(tokens=0))
    kernels.launch_rotary(None, None, None, None, None, rotary, qk(q_heads=0, k_heads=0))
    kernels.launch_qk_norm_rotary(None, None, None, None, QkNorm(), None, None, qk(tokens=0))


@pytest.mark.parametrize("changes,message", [
    (dict(tokens=-1), "negative"), (dict(k_heads=-2), "negative"),
    (dict(head_dim=7), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(head_dim=258), "head_dim"),
    (dict(dtype=kernels.DTYPE_TF32), "F32 or BF16"), (dict(dtype=9), "F32 or BF16"),
    (dict(head_dim=6), "more pairs"), (dict(q_stride=15), "stride"),
    (dict(k_out_stride=-16), "stride"), (dict(position_stride=-1), "position stride")])
def test_rotary_refusals(changes, message):
    rotary = kernels.rotary_axes([4])
    with pytest.raises(InvalidArgument, match=message):
        kernels.launch_rotary(FAKE, 2 * FAKE, 3 * FAKE, 4 * FAKE, 5 * FAKE, rotary, qk(**changes))


def test_rotary_pointer_refusals():
    rotary = kernels.rotary_axes([4])
    call = kernels.launch_rotary
    with pytest.raises(InvalidArgument, match="rotary axes cannot be null"):
        call(FAKE, 2 * FAKE, 3 * FAKE, 4 * FAKE, 5 * FAKE, None, qk())
    with pytest.raises(InvalidArgument, match="positions"):
        call(FAKE, 2 * FAKE, 3 * FAKE, 4 * FAKE, None, rotary, qk())
    with pytest.raises(InvalidArgument, match="cannot be null"):
        call(None, 2 * FAKE, 3 * FAKE, 4 * FAKE, 5 * FAKE, rotary, qk())
    with pytest.raises(InvalidArgument, match="aligned"):
        call(FAKE + 2, 2 * FAKE, 3 * FAKE, 4 * FAKE, 5 * FAKE, rotary, qk())
    # An output may be its own input, but not the other one, nor shifted, nor the other output.
    with pytest.raises(InvalidArgument, match="not its own"):
        call(FAKE, 2 * FAKE, 2 * FAKE, 4 * FAKE, 5 * FAKE, rotary, qk())
    with pytest.raises(InvalidArgument, match="not its own"):
        call(FAKE, 2 * FAKE, FAKE + 4, 4 * FAKE, 5 * FAKE, rotary, qk())
    with pytest.raises(InvalidArgument, match="not its own"):
        call(FAKE, 2 * FAKE, FAKE, 4 * FAKE, 5 * FAKE, rotary, qk(q_out_stride=32))
    with pytest.raises(InvalidArgument, match="outputs overlap"):
        call(FAKE, 2 * FAKE, 4 * FAKE, 4 * FAKE + 8, 5 * FAKE, rotary, qk())
    with pytest.raises(LengthError):
        call(FAKE, 2 * FAKE, 3 * FAKE, 4 * FAKE, 5 * FAKE, rotary, qk(q_stride=2 ** 60))
    broken = kernels.rotary_axes([4])
    broken.first[1] = 200
    with pytest.raises(InvalidArgument, match="cuvit_rotary_init"):
        call(FAKE, 2 * FAKE, 3 * FAKE, 4 * FAKE, 5 * FAKE, broken, qk())


@pytest.mark.parametrize("norm", [QkNorm(kind=2), QkNorm(epsilon=-1.0),
                                  QkNorm(epsilon=float("nan")), QkNorm(epsilon=float("inf"))])
def test_norm_refusals(norm):
    with pytest.raises(InvalidArgument, match="unknown norm"):
        kernels.launch_qk_norm_rotary(FAKE, 2 * FAKE, 3 * FAKE, 4 * FAKE, norm, None, None, qk())


def test_norm_gain_alignment():
    with pytest.raises(InvalidArgument, match="gains"):
        kernels.launch_qk_norm_rotary(FAKE, 2 * FAKE, 3 * FAKE, 4 * FAKE, QkNorm(k_beta=FAKE + 1),
                                      None, None, qk())


def test_attention_no_ops():
    for changes in (dict(batch=0), dict(q_tokens=0), dict(q_heads=0)):
        kernels.launch_attention_varlen(None, None, None, None, None, None, attention(**changes))
        assert kernels.attention_varlen_workspace(attention(**changes)) == 0


@pytest.mark.parametrize("changes,message", [
    (dict(batch=-1), "negative"), (dict(q_tokens=-5), "negative"), (dict(kv_heads=-1), "negative"),
    (dict(head_dim=0), "head_dim"), (dict(head_dim=129), "head_dim"),
    (dict(dtype=kernels.DTYPE_TF32), "F32 or BF16"), (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(kv_heads=3), "divide"), (dict(kv_heads=0), "divide"),
    (dict(q_stride=31), "stride"), (dict(v_stride=-16), "stride")])
def test_attention_refusals(changes, message):
    with pytest.raises(InvalidArgument, match=message):
        kernels.launch_attention_varlen(FAKE, 2 * FAKE, 3 * FAKE, 4 * FAKE, FAR, FAR,
                                        attention(**changes))
    with pytest.raises(InvalidArgument, match=message):
        kernels.attention_varlen_workspace(attention(**changes))


def test_attention_pointer_refusals():
    call = kernels.launch_attention_varlen
    with pytest.raises(InvalidArgument, match="cannot be null"):
        call(None, FAKE, FAKE, 2 * FAKE, FAR, FAR, attention())
    with pytest.raises(InvalidArgument, match="cannot be null"):
        call(FAKE, FAKE, None, 2 * FAKE, FAR, FAR, attention())
    with pytest.raises(InvalidArgument, match="cannot be null"):
        call(FAKE, FAKE, FAKE, 2 * FAKE, None, FAR, attention())
    with pytest.raises(InvalidArgument, match="as many keys"):
        call(FAKE, FAKE, FAKE, 2 * FAKE, FAR, None, attention(kv_tokens=9))
    with pytest.raises(InvalidArgument, match="aligned"):
        call(FAKE + 2, FAKE, FAKE, 2 * FAKE, FAR, FAR, attention())
    with pytest.raises(InvalidArgument, match="offsets must be aligned"):
        call(FAKE, FAKE, FAKE, 2 * FAKE, FAR + 2, FAR, attention())
    for shared in range(3):
        operands = [FAKE, 2 * FAKE, 3 * FAKE]
        with pytest.raises(InvalidArgument, match="overlaps"):
            call(*operands, operands[shared], FAR, FAR, attention())
    with pytest.raises(LengthError):
        call(FAKE, 2 * FAKE, 3 * FAKE, 4 * FAKE, FAR, FAR, attention(q_tokens=2 ** 31 - 1))
    with pytest.raises(LengthError):
        call(FAKE, 2 * FAKE, 3 * FAKE, 4 * FAKE, FAR, FAR, attention(k_stride=2 ** 60))


def test_attention_scale_times_log2e_is_finite():
    """The kernels scale scores for powers of two; 3e38 log2(e) is no float."""
    for scale in (3.0e38, 2.4e38):
        with pytest.raises(InvalidArgument, match="scale"):
            kernels.launch_attention_varlen(FAKE, 2 * FAKE, 3 * FAKE, 4 * FAKE, FAR, FAR,
                                            attention(scale=scale))
    with pytest.raises(Exception) as caught:
        kernels.launch_attention_varlen(FAKE, 2 * FAKE, 3 * FAKE, 4 * FAKE, FAR, FAR,
                                        attention(scale=2.3e38))
    assert "scale" not in str(caught.value)


def test_linear_no_ops():
    for changes in (dict(m=0), dict(n=0)):
        kernels.launch_linear(None, None, None, None, None, None, linear(**changes))


@pytest.mark.parametrize("changes,message", [
    (dict(m=-1), "negative"), (dict(k=-1), "negative"), (dict(math=3), "math mode"),
    (dict(out_dtype=3), "output data type"), (dict(activation=4), "activation"),
    (dict(activation=-1), "activation"), (dict(ldx=15), "row distance"),
    (dict(ldo=-8), "row distance"), (dict(ldr=7), "row distance")])
def test_linear_refusals(changes, message):
    with pytest.raises(InvalidArgument, match=message):
        kernels.launch_linear(FAKE, 2 * FAKE, None, None, None, 3 * FAKE, linear(**changes))


def test_linear_pointer_refusals():
    call = kernels.launch_linear
    with pytest.raises(InvalidArgument, match="cannot be null"):
        call(FAKE, None, None, None, None, 2 * FAKE, linear())
    with pytest.raises(InvalidArgument, match="cannot be null"):
        call(FAKE, FAKE, None, None, None, None, linear())
    with pytest.raises(InvalidArgument, match="aligned"):
        call(FAKE, FAKE, FAR + 2, None, None, 2 * FAKE, linear())
    for at in range(5):
        operands = [FAKE, 2 * FAKE, 3 * FAKE, 4 * FAKE, 5 * FAKE]
        out = operands[at] + (4 if at == 4 else 0)  # the residual itself is allowed
        with pytest.raises(InvalidArgument, match="overlaps"):
            call(*operands, out, linear())
    with pytest.raises(InvalidArgument, match="overlaps"):  # the up half of a gated bias
        call(FAKE, 2 * FAKE, FAR, None, None, FAR + 4 * 12, linear(gated=True))
    with pytest.raises(LengthError):
        call(FAKE, 2 * FAKE, None, None, None, FAR, linear(m=2 ** 31 - 1))


@pytest.mark.parametrize("extent", ["m", "n", "k"])
def test_linear_extents_whose_steps_pass_32_bits(extent):
    """The kernels count up to 8192 elements past an extent's end; what that takes past 2^31 - 1 is
    refused."""
    largest = 2 ** 31 - 1 - 65536
    sizes = dict(m=1, n=1, k=8)
    if extent == "n":
        largest //= 2
    for size in (largest + 1, 2 ** 31 - 1 - 4096 if extent != "n" else (2 ** 31 - 1 - 4096) // 2):
        with pytest.raises(LengthError):
            kernels.launch_linear(FAKE, 2 * FAKE, None, None, None, 2 ** 48,
                                  linear(**{**sizes, extent: size}))
    # The next smaller one passes this check (and fails only later, for the fake addresses).
    with pytest.raises(Exception) as caught:
        kernels.launch_linear(FAKE, 2 ** 40, None, None, None, 2 ** 48,
                              linear(**{**sizes, extent: largest}))
    assert "too large" not in str(caught.value)


def test_interleaved_columns_do_not_overlap():
    """Outputs in other columns of their inputs' rows pass the overlap check (and fail only
    later, on a machine without a device or for the fake addresses)."""
    rotary = kernels.rotary_axes([4])
    problem = qk(q_stride=64, k_stride=64, q_out_stride=64, k_out_stride=64)
    with pytest.raises(Exception) as caught:
        kernels.launch_rotary(FAKE, FAKE + 64, FAKE + 128, FAKE + 192, FAR, rotary, problem)
    assert "overlap" not in str(caught.value)
    with pytest.raises(InvalidArgument, match="overlap"):
        kernels.launch_rotary(FAKE, FAKE + 64, FAKE + 96, FAKE + 192, FAR, rotary, problem)


def test_positions_wrap_exactly():
    """position * turns modulo 2^64 is the fraction of a turn, for every 32-bit position."""
    rotary = kernels.rotary_axes([16])
    for position in (0, 1, -1, 12345, 2 ** 31 - 1, -2 ** 31):
        for i in (0, 5, 15):
            fraction = ((position * int(rotary.turns[i])) % 2 ** 64) / 2.0 ** 64
            want = math.fmod(position * 10000.0 ** (-i / 16), 2 * math.pi)
            difference = np.remainder(fraction * 2 * math.pi - want + math.pi, 2 * math.pi) - math.pi
            # A double's angle: 2^-53 relative, twice (the power and the product).
            assert abs(difference) <= 4 * 2.0 ** -53 * max(abs(position), 8.0)


def test_outputs_over_what_every_block_reads_are_refused():
    rotary = kernels.rotary_axes([4])
    with pytest.raises(InvalidArgument, match="overlaps the positions"):
        kernels.launch_rotary(FAKE, None, FAR, None, FAR + 8, rotary, qk(k_heads=0))
    for gains in ((FAR + 4, None), (None, FAR + 4)):
        with pytest.raises(InvalidArgument, match="overlaps the positions"):
            kernels.launch_qk_norm_rotary(FAKE, None, FAR, None,
                                          QkNorm(kernels.NORM_RMS, 1e-6, *gains, None, None), None,
                                          None, qk(k_heads=0))
    for at in (0, 1):
        offsets = [2 * FAR, 3 * FAR]
        offsets[at] = FAR + 4
        with pytest.raises(InvalidArgument, match="overlaps"):
            kernels.launch_attention_varlen(FAKE, 2 * FAKE, 3 * FAKE, FAR, *offsets, attention())


CPP = r"""
#include "cuvit/kernels.hpp"
#include <cstdio>
template <typename Call> static bool refused(Call call) {
    try { call(); } catch (const std::invalid_argument&) { return true; }
    return false;
}
int main() {
    cuvit_rotary rotary;
    const int sections[2] = {8, 8};
    if (cuvit_rotary_init(&rotary, 2, sections, 10000.0, CUVIT_ROTARY_HALVES,
                          CUVIT_ROTARY_LADDER_AXIS) != CUVIT_OK) return 1;
    cuvit_qk_problem qk{};
    qk.tokens = -1; qk.head_dim = 32;
    cuvit_qk_norm norm{};
    cuvit_attention_problem attention{};
    attention.batch = -1;
    cuvit_linear_problem linear{};
    linear.m = -1;
    if (!refused([&] { cuvit::launch_rotary(nullptr, nullptr, nullptr, nullptr, nullptr, rotary, qk); }))
        return 2;
    if (!refused([&] { cuvit::launch_qk_norm_rotary(nullptr, nullptr, nullptr, nullptr, norm, nullptr,
                                                   &rotary, qk); })) return 3;
    if (!refused([&] { cuvit::attention_varlen_workspace(attention); })) return 4;
    if (!refused([&] { cuvit::launch_attention_varlen(nullptr, nullptr, nullptr, nullptr, nullptr,
                                                     nullptr, attention); })) return 5;
    if (!refused([&] { cuvit::launch_linear(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr,
                                           linear); })) return 6;
    linear.m = 0;
    cuvit::launch_linear(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, linear);
    return 0;
}
"""


def test_cpp_wrappers_compile_and_refuse(tmp_path):
    """The header-only wrappers of include/cuvit/kernels.hpp raise what the C entries report."""
    root = pathlib.Path(__file__).resolve().parent.parent
    source = tmp_path / "wrappers.cpp"
    source.write_text(CPP)
    program = tmp_path / "wrappers"
    library = _lib.LIBRARY_PATH
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", f"-I{root / 'include'}",
                    "-I/usr/local/cuda/include", str(source), "-o", str(program), str(library),
                    f"-Wl,-rpath,{library.parent}", "-L/usr/local/cuda/lib64", "-lcudart"],
                   check=True, timeout=120)
    assert subprocess.run([str(program)], timeout=60).returncode == 0
