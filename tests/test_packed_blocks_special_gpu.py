"""The operators over packed images and videos on NaN, infinities and the ends of their ranges: what
each formula gives there, through every kernel a call may take."""

from __future__ import annotations

import math
import pathlib
import subprocess
import sys

import pytest

from cuvit import kernels
from cuvit.kernels import AttentionProblem, LinearProblem, QkNorm, QkProblem
from test_packed_blocks_gpu import (TYPES, attention_64, check, dtype_of, normal, offsets,
                                    run_attention, torch_type)

pytestmark = pytest.mark.gpu

# Places of a key: every one of a group of eight, ends of 32, 64 and 128 keys, a sequence's last.
PLACES = [*range(8), 14, 15, 30, 31, 62, 63, 94, 95, 110, 126, 127, 128, 134, 143, 200, 255, 256, 299]


def attention_case(torch, kind, queries, keys, dim, causal, seed=0):
    heads = 2
    q = normal(torch, (queries, heads, dim), seed + 1, kind)
    k, v = (normal(torch, (keys, heads, dim), seed + i, kind) for i in (2, 3))
    problem = AttentionProblem(1, queries, keys, heads, heads, dim, dtype_of(kind), causal, 0.125)
    return q, k, v, problem


# ---- attention: NaN and infinite keys ------------------------------------------------------


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("queries", [2, 300])
@pytest.mark.parametrize("dim", [32, 64, 80, 128, 13])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_nan_key_reaches_every_query_that_sees_it(causal, dim, queries, kind, cuda):
    """Wherever the key stands in its tile. The other head keeps its results, and so do, but for
    roundings, the queries that do not see the key: rows that share a warp with one that reads its
    scores again do so too, and take all their exponentials in the exact form, where a quarter of
    them may have come from the polynomial that attention_64's bound counts."""
    torch = cuda
    keys = 300
    q, k, v, problem = attention_case(torch, kind, queries, keys, dim, causal)
    places = offsets(torch, [queries]), offsets(torch, [keys])
    clean = run_attention(torch, q, k, v, *places, problem)
    assert clean.isfinite().all()
    want, bound = attention_64(torch, q, k, v, [queries], [keys], 0.125, causal, kind)
    for at in PLACES:
        poisoned = k.clone()
        poisoned[at, 0, dim // 2] = float("nan")
        got = run_attention(torch, q, poisoned, v, *places, problem)
        sees = torch.ones(queries, dtype=torch.bool, device="cuda")
        if causal:
            sees = torch.arange(queries, device="cuda") + keys - queries >= at
        assert got[sees, 0].isnan().all(), f"key {at}"
        check(got[~sees], want[~sees], bound[~sees], f"key {at}")
        assert torch.equal(got[:, 1], clean[:, 1])


@pytest.mark.parametrize("queries", [2, 300])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_infinite_keys(queries, dim, cuda):
    """A score of plus infinity leaves no weight to divide by, one of minus infinity leaves its key
    out; a query whose scores are all minus infinity counts as one that sees no key, also where
    only its first tile's are."""
    torch = cuda
    keys = 300
    q, k, v, problem = attention_case(torch, "bf16", queries, keys, dim, False)
    q[:, :, 0] = q[:, :, 0].abs() + 0.5
    q[queries // 2, :, 0] = -1.0
    places = offsets(torch, [queries]), offsets(torch, [keys])
    for out_of, left in ((range(7, 8), None), (range(0, 130), None), (range(0, keys), 0)):
        poisoned = k.clone()
        poisoned[out_of.start:out_of.stop, 0, 0] = -float("inf")
        got = run_attention(torch, q, poisoned, v, *places, problem)
        assert got[queries // 2, 0].isnan().all()
        rest = [i for i in range(queries) if i != queries // 2]
        if left == 0:
            assert (got[rest, 0] == 0.0).all()
            continue
        kept = [j for j in range(keys) if j not in out_of]
        want, bound = attention_64(torch, q, k[kept], v[kept], [queries], [len(kept)], 0.125, False,
                                   "bf16")
        check(got[rest, 0], want[rest, 0], bound[rest, 0], f"without {out_of}")


@pytest.mark.parametrize("queries", [2, 300])
def test_attention_first_tile_minus_infinity_then_low_scores(queries, cuda):
    """The first tile's keys are left out and the next ones' scores lie thousands below zero: the
    maximum has to come down to them."""
    torch = cuda
    keys, dim = 300, 64
    q, k, v, _ = attention_case(torch, "bf16", queries, keys, dim, False)
    q[:, :, 0] = 64.0
    k[:, :, 0] = -64.0
    k[:130, :, 0] = -float("inf")
    problem = AttentionProblem(1, queries, keys, 2, 2, dim, dtype_of("bf16"), False, 1.0)
    got = run_attention(torch, q, k, v, offsets(torch, [queries]), offsets(torch, [keys]), problem)
    want, bound = attention_64(torch, q, k[130:], v[130:], [queries], [keys - 130], 1.0, False, "bf16")
    check(got, want, bound)


# ---- rotary: elements past the rotated pairs -----------------------------------------------


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("pairing", [kernels.ROTARY_HALVES, kernels.ROTARY_ADJACENT],
                         ids=["halves", "adjacent"])
@pytest.mark.parametrize("dim,pairs", [(64, 16), (64, 8), (72, 32), (80, 12), (24, 5), (96, 44), (12, 2),
                                       (64, 31), (10, 3)])
@pytest.mark.parametrize("shift", [0, 1])
def test_rotary_copies_what_it_does_not_turn(shift, dim, pairs, pairing, kind, cuda):
    """Bit for bit, whatever their neighbours hold: NaN, infinities and negative zeros beside the
    elements that turn and beside each other. At any alignment."""
    torch = cuda
    tokens, heads = 5, 3
    buffer = normal(torch, (tokens * heads * dim + shift,), dim + pairs, kind)
    x = buffer[shift:].view(tokens, heads, dim)
    rest = x[..., 2 * pairs:]
    for i, value in enumerate((float("nan"), float("inf"), -float("inf"), -0.0)):
        rest[:, :, i::7] = value
    x[2, 1, 0] = float("nan")
    out = torch.zeros_like(x)
    positions = torch.arange(1, tokens + 1, dtype=torch.int32, device="cuda")
    problem = QkProblem(tokens, heads, 0, dim, dtype_of(kind))
    kernels.launch_rotary(x, None, out, None, positions, kernels.rotary_axes([pairs], 10.0, pairing),
                          problem)
    torch.cuda.synchronize()
    bits = torch.int16 if kind == "bf16" else torch.int32
    got, want = (t[..., 2 * pairs:] for t in (out, x))
    alike = (got.contiguous().view(bits) == want.contiguous().view(bits)) | (got.isnan() & want.isnan())
    assert alike.all()
    clean = torch.ones_like(out[..., :2 * pairs], dtype=torch.bool)
    clean[2, 1] = False
    assert out[..., :2 * pairs][clean].isfinite().all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("norm", [kernels.NORM_RMS, kernels.NORM_LAYER], ids=["rms", "layer"])
@pytest.mark.parametrize("pairs", [0, 8])
@pytest.mark.parametrize("shift", [0, 1])
def test_norm_of_gains_that_are_not_finite(shift, pairs, norm, kind, cuda):
    """An infinite or NaN gain of an element that does not turn reaches that element alone, with
    and without a rotation."""
    torch = cuda
    tokens, heads, dim = 4, 2, 64
    buffer = normal(torch, (tokens * heads * dim + shift,), 3, kind)
    x = buffer[shift:].view(tokens, heads, dim)
    gamma = normal(torch, (dim,), 4)
    gamma[20], gamma[43] = float("nan"), float("inf")
    out = torch.zeros_like(x)
    positions = torch.arange(tokens, dtype=torch.int32, device="cuda")
    kernels.launch_qk_norm_rotary(x, None, out, None, QkNorm(norm, 1e-6, gamma), positions,
                                  kernels.rotary_axes([pairs]) if pairs else None,
                                  QkProblem(tokens, heads, 0, dim, dtype_of(kind)))
    torch.cuda.synchronize()
    clean = torch.ones(dim, dtype=torch.bool, device="cuda")
    clean[20] = clean[43] = False
    assert out[..., clean].isfinite().all()
    assert out[..., 20].isnan().all() and out[..., 43].isinf().all()


# ---- linear layers: activations at infinities and in their tails ---------------------------

ACTIVATIONS = pytest.mark.parametrize("activation", range(4), ids=["none", "gelu", "gelu_tanh", "silu"])
# A few rows; a cluster's slices of k; whole tiles; operands that TMA cannot describe.
PATHS = pytest.mark.parametrize("m,k,shift", [(3, 64, 0), (24, 2048, 0), (300, 64, 0), (20, 64, 1)],
                                ids=["rows", "slices", "tiles", "simt"])
MODES = pytest.mark.parametrize("kind,out_kind", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32"),
                                                  ("f32", "bf16")])


def activated(torch, activation, y):
    """The formulas in 64 bits, none of which cancels for negative y."""
    if activation == kernels.ACTIVATION_GELU:
        return y * torch.special.erfc(y * -math.sqrt(0.5)) / 2
    if activation == kernels.ACTIVATION_GELU_TANH:
        return y / (1 + (-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)).exp())
    return y / (1 + (-y).exp()) if activation == kernels.ACTIVATION_SILU else y


def run_layer(torch, m, k, shift, w0, kind, out_kind, activation, gated, bias=None):
    """x has a one at the first place and zeros after: every sum is the one product w0[column]."""
    n = w0.numel() // (2 if gated else 1)
    x = torch.zeros(m * (k + shift), dtype=torch_type(torch, kind), device="cuda").view(m, k + shift)
    w = torch.zeros(w0.numel(), k + shift, dtype=x.dtype, device="cuda")
    x[:, 0] = 1.0
    w[:, 0] = w0
    out = torch.full((m, n), 3.0, dtype=torch_type(torch, out_kind), device="cuda")
    kernels.launch_linear(x, w, bias, None, None, out,
                          LinearProblem(m, n, k, kernels.MATH_BF16 if kind == "bf16"
                                        else kernels.MATH_FP32, dtype_of(out_kind), activation, gated,
                                        k + shift, k + shift))
    torch.cuda.synchronize()
    return out


@ACTIVATIONS
@MODES
@PATHS
@pytest.mark.parametrize("gated", [False, True], ids=["plain", "gated"])
def test_linear_infinite_sums(gated, m, k, shift, kind, out_kind, activation, cuda):
    """What the formula gives for a sum of plus infinity (itself), minus infinity (NaN, but for no
    activation) and NaN, whichever kernel a call takes; its neighbours keep their values."""
    torch = cuda
    n = 96
    w0 = torch.linspace(-4, 4, 2 * n if gated else n, device="cuda")
    bias = torch.zeros(w0.numel(), device="cuda")
    clean = run_layer(torch, m, k, shift, w0, kind, out_kind, activation, gated, bias)
    bias[5], bias[42], bias[77] = float("inf"), -float("inf"), float("nan")
    if gated:
        w0[n + 5] = w0[n + 42] = 1.0
    got = run_layer(torch, m, k, shift, w0, kind, out_kind, activation, gated, bias)
    assert (got[:, 5] == float("inf")).all()
    if activation == kernels.ACTIVATION_NONE:
        assert (got[:, 42] == -float("inf")).all()
    else:
        assert got[:, 42].isnan().all()
    assert got[:, 77].isnan().all()
    same = [c for c in range(n) if c not in (5, 42, 77)]
    assert clean.isfinite().all() and torch.equal(got[:, same], clean[:, same])


@ACTIVATIONS
@MODES
@PATHS
def test_linear_large_finite_sums(m, k, shift, kind, out_kind, activation, cuda):
    """Sums up to the largest bfloat16, where squares and cubes are infinite: themselves, or zero."""
    torch = cuda
    sizes = torch.tensor([1e2, 1e6, 1e12, 9e17, 2e18, 1e19, 1e20, 1e30, 1e37, 3.3e38], device="cuda")
    w0 = torch.cat([sizes, -sizes])
    got = run_layer(torch, m, k, shift, w0, kind, out_kind, activation, False).double()
    y = w0.to(torch_type(torch, kind)).double()
    want = activated(torch, activation, y) if activation == kernels.ACTIVATION_NONE else y.clamp_min(0.0)
    want = want.to(torch_type(torch, out_kind)).double()
    # The value itself, times a factor that is 1 to within a few steps.
    step = 2.0 ** -7 if out_kind == "bf16" else 32 * 2.0 ** -24
    check(got, want.expand_as(got), (step * want.abs() + 1e-30).expand_as(got))


@pytest.mark.parametrize("activation", range(1, 4), ids=["gelu", "gelu_tanh", "silu"])
@MODES
@PATHS
@pytest.mark.parametrize("short", [False, True], ids=["full", "short"])
def test_linear_activation_tails(short, m, k, shift, kind, out_kind, activation, cuda):
    """Relative accuracy alone, into the negative tail: every sum is one product by 1, so the
    activation sees just that value. Float outputs: 12 u32 (six of them the polynomial of the erf
    form, the others a power, a reciprocal and products), bfloat16 ones 2^-12 and the store's half
    step, within a factor of 1 + 2^-8. Powers of two below 2^-126 may be flushed, with them values
    below |y| times that.
    The products of TF32 halves keep all but 2^-23 of a float, which the activation's slope passes on
    (in the tail of GELU y^2 times as much of the value); short values, of eight bits, are kept
    whole."""
    torch = cuda
    y = torch.cat([torch.linspace(-95.0, 12.0, 700), torch.linspace(-14.5, -0.01, 500),
                   torch.logspace(-30, 0, 60), -torch.logspace(-30, 0, 60)]).cuda()
    if short:
        y = y.bfloat16().float()
    got = run_layer(torch, m, k, shift, y, kind, out_kind, activation, False)
    y = y.to(torch_type(torch, kind)).double().requires_grad_()
    want = activated(torch, activation, y)
    slope, = torch.autograd.grad(want.sum(), y)
    slope = slope.nan_to_num(0.0)  # infinite over infinite where a double's power is: below 1e-150
    y, want = y.detach(), want.detach()
    if out_kind == "bf16":
        bound = (2.0 ** -12 * (1 + 2.0 ** -8) + 2.0 ** -8) * want.abs()
    else:
        bound = 12 * 2.0 ** -24 * want.abs()
    bound = bound + 128 * 2.0 ** -126
    if kind == "f32" and not short:
        bound = bound + 1.01 * 2.0 ** -23 * (slope * y).abs()
    check(got, want.expand(m, -1), bound.expand(m, -1))


# ---- float products of TF32 halves: every NaN ----------------------------------------------


@pytest.mark.parametrize("bits", [0x7F800001, 0x7F801FFF, 0x7FC00000, 0x7FFFFFFF, -0x7FFFFF, -1],
                         ids=lambda b: f"{b & 0xFFFFFFFF:08x}")
def test_float_nan_of_any_payload(bits, cuda):
    """A NaN with its payload in the last bits only is one all the same."""
    torch = cuda
    for m, n, k in ((40, 64, 96), (300, 200, 64), (12, 64, 4096)):
        for side in range(2):
            x, w = normal(torch, (m, k), 1), normal(torch, (n, k), 2)
            (x, w)[side].view(torch.int32)[5, 33] = bits
            out = torch.zeros(m, n, device="cuda")
            kernels.launch_linear(x, w, None, None, None, out,
                                  LinearProblem(m, n, k, kernels.MATH_FP32, kernels.DTYPE_F32))
            torch.cuda.synchronize()
            bad = torch.zeros_like(out, dtype=torch.bool)
            (bad if side == 0 else bad.t())[5] = True
            assert out[bad].isnan().all() and out[~bad].isfinite().all()
    for dim in (64, 128):
        for queries in (2, 200):
            q, k, v, problem = attention_case(torch, "f32", queries, 300, dim, False)
            places = offsets(torch, [queries]), offsets(torch, [300])
            for side in range(3):
                operands = [t.clone() for t in (q, k, v)]
                operands[side].view(torch.int32)[1, 0, 7] = bits
                got = run_attention(torch, *operands, *places, problem)
                bad = torch.zeros_like(got, dtype=torch.bool)
                if side == 0:
                    bad[1, 0] = True
                elif side == 1:
                    bad[:, 0] = True
                else:
                    bad[:, 0, 7] = True
                assert got[bad].isnan().all() and got[~bad].isfinite().all()


# ---- attention: more query heads to a key head than the few-row kernels take at once -------


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("group", [9, 12, 16, 17, 40])
@pytest.mark.parametrize("empty", [0, 1, 5], ids=lambda n: f"{n}empty")
def test_attention_wide_groups_of_single_queries(empty, group, kind, cuda):
    """One query a sequence, with and without sequences that have none: on the average over the
    batch the former have more rows than the few-row kernels take, the latter few enough, so that
    their blocks divide a key head's query heads into chunks of eight."""
    torch = cuda
    kv_heads, dim = 2, 64
    queries = ([1] + [0] * empty) * 3
    keys = ([300, *[0] * empty, 17, *[4] * empty, 2000, *[64] * empty])
    q = normal(torch, (sum(queries), kv_heads * group, dim), 1, kind)
    k, v = (normal(torch, (sum(keys), kv_heads, dim), seed, kind) for seed in (2, 3))
    for causal in (False, True):
        problem = AttentionProblem(len(queries), sum(queries), sum(keys), kv_heads * group, kv_heads,
                                   dim, dtype_of(kind), causal, 0.2)
        want, bound = attention_64(torch, q, k, v, queries, keys, 0.2, causal, kind)
        for workspace in (True, False):
            got = run_attention(torch, q, k, v, offsets(torch, queries), offsets(torch, keys), problem,
                                workspace)
            check(got, want, bound, f"causal {causal} workspace {workspace}")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("long", [40, 700])
def test_attention_one_long_sequence_among_single_queries(long, kind, cuda):
    """A prompt beside new tokens of other sequences: the average sends it to the few-row kernels in
    one batch and the new tokens to the tile kernels in the other."""
    torch = cuda
    queries = [1] * 20 + [long] + [1] * 20
    keys = [37 * i % 400 + 1 for i in range(20)] + [long + 5] + [91 * i % 700 + 1 for i in range(20)]
    heads, kv_heads, dim = 4, 2, 64
    q = normal(torch, (sum(queries), heads, dim), 1, kind)
    k, v = (normal(torch, (sum(keys), kv_heads, dim), seed, kind) for seed in (2, 3))
    for causal in (False, True):
        problem = AttentionProblem(len(queries), sum(queries), sum(keys), heads, kv_heads, dim,
                                   dtype_of(kind), causal, 0.2)
        want, bound = attention_64(torch, q, k, v, queries, keys, 0.2, causal, kind)
        got = run_attention(torch, q, k, v, offsets(torch, queries), offsets(torch, keys), problem)
        check(got, want, bound, f"causal {causal}")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("group", [16, 24])
def test_attention_single_queries_of_a_wide_group_share_their_keys(group, kind, cuda):
    """The few-row kernels take a wide group's heads eight at a time: without a split of the keys that
    is bit for bit the calls of eight heads each."""
    torch = cuda
    keys, dim = [300, 17, 1000], 128
    q = normal(torch, (3, group, dim), 1, kind)
    k, v = (normal(torch, (sum(keys), 1, dim), seed, kind) for seed in (2, 3))
    places = offsets(torch, [1, 1, 1]), offsets(torch, keys)

    def run(part):
        problem = AttentionProblem(3, 3, sum(keys), part.shape[1], 1, dim, dtype_of(kind), True, 0.1)
        return run_attention(torch, part, k, v, *places, problem, workspace=False)

    whole = run(q)
    for first in range(0, group, 8):
        assert torch.equal(whole[:, first:first + 8], run(q[:, first:first + 8].contiguous()))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("queries", [20, 150, 300])
def test_attention_rows_behind_a_sequence_change_no_bit_of_it(queries, dim, kind, cuda):
    """The next sequence's queries stand in the same tile: what they are, or that they are large,
    infinite or NaN, leaves this one's results as they are, also in their roundings."""
    torch = cuda
    keys = 700
    q, k, v, _ = attention_case(torch, kind, queries + 100, keys, dim, False)
    problem = AttentionProblem(2, queries + 100, keys, 2, 2, dim, dtype_of(kind), False, 0.125)
    places = offsets(torch, [queries, 100]), offsets(torch, [600, 100])
    want = run_attention(torch, q, k, v, *places, problem)[:queries]
    for tail in (1000.0 * q[queries:], torch.full_like(q[queries:], 1e30),
                 torch.full_like(q[queries:], float("inf")),
                 torch.full_like(q[queries:], float("nan"))):
        other = torch.cat([q[:queries], tail])
        assert torch.equal(run_attention(torch, other, k, v, *places, problem)[:queries], want)


# ---- a process whose first call is a captured one ------------------------------------------

FIRST_CALL = r"""
import sys
sys.path[:0] = {paths!r}
import torch
from cuvit import kernels as K
from test_packed_blocks_gpu import dtype_of, normal, offsets
kind, name = {kind!r}, {name!r}
torch.zeros(1, device="cuda")  # the caller's context, nothing of the library's
math = K.MATH_BF16 if kind == "bf16" else K.MATH_FP32
if name.startswith("linear"):
    m, k, n = dict(rows=(3, 64, 96), slices=(24, 4096, 96), tiles=(300, 64, 96), pairs=(9000, 64, 2048),
                   simt=(20, 65, 96))[name[7:]]
    x, w = normal(torch, (m, k), 1, kind), normal(torch, (n, k), 2, kind)
    out = torch.zeros(m, n, dtype=x.dtype, device="cuda")
    problem = K.LinearProblem(m, n, k, math, dtype_of(kind))
    call = lambda stream: K.launch_linear(x, w, None, None, None, out, problem, stream)
elif name.startswith("attention"):
    queries, keys, dim = dict(few=(1, 9000, 64), many=(300, 5000, 64), wide=(300, 300, 128),
                              odd=(70, 90, 13))[name[10:]]
    q = normal(torch, (queries, 2, dim), 1, kind)
    k, v = (normal(torch, (keys, 2, dim), i, kind) for i in (2, 3))
    out, places = torch.zeros_like(q), (offsets(torch, [queries]), offsets(torch, [keys]))
    area = torch.zeros(32 << 20, dtype=torch.uint8, device="cuda")
    problem = K.AttentionProblem(1, queries, keys, 2, 2, dim, dtype_of(kind), False, 0.1)
    call = lambda stream: K.launch_attention_varlen(q, k, v, out, *places, problem, area,
                                                    area.numel(), stream)
else:
    x = normal(torch, (40, 3, 64), 1, kind)
    out, positions = torch.zeros_like(x), torch.arange(40, dtype=torch.int32, device="cuda")
    rotary, problem = K.rotary_axes([16]), K.QkProblem(40, 3, 0, 64, dtype_of(kind))
    call = lambda stream: K.launch_qk_norm_rotary(x, None, out, None, K.QkNorm(), positions, rotary,
                                                  problem, stream)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    call(torch.cuda.current_stream())
graph.replay()
torch.cuda.synchronize()
got = out.clone()
out.zero_()
torch.cuda.synchronize()
call(None)
torch.cuda.synchronize()
assert got.abs().sum() > 0 and torch.equal(got, out) and K.device_status() == 0
print("same")
"""


@pytest.mark.parametrize("name,kind", [("rotary", "bf16"), ("linear_slices", "bf16"),
                                       ("linear_pairs", "bf16"), ("linear_tiles", "f32"),
                                       ("attention_few", "bf16"), ("attention_wide", "bf16"),
                                       ("attention_many", "f32")])
def test_first_call_of_a_process_is_captured(name, kind, cuda):
    """Nothing that a call sets up once (context, function attributes, cluster sizes, tensor maps) is
    forbidden under capture."""
    here = pathlib.Path(__file__).resolve().parent
    program = FIRST_CALL.format(paths=[str(here), str(here.parent / "cu-vit_b200")], kind=kind, name=name)
    run = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "same" in run.stdout, run.stderr[-2000:]
