"""The operators over packed images and videos on the GPU, against their formulas in 64 bits.

Tolerances are sums of rounding steps (u32 = 2^-24 for FP32, ub = 2^-8 for bfloat16, half a step
each), derived at each operator; none is fitted to what a kernel returns.
"""

from __future__ import annotations

import math

import pytest

from cuvit import kernels
from cuvit.errors import InvalidArgument
from cuvit.kernels import AttentionProblem, LinearProblem, QkNorm, QkProblem

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
UB = 2.0 ** -8
TYPES = ["f32", "bf16"]


def dtype_of(kind):
    return kernels.DTYPE_BF16 if kind == "bf16" else kernels.DTYPE_F32


def torch_type(torch, kind):
    return torch.bfloat16 if kind == "bf16" else torch.float32


def normal(torch, shape, seed, kind="f32", std=1.0):
    generator = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=generator) * std).to(torch_type(torch, kind)).cuda()


def check(got, want, bound, what=""):
    """|got - want| <= bound, elementwise; NaN never passes."""
    difference = (got.double() - want).abs()
    bad = ~(difference <= bound)
    if bad.any():
        at = bad.nonzero()[0].tolist()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; first at {at}: "
                             f"{got[tuple(at)].item()} for {want[tuple(at)].item()}, bound "
                             f"{bound[tuple(at)].item() if bound.ndim else bound.item()}")


# ---- rotary positions and norms ------------------------------------------------------------


def turned(torch, x, positions, sections, base, pairing, ladder):
    """x [tokens, heads, dim] in 64 bits, turned."""
    pairs = sum(sections)
    rate, axis_of = [], []
    for axis, n in enumerate(sections):
        for j in range(n):
            exponent = j / n if ladder == kernels.ROTARY_LADDER_AXIS else (
                sum(sections[:axis]) + j) / pairs
            rate.append(base ** -exponent)
            axis_of.append(axis)
    rate = torch.tensor(rate, dtype=torch.float64, device="cuda")
    angle = (positions[axis_of].double().t() * rate)[:, None]
    index = torch.arange(pairs, device="cuda")
    first, second = ((index, index + pairs) if pairing == kernels.ROTARY_HALVES
                     else (2 * index, 2 * index + 1))
    out = x.clone()
    out[..., first] = x[..., first] * angle.cos() - x[..., second] * angle.sin()
    out[..., second] = x[..., first] * angle.sin() + x[..., second] * angle.cos()
    return out


def normed(torch, x, kind, epsilon, gamma, beta):
    if kind == kernels.NORM_LAYER:
        x = x - x.mean(-1, keepdim=True)
    x = x / ((x * x).mean(-1, keepdim=True) + epsilon).sqrt()
    if gamma is not None:
        x = x * gamma.double()
    return x if beta is None else x + beta.double()


def pair_norm(x):
    """An upper bound for what a rotation can make of any element: the head's largest pair."""
    return math.sqrt(2.0) * x.abs().amax(-1, keepdim=True)


def rotary_bound(torch, x, want, kind, dim, normalise):
    """FP32: sin and cos within 2 u32 of the angle's, the angle within 2^-25 half turns (pi
    2^-25 <= 2 u32), two products and a sum: 8 u32 of the pair's length in all; a norm's mean
    and sum of squares (dim additions) and its five further operations come on top. Positions
    near 2^31 are off by 2^-53 relative in the 64-bit angle itself: 2^31 2^-52 < 9 u32 more.
    Then the store's rounding."""
    steps = 17.0 + (2.0 * dim + 12.0 if normalise else 0.0)
    bound = steps * U32 * pair_norm(x)
    return bound + (UB if kind == "bf16" else U32) * want.abs()


SHAPES = [  # tokens, q_heads, k_heads, dim, sections
    (1, 1, 1, 2, [1]), (3, 2, 1, 6, [1, 1]), (197, 12, 12, 64, [16, 16]), (33, 3, 3, 32, [16]),
    (50, 16, 4, 72, [16, 16]), (41, 4, 4, 72, [12, 12, 12]), (130, 8, 2, 80, [8, 16, 16]),
    (64, 6, 0, 96, [24, 24]), (7, 0, 5, 128, [64]), (1, 24, 24, 128, [16, 24, 24]),
    (29, 2, 3, 256, [40, 40, 48]), (19, 3, 1, 100, [10, 7, 3, 5]), (11, 5, 5, 20, [0, 3, 4]),
    (500, 2, 2, 10, [5])]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("pairing", [kernels.ROTARY_HALVES, kernels.ROTARY_ADJACENT],
                         ids=["halves", "adjacent"])
@pytest.mark.parametrize("norm", [None, kernels.NORM_RMS, kernels.NORM_LAYER],
                         ids=["plain", "rms", "layer"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_rotary_and_norms(shape, norm, pairing, kind, cuda):
    torch = cuda
    tokens, q_heads, k_heads, dim, sections = shape
    ladder = (tokens + dim) % 2
    seed = tokens * 31 + dim
    x = normal(torch, (tokens, q_heads + k_heads, dim), seed, kind)
    q, k = x[:, :q_heads], x[:, q_heads:]
    generator = torch.Generator().manual_seed(seed + 1)
    positions = torch.randint(0, 1000, (len(sections), tokens), generator=generator,
                              dtype=torch.int32)
    positions[0, 0] = -7
    positions[-1, -1] = 2 ** 31 - 1
    positions = positions.cuda()
    problem = QkProblem(tokens, q_heads, k_heads, dim, dtype_of(kind), q_stride=x.stride(0),
                        k_stride=x.stride(0))
    rotary = kernels.rotary_axes(sections, 10000.0, pairing, ladder)
    outs = [torch.full((tokens, h, dim), float("nan"), dtype=x.dtype, device="cuda")
            for h in (q_heads, k_heads)]
    gains = [normal(torch, (dim,), seed + 2 + i, "f32", 0.3) for i in range(4)]
    if norm is None:
        kernels.launch_rotary(q, k, *outs, positions, rotary, problem)
    else:
        kernels.launch_qk_norm_rotary(q, k, *outs, QkNorm(norm, 1e-5, *gains), positions, rotary,
                                      problem)
    torch.cuda.synchronize()
    for side, out in enumerate(outs):
        y = (q, k)[side].double()
        if y.numel() == 0:
            continue
        if norm is not None:
            y = normed(torch, y, norm, 1e-5, gains[2 * side], gains[2 * side + 1])
        want = turned(torch, y, positions, sections, 10000.0, pairing, ladder)
        # The gains of a pair's two elements differ, and beta cancels: count what is added up.
        size = y.abs() if norm is None else y.abs() + 2 * gains[2 * side + 1].abs().double()
        check(out, want, rotary_bound(torch, size, want, kind, dim, norm is not None),
              f"side {side}")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("dim,shift", [(64, 0), (64, 1), (72, 4), (128, 2), (48, 8)])
def test_rotary_in_place_strided_and_unaligned(dim, shift, kind, cuda):
    """In place inside packed projection rows whose base is off any vector boundary; values,
    neighbours and padding stay untouched, and a norm without gains follows."""
    torch = cuda
    tokens, heads = 37, 3
    width = 3 * heads * dim + 5 * (shift % 2) + 8
    buffer = normal(torch, (tokens * width + shift,), 5 + shift, kind)
    before = buffer.clone()
    rows = buffer[shift:].view(tokens, width)
    q = rows[:, :heads * dim]
    k = rows[:, heads * dim:2 * heads * dim]
    positions = torch.arange(tokens, dtype=torch.int32, device="cuda").repeat(2, 3)[:, :tokens * 2]
    problem = QkProblem(tokens, heads, heads, dim, dtype_of(kind), width, width, width, width,
                        position_stride=positions.stride(0))
    rotary = kernels.rotary_axes([8, 8], 100.0, kernels.ROTARY_HALVES)
    kernels.launch_qk_norm_rotary(q, k, q, k, QkNorm(kernels.NORM_RMS, 0.0), positions, rotary,
                                  problem)
    torch.cuda.synchronize()
    old = before[shift:].view(tokens, width)
    for side in range(2):
        x = old[:, side * heads * dim:(side + 1) * heads * dim].reshape(tokens, heads, dim).double()
        y = normed(torch, x, kernels.NORM_RMS, 0.0, None, None)
        want = turned(torch, y, positions[:, :tokens], [8, 8], 100.0, kernels.ROTARY_HALVES,
                      kernels.ROTARY_LADDER_AXIS)
        got = rows[:, side * heads * dim:(side + 1) * heads * dim].reshape(tokens, heads, dim)
        check(got, want, rotary_bound(torch, y, want, kind, dim, True), f"side {side}")
    rest = torch.ones(width, dtype=torch.bool)
    rest[:2 * heads * dim] = False
    assert torch.equal(rows[:, rest.cuda()], old[:, rest.cuda()])
    assert torch.equal(buffer[:shift], before[:shift])


def test_norm_alone_and_of_one_side(cuda):
    torch = cuda
    x = normal(torch, (9, 4, 64), 3)
    x[0, 0] = 0.0  # epsilon alone keeps this head finite
    x[1, 1] += 1000.0  # a common offset must not swamp the layer norm's spread
    out = torch.empty_like(x)
    kernels.launch_qk_norm_rotary(x, None, out, None, QkNorm(kernels.NORM_LAYER, 1e-6), None, None,
                                  QkProblem(9, 4, 0, 64, kernels.DTYPE_F32))
    torch.cuda.synchronize()
    want = normed(torch, x.double(), kernels.NORM_LAYER, 1e-6, None, None)
    # Deviations x - mean carry the mean's error, 64 u32 of 1000, against a spread near 1.
    bound = torch.full_like(want, 200 * U32)
    bound[1, 1] = 200 * U32 * 1000
    check(out, want, bound)


def test_rotary_operand_on_host_is_refused(cuda):
    torch = cuda
    from cuvit.errors import InvalidArgument
    x = torch.zeros(4, 1, 8)
    out = torch.zeros(4, 1, 8, device="cuda")
    positions = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
    with pytest.raises(InvalidArgument, match="not device memory"):
        kernels.launch_rotary(x, None, out, None, positions, kernels.rotary_axes([4]),
                              QkProblem(4, 1, 0, 8, kernels.DTYPE_F32))


# ---- attention over packed sequences -------------------------------------------------------


def offsets(torch, lengths, first=0):
    total = [first]
    for length in lengths:
        total.append(total[-1] + length)
    return torch.tensor(total, dtype=torch.int32, device="cuda")


def attention_64(torch, q, k, v, queries, keys, scale, causal, kind, q0=0, k0=0):
    """Outputs in 64 bits and the bound of each: scores are off by (dim + 3) u32 of their terms'
    magnitudes (times scale and log2 e, the maximum subtracted: twice), weights by that, by the
    exponential (7.5e-5 for the bfloat16 path's polynomial, 4 u32 for float) and by their
    rounding (bfloat16: ub); the sums add at most one u32 a key and rescaling; the store rounds
    once more."""
    want = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(want)
    group = q.shape[1] // k.shape[1]
    dim = q.shape[2]
    for n_q, n_k in zip(queries, keys):
        if n_q and n_k:
            qs = q[q0:q0 + n_q].double().transpose(0, 1)
            ks = k[k0:k0 + n_k].double().repeat_interleave(group, 1).transpose(0, 1)
            vs = v[k0:k0 + n_k].double().repeat_interleave(group, 1).transpose(0, 1)
            scores = qs @ ks.transpose(1, 2) * scale
            size = qs.abs() @ ks.abs().transpose(1, 2) * scale
            if causal:
                row = torch.arange(n_q, device="cuda")[:, None] + n_k - n_q
                hidden = torch.arange(n_k, device="cuda")[None] > row
                scores = scores.masked_fill(hidden, -math.inf)
                size = size.masked_fill(hidden, 0.0)
            top = scores.amax(-1, keepdim=True)
            weights = (scores - torch.where(top.isinf(), torch.zeros_like(top), top)).exp()
            total = weights.sum(-1, keepdim=True)
            weights = torch.where(total > 0, weights / total, torch.zeros_like(weights))
            out = weights @ vs
            spread = 2 * (dim + 5) * U32 * size.amax(-1, keepdim=True)
            spread = spread + (2 * n_k + 64) * U32
            spread = spread + (2 * 7.5e-5 + UB if kind == "bf16" else 8 * U32)
            limit = spread * (weights @ vs.abs() + out.abs())
            limit = limit + (UB if kind == "bf16" else U32) * out.abs()
            want[q0:q0 + n_q] = out.transpose(0, 1)
            bound[q0:q0 + n_q] = limit.transpose(0, 1)
        q0, k0 = q0 + n_q, k0 + n_k
    return want, bound


def run_attention(torch, q, k, v, q_offsets, kv_offsets, problem, workspace=True, stream=None):
    out = torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda")
    size = kernels.attention_varlen_workspace(problem) if workspace else 0
    area = torch.full((max(size, 16),), 0xFF, dtype=torch.uint8, device="cuda")
    kernels.launch_attention_varlen(q, k, v, out, q_offsets, kv_offsets, problem,
                                    area if size else None, size, stream)
    torch.cuda.synchronize()
    return out


ATTENTION = [  # queries, keys (None: the queries), q_heads, kv_heads, dim, causal
    ([1], None, 1, 1, 64, False), ([1], None, 2, 1, 16, True), ([17], None, 2, 2, 64, False),
    ([64], None, 3, 3, 64, True), ([65, 1, 127, 128, 129], None, 2, 2, 64, False),
    ([65, 1, 127, 128, 129], None, 2, 2, 64, True), ([197] * 3, None, 3, 3, 64, False),
    ([255, 256, 257], None, 2, 1, 128, False), ([255, 256, 257], None, 2, 1, 128, True),
    ([300, 0, 20], None, 4, 2, 72, False), ([300, 0, 20], None, 4, 2, 72, True),
    ([130, 70], None, 2, 2, 80, True), ([640], None, 1, 1, 32, False), ([1025], None, 2, 2, 96, True),
    ([513, 100], None, 2, 1, 128, False), ([40, 50], None, 2, 2, 1, False),
    ([40, 50], None, 2, 2, 13, True), ([77], None, 3, 1, 100, False),
    # Other numbers of keys than queries: pooling, cross, keys or queries missing.
    ([1] * 5, [197, 1, 0, 300, 64], 4, 4, 64, False), ([1] * 3, [1000, 33, 0], 8, 2, 128, True),
    ([3, 5], [700, 100], 4, 1, 64, True), ([1], [9000], 4, 2, 64, False),
    ([2, 1], [5000, 4100], 3, 3, 72, True), ([100, 64], [30, 500], 2, 2, 64, False),
    ([100, 64], [30, 500], 2, 2, 64, True), ([200, 10], [0, 0], 2, 2, 64, False),
    ([0, 0, 5], [3, 0, 2], 2, 2, 64, False), ([300], [7], 1, 1, 128, True),
    ([260], [2600], 2, 1, 64, False), ([129], [4000], 2, 2, 128, True),
    ([12, 16], [3000, 3100], 16, 2, 96, False), ([33] * 40, None, 2, 2, 64, False)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: f"{c[0][:3]}x{len(c[0])}-{(c[1] or ['same'])[:3]}"
                         f"-{c[2]}-{c[3]}-{c[4]}-{'causal' if c[5] else 'full'}".replace(" ", ""))
def test_attention(case, kind, cuda):
    torch = cuda
    queries, keys, q_heads, kv_heads, dim, causal = case
    seed = sum(queries) + dim
    same = keys is None
    keys = queries if same else keys
    q = normal(torch, (sum(queries), q_heads, dim), seed, kind)
    k = normal(torch, (sum(keys), kv_heads, dim), seed + 1, kind)
    v = normal(torch, (sum(keys), kv_heads, dim), seed + 2, kind)
    scale = 2.0 / math.sqrt(dim)
    problem = AttentionProblem(len(queries), sum(queries), sum(keys), q_heads, kv_heads, dim,
                               dtype_of(kind), causal, scale)
    want, bound = attention_64(torch, q, k, v, queries, keys, scale, causal, kind)
    kv = None if same else offsets(torch, keys)
    for workspace in (True, False):
        got = run_attention(torch, q, k, v, offsets(torch, queries), kv, problem, workspace)
        check(got, want, bound, f"workspace {workspace}")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("dim", [64, 72, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_rows_outside_sequences(dim, causal, kind, cuda):
    """Offsets that start past zero and end before the last row: rows outside every sequence
    hold NaN in q, k and v, reach nothing, and stay as they were in the output; so do the keys
    of the other sequences, which end inside a tile."""
    torch = cuda
    queries, keys, q_first, k_first = [70, 150, 1], [90, 161, 130], 13, 37
    heads = 2
    q = normal(torch, (sum(queries) + 40, heads, dim), 1, kind)
    k = normal(torch, (sum(keys) + 60, heads, dim), 2, kind)
    v = normal(torch, (sum(keys) + 60, heads, dim), 3, kind)
    for x, first, n in ((q, q_first, sum(queries)), (k, k_first, sum(keys)), (v, k_first, sum(keys))):
        x[:first] = float("nan")
        x[first + n:] = float("inf")
    problem = AttentionProblem(3, q.shape[0], k.shape[0], heads, heads, dim, dtype_of(kind), causal,
                               0.125)
    want, bound = attention_64(torch, q, k, v, queries, keys, 0.125, causal, kind, q_first, k_first)
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    kernels.launch_attention_varlen(q, k, v, out, offsets(torch, queries, q_first),
                                    offsets(torch, keys, k_first), problem)
    torch.cuda.synchronize()
    live = slice(q_first, q_first + sum(queries))
    check(out[live], want[live], bound[live])
    assert (out[:q_first] == 7.0).all() and (out[live.stop:] == 7.0).all()
    # One sequence at a time poisons the others' keys and values.
    for poisoned in range(3):
        k2, v2 = k.clone(), v.clone()
        start = k_first + sum(keys[:poisoned])
        k2[start:start + keys[poisoned]] = float("nan")
        v2[start:start + keys[poisoned]] = float("inf")
        again = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
        kernels.launch_attention_varlen(q, k2, v2, again, offsets(torch, queries, q_first),
                                        offsets(torch, keys, k_first), problem)
        torch.cuda.synchronize()
        for s in range(3):
            rows = slice(q_first + sum(queries[:s]), q_first + sum(queries[:s + 1]))
            if s != poisoned:
                assert torch.equal(again[rows], out[rows])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("shift", [0, 1, 4, 8])
def test_attention_packed_projection_rows(shift, kind, cuda):
    """q, k and v as columns of packed projection rows at any alignment, out in wider rows."""
    torch = cuda
    heads, dim, lengths = 3, 64, [150, 47]
    tokens = sum(lengths)
    width = 3 * heads * dim + 2 * shift
    buffer = normal(torch, (tokens * width + shift,), 11, kind)
    rows = buffer[shift:].view(tokens, width)[:, :3 * heads * dim]
    q, k, v = rows.unflatten(1, (3, heads, dim)).unbind(1)
    wide = torch.full((tokens, heads * dim + shift), 3.0, dtype=q.dtype, device="cuda")
    problem = AttentionProblem(2, tokens, tokens, heads, heads, dim, dtype_of(kind), False, 0.125,
                               width, width, width, wide.shape[1])
    kernels.launch_attention_varlen(q, k, v, wide, offsets(torch, lengths), None, problem)
    torch.cuda.synchronize()
    want, bound = attention_64(torch, q, k, v, lengths, lengths, 0.125, False, kind)
    check(wide[:, :heads * dim].unflatten(1, (heads, dim)), want, bound)
    assert (wide[:, heads * dim:] == 3.0).all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("queries,keys", [([300], [300]), ([2], [3000])])
def test_attention_large_scores(queries, keys, kind, cuda):
    """Scores of +-1e4 with the largest in a late tile, and rows whose scores all lie near the
    lowest float: the running maximum has to follow without overflow."""
    torch = cuda
    dim, heads = 64, 2
    q = normal(torch, (queries[0], heads, dim), 21, kind, 40.0)
    k = normal(torch, (keys[0], heads, dim), 22, kind, 40.0)
    v = normal(torch, (keys[0], heads, dim), 23, kind)
    k[keys[0] - 5] = 3 * q[queries[0] // 2]  # one query's maximum in the last tile
    q[0] = -1e18
    k[:, 0] = k[:, 0].abs() + 1.0
    problem = AttentionProblem(1, queries[0], keys[0], heads, heads, dim, dtype_of(kind), False, 1.0)
    got = run_attention(torch, q, k, v, offsets(torch, queries), offsets(torch, keys), problem)
    assert got.isfinite().all()
    # Where the largest weight is nearly all of it, the output is that value row.
    scores = torch.einsum("qhd,khd->hqk", q.double(), k.double())
    top = scores.topk(2, -1)
    size = torch.einsum("qhd,khd->hqk", q.double().abs(), k.double().abs()).amax(-1)
    clear = top.values[..., 0] - top.values[..., 1] > 40.0 + 2 * 70 * U32 * size
    assert clear.any()
    picked = v.double().transpose(0, 1).gather(
        1, top.indices[..., :1].expand(-1, -1, dim)).transpose(0, 1)
    clear = clear.t()[..., None].expand_as(picked)
    step = (2 * UB + 1e-3) if kind == "bf16" else 64 * U32
    check(got[clear], picked[clear], step * picked[clear].abs() + 1e-9)


def test_attention_offsets_out_of_range_stay_inside(cuda):
    """Offsets past the matrices or decreasing are clamped: whatever the rows hold, nothing
    outside the output is written and the call returns."""
    torch = cuda
    for kind in TYPES:
        q = normal(torch, (64, 2, 64), 1, kind)
        guard = torch.full((192, 2, 64), 5.0, dtype=q.dtype, device="cuda")
        out = guard[64:128]
        problem = AttentionProblem(3, 64, 64, 2, 2, 64, dtype_of(kind), False, 0.125)
        for bad in ([-100, 10, 5, 1000], [0, 2 ** 31 - 1, -2 ** 31, 64], [64, 0, 64, 0]):
            bad = torch.tensor(bad, dtype=torch.int32, device="cuda")
            kernels.launch_attention_varlen(q, q, q, out, bad, None, problem)
            torch.cuda.synchronize()
            assert (guard[:64] == 5.0).all() and (guard[128:] == 5.0).all()


# ---- linear layers -------------------------------------------------------------------------


def activation_64(torch, activation, x):
    if activation == kernels.ACTIVATION_GELU:
        return x * torch.special.ndtr(x)
    if activation == kernels.ACTIVATION_GELU_TANH:
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))
    return x * torch.sigmoid(x) if activation == kernels.ACTIVATION_SILU else x


def linear_64(torch, x, w, bias, scale, residual, activation, gated, kind, out_kind, n):
    """Outputs in 64 bits and their bound. Sums: (k + 4) u32 of the terms' magnitudes, plus, for
    float operands, three roundings to 22 bits of a split product (3 2^-22). Activations have
    slopes below 1.2 and cost 32 u32 of their value (bfloat16 outputs: 2^-12), the gate's
    product, scale and residual one u32 each; then the store."""
    k = x.shape[1]
    size = x.double().abs() @ w.double().abs().t()
    y = x.double() @ w.double().t()
    error = ((k + 4) * U32 + (3 * 2.0 ** -22 if kind == "f32" else 0.0)) * size
    if bias is not None:
        y = y + bias.double()
        error = error + U32 * (y.abs() + bias.double().abs())
    value = activation_64(torch, activation, y[:, :n])
    off = 1.2 * error[:, :n]
    if activation != kernels.ACTIVATION_NONE:
        off = off + (2.0 ** -12 if out_kind == "bf16" else 32 * U32) * value.abs()
    if gated:
        off = off * (y[:, n:].abs() + error[:, n:]) + value.abs() * error[:, n:]
        value = value * y[:, n:]
        off = off + U32 * value.abs()
    if scale is not None:
        value, off = value * scale.double(), off * scale.double().abs()
        off = off + U32 * value.abs()
    if residual is not None:
        value = value + residual.double()
        off = off + U32 * (value.abs() + residual.double().abs())
    step = dict(bf16=UB, f32=U32, tf32=2.0 ** -11)[out_kind]
    return value, off * (1 + 2 * step) + step * value.abs() + 1e-30


LINEAR = [  # m, n, k
    (1, 1, 1), (1, 8, 16), (1, 1000, 192), (2, 33, 40), (3, 130, 1280), (5, 64, 72), (16, 257, 136),
    (17, 100, 64), (63, 64, 65), (64, 65, 200), (127, 129, 128), (128, 256, 64), (129, 1, 8),
    (197, 384, 192), (200, 130, 1032), (257, 520, 264), (300, 7, 15), (1000, 96, 0), (640, 1152, 72)]


@pytest.mark.parametrize("kind,out_kind", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32"),
                                           ("f32", "bf16"), ("f32", "tf32")])
@pytest.mark.parametrize("gated", [False, True], ids=["plain", "gated"])
@pytest.mark.parametrize("shape", LINEAR, ids=str)
def test_linear(shape, gated, kind, out_kind, cuda):
    torch = cuda
    m, n, k = shape
    seed = m + 3 * n + 7 * k
    activation = seed % 4
    extras = seed % 8  # bias, scale, residual in every combination over the shapes
    x = normal(torch, (m, k), seed, kind)
    w = normal(torch, ((2 if gated else 1) * n, k), seed + 1, kind, max(k, 1) ** -0.5)
    bias = normal(torch, (w.shape[0],), seed + 2) if extras & 1 else None
    scale = normal(torch, (n,), seed + 3) if extras & 2 else None
    store = "bf16" if out_kind == "bf16" else "f32"
    residual = normal(torch, (m, n), seed + 4, store) if extras & 4 else None
    out = torch.full((m, n), float("nan"), dtype=torch_type(torch, store), device="cuda")
    problem = LinearProblem(m, n, k, kernels.MATH_BF16 if kind == "bf16" else kernels.MATH_FP32,
                            dict(bf16=kernels.DTYPE_BF16, f32=kernels.DTYPE_F32,
                                 tf32=kernels.DTYPE_TF32)[out_kind], activation, gated)
    kernels.launch_linear(x, w, bias, scale, residual, out, problem)
    torch.cuda.synchronize()
    want, bound = linear_64(torch, x, w, bias, scale, residual, activation, gated, kind, out_kind, n)
    check(out, want, bound, f"activation {activation} extras {extras}")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("activation", range(4), ids=["none", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("m", [2, 130])
def test_linear_activations_over_their_range(m, activation, kind, cuda):
    """Sums from -30 to 30 in FP32 outputs and bfloat16 ones: tails as well as the middle."""
    torch = cuda
    n, k = 256, 64
    x = torch.zeros(m, k)
    x[:, 0] = 1.0
    w = torch.zeros(n, k)
    w[:, 0] = torch.linspace(-30, 30, n)
    x, w = (t.to(torch_type(torch, kind)).cuda() for t in (x, w))
    out = torch.empty(m, n, dtype=torch_type(torch, kind), device="cuda")
    problem = LinearProblem(m, n, k, kernels.MATH_BF16 if kind == "bf16" else kernels.MATH_FP32,
                            dtype_of(kind), activation, False)
    kernels.launch_linear(x, w, None, None, None, out, problem)
    torch.cuda.synchronize()
    want, bound = linear_64(torch, x, w, None, None, None, activation, False, kind, kind, n)
    check(out, want, bound + 2.0 ** -126)  # denormals may be flushed


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("m,n,k,shift", [(3, 40, 64, 1), (70, 72, 64, 1), (130, 200, 96, 2),
                                         (140, 136, 64, 8), (1, 96, 128, 4)])
def test_linear_strides_and_in_place_residual(m, n, k, shift, kind, cuda):
    torch = cuda
    x = normal(torch, (m, k + 3 * shift), 1, kind)[:, :k]
    w = normal(torch, (n, k + shift), 2, kind, 0.1)[:, :k]
    buffer = normal(torch, (m * (n + shift) + shift,), 3, kind)
    before = buffer.clone()
    rows, old = (t[shift:].view(m, n + shift) for t in (buffer, before))
    problem = LinearProblem(m, n, k, kernels.MATH_BF16 if kind == "bf16" else kernels.MATH_FP32,
                            dtype_of(kind), kernels.ACTIVATION_NONE, False, x.stride(0), w.stride(0),
                            n + shift, n + shift)
    kernels.launch_linear(x, w, None, None, rows, rows, problem)
    torch.cuda.synchronize()
    want, bound = linear_64(torch, x, w, None, None, old[:, :n], 0, False, kind, kind, n)
    check(rows[:, :n], want, bound)
    assert torch.equal(rows[:, n:], old[:, n:]) and torch.equal(buffer[:shift], before[:shift])


def test_linear_nan_rows_stay_in_their_rows(cuda):
    """A NaN row of x reaches its own output row only; a NaN gate row its own column."""
    torch = cuda
    for kind in TYPES:
        for m in (4, 200):
            x, w = normal(torch, (m, 64), 1, kind), normal(torch, (2 * 40, 64), 2, kind)
            x[1] = float("nan")
            w[3] = float("inf")
            out = torch.empty(m, 40, dtype=x.dtype, device="cuda")
            problem = LinearProblem(m, 40, 64, kernels.MATH_BF16 if kind == "bf16"
                                    else kernels.MATH_FP32, dtype_of(kind),
                                    kernels.ACTIVATION_NONE, True)
            kernels.launch_linear(x, w, None, None, None, out, problem)
            torch.cuda.synchronize()
            clean = torch.ones_like(out, dtype=torch.bool)
            clean[1] = False
            clean[:, 3] = False
            assert out[clean].isfinite().all() and not out[1].isfinite().any()


# ---- together ------------------------------------------------------------------------------


def block(torch, state, stream=None):
    """One encoder block over packed images: projection, per-head norms with rotary positions,
    attention, output projection with column scale and residual, gated feed-forward layer."""
    p, s = state["problems"], state
    kernels.launch_linear(s["x"], s["w_qkv"], s["b_qkv"], None, None, s["qkv"], p["qkv"], stream)
    q, k, v = s["qkv"].unflatten(1, (3, s["heads"], s["dim"])).unbind(1)
    kernels.launch_qk_norm_rotary(q, k, q, k, s["norm"], s["positions"], s["rotary"], p["norm"],
                                  stream)
    kernels.launch_attention_varlen(q, k, v, s["context"], s["offsets"], None, p["attention"],
                                    s["workspace"], s["workspace"].numel(), stream)
    kernels.launch_linear(s["context"], s["w_out"], s["b_out"], s["scale"], s["x"], s["y"],
                          p["out"], stream)
    kernels.launch_linear(s["y"], s["w_gate"], s["b_gate"], None, None, s["hidden"], p["gate"],
                          stream)
    kernels.launch_linear(s["hidden"], s["w_down"], None, s["scale"], s["y"], s["y"], p["down"],
                          stream)
    return s["y"]


def block_state(torch, kind, lengths, heads=4, dim=64, hidden=344, seed=0):
    width, tokens = heads * dim, sum(lengths)
    math_mode = kernels.MATH_BF16 if kind == "bf16" else kernels.MATH_FP32
    dtype = dtype_of(kind)

    def linear(n, k, **more):
        return LinearProblem(tokens, n, k, math_mode, dtype, **more)

    def empty(*shape):
        return torch.empty(shape, dtype=torch_type(torch, kind), device="cuda")

    s = dict(heads=heads, dim=dim, x=normal(torch, (tokens, width), seed, kind),
             w_qkv=normal(torch, (3 * width, width), seed + 1, kind, width ** -0.5),
             b_qkv=normal(torch, (3 * width,), seed + 2),
             w_out=normal(torch, (width, width), seed + 3, kind, width ** -0.5),
             b_out=normal(torch, (width,), seed + 4), scale=normal(torch, (width,), seed + 5),
             w_gate=normal(torch, (2 * hidden, width), seed + 6, kind, width ** -0.5),
             b_gate=normal(torch, (2 * hidden,), seed + 7),
             w_down=normal(torch, (width, hidden), seed + 8, kind, hidden ** -0.5),
             qkv=empty(tokens, 3 * width), context=empty(tokens, width), y=empty(tokens, width),
             hidden=empty(tokens, hidden), offsets=offsets(torch, lengths),
             rotary=kernels.rotary_axes([dim // 4, dim // 4]),
             positions=torch.stack([torch.cat([torch.arange(n) // 16 for n in lengths]),
                                    torch.cat([torch.arange(n) % 16 for n in lengths])]).to(
                                        torch.int32).cuda())
    gains = [normal(torch, (dim,), seed + 9 + i, "f32", 0.2) + 1.0 for i in range(2)]
    s["gains"] = gains
    s["norm"] = QkNorm(kernels.NORM_RMS, 1e-6, gains[0], None, gains[1], None)
    s["problems"] = dict(
        qkv=linear(3 * width, width),
        norm=QkProblem(tokens, heads, heads, dim, dtype, 3 * width, 3 * width, 3 * width, 3 * width),
        attention=AttentionProblem(len(lengths), tokens, tokens, heads, heads, dim, dtype, False,
                                   dim ** -0.5, 3 * width, 3 * width, 3 * width),
        out=linear(width, width), gate=linear(hidden, width, activation=kernels.ACTIVATION_SILU,
                                              gated=True), down=linear(width, hidden))
    s["workspace"] = torch.empty(
        max(16, kernels.attention_varlen_workspace(s["problems"]["attention"])), dtype=torch.uint8,
        device="cuda")
    return s


def block_64(torch, s, lengths):
    heads, dim = s["heads"], s["dim"]
    d = {key: value.double() for key, value in s.items()
         if torch.is_tensor(value) and value.is_floating_point()}
    qkv = (d["x"] @ d["w_qkv"].t() + d["b_qkv"]).unflatten(1, (3, heads, dim))
    q, k = (turned(torch, normed(torch, qkv[:, i], kernels.NORM_RMS, 1e-6, s["gains"][i], None),
                   s["positions"], [dim // 4, dim // 4], 10000.0, kernels.ROTARY_HALVES,
                   kernels.ROTARY_LADDER_AXIS) for i in range(2))
    context, start = [], 0
    for n in lengths:
        part = slice(start, start + n)
        weights = torch.softmax(torch.einsum("qhd,khd->hqk", q[part], k[part]) * dim ** -0.5, -1)
        context.append(torch.einsum("hqk,khd->qhd", weights, qkv[part, 2]))
        start += n
    y = d["x"] + d["scale"] * (torch.cat(context).flatten(1) @ d["w_out"].t() + d["b_out"])
    gate, up = (y @ d["w_gate"].t() + d["b_gate"]).chunk(2, 1)
    return y + d["scale"] * ((gate * torch.sigmoid(gate) * up) @ d["w_down"].t())


@pytest.mark.parametrize("kind", TYPES)
def test_block_of_all_four(kind, cuda):
    """The chain as an encoder runs it. Six stages each round their outputs once (a relative step
    u of values near 1 to 4); a stage passes errors on with a gain of at most about 3 in RMS
    (gate: |silu' up| + |silu|): the RMS error stays below 40 u, and the first-order 64-bit
    chain is the reference."""
    torch = cuda
    lengths = [49, 197, 1, 130, 256]
    s = block_state(torch, kind, lengths)
    want = block_64(torch, s, lengths)
    got = block(torch, s).double()
    torch.cuda.synchronize()
    step = UB if kind == "bf16" else 64 * U32
    rms = (got - want).square().mean().sqrt() / want.square().mean().sqrt()
    assert rms <= 40 * step and got.isfinite().all()


@pytest.mark.parametrize("kind", TYPES)
def test_block_captured_and_replayed(kind, cuda):
    """Captured in a CUDA graph and replayed on new inputs, the block gives bitwise what eager
    calls give; eager calls on a second stream run beside it."""
    torch = cuda
    lengths = [80, 300, 17]
    eager, captured, beside = (block_state(torch, kind, lengths, seed=7) for _ in range(3))
    block(torch, captured)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block(torch, captured, torch.cuda.current_stream())
    other = torch.cuda.Stream()
    for seed in (100, 200):
        x = normal(torch, eager["x"].shape, seed, kind)
        for state in (eager, captured, beside):
            state["x"].copy_(x)
        torch.cuda.synchronize()
        graph.replay()
        block(torch, beside, other)
        torch.cuda.synchronize()
        block(torch, eager)
        torch.cuda.synchronize()
        for state in (captured, beside):
            assert torch.equal(state["y"], eager["y"])
            assert torch.equal(state["context"], eager["context"])


def test_linear_f32_special_values(cuda):
    """Operands are split into TF32 values: infinities, NaN and the largest float among them."""
    torch = cuda
    m, n, k = 140, 150, 68
    gen = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(m, k, device="cuda", generator=gen)
    w = torch.randn(n, k, device="cuda", generator=gen)
    x[3, 7] = float("nan")
    x[130, 67] = float("inf")
    w[149, 1] = float("nan")
    largest = torch.finfo(torch.float32).max
    x[5] = 0.0
    x[5, 9] = largest
    w[:, 9] = 0.5 * torch.sign(w[:, 9])
    out = torch.empty(m, n, device="cuda")
    torch.cuda.synchronize()
    kernels.launch_linear(x, w, None, None, None, out,
                          LinearProblem(m=m, n=n, k=k, math=kernels.MATH_FP32,
                                        out_dtype=kernels.DTYPE_F32))
    torch.cuda.synchronize()
    assert out[3].isnan().all() and out[:, 149].isnan().all()
    assert not out[130, :149].isfinite().any()
    rows = [r for r in range(m) if r not in (3, 130)]
    assert out[rows, :149].isfinite().all()
    # The head of the largest float is cut, not rounded to infinity: 2^-10 remain to the rest,
    # which the tensor core holds to 2^-11 of that.
    expected = largest * w[:149, 9].double()
    error = (out[5, :149].double() - expected).abs()
    assert (error <= 2.0 ** -20 * expected.abs()).all()


@pytest.mark.parametrize("k", [60, 1000, 16388])
def test_linear_f32_long_rows(k, cuda):
    torch = cuda
    m, n = 200, 170
    gen = torch.Generator(device="cuda").manual_seed(k)
    # All products positive: what a summation loses in one direction adds up.
    x = torch.rand(m, k, device="cuda", generator=gen)
    w = torch.rand(n, k, device="cuda", generator=gen)
    out = torch.empty(m, n, device="cuda")
    torch.cuda.synchronize()
    kernels.launch_linear(x, w, None, None, None, out,
                          LinearProblem(m=m, n=n, k=k, math=kernels.MATH_FP32,
                                        out_dtype=kernels.DTYPE_F32))
    torch.cuda.synchronize()
    exact = x.double() @ w.double().T
    # Operands: 2^-23 each, and the product of the remainders, 2^-22. 64 of k in the accumulator:
    # 24 additions, each cutting off less than 2^-23 of the partial sum, which grows from 0 to the
    # whole: half of 24 2^-23. Then k / 64 additions rounded to 2^-24 of a sum that grows from 0
    # to the whole: half of k / 64 2^-24, at most.
    bound = 4 * 2.0 ** -23 + 13 * 2.0 ** -23 + (k / 128 + 1) * 2.0 ** -24
    assert ((out.double() - exact).abs() <= bound * exact).all()


# ---- calls around the edges ----------------------------------------------------------------


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("group", [1, 3, 5, 8, 16])
def test_attention_many_ragged_causal_sequences(group, kind, cuda):
    """More sequences than are ordered by length, some empty, some of one token."""
    torch = cuda
    lengths = [(17 * i * i) % 211 for i in range(45)] + [1, 0, 400]
    dim, kv_heads = 64, 2
    tokens = sum(lengths)
    q = normal(torch, (tokens, kv_heads * group, dim), 1, kind)
    k, v = (normal(torch, (tokens, kv_heads, dim), seed, kind) for seed in (2, 3))
    problem = AttentionProblem(len(lengths), tokens, tokens, kv_heads * group, kv_heads, dim,
                               dtype_of(kind), True, 0.2)
    want, bound = attention_64(torch, q, k, v, lengths, lengths, 0.2, True, kind)
    got = run_attention(torch, q, k, v, offsets(torch, lengths), None, problem)
    check(got, want, bound)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("group,queries", [(1, 8), (2, 3), (3, 2), (5, 1), (7, 1), (8, 1), (3, 1)])
@pytest.mark.parametrize("dim", [8, 40, 64, 88, 128])
def test_attention_few_rows(group, queries, dim, kind, cuda):
    """Every division of eight rows into queries and heads, lengths on both sides of the steps."""
    torch = cuda
    keys = [1, 15, 16, 17, 33, 64, 65, 700, 0, 5]
    rows = [queries] * len(keys)
    kv_heads = 2
    q = normal(torch, (sum(rows), kv_heads * group, dim), 4, kind)
    k, v = (normal(torch, (sum(keys), kv_heads, dim), seed, kind) for seed in (5, 6))
    for causal in (False, True):
        problem = AttentionProblem(len(keys), sum(rows), sum(keys), kv_heads * group, kv_heads, dim,
                                   dtype_of(kind), causal, 0.3)
        want, bound = attention_64(torch, q, k, v, rows, keys, 0.3, causal, kind)
        got = run_attention(torch, q, k, v, offsets(torch, rows), offsets(torch, keys), problem)
        check(got, want, bound, f"causal {causal}")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("queries", [1, 150])
def test_attention_offsets_past_32_bits(queries, kind, cuda):
    """Rows whose element offsets pass 2^32: the keys of the last sequence lie there."""
    torch = cuda
    stride, tokens, heads, dim = 2 ** 16, 70000, 1, 64
    rows = torch.empty(tokens * stride, dtype=torch_type(torch, kind), device="cuda").view(tokens,
                                                                                          stride)
    keys = [tokens - 200, 200]
    live = rows[tokens - 200:]
    live[:, :dim] = normal(torch, (200, dim), 1, kind)
    live[:, dim:2 * dim] = normal(torch, (200, dim), 2, kind)
    k, v = rows[:, :dim].unsqueeze(1), rows[:, dim:2 * dim].unsqueeze(1)
    q = normal(torch, (queries, heads, dim), 3, kind)
    problem = AttentionProblem(2, queries, tokens, heads, heads, dim, dtype_of(kind), False, 0.125,
                               0, stride, stride)
    want, bound = attention_64(torch, q, k[tokens - 200:], v[tokens - 200:], [queries], [200], 0.125,
                               False, kind)
    got = run_attention(torch, q, k, v, offsets(torch, [0, queries]), offsets(torch, keys), problem)
    check(got, want, bound)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("queries", [1, 100])
def test_attention_split_calls_on_two_streams(queries, kind, cuda):
    """Calls that split their keys, at the same time and captured, each with its own workspace."""
    torch = cuda
    dim, heads, keys = 64, 4, 6000
    problem = AttentionProblem(1, queries, keys, heads, heads, dim, dtype_of(kind), False, 0.125)
    size = kernels.attention_varlen_workspace(problem)
    assert size > 0
    q_offsets, kv_offsets = offsets(torch, [queries]), offsets(torch, [keys])
    sides = []
    for seed in (1, 2):
        q = normal(torch, (queries, heads, dim), seed, kind)
        k, v = (normal(torch, (keys, heads, dim), 10 * seed + i, kind) for i in range(2))
        sides.append(dict(q=q, k=k, v=v, out=torch.empty_like(q),
                          area=torch.empty(size, dtype=torch.uint8, device="cuda")))

    def launch(side, stream):
        kernels.launch_attention_varlen(side["q"], side["k"], side["v"], side["out"], q_offsets,
                                        kv_offsets, problem, side["area"], size, stream)

    want = []
    for side in sides:
        launch(side, None)
        torch.cuda.synchronize()
        want.append(side["out"].clone())
    streams = [torch.cuda.Stream() for _ in sides]
    for _ in range(20):
        for side, stream in zip(sides, streams):
            launch(side, stream)
    torch.cuda.synchronize()
    for side, expected in zip(sides, want):
        assert torch.equal(side["out"], expected)
    graphs = []
    for side in sides:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            launch(side, torch.cuda.current_stream())
        side["out"].zero_()
        side["area"].fill_(0xFF)
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for side, expected in zip(sides, want):
        assert torch.equal(side["out"], expected)


def test_attention_workspace_refusals(cuda):
    torch = cuda
    problem = AttentionProblem(1, 1, 9000, 2, 2, 64, kernels.DTYPE_BF16, False, 0.125)
    size = kernels.attention_varlen_workspace(problem)
    q = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(9000, 2, 64, dtype=torch.bfloat16, device="cuda")
    area = torch.empty(size + 16, dtype=torch.uint8, device="cuda")
    one, many = offsets(torch, [1]), offsets(torch, [9000])
    out = torch.zeros_like(q)
    for workspace, given in ((area, 16), (area[1:], size), (k, size), (area.cpu(), size)):
        with pytest.raises(InvalidArgument):
            kernels.launch_attention_varlen(q, k, k, out, one, many, problem, workspace, given)
    torch.cuda.synchronize()
    assert (out == 0).all()


def test_operands_of_another_device_are_refused(cuda):
    torch = cuda
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    x = torch.zeros(4, 1, 8, device="cuda:1")
    out = torch.zeros(4, 1, 8, device="cuda:0")
    with torch.cuda.device(0), pytest.raises(InvalidArgument, match="another device"):
        kernels.launch_rotary(x, None, out, None, torch.zeros(4, dtype=torch.int32, device="cuda:0"),
                              kernels.rotary_axes([4]), QkProblem(4, 1, 0, 8, kernels.DTYPE_F32))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("gated", [False, True], ids=["plain", "gated"])
@pytest.mark.parametrize("m,n,k", [(9, 48, 64), (12, 16, 4), (15, 145, 96), (128, 289, 32),
                                   (130, 1000, 260), (2000, 100, 64)])
def test_linear_around_the_tiles(m, n, k, gated, kind, cuda):
    """Tile widths from one step of columns to the widest, all with every optional operand."""
    torch = cuda
    x = normal(torch, (m, k), 1, kind)
    w = normal(torch, ((2 if gated else 1) * n, k), 2, kind, k ** -0.5)
    bias = normal(torch, (w.shape[0],), 3)
    scale = normal(torch, (n,), 4)
    residual = normal(torch, (m, n), 5, kind)
    out = torch.empty_like(residual)
    math_mode = kernels.MATH_BF16 if kind == "bf16" else kernels.MATH_FP32
    kernels.launch_linear(x, w, bias, scale, residual, out,
                          LinearProblem(m, n, k, math_mode, dtype_of(kind), kernels.ACTIVATION_GELU,
                                        gated))
    torch.cuda.synchronize()
    want, bound = linear_64(torch, x, w, bias, scale, residual, kernels.ACTIVATION_GELU, gated, kind,
                            kind, n)
    check(out, want, bound)


@pytest.mark.parametrize("kind,out_kind", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32"),
                                           ("f32", "bf16")])
@pytest.mark.parametrize("gated", [False, True], ids=["plain", "gated"])
@pytest.mark.parametrize("m,n,k", [(9, 1000, 4104), (16, 64, 512), (33, 200, 2048), (128, 31, 1024),
                                   (130, 70, 1160), (197, 768, 3848), (300, 130, 520), (12, 9, 8192)])
def test_linear_with_divided_k(m, n, k, gated, kind, out_kind, cuda):
    """Few tiles and a long k: the CTAs of a cluster share a tile. Twice, bitwise the same."""
    torch = cuda
    x = normal(torch, (m, k), 1, kind)
    w = normal(torch, ((2 if gated else 1) * n, k), 2, kind, k ** -0.5)
    bias = normal(torch, (w.shape[0],), 3)
    scale = normal(torch, (n,), 4)
    residual = normal(torch, (m, n), 5, out_kind)
    outs = [torch.full((m, n), float("nan"), dtype=torch_type(torch, out_kind), device="cuda")
            for _ in range(2)]
    math_mode = kernels.MATH_BF16 if kind == "bf16" else kernels.MATH_FP32
    for out in outs:
        kernels.launch_linear(x, w, bias, scale, residual, out,
                              LinearProblem(m, n, k, math_mode, dtype_of(out_kind),
                                            kernels.ACTIVATION_SILU, gated))
    torch.cuda.synchronize()
    want, bound = linear_64(torch, x, w, bias, scale, residual, kernels.ACTIVATION_SILU, gated, kind,
                            out_kind, n)
    check(outs[0], want, bound)
    assert torch.equal(*outs)


@pytest.mark.parametrize("kind", TYPES)
def test_linear_with_divided_k_captured_beside_others(kind, cuda):
    """Clusters on two streams at once, captured and replayed on new inputs."""
    torch = cuda
    m, n, k = 40, 300, 4096
    math_mode = kernels.MATH_BF16 if kind == "bf16" else kernels.MATH_FP32
    problem = LinearProblem(m, n, k, math_mode, dtype_of(kind))
    sides = [dict(x=normal(torch, (m, k), seed, kind), w=normal(torch, (n, k), seed + 1, kind, 0.02),
                  out=torch.zeros(m, n, dtype=torch_type(torch, kind), device="cuda"),
                  stream=torch.cuda.Stream(), graph=torch.cuda.CUDAGraph()) for seed in (1, 3)]
    torch.cuda.synchronize()
    for side in sides:
        with torch.cuda.graph(side["graph"]):
            kernels.launch_linear(side["x"], side["w"], None, None, None, side["out"], problem,
                                  torch.cuda.current_stream())
    for side in sides:
        side["x"].copy_(normal(torch, (m, k), 9, kind))
    torch.cuda.synchronize()
    for _ in range(10):
        for side in sides:
            with torch.cuda.stream(side["stream"]):
                side["graph"].replay()
    torch.cuda.synchronize()
    for side in sides:
        want, bound = linear_64(torch, side["x"], side["w"], None, None, None, 0, False, kind, kind, n)
        check(side["out"], want, bound)


@pytest.mark.parametrize("gated", [False, True], ids=["plain", "gated"])
@pytest.mark.parametrize("m,n,k", [(3, 40, 64), (130, 200, 72), (700, 300, 500), (40, 33, 30)])
def test_linear_tf32(m, n, k, gated, cuda):
    """One product of TF32 values: each operand keeps 11 bits, cut off at most: 2^-10 of it, twice.
    Few rows and rows that are not whole 16-byte vectors have FP32 products, which is within that."""
    torch = cuda
    x, residual = normal(torch, (m, k), 1, "f32"), normal(torch, (m, n), 2, "f32")
    w = normal(torch, ((2 if gated else 1) * n, k), 3, "f32")
    out = torch.empty_like(residual)
    kernels.launch_linear(x, w, None, None, residual, out,
                          LinearProblem(m, n, k, kernels.MATH_TF32, kernels.DTYPE_F32,
                                        kernels.ACTIVATION_NONE, gated))
    torch.cuda.synchronize()
    y = x.double() @ w.double().t()
    # The sum's k additions cut off less than 2^-23 of the partial sums each.
    error = (2.0 ** -9 + 2.0 ** -20 + (k + 4) * 2.0 ** -23) * (x.double().abs() @ w.double().abs().t())
    value, off = y[:, :n], error[:, :n]
    if gated:
        off = off * (y[:, n:].abs() + error[:, n:]) + value.abs() * error[:, n:]
        value = value * y[:, n:]
    want = value + residual.double()
    check(out, want, off + 4 * U32 * (value.abs() + residual.double().abs()))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("dim", [3, 9, 17, 24, 33, 48, 56, 65, 81, 88, 104, 112, 113, 120, 127])
def test_attention_head_widths(dim, kind, cuda):
    """Widths on both sides of the kernels' groups of columns, with and without whole vectors."""
    torch = cuda
    lengths, heads = [130, 40, 67, 1], 2
    q, k, v = (normal(torch, (sum(lengths), heads, dim), seed, kind) for seed in (1, 2, 3))
    for causal in (False, True):
        problem = AttentionProblem(len(lengths), sum(lengths), sum(lengths), heads, heads, dim,
                                   dtype_of(kind), causal, dim ** -0.5)
        want, bound = attention_64(torch, q, k, v, lengths, lengths, dim ** -0.5, causal, kind)
        got = run_attention(torch, q, k, v, offsets(torch, lengths), None, problem)
        check(got, want, bound, f"causal {causal}")
