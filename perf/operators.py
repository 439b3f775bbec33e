"""What the operators of an encoder block over packed images and videos cost.

The four operators and the calls a user makes of them:

* rotary positions with several axes (time, height, width) on queries and keys,
* per-head norms of queries and keys with that rotation in the same pass,
* attention over packed sequences of any length,
* a linear layer with bias, activation (gated too), column scale and residual.

`run` computes them either in plain 32-bit torch operations (`own = False`) or through the
library's entry points (`own = True`); `exact` is the definition in 64 bits.
"""

import math
import os
import sys

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _library():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                           "cu-vit_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from cuvit import kernels
    return kernels


# ---- cases --------------------------------------------------------------------------------

def listed():
    return [
        # One new token of a 12-head model: nothing but latency.
        dict(name="rotary-token", op="rotary", type="bf16", tokens=1, heads=12, kv_heads=12,
             dim=64, sections="32", pairing="halves", ladder="shared", reach=5000),
        # A clip: 16 frames of 28 x 28 patches, time / height / width, queries and keys of 16
        # heads of 80 taken out of packed projection rows.
        dict(name="rotary-clip", op="rotary", type="bf16", tokens=12544, heads=16, kv_heads=16,
             dim=80, sections="8+16+16", pairing="halves", ladder="axis", reach=64),
        # 256 images of the base model (197 tokens, 12 heads of 64), RMS norms.
        dict(name="norm-batch", op="norm", type="bf16", tokens=50432, heads=12, kv_heads=12,
             dim=64, sections="16+16", pairing="halves", ladder="axis", reach=64, norm="rms"),
        # A ragged float batch, heads of 72 with part of each head left unturned, fewer key heads.
        dict(name="norm-ragged-f32", op="norm", type="f32", tokens=5003, heads=16, kv_heads=4,
             dim=72, sections="16+16", pairing="halves", ladder="axis", reach=64, norm="layer"),
        # One new token over a long context with shared key heads: split over the keys.
        dict(name="attention-token", op="attention", type="bf16", queries="1*2",
             keys="16001+9000", heads=16, kv_heads=4, dim=128, causal=True),
        # Images in their own sizes packed into one batch.
        dict(name="attention-mixed", op="attention", type="bf16",
             queries="4096+196+1369*2+2500+729+64*8+1023+3025", heads=16,
             kv_heads=16, dim=72, causal=False),
        # A long clip, one sequence.
        dict(name="attention-clip", op="attention", type="bf16", queries="16384",
             heads=16, kv_heads=16, dim=128, causal=False),
        # Float activations: 8 images of the base model.
        dict(name="attention-f32", op="attention", type="f32", queries="197*8",
             heads=12, kv_heads=12, dim=64, causal=False),
        # One token through a gated layer: weights streamed once.
        dict(name="linear-token-gated", op="linear", type="bf16", m=1, n=4096, k=1280,
             activation="silu", gated=True, bias=False, scale=False, residual=False),
        # A gated layer over a packed batch, ragged rows and columns.
        dict(name="linear-gated", op="linear", type="bf16", m=16411, n=3420, k=1280,
             activation="silu", gated=True, bias=True, scale=False, residual=False),
        # The output projection of 256 images of the base model: bias, column scale, residual.
        dict(name="linear-residual", op="linear", type="bf16", m=50432, n=768, k=768,
             activation="none", gated=False, bias=True, scale=True, residual=True),
        # The small model's first feed-forward layer over 8 images in float.
        dict(name="linear-f32", op="linear", type="f32", m=1576, n=1536, k=384,
             activation="gelu", gated=False, bias=True, scale=False, residual=False),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rotary", "norm", "attention", "linear"])
    kind = "f32" if rng.random() < 0.25 else "bf16"
    if op in ("rotary", "norm"):
        dim = rng.choice([32, 64, 72, 80, 96, 128])
        heads = rng.choice([3, 6, 8, 12, 16, 24])
        axes = rng.choice([1, 2, 3])
        # Even sections of up to the whole head; what is left over of a head is not turned.
        unit = dim // 2 // (4 * axes) * 4
        case = dict(op=op, type=kind, tokens=_spread(rng, 1, 30000), heads=heads,
                    kv_heads=rng.choice([heads, heads, 1]), dim=dim,
                    sections="+".join([str(max(unit, 4))] * axes),
                    pairing=rng.choice(["halves", "adjacent"]),
                    ladder=rng.choice(["axis", "shared"]), reach=_spread(rng, 16, 100000))
        if op == "norm":
            case["norm"] = rng.choice(["rms", "layer"])
        return case
    if op == "attention":
        dim = rng.choice([32, 64, 72, 80, 96, 128])
        heads = rng.choice([4, 8, 12, 16])
        count = _spread(rng, 1, 64)
        causal = rng.random() < 0.3
        single = rng.random() < 0.3
        longest = 20000 if single else (4000 if kind == "f32" else 12000)
        budget = longest  # keys of the whole batch
        keys = []
        for _ in range(count):
            if budget < 1:
                break
            keys.append(min(_spread(rng, 1, longest), budget))
            budget -= keys[-1]
        keys = "+".join(map(str, keys))
        return dict(op=op, type=kind,
                    queries="1*%d" % len(keys.split("+")) if single else keys, keys=keys,
                    heads=heads, kv_heads=rng.choice([heads, heads, heads // 2, heads // 4]),
                    dim=dim, causal=causal)
    # Linear layers: widths of a model (multiples of 8 in), any number of columns out.
    m, k = _spread(rng, 1, 30000), 8 * _spread(rng, 8, 640)
    n = _spread(rng, 32, 6000)
    while 2.0 * m * n * k > 1.2e11 * (1 if kind == "bf16" else 0.25):
        m = max(1, m // 2)
    gated = rng.random() < 0.4
    return dict(op="linear", type=kind, m=m, n=n, k=k,
                activation=rng.choice(["none", "gelu", "gelu_tanh", "silu"]), gated=gated,
                bias=rng.random() < 0.7, scale=rng.random() < 0.4, residual=rng.random() < 0.5)


def _lengths(text):
    out = []
    for part in text.split("+"):
        value, _, times = part.partition("*")
        out += [int(value)] * int(times or 1)
    return out


def _sequences(case):
    queries = _lengths(case["queries"])
    return queries, _lengths(case["keys"]) if "keys" in case else queries


def _sections(case):
    return [int(x) for x in case["sections"].split("+")]


# ---- inputs -------------------------------------------------------------------------------

def _normal(shape, seed, kind, std=1.0):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=generator, device="cuda") * std).to(TYPES[kind])


def _offsets(lengths):
    total = [0]
    for length in lengths:
        total.append(total[-1] + length)
    return torch.tensor(total, dtype=torch.int32, device="cuda")


def _prepare(case, seed):
    """The tensors alone; `exact` starts from these too."""
    kind, seed = case["type"], seed * 16 + 1
    state = {}
    if case["op"] in ("rotary", "norm"):
        heads = case["heads"] + 2 * case["kv_heads"]
        # Rows as a projection leaves them: queries, keys and values of one token.
        state["qkv"] = _normal((case["tokens"], heads, case["dim"]), seed, kind)
        generator = torch.Generator(device="cuda").manual_seed(seed + 1)
        state["positions"] = torch.randint(0, case["reach"],
                                           (len(_sections(case)), case["tokens"]),
                                           generator=generator, device="cuda", dtype=torch.int32)
        if case["op"] == "norm":
            for i, name in enumerate(("q_gamma", "q_beta", "k_gamma", "k_beta")):
                if name.endswith("gamma") or case["norm"] == "layer":
                    value = _normal((case["dim"],), seed + 2 + i, "f32", 0.2)
                    state[name] = value + 1.0 if name.endswith("gamma") else value
    elif case["op"] == "attention":
        queries, keys = _sequences(case)
        state["q"] = _normal((sum(queries), case["heads"], case["dim"]), seed, kind)
        state["k"] = _normal((sum(keys), case["kv_heads"], case["dim"]), seed + 1, kind)
        state["v"] = _normal((sum(keys), case["kv_heads"], case["dim"]), seed + 2, kind)
        state["q_offsets"], state["kv_offsets"] = _offsets(queries), _offsets(keys)
    else:
        rows = case["n"] * (2 if case["gated"] else 1)
        state["x"] = _normal((case["m"], case["k"]), seed, kind)
        state["w"] = _normal((rows, case["k"]), seed + 1, kind, case["k"] ** -0.5)
        if case["bias"]:
            state["bias"] = _normal((rows,), seed + 2, "f32", 0.5)
        if case["scale"]:
            state["scale"] = _normal((case["n"],), seed + 3, "f32", 0.5)
        if case["residual"]:
            state["residual"] = _normal((case["m"], case["n"]), seed + 4, kind)
    return state


def prepare(case, seed):
    state = _prepare(case, seed)
    state["case"] = case
    if own:
        _plan(state)
    return state


# ---- the library's kernels ----------------------------------------------------------------

def _plan(state):
    """What a program keeps between calls: the problem, the output buffers, the workspace."""
    kernels, case = _library(), state["case"]
    dtype = kernels.DTYPE_BF16 if case["type"] == "bf16" else kernels.DTYPE_F32
    kind = TYPES[case["type"]]
    if case["op"] in ("rotary", "norm"):
        h, g, d = case["heads"], case["kv_heads"], case["dim"]
        stride = (h + 2 * g) * d
        state["problem"] = kernels.QkProblem(tokens=case["tokens"], q_heads=h, k_heads=g,
                                             head_dim=d, dtype=dtype, q_stride=stride,
                                             k_stride=stride)
        state["rotary"] = kernels.rotary_axes(
            _sections(case), base=10000.0,
            pairing=kernels.ROTARY_HALVES if case["pairing"] == "halves"
            else kernels.ROTARY_ADJACENT,
            ladder=kernels.ROTARY_LADDER_AXIS if case["ladder"] == "axis"
            else kernels.ROTARY_LADDER_SHARED)
        state["q_in"], state["k_in"] = state["qkv"][:, :h], state["qkv"][:, h:h + g]
        state["q_out"] = torch.empty((case["tokens"], h, d), dtype=kind, device="cuda")
        state["k_out"] = torch.empty((case["tokens"], g, d), dtype=kind, device="cuda")
        if case["op"] == "norm":
            state["norm"] = kernels.QkNorm(
                kind=kernels.NORM_RMS if case["norm"] == "rms" else kernels.NORM_LAYER,
                epsilon=1e-6, q_gamma=state["q_gamma"], q_beta=state.get("q_beta"),
                k_gamma=state["k_gamma"], k_beta=state.get("k_beta"))
    elif case["op"] == "attention":
        queries, keys = _sequences(case)
        state["problem"] = kernels.AttentionProblem(
            batch=len(queries), q_tokens=sum(queries), kv_tokens=sum(keys),
            q_heads=case["heads"], kv_heads=case["kv_heads"], head_dim=case["dim"], dtype=dtype,
            scale=case["dim"] ** -0.5, causal=case["causal"])
        state["out"] = torch.empty_like(state["q"])
        state["workspace"] = torch.empty(
            max(kernels.attention_varlen_workspace(state["problem"]), 1), dtype=torch.uint8,
            device="cuda")
    else:
        activation = dict(none=kernels.ACTIVATION_NONE, gelu=kernels.ACTIVATION_GELU,
                          gelu_tanh=kernels.ACTIVATION_GELU_TANH, silu=kernels.ACTIVATION_SILU)
        state["problem"] = kernels.LinearProblem(
            m=case["m"], n=case["n"], k=case["k"],
            math=kernels.MATH_BF16 if case["type"] == "bf16" else kernels.MATH_FP32,
            out_dtype=dtype, activation=activation[case["activation"]], gated=case["gated"])
        state["out"] = torch.empty((case["m"], case["n"]), dtype=kind, device="cuda")


def _run_own(state):
    kernels, case = _library(), state["case"]
    stream = torch.cuda.current_stream()
    if case["op"] == "rotary":
        kernels.launch_rotary(state["q_in"], state["k_in"], state["q_out"], state["k_out"],
                              state["positions"], state["rotary"], state["problem"], stream)
        return [state["q_out"], state["k_out"]]
    if case["op"] == "norm":
        kernels.launch_qk_norm_rotary(state["q_in"], state["k_in"], state["q_out"],
                                      state["k_out"], state["norm"], state["positions"],
                                      state["rotary"], state["problem"], stream)
        return [state["q_out"], state["k_out"]]
    if case["op"] == "attention":
        kernels.launch_attention_varlen(state["q"], state["k"], state["v"], state["out"],
                                        state["q_offsets"], state["kv_offsets"],
                                        state["problem"], state["workspace"],
                                        state["workspace"].numel(), stream)
        return state["out"]
    kernels.launch_linear(state["x"], state["w"], state.get("bias"), state.get("scale"),
                          state.get("residual"), state["out"], state["problem"], stream)
    return state["out"]


# ---- plain forms --------------------------------------------------------------------------

def _plain_tables(case, positions):
    """cos and sin [tokens, 1, pairs] in 64-bit angles, held in 32 bits."""
    sections = _sections(case)
    total, angles = sum(sections), []
    for axis, pairs in enumerate(sections):
        index = torch.arange(pairs, device="cuda", dtype=torch.float64)
        if case["ladder"] == "axis":
            exponent = index / pairs
        else:
            exponent = (index + sum(sections[:axis])) / total
        frequency = torch.exp(exponent * -math.log(10000.0))
        angles.append(positions[axis].double()[:, None] * frequency)
    angle = torch.cat(angles, 1)[:, None]
    return torch.cos(angle).float(), torch.sin(angle).float()


def _plain_turn(case, x, cos, sin):
    half = cos.shape[-1]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if case["pairing"] == "halves":
        a, b = turned[..., :half], turned[..., half:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, rest], -1)
    a, b = turned[..., 0::2], turned[..., 1::2]
    both = torch.stack([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([both.flatten(-2), rest], -1)


def _plain_norm(case, x, gamma, beta):
    if case["norm"] == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * gamma
    return x if beta is None else x + beta


def _plain_attention(case, state):
    queries, keys = _sequences(case)
    group = case["heads"] // case["kv_heads"]
    out = torch.empty_like(state["q"])
    if len(set(queries)) == 1 and len(set(keys)) == 1:
        # Equal lengths: one batch of matrices.
        pieces = [(0, len(queries), 0, queries[0], keys[0])]
    else:
        pieces, q0, k0 = [], 0, 0
        for n_q, n_k in zip(queries, keys):
            pieces.append((q0, 1, k0, n_q, n_k))
            q0, k0 = q0 + n_q, k0 + n_k
    for q0, count, k0, n_q, n_k in pieces:
        if n_q == 0:
            continue
        # Whole heads at a time, as many as keep the scores within a few GB.
        step = max(1, min(case["kv_heads"], int(1e9 // max(1, count * n_q * n_k * group))))
        q = state["q"][q0:q0 + count * n_q].view(count, n_q, case["kv_heads"], group, -1)
        k = state["k"][k0:k0 + count * n_k].view(count, n_k, case["kv_heads"], -1)
        v = state["v"][k0:k0 + count * n_k].view(count, n_k, case["kv_heads"], -1)
        o = out[q0:q0 + count * n_q].view(count, n_q, case["kv_heads"], group, -1)
        for h in range(0, case["kv_heads"], step):
            qh = q[:, :, h:h + step].permute(0, 2, 3, 1, 4).float() * case["dim"] ** -0.5
            kh = k[:, :, h:h + step].permute(0, 2, 1, 3)[:, :, None].float()
            vh = v[:, :, h:h + step].permute(0, 2, 1, 3)[:, :, None].float()
            scores = torch.matmul(qh, kh.transpose(-1, -2))
            if case["causal"] and n_q > 1:
                row = torch.arange(n_q, device="cuda")[:, None] + (n_k - n_q)
                scores.masked_fill_(torch.arange(n_k, device="cuda")[None] > row, -math.inf)
            scores -= scores.amax(-1, keepdim=True)
            scores.exp_()
            total = scores.sum(-1, keepdim=True)
            o[:, :, h:h + step] = (torch.matmul(scores, vh) / total).permute(
                0, 3, 1, 2, 4).to(out.dtype)
    return out


def _plain_activation(name, x):
    if name == "gelu":
        return 0.5 * x * torch.erfc(x * -math.sqrt(0.5))
    if name == "gelu_tanh":
        return 0.5 * x * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (x + 0.044715 * x ** 3)))
    return x * torch.sigmoid(x) if name == "silu" else x


def run(state):
    if own:
        return _run_own(state)
    case, kind = state["case"], TYPES[state["case"]["type"]]
    if case["op"] in ("rotary", "norm"):
        h, g = case["heads"], case["kv_heads"]
        cos, sin = _plain_tables(case, state["positions"])
        out = []
        for name, x in (("q", state["qkv"][:, :h]), ("k", state["qkv"][:, h:h + g])):
            x = x.float()
            if case["op"] == "norm":
                x = _plain_norm(case, x, state[name + "_gamma"], state.get(name + "_beta"))
            out.append(_plain_turn(case, x, cos, sin).to(kind))
        return out
    if case["op"] == "attention":
        return _plain_attention(case, state)
    product = state["x"].float() @ state["w"].float().t()
    if "bias" in state:
        product = product + state["bias"]
    if case["gated"]:
        value = _plain_activation(case["activation"], product[:, :case["n"]])
        value = value * product[:, case["n"]:]
    else:
        value = _plain_activation(case["activation"], product)
    if "scale" in state:
        value = value * state["scale"]
    if "residual" in state:
        value = value + state["residual"].float()
    return value.to(kind)


# ---- the least work -----------------------------------------------------------------------

def _visible(case):
    """Pairs of a query and a key it sees, over the batch, per head."""
    total = 0
    for n_q, n_k in zip(*_sequences(case)):
        if not case["causal"]:
            total += n_q * n_k
        else:
            first = n_k - n_q + 1  # keys the first query sees
            low = max(0, min(n_q, 1 - first))  # queries that see none
            total += (n_q - low) * (first + low + n_k) // 2 if n_q > low else 0
    return total


def work(case):
    size = 2 if case["type"] == "bf16" else 4
    if case["op"] in ("rotary", "norm"):
        rows, d = case["tokens"] * (case["heads"] + case["kv_heads"]), case["dim"]
        total = 2 * rows * d * size + 4 * case["tokens"] * len(_sections(case))
        flops = 6 * rows * sum(_sections(case))
        if case["op"] == "norm":
            layer = case["norm"] == "layer"
            total += 4 * d * (4 if layer else 2)
            flops += rows * d * (7 if layer else 4)
        return {"bytes": total, "flops": flops}
    if case["op"] == "attention":
        queries, keys = _sequences(case)
        d = case["dim"]
        total = size * d * (2 * sum(queries) * case["heads"] + 2 * sum(keys) * case["kv_heads"])
        total += 4 * 2 * (len(queries) + 1)
        return {"bytes": total, "flops": 4 * _visible(case) * d * case["heads"]}
    rows = case["n"] * (2 if case["gated"] else 1)
    m, n, k = case["m"], case["n"], case["k"]
    total = size * (m * k + rows * k + m * n * (2 if case["residual"] else 1))
    total += 4 * ((rows if case["bias"] else 0) + (n if case["scale"] else 0))
    return {"bytes": total, "flops": 2 * m * rows * k}


# ---- the definition in 64 bits ------------------------------------------------------------

def exact(case, seed):
    data = {key: value.double() if value.is_floating_point() else value
            for key, value in _prepare(case, seed).items()}
    if case["op"] in ("rotary", "norm"):
        return _exact_rotary(case, data)
    if case["op"] == "attention":
        return _exact_attention(case, data)
    return _exact_linear(case, data)


def _exact_rotary(case, data):
    d, sections = case["dim"], _sections(case)
    pairs = sum(sections)
    # One complex number a pair: multiplying by exp(i angle) turns it.
    axis_of = [a for a, n in enumerate(sections) for _ in range(n)]
    rate = torch.tensor([10000.0 ** (-(j / n if case["ladder"] == "axis"
                                       else (sum(sections[:a]) + j) / pairs))
                         for a, n in enumerate(sections) for j in range(n)],
                        dtype=torch.float64, device="cuda")
    angle = data["positions"][axis_of].double().t() * rate
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    if case["pairing"] == "halves":
        first = torch.arange(pairs, device="cuda")
        second = first + pairs
    else:
        first = 2 * torch.arange(pairs, device="cuda")
        second = first + 1
    out, start = [], 0
    for name, heads in (("q", case["heads"]), ("k", case["kv_heads"])):
        x = data["qkv"][:, start:start + heads].clone()
        start += heads
        if case["op"] == "norm":
            if case["norm"] == "layer":
                spread = x.var(-1, unbiased=False, keepdim=True)
                x = (x - x.sum(-1, keepdim=True) / d) * (spread + 1e-6).rsqrt()
            else:
                x = x * (x.square().sum(-1, keepdim=True) / d + 1e-6).rsqrt()
            x = x * data[name + "_gamma"]
            if name + "_beta" in data:
                x = x + data[name + "_beta"]
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        out.append(x)
    return out


def _exact_attention(case, data):
    group, out = case["heads"] // case["kv_heads"], torch.zeros_like(data["q"])
    q0 = k0 = 0
    for n_q, n_k in zip(*_sequences(case)):
        for head in range(case["heads"]):
            k = data["k"][k0:k0 + n_k, head // group]
            v = data["v"][k0:k0 + n_k, head // group]
            for row in range(0, n_q if n_k else 0, 4096):
                q = data["q"][q0 + row:q0 + min(row + 4096, n_q), head]
                logits = (q @ k.T) / math.sqrt(case["dim"])
                if case["causal"]:
                    last = torch.arange(row, row + q.shape[0], device="cuda") + n_k - n_q
                    hidden = torch.arange(n_k, device="cuda")[None] > last[:, None]
                    logits = logits.masked_fill(hidden, -math.inf)
                out[q0 + row:q0 + row + q.shape[0], head] = torch.softmax(logits, -1) @ v
        q0, k0 = q0 + n_q, k0 + n_k
    return out


def _exact_linear(case, data):
    n = case["n"]

    def part(rows):
        value = torch.einsum("mk,nk->mn", data["x"], data["w"][rows])
        return value + data["bias"][rows] if case["bias"] else value

    def activated(x):
        if case["activation"] == "gelu":
            return x * torch.special.ndtr(x)
        if case["activation"] == "silu":
            return x / (1.0 + torch.exp(-x))
        if case["activation"] == "gelu_tanh":
            # (1 + tanh u) / 2 = 1 / (1 + exp(-2u))
            return x / (1.0 + torch.exp(-math.sqrt(8.0 / math.pi) * (x + 0.044715 * x ** 3)))
        return x

    value = activated(part(slice(0, n)))
    if case["gated"]:
        value = value * part(slice(n, 2 * n))
    if case["scale"]:
        value = value * data["scale"]
    return value + data["residual"] if case["residual"] else value
