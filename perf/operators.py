"""Performance cases of the decoder operators: rotary positions, attention whose scores go by positions, the gated
feed-forward block.

A program that serves or evaluates a decoder keeps its weights and its cache on the device and calls the entry points of
``include/fluidml_hip.h`` through ``fluidml_amd.cabi`` for every layer and every step.  A pass here is one such call, on the
stream that torch uses, into result tensors that stay from step to step.
"""
from __future__ import annotations

import ctypes
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # ---- rotary positions of queries and keys, before the keys go into the cache --------------------------------------
        # one token for each of 64 requests, far into long contexts: nothing but the launch
        rotary("rotary_token_b64", "bf16", batch=64, length=1, heads=32, kv_heads=8, size=128, dims=128, interleaved=True,
               scaling="wavelength", far=131072),
        # the decoder of fluidml_amd.models at its context: a quarter of each head
        rotary("rotary_neox_s256", "fp32", batch=1, length=256, heads=8, kv_heads=8, size=64, dims=16, interleaved=False,
               scaling="none", far=256),
        # the prompts of a batch in one pass
        rotary("rotary_prompt_s8192", "bf16", batch=2, length=8192, heads=32, kv_heads=8, size=128, dims=128,
               interleaved=False, scaling="dimension", far=65536),
        # ---- attention ----------------------------------------------------------------------------------------------------
        # one token for each of 24 requests over caches of all lengths up to 8192, scores capped
        attention("attention_token_b24", "bf16", batch=24, length=1, keys=8192, heads=32, kv_heads=8, size=128, cap=50.0,
                  ragged=True),
        # the decoder's heads with a distance bias in place of positions, an odd length, in fp32
        attention("attention_bias_s509", "fp32", batch=2, length=509, keys=509, heads=12, kv_heads=12, size=64, bias=True),
        # instruction and input seen both ways, the answer causally; a head size that is no power of two
        attention("attention_prefix_s1900", "bf16", batch=2, length=1900, keys=1900, heads=32, kv_heads=32, size=80,
                  prefix=700),
        # a layer with a sliding window and capped scores over a long prompt, large heads
        attention("attention_window_s5000", "bf16", batch=1, length=5000, keys=5000, heads=16, kv_heads=8, size=256,
                  cap=50.0, window=1024),
        # documents packed into one row of 8192 tokens
        attention("attention_documents_s8192", "fp16", batch=1, length=8192, keys=8192, heads=32, kv_heads=8, size=128,
                  documents=12),
        # ---- gated feed-forward block -------------------------------------------------------------------------------------
        # the tokens of a small decoding batch: the weights are all there is to read
        feed_forward("ffn_rows4", "bf16", rows=4, width=4096, hidden=11008, activation="silu", biased=False, rows_first=True),
        # the decoder of fluidml_amd.models at its context, in fp32
        feed_forward("ffn_neox_rows256", "fp32", rows=256, width=512, hidden=2048, activation="gelu", biased=True,
                     rows_first=False),
        # sizes that no tile divides
        feed_forward("ffn_rows333", "fp16", rows=333, width=1000, hidden=2731, activation="gelu_tanh", biased=True,
                     rows_first=True),
        # a long prompt through a large layer: the most arithmetic
        feed_forward("ffn_rows8192", "bf16", rows=8192, width=4096, hidden=14336, activation="silu", biased=False,
                     rows_first=True),
    ]


def rotary(name, dtype, **sizes):
    return {"name": name, "operator": "rotary", "dtype": dtype, **sizes}


def attention(name, dtype, **sizes):
    return {"name": name, "operator": "attention", "dtype": dtype,
            **{"cap": 0.0, "bias": False, "prefix": 0, "window": 0, "documents": 0, "ragged": False, **sizes}}


def feed_forward(name, dtype, **sizes):
    return {"name": name, "operator": "feed_forward", "dtype": dtype, **sizes}


def draw(rng):
    def spread(low, high):
        return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))

    dtype = rng.choice(["fp32", "fp16", "bf16", "bf16"])
    operator = rng.choice(["rotary", "attention", "attention", "feed_forward", "feed_forward"])
    heads, kv_heads = rng.choice([(8, 8), (12, 12), (16, 8), (32, 8), (28, 4), (32, 32), (25, 5)])
    if operator == "rotary":
        size = rng.choice([64, 80, 96, 128, 256])
        dims = rng.choice([size, size, size // 2, size // 4])
        batch = spread(1, 64)
        case = rotary("", dtype, batch=batch, length=min(spread(1, 8192), 16384 * 128 // (batch * size)), heads=heads,
                      kv_heads=kv_heads, size=size, dims=dims, interleaved=rng.random() < 0.5,
                      scaling=rng.choice(["none", "linear", "base", "wavelength", "dimension"]), far=spread(8192, 131072))
    elif operator == "attention":
        size = rng.choice([64, 80, 96, 128, 256])
        more = {"size": size, "heads": heads, "kv_heads": kv_heads, "cap": rng.choice([0.0, 30.0, 50.0]),
                "bias": rng.random() < 0.3}
        if rng.random() < 0.4:  # a step of decoding: one token, or a few drafted ones
            case = attention("", dtype, batch=spread(1, 24), length=rng.choice([1, 1, 1, spread(2, 8)]),
                             keys=spread(64, 8192), ragged=True, **more)
        else:
            length = spread(16, 8192 if size <= 128 else 5000)
            if dtype == "fp32":
                length = min(length, 3000)
            batch = max(1, min(spread(1, 8), 8192 * 2048 // length ** 2))
            kind = rng.choice(["none", "prefix", "window", "documents"])
            case = attention("", dtype, batch=batch, length=length, keys=length,
                             prefix=spread(1, length) if kind == "prefix" else 0,
                             window=spread(1, length) if kind == "window" else 0,
                             documents=spread(1, max(1, length // 16)) if kind == "documents" else 0, **more)
    else:
        rows, width, hidden = spread(1, 8192), spread(64, 4096), spread(64, 14336)
        if dtype == "fp32":
            rows = min(rows, 1024)
        case = feed_forward("", dtype, rows=rows, width=width, hidden=hidden, biased=rng.random() < 0.5,
                            activation=rng.choice(["silu", "gelu", "gelu_tanh", "relu"]), rows_first=rng.random() < 0.5)
    del case["name"]
    return case


# ---- inputs -------------------------------------------------------------------------------------------------------------


def _document_ends(case):
    """Ends of the packed documents: every length from a short note to a long text, the same for all seeds."""
    weights = [1.5 ** (3 * i % 7) for i in range(case["documents"])]
    ends, total = [], 0.0
    for w in weights:
        total += w
        ends.append(max(1, round(case["length"] * total / sum(weights))))
    return ends


def _key_counts(case):
    """Keys in use for each request: spread over the cache where it is ragged."""
    if not case["ragged"]:
        return [case["keys"]] * case["batch"]
    low = min(case["length"], case["keys"])
    return [low + (case["keys"] - low) * (i + 1) // case["batch"] for i in range(case["batch"])]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, spread=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * spread).to(dtype)

    state = {"case": case}
    if case["operator"] == "rotary":
        B, S, H, KV, D = (case[k] for k in ("batch", "length", "heads", "kv_heads", "size"))
        state["q"] = normal(B, S, H, D).transpose(1, 2)  # as the projections leave them
        state["k"] = normal(B, S, KV, D).transpose(1, 2)
        start = torch.randint(0, max(1, case["far"] - S + 1), (B, 1), generator=g, device="cuda")
        state["positions"] = start + torch.arange(S, device="cuda")
        state["q_out"], state["k_out"] = torch.empty_like(state["q"]), torch.empty_like(state["k"])
    elif case["operator"] == "attention":
        B, S, T, H, KV, D = (case[k] for k in ("batch", "length", "keys", "heads", "kv_heads", "size"))
        state["q"] = normal(B, S, H, D).transpose(1, 2)
        state["k"], state["v"] = normal(B, T, KV, D).transpose(1, 2), normal(B, T, KV, D).transpose(1, 2)
        state["out"] = torch.empty_like(state["q"])
        if case["ragged"]:
            counts = torch.tensor(_key_counts(case), dtype=torch.int32, device="cuda")
            state["key_lengths"] = counts[torch.randperm(B, generator=g, device="cuda")]
        if case["bias"]:
            state["slopes"] = 2.0 ** (-8.0 * torch.arange(1, H + 1, device="cuda", dtype=torch.float32) / H)
        if case["prefix"]:
            state["prefix_lengths"] = torch.full((B,), case["prefix"], dtype=torch.int32, device="cuda")
        if case["documents"]:
            ends = torch.tensor(_document_ends(case), device="cuda")
            ids = torch.searchsorted(ends, torch.arange(S, device="cuda"), right=True).int()
            state["documents"] = ids.expand(B, S).contiguous()
        state["scratch"] = torch.empty(32 << 20, dtype=torch.uint8, device="cuda")
    else:
        M, K, N = case["rows"], case["width"], case["hidden"]
        state["x"] = normal(M, K)
        if case["rows_first"]:  # a row for each output, as checkpoints store them
            state["gate"], state["up"] = normal(N, K, spread=K ** -0.5).t(), normal(N, K, spread=K ** -0.5).t()
            state["down"] = normal(K, N, spread=N ** -0.5).t()
        else:
            state["gate"], state["up"] = normal(K, N, spread=K ** -0.5), normal(K, N, spread=K ** -0.5)
            state["down"] = normal(N, K, spread=N ** -0.5)
        if case["biased"]:
            state["gate_bias"], state["up_bias"], state["down_bias"] = normal(N), normal(N), normal(K)
        state["products"] = torch.empty(M, N, dtype=dtype, device="cuda")
        state["out"] = torch.empty(M, K, dtype=dtype, device="cuda")
    return state


def run(state):
    operator = state["case"]["operator"]
    if operator == "rotary":
        return _rotary_own(state) if own else _rotary_plain(state)
    if operator == "attention":
        return _attention_own(state) if own else _attention_plain(state)
    return _feed_forward_own(state) if own else _feed_forward_plain(state)


# ---- the framework's calls ----------------------------------------------------------------------------------------------


def _view(t):
    from fluidml_amd import cabi

    return ctypes.byref(cabi.view(t))


def _optional(state, name):
    from fluidml_amd import cabi

    return ctypes.pointer(cabi.view(state[name])) if name in state else None


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


# context of the model before it was stretched, and by how much
BASE, FACTOR, ORIGINAL = 500000.0, 8.0, 8192


def _rotary_own(state):
    from fluidml_amd import cabi

    case = state["case"]
    plan = cabi.FlRotaryPlan()
    plan.interleaved, plan.dims, plan.base, plan.amplitude = int(case["interleaved"]), case["dims"], BASE, 1.0
    plan.scaling = {"none": cabi.FL_ROTARY_PLAIN, "linear": cabi.FL_ROTARY_LINEAR, "base": cabi.FL_ROTARY_BASE,
                    "wavelength": cabi.FL_ROTARY_WAVELENGTH, "dimension": cabi.FL_ROTARY_DIMENSION}[case["scaling"]]
    plan.factor, plan.original_length = FACTOR, ORIGINAL
    if case["scaling"] == "wavelength":
        plan.low, plan.high = 1.0, 4.0
    elif case["scaling"] == "dimension":
        plan.low, plan.high, plan.amplitude = 1.0, 32.0, 0.1 * math.log(FACTOR) + 1.0
    cabi.call("rotary_positions_pair", _view(state["q"]), _view(state["q_out"]), _view(state["k"]), _view(state["k_out"]),
              _view(state["positions"]), ctypes.byref(plan), _stream())
    return {"q": state["q_out"], "k": state["k_out"]}


def _attention_own(state):
    from fluidml_amd import cabi

    case = state["case"]
    scores = cabi.FlAttentionScores()
    scores.scale, scores.cap = case["size"] ** -0.5, case["cap"]
    scores.causal, scores.window = 1, case["window"]
    scores.slopes = _optional(state, "slopes")
    scores.prefix_lengths = _optional(state, "prefix_lengths")
    scores.query_documents = scores.key_documents = _optional(state, "documents")
    scores.key_lengths = _optional(state, "key_lengths")
    scratch = state["scratch"]
    cabi.call("attention_positions", _view(state["q"]), _view(state["k"]), _view(state["v"]), _view(state["out"]),
              ctypes.byref(scores), scratch.data_ptr(), scratch.numel(), _stream())
    return state["out"]


def _feed_forward_own(state):
    from fluidml_amd import cabi

    activation = {"silu": cabi.FL_GATE_SILU, "gelu": cabi.FL_GATE_GELU, "gelu_tanh": cabi.FL_GATE_GELU_TANH,
                  "relu": cabi.FL_GATE_RELU}[state["case"]["activation"]]
    cabi.call("gated_feed_forward", _view(state["x"]), _view(state["gate"]), _view(state["up"]),
              _optional(state, "gate_bias"), _optional(state, "up_bias"), _view(state["down"]),
              _optional(state, "down_bias"), None, _view(state["products"]), _view(state["out"]), activation, _stream())
    return {"products": state["products"], "out": state["out"]}


# ---- the plain forms ----------------------------------------------------------------------------------------------------


def _frequencies(case):
    """Radians per position of each pair of columns."""
    R = case["dims"]
    j = torch.arange(R // 2, device="cuda", dtype=torch.float64)
    f = BASE ** (-2.0 * j / R)
    if case["scaling"] == "linear":
        return f / FACTOR
    if case["scaling"] == "base":
        return (BASE * FACTOR ** (R / (R - 2.0))) ** (-2.0 * j / R)
    if case["scaling"] == "wavelength":  # long waves stretched, short ones kept, a ramp between
        turns = ORIGINAL * f / (2.0 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0.0, 1.0)
        return f / FACTOR * (1.0 - keep) + f * keep
    if case["scaling"] == "dimension":  # the same by a ramp over the columns
        at = [R * math.log(ORIGINAL / (turns * 2.0 * math.pi)) / (2.0 * math.log(BASE)) for turns in (32.0, 1.0)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), R - 1)
        stretch = ((j - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        return f / FACTOR * stretch + f * (1.0 - stretch)
    return f


def _rotary_plain(state):
    case = state["case"]
    R, D = case["dims"], case["size"]
    angle = state["positions"].double()[:, None, :, None] * _frequencies(case)
    amplitude = 0.1 * math.log(FACTOR) + 1.0 if case["scaling"] == "dimension" else 1.0
    cos, sin = (angle.cos() * amplitude).float(), (angle.sin() * amplitude).float()

    def turned(x):
        x = x.float()
        if case["interleaved"]:
            a, b = x[..., 0:R:2], x[..., 1:R:2]
            front = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = x[..., :R // 2], x[..., R // 2:R]
            front = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([front, x[..., R:]], -1)

    dtype = DTYPES[case["dtype"]]
    return {"q": turned(state["q"]).to(dtype), "k": turned(state["k"]).to(dtype)}


def _visible(state, S, T):
    """Which keys each query sees, [B, 1, 1, S, T], and how far away they are."""
    case = state["case"]
    counts = state["key_lengths"] if "key_lengths" in state else torch.full((case["batch"],), T, device="cuda")
    at = (counts[:, None] - S + torch.arange(S, device="cuda"))[:, None, None, :, None]
    key = torch.arange(T, device="cuda")
    seen = key <= at
    if case["window"]:
        seen = seen & (key > at - case["window"])
    if "prefix_lengths" in state:
        seen = seen | (key < state["prefix_lengths"][:, None, None, None, None])
    seen = seen & (key < counts[:, None, None, None, None])
    if "documents" in state:
        ids = state["documents"]
        seen = seen & (ids[:, None, None, :, None] == ids[:, None, None, None, :])
    return seen, (at - key).abs()


def _attention_plain(state):
    case = state["case"]
    B, S, T, H, KV, D = (case[k] for k in ("batch", "length", "keys", "heads", "kv_heads", "size"))
    q = state["q"].float().reshape(B, KV, H // KV * S, D)
    kt = state["k"].float().transpose(2, 3).contiguous()
    s = torch.matmul(q, kt).view(B, KV, H // KV, S, T) * case["size"] ** -0.5
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    seen, distance = _visible(state, S, T)
    if case["bias"]:
        s = s - state["slopes"].view(KV, H // KV, 1, 1) * distance
    s = s.masked_fill(~seen, -math.inf)
    most = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(most == -math.inf, 0.0, most))
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total == 0.0, 1.0, total)).view(B, KV, H // KV * S, T)
    out = torch.matmul(p, state["v"].float().contiguous())
    return out.view(B, H, S, D).transpose(1, 2).to(DTYPES[case["dtype"]]).transpose(1, 2)


def _feed_forward_plain(state):
    case, dtype = state["case"], DTYPES[state["case"]["dtype"]]
    x = state["x"].float()
    gate, up = x @ state["gate"].float(), x @ state["up"].float()
    if case["biased"]:
        gate, up = gate + state["gate_bias"].float(), up + state["up_bias"].float()
    if case["activation"] == "silu":
        gate = gate / (1.0 + torch.exp(-gate))
    elif case["activation"] == "gelu":
        gate = 0.5 * gate * (1.0 + torch.erf(gate * math.sqrt(0.5)))
    elif case["activation"] == "gelu_tanh":
        gate = 0.5 * gate * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (gate + 0.044715 * gate * gate * gate)))
    else:
        gate = torch.where(gate > 0.0, gate, 0.0 * gate)
    products = (gate * up).to(dtype)
    out = products.float() @ state["down"].float()
    if case["biased"]:
        out = out + state["down_bias"].float()
    return {"products": products, "out": out.to(dtype)}


# ---- what has to be read, written and computed --------------------------------------------------------------------------


def work(case):
    item = 4 if case["dtype"] == "fp32" else 2
    if case["operator"] == "rotary":
        tokens, values = case["batch"] * case["length"], case["heads"] + case["kv_heads"]
        return {"bytes": tokens * (values * case["size"] * 2 * item + 8), "flops": tokens * values * case["dims"] * 3}
    if case["operator"] == "attention":
        B, S, T, H, KV, D = (case[k] for k in ("batch", "length", "keys", "heads", "kv_heads", "size"))
        pairs, read = 0, 0
        for count in _key_counts(case):
            pairs += _pairs(case, S, count)
            read += min(count, _keys_seen(case, S, count))
        return {"bytes": item * D * (2 * B * S * H + 2 * read * KV), "flops": 4 * D * H * pairs}
    M, K, N = case["rows"], case["width"], case["hidden"]
    return {"bytes": item * (2 * M * K + M * N + 3 * K * N + (2 * N + K if case["biased"] else 0)), "flops": 6 * M * K * N}


def _pairs(case, S, T):
    """Pairs of a query and a key that it sees, for one head of one request."""
    if case["documents"]:
        ends = [0] + _document_ends(case)
        return sum((b - a) * (b - a + 1) // 2 for a, b in zip(ends, ends[1:]))
    total = 0
    for i in range(S):
        at = T - S + i
        low = max(0, at - case["window"] + 1) if case["window"] else 0
        prefix = min(case["prefix"], T)
        total += max(0, at + 1 - low) + max(0, prefix - max(at + 1, 0)) + min(low, prefix)
    return total


def _keys_seen(case, S, T):
    """Keys that any query of one request sees."""
    return min(T, S + case["window"] - 1) if case["window"] and not case["prefix"] else T


# ---- the same from the definitions, in 64 bits --------------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    return {"rotary": _rotary_exact, "attention": _attention_exact, "feed_forward": _feed_forward_exact}[case["operator"]](state, case)


def _rotary_exact(state, case):
    """Each pair of columns is a complex number, turned by exp(i angle)."""
    R, half = case["dims"], case["dims"] // 2
    rate = []
    for j in range(half):
        f = BASE ** (-2.0 * j / R)
        if case["scaling"] == "linear":
            f /= FACTOR
        elif case["scaling"] == "base":
            f = (BASE * FACTOR ** (R / (R - 2))) ** (-2.0 * j / R)
        elif case["scaling"] == "wavelength":
            wave = 2 * math.pi / f
            if wave > ORIGINAL / 1.0:
                f /= FACTOR
            elif wave > ORIGINAL / 4.0:
                share = (ORIGINAL / wave - 1.0) / 3.0
                f = (1 - share) * f / FACTOR + share * f
        elif case["scaling"] == "dimension":
            column = lambda turns: R * math.log(ORIGINAL / (2 * math.pi * turns)) / (2 * math.log(BASE))  # noqa: E731
            low, high = max(0, math.floor(column(32.0))), min(R - 1, math.ceil(column(1.0)))
            share = min(1.0, max(0.0, (j - low) / max(high - low, 0.001)))
            f = share * f / FACTOR + (1 - share) * f
        rate.append(f)
    angle = state["positions"].double().unsqueeze(-1) * torch.tensor(rate, dtype=torch.float64, device="cuda")
    size = torch.full_like(angle, 1.0 + 0.1 * math.log(FACTOR) if case["scaling"] == "dimension" else 1.0)
    turn = torch.polar(size, angle).unsqueeze(1)
    result = {}
    for name in ("q", "k"):
        x = state[name].double()
        out = x.clone()
        if case["interleaved"]:
            z = turn * torch.complex(x[..., 0:R:2], x[..., 1:R:2])
            out[..., 0:R:2], out[..., 1:R:2] = z.real, z.imag
        else:
            z = turn * torch.complex(x[..., :half], x[..., half:R])
            out[..., :half], out[..., half:R] = z.real, z.imag
        result[name] = out
    return result


def _attention_exact(state, case):
    """A head of a request at a time, its queries in runs, over the keys from its first to its last."""
    B, S, H, KV = (case[k] for k in ("batch", "length", "heads", "kv_heads"))
    if 4.0 * case["size"] * S * case["keys"] * B * H > 4e13:
        return None
    out = torch.empty(B, H, S, case["size"], dtype=torch.float64, device="cuda")
    counts = state["key_lengths"].tolist() if "key_lengths" in state else [case["keys"]] * B
    for b in range(B):
        n = counts[b]
        key = torch.arange(n, device="cuda")
        for first in range(0, S, 2048):
            last = min(S, first + 2048)
            at = torch.arange(first, last, device="cuda").unsqueeze(1) + (n - S)
            hidden = key > at
            if case["window"]:
                hidden |= key <= at - case["window"]
            if case["prefix"]:
                hidden &= key >= case["prefix"]
            if case["documents"]:
                hidden |= state["documents"][b, first:last].unsqueeze(1) != state["documents"][b, :n]
            nothing = hidden.all(1, keepdim=True)
            for h in range(H):
                k, v = state["k"][b, h * KV // H, :n].double(), state["v"][b, h * KV // H, :n].double()
                s = state["q"][b, h, first:last].double() @ k.t() / math.sqrt(case["size"])
                if case["cap"]:
                    s = torch.tanh(s / case["cap"]) * case["cap"]
                if case["bias"]:
                    s -= (at - key).abs() * state["slopes"][h].double()
                s[hidden] = -math.inf
                s = torch.softmax(s, 1)
                out[b, h, first:last] = torch.where(nothing, 0.0, s) @ v
    return out


def _feed_forward_exact(state, case):
    if 6.0 * case["rows"] * case["width"] * case["hidden"] > 1e13:
        return None
    wide = {k: v.double() for k, v in state.items() if torch.is_tensor(v)}
    a, b = wide["x"] @ wide["gate"], wide["x"] @ wide["up"]
    if case["biased"]:
        a += wide["gate_bias"]
        b += wide["up_bias"]
    kind = case["activation"]
    a = (a * torch.sigmoid(a) if kind == "silu" else a * torch.special.ndtr(a) if kind == "gelu" else a.clamp(min=0)
         if kind == "relu" else a * torch.sigmoid(math.sqrt(8.0 / math.pi) * (a + 0.044715 * a ** 3)))
    out = (a * b) @ wide["down"]
    return {"products": a * b, "out": out + wide["down_bias"] if case["biased"] else out}
