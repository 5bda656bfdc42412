"""Attention by positions and the gated block from their definitions, in 64 bits on the CPU."""
import ctypes
import math


def visible(B, Sq, Skv, causal=False, window=0, prefix=None, documents=None, starts=None, query_lengths=None, key_lengths=None):
    """Which keys each query sees [B, Sq, Skv], the distances, and which rows are written [B, Sq]."""
    import torch

    lengths = torch.full((B,), Skv) if key_lengths is None else key_lengths.cpu().long().clamp(0, Skv)
    rows = torch.full((B,), Sq) if query_lengths is None else query_lengths.cpu().long().clamp(0, Sq)
    first = lengths - rows if starts is None else starts.cpu().long()
    at = (first[:, None] + torch.arange(Sq))[:, :, None]
    j = torch.arange(Skv)[None, None, :]
    seen = torch.ones(B, Sq, Skv, dtype=torch.bool)
    if causal:
        seen &= j <= at
    if window:
        seen &= (j > at - window) & (j < at + window)
    if prefix is not None:
        seen |= j < prefix.cpu().long()[:, None, None]
    seen &= j < lengths[:, None, None]
    if documents is not None:
        dq, dk = documents[0].cpu()[:, :, None], documents[1].cpu()[:, None, :]
        seen &= (dq == dk) & (dq >= 0)
    return seen, (at - j).abs(), torch.arange(Sq)[None, :] < rows[:, None]


def attention(q, k, v, scale, cap=0.0, slopes=None, **masks):
    """(result, largest |v| that a row sees, rows that are written)"""
    import torch

    B, H, Sq, D = q.shape
    KV, Skv = k.shape[1], k.shape[2]
    seen, distance, written = visible(B, Sq, Skv, **masks)
    q, k, v = (t.double().cpu() for t in (q, k, v))
    out, most = torch.zeros(B, H, Sq, D, dtype=torch.float64), torch.zeros(B, H, Sq, dtype=torch.float64)
    if q.isfinite().all() and k.isfinite().all() and v.isfinite().all():  # whole heads at a time: the hidden weights are zeros
        for b in range(B):
            for h in range(H):
                kk, vv = k[b, h // (H // KV)], v[b, h // (H // KV)]
                s = q[b, h] @ kk.t() * scale
                if cap:
                    s = cap * torch.tanh(s / cap)
                if slopes is not None:
                    s = s - slopes[h].double().cpu() * distance[b]
                some = seen[b].any(1, keepdim=True)
                weights = torch.softmax(s.masked_fill(~seen[b], -math.inf), 1).masked_fill(~some, 0.0)
                out[b, h] = weights @ vv
                most[b, h] = torch.where(seen[b], vv.abs().amax(1)[None, :], torch.zeros(())).amax(1)
        return out, most, written
    for b in range(B):
        for h in range(H):
            kk, vv = k[b, h // (H // KV)], v[b, h // (H // KV)]
            for i in range(Sq):
                keys = seen[b, i].nonzero().flatten()
                if len(keys) == 0:
                    continue
                s = kk[keys] @ q[b, h, i] * scale
                if cap:
                    s = cap * torch.tanh(s / cap)
                if slopes is not None:
                    s = s - slopes[h].double().cpu() * distance[b, i, keys]
                out[b, h, i] = torch.softmax(s, 0) @ vv[keys]
                most[b, h, i] = vv[keys].abs().max()
    return out, most, written


def attention_bound(want, most, dtype, D, Skv, scale, cap, reach, peak=1.0):
    """What the kernel may be off by, for operands up to `peak` in magnitude.  A score is a sum of D products of up to peak^2: D / 4 roundings
    of its largest value 2^-24 D peak^2, then scale, cap and bias, each a few roundings of the score's own size (cap, or D scale peak^2;
    `reach`: the largest bias).  An error e of the scores moves a mean of values up to m by 2 e m.  The sums over the keys: one rounding
    per 16 keys, and exp and the division.  With 16-bit operands the weights are rounded once (half a step of a mean of values up
    to m) and so is the result; fp16 has steps of 2^-24 where it is denormal, for each of Skv weights (the largest is 1 or more) and the result."""
    import torch

    size = D * abs(scale) * peak * peak
    e = 2.0 ** -24 * (size * (D / 4 + 8) + 8 * (min(cap, size) if cap else 0.0) + (8 * cap if cap else 0) + 4 * reach)
    off = most[..., None] * (2 * e + 2.0 ** -24 * (Skv / 16 + 24))
    if dtype != torch.float32:
        off = off + torch.finfo(dtype).eps / 2 * (most[..., None] + want.abs())
        if dtype == torch.float16:
            off = off + 2.0 ** -25 * (Skv * most[..., None] + 1)
    return off


def call_attention(q, k, v, out, scale, cap=0.0, slopes=None, causal=False, window=0, prefix=None, documents=None, starts=None,
                   query_lengths=None, key_lengths=None, stream=None, scratch=None):
    """The entry point, with scratch of exactly the size it asks for (whose contents it must not care about)."""
    import torch

    from fluidml_amd import cabi

    def optional(t):
        return None if t is None else ctypes.pointer(cabi.view(t))

    scores = cabi.FlAttentionScores(scale, cap, optional(slopes), int(causal), window, optional(prefix),
                                    *(map(optional, documents) if documents is not None else (None, None)), optional(starts),
                                    optional(query_lengths), optional(key_lengths))
    views = [ctypes.byref(cabi.view(t)) for t in (q, k, v, out)]
    need = ctypes.c_size_t()
    cabi.call("attention_positions_scratch", views[0], views[1], ctypes.byref(scores), ctypes.byref(need))
    if scratch is None:
        scratch = torch.full((max(need.value, 16),), 0xff, dtype=torch.uint8, device=q.device)
    cabi.call("attention_positions", *views, ctypes.byref(scores), scratch.data_ptr(), need.value, stream)
    return scratch


ACTIVATIONS = ("silu", "gelu", "gelu_tanh", "relu", "sigmoid", "identity")


def activated(kind, a):
    import torch

    return {"silu": lambda: a * torch.sigmoid(a), "gelu": lambda: 0.5 * a * (1 + torch.erf(a / math.sqrt(2))),
            "gelu_tanh": lambda: 0.5 * a * (1 + torch.tanh(math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3))),
            "relu": lambda: torch.relu(a), "sigmoid": lambda: torch.sigmoid(a), "identity": lambda: a}[kind]()


def gated(x, gate, up, gate_bias, up_bias, kind):
    """(products, their bound): sums of K products, each rounding 2^-24 of the sum of the magnitudes; an activation's slope is at most
    1.13, and its value is off by a few roundings of itself (8; the arguments of exp, erf and tanh are rounded too) and never by less
    than 2^-24 of the gate's own."""
    import torch

    x, gate, up = x.double().cpu(), gate.double().cpu(), up.double().cpu()
    K = x.shape[1]
    g, u = x @ gate, x @ up
    eg, eu = 2.0 ** -24 * (K + 4) * (x.abs() @ gate.abs()), 2.0 ** -24 * (K + 4) * (x.abs() @ up.abs())
    for bias, value, err in ((gate_bias, g, eg), (up_bias, u, eu)):
        if bias is not None:
            value += bias.double().cpu()
            err += 2.0 ** -24 * value.abs()
    act = activated(kind, g)
    ea = 1.13 * eg + 2.0 ** -24 * 8 * (act.abs() + g.abs() + (1.0 if kind == "sigmoid" else 0.0))
    return act * u, ea * u.abs() + act.abs() * eu + ea * eu + 2.0 ** -24 * 2 * (act * u).abs()


def rounded(bound, want, dtype):
    import torch

    if dtype == torch.float32:
        return bound + 2.0 ** -140
    # half a step; fp16 has steps of 2^-24 where it is denormal
    return bound + torch.finfo(dtype).eps / 2 * (want.abs() + bound) + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134)
