"""Attention by positions against its definition in 64 bits: types, head layouts, lengths, masks that leave rows empty, strides, what is
hidden holding infinities and NaN, capture."""
import ctypes

import pytest

from tests import decoder_oracle as oracle

pytestmark = pytest.mark.gpu


def dtype_of(name):
    import torch

    return {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}[name]


def draw(device, dtype, *shapes, seed=0):
    """uniform in -1 .. 1"""
    import torch

    g = torch.Generator(device=device).manual_seed(seed)
    return [(torch.rand(*s, device=device, generator=g) * 2 - 1).to(dtype) for s in shapes]


def check(q, k, v, out, scale, cap=0.0, slopes=None, peak=1.0, **masks):
    import torch

    want, most, written = oracle.attention(q, k, v, scale, cap, slopes, **masks)
    reach = 0.0
    if slopes is not None:
        reach = float(slopes.abs().max()) * float(oracle.visible(q.shape[0], q.shape[2], k.shape[2], **masks)[1].max())
    bound = oracle.attention_bound(want, most, q.dtype, q.shape[3], k.shape[2], scale, cap, reach, peak)
    got = out.double().cpu()
    far = ((got - want).abs() - bound)[written[:, None, :].expand(got.shape[:3])]
    assert not far.isnan().any() and far.max() <= 0, f"{far.max()} over"
    return got, written


def options(name, device, B, H, Sq, Skv):
    import torch

    def ints(values):
        return torch.tensor([values[i % len(values)] for i in range(B)], dtype=torch.int32, device=device)

    if name == "plain":
        return {}
    if name == "causal":
        return {"causal": True}
    if name == "cap":
        return {"causal": True, "cap": 0.7}
    if name == "slopes":
        return {"causal": True, "slopes": 2.0 ** -(1 + torch.arange(H, device=device, dtype=torch.float32) % 8)}
    if name == "slopes both ways":
        return {"cap": 20.0, "slopes": 2.0 ** -(2 + torch.arange(H, device=device, dtype=torch.float32) % 8)}
    if name == "window":
        return {"causal": True, "window": max(1, Skv // 3)}
    if name == "window both ways":
        return {"window": 1 + Skv // 5}
    if name == "prefix":
        return {"causal": True, "prefix": ints([Skv // 2, 0, Skv + 3, -2])}
    if name == "prefix and window":
        return {"causal": True, "window": 5, "prefix": ints([3, 70])}
    if name == "documents":
        g = torch.Generator(device=device).manual_seed(Skv)
        cut = torch.sort(torch.randint(0, Skv + 1, (B, 4), device=device, generator=g)).values
        ids = torch.searchsorted(cut, torch.arange(Skv, device=device).expand(B, Skv).contiguous(), right=True).int()
        ids[:, -1] = -1  # padding
        return {"causal": True, "documents": (ids[:, Skv - min(Sq, Skv):].repeat(1, -(-Sq // Skv))[:, :Sq].contiguous(), ids)}
    if name == "documents in any order":
        g = torch.Generator(device=device).manual_seed(Skv)
        return {"documents": tuple(torch.randint(-1, 3, (B, n), device=device, generator=g, dtype=torch.int32) for n in (Sq, Skv))}
    if name == "lengths":
        return {"causal": True, "cap": 30.0, "key_lengths": ints([Skv, 1, 0, Skv // 2, Skv + 9, -4])}
    if name == "starts":
        return {"causal": True, "starts": ints([0, Skv // 2, -Sq, 3 * Skv]), "window": Skv}
    if name == "query lengths":
        return {"causal": True, "query_lengths": ints([Sq, 0, Sq // 2, Sq + 1, -1]), "key_lengths": ints([Skv, Skv // 2])}
    raise KeyError(name)


ALL = ("plain", "causal", "cap", "slopes", "slopes both ways", "window", "window both ways", "prefix", "prefix and window", "documents",
       "documents in any order", "lengths", "starts", "query lengths")


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("name", ALL)
@pytest.mark.parametrize("B,H,KV,Sq,Skv,D", [
    (3, 4, 2, 1, 300, 64),      # a token
    (2, 8, 1, 5, 333, 128),     # drafted tokens, one key head
    (3, 2, 2, 77, 77, 64),      # odd lengths
    (2, 6, 2, 130, 200, 80),    # more keys than queries, a head that is no power of two
], ids=["token", "drafted", "odd", "cached"])
def test_attention_positions(device, dtype, name, B, H, KV, Sq, Skv, D):
    import torch

    print("[case]", dtype, name, B, H, KV, Sq, Skv, D, flush=True)
    q, k, v = draw(device, dtype_of(dtype), (B, H, Sq, D), (B, KV, Skv, D), (B, KV, Skv, D))
    more = options(name, device, B, H, Sq, Skv)
    out = torch.full_like(q, 7.0)
    oracle.call_attention(q, k, v, out, D ** -0.5, **more)
    got, written = check(q, k, v, out, D ** -0.5, **more)
    assert (got[~written[:, None, :].expand(got.shape[:3])] == 7.0).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("B,H,KV,Sq,Skv,D", [
    (1, 1, 1, 1, 1, 1), (1, 2, 1, 3, 2, 3), (1, 3, 3, 1, 64, 17), (1, 2, 2, 65, 65, 33), (2, 2, 1, 64, 128, 256), (1, 25, 5, 9, 130, 200),
    (1, 40, 1, 3, 260, 96),     # more heads to a key head than a tile has rows
    (1, 2, 1, 1, 4100, 128),    # a long cache for few rows
    (2, 4, 4, 2, 1500, 256),
    (1, 2, 2, 520, 520, 128),
])
def test_attention_positions_sizes(device, dtype, B, H, KV, Sq, Skv, D):
    import torch

    print("[case]", dtype, B, H, KV, Sq, Skv, D, flush=True)
    q, k, v = draw(device, dtype_of(dtype), (B, H, Sq, D), (B, KV, Skv, D), (B, KV, Skv, D), seed=D)
    out = torch.full_like(q, 7.0)
    oracle.call_attention(q, k, v, out, 0.3, causal=True)
    check(q, k, v, out, 0.3, causal=True)


def kernels(q, k, v, out, scale, **more):
    """Names of what a call launches."""
    from tests.util import launches

    scratch = oracle.call_attention(q, k, v, out, scale, **more)
    return [name for name, _ in launches(lambda stream: oracle.call_attention(q, k, v, out, scale, **more, stream=stream, scratch=scratch))]


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("name", ALL)
@pytest.mark.parametrize("B,H,KV,Sq,Skv,D", [
    (6, 16, 8, 250, 250, 64),      # 500 rows to a key head, the last tile of rows not full
    (7, 12, 12, 300, 389, 128),    # key heads that do not spread evenly over eight
    (5, 9, 3, 1200, 330, 72),      # more queries than keys; columns that no sixteen divides
    (8, 8, 8, 270, 300, 256),
], ids=["grouped", "cached", "long", "wide"])
def test_attention_positions_many_rows(device, dtype, name, B, H, KV, Sq, Skv, D):
    import torch

    print("[case]", dtype, name, B, H, KV, Sq, Skv, D, flush=True)
    q, k, v = draw(device, dtype_of(dtype), (B, Sq, H, D), (B, Skv, KV, D), (B, Skv, KV, D))
    q, k, v = q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)
    more = options(name, device, B, H, Sq, Skv)
    out = torch.full_like(q, 7.0)
    assert any("AttentionRowsKernel" in n for n in kernels(q, k, v, out, D ** -0.5, **more))
    out.fill_(7.0)
    oracle.call_attention(q, k, v, out, D ** -0.5, **more)
    got, written = check(q, k, v, out, D ** -0.5, **more)
    assert (got[~written[:, None, :].expand(got.shape[:3])] == 7.0).all()


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("name", ["causal", "window", "documents", "prefix", "lengths"])
def test_attention_positions_many_rows_hidden_values(device, dtype, name):
    """The same with infinities and NaN in keys that no query sees and in values that some do not see."""
    import torch

    B, H, KV, Sq, D = 12, 8, 8, 280, 64
    q, k, v = draw(device, dtype_of(dtype), (B, H, Sq, D), (B, KV, Sq, D), (B, KV, Sq, D))
    more = options(name, device, B, H, Sq, Sq)
    if name == "window":
        more["window"] = 20
    seen, _, _ = oracle.visible(B, Sq, Sq, **{a: b for a, b in more.items() if a not in ("cap", "slopes")})
    for b in range(B):
        k[b, :, ~seen[b].any(0)], v[b, :, ~seen[b].any(0)] = float("nan"), float("inf")
    some = (seen[3].any(0) & ~seen[3].all(0)).nonzero().flatten()
    if len(some):
        v[3, 0, int(some[-1]), 5], v[3, 1, int(some[0]), 7], k[3, 2, int(some[-1]), 9] = float("nan"), float("inf"), float("nan")
    out = torch.full_like(q, 7.0)
    assert any("AttentionRowsKernel" in n for n in kernels(q, k, v, out, D ** -0.5, **more))
    pick = [0, 3, 5]  # (the definition's way takes its time: three sequences of the batch, three heads)
    more = {a: tuple(t[pick] for t in b) if a == "documents" else b[pick] if hasattr(b, "shape") and a != "slopes" else b for a, b in more.items()}
    q, k, v, out = (t[pick][:, :3] for t in (q, k, v, out))
    want, most, _ = oracle.attention(q, k, v, D ** -0.5, **more)
    got = out.double().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    fine = want.isfinite()
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    bound = oracle.attention_bound(want, torch.ones_like(most), q.dtype, D, Sq, D ** -0.5, more.get("cap", 0.0), 0.0)
    assert ((got - want).abs() <= bound)[fine].all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_attention_positions_many_rows_far_scores(device, dtype):
    import torch

    for order in (1, -1):
        q, k, v = draw(device, dtype_of(dtype), (3, 8, 1100, 64), (3, 8, 300, 64), (3, 8, 300, 64))
        ramp = torch.arange(300, device=device).to(torch.float32) / 300
        ramp = ramp if order == 1 else ramp.flip(0)
        k = (k * 0.1 + ramp[:, None] * torch.sign(q[:, :, :1].float())).to(q.dtype)
        out = torch.full_like(q, 7.0)
        oracle.call_attention(q, k, v, out, -8.0)
        check(q, k, v, out, -8.0, peak=1.1)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("Sq", [1, 40])
@pytest.mark.parametrize("D", [64, 128, 72])
def test_attention_positions_views(device, dtype, Sq, D):
    """Projections as they lie; a cache whose tokens lie apart; odd addresses; columns at a stride; one sequence's keys for all."""
    import torch

    B, H, KV, T = 2, 4, 2, 150
    kind = dtype_of(dtype)
    q, k, v = draw(device, kind, (B, Sq, H, D), (B, T, KV, D), (B, T, KV, D))
    views = {
        "tokens first": (q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)),
        "one tensor": tuple(draw(device, kind, (B, T, KV, 3 * D))[0].transpose(1, 2)[..., i * D:(i + 1) * D] for i in (1, 2)),
        "odd address": tuple(torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape).transpose(1, 2) for t in (k, v)),
        "columns apart": tuple(t.permute(0, 2, 3, 1).contiguous().transpose(2, 3) for t in (k, v)),
        "one for all": tuple(t[:1].transpose(1, 2).expand(B, KV, T, D) for t in (k, v)),
        "one key": tuple(t[:, :1].transpose(1, 2).expand(B, KV, T, D) for t in (k, v)),
    }
    for name, t in views.items():
        kk, vv = t[-2:]
        for turned in (False, True):
            qq = q.transpose(1, 2)
            if turned:
                qq = qq.transpose(2, 3).contiguous().transpose(2, 3)
            out = torch.full((B, Sq, D, H), 7.0, device=device, dtype=kind).permute(0, 3, 1, 2) if turned else torch.full_like(qq, 7.0)
            print("[case]", dtype, Sq, D, name, turned, flush=True)
            oracle.call_attention(qq, kk, vv, out, D ** -0.5, causal=True, cap=3.0)
            check(qq, kk, vv, out, D ** -0.5, causal=True, cap=3.0)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("Sq", [1, 3, 150])
@pytest.mark.parametrize("name", ["causal", "window", "documents", "lengths", "prefix"])
def test_attention_positions_hidden_values(device, dtype, Sq, name):
    """Infinities and NaN where a query does not look reach neither its weights nor its sums."""
    import torch

    B, H, KV, T, D = 3, 4, 2, 200, 64
    q, k, v = draw(device, dtype_of(dtype), (B, H, Sq, D), (B, KV, T, D), (B, KV, T, D))
    more = options(name, device, B, H, Sq, T)
    if name == "window":
        more["window"] = 20
    seen, _, _ = oracle.visible(B, Sq, T, **{a: b for a, b in more.items() if a not in ("cap", "slopes")})
    for b in range(B):
        hidden = (~seen[b].any(0)).nonzero().flatten()
        for n, j in enumerate(hidden.tolist()):  # seen by no query
            k[b, :, j], v[b, :, j] = (float("nan"), float("inf"), -float("inf"))[n % 3], (float("inf"), float("nan"))[n % 2]
    if Sq > 1 and name != "lengths":  # seen by some: these rows have it, the others do not
        for b in range(B):
            some = (seen[b].any(0) & ~seen[b].all(0)).nonzero().flatten()
            if len(some):
                v[b, 0, int(some[-1]), 5], v[b, 1, int(some[0]), 7], v[b, 1, int(some[-1]), 9] = float("nan"), float("inf"), -float("inf")
    out = torch.full_like(q, 7.0)
    oracle.call_attention(q, k, v, out, D ** -0.5, **more)
    want, most, _ = oracle.attention(q, k, v, D ** -0.5, **more)
    got = out.double().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    fine = want.isfinite()
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    size = torch.where(v.isfinite(), v, torch.zeros_like(v)).abs().max().item()
    bound = oracle.attention_bound(want, torch.full_like(most, size), q.dtype, D, T, D ** -0.5, more.get("cap", 0.0), 0.0)
    assert ((got - want).abs() <= bound)[fine].all()


def test_attention_positions_scores_not_finite(device):
    """A NaN in a query or a key makes its rows NaN and no others; scores beyond every float are what a softmax makes of them."""
    import torch

    for Sq in (1, 100):
        q, k, v = draw(device, torch.float32, (1, 2, Sq, 64), (1, 2, 130, 64), (1, 2, 130, 64))
        q[0, 0, 0, 3] = float("nan")
        k[0, 1, 129, 5] = float("nan")  # the last query's own
        out = torch.full_like(q, 7.0)
        oracle.call_attention(q, k, v, out, 0.125, causal=True)
        bad = out.isnan().all(-1)
        assert bad[0, 0].tolist() == [True] + [False] * (Sq - 1) and bad[0, 1].tolist() == [False] * (Sq - 1) + [True]
        assert torch.equal(out.isnan().any(-1), bad)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("Sq", [1, 140])
def test_attention_positions_far_scores(device, dtype, Sq):
    """Scores of several hundreds, whose largest comes last or first: sums are scaled as the maximum moves."""
    import torch

    kind = dtype_of(dtype)
    for order in (1, -1):
        q, k, v = draw(device, kind, (1, 2, Sq, 64), (1, 2, 300, 64), (1, 2, 300, 64))
        ramp = torch.arange(300, device=device).to(torch.float32) / 300
        ramp = ramp if order == 1 else ramp.flip(0)
        k = (k * 0.1 + ramp[:, None] * torch.sign(q[:, :, :1].float())).to(kind)
        out = torch.full_like(q, 7.0)
        oracle.call_attention(q, k, v, out, 8.0)
        check(q, k, v, out, 8.0, peak=1.1)


def test_attention_positions_large_offsets(device):
    """A cache whose last keys lie beyond 2^31 elements, one head a row of it."""
    import torch

    T, D = 70, 64
    pool = torch.zeros(2 ** 31 + (1 << 24), dtype=torch.bfloat16, device=device)
    stride = (2 ** 31) // (T - 1)
    k = pool.as_strided((1, 1, T, D), (0, 0, stride, 1))
    q, kk, vv = draw(device, torch.bfloat16, (1, 1, 5, D), (1, 1, T, D), (1, 1, T, D))
    v = pool.as_strided((1, 1, T, D), (0, 0, stride, 1), 4096)
    k.copy_(kk)
    v.copy_(vv)
    out = torch.empty_like(q)
    oracle.call_attention(q, k, v, out, 0.125, causal=True)
    check(q, kk, vv, out, 0.125, causal=True)


def test_attention_positions_captured(device):
    """A token's call recorded once and replayed as the cache grows, and the same on a stream that the library has never seen."""
    import torch

    B, H, KV, T, D = 2, 8, 2, 900, 128
    q, k, v = draw(device, torch.bfloat16, (B, H, 1, D), (B, KV, T, D), (B, KV, T, D))
    lengths = torch.tensor([1, 2], dtype=torch.int32, device=device)
    ids = torch.zeros(B, T, dtype=torch.int32, device=device)
    out, stream, graph = torch.empty_like(q), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    more = {"causal": True, "key_lengths": lengths, "documents": (ids[:, :1], ids)}
    scratch = oracle.call_attention(q, k, v, out, 0.1, **more)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        oracle.call_attention(q, k, v, out, 0.1, **more, stream=ctypes.c_void_p(torch.cuda.current_stream().cuda_stream), scratch=scratch)
    for step in (3, 150, 897):
        lengths.copy_(torch.tensor([step, step + 3], device=device))
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        check(q, k, v, got, 0.1, **more)
        oracle.call_attention(q, k, v, out, 0.1, **more)
        torch.cuda.synchronize()
        assert torch.equal(out, got)  # the same bits, every time


@pytest.mark.parametrize("B,H,KV,Sq,Skv", [(6, 2, 1, 3, 200), (6, 32, 32, 130, 90)], ids=["few", "many"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_attention_positions_far_starts(device, dtype, B, H, KV, Sq, Skv):
    """Starts up to the ends of 32 bits with windows that reach as far and windows of any 64-bit width, and biases of such distances."""
    import torch

    q, k, v = draw(device, dtype_of(dtype), (B, H, Sq, 64), (B, KV, Skv, 64), (B, KV, Skv, 64))
    starts = torch.tensor([2 ** 31 - 1, -2 ** 31, 2 ** 30 - 1, 40, 1 - 2 ** 30, -Sq], dtype=torch.int32, device=device)
    for causal in (True, False):
        for window in (0, 7, 2 ** 30, 2 ** 30 + 5, 2 ** 31 - 1, 2 ** 31 + 50, 2 ** 62):
            print("[case]", dtype, causal, window, flush=True)
            out = torch.full_like(q, 7.0)
            oracle.call_attention(q, k, v, out, 0.125, causal=causal, window=window, starts=starts)
            check(q, k, v, out, 0.125, causal=causal, window=window, starts=starts)
    # a bias of a far query is one number for all its keys: small slopes, so that its roundings (2^-24 of it) stay below the scores
    slopes = 2.0 ** -(24 + torch.arange(H, device=device, dtype=torch.float32) % 4)
    out = torch.full_like(q, 7.0)
    near = starts.clamp(-2 ** 24, 2 ** 24)
    oracle.call_attention(q, k, v, out, 0.125, slopes=slopes, starts=near)
    check(q, k, v, out, 0.125, slopes=slopes, starts=near)


def test_attention_positions_many_rows_large_offsets(device):
    """Keys and values beyond 2^31 elements where a workgroup has 128 rows: steps that 32 bits hold and steps that they do not."""
    import torch

    D, H, Sq = 64, 12, 2100
    pool = torch.zeros(2 ** 31 + (1 << 24), dtype=torch.bfloat16, device=device)
    for T in (70, 300):
        stride = (2 ** 31) // (T - 1) // 8 * 8
        k, v = (pool.as_strided((1, 1, T, D), (0, 0, stride, 1), at) for at in (0, 4096))
        q, kk, vv = draw(device, torch.bfloat16, (1, H, Sq, D), (1, 1, T, D), (1, 1, T, D))
        k.copy_(kk)
        v.copy_(vv)
        out = torch.empty_like(q)
        assert any("AttentionRowsKernel" in name for name in kernels(q, k, v, out, 0.125))
        oracle.call_attention(q, k, v, out, 0.125)
        check(q, kk, vv, out, 0.125)
