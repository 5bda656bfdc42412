"""The decoder operators as a layer uses them: rotary positions into a cache, attention over it, the gated block; a prompt, tokens from a
recorded graph, two layers at once.  Each stage is held to its own bound against 64 bits, from the operands that it really had."""
import ctypes

import pytest

from tests import decoder_oracle as oracle, test_gpu_gated as blocks, test_gpu_rotary_positions as rotary

pytestmark = pytest.mark.gpu
B, H, KV, D, WIDTH, INNER, ROOM = 3, 8, 2, 64, 512, 1376, 160


class Layer:
    """Weights of one layer, its cache [B, KV, ROOM, D] and how far each sequence has come."""

    def __init__(self, device, kind, seed=0):
        import torch

        g = torch.Generator(device=device).manual_seed(seed)

        def normal(*shape, by):
            return (torch.randn(*shape, device=device, generator=g) * by).to(kind)

        self.kind, self.device = kind, device
        self.qkv = normal(WIDTH, (H + 2 * KV) * D, by=WIDTH ** -0.5)
        self.back = normal(H * D, WIDTH, by=(H * D) ** -0.5)
        self.gate, self.up = (normal(INNER, WIDTH, by=WIDTH ** -0.5).t() for _ in range(2))
        self.down = normal(WIDTH, INNER, by=INNER ** -0.5).t()
        self.keys, self.values = (torch.zeros(B, KV, ROOM, D, device=device, dtype=kind) for _ in range(2))
        self.lengths = torch.zeros(B, dtype=torch.int32, device=device)
        self.plan = rotary.plan_of(D, base=10000.0)

    def run(self, x, rows=None, stream=None):
        """x [B, S, WIDTH] of the next tokens; rows [B]: how many of the S are tokens.  Returns all that passes between the operators."""
        import torch

        S = x.shape[1]
        rows = torch.full((B,), S, dtype=torch.int32, device=self.device) if rows is None else rows
        q, k, v = (x @ self.qkv).split([H * D, KV * D, KV * D], 2)
        q, k, v = (t.unflatten(2, (-1, D)).transpose(1, 2) for t in (q, k, v))
        positions = self.lengths[:, None] + torch.arange(S, device=self.device, dtype=torch.int32)
        turned_q, turned_k = torch.empty_like(q), torch.empty_like(k)
        rotary.call_pair(q, turned_q, k, turned_k, positions, self.plan, stream)
        # behind a shorter sequence's rows the cache takes what the next call writes over
        at = positions.long().clamp(max=ROOM - 1)[:, None, :, None].expand(B, KV, S, D)
        self.keys.scatter_(2, at, turned_k)
        self.values.scatter_(2, at, v)
        self.lengths += rows
        mixed = torch.zeros(B, H, S, D, device=self.device, dtype=self.kind)
        scratch = oracle.call_attention(turned_q, self.keys, self.values, mixed, D ** -0.5, causal=True, query_lengths=rows,
                                        key_lengths=self.lengths, stream=stream)
        residual = (x + mixed.transpose(1, 2).flatten(2) @ self.back).view(B * S, WIDTH)
        products = torch.empty(B * S, INNER, device=self.device, dtype=self.kind)
        out = torch.empty_like(residual)
        blocks.call_block(residual, self.gate, self.up, None, None, self.down, None, residual, products, out, "silu", stream)
        return {"q": q, "k": k, "turned_q": turned_q, "turned_k": turned_k, "positions": positions, "mixed": mixed, "rows": rows,
                "residual": residual, "products": products, "out": out, "scratch": scratch}

    def again(self, r, attention=True):
        """The same calls one after the other, from the same operands: the same bits."""
        import torch

        new = {name: torch.zeros_like(r[name]) for name in ("turned_q", "turned_k", "mixed", "products", "out")}
        rotary.call_pair(r["q"], new["turned_q"], r["k"], new["turned_k"], r["positions"], self.plan)
        blocks.call_block(r["residual"], self.gate, self.up, None, None, self.down, None, r["residual"], new["products"], new["out"], "silu")
        if attention:  # (the cache and the lengths are still those of this step)
            oracle.call_attention(r["turned_q"], self.keys, self.values, new["mixed"], D ** -0.5, causal=True, query_lengths=r["rows"],
                                  key_lengths=self.lengths)
        torch.cuda.synchronize()
        for name, t in new.items():
            assert torch.equal(t, r[name]) or (name == "mixed" and not attention), name

    def check(self, r):
        import torch

        rotary.check(r["turned_q"], r["q"], r["positions"], self.plan)
        rotary.check(r["turned_k"], r["k"], r["positions"], self.plan)
        masks = {"causal": True, "query_lengths": r["rows"], "key_lengths": self.lengths}
        want, most, written = oracle.attention(r["turned_q"], self.keys, self.values, D ** -0.5, **masks)
        peak = float(max(r["turned_q"].abs().max(), self.keys.abs().max()))
        bound = oracle.attention_bound(want, most, self.kind, D, ROOM, D ** -0.5, 0.0, 0.0, peak)
        seen = written[:, None, :].expand(r["mixed"].shape[:3])
        blocks.check(r["mixed"].cpu()[seen], want[seen], bound[seen])
        assert (r["mixed"].cpu()[~seen] == 0).all()
        want, bound = oracle.gated(r["residual"], self.gate, self.up, None, None, "silu")
        blocks.check(r["products"], want, oracle.rounded(bound, want, self.kind))
        h, d, x = r["products"].double().cpu(), self.down.double().cpu(), r["residual"].double().cpu()
        want = h @ d + x
        bound = 2.0 ** -24 * (INNER + 4) * (h.abs() @ d.abs()) + 2.0 ** -24 * 2 * (want.abs() + x.abs())
        blocks.check(r["out"], want, oracle.rounded(bound, want, self.kind))


def tokens(device, kind, S, seed):
    import torch

    return torch.randn(B, S, WIDTH, device=device, generator=torch.Generator(device=device).manual_seed(seed)).to(kind)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_prompt_and_tokens(device, dtype):
    """A ragged prompt, then tokens one by one, then several at once."""
    import torch

    kind = rotary.dtype_of(dtype)
    layer = Layer(device, kind)
    for step, (S, rows) in enumerate([(70, [70, 1, 33]), (1, None), (1, None), (5, [5, 3, 4]), (40, None)]):
        print("[case]", dtype, step, S, flush=True)
        rows = None if rows is None else torch.tensor(rows, dtype=torch.int32, device=device)
        layer.check(layer.run(tokens(device, kind, S, step), rows))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_recorded_token(device, dtype):
    """A token's whole step in a graph, replayed as the cache grows."""
    import torch

    kind = rotary.dtype_of(dtype)
    layer = Layer(device, kind)
    x = tokens(device, kind, 1, 1)
    layer.run(tokens(device, kind, 20, 0))
    layer.run(x)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        r = layer.run(x, stream=ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    for step in range(4):
        print("[case]", dtype, step, flush=True)
        x.copy_(tokens(device, kind, 1, 10 + step))
        graph.replay()
        torch.cuda.synchronize()
        assert layer.lengths.tolist() == [22 + step] * B
        layer.check(r)
        layer.again(r)


def test_two_layers_at_once(device):
    """Two layers on two streams, each with scratch of its own."""
    import torch

    kind = torch.bfloat16
    inputs = [tokens(device, kind, S, seed) for seed, S in enumerate((60, 1, 1, 7, 1))]
    layers, streams, found = [Layer(device, kind, seed) for seed in (1, 2)], [torch.cuda.Stream() for _ in range(2)], [[], []]
    torch.cuda.synchronize()
    for x in inputs:
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                found[i].append(layers[i].run(x, stream=ctypes.c_void_p(streams[i].cuda_stream)))
    torch.cuda.synchronize()
    for i in range(2):
        layers[i].check(found[i][-1])
        for step, r in enumerate(found[i]):
            layers[i].again(r, attention=step == len(inputs) - 1)
