"""Rotary positions from positions: both layouts, part of the head, every stretch, far and negative positions, strides, in place,
against 64-bit angles and products."""
import ctypes
import math

import pytest

pytestmark = pytest.mark.gpu
KINDS = ("plain", "linear", "base", "wavelength", "dimension")


def plan_of(dims, interleaved=0, kind="plain", base=10000.0, amplitude=1.0):
    from fluidml_amd import cabi

    return cabi.FlRotaryPlan(interleaved, KINDS.index(kind), dims, base, 8.0, 2048.0, 1.0, 32.0 if kind == "dimension" else 4.0, amplitude)


def rates(plan):
    R, two_pi = plan.dims, 2 * math.pi
    found = []
    for j in range(R // 2):
        f = plan.base ** (-2.0 * j / R)
        if plan.scaling == 1:
            f /= plan.factor
        elif plan.scaling == 2 and R > 2:
            f = (plan.base * plan.factor ** (R / (R - 2.0))) ** (-2.0 * j / R)
        elif plan.scaling == 3:
            m = min(1.0, max(0.0, (plan.original_length * f / two_pi - plan.low) / (plan.high - plan.low)))
            f *= m + (1 - m) / plan.factor
        elif plan.scaling == 4:
            def at(turns):
                return R * math.log(plan.original_length / (two_pi * turns)) / (2 * math.log(plan.base))
            first, last = max(0, math.floor(at(plan.high))), min(R - 1, math.ceil(at(plan.low)))
            m = 1 - min(1.0, max(0.0, (j - first) / max(last - first, 0.001)))
            f *= m + (1 - m) / plan.factor
        found.append(f)
    return found


def oracle(x, positions, plan):
    """(result, what an error is measured against: |a| + |b| of each pair)"""
    import torch

    x, R = x.double().cpu(), plan.dims
    angle = positions.cpu().double().expand(x.shape[0], x.shape[2])[:, None, :, None] * torch.tensor(rates(plan), dtype=torch.float64)
    c, s = angle.cos() * plan.amplitude, angle.sin() * plan.amplitude
    first = torch.arange(0, R, 2) if plan.interleaved else torch.arange(R // 2)
    second = first + 1 if plan.interleaved else first + R // 2
    out, size = x.clone(), torch.zeros_like(x)
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * c - b * s, b * c + a * s
    size[..., first] = size[..., second] = (a.abs() + b.abs()) * abs(plan.amplitude)
    return out, size


def check(got, x, positions, plan):
    import torch

    want, size = oracle(x, positions, plan)
    # what is left of the angle is rounded to 32 bits (half a turn: 2^-26 of a turn, 2^-23.3 in the angle), sine and cosine and their
    # product with the amplitude (2^-23), the two products and their sum (2^-24 each); then the result to its type, half a step of the value, in fp16 below 2^-14, whose steps are 2^-24 there, half of that
    bound = size * 2.0 ** -21 + want.abs() * (torch.finfo(x.dtype).eps / 2 if x.dtype != torch.float32 else 0.0)
    bound = bound + (2.0 ** -25 if x.dtype == torch.float16 else 0.0)
    far = (got.double().cpu() - want).abs() - bound
    assert far.max() <= 0, f"{far.max()} over"
    assert torch.equal(got[..., plan.dims:].cpu(), x[..., plan.dims:].cpu())


def call(x, positions, out, plan, stream=None):
    from fluidml_amd import cabi

    cabi.call("rotary_positions", ctypes.byref(cabi.view(x)), ctypes.byref(cabi.view(positions)), ctypes.byref(cabi.view(out)), ctypes.byref(plan), stream)


def call_pair(x0, out0, x1, out1, positions, plan, stream=None):
    from fluidml_amd import cabi

    v = [ctypes.byref(cabi.view(t)) for t in (x0, out0, x1, out1, positions)]
    cabi.call("rotary_positions_pair", *v, ctypes.byref(plan), stream)


def dtype_of(name):
    import torch

    return {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}[name]


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("B,H,S,D,R", [
    (1, 1, 1, 2, 2), (1, 3, 5, 7, 2), (2, 3, 7, 64, 16), (3, 2, 9, 80, 20), (2, 5, 3, 96, 36), (1, 8, 33, 128, 128),
    (2, 2, 2, 1040, 1024),   # as many angles as a workgroup keeps
    (5, 2, 431, 64, 64),     # several tokens to a workgroup, sequences that end inside one
    (1, 70, 2100, 16, 12),
])
def test_rotary_positions(device, dtype, interleaved, B, H, S, D, R):
    import torch

    print("[case]", dtype, interleaved, B, H, S, D, R, flush=True)
    g = torch.Generator(device=device).manual_seed(S + D)
    x = torch.randn(B, H, S, D, device=device, generator=g).to(dtype_of(dtype))
    positions = torch.randint(-100, 100000, (B, S), device=device, generator=g)
    out = torch.full_like(x, 7.0)
    plan = plan_of(R, interleaved)
    call(x, positions, out, plan)
    check(out, x, positions, plan)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dims", [2, 64, 100])
def test_rotary_positions_scaled(device, kind, dims):
    import torch

    g = torch.Generator(device=device).manual_seed(dims)
    x = torch.randn(2, 3, 40, 112, device=device, generator=g)
    # far enough that an angle in 32 bits would be wrong in every bit
    positions = torch.randint(0, 1 << 30, (2, 40), device=device, generator=g, dtype=torch.int32)
    positions[0, :4] = torch.tensor([0, 1, 2047, 2048], device=device)
    out = torch.empty_like(x)
    plan = plan_of(dims, 0, kind, 500000.0, 1.25)
    call(x, positions, out, plan)
    check(out, x, positions, plan)


def test_rotary_positions_views(device):
    """Projections as they lie, one position list for all sequences, columns at a stride, addresses at odd elements, in place."""
    import torch

    g = torch.Generator(device=device).manual_seed(5)
    for dtype in (torch.float32, torch.bfloat16):
        for interleaved in (0, 1):
            flat = torch.randn(3 * 11 * 9 * 64 + 1, device=device, generator=g).to(dtype)
            plan = plan_of(32, interleaved)
            positions = torch.randint(0, 5000, (1, 11), device=device, generator=g, dtype=torch.int32)
            x = flat[1:].view(3, 11, 9, 64).transpose(1, 2)                     # odd address
            out = torch.empty(3, 9, 64, 11, device=device, dtype=dtype).transpose(2, 3)  # columns at a stride
            call(x, positions, out, plan)
            check(out, x, positions, plan)
            x = flat[:-1].view(3, 11, 9, 64).transpose(1, 2)
            want = torch.empty_like(x)
            call(x, positions[0], want, plan)
            check(want, x, positions, plan)
            whole = flat.clone()
            call(whole[:-1].view(3, 11, 9, 64).transpose(1, 2), positions[0], whole[:-1].view(3, 11, 9, 64).transpose(1, 2), plan)
            assert torch.equal(whole[:-1].view(3, 11, 9, 64).transpose(1, 2), want)
            x = torch.randn(1, 9, 11, 64, device=device, generator=g).to(dtype).expand(3, 9, 11, 64)  # one operand for three results
            out = torch.empty(3, 9, 11, 64, device=device, dtype=dtype)
            call(x, positions, out, plan)
            check(out, x, positions, plan)


def test_rotary_positions_pair(device):
    """Queries and keys of one launch are what two launches give, a token or many; the values beside a result stay."""
    import torch

    g = torch.Generator(device=device).manual_seed(6)
    for B, S in ((6, 1), (3, 1000)):
        q = torch.randn(B, S, 8, 64, device=device, generator=g).bfloat16().transpose(1, 2)
        k = torch.randn(B, S, 2, 64, device=device, generator=g).bfloat16().transpose(1, 2)
        cache = torch.full((B, 2, S + 5, 64), 3.0, device=device, dtype=torch.bfloat16)
        positions = torch.randint(0, 9000, (B, S), device=device, generator=g)
        q_out, alone, plan = torch.empty_like(q), torch.empty_like(q), plan_of(64, 1)
        call_pair(q, q_out, k, cache[:, :, 2:2 + S], positions, plan)
        call(q, positions, alone, plan)
        assert torch.equal(q_out, alone)
        check(q_out, q, positions, plan)
        check(cache[:, :, 2:2 + S], k, positions, plan)
        assert (cache[:, :, :2] == 3).all() and (cache[:, :, 2 + S:] == 3).all()


def test_rotary_positions_not_finite(device):
    """An infinity or a NaN stays in its pair."""
    import torch

    x = torch.ones(1, 1, 4, 64, device=device)
    x[0, 0, 1, 3], x[0, 0, 2, 40], x[0, 0, 3, 63] = float("nan"), float("inf"), float("nan")
    out = torch.empty_like(x)
    call(x, torch.tensor([1, 2, 3, 4], device=device), out, plan_of(32))
    bad = ~out.isfinite().cpu()[0, 0]
    assert bad.nonzero().tolist() == [[1, 3], [1, 19], [2, 40], [3, 63]]


def test_rotary_positions_captured(device):
    import torch

    g = torch.Generator(device=device).manual_seed(7)
    q, k = torch.randn(4, 8, 3, 64, device=device, generator=g), torch.randn(4, 2, 3, 64, device=device, generator=g)
    positions, plan = torch.zeros(4, 3, dtype=torch.int64, device=device), plan_of(64)
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call_pair(q, q_out, k, k_out, positions, plan, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    for step in range(3):
        positions.copy_(torch.randint(0, 1000, (4, 3), device=device, generator=g))
        q.mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        check(q_out, q, positions, plan)
        check(k_out, k, positions, plan)
