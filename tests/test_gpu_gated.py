"""The gated feed-forward block against 64 bits: types, activations, biases, layouts of the weights, sizes that no tile divides."""
import ctypes

import pytest

from tests import decoder_oracle as oracle

pytestmark = pytest.mark.gpu


def dtype_of(name):
    import torch

    return {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}[name]


def ref(t):
    from fluidml_amd import cabi

    return None if t is None else ctypes.byref(cabi.view(t))


def call(x, gate, up, gate_bias, up_bias, products, kind, stream=None):
    from fluidml_amd import cabi

    cabi.call("gated_matmul", ref(x), ref(gate), ref(up), ref(gate_bias), ref(up_bias), ref(products), oracle.ACTIVATIONS.index(kind), stream)


def call_block(x, gate, up, gate_bias, up_bias, down, down_bias, addend, products, out, kind, stream=None):
    from fluidml_amd import cabi

    cabi.call("gated_feed_forward", ref(x), ref(gate), ref(up), ref(gate_bias), ref(up_bias), ref(down), ref(down_bias), ref(addend), ref(products),
              ref(out), oracle.ACTIVATIONS.index(kind), stream)


def make(device, dtype, M, K, N, turned, biased, seed=0):
    import torch

    g = torch.Generator(device=device).manual_seed(seed + M + K + N)

    def normal(*shape, by=1.0):
        return (torch.randn(*shape, device=device, generator=g) * by).to(dtype)

    x = normal(M, K)
    gate, up = (normal(N, K, by=K ** -0.5).t() if turned else normal(K, N, by=K ** -0.5) for _ in range(2))
    return x, gate, up, *((normal(N), normal(N)) if biased else (None, None))


def check(got, want, bound):
    far = (got.double().cpu() - want).abs() - bound
    assert not far.isnan().any() and (far <= 0).all(), f"{far.max()} over at {far.argmax()}"


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("turned", [True, False], ids=["rows", "columns"])
@pytest.mark.parametrize("M,K,N", [
    (1, 1, 1), (1, 64, 64), (2, 100, 33), (5, 512, 200), (16, 1024, 96), (17, 72, 130), (31, 256, 515), (33, 999, 77), (64, 96, 256), (100, 640, 640),
    (129, 200, 129), (257, 64, 1000), (300, 1032, 264), (513, 520, 520), (1, 11008, 40), (3, 8200, 24),
])
def test_gated_matmul(device, dtype, turned, M, K, N):
    import torch

    print("[case]", dtype, turned, M, K, N, flush=True)
    kind = dtype_of(dtype)
    biased = M % 2 == 1
    x, gate, up, gb, ub = make(device, kind, M, K, N, turned, biased)
    out = torch.full((M, N), 7.0, device=device, dtype=kind)
    call(x, gate, up, gb, ub, out, "silu")
    want, bound = oracle.gated(x, gate, up, gb, ub, "silu")
    check(out, want, oracle.rounded(bound, want, kind))


def kernels(run):
    """Names of what run(stream) launches."""
    from tests.util import launches

    run(None)
    return [name for name, _ in launches(run)]


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("turned", [True, False], ids=["rows", "columns"])
@pytest.mark.parametrize("M,K,N,tile", [
    (2003, 200, 1100, 128), (2100, 71, 1111, 128),    # tiles of 128 rows: columns, depth and rows that they do not divide
    (3400, 136, 2000, 256), (3333, 70, 1999, 256), (3500, 64, 1984, 256), (3400, 192, 2000, 256), (3601, 448, 1920, 256),
])
def test_gated_matmul_many_rows(device, dtype, turned, M, K, N, tile):
    import torch

    print("[case]", dtype, turned, M, K, N, flush=True)
    kind = dtype_of(dtype)
    x, gate, up, gb, ub = make(device, kind, M, K, N, turned, M % 2 == 1)
    out = torch.full((M, N), 7.0, device=device, dtype=kind)
    name, = kernels(lambda stream: call(x, gate, up, gb, ub, out, "silu", stream))
    if dtype == "fp32" or K % 64 != 0:  # tiles of 256 rows are for 16-bit operands and whole stages
        tile = 128
    assert f"Li{tile}ELi{tile}E" in name
    out.fill_(7.0)
    call(x, gate, up, gb, ub, out, "silu")
    want, bound = oracle.gated(x, gate, up, gb, ub, "silu")
    check(out, want, oracle.rounded(bound, want, kind))
    # one matrix, from the products on
    down = (torch.randn(K, N, device=device) * N ** -0.5).to(kind).t()
    if not turned:
        down = down.contiguous()
    addend, products, back = torch.randn(M, K, device=device).to(kind), torch.empty_like(out), torch.full((M, K), 7.0, device=device, dtype=kind)
    call_block(x, gate, up, gb, ub, down, None, addend, products, back, "silu")
    assert torch.equal(products, out)
    h, d = products.double().cpu(), down.double().cpu()
    want = h @ d + addend.double().cpu()
    check(back, want, oracle.rounded(2.0 ** -24 * (N + 4) * (h.abs() @ d.abs()) + 2.0 ** -24 * 2 * (want.abs() + addend.double().cpu().abs()), want, kind))


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_gated_down_many_rows(device, dtype):
    """The projection back in the largest tiles, with a bias."""
    import torch

    kind = dtype_of(dtype)
    M, K, N, Oc = 3400, 64, 192, 4000
    x, gate, up, gb, ub = make(device, kind, M, K, N, True, True)
    for turned in (True, False):
        down = (torch.randn(Oc, N, device=device) * N ** -0.5).to(kind).t()
        if not turned:
            down = down.contiguous()
        bias, products, out = torch.randn(Oc, device=device).to(kind), torch.empty(M, N, device=device, dtype=kind), torch.empty(M, Oc, device=device, dtype=kind)
        names = kernels(lambda stream: call_block(x, gate, up, gb, ub, down, bias, None, products, out, "gelu", stream))
        assert dtype == "fp32" or "Li256ELi256E" in names[1]
        h, d = products.double().cpu(), down.double().cpu()
        want = h @ d + bias.double().cpu()
        check(out, want, oracle.rounded(2.0 ** -24 * (N + 4) * (h.abs() @ d.abs()) + 2.0 ** -24 * 2 * (want.abs() + bias.double().cpu().abs()), want, kind))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_gated_many_rows_not_finite(device, dtype):
    import torch

    x, gate, up, _, _ = make(device, dtype_of(dtype), 3400, 72, 2000, True, False)
    gate[50, 7], up[3, 1960], x[3399, 71], x[5, 0] = float("nan"), float("inf"), float("nan"), -float("inf")
    out = torch.empty(3400, 2000, device=device, dtype=x.dtype)
    call(x, gate, up, None, None, out, "relu")
    want, bound = oracle.gated(x, gate, up, None, None, "relu")
    assert torch.equal(out.isnan().cpu(), want.isnan()) and torch.equal(out.isinf().cpu(), want.isinf())
    fine = want.isfinite()
    assert ((out.double().cpu() - want).abs() <= oracle.rounded(torch.nan_to_num(bound, nan=0.0, posinf=0.0) + 1e-6 * 72, want, x.dtype))[fine].all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("kind", oracle.ACTIVATIONS)
def test_gated_activations(device, dtype, kind):
    """Over the gates' whole range: sums from none to large ones of either sign."""
    import torch

    for M in (3, 130):
        x, gate, up, gb, ub = make(device, dtype_of(dtype), M, 128, 192, True, True)
        gb = (torch.linspace(-30, 30, 192, device=device)).to(x.dtype)
        out = torch.empty(M, 192, device=device, dtype=x.dtype)
        call(x, gate, up, gb, ub, out, kind)
        want, bound = oracle.gated(x, gate, up, gb, ub, kind)
        check(out, want, oracle.rounded(bound, want, x.dtype))


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_gated_far_gates(device, dtype):
    """Gates of the type's largest values and infinities give what the activation tends to, never a NaN from an overflow inside."""
    import torch

    kind = dtype_of(dtype)
    big = torch.finfo(kind).max
    gates = torch.tensor([big, -big, 1000.0, -1000.0, 0.0, float("inf"), float("nan")], dtype=kind, device=device)
    x, gate, up = torch.ones(2, 1, device=device, dtype=kind), gates[None, :].contiguous(), torch.ones(1, 7, device=device, dtype=kind)
    for name in oracle.ACTIVATIONS:
        out = torch.empty(2, 7, device=device, dtype=kind)
        call(x, gate, up, None, None, out, name)
        got = out.double().cpu()
        limit = {"sigmoid": [1, 0, 1, 0, 0.5, 1]}.get(name, [float(big), -float(big) if name == "identity" else 0, 1000,
                                                               -1000 if name == "identity" else 0, 0, float("inf")])
        assert got[0, :6].tolist() == [float(v) for v in limit], name
        assert got[:, 6].isnan().all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("M", [1, 20, 200])
def test_gated_views(device, dtype, M):
    """The halves of one tensor, rows apart, odd addresses, operands with neither side at a unit stride, results at a stride."""
    import torch

    kind = dtype_of(dtype)
    K, N = 264, 136
    x, gate, up, gb, ub = make(device, kind, M, K, N, True, True)
    both = torch.cat([gate.t(), up.t()])                       # [2 N, K]
    wide = torch.cat([gate, up], 1).contiguous()               # [K, 2 N]
    spread = torch.zeros(2 * K, 3 * N, device=device, dtype=kind)[::2, ::3]
    spread.copy_(gate)
    odd = torch.cat([up.t().flatten()[:1], up.t().flatten()])[1:].view(N, K).t()
    rows = torch.zeros(M, K + 24, device=device, dtype=kind)[:, :K]
    rows.copy_(x)
    apart = x.t().contiguous().t()
    want, bound = oracle.gated(x, gate, up, gb, ub, "gelu")
    bound = oracle.rounded(bound, want, kind)
    for name, xx, g, u in [("halves", x, both[:N].t(), both[N:].t()), ("wide", rows, wide[:, :N], wide[:, N:]), ("spread", x, spread, up),
                           ("odd", rows, gate, odd), ("columns first", apart, gate, up), ("two layouts", x, gate, up.contiguous())]:
        for out in (torch.full((M, N), 7.0, device=device, dtype=kind), torch.full((N, M), 7.0, device=device, dtype=kind).t(),
                    torch.full((M, N + 7), 7.0, device=device, dtype=kind)[:, :N]):
            print("[case]", dtype, M, name, tuple(out.stride()), flush=True)
            call(xx, g, u, gb, ub[:1].expand(N) if name == "spread" else ub, out, "gelu")
            if name != "spread":
                check(out, want, bound)
            if out.stride(0) == N + 7:
                assert (out.as_strided((M, 7), (N + 7, 1), N) == 7.0)[:-1].all()
    want, bound = oracle.gated(x, gate, up, gb, ub[:1].expand(N), "gelu")
    out = torch.empty(M, N, device=device, dtype=kind)
    call(x, spread, up, gb, ub[:1].expand(N), out, "gelu")
    check(out, want, oracle.rounded(bound, want, kind))


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("turned", [True, False], ids=["rows", "columns"])
@pytest.mark.parametrize("M,K,N,O", [(1, 256, 704, 256), (7, 130, 99, 61), (40, 512, 1376, 512), (260, 320, 300, 328), (2, 64, 20000, 16)])
def test_gated_feed_forward(device, dtype, turned, M, K, N, O):
    import torch

    print("[case]", dtype, turned, M, K, N, O, flush=True)
    kind = dtype_of(dtype)
    x, gate, up, gb, ub = make(device, kind, M, K, N, turned, True)
    g = torch.Generator(device=device).manual_seed(9)
    down = (torch.randn(O, N, device=device, generator=g) * N ** -0.5).to(kind).t()
    if not turned:
        down = down.contiguous()
    for with_addend in (False, True):
        bias = torch.randn(O, device=device, generator=g).to(kind) if with_addend else None
        addend = torch.randn(M, O, device=device, generator=g).to(kind) if with_addend else None
        products, out = torch.full((M, N), 7.0, device=device, dtype=kind), addend.clone() if with_addend else torch.full((M, O), 7.0, device=device, dtype=kind)
        call_block(x, gate, up, gb, ub, down, bias, out if with_addend else None, products, out, "silu")
        want, bound = oracle.gated(x, gate, up, gb, ub, "silu")
        check(products, want, oracle.rounded(bound, want, kind))
        h, d = products.double().cpu(), down.double().cpu()  # (the products themselves are held to their own bound)
        want = h @ d
        bound = 2.0 ** -24 * (N + 4) * (h.abs() @ d.abs())
        if with_addend:
            want = want + bias.double().cpu() + addend.double().cpu()
            bound = bound + 2.0 ** -24 * 2 * (want.abs() + addend.double().cpu().abs() + bias.double().cpu().abs())
        check(out, want, oracle.rounded(bound, want, kind))


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("M", [2, 150])
def test_gated_not_finite(device, dtype, M):
    """An infinity or a NaN of x reaches its row, one of a weight its column, and nothing else."""
    import torch

    kind = dtype_of(dtype)
    x, gate, up, _, _ = make(device, kind, M, 100, 90, True, False)
    clean = torch.empty(M, 90, device=device, dtype=kind)
    call(x, gate, up, None, None, clean, "silu")
    gate[50, 7], up[3, 60] = float("nan"), float("inf")
    x[M - 1, 99] = float("nan")
    out = torch.empty_like(clean)
    call(x, gate, up, None, None, out, "silu")
    want, _ = oracle.gated(x, gate, up, None, None, "silu")
    assert torch.equal(out.isnan().cpu(), want.isnan()) and torch.equal(out.isinf().cpu(), want.isinf())
    fine = want.isfinite()
    assert torch.equal(out.cpu()[fine], clean.cpu()[fine])


def test_gated_small_and_large_values(device):
    """fp32 operands near both ends of the range."""
    import torch

    for M in (2, 150):
        for by_x, by_w in ((1e-18, 1e-18), (1e18, 1e-18), (1e15, 1e15), (1.0, 1e-30)):
            x, gate, up, _, _ = make(device, torch.float32, M, 96, 80, True, False)
            x, gate = x * by_x, gate * by_w
            out = torch.empty(M, 80, device=device)
            call(x, gate, up, None, None, out, "identity")
            want, bound = oracle.gated(x, gate, up, None, None, "identity")
            beyond = want.abs() > torch.finfo(torch.float32).max  # (rounded to fp32: an infinity; 1e15 three times)
            assert torch.equal(out.double().cpu()[beyond], want.float().double()[beyond])
            fine = ~beyond
            check(out.cpu()[fine], want[fine], (bound + 2.0 ** -126 * 96)[fine])  # (a denormal number may be taken for none)


def test_gated_captured(device):
    import torch

    x, gate, up, gb, ub = make(device, torch.bfloat16, 8, 512, 768, True, True)
    down = torch.randn(512, 768, device=device).mul(0.03).bfloat16().t()
    products, out = torch.empty(8, 768, device=device, dtype=torch.bfloat16), torch.empty(8, 512, device=device, dtype=torch.bfloat16)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call_block(x, gate, up, gb, ub, down, None, None, products, out, "silu", ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    for _ in range(3):
        x.mul_(-0.75)
        graph.replay()
        torch.cuda.synchronize()
        got = products.clone(), out.clone()
        call_block(x, gate, up, gb, ub, down, None, None, products, out, "silu")
        torch.cuda.synchronize()
        assert torch.equal(got[0], products) and torch.equal(got[1], out)
        want, bound = oracle.gated(x, gate, up, gb, ub, "silu")
        check(products, want, oracle.rounded(bound, want, torch.bfloat16))


MIDDLE = [(500, 200, 1500), (497, 71, 1501), (512, 1032, 1536), (450, 4200, 1500)]  # too few rows for tiles of 128


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("turned", [True, False], ids=["rows", "columns"])
@pytest.mark.parametrize("M,K,N", MIDDLE)
def test_gated_middle_tiles(device, dtype, turned, M, K, N):
    """Tiles of 64 rows, whose waves share the depth, with two matrices and with one."""
    import torch

    print("[case]", dtype, turned, M, K, N, flush=True)
    kind = dtype_of(dtype)
    x, gate, up, gb, ub = make(device, kind, M, K, N, turned, M % 2 == 1)
    Oc = 2010 + K % 2
    down = (torch.randn(Oc, N, device=device) * N ** -0.5).to(kind).t()
    if not turned:
        down = down.contiguous()
    bias, addend = torch.randn(Oc, device=device).to(kind), torch.randn(M, Oc, device=device).to(kind)
    products, out = torch.full((M, N), 7.0, device=device, dtype=kind), torch.full((M, Oc), 7.0, device=device, dtype=kind)
    names = kernels(lambda stream: call_block(x, gate, up, gb, ub, down, bias, addend, products, out, "silu", stream))
    tile = "Li64ELi128E" if dtype == "fp32" else "Li64ELi64E"
    assert len(names) == 2 and all(tile in name for name in names), names
    products.fill_(7.0), out.fill_(7.0)
    call_block(x, gate, up, gb, ub, down, bias, addend, products, out, "silu")
    want, bound = oracle.gated(x, gate, up, gb, ub, "silu")
    check(products, want, oracle.rounded(bound, want, kind))
    h, d = products.double().cpu(), down.double().cpu()
    want = h @ d + bias.double().cpu() + addend.double().cpu()
    bound = 2.0 ** -24 * (N + 4) * (h.abs() @ d.abs()) + 2.0 ** -24 * 2 * (want.abs() + addend.double().cpu().abs() + bias.double().cpu().abs())
    check(out, want, oracle.rounded(bound, want, kind))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_gated_middle_tiles_not_finite(device, dtype):
    import torch

    M, K, N = 500, 136, 1500
    x, gate, up, _, _ = make(device, dtype_of(dtype), M, K, N, True, False)
    gate[50, 7], up[3, 1460], x[M - 1, K - 1], x[5, 0], up[0, 9] = float("nan"), float("inf"), float("nan"), -float("inf"), 0.0
    out = torch.empty(M, N, device=device, dtype=x.dtype)
    call(x, gate, up, None, None, out, "relu")
    want, bound = oracle.gated(x, gate, up, None, None, "relu")
    assert torch.equal(out.isnan().cpu(), want.isnan()) and torch.equal(out.isinf().cpu(), want.isinf())
    fine = want.isfinite()  # (what is finite here saw finite operands alone, unless an infinite gate was shut: 0 times a finite sum)
    assert ((out.double().cpu() - want).abs() <= oracle.rounded(torch.nan_to_num(bound, nan=0.0, posinf=0.0), want, x.dtype))[fine].all()


@pytest.mark.parametrize("M", [500, 2003])
def test_gated_tiles_small_and_large_values(device, M):
    """fp32 operands near both ends of the range, in tiles whose products are made of parts."""
    import torch

    for by_x, by_w in ((1e-18, 1e-18), (1e18, 1e-18), (1e15, 1e15), (1.0, 1e-30)):
        x, gate, up, _, _ = make(device, torch.float32, M, 96, 1500, True, False)
        x, gate = x * by_x, gate * by_w
        out = torch.empty(M, 1500, device=device)
        call(x, gate, up, None, None, out, "identity")
        want, bound = oracle.gated(x, gate, up, None, None, "identity")
        beyond = want.abs() > torch.finfo(torch.float32).max
        assert torch.equal(out.double().cpu()[beyond], want.float().double()[beyond])
        fine = ~beyond
        # a product of the first sum below the normal numbers may be taken for none, 96 of them, and the other sum multiplies what is lost
        lost = 2.0 ** -126 * 96 * (1 + (x.double().cpu() @ up.double().cpu()).abs())
        check(out.cpu()[fine], want[fine], (bound + lost)[fine])


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("M", [500, 2003])
def test_gated_tiles_views(device, dtype, M):
    """Operands at odd addresses and odd strides, halves of one tensor, rows apart, results in columns, in tiles."""
    import torch

    kind = dtype_of(dtype)
    K, N = 264, 1500
    x, gate, up, gb, ub = make(device, kind, M, K, N, True, True)

    def shifted(t, by):  # the same values `by` values behind an aligned address, rows an odd number of values apart
        rows, columns = t.shape
        flat = torch.full((rows * (columns + 3) + by,), float("nan"), device=device, dtype=kind)
        view = flat[by:].as_strided((rows, columns), (columns + 3, 1))
        return view.copy_(t)

    spread = torch.zeros(M, 2 * K, device=device, dtype=kind)[:, ::2]
    spread.copy_(x)
    wide = torch.cat([gate, up], 1).contiguous()
    want, bound = oracle.gated(x, gate, up, gb, ub, "gelu")
    bound = oracle.rounded(bound, want, kind)
    for name, xx, g, u in [("odd rows", shifted(x, 1), shifted(gate.t(), 3).t(), shifted(up.t(), 1).t()), ("wide", x, wide[:, :N], wide[:, N:]),
                           ("odd columns", shifted(x, 2), shifted(gate, 1), shifted(up, 5)), ("spread", spread, gate, up),
                           ("columns first", x.t().contiguous().t(), gate, up), ("two layouts", x, gate, up.contiguous())]:
        for out in (torch.full((M, N), 7.0, device=device, dtype=kind), torch.full((N, M), 7.0, device=device, dtype=kind).t(),
                    torch.full((M, N + 7), 7.0, device=device, dtype=kind)[:, :N]):
            print("[case]", dtype, M, name, tuple(out.stride()), flush=True)
            call(xx, g, u, gb, ub, out, "gelu")
            check(out, want, bound)
            if out.stride(0) == N + 7:
                assert (out.as_strided((M, 7), (N + 7, 1), N) == 7.0)[:-1].all()


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("turned", [True, False], ids=["rows", "columns"])
@pytest.mark.parametrize("M,K,N", [(500, 1, 1500), (500, 5, 1500), (2003, 7, 1100), (20001, 40, 3), (33000, 71, 1), (20000, 3, 5)])
def test_gated_tiles_thin(device, dtype, turned, M, K, N):
    """A depth or columns below one load's values, in tiles."""
    import torch

    print("[case]", dtype, turned, M, K, N, flush=True)
    kind = dtype_of(dtype)
    x, gate, up, gb, ub = make(device, kind, M, K, N, turned, True)
    out = torch.full((M, N), 7.0, device=device, dtype=kind)
    name, = kernels(lambda stream: call(x, gate, up, gb, ub, out, "silu", stream))
    assert "GatedTileKernel" in name
    out.fill_(7.0)
    call(x, gate, up, gb, ub, out, "silu")
    want, bound = oracle.gated(x, gate, up, gb, ub, "silu")
    check(out, want, oracle.rounded(bound, want, kind))
