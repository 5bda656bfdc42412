"""Arguments that the decoder operators refuse before anything is launched (no GPU: the addresses are never read)."""
import ctypes

import pytest

HERE = ctypes.create_string_buffer(4096)
NULL, RANK, SHAPE, DTYPE, ATTR, LARGE, SCRATCH, UNSUPPORTED = -1, -2, -3, -4, -5, -6, -7, -8


@pytest.fixture
def cabi():
    import torch  # noqa: F401  (before fluidml_amd: the process then has one HIP runtime)
    from fluidml_amd import cabi

    return cabi


def tensor(cabi, *shape, dtype=None, strides=None):
    base = (ctypes.addressof(HERE) + 255) // 256 * 256
    return cabi.make_tensor(base, cabi.FL_BFLOAT16 if dtype is None else dtype, shape, strides)


def p(t):
    return None if t is None else ctypes.byref(t)


def test_rotary_refusals(cabi):
    def rc(x=None, out=None, positions=None, **plan):
        x = tensor(cabi, 2, 3, 5, 64) if x is None else x
        out = tensor(cabi, 2, 3, 5, 64) if out is None else out
        positions = tensor(cabi, 2, 5, dtype=cabi.FL_INT32) if positions is None else positions
        values = dict(interleaved=0, scaling=cabi.FL_ROTARY_WAVELENGTH, dims=32, base=1e4, factor=4.0, original_length=100.0, low=1.0, high=4.0, amplitude=1.0)
        values.update(plan)
        return cabi.lib.fluidml_hip_rotary_positions(p(x), p(positions), p(out), p(cabi.FlRotaryPlan(**values)), None)

    nan, inf = float("nan"), float("inf")
    for plan in (dict(dims=31), dict(dims=0), dict(dims=-2), dict(dims=66), dict(interleaved=2), dict(scaling=5), dict(scaling=-1), dict(base=1.0), dict(base=nan),
                 dict(base=inf), dict(factor=0.5), dict(factor=nan), dict(original_length=0.0), dict(low=0.0), dict(low=4.0), dict(high=inf), dict(amplitude=nan)):
        assert rc(**plan) == ATTR, plan
    assert rc(x=tensor(cabi, 2, 3, 5, 2048), out=tensor(cabi, 2, 3, 5, 2048), dims=1026) == UNSUPPORTED
    assert rc(x=tensor(cabi, 3, 5, 64)) == RANK
    assert rc(out=tensor(cabi, 2, 3, 5, 32)) == SHAPE
    assert rc(out=tensor(cabi, 2, 3, 5, 64, strides=(0, 320, 64, 1))) == SHAPE  # results in one place
    assert rc(out=tensor(cabi, 2, 3, 5, 64, strides=(960, 320, 64, -1))) == SHAPE
    assert rc(out=tensor(cabi, 2, 3, 5, 64, dtype=cabi.FL_FLOAT32)) == DTYPE
    assert rc(x=tensor(cabi, 2, 3, 5, 64, dtype=cabi.FL_INT32), out=tensor(cabi, 2, 3, 5, 64, dtype=cabi.FL_INT32)) == DTYPE
    assert rc(positions=tensor(cabi, 2, 5, dtype=cabi.FL_FLOAT32)) == DTYPE
    assert rc(positions=tensor(cabi, 5, 2, dtype=cabi.FL_INT32)) == SHAPE
    assert rc(positions=tensor(cabi, 3, 5, dtype=cabi.FL_INT64)) == SHAPE
    assert rc(positions=tensor(cabi, 1, 2, 5, dtype=cabi.FL_INT64)) == RANK
    x, i, plan = tensor(cabi, 1, 1, 1, 8), tensor(cabi, 1, dtype=cabi.FL_INT32), cabi.FlRotaryPlan(0, 0, 8, 1e4, 1, 1, 1, 4, 1)
    lib = cabi.lib
    assert lib.fluidml_hip_rotary_positions(None, p(i), p(x), p(plan), None) == NULL
    assert lib.fluidml_hip_rotary_positions(p(x), None, p(x), p(plan), None) == NULL
    assert lib.fluidml_hip_rotary_positions(p(x), p(i), p(x), None, None) == NULL
    for other in ((2, 1, 1, 8), (1, 1, 2, 8), (1, 1, 1, 16)):
        o = tensor(cabi, *other)
        assert lib.fluidml_hip_rotary_positions_pair(p(x), p(x), p(o), p(o), p(i), p(plan), None) == SHAPE
    assert lib.fluidml_hip_rotary_positions(p(tensor(cabi, 1, 1, 1, 1 << 29)), p(i), p(x), p(plan), None) == LARGE


def test_attention_refusals(cabi):
    def rc(q=(2, 4, 5, 64), k=(2, 2, 9, 64), v=None, out=None, dtype=None, scratch=1 << 20, scratch_at=None, **scores):
        q, k = (tensor(cabi, *t, dtype=dtype) if isinstance(t, tuple) else t for t in (q, k))
        v, out = k if v is None else v, q if out is None else out
        values = dict(scale=1.0, cap=0.0, causal=1, window=0)
        values.update({a: ctypes.pointer(b) if isinstance(b, cabi.FlTensor) else b for a, b in scores.items()})
        s = cabi.FlAttentionScores(**values)
        at = (ctypes.addressof(HERE) + 255) // 256 * 256 if scratch_at is None else scratch_at
        return cabi.lib.fluidml_hip_attention_positions(p(q), p(k), p(v), p(out), p(s), at, scratch, None)

    def ints(*shape):
        return tensor(cabi, *shape, dtype=cabi.FL_INT32)

    nan, inf = float("nan"), float("inf")
    for bad in (dict(scale=nan), dict(scale=inf), dict(scale=1e300), dict(cap=-1.0), dict(cap=nan), dict(cap=inf), dict(causal=2), dict(window=-1)):
        assert rc(**bad) == ATTR, bad
    assert rc(q=(2, 3, 5, 64)) == SHAPE          # 3 heads on 2
    assert rc(q=(2, 1, 5, 64)) == SHAPE
    assert rc(k=(3, 2, 9, 64)) == SHAPE
    assert rc(k=(2, 2, 9, 32)) == SHAPE
    assert rc(k=(2, 2, 0, 64)) == SHAPE
    assert rc(q=(4, 5, 64)) == RANK
    assert rc(v=tensor(cabi, 2, 2, 8, 64)) == SHAPE
    assert rc(out=tensor(cabi, 2, 4, 6, 64)) == SHAPE
    assert rc(out=tensor(cabi, 2, 4, 5, 64, strides=(1280, 0, 64, 1))) == SHAPE
    assert rc(q=(2, 4, 5, 257), k=(2, 2, 9, 257)) == UNSUPPORTED
    assert rc(dtype=cabi.FL_FLOAT64) == DTYPE
    assert rc(v=tensor(cabi, 2, 2, 9, 64, dtype=cabi.FL_FLOAT16)) == DTYPE
    assert rc(slopes=tensor(cabi, 2, dtype=cabi.FL_FLOAT32)) == SHAPE
    assert rc(slopes=tensor(cabi, 4)) == DTYPE
    assert rc(slopes=tensor(cabi, 1, 4, dtype=cabi.FL_FLOAT32)) == RANK
    for name in ("prefix_lengths", "query_starts", "query_lengths", "key_lengths"):
        assert rc(**{name: ints(3)}) == SHAPE and rc(**{name: ints(2, 1)}) == RANK
        assert rc(**{name: tensor(cabi, 2, dtype=cabi.FL_INT64)}) == DTYPE
    assert rc(query_documents=ints(2, 5)) == NULL and rc(key_documents=ints(2, 9)) == NULL
    assert rc(query_documents=ints(2, 5), key_documents=ints(2, 5)) == SHAPE
    assert rc(query_documents=ints(2, 9), key_documents=ints(2, 9)) == SHAPE
    assert rc(query_documents=ints(2, 5), key_documents=tensor(cabi, 2, 9, dtype=cabi.FL_INT64)) == DTYPE
    size, s = ctypes.c_size_t(), cabi.FlAttentionScores(1.0)
    q, k = tensor(cabi, 2, 4, 5, 64), tensor(cabi, 2, 2, 9, 64)
    call = cabi.lib.fluidml_hip_attention_positions_scratch
    assert call(p(q), p(k), p(s), None) == NULL and call(p(q), p(k), None, p(size)) == NULL and call(None, p(k), p(s), p(size)) == NULL
    assert call(p(q), p(q), p(s), p(size)) == 0


def test_gated_refusals(cabi):
    f32, bf = cabi.FL_FLOAT32, cabi.FL_BFLOAT16

    def rc(x=(3, 8), gate=(8, 16), up=(8, 16), down=(16, 4), out=(3, 4), products=(3, 16), gb=None, ub=None, db=None, addend=None, activation=0, dtype=bf):
        t = [tensor(cabi, *s, dtype=dtype) if isinstance(s, tuple) else s for s in (x, gate, up, gb, ub, down, db, addend, products, out)]
        return cabi.lib.fluidml_hip_gated_feed_forward(*map(p, t), activation, None)

    assert rc(gate=(7, 16)) == SHAPE and rc(up=(8, 15)) == SHAPE and rc(products=(3, 15)) == SHAPE and rc(products=(2, 16)) == SHAPE
    assert rc(down=(15, 4)) == SHAPE and rc(out=(3, 5)) == SHAPE and rc(addend=(3, 5)) == SHAPE and rc(db=(5,)) == SHAPE
    assert rc(gb=(15,)) == SHAPE and rc(ub=(17,)) == SHAPE and rc(ub=(16, 1)) == RANK
    assert rc(x=(1, 3, 8)) == RANK and rc(gate=(8,)) == RANK and rc(down=(16, 4, 1)) == RANK
    assert rc(dtype=cabi.FL_INT32) == DTYPE
    for name in ("gate", "up", "down", "products", "out"):
        shape = dict(gate=(8, 16), up=(8, 16), down=(16, 4), products=(3, 16), out=(3, 4))[name]
        assert rc(**{name: tensor(cabi, *shape, dtype=f32)}) == DTYPE, name
    assert rc(gb=tensor(cabi, 16, dtype=f32)) == DTYPE and rc(addend=tensor(cabi, 3, 4, dtype=f32)) == DTYPE
    assert rc(activation=6) == ATTR and rc(activation=-1) == ATTR
    assert rc(out=tensor(cabi, 3, 4, strides=(0, 1))) == SHAPE and rc(products=tensor(cabi, 3, 16, strides=(16, 0))) == SHAPE
    x, w, o = tensor(cabi, 3, 8), tensor(cabi, 8, 16), tensor(cabi, 3, 16)
    for i in (0, 1, 2, 5):
        t = [p(x), p(w), p(w), None, None, p(o)]
        t[i] = None
        assert cabi.lib.fluidml_hip_gated_matmul(*t, 0, None) == NULL
    assert rc(x=(0, 8)) == SHAPE


def test_extents_beyond_a_grid(cabi):
    """What no grid counts is refused before anything is launched, and no size is computed that 64 bits do not hold.  (Views of overlapping
    places: nothing is read.)"""
    lib, size = cabi.lib, ctypes.c_size_t()
    scores = cabi.FlAttentionScores(1.0)
    # (the fourth: tiles of one row each; with one key head its 2^24 rows would be 2^20 tiles of sixteen, which a grid counts)
    for B, H, KV, S, D in ((1, 1 << 28, 1, 1 << 28, 254), (1, 1 << 28, 1 << 28, 1 << 28, 254), (1 << 16, 1 << 12, 1, 1 << 28, 2), (1, 1 << 24, 1 << 24, 1, 8),
                           (65536, 1, 1, 1, 8), (1, 1, 1, 1 << 28, 8)):
        q, k = tensor(cabi, B, H, S, D, strides=(1, 1, 1, 1)), tensor(cabi, B, KV, 9, D, strides=(1, 1, 1, 1))
        assert lib.fluidml_hip_attention_positions_scratch(p(q), p(k), p(scores), p(size)) == LARGE
        assert lib.fluidml_hip_attention_positions(p(q), p(k), p(k), p(q), p(scores), None, 0, None) == LARGE
    x, w, o = tensor(cabi, 1, 8), tensor(cabi, 8, 1 << 27), tensor(cabi, 1, 1 << 27)
    assert lib.fluidml_hip_gated_matmul(p(x), p(w), p(w), None, None, p(o), 0, None) == LARGE
    x, w, o = tensor(cabi, 1 << 28, 8), tensor(cabi, 8, 512), tensor(cabi, 1 << 28, 512)
    assert lib.fluidml_hip_gated_matmul(p(x), p(w), p(w), None, None, p(o), 0, None) == LARGE
    x, w, down, small, o = tensor(cabi, 1 << 28, 8), tensor(cabi, 8, 16), tensor(cabi, 16, 512), tensor(cabi, 1 << 28, 16), tensor(cabi, 1 << 28, 512)
    assert lib.fluidml_hip_gated_feed_forward(p(x), p(w), p(w), None, None, p(down), None, None, p(small), p(o), 0, None) == LARGE
    plan = cabi.FlRotaryPlan(0, 0, 8, 1e4, 1, 1, 1, 4, 1)
    x, i = tensor(cabi, 1 << 12, 4096, 1 << 13, 8), tensor(cabi, 1 << 13, dtype=cabi.FL_INT32)
    assert lib.fluidml_hip_rotary_positions(p(x), p(i), p(x), p(plan), None) == LARGE


def test_factors_beyond_32_bits(cabi):
    q, k = tensor(cabi, 2, 4, 5, 64), tensor(cabi, 2, 2, 9, 64)
    for scale, cap in ((3e38, 0.0), (-3e38, 0.0), (1.0, 3e38), (1.0, 1e300), (1e30, 1e-30)):
        scores = cabi.FlAttentionScores(scale, cap)
        assert cabi.lib.fluidml_hip_attention_positions(p(q), p(k), p(k), p(q), p(scores), None, 0, None) == ATTR, (scale, cap)
    x, i, plan = tensor(cabi, 1, 1, 1, 8), tensor(cabi, 1, dtype=cabi.FL_INT32), cabi.FlRotaryPlan(0, 0, 8, 1e4, 1, 1, 1, 4, 1e39)
    assert cabi.lib.fluidml_hip_rotary_positions(p(x), p(i), p(x), p(plan), None) == ATTR


def test_view_refusals(cabi):
    """Host memory has no view: a kernel that got its address would fault."""
    import torch

    for t in (torch.zeros(2, 3), torch.zeros(2, dtype=torch.complex64), torch.zeros(2, device="meta")):
        with pytest.raises(ValueError):
            cabi.view(t)


@pytest.mark.gpu
def test_views(cabi, device):
    import torch

    for dtype, code in ((torch.bfloat16, cabi.FL_BFLOAT16), (torch.float16, cabi.FL_FLOAT16), (torch.float32, cabi.FL_FLOAT32), (torch.int64, cabi.FL_INT64)):
        t = torch.zeros(5, 7, 3, dtype=dtype, device=device)[1:, ::2].transpose(0, 2)
        v = cabi.view(t)
        assert (v.base, v.dtype, v.rank) == (t.data_ptr(), code, 3)
        assert tuple(v.shape[:3]) == tuple(t.shape) and tuple(v.strides[:3]) == t.stride()
    for t in (torch.zeros(2, dtype=torch.complex64, device=device), torch.zeros([1] * (cabi.FL_MAX_RANK + 1), device=device)):
        with pytest.raises(ValueError):
            cabi.view(t)
