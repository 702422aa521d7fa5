"""Rotary positions against a float64 implementation: layouts, partial heads, positions, scalings, strides, gradients, refusals.

Tolerances.  A turned value is m (a c - b s).  The turn count is rounded to float32 below half a turn (2^-26 of a turn,
2 pi 2^-26 rad), sine and cosine to 2 units in the last place (2^-23), m c and m s once more (2^-24): each factor is off by
less than 2 pi 2^-26 + 2^-23 + 2^-24 < 2^-21.6; the two products and the sum round by 2^-24 each.  Together below
2^-21 m (|a| + |b|), and half a step of the output's type on top.  In float64 the angle itself is what is off: frequency,
its division by 2 pi and its product with the position p are rounded here and there, less than 8 times 2^-53 |p| (f <= 1)."""
import math

import numpy as np
import pytest

import orthon_b200 as ob
from orthon_b200 import _C, nn

HALF_STEP = {"float64": 0.0, "float32": 0.0, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
SUBNORMAL = {"float64": 0.0, "float32": 0.0, "float16": 2.0 ** -25, "bfloat16": 0.0}


def make(rng, shape, dtype, device):
    t = _C.from_numpy(rng.standard_normal(shape).astype(np.float64 if dtype == "float64" else np.float32), dtype)
    return (t if device == "cpu" else t.to(device)), t.cast("float32").numpy().astype(np.float64) if dtype not in ("float64",) else t.numpy()


def frequencies(R, base=10000.0, scaling=None):
    i = np.arange(R // 2)
    kind, s = (scaling or {}).get("type"), (scaling or {}).get("factor")
    if kind == "ntk":
        base *= s ** (R / (R - 2))
    f = np.exp(-2 * i / R * np.log(base))
    if kind == "linear":
        return f / s, 1.0
    if kind == "yarn":
        L = scaling["original_length"]
        turns_over_length = lambda n: R * np.log(L / (n * 2 * np.pi)) / (2 * np.log(base))  # noqa: E731
        lo, hi = max(np.floor(turns_over_length(32.0)), 0), min(np.ceil(turns_over_length(1.0)), R - 1)
        r = np.clip((i - lo) / max(hi - lo, 1e-3), 0, 1)
        return f * (1 - r) + f / s * r, 0.1 * np.log(s) + 1
    return f, 1.0


def reference(x, positions, R, heads, inter=False, base=10000.0, scaling=None, sign=1.0):
    """(turned values, m (|a| + |b|) per value) in float64."""
    f, m = frequencies(R, base, scaling)
    a = (positions[..., None].astype(np.float64) * f)[:, :, None, :]
    z = np.exp(1j * sign * a) * m
    part = x[:, :, :heads, :R]
    u, v = (part[..., 0::2], part[..., 1::2]) if inter else (part[..., :R // 2], part[..., R // 2:])
    w = (u + 1j * v) * z
    size = m * (abs(u) + abs(v))
    y, e = x.copy(), np.zeros_like(x)
    if inter:
        y[:, :, :heads, 0:R:2], y[:, :, :heads, 1:R:2] = w.real, w.imag
        e[:, :, :heads, 0:R:2] = e[:, :, :heads, 1:R:2] = size
    else:
        y[:, :, :heads, :R // 2], y[:, :, :heads, R // 2:R] = w.real, w.imag
        e[:, :, :heads, :R // 2] = e[:, :, :heads, R // 2:R] = size
    return y, e


def close(got, want, size, dtype, far=1e6):
    got = got.to("cpu").cast("float32").numpy().astype(np.float64) if dtype != "float64" else got.numpy()
    tol = size * (2.0 ** -21 if dtype != "float64" else 2.0 ** -50 * far) + abs(want) * HALF_STEP[dtype] * (1 + 2.0 ** -10) + SUBNORMAL[dtype]
    bad = ~(abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), float(abs(got - want).max()))


DEVICES = [pytest.param("cpu", "float32"), pytest.param("cpu", "float64")] + [
    pytest.param("cuda:0", t, marks=pytest.mark.gpu) for t in ("float32", "float16", "bfloat16")]
SHAPES = [(1, 1, 1, 2, 2, 1), (2, 3, 4, 64, 64, 4), (1, 5, 3, 128, 64, 2), (3, 1, 48, 128, 128, 32), (2, 7, 5, 80, 40, 5), (1, 300, 2, 36, 20, 1),
          (2, 2, 3, 33, 32, 3), (1, 2, 2, 30, 6, 2), (1, 2, 2, 512, 512, 2)]


@pytest.mark.parametrize("device,dtype", DEVICES)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("B,T,H,D,R,heads", SHAPES)
def test_turn_matches_the_definition(device, dtype, inter, B, T, H, D, R, heads):
    rng = np.random.default_rng(B * T + D + inter)
    x, xs = make(rng, (B, T, H, D), dtype, device)
    pos = rng.integers(-5, 100000, (B, T))
    p = _C.from_numpy(pos.astype(np.int32 if inter else np.int64)).to(device)
    for back in (False, True):
        got = ob.rotary_embedding(x, p, rotary_dim=R, rotary_heads=heads, interleaved=inter, transposed=back)
        want, size = reference(xs, pos, R, heads, inter, sign=-1.0 if back else 1.0)
        assert got.shape == x.shape and got.dtype == dtype and got.is_contiguous
        close(got, want, size, dtype)
    kept = ob.rotary_embedding(x, p, rotary_dim=R, rotary_heads=heads, interleaved=inter)
    ob.rotary_embedding_(x, p, rotary_dim=R, rotary_heads=heads, interleaved=inter)  # the same values, in place
    assert x.tolist() == kept.tolist()


@pytest.mark.parametrize("device,dtype", DEVICES)
@pytest.mark.parametrize("scaling", [None, {"type": "linear", "factor": 4.0}, {"type": "ntk", "factor": 8.0},
                                     {"type": "yarn", "factor": 16.0, "original_length": 4096},
                                     {"type": "yarn", "factor": 2.0, "original_length": 8}])
def test_scalings_and_far_positions(device, dtype, scaling):
    rng = np.random.default_rng(5)
    x, xs = make(rng, (2, 9, 2, 64), dtype, device)
    pos = np.stack([np.arange(9) + 10 ** 6, np.arange(9) * 12345])
    got = ob.rotary_embedding(x, _C.from_numpy(pos.astype(np.int64)).to(device), scaling=scaling, base=500000.0)
    close(got, *reference(xs, pos, 64, 2, base=500000.0, scaling=scaling), dtype)


@pytest.mark.parametrize("device,dtype", DEVICES)
def test_strided_inputs_and_default_positions(device, dtype):
    rng = np.random.default_rng(6)
    packed, ps = make(rng, (2, 6, 9, 24), dtype, device)
    default = np.broadcast_to(np.arange(6), (2, 6))
    for view, arr in ((packed.slice(2, 3, 6), ps[:, :, 3:6]), (packed.slice(3, 1, 17), ps[..., 1:17]), (packed.slice(1, 2, 5), ps[:, 2:5]),
                      (packed.transpose(1, 2), ps.transpose(0, 2, 1, 3)), (packed.transpose(2, 3), ps.transpose(0, 1, 3, 2))):
        n, heads, D = arr.shape[1], arr.shape[2], arr.shape[3]
        R = D - D % 2
        for inter in (False, True):
            got = ob.rotary_embedding(view, rotary_dim=R, interleaved=inter)
            pos = np.broadcast_to(np.arange(n), (2, n))
            close(got, *reference(np.ascontiguousarray(arr), pos, R, heads, inter), dtype)
    row = _C.from_numpy(np.arange(6, dtype=np.int32)).to(device)
    close(ob.rotary_embedding(packed, row), *reference(ps, default, 24, 9), dtype)
    before = packed.to("cpu").cast("float32").numpy()
    ob.rotary_embedding_(packed.slice(2, 0, 3), row, rotary_dim=8)
    after = packed.to("cpu").cast("float32").numpy()
    want, size = reference(ps, default, 8, 3)
    assert np.array_equal(after[:, :, 3:], before[:, :, 3:]) and np.array_equal(after[:, :, :3, 8:], before[:, :, :3, 8:])
    close(packed, want, size, dtype)


@pytest.mark.parametrize("device,dtype", DEVICES)
@pytest.mark.parametrize("inter", [False, True])
def test_gradient_is_the_transposed_map(device, dtype, inter):
    rng = np.random.default_rng(7)
    x, xs = make(rng, (2, 5, 3, 16), dtype, device)
    w, ws = make(rng, (2, 5, 3, 16), dtype, device)
    yarn = {"type": "yarn", "factor": 4.0, "original_length": 32}
    x.requires_grad_()
    y = ob.rotary_embedding(x, rotary_dim=12, rotary_heads=2, interleaved=inter, scaling=yarn, base=100.0)
    (y * w).backward()
    pos = np.broadcast_to(np.arange(5), (2, 5))
    close(x.grad, *reference(ws, pos, 12, 2, inter, base=100.0, scaling=yarn, sign=-1.0), dtype)
    with pytest.raises(RuntimeError, match="no_grad"):
        ob.rotary_embedding_(y)


def test_gradient_matches_differences():
    rng = np.random.default_rng(8)
    xs, ws = rng.standard_normal((1, 4, 2, 10)), rng.standard_normal((1, 4, 2, 10))
    loss = lambda v: float((ob.rotary_embedding(_C.from_numpy(v), rotary_dim=6, interleaved=True).numpy() * ws).sum())  # noqa: E731
    x = _C.from_numpy(xs).requires_grad_()
    (ob.rotary_embedding(x, rotary_dim=6, interleaved=True) * _C.from_numpy(ws)).sum().backward()
    got = x.grad.numpy()
    for at in [(0, 0, 0, 0), (0, 1, 1, 3), (0, 3, 0, 5), (0, 2, 1, 9)]:
        step = np.zeros_like(xs)
        step[at] = 1e-5
        # The map is linear: the difference quotient has no truncation error, rounding gives 1e-16 * |loss| / 1e-5.
        assert abs((loss(xs + step) - loss(xs - step)) / 2e-5 - got[at]) < 1e-8


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
def test_refusals(device):
    x = ob.zeros([2, 3, 4, 8]).to(device)
    ids = lambda *s: ob.zeros(list(s), "int32").to(device)  # noqa: E731
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=10), dict(rotary_heads=0), dict(rotary_heads=5), dict(base=1.0), dict(base=math.inf),
                dict(scaling={"type": "other"}), dict(scaling={"type": "linear"}), dict(scaling={"type": "yarn", "factor": 2.0}),
                dict(scaling={"type": "linear", "factor": -1.0}), dict(scaling={"type": "linear", "factor": 2.0, "original_length": 4}),
                dict(rotary_dim=2, scaling={"type": "ntk", "factor": 2.0}),
                dict(positions=ids(4)), dict(positions=ids(3, 2)), dict(positions=ids(2, 3, 1)), dict(positions=ob.zeros([3]).to(device))):
        with pytest.raises(ValueError):
            ob.rotary_embedding(x, **bad)
    with pytest.raises(ValueError):
        ob.rotary_embedding(x.reshape([6, 4, 8]))
    with pytest.raises(ob.UnsupportedOperation):
        ob.rotary_embedding(ob.zeros([1, 1, 1, 8], "int32").to(device))
    with pytest.raises(ValueError):
        ob.rotary_embedding_(x.transpose(2, 3))
    assert ob.rotary_embedding(ob.zeros([0, 3, 4, 8]).to(device)).shape == (0, 3, 4, 8)
    assert ob.rotary_embedding(ob.zeros([2, 0, 4, 8]).to(device)).shape == (2, 0, 4, 8)


def test_module_holds_the_settings():
    x = _C.from_numpy(np.random.default_rng(1).standard_normal((1, 3, 2, 8)))
    m = nn.RotaryEmbedding(6, base=50.0, interleaved=True, scaling={"type": "linear", "factor": 2.0})
    want = ob.rotary_embedding(x, rotary_dim=6, base=50.0, interleaved=True, scaling={"type": "linear", "factor": 2.0}, rotary_heads=1)
    assert np.array_equal(m(x, rotary_heads=1).numpy(), want.numpy())
    assert list(m.parameters()) == [] and m.state_dict() == {}
    m.forward_(x, rotary_heads=1)
    assert np.array_equal(x.numpy(), want.numpy())
    with pytest.raises(ValueError):
        nn.RotaryEmbedding(5)


@pytest.mark.parametrize("device,dtype", DEVICES)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("B,T,H,D,R,heads", [(1, 8191, 1, 32, 32, 1), (4000, 1, 2, 16, 8, 1), (1500, 3, 1, 20, 12, 1), (3, 1999, 8, 64, 48, 8),
                                             (1, 20011, 5, 8, 8, 1), (700, 5, 1, 33, 2, 1), (2, 1300, 20, 128, 128, 3)])
def test_many_narrow_rows(device, dtype, inter, B, T, H, D, R, heads):
    """Rows that lie beside each other in one block: sequences that end inside it, the last block, more to pass on than to turn."""
    rng = np.random.default_rng(B + T)
    x, x64 = make(rng, (B, T, H, D), dtype, device)
    positions = rng.integers(0, 5000, (B, T))
    p = _C.from_numpy(positions)
    module = dict(rotary_dim=R, rotary_heads=heads, interleaved=inter)
    want, size = reference(x64, positions, R, heads, inter)
    close(ob.rotary_embedding(x, p if device == "cpu" else p.to(device), **module), want, size, dtype)
    want, size = reference(x64, np.broadcast_to(np.arange(T), (B, T)), R, heads, inter)
    close(ob.rotary_embedding_(x, **module), want, size, dtype)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("factor", [0.5, 1e-6, 1.0])
def test_yarn_does_not_shrink_below_a_factor_of_one(device, factor):
    """The enlargement is 0.1 ln(factor) + 1 from a factor of 1 on, and 1 below: turned pairs keep their length.  Their length is
    off by the rounding of two products, a sum, sine and cosine (2^-22 in all) and of the results (2^-24 each)."""
    rng = np.random.default_rng(7)
    x = rng.standard_normal((2, 5, 2, 8)).astype(np.float32)
    scaling = {"type": "yarn", "factor": factor, "original_length": 64}
    give = lambda s: ob.rotary_embedding(_C.from_numpy(x).to(device), scaling=s).to("cpu").numpy().astype(np.float64)  # noqa: E731
    y = give(scaling)
    size = lambda a: np.hypot(a[..., :4], a[..., 4:])  # noqa: E731
    want = size(x.astype(np.float64))
    assert (abs(size(y) - want) <= want * 2.0 ** -21).all()
    assert np.array_equal(give({**scaling, "attention_factor": 1.0}), y)
    assert not np.array_equal(give({**scaling, "attention_factor": 0.75}), y)


@pytest.mark.parametrize("scaling", [{"type": "linear", "factor": None}, {"type": "yarn", "factor": None, "original_length": 8},
                                     {"type": "yarn", "factor": 2.0, "original_length": None}])
def test_a_scaling_without_its_numbers_is_refused(scaling):
    with pytest.raises(ValueError, match="needs"):
        ob.rotary_embedding(ob.zeros([1, 2, 1, 4]), scaling=scaling)
