"""Writes into the paged cache, page copies and attention over the pages, against plain NumPy loops in float64.

Tolerances of attention.  A score is a sum of D products of values that the type holds exactly; in float32 it is off by at
most (D + 2) 2^-24 s with s = scale sum |q||k|, plus 2^-24 |score| for the change of base.  A weight exp(score - max) is then
off by that much relative (twice: score and maximum), plus 2^-22 for exp2 and the running rescaling, and in 16-bit types half a
step for the rounding of the weights that the tensor cores multiply.  The output is a weighted mean: its error is at most
(weight error) * 2 * sum_j p_j |v_j| + the summation's (n + 2) 2^-24 sum_j p_j |v_j|, and half a step of the output."""
import numpy as np
import pytest

import orthon_b200 as ob
from orthon_b200 import _C

HALF_STEP = {"float64": 2.0 ** -53, "float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
ONE = {"float64": 2.0 ** -53, "float32": 2.0 ** -24, "float16": 2.0 ** -24, "bfloat16": 2.0 ** -24}
TINY = {"float64": 0.0, "float32": 0.0, "float16": 2.0 ** -24, "bfloat16": 0.0}
DEVICES = [pytest.param("cpu", "float32"), pytest.param("cpu", "float64")] + [
    pytest.param("cuda:0", t, marks=pytest.mark.gpu) for t in ("float32", "float16", "bfloat16")]
PLACES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


def give(a, dtype, device):
    t = _C.from_numpy(np.ascontiguousarray(a), dtype)
    return t if device == "cpu" else t.to(device)


def seen(t):
    t = t.to("cpu")
    return t.numpy() if t.dtype == "float64" else t.cast("float32").numpy().astype(np.float64)


def index_errors():
    _C.cuda_synchronize()
    return _C._cuda_index_errors()


def whole(a, device):
    return give(np.asarray(a, dtype=np.int32), "int32", device)


def make_table(rng, lengths, page, spare=2):
    need = [-(-n // page) for n in lengths]
    order = rng.permutation(sum(need) + spare)
    table = np.zeros((len(lengths), max(need + [1])), dtype=np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(need) + spare


def attend(q, k_pages, v_pages, table, lengths, scale):
    """(output, tolerance without the output's rounding per unit of ONE, weights' rounding) in float64."""
    B, H, D = q.shape
    group, P = H // k_pages.shape[1], k_pages.shape[2]
    out, size = np.zeros((B, H, D)), np.zeros((B, H, D))
    spread = np.zeros((B, H))
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        pages = table[b, :-(-n // P)]
        for h in range(H):
            k = k_pages[pages, h // group].reshape(-1, D)[:n]
            v = v_pages[pages, h // group].reshape(-1, D)[:n]
            s = k @ q[b, h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[b, h], size[b, h] = p @ v, p @ abs(v)
            spread[b, h] = (abs(k) @ abs(q[b, h])).max() * abs(scale)
    return out, size, spread


def check_attention(got, q, kp, vp, table, lengths, scale, dtype):
    want, size, spread = attend(q, kp, vp, table, lengths, scale)
    n = max(list(lengths) + [1])
    one = ONE[dtype]
    weight = 2 * (q.shape[2] + 4) * one * spread[..., None] + 8 * one + (HALF_STEP[dtype] if dtype in ("float16", "bfloat16") else 0.0)
    tol = 2 * weight * size + (n + 2) * one * size + abs(want) * HALF_STEP[dtype] * 1.001 + TINY[dtype]
    got = seen(got)
    bad = ~(abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), float(abs(got - want).max()), float(tol.min()))


CASES = [  # lengths, query heads, cached heads, head size, page size
    ([1], 1, 1, 64, 16), ([0], 2, 1, 64, 16), ([5, 0, 33, 1], 4, 4, 128, 16), ([333], 16, 16, 128, 16), ([64, 65, 63, 128], 8, 2, 64, 64),
    ([100, 7], 8, 1, 128, 8), ([17, 31, 2], 6, 3, 80, 16), ([50, 1, 200], 5, 1, 96, 32), ([9, 70], 12, 4, 20, 4), ([40, 13], 3, 3, 33, 5),
    ([260, 3], 20, 1, 128, 32), ([77], 40, 2, 64, 16), ([1000, 1, 0, 513], 2, 2, 256, 64), ([2500], 4, 1, 64, 1), ([15] * 70, 2, 2, 64, 16),
    ([4097, 31], 4, 2, 128, 128),
]


@pytest.mark.parametrize("device,dtype", DEVICES)
@pytest.mark.parametrize("lengths,H,K,D,P", CASES)
def test_attention_matches_the_definition(device, dtype, lengths, H, K, D, P):
    rng = np.random.default_rng(len(lengths) + H + D)
    table, pages = make_table(rng, lengths, P)
    q = give(rng.standard_normal((len(lengths), H, D)) * 2, dtype, device)
    raw = rng.standard_normal((2, pages, K, P, D))
    kp, vp = (give(x, dtype, device) for x in raw)
    got = ob.paged_attention(q, kp, vp, whole(table, device), whole(lengths, device))
    assert got.shape == q.shape and got.dtype == dtype and got.is_contiguous
    check_attention(got, seen(q), seen(kp), seen(vp), table, lengths, D ** -0.5, dtype)


@pytest.mark.parametrize("device,dtype", DEVICES)
@pytest.mark.parametrize("room", [0, 5000])
@pytest.mark.parametrize("lengths,H,K,D,P", CASES[:5] + [
    ([100, 7, 24, 0, 49], 8, 1, 128, 8), ([30, 70, 1, 25], 4, 2, 64, 24), ([90, 8], 20, 1, 80, 8), ([60, 0, 16], 10, 1, 256, 16), ([31] * 3, 40, 1, 96, 40),
    ([77, 3], 40, 2, 64, 16), ([50, 1, 200], 5, 1, 96, 32), ([9, 70], 12, 4, 20, 4), ([40, 13], 6, 1, 33, 5), ([1000, 1, 0, 513], 2, 2, 256, 64),
    ([700, 0, 3] * 12, 4, 2, 128, 16), ([17, 0, 40, 1, 5, 16, 33] * 300, 2, 1, 64, 16)])
def test_tables_with_room_for_more(device, dtype, room, lengths, H, K, D, P):
    """The result does not depend on the table's width, by which the kernel chooses how it divides the work."""
    rng = np.random.default_rng(len(lengths) + H + D + 1)
    table, pages = make_table(rng, lengths, P)
    table = np.pad(table, ((0, 0), (0, max(0, -(-room // P) - table.shape[1]))), constant_values=pages - 1)
    q = give(rng.standard_normal((len(lengths), H, D)) * 2, dtype, device)
    kp, vp = (give(x, dtype, device) for x in rng.standard_normal((2, pages, K, P, D)))
    got = ob.paged_attention(q, kp, vp, whole(table, device), whole(lengths, device))
    check_attention(got, seen(q), seen(kp), seen(vp), table, lengths, D ** -0.5, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("spare", [16, 24, 17])
def test_pages_beyond_32_bits(spare):
    """Pages of more than 2^31 values: zeros but for the last three tokens."""
    N, D, dev = 2 ** 24 + spare, 128, "cuda:0"
    rng = np.random.default_rng(spare)
    kp, vp = (_C._zeros_on([2, 1, N, D], "bfloat16", dev) for _ in range(2))
    k, v, q = (give(rng.standard_normal(s), "bfloat16", dev) for s in ((1, 3, 1, D), (1, 3, 1, D), (1, 2, D)))
    table, n = whole([[1]], dev), whole([N], dev)
    ob.paged_append_(kp, vp, k, v, table, whole([N - 3], dev))
    got = seen(ob.paged_attention(q, kp, vp, table, n, scale=1.0))
    s = np.einsum("hd,td->ht", seen(q)[0], seen(k)[0, :, 0])
    top = np.maximum(s.max(-1, keepdims=True), 0.0)
    p = np.exp(s - top)
    total = p.sum(-1, keepdims=True) + (N - 3) * np.exp(-top)
    want = p / total @ seen(v)[0, :, 0]
    # Half a step for a weight, half a step for the result, and the sums of N zeros' equal weights: at most N 2^-24 = 1 step
    # of float32 for each of the few thousand that a warp adds, which the half steps of bfloat16 leave room for.
    size = p / total @ abs(seen(v)[0, :, 0])
    assert (abs(got[0] - want) <= 2.0 ** -8 * abs(want) + (2.0 ** -8 + 2 ** -9) * size).all()
    ob.copy_pages_(kp, [1], [0])
    assert np.array_equal(seen(kp.slice(0, 0, 1).slice(2, N - 3, N))[0, 0], seen(k)[0, :, 0])


@pytest.mark.parametrize("device,dtype", DEVICES)
def test_head_sizes_one_after_another(device, dtype):
    """Small heads first: what a launch asks the device for does not depend on what was asked before."""
    rng = np.random.default_rng(6)
    for D in (24, 33, 60, 64, 65, 120, 128, 130, 256):
        for H in (1, 2, 3, 8):
            table, pages = make_table(rng, [20, 3], 16)
            q, kp, vp = (give(rng.standard_normal(s), dtype, device) for s in ((2, H, D), (pages, 1, 16, D), (pages, 1, 16, D)))
            got = ob.paged_attention(q, kp, vp, whole(table, device), whole([20, 3], device))
            check_attention(got, seen(q), seen(kp), seen(vp), table, [20, 3], D ** -0.5, dtype)


@pytest.mark.parametrize("device,dtype", DEVICES)
@pytest.mark.parametrize("D,P,H", [(64, 16, 4), (128, 32, 2), (40, 8, 2)])
def test_what_lies_behind_the_length_does_not_matter(device, dtype, D, P, H):
    """NaN and infinities in the unused rows of the last page, in pages that belong to nobody, and in wrong table entries
    behind the length."""
    rng = np.random.default_rng(3)
    lengths = [P + 3, 2 * P, 1, 0, 3 * P - 1]
    table, pages = make_table(rng, lengths, P)
    raw = rng.standard_normal((2, pages, 2, P, D))
    used = np.zeros((pages, P), dtype=bool)
    for b, n in enumerate(lengths):
        for j in range(n):
            used[table[b, j // P], j % P] = True
    raw[:, ~used.any(1)] = np.nan
    for i, (pg, slot) in enumerate(np.argwhere(~used)):
        raw[:, pg, :, slot] = [np.nan, np.inf, -np.inf][i % 3]
    for b, n in enumerate(lengths):
        table[b, -(-n // P):] = -7 if device != "cpu" else 0
    q = give(rng.standard_normal((5, H, D)), dtype, device)
    kp, vp = (give(x.astype(np.float32), dtype, device) for x in raw)
    got = ob.paged_attention(q, kp, vp, whole(table, device), whole(lengths, device), scale=0.3)
    kz, vz = (np.nan_to_num(seen(t), nan=0, posinf=0, neginf=0) for t in (kp, vp))
    check_attention(got, seen(q), kz, vz, np.maximum(table, 0), lengths, 0.3, dtype)
    assert not seen(got)[3].any()
    if device != "cpu":
        assert index_errors() == 0


@pytest.mark.parametrize("device,dtype", DEVICES)
def test_values_that_are_seen_do_matter(device, dtype):
    """A NaN among the seen keys or values reaches the output of its head only; a weight of zero stays zero."""
    rng = np.random.default_rng(4)
    table, pages = make_table(rng, [20, 20], 16)
    raw = rng.standard_normal((2, pages, 2, 16, 64)).astype(np.float32)
    raw[0, table[0, 1], 1, 2, 5] = np.nan
    raw[1, table[1, 0], 0, 3, 7] = np.inf
    q = give(np.abs(rng.standard_normal((2, 2, 64))) + 0.5, dtype, device)
    big = raw.copy()
    big[0, table[1, 1], 1, 1] = -60000.0  # the score is about -1e6: its weight vanishes
    kp, vp = (give(x, dtype, device) for x in big)
    got = seen(ob.paged_attention(q, kp, vp, whole(table, device), whole([20, 20], device)))
    assert np.isnan(got[0, 1]).all() and np.isfinite(got[0, 0]).all()
    assert np.isinf(got[1, 0, 7]) and np.isfinite(np.delete(got[1, 0], 7)).all() and np.isfinite(got[1, 1]).all()


@pytest.mark.parametrize("device,dtype", DEVICES)
def test_strided_queries_and_pages(device, dtype):
    """Queries inside a packed projection; keys and values page by page in one pool."""
    rng = np.random.default_rng(9)
    lengths, P, D = [37, 5, 64], 16, 64
    table, pages = make_table(rng, lengths, P)
    packed = give(rng.standard_normal((3, 6, D)), dtype, device)
    pool = give(rng.standard_normal((pages, 2, 2, P, D)), dtype, device).reshape([pages, 4, P, D])
    kp, vp = pool.slice(1, 0, 2), pool.slice(1, 2, 4)
    q = packed.slice(1, 1, 5)
    args = whole(table, device), whole(lengths, device)
    got = ob.paged_attention(q, kp, vp, *args)
    check_attention(got, seen(q.contiguous()), seen(kp.contiguous()), seen(vp.contiguous()), table, lengths, D ** -0.5, dtype)
    wide = packed.transpose(1, 2).contiguous().transpose(1, 2)  # the last dimension is strided: a copy is read
    assert np.array_equal(seen(ob.paged_attention(wide.slice(1, 1, 5), kp, vp, *args)), seen(got))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_results_do_not_depend_on_the_company(dtype):
    """The same calls give the same bits, twice in a row and from two threads."""
    import threading
    rng = np.random.default_rng(10)
    lengths = [3000, 1, 700, 64]
    table, pages = make_table(rng, lengths, 16)
    kp, vp = (give(rng.standard_normal((pages, 2, 16, 128)), dtype, "cuda:0") for _ in range(2))
    q = give(rng.standard_normal((4, 8, 128)), dtype, "cuda:0")
    args = q, kp, vp, whole(table, "cuda:0"), whole(lengths, "cuda:0")
    first = ob.paged_attention(*args).tolist()
    found = []
    work = [threading.Thread(target=lambda: found.append([ob.paged_attention(*args).tolist() for _ in range(5)])) for _ in range(2)]
    for w in work:
        w.start()
    for w in work:
        w.join()
    assert all(x == first for f in found for x in f)


@pytest.mark.gpu
def test_bad_pages_are_counted_and_not_followed():
    rng = np.random.default_rng(11)
    kp, vp = (give(rng.standard_normal((4, 1, 16, 64)), "bfloat16", "cuda:0") for _ in range(2))
    q = give(rng.standard_normal((1, 1, 64)), "bfloat16", "cuda:0")
    index_errors()
    ob.paged_attention(q, kp, vp, whole([[1, 4]], "cuda:0"), whole([32], "cuda:0"))
    assert index_errors() > 0
    ob.paged_attention(q, kp, vp, whole([[1, 2]], "cuda:0"), whole([33], "cuda:0"))  # longer than the table
    assert index_errors() > 0
    assert not seen(ob.paged_attention(q, kp, vp, whole([[1, 2]], "cuda:0"), whole([-1], "cuda:0"))).any()
    assert index_errors() > 0
    before = seen(kp)
    row = give(np.ones((1, 3, 1, 64)), "bfloat16", "cuda:0")
    ob.paged_append_(kp, vp, row, row, whole([[9, -1]], "cuda:0"), whole([15], "cuda:0"))
    assert index_errors() == 3 and np.array_equal(seen(kp), before)
    ob.paged_append_(kp, vp, row, row, whole([[0]], "cuda:0"), whole([14], "cuda:0"))  # the third token has no page
    assert index_errors() == 1
    before[0, :, 14:] = 1
    assert np.array_equal(seen(kp), before)
    ob.paged_append_(kp, vp, row, row, whole([[0]], "cuda:0"), whole([-2], "cuda:0"))
    assert index_errors() == 2
    before[0, :, 0] = 1
    assert np.array_equal(seen(kp), before)


@pytest.mark.parametrize("device,dtype", DEVICES)
@pytest.mark.parametrize("T,H,D,P,counts", [(1, 4, 64, 16, None), (7, 3, 80, 4, [7, 0, 3]), (40, 2, 128, 16, [40, 1, 17]), (5, 1, 33, 3, None), (6, 2, 12, 8, [9, -1, 6])])
def test_append_writes_exactly_its_rows(device, dtype, T, H, D, P, counts):
    rng = np.random.default_rng(T + H)
    starts = [0, 5, 13]
    table, pages = make_table(rng, [s + T for s in starts], P)
    packed = give(rng.standard_normal((3, T, 3 * H, D)), dtype, device)
    kp, vp = (give(rng.standard_normal((pages, H, P, D)), dtype, device) for _ in range(2))
    k, v = packed.slice(2, H, 2 * H), packed.slice(2, 2 * H, 3 * H)
    want = [seen(kp), seen(vp)]
    rows = seen(packed)
    for b in range(3):
        for t in range(T if counts is None else min(T, counts[b])):
            at = starts[b] + t
            for i in range(2):
                want[i][table[b, at // P], :, at % P] = rows[b, t, (i + 1) * H:(i + 2) * H]
    ob.paged_append_(kp, vp, k, v, whole(table, device), whole(starts, device), None if counts is None else whole(counts, device))
    assert np.array_equal(seen(kp), want[0]) and np.array_equal(seen(vp), want[1])
    if device != "cpu":
        assert index_errors() == 0


@pytest.mark.parametrize("device", PLACES)
@pytest.mark.parametrize("dtype", ["float32", "float16", "int64", "int8", "bool"])
@pytest.mark.parametrize("shape,dim", [((6, 5), 0), ((3, 6, 4, 16), 1), ((2, 3, 6, 33), 2), ((6, 1), 0), ((2, 6), 1), ((6, 70000), 0)])
def test_page_copies(device, dtype, shape, dim):
    rng = np.random.default_rng(1)
    a = rng.integers(0, 2 if dtype == "bool" else 100, shape)
    np_type = {"float16": "float16"}.get(dtype, dtype)
    t = _C.from_numpy(a.astype(np_type))
    t = t if device == "cpu" else t.to(device)
    out = ob.copy_pages_(t, [4, 1, 4], [0, 5, 2], dim=dim)
    want = a.astype(np_type)
    np.moveaxis(want, dim, 0)[[0, 5, 2]] = np.moveaxis(want, dim, 0)[[4, 1, 4]]
    assert np.array_equal(t.to("cpu").numpy(), want) and out.shape == t.shape
    ob.copy_pages_(t, [], [], dim=dim)
    assert np.array_equal(t.to("cpu").numpy(), want)


@pytest.mark.parametrize("device", PLACES)
def test_many_page_copies(device):
    a = np.random.default_rng(2).standard_normal((3, 2000, 8)).astype(np.float32)
    t = give(a, "float32", device)
    order = np.random.default_rng(3).permutation(2000)
    ob.copy_pages_(t, order[:1000].tolist(), order[1000:].tolist(), dim=1)
    a[:, order[1000:]] = a[:, order[:1000]]
    assert np.array_equal(t.to("cpu").numpy(), a)


@pytest.mark.parametrize("device", PLACES)
def test_refusals(device):
    z = lambda *s, d="float32": ob.zeros(list(s), d).to(device)  # noqa: E731
    i = lambda *s: ob.zeros(list(s), "int32").to(device)  # noqa: E731
    kp, vp, q, table, n = z(4, 2, 8, 16), z(4, 2, 8, 16), z(3, 4, 16), i(3, 2), i(3)
    rows = z(3, 5, 2, 16)
    for bad in ((z(3, 4, 8), kp, vp, table, n), (z(3, 3, 16), kp, vp, table, n), (z(3, 16), kp, vp, table, n), (q, z(4, 2, 8, 8), vp, table, n),
                (q, kp, vp, i(2, 2), n), (q, kp, vp, i(6), n), (q, kp, vp, table, i(2)), (q, kp, vp, table, z(3)), (q, kp, vp, z(3, 2), n),
                (q, z(4, 8, 2, 16).transpose(1, 2), vp, table, n), (q, z(2, 8, 16), z(2, 8, 16), table, n)):
        with pytest.raises((ValueError, RuntimeError)):
            ob.paged_attention(*bad)
    with pytest.raises(ValueError):
        ob.paged_attention(q, kp, vp, table, n, scale=float("nan"))
    with pytest.raises((ValueError, RuntimeError)):
        ob.paged_attention(q, kp, z(4, 2, 8, 16, d="float16") if device != "cpu" else z(4, 2, 8, 16, d="float64"), table, n)
    with pytest.raises(RuntimeError, match="no_grad"):
        ob.paged_attention(z(3, 4, 16).requires_grad_(), kp, vp, table, n)
    with pytest.raises(ob.UnsupportedOperation):
        ob.paged_attention(z(3, 4, 16, d="int32"), z(4, 2, 8, 16, d="int32"), z(4, 2, 8, 16, d="int32"), table, n)
    for bad in ((kp, vp, z(3, 5, 4, 16), rows, table, n), (kp, vp, rows, z(3, 4, 2, 16), table, n), (kp, vp, z(3, 2, 16), z(3, 2, 16), table, n),
                (kp, vp, rows, rows, table, i(2)), (kp, kp, rows, rows, table, n), (kp, vp, kp.slice(0, 0, 3).transpose(1, 2), rows, table, n)):
        with pytest.raises(ValueError):
            ob.paged_append_(*bad)
    with pytest.raises(ValueError):
        ob.paged_append_(kp, vp, rows, rows, table, n, i(2))
    with pytest.raises(RuntimeError, match="no_grad"):
        ob.paged_append_(kp, vp, z(3, 5, 2, 16).requires_grad_(), rows, table, n)
    for s, d, e in (([0], [0], ValueError), ([0, 1], [2, 2], ValueError), ([0, 1], [1, 2], ValueError), ([0], [1, 2], ValueError), ([4], [0], IndexError),
                    ([0], [-1], IndexError)):
        with pytest.raises(e):
            ob.copy_pages_(kp, s, d)
    with pytest.raises(ValueError):
        ob.copy_pages_(kp.transpose(0, 1), [0], [1])
    with pytest.raises(ValueError):
        ob.copy_pages_(kp, [0], [1], dim=4)
    if device == "cpu":
        for bad_table, start in (([[4, 0]] * 3, 0), ([[-1, 0]] * 3, 0), ([[0, 0]] * 3, 12), ([[0, 0]] * 3, -1)):
            with pytest.raises(IndexError):
                ob.paged_append_(kp, vp, rows, rows, whole(bad_table, device), whole([start] * 3, device))
        for bad_table, length in (([[4, 0]] * 3, 1), ([[0, 0]] * 3, 17), ([[0, 0]] * 3, -1)):
            with pytest.raises(IndexError):
                ob.paged_attention(q, kp, vp, whole(bad_table, device), whole([length] * 3, device))
    else:
        with pytest.raises(ValueError):
            ob.paged_attention(z(1, 1, 264), z(2, 1, 8, 264), z(2, 1, 8, 264), i(1, 1), i(1))
    assert ob.paged_attention(z(0, 4, 16), kp, vp, i(0, 2), i(0)).shape == (0, 4, 16)
    assert not ob.paged_attention(q, z(0, 2, 8, 16), z(0, 2, 8, 16), i(3, 0), n).cpu().numpy().any()
    ob.paged_append_(kp, vp, z(3, 0, 2, 16), z(3, 0, 2, 16), table, n)


@pytest.mark.parametrize("device,dtype", DEVICES)
@pytest.mark.parametrize("B,T,H,D,P,longest", [(1, 4099, 1, 64, 16, 4099), (3, 1000, 2, 33, 16, 700), (300, 13, 1, 8, 4, 13), (2, 2500, 20, 128, 32, 2500)])
def test_append_of_many_tokens(device, dtype, B, T, H, D, P, longest):
    """Tokens that lie beside each other in one block, with counts that end inside it and sequences of no new token."""
    rng = np.random.default_rng(B + T)
    starts, counts = rng.integers(0, 40, B), rng.integers(0, longest + 1, B)
    counts[0], counts[-1] = (T, 0) if B > 1 else (T, T)
    table, pages = make_table(rng, [int(s) + T for s in starts], P)
    k, v = (give(rng.standard_normal((B, T, H, D)), dtype, device) for _ in range(2))
    kp, vp = (give(rng.standard_normal((pages, H, P, D)), dtype, device) for _ in range(2))
    want = [seen(kp), seen(vp)]
    for rows, side in zip((seen(k), seen(v)), want):
        for b in range(B):
            at = starts[b] + np.arange(counts[b])
            side[table[b, at // P], :, at % P] = rows[b, :counts[b]]
    ob.paged_append_(kp, vp, k, v, whole(table, device), whole(starts, device), whole(counts, device))
    assert np.array_equal(seen(kp), want[0]) and np.array_equal(seen(vp), want[1])
    if device != "cpu":
        assert index_errors() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("room", [0, 5000])
@pytest.mark.parametrize("H,K,D", [(8, 4, 64), (24, 2, 128), (6, 6, 96)])
def test_weights_keep_more_bits_than_the_cache(dtype, room, H, K, D):
    """One value of each query and key is not zero, so a score is a product and no sum: off by 2^-24 of itself for each of three
    roundings (scale, base, difference to the maximum), and its weight by that, twice (own and sum), and 2^-21 for exp2 and the
    running rescaling.  Two terms of the type, the first rounded down (a step) and the second to the nearest (half a step of what
    is left), hold a weight to 2 half steps^2.  With the sums of n < 100 weights and
    products, (n + 2) 2^-24 each, that is far below half a step of the weights; what is left is half a step of the output."""
    rng, lengths, P = np.random.default_rng(H + D), [48, 31, 64, 96], 16
    table, pages = make_table(rng, lengths, P)
    table = np.pad(table, ((0, 0), (0, max(0, -(-room // P) - table.shape[1]))))
    raw = np.zeros((2, pages, K, P, D))
    raw[0, ..., 5] = rng.uniform(-2, 2, (pages, K, P))
    raw[1] = rng.standard_normal((pages, K, P, D))
    queries = np.zeros((len(lengths), H, D))
    queries[..., 5] = rng.uniform(0.5, 1.5, (len(lengths), H))
    q, kp, vp = (give(x, dtype, "cuda:0") for x in (queries, raw[0], raw[1]))
    got = seen(ob.paged_attention(q, kp, vp, whole(table, "cuda:0"), whole(lengths, "cuda:0"), scale=1.0))
    want, size, spread = attend(seen(q), seen(kp), seen(vp), table, lengths, 1.0)
    weight = 2 * 3 * 2.0 ** -24 * 2 * spread[..., None] + 2.0 ** -21 + 2 * HALF_STEP[dtype] ** 2 + 2 * (max(lengths) + 2) * 2.0 ** -24
    bad = ~(abs(got - want) <= weight * size + abs(want) * HALF_STEP[dtype] * 1.001 + TINY[dtype])
    assert not bad.any(), (int(bad.sum()), bad.size, float(abs(got - want).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("B,at,long,H,K,D", [(700, 0, 30000, 2, 1, 64), (600, 599, 40001, 3, 1, 40), (300, 150, 20000, 8, 2, 128), (1100, 7, 70000, 1, 1, 128)])
def test_one_sequence_far_longer_than_the_rest(dtype, B, at, long, H, K, D):
    """Its many shares are joined by more than one warp."""
    rng = np.random.default_rng(B)
    lengths = [int(n) for n in rng.integers(0, 40, B)]
    lengths[at], lengths[(at + 1) % B] = long, long // 3
    table, pages = make_table(rng, lengths, 16)
    q = give(rng.standard_normal((B, H, D)) * 2, dtype, "cuda:0")
    kp, vp = (give(rng.standard_normal((pages, K, 16, D), dtype=np.float32), dtype, "cuda:0") for _ in range(2))
    args = q, kp, vp, whole(table, "cuda:0"), whole(lengths, "cuda:0")
    got = ob.paged_attention(*args)
    check_attention(got, seen(q), seen(kp), seen(vp), table, lengths, D ** -0.5, dtype)
    assert np.array_equal(seen(got), seen(ob.paged_attention(*args)))


@pytest.mark.parametrize("device", PLACES)
@pytest.mark.parametrize("pairs", [439, 440, 441, 508, 509, 510, 1018, 1019])
def test_lists_of_copies_at_the_ends_of_a_launch(device, pairs):
    rng = np.random.default_rng(pairs)
    a = rng.integers(0, 1000, (2, 2 * pairs + 3, 5)).astype(np.int32)
    order = rng.permutation(2 * pairs + 3)
    t = give(a, "int32", device)
    ob.copy_pages_(t, order[:pairs].tolist(), order[pairs:2 * pairs].tolist(), dim=1)
    a[:, order[pairs:2 * pairs]] = a[:, order[:pairs]]
    assert np.array_equal(t.to("cpu").numpy(), a)
