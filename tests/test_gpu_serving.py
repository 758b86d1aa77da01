"""The operators for many continuations of one prefix (attention_sinks,
attention_shared, logits_rules) against plain float64 implementations.

Attention tolerances, per output element, from the kernels' arithmetic (u =
2^-24 the half step of f32, e = the half step of the tensors' type):
  scores    a sum of D products in f32, any order: off by D u sum|q_d k_d|
            scale, and a few u of itself through scaling and the exponent's
            argument, so that a weight is off by about (D + 8) u S relative,
            S the row's largest sum|q k| scale over its keys;
  exp       a few u; numerator and denominator each carry both;
  sums      n keys in any order: n u, over weights and over products;
  weights   rounded to the tensors' type before the product with V: e;
  output    one rounding: e of the value (for f32, u).
All but the last are relative to sum_j w_j |v_j|.
"""
import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

F32, F16, BF16 = 0, 1, 2
KINDS = pytest.mark.parametrize("kind", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
U = 2.0 ** -24


def pack(x, kind):
    """Float values in the kind's storage (bf16 as uint16 bits), rounded to nearest even."""
    x = np.asarray(x, np.float32)
    if kind == F32:
        return x
    if kind == F16:
        return x.astype(np.float16)
    b = x.view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def unpack(x, kind):
    if kind != BF16:
        return np.asarray(x, np.float64)
    return (np.asarray(x, np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def attend64(q, k, v, visible):
    """One row: q [H, D], k and v [n, KV, D], visible [n]: (output, tolerance
    without the output's rounding), float64."""
    H, D = q.shape
    KV = k.shape[1]
    out, tol = np.zeros((H, D)), np.zeros((H, D))
    k, v = k[visible], v[visible]
    n = len(k)
    if n == 0:
        return out, tol
    for h in range(H):
        kh, vh = k[:, h * KV // H], v[:, h * KV // H]
        s = kh @ q[h] / np.sqrt(D)
        w = np.exp(s - s.max())
        w /= w.sum()
        out[h] = w @ vh
        big = (np.abs(kh) @ np.abs(q[h])).max() / np.sqrt(D)
        tol[h] = (w @ np.abs(vh)) * (2 * ((D + 8) * U * big + 8 * U) + 2 * (n + 8) * U)
    return out, tol


def near(got, want, tol, w_tol, kind):
    """|got - want| within the derived tolerance, values not finite equal."""
    e = HALF_STEP[kind]
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    lim = tol + (w_tol * e if kind != F32 else 0) + np.abs(want) * e * 1.01 + (2.0 ** -25 if kind == F16 else 1e-38)
    d = np.abs(got - want)
    bad = fine & ~(d <= lim)
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {np.max(d[bad] / lim[bad]):.3g} of the tolerance"


def check_rows(got, q, rows, kind):
    """rows: (k, v, visible) of each row of q [n, H, D]."""
    got = unpack(got, kind).reshape(q.shape)
    for i, (k, v, visible) in enumerate(rows):
        want, tol = attend64(q[i], k, v, visible)
        absw = attend64(q[i], k, np.abs(v), visible)[0]
        near(got[i], want, tol, absw, kind)


def sinks_visible(ctx, p, window, n_sink):
    j = np.arange(ctx)
    return (j <= p) & ((j < n_sink) | (j > p - window) if window else True)


HEADS = [(4, 4, 64), (32, 4, 64), (8, 2, 128), (10, 2, 128), (8, 4, 256), (3, 1, 256)]
SINKS = [(0, 1, 0, 0), (0, 1, 1, 0), (5, 1, 3, 2), (37, 1, 16, 4), (15, 1, 0, 0), (16, 1, 0, 0), (31, 2, 5, 1),
         (0, 33, 8, 3), (63, 17, 64, 4), (130, 70, 64, 4), (300, 5, 1, 0), (200, 129, 0, 0), (777, 1, 100, 1000),
         (777, 1, 1, 0), (1200, 9, 500, 3), (95, 3, 32, 33), (0, 200, 1, 1)]


@KINDS
@pytest.mark.parametrize("nh,nkv,hd", HEADS, ids=str)
def test_sinks(aotk, kind, nh, nkv, hd):
    for case, (pos0, m, window, n_sink) in enumerate(SINKS):
        rng = np.random.default_rng(1000 * kind + 10 * nh + case)
        ctx = pos0 + m + case % 3
        q = pack(rng.standard_normal((m, nh, hd)) * 1.5, kind)
        k, v = (pack(rng.standard_normal((2, ctx, nkv, hd)), kind) for _ in range(2))
        # what no row sees is not read
        seen = np.zeros(ctx, bool)
        for i in range(m):
            seen |= sinks_visible(ctx, pos0 + i, window, n_sink)
        bad = pack(np.array([np.nan, np.inf, -np.inf]), kind)
        for c in (k, v):
            c[0] = bad[0]
            c[1][~seen] = bad[np.arange((~seen).sum()) % 3][:, None, None]
        got = aotk.attention_sinks(q, k, v, nh, nkv, hd, ctx, 1, pos0, m, window, n_sink, kind)
        q64, k64, v64 = unpack(q, kind), unpack(k[1], kind), unpack(v[1], kind)
        check_rows(got, q64, [(k64, v64, sinks_visible(ctx, pos0 + i, window, n_sink)) for i in range(m)], kind)


@KINDS
@pytest.mark.parametrize("nh,nkv,hd", [(8, 4, 64), (8, 2, 128), (2, 2, 256), (2, 2, 128), (1, 1, 64)], ids=str)
def test_sinks_values_not_finite_reach_only_rows_that_see_them(aotk, kind, nh, nkv, hd):
    """Positions that some rows of a call see and others do not hold NaN and
    infinities in K or V; also a long window's far rows."""
    for case, (pos0, m, window, n_sink, marks) in enumerate([
            (3, 40, 6, 2, {10: "vnan", 20: "vinf", 30: "knan"}), (100, 70, 16, 0, {101: "vinf", 150: "vnan", 169: "knan"}),
            (0, 150, 0, 0, {70: "vnan", 149: "vinf"}), (40, 7, 5, 1, {41: "vinf", 44: "vnan", 46: "knan"}),
            (40, 9, 0, 0, {30: "vinf", 42: "vnan", 47: "kinf"}), (64, 64, 32, 5, {64: "vnan", 4: "vinf", 127: "kinf"})]):
        rng = np.random.default_rng(77 + case)
        ctx = pos0 + m
        q = pack(rng.standard_normal((m, nh, hd)), kind)
        k, v = rng.standard_normal((2, 1, ctx, nkv, hd))
        q = np.abs(q) if kind != BF16 else q & 0x7FFF  # +inf keys give +inf scores
        for j, what in marks.items():
            c = k if what[0] == "k" else v
            # one value of V, in one dimension: only that dimension of a row that sees it
            c[0, j, :, 5 if what[0] == "v" else slice(None)] = np.nan if what[1:] == "nan" else np.inf
        k, v = pack(k, kind), pack(v, kind)
        got = aotk.attention_sinks(q, k, v, nh, nkv, hd, ctx, 0, pos0, m, window, n_sink, kind)
        q64, k64, v64 = unpack(q, kind), unpack(k[0], kind), unpack(v[0], kind)
        got = unpack(got, kind).reshape(m, nh, hd)
        with np.errstate(invalid="ignore"):
            for i in range(m):
                vis = sinks_visible(ctx, pos0 + i, window, n_sink)
                want, tol = attend64(q64[i], k64, v64, vis)
                absw = attend64(q64[i], k64, np.abs(v64), vis)[0]
                fine = np.isfinite(want)
                assert np.array_equal(np.isfinite(got[i]), fine), f"case {case} row {i}"
                near(np.where(fine, got[i], 0), np.where(fine, want, 0), np.where(fine, tol, 0), np.where(fine, absw, 0), kind)


@KINDS
@pytest.mark.parametrize("nh,nkv,hd", [(4, 2, 64), (8, 2, 128), (2, 1, 256)], ids=str)
@pytest.mark.parametrize("m", [1, 5, 200])
def test_sinks_infinite_values_that_every_row_sees(aotk, kind, nh, nkv, hd, m):
    """In tiles that lie wholly before the rows: infinities stay infinities,
    two of both signs and a NaN become NaN, in their dimensions alone."""
    rng = np.random.default_rng(11)
    ctx = 300 + m
    q = pack(rng.standard_normal((m, nh, hd)), kind)
    k, v = rng.standard_normal((2, 1, ctx, nkv, hd))
    for j, d, x in [(10, 5, np.inf), (99, 6, -np.inf), (20, 7, np.inf), (70, 7, -np.inf), (140, 9, np.nan)]:
        v[0, j, :, d] = x
    k, v = pack(k, kind), pack(v, kind)
    got = aotk.attention_sinks(q, k, v, nh, nkv, hd, ctx, 0, 300, m, 0, 0, kind)
    k64, v64 = unpack(k[0], kind), unpack(v[0], kind)
    with np.errstate(invalid="ignore"):
        check_rows(got, unpack(q, kind), [(k64, v64, np.arange(ctx) <= 300 + i) for i in range(m)], kind)


@KINDS
def test_sinks_scores_far_apart(aotk, kind):
    """One key far above the others, many equal keys far below the largest
    (weights of 2^-15 whose sum still counts), scores of hundreds."""
    hd, n = 128, 4096
    q = np.zeros((1, 2, hd))
    q[:, :, 0] = np.sqrt(hd)
    k = np.zeros((1, n, 1, hd))
    v = np.ones((1, n, 1, hd))
    k[0, 7, 0, 0] = 15 * np.log(2)
    v[0, 7] = -1
    for offset in (0.0, 300.0, -300.0):
        kk = k.copy()
        kk[0, :, 0, 1] = offset
        qq = q.copy()
        qq[:, :, 1] = np.sqrt(hd)
        qp, kp, vp = pack(qq, kind), pack(kk, kind), pack(v, kind)
        got = aotk.attention_sinks(qp, kp, vp, 2, 1, hd, n, 0, n - 1, 1, 0, 0, kind)
        check_rows(got, unpack(qp, kind), [(unpack(kp[0], kind), unpack(vp[0], kind), np.ones(n, bool))], kind)


@KINDS
@pytest.mark.parametrize("m", [1, 40])
def test_sinks_many_small_weights_beside_a_large_one(aotk, kind, m):
    """65536 equal weights of 1.37 x 2^-18 of the largest, a quarter of the sum."""
    hd, n = 64, 65536
    c = np.sqrt(hd) / 8
    q, k, v = np.zeros((m, 1, hd)), np.zeros((1, n, 1, hd)), np.ones((1, n, 1, hd))
    q[:, :, :2] = 8, 1
    k[0, 7, 0, :2] = 1.5 * c, np.log(2 ** 18 / 1.37) * 8 - 12
    v[0, 7] = -1
    qp, kp, vp = pack(q, kind), pack(k, kind), pack(v, kind)
    got = aotk.attention_sinks(qp, kp, vp, 1, 1, hd, n, 0, n - m, m, 0, 0, kind)
    k64, v64 = unpack(kp[0], kind), unpack(vp[0], kind)
    check_rows(got, unpack(qp, kind), [(k64, v64, np.arange(n) <= n - m + i) for i in range(m)], kind)


@KINDS
def test_sinks_rows_whose_scores_are_all_minus_infinity(aotk, kind):
    """Like the formula: such a row is NaN (no weight to divide by)."""
    q = pack(np.ones((1, 2, 64)), kind)
    k, v = pack(np.full((1, 20, 1, 64), -np.inf), kind), pack(np.ones((1, 20, 1, 64)), kind)
    assert np.isnan(unpack(aotk.attention_sinks(q, k, v, 2, 1, 64, 20, 0, 19, 1, 4, 2, kind), kind)).all()


def test_sinks_long_context(aotk):
    """A cache whose bytes pass 32 bits of offset, far behind a window."""
    nkv, hd, ctx = 8, 128, 1_100_000  # 2.25 GB of bf16 each
    rng = np.random.default_rng(5)
    lib = aotk.abi.load()
    row = nkv * hd * 2
    kn, vn = pack(rng.standard_normal((2, 600, nkv, hd)), BF16)
    caches = []
    for x in (kn, vn):
        c = aotk.DeviceBuffer(ctx * row)
        aotk.abi.check(lib.aotk_memset(c.ptr, 0xFF, c.nbytes))  # NaN
        for at, part in ((0, x[:10]), (ctx - 590, x[10:])):
            aotk.abi.check(lib.aotk_h2d(c.ptr + at * row, np.ascontiguousarray(part).ctypes.data, part.nbytes))
        caches.append(c)
    q = pack(rng.standard_normal((3, 16, hd)), BF16)
    qd, out = aotk.DeviceBuffer.from_numpy(q), aotk.DeviceBuffer(q.nbytes)
    aotk.abi.check(lib.aotk_attention_sinks(out.ptr, qd.ptr, caches[0].ptr, caches[1].ptr, BF16, 16, nkv, hd, ctx, 0, ctx - 3,
                                            3, 500, 10))
    got = out.to_numpy(np.uint16)
    k64, v64, q64 = (unpack(x, BF16) for x in (kn, vn, q))
    rows = []
    for i in range(3):
        vis = np.zeros(600, bool)
        vis[:10] = True
        last = 600 - 3 + i
        vis[last - 499:last + 1] = True
        rows.append((k64, v64, vis))
    check_rows(got, q64, rows, BF16)


def shared_inputs(rng, kind, nh, nkv, hd, prefix_ctx, n_prefix, tail_ctx, tail_len, rows, layers=2, layer=1):
    """Inputs with everything that no row may see set to NaN or infinity."""
    total = sum(rows)
    q = pack(rng.standard_normal((total, nh, hd)) * 1.5, kind)
    kp, vp = (pack(rng.standard_normal((layers, prefix_ctx, nkv, hd)), kind) for _ in range(2))
    kt, vt = (pack(rng.standard_normal((layers, len(tail_len), tail_ctx, nkv, hd)), kind) for _ in range(2))
    bad = pack(np.array([np.nan, np.inf, -np.inf]), kind)
    for x in (kp, vp):
        x[layer, n_prefix:] = bad[0]
        x[:layer] = bad[1]
    for x in (kt, vt):
        x[:layer] = bad[2]
        for b, n in enumerate(tail_len):
            x[layer, b, n:] = bad[b % 3]
    return q, kp, vp, kt, vt


def shared_rows(kp, vp, kt, vt, n_prefix, tail_len, rows, kind, layer=1):
    kp, vp, kt, vt = (unpack(x[layer], kind) for x in (kp, vp, kt, vt))
    out = []
    for b, (n, r) in enumerate(zip(tail_len, rows)):
        k, v = np.concatenate([kp[:n_prefix], kt[b, :n]]), np.concatenate([vp[:n_prefix], vt[b, :n]])
        for i in range(r):
            out.append((k, v, np.arange(len(k)) < n_prefix + max(0, n - r + i + 1)))
    return out


SHARED = [  # n_prefix, tail_len, rows
    (1, [0], None), (0, [1], None), (0, [0, 3, 0], None), (7, [0, 1, 2], None), (16, [16, 17], None),
    (100, [5, 33, 64, 1, 0], None), (333, [20], None), (0, [0, 5], [2, 3]), (64, [9, 40, 0, 3], [4, 40, 0, 5]),
    (50, [12, 30, 70], [1, 20, 70]), (1000, [3, 1, 4, 1, 5, 9, 2, 6, 5, 3, 5, 8, 9, 7, 9, 3, 2], None),
    (0, [300, 2], [130, 1]), (513, [1] * 70, None),
]


@KINDS
@pytest.mark.parametrize("nh,nkv,hd", HEADS, ids=str)
def test_shared(aotk, kind, nh, nkv, hd):
    for case, (n_prefix, tail_len, rows) in enumerate(SHARED):
        rng = np.random.default_rng(5000 * kind + 7 * nh + case)
        prefix_ctx, tail_ctx = n_prefix + case % 2, max(tail_len) + case % 3
        nr = rows or [1] * len(tail_len)
        q, kp, vp, kt, vt = shared_inputs(rng, kind, nh, nkv, hd, prefix_ctx, n_prefix, tail_ctx, tail_len, nr)
        got = aotk.attention_shared(q, kp, vp, kt, vt, nh, nkv, hd, prefix_ctx, n_prefix, tail_ctx, 1, tail_len, rows, kind)
        check_rows(got, unpack(q, kind), shared_rows(kp, vp, kt, vt, n_prefix, tail_len, nr, kind), kind)


def test_shared_many_sequences_and_rows_left_alone(aotk):
    """More sequences than one launch's arguments hold, most without rows;
    what lies behind the last row stays."""
    nh, nkv, hd, n = 4, 2, 64, 300
    rng = np.random.default_rng(9)
    tail_len = [int(x) for x in rng.integers(0, 20, n)]
    rows = [int(x) if b % 3 else 0 for b, x in enumerate(rng.integers(0, 4, n))]
    q, kp, vp, kt, vt = shared_inputs(rng, F32, nh, nkv, hd, 40, 40, 20, tail_len, rows)
    total = sum(rows)
    t = [aotk.DeviceBuffer.from_numpy(x) for x in (q, kp, vp, kt, vt)]
    out = aotk.DeviceBuffer.from_numpy(np.full((total + 3, nh, hd), 7.0, np.float32))
    tl, nr = np.array(tail_len, np.uint32), np.array(rows, np.uint32)
    lib = aotk.abi.load()
    aotk.abi.check(lib.aotk_attention_shared(out.ptr, *[x.ptr for x in t], F32, nh, nkv, hd, 40, 40, 20, 1, n,
                                             tl.ctypes.data, nr.ctypes.data))
    got = out.to_numpy(np.float32).reshape(total + 3, nh, hd)
    assert (got[total:] == 7.0).all()
    check_rows(got[:total], q.astype(np.float64), shared_rows(kp, vp, kt, vt, 40, tail_len, rows, F32), F32)


SHAPES = [  # nh, nkv, hd, prefix, tail lengths, rows: every pairing of the kernels' row tiles, prefix / tails
    (2, 2, 64, 70, [9, 40, 3], None),  # 3 rows / 1
    (8, 1, 128, 90, [30, 50, 7], None),  # 24 / 8
    (20, 1, 128, 40, [5, 9], [1, 1]),  # 40 / 20 of 64
    (4, 1, 64, 130, [40, 33, 2, 9], [9, 2, 1, 3]),  # 60 / 36
    (8, 1, 256, 100, [33, 70, 5], None),  # 24 / 8, heads of 256
    (24, 1, 256, 33, [64, 5], None),  # 48 / 24, heads of 256
    (16, 2, 128, 300, [70, 1, 20] * 6, None),  # 144 / 8
    (24, 1, 128, 200, [70, 33, 1, 9, 20, 64], None),  # 144 / 24
    (4, 1, 128, 65, [50, 100, 3], [40, 90, 3]),  # 532 / 360
    (6, 3, 256, 97, [50, 130, 3], [40, 90, 1]),  # 262 / 180, heads of 256
    (128, 1, 64, 31, [2, 40], None),  # a group wider than a tile
]


@KINDS
@pytest.mark.parametrize("nh,nkv,hd,n_prefix,tail_len,rows", SHAPES, ids=str)
def test_shared_row_tiles(aotk, kind, nh, nkv, hd, n_prefix, tail_len, rows):
    rng = np.random.default_rng(nh + hd)
    nr = rows or [1] * len(tail_len)
    tail_ctx = max(tail_len)
    q, kp, vp, kt, vt = shared_inputs(rng, kind, nh, nkv, hd, n_prefix + 3, n_prefix, tail_ctx, tail_len, nr)
    got = aotk.attention_shared(q, kp, vp, kt, vt, nh, nkv, hd, n_prefix + 3, n_prefix, tail_ctx, 1, tail_len, rows, kind)
    check_rows(got, unpack(q, kind), shared_rows(kp, vp, kt, vt, n_prefix, tail_len, nr, kind), kind)


@KINDS
def test_shared_one_tail_far_longer_than_the_others(aotk, kind):
    """A sequence whose run of keys is cut while the others' are whole, with
    more blocks than fit the chip; one with many rows beside one with many keys."""
    rng = np.random.default_rng(21)
    nh, nkv, hd, n = 8, 2, 64, 300
    tail_len = [3] * 150 + [1200] + [2] * 149
    q, kp, vp = (pack(rng.standard_normal(s), kind) for s in ((n, nh, hd), (1, 5, nkv, hd), (1, 5, nkv, hd)))
    kt, vt = (np.zeros((1, n, 1200, nkv, hd), q.dtype) for _ in range(2))
    for c in (kt, vt):
        for b, m in enumerate(tail_len):
            c[0, b, :m] = pack(rng.standard_normal((m, nkv, hd)), kind)
    got = aotk.attention_shared(q, kp, vp, kt, vt, nh, nkv, hd, 5, 5, 1200, 0, tail_len, None, kind)
    keys = [np.concatenate([unpack(p[0], kind), unpack(t[0, b, :m], kind)]) for b, m in enumerate(tail_len) for p, t in ((kp, kt), (vp, vt))]
    check_rows(got, unpack(q, kind), [(keys[2 * b], keys[2 * b + 1], np.ones(5 + m, bool)) for b, m in enumerate(tail_len)], kind)
    kt, vt = (pack(rng.standard_normal((1, 3, 9000, nkv, hd)), kind) for _ in range(2))
    lens, rows = [2, 9000, 1], [300, 1, 0]
    q = pack(rng.standard_normal((301, nh, hd)), kind)
    got = aotk.attention_shared(q, kp, vp, kt, vt, nh, nkv, hd, 5, 5, 9000, 0, lens, rows, kind)
    check_rows(got, unpack(q, kind), shared_rows(kp, vp, kt, vt, 5, lens, rows, kind, 0), kind)


@KINDS
@pytest.mark.parametrize("rows", [[1100, 1100, 1000, 1200], [4300, 1, 0, 99]], ids=str)
def test_shared_many_rows_of_every_sequence(aotk, kind, rows):
    """More than a thousand tiles of rows; a sample of the rows is checked."""
    nh, nkv, hd, n_prefix, tail_len = 32, 4, 64, 70, [1200, 1100, 900, 1300]
    rng = np.random.default_rng(33)
    q, kp, vp, kt, vt = shared_inputs(rng, kind, nh, nkv, hd, 72, n_prefix, 1300, tail_len, rows)
    got = aotk.attention_shared(q, kp, vp, kt, vt, nh, nkv, hd, 72, n_prefix, 1300, 1, tail_len, rows, kind)
    ends = np.cumsum(rows)
    some = sorted({int(x) for x in [0, *(ends - 1), *ends[:-1], *rng.integers(0, ends[-1], 30)]})
    want = shared_rows(kp, vp, kt, vt, n_prefix, tail_len, rows, kind)
    check_rows(got.reshape(q.shape)[some], unpack(q, kind)[some], [want[i] for i in some], kind)


def test_shared_more_rows_than_one_join_takes(aotk):
    """Two parts for each of 66000 x 32 rows."""
    nh, nkv, hd, rows = 32, 4, 64, [33001, 32999]
    rng = np.random.default_rng(34)
    few = rng.standard_normal((250, nh, hd)).astype(np.float32)
    q = np.tile(few, (264, 1, 1))
    kp, vp = rng.standard_normal((2, 1, 3, nkv, hd)).astype(np.float32)
    kt, vt = rng.standard_normal((2, 1, 2, 5, nkv, hd)).astype(np.float32)
    got = aotk.attention_shared(q, kp, vp, kt, vt, nh, nkv, hd, 3, 3, 5, 0, [5, 2], rows, F32).reshape(q.shape)
    some = [0, 249, 32995, 32998, 33000, 33001, 65533, 65534, 65535, 65536, 65537, 65998, 65999]
    want = shared_rows(kp, vp, kt, vt, 3, [5, 2], rows, F32, 0)
    check_rows(got[some], q[some].astype(np.float64), [want[i] for i in some], F32)
    # rows that see the prefix alone: the same for the same query
    assert (got[250:32500].reshape(-1, 250, nh, hd) == got[:250]).all()


def test_shared_without_rows_is_no_work(aotk):
    z = np.zeros((1, 1, 1, 64), np.float32)
    got = aotk.attention_shared(np.zeros((0, 1, 64), np.float32), z, z, np.zeros((1, 2, 1, 1, 64), np.float32),
                                np.zeros((1, 2, 1, 1, 64), np.float32), 1, 1, 64, 1, 1, 1, 0, [1, 0], [0, 0])
    assert got.size == 0


@KINDS
def test_shared_equals_one_sequence_of_prefix_and_tail(aotk, kind):
    """The same keys as one range and as two."""
    nh, nkv, hd = 16, 4, 128
    rng = np.random.default_rng(3)
    for n_prefix, n, r in ((130, 9, 9), (31, 200, 1), (512, 64, 33)):
        ctx = n_prefix + n
        q = pack(rng.standard_normal((r, nh, hd)), kind)
        k, v = (pack(rng.standard_normal((ctx, nkv, hd)), kind) for _ in range(2))
        one = aotk.attention_sinks(q, k, v, nh, nkv, hd, ctx, 0, ctx - r, r, 0, 0, kind)
        two = aotk.attention_shared(q, k[:n_prefix], v[:n_prefix], k[n_prefix:], v[n_prefix:], nh, nkv, hd, n_prefix, n_prefix,
                                    n, 0, [n], [r], kind)
        q64, k64, v64 = (unpack(x, kind) for x in (q, k, v))
        for i in range(r):
            vis = np.arange(ctx) <= ctx - r + i
            _, tol = attend64(q64[i], k64, v64, vis)
            absw = attend64(q64[i], k64, np.abs(v64), vis)[0]
            a, b = (unpack(x, kind).reshape(r, nh, hd)[i] for x in (one, two))
            e = HALF_STEP[kind]
            assert (np.abs(a - b) <= 2 * (tol + (absw * e if kind else 0) + absw * e)).all()


# ------------------------------------------------------------------- rules
def rules64(x, rules, masks, kind):
    """(values before rounding, float64; exact where no penalty applies)."""
    y = unpack(x, kind)
    for i, r in enumerate(rules):
        seen = {}
        for t in r.get("history", ()):
            seen[int(t)] = seen.get(int(t), 0) + 1
        rep = float(np.float32(r.get("repetition", 1.0)))
        pres, freq = float(np.float32(r.get("presence", 0.0))), float(np.float32(r.get("frequency", 0.0)))
        for t, c in seen.items():
            if t < y.shape[1]:
                v = y[i, t]
                y[i, t] = (v / rep if v > 0 else v * rep) - (pres + freq * c)
        bias = r.get("bias", ())
        for t, b in dict(bias).items():
            if t < y.shape[1]:
                y[i, t] += float(np.float32(b))
        if r.get("mask", -1) >= 0:
            bits = np.unpackbits(masks[r["mask"]].view(np.uint8), bitorder="little")[:y.shape[1]]
            y[i, bits == 0] = -np.inf
    return y


def pick(row):
    row = np.where(np.isnan(row), -np.inf, row)
    return int(np.argmax(row)) if row.max() > -np.inf else 0xFFFFFFFF


def check_rules(aotk, x, rules, masks, kind):
    got, tok = aotk.logits_rules(x, rules, masks, kind)
    want = rules64(x, rules, masks, kind)
    g = unpack(got, kind)
    # f32: at most four roundings (quotient or product, product and sum of the
    # penalties, their difference, the bias), each half a step of a value no
    # larger than this magnitude; then one rounding to the type
    with np.errstate(invalid="ignore"):
        mag = np.abs(unpack(x, kind)) * max([1.0] + [r.get("repetition", 1.0) for r in rules] + [1 / r.get("repetition", 1.0) for r in rules])
        for i, r in enumerate(rules):
            mag[i] += abs(r.get("presence", 0)) + abs(r.get("frequency", 0)) * len(r.get("history", ()))
            mag[i] += max([0.0] + [abs(b) for _, b in (r["bias"].items() if isinstance(r.get("bias"), dict) else r.get("bias", ()))])
        near(g, want, 5 * U * np.where(np.isfinite(mag), mag, 0), 0.0, kind)
    # a value that no rule names keeps its bits, and picks are of the values as written
    for i, r in enumerate(rules):
        named = {int(t) for t in r.get("history", ())} | {int(t) for t, _ in (r["bias"].items() if isinstance(r.get("bias"), dict) else r.get("bias", ()))}
        free = np.ones(x.shape[1], bool)
        free[[t for t in named if t < x.shape[1]]] = False
        free &= ~np.isneginf(want[i])
        size = np.uint32 if kind == F32 else np.uint16
        same = got[i].view(size)[free] == x[i].view(size)[free]
        assert (same | np.isnan(unpack(x[i], kind)[free])).all()
        assert tok[i] == pick(g[i]), f"row {i}"


@KINDS
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 31), (2, 33), (3, 1000), (5, 4096), (2, 4097), (1, 32000), (70, 517),
                                        (4, 20481)], ids=str)
def test_rules(aotk, kind, rows, vocab):
    rng = np.random.default_rng(rows * 31 + vocab)
    x = pack(rng.standard_normal((rows, vocab)) * 3, kind)
    words = (vocab + 31) // 32
    masks = rng.integers(0, 1 << 32, (3, words), dtype=np.uint32)
    masks[1] = 0  # nothing is allowed
    masks[2] = 0xFFFFFFFF  # bits past the vocabulary are set and mean nothing
    rules = []
    for i in range(rows):
        h = [int(t) for t in rng.integers(0, vocab, int(rng.integers(0, 3000 if i == 0 else 40)))]
        b = [(int(t), float(np.float32(s))) for t, s in zip(rng.integers(0, vocab, 12), rng.standard_normal(12) * 5)]
        rules.append({"repetition": [1.0, 1.3, 0.7][i % 3], "presence": [0.0, 0.5][i % 2], "frequency": [0.25, 0.0, -0.1][i % 3],
                      "history": h if i % 4 != 3 else [], "bias": b if i % 5 != 1 else [], "mask": i % 4 - 1})
    check_rules(aotk, x, rules, masks, kind)
    check_rules(aotk, x, [{}] * rows, None, kind)


@KINDS
def test_rules_last_bias_of_a_token_and_names_outside(aotk, kind):
    x = pack(np.array([[1.0, 2.0, 3.0, -1.0, 0.0]]), kind)
    out = [5, 6, 4095, 4096, 0xFFFFFFFF]
    rules = [{"repetition": 2.0, "presence": 0.25, "frequency": 0.5, "history": [3, 0, 0, 3, 3] + out,
              "bias": [(1, 9.0), (2, 1.0), (1, -4.0)] + [(t, 50.0) for t in out], "mask": -1}]
    got, tok = aotk.logits_rules(x, rules, None, kind)
    want = [0.5 - 0.25 - 1.0, 2.0 - 4.0, 4.0, -2.0 - 0.25 - 1.5, 0.0]
    assert np.array_equal(unpack(got, kind)[0], want)
    assert tok[0] == 2


@KINDS
def test_rules_values_not_finite_and_ties(aotk, kind):
    inf, nan = np.inf, np.nan
    rows = np.array([[nan, inf, 1.0, -inf], [nan, nan, nan, nan], [-inf, -inf, nan, -inf], [0.0, 2.0, 2.0, 1.0],
                     [-0.0, 0.0, -1.0, -0.0], [nan, inf, inf, -inf], [-1.0, -3.0, -1.0, -2.0]], np.float32)
    x = pack(rows, kind)
    masks = np.array([[0b1100], [0b0100]], np.uint32)
    plain, tok = aotk.logits_rules(x, [{}] * 7, None, kind)
    assert list(tok) == [1, 0xFFFFFFFF, 0xFFFFFFFF, 1, 0, 1, 0]
    assert np.array_equal(np.isnan(unpack(plain, kind)), np.isnan(rows))
    got, tok = aotk.logits_rules(x, [{"mask": i % 2} for i in range(7)], masks, kind)
    want = rows.copy()
    want[0::2, :2] = -inf
    want[1::2, [0, 1, 3]] = -inf
    g = unpack(got, kind)
    assert np.array_equal(np.isnan(g), np.isnan(want)) and np.array_equal(g[~np.isnan(g)], want[~np.isnan(want)])
    assert list(tok) == [2, 0xFFFFFFFF, 0xFFFFFFFF, 2, 3, 2, 2]


def test_rules_stride_in_place_and_no_picks(aotk):
    rng = np.random.default_rng(2)
    rows, vocab, stride = 5, 4100, 4111
    x = rng.standard_normal((rows, stride)).astype(np.float32)
    t = aotk.DeviceBuffer.from_numpy(x)
    hist = aotk.DeviceBuffer.from_numpy(np.arange(10, dtype=np.uint32))
    rules = np.zeros(rows, aotk.LOGITS_RULE_DTYPE)
    rules["repetition"], rules["presence"], rules["mask"] = 1.0, 2.0, -1
    rules["hist_off"], rules["hist_len"] = [0, 2, 4, 9, 10], [10, 3, 0, 1, 0]
    lib = aotk.abi.load()
    aotk.abi.check(lib.aotk_logits_rules(t.ptr, t.ptr, F32, rows, vocab, stride, rules.ctypes.data, hist.ptr,
                                         10, None, None, 0, None, 0, None))
    want = x.copy()
    for i, (a, n) in enumerate(zip(rules["hist_off"], rules["hist_len"])):
        want[i, a:a + n] -= np.float32(2.0)
    assert np.array_equal(t.to_numpy(np.float32).reshape(rows, stride), want)


# ---------------------------------------------------------------- together
def test_decoding_a_batch_behind_a_prefix_under_rules(aotk, oracle):
    """As they are used: continuations of one prefix decode greedily, each
    step attending to prefix and tail, projecting to logits, applying each
    row's penalties, biases and mask; and the same step by step in float64."""
    nh, nkv, hd, vocab, batch, n_prefix, steps = 4, 2, 64, 300, 5, 37, 6
    rng = np.random.default_rng(11)
    embed = rng.standard_normal((vocab, nh * hd)).astype(np.float32)
    wk, wv = (rng.standard_normal((nkv * hd, nh * hd)).astype(np.float32) / 16 for _ in range(2))
    head = rng.standard_normal((vocab, nh * hd)).astype(np.float32)
    w = aotk.Weight(F32, head.view(np.uint8).reshape(-1), vocab, nh * hd)
    kp, vp = (rng.standard_normal((1, n_prefix, nkv, hd)).astype(np.float32) for _ in range(2))
    kt, vt = (np.full((1, batch, steps, nkv, hd), np.nan, np.float32) for _ in range(2))
    masks = np.stack([aotk.allowed_mask(range(b, vocab, 7), vocab) for b in range(batch)])
    toks = [[b] for b in range(batch)]
    for step in range(steps):
        x = embed[[t[-1] for t in toks]]
        kt[0, :, step] = (x @ wk.T).reshape(batch, nkv, hd)
        vt[0, :, step] = (x @ wv.T).reshape(batch, nkv, hd)
        o = aotk.attention_shared(x.reshape(batch, nh, hd), kp, vp, kt, vt, nh, nkv, hd, n_prefix, n_prefix, steps, 0,
                                  [step + 1] * batch)
        logits = aotk.matmul(w, o.reshape(batch, nh * hd), batch)
        rules = [{"repetition": 1.2, "presence": 0.3, "frequency": 0.1, "history": t, "bias": {5 + b: 0.5}, "mask": b}
                 for b, t in enumerate(toks)]
        out, picks = aotk.logits_rules(logits, rules, masks)
        # the same in float64 from the same inputs
        o64, tol = np.zeros((batch, nh * hd)), np.zeros((batch, nh * hd))
        for b in range(batch):
            k = np.concatenate([kp[0], kt[0, b, :step + 1]]).astype(np.float64)
            v = np.concatenate([vp[0], vt[0, b, :step + 1]]).astype(np.float64)
            a, e = attend64(x[b].reshape(nh, hd).astype(np.float64), k, v, np.ones(len(k), bool))
            o64[b], tol[b] = a.reshape(-1), e.reshape(-1) + np.abs(a.reshape(-1)) * U
        h64 = head.astype(np.float64)
        # the attention's error through the projection, and the projection's own
        lim = tol @ np.abs(h64).T + (nh * hd + 8) * U * (np.abs(o64) @ np.abs(h64).T)
        want = rules64(o64 @ h64.T, rules, masks, F32)
        fine = np.isfinite(want)
        assert np.array_equal(np.isfinite(out), fine)
        assert (np.abs(np.where(fine, out, 0) - np.where(fine, want, 0))[fine] <= (1.3 * lim + 8 * U * (np.abs(np.where(fine, want, 0)) + 2))[fine]).all()
        for b in range(batch):
            assert picks[b] == pick(out[b].astype(np.float64)) and picks[b] % 7 == b % 7
            toks[b].append(int(picks[b]))
    assert len({tuple(t[1:]) for t in toks}) == batch


def test_state_rules_before_the_pick(aotk):
    """A model's logits under a mask: greedy and sampled tokens keep to it."""
    spec = aotk.configs.build("tiny-q4km")
    model = aotk.Model(spec, seed=3)
    st = aotk.State(model, 32, 8)
    prompt = aotk.configs.prompt_tokens(1, 6, spec.d["vocab"])
    st.prompt(prompt, batch=8)
    before = st.logits()
    allowed = [3, 77, 400]
    got = st.apply_rules({"history": prompt, "frequency": 0.01}, aotk.allowed_mask(allowed, spec.d["vocab"]))
    after = st.logits()
    assert got == st.greedy() and got in allowed
    assert np.array_equal(np.flatnonzero(np.isfinite(after)), allowed)
    for t in allowed:
        assert after[t] == before[t] if t not in prompt else after[t] < before[t]
    sampler = aotk.Sampler(temperature=1.0, top_k=2, top_p=1.0)
    assert {st.sample(sampler) for _ in range(20)} <= set(allowed)
    st.set_logits(before)
    assert st.apply_rules({}) == st.greedy()
    assert st.apply_rules({}, aotk.allowed_mask([], spec.d["vocab"])) == aotk.NO_TOKEN


def test_calls_from_several_threads(aotk):
    """Calls of all three at once give what they give alone."""
    rng = np.random.default_rng(8)
    q = rng.standard_normal((3, 8, 128)).astype(np.float32)
    k, v = rng.standard_normal((2, 900, 2, 128)).astype(np.float32)
    kt, vt = rng.standard_normal((2, 3, 8, 2, 128)).astype(np.float32)
    x = rng.standard_normal((3, 9000)).astype(np.float32)
    jobs = [lambda: aotk.attention_sinks(q, k, v, 8, 2, 128, 900, 0, 897, 3, 0, 0),
            lambda: aotk.attention_shared(q, k, v, kt, vt, 8, 2, 128, 900, 900, 8, 0, [8, 1, 4]),
            lambda: aotk.logits_rules(x, [{"history": [1, 2], "frequency": 1.0}] * 3)[0]]
    alone = [j() for j in jobs]
    wrong = []

    def work(n):
        for i in range(6):
            w = (i + n) % 3
            if not np.array_equal(jobs[w](), alone[w]):
                wrong.append(w)

    threads = [threading.Thread(target=work, args=(n,)) for n in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_a_stream_under_capture_is_refused(aotk):
    """Nothing is queued, and the capture goes on."""
    import ctypes as C
    hip = C.CDLL("libamdhip64.so")
    stream, graph = C.c_void_p(aotk.stream()), C.c_void_p()
    lib = aotk.abi.load()
    b = aotk.DeviceBuffer.from_numpy(np.ones(4096, np.float32))
    out = aotk.DeviceBuffer(4096)
    table = aotk.logits_rules_table([{}])[0]
    lens = np.array([1], np.uint32)
    calls = [lambda: lib.aotk_attention_sinks(out.ptr, b.ptr, b.ptr, b.ptr, F32, 1, 1, 64, 4, 0, 3, 1, 0, 0),
             lambda: lib.aotk_attention_shared(out.ptr, b.ptr, b.ptr, b.ptr, b.ptr, b.ptr, F32, 1, 1, 64, 4, 4, 4, 0, 1,
                                               lens.ctypes.data, None),
             lambda: lib.aotk_logits_rules(out.ptr, b.ptr, F32, 1, 64, 64, table.ctypes.data, None, 0, None, None, 0, None, 0, None)]
    assert [c() for c in calls] == [0, 0, 0]
    assert hip.hipStreamBeginCapture(stream, 1) == 0
    try:
        got = [(c(), lib.aotk_last_error()) for c in calls]
    finally:
        assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
        hip.hipGraphDestroy(graph)
    assert all(rc == -1 and b"captured" in why for rc, why in got)
    assert [c() for c in calls] == [0, 0, 0]


def test_calls_beside_a_state_that_generates(aotk):
    """One thread generates on fresh states, each of which captures its decode
    step (greedy) and its sampling step; another makes the three calls: what
    both give is what they give alone."""
    spec = aotk.configs.build("tiny-q4km")
    model = aotk.Model(spec, seed=3)
    prompt = aotk.configs.prompt_tokens(1, 6, spec.d["vocab"])
    rng = np.random.default_rng(12)
    q = rng.standard_normal((3, 8, 128)).astype(np.float32)
    k, v = rng.standard_normal((2, 900, 2, 128)).astype(np.float32)
    kt, vt = rng.standard_normal((2, 3, 8, 2, 128)).astype(np.float32)
    x = rng.standard_normal((3, 9000)).astype(np.float32)
    jobs = [lambda: aotk.attention_sinks(q, k, v, 8, 2, 128, 900, 0, 897, 3, 0, 0),
            lambda: aotk.attention_shared(q, k, v, kt, vt, 8, 2, 128, 900, 900, 8, 0, [8, 1, 4]),
            lambda: aotk.logits_rules(x, [{"history": [1, 2], "frequency": 1.0}] * 3)[0]]

    def tokens():
        st = aotk.State(model, 64, 8)
        st.prompt(prompt, batch=8)
        greedy = st.generate(len(prompt), 8)
        st.prompt(prompt, batch=8)
        return list(greedy) + list(st.generate_sampled(aotk.Sampler(temperature=1.0, top_k=8, seed=5), len(prompt), 8, prompt))

    alone, alone_tokens = [j() for j in jobs], tokens()
    wrong, errors, done = [], [], threading.Event()

    def generate():
        try:
            for i in range(12):
                if tokens() != alone_tokens:
                    wrong.append(("tokens", i))
        except Exception as e:  # noqa: BLE001
            errors.append(repr(e))
        done.set()

    def operators():
        try:
            for i in range(3000):
                if done.is_set():
                    break
                if not np.array_equal(jobs[i % 3](), alone[i % 3]):
                    wrong.append(i)
        except Exception as e:  # noqa: BLE001
            errors.append(repr(e))

    threads = [threading.Thread(target=f) for f in (generate, operators)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and not wrong, (errors, wrong)


# --------------------------------------------- many slices, rows and launches
def rules_of_rows(rng, rows, vocab, n_mask):
    rules = []
    for i in range(rows):
        h = [int(t) for t in rng.integers(0, vocab, int(rng.integers(0, 50)))]
        b = [(int(t), float(np.float32(s))) for t, s in zip(rng.integers(0, vocab, 9), rng.standard_normal(9) * 5)]
        rules.append({"repetition": [1.0, 1.3, 0.7][i % 3], "presence": [0.0, 0.5][i % 2], "frequency": [0.25, 0.0, -0.1][i % 3],
                      "history": h if i % 4 != 3 else [], "bias": b if i % 5 != 1 else [], "mask": i % (n_mask + 1) - 1})
    return rules


@KINDS
@pytest.mark.parametrize("rows,vocab", [(70, 70001), (70, 69001), (1100, 9000)], ids=str)
def test_rules_blocks_of_several_slices(aotk, kind, rows, vocab):
    """More rows x slices than blocks: 9 blocks of 2 slices a row, the last of
    them short or alone, and one block a row. The largest values lie in any
    slice, some twice, next to each other or slices apart."""
    rng = np.random.default_rng(rows + vocab)
    x = rng.standard_normal((rows, vocab)) * 3
    for i in range(rows):
        at = [int(t) for t in rng.integers(0, vocab, 1 + i % 3)] + [vocab - 1] * (i % 4 == 0)
        x[i, at + ([min(at[0] + 1, vocab - 1)] if i % 5 == 0 else [])] = 100.0
    masks = rng.integers(0, 1 << 32, (2, (vocab + 31) // 32), dtype=np.uint32)
    check_rules(aotk, pack(x, kind), rules_of_rows(rng, rows, vocab, 2), masks, kind)


@KINDS
def test_rules_of_more_rows_than_the_arguments_hold(aotk, kind):
    """Calls of growing and shrinking batches, each with rules of its own."""
    rng = np.random.default_rng(40)
    for rows, vocab in ((97, 1500), (300, 700), (97, 4100), (96, 900), (1200, 300), (130, 5000)):
        x = pack(rng.standard_normal((rows, vocab)) * 3, kind)
        masks = rng.integers(0, 1 << 32, (3, (vocab + 31) // 32), dtype=np.uint32)
        check_rules(aotk, x, rules_of_rows(rng, rows, vocab, 3), masks, kind)


def test_rules_of_more_rows_than_a_launch(aotk):
    """65535 rows in the first launch: values and picks of all, exactly."""
    rows, vocab = 65540, 40
    rng = np.random.default_rng(41)
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    masks = rng.integers(0, 1 << 32, (2, 2), dtype=np.uint32)
    masks[0] = 0
    i = np.arange(rows)
    got, tok = aotk.logits_rules(x, [{"presence": 0.25 * (n % 7), "history": [n % vocab], "mask": n % 3 - 1} for n in range(rows)], masks)
    want = x.copy()
    want[i, i % vocab] -= (0.25 * (i % 7)).astype(np.float32)
    bits = np.unpackbits(masks.view(np.uint8), axis=1, bitorder="little")[:, :vocab]
    for m in range(2):
        want[i % 3 == m + 1] = np.where(bits[m], want[i % 3 == m + 1], -np.inf)
    assert np.array_equal(got, want)
    assert np.array_equal(tok, np.where(want.max(1) > -np.inf, want.argmax(1), 0xFFFFFFFF))


# ------------------------------------------------------- weights and range
@pytest.mark.parametrize("kind", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("what,nh,hd", [("sinks", 1, 64), ("sinks", 16, 128), ("sinks", 16, 256), ("sinks", 32, 128),
                                        ("sinks", 32, 64), ("shared", 8, 256), ("shared", 8, 128), ("shared", 16, 64)], ids=str)
def test_weights_of_few_rows_keep_both_parts(aotk, kind, what, nh, hd):
    """Up to 32 rows (16 with heads of 256) a 16-bit weight enters the second
    product as its rounding and the rest's rounding: off by e^2, not by e. Two
    sets of keys, values 1 and -1, whose weights differ by less than half a step
    of the type: rounded weights alone would give 0."""
    e = HALF_STEP[kind]
    delta = {BF16: 0.0015, F16: 2e-4}[kind]  # e^-delta is nearer to 1 than to the type's next value below
    n = 64
    batch = 1 if what == "sinks" else 2
    q = np.zeros((batch, nh, hd))
    q[..., 0] = 1
    k, v = np.zeros((n, 1, hd)), np.ones((n, 1, hd))
    k[::2, 0, 0] = delta * np.sqrt(hd)
    v[1::2] = -1
    q, k, v = pack(q, kind), pack(k, kind), pack(v, kind)
    if what == "sinks":
        got = aotk.attention_sinks(q, k, v, nh, 1, hd, n, 0, n - 1, 1, 0, 0, kind)
    else:
        tails = [np.stack([x[44:], x[44:]]) for x in (k, v)]
        got = aotk.attention_shared(q, k[:44], v[:44], *tails, nh, 1, hd, 44, 44, 20, 0, [20, 20], None, kind)
    q64, k64, v64 = (unpack(x, kind) for x in (q, k, v))
    s = k64[:, 0, 0] / np.sqrt(hd)
    w = np.exp(s - s.max())
    rounded = np.abs((unpack(pack(w, kind), kind) @ v64[:, 0, 0]) / w.sum() - (w @ v64[:, 0, 0]) / w.sum())
    for b in range(batch):
        want, tol = attend64(q64[b], k64, v64, np.ones(n, bool))
        # the rest's rounding, e of at most e of a weight, and f16's smallest steps
        tol = tol + 1.01 * e * e + (n * 2.0 ** -31 if kind == F16 else 0)
        assert (rounded > 4 * (tol + np.abs(want) * e)).all()
        near(unpack(got, kind).reshape(q.shape)[b], want, tol, 0.0, kind)


@pytest.mark.parametrize("kind", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("m", [1, 40, 70])
def test_large_values_overflow_no_earlier_than_the_formula(aotk, kind, hd, m):
    """512 values of up to 4e35: their sum with weights of at most 1 stays in
    f32's range. The latest keys score 5.2 above the earliest, so that a
    maximum that lags behind would give them weights of 180."""
    nh, n = 512, 512  # so many heads that a block takes all keys of its own
    rng = np.random.default_rng(17)
    q = np.zeros((m, nh, hd))
    q[..., 0] = np.sqrt(hd)
    k, v = np.zeros((n, nh, hd), np.float32), rng.uniform(2e35, 4e35, (n, nh, hd)).astype(np.float32)
    k[128:, :, 0] = 5.2
    q, k, v = pack(q, kind), pack(k, kind), pack(v, kind)
    got = unpack(aotk.attention_sinks(q, k, v, nh, nh, hd, n, 0, n - m, m, 0, 0, kind), kind).reshape(m, nh, hd)
    assert (~np.isfinite(got)).sum() == 0
    some = [0, 200, 511]
    k64, v64 = unpack(k[:, some], kind), unpack(v[:, some], kind)
    for i in sorted({0, m // 2, m - 1}):
        visible = np.arange(n) <= n - m + i
        want, tol = attend64(unpack(q[i, some], kind), k64, v64, visible)
        near(got[i, some], want, tol, attend64(unpack(q[i, some], kind), k64, v64, visible)[0], kind)


# -------------------------------------------------------- the largest counts
@KINDS
@pytest.mark.parametrize("nkv", [16384, 1, 128])
def test_the_most_heads(aotk, kind, nkv):
    """16384 query heads, each with its own keys or sharing them; a sample."""
    nh, hd, ctx, m = 16384, 64, 70, 3
    rng = np.random.default_rng(nkv)
    q = pack(rng.standard_normal((m, nh, hd), np.float32), kind)
    k, v = (pack(rng.standard_normal((ctx, nkv, hd), np.float32), kind) for _ in range(2))
    got = aotk.attention_sinks(q, k, v, nh, nkv, hd, ctx, 0, ctx - m, m, 40, 2, kind).reshape(q.shape)
    some = [0, 1, 127, 128, 8191, 8192, 16255, 16383]
    kv = [h * nkv // nh for h in some]
    k64, v64 = unpack(k[:, kv], kind), unpack(v[:, kv], kind)
    check_rows(got[:, some], unpack(q[:, some], kind), [(k64, v64, sinks_visible(ctx, ctx - m + i, 40, 2)) for i in range(m)], kind)


def test_the_most_sequences(aotk):
    """65535 sequences behind one prefix, tails of 0 to 2; a sample."""
    nh, nkv, hd, n = 2, 1, 64, 65535
    rng = np.random.default_rng(50)
    tail_len = np.arange(n) % 3
    q = rng.standard_normal((n, nh, hd), np.float32)
    kp, vp = rng.standard_normal((2, 1, 37, nkv, hd), np.float32)
    kt, vt = rng.standard_normal((2, 1, n, 2, nkv, hd), np.float32)
    got = aotk.attention_shared(q, kp, vp, kt, vt, nh, nkv, hd, 37, 37, 2, 0, tail_len, None, F32).reshape(q.shape)
    for b in [0, 1, 2, 63, 64, 65, 4095, 32767, 65471, 65472, 65533, 65534]:
        k, v = (np.concatenate([p[0], t[0, b, :tail_len[b]]]).astype(np.float64) for p, t in ((kp, kt), (vp, vt)))
        check_rows(got[b:b + 1], q[b:b + 1].astype(np.float64), [(k, v, np.ones(len(k), bool))], F32)
    # every row, by the sum of its weights: all values equal
    one = aotk.attention_shared(q, kp, np.ones_like(vp), kt, np.ones_like(vt), nh, nkv, hd, 37, 37, 2, 0, tail_len, None, F32)
    assert np.abs(one - 1).max() <= 39 * 4 * U


# ------------------------------------------- decode rows in batches of any size
def near_equal_weights(kind, n, hd):
    """Two sets of keys, values 1 and -1, whose weights differ by less than half
    a step of the type: q [hd], k and v [n, 1, hd]."""
    q, k, v = np.zeros(hd), np.zeros((n, 1, hd)), np.ones((n, 1, hd))
    q[0] = 1
    k[::2, 0, 0] = {BF16: 0.0015, F16: 2e-4}[kind] * np.sqrt(hd)
    v[1::2] = -1
    return pack(q, kind), pack(k, kind), pack(v, kind)


@pytest.mark.parametrize("kind", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("nh,hd,batch", [(4, 64, 9), (8, 128, 5), (16, 128, 3), (8, 128, 40), (32, 64, 8), (20, 128, 70), (8, 256, 5),
                                         (16, 256, 40), (20, 128, 3), (24, 64, 2), (32, 128, 2), (16, 128, 1), (8, 64, 4)], ids=str)
def test_weights_of_decode_rows_keep_both_parts_in_any_batch(aotk, kind, nh, hd, batch):
    """A sequence's row is as exact in a large batch as alone: also the prefix's
    blocks, over all sequences' rows, take 16-bit weights in two parts."""
    e, n_prefix, n_tail = HALF_STEP[kind], 150, 10
    q, k, v = near_equal_weights(kind, n_prefix + n_tail, hd)
    q = np.broadcast_to(q, (batch, nh, hd))
    tails = [np.broadcast_to(x[n_prefix:], (batch, n_tail, 1, hd)) for x in (k, v)]
    got = aotk.attention_shared(q, k[:n_prefix], v[:n_prefix], *tails, nh, 1, hd, n_prefix, n_prefix, n_tail, 0, [n_tail] * batch, None,
                                kind)
    got = unpack(got, kind).reshape(batch, nh, hd)
    q64, k64, v64 = (unpack(x, kind) for x in (q, k, v))
    want, tol = attend64(q64[0], k64, v64, np.ones(n_prefix + n_tail, bool))
    s = k64[:, 0, 0] / np.sqrt(hd)
    w = np.exp(s - s.max())
    rounded = np.abs((unpack(pack(w, kind), kind) @ v64[:, 0, 0]) / w.sum() - want)
    tol = tol + 1.01 * e * e + (len(s) * 2.0 ** -31 if kind == F16 else 0)
    assert (rounded > 2 * (tol + np.abs(want) * e)).all()
    for b in range(batch):
        near(got[b], want, tol, 0.0, kind)


@KINDS
@pytest.mark.parametrize("nh,hd,batch", [(4, 64, 9), (8, 128, 5), (16, 128, 40), (8, 256, 5), (16, 256, 40), (20, 128, 3), (32, 64, 2),
                                         (24, 128, 9)], ids=str)
def test_infinite_values_of_the_prefix_in_decode_batches(aotk, kind, nh, hd, batch):
    """Infinities stay infinities, two of both signs and a NaN become NaN, in
    their dimensions alone; also in the prefix's last, short tile."""
    rng = np.random.default_rng(60)
    n_prefix, n_tail = 330, 3
    q = pack(rng.standard_normal((batch, nh, hd)), kind)
    k, v = rng.standard_normal((2, 1, n_prefix, 1, hd))
    for j, d, x in [(10, 5, np.inf), (99, 6, -np.inf), (20, 7, np.inf), (170, 7, -np.inf), (140, 9, np.nan), (329, 12, np.inf),
                    (200, 63, -np.inf), (64, 0, np.inf), (65, 0, np.inf)]:
        v[0, j, 0, d] = x
    kp, vp = pack(k, kind), pack(v, kind)
    kt, vt = (pack(rng.standard_normal((1, batch, n_tail, 1, hd)), kind) for _ in range(2))
    got = aotk.attention_shared(q, kp, vp, kt, vt, nh, 1, hd, n_prefix, n_prefix, n_tail, 0, [n_tail] * batch, None, kind)
    with np.errstate(invalid="ignore"):
        check_rows(got, unpack(q, kind), shared_rows(kp, vp, kt, vt, n_prefix, [n_tail] * batch, [1] * batch, kind, 0), kind)


def test_a_states_cache_as_the_prefix(aotk):
    """What kv_download reads is the prefix of continuations, layer by layer."""
    d = aotk.configs.build("tiny-q4km").d
    nh, nkv, hd, n, n_pos = d["n_head"], d["n_kv_head"], d["head_dim"], 12, 15
    st = aotk.State(aotk.Model(aotk.configs.build("tiny-q4km"), seed=3), 32, 8)
    st.prompt(aotk.configs.prompt_tokens(1, n, d["vocab"]), batch=8)
    kp, vp = (x.reshape(d["n_layer"], n_pos, nkv, hd) for x in st.kv_download(n_pos))
    rng = np.random.default_rng(70)
    q = rng.standard_normal((3, nh, hd)).astype(np.float32)
    kt, vt = rng.standard_normal((2, d["n_layer"], 3, 4, nkv, hd)).astype(np.float32)
    for layer in range(d["n_layer"]):
        got = aotk.attention_shared(q, kp, vp, kt, vt, nh, nkv, hd, n_pos, n, 4, layer, [4, 0, 2])
        check_rows(got, q.astype(np.float64), shared_rows(kp, vp, kt, vt, n, [4, 0, 2], [1] * 3, F32, layer), F32)
