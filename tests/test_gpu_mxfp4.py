"""MXFP4 rows, products and expert products on the GPU against their restatement in 64 bits (mx_ref.py: where the tolerances come from)."""
import ctypes as C

import numpy as np
import pytest

import harness as T
import llama_box_amd as L
import mx_ref

pytestmark = pytest.mark.gpu


def rng_of(*key):
    return np.random.default_rng([abs(hash(k)) % (1 << 31) if isinstance(k, str) else k for k in key])


def weights(r, *shape):
    return mx_ref.quantise((r.standard_normal(shape) / np.sqrt(shape[-1])).astype(np.float32))


def acts(r, *shape):
    x = r.standard_normal(shape).astype(np.float32)
    x[..., r.integers(0, shape[-1], max(1, shape[-1] // 100))] *= 12.0
    return x


def rows_of(raw, K):
    return np.asarray(raw).view(np.uint8).reshape(-1, K // 32 * 17)


# ------------------------------------------------------------------------------------------ rows
def hard_rows(K):
    """rows of the values that a quantisation can get wrong"""
    f = np.float32
    r = rng_of(5, K)
    x = r.standard_normal((24, K)).astype(f)
    x[0] = 0
    x[1] = -0.0
    x[2] = np.tile(np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, -4.0], f), K // 16)
    x[3] = np.nextafter(x[2], f(10))
    x[4] = np.nextafter(x[2], f(-10))
    x[5] *= f(1e-38)
    x[6] = r.integers(0, 9, K).astype(f) * f(1.4e-45)
    x[7] *= f(2e37)
    x[8, K // 2] = np.inf
    x[9, K - 1] = -np.inf
    x[10, 0] = np.nan
    x[11] = f(3.4028235e38) * np.where(r.random(K) < 0.5, -1, 1)
    x[12] = f(2.0) ** r.integers(-126, 120, K)
    x[13] = np.nextafter(f(2.0) ** r.integers(-120, 120, K).astype(f), f(0))  # just below a power of two: the exponent of the largest
    x[14:] *= np.exp2(r.integers(-40, 40, (10, 1))).astype(f)
    return x


@pytest.mark.parametrize("K", [32, 64, 96, 1056])
def test_convert(backend, K):
    x = hard_rows(K)

    def build(g):
        q = g.H.ggml_cast(g.ctx, g.new(L.F32, (K, len(x)), x), L.MXFP4)
        return [q, g.H.ggml_cast(g.ctx, q, L.F32)]

    raw, back = T.run_case(build, backend)
    want = mx_ref.quantise(x)
    assert np.array_equal(rows_of(raw, K), want)
    assert np.array_equal(back.reshape(-1, K), mx_ref.values(want).astype(np.float32), equal_nan=True)


@pytest.mark.parametrize("rows", [1, 31, 33, 300])
def test_convert_sizes(backend, rows):
    x = acts(rng_of(6, rows), rows, 160)
    back, = T.run_case(lambda g: g.H.ggml_cast(g.ctx, g.H.ggml_cast(g.ctx, g.new(L.F32, (160, rows), x), L.MXFP4), L.F32), backend)
    assert np.array_equal(back.reshape(-1, 160), mx_ref.values(mx_ref.quantise(x)).astype(np.float32))


@pytest.mark.parametrize("first", [1, 16])
def test_convert_in_place_of_rows(backend, first):
    """some rows of a table written and read back: blocks that start at any byte"""
    r = rng_of(33, first)
    K, R, n = 96, 40, 9
    table, x = weights(r, R, K), acts(r, n, K)

    def build(g):
        H = g.H
        t = g.new(L.MXFP4, (K, R), table)
        put = H.ggml_cpy(g.ctx, g.new(L.F32, (K, n), x), H.ggml_view_2d(g.ctx, t, K, n, t.contents.nb[1], first * t.contents.nb[1]))
        return [H.ggml_cast(g.ctx, put, L.F32), H.ggml_cast(g.ctx, H.ggml_view_2d(g.ctx, t, K, R - 1, t.contents.nb[1], t.contents.nb[1]), L.F32)]

    part, rest = T.run_case(build, backend)
    want = table.copy()
    want[first:first + n] = mx_ref.quantise(x)
    assert np.array_equal(part.reshape(n, K), mx_ref.values(want[first:first + n]).astype(np.float32))
    assert np.array_equal(rest.reshape(R - 1, K), mx_ref.values(want[1:]).astype(np.float32))


@pytest.mark.parametrize("scale", [0, 1, 2, 127, 253, 254, 255])
def test_every_code(backend, scale):
    codes = np.arange(16, dtype=np.uint8)
    p = np.concatenate([[scale], codes | (codes[::-1] << 4)]).astype(np.uint8)[None]
    back, = T.run_case(lambda g: g.H.ggml_cast(g.ctx, g.new(L.MXFP4, (32, 1), p), L.F32), backend)
    with np.errstate(over="ignore"):  # (6 and 4 times 2^127: infinities)
        assert np.array_equal(back.ravel(), mx_ref.values(p).astype(np.float32).ravel(), equal_nan=True)


@pytest.mark.parametrize("K,rows,taken", [(32, 1, 1), (96, 40, 7), (1056, 129, 129), (4096, 33, 5)])
def test_store_and_read(backend, K, rows, taken):
    r = rng_of(7, K, rows)
    table, x = weights(r, rows, K), acts(r, taken, K)
    slots = r.permutation(rows)[:taken].astype(np.int64)
    order = np.concatenate([r.permutation(rows), slots, slots]).astype(np.int32)  # every row, some of them more than once

    def build(g):
        t = g.H.ggml_set_rows(g.ctx, g.new(L.MXFP4, (K, rows), table), g.new(L.F32, (K, taken), x), g.new(L.I64, (taken,), slots))
        return [g.H.ggml_get_rows(g.ctx, t, g.new(L.I32, (len(order),), order)), t]

    got, raw = T.run_case(build, backend)
    want = table.copy()
    want[slots] = mx_ref.quantise(x)
    assert np.array_equal(rows_of(raw, K), want)
    assert np.array_equal(got.reshape(-1, K), mx_ref.values(want)[order].astype(np.float32))


def test_store_strided_batches(backend):
    """rows that are views (any whole number of floats apart), batches of tables, indices shared by them; rows that no index names stay as they were, an index outside the table stores nothing"""
    r = rng_of(8)
    K, R, n, B = 64, 20, 6, 3
    table, x = weights(r, B, R, K), acts(r, B, n, K + 7)
    slots = np.array([3, 19, -1, 0, 20, 7], np.int64)

    def build(g):
        src = g.new(L.F32, ((K + 7), n, B), x)
        v = g.H.ggml_view_3d(g.ctx, src, K, n, B, src.contents.nb[1], src.contents.nb[2], 12)
        t = g.H.ggml_set_rows(g.ctx, g.new(L.MXFP4, (K, R, B), table), v, g.new(L.I64, (n,), slots))
        ids = np.array([[19, 1, 3], [0, 0, 7], [18, 19, 5]], np.int32)
        return [t, g.H.ggml_get_rows(g.ctx, t, g.new(L.I32, (3, B), ids))]

    raw, got = T.run_case(build, backend)
    want = table.copy()
    for b in range(B):
        for i, s in enumerate(slots):
            if 0 <= s < R:
                want[b, s] = mx_ref.quantise(x[b, i, 3:3 + K])
    assert np.array_equal(np.asarray(raw).reshape(want.shape), want)
    ids = np.array([[19, 1, 3], [0, 0, 7], [18, 19, 5]])
    assert np.array_equal(got.reshape(B, 3, K), np.stack([mx_ref.values(want[b])[ids[b]] for b in range(B)]).astype(np.float32))


def test_read_outside_leaves_rows(backend):
    table = weights(rng_of(9), 5, 64)
    ids = np.array([4, 5, -1, 0], np.int32)
    got, = T.run_case(lambda g: g.H.ggml_get_rows(g.ctx, g.new(L.MXFP4, (64, 5), table), g.new(L.I32, (4,), ids)), backend)
    want = np.zeros((4, 64), np.float32)  # (the harness clears its buffers)
    want[0], want[3] = mx_ref.values(table)[[4, 0]]
    assert np.array_equal(got.reshape(4, 64), want)


# ------------------------------------------------------------------------------------------ MUL_MAT
SHAPES = [(32, 1, 1), (32, 33, 3), (64, 31, 2), (96, 129, 1), (128, 16, 16), (160, 64, 17), (224, 257, 33), (256, 100, 64), (2080, 1001, 5), (512, 300, 65), (1056, 70, 129),
          (4096, 512, 1), (4096, 512, 4), (4096, 130, 31), (4096, 260, 32), (640, 515, 200), (14336, 96, 1), (14336, 40, 2), (1024, 1024, 300), (288, 640, 513), (1536, 2050, 513), (2048, 6200, 1000)]


def mul_mat(backend, w, x, K, N, M, **kw):
    return T.run_case(lambda g: g.H.ggml_mul_mat(g.ctx, g.new(L.MXFP4, (K, N), w), g.new(L.F32, (K, M), x)), backend, **kw)[0].reshape(M, N)


@pytest.mark.parametrize("K,N,M", SHAPES)
def test_product(backend, K, N, M, plog):
    r = rng_of(10, K, N, M)
    w, x = weights(r, N, K), acts(r, M, K)
    want, mags = mx_ref.product(x, w)
    plog(f"mxfp4 product K={K} N={N} M={M}: rel {mx_ref.check('product', mul_mat(backend, w, x, K, N, M), want, mags, K):.2e}")


@pytest.mark.parametrize("K,N,M", [(96, 40, 1), (288, 130, 5), (1056, 300, 40), (2048, 600, 200)])
def test_product_of_wide_range(backend, K, N, M):
    """blocks of all sizes beside each other, zeros, rows and columns of zeros"""
    r = rng_of(11, K, N, M)
    w = mx_ref.quantise((r.standard_normal((N, K // 32, 32)) * np.exp2(r.integers(-20, 20, (N, K // 32, 1)))).astype(np.float32).reshape(N, K))
    x = (r.standard_normal((M, K // 32, 32)) * np.exp2(r.integers(-20, 20, (M, K // 32, 1)))).astype(np.float32).reshape(M, K)
    x[0, : K // 2] = 0
    w[N // 2] = 0
    want, mags = mx_ref.product(x, w)
    got = mul_mat(backend, w, x, K, N, M)
    over = np.abs(got - want) > 2.0**-24 * (2 * K + 1) * mags
    assert not over.any()
    assert not got[:, N // 2].any()


@pytest.mark.parametrize("M", [1, 3, 40, 200])
def test_product_infinities_and_nan_stay_in_their_rows_and_columns(backend, M):
    r = rng_of(12, M)
    K, N = 160, 70
    w, x = weights(r, N, K), acts(r, M, K)
    w[13, 17 * 4] = 255                      # a NaN block: row 13
    x[0, 159] = np.inf
    if M > 2:
        x[2, 3] = np.nan
        x[1] *= np.float32(1e-38)            # (below the smallest step: zeros)
    want, mags = mx_ref.product(x, w)
    assert np.isnan(want[0]).all() and np.isnan(want[:, 13]).all()
    mx_ref.check("nan", mul_mat(backend, w, x, K, N, M), want, mags, K)


def test_product_strided_and_batched_activations(backend):
    """columns of a 4-d tensor, their rows a whole number of floats apart; a matrix that is some rows of another"""
    r = rng_of(13)
    K, N = 96, 75
    w, x = weights(r, N + 20, K), acts(r, 2, 3, 5, K + 9)

    def build(g):
        src, m = g.new(L.F32, (K + 9, 5, 3, 2), x), g.new(L.MXFP4, (K, N + 20), w)
        nb = src.contents.nb
        v = g.H.ggml_view_4d(g.ctx, src, K, 4, 3, 2, nb[1], nb[2], nb[3], 4 * 5)
        p = g.H.ggml_permute(g.ctx, v, 0, 2, 1, 3)  # [K, 3, 4, 2]
        part = g.H.ggml_view_2d(g.ctx, m, K, N, m.contents.nb[1], 11 * m.contents.nb[1])
        return [g.H.ggml_mul_mat(g.ctx, part, v), g.H.ggml_mul_mat(g.ctx, part, p)]

    a, b = T.run_case(build, backend)
    want, mags = mx_ref.product(x[:, :, :4, 5:5 + K], w[11:11 + N])
    mx_ref.check("strided", a, want, mags, K)
    mx_ref.check("permuted", b, want.swapaxes(1, 2), mags.swapaxes(1, 2), K)


# rows and columns that take tiles of 64, 128 and 256 rows; K: whole 16-byte pieces, whole dwords, anything
@pytest.mark.parametrize("N,M", [(1001, 600), (2083, 1000), (4129, 1000)])
@pytest.mark.parametrize("K", [1024, 384, 160])
def test_product_tiles(backend, K, N, M):
    r = rng_of(34, K, N)
    w, x = weights(r, N, K), acts(r, M, K)
    want, mags = mx_ref.product(x, w)
    mx_ref.check("tiles", mul_mat(backend, w, x, K, N, M), want, mags, K)


@pytest.mark.parametrize("K,N,M", [(512, 8200, 1100), (1024, 4300, 2500)])
def test_product_low_tiles_behind_tall_ones(backend, K, N, M):
    """products whose last rows are in tiles of 64 and of 128 rows behind whole rounds of tiles of 256"""
    r = rng_of(42, K, N)
    w, x = weights(r, N, K), acts(r, M, K)
    want, mags = mx_ref.product(x, w)
    mx_ref.check("low tiles", mul_mat(backend, w, x, K, N, M), want, mags, K)


@pytest.mark.parametrize("M", [1, 20, 700])
def test_product_rows_far_apart(backend, M):
    """a matrix that is some columns of a much wider one: its rows lie half a megabyte apart"""
    r = rng_of(35, M)
    K, N, wide = 512, 300, 1 << 20
    w, x = weights(r, N, K), acts(r, M, K)
    block = np.zeros((N, wide // 32 * 17), np.uint8)
    block[:, 17 * 64:17 * 80] = w

    def build(g):
        m = g.new(L.MXFP4, (wide, N), block)
        return g.H.ggml_mul_mat(g.ctx, g.H.ggml_view_2d(g.ctx, m, K, N, m.contents.nb[1], 17 * 64), g.new(L.F32, (K, M), x))

    want, mags = mx_ref.product(x, w)
    mx_ref.check("far", T.run_case(build, backend)[0].reshape(M, N), want, mags, K)


def test_product_one_column_like_many(backend):
    """what a token gets does not hang on the kernel that its batch takes by more than the sums' roundings"""
    r = rng_of(14)
    K, N = 1056, 333
    w, x = weights(r, N, K), acts(r, 300, K)
    want, mags = mx_ref.product(x, w)
    for M in (1, 2, 4, 8, 16, 17, 32, 33, 64, 65, 128, 129, 256, 300):
        mx_ref.check(f"M={M}", mul_mat(backend, w, x[:M], K, N, M), want[:M], mags[:M], K)


def test_shared_activations(backend):
    """two matrices over one input, then the input's memory written anew between two products"""
    r = rng_of(15)
    K, N, M = 320, 200, 6
    w0, w1, x = weights(r, N, K), weights(r, K, K), acts(r, M, K)

    def build(g):
        H = g.H
        a, m0, m1 = g.new(L.F32, (K, M), x), g.new(L.MXFP4, (K, N), w0), g.new(L.MXFP4, (K, K), w1)
        y0, y1 = H.ggml_mul_mat(g.ctx, m0, a), H.ggml_mul_mat(g.ctx, m1, a)
        a2 = H.ggml_scale(g.ctx, y1, 2.0)
        g.pair = (a2, y1)
        return [y0, H.ggml_mul_mat(g.ctx, m0, y1), H.ggml_mul_mat(g.ctx, m0, a2), y1]

    y0, y1, y2, mid = T.run_case(build, backend)
    for got, src, m in ((y0, x, w0), (y1, mid, w0), (y2, 2 * mid, w0), (mid, x, w1)):
        want, mags = mx_ref.product(np.asarray(src).reshape(M, K), m)
        mx_ref.check("shared", got.reshape(want.shape), want, mags, K)


# ------------------------------------------------------------------------------------------ MUL_MAT_ID, ADD_ID
def run_experts(backend, w, x, ids, bias, K, N, view_ids=False, **kw):
    E, (Tn, U) = w.shape[0], ids.shape

    def build(g):
        H = g.H
        if view_ids:  # (as top-k leaves them: the first U of a longer row)
            long = np.full((Tn, U + 3), 1 << 20, np.int32)
            long[:, :U] = ids
            t = g.new(L.I32, (U + 3, Tn), long)
            i = H.ggml_view_2d(g.ctx, t, U, Tn, t.contents.nb[1], 0)
        else:
            i = g.new(L.I32, (U, Tn), ids)
        y = H.ggml_mul_mat_id(g.ctx, g.new(L.MXFP4, (K, N, E), w), g.new(L.F32, (K, x.shape[1], Tn), x), i)
        return H.ggml_add_id(g.ctx, y, g.new(L.F32, (N, E), bias), i) if bias is not None else y

    return T.run_case(build, backend, **kw)[0].reshape(Tn, U, N)


def choose(r, Tn, U, E, skew=0.7):
    return np.argsort(-(r.standard_normal((Tn, E)) + skew * r.standard_normal(E)), axis=1)[:, :U].astype(np.int32)


ID_SHAPES = [(32, 1, 1, 1, 1, False), (96, 33, 5, 3, 7, False), (64, 40, 4, 2, 1, True), (2048, 256, 32, 4, 1, True), (1056, 333, 5, 3, 7, True), (160, 130, 32, 4, 16, True),
             (288, 100, 8, 2, 40, False), (512, 200, 8, 2, 150, True), (256, 140, 64, 8, 33, False), (1024, 260, 4, 1, 300, True), (64, 64, 1, 1, 70, True), (96, 50, 200, 6, 50, True)]


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("K,N,E,U,Tn,shared", ID_SHAPES)
def test_experts(backend, K, N, E, U, Tn, shared, bias, plog):
    r = rng_of(20, K, N, E, Tn)
    w, x, ids = weights(r, E, N, K), acts(r, Tn, 1 if shared else U, K), choose(r, Tn, U, E)
    b = r.standard_normal((E, N)).astype(np.float32) if bias else None
    want, mags = mx_ref.experts(x, w, ids, b)
    got = run_experts(backend, w, x, ids, b, K, N, view_ids=bias)
    rel = mx_ref.check("experts", got, want, mags, K, extra=np.abs(b[ids]) if bias else 0.0)
    plog(f"mxfp4 experts K={K} N={N} E={E} U={U} T={Tn}: rel {rel:.2e}")


@pytest.mark.parametrize("N", [1001, 2083, 4129])
@pytest.mark.parametrize("K", [1024, 384, 160])
def test_experts_tiles(backend, K, N):
    """tiles of 64, 128 and 256 rows; two experts, of which one has one column more than whole tiles"""
    r = rng_of(36, K, N)
    Tn = 900
    w, x, b = weights(r, 2, N, K), acts(r, Tn, 1, K), r.standard_normal((2, N)).astype(np.float32)
    ids = (np.arange(Tn) >= 385).astype(np.int32)[r.permutation(Tn)][:, None]
    want, mags = mx_ref.experts(x, w, ids, b)
    mx_ref.check("tiles", run_experts(backend, w, x, ids, b, K, N), want, mags, K, extra=np.abs(b[ids]))


@pytest.mark.parametrize("K", [512, 1536])
def test_experts_short_tiles(backend, K):
    """tall tiles of one, two, three and four groups of columns, beside an expert without any"""
    r = rng_of(43, K)
    N, counts = 2500, [129, 1, 0, 33, 200, 96, 310, 64, 512, 65, 127, 160]
    E, Tn = len(counts), sum(counts)
    w, x, b = weights(r, E, N, K), acts(r, Tn, 1, K), r.standard_normal((E, N)).astype(np.float32)
    ids = np.repeat(np.arange(E, dtype=np.int32), counts)[r.permutation(Tn)][:, None]
    want, mags = mx_ref.experts(x, w, ids, b)
    mx_ref.check("short", run_experts(backend, w, x, ids, b, K, N), want, mags, K, extra=np.abs(b[ids]))


def test_bias_of_fewer_experts(backend):
    """ids behind the bias rows' last: the product alone (ADD_ID), also where the two could be one launch"""
    r = rng_of(37)
    K, N, E, U, Tn = 128, 70, 6, 2, 40
    w, x, ids, b = weights(r, E, N, K), acts(r, Tn, 1, K), choose(r, Tn, U, E), r.standard_normal((4, N)).astype(np.float32)

    def build(g):
        i = g.new(L.I32, (U, Tn), ids)
        y = g.H.ggml_mul_mat_id(g.ctx, g.new(L.MXFP4, (K, N, E), w), g.new(L.F32, (K, 1, Tn), x), i)
        return g.H.ggml_add_id(g.ctx, y, g.new(L.F32, (N, 4), b), i)

    want, mags = mx_ref.experts(x, w, ids, np.concatenate([b, np.zeros((2, N), np.float32)]))
    mx_ref.check("bias", T.run_case(build, backend)[0].reshape(Tn, U, N), want, mags, K, extra=np.abs(want))


@pytest.mark.parametrize("Tn", [1, 60])
def test_bias_result_in_the_activations_memory(backend, Tn):
    """the block of activations that nobody reads any more taken for the sum with the bias, as the graph allocator does"""
    r = rng_of(38, Tn)
    K, N, E = 2048, 2048, 4
    w, x, b = weights(r, E, N, K), acts(r, Tn, 1, K), r.standard_normal((E, N)).astype(np.float32)
    ids = r.integers(0, E, (Tn, 1)).astype(np.int32)
    g = T.G(backend)
    try:
        H, i, src = g.H, g.new(L.I32, (1, Tn), ids), g.new(L.F32, (K, 1, Tn), x)
        y = H.ggml_add_id(g.ctx, H.ggml_mul_mat_id(g.ctx, g.new(L.MXFP4, (K, N, E), w), src, i), g.new(L.F32, (N, E), b), i)
        got, = g.compute([y], same_block=[(y, src)])
    finally:
        g.free()
    want, mags = mx_ref.experts(x, w, ids, b)
    mx_ref.check("in place", got.reshape(Tn, 1, N), want, mags, K, extra=np.abs(b[ids]))


@pytest.mark.parametrize("Tn", [1, 5, 90])
def test_experts_uneven(backend, Tn):
    """all tokens at one expert, an expert twice for one token, experts without a token, ids that name none (their rows stay as they were)"""
    r = rng_of(21, Tn)
    K, N, E, U = 160, 90, 6, 3
    w, x = weights(r, E, N, K), acts(r, Tn, 1, K)
    for ids in (np.full((Tn, U), 4), np.tile([5, 5, 0], (Tn, 1)), np.tile([-1, 2, 6], (Tn, 1)), np.full((Tn, U), 1 << 30)):
        ids = ids.astype(np.int32)
        want, mags = mx_ref.experts(x, w, ids)
        mx_ref.check(str(ids[0]), run_experts(backend, w, x, ids, None, K, N), want, mags, K)  # (the harness clears its buffers: zeros)


@pytest.mark.parametrize("N,U,Tn,E", [(1, 1, 1, 1), (257, 3, 5, 4), (4096, 4, 9, 32)])
def test_add_id(backend, N, U, Tn, E):
    r = rng_of(22, N)
    a, b, ids = r.standard_normal((Tn, U, N)).astype(np.float32), r.standard_normal((E, N)).astype(np.float32), r.integers(0, E, (Tn, U)).astype(np.int32)
    ids[-1, -1] = E  # (names no row: a's row alone)

    def build(g):
        wide = np.full((Tn, U, N + 5), 7.0, np.float32)
        wide[:, :, 2:2 + N] = a
        t = g.new(L.F32, (N + 5, U, Tn), wide)
        v = g.H.ggml_view_3d(g.ctx, t, N, U, Tn, t.contents.nb[1], t.contents.nb[2], 8)
        i = g.new(L.I32, (U, Tn), ids)
        return [g.H.ggml_add_id(g.ctx, g.new(L.F32, (N, U, Tn), a), g.new(L.F32, (N, E), b), i), g.H.ggml_add_id(g.ctx, v, g.new(L.F32, (N, E), b), i)]

    want = a.copy()
    for t in range(Tn):
        for u in range(U):
            if ids[t, u] < E:
                want[t, u] += b[ids[t, u]]
    for got in T.run_case(build, backend):
        assert np.array_equal(got.reshape(want.shape), want)


# ------------------------------------------------------------------------------------------ together
def ffn_block(g, z, stages=False):
    """router -> the experts' gate and up with their biases -> limited SwiGLU -> down with its bias -> weighted sum of a token's experts"""
    H, c = g.H, g.ctx
    K, F, E, U, Tn = z["K"], z["F"], z["E"], z["U"], z["T"]
    x = g.new(L.F32, (K, Tn), z["x"])
    logits = H.ggml_mul_mat(c, g.new(L.F32, (K, E), z["router"]), x)
    ids = H.ggml_top_k(c, logits, U)
    p = H.ggml_get_rows(c, H.ggml_reshape_3d(c, logits, 1, E, Tn), ids)             # [1, U, T]
    p = H.ggml_reshape_3d(c, H.ggml_soft_max(c, H.ggml_reshape_2d(c, p, U, Tn)), 1, U, Tn)
    x3 = H.ggml_reshape_3d(c, x, K, 1, Tn)
    gate = H.ggml_add_id(c, H.ggml_mul_mat_id(c, g.new(L.MXFP4, (K, F, E), z["gate"]), x3, ids), g.new(L.F32, (F, E), z["gate_b"]), ids)
    up = H.ggml_add_id(c, H.ggml_mul_mat_id(c, g.new(L.MXFP4, (K, F, E), z["up"]), x3, ids), g.new(L.F32, (F, E), z["up_b"]), ids)
    act = H.ggml_reshape_3d(c, H.ggml_swiglu_oai(c, H.ggml_reshape_2d(c, gate, F, U * Tn), H.ggml_reshape_2d(c, up, F, U * Tn), 1.702, 7.0), F, U, Tn)
    down = H.ggml_add_id(c, H.ggml_mul_mat_id(c, g.new(L.MXFP4, (F, K, E), z["down"]), act, ids), g.new(L.F32, (K, E), z["down_b"]), ids)
    y = H.ggml_mul(c, down, p)
    s = None
    for u in range(U):
        v = H.ggml_view_2d(c, y, K, Tn, y.contents.nb[2], u * y.contents.nb[1])
        s = v if s is None else H.ggml_add(c, s, v)
    if U == 1:
        s = H.ggml_cont(c, s)
    return [s] + ([gate, up, act, down, ids, p] if stages else [])


def ffn_data(seed, K, F, E, U, Tn):
    r = rng_of(30, seed, K, F, E, Tn)
    return dict(K=K, F=F, E=E, U=U, T=Tn, x=acts(r, Tn, K), router=(r.standard_normal((E, K)) / np.sqrt(K)).astype(np.float32), gate=weights(r, E, F, K), up=weights(r, E, F, K),
                down=weights(r, E, K, F), gate_b=r.standard_normal((E, F)).astype(np.float32), up_b=r.standard_normal((E, F)).astype(np.float32), down_b=r.standard_normal((E, K)).astype(np.float32))


@pytest.mark.parametrize("K,F,E,U,Tn", [(128, 96, 4, 2, 1), (256, 288, 8, 4, 3), (288, 160, 8, 2, 50), (512, 256, 32, 4, 130)])
def test_expert_block(backend, K, F, E, U, Tn):
    """every stage of the block against 64 bits on what the stage was given, and the block as a model runs it (fused, nothing else kept) against the stages"""
    z = ffn_data(1, K, F, E, U, Tn)
    s, gate, up, act, down, ids, p = [np.asarray(o) for o in T.run_case(lambda g: ffn_block(g, z, True), backend)]
    ids, x3 = ids.reshape(-1).view(np.int32), z["x"][:, None]
    ids = np.stack([ids[t * E:t * E + U] for t in range(Tn)])  # (a view of the sorted rows: the first U of E)
    for name, got, src, k in (("gate", gate, x3, K), ("up", up, x3, K), ("down", down, act.reshape(Tn, U, F), F)):
        want, mags = mx_ref.experts(src, z[name], ids, z[name + "_b"])
        mx_ref.check(name, got.reshape(want.shape), want, mags, k, extra=np.abs(z[name + "_b"][ids]))
    gg, uu = np.minimum(gate.astype(np.float64), 7.0), np.clip(up.astype(np.float64), -7.0, 7.0)
    want = gg / (1 + np.exp(-1.702 * gg)) * (uu + 1)
    assert np.allclose(act.reshape(want.shape), want, rtol=2.0**-20, atol=2.0**-20)
    fused, = T.run_case(lambda g: ffn_block(g, z), backend)
    assert np.array_equal(np.asarray(fused), s)


def test_fusion_off_gives_the_same(backend):
    """up to the down projection's rows: their weights come from the router's soft-max, whose fused form rounds in another order"""
    z = ffn_data(2, 256, 288, 8, 4, 60)
    a, = T.run_case(lambda g: ffn_block(g, z, True)[4:5], backend)
    backend.set_option("fusion", 0)
    try:
        b, = T.run_case(lambda g: ffn_block(g, z, True)[4:5], backend)
    finally:
        backend.set_option("fusion", 1)
    assert np.array_equal(np.asarray(a), np.asarray(b))


@pytest.mark.parametrize("Tn", [1, 3, 40, 150])
def test_feed_forward_of_a_dense_model(backend, Tn):
    """norm -> gate, up -> SwiGLU -> down -> + input, alone in its graph (whatever is fused there) and with every stage kept: each product against 64 bits on what it was given"""
    r = rng_of(39, Tn)
    K, F = 512, 736
    x, nw, gw, uw, dw = acts(r, Tn, K), r.standard_normal(K).astype(np.float32), weights(r, F, K), weights(r, F, K), weights(r, K, F)

    def build(g, stages):
        H, c = g.H, g.ctx
        src = g.new(L.F32, (K, Tn), x)
        n = H.ggml_mul(c, H.ggml_rms_norm(c, src, 1e-5), g.new(L.F32, (K,), nw))
        gate, up = H.ggml_mul_mat(c, g.new(L.MXFP4, (K, F), gw), n), H.ggml_mul_mat(c, g.new(L.MXFP4, (K, F), uw), n)
        act = H.ggml_swiglu_split(c, gate, up)
        down = H.ggml_mul_mat(c, g.new(L.MXFP4, (F, K), dw), act)
        return [H.ggml_add(c, down, src)] + ([n, gate, up, act, down] if stages else [])

    y, n, gate, up, act, down = [np.asarray(o).reshape(Tn, -1) for o in T.run_case(lambda g: build(g, True), backend)]
    for name, got, src, m, k in (("gate", gate, n, gw, K), ("up", up, n, uw, K), ("down", down, act, dw, F)):
        want, mags = mx_ref.product(src, m)
        mx_ref.check(name, got, want, mags, k)
    assert np.array_equal(y, down + x)
    alone, = T.run_case(lambda g: build(g, False), backend)
    assert np.array_equal(np.asarray(alone).reshape(y.shape), y)


@pytest.mark.parametrize("M", [1, 8, 40])
@pytest.mark.parametrize("kind", [L.Q4_K, L.Q8_0])
def test_between_products_of_other_formats(backend, kind, M):
    """normed rows whose readers are products by another block format, and a product by an MXFP4 matrix between the two: both use the scratch for activations..
    The other format moves an activation i by at most half a step of its block, d_i = top_i / 254 (blocks of 256 for Q4_K, 32 for Q8_0).  A sum of w_ji e_i with |e_i| <= d_i and no common sign has a
    mean square of at most sum w_ji^2 d_i^2, so the whole is off by at most the 2-norm of sqrt(sum_i w_ji^2 d_i^2) (even steps would leave 1 / sqrt 3 of it): with the values twelve times the others
    some tenth of the whole, where digits of the other product would leave nothing right."""
    r = rng_of(40, M, kind)
    K, N = 512, 256
    x, z, nw, mw = acts(r, M, K), acts(r, M, K), r.standard_normal(K).astype(np.float32), weights(r, N, K)
    ws = [T.rand_blocks(kind, N * K // L.TYPE_BLCK[kind], K, r) for _ in range(2)]

    def build(g):
        H, c = g.H, g.ctx
        n = H.ggml_mul(c, H.ggml_rms_norm(c, g.new(L.F32, (K, M), x), 1e-5), g.new(L.F32, (K,), nw))
        a = H.ggml_mul_mat(c, g.new(kind, (K, N), ws[0]), n)
        m = H.ggml_mul_mat(c, g.new(L.MXFP4, (K, N), mw), g.new(L.F32, (K, M), z))
        b = H.ggml_mul_mat(c, g.new(kind, (K, N), ws[1]), n)
        return [a, m, b]

    a, m, b = [np.asarray(o).reshape(M, N) for o in T.run_case(build, backend)]
    want, mags = mx_ref.product(z, mw)
    mx_ref.check("between", m, want, mags, K)
    x64 = x.astype(np.float64)
    n = x64 / np.sqrt((x64 * x64).mean(-1, keepdims=True) + 1e-5) * nw
    for got, blocks in ((a, ws[0]), (b, ws[1])):
        f = np.empty((N, K), np.float32)
        T.oracle().oracle_dequantize_row(kind, np.ascontiguousarray(blocks).ctypes.data_as(C.c_void_p), f.ctypes.data_as(C.c_void_p), N * K)
        f, size = f.astype(np.float64), 256 if kind == L.Q4_K else 32
        d = np.repeat(np.abs(n).reshape(M, K // size, size).max(-1), size, axis=-1) / 254
        want, off = n @ f.T, np.linalg.norm(np.sqrt(d * d @ (f * f).T))
        assert off < 0.25 * np.linalg.norm(want) and np.linalg.norm(got - want) <= off


@pytest.mark.parametrize("Tn", [1, 6, 80])
def test_replayed_graphs(backend, Tn):
    """two blocks' graphs in turn through the one scratch, captured and replayed, with new inputs each time; every replay against the eager result of the same inputs"""
    H = L.host()
    zs = [ffn_data(3, 256, 96, 8, 2, Tn), ffn_data(4, 160, 288, 5, 3, Tn)]
    gs = []
    for z in zs:
        g = T.G(backend)
        out = ffn_block(g, z)
        xt = g.inputs[0][0]
        first = g.compute(out)
        gs.append((g, out[0], xt, first[0]))
    r = rng_of(31, Tn)
    xs = [[acts(r, Tn, z["K"]) for _ in range(4)] for z in zs]
    want = [[np.asarray(T.run_case(lambda g, z=z, x=x: ffn_block(g, dict(z, x=x)), backend)[0]) for x in row] for z, row in zip(zs, xs)]
    try:
        for turn in range(4):
            for k, (g, out, xt, _) in enumerate(gs):
                x = xs[k][turn]
                H.ggml_backend_tensor_set(xt, x.ctypes.data_as(C.c_void_p), 0, x.nbytes)
                assert H.ggml_backend_graph_compute_async(backend.backend, g.gf) == 0
            backend.synchronize()
            for k, (g, out, xt, _) in enumerate(gs):
                assert np.array_equal(g.read(out), want[k][turn]), (turn, k)
    finally:
        for g, *_ in gs:
            g.free()


def test_two_backends_at_once(built, backend):
    """two backends of one device, each with its own stream and scratch, computing at the same time"""
    H = L.host()
    other = built.Backend(0)
    r = rng_of(32)
    K, N, M = 1024, 700, 40
    made = []
    try:
        for be in (backend, other):
            w, x = weights(r, N, K), acts(r, M, K)
            g = T.G(be)
            out = H.ggml_mul_mat(g.ctx, g.new(L.MXFP4, (K, N), w), g.new(L.F32, (K, M), x))
            g.compute([out])
            made.append((be, g, out, mx_ref.product(x, w)))
        for _ in range(5):
            for be, g, out, _ in made:
                assert H.ggml_backend_graph_compute_async(be.backend, g.gf) == 0
        for be, g, out, (want, mags) in made:
            be.synchronize()
            mx_ref.check("two", g.read(out).reshape(M, N), want, mags, K)
    finally:
        for be, g, out, _ in made:
            g.free()
        other.close()


def test_same_result_every_time(backend):
    z = ffn_data(5, 512, 256, 16, 4, 100)
    a, = T.run_case(lambda g: ffn_block(g, z), backend)
    for _ in range(3):
        assert np.array_equal(np.asarray(a), np.asarray(T.run_case(lambda g: ffn_block(g, z), backend)[0]))


@pytest.mark.parametrize("K,N,M", [(256, 300, 2), (256, 1027, 40), (512, 4100, 700), (160, 2048, 500)])
def test_result_in_host_memory(backend, K, N, M):
    """a graph whose last node is such a product, asked to leave its result in pinned host memory: every form stores there, in rows that are whole 16-byte pieces and that are not"""
    H = L.host()
    result_to = backend.proc("ggml_backend_mi355x_result_to", C.c_int, [C.c_void_p, L.TP, C.c_void_p, C.c_size_t])
    r = rng_of(41, K, N)
    g, pin = T.G(backend), None
    try:
        w, x = weights(r, N, K), acts(r, M, K)
        out = H.ggml_mul_mat(g.ctx, g.new(L.MXFP4, (K, N), w), g.new(L.F32, (K, M), x))
        ref = g.compute([out])[0].reshape(M, N)
        pin = H.ggml_backend_buft_alloc_buffer(H.ggml_backend_dev_host_buffer_type(backend.dev), M * N * 4)
        base = H.ggml_backend_buffer_get_base(pin)
        for _ in range(3):
            C.memset(base, 0x55, M * N * 4)
            assert result_to(backend.backend, out, base, M * N * 4) == 1
            assert H.ggml_backend_graph_compute_async(backend.backend, g.gf) == 0
            backend.synchronize()
            assert np.array_equal(np.ctypeslib.as_array(C.cast(base, C.POINTER(C.c_float)), (M, N)), ref)
    finally:
        if pin:
            H.ggml_backend_buffer_free(pin)
        g.free()
