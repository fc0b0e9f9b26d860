"""MXFP4 products whose kernels take several turns over what one turn does not hold, rows that are neither whole pieces nor whole dwords in every form, and two backends whose rounds all count;
against the restatement in 64 bits (mx_ref.py: where the tolerances come from)."""
import ctypes as C

import numpy as np
import pytest

import harness as T
import llama_box_amd as L
import mx_ref
from test_gpu_mxfp4 import acts, choose, mul_mat, rng_of, run_experts, weights

pytestmark = pytest.mark.gpu


def check_experts(backend, r, K, N, E, ids, bias, shared=True):
    Tn, U = ids.shape
    w, x = weights(r, E, N, K), acts(r, Tn, 1 if shared else U, K)
    b = r.standard_normal((E, N)).astype(np.float32) if bias else None
    named = (ids >= 0) & (ids < E)
    want, mags = mx_ref.experts(x, w, ids, b)
    got = run_experts(backend, w, x, ids.astype(np.int32), b, K, N)
    extra = np.where(named[..., None], np.abs(b[np.where(named, ids, 0)]), 0.0) if bias else 0.0
    mx_ref.check("experts", got, want, mags, K, extra=extra)  # (the harness clears its buffers: rows that no id names are zeros, as mx_ref.experts leaves them)


# columns of one expert beyond the 16 that the one-launch form has at a time (fewer for long rows)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("K,N,E,counts", [(96, 40, 3, [0, 17, 0]), (256, 300, 4, [33, 0, 5, 1]), (96, 50, 2, [64, 0]), (160, 70, 2, [31, 33]), (14336, 48, 2, [0, 5]), (14336, 33, 3, [3, 7, 1])])
def test_one_experts_columns_in_turns(backend, K, N, E, counts, bias):
    r = rng_of(50, K, N, sum(counts))
    ids = np.repeat(np.arange(E), counts)[r.permutation(sum(counts))][:, None]
    check_experts(backend, r, K, N, E, ids, bias)


# ids beyond the 4096 that the grouping takes a round
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("K,N,E,U,Tn", [(32, 33, 3, 1, 4096), (64, 20, 5, 1, 4097), (32, 40, 7, 3, 3001), (64, 17, 300, 2, 6000)])
def test_ids_in_rounds(backend, K, N, E, U, Tn, bias):
    r = rng_of(51, E, Tn)
    ids = r.integers(0, E, (Tn, U))
    ids[r.random((Tn, U)) < 0.05] = -1
    ids[r.random((Tn, U)) < 0.05] = E
    if not bias:
        return check_experts(backend, r, K, N, E, ids, False, shared=False)
    ids = np.clip(ids, 0, E - 1)  # (with a bias a row that no id names is ADD_ID's affair)
    check_experts(backend, r, K, N, E, ids, True)


@pytest.mark.parametrize("K", [38912, 40960])
def test_one_column_of_a_row_beyond_lds(backend, K):
    r = rng_of(52, K)
    w, x = weights(r, 70, K), acts(r, 1, K)
    want, mags = mx_ref.product(x, w)
    mx_ref.check("long", mul_mat(backend, w, x, K, 70, 1), want, mags, K)


# rows of 1530 bytes: they start at even bytes only, and end inside a step
@pytest.mark.parametrize("N,M", [(100, 1), (2880, 1), (2880, 3), (300, 12), (2880, 32), (700, 100), (2880, 300), (2880, 1100), (5000, 900)])
def test_product_of_rows_at_even_bytes(backend, N, M):
    K = 2880
    r = rng_of(53, N, M)
    w, x = weights(r, N, K), acts(r, M, K)
    want, mags = mx_ref.product(x, w)
    mx_ref.check("even", mul_mat(backend, w, x, K, N, M), want, mags, K)


@pytest.mark.parametrize("N,E,U,Tn", [(720, 32, 4, 1), (360, 8, 4, 8), (360, 8, 4, 64), (1440, 4, 4, 300), (130, 128, 4, 500), (2880, 3, 1, 700)])
def test_experts_of_rows_at_even_bytes(backend, N, E, U, Tn):
    K = 2880
    r = rng_of(54, N, E, Tn)
    check_experts(backend, r, K, N, E, choose(r, Tn, U, E), True)


def test_two_backends_with_new_inputs_each_round(built, backend):
    """two backends of one device at the same time, of other sizes each; every round has inputs of its own and finds the output cleared"""
    H = L.host()
    other = built.Backend(0)
    r = rng_of(55)
    made = []
    try:
        for be, (K, N, M) in ((backend, (1024, 700, 40)), (other, (1536, 900, 300))):
            w, xs = weights(r, N, K), [acts(r, M, K) for _ in range(4)]
            g = T.G(be)
            out = H.ggml_mul_mat(g.ctx, g.new(L.MXFP4, (K, N), w), g.new(L.F32, (K, M), xs[0]))
            xt = g.inputs[1][0]
            g.compute([out])
            made.append((be, g, out, xt, K, N, M, xs, [mx_ref.product(x, w) for x in xs]))
        for turn in range(4):
            for be, g, out, xt, K, N, M, xs, want in made:
                H.ggml_backend_tensor_set(xt, xs[turn].ctypes.data_as(C.c_void_p), 0, xs[turn].nbytes)
                H.ggml_backend_tensor_memset(out, 0x7F, 0, M * N * 4)
            for be, g, out, *_ in made:
                assert H.ggml_backend_graph_compute_async(be.backend, g.gf) == 0
            for be, g, out, xt, K, N, M, xs, want in made:
                be.synchronize()
                mx_ref.check("two", g.read(out).reshape(M, N), *want[turn], K)
    finally:
        for be, g, *_ in made:
            g.free()
        other.close()
