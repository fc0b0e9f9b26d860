"""MXFP4 on the host: sizes, names, and what supports_op takes and refuses (host arithmetic, no device)."""
import ctypes as C

import numpy as np
import pytest

import llama_box_amd as L
import mx_ref


@pytest.fixture(scope="module")
def ask(built):
    H = L.host()
    lib = C.CDLL(L.BACKEND_SO)
    lib.ggml_backend_mi355x_reg.restype = C.c_void_p
    return C.CFUNCTYPE(C.c_int, L.TP)(H.ggml_backend_reg_get_proc_address(lib.ggml_backend_mi355x_reg(), b"ggml_backend_mi355x_supports_probe"))


@pytest.fixture()
def g(built):
    H = L.host()
    ctx = H.ggml_init(L.InitParams(0, None, True))

    class Ctx:
        def new(self, kind, *ne):
            return H.ggml_new_tensor_4d(ctx, kind, *(list(ne) + [1] * (4 - len(ne))))

        def __getattr__(self, name):
            return lambda *a: getattr(H, "ggml_" + name)(ctx, *a)

    yield Ctx()
    H.ggml_free(ctx)


def test_sizes(H, g):
    assert H.ggml_row_size(L.MXFP4, 4096) == 4096 // 32 * 17 == L.TYPE_SIZE[L.MXFP4] * 128
    t = g.new(L.MXFP4, 96, 7)
    assert H.ggml_nbytes(t) == 7 * 51 and t.contents.nb[1] == 51 and t.contents.nb[0] == 17


def test_reference_round_trip():
    # (the restatement itself: every value of every scale comes back, and a quantised row is what it stands for)
    codes = np.arange(16, dtype=np.uint8)
    for e in (0, 1, 2, 100, 127, 200, 252):
        p = np.concatenate([[e], codes | (codes[::-1] << 4)]).astype(np.uint8)[None]
        v = mx_ref.values(p)
        assert np.array_equal(mx_ref.values(mx_ref.quantise(v.astype(np.float32))), v)
    x = np.array([[1.0, 0.25, -0.25, 0.26, 3.5, 4.0, 7.9, -5.0] * 4], np.float32)  # 2^(e - 127) = 1 (largest 7.9)
    assert mx_ref.values(mx_ref.quantise(x))[0, :8].tolist() == [1.0, 0.0, 0.0, 0.5, 3.0, 4.0, 6.0, -4.0]
    a = np.zeros((1, 32), np.float32)
    for top, q in ((255.0, 255.0), (255.49, 255.0), (255.5, 256.0), (1e-45, 0.0), (3.4e38, 3.4e38)):
        a[0, 3] = top
        assert abs(mx_ref.activations(a)[0, 3] - q) <= (0 if q < 1e9 else 2.0**-8 * q)


def test_rows_taken_and_refused(ask, g):
    table, rows = g.new(L.MXFP4, 96, 50), g.new(L.F32, 96, 4)
    assert ask(g.set_rows(table, rows, g.new(L.I64, 4)))
    assert ask(g.get_rows(table, g.new(L.I32, 9)))
    assert ask(g.cast(rows, L.MXFP4)) and ask(g.cast(table, L.F32))
    assert not ask(g.cast(table, L.F16)) and not ask(g.cast(g.new(L.F16, 96, 4), L.MXFP4)) and not ask(g.cast(g.new(L.Q8_0, 96, 4), L.MXFP4))
    strided = g.view_2d(g.new(L.F32, 128, 4), 96, 4, 512, 0)
    assert not ask(g.cast(strided, L.MXFP4)) and ask(g.set_rows(table, strided, g.new(L.I64, 4)))
    assert not ask(g.set_rows(table, g.transpose(g.new(L.F32, 4, 96)), g.new(L.I64, 4)))


def test_products_taken_and_refused(ask, g):
    w, x = g.new(L.MXFP4, 96, 50), g.new(L.F32, 96, 4)
    assert ask(g.mul_mat(w, x)) and ask(g.mul_mat(w, g.new(L.F32, 96, 4, 3, 2)))
    assert not ask(g.mul_mat(w, g.new(L.F16, 96, 4)))                              # activations are f32
    assert not ask(g.mul_mat(g.new(L.MXFP4, 96, 50, 2), g.new(L.F32, 96, 4, 2)))   # one matrix
    assert not ask(g.mul_mat(w, g.transpose(g.new(L.F32, 4, 96))))                 # dense rows
    assert not ask(g.mul_mat(w, g.new(L.F32, 96, 1 << 22)))                        # more columns than a launch has
    odd = g.new(L.F32, 96, 4)
    odd.contents.nb[1] = 97 * 4 - 1
    assert not ask(g.mul_mat(w, odd))                                              # rows at whole floats
    assert ask(g.mul_mat(g.view_2d(w, 96, 20, w.contents.nb[1], 7 * 51), x))       # some of the rows


def test_expert_products_taken_and_refused(ask, g):
    w, ids = g.new(L.MXFP4, 64, 40, 8), g.new(L.I32, 3, 5)
    one, three = g.new(L.F32, 64, 1, 5), g.new(L.F32, 64, 3, 5)
    y = g.mul_mat_id(w, one, ids)
    assert ask(y) and ask(g.mul_mat_id(w, three, ids))
    assert not ask(g.mul_mat_id(w, g.new(L.F16, 64, 1, 5), ids))
    assert not ask(g.mul_mat_id(g.new(L.MXFP4, 64, 40, 1025), one, ids))           # more experts than the lists hold
    assert not ask(g.mul_mat_id(g.new(L.Q8_0, 64, 40, 8), one, ids))               # (no other block format)
    assert ask(g.add_id(y, g.new(L.F32, 40, 8), ids))
    assert not ask(g.add_id(y, g.new(L.F16, 40, 8), ids))
    bad = g.add_id(y, g.new(L.F32, 40, 8), ids)
    bad.contents.src[2].contents.ne[0] = 2
    assert not ask(bad)                                                            # an id for every row


def test_sizes_refused(ask, g):
    """what the launches and the kernels' 32-bit offsets do not hold"""
    x = g.new(L.F32, 96, 4)
    assert not ask(g.mul_mat(g.new(L.MXFP4, 1 << 24, 2), g.new(L.F32, 1 << 24, 1)))        # rows of more than 8 MiB
    far = g.new(L.MXFP4, 96, 50)
    far.contents.nb[1] = (1 << 23) + 17
    assert not ask(g.mul_mat(far, x))
    far.contents.nb[1] = (1 << 23) - 3
    assert ask(g.mul_mat(far, x))
    assert not ask(g.mul_mat(g.new(L.MXFP4, 96, 1 << 26), x))                              # rows, and rows times columns
    assert not ask(g.mul_mat(g.new(L.MXFP4, 96, 1 << 20), g.new(L.F32, 96, 1 << 18)))
    assert not ask(g.set_rows(g.new(L.MXFP4, 32, 50), g.new(L.F32, 32, 1 << 24), g.new(L.I64, 1 << 24)))
    w, one = g.new(L.MXFP4, 64, 40, 8), g.new(L.F32, 64, 1, 5)
    y = g.mul_mat_id(w, one, g.new(L.I32, 3, 5))
    y.contents.src[0].contents.ne[2] = 0                                                   # no experts
    assert not ask(y)
