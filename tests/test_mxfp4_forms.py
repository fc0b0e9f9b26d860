"""The forms that MXFP4 products choose (host arithmetic, no device): a tile's height is one that a kernel exists for."""
import ctypes as C

import pytest

import llama_box_amd as L


@pytest.fixture(scope="module")
def rows(built):
    H = L.host()
    lib = C.CDLL(L.BACKEND_SO)
    lib.ggml_backend_mi355x_reg.restype = C.c_void_p
    return C.CFUNCTYPE(C.c_int, C.c_int64, C.c_int64, C.c_int64, C.c_int64)(H.ggml_backend_reg_get_proc_address(lib.ggml_backend_mi355x_reg(), b"ggml_backend_mi355x_mx_tile_rows"))


COLS = (1, 2, 16, 17, 33, 64, 100, 128, 200, 256, 384, 512, 700, 1024, 1536, 2048, 4096, 20000)


@pytest.mark.parametrize("K", [32, 512, 1536, 2080, 2880, 4064, 4096, 4224])
@pytest.mark.parametrize("experts", [0, 1, 5, 32, 128])
def test_heights_exist(rows, K, experts):
    for N in (1, 33, 64, 65, 127, 128, 200, 255, 256, 1001, 2080, 4096, 14336):
        for cols in COLS:
            h = rows(K, N, experts, cols)
            assert h in (0, 64, 128, 256)
            if K % 512:  # rows that are not whole 16-byte pieces: no tiles of 256, and none of 128 for what one of 64 holds
                assert h <= 128 and (h < 128 or N > 64), (N, cols, h)
            else:  # a tall tile takes its rows from the matrix, whole
                assert h <= 64 or N >= h, (N, cols, h)


def test_heights_of_rows_that_are_not_whole_pieces(rows):
    """128 rows from 512 tiles of 64 on (two a CU), and of experts with few columns from 2200 on"""
    assert rows(4064, 4096, 0, 1536) == 128 and rows(4064, 4096, 0, 1024) == 128 and rows(4064, 4096, 0, 512) == 64 and rows(4224, 2080, 0, 1024) == 64 and rows(2880, 2880, 0, 2048) == 128
    assert rows(2080, 2080, 32, 80) == 64 and rows(2080, 2080, 32, 2000) == 128 and rows(2080, 2080, 128, 2000) == 128 and rows(1056, 4096, 32, 240) == 64
    assert rows(512, 4096, 0, 2048) > 0  # (whole pieces: by their own costs)
