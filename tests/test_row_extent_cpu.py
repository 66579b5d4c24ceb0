"""More rows than a tile's 32-bit row index holds are refused before any device call."""

from __future__ import annotations

import ctypes

import pytest

# the first extents whose last tile has a row index past 2^31 - 1
TOO_MANY = [2 ** 31 - 256, 2 ** 31 - 129, 2 ** 31 - 1, 2 ** 31, 2 ** 40]


@pytest.mark.parametrize("rows", TOO_MANY)
@pytest.mark.parametrize("epilogue", [0, 1, 2, 3])
def test_grouped_product(rows, epilogue):
    from ctypes_ext import MgfGemmDesc
    from cutlass_op.bf16_grouped_mm._ext import lib

    d = MgfGemmDesc(epilogue=epilogue, num_groups=1, total_rows=rows, m=64, n=64, k=64, a=4096, lda=64, b=4096, ldb=64,
                    ldb_batch=4096, b_mn_major=1, offs=4096, bias=4096, d=4096, ldd=128, ldd_batch=4096, d2=4096, ldd2=64,
                    aux=4096, ld_aux=128)
    lib.mgf_grouped_gemm_launch.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    assert lib.mgf_grouped_gemm_launch(ctypes.byref(d), None) == -1


@pytest.mark.parametrize("rows", TOO_MANY)
@pytest.mark.parametrize("epilogue", [0, 1, 2])
def test_block_scaled_product(rows, epilogue):
    from cutlass_op.bf16_grouped_mm._ext import lib

    i32, i64, ptr, f32 = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p, ctypes.c_float

    class Desc(ctypes.Structure):  # include/moe_gemm.h: mgf_block_gemm_desc
        _fields_ = [("epilogue", i32), ("num_groups", i32), ("total_rows", i64), ("n", i64), ("k", i64), ("a", ptr),
                    ("lda", i64), ("b", ptr), ("ldb", i64), ("ldb_batch", i64), ("b_mn_major", i32),
                    ("sm_carveout", i32), ("offs", ptr), ("scale_a", ptr), ("scale_a_stride", i64), ("scale_b", ptr),
                    ("scale_b_stride_e", i64), ("scale_b_stride_k", i64), ("scale_b_stride_n", i64), ("bias", ptr),
                    ("bias_stride", i64), ("d", ptr), ("ldd", i64), ("d2", ptr), ("ldd2", i64), ("aux", ptr),
                    ("ld_aux", i64), ("swiglu_alpha", f32), ("swiglu_limit", f32), ("workspace", ptr)]

    lib.mgf_block_gemm_desc_size.restype = ctypes.c_size_t
    assert ctypes.sizeof(Desc) == lib.mgf_block_gemm_desc_size()
    p = 4096
    d = Desc(epilogue, 1, rows, 64, 64, p, 64, p, 64, 4096, 1, 0, p, p, 1, p, 1, 1, 1, p, 64, p, 128, p, 64, p, 128, 1.0,
             7.0, None)
    lib.mgf_block_gemm_launch.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    assert lib.mgf_block_gemm_launch(ctypes.byref(d), None) == -1
