"""The FP8 tiles refuse rows that their epilogue would run past, before they look at a device."""
import ctypes
import struct

import pytest


@pytest.mark.parametrize("rows", [64, 192, 4032, 0])
def test_rows_that_are_no_multiple_of_128_are_refused(rows):
    from mimo_prismwing_b200 import load
    # launch_fp8_gemm(Fp8CodesArgs const &, int, cudaStream_t): weight, its scales, codes, scales; rows, K, layout, width
    launch = getattr(load(), "_ZN2pw15launch_fp8_gemmERKNS_12Fp8CodesArgsEiP11CUstream_st")
    args = ctypes.create_string_buffer(struct.pack("=QQQQIIII", 0, 0, 0, 0, rows, 256, 0, 300), 256)
    launch.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p]
    assert launch(args, 148, None) == 1  # cudaErrorInvalidValue
