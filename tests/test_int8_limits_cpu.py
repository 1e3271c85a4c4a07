"""The longest K that the 8-bit products admit — no GPU."""
import ctypes

import kebab_b200 as kb

P = ctypes.c_void_p(64)


def test_longest_k():
    from kebab_b200._call import function

    def gemm(K, M):
        return function("kebab_gemm_i8")(kb.F16, P, K, P, P, K, P, None, P, 64, M, 64, K, None)

    def grouped(K, M):
        return function("kebab_gemm_grouped_i8")(kb.F16, P, K, P, P, K, 64 * K, P, P, 64, P, 2, M, 64, K, None)

    def linear(K, M):
        return function("kebab_linear_i8")(kb.F16, P, K, P, K, 0, P, None, P, 64, None, 1, M, 64, K, P, 1 << 20, None)

    for call, most in ((gemm, 131071), (grouped, 131071), (linear, 131072)):
        assert call(most, 0) == kb.OK  # no rows: nothing but the checks
        for M in (0, 4):
            assert call(most + 1, M) == kb.EINVAL and "overflow" in kb.last_error()
