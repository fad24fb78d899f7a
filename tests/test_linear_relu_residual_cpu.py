"""A relu that keeps z reads its residual a second time: one in the result's place is refused, on the host."""
import ctypes


def test_residual_in_the_results_place_is_refused():
    from gridbook_b200 import _native
    lib = _native.load()
    at, null = ctypes.c_void_p(4096), ctypes.c_void_p(0)
    other = ctypes.c_void_p(8192)
    # (x, x_ld, w, bias, r, r_ld, dtype, M, N, K, act, y, z, stream)
    assert lib.gb_linear_act(at, 64, at, null, other, 8, 0, 300, 8, 64, _native.EPI_RELU, other, at, null) != 0
    assert "residual twice" in lib.gb_last_error().decode()
