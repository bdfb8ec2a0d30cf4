"""What the C entries of the microscaled operators, the norm and the rotary positions refuse before anything is launched (no device is
touched)."""
from crowdsam_amd import hip


def refused(name, match, *args):
    lib = hip.lib()
    assert getattr(lib, name)(None, *args) == -1, name
    assert match in lib.csam_last_error(), lib.csam_last_error()


def gemm(M, N, K=32, act=0, fmt=1):
    return (64, 256, 64, 4 * M, fmt, 64, 128, 64, 4 * N, 64, N, 0, None, None, 0, 0, act, M, N, K)


def test_the_two_choices_exclude_each_other():
    refused("csam_mx_gemm", b"exclude", *gemm(4, 4, act=16 | 32))
    refused("csam_mx_gemm", b"activation", *gemm(4, 4, act=64))
