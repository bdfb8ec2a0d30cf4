"""What the C entries of the microscaled operators, the norm and the rotary positions refuse before anything is launched (no device is
touched)."""
import pytest

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


def test_calls_of_too_many_work_items_are_refused():
    """HIP launches fewer than 2^32 work items; what needs more is refused, not left to the runtime."""
    big = (1 << 31) - 256
    refused("csam_mx_quantize", b"one launch", 64, 1, 0, 64, 128, 64, 1 << 33, 0, big, 1)
    refused("csam_mx_quantize", b"one launch", 64, 1 << 20, 0, 64, 1 << 20, 64, 1 << 33, 1, 1 << 19, 1 << 20)
    refused("csam_mx_dequantize", b"one launch", 64, 128, 64, 1 << 33, 0, 64, 1, 0, big, 1)
    refused("csam_mx_dequantize", b"one launch", 64, 256, 64, 1 << 33, 1, 64, 256, 1, 1 << 28, 256)
    refused("csam_mx_gemm", b"one launch", *gemm(1, big))
    refused("csam_mx_gemm", b"one launch", *gemm(big, 300))
    refused("csam_mx_gemm", b"one launch", *gemm(1 << 20, 1 << 20, act=16))
    refused("csam_mx_gemm", b"one launch", *gemm(1 << 20, 1 << 20, act=32))
    for rows, d in ((1 << 26, 64), (1 << 26, 2048), (1 << 24, 2056), (1 << 24, 8192), (1 << 22, 8200), (1 << 22, 32768)):
        refused("csam_rms_norm", b"one launch", 64, d, 0, None, 0, 0, None, 0, 64, 1e-6, 64, d, 0, rows, d)
        refused("csam_rms_norm_mx", b"one launch", 64, d, 0, None, 0, 0, None, 0, 64, 1e-6, 64, 1 << 15, 64, 1 << 33, 1, rows, d)
    refused("csam_rotary", b"one launch", 64, 1 << 14, 8, 64, 1 << 14, 8, 1 << 8, None, 0, 0, None, 0, 0, 0, 0, 64, big, 0, 64, 64, 1, 1, 0, big, big, 8)


def test_a_refusal_is_a_value_error():
    for kind in (ValueError, RuntimeError):
        with pytest.raises(kind, match="one launch"):
            hip.call("csam_mx_gemm", None, *gemm(1, (1 << 31) - 256))
