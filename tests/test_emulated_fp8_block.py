"""GPU tests of the FP8 block operators' details, run on the kernels' source on the CPU (see tests/test_emulated_routing.py)."""
import test_kernel_source_emulation as E
from test_emulated_routing import library, on_cpu  # noqa: F401  (fixtures)


def test_emulated_rounding(on_cpu):  # noqa: F811
    import test_gpu_fp8_block_rounding as G
    assert E.run_gpu_tests(G) > 50


def test_emulated_forward_mode(on_cpu):  # noqa: F811
    import test_gpu_moe_forward_mode as G
    assert E.run_gpu_tests(G) == 4


def test_emulated_saved_rows(on_cpu):  # noqa: F811
    import test_gpu_moe_saved_rows as G
    assert E.run_gpu_tests(G) == 4
