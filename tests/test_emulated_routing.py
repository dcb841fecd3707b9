"""The source of the FP8 block quantizer and of the routing kernels, executed on the CPU: the GPU tests of both, called
with all their parameters on host tensors (how the emulation works: tests/test_kernel_source_emulation.py)."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

import test_kernel_source_emulation as E


@pytest.fixture(scope='module')
def library(tmp_path_factory):
    if shutil.which('g++') is None or not os.path.exists(os.path.join(E.CUDA_INCLUDE, 'cuda_fp8.h')):
        pytest.skip('needs g++ and the CUDA headers')
    out = str(tmp_path_factory.mktemp('emu_routing') / 'libamct_emu_routing.so')
    subprocess.check_call(['g++', '-std=c++17', '-O1', '-w', '-ffp-contract=off', '-fsanitize=alignment', '-fno-sanitize-recover=alignment',
                           '-fPIC', '-shared', '-x', 'c++', '-include', os.path.join(E.EMU, 'cuda_emu_routing.h'), '-I', E.CUDA_INCLUDE,
                           os.path.join(E.CSRC, 'fp8_block_quant.cu'), os.path.join(E.CSRC, 'moe_permute.cu'), '-o', out, '-lpthread'])
    handle = ctypes.CDLL(out)
    from amct_b200.backend import lib
    monkeypatch = pytest.MonkeyPatch()
    monkeypatch.setattr(lib, '_SIGNATURES', {n: s for n, s in lib._SIGNATURES.items() if hasattr(handle, n)})
    lib.declare(handle)
    monkeypatch.undo()
    return handle


@pytest.fixture
def on_cpu(library, monkeypatch):
    ops = E.patch_ops(monkeypatch, library)
    monkeypatch.setattr(ops, '_raw_stream', lambda: 0)
    return ops


def test_emulated_fp8_block_quant(on_cpu):
    import test_gpu_fp8_block_quant as G
    assert E.run_gpu_tests(G) > 90


def test_emulated_routing(on_cpu):
    import test_gpu_moe_permute as G
    assert E.run_gpu_tests(G, skip=("test_many_chunks_of_assignments", "test_more_than_two_gigabytes_of_rows", "test_backward_captured_and_replayed")) > 150


def test_emulated_many_chunks(on_cpu):
    import test_gpu_moe_permute as G
    G.test_many_chunks_of_assignments(2600, 4, 40)
