"""The FP8 block product behind a bounded wait that runs out: whatever the wait left unknown is NaN, the status word has its bit,
everything else is right, and the next call is as if nothing had been.  The kernels' source is built once more with a limit
that is set at run time and looked at after every poll; all waits are there, they give up sooner."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
SOURCE = r'''
static __device__ unsigned long long wait_limit_ns = 2000000000ull;
#define AMCT_WAIT_LIMIT_NS wait_limit_ns
#define AMCT_WAIT_POLLS 1
#define AMCT_WAIT_PTX "mbarrier.test_wait"
#include "gemm_fp8_block.cu"
extern "C" int set_wait_limit(unsigned long long ns) { return cudaMemcpyToSymbol(wait_limit_ns, &ns, sizeof(ns)) != cudaSuccess; }
'''
PATIENT = 2000000000


@pytest.fixture(scope='module')
def library(tmp_path_factory):
    from amct_b200.csrc import build
    nvcc = os.environ.get('NVCC', '/usr/local/cuda/bin/nvcc')
    if shutil.which(nvcc) is None:
        pytest.skip('needs nvcc')
    folder = tmp_path_factory.mktemp('wait_limit')
    (folder / 'impatient.cu').write_text(SOURCE)
    out = str(folder / 'impatient.so')
    subprocess.check_call([nvcc, '-gencode', 'arch=compute_100a,code=sm_100a', '-O3', '-std=c++17', '-Xcompiler', '-fPIC', '-shared', '--expt-relaxed-constexpr',
                           '-I', build.INCLUDE, '-I', build.HERE, '-cudart', 'static', '-o', out, str(folder / 'impatient.cu')])
    from amct_b200.backend import lib
    handle = ctypes.CDLL(out)
    for name in ('amct_gemm_fp8_block', 'amct_gemm_fp8_block_grouped'):
        getattr(handle, name).argtypes = [lib._CTYPES[c] for c in lib._SIGNATURES[name]]
    handle.set_wait_limit.argtypes = [ctypes.c_ulonglong]
    return handle


def operands(m, n, k, experts, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)

    def codes(*shape):
        return (torch.randn(*shape, generator=gen, device='cuda') * 50).clamp(-448, 448).to(F8)

    def scales(*shape):
        return torch.rand(*shape, generator=gen, device='cuda') + 0.5
    kb, nb = -(-k // 128), -(-n // 128)
    lead = (experts,) if experts else ()
    return codes(m, k), scales(m, kb), codes(*lead, n, k), scales(*lead, nb, kb)


# decode with K split over a cluster, more tokens, the wide kernel with ragged tiles and a bias, and with several tiles a CTA
SHAPES = [(1, 1024, 4096, 0, False), (40, 300, 2048, 0, True), (100, 512, 1024, 0, False), (300, 5001, 512, 0, True), (4096, 4096, 256, 0, False),
          (64, 512, 2048, 8, False), (900, 2048, 512, 3, False)]


@pytest.mark.parametrize('out_dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('m,n,k,experts,bias', SHAPES)
def test_unknown_outputs_are_nan(m, n, k, experts, bias, out_dtype, library, monkeypatch):
    from amct_b200.backend import lib, ops
    a, a_scale, b, b_scale = operands(m, n, k, experts, m + n)
    b_bias = torch.randn(n, device='cuda') if bias else None
    offsets = torch.tensor([m * e // (experts + 1) for e in range(experts + 1)], dtype=torch.int32, device='cuda') if experts else None
    end = int(offsets[-1]) if experts else m

    def run():
        out, status = torch.full((m, n), 7.0, dtype=out_dtype, device='cuda'), torch.zeros(1, dtype=torch.int32, device='cuda')
        if experts:
            ops.gemm_fp8_block_grouped(a, a_scale, offsets, b, b_scale, out=out, status=status)
        else:
            ops.gemm_fp8_block(a, a_scale, b, b_scale, bias=b_bias, out=out, status=status)
        torch.cuda.synchronize()
        return out, int(status)

    want, status = run()
    assert status == 0 and not bool(want.isnan().any()) and bool((want[end:] == 7).all())
    monkeypatch.setattr(lib, 'load', lambda: library)
    for limit in (PATIENT, 0, 500, 1500, 4000, 12000, PATIENT):
        assert library.set_wait_limit(limit) == 0
        got, status = run()
        unknown = got.isnan()
        assert torch.equal(torch.where(unknown, want, got), want)
        assert not bool(unknown[end:].any())
        if limit == PATIENT:
            assert status == 0 and not bool(unknown.any())
        if limit == 0:
            assert bool(unknown[:end].any())
        assert status in (0, 2) and (status == 2 or not bool(unknown.any()))
    assert library.set_wait_limit(PATIENT) == 0
