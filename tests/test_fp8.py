"""CPU tests of the 8-bit cache's C ABI (include/clove_fp8.h): bindings,
refusals that need no device, and the scale and rounding rules against
torch's own e4m3 conversion."""
import ctypes as C
import re

import pytest
import torch

from clove_b200 import _lib
from conftest import ROOT, cuda_ok
from fp8_reference import round_e4m3, scale_for


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        from clove_b200 import build
        build.build()
    return _lib.load()


def test_bindings_cover_header():
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "clove_fp8.h").read_text(), flags=re.S)
    assert set(re.findall(r"\b(clove_\w+)\s*\(", text)) == set(_lib.FP8_SIGNATURES)


@pytest.mark.parametrize("nb,bs,h,d,rc", [(4, 4, 1, 64, -2), (4, 12, 1, 64, -2), (4, 512, 1, 64, -2), (4, 16, 1, 96, -2),
                                          (0, 16, 1, 64, -1), (4, 16, 0, 64, -1), (1 << 28, 16, 1, 64, -1),
                                          (1 << 24, 64, 4, 64, -1)])
def test_pool_shapes_refused(lib, nb, bs, h, d, rc):
    out = C.c_void_p(1)
    assert lib.clove_fp8_pool_create(0, nb, bs, h, d, 0, C.byref(out)) == rc
    assert not out.value and _lib.last_error()
    out = C.c_void_p(1)
    assert lib.clove_fp8_pool_wrap(0, 4096, 4096, None, nb, bs, h, d, C.byref(out)) == rc
    assert not out.value


def test_misaligned_and_null_storage_refused(lib):
    out = C.c_void_p()
    assert lib.clove_fp8_pool_wrap(0, 4096 + 64, 4096, None, 4, 16, 1, 64, C.byref(out)) == -1
    assert lib.clove_fp8_pool_wrap(0, 4096, 4096 + 4, None, 4, 16, 1, 64, C.byref(out)) == -1
    assert lib.clove_fp8_pool_wrap(0, 4096, 4096, 4104, 4, 16, 1, 64, C.byref(out)) == -1
    assert lib.clove_fp8_pool_wrap(0, None, 4096, None, 4, 16, 1, 64, C.byref(out)) == -1
    assert lib.clove_fp8_pool_wrap(0, 4096, None, None, 4, 16, 1, 64, C.byref(out)) == -1
    assert lib.clove_fp8_pool_create(0, 4, 16, 1, 64, 0, None) == -1


@pytest.mark.skipif(cuda_ok(), reason="checks the no-device path")
def test_no_device_reported(lib):
    out = C.c_void_p()
    assert lib.clove_fp8_pool_create(0, 4, 16, 1, 64, 0, C.byref(out)) == -7


def test_null_pool_refused(lib):
    assert lib.clove_fp8_pool_destroy(None) == 0
    assert lib.clove_fp8_pool_info(None, None) == -1
    assert lib.clove_fp8_pool_status(None, None, None) == -1
    assert lib.clove_fp8_append_workspace_size(None, 5) == 0
    assert lib.clove_fp8_append(None, 0, None, None, None, 1, None, 0, None) == -1
    assert lib.clove_fp8_gather(None, None, 1, None, 1, 1, None, None, None) == -1
    assert lib.clove_fp8_decode_workspace_size(None, 1, 1, 1, 0) == 0
    assert lib.clove_fp8_decode(None, 0, None, None, None, 1, None, 1, None, 1, 1.0, 1, None, None, None, 0, None) == -1
    assert lib.clove_fp8_evict_workspace_size(None, 1, 1, 1) == 0
    assert lib.clove_fp8_evict(None, None, 1, None, 1, 1, None, 1, 1, 0, None, None, None, 0, None) == -1
    assert lib.clove_fp8_copy_blocks(None, None, None, 1, None) == -1


def test_pool_needs_a_cuda_device():
    from clove_b200 import Fp8KVPool
    with pytest.raises(ValueError):
        Fp8KVPool(4, 16, 1, 64, device="cpu")


def test_backend_refuses_the_16_bit_only_calls():
    from clove_b200.backend import CudaBackend
    from clove_b200.fp8 import Fp8KVPool
    with pytest.raises(TypeError):
        CudaBackend._pool(Fp8KVPool.__new__(Fp8KVPool))


def test_reference_rounding_is_e4m3():
    x = torch.cat([torch.linspace(-500, 500, 20011), torch.linspace(-0.04, 0.04, 8009),
                   torch.tensor([448.0, 464.0, 1e9, 2.0 ** -10, 3 * 2.0 ** -11, 0.0])])
    want = x.clamp(-448, 448).to(torch.float8_e4m3fn).double()
    assert torch.equal(round_e4m3(x.double()), want)


@pytest.mark.parametrize("amax,e", [(448.0, 0), (448.1, 1), (449.0, 1), (224.0, -1), (1.75, -8), (1.0, -8), (1.76, -7),
                                    (0.0, -126), (1e-45, -126), (3.4e38, 120)])
def test_reference_scale(amax, e):
    assert scale_for(amax) == 2.0 ** e
