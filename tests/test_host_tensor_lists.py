"""Lists of tensors that the optimizer's entry points refuse before any launch, through the C ABI."""
import ctypes as C

import pytest

from diffusion_model_amd import _lib


@pytest.mark.parametrize("count", [64, 88, 500])
def test_lists_of_more_chunks_than_32_bits_count(count):
    """2^36 elements are 2^25 chunks of an Adam step: 64 such tensors in a launch would wrap its count around."""
    buf = (C.c_char * 128)()
    at = C.addressof(buf) + -C.addressof(buf) % 64
    p, n = (C.c_void_p * count)(*[at] * count), (C.c_int64 * count)(*[1 << 36] * count)
    L = _lib.lib()
    scalars = (1e-3, 0.9, 0.999, 1e-8, 0.0, 1)
    assert L.ddpm_adam_step(count, p, p, p, p, n, *scalars, None) == -1
    assert L.ddpm_adam_step_clipped(count, p, p, p, p, n, *scalars, C.c_void_p(at), None) == -1
    assert b"chunks_fit" in L.ddpm_last_error()
