"""What the Python binding takes for an argument. Sizes of zero end a call before anything is looked at, so no GPU is needed."""
import ctypes

import numpy as np
import pytest

import skl_amd
from skl_amd import DeviceBuffer, Epilogue, MoeLayer


class Buffer(DeviceBuffer):
    """A buffer that is only an address."""

    def __init__(self):
        self.nbytes, self.ptr = 64, 4096

    def free(self):
        pass


REFUSED = (ctypes.ArgumentError, TypeError)


def gemm(lib, **change):
    """An MXFP4 product without rows; change: position by name."""
    names = "m n k alpha a lda sa lsa b ldb sb lsb beta c rsc csc".split()
    args = dict(zip(names, (0, 4, 4, 1.0, Buffer(), 4, Buffer(), 1, Buffer(), 4, Buffer(), 1, 0.0, Buffer(), 4, 1)), **change)
    lib.skl_gemm_mxf4e2m1r_mxf4e2m1c_f32rc_gfx950(*args.values())


def fused(lib, epilogue):
    b = Buffer()
    lib.skl_gemm_fused_i8rc_i8rc_i32rc_gfx950(0, 4, 4, 1, b, 4, 1, b, 4, 1, 0, b, 4, 1, epilogue)


def experts(lib, layer):
    b = Buffer()
    lib.skl_moe_bf16_mxf4e2m1_f32_gfx950(layer, 0, b, 4, 0.0, None, 0, b, 4)


def test_what_is_meant_is_taken():
    lib = skl_amd.load()
    gemm(lib)
    gemm(lib, a=np.zeros(4, np.uint8), b=4096, sa=None)
    fused(lib, Epilogue(bias=Buffer()))
    fused(lib, None)
    experts(lib, MoeLayer(hidden=32, inter=32, router=Buffer(), gate=np.zeros(4, np.uint8)))
    assert lib.skl_hip_last_error() == 0


@pytest.mark.parametrize("position", ("n", "k", "alpha", "lda", "lsb", "beta", "rsc"))
def test_a_buffer_is_no_number(position):
    for wrong in (Buffer(), MoeLayer(hidden=32), np.zeros(2)):
        with pytest.raises(REFUSED):
            gemm(skl_amd.load(), **{position: wrong})


def test_descriptors_are_of_their_own_kind():
    lib = skl_amd.load()
    for wrong in (4096, Buffer(), MoeLayer(hidden=32), np.zeros(64, np.uint8)):
        with pytest.raises(REFUSED):
            fused(lib, wrong)
    for wrong in (4096, Buffer(), Epilogue(), np.zeros(64, np.uint8)):
        with pytest.raises(REFUSED):
            experts(lib, wrong)


def test_the_number_of_arguments():
    with pytest.raises(TypeError, match="expected 9 arguments, got 8"):
        skl_amd.load().skl_moe_bf16_mxf4e2m1_f32_gfx950(None, 0, None, 4, 0.0, None, 0, None)


def test_every_argument_is_looked_at_once():
    """Also where some are addresses, others buffers, halves or descriptors: none is converted, found wanting and converted again."""
    lib, looked = skl_amd.load(), []

    class Counted(Buffer):
        @property
        def ptr(self):
            looked.append("buffer")
            return 4096

        @ptr.setter
        def ptr(self, value):
            pass

    class Half:
        def __float__(self):
            looked.append("half")
            return 1.5

    class CountedEpilogue(Epilogue):
        def as_struct(self):
            looked.append("epilogue")
            return super().as_struct()

    a = Counted()
    lib.skl_gemm_f16_f16_f16_gfx950(0, 4, 4, Half(), 4096, 4, a, 4, Half(), np.zeros(4, np.float16), 4)
    assert sorted(looked) == ["buffer", "half", "half"]
    looked.clear()
    lib.skl_gemm_fused_i8rc_i8rc_i32rc_gfx950(0, 4, 4, 1, a, 4, 1, 4096, 4, 1, 0, np.zeros(4, np.int32), 4, 1, CountedEpilogue())
    assert sorted(looked) == ["buffer", "epilogue"]
