"""What the products grouped by expert refuse. Arguments are looked at before anything reaches the device, so no GPU is needed."""
import pytest

import skl_amd
from skl_amd import U4Weights

P = 4096  # an address that is never followed


def refused(lib):
    return lib.skl_hip_last_error() == -2


@pytest.fixture()
def lib():
    lib = skl_amd.load()
    lib.skl_hip_last_error()
    lib.skl_hip_set_pointer_mode(1)
    yield lib
    lib.skl_hip_set_pointer_mode(0)
    lib.skl_hip_last_error()


BIG = (1 << 30) + 1


@pytest.mark.parametrize("change", [dict(groups=0), dict(groups=4097), dict(count=BIG), dict(offsets=None), dict(ids=None), dict(per_row=0)], ids=str)
def test_group_rows(lib, change):
    args = dict(count=4, ids=P, per_row=2, groups=3, offsets=P, order=P, rows=P, place=P)
    args.update(change)
    lib.skl_group_rows_gfx950(*args.values())
    assert refused(lib)


@pytest.mark.parametrize("change", [dict(groups=4097), dict(offsets=None), dict(m=BIG), dict(n=BIG), dict(k=BIG), dict(a_rows=BIG), dict(a=None), dict(b=None), dict(c=None), dict(rsc=15),
                                    dict(rows=P, a_rows=3, a=None)], ids=str)
@pytest.mark.parametrize("name", ("bf16_bf16rc_f32", "bf16_bf16rc_bf16", "f16_f16rc_f32", "f16_f16rc_f16"))
def test_grouped(lib, name, change):
    args = dict(groups=3, offsets=P, m=8, n=16, k=32, alpha=1.0, a=P, rsa=32, rows=None, a_rows=0, b=P, rsb=1, csb=32, gsb=512, beta=0.0, c=P, rsc=16)
    args.update(change)
    getattr(lib, f"skl_gemm_grouped_{name}_gfx950")(*args.values())
    assert refused(lib)


@pytest.mark.parametrize("change", [dict(groups=4097), dict(offsets=None), dict(m=BIG), dict(n=BIG), dict(total=BIG), dict(a_rows=BIG), dict(b_rows=BIG), dict(a=None), dict(b=None), dict(c=None),
                                    dict(rsc=15), dict(gsc=127), dict(rows_b=P, b_rows=3, b=None)], ids=str)
@pytest.mark.parametrize("name", ("bf16c_bf16_f32", "bf16c_bf16_bf16", "f16c_f16_f32", "f16c_f16_f16"))
def test_groupedk(lib, name, change):
    args = dict(groups=3, offsets=P, m=8, n=16, total=40, alpha=1.0, a=P, rsa=8, rows_a=None, a_rows=0, b=P, rsb=16, rows_b=None, b_rows=0, beta=0.0, c=P, rsc=16, gsc=128)
    args.update(change)
    getattr(lib, f"skl_gemm_groupedk_{name}_gfx950")(*args.values())
    assert refused(lib)


@pytest.mark.parametrize("change", [dict(groups=4097), dict(offsets=None), dict(m=BIG), dict(k=BIG), dict(a=None), dict(c=None), dict(rsc=15)], ids=str)
@pytest.mark.parametrize("name", ("bf16_u4c_f32", "bf16_u4c_bf16", "f16_u4c_f32", "f16_u4c_f16"))
def test_u4(lib, name, change):
    w = U4Weights(group_k=32, codes=P, ld=64, expert=1024, scales=P, zeros=None, ld_scales=2, expert_scales=32)
    args = dict(groups=3, offsets=P, m=8, n=16, k=64, alpha=1.0, a=P, rsa=64, rows=None, a_rows=0, w=w, beta=0.0, c=P, rsc=16)
    args.update(change)
    getattr(lib, f"skl_gemm_grouped_{name}_gfx950")(*args.values())
    assert refused(lib)


@pytest.mark.parametrize("change", [dict(group_k=0), dict(group_k=48), dict(codes=None), dict(scales=None), dict(ld=63), dict(ld=62), dict(expert=1023), dict(ld_scales=1)], ids=str)
def test_u4_weights(lib, change):
    members = dict(group_k=32, codes=P, ld=64, expert=1024, scales=P, zeros=P, ld_scales=2, expert_scales=32)
    members.update(change)
    lib.skl_gemm_grouped_bf16_u4c_f32_gfx950(3, P, 8, 16, 64, 1.0, P, 64, None, 0, U4Weights(**members), 0.0, P, 16)
    assert refused(lib)
    lib.skl_gemm_grouped_bf16_u4c_f32_gfx950(3, P, 8, 16, 64, 1.0, P, 64, None, 0, None, 0.0, P, 16)
    assert refused(lib)


def test_unknown_member():
    with pytest.raises(TypeError, match="skl_gfx950_u4_t has no member wrong"):
        U4Weights(wrong=1)


def test_nothing_to_do_is_no_error(lib):
    for m, n, groups in ((0, 16, 3), (8, 0, 3), (8, 16, 0)):
        lib.skl_gemm_grouped_bf16_bf16rc_f32_gfx950(groups, None, m, n, 32, 1.0, None, 32, None, 0, None, 1, 32, 512, 0.0, None, 16)
        lib.skl_gemm_groupedk_bf16c_bf16_f32_gfx950(groups, None, m, n, 32, 1.0, None, 32, None, 0, None, 1, None, 0, 0.0, None, 16, 128)
        lib.skl_gemm_grouped_bf16_u4c_f32_gfx950(groups, None, m, n, 32, 1.0, None, 32, None, 0, None, 0.0, None, 16)
    assert lib.skl_hip_last_error() == 0

