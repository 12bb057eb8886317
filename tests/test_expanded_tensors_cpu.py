"""The C entry points refuse an x whose tokens are one place, before anything is launched."""
import ctypes

import pytest

import cabi
import cabi_ops

FAKE = 0x10000


@pytest.fixture(scope="module")
def lib():
    return cabi_ops.load()


def strides(name):
    return {f"{name}_batch_stride": 64, f"{name}_c_stride": 1, f"{name}_l_stride": 0}


def test_one_token_expanded_over_the_sequence(lib):
    common = dict(itype=cabi.BF16, wtype=cabi.F32, width=4, batch=2, dim=64, seqlen=32, x=FAKE, **strides("x"),
                  weight=FAKE, weight_c_stride=4, weight_width_stride=1)
    f = cabi.FwdParams(**common, out=FAKE, out_batch_stride=2048, out_c_stride=32, out_l_stride=1)
    codes = cabi_ops.Codes(codes=FAKE, scales=FAKE)
    assert lib.cc1d_fwd(ctypes.byref(f), None) == 5
    assert lib.cc1d_fwd_e4m3(ctypes.byref(f), ctypes.byref(codes), None) == 5
    assert lib.cc1d_checkpoint_e4m3(ctypes.byref(f), ctypes.byref(codes), None) == 5
    assert lib.cc1d_restore_e4m3(ctypes.byref(f), FAKE, ctypes.byref(codes), None) == 5
    b = cabi.BwdParams(**common, dout=FAKE, dout_batch_stride=2048, dout_c_stride=32, dout_l_stride=1,
                       dx=FAKE, dx_batch_stride=2048, dx_c_stride=32, dx_l_stride=1,
                       dweight=FAKE, dweight_c_stride=4, dweight_width_stride=1, workspace=FAKE, workspace_bytes=1 << 40)
    assert lib.cc1d_bwd(ctypes.byref(b), None) == 5
