"""The C ABI of the delta rule and of the 8-bit checkpoint without a GPU: plain C headers, layouts, exports, and
every refusal with its status before CUDA is touched."""
import ctypes
import os
import shutil
import subprocess

import pytest

import cabi
import cabi_ops as ops

FAKE = 0x10000  # never dereferenced: validation fails first, or there is nothing to do


@pytest.fixture(scope="module")
def lib():
    import causal_conv1d_b200._build as b
    b.build_kernels()
    return ops.load()


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_headers_are_plain_c_and_match_the_mirrors(tmp_path):
    lines = ['#include <stdio.h>', '#include "cc1d_gdr.h"', '#include "cc1d_checkpoint.h"', "int main(void) {"]
    for cname, st in ops.BLOCKS.items():
        lines.append(f'    printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'    printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in st._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["    return 0;", "}"]) + "\n")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-pedantic", "-I", os.path.join(ops.ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    for cname, st in ops.BLOCKS.items():
        assert int(got[cname]) == ctypes.sizeof(st), cname
        for f, _ in st._fields_:
            assert int(got[f"{cname}.{f}"]) == getattr(st, f).offset, f"{cname}.{f}"


def test_exports(lib):
    names = ops.declared_symbols()
    assert len(names) == 10
    for n in names:
        assert hasattr(lib, n), n
    assert lib.cc1d_abi_version() >= 5
    assert "multiples of 8" in lib.cc1d_status_str(20).decode() and "multiple of the number of key heads" in lib.cc1d_status_str(21).decode()


def gdr(**kw):
    p = ops.GdrParams(itype=cabi.BF16, gtype=cabi.F32, btype=cabi.BF16, scale=1.0, batch=2, seqlen=70, heads_k=2, heads_v=4, dim_k=64, dim_v=32,
                      state_rows=2, final_states=FAKE, final_states_batch_stride=4 * 64 * 32, final_states_h_stride=64 * 32,
                      workspace=FAKE, workspace_bytes=1 << 40)
    for n, h, d in (("q", 2, 64), ("k", 2, 64), ("v", 4, 32), ("g", 4, 1), ("beta", 4, 1), ("out", 4, 32)):
        setattr(p, n, FAKE)
        setattr(p, n + "_batch_stride", 70 * h * d); setattr(p, n + "_l_stride", h * d); setattr(p, n + "_h_stride", d)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


COMMON = [(dict(itype=5), 2), (dict(gtype=-1), 2), (dict(btype=3), 2), (dict(batch=-1), 4), (dict(seqlen=-1), 4), (dict(dim_k=60), 20),
          (dict(dim_k=136), 20), (dict(dim_v=0), 20), (dict(heads_v=3), 21), (dict(heads_k=0), 21), (dict(heads_v=0), 21), (dict(q=0), 1), (dict(out=0), 1),
          (dict(beta=0), 1), (dict(g=FAKE + 2), 12), (dict(final_states=FAKE + 4), 12), (dict(final_states_batch_stride=6), 12),
          (dict(seqlen=1 << 31), 13)]


@pytest.mark.parametrize("kw,code", COMMON + [(dict(final_states=0), 1), (dict(v=FAKE + 1), 12)])
def test_update_refuses(lib, kw, code):
    assert lib.cc1d_gdr_update(ctypes.byref(gdr(**kw)), None) == code


@pytest.mark.parametrize("kw,code", COMMON + [(dict(k=FAKE + 2), 12), (dict(v_l_stride=132), 12), (dict(out_h_stride=33), 12), (dict(q_batch_stride=4), 12),
                                              (dict(nseq=3), 1), (dict(cu_seqlens=FAKE, nseq=2), 4), (dict(workspace=0), 11), (dict(workspace_bytes=64), 11),
                                              (dict(workspace=FAKE + 8), 11), (dict(initial_states=FAKE, initial_states_h_stride=2), 12)])
def test_forward_refuses(lib, kw, code):
    assert lib.cc1d_gdr_fwd(ctypes.byref(gdr(**kw)), None) == code


BWD = dict(dout=FAKE, dout_batch_stride=70 * 128, dout_l_stride=128, dout_h_stride=32, dq=FAKE, dk=FAKE, dv=FAKE, dg=FAKE, dbeta=FAKE,
           workspace=FAKE, workspace_bytes=1 << 40)


@pytest.mark.parametrize("kw,code", [(dict(dout=0), 1), (dict(dg=0), 1), (dict(dq=FAKE + 8), 12), (dict(dout_l_stride=130), 12), (dict(dbeta=FAKE + 1), 12),
                                     (dict(workspace=0), 11), (dict(workspace_bytes=1000), 11)])
def test_backward_refuses(lib, kw, code):
    p = ops.GdrBwdParams(fwd=gdr(), **{**BWD, **kw})
    assert lib.cc1d_gdr_bwd(ctypes.byref(p), None) == code


@pytest.mark.parametrize("kw,code", [c for c in COMMON if not {"out", "final_states", "final_states_batch_stride"} & set(c[0])])
def test_backward_refuses_a_bad_forward(lib, kw, code):
    p = ops.GdrBwdParams(fwd=gdr(**kw), **BWD)
    assert lib.cc1d_gdr_bwd(ctypes.byref(p), None) == code


def test_nothing_to_do_launches_nothing(lib):
    assert lib.cc1d_gdr_update(ctypes.byref(gdr(batch=0)), None) == 0
    assert lib.cc1d_gdr_update(ctypes.byref(gdr(seqlen=0)), None) == 0
    assert lib.cc1d_gdr_fwd(ctypes.byref(gdr(batch=0)), None) == 0
    assert lib.cc1d_gdr_fwd(ctypes.byref(gdr(seqlen=0, final_states=0)), None) == 0
    assert lib.cc1d_gdr_bwd(ctypes.byref(ops.GdrBwdParams(fwd=gdr(batch=0), **BWD)), None) == 0
    assert lib.cc1d_gdr_update(None, None) == lib.cc1d_gdr_fwd(None, None) == lib.cc1d_gdr_bwd(None, None) == 1
    assert lib.cc1d_gdr_fwd_workspace_bytes(None) == lib.cc1d_gdr_bwd_workspace_bytes(None) == 0
    assert lib.cc1d_gdr_fwd_workspace_bytes(ctypes.byref(gdr(dim_k=60))) == 0


def test_workspace_grows_with_the_chunks(lib):
    small, large = (lib.cc1d_gdr_fwd_workspace_bytes(ctypes.byref(gdr(seqlen=n))) for n in (64, 6400))
    assert 0 < small and 50 * small <= large
    # packed: every sequence may leave one chunk partly filled
    a = lib.cc1d_gdr_fwd_workspace_bytes(ctypes.byref(gdr(batch=1, cu_seqlens=FAKE, nseq=3)))
    b = lib.cc1d_gdr_fwd_workspace_bytes(ctypes.byref(gdr(batch=1, cu_seqlens=FAKE, nseq=40)))
    assert b > a
    assert lib.cc1d_gdr_bwd_workspace_bytes(ctypes.byref(ops.GdrBwdParams(fwd=gdr(), **BWD))) > 4 * lib.cc1d_gdr_fwd_workspace_bytes(ctypes.byref(gdr()))


def conv(**kw):
    p = cabi.FwdParams(itype=cabi.BF16, wtype=cabi.BF16, width=4, silu=1, batch=2, dim=64, seqlen=128, x=FAKE, x_batch_stride=64 * 128, x_c_stride=128, x_l_stride=1,
                       weight=FAKE, weight_c_stride=4, weight_width_stride=1, out=FAKE, out_batch_stride=64 * 128, out_c_stride=128, out_l_stride=1)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,codes,code", [(dict(itype=9), {}, 2), (dict(batch=-1), {}, 4), (dict(x_c_stride=3, x_l_stride=2), {}, 5), (dict(), dict(codes=0), 1),
                                           (dict(), dict(scales=0), 1), (dict(), dict(codes=FAKE + 8), 12), (dict(x=0), {}, 1), (dict(x=FAKE + 1), {}, 12)])
def test_checkpoint_refuses(lib, kw, codes, code):
    c = ops.Codes(**{**dict(codes=FAKE, scales=FAKE), **codes})
    p = conv(**kw)
    assert lib.cc1d_checkpoint_e4m3(ctypes.byref(p), ctypes.byref(c), None) == code
    assert lib.cc1d_restore_e4m3(ctypes.byref(p), p.x, ctypes.byref(c), None) == code
    assert lib.cc1d_fwd_e4m3(ctypes.byref(p), ctypes.byref(c), None) == code


def test_checkpointed_convolution_keeps_the_convolutions_checks(lib):
    c = ops.Codes(codes=FAKE, scales=FAKE)
    for kw, code in ((dict(width=5), 3), (dict(seq_idx=FAKE), 8), (dict(out=0), 1), (dict(dim=60, x_c_stride=1, x_l_stride=64), 6)):
        assert lib.cc1d_fwd_e4m3(ctypes.byref(conv(**kw)), ctypes.byref(c), None) == code
    assert lib.cc1d_fwd_e4m3(ctypes.byref(conv(batch=0)), ctypes.byref(c), None) == 0
    b = dict(itype=cabi.BF16, wtype=cabi.BF16, width=4, silu=1, batch=2, dim=64, seqlen=128, x_c_stride=128, x_l_stride=1, weight=FAKE, weight_c_stride=4, weight_width_stride=1,
             dout=FAKE, dout_batch_stride=64 * 128, dout_c_stride=128, dout_l_stride=1, dx=FAKE, dx_batch_stride=64 * 128, dx_c_stride=128, dx_l_stride=1, dweight=FAKE,
             dweight_c_stride=4, dweight_width_stride=1, workspace=FAKE, workspace_bytes=1 << 30)
    call = lambda codes=c, restored=0, **kw: lib.cc1d_bwd_e4m3(ctypes.byref(cabi.BwdParams(**{**b, **kw})), ctypes.byref(codes), restored, None)  # noqa: E731
    need = lambda **kw: lib.cc1d_bwd_e4m3_restore_bytes(ctypes.byref(cabi.BwdParams(**{**b, **kw})))  # noqa: E731
    assert need() == 0                                    # 16-bit, channel-first, a multiple of 16 long: read as they are
    assert need(seqlen=120) == 2 * 64 * 120 * 2 and need(itype=cabi.F32) == 2 * 64 * 128 * 4
    assert call(width=7) == 3 and call(dweight=0) == 1 and call(workspace=0) == 11
    assert call(ops.Codes(codes=0, scales=FAKE)) == 1 and call(ops.Codes(codes=FAKE + 4, scales=FAKE)) == 12
    assert call(itype=cabi.F32) == 11                     # needs room for x
    assert call(itype=cabi.F32, restored=FAKE + 16) == 12
    assert call(itype=cabi.F32, restored=FAKE, width=7) == 3 and call(itype=cabi.F32, restored=FAKE, dbias=FAKE) == 1
