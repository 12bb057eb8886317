"""ctypes mirrors of include/cc1d_gdr.h and include/cc1d_checkpoint.h."""
import ctypes
import re
import os

import cabi
from cabi import i32, i64, vp, sz

ROOT = cabi.ROOT
HEADERS = [os.path.join(ROOT, "include", h) for h in ("cc1d_gdr.h", "cc1d_checkpoint.h")]


def _s(name):
    return [(name, vp)] + [(f"{name}_{d}_stride", i64) for d in ("batch", "l", "h")]


class GdrParams(ctypes.Structure):
    _fields_ = ([("itype", i32), ("gtype", i32), ("btype", i32), ("scale", ctypes.c_float)] +
                [(n, i64) for n in ("batch", "seqlen", "nseq", "heads_k", "heads_v", "dim_k", "dim_v")] +
                _s("q") + _s("k") + _s("v") + _s("g") + _s("beta") + _s("out") +
                [("cu_seqlens", vp), ("state_indices", vp), ("has_initial_state", vp), ("state_rows", i64),
                 ("initial_states", vp), ("initial_states_batch_stride", i64), ("initial_states_h_stride", i64),
                 ("final_states", vp), ("final_states_batch_stride", i64), ("final_states_h_stride", i64),
                 ("workspace", vp), ("workspace_bytes", sz)])


class GdrBwdParams(ctypes.Structure):
    _fields_ = ([("fwd", GdrParams)] + _s("dout") +
                [("dfinal_states", vp), ("dq", vp), ("dk", vp), ("dv", vp), ("dg", vp), ("dbeta", vp), ("dinitial_states", vp),
                 ("workspace", vp), ("workspace_bytes", sz)])


class Codes(ctypes.Structure):
    _fields_ = [("codes", vp), ("scales", vp)]


BLOCKS = {"cc1d_gdr_params": GdrParams, "cc1d_gdr_bwd_params": GdrBwdParams, "cc1d_codes": Codes}


def declared_symbols():
    names = set()
    for h in HEADERS:
        text = re.sub(r"/\*.*?\*/", "", open(h).read(), flags=re.S)
        names |= set(re.findall(r"\b(cc1d_[a-z0-9_]+)\s*\(", text))
    return sorted(names)


def load():
    lib = cabi.load()
    P = ctypes.POINTER
    for name, args, res in (("cc1d_gdr_update", [P(GdrParams), vp], ctypes.c_int), ("cc1d_gdr_fwd", [P(GdrParams), vp], ctypes.c_int),
                            ("cc1d_gdr_fwd_workspace_bytes", [P(GdrParams)], sz), ("cc1d_gdr_bwd", [P(GdrBwdParams), vp], ctypes.c_int),
                            ("cc1d_gdr_bwd_workspace_bytes", [P(GdrBwdParams)], sz),
                            ("cc1d_checkpoint_e4m3", [P(cabi.FwdParams), P(Codes), vp], ctypes.c_int),
                            ("cc1d_restore_e4m3", [P(cabi.FwdParams), vp, P(Codes), vp], ctypes.c_int),
                            ("cc1d_fwd_e4m3", [P(cabi.FwdParams), P(Codes), vp], ctypes.c_int),
                            ("cc1d_bwd_e4m3_restore_bytes", [P(cabi.BwdParams)], sz),
                            ("cc1d_bwd_e4m3", [P(cabi.BwdParams), P(Codes), vp, vp], ctypes.c_int)):
        f = getattr(lib, name)
        f.argtypes, f.restype = args, res
    return lib
