"""The quantised cache's binding without a GPU: its argument structs are laid
out as the header's, and calls fail loudly."""
import ctypes
import os
import shutil
import struct
import subprocess

import pytest

from conftest import ROOT, cuda_ok
from chonklm_b200 import _lib, kv_cache

STRUCTS = {"ck_kv_store_args": (kv_cache._STORE, ["q", "k", "v", "q_out", "table", "seq", "pos", "q_norm", "k_norm", "inv_freq", "eps", "interleaved", "n"]),
           "ck_kv_load_args": (kv_cache._LOAD, ["k", "v", "table", "seq", "pos", "n"]),
           "ck_kv_attend_args": (kv_cache._ATTEND, ["q", "out", "table", "len", "seq", "n", "window", "scale"])}
# fields of a packed struct that begin a member of the C one
FIRST = {"ck_kv_store_args": [0, 5, 10, 15, 20, 23, 24, 25, 26, 27, 28, 29, 30], "ck_kv_load_args": [0, 5, 10, 13, 14, 15],
         "ck_kv_attend_args": [0, 5, 10, 13, 14, 15, 16, 17]}


@pytest.mark.skipif(not shutil.which("gcc"), reason="needs a C compiler")
def test_packed_structs_match_the_header(tmp_path):
    lines = "".join(f'printf("{s} %zu", sizeof({s}));' + "".join(f'printf(" %zu", offsetof({s}, {m}));' for m in ms) + 'printf("\\n");'
                    for s, (_, ms) in STRUCTS.items())
    src = tmp_path / "s.c"
    src.write_text(f'#include <stdio.h>\n#include "{os.path.join(ROOT, "include", "chonk_b200.h")}"\nint main(void) {{ {lines} return 0; }}')
    exe = str(tmp_path / "s")
    subprocess.check_call(["gcc", str(src), "-o", exe])
    for line in subprocess.check_output([exe], text=True).splitlines():
        name, size, *offsets = line.split()
        packed = STRUCTS[name][0]
        assert packed.size == int(size)
        fmt = packed.format
        codes = [c for c in fmt if c != "@"]
        for field, off in zip(FIRST[name], offsets):
            # the offset of field i: pack everything before it, with its own alignment at the end
            before = struct.calcsize("@" + "".join(codes[:field]) + "0" + codes[field])
            assert before == int(off), (name, field)


@pytest.mark.skipif(cuda_ok(), reason="checks the no-GPU failure path")
def test_fails_loudly_without_gpu():
    with pytest.raises(_lib.CkError):
        kv_cache.QuantKvCache(4, 2, 64, 4)


def test_geometry_is_checked_before_the_device():
    for args, word in [((4, 2, 80, 4), "head_dim"), ((5, 2, 64, 4), "heads"), ((4, 2, 64, 0), "blocks")]:
        with pytest.raises(_lib.CkError, match=word):
            kv_cache.QuantKvCache(*args)
    with pytest.raises(_lib.CkError, match="positions"):
        kv_cache.QuantKvCache(4, 2, 64, 4, block=8)
    with pytest.raises(_lib.CkError, match="bits"):
        kv_cache.QuantKvCache(4, 2, 64, 4, v_bits=2)


def test_null_arguments_are_refused():
    L = _lib.lib()
    for rc in (L.ck_kv_create(None, 0, None), L.ck_kv_store(None, None, None), L.ck_kv_load(None, None, None), L.ck_kv_attend(None, None, None),
               L.ck_kv_attend_prompt(None, None, None, 0, None), L.ck_kv_check(None, None), L.ck_kv_bytes(None, None)):
        assert rc == _lib.CK_EINVAL
    assert L.ck_kv_destroy(None) == _lib.CK_OK
    assert b"ck_kv" in L.ck_global_error()
    assert ctypes.sizeof(ctypes.c_void_p) == 8
