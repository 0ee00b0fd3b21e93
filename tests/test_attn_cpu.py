"""The attention operators' C entries and their ctypes descriptions without a GPU: null handles, a device that
is not there, the layout of exn_kv_cache."""
import ctypes
import os
import subprocess

import pytest

import exn_b200 as E

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_null_handles_are_refused():
    L = E.lib()
    c = E.KvCache()
    n = ctypes.c_size_t()
    assert L.exn_attn_packed(None, 30, 8, 2, 1, None, None, 1, 1, None, 0, None, 0, None, 0, None, 0, 0.0, None) == 1
    assert b"exn_attn_packed: null handle" in L.exn_attn_last_error(None)
    assert L.exn_attn_cache_write(None, ctypes.byref(c), 30, None, 1, None, 0, None, 0, None) == 1
    assert L.exn_attn_cache_read(None, ctypes.byref(c), 30, None, 1, None, 0, None, 0, None) == 1
    assert L.exn_attn_cache_attend(None, ctypes.byref(c), 30, 8, None, 1, None, 0, None, 0, 0.0, None, 0, None) == 1
    assert L.exn_attn_cache_workspace(None, ctypes.byref(c), 8, 1, ctypes.byref(n)) == 1
    assert L.exn_attn_sync(None, None) == 1
    assert b"exn_attn_sync: null handle" in L.exn_attn_last_error(None)
    assert L.exn_attn_open(0, None) == 1
    L.exn_attn_close(None)
    L.exn_enc_cache_close(None)
    assert L.exn_enc_cache_length(None, 0) == -1
    assert L.exn_enc_cache_open(None, 1, 64, ctypes.byref(ctypes.c_void_p())) == 1
    assert L.exn_enc_extend(None, None, None, None, None, None) == 1
    assert L.exn_enc_cache_trim(None, None, 0, 0) == 1
    assert L.exn_enc_states_packed(None, None, 1, None, None, None) == 1
    assert L.exn_enc_states_packed_device(None, None, 1, None, None, 0, None, None) == 1


def test_a_device_that_is_not_there_is_refused():
    with pytest.raises(E.ExnError) as e:
        E.Attention(device=99)
    assert e.value.code == 2 and "no CUDA device 99" in str(e.value)


def test_kv_cache_has_the_headers_layout(tmp_path):
    src = tmp_path / "layout.c"
    names = [f[0] for f in E.KvCache._fields_]
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "exn_b200.h"\nint main(void) {\n'
                   + "".join('  printf("%%d ", (int)offsetof(exn_kv_cache, %s));\n' % n for n in names)
                   + '  printf("%d\\n", (int)sizeof(exn_kv_cache));\n  return 0;\n}\n')
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", exe, str(src)], check=True)
    got = [int(x) for x in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [getattr(E.KvCache, n).offset for n in names] + [ctypes.sizeof(E.KvCache)]


@pytest.mark.parametrize("status,code,words", [
    (0, 0, []), (4, 1, ["offsets", "left them out"]), (2, 6, ["gave up", "0x2"]), (6, 6, ["gave up", "out of range"]),
    (8, 6, ["gave up"])])
def test_a_kernel_that_gave_up_is_reported_before_anything_else(status, code, words):
    text = ctypes.create_string_buffer(512)
    assert E.lib().exn_test_attn_report(status, text, len(text)) == code
    assert all(w in text.value.decode() for w in words)
    assert (code == 1) == ("left them out" in text.value.decode())
