"""Libraries without the table of include/h3lm.h, or with a shorter one, serve what they have. CPU only: the libraries here are stubs."""
import ctypes as C
import subprocess

import pytest

from sycl_minimax_h3_amd import api as A


def stub(tmp_path, more):
    src, lib = tmp_path / "stub.c", tmp_path / "libstub.so"
    src.write_text("".join(f"int {n}(void) {{ return 7; }}\n" for n in {**A.REFERENCE, **A.ADDITIONS}) + more)
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(lib), str(src)], check=True)
    return A.Api(str(lib))


def test_a_library_without_the_table(tmp_path):
    api = stub(tmp_path, "")
    assert api.lib.h3s_wait(None) == 7 and api.lm is None
    for name, _ in A.LmApi._fields_[1:]:
        with pytest.raises(OSError, match=f"h3lm's {name} is missing"):
            getattr(api, "lm_" + name)(None, None)


def test_a_library_with_a_shorter_table(tmp_path):
    api = stub(tmp_path, "static int f(void) { return 5; }\nstruct { long long size; void* f[2]; } h3lm = {sizeof h3lm, {(void*) f, (void*) f}};\n")
    cache = C.byref(A.KvCache())
    assert api.lm_kv_write(None, cache, None, None, None, 0, None, 0, 0) == 5
    assert api.lm_kv_read(None, cache, None, None, None, 0, None, 0, 0) == 5
    with pytest.raises(OSError, match="h3lm's kv_attention is missing"):
        api.lm_kv_attention(None)
    with pytest.raises(OSError, match="h3lm's linear4 is missing"):
        api.lm_linear4(None)


def test_this_library_has_all(tmp_path):
    api = A.load()
    assert api.lm.size >= C.sizeof(A.LmApi)
    assert api.lm_linear4(None, None, 9, 1, 1, None, 1, None, None, 0, 32, None, None, 0) == -1 and "element type" in api.error()
