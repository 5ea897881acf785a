"""The in-tree build: what a change compiles again, and the C ABI's structs as the bindings hold them."""
import ctypes
import os
import subprocess
import types

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize('changed,again', ((None, 0), ('openpvsg_amd/csrc/a.hip', 1), ('openpvsg_amd/csrc/a.h', 2), ('include/openpvsg_hip.h', 2)))
def test_a_changed_header_compiles_what_includes_it(tmp_path, monkeypatch, changed, again):
    """the public header too: kernels take its structs by value, so a library of old objects reads them wrongly"""
    from openpvsg_amd import build
    for f in ('openpvsg_amd/csrc/a.hip', 'openpvsg_amd/csrc/b.hip', 'openpvsg_amd/csrc/a.h', 'include/openpvsg_hip.h'):
        (tmp_path / f).parent.mkdir(parents=True, exist_ok=True)
        (tmp_path / f).write_text('')
        os.utime(tmp_path / f, (1000, 1000))
    lib = tmp_path / 'openpvsg_amd' / 'lib'
    (lib / 'obj').mkdir(parents=True)
    for f in ('obj/a.o', 'obj/b.o', build.LIBNAME):
        (lib / f).write_text('')
        os.utime(lib / f, (2000, 2000))
    if changed:
        os.utime(tmp_path / changed, (3000, 3000))
    ran = []

    def run(cmd, **kw):
        ran.append(cmd)
        open(cmd[cmd.index('-o') + 1], 'w').close()
        return types.SimpleNamespace(returncode=0, stdout='', stderr='')

    here = str(tmp_path / 'openpvsg_amd')
    for name, value in (('HERE', here), ('CSRC', here + '/csrc'), ('LIBDIR', str(lib)), ('OBJDIR', str(lib / 'obj')), ('INCLUDE', str(tmp_path / 'include'))):
        monkeypatch.setattr(build, name, value, raising=False)
    monkeypatch.setattr(build.subprocess, 'run', run)
    build.build_hip_lib(verbose=False)
    assert sum('-c' in c for c in ran) == again and len(ran) == again + bool(again)       # and the link


def test_the_pool_struct_is_laid_out_as_the_header_says(tmp_path):
    from openpvsg_amd import _lib
    names = [n for n, _ in _lib.KvPages._fields_]
    src = tmp_path / 'layout.c'
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "openpvsg_hip.h"\nint main(void) {\n  printf("%zu", sizeof(pvsg_kv_pages));\n'
                   + ''.join('  printf(" %%zu", offsetof(pvsg_kv_pages, %s));\n' % n for n in names) + '  return 0;\n}\n')
    subprocess.run(['gcc', '-I', os.path.join(ROOT, 'include'), str(src), '-o', str(tmp_path / 'layout')], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / 'layout')], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(_lib.KvPages)] + [getattr(_lib.KvPages, n).offset for n in names]
