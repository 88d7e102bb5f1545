"""The in-tree build of the native libraries: what is compiled again, and with which flags."""
import importlib.util
import os
import stat

import pytest

import paddle


@pytest.fixture
def build(tmp_path, monkeypatch):
    """The build module over two sources and a compiler that writes its arguments to a log."""
    spec = importlib.util.spec_from_file_location('_pa_build', os.path.join(os.path.dirname(paddle.__file__), '_build.py'))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    csrc, log, cc = tmp_path / 'csrc', tmp_path / 'log', tmp_path / 'cc'
    csrc.mkdir()
    for name in ('a.hip', 'b.hip'):
        (csrc / name).write_text('')
    cc.write_text(f'#!/bin/sh\necho "$@" >> {log}\nwhile [ $# -gt 0 ]; do [ "$1" = -o ] && echo > "$2"; shift; done\n')
    cc.chmod(cc.stat().st_mode | stat.S_IXUSR)
    for k, v in dict(CSRC=csrc, LIB=tmp_path / 'lib', OBJ=tmp_path / 'lib' / 'obj', HIPCC=cc,
                     KERNEL_LIB=tmp_path / 'lib' / 'k.so').items():
        monkeypatch.setattr(mod, k, str(v))

    def compiled():
        log.write_text('')
        mod.build_kernels()
        lines = log.read_text().splitlines()
        return sorted(os.path.basename(w) for line in lines for w in line.split() if w.endswith('.hip')), \
            sum(' -shared ' in f' {line} ' for line in lines), lines
    return mod, compiled


def test_objects_follow_their_flags(build, monkeypatch):
    mod, compiled = build
    assert compiled()[:2] == (['a.hip', 'b.hip'], 1)
    assert compiled()[:2] == ([], 0)
    monkeypatch.setitem(mod.FILE_FLAGS, 'b.hip', ['-fextra'])
    names, links, lines = compiled()
    assert (names, links) == (['b.hip'], 1) and ' -fextra' in lines[0]
    assert compiled()[:2] == ([], 0)
    monkeypatch.setattr(mod, 'FLAGS', [*mod.FLAGS, '-fmore'])
    assert compiled()[:2] == (['a.hip', 'b.hip'], 1)
    monkeypatch.setattr(mod, 'ARCH', 'gfx942')
    assert compiled()[:2] == (['a.hip', 'b.hip'], 1)
    os.remove(os.path.join(mod.CSRC, 'a.hip'))
    assert compiled()[:2] == ([], 1)                        # a source that is gone is linked no more
    assert compiled()[:2] == ([], 0)


def test_a_failed_compile_is_not_taken_for_done(build, monkeypatch):
    mod, compiled = build
    compiled()
    good = mod.HIPCC
    monkeypatch.setattr(mod, 'FLAGS', [*mod.FLAGS, '-fmore'])
    monkeypatch.setattr(mod, 'HIPCC', '/bin/false')
    with pytest.raises(RuntimeError, match='build failed'):
        mod.build_kernels()
    monkeypatch.setattr(mod, 'HIPCC', good)
    assert compiled()[:2] == (['a.hip', 'b.hip'], 1)


def test_kernels_have_no_packed_fp32(build):
    _, compiled = build
    for line in compiled()[2]:
        assert ' -shared ' in line or '-Xclang -target-feature -Xclang -packed-fp32-ops' in line
