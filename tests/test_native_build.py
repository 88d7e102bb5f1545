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


def test_custom_operators_have_no_packed_fp32(tmp_path, monkeypatch):
    """A user's own kernels get the flag too, by each of the ways to build them."""
    from paddle.utils import cpp_extension as X
    log, cc, src = tmp_path / 'log', tmp_path / 'cc', tmp_path / 'k.hip'
    cc.write_text(f'#!/bin/sh\necho "$@" >> {log}\nexec /opt/rocm/bin/hipcc "$@"\n')
    cc.chmod(cc.stat().st_mode | stat.S_IXUSR)
    src.write_text('#include <hip/hip_runtime.h>\n__global__ void k(float2* x) { x[threadIdx.x].x *= 2; x[threadIdx.x].y *= 3; }\n'
                   'extern "C" int answer() { return 42; }\n')
    monkeypatch.setenv('HIPCC', str(cc))
    lib = X.load_hip_library('t', [str(src)], extra_cflags=['-DA=1'], build_directory=str(tmp_path / 'b'))
    assert lib.answer() == 42
    args = log.read_text().split()
    at = args.index('-packed-fp32-ops')
    assert args[at - 3:at] == ['-Xclang', '-target-feature', '-Xclang'] and '-DA=1' in args
    seen = {}
    from torch.utils import cpp_extension as tce
    monkeypatch.setattr(tce, 'load', lambda **kw: seen.update(kw))
    X.load('t', [str(src)], extra_cuda_cflags=['-DB'], build_directory=str(tmp_path / 'c'))
    assert '-packed-fp32-ops' in seen['extra_cuda_cflags'] and '-DB' in seen['extra_cuda_cflags']
    monkeypatch.setattr(tce, 'CUDAExtension', lambda name, sources, *a, **kw: kw)
    for given in (None, ['-DC'], {'cxx': ['-DC']}, {'nvcc': ['-DC']}):
        got = X.CUDAExtension([str(src)], **({} if given is None else dict(extra_compile_args=given)))['extra_compile_args']
        assert '-packed-fp32-ops' in got['nvcc'] and '-packed-fp32-ops' not in got.get('cxx', [])
        if given is not None:
            assert all('-DC' in got[k] for k in (('cxx', 'nvcc') if isinstance(given, list) else given))
