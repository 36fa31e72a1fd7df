"""The build: the kernels' library needs hipcc alone; _tensor_list.so needs the installed torch's headers and is left out where
there is no torch.  The compilers are stand-ins that write what they were called with."""
import importlib.util
import stat

import pytest

HIPCC = '''#!/bin/sh
echo hipcc "$@" >> "$LOG"
[ -n "$FAIL" ] && exit 1
while [ $# -gt 0 ]; do [ "$1" = -o ] && echo built > "$2"; shift; done
'''


@pytest.fixture
def tree(tmp_path, monkeypatch):
    from pde_surrogate_amd import build
    src = tmp_path / 'csrc'
    src.mkdir()
    (src / 'a.hip').write_text('')
    (src / 'multi_tensor.hip').write_text('')
    (src / 'tensor_list.cpp').write_text('')
    for name, text in (('hipcc', HIPCC), ('g++', HIPCC.replace('hipcc', 'host').replace('$FAIL', '$FAIL_HOST'))):
        (tmp_path / name).write_text(text)
        (tmp_path / name).chmod(0o755 | stat.S_IXUSR)
    monkeypatch.setenv('HIPCC', str(tmp_path / 'hipcc'))
    monkeypatch.setenv('CXX', str(tmp_path / 'g++'))
    monkeypatch.setenv('LOG', str(tmp_path / 'log'))
    for k, v in (('HERE', tmp_path), ('CSRC', src), ('LIB', tmp_path / 'libpdes_hip.so'), ('HOST_SRC', src / 'tensor_list.cpp'), ('HOST_LIB', tmp_path / '_tensor_list.so')):
        monkeypatch.setattr(build, k, str(v))

    def calls():
        log = tmp_path / 'log'
        text = log.read_text().splitlines() if log.exists() else []
        log.unlink(missing_ok=True)
        return text
    return build, tmp_path, calls


def test_everything_is_built_once(tree):
    build, path, calls = tree
    assert build.needs_build()
    build.build(verbose=False)
    got = calls()
    assert sum(x.startswith('hipcc') and ' -c ' in x for x in got) == 2 and sum('libpdes_hip.so' in x for x in got) == 1
    assert sum(x.startswith('host') for x in got) == 1 and any('tensor_list.cpp' in x and '-ltorch_python' in x for x in got)
    assert not build.needs_build()
    build.build(verbose=False)
    assert not calls()
    build.build(force=True, verbose=False)
    assert len(calls()) == 4


def test_without_torch_the_kernels_are_built(tree, monkeypatch):
    build, path, calls = tree
    real = importlib.util.find_spec

    def none():
        raise ModuleNotFoundError("No module named 'torch'")
    monkeypatch.setattr(importlib.util, 'find_spec', lambda name, *a: None if name == 'torch' else real(name, *a))
    monkeypatch.setattr(build, 'host_command', none)                  # (which imports it)
    for force in (False, True):
        build.build(force=force, verbose=False)
        got = calls()
        assert len(got) == 3 and all(x.startswith('hipcc') for x in got)
        assert (path / 'libpdes_hip.so').exists() and not (path / '_tensor_list.so').exists()
        assert not build.needs_build()
    build.build(verbose=False)
    assert not calls()


@pytest.mark.parametrize('which', ['FAIL', 'FAIL_HOST'])
def test_a_compiler_that_fails_is_reported(tree, monkeypatch, which):
    build, path, calls = tree
    monkeypatch.setenv(which, '1')
    with pytest.raises(RuntimeError, match='failed on'):
        build.build(verbose=False)
    monkeypatch.delenv(which)
    build.build(verbose=False)
    assert (path / 'libpdes_hip.so').exists() and (path / '_tensor_list.so').exists() and not build.needs_build()
