"""Build libpdes_hip.so (all HIP kernels + the C ABI) in-tree with hipcc for gfx950, and _tensor_list.so (host code that reads
Python lists of tensors, against the installed torch's headers) with g++.  Where torch is not installed the kernels' library is
all that is built.

    python -m pde_surrogate_amd.build            # rebuild if any source is newer than the .so
    python -m pde_surrogate_amd.build --force

Both are git-ignored: the history stays source-only.
hipcc cross-compiles gfx950 without a GPU.
"""
import glob
import importlib.util
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, 'csrc')
LIB = os.path.join(HERE, 'libpdes_hip.so')
HOST_SRC = os.path.join(CSRC, 'tensor_list.cpp')
HOST_LIB = os.path.join(HERE, '_tensor_list.so')
FLAGS = ['--offload-arch=gfx950', '-O3', '-std=c++17', '-fPIC', '-shared', '-ffp-contract=fast',
         '-Wno-unused-result', '-munsafe-fp-atomics']
# added for one source: the list operators round every product and sum once (no contraction), and use no packed fp32
# instructions
FILE_FLAGS = {'multi_tensor.hip': ['-ffp-contract=off', '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops']}


def sources():
    return sorted(glob.glob(os.path.join(CSRC, '*.hip')))


def headers():
    return glob.glob(os.path.join(CSRC, '*.h')) + glob.glob(os.path.join(CSRC, '*.inc')) + glob.glob(os.path.join(os.path.dirname(HERE), 'include', '*.h'))


def has_torch():
    return importlib.util.find_spec('torch') is not None


def needs_host_build():
    return has_torch() and (not os.path.exists(HOST_LIB) or os.path.getmtime(HOST_SRC) > os.path.getmtime(HOST_LIB))


def needs_build():
    if not os.path.exists(LIB) or needs_host_build():
        return True
    t = os.path.getmtime(LIB)
    return any(os.path.getmtime(p) > t for p in sources() + headers())


def host_command():
    import sysconfig
    import torch
    from torch.utils.cpp_extension import include_paths, library_paths
    return ([os.environ.get('CXX', 'g++'), '-O2', '-std=c++17', '-fPIC', '-shared', '-fvisibility=hidden',
             f'-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}'] + ['-I' + d for d in include_paths()] +
            ['-I' + sysconfig.get_paths()['include'], HOST_SRC] + ['-L' + d for d in library_paths()] +
            ['-ltorch_python', '-ltorch_cpu', '-lc10', '-o', HOST_LIB])


def build(force=False, verbose=True):
    if not force and not needs_build():
        return LIB
    hipcc = os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')
    objs = []
    host = None
    if needs_host_build() or (force and has_torch()):
        host = subprocess.Popen(host_command(), stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    # one object per source, compiled in parallel, then linked: keeps rebuilds to seconds
    procs = []
    for src in sources():
        obj = os.path.join(CSRC, os.path.basename(src)[:-4] + '.o')
        objs.append(obj)
        if force or not os.path.exists(obj) or os.path.getmtime(obj) < max(
                [os.path.getmtime(src)] + [os.path.getmtime(h) for h in headers()]):
            cmd = [hipcc] + [f for f in FLAGS if f != '-shared'] + FILE_FLAGS.get(os.path.basename(src), []) + os.environ.get('PDES_EXTRA_FLAGS', '').split() + ['-c', src, '-o', obj]
            if verbose:
                print(' '.join(cmd), flush=True)
            procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
    failed = []
    for src, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            sys.stderr.write(out.decode())
            failed.append(f'hipcc failed on {src}')
    if host is not None:
        host_out, _ = host.communicate()
    if failed:
        raise RuntimeError('; '.join(failed))
    cmd = [hipcc, '--offload-arch=gfx950', '-shared', '-fPIC'] + objs + ['-o', LIB]
    if verbose:
        print(' '.join(cmd), flush=True)
    subprocess.check_call(cmd)
    if host is not None and host.returncode != 0:             # (the kernels' library is whole)
        sys.stderr.write(host_out.decode())
        raise RuntimeError(f'{os.environ.get("CXX", "g++")} failed on {HOST_SRC}')
    return LIB


if __name__ == '__main__':
    build(force='--force' in sys.argv)
    print(LIB)
