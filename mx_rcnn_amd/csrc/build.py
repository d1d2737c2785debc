"""In-tree build of the gfx950 extension ``mx_rcnn_amd/_C*.so``.

Explicit hipcc pipeline (no hipify, no JIT cache): every ``hip/*.hip`` is compiled with
``hipcc --offload-arch=gfx950`` into a PIC object, ``bindings.cpp`` (host-only glue)
with the host compiler against the PyTorch headers, and everything is linked into one
shared object next to the package so it travels with the repo snapshot to the GPU box.
Incremental: an object is kept only while what it was made from -- compile command, compiler, source and in-tree headers,
by content -- is unchanged (``<object>.made``), so a changed flag or an older file checked out over a newer one rebuilds.

Usage: ``python -m mx_rcnn_amd.csrc.build [--force] [--jobs N] [--debug]``
"""
import argparse
import glob
import hashlib
import os
import re
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(HERE)
BUILD = os.path.join(HERE, '_build')
ROCM = os.environ.get('ROCM_PATH', '/opt/rocm')
ARCH = os.environ.get('MXR_OFFLOAD_ARCH', 'gfx950')


def _torch_paths():
    import torch
    root = os.path.dirname(torch.__file__)
    inc = [os.path.join(root, 'include'), os.path.join(root, 'include', 'torch', 'csrc', 'api', 'include')]
    return root, inc, os.path.join(root, 'lib'), int(torch._C._GLIBCXX_USE_CXX11_ABI)


def ext_path():
    """The in-tree extension, or MXR_EXT_OUT when set (a staging path: link elsewhere while the
    in-tree .so is in use, then copy it in)."""
    if os.environ.get('MXR_EXT_OUT'):
        return os.environ['MXR_EXT_OUT']
    suffix = sysconfig.get_config_var('EXT_SUFFIX') or '.so'
    return os.path.join(PKG, '_C' + suffix)


def _made_from(parts, files):
    """Digest of texts and of files' contents."""
    h = hashlib.sha256()
    for p in parts:
        h.update(p.encode() + b'\0')
    for f in files:
        with open(f, 'rb') as fh:
            h.update(hashlib.sha256(fh.read()).digest())
    return h.hexdigest()


def _record(target):
    """What ``target`` was made from, or None."""
    try:
        with open(target + '.made') as f:
            return f.read()
    except OSError:
        return None


def _forget(target):
    if os.path.exists(target + '.made'):
        os.remove(target + '.made')


def _remember(target, digest):
    with open(target + '.made', 'w') as f:
        f.write(digest)


def _run(cmd):
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode != 0:
        raise RuntimeError('build step failed:\n%s\n%s' % (' '.join(cmd), r.stdout))
    return r.stdout


_INC = re.compile(r'^\s*#\s*include\s+"([^"]+)"', re.M)


def _local_deps(src, seen=None):
    """The in-tree headers ``src`` includes, transitively (quoted includes resolved next to the
    including file, then in csrc/ and csrc/hip/): an object rebuilds only when one of ITS headers
    changes (a conv-body edit does not rebuild every kernel file)."""
    seen = set() if seen is None else seen
    try:
        text = open(src).read()
    except OSError:
        return seen
    for name in _INC.findall(text):
        for d in (os.path.dirname(src), HERE, os.path.join(HERE, 'hip')):
            path = os.path.normpath(os.path.join(d, name))
            if os.path.exists(path):
                if path not in seen:
                    seen.add(path)
                    _local_deps(path, seen)
                break
    return seen


def build(force=False, jobs=None, debug=False, verbose=False):
    os.makedirs(BUILD, exist_ok=True)
    troot, tinc, tlib, abi = _torch_paths()
    hipcc = os.path.join(ROCM, 'bin', 'hipcc')
    opt = ['-O0', '-g'] if debug else ['-O3']
    hip_flags = opt + ['--offload-arch=%s' % ARCH, '-fPIC', '-std=c++17', '-ffp-contract=off',
                       # no packed fp32 instructions: some of their forms have given wrong results on gfx950
                       '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops',
                       '-D_GLIBCXX_USE_CXX11_ABI=%d' % abi, '-I', HERE, '-I', os.path.join(HERE, 'hip')]
    if os.environ.get('MXR_SYNC_DEBUG'):
        hip_flags.append('-DMXR_SYNC_DEBUG=1')
    jobs_list = []  # (object, digest, command)
    objs = []

    def add(src, obj, versions, cmd):
        objs.append(obj)
        digest = _made_from(versions + cmd, [src] + sorted(_local_deps(src)))
        if force or not os.path.exists(obj) or _record(obj) != digest:
            jobs_list.append((obj, digest, cmd))

    hip_versions = [_run([hipcc, '--version'])]
    for src in sorted(glob.glob(os.path.join(HERE, 'hip', '*.hip'))):
        obj = os.path.join(BUILD, os.path.basename(src) + '.o')
        add(src, obj, hip_versions, [hipcc] + hip_flags + ['-c', src, '-o', obj])
    py_inc = sysconfig.get_paths()['include']
    glue = os.path.join(HERE, 'bindings.cpp')
    glue_obj = os.path.join(BUILD, 'bindings.o')
    cxx = os.environ.get('CXX', 'g++')
    flags = opt + ['-fPIC', '-std=c++17', '-D__HIP_PLATFORM_AMD__=1', '-DUSE_ROCM=1',
                   '-DTORCH_EXTENSION_NAME=_C', '-DTORCH_API_INCLUDE_EXTENSION_H',
                   '-D_GLIBCXX_USE_CXX11_ABI=%d' % abi, '-I', HERE, '-I', os.path.join(ROCM, 'include'),
                   '-I', py_inc] + sum([['-I', p] for p in tinc], []) + ['-w']
    import torch
    add(glue, glue_obj, [torch.__version__, _run([cxx, '--version'])], [cxx] + flags + ['-c', glue, '-o', glue_obj])

    def compile_one(job):
        obj, digest, cmd = job
        _forget(obj)  # (a step that fails or is killed leaves nothing that counts as made)
        out = _run(cmd)
        _remember(obj, digest)
        return out

    n = jobs or min(8, max(1, len(jobs_list)))
    with ThreadPoolExecutor(n) as ex:
        for out in ex.map(compile_one, jobs_list):
            if verbose and out.strip():
                print(out)
    target = ext_path()
    link = ['g++', '-shared', '-o', target] + objs + [
        '-L', tlib, '-Wl,-rpath,' + tlib, '-lc10', '-lc10_hip', '-ltorch', '-ltorch_cpu', '-ltorch_hip',
        '-ltorch_python', '-lamdhip64']
    made = os.path.join(BUILD, os.path.basename(target))  # (its record stays with the objects')
    digest = _made_from(link, objs)
    if force or jobs_list or not os.path.exists(target) or _record(made) != digest + _made_from([], [target]):
        _forget(made)
        _run(link)
        _remember(made, digest + _made_from([], [target]))
    return target


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument('--force', action='store_true')
    ap.add_argument('--jobs', type=int, default=None)
    ap.add_argument('--debug', action='store_true')
    ap.add_argument('-v', '--verbose', action='store_true')
    a = ap.parse_args()
    print(build(force=a.force, jobs=a.jobs, debug=a.debug, verbose=a.verbose))


if __name__ == '__main__':
    sys.exit(main())
