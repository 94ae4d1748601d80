"""Builds libasrn_hip.so (the C-ABI library of HIP kernels for gfx950) in-tree with hipcc, and _nodos.so (autograd nodes
in C++ over its entry points, host code only) with the C++ compiler against the installed PyTorch.

    python -m asrn_amd.build            # or asrn_amd.build.build()

Every source is compiled with packed-fp32 instructions disabled; ngram.hip and decode.hip also with -ffp-contract=off
because the n-gram keys must round each fp64 multiply and add separately, exactly as the reference does.
"""
import os
import shutil
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, 'csrc')
LIB = os.path.join(HERE, 'libasrn_hip.so')
NODOS = os.path.join(HERE, '_nodos.so')
SOURCES = ['errors.hip', 'graph.hip', 'bucket_sort.hip', 'ngram.hip', 'scan.hip', 'candidates.hip', 'decode.hip',
           'decode_produce.hip', 'gate.hip', 'context.hip', 'hidden.hip', 'reduce.hip', 'small_gemm.hip', 'gemm.hip', 'blocks.hip',
           'phi.hip', 'sampling.hip', 'block_step.hip', 'cross_entropy.hip', 'conv_window.hip',
           'layernorm.hip', 'clip.hip', 'embedding.hip', 'key_rows.hip',
           'token_logp.hip', 'preference.hip', 'policy.hip', 'eight_bits.hip']
ARCH = os.environ.get('ASRN_OFFLOAD_ARCH', 'gfx950')
INCLUDE = os.path.join(os.path.dirname(HERE), 'include')
COMMON = ['-O3', '-fPIC', '-std=c++17', f'--offload-arch={ARCH}', '-Xclang', '-target-feature', '-Xclang',
          '-packed-fp32-ops', '-Wno-unused-command-line-argument', f'-I{INCLUDE}']
PER_FILE = {'ngram.hip': ['-ffp-contract=off'], 'decode.hip': ['-ffp-contract=off']}


def hipcc():
    for cand in (shutil.which('hipcc'), '/opt/rocm/bin/hipcc'):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError('hipcc not found: the ASRN HIP library needs ROCm')


def orden_nodos(salida):
    """The command that compiles csrc/nodos.cpp into `salida`."""
    import sysconfig

    import torch
    raiz = os.path.dirname(torch.__file__)
    rocm = os.path.dirname(os.path.dirname(os.path.realpath(hipcc())))
    return [os.environ.get('CXX') or shutil.which('g++') or os.path.join(rocm, 'llvm', 'bin', 'clang++'),
            '-O2', '-std=c++17', '-shared', '-fPIC', '-fvisibility=hidden', '-D__HIP_PLATFORM_AMD__=1', '-DUSE_ROCM=1',
            f'-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}', f'-I{INCLUDE}',
            f"-I{os.path.join(raiz, 'include')}", f"-I{os.path.join(raiz, 'include', 'torch', 'csrc', 'api', 'include')}",
            f"-I{os.path.join(rocm, 'include')}", f"-I{sysconfig.get_paths()['include']}", os.path.join(CSRC, 'nodos.cpp'),
            '-o', salida, f"-L{os.path.join(raiz, 'lib')}", '-ltorch', '-ltorch_cpu', '-lc10', '-lc10_hip', '-ltorch_hip',
            '-ltorch_python']


def _colocar(hecho, sitio):
    shutil.copyfile(hecho, sitio + '.tmp')
    os.replace(sitio + '.tmp', sitio)


def _salida(cmd):
    return subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)


def build(verbose=False, jobs=None):
    """Compiles every source (in parallel), links the shared library and places it and the nodes atomically. Raises on any
    error. The library needs hipcc alone: it is placed also where the nodes cannot be compiled (PyTorch's, Python's or
    HIP's C++ headers missing), and the error says so."""
    cc = hipcc()
    with tempfile.TemporaryDirectory(prefix='asrn_build_') as tmp:
        tmp_nodos = os.path.join(tmp, '_nodos.so')
        try:
            nodos, error_nodos = _salida(orden_nodos(tmp_nodos)), None
        except (ImportError, OSError) as e:
            nodos, error_nodos = None, str(e)
        procs = []
        objs = []
        for src in SOURCES:
            obj = os.path.join(tmp, src.replace('.hip', '.o'))
            cmd = [cc, *COMMON, *PER_FILE.get(src, []), '-c', os.path.join(CSRC, src), '-o', obj]
            if verbose:
                print(' '.join(cmd), flush=True)
            procs.append((src, _salida(cmd)))
            objs.append(obj)
        errors = []
        for src, p in procs:
            out, _ = p.communicate()
            if p.returncode != 0:
                errors.append(f'--- {src} ---\n{out}')
            elif verbose and out.strip():
                print(out)
        if nodos is not None:
            out, _ = nodos.communicate()
            if nodos.returncode != 0:
                error_nodos = out
            elif verbose and out.strip():
                print(out)
        if errors:
            raise RuntimeError('hipcc failed:\n' + '\n'.join(errors))
        tmp_lib = os.path.join(tmp, 'libasrn_hip.so')
        cmd = [cc, '-shared', '-fPIC', f'--offload-arch={ARCH}', *objs, '-o', tmp_lib]
        r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
        if r.returncode != 0:
            raise RuntimeError('link failed:\n' + r.stdout)
        _colocar(tmp_lib, LIB)
        if error_nodos is not None:
            if os.path.exists(NODOS):         # nodes of another build may call this library by other signatures
                os.remove(NODOS)
            raise RuntimeError(f'{LIB} is built; the autograd nodes are not (csrc/nodos.cpp):\n{error_nodos}')
        _colocar(tmp_nodos, NODOS)
    return LIB


if __name__ == '__main__':
    print(build(verbose='-v' in sys.argv))
