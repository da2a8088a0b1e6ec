"""Build the gfx950 C-ABI shared libraries IN-TREE: lib/libuh_hotpath.so (include/uh_hotpath.h) and lib/libuh_model_ops.so
(include/uh_model_ops.h).

hipcc cross-compiles without a GPU.  The built .so is git-ignored but travels to the GPU box with
the gpurun snapshot.  `-ffp-contract=off` is part of the numerics contract: the forward
kernels must round once per written operation, like the un-fused TF-CPU graph.
"""
import hashlib
import os
import shutil
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, 'csrc')
LIBDIR = os.path.join(HERE, 'lib')
LIB = os.path.join(LIBDIR, 'libuh_hotpath.so')
SOURCES = ['uh_dlt.hip', 'uh_warp.hip', 'uh_misc.hip', 'uh_patch.hip', 'uh_losses.hip', 'uh_inputs.hip', 'uh_tail.hip', 'uh_epilogue.hip']
HEADERS = ['uh_device.h', 'uh_host.h', os.path.join('..', '..', 'include', 'uh_hotpath.h')]
# the operators around the regressor are a library of their own: the hot path's fingerprint (its committed measurements carry
# it) does not change with them
MODEL_OPS_LIB = os.path.join(LIBDIR, 'libuh_model_ops.so')
MODEL_OPS_SOURCES = ['uhm_multi.hip', 'uhm_int8.hip']
MODEL_OPS_HEADERS = [os.path.join('..', '..', 'include', 'uh_model_ops.h')]
TORCH_OPS_LIB = os.path.join(LIBDIR, '_uhm_torch.so')
TORCH_OPS_SOURCES = ['uhm_torch.cpp']
# `-packed-fp32-ops`: no v_pk_{add,mul,fma}_f32 anywhere -- some of their forms have given wrong results now and then on gfx950.
# The scalar forms round the same, and every kernel keeps its register count (the warp and patch kernels lose 224 packed
# instructions, the others had none).  hipcc's host pass warns that it does not know the feature: harmless.
FLAGS = ['--offload-arch=gfx950', '-O3', '-std=c++17', '-ffp-contract=off', '-fno-slp-vectorize', '-fPIC', '-shared',
         '-fvisibility=hidden', '-Wall', '-Wno-unused-function', '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops']


def _fingerprint(files=None):
    h = hashlib.sha256(' '.join(FLAGS).encode())
    for f in SOURCES + HEADERS if files is None else files:
        with open(os.path.join(CSRC, f), 'rb') as fh:
            h.update(fh.read())
    return h.hexdigest()


def find_hipcc():
    for c in (os.environ.get('HIPCC'), shutil.which('hipcc'), '/opt/rocm/bin/hipcc'):
        if c and os.path.exists(c):
            return c
    raise RuntimeError('hipcc not found: cannot build libuh_hotpath.so')


def _build(lib, sources, headers, force, verbose, command=None):
    os.makedirs(LIBDIR, exist_ok=True)
    stamp = lib + '.sha256'
    fp = _fingerprint(sources + headers)
    if not force and os.path.exists(lib) and os.path.exists(stamp) and open(stamp).read().strip() == fp:
        return lib
    before, after = command() if command else ([find_hipcc()] + FLAGS, [])
    cmd = before + [os.path.join(CSRC, s) for s in sources] + after + ['-o', lib + '.tmp']
    if verbose:
        print(' '.join(cmd))
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError('%s failed:\n' % os.path.basename(cmd[0]) + res.stdout + res.stderr)
    os.replace(lib + '.tmp', lib)
    with open(stamp, 'w') as fh:
        fh.write(fp)
    return lib


def build_library(force=False, verbose=False):
    """Compile csrc/uh_*.hip -> lib/libuh_hotpath.so.  Returns the library path."""
    return _build(LIB, SOURCES, HEADERS, force, verbose)


def build_model_ops(force=False, verbose=False):
    """Compile csrc/uhm_*.hip -> lib/libuh_model_ops.so, and csrc/uhm_torch.cpp -> lib/_uhm_torch.so on top of it.  Returns the
    library path."""
    lib = _build(MODEL_OPS_LIB, MODEL_OPS_SOURCES, MODEL_OPS_HEADERS, force, verbose)
    _build(TORCH_OPS_LIB, TORCH_OPS_SOURCES, MODEL_OPS_HEADERS, force, verbose, torch_command)
    return lib


def torch_command():
    """The host compiler's command for a Python module on torch's and this package's libraries."""
    import sysconfig
    import torch
    base = os.path.dirname(torch.__file__)
    cxx = os.environ.get('CXX') or shutil.which('g++') or shutil.which('c++')
    if not cxx:
        raise RuntimeError('no C++ compiler: cannot build _uhm_torch.so')
    includes = [os.path.join(base, 'include'), os.path.join(base, 'include', 'torch', 'csrc', 'api', 'include'),
                os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(find_hipcc()))), 'include'), sysconfig.get_paths()['include']]
    return ([cxx, '-O2', '-std=c++17', '-fPIC', '-shared', '-fvisibility=hidden', '-D__HIP_PLATFORM_AMD__=1', '-DUSE_ROCM=1',
             '-D_GLIBCXX_USE_CXX11_ABI=%d' % torch._C._GLIBCXX_USE_CXX11_ABI] + ['-I' + i for i in includes],
            ['-L' + LIBDIR, '-luh_model_ops', '-L' + os.path.join(base, 'lib'), '-lc10', '-lc10_hip', '-ltorch_cpu', '-ltorch', '-ltorch_python',
             '-Wl,-rpath,$ORIGIN'])


def kernel_resources(force=False, sources=None, headers=None):
    """Register / LDS / scratch budget of EVERY kernel of the library, from the code-object metadata hipcc emits
    (`-S --cuda-device-only`: device assembly only, ~10 s for uh_warp.hip, the files in parallel), cached beside the library
    under the same source fingerprint.  -> {demangled kernel name: {'file', 'vgpr', 'agpr', 'sgpr', 'vgpr_spill', 'sgpr_spill',
    'scratch_bytes', 'lds_bytes', 'dynamic_stack', 'max_threads'}}.  tests/test_kernel_resources.py holds the budgets.
    sources / headers: those of another library (MODEL_OPS_SOURCES, MODEL_OPS_HEADERS), not cached."""
    import json
    import re
    import tempfile
    from concurrent.futures import ThreadPoolExecutor
    import yaml
    os.makedirs(LIBDIR, exist_ok=True)
    cache = os.path.join(LIBDIR, 'kernel_resources.json') if sources is None else None
    sources, headers = (SOURCES, HEADERS) if sources is None else (sources, headers)
    fp = _fingerprint(sources + headers)
    if cache and not force and os.path.exists(cache):
        try:
            with open(cache) as fh:
                c = json.load(fh)
            if c.get('fingerprint') == fp:
                return c['kernels']
        except Exception:
            pass
    dev_flags = [f for f in FLAGS if f not in ('-shared', '-fPIC')] + ['-S', '--cuda-device-only', '-Wno-unused-command-line-argument']
    hipcc = find_hipcc()
    out = {}
    with tempfile.TemporaryDirectory() as td:
        def one(src):
            asm = os.path.join(td, src + '.s')
            res = subprocess.run([hipcc] + dev_flags + [os.path.join(CSRC, src), '-o', asm], capture_output=True, text=True)
            if res.returncode != 0:
                raise RuntimeError('hipcc -S failed for %s:\n%s%s' % (src, res.stdout, res.stderr))
            with open(asm) as fh:
                text = fh.read()
            m = re.search(r'\.amdgpu_metadata\n---\n(.*?)\n\.\.\.\n', text, re.S)
            return src, (yaml.safe_load(m.group(1)).get('amdhsa.kernels', []) if m else [])
        with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
            per_file = list(ex.map(one, sources))
    names = [k['.name'] for _, ks in per_file for k in ks]
    filt = shutil.which('c++filt')
    dem = subprocess.run([filt] + names, capture_output=True, text=True).stdout.split('\n') if (filt and names) else names
    i = 0
    for src, ks in per_file:
        for k in ks:
            name = re.sub(r'\(.*$', '', dem[i]).replace('void ', '') or k['.name']
            i += 1
            # a key the toolchain did not emit is None (NOT 0): tests/test_kernel_resources.py must fail on it instead of reading
            # "no spills" out of a renamed metadata field
            out[name] = {'file': src, 'vgpr': k.get('.vgpr_count'), 'agpr': k.get('.agpr_count', 0), 'sgpr': k.get('.sgpr_count'),
                         'vgpr_spill': k.get('.vgpr_spill_count'), 'sgpr_spill': k.get('.sgpr_spill_count'),
                         'scratch_bytes': k.get('.private_segment_fixed_size'), 'lds_bytes': k.get('.group_segment_fixed_size'),
                         'dynamic_stack': bool(k.get('.uses_dynamic_stack', False)),
                         'max_threads': k.get('.max_flat_workgroup_size')}
    if cache is None:
        return out
    with open(cache, 'w') as fh:
        json.dump({'fingerprint': fp, 'kernels': out}, fh, indent=0, sort_keys=True)
    return out


if __name__ == '__main__':
    print(build_library(force=True, verbose=True))
    print(build_model_ops(force=True, verbose=True))
