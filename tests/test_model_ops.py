"""CPU: the library of the operators around the regressor (include/uh_model_ops.h): it builds, exports what its header declares,
checks arguments before any HIP call, keeps its register budgets, and the Python entry points refuse what they cannot compute."""
import ctypes as C
import os
import re
from array import array

import pytest

torch = pytest.importorskip('torch')

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def declared_symbols():
    src = open(os.path.join(ROOT, 'include', 'uh_model_ops.h')).read()
    return sorted(set(re.findall(r'^UHM_API\s+[\w\s\*]+?\b(uhm_\w+)\s*\(', src, flags=re.M)))


@pytest.fixture(scope='module')
def lib():
    from unsuperviseddeephomographyral2018_amd import _lib, build
    if not os.path.exists(build.MODEL_OPS_LIB):
        build.build_model_ops()
    return _lib.load_model_ops()


def test_binding_covers_header_and_library(lib):
    from unsuperviseddeephomographyral2018_amd import _lib
    assert sorted(_lib.MODEL_OPS_SIGNATURES) == declared_symbols()
    assert lib.uhm_abi_version() == _lib.UHM_ABI_VERSION


def test_header_is_plain_c(tmp_path):
    import shutil
    import subprocess
    if shutil.which('gcc') is None:
        pytest.skip('no gcc')
    src = tmp_path / 'caller.c'
    src.write_text('#include "uh_hotpath.h"\n#include "uh_model_ops.h"\nint main(void) { return UHM_ABI_VERSION - 1; }\n')
    r = subprocess.run(['gcc', '-std=c99', '-Wall', '-Werror', '-pedantic', '-I', os.path.join(ROOT, 'include'), '-fsyntax-only',
                        str(src)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_no_kernel_spills_or_uses_scratch():
    from unsuperviseddeephomographyral2018_amd import build
    res = build.kernel_resources(sources=build.MODEL_OPS_SOURCES, headers=build.MODEL_OPS_HEADERS)
    assert {v['file'] for v in res.values()} == set(build.MODEL_OPS_SOURCES)
    for name, v in res.items():
        for f in ('vgpr_spill', 'sgpr_spill', 'scratch_bytes', 'lds_bytes'):
            assert v[f] is not None, (name, f)
        assert not (v['vgpr_spill'] or v['sgpr_spill'] or v['scratch_bytes'] or v['dynamic_stack']), (name, v)
        assert v['lds_bytes'] <= 160 * 1024, (name, v)


def test_packed_f32_instructions_are_off():
    from unsuperviseddeephomographyral2018_amd import build
    assert '-packed-fp32-ops' in build.FLAGS


# addresses that are never dereferenced: validation fails first
def _ptrs(*addr):
    return array('Q', addr)


def _at(a):
    return a.buffer_info()[0]


def test_list_argument_errors_without_gpu(lib):
    one, n4, f32 = _ptrs(4096), array('q', [4]), array('i', [0])
    ws, big = 1 << 20, lib.uhm_multi_workspace_bytes(1)
    norm = 64

    def call(p=one, n=n4, t=f32, count=1, out=norm, w=ws, nbytes=big):
        return lib.uhm_global_norm(_at(p) if p else None, _at(n) if n else None, _at(t) if t else None, count, out, w, nbytes, None)
    assert lib.uhm_multi_workspace_bytes(0) == 0 and lib.uhm_multi_workspace_bytes(1) >= 8
    assert lib.uhm_multi_workspace_bytes(1000) > big
    assert call(p=None) == -1 and call(n=None) == -1 and call(t=None) == -1 and call(out=None) == -1
    assert call(p=_ptrs(0)) == -1                                          # NULL tensor with elements
    assert call(count=0) == -2 and call(count=-3) == -2 and call(n=array('q', [-1])) == -2
    assert call(w=None) == -4 and call(nbytes=big - 1) == -4
    assert call(n=array('q', [1 << 60])) == -5 and call(n=array('q', [1 << 44])) == -5      # more chunks than 31 bits count
    assert call(t=array('i', [3])) == -7 and call(t=array('i', [-1])) == -7
    assert call(p=_ptrs(4098)) == -9 and call(p=_ptrs(4097), t=array('i', [1])) == -9 and call(w=ws + 4) == -9
    assert b'UHM_E_OVERLAP' in lib.uhm_error_string(-8) and lib.uhm_error_string(0) == b'ok'


def test_clip_argument_errors_without_gpu(lib):
    big = lib.uhm_multi_workspace_bytes(2)
    n, t = array('q', [256, 256]), array('i', [0, 0])

    def call(src, dst, clip=1.0, use=None, norm=64, w=1 << 20, nbytes=big, n=n, t=t):
        return lib.uhm_clip_by_global_norm(_at(src), _at(dst) if dst else None, _at(n), _at(t), 2, clip, use, norm, w, nbytes, None)
    a = _ptrs(4096, 8192)
    assert call(a, None) == -1 and call(a, _ptrs(0, 12288)) == -1
    for bad in (0.0, -1.0, float('nan')):
        assert call(a, a, clip=bad) == -10
    assert call(a, a, w=None) == -4
    assert call(_ptrs(4096, 4096), _ptrs(4096, 4096)) == -8                  # the same tensor twice, in place
    assert call(_ptrs(4096, 4096 + 512), _ptrs(4096, 4096 + 512)) == -8      # ... and two that overlap
    assert call(a, _ptrs(16384, 16384)) == -8                               # one output for two tensors
    assert call(a, _ptrs(8192, 16384)) == -8                                # the first output is the second input
    assert call(a, _ptrs(4096 + 16, 16384)) == -8                           # partly over its own input


def test_adam_argument_errors_without_gpu(lib):
    big = lib.uhm_multi_workspace_bytes(1)

    def call(p=4096, g=8192, m=12288, v=16384, n=256, t=0, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, step=1, clip=1.0, flags=0, w=1 << 20,
             nbytes=big):
        P, G, M, V, N, T = _ptrs(p), _ptrs(g), _ptrs(m), _ptrs(v), array('q', [n]), array('i', [t])
        return lib.uhm_adam_clip_update(_at(P), _at(G), _at(M), _at(V), _at(N), _at(T), 1, lr, b1, b2, eps,
                                        step, clip, flags, None, 64, w, nbytes, None)
    assert call(p=0) == -1 and call(g=0) == -1 and call(m=0) == -1 and call(v=0) == -1
    assert call(w=None) == -4 and call(nbytes=8) == -4
    assert call(p=4098) == -9 and call(m=12290) == -9 and call(g=8194) == -9
    for kw in (dict(clip=0.0), dict(clip=float('nan')), dict(step=0), dict(b1=1.0), dict(b2=-0.1), dict(eps=-1e-8), dict(lr=float('inf')),
               dict(lr=float('nan')), dict(flags=2), dict(eps=float('nan'))):
        assert call(**kw) == -10, kw
    assert call(m=4096) == -8 and call(v=12288) == -8 and call(g=4096) == -8 and call(p=8192 + 512) == -8


def test_int8_argument_errors_without_gpu(lib):
    def q(x=4096, t=0, x_ld=64, out=8192, q_ld=64, scale=64, rows=2, K=64):
        return lib.uhm_quantize_rows(x, t, x_ld, out, q_ld, scale, rows, K, None)
    assert q(rows=-1) == -2 and q(K=0) == -2 and q(x_ld=63) == -2 and q(q_ld=48) == -2
    assert q(t=5) == -7 and q(x=None) == -1 and q(out=None) == -1 and q(scale=None) == -1
    assert q(out=8193) == -9 and q(q_ld=72) == -9 and q(x=4098) == -9
    assert q(rows=1 << 40) == -5 and q(rows=0, x=None, out=None, scale=None) == 0

    def mm(a=4096, a_ld=64, sa=64, b=8192, b_ld=64, sb=64, bias=None, out=16384, t=0, M=2, N=2, K=64, flags=0, w=None, nbytes=0):
        return lib.uhm_int8_matmul(a, a_ld, sa, b, b_ld, sb, bias, out, t, M, N, K, flags, w, nbytes, None)
    assert mm(M=-1) == -2 and mm(N=-1) == -2 and mm(K=0) == -2 and mm(a_ld=48) == -2 and mm(b_ld=16) == -2
    assert mm(K=131072, a_ld=131072, b_ld=131072) == -5 and mm(M=1 << 40) == -5
    assert mm(t=3) == -7 and mm(flags=2) == -10
    assert mm(a=None) == -1 and mm(sb=None) == -1 and mm(out=None) == -1
    assert mm(a=4100) == -9 and mm(a_ld=72) == -9 and mm(bias=66) == -9 and mm(out=16386) == -9
    assert mm(M=0) == 0 and mm(N=0) == 0
    need = lib.uhm_int8_matmul_workspace_bytes(1, 1024, 32768)
    if need:
        assert mm(M=1, N=1024, K=32768, a_ld=32768, b_ld=32768, w=None) == -4
        assert mm(M=1, N=1024, K=32768, a_ld=32768, b_ld=32768, w=1 << 20, nbytes=need - 1) == -4
        assert mm(M=1, N=1024, K=32768, a_ld=32768, b_ld=32768, w=(1 << 20) + 4, nbytes=need) == -9
    assert lib.uhm_int8_matmul_workspace_bytes(0, 8, 8) == 0 and lib.uhm_int8_matmul_workspace_bytes(8, 8, 0) == 0


def test_entry_points_refuse_cpu_tensors_and_bad_arguments(lib):
    from unsuperviseddeephomographyral2018_amd import ops
    from unsuperviseddeephomographyral2018_amd._lib import UHError
    t = torch.ones(4)
    for f in (ops.global_norm, lambda x: ops.clip_by_global_norm(x, 1.0), lambda x: ops.clip_by_global_norm_(x, 1.0)):
        with pytest.raises(UHError, match='no CPU fallback'):
            f([t])
        with pytest.raises(UHError, match='at least one'):
            f([])
    for bad in (0.0, -1.0, float('nan')):
        with pytest.raises(UHError, match='clip_norm'):
            ops.clip_by_global_norm([t], bad)
        with pytest.raises(UHError, match='clip_norm'):
            ops.adam_clip_update_([t], [t], [t], [t], lr=1e-3, clip_norm=bad)
    with pytest.raises(UHError, match='no CPU fallback'):
        ops.adam_clip_update_([t], [t], [t], [t], lr=1e-3)
    q = torch.ones(2, 4, dtype=torch.int8)
    with pytest.raises(UHError, match='no CPU fallback'):
        ops.quantize_rows(torch.ones(2, 4))
    with pytest.raises(UHError, match='no CPU fallback'):
        ops.int8_linear(torch.ones(2, 4), q, torch.ones(2))
    with pytest.raises(UHError, match='no CPU fallback'):
        ops.int8_matmul(q, torch.ones(2), q, torch.ones(2))
    with pytest.raises(UHError, match='out_dtype'):
        ops.int8_matmul(q, torch.ones(2), q, torch.ones(2), out_dtype=torch.float64)
