"""CPU: memory that a call of include/uh_model_ops.h writes overlaps nothing else of the call: refused before anything is enqueued."""
import os
from array import array

import pytest

pytest.importorskip('torch')

OVERLAP = -8
MB = 1 << 20


@pytest.fixture(scope='module')
def lib():
    from unsuperviseddeephomographyral2018_amd import _lib, build
    if not os.path.exists(build.MODEL_OPS_LIB):
        build.build_model_ops()
    return _lib.load_model_ops()


# addresses that are never dereferenced: validation fails first.  One argument at a time is moved over another.
def product(lib, M=64, N=1024, K=32768, a=64 * MB, sa=96 * MB, b=128 * MB, sb=192 * MB, bias=200 * MB, out=256 * MB, w=512 * MB, nbytes=None):
    if nbytes is None:
        nbytes = lib.uhm_int8_matmul_workspace_bytes(M, N, K)
    return lib.uhm_int8_matmul(a, K, sa, b, K, sb, bias, out, 0, M, N, K, 0, w, nbytes, None)


@pytest.mark.parametrize('M', [1, 2, 64, 3000])                            # each kernel, with and without a workspace
def test_products_refuse_an_output_over_the_tokens_scales(lib, M):
    assert product(lib, M=M, sa=256 * MB) == OVERLAP
    assert product(lib, M=M, sa=256 * MB + M * 1024 * 4 - 4) == OVERLAP
    assert product(lib, M=M, out=96 * MB + 4 * (M - 1)) == OVERLAP


def layer(lib, M=64, N=1024, K=32768, x=64 * MB, b=128 * MB, sb=192 * MB, bias=200 * MB, out=256 * MB, w=512 * MB, nbytes=None, dtype=0):
    if nbytes is None:
        nbytes = lib.uhm_int8_linear_workspace_bytes(M, N, K)
    return lib.uhm_int8_linear(x, dtype, K, b, K, sb, bias, out, M, N, K, 0, w, nbytes, None)


def over(begin, size, need):
    """Workspaces that end just inside a span, lie in it, and begin with its last bytes."""
    return [begin - need + 16, begin, begin + size // 32 * 16, begin + (size - 1) // 16 * 16]


def test_products_refuse_a_workspace_over_anything_else(lib):
    M, N, K = 64, 1024, 32768
    need = lib.uhm_int8_matmul_workspace_bytes(M, N, K)
    assert need > 0
    for begin, size in ((64 * MB, M * K), (96 * MB, 4 * M), (128 * MB, N * K), (192 * MB, 4 * N), (200 * MB, 4 * N), (256 * MB, 4 * M * N)):
        for w in over(begin, size, need):
            assert product(lib, w=w) == OVERLAP, (begin, w)
    assert product(lib, bias=None, w=256 * MB) == OVERLAP


def test_layers_refuse_a_workspace_over_anything_else(lib):
    M, N, K = 64, 1024, 32768
    for dtype, size in ((0, 4), (1, 2), (2, 2)):
        need = lib.uhm_int8_linear_workspace_bytes(M, N, K)
        for begin, length in ((64 * MB, M * K * size), (128 * MB, N * K), (192 * MB, 4 * N), (200 * MB, 4 * N), (256 * MB, size * M * N)):
            for w in over(begin, length, need):
                assert layer(lib, w=w, dtype=dtype) == OVERLAP, (begin, w)


def test_products_refuse_missing_workspaces(lib):
    need = lib.uhm_int8_matmul_workspace_bytes(64, 1024, 32768)
    assert need > 0
    assert product(lib, w=None) == -4 and product(lib, nbytes=need - 1) == -4 and product(lib, w=512 * MB + 4) == -9
    need = lib.uhm_int8_linear_workspace_bytes(64, 1024, 32768)
    assert layer(lib, w=None) == -4 and layer(lib, nbytes=need - 1) == -4 and layer(lib, w=512 * MB + 4) == -9


# ---- lists ------------------------------------------------------------------------------------------------------------------------
def address(values, kind='Q'):
    a = array(kind, values)
    return a.buffer_info()[0], a


def lists(count=2, n=1000, **at):
    """Pointers to `count` tensors of n f32 elements each, 1 MB apart from the given addresses on, with their lengths and types."""
    out = {k: address([base + i * MB for i in range(count)]) for k, base in at.items()}
    out['n'], out['t'] = address([n] * count, 'q'), address([0] * count, 'i')
    return out


def norm_of(lib, tensors=64 * MB, norm=32 * MB, w=512 * MB, count=2):
    l = lists(count, p=tensors)
    return lib.uhm_global_norm(l['p'][0], l['n'][0], l['t'][0], count, norm, w, lib.uhm_multi_workspace_bytes(count), None)


def clip(lib, tensors=64 * MB, out=128 * MB, norm=32 * MB, use=None, w=512 * MB, count=2):
    l = lists(count, p=tensors, o=out)
    return lib.uhm_clip_by_global_norm(l['p'][0], l['o'][0], l['n'][0], l['t'][0], count, 1.0, use, norm, w, lib.uhm_multi_workspace_bytes(count), None)


def adam(lib, p=64 * MB, g=128 * MB, m=192 * MB, v=256 * MB, norm=32 * MB, use=None, w=512 * MB, count=2):
    l = lists(count, p=p, g=g, m=m, v=v)
    return lib.uhm_adam_clip_update(l['p'][0], l['g'][0], l['m'][0], l['v'][0], l['n'][0], l['t'][0], count, 1e-3, 0.9, 0.999, 1e-8, 1, 1.0, 0, use,
                                    norm, w, lib.uhm_multi_workspace_bytes(count), None)


def list_workspaces(lib, tensors, count=2):
    need = lib.uhm_multi_workspace_bytes(count)
    return [w for base in tensors for w in (base + MB - need + 8, base + MB, base + MB + 2000, base + MB + 3992)]      # over the second tensor


def test_lists_refuse_a_workspace_over_their_tensors(lib):
    for w in list_workspaces(lib, [64 * MB]):
        assert norm_of(lib, w=w) == OVERLAP and clip(lib, w=w) == OVERLAP and adam(lib, w=w) == OVERLAP
        assert clip(lib, out=64 * MB, w=w) == OVERLAP                      # in place
    for w in list_workspaces(lib, [128 * MB]):
        assert clip(lib, w=w) == OVERLAP and adam(lib, w=w) == OVERLAP
    for w in list_workspaces(lib, [192 * MB, 256 * MB]):
        assert adam(lib, w=w) == OVERLAP


def test_lists_refuse_a_norm_in_their_workspace(lib):
    need = lib.uhm_multi_workspace_bytes(2)
    for call in (norm_of, clip, adam):
        for norm in (512 * MB, 512 * MB + 1000, 512 * MB + need - 4, 512 * MB - 2):
            assert call(lib, norm=norm) == OVERLAP, (call, norm)


def test_the_norm_is_not_written_over_a_tensor(lib):
    for norm in (64 * MB, 65 * MB + 3996):
        assert norm_of(lib, norm=norm) == OVERLAP
