"""CPU: refusals of include/uh_model_ops.h that take no GPU: outputs over operands, sizes past what the grids and indexes reach."""
import os
from array import array

import pytest

pytest.importorskip('torch')


@pytest.fixture(scope='module')
def lib():
    from unsuperviseddeephomographyral2018_amd import _lib, build
    if not os.path.exists(build.MODEL_OPS_LIB) or not os.path.exists(build.TORCH_OPS_LIB):
        build.build_model_ops()
    return _lib.load_model_ops()


# addresses that are never dereferenced: validation fails first
def product(lib, a=1 << 20, b=1 << 21, out=1 << 22, M=4, N=4, K=64, ld=64, sa=64, sb=128, bias=None, w=None, nbytes=0):
    return lib.uhm_int8_matmul(a, ld, sa, b, ld, sb, bias, out, 0, M, N, K, 0, w, nbytes, None)


def layer(lib, x=1 << 20, b=1 << 21, out=1 << 22, M=4, N=4, K=64, ld=64, dtype=0, sb=128, bias=None, w=None, nbytes=0, flags=0):
    return lib.uhm_int8_linear(x, dtype, ld, b, ld, sb, bias, out, M, N, K, flags, w, nbytes, None)


def test_products_refuse_outputs_over_operands(lib):
    assert product(lib, out=1 << 20) == -8 and product(lib, out=(1 << 21) + 16) == -8 and product(lib, out=(1 << 20) - 32) == -8
    assert product(lib, bias=(1 << 22) + 60) == -8 and product(lib, sb=(1 << 22)) == -8
    assert layer(lib, out=(1 << 20) + 4 * 64 * 3, w=1 << 23, nbytes=1 << 20) == -8
    assert layer(lib, sb=(1 << 22) + 4, w=1 << 23, nbytes=1 << 20) == -8


def test_products_refuse_sizes_past_their_grids(lib):
    assert product(lib, N=(1 << 27) + 1) == -5 and product(lib, M=1 << 28) == -5 and product(lib, M=1 << 20, N=1 << 20) == -5
    far = (1 << 23) + 16
    assert product(lib, ld=far) == -5 and layer(lib, ld=far, w=1 << 23, nbytes=1 << 20) == -5
    assert lib.uhm_int8_matmul_workspace_bytes(1 << 20, 1 << 20, 64) == 0
    assert lib.uhm_quantize_rows(4096, 0, 1 << 31, 8192, 1 << 31, 64, 2, (1 << 31) - 1024, None) == -5


def test_layer_argument_errors(lib):
    assert layer(lib, x=None) == -1 and layer(lib, b=None) == -1 and layer(lib, sb=None) == -1 and layer(lib, out=None) == -1
    assert layer(lib, M=-1) == -2 and layer(lib, K=0) == -2 and layer(lib, ld=63) == -2
    assert layer(lib, dtype=3) == -7 and layer(lib, flags=2) == -10 and layer(lib, K=131072, ld=131072) == -5
    need = lib.uhm_int8_linear_workspace_bytes(4, 4, 64)
    assert need >= 4 * 128 + 16 and layer(lib) == -4 and layer(lib, w=1 << 23, nbytes=need - 1) == -4
    assert layer(lib, w=(1 << 23) + 4, nbytes=need) == -9 and layer(lib, x=(1 << 20) + 2, w=1 << 23, nbytes=need) == -9
    assert layer(lib, M=0) == 0 and layer(lib, N=0) == 0
    assert lib.uhm_int8_linear_workspace_bytes(1, 1000, 5000) == 0             # one token is quantised on the way


def test_norms_that_overlap_what_is_written_are_refused(lib):
    n, t = array('q', [256]), array('i', [0])
    src, dst = array('Q', [1 << 20]), array('Q', [1 << 21])
    at = lambda x: x.buffer_info()[0]
    big = lib.uhm_multi_workspace_bytes(1)

    def clip(use, norm):
        return lib.uhm_clip_by_global_norm(at(src), at(dst), at(n), at(t), 1, 1.0, use, norm, 1 << 23, big, None)
    assert clip((1 << 21) + 8, 64) == -8 and clip(None, (1 << 21) + 1020) == -8 and clip(None, (1 << 20) + 4) == -8

    m, v = array('Q', [1 << 24]), array('Q', [1 << 25])

    def adam(use, norm):
        return lib.uhm_adam_clip_update(at(dst), at(src), at(m), at(v), at(n), at(t), 1, 1e-3, 0.9, 0.999, 1e-8, 1, 1.0, 0, use, norm, 1 << 23, big, None)
    assert adam((1 << 24) + 8, 64) == -8 and adam(None, 1 << 25) == -8 and adam(None, 1 << 20) == -8


def test_quantiser_refuses_overlaps(lib):
    def q(x=1 << 20, out=1 << 21, scale=64, rows=4, K=60, q_ld=64):
        return lib.uhm_quantize_rows(x, 0, 60, out, q_ld, scale, rows, K, None)
    assert q(out=(1 << 20) + 16) == -8 and q(out=(1 << 20) - 16) == -8 and q(out=(1 << 20) + 944) == -8     # x ends at + 960
    assert q(scale=(1 << 20) + 8) == -8 and q(scale=(1 << 21) + 252) == -8 and q(scale=(1 << 21) - 4) == -8
