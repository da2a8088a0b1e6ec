"""GPU: the operators around the regressor at the sizes where their variants change: tiles and splits of the 8-bit products, segments of
the quantiser, lists that the caches hold and lists that they do not, shared allocations, lazily negated tensors."""
import math

import pytest

torch = pytest.importorskip('torch')

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
INF = float('inf')


@pytest.fixture(scope='module')
def dev():
    if not torch.cuda.is_available():
        pytest.skip('no HIP device')
    return torch.device('cuda:0')


@pytest.fixture(scope='module')
def ops(dev):
    from unsuperviseddeephomographyral2018_amd import ops
    return ops


@pytest.fixture(scope='module')
def UHError():
    from unsuperviseddeephomographyral2018_amd._lib import UHError
    return UHError


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def int_rows(dev, rows, K, seed):
    ld = -(-K // 128) * 128
    return torch.randint(-128, 128, (rows, ld), generator=gen(dev, seed), device=dev, dtype=torch.int8)[:, :K]


# 128 x 128 tiles: from 200 of them; 256 x 256 tiles: from 200; 64 x 64 split and not; rows and columns that end inside a tile; a tile of
# K that is whole, that ends after 1, 16, 17 and 127 bytes; fewer tiles of K than buffers
@pytest.mark.parametrize('M,N,K', [(2000, 1700, 129), (1921, 1921, 640), (1900, 1800, 16), (3700, 3650, 127), (3713, 3841, 272), (3600, 3900, 385),
                                   (3841, 3600, 1024), (64, 64, 5000), (65, 700, 8192), (500, 60, 2049), (960, 1000, 1100), (33, 129, 4096), (32, 4000, 1153),
                                   (3, 3, 3), (3, 1000, 32768), (4, 8, 1024), (2, 1000, 32769), (2, 600, 5000), (1, 600, 70000), (1, 1, 131071)])
def test_int8_sums_of_every_variant(ops, dev, M, N, K):
    a, b = int_rows(dev, M, K, 1 + M), int_rows(dev, N, K, 2 + N)
    want = (a.double() @ b.double().t().contiguous()).float()              # sums below 2^31: exact in 64 bits, one rounding
    ones = lambda n: torch.ones(n, device=dev)
    assert torch.equal(ops.int8_matmul(a, ones(M), b, ones(N)), want)
    sa, sb = torch.rand(M, generator=gen(dev, 3), device=dev) + 0.5, torch.rand(N, generator=gen(dev, 4), device=dev) + 0.5
    for bias in (None, torch.randn(N, generator=gen(dev, 5), device=dev) * 1000):
        # the epilogue's roundings, one by one
        full = (want * sa[:, None]) * sb
        full = full if bias is None else full + bias
        assert torch.equal(ops.int8_matmul(a, sa, b, sb, bias=bias), full)
        for dtype in (torch.bfloat16, torch.float16):
            assert torch.equal(ops.int8_matmul(a, sa, b, sb, bias=bias, relu=True, out_dtype=dtype), full.clamp(min=0).to(dtype))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize('rows,K,offset', [(2, 2048, 0), (2, 2052, 0), (3, 8192, 4), (3, 8196, 1), (2, 32768, 0), (2, 32772, 0), (1, 131071, 0), (1, 70004, 2),
                                           (2, 200001, 0), (5, 4, 0), (5, 8, 3), (1, 100, 1)])
def test_quantiser_segments(ops, dev, rows, K, offset, dtype):
    base = torch.randn(rows * K + offset, generator=gen(dev, K), device=dev).to(dtype)
    x = base[offset:].view(rows, K)
    for at in (0, K - 1, K // 2):                                          # the maximum wherever it may be
        y = x.clone() if offset == 0 else torch.cat([base[:offset], x.reshape(-1)])[offset:].view(rows, K)
        y[:, at] = 9.0
        q, s = ops.quantize_rows(y)
        inverse = torch.tensor(127.0 / 9.0, dtype=torch.float64).float().double().item()
        assert torch.equal(q, torch.round(y.double() * inverse).to(torch.int8)) and bool((s == torch.tensor(9.0 / 127.0, dtype=torch.float64).float().item()).all())


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize('N,K,offset', [(1, 1, 0), (7, 4, 0), (600, 4096, 0), (1024, 4100, 0), (1030, 4097, 0), (500, 16384, 1), (1100, 16388, 0), (3, 32768, 0),
                                        (1025, 32772, 4), (40, 70001, 0), (520, 100000, 0), (9, 131071, 0)])
def test_layer_for_one_token(ops, dev, N, K, offset, dtype):
    """One float row: the fused kernel gives the bits of quantising first."""
    x = torch.randn(K + offset, generator=gen(dev, N), device=dev).to(dtype)[offset:]
    w, ws = ops.quantize_rows(torch.randn(N, K, generator=gen(dev, K), device=dev) if N * K < 4e7 else torch.randn(N, K, device=dev))
    q, s = ops.quantize_rows(x)
    want = ops.int8_matmul(q[None], s[None], w, ws, out_dtype=dtype)[0]
    sums = (q.double()[None] @ w.double().t().contiguous())[0].float()
    assert torch.equal(want, ((sums * s) * ws).to(dtype))
    assert torch.equal(ops.int8_linear(x, w, ws), want)
    x[K // 3] = INF
    assert bool(ops.int8_linear(x, w, ws, relu=True).isnan().all())
    assert bool((ops.int8_linear(torch.zeros_like(x), w, ws) == 0).all())


def norm64(ts):
    return math.sqrt(math.fsum(float((t.double() ** 2).sum()) for t in ts))


@pytest.mark.parametrize('scale', [1.0, 1e-30], ids=['ordinary', 'small'])
@pytest.mark.parametrize('offset', [0, 1])
def test_lists_past_the_caches(ops, dev, offset, scale):
    """More than 192 MB moved: chunks in the other order, loads and stores past the caches."""
    sizes = [12_000_001, 3, 5_000_000, 0, 4097]
    make = lambda k: [(torch.randn(n + offset, generator=gen(dev, 10 * k + i), device=dev) * scale)[offset:] for i, n in enumerate(sizes)]
    ts = make(1)
    n = norm64(ts)
    out, told = ops.clip_by_global_norm(ts, n / 2)
    assert abs(float(told) - n) <= 1.01 * U * n
    f = torch.tensor(n / 2, dtype=torch.float64).float() / told.cpu()
    for t, o in zip(ts, out):
        assert torch.equal(o, t * f.item())
    p, m, v = make(2), make(3), [t.square() for t in make(4)]
    q, m1, v1 = ([t.clone() for t in x] for x in (p, m, v))
    ops.adam_clip_update_(p, ts, m, v, lr=1e-2, clip_norm=n / 2, eps=1e-3 * scale)
    for i in range(len(sizes)):                                            # the same list cut into short ones: the other order
        cut = [slice(a, a + 1_000_000) for a in range(0, sizes[i], 1_000_000)]
        for c in cut:
            ops.adam_clip_update_([q[i][c]], [ts[i][c]], [m1[i][c]], [v1[i][c]], lr=1e-2, clip_norm=n / 2, eps=1e-3 * scale, use_norm=told)
    assert all(torch.equal(a, b) for x, y in ((p, q), (m, m1), (v, v1)) for a, b in zip(x, y))
    ops.clip_by_global_norm_(ts, n / 2)                                    # in place, and what is clipped already stays
    assert all(torch.equal(a, b) for a, b in zip(ts, out))


def test_small_results_share_memory_but_not_values(ops, dev):
    ts = [torch.randn(n, generator=gen(dev, n), device=dev).to(d) for n, d in ((5, torch.float32), (0, torch.float16), (70000, torch.bfloat16), (9, torch.float16),
                                                                              (100, torch.float32), (70000, torch.float32))]
    out, _ = ops.clip_by_global_norm(ts, INF)
    for i, o in enumerate(out):
        assert o.data_ptr() % 16 == 0 and o.is_contiguous() and o.dtype == ts[i].dtype
        kept = [x.clone() for x in out]
        version = [x._version for x in out]
        o.zero_()
        assert all(torch.equal(a, b) for j, (a, b) in enumerate(zip(out, kept)) if j != i)
        assert [x._version for x in out] == [v + (j == i) for j, v in enumerate(version)]
        o.copy_(kept[i])
    assert all(torch.equal(a, b) for a, b in zip(out, ts))
    out[0].requires_grad_()
    (out[0] * 2).sum().backward()
    assert torch.equal(out[0].grad, torch.full_like(ts[0], 2.0))


def test_lazily_negated_tensors(ops, dev):
    z = torch.randn(50, dtype=torch.complex64, generator=gen(dev, 1), device=dev)
    t = z.conj().imag                                                      # negative of memory, twice as far apart
    assert t.is_neg()
    want = t.clone()
    n = norm64([want])
    assert abs(float(ops.global_norm([t])) - n) <= 1.01 * U * n
    out, _ = ops.clip_by_global_norm([t], INF)
    assert torch.equal(out[0], want)
    q, s = ops.quantize_rows(t)
    wq, ws = ops.quantize_rows(want)
    assert torch.equal(q, wq) and torch.equal(s, ws)
    ops.clip_by_global_norm_([t], n / 2)
    assert bool(((t.double() - want.double() / 2).abs() <= want.double().abs() * 3 * U).all())


def test_strided_tensors_given_twice_are_refused(ops, dev, UHError):
    big = torch.ones(8, 8, device=dev)
    with pytest.raises(UHError, match='twice'):
        ops.clip_by_global_norm_([big[:, :3], big[:, :3]], 1.0)
    assert bool((big == 1).all())


def test_inference_mode(ops, dev):
    with torch.inference_mode():
        t = torch.ones(10, device=dev)
        n = ops.clip_by_global_norm_([t], 1.0)
        assert abs(float(n) - math.sqrt(10)) < 1e-6 and abs(float(t[0]) - 1 / math.sqrt(10)) < 1e-6
        p, g, m, v = (torch.ones(10, device=dev) for _ in range(4))
        ops.adam_clip_update_([p], [g], [m], [v], lr=1e-2)
        assert float(p[0]) < 1.0
        out, _ = ops.clip_by_global_norm([t], 0.5)
        assert out[0].shape == (10,)


def test_refused_calls_leave_everything_alone(ops, dev, UHError):
    p, g, m, v = (torch.ones(10, device=dev) for _ in range(4))
    with pytest.raises(UHError, match='no gradient'):
        ops.clip_by_global_norm([g], 1.0, use_norm=torch.ones((), device=dev).requires_grad_())
    with pytest.raises(UHError):
        ops.adam_clip_update_([p], [g], [m], [m], lr=1e-2)
    with pytest.raises(TypeError):
        ops.global_norm(3)
    assert all(bool((t == 1).all()) and t._version == 0 for t in (p, g, m, v))
    ops.global_norm(t for t in (p, g))                                     # any iterable


def test_rows_that_are_far_apart_or_few(ops, dev):
    """Strides past what 256 rows of 32-bit offsets reach are copied; a single row may carry any."""
    wide = torch.randint(-128, 128, (2, (1 << 23) + 64), generator=gen(dev, 7), device=dev, dtype=torch.int8)
    a = wide[:, 16:400]
    b = int_rows(dev, 5, 384, 9)
    one = torch.ones(5, device=dev)
    want = (a.double() @ b.double().t().contiguous()).float()
    assert torch.equal(ops.int8_matmul(a, one[:2], b, one), want)
    assert torch.equal(ops.int8_matmul(b, one, a, one[:2]), want.t())
    assert torch.equal(ops.int8_matmul(a[1:], one[:1], b, one), want[1:])


def test_graph_replays_of_split_products_and_lists(ops, dev):
    """Split products, the fused single row and a long list in one graph: replayed on new inputs with eager calls in between."""
    x, y = torch.randn(70, 8192, device=dev), torch.randn(1, 8192, device=dev)
    w, ws = ops.quantize_rows(torch.randn(300, 8192, generator=gen(dev, 4), device=dev))
    g = [torch.randn(9_000_000, device=dev), torch.randn(11, device=dev)]

    def run():
        return [ops.int8_linear(x, w, ws), ops.int8_linear(y, w, ws), ops.global_norm(g)] + ops.clip_by_global_norm(g, 1.0)[0]
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for _ in range(4):
        for t in [x, y] + g:
            t.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, run()))
