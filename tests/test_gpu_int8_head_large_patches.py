"""GPU: fc1 in 8 bits where one product may not add up all of its columns in 32 bits (patches of 256 px and more)."""
import pytest

torch = pytest.importorskip('torch')

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope='module')
def dev():
    if not torch.cuda.is_available():
        pytest.skip('no HIP device')
    return torch.device('cuda:0')


@pytest.fixture(scope='module')
def head(dev):
    from unsuperviseddeephomographyral2018_amd.homography_model import VGGRegressor

    def make(K):
        net = VGGRegressor(32)
        net.fc1 = torch.nn.Linear(K, 1024)
        return net.to(dev).eval()
    return make


def head64(net, x, columns):
    """relu(fc1) in 64 bits and how far 8 bits may be off: in each part half a step of either factor's scale; the factors and scales are
    rounded (4 u), the epilogue (4 u) and the sums of the parts (2 u each) too."""
    w = net.fc1.weight.detach()
    full = net.fc1.bias.detach().double().expand(x.shape[0], 1024).clone()
    bound, size = torch.zeros_like(full), full.abs()
    for c in columns:
        xs, ws = x[:, c].double(), w[:, c].double()
        sx, sw = xs.abs().amax(1) / 127, ws.abs().amax(1) / 127
        product = torch.mm(xs, ws.t().contiguous())
        full += product
        size = torch.maximum(size, full.abs()) + product.abs()
        bound += 0.5 * sx[:, None] * ws.abs().sum(1) + 0.5 * sw * xs.abs().sum(1)[:, None] + 0.25 * xs.shape[1] * sx[:, None] * sw
    return full.clamp(min=0), bound * 1.001 + (8 + 2 * len(columns)) * U * (size + bound)


@pytest.mark.parametrize('K,parts', [(2048, 1), (131071, 1), (131072, 2), (139392, 2), (261888, 2), (262142, 3)])
def test_fc1_in_parts(head, dev, K, parts):
    from unsuperviseddeephomographyral2018_amd import ops
    net = head(K)
    g = torch.Generator(device=dev).manual_seed(K)
    x = torch.randn(3, K, generator=g, device=dev).relu() * torch.linspace(0.1, 2.0, K, device=dev)
    with torch.no_grad(), net.int8_head():
        y = net._fc1_relu(x).double()
        columns = [c for c, _, _ in net._int8_fc1]
        assert len(columns) == parts and columns[0].start == 0 and columns[-1].stop >= K
        assert all(a.stop == b.start and a.stop % 128 == 0 for a, b in zip(columns, columns[1:]))
    assert net._int8_fc1 is None
    want, bound = head64(net, x, columns)
    assert bool(((y - want).abs() <= bound).all())
    if parts == 1:
        q, s = ops.quantize_rows(net.fc1.weight.detach())
        assert torch.equal(y, ops.int8_linear(x, q, s, bias=net.fc1.bias.detach(), relu=True).double())


def test_a_regressor_for_256_px(dev):
    from unsuperviseddeephomographyral2018_amd.homography_model import VGGRegressor
    torch.manual_seed(1)
    net = VGGRegressor(256).to(dev).to(memory_format=torch.channels_last).eval()
    x = torch.randn(2, 256, 256, 2, device=dev)
    seen, call = [], net._fc1_relu
    net._fc1_relu = lambda t: (seen.append(t), call(t))[1]
    with torch.no_grad(), net.int8_head():
        y = net(x)
        columns = [c for c, _, _ in net._int8_fc1]
    assert len(columns) == 2 and seen[0].shape == (2, 131072)
    hidden, bound = head64(net, seen[0], columns)
    w2 = net.fc2.weight.detach().double()
    want = torch.mm(hidden, w2.t().contiguous()) + net.fc2.bias.detach().double()
    rounding = 1026 * U * (torch.mm(hidden + bound, w2.t().abs().contiguous()) + net.fc2.bias.detach().double().abs())      # fc2 in float32
    assert bool(((y.double() - want).abs() <= torch.mm(bound, w2.t().abs().contiguous()) + rounding).all())
