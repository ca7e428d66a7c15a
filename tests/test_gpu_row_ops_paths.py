"""GPU: the framework's own paths through the row operators: the flat bucket's clip, pointwise
sparse convs under ops.conv_math("f8") and spconv.RMSNorm inside a SparseSequential."""
import pytest
import torch
from torch import nn

import row_reference as ref
from objectdetection_amd import ops, spconv
from objectdetection_amd.dist import FlatGradAllReduce

pytestmark = pytest.mark.gpu


def _tensor(cuda, n=500, c=256, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    f = torch.randn((n, c), generator=g).to(dtype).to(cuda)
    cells = torch.randperm(20 * 20 * 20, generator=g)[:n]
    idx = torch.stack([torch.zeros_like(cells), cells // 400, cells // 20 % 20, cells % 20], 1)
    return spconv.SparseConvTensor(f, idx.int().to(cuda), [20, 20, 20], 1)


def _q(v, h=1):
    return ref.value(*ref.quantise(v.detach().float(), h=h), h)


def _near(got, want, share=1e-3):
    got, want = got.detach().double().cpu(), want.double().cpu()
    assert (got - want).norm() <= share * want.norm(), ((got - want).norm() / want.norm()).item()


def test_bucket_clip_takes_gradients_straight_into_the_buffer(cuda):
    torch.manual_seed(0)
    net = nn.Sequential(nn.Conv2d(3, 8, 3), nn.Conv2d(8, 5, 1), nn.Flatten(), nn.Linear(5 * 36, 7)).to(cuda)
    net[0].to(memory_format=torch.channels_last)
    x = torch.randn((4, 3, 8, 8), device=cuda).contiguous(memory_format=torch.channels_last)
    for max_norm in (0.1, 1e6):
        results = []
        for fused in (False, True):
            bucket = FlatGradAllReduce(net.parameters(), attach=False)
            bucket.zero()
            (net(x).square().sum()).backward()
            if fused:
                total = bucket.collect_clip_(max_norm)
            else:
                bucket.collect()
                total = torch.linalg.vector_norm(bucket.flat)
                bucket.flat.mul_(torch.clamp(max_norm / (total + 1e-6), max=1.0))
            results.append((total.clone(), bucket.flat.clone(), [p.grad.clone() for p in net.parameters()]))
            assert all(p.grad is v for p, v in zip(bucket.params, bucket.views[0]))
        (ta, fa, ga), (tb, fb, gb) = results
        assert torch.allclose(ta, tb, rtol=1e-5) and torch.allclose(fa, fb, rtol=1e-4, atol=1e-7)
        assert all(torch.allclose(a, b, rtol=1e-4, atol=1e-7) for a, b in zip(ga, gb))
    # a parameter without a gradient contributes zeros
    bucket = FlatGradAllReduce(net.parameters(), attach=False)
    bucket.zero()
    net[0](x).square().sum().backward()
    total = bucket.collect_clip_(0.5)
    assert total > 0.5 and abs(torch.linalg.vector_norm(bucket.flat).item() - 0.5) < 1e-4
    assert bool((net[3].weight.grad == 0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pointwise_conv_in_8_bit_form_trains(cuda, dtype):
    x = _tensor(cuda, dtype=dtype)
    conv = spconv.SubMConv3d(256, 64, 1, bias=True).to(cuda)
    feats = x.features.clone().requires_grad_(True)
    x.features = feats
    with ops.conv_math("f8"):
        y = conv(x).features
    assert y.dtype == dtype
    g = torch.randn(y.shape, generator=torch.Generator().manual_seed(1)).to(dtype)
    y.backward(g.to(cuda))
    w = conv.weight.detach().view(256, 64)
    share = 1e-5 if dtype == torch.float32 else 4e-3
    _near(y, _q(feats) @ _q(w, 128) + conv.bias.detach().double().cpu(), share)
    _near(feats.grad, _q(g) @ _q(w, 128).t(), share)
    _near(conv.weight.grad.view(256, 64), _q(feats.detach().t()) @ _q(g.t()).t(), 1e-5)
    _near(conv.bias.grad, g.double().sum(0), 1e-5)
    # a bias that alone wants a gradient gets one
    conv.weight.requires_grad_(False)
    conv.bias.grad = None
    x.features = feats.detach()
    with ops.conv_math("f8"):
        conv(x).features.backward(g.to(cuda))
    _near(conv.bias.grad, g.double().sum(0), 1e-5)
    plain = conv(x).features  # the default mode is what it was
    assert torch.equal(plain, torch.mm(feats, w.to(dtype)) + conv.bias.to(dtype))


def test_pointwise_conv_in_8_bit_form_serves_with_its_epilogue(cuda):
    torch.manual_seed(3)
    seq = spconv.SparseSequential(spconv.SubMConv3d(256, 64, 1, bias=False), nn.BatchNorm1d(64), nn.ReLU(),
                                  spconv.SubMConv3d(64, 256, 1, bias=True)).to(cuda).eval()
    with torch.no_grad():
        seq[1].running_mean.normal_()
        seq[1].running_var.uniform_(0.5, 2.0)
        x = _tensor(cuda)
        with ops.conv_math("f8"):
            got = seq(x).features
            again = seq(x).features
        bn = seq[1]
        a = _q(x.features) @ _q(seq[0].weight.view(256, 64), 128)
        a = torch.relu((a - bn.running_mean.double().cpu()) * (bn.running_var.double().cpu() + bn.eps) ** -0.5
                       * bn.weight.double().cpu() + bn.bias.double().cpu())
        want = _q(a.float()) @ _q(seq[3].weight.view(64, 256), 128) + seq[3].bias.double().cpu()
        # a few values within fp32 rounding of an 8-bit border may fall on its other side
        _near(got, want, 2e-3)
        assert torch.equal(got, again)
        seq[0].weight.mul_(2.0)  # the kept image follows the parameter
        with ops.conv_math("f8"):
            assert not torch.equal(seq(x).features, got)


@pytest.mark.parametrize("math", ["f32", "f8"])
def test_rms_norm_module_in_a_sequence(cuda, math):
    torch.manual_seed(4)
    seq = spconv.SparseSequential(spconv.RMSNorm(256), spconv.SubMConv3d(256, 64, 1, bias=False), nn.ReLU()).to(cuda)
    with torch.no_grad():
        seq[0].weight.normal_(1.0, 0.2)
    x = _tensor(cuda, 300)
    eps = torch.finfo(torch.float32).eps
    y, _, _ = ref.rms_norm(x.features, seq[0].weight.detach(), eps)
    w = seq[1].weight.detach().view(256, 64)
    if math == "f8":
        want = torch.relu(_q(y.float()) @ _q(w, 128))
    else:
        want = torch.relu(y @ w.double().cpu())
    with ops.conv_math(math):
        with torch.no_grad():
            served = seq(_tensor(cuda, 300)).features
        # (a sequence that begins with an ordinary module writes its result to the tensor it was given)
        x = _tensor(cuda, 300)
        x.features = leaf = x.features.requires_grad_(True)
        trained = seq(x).features
        trained.square().sum().backward()
    _near(served, want, 2e-3 if math == "f8" else 1e-5)
    _near(trained, want, 2e-3 if math == "f8" else 1e-5)
    assert leaf.grad.shape == (300, 256) and bool(torch.isfinite(leaf.grad).all())
    assert seq[0].weight.grad.shape == (256,) and float(seq[1].weight.grad.abs().sum()) > 0
    # and with the residual, as a residual block calls it
    r = torch.randn((300, 256), generator=torch.Generator().manual_seed(5)).to(cuda)
    yy, h = seq[0](leaf.detach(), r)
    assert torch.equal(h, leaf.detach() + r)
    _near(yy, ref.rms_norm(leaf.detach(), seq[0].weight.detach(), eps, r)[0], 1e-5)


def test_rms_norm_module_is_what_nn_rms_norm_is(cuda):
    a, b = spconv.RMSNorm(96, eps=1e-5).to(cuda), nn.RMSNorm(96, eps=1e-5).to(cuda)
    b.load_state_dict(a.state_dict())
    x = torch.randn((77, 96), generator=torch.Generator().manual_seed(6)).to(cuda)
    assert torch.allclose(a(x), b(x), rtol=1e-5, atol=1e-6)


def test_weight_images_follow_replaced_weights_streams_copies_and_captures(cuda):
    import copy
    import io
    x = _tensor(cuda)
    feats = x.features

    def run(conv):
        x.features = feats
        with torch.no_grad(), ops.conv_math("f8"):
            return conv(x).features.clone()

    def want(conv):
        return ops.f8_product(feats, ops.f8_weight_image(conv.weight.detach().view(256, 64), transpose=True))
    conv = spconv.SubMConv3d(256, 64, 1, bias=False).to(cuda)
    conv.weight = nn.Parameter(conv.weight.detach().clone())
    assert torch.equal(run(conv), want(conv))
    # replaced twice between two calls: the second takes the first one's memory, if that is free
    conv.weight = nn.Parameter(conv.weight.detach() * 2)
    conv.weight = nn.Parameter(conv.weight.detach() * 3)
    assert torch.equal(run(conv), want(conv))
    # copies and pickles
    for twin in (copy.deepcopy(conv), torch.load(_saved(conv, io.BytesIO()), weights_only=False)):
        with torch.no_grad():
            twin.weight.mul_(0.5)
        assert torch.equal(run(twin), want(twin))
    # first used on another stream, then here, and the other way round
    side = torch.cuda.Stream()
    with torch.no_grad():
        conv.weight.mul_(2.0)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = run(conv)
    here = run(conv)
    torch.cuda.synchronize()
    assert torch.equal(there, want(conv)) and torch.equal(here, there)
    # first used in a capture: the graph's image is the graph's
    run(spconv.SubMConv3d(256, 64, 1, bias=False).to(cuda))
    with torch.no_grad():
        conv.weight.mul_(0.25)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(conv)
    right = want(conv)
    assert torch.equal(run(conv), right)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, right) and torch.equal(run(conv), right)


def _saved(module, file):
    torch.save(module, file)
    file.seek(0)
    return file


@pytest.mark.parametrize("size", [1.0, 0.03, 0.001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_rms_norm_module_without_eps_takes_that_of_float32(cuda, dtype, size):
    """nn.RMSNorm's own default: the epsilon of the 32 bits that the norm is taken in, whatever the rows'
    type (bf16 rows of RMS 0.03 under bf16's own epsilon of 2^-7 would come out a third as large)."""
    x = (torch.randn((77, 96), generator=torch.Generator().manual_seed(7)) * size).to(dtype)
    want, _, inv = ref.rms_norm(x, None, torch.finfo(torch.float32).eps)
    # one store, and a chain of 96 squares, mean, root and division in fp32
    bound = (ref.half_step(dtype) + 2.0 ** -24 * 120) * want.abs() + torch.finfo(dtype).tiny
    y = spconv.RMSNorm(96).to(cuda)(x.to(cuda)).detach()
    assert y.dtype == dtype and bool(((y.double().cpu() - want).abs() <= bound).all())
    theirs = nn.RMSNorm(96, dtype=dtype)(x).detach().double()  # stored once as well
    assert bool(((y.double().cpu() - theirs).abs() <= 2 * bound).all())
    # straight to 8-bit rows, in front of a pointwise conv (values on a border of the format fall either way)
    seq = spconv.SparseSequential(spconv.RMSNorm(96), spconv.SubMConv3d(96, 32, 1, bias=False)).to(cuda)
    t = _tensor(cuda, 77, 96)
    t.features = x.to(cuda)
    with torch.no_grad(), ops.conv_math("f8"):
        got = seq(t).features
    _near(got, _q(want) @ _q(seq[1].weight.view(96, 32), 128), 2e-3 + ref.half_step(dtype))


@pytest.mark.parametrize("math", ["f8", "f32", "bf16x3"])
def test_a_captured_graph_makes_its_own_weight_image(cuda, math):
    """Warmed up, captured, then the weight changes and an ordinary call replaces the kept image: replays
    follow the weight and read nothing that was freed."""
    cin, cout, kernel = (256, 64, 1) if math == "f8" else (32, 32, 3)
    conv = spconv.SubMConv3d(cin, cout, kernel, bias=False, indice_key="a").to(cuda)
    x = _tensor(cuda, c=cin)
    feats = x.features

    def run():
        x.features = feats
        with torch.no_grad(), ops.conv_math(math):
            return conv(x).features
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            run()
    torch.cuda.current_stream().wait_stream(side)
    before = run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, before)
    for factor in (2.0, -0.5, 4.0):
        with torch.no_grad():
            conv.weight.mul_(factor)
        scaled, before = before * factor, run()
        # powers of two are exact in every mode; with the other sign the matrix cores may round a sum to
        # its other neighbour (32 channels x 27 offsets x 3 products, 2^-23 each)
        if factor > 0:
            assert torch.equal(before, scaled)
        assert float((before - scaled).abs().max()) <= 27 * 32 * 3 * 2.0 ** -23 * float(scaled.abs().max())
        for _ in range(20):  # what was freed is somebody else's now
            torch.full((cin * cout * kernel ** 3,), float("nan"), device=cuda)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, before) and torch.equal(run(), before)


class _Doubled(spconv.RMSNorm):
    def forward(self, x, residual=None):
        return 2 * super().forward(x, residual)


class _Counted(spconv.SubMConv3d):
    calls = 0

    def forward(self, input):
        _Counted.calls += 1
        return super().forward(input)


def test_norm_before_a_pointwise_conv_is_called_where_it_is_more_than_the_norm(cuda):
    """A subclass's forward and forward hooks, of the norm or the conv, act under conv_math('f8') without
    gradients as they do in every other mode."""
    torch.manual_seed(8)
    x = _tensor(cuda, 200, 64).features

    def run(norm, conv):
        t = _tensor(cuda, 200, 64)
        with torch.no_grad(), ops.conv_math("f8"):
            return spconv.SparseSequential(norm, conv)(t).features
    conv = spconv.SubMConv3d(64, 32, 1, bias=False).to(cuda)
    plain, twice = spconv.RMSNorm(64).to(cuda), _Doubled(64).to(cuda)
    y = ref.rms_norm(x, None, torch.finfo(torch.float32).eps)[0]
    w = _q(conv.weight.view(64, 32), 128)
    _near(run(plain, conv), _q(y) @ w, 2e-3)
    _near(run(twice, conv), _q(2 * y) @ w, 2e-3)
    seen = []
    plain.register_forward_pre_hook(lambda m, args: seen.append(args[0].shape))
    _near(run(plain, conv), _q(y) @ w, 2e-3)
    assert seen == [(200, 64)]
    hooked = spconv.RMSNorm(64).to(cuda)
    hooked.register_forward_hook(lambda m, args, out: out * 4)
    _near(run(hooked, conv), _q(4 * y) @ w, 2e-3)
    own = _Counted(64, 32, 1, bias=False).to(cuda)
    own.load_state_dict(conv.state_dict())
    _near(run(spconv.RMSNorm(64).to(cuda), own), _q(y) @ w, 2e-3)
    assert _Counted.calls == 1
    rows = []
    conv.register_forward_pre_hook(lambda m, args: rows.append(args[0].features))
    _near(run(spconv.RMSNorm(64).to(cuda), conv), _q(y) @ w, 2e-3)
    _near(rows[0], y, 1e-6)  # the normed rows, not those in front of the norm
