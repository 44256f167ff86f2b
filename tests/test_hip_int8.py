"""The int8 linear layer on the GPU (mmearth_train_amd.int8) against the definition in 64 bits on the CPU.

Tolerances. The codes are whole numbers and equal. y: the exact integer sum is rounded to fp32 (2^-24), multiplied by two scales that are rounded
to fp32 (2^-24 each, two products: 2^-24 each), added to the bias (2^-24 of the result) and rounded once to the type: at most 6 * 2^-24 of |q-product| and
of |y| + half a step of the type.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def ref_codes(x):
    x = x.detach().double().cpu()
    a = x.abs().amax(-1)
    q = torch.round(127.0 * x / torch.where(a == 0, 1.0, a)[..., None])
    return q, (a / 127.0).float().double()


def ref_linear(x, w, b):
    (qx, sx), (qw, sw) = ref_codes(x), ref_codes(w)
    part = (qx @ qw.t()) * sx[..., None] * sw
    return part + (0 if b is None else b.double().cpu()), part


def check(x, w, b, y):
    want, part = ref_linear(x, w, b)
    assert y.dtype == x.dtype and y.shape == want.shape
    tol = 6 * U * (part.abs() + want.abs()) + (0 if x.dtype == torch.float32 else torch.finfo(x.dtype).eps / 2) * want.abs()
    if x.dtype == torch.float16:
        tol = tol + 2.0 ** -25                 # half a step among its subnormals
    off = (y.double().cpu() - want).abs()
    assert bool((off <= tol).all()), (tuple(x.shape), tuple(w.shape), x.dtype, float((off - tol).max()))


def data(m, k, n, dtype, bias, seed=0):
    gen = torch.Generator("cuda").manual_seed(seed + 7 * m + 11 * k + 13 * n)
    x = (torch.randn(m, k, device="cuda", generator=gen) * torch.exp(torch.randn(m, 1, device="cuda", generator=gen))).to(dtype)
    w = torch.randn(n, k, device="cuda", generator=gen) * 0.03
    return x, w, 0.1 * torch.randn(n, device="cuda", generator=gen) if bias else None


@pytest.mark.parametrize("k", [1, 7, 128, 129, 333, 1000, 2048, 2049, 5000, 16384, 16385])
@pytest.mark.parametrize("dtype", list(DT))
def test_codes_and_scales(k, dtype):
    from mmearth_train_amd.int8 import quantize_weight
    for rows in (1, 5, 67):
        x, _, _ = data(rows, k, 1, DT[dtype], False, 1)
        if rows > 2:
            x[1] = 0.0
            x[2] *= 1e-3 if dtype == "fp16" else 1e-36
            x[3, ::2] = x[3].abs().amax() / 2         # 63.5: exact ties, to even
        w = quantize_weight(x)
        q, s = ref_codes(x)
        assert torch.equal(w.q[:, :k].cpu().double(), q), (rows, k, dtype)
        assert torch.equal(w.scale.cpu().double(), s)
        assert not w.q[:, k:].any()


SHAPES = [(1, 1, 1), (1, 16, 16), (1, 1024, 4096), (1, 11264, 40), (2, 77, 1000), (3, 2816, 1000), (8, 2816, 1000), (15, 640, 129), (16, 640, 128), (17, 129, 640),
          (33, 1000, 257), (49, 2816, 1408), (64, 320, 1280), (65, 320, 1280), (100, 43, 1009), (127, 160, 640), (128, 640, 160), (129, 5000, 255),
          (255, 128, 512), (256, 512, 256), (257, 513, 259), (300, 1, 300), (1003, 333, 77), (511, 1024, 1025), (2000, 384, 96), (4099, 80, 320)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear(m, k, n, dtype):
    from mmearth_train_amd.int8 import linear_int8, quantize_weight
    for bias in (True, False):
        x, w, b = data(m, k, n, DT[dtype], bias)
        check(x, w, b, linear_int8(x, quantize_weight(w, b)))


@pytest.mark.parametrize("m", [1, 2, 5, 16, 17, 40, 64, 65, 200, 1030])
def test_row_counts_around_every_variant(m):
    from mmearth_train_amd.int8 import linear_int8, quantize_weight
    for k, n in ((640, 1000), (2816, 704), (130, 4096)):
        x, w, b = data(m, k, n, torch.bfloat16, True, 3)
        check(x, w, b, linear_int8(x, quantize_weight(w, b)))


@pytest.mark.parametrize("m,k,n", [
    (1500, 300, 1300), (3000, 200, 2300), (3000, 1100, 2300), (20000, 130, 2600), (4100, 2050, 4100), (4100, 2050, 4000), (5600, 2050, 5500), (8192, 2048, 2048),
    (49, 11264, 2816), (20, 4097, 130), (100, 9000, 333), (33, 5000, 61), (9, 16384, 8300), (5, 3064, 515), (8, 2050, 70), (7, 1032, 333), (3, 6136, 100)])
def test_every_variant_of_the_product(m, k, n):
    """Sizes on both sides of every rule that chooses a kernel, against the products of the codes in 64 bits (exact: below 2^53) on the GPU."""
    from mmearth_train_amd.int8 import linear_int8, quantize_weight
    x, w, b = data(m, k, n, torch.bfloat16, True, 9)
    p, q = quantize_weight(w, b), quantize_weight(x)
    qx, _ = ref_codes(x[:50])
    assert torch.equal(q.q[:50, :k].cpu().double(), qx)
    part = (q.q[:, :k].double() @ p.q[:, :k].double().t().contiguous()) * q.scale.double()[:, None] * p.scale.double()
    want = part + b.double()
    y = linear_int8(x, p)
    tol = 6 * U * (part.abs() + want.abs()) + torch.finfo(torch.bfloat16).eps / 2 * want.abs()
    assert bool(((y.double() - want).abs() <= tol).all())


def test_leading_dimensions_strides_and_offsets():
    from mmearth_train_amd.int8 import linear_int8, quantize_weight
    gen = torch.Generator("cuda").manual_seed(5)
    w = torch.randn(90, 70, device="cuda", generator=gen)
    p = quantize_weight(w)
    for dtype in DT.values():
        room = torch.randn(6, 5, 4, 200, device="cuda", generator=gen).to(dtype)
        for x in (room[..., :70], room[..., 3:73], room[2, 1, 0, 1:71], room[0, 0, :, 5:75], room.permute(3, 0, 1, 2)[:4, :, :, 0].new_tensor(0).expand(3, 70),
                  room[0, 0, :, :70].t().contiguous().t(), room[:0, ..., :70], room[:, :, :, :70].transpose(0, 2), room[0, 0, :1, 2:72].expand(9, 70)):
            y = linear_int8(x, p)
            assert y.shape == x.shape[:-1] + (90,)
            if x.numel():
                check(x.reshape(-1, 70), w, None, y.reshape(-1, 90))
    # a weight that is a view of another order
    q = quantize_weight(w.t().contiguous().t())
    assert torch.equal(q.q, p.q) and torch.equal(q.scale, p.scale)


@pytest.mark.parametrize("m", [3, 70, 600])
def test_bad_rows_stay_alone(m):
    from mmearth_train_amd.int8 import linear_int8, quantize_weight
    for dtype in DT.values():
        x, w, b = data(m, 300, 130, dtype, True, 4)
        p = quantize_weight(w, b)
        x[0] = 0.0
        clean = linear_int8(x, p)
        assert torch.equal(clean[0].float(), b.to(dtype).float())
        x[1, 299] = float("inf")
        x[m - 1, 0] = float("nan")
        y = linear_int8(x, p)
        assert bool(torch.isnan(y[1]).all()) and bool(torch.isnan(y[m - 1]).all())
        rest = [i for i in range(m) if i not in (1, m - 1)]
        assert torch.equal(y[rest], clean[rest])


def test_sums_of_the_largest_codes():
    """Every product 127 * 127, the longest row whose sum fits 32 bits, both signs."""
    from mmearth_train_amd.int8 import MAX_K, linear_int8, quantize_weight
    for k in (MAX_K, MAX_K - 130):
        for m in (1, 20, 300):
            x, w = torch.ones(m, k, device="cuda", dtype=torch.bfloat16), torch.ones(3, k, device="cuda")
            w[1] = -1.0
            x[m - 1] = -2.0
            check(x, w, None, linear_int8(x, quantize_weight(w)))


def test_rows_past_31_bits():
    """x of more than 2^31 elements: offsets of rows need 64 bits, in x, in the codes and in y."""
    from mmearth_train_amd.int8 import linear_int8, quantize_weight
    m, k, n = 2 ** 31 // 128 + 77, 128, 136
    x = torch.zeros(m, k, device="cuda", dtype=torch.bfloat16)
    tail = torch.randn(300, k, device="cuda", generator=torch.Generator("cuda").manual_seed(6)).to(torch.bfloat16)
    x[-300:] = tail
    w = torch.randn(n, k, device="cuda", generator=torch.Generator("cuda").manual_seed(7))
    p = quantize_weight(w)
    y = linear_int8(x, p)
    check(tail, w, None, y[-300:])
    assert not bool(y[:-300].any())


def test_streams_and_graphs():
    from mmearth_train_amd.int8 import linear_int8, quantize_weight
    for m in (1, 40, 700):
        x, w, b = data(m, 640, 512, torch.bfloat16, True, 8)
        p = quantize_weight(w, b)
        want = linear_int8(x, p)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            y = linear_int8(x, p)
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(y, want)
        one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()       # two graphs over one weight, replayed in turn
        torch.cuda.synchronize()
        with torch.cuda.graph(one):
            y1 = linear_int8(x, p)
        x2 = x.clone()
        torch.cuda.synchronize()
        with torch.cuda.graph(two):
            y2 = linear_int8(x2, p)
        for k in range(3):
            x.normal_(generator=torch.Generator("cuda").manual_seed(k))
            x2.normal_(generator=torch.Generator("cuda").manual_seed(90 + k))
            one.replay()
            two.replay()
            torch.cuda.synchronize()
            assert torch.equal(y1, linear_int8(x, p)) and torch.equal(y2, linear_int8(x2, p))


def test_refusals_on_the_device():
    from mmearth_train_amd.int8 import linear_int8, quantize_weight
    w = torch.zeros(8, 16, device="cuda")
    p = quantize_weight(w)
    with pytest.raises(ValueError, match="end in 16"):
        linear_int8(torch.zeros(2, 17, device="cuda"), p)
    with pytest.raises(ValueError, match="end in 16"):
        linear_int8(torch.zeros((), device="cuda"), p)
    with pytest.raises(ValueError, match="fp32, bf16 or fp16"):
        linear_int8(torch.zeros(2, 16, device="cuda", dtype=torch.float64), p)
    with pytest.raises(ValueError, match="the input is on cpu"):
        linear_int8(torch.zeros(2, 16), p)
    x = torch.zeros(2, 16, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward"):
        linear_int8(x, p)
    with torch.no_grad():
        assert linear_int8(x, p).shape == (2, 8)
    with pytest.raises(ValueError, match="bias"):
        quantize_weight(w, torch.zeros(9, device="cuda"))
    from mmearth_train_amd.int8 import Int8Weight
    q, f = p.q, p.scale
    for bad in (Int8Weight(q.float(), f, None, 16), Int8Weight(q, f.half(), None, 16), Int8Weight(q, f[:7], None, 16), Int8Weight(q[:, :100], f, None, 16),
                Int8Weight(q[:, :64].contiguous(), f, None, 16), Int8Weight(q, f, f.double(), 16), Int8Weight(q, f.cpu(), None, 16)):
        with pytest.raises(ValueError, match="quantize_weight makes"):
            linear_int8(torch.zeros(2, 16, device="cuda"), bad)


def test_wider_rows_of_codes_are_refused():
    """Codes padded further than K rounded up: refused on the host, before anything is launched."""
    from mmearth_train_amd.int8 import Int8Weight, linear_int8, quantize_weight
    for k, wide, m in ((3900, 4096, 64), (7, 256, 3), (100, 384, 20)):
        p = quantize_weight(torch.ones(5, k, device="cuda"))
        q = torch.zeros(5, wide, device="cuda", dtype=torch.int8)
        q[:, :p.q.shape[1]] = p.q
        with pytest.raises(ValueError, match="quantize_weight makes"):
            linear_int8(torch.ones(m, k, device="cuda"), Int8Weight(q, p.scale, None, k))


def test_a_network_is_trained_with_8_bit_moments_and_served_in_int8(tmp_path):
    """The dense network as a user has it: fine-tuned by the 8-bit AdamW, then quantised, saved, loaded and served."""
    from mmearth_train_amd import convnextv2
    from mmearth_train_amd.helpers import param_groups_weight_decay
    from mmearth_train_amd.int8 import Int8Linear, quantize_model
    from mmearth_train_amd.optim import AdamW
    torch.manual_seed(0)
    net = convnextv2.convnextv2_atto(num_classes=5).cuda()
    opt = AdamW(param_groups_weight_decay(net, 0.05), lr=1e-3, betas=(0.9, 0.95), state_bits=8, max_norm=1.0)
    x, t = torch.randn(6, 12, 56, 56, device="cuda"), torch.tensor([0, 1, 2, 3, 4, 0], device="cuda")
    for _ in range(3):
        loss = nn_loss(net(x), t)
        loss.backward()
        assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in net.parameters())
        opt.step()
        opt.zero_grad()
    assert opt.plan.steps.tolist() == [3] * len(opt.plan.params) and math.isfinite(float(opt.grad_norm))
    with torch.no_grad():
        # the same network with its weights and activations rounded as the definition rounds them
        taken = {}
        hooks = [mod.register_forward_hook(lambda mod, i, o, name=name: taken.__setitem__(name, (i[0], mod))) for name, mod in net.named_modules()
                 if isinstance(mod, torch.nn.Linear)]
        net(x)
        for h in hooks:
            h.remove()
        assert len(taken) == 2 * 12 + 1
        served = quantize_model(net)
        mods = dict(served.named_modules())
        assert sum(isinstance(v, Int8Linear) for v in mods.values()) == len(taken) and not any(isinstance(v, torch.nn.Linear) for v in mods.values())
        for name, (i, linear) in taken.items():
            check(i.reshape(-1, i.shape[-1]), linear.weight, linear.bias, mods[name](i).reshape(-1, linear.out_features))
        y = served(x)
        assert y.shape == (6, 5) and bool(torch.isfinite(y).all())
        torch.save(served.state_dict(), tmp_path / "served.pth")
        other = quantize_model(convnextv2.convnextv2_atto(num_classes=5).cuda())
        other.load_state_dict(torch.load(tmp_path / "served.pth", map_location="cuda", weights_only=True))
        # (F.layer_norm and the convolutions are the same calls on the same inputs)
        assert torch.equal(other(x), y)
        import copy
        twin = copy.deepcopy(other)              # its own buffers, read by its own calls
        for buf in other.buffers():
            if buf.dtype == torch.int8:
                buf.zero_()
        assert torch.equal(twin(x), y) and not torch.equal(other(x), y)
        half = twin.half()
        lin = half.head
        assert lin.scale.dtype == torch.float32 and lin.q.dtype == torch.int8
        assert half(x.half()).dtype == torch.float16


def test_shared_and_foreign_layers_of_a_model():
    from mmearth_train_amd.int8 import Int8Linear, quantize_model

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.a = torch.nn.Linear(16, 16)
            self.b = self.a
            self.c = torch.nn.Sequential(self.a, torch.nn.ReLU())
            self.d = torch.nn.MultiheadAttention(16, 2)
            self.e = None

        def forward(self, x):
            return self.c(self.b(self.a(x)))

    net = quantize_model(Net().cuda())
    assert isinstance(net.a, Int8Linear) and net.a is net.b and net.a is net.c[0]
    assert not isinstance(net.d.out_proj, Int8Linear)
    with torch.no_grad():
        assert net(torch.randn(3, 16, device="cuda")).shape == (3, 16)
        net.d(*[torch.randn(3, 1, 16, device="cuda")] * 3)


def test_a_quantised_weight_is_a_copy():
    """Training on after the quantisation changes neither the codes nor the bias."""
    from mmearth_train_amd.int8 import linear_int8, quantize_weight
    layer = torch.nn.Linear(40, 24).cuda()
    x = torch.randn(5, 40, device="cuda")
    for bias in (layer.bias, layer.bias.detach()[:1].expand(24)):
        with torch.no_grad():
            p = quantize_weight(layer.weight, bias)
            y = linear_int8(x, p)
            layer.weight.add_(1.0)
            layer.bias.add_(1.0)
            assert torch.equal(y, linear_int8(x, p))


def nn_loss(y, t):
    return torch.nn.functional.cross_entropy(y, t)


def test_hub_serves_in_int8():
    import hubconf
    from mmearth_train_amd.int8 import Int8Linear
    net = hubconf.MPMAE("convnextv2_atto", pretrained=False, num_classes=7, int8=True)
    assert isinstance(net.head, Int8Linear) and isinstance(net.stages[0][0].pwconv1, Int8Linear) and net.head.q.is_cuda
    with torch.no_grad():
        assert net(torch.randn(1, 12, 56, 56, device="cuda")).shape == (1, 7)


def test_traced_and_exported_layers_compute(tmp_path):
    """The operator is in the graph, with other inputs and row counts than the traced ones, from a file, and next to the eager call bit for bit."""
    import warnings
    from torch.fx.experimental.proxy_tensor import make_fx
    from mmearth_train_amd.int8 import linear_int8, quantize_model, quantize_weight
    torch.manual_seed(0)
    net = quantize_model(torch.nn.Sequential(torch.nn.Linear(96, 200), torch.nn.GELU(), torch.nn.Linear(200, 33)).cuda())
    xs = [torch.randn(n, 96, device="cuda") for n in (5, 1, 300)]
    w = torch.randn(40, 96, device="cuda")
    with torch.no_grad(), warnings.catch_warnings():
        warnings.simplefilter("error", torch.jit.TracerWarning)
        want = [net(x) for x in xs]
        traced = torch.jit.trace(net, xs[0])
        assert str(traced.inlined_graph).count("mpmae::linear_int8") == 2
        traced.save(str(tmp_path / "net.pt"))
        loaded = torch.jit.load(str(tmp_path / "net.pt"))
        fx = make_fx(net)(xs[0])
        exported = torch.export.export(net, (xs[0],), strict=False).module()
        for f, count in ((traced, 3), (loaded, 3), (fx, 1), (exported, 1)):
            for _ in range(3):
                for x, y in list(zip(xs, want))[:count]:
                    junk = torch.full_like(y, 5.0)              # (what an output that nothing writes would hold)
                    del junk
                    assert torch.equal(f(x), y)
        warnings.simplefilter("ignore")                         # (the quantiser's checks of sizes in Python hold for the traced ones)
        both = torch.jit.trace(lambda x, w: linear_int8(x, quantize_weight(w)), (xs[0], w))
        assert "mpmae::quantize_int8" in str(both.graph) and "aten::empty" not in str(both.graph)
        for _ in range(2):
            assert torch.equal(both(xs[2], 2 * w), linear_int8(xs[2], quantize_weight(2 * w)))
        # rows under vmap are the rows of the whole call
        p = quantize_weight(w)
        assert torch.equal(torch.vmap(lambda x: linear_int8(x, p))(xs[2].view(10, 30, 96)), linear_int8(xs[2], p).view(10, 30, 40))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            y = traced(xs[2])
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(y, want[2])


def test_quantised_layers_keep_their_hooks():
    """Forward hooks and pre-hooks run on the new layer as on the old one, and their handles remove them; layers whose weight a hook computes or whose forward was
    replaced stay as they are."""
    import torch.nn.utils.prune as prune
    from mmearth_train_amd.int8 import Int8Linear, quantize_model
    torch.manual_seed(1)
    net = torch.nn.Sequential(*[torch.nn.Linear(16, 16) for _ in range(5)]).cuda().eval()
    seen = []
    pre = net[0].register_forward_pre_hook(lambda m, a: (seen.append("pre"), (a[0] * 2,))[1])
    post = net[0].register_forward_hook(lambda m, a, kw, y: (seen.append(type(m)), y + 1)[1], with_kwargs=True)
    prune.random_unstructured(net[1], "weight", 0.5)
    net[2] = torch.nn.utils.spectral_norm(net[2])
    was = net[3].forward
    net[3].forward = lambda x: was(x) - 1
    net[3].register_forward_hook(lambda m, a, y: -y)
    x = torch.randn(4, 16, device="cuda")
    with torch.no_grad():
        quantize_model(net)
        assert [isinstance(m, Int8Linear) for m in net] == [True, False, False, False, True] and not net[0].training
        y = net[0](x)
        assert seen == ["pre", Int8Linear]
        post.remove()
        assert torch.equal(net[0](x) + 1, y) and seen == ["pre", Int8Linear, "pre"]
        pre.remove()
        assert torch.equal(net[0](2 * x) + 1, y) and len(seen) == 3
        net(x)


def test_a_refused_layer_leaves_the_model_as_it_was():
    from mmearth_train_amd.int8 import Int8Linear, quantize_model
    net = torch.nn.Sequential(torch.nn.Linear(16, 16), torch.nn.Sequential(torch.nn.Linear(16, 8)), torch.nn.Linear(8, 4).double()).cuda()
    with pytest.raises(ValueError, match="fp32, bf16 or fp16"):
        quantize_model(net)
    assert not any(isinstance(m, Int8Linear) for m in net.modules())
    net[2].float()
    assert [isinstance(m, Int8Linear) for m in (quantize_model(net)[0], net[1][0], net[2])] == [True] * 3
    assert isinstance(quantize_model(torch.nn.Linear(4, 4).cuda()), Int8Linear)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("k", [7, 130, 1000, 9000, 20000])
def test_codes_of_rows_near_the_largest_number(dtype, k):
    """Rows whose maximum times 127 is no number of fp32, among them exact ties (63.5: half the maximum) and the type's
    lowest value."""
    from mmearth_train_amd.int8 import quantize_weight
    t = DT[dtype]
    x, _, _ = data(6, k, 1, t, False, 2)
    x = (x.float() / x.float().abs().amax(1, keepdim=True) * torch.tensor([3.3e38, 1e38, 2.7e36, 2.6e36, 1e31, 1e30], device="cuda")[:, None]).to(t)
    x[0, 0] = torch.finfo(t).min
    for r in range(6):
        a = float(x[r].abs().amax())
        x[r, 1:k:5] = a / 2                                   # 63.5 -> 64
        x[r, 2:k:5] = -a / 2
        if dtype == "fp32" or r:
            x[r, -1] = (2.0 ** math.floor(math.log2(a)))      # a power of two near the top
    w = quantize_weight(x)
    q, s = ref_codes(x)
    assert torch.equal(w.q[:, :k].cpu().double(), q) and torch.equal(w.scale.cpu().double(), s)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("m,k,n", [(1, 130, 40), (6, 1000, 33), (8, 3080, 40), (12, 640, 100), (40, 640, 100), (40, 4096, 100), (700, 130, 600)])
def test_outputs_of_rows_that_hold_the_lowest_value(m, k, n, dtype):
    """Every form of the product: outputs that are numbers of the type come out as such, also where the scale of x times the integer sum is none."""
    from mmearth_train_amd.int8 import linear_int8, quantize_weight
    t = DT[dtype]
    x, w, b = data(m, k, n, t, True, 12)
    x[:, ::3] = torch.finfo(t).min
    x[m - 1] = torch.finfo(t).max / 3
    w = w / (k if dtype == "fp16" else 64 * k)                # (sums of k products stay below the largest number)
    y = linear_int8(x, quantize_weight(w, b))
    assert bool(torch.isfinite(y).all())
    check(x, w, b, y)
