"""AdamW over many tensors on the GPU (mmearth_train_amd.optim) against the formulas in 64 bits on the CPU.

Tolerances. u = 2^-24 is half a step of fp32. A 32-bit moment is two products and a sum of fp32-rounded factors: at most 5 roundings of
|b1 m| + |c1 g| per step, and the last step's error enters the next one scaled by b1 < 1, so `steps * 5 u` of the largest such sum bounds it. The
parameter adds p * decay (3 roundings of |p|) and the quotient step * m / (sqrt(v) * isbc2 + eps): at most 10 roundings of its own on top of the
moments' relative errors (that of v halved by the root). A parameter of fewer bits is rounded once per step on both sides: next to a border the two
round apart, one whole step of its type (eps). Codes and scales of the 8-bit moments are formed in 64 bits on both sides,
operation by operation, and have to be equal.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BLOCK = 256
DT = [torch.float32, torch.bfloat16, torch.float16]


class Ref:
    """One tensor of the definition in 64 bits; the parameter is rounded to its type after every step."""

    def __init__(self, p, bits):
        self.type, self.bits, self.t = p.dtype, bits, 0
        self.p = p.detach().double().cpu().reshape(-1)
        self.m, self.v = torch.zeros_like(self.p), torch.zeros_like(self.p)
        self.tol_m, self.tol_v, self.tol_p = (torch.zeros_like(self.p) for _ in range(3))

    def step(self, g, coef, lr, b1, b2, eps, wd):
        self.t += 1
        g = g.detach().double().cpu().reshape(-1) * coef
        size_m, size_v = b1 * self.m.abs() + (1 - b1) * g.abs(), b2 * self.v + (1 - b2) * g * g
        m, v = b1 * self.m + (1 - b1) * g, b2 * self.v + (1 - b2) * g * g
        self.tol_m = b1 * self.tol_m + (0 if self.bits == 8 else 5 * U) * size_m
        self.tol_v = b2 * self.tol_v + (0 if self.bits == 8 else 6 * U) * size_v
        denom = v.sqrt() / math.sqrt(1 - b2 ** self.t) + eps
        step = lr / (1 - b1 ** self.t)
        up = step * m / denom
        self.tol_p = self.tol_p + 3 * U * self.p.abs() + step * (self.tol_m + U * m.abs()) / denom + up.abs() * (12 * U + torch.nan_to_num(self.tol_v / v))
        self.p = (self.p * (1 - lr * wd) - up)
        self.tol_p = self.tol_p + (U if self.type == torch.float32 else torch.finfo(self.type).eps) * self.p.abs()
        if self.type == torch.float16:
            self.tol_p = self.tol_p + 2.0 ** -24           # a whole step among its subnormals
        self.p = self.p.to(self.type).double()
        if self.bits == 32:
            self.m, self.v = m, v
        else:
            (self.km, self.sm), (self.kv, self.sv) = codes(m, False), codes(v, True)
            self.m, self.v = values(self.km, self.sm, False)[:m.numel()], values(self.kv, self.sv, True)[:m.numel()]


def codes(x, fourth):
    n = x.numel()
    x = torch.cat([x, x.new_zeros(-n % BLOCK)]).reshape(-1, BLOCK).numpy()
    s = np.abs(x).max(1).astype(np.float32).astype(np.float64)
    r = np.divide(np.abs(x), s[:, None], out=np.zeros_like(x), where=s[:, None] > 0)
    k = np.floor(255 * r ** 0.25 + 0.5).clip(0, 255) if fourth else np.floor(127 * r ** 0.5 + 0.5).clip(0, 127) * np.sign(x)
    if fourth:
        k = np.where((x > 0) & (s[:, None] > 0), np.maximum(k, 1), k)        # (a block whose scale rounds to 0 holds nothing)
    return k, s


def values(k, s, fourth):
    x = k ** 4 * (s * (1 / 255 ** 4))[:, None] if fourth else k * np.abs(k) * (s * (1 / 127 ** 2))[:, None]
    return torch.from_numpy(x.reshape(-1))


def params_of(sizes, types, seed, odd=False):
    gen = torch.Generator("cuda").manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        d = types[i % len(types)]
        room = torch.randn(n + 1, device="cuda", generator=gen)
        room = (0.1 * room).to(d)
        out.append(torch.nn.Parameter(room[1:] if odd else room[:n]))         # odd: rows that begin at no vector boundary
    return out


def grads_for(params, seed, odd=False, scale=1.0):
    gen = torch.Generator("cuda").manual_seed(seed)
    for p in params:
        room = torch.randn(p.numel() + 1, device="cuda", generator=gen) * torch.exp(torch.randn(p.numel() + 1, device="cuda", generator=gen))
        room = (scale * 0.02 * room).to(p.dtype)
        p.grad = (room[1:] if odd else room[:p.numel()]).view(p.shape)


def check(opt, params, refs, bits):
    m, v = (x.cpu().double() for x in opt.flat_moments())
    for p, o, r in zip(params, opt.offsets, refs):
        n = p.numel()
        dp = (p.detach().double().cpu().reshape(-1) - r.p).abs()
        assert bool((dp <= r.tol_p).all()), (n, p.dtype, float((dp - r.tol_p).max()))
        if bits == 8:
            plan = opt.plan
            nb = -(-n // BLOCK)
            assert torch.equal(plan.m[o:o + nb * BLOCK].cpu().double(), torch.from_numpy(r.km.reshape(-1))), (n, p.dtype)
            assert torch.equal(plan.v[o:o + nb * BLOCK].cpu().double(), torch.from_numpy(r.kv.reshape(-1))), (n, p.dtype)
            assert torch.equal(plan.ms[o // BLOCK:o // BLOCK + nb].cpu().double(), torch.from_numpy(r.sm))
            assert torch.equal(plan.vs[o // BLOCK:o // BLOCK + nb].cpu().double(), torch.from_numpy(r.sv))
            # read back in fp32: one rounding of the value, half a step: 2^-24 of it, or 2^-150 where it is subnormal (those are 2^-149 apart)
            assert bool(((m[o:o + n] - r.m).abs() <= 1.01 * U * r.m.abs() + 2.0 ** -150).all())
            assert bool(((v[o:o + n] - r.v).abs() <= 1.01 * U * r.v.abs() + 2.0 ** -150).all())
        else:
            assert bool(((m[o:o + n] - r.m).abs() <= r.tol_m + 1e-45).all()), (n, p.dtype)
            assert bool(((v[o:o + n] - r.v).abs() <= r.tol_v + 1e-45).all()), (n, p.dtype)
        assert not m[o + n:o + -(-n // BLOCK) * BLOCK].any() and not v[o + n:o + -(-n // BLOCK) * BLOCK].any()


def run_steps(opt, params, refs, steps, clip=None, odd=False, lacking=()):
    for k in range(steps):
        grads_for(params, 100 + k, odd, scale=10.0 if k == 1 else 1.0)
        for i in lacking:
            if (i + k) % 2 == 0:
                params[i].grad = None
        before = [p.grad.clone() for p in params if p.grad is not None]
        coef = 1.0
        if clip:
            norm = math.sqrt(sum(float(p.grad.double().square().sum()) for p in params if p.grad is not None))
            coef = float(np.float32(min(1.0, clip / (norm + 1e-6))))
        opt.step()
        if clip:
            assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm
        assert all(torch.equal(a, b) for a, b in zip(before, (p.grad for p in params if p.grad is not None)))
        i = 0
        for g in opt.param_groups:
            for p in g["params"]:
                if p.grad is not None:
                    refs[i].step(p.grad, coef, g["lr"], *g["betas"], g["eps"], g["weight_decay"])
                i += 1


SIZES = [1, 7, 255, 256, 257, 2047, 4096, 4097, 10007, 3, 65536 + 13]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("types", [DT[:1], DT[1:2], DT[2:], DT], ids=["fp32", "bf16", "fp16", "mixed"])
@pytest.mark.parametrize("odd", [False, True], ids=["aligned", "odd"])
def test_steps_match_the_definition(bits, types, odd):
    from mmearth_train_amd.optim import AdamW
    params = params_of(SIZES, types, 3, odd)
    refs = [Ref(p, bits) for p in params]
    opt = AdamW([{"params": params[:4], "weight_decay": 0.0}, {"params": params[4:], "betas": (0.8, 0.999), "lr": 3e-3}], lr=1e-3, betas=(0.9, 0.95),
                weight_decay=0.05, state_bits=bits)
    run_steps(opt, params, refs, 4, odd=odd, lacking=(2, 5))
    check(opt, params, refs, bits)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("clip", [0.05, 1e4])
def test_clip_uses_the_norm_of_every_gradient(bits, clip):
    from mmearth_train_amd.optim import AdamW
    params = params_of(SIZES, DT, 4)
    refs = [Ref(p, bits) for p in params]
    opt = AdamW(params, lr=1e-3, state_bits=bits, max_norm=clip)
    run_steps(opt, params, refs, 3, clip=clip, lacking=(1,))
    assert float(opt.skipped) == 0.0
    check(opt, params, refs, bits)


@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_and_groups_than_one_launch_takes(bits):
    from mmearth_train_amd.optim import AdamW
    sizes = [1 + (i * 37) % 700 for i in range(1100)]
    params = params_of(sizes, DT, 5)
    refs = [Ref(p, bits) for p in params]
    opt = AdamW([{"params": params[i:i + 8], "lr": 1e-3 * (1 + i / 100), "weight_decay": 0.01 * (i % 3)} for i in range(0, 1100, 8)], state_bits=bits,
                max_norm=0.5)
    run_steps(opt, params, refs, 2, clip=0.5)
    check(opt, params, refs, bits)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_norm_that_is_not_finite_changes_nothing(bits):
    from mmearth_train_amd.optim import AdamW
    params = params_of([300, 5000], DT[:2], 6)
    opt = AdamW(params, state_bits=bits, max_norm=1.0)
    grads_for(params, 1)
    opt.step()
    keep = [p.detach().clone() for p in params], [x.clone() for x in opt.flat_moments()], opt.plan.steps.clone()
    for bad in (float("inf"), float("nan"), -float("inf")):
        grads_for(params, 2)
        params[1].grad[4321] = bad
        opt.step()
        assert float(opt.skipped) == 1.0 and not math.isfinite(float(opt.grad_norm))
        assert all(torch.equal(a, b.detach()) for a, b in zip(keep[0], params))
        assert all(torch.equal(a, b) for a, b in zip(keep[1], opt.flat_moments()))
        assert torch.equal(keep[2], opt.plan.steps)
    grads_for(params, 3)
    opt.step()
    assert float(opt.skipped) == 0.0 and opt.plan.steps.tolist() == [2, 2]


def test_without_a_clip_a_bad_gradient_stays_in_its_block():
    from mmearth_train_amd.optim import AdamW
    params = params_of([1024], DT[:1], 7)
    opt = AdamW(params, state_bits=8)
    grads_for(params, 1)
    params[0].grad[300] = float("nan")
    opt.step()
    m, v = opt.flat_moments()
    bad = torch.zeros(1024, dtype=torch.bool, device="cuda")
    bad[256:512] = True
    assert torch.equal(torch.isnan(m), bad) and torch.equal(torch.isnan(v), bad)
    assert torch.isnan(params[0]).nonzero().flatten().tolist() == [300]


def test_tiny_and_zero_gradients():
    """Blocks whose scale is far below fp32's normal range, or nothing at all."""
    from mmearth_train_amd.optim import AdamW
    params = params_of([256 * 6], DT[:1], 8)
    refs = [Ref(params[0], 8)]
    opt = AdamW(params, state_bits=8, eps=1e-8)
    for k in range(3):
        grads_for(params, 20 + k)
        g = params[0].grad.view(6, 256)
        g[0] = 0.0
        g[1] *= 1e-18              # v near 1e-39: subnormal scale
        g[2] *= 1e-30              # v under every fp32 number, m still normal
        g[3, 1:] = 0.0
        g[4, ::2] *= 1e-12
        opt.step()
        refs[0].step(params[0].grad, 1.0, 1e-3, 0.9, 0.999, 1e-8, 1e-2)
    check(opt, params, refs, 8)


def test_other_element_orders():
    """Parameters that are dense in another order than row-major, gradients in a third one."""
    from mmearth_train_amd.optim import AdamW
    for bits in (32, 8):
        gen = torch.Generator("cuda").manual_seed(9)
        w = torch.nn.Parameter(torch.randn(8, 12, 5, 5, device="cuda", generator=gen).contiguous(memory_format=torch.channels_last))
        q = torch.nn.Parameter(torch.randn(40, 30, device="cuda", generator=gen).t())
        g, h = torch.randn(8, 12, 5, 5, device="cuda", generator=gen), torch.randn(30, 40, device="cuda", generator=gen)
        w.grad, q.grad = g.clone(), h.clone()
        a = torch.nn.Parameter(w.detach().clone().contiguous())
        b = torch.nn.Parameter(q.detach().clone().contiguous())
        a.grad, b.grad = g.clone(), h.clone()
        one, two = AdamW([w, q], state_bits=32), AdamW([a, b], state_bits=32)
        for _ in range(2):
            one.step()
            two.step()
        assert torch.equal(w, a) and torch.equal(q, b)
        s, t = one.state_dict()["state"], two.state_dict()["state"]
        assert all(torch.equal(s[i][k], t[i][k]) for i in (0, 1) for k in ("exp_avg", "exp_avg_sq"))


@pytest.mark.parametrize("bits", [32, 8])
def test_checkpoints_go_both_ways_with_torch(bits):
    from mmearth_train_amd.optim import AdamW
    params = params_of([33, 4500, 257], DT[:1], 10)
    mine = AdamW(params, lr=2e-3, betas=(0.9, 0.95), weight_decay=0.05, state_bits=bits)
    for k in range(3):
        grads_for(params, 30 + k)
        mine.step()
    sd = mine.state_dict()
    theirs = torch.optim.AdamW([torch.nn.Parameter(p.detach().clone()) for p in params], lr=1.0)
    theirs.load_state_dict(sd)
    assert theirs.param_groups[0]["lr"] == 2e-3
    again = AdamW([torch.nn.Parameter(p.detach().clone()) for p in params], lr=1.0, state_bits=bits)
    again.load_state_dict(theirs.state_dict())
    assert all(torch.equal(a, b) for a, b in zip(mine.flat_moments(), again.flat_moments()))
    if bits == 8:
        assert torch.equal(mine.plan.m, again.plan.m) and torch.equal(mine.plan.v, again.plan.v)
    grads_for(params, 40)
    for p, q, r in zip(params, theirs.param_groups[0]["params"], again.param_groups[0]["params"]):
        q.grad, r.grad = p.grad.clone(), p.grad.clone()
    mine.step(), theirs.step(), again.step()
    for p, q, r in zip(params, theirs.param_groups[0]["params"], again.param_groups[0]["params"]):
        assert torch.equal(p, r)
        # both round p * decay and the update of at most lr * sqrt(10) or so a few times: 16 roundings of |p| + 0.01 leave room for either order
        assert bool(((p - q).abs() <= 16 * U * (p.abs() + 0.01)).all())


def test_a_captured_step_replays_as_the_next_one():
    from mmearth_train_amd.optim import AdamW
    for bits in (32, 8):
        params, eager = params_of([700, 9000], DT[:2], 11), params_of([700, 9000], DT[:2], 11)
        a, b = (AdamW(ps, lr=1e-3, state_bits=bits, max_norm=0.7) for ps in (params, eager))
        for ps in (params, eager):
            grads_for(ps, 50)
        a.step(), b.step()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            a.step()
        for k in range(4):
            for p, q in zip(params, eager):
                q.grad.normal_(generator=torch.Generator("cuda").manual_seed(60 + k))
                p.grad.copy_(q.grad)
            graph.replay()
            b.step()
            torch.cuda.synchronize()
            assert torch.equal(a.plan.steps, b.plan.steps)
            assert all(torch.equal(p, q) for p, q in zip(params, eager))
            assert all(torch.equal(x, y) for x, y in zip(a.flat_moments(), b.flat_moments()))
            torch.zeros(1 << 20, device="cuda").sum().item()


def test_state_must_exist_before_a_capture():
    from mmearth_train_amd.optim import AdamW
    params = params_of([10], DT[:1], 12)
    grads_for(params, 1)
    opt = AdamW(params)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager step"):
        with torch.cuda.graph(graph):
            opt.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_edges_of_the_settings(bits):
    """betas of 0, eps of 0 and tiny, a decay, one element: the update of the definition."""
    from mmearth_train_amd.optim import AdamW
    for betas, eps in (((0.0, 0.0), 1e-8), ((0.9, 0.999), 0.0), ((0.9, 0.999), 1e-20), ((0.0, 0.5), 1e-3)):
        params = params_of([1, 700], DT[:1], 18)
        refs = [Ref(p, bits) for p in params]
        opt = AdamW(params, lr=1e-3, betas=betas, eps=eps, weight_decay=0.3, state_bits=bits)
        run_steps(opt, params, refs, 3)
        check(opt, params, refs, bits)


def test_own_stream_and_determinism():
    from mmearth_train_amd.optim import AdamW
    got = []
    for k in range(2):
        params = params_of(SIZES, DT, 13)
        opt = AdamW(params, state_bits=8, max_norm=0.1)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for i in range(3):
                grads_for(params, 70 + i)
                opt.step()
        torch.cuda.current_stream().wait_stream(s)
        got.append([p.detach().clone() for p in params] + list(opt.flat_moments()) + [opt.grad_norm.clone()])
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("bits", [32, 8])
def test_groups_added_later_and_schedulers(bits):
    from mmearth_train_amd.optim import AdamW
    params = params_of([500, 300, 1000], DT[:1], 14)
    refs = [Ref(p, bits) for p in params]
    opt = AdamW(params[:2], lr=1e-3, state_bits=bits)
    sched = torch.optim.lr_scheduler.StepLR(opt, 1, 0.5)
    run_steps(opt, params[:2], refs, 2)
    sched.step()
    assert opt.param_groups[0]["lr"] == 5e-4
    opt.add_param_group({"params": [params[2]], "lr": 1e-2})
    run_steps(opt, params, refs, 2)
    check(opt, params, refs, bits)
    assert opt.plan.steps.tolist() == [4, 4, 2]
    with pytest.raises(ValueError, match="more than one parameter group|twice"):
        opt.add_param_group({"params": [params[0]]})
    assert len(opt.param_groups) == 2


def test_refusals_on_the_device():
    from mmearth_train_amd.optim import AdamW
    x = torch.zeros(64, device="cuda")
    mk = torch.nn.Parameter
    with pytest.raises(ValueError, match="share memory"):
        AdamW([mk(x[:40]), mk(x[30:])])
    with pytest.raises(ValueError, match="densely"):
        AdamW([mk(x[::2])])
    with pytest.raises(ValueError, match="twice"):
        p = mk(x)
        AdamW([p, p])
    p = mk(torch.zeros(8, device="cuda"))
    opt = AdamW([p, mk(torch.zeros(0, device="cuda"))])
    opt.step()                                          # no gradient anywhere: nothing happens
    assert opt.state_dict()["state"] == {}
    p.grad = torch.ones(8, device="cuda")
    opt.step()
    p.data = torch.zeros(9, device="cuda")
    p.grad = None
    with pytest.raises(ValueError, match="another size"):
        opt.step()
    e = torch.nn.Embedding(4, 4, sparse=True).cuda()
    e(torch.tensor([1], device="cuda")).sum().backward()
    with pytest.raises(ValueError, match="sparse"):
        AdamW(e.parameters()).step()
    with pytest.raises(RuntimeError, match="max_norm"):
        opt.grad_norm
    with pytest.raises(TypeError, match="state_dict"):
        import copy
        copy.deepcopy(opt)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_tensor_longer_than_31_bits(bits):
    """Element offsets past 2^31: the last elements against a small tensor that holds the same values in the same block places."""
    from mmearth_train_amd.optim import AdamW
    n, tail = 2 ** 31 + 5003, 5003 + 256
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device="cuda"))
    p.grad = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    start = 2 ** 31 - 256
    small = params_of([tail], DT[1:2], 15)
    grads_for(small, 16)
    p.data[start:] = small[0].data
    p.grad[start:] = small[0].grad
    a, b = AdamW([p], state_bits=bits, max_norm=0.5), AdamW(small, state_bits=bits, max_norm=0.5)
    for _ in range(2):
        a.step()
        b.step()
    assert torch.equal(a.grad_norm, b.grad_norm)
    assert torch.equal(p.data[start:], small[0].data) and not bool(p.data[:start].any())
    if bits == 8:
        assert torch.equal(a.plan.m[start:start + tail], b.plan.m[:tail]) and torch.equal(a.plan.v[start:start + tail], b.plan.v[:tail])
    else:
        assert torch.equal(a.plan.m[start:start + tail], b.plan.m[:tail]) and torch.equal(a.plan.v[start:start + tail], b.plan.v[:tail])


def test_autograd_notices_the_update():
    """A step between forward and backward of a graph that saved the parameter is an error, as with torch's own optimizers."""
    from mmearth_train_amd.optim import AdamW
    w = torch.nn.Parameter(torch.randn(4, 4, device="cuda"))
    x = torch.randn(4, 4, device="cuda", requires_grad=True)
    w.grad = torch.ones_like(w)
    y = (x @ w).sum()
    AdamW([w]).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    y = (x @ w).sum()
    AdamW([w]).flat_moments()                # (making the state writes no parameter)
    y.backward()


def test_a_step_beside_a_live_graph_of_the_same_leaves():
    """Backward under capture while an eager graph of the same parameters is alive is not this optimizer's business; its own capture is."""
    from mmearth_train_amd.optim import AdamW
    w = torch.nn.Parameter(torch.randn(64, 64, device="cuda"))
    opt = AdamW([w], lr=1e-2)
    (w * w).sum().backward()
    opt.step()
    alive = (w * w).sum()                    # an eager graph over w that nothing ever runs backward
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    before = w.detach().clone()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
    assert not torch.equal(before, w) and opt.plan.steps.tolist() == [4] and alive.requires_grad


@pytest.mark.parametrize("opt", ["adamw", "adamw8bit"])
def test_main_pretrain_trains_and_resumes_with_it(opt, tmp_path):
    """--fast_path False --opt adamw / adamw8bit --clip_grad: two epochs, the second one resumed from the first one's checkpoint."""
    import main_pretrain
    common = ["--model", "convnextv2_atto", "--input_size", "56", "--patch_size", "8", "--batch_size", "2", "--update_freq", "2", "--steps_per_epoch", "4",
              "--lr", "1e-3", "--norm_pix_loss", "True", "--fast_path", "False", "--out_modalities", "pix_mod", "--opt", opt, "--clip_grad", "1.0",
              "--warmup_epochs", "0", "--output_dir", str(tmp_path)]
    for epochs in ("1", "2"):
        stats = main_pretrain.main(main_pretrain.get_args_parser().parse_args(common + ["--epochs", epochs]))
        assert math.isfinite(stats[0]["loss"])
    ck = [torch.load(tmp_path / f"checkpoint-{i}.pth", map_location="cpu", weights_only=False) for i in (0, 1)]
    assert [float(c["optimizer"]["state"][0]["step"]) for c in ck] == [2.0, 4.0]
    assert not torch.equal(ck[0]["model"]["proj.weight"], ck[1]["model"]["proj.weight"])


def test_main_pretrain_refuses_settings_that_would_do_nothing():
    import main_pretrain
    base = ["--model", "convnextv2_atto", "--input_size", "56", "--patch_size", "8"]
    for extra in (["--opt", "adamw"], ["--clip_grad", "1.0"], ["--fast_path", "False", "--clip_grad", "1.0"]):
        with pytest.raises(ValueError, match="--opt|--clip_grad"):
            main_pretrain.main(main_pretrain.get_args_parser().parse_args(base + extra))


def test_parameters_that_move_in_memory():
    """`p.data = other`: the step follows the parameter; a capture right after it is refused (the device table has to be written first)."""
    from mmearth_train_amd.optim import AdamW
    params, twin = params_of([300, 5000], DT[:2], 17), params_of([300, 5000], DT[:2], 17)
    a, b = AdamW(params, state_bits=8), AdamW(twin, state_bits=8)
    for k in range(3):
        for ps in (params, twin):
            grads_for(ps, 80 + k)
        old = params[1].data
        if k:
            params[1].data = old.clone()
        kept = old.clone()
        a.step(), b.step()
        assert all(torch.equal(p, q) for p, q in zip(params, twin))
        assert k == 0 or torch.equal(old, kept)
    params[0].data = params[0].data.clone()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="moved"):
        with torch.cuda.graph(graph):
            a.step()
    a.step(), b.step()
    assert all(torch.equal(p, q) for p, q in zip(params, twin))
    x = torch.zeros(600, device="cuda")
    p, q = torch.nn.Parameter(x[:300]), torch.nn.Parameter(torch.zeros(300, device="cuda"))
    c = AdamW([p, q])
    p.grad, q.grad = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
    c.step()
    q.data = x[100:400]
    with pytest.raises(ValueError, match="share memory"):
        c.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_another_element_order_is_refused(bits):
    """The moments lie in the parameter's element order of the first step: a parameter that is laid out anew afterwards is not updated with misplaced ones."""
    from mmearth_train_amd.optim import AdamW
    w = torch.nn.Parameter(torch.randn(6, 4, 3, 3, device="cuda"))
    w.grad = torch.randn_like(w)
    opt = AdamW([w], state_bits=bits)
    opt.step()
    w.data = w.data.contiguous(memory_format=torch.channels_last)
    before = w.detach().clone()
    with pytest.raises(ValueError, match="another order"):
        opt.step()
    assert torch.equal(before, w)
    w.data = w.data.contiguous()
    opt.step()
    assert opt.plan.steps.tolist() == [2]


@pytest.mark.parametrize("bits", [32, 8])
def test_loading_views_of_the_state_itself_and_lists_with_holes(bits):
    from mmearth_train_amd.optim import AdamW
    params = params_of([300, 700, 5], DT[:1], 19)
    opt = AdamW([{"params": []}, {"params": params}], state_bits=bits)
    grads_for(params, 1)
    params[1].grad = None
    opt.step()
    sd = opt.state_dict()
    assert sorted(sd["state"]) == [0, 2]
    m, v = opt.flat_moments()
    keep = m.clone(), v.clone()
    for i in (0, 2):
        o, n = opt.offsets[i], params[i].numel()
        sd["state"][i]["exp_avg"], sd["state"][i]["exp_avg_sq"] = m[o:o + n], v[o:o + n]
    opt.load_state_dict(sd)
    assert all(torch.equal(a, b) for a, b in zip(keep, opt.flat_moments())) and opt.plan.steps.tolist() == [1, 0, 1]
    grads_for(params, 2)
    opt.step()
    opt.load_state_dict(sd | {"state": {0: sd["state"][0]}})
    m, v = opt.flat_moments()
    assert not m[opt.offsets[1]:].any() and not v[opt.offsets[1]:].any() and opt.plan.steps.tolist() == [1, 0, 0]


@pytest.mark.parametrize("bits", [32, 8])
def test_a_parameter_laid_out_anew_keeps_its_moments_in_place(bits):
    """Its moments stay in the order of the first step: in a checkpoint, and a list that grows does not take them over misplaced."""
    from mmearth_train_amd.optim import AdamW
    w, more = torch.nn.Parameter(torch.randn(6, 4, 3, 3, device="cuda")), torch.nn.Parameter(torch.randn(40, device="cuda"))
    w.grad = torch.randn_like(w)
    opt = AdamW([w], state_bits=bits)
    opt.step()
    before = opt.state_dict()["state"][0]
    w.data = w.data.contiguous(memory_format=torch.channels_last)
    after = opt.state_dict()["state"][0]
    assert torch.equal(before["exp_avg"], after["exp_avg"]) and torch.equal(before["exp_avg_sq"], after["exp_avg_sq"])
    with pytest.raises(ValueError, match="another order"):
        opt.add_param_group({"params": [more]})
    assert len(opt.param_groups) == 1
    w.data = w.data.contiguous()
    opt.add_param_group({"params": [more]})
    more.grad = torch.ones_like(more)
    opt.step()
    assert opt.plan.steps.tolist() == [2, 1]


def test_edited_lists_are_refused():
    from mmearth_train_amd.optim import AdamW
    a, b = (torch.nn.Parameter(torch.ones(300, device="cuda")) for _ in range(2))
    a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
    opt = AdamW([{"params": [a]}, {"params": []}])
    opt.step()
    opt.param_groups[0]["params"].append(b)
    with pytest.raises(RuntimeError, match="add_param_group"):
        opt.step()
    assert torch.equal(b, torch.ones_like(b))
    opt.param_groups[0]["params"].pop()
    opt.step()
    assert opt.plan.steps.tolist() == [2]


@pytest.mark.parametrize("bits", [32, 8])
def test_a_refused_step_does_not_lose_what_has_moved(bits):
    """A parameter moves and a later one's gradient is refused: once that is put right, the step writes the new memory and leaves the old."""
    from mmearth_train_amd.optim import AdamW
    params, twin = params_of([300, 5000], DT[:1], 20), params_of([300, 5000], DT[:1], 20)
    a, b = AdamW(params, state_bits=bits), AdamW(twin, state_bits=bits)
    for ps in (params, twin):
        grads_for(ps, 90)
    a.step(), b.step()
    old = params[0].data
    kept = old.clone()
    params[0].data = old.clone()
    good = params[1].grad
    params[1].grad = good.to_sparse()
    with pytest.raises(ValueError, match="parameter 1 has a sparse"):
        a.step()
    params[1].grad = good
    a.step(), b.step()
    assert torch.equal(old, kept) and all(torch.equal(p, q) for p, q in zip(params, twin)) and a.plan.steps.tolist() == [2, 2]


def test_replaced_and_exchanged_parameters_are_refused():
    """Lists of the same lengths that hold other parameters: nothing is updated, nothing saved or loaded under a wrong index."""
    from mmearth_train_amd.optim import AdamW
    a, b, new = (torch.nn.Parameter(torch.ones(300, device="cuda")) for _ in range(3))
    for p in (a, b, new):
        p.grad = torch.ones_like(p)
    opt = AdamW([{"params": [a], "lr": 1e-3}, {"params": [b], "lr": 1e-1}])
    opt.step()
    keep = [p.detach().clone() for p in (a, b, new)]
    one, two = opt.param_groups
    saved = opt.state_dict()

    def put(x, y):
        one["params"][0], two["params"][0] = x, y

    for x, y in ((new, b), (b, a)):
        put(x, y)
        for call in (opt.step, opt.state_dict, opt.flat_moments, lambda: opt.load_state_dict(saved), lambda: opt.add_param_group({"params": [new]})):
            with pytest.raises(RuntimeError, match="add_param_group"):
                call()
        assert all(torch.equal(p, q) for p, q in zip((a, b, new), keep)) and len(opt.param_groups) == 2
    put(a, b)
    opt.param_groups.reverse()
    with pytest.raises(RuntimeError, match="add_param_group"):
        opt.step()
    opt.param_groups.reverse()
    opt.step()
    assert opt.plan.steps.tolist() == [2, 2]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("size", [1e18, 1e20, 1e22, 1e30, 1e34])
@pytest.mark.parametrize("types", [DT[:1], DT[1:2]], ids=["fp32", "bf16"])
def test_clip_of_large_finite_norms(bits, size, types):
    """coef * g is an ordinary number, coef^2 and g^2 are not: the moments take the clipped gradient's square, on the first step and after."""
    from mmearth_train_amd.optim import AdamW
    params = params_of([257, 4100], types, 21)
    refs = [Ref(p, bits) for p in params]
    opt = AdamW(params, lr=1e-3, state_bits=bits, max_norm=1.0)
    for k in range(2):
        grads_for(params, 110 + k, scale=size)
        norm = math.sqrt(sum(float(p.grad.double().square().sum()) for p in params))
        coef = float(np.float32(min(1.0, 1.0 / (norm + 1e-6))))
        opt.step()
        assert float(opt.skipped) == 0.0 and abs(float(opt.grad_norm) - norm) <= 2 * U * norm
        for p, r in zip(params, refs):
            r.step(p.grad, coef, 1e-3, 0.9, 0.999, 1e-8, 1e-2)
    check(opt, params, refs, bits)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_norm_past_the_range_of_fp32_skips_the_step(bits):
    """Every element finite, the norm not a number of fp32: `grad_norm` reads infinity, `skipped` 1, and nothing has changed."""
    from mmearth_train_amd.optim import AdamW
    params = params_of([300, 5000], DT[:2], 22)
    opt = AdamW(params, state_bits=bits, max_norm=1.0)
    grads_for(params, 1)
    opt.step()
    keep = [p.detach().clone() for p in params], [x.clone() for x in opt.flat_moments()], opt.plan.steps.clone()
    for p in params:
        p.grad.fill_(1e37)                                     # 5300 of them: a norm of 7.3e38
    opt.step()
    assert float(opt.skipped) == 1.0 and float(opt.grad_norm) == float("inf")
    assert all(torch.equal(a, b.detach()) for a, b in zip(keep[0], params))
    assert all(torch.equal(a, b) for a, b in zip(keep[1], opt.flat_moments())) and torch.equal(keep[2], opt.plan.steps)


@pytest.mark.parametrize("bits", [32, 8])
def test_no_group_is_added_behind_a_captured_step(bits):
    """A longer list takes new buffers; a graph would go on writing the old, freed ones. The refusal leaves optimizer and graph as they were."""
    from mmearth_train_amd.optim import AdamW
    params, twin = params_of([700, 300, 40], DT[:1], 23), params_of([700, 300, 40], DT[:1], 23)
    a, b = AdamW(params[:2], state_bits=bits), AdamW(twin[:2], state_bits=bits)
    for ps in (params, twin):
        grads_for(ps, 120)
    a.step(), b.step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        a.step()
    with pytest.raises(RuntimeError, match="captured"):
        a.add_param_group({"params": [params[2]]})
    assert len(a.param_groups) == 1
    for _ in range(2):
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(params, twin))
        assert all(torch.equal(x, y) for x, y in zip(a.flat_moments(), b.flat_moments()))
    b.add_param_group({"params": [twin[2]]})                   # (nothing was captured here)
    b.step()
    assert b.plan.steps.tolist() == [4, 4, 1]


@pytest.mark.parametrize("bits", [32, 8])
def test_a_group_added_on_another_stream(bits):
    """The old state is read on that stream and freed on the first one's: the reads are done when the call returns, and the values are the ones they were."""
    from mmearth_train_amd.optim import AdamW
    params = params_of([5_000_000, 300], DT[:1], 24)
    opt = AdamW(params[:1], state_bits=bits)
    grads_for(params, 130)
    opt.step()
    m, v = (x.clone() for x in opt.flat_moments())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        opt.add_param_group({"params": params[1:]})
        assert s.query()
    fill = [torch.full_like(x, 7.0) for x in (m, v) for _ in range(2)]
    assert all(torch.equal(x[:5_000_000], y[:5_000_000]) for x, y in zip((m, v), opt.flat_moments())) and len(fill) == 4
    assert opt.plan.steps.tolist() == [1, 0]


@pytest.mark.parametrize("bits", [32, 8])
def test_a_refused_checkpoint_changes_nothing(bits):
    from mmearth_train_amd.optim import AdamW
    params = params_of([300, 700], DT[:1], 25)
    opt = AdamW(params, lr=1e-3, state_bits=bits)
    grads_for(params, 140)
    opt.step()
    keep = [x.clone() for x in opt.flat_moments()]

    def spoiled(i, key, value):
        sd = opt.state_dict()
        sd["param_groups"][0]["lr"] = 5.0
        for st in sd["state"].values():
            st["exp_avg"] = st["exp_avg"] + 1.0
        if value is None:
            del sd["state"][i][key]
        else:
            sd["state"][i][key] = value
        return sd

    for i, key, value in ((1, "step", None), (1, "step", torch.tensor(float("nan"))), (1, "step", -1), (0, "step", 2.5), (1, "step", 2.0 ** 31), (1, "exp_avg_sq", None),
                          (1, "exp_avg_sq", torch.zeros(699, device="cuda")), (0, "exp_avg", 3.0), (0, "exp_avg", torch.zeros(300, dtype=torch.complex64))):
        with pytest.raises(ValueError, match="loaded"):
            opt.load_state_dict(spoiled(i, key, value))
        assert opt.param_groups[0]["lr"] == 1e-3 and opt.plan.steps.tolist() == [1, 1]
        assert all(torch.equal(a, b) for a, b in zip(keep, opt.flat_moments())), (i, key)


def test_hooks_of_checkpoints_run():
    from mmearth_train_amd.optim import AdamW
    params = params_of([30], DT[:1], 26)
    opt, seen = AdamW(params), []
    grads_for(params, 150)
    opt.step()
    opt.register_state_dict_pre_hook(lambda o: seen.append("before"))
    opt.register_state_dict_post_hook(lambda o, sd: {**sd, "note": 3})
    opt.register_load_state_dict_pre_hook(lambda o, sd: (seen.append(sd["note"]), {k: v for k, v in sd.items() if k != "note"})[1])
    opt.register_load_state_dict_post_hook(lambda o: seen.append("after"))
    opt.load_state_dict(opt.state_dict())
    assert seen == ["before", 3, "after"] and opt.plan.steps.tolist() == [1]


def test_settings_of_the_whole_optimizer_are_fixed():
    from mmearth_train_amd.optim import AdamW
    opt = AdamW(params_of([30], DT[:1], 27), state_bits=8, max_norm=0.5)
    assert opt.state_bits == 8 and opt.max_norm == 0.5
    for name, value in (("max_norm", 1.0), ("state_bits", 32)):
        with pytest.raises(AttributeError):
            setattr(opt, name, value)
    assert opt.state_bits == 8 and opt.max_norm == 0.5


def test_settings_changed_to_impossible_ones_are_refused():
    from mmearth_train_amd.optim import AdamW
    params = params_of([300], DT[:1], 28)
    opt = AdamW(params, lr=1e-3)
    grads_for(params, 160)
    opt.step()
    keep = params[0].detach().clone()
    for key, value, what in (("betas", (1.0, 0.999), "betas"), ("lr", float("nan"), "lr"), ("lr", -1.0, "lr"), ("eps", float("inf"), "eps"), ("weight_decay", -1.0, "weight_decay")):
        old = opt.param_groups[0][key]
        opt.param_groups[0][key] = value
        with pytest.raises(ValueError, match=what):
            opt.step()
        opt.param_groups[0][key] = old
        assert torch.equal(keep, params[0].detach()) and opt.plan.steps.tolist() == [1]
    opt.step()
    assert opt.plan.steps.tolist() == [2]


def test_settings_of_any_numeric_type():
    """What a configuration or a scheduler puts into the groups: numpy numbers, betas as a list or an array; what is no number is refused with its own error."""
    from mmearth_train_amd.optim import AdamW
    params, twin = params_of([300], DT[:1], 29), params_of([300], DT[:1], 29)
    a, b = AdamW(params, lr=1e-3, betas=(0.9, 0.99)), AdamW(twin, lr=1e-3, betas=(0.9, 0.99))
    for ps in (params, twin):
        grads_for(ps, 170)
    for betas in ([0.9, 0.99], np.array([0.9, 0.99]), iter_twice(0.9, 0.99)):
        a.param_groups[0].update(lr=np.float64(1e-3), betas=betas, weight_decay=np.float64(1e-2))
        a.step(), b.step()
        assert torch.equal(params[0], twin[0])
    for key, value, error in (("betas", (0.9,), ValueError), ("betas", 0.9, TypeError), ("lr", "fast", TypeError), ("lr", torch.tensor(1e-3), ValueError), ("eps", None, TypeError)):
        old = a.param_groups[0][key]
        a.param_groups[0][key] = value
        with pytest.raises(error):
            a.step()
        a.param_groups[0][key] = old
    del a.param_groups[0]["eps"]
    with pytest.raises(KeyError, match="eps"):
        a.step()
    assert a.plan.steps.tolist() == [3] and torch.equal(params[0], twin[0])


def iter_twice(*numbers):
    """A sequence that is neither a list nor a tuple."""
    class Seq:
        def __len__(self):
            return len(numbers)

        def __getitem__(self, i):
            return numbers[i]
    return Seq()


def test_an_empty_entry_of_a_checkpoint_is_none():
    """`optimizer.state[p]` on torch's own class makes one for a parameter that was never stepped."""
    from mmearth_train_amd.optim import AdamW
    params = params_of([30, 40], DT[:1], 30)
    theirs = torch.optim.AdamW([torch.nn.Parameter(p.detach().clone()) for p in params])
    p, q = theirs.param_groups[0]["params"]
    p.grad = torch.ones_like(p)
    theirs.step()
    assert theirs.state[q] == {}
    opt = AdamW(params)
    opt.load_state_dict(theirs.state_dict())
    assert opt.plan.steps.tolist() == [1, 0] and sorted(opt.state_dict()["state"]) == [0]
