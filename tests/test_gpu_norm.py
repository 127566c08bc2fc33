"""Group norm with an activation on channels-last maps against its definition in float64, its gradients against the
formula and against differences, and the head towers that run on it."""
from functools import partial

import pytest
import torch
from torch import nn

from object_detection_amd import _C
from object_detection_amd.norm import GroupNormAct, group_norm_act

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# Roundings a value passes on its way: a thread adds at most 64 pixels in these tests, the rows of a workgroup, the chunks
# and the channels of a group are added behind them (below 64 more), normalising and the two averages take a dozen; the
# spread of the sums by the thread's own shift costs a factor of two.  256 half steps of fp32 cover that.
CHAIN = 256 * U32


def _ref(x, groups, gamma, beta, eps, act, dy=None):
    """(y, u, xhat, mean, rstd[, dx, dgamma, dbeta]) in float64 for x [B, C, H, W]."""
    B, C, H, W = x.shape
    v = x.double().reshape(B, groups, -1)
    mean = v.mean(dim=2, keepdim=True)
    rstd = ((v - mean).pow(2).mean(dim=2, keepdim=True) + eps).rsqrt()
    xhat = ((v - mean) * rstd).view(B, C, H, W)
    g = torch.ones(C, dtype=torch.float64, device=x.device) if gamma is None else gamma.double()
    b = torch.zeros(C, dtype=torch.float64, device=x.device) if beta is None else beta.double()
    g, b = g.view(1, C, 1, 1), b.view(1, C, 1, 1)
    u = xhat * g + b
    s = torch.sigmoid(u)
    y = {"none": u, "relu": u.clamp(min=0), "silu": u * s}[act]
    spread = (1.0 / rstd).expand(B, groups, C // groups).reshape(B, C, 1, 1)
    out = dict(y=y, u=u, xhat=xhat, rstd=(1.0 / spread), scale=(xhat.abs() + 1.0) * g.abs() + b.abs(), g=g)
    if dy is not None:
        du = dy.double() * {"none": torch.ones_like(u), "relu": (u > 0).double(), "silu": s * (1 + u * (1 - s))}[act]

        def avg(t):
            return t.reshape(B, groups, -1).mean(dim=2).repeat_interleave(C // groups, dim=1).view(B, C, 1, 1)
        out.update(dx=out["rstd"] * (g * du - avg(g * du) - xhat * avg(g * du * xhat)),
                   dx_scale=out["rstd"] * (1 + xhat.abs()) * ((g * du).abs() + avg((g * du).abs())
                                                              + avg((g * du * xhat).abs())),
                   dgamma=(du * xhat).sum(dim=(0, 2, 3)), dbeta=du.sum(dim=(0, 2, 3)),
                   dgamma_scale=(dy.double().abs() * 1.1 * (xhat.abs() + 1)).sum(dim=(0, 2, 3)),
                   dbeta_scale=(dy.double().abs() * 1.1 * (1 + xhat.abs())).sum(dim=(0, 2, 3)))
    return out


def _close(got, want, tol, what):
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"{what}: off by {float((err - tol).max())} more than allowed, {float(err.max())} in all"


def _case(device, B, C, H, W, groups, act, dtype, affine, seed, pdtype=torch.float32, offset=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn((B, C, H, W), generator=gen) * (0.5 + torch.rand((1, C, 1, 1), generator=gen))
         + offset * torch.randn((1, C, 1, 1), generator=gen)).to(device, dtype)
    dy = torch.randn((B, C, H, W), generator=gen).to(device, dtype)
    gamma = (torch.rand((C,), generator=gen) + 0.5).to(device, pdtype) if affine else None
    beta = (torch.randn((C,), generator=gen) * 0.3).to(device, pdtype) if affine else None
    # a value next to the rectifier's corner may fall on either side of it: no gradient arrives there
    if act == "relu":
        r = _ref(x, groups, gamma, beta, 1e-5, act)
        dy = torch.where(r["u"].abs() < 1e-3 * r["scale"], torch.zeros_like(dy), dy)
    return x, dy, gamma, beta


def _check(x, dy, groups, gamma, beta, act, eps=1e-5):
    dtype, C = x.dtype, x.shape[1]
    xl = x.clone(memory_format=torch.preserve_format).requires_grad_(True)
    leaves = [xl] + [p.clone().requires_grad_(True) for p in (gamma, beta) if p is not None]
    y = group_norm_act(xl, groups, *(leaves[1:] if gamma is not None else (None, None)), eps, act)
    assert y.dtype == dtype and y.shape == x.shape and y.permute(0, 2, 3, 1).is_contiguous()
    grads = torch.autograd.grad(y, leaves, dy)
    r = _ref(x, groups, gamma, beta, eps, act, dy)
    # the hardware exponential and reciprocal of silu: a relative 2^-20 of the value at the arguments met here
    more = 2.0 ** -20 if act == "silu" else 0.0
    _close(y.detach(), r["y"], HALF[dtype] * r["y"].abs() * 1.01 + (CHAIN + more) * r["scale"] + 1e-7 * (dtype == torch.float16), "y")
    _close(grads[0], r["dx"], HALF[dtype] * r["dx"].abs() * 1.01 + (CHAIN + 4 * more) * r["dx_scale"]
           + 1e-7 * (dtype == torch.float16), "dx")
    if gamma is not None:
        half = HALF[gamma.dtype]
        _close(grads[1], r["dgamma"], half * r["dgamma"].abs() * 1.01 + (CHAIN + more) * r["dgamma_scale"], "dgamma")
        _close(grads[2], r["dbeta"], half * r["dbeta"].abs() * 1.01 + (CHAIN + more) * r["dbeta_scale"], "dbeta")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,C,H,W,groups,act,affine", [
    (2, 256, 8, 8, 32, "relu", True),          # coarse pyramid level: the one-launch form
    (3, 256, 32, 32, 32, "relu", True),
    (2, 256, 64, 64, 32, "silu", True),        # the two-pass form
    (1, 96, 61, 47, 12, "silu", True),         # sizes that divide nothing
    (2, 24, 33, 5, 8, "relu", True),           # groups of 3 channels: vectors across group borders
    (2, 7, 9, 11, 7, "none", True),            # one channel a group, scalar accesses
    (5, 12, 3, 3, 4, "relu", False),
    (1, 48, 1, 1, 4, "none", True),            # one pixel
    (1, 512, 40, 40, 1, "silu", True),         # one group
    (2, 2048, 7, 3, 32, "relu", True),         # the channel limit
    (1, 300, 70, 70, 300, "relu", True),       # more groups than a workgroup has threads
])
def test_group_norm_act_matches_definition(device, B, C, H, W, groups, act, affine, dtype):
    x, dy, gamma, beta = _case(device, B, C, H, W, groups, act, dtype, affine, seed=B * 1000 + C + H)
    _check(x.contiguous(memory_format=torch.channels_last), dy.contiguous(memory_format=torch.channels_last), groups, gamma,
           beta, act)


def test_many_images_of_many_groups(device):
    """More groups than threads, whose few chunks an image's own workgroups join."""
    x, dy, gamma, beta = _case(device, 300, 288, 33, 33, 288, "silu", torch.bfloat16, True, seed=17)
    _check(x.contiguous(memory_format=torch.channels_last), dy.contiguous(memory_format=torch.channels_last), 288, gamma, beta,
           "silu")


def test_offsets_past_32_bits(device):
    """An image of 2.3 G elements: a thread adds 6000 * 6000 / 256 / 32 = 4395 pixels, so that many half steps of fp32 more
    in the statistics (twice, by the thread's own shift) and in the sums of the gradients."""
    C, side, groups = 64, 6000, 4
    gen = torch.Generator(device=device).manual_seed(2)
    x = torch.empty((1, side, side, C), dtype=torch.bfloat16, device=device).normal_(0.5, 1.0, generator=gen)
    x = x.permute(0, 3, 1, 2).requires_grad_(True)
    y = group_norm_act(x, groups, None, None, 1e-5, "silu")
    dx = torch.autograd.grad(y, x, torch.ones_like(y))[0]
    per = C // groups
    chain = CHAIN + 2 * 4395 * U32
    for g in (0, groups - 1):
        v = x.detach()[:, g * per:(g + 1) * per]
        mean = v.mean(dtype=torch.float64)
        parts = [v[:, c].double() for c in range(per)]
        rstd = (sum((q - mean).pow(2).sum() for q in parts) / (per * side * side) + 1e-5).rsqrt()
        a = b = 0.0
        for q in parts:
            h = (q - mean) * rstd
            s = torch.sigmoid(h)
            du = s * (1 + h * (1 - s))
            a, b = a + du.sum() / (per * side * side), b + (du * h).sum() / (per * side * side)
        for rows in (slice(0, 2), slice(side - 2, side)):
            h = (v[:, :, rows].double() - mean) * rstd
            s = torch.sigmoid(h)
            _close(y.detach()[:, g * per:(g + 1) * per, rows], h * s,
                   2.0 ** -8 * (h * s).abs() * 1.01 + (chain + 2.0 ** -20) * (h.abs() + 1), "y")
            want = rstd * (s * (1 + h * (1 - s)) - a - h * b)
            _close(dx[:, g * per:(g + 1) * per, rows], want,
                   2.0 ** -8 * want.abs() * 1.01 + (chain + 2.0 ** -18) * rstd * (1 + h.abs()) * 3, "dx")


@pytest.mark.parametrize("pdtype", [torch.float16, torch.bfloat16])
def test_parameter_types_and_memory_orders(device, pdtype):
    x, dy, gamma, beta = _case(device, 2, 64, 12, 10, 8, "relu", torch.bfloat16, True, seed=5, pdtype=pdtype)
    _check(x, dy, 8, gamma, beta, "relu")                                          # NCHW
    _check(x.transpose(2, 3), dy.transpose(2, 3), 8, gamma, beta, "relu")          # width before height
    wide = torch.zeros((2, 80, 12, 10), dtype=x.dtype, device=device).contiguous(memory_format=torch.channels_last)
    wide[:, 8:72] = x
    _check(wide[:, 8:72], dy, 8, gamma, beta, "relu")                              # a slice of the channels
    flat = torch.zeros(x.numel() + 1, dtype=x.dtype, device=device)                # rows off the 16-byte grid
    odd = flat[1:].view(2, 12, 10, 64).permute(0, 3, 1, 2)
    odd.copy_(x)
    _check(odd, dy, 8, gamma[1:].clone().new_tensor(gamma.tolist()), beta, "relu")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_offset_far_above_the_spread(device, dtype):
    """Mean 300 times the spread: the statistics must not come from a difference of large sums."""
    gen = torch.Generator().manual_seed(9)
    x = (300.0 + torch.randn((2, 64, 50, 50), generator=gen)).to(device, dtype).contiguous(memory_format=torch.channels_last)
    x[0, 0, 0, 0] = -5000.0                                                          # an outlier in a shift's place
    y = group_norm_act(x, 8, None, None, 1e-5, "none")
    r = _ref(x, 8, None, None, 1e-5, "none")
    # what the kernel subtracts is the mean rounded to fp32, 302 * 2^-24 of the spread's units at most; 1/std comes from the
    # outlier's own thread among others, whose mean is 5300 / 64 off its shift: a factor n = 64 on its half steps
    tol = HALF[dtype] * r["y"].abs() * 1.01 + CHAIN * r["scale"] + 64 * CHAIN * r["xhat"].abs() + 302 * U32 * r["rstd"]
    _close(y, r["y"], tol, "y")


def test_rectifier_decides_as_64_bits_do(device):
    """A bf16 map holds few different values: at mean 0, 1/std 1 and a bias that is a value of the map, hundreds of pixels of
    a channel lie next to the corner, on the side that the statistics' last digits decide."""
    gen = torch.Generator().manual_seed(4)
    x = torch.randn((4, 32, 64, 64), generator=gen).to(device, torch.bfloat16).contiguous(memory_format=torch.channels_last)
    dy = torch.ones_like(x)
    gamma = torch.ones(32, device=device)
    for trial in range(4):
        v = x.double().reshape(4, 8, -1)
        mean, std = v.mean(2), (v.var(2, unbiased=False) + 1e-5).sqrt()
        at = x[trial, ::4, trial, trial].double()                                # a value of each group of image `trial`
        beta = -((at - mean[trial]) / std[trial]).repeat_interleave(4).float()   # u of that value: a rounding of zero
        xl, bl = x.clone(memory_format=torch.preserve_format).requires_grad_(True), beta.clone().requires_grad_(True)
        y = group_norm_act(xl, 8, gamma, bl)
        db = torch.autograd.grad(y, bl, dy)[0]
        u = (x.double() - mean.repeat_interleave(4, 1)[..., None, None]) / std.repeat_interleave(4, 1)[..., None, None] \
            + beta.double()[None, :, None, None]
        # the side of a value is certain where u is further from zero than the sums' own error, 64 additions of 2^-24
        # averaged over the 16384 * 4 values of a group: 1e-8
        low, high = (u > 1e-8).sum(dim=(0, 2, 3)), (u > -1e-8).sum(dim=(0, 2, 3))
        assert bool(((db >= low) & (db <= high)).all())
        assert int((u.abs() < 1e-6).sum()) > 100                                # and the case is there


def test_nan_and_inf_stay_in_their_group(device):
    x = torch.randn((2, 32, 9, 9), device=device).contiguous(memory_format=torch.channels_last)
    clean = group_norm_act(x, 4, None, None, 1e-5, "relu")
    x[1, 9, 3, 3] = float("nan")
    x[0, 30, 0, 0] = float("inf")
    y = group_norm_act(x, 4, None, None, 1e-5, "relu")
    bad = torch.zeros((2, 32), dtype=torch.bool, device=device)
    bad[1, 8:16] = True
    bad[0, 24:32] = True
    assert bool(y.isnan().all(dim=(2, 3)).eq(bad).all())
    assert torch.equal(y[~bad], clean[~bad])


def test_empty_maps_and_single_values(device):
    gamma = torch.ones(8, device=device, requires_grad=True)
    beta = torch.zeros(8, device=device, requires_grad=True)
    for shape in ((0, 8, 4, 4), (2, 8, 0, 4)):
        x = torch.zeros(shape, device=device, requires_grad=True)
        y = group_norm_act(x, 4, gamma, beta)
        dx, dg, db = torch.autograd.grad(y, [x, gamma, beta], torch.zeros_like(y))
        assert y.shape == dx.shape == torch.Size(shape) and not dg.any() and not db.any()
    x = torch.full((1, 4, 1, 1), 3.0, device=device, requires_grad=True)       # one value a group: nothing is left of it
    y = group_norm_act(x, 4, None, None, 1e-5, "none")
    assert not y.any() and not torch.autograd.grad(y.sum(), x)[0].any()


def test_gradient_against_differences(device):
    """Central differences of L = sum(y r) along the gradient itself (entries up to 1, step 1e-2).  Noise: 560 terms off by
    4e-6 / 1e-2 at most, 0.25 in all; the third derivative's term is below 1e-4 / 6 * 560 * 10 = 0.1; L' is above 100."""
    gen = torch.Generator().manual_seed(3)
    x = torch.randn((2, 8, 5, 7), generator=gen).to(device).contiguous(memory_format=torch.channels_last)
    r = torch.randn((2, 8, 5, 7), generator=gen).to(device)
    gamma = (torch.rand(8, generator=gen) + 0.5).to(device)
    beta = torch.randn(8, generator=gen).to(device)
    leaves = [t.clone().requires_grad_(True) for t in (x, gamma, beta)]
    grads = torch.autograd.grad((group_norm_act(leaves[0], 4, leaves[1], leaves[2], 1e-5, "silu") * r).sum(), leaves)

    def loss(*a):
        return float((group_norm_act(a[0], 4, a[1], a[2], 1e-5, "silu").double() * r.double()).sum())
    for k in range(3):
        v = grads[k] / grads[k].abs().max()
        args = [x, gamma, beta]
        up, down = list(args), list(args)
        up[k], down[k] = args[k] + 1e-2 * v, args[k] - 1e-2 * v
        slope = (loss(*up) - loss(*down)) / 2e-2
        want = float((grads[k].double() * v.double()).sum())
        assert abs(slope - want) <= 0.35, (k, slope, want)


def test_partial_gradients_and_repeated_results(device):
    x, dy, gamma, beta = _case(device, 4, 64, 60, 60, 8, "relu", torch.bfloat16, True, seed=11)
    x = x.contiguous(memory_format=torch.channels_last)
    xl, gl = x.clone().requires_grad_(True), gamma.clone().requires_grad_(True)
    full = torch.autograd.grad(group_norm_act(xl, 8, gl, beta), [xl, gl], dy)
    only = torch.autograd.grad(group_norm_act(x, 8, gl, beta), [gl], dy)[0]
    frozen = torch.autograd.grad(group_norm_act(xl, 8, gamma, beta), [xl], dy)[0]
    assert torch.equal(only, full[1]) and torch.equal(frozen, full[0])       # and the same bits every time
    with pytest.raises(RuntimeError, match="once_differentiable"):
        y = group_norm_act(xl, 8, gl, beta)
        g = torch.autograd.grad(y, xl, dy.clone().requires_grad_(True), create_graph=True)[0]
        g.sum().backward()


def test_refusals(device):
    x = torch.zeros((1, 8, 2, 2), device=device)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        group_norm_act(x.cpu(), 4)
    with pytest.raises(ValueError, match="groups"):
        group_norm_act(x, 3)
    with pytest.raises(ValueError, match="groups"):
        group_norm_act(x, 0)
    with pytest.raises(ValueError, match="map"):
        group_norm_act(x[0], 4)
    with pytest.raises(ValueError, match="activation"):
        group_norm_act(x, 4, activation="gelu")
    with pytest.raises(ValueError, match="eps"):
        group_norm_act(x, 4, eps=float("nan"))
    with pytest.raises(ValueError, match="weight must be"):
        group_norm_act(x, 4, torch.ones(4, device=device))
    with pytest.raises(RuntimeError, match="weight is on"):
        group_norm_act(x, 4, torch.ones(8))
    with pytest.raises(TypeError, match="bias"):
        group_norm_act(x, 4, torch.ones(8, device=device), torch.ones(8, device=device, dtype=torch.float16))
    with pytest.raises(TypeError, match="float64"):
        group_norm_act(x.double(), 4)
    with pytest.raises(_C.OdBoxesError, match="2048"):
        group_norm_act(torch.zeros((1, 4096, 1, 1), device=device), 4)


def test_another_stream_and_a_captured_step(device):
    x, dy, gamma, beta = _case(device, 2, 64, 40, 40, 8, "silu", torch.bfloat16, True, seed=21)
    x, dy = (t.contiguous(memory_format=torch.channels_last) for t in (x, dy))

    def step(x, g, b):
        y = group_norm_act(x, 8, g, b, 1e-5, "silu")
        return [y.detach()] + list(torch.autograd.grad(y, [x, g, b], dy))
    want = [t.clone() for t in step(*[t.clone().requires_grad_(True) for t in (x, gamma, beta)])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(*[t.clone().requires_grad_(True) for t in (x, gamma, beta)])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))

    from object_detection_amd.graph_step import capture
    leaves = [t.clone(memory_format=torch.preserve_format).requires_grad_(True) for t in (x, gamma, beta)]
    first, second = capture(lambda: step(*leaves), device), capture(lambda: step(*leaves), device)
    for k in range(3):                                # replays with eager work of the same operator between them
        with torch.no_grad():
            leaves[0].copy_(x + 0.25 * k)
        outs = [t.clone() for t in first.replay()]
        eager = step(*[t.detach().clone(memory_format=torch.preserve_format).requires_grad_(True) for t in leaves])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager))
        other = [t.clone() for t in second.replay()]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(other, eager))


@pytest.mark.parametrize("arch", ["retinanet", "fcos"])
def test_towers_of_the_models(device, arch):
    """The heads with the fused norm load the plain heads' checkpoints and give the plain heads' outputs, losses and
    gradients; both forms run in fp32 with every convolution in the same library, whose own choice of algorithm for the
    two memory orders is what the 1e-3 covers (four convolutions of 288 products each, 2^-24 * 288 * 4 = 7e-5 at most of
    the largest value, times the condition of the normalisation between them)."""
    from object_detection_amd.retinanet_model import get_model
    torch.manual_seed(0)
    kw = dict(arch=arch, backbone="pyramid_stub", out_channels=64, layers=[0, 1], min_size=128, max_size=128)
    plain = get_model(5, **kw).to(device)
    fused = get_model(5, norm_layer=partial(GroupNormAct, 32), **kw).to(device)
    assert sum(isinstance(m, GroupNormAct) for m in fused.modules()) == 8
    fused.load_state_dict(plain.state_dict())
    fused = fused.to(memory_format=torch.channels_last)
    gen = torch.Generator().manual_seed(1)
    images = [torch.rand((3, 128, 128), generator=gen).to(device) for _ in range(2)]
    targets = [{"boxes": torch.tensor([[10., 12., 60., 70.], [30., 40., 110., 120.]], device=device),
                "labels": torch.tensor([1, 3], device=device)} for _ in range(2)]
    a, b = plain.train()(images, targets), fused.train()(images, targets)
    for k in a:
        assert abs(float(a[k].detach()) - float(b[k].detach())) <= 1e-3 * max(1.0, abs(float(a[k].detach()))), k
    ga = torch.autograd.grad(sum(a.values()), list(plain.parameters()))
    gb = torch.autograd.grad(sum(b.values()), list(fused.parameters()))
    for (name, _), p, q in zip(plain.named_parameters(), ga, gb):
        assert float((p - q).abs().max()) <= 1e-2 * float(p.abs().max()) + 1e-7, name
    with torch.no_grad():
        feats = [torch.randn((2, 64, s, s), generator=gen).to(device) for s in (16, 8, 4)]
        pm, fm = plain.eval().head.forward_maps(feats), fused.eval().head.forward_maps(feats)
        for k in pm:
            for p, q in zip(pm[k], fm[k]):
                assert float((p - q).abs().max()) <= 1e-3 * max(1.0, float(p.abs().max())), k
        dp, df = plain(images), fused(images)
    assert len(dp) == len(df) == 2 and all(set(d) == {"boxes", "scores", "labels"} for d in df)


@pytest.mark.parametrize("arch", ["retinanet", "fcos"])
def test_channels_last_maps_are_selected_in_place(device, arch):
    """postprocess of channels-last maps equals postprocess of the same values in NCHW."""
    from object_detection_amd.retinanet_model import get_model
    torch.manual_seed(3)
    model = get_model(5, arch=arch, backbone="pyramid_stub", out_channels=32, layers=[0, 1], min_size=128, max_size=128,
                      score_thresh=0.3, norm_layer=partial(GroupNormAct, 32)).to(device).eval()
    images = [torch.rand((3, 128, 128), device=device) for _ in range(2)]
    nn.init.normal_(model.head.classification_head.cls_logits.weight, std=0.5)
    with torch.no_grad():
        maps = model.head.forward_maps

        def nchw(features):
            return {k: [m.contiguous() for m in v] for k, v in maps(features).items()}
        last = model(images)
        model.head.forward_maps = nchw
        plain = model(images)
    assert sum(int(d["scores"].numel()) for d in last) > 0
    for p, q in zip(plain, last):
        assert all(torch.equal(p[k], q[k]) for k in p)


@pytest.mark.parametrize("gamma,beta,value", [(0.0, 0.0, None), (0.0, 0.5, None), (0.0, -0.5, None), (1.0, 0.0, 0.0),
                                              (1.0, 0.0, 0.375), (-0.5, 0.0, None)])
def test_fresh_parameters_and_constant_maps(device, gamma, beta, value):
    """A zero-initialised norm and a map of one value put every pixel on the rectifier's corner: the gradients are those of the
    definition, and the backward pass does not go over the map once more for it."""
    gen = torch.Generator().manual_seed(41)
    C, groups = 256, 32
    x = torch.randn((16, C, 64, 64), generator=gen).to(device, torch.bfloat16)
    if value is not None:
        x.fill_(value)
    x = x.contiguous(memory_format=torch.channels_last)
    dy = torch.randn((16, C, 64, 64), generator=gen).to(device, torch.bfloat16).contiguous(memory_format=torch.channels_last)
    g, b = torch.full((C,), gamma, device=device), torch.full((C,), beta, device=device)
    if gamma < 0:
        # away from the corner: a value next to it may fall on either side
        r = _ref(x, groups, g, b, 1e-5, "relu")
        dy = torch.where(r["u"].abs() < 1e-3 * r["scale"], torch.zeros_like(dy), dy)
    _check(x, dy, groups, g, b, "relu")

    def spent(g, b, x):
        leaves = [t.detach().clone(memory_format=torch.preserve_format).requires_grad_(True) for t in (x, g, b)]
        y = group_norm_act(*leaves[:1], groups, *leaves[1:])
        times = []
        for _ in range(6):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            for _ in range(20):
                torch.autograd.grad(y, leaves, dy, retain_graph=True)
            end.record()
            end.synchronize()
            times.append(start.elapsed_time(end))
        return min(times)
    ordinary = spent(torch.linspace(0.5, 1.5, C, device=device), torch.linspace(-0.3, 0.4, C, device=device),
                     torch.randn((16, C, 64, 64), device=device).to(x).contiguous(memory_format=torch.channels_last))
    assert spent(g, b, x) < 2 * ordinary                            # the second sweep: 3 times and more


def test_channels_last_maps_that_do_not_belong_together_are_refused(device):
    """As in NCHW memory: a box map smaller than its class map, or anchors of another size, raise before anything is read."""
    from object_detection_amd.retinanet import postprocess_batched
    last = torch.channels_last

    def call(side, anchors, memory):
        cls = [torch.zeros((2, 3 * 5, 8, 8), device=device).contiguous(memory_format=memory)]
        reg = [torch.zeros((2, 3 * 4, side, side), device=device).contiguous(memory_format=memory)]
        return postprocess_batched(cls, reg, [[torch.zeros((anchors, 4), device=device)]] * 2, [(64, 64)] * 2, 0.05, 100, 0.5, 10,
                                   0, 4.0, planar_classes=5)
    assert len(call(8, 192, last)) == len(call(8, 192, torch.contiguous_format)) == 2
    for side, anchors in ((4, 192), (8, 100)):
        for memory in (last, torch.contiguous_format):
            with pytest.raises((ValueError, _C.OdBoxesError)):
                call(side, anchors, memory)
