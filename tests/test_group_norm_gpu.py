"""Group norm with an activation: the kernels against the formula in 64 bits.

Bounds count roundings.  u = 2^-24 is half a step of fp32 and h half a step of the tensor's type.  In the tests' sizes no
thread adds more than 64 rows of a channel and no tree is deeper than 16, so a mean is off by at most 100 u of the spread
and an inverse deviation by 100 u of itself; a value costs 8 more roundings of its parts."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from pytorch_distributed_amd import ops

DEV = "cuda"
U = 2.0 ** -24
INF = float("inf")
TYPES = [torch.float32, torch.float16, torch.bfloat16]
# least difference that the type can show
TINY = {torch.float32: 1e-40, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-38}


def exact(x, groups, w, b, res, act, eps, dy=None):
    """Everything in 64 bits; act'(z) by its formula."""
    N, C = x.shape[0], x.shape[-1]
    x64 = x.detach().double().reshape(N, -1, groups, C // groups)
    m = x64.shape[1] * x64.shape[3]
    mean = x64.sum((1, 3), keepdim=True) / m
    r = 1.0 / torch.sqrt(((x64 - mean) ** 2).sum((1, 3), keepdim=True) / m + eps)
    xh = (x64 - mean) * r
    ga = torch.ones(C, device=x.device).double() if w is None else w.detach().double()
    be = torch.zeros(C, device=x.device).double() if b is None else b.detach().double()
    ga, be = ga.view(1, 1, groups, -1), be.view(1, 1, groups, -1)
    rs = torch.zeros_like(x64) if res is None else res.detach().double().reshape(x64.shape)
    z = xh * ga + be + rs
    s = torch.sigmoid(z)
    out, slope = {False: (z, torch.ones_like(z)), True: (z.clamp_min(0), (z > 0).double()),
                  6.0: (z.clamp(0, 6), ((z > 0) & (z < 6)).double()), "silu": (z * s, s * (1 + z * (1 - s)))}[act]
    # what one rounding step of each part may do to z
    ez = U * (100 * (xh * ga).abs() + 100 * ga.abs() + 8 * (be.abs() + rs.abs()))
    eo = ez * 1.2 + (U * (z.abs() + 8) * out.abs() if act == "silu" else 0)
    e = {"out": (out, eo)}
    if dy is not None:
        d = dy.detach().double().reshape(x64.shape)
        g = d * slope
        # the slope of silu changes by at most half of what z does, and its own roundings count (4 + |z|) each
        eg = d.abs() * (0.6 * ez + U * (4 + z.abs()) ** 2) if act == "silu" else torch.zeros_like(g)
        gx = g * xh
        egx = eg * xh.abs() + g.abs() * U * (100 + 104 * xh.abs())
        A, B = ((t * ga).sum((1, 3), keepdim=True) / m for t in (g, gx))
        eA = (((100 * U * g.abs() + eg) * ga.abs()).sum((1, 3), keepdim=True)) / m
        eB = (((100 * U * gx.abs() + egx) * ga.abs()).sum((1, 3), keepdim=True)) / m
        dx = r * (ga * g - A - xh * B)
        edx = r * (ga.abs() * eg + eA + xh.abs() * eB + 100 * U * B.abs() +
                   U * (108 * (ga * g).abs() + 108 * A.abs() + 208 * (xh * B).abs()))
        e["dx"] = (dx, edx)
        e["dres"] = (g, eg)
        e["dgamma"] = (gx.sum((0, 1)).reshape(-1), (100 * U * gx.abs() + egx).sum((0, 1)).reshape(-1))
        e["dbeta"] = (g.sum((0, 1)).reshape(-1), (100 * U * g.abs() + eg).sum((0, 1)).reshape(-1))
    return e


def close(name, got, want):
    ref, err = want
    half = torch.finfo(got.dtype).eps / 2
    diff = (got.double().reshape(ref.shape) - ref).abs()
    lim = half * (ref.abs() + err) + err + TINY[got.dtype]
    worst = float((diff / lim).max())
    assert worst <= 1.0, f"{name}: {worst:.2f} times the bound"


def make(shape, dtype, seed, offset=0.5, residual=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    C = shape[-1]

    def rand(*s):
        return torch.randn(s, device=DEV, generator=g)

    x = (rand(*shape) * (0.5 + rand(C).abs()) + offset).to(dtype)
    res = rand(*shape).to(dtype) if residual else None
    return x, 1 + 0.3 * rand(C), 0.3 * rand(C), res, rand(*shape).to(dtype)


def check(x, groups, w, b, res, dy, act, eps=1e-5):
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b, res)]
    out = ops.group_norm_act(leaves[0], groups, leaves[1], leaves[2], leaves[3], act, eps)
    want = exact(x, groups, w, b, res, act, eps, dy)
    close("out", out, want["out"])
    some = [t for t in leaves if t is not None]
    grads = dict(zip([n for n, t in zip(("dx", "dgamma", "dbeta", "dres"), leaves) if t is not None],
                     torch.autograd.grad(out, some, dy)))
    for n, t in grads.items():
        close(n, t, want[n])
    return out, grads


SHAPES = [  # shape, groups
    ((1, 1, 1, 8), 8),          # one value a group
    ((1, 1, 1, 1), 1),
    ((2, 1, 1, 64), 32),
    ((3, 1, 7, 24), 3),
    ((2, 7, 7, 2048), 32),
    ((5, 8, 8, 64), 32),        # two channels a group
    ((2, 14, 14, 256), 32),
    ((2, 28, 28, 116), 4),      # 29 channels a group, no whole vectors
    ((2, 9, 11, 58), 2),
    ((2, 5, 3, 7), 7),          # odd channels
    ((2, 33, 31, 3), 1),
    ((1, 56, 56, 64), 1),       # one group
    ((2, 56, 56, 256), 32),
    ((1, 3, 3, 4104), 1),       # wider than a block, one group over it
    ((1, 112, 112, 16), 16),
    ((257, 2, 2, 512), 32),     # many small samples
    ((3, 40), 5),               # no positions at all
    ((2, 50, 24), 4),
    ((3, 6, 6, 58), 2),         # several positions make up whole vectors
    ((2, 4, 4, 7), 7),
    ((2, 8, 3, 12), 3),
    ((1, 120, 120, 24), 3),     # too many positions for registers
    ((9, 28, 28, 64), 32),
    ((40, 2, 2, 512), 512),     # a group a channel, rows as wide as a wave
    ((1500, 1, 3, 512), 512),
    ((1100, 1, 2, 4096), 4096),
    ((3, 2, 3, 2048), 128),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_group_norm_act_sizes(shape, groups, dtype):
    x, w, b, res, dy = make(shape, dtype, 5, residual=True)
    check(x, groups, w, b, res, dy, True)
    check(x, groups, w, b, None, dy, "silu")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", [False, True, 6.0, "silu"])
@pytest.mark.parametrize("residual", [False, True])
def test_group_norm_act_activations(act, residual, dtype):
    x, w, b, res, dy = make((3, 13, 11, 48), dtype, 6, residual=residual)
    check(x, 6, 3 * w, b, res, dy, act)
    check(x, 6, None, None, res, dy, act)


@pytest.mark.parametrize("offset", [100.0, -3000.0])
def test_group_norm_act_mean_far_from_zero(offset):
    x, w, b, _, dy = make((2, 20, 20, 32), torch.float32, 7, offset=offset)
    check(x, 4, w, b, None, dy, True)
    x[0, 0, 0] += 1e4   # an outlier in the first row
    check(x, 4, w, b, None, dy, "silu")


@pytest.mark.parametrize("shape,groups", [((2, 20, 20, 32), 4), ((2, 20, 20, 8), 4), ((3, 6, 6, 58), 2), ((2, 14, 14, 48), 8),
                                          ((2, 13, 7, 3), 1), ((2, 120, 120, 24), 3), ((2, 120, 120, 24), 12),
                                          ((2, 56, 56, 64), 1)])
@pytest.mark.parametrize("dtype,offset,spread", [(torch.float32, 123457.0, 1.0), (torch.float32, -2000003.0, 1.0),
                                                 (torch.float16, 40000.0, 156.25), (torch.bfloat16, -189.0 * 2 ** 25, 2.0 ** 26)])
def test_group_norm_act_spread_far_below_the_mean(shape, groups, dtype, offset, spread):
    """Values whose spread is a small part of their mean, and none at all in the last sample (r = 1/sqrt(eps) there).  With
    differences to one of a group's m elements, p, a variance is off by some 2^-53 ((p - mean)^2 + spread^2), and (p - mean)^2 is at
    most m <= 14400 * 64 times spread^2: 2^-33 of it, far inside the bounds.  The oracle's values have the offset taken off
    first, which is exact in 64 bits."""
    x, w, b, _, dy = make(shape, dtype, 51)
    x = ((x.float() * 8).round() / 8 * spread + offset).to(dtype)
    x[-1] = offset
    left = x.double() - offset
    assert bool(torch.isfinite(x).all()) and not bool(left[-1].any())
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    for act in (False, "silu"):
        out = ops.group_norm_act(x, groups, w, b, None, act)
        want = exact(left, groups, w, b, None, act, 1e-5, dy)
        close("out", out.detach(), want["out"])
        for n, t in zip(("dx", "dgamma", "dbeta"), torch.autograd.grad(out, leaves, dy)):
            close(n, t, want[n])


def test_group_norm_act_borders_of_the_activation():
    """res such that z is the rounding of an fp32 number, to either side of 0.  x is a multiple of 2^-6 below 4 in size: sums of
    four such and of their squares are exact in fp32, so the statistics are those of fp64, good to 1e-12."""
    N, S, C = 2, 512, 8
    x, w, b, _, dy = make((N, S, C), torch.float32, 8)
    x = ((x * 64).round() / 64).clamp(-3.5, 3.5)
    z = exact(x, 2, w, b, None, False, 1e-5)["out"][0].reshape(x.shape)
    res = (-z).float()
    left = z + res.double()
    sure = left.abs() > 1e-10
    assert int(sure.sum()) > 4000
    rl = res.requires_grad_(True)
    out = ops.group_norm_act(x, 2, w, b, rl, True)
    dres = torch.autograd.grad(out, rl, dy)[0]
    assert torch.equal((dres != 0)[sure], (left > 0)[sure] & (dy != 0)[sure])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,groups", [((2, 6, 6, 32), 4), ((2, 9, 11, 58), 29), ((1, 120, 120, 24), 3)])
@pytest.mark.parametrize("act,border", [(True, 0.0), (6.0, 0.0), (6.0, 6.0), (0.5, 0.5)])
def test_group_norm_act_no_gradient_on_a_border(act, border, shape, groups, dtype):
    x, _, _, _, dy = make(shape, dtype, 52)
    for by_beta in (True, False):
        beta, res = (border, 0.0) if by_beta else (0.0, border)
        leaves = [t.requires_grad_(True) for t in (x.clone(), torch.zeros(shape[-1], device=DEV),
                                                   torch.full((shape[-1],), beta, device=DEV), torch.full_like(x, res))]
        out = ops.group_norm_act(leaves[0], groups, leaves[1], leaves[2], leaves[3], act)
        assert torch.equal(out, torch.full_like(out, border))
        assert not any(bool(t.any()) for t in torch.autograd.grad(out, leaves, dy))


@pytest.mark.parametrize("shape,groups", [((2, 300, 8), 2), ((3, 28, 28, 64), 8), ((2, 56, 56, 32), 16), ((2, 15000, 8), 2),
                                          ((2, 9, 11, 58), 29)])
@pytest.mark.parametrize("act", [True, 6.0])
def test_group_norm_act_side_of_a_border_is_that_of_fp64(shape, groups, act):
    """As above with values of full precision: sums of x and x^2 in fp64 are off by 1e-16 times the root of their number at
    most (300 here), z by a few of those; 1e-12 is beyond it."""
    x, w, b, _, dy = make(shape, torch.float32, 31)
    z = exact(x, groups, w, b, None, False, 1e-5)["out"][0].reshape(shape)
    border = 0.0 if act is True else 6.0
    res = (border - z).float()
    left = z + res.double() - border
    sure = left.abs() > 1e-12
    assert float(sure.double().mean()) > 0.9
    rl = res.requires_grad_(True)
    dres, = torch.autograd.grad(ops.group_norm_act(x, groups, w, b, rl, act), rl, dy)
    inside = left > 0 if act is True else left < 0
    assert torch.equal((dres != 0)[sure], inside[sure] & (dy != 0)[sure])


# as many positions as registers hold
LONG = [((600, 1500, 32), 4, torch.float32), ((2, 6500, 8), 1, torch.float32), ((2, 6272, 32), 2, torch.float16), ((3, 12999, 8), 1, torch.bfloat16),
        ((300, 3136, 64), 8, torch.float16), ((2, 6400, 16), 2, torch.bfloat16)]


@pytest.mark.parametrize("act", [False, True, 6.0, "silu"])
@pytest.mark.parametrize("shape,groups,dtype", LONG)
def test_group_norm_act_long_samples(shape, groups, dtype, act):
    x, w, b, res, dy = make(shape, dtype, 41, residual=act != 6.0)
    if act is True or act == 6.0:  # whole vectors and single elements of zero
        dy[:, 7::50] = 0
        dy[..., 3] = 0
    check(x, groups, w, b, res, dy, act)


@pytest.mark.parametrize("act", [True, 6.0])
@pytest.mark.parametrize("shape,groups", [(s, g) for s, g, t in LONG if t == torch.float32])
def test_group_norm_act_long_samples_all_next_to_a_border(shape, groups, act):
    """Every element lies next to the border and is decided in fp64; the sums have to follow.  dy is 0 where z is nearer than
    1e-12.  With g known the bounds are those of sums of g and g xh, each term good to 104 u."""
    x, w, b, _, dy = make(shape, torch.float32, 43)
    z = exact(x, groups, w, b, None, False, 1e-5)["out"][0].reshape(shape)
    border = 0.0 if act is True else 6.0
    res = (border - z).float()
    left = z + res.double() - border
    dy = torch.where(left.abs() > 1e-12, dy, 0.0)
    leaves = [t.requires_grad_(True) for t in (x, w, b, res)]
    out = ops.group_norm_act(x, groups, w, b, res, act)
    dx, dw, db, dres = torch.autograd.grad(out, leaves, dy)
    g = dy.double() * (left > 0 if act is True else left < 0)
    assert torch.equal(dres, g.float())
    # the same gradient through the norm alone
    want = exact(x, groups, w, b, None, False, 1e-5, g)
    close("dbeta", db, want["dbeta"])
    close("dgamma", dw, want["dgamma"])
    close("dx", dx, want["dx"])


def test_group_norm_act_constant_groups_and_nan():
    x = torch.full((2, 6, 6, 16), 3.0, device=DEV)
    w, b = torch.full((16,), 2.0, device=DEV), torch.linspace(-1, 1, 16, device=DEV)
    out = ops.group_norm_act(x, 4, w, b)
    assert torch.equal(out, b.expand_as(out))       # no spread: the shift alone
    x[1, 2, 3, 5] = float("nan")
    out = ops.group_norm_act(x, 4, w, b, None, True)
    bad = torch.isnan(out)
    assert bool(bad[1, :, :, 4:8].all()) and int(bad.sum()) == 6 * 6 * 4
    x[1, 2, 3, 5] = float("inf")
    assert int(torch.isnan(ops.group_norm_act(x, 4, w, b, None, "silu")).sum()) == 6 * 6 * 4


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,groups", [((2, 6, 6, 32), 4), ((2, 14, 14, 48), 8), ((3, 6, 6, 58), 2), ((2, 120, 120, 24), 3)])
def test_group_norm_act_no_number_in_first_place(shape, groups, dtype):
    """The first value of a group, from which its sums are taken, and the last one: NaN in that group alone, the others as before."""
    x, w, b, _, dy = make(shape, dtype, 53)
    D = shape[-1] // groups
    leaf = x.clone().requires_grad_(True)
    ref = ops.group_norm_act(leaf, groups, w, b, None, "silu")
    dref, = torch.autograd.grad(ref, leaf, dy)
    for bad in (float("nan"), INF, -INF):
        for at in ((1, 0, 0, D), (1, shape[1] - 1, shape[2] - 1, 2 * D - 1)):
            y = x.clone()
            y[at] = bad
            y.requires_grad_(True)
            out = ops.group_norm_act(y, groups, w, b, None, "silu")
            dx, = torch.autograd.grad(out, y, dy)
            for got, was in ((out, ref), (dx, dref)):
                assert bool(got[1, ..., D:2 * D].isnan().all())
                keep = torch.ones_like(got, dtype=torch.bool)
                keep[1, ..., D:2 * D] = False
                assert torch.equal(got[keep], was[keep])


@pytest.mark.parametrize("dtype", TYPES)
def test_group_norm_act_strides_and_alignment(dtype):
    x, w, b, res, dy = make((3, 10, 10, 64), dtype, 9, residual=True)
    # channels first in memory, a sliced residual, an upstream gradient with strides 0
    xs = x.permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1)
    big = torch.zeros((3, 10, 10, 72), device=DEV, dtype=dtype)
    big[..., 4:68] = res
    out, grads = check(xs, 8, w, b, big[..., 4:68], dy, True)
    check(x, 8, w, b, res, dy[:1, :1, :1].expand(3, 10, 10, 64), True)
    # a base address that no vector access may use
    flat = torch.zeros(x.numel() + 1, device=DEV, dtype=dtype)
    flat[1:] = x.reshape(-1)
    out2, grads2 = check(flat[1:].view_as(x), 8, w, b, res, dy, True)
    assert torch.equal(out, out2) or dtype == torch.float32 or float((out - out2).abs().max()) < 1e-1


def test_group_norm_act_gradient_subsets_and_parameter_types():
    x, w, b, res, dy = make((2, 6, 6, 32), torch.float16, 10, residual=True)
    want = exact(x, 4, w.half(), b.half(), res, True, 1e-5, dy)
    wl, bl = w.half().requires_grad_(True), b.half().requires_grad_(True)
    out = ops.group_norm_act(x, 4, wl, bl, res, True)
    dg, = torch.autograd.grad(out, wl, dy)
    assert dg.dtype == torch.float16
    close("dgamma", dg, want["dgamma"])
    rl = res.clone().requires_grad_(True)
    close("dres", torch.autograd.grad(ops.group_norm_act(x, 4, wl.detach(), bl.detach(), rl, True), rl, dy)[0], want["dres"])
    xl = x.clone().requires_grad_(True)
    close("dx", torch.autograd.grad(ops.group_norm_act(xl, 4, wl.detach(), bl.detach(), res, True), xl, dy)[0], want["dx"])
    # no activation: the residual's gradient is the upstream one
    r2 = res.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(ops.group_norm_act(x, 4, None, None, r2), r2, dy)[0], dy)


@pytest.mark.parametrize("shape", [(1400, 56, 56, 512), (160, 14400, 1024)])
def test_group_norm_act_offsets_beyond_32_bits(shape):
    """The last sample lies behind 2^31 elements (in registers, and by row chunks)."""
    g = torch.Generator(device=DEV).manual_seed(16)
    one, w, b, _, dy = make((1,) + shape[1:], torch.float16, 17)
    x = torch.zeros(shape, device=DEV, dtype=torch.float16)
    x[-1:] = one
    up = torch.zeros_like(x)
    up[-1:] = dy
    xl, wl = x.requires_grad_(True), w.requires_grad_(True)
    out = ops.group_norm_act(xl, 32, wl, b, None, True)
    dx, dw = torch.autograd.grad(out, (xl, wl), up)
    want = exact(one, 32, w, b, None, True, 1e-5, dy)
    close("out", out[-1:], want["out"])
    close("dx", dx[-1:], want["dx"])
    close("dgamma", dw, want["dgamma"])
    assert not bool(dx[:-1].any())


@pytest.mark.parametrize("shape,groups,dtype", [(((1 << 25) + 3, 16), 2, torch.float16), (((1 << 24) + 3, 2, 5), 1, torch.bfloat16)])
def test_group_norm_act_more_samples_than_one_launch_holds(shape, groups, dtype):
    x = torch.ones(shape, device=DEV, dtype=dtype)
    at = torch.tensor([0, 1, (1 << 21) - 1, 1 << 21, 1 << 23, (1 << 24) - 1, 1 << 24, shape[0] - 1], device=DEV)
    some, w, b, _, dy = make((8,) + shape[1:], dtype, 29)
    x[at] = some
    full = torch.zeros(shape, device=DEV, dtype=dtype)
    full[at] = dy
    x.requires_grad_(True), some.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)
    out, few = ops.group_norm_act(x, groups, w, b, None, "silu"), ops.group_norm_act(some, groups, w, b, None, "silu")
    got, want = torch.autograd.grad(out, (x, w, b), full), exact(some, groups, w, b, None, "silu", 1e-5, dy)
    close("out", out[at].detach(), want["out"])
    close("few", few.detach(), want["out"])
    close("dx", got[0][at], want["dx"])
    close("dgamma", got[1], want["dgamma"])
    close("dbeta", got[2], want["dbeta"])


@pytest.mark.parametrize("shape,groups", [((4096, 1, 16), 2), ((4097, 1, 16), 2), ((5000, 2, 2, 30), 3), ((600000, 24), 3)])
def test_group_norm_act_parameter_sums_over_many_samples(shape, groups):
    x, w, b, _, dy = make(shape, torch.float32, 44)
    check(x, groups, w, b, None, dy, "silu")


def test_group_norm_act_is_differentiable_once():
    x, w, b, _, dy = make((2, 3, 3, 16), torch.float32, 15)
    xl = x.requires_grad_(True)
    out = ops.group_norm_act(xl, 4, w, b, None, "silu")
    g, = torch.autograd.grad(out, xl, dy, create_graph=True)
    close("dx", g.detach(), exact(x, 4, w, b, None, "silu", 1e-5, dy)["dx"])
    with pytest.raises(RuntimeError):
        g.sum().backward()
    out = ops.group_norm_act(xl, 4, w, b, None, True)
    with torch.no_grad():
        xl += 1.0
    with pytest.raises(RuntimeError):    # changed in place since the forward pass
        torch.autograd.grad(out, xl, dy)


def test_group_norm_act_same_tensor_twice_and_retained_graph():
    x, w, b, _, dy = make((2, 9, 9, 32), torch.float32, 11)
    xl = x.clone().requires_grad_(True)
    out = ops.group_norm_act(xl, 8, w, b, xl, True)     # the residual is x itself
    g1, = torch.autograd.grad(out, xl, dy, retain_graph=True)
    g2, = torch.autograd.grad(out, xl, dy)
    assert torch.equal(g1, g2)
    e = exact(x, 8, w, b, x, True, 1e-5, dy)
    close("dx", g1, (e["dx"][0] + e["dres"][0], e["dx"][1] + e["dres"][1] + 2 * U * (e["dx"][0].abs() + e["dres"][0].abs())))


def test_group_norm_act_repeats_bit_for_bit_on_other_streams():
    x, w, b, res, dy = make((64, 14, 14, 128), torch.float16, 12, residual=True)
    ref, gref = check(x, 32, w, b, res, dy, True)
    side = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            leaves = [t.detach().requires_grad_(True) for t in (x, w, b, res)]
            o = ops.group_norm_act(leaves[0], 32, leaves[1], leaves[2], leaves[3], True)
            outs.append((o, torch.autograd.grad(o, leaves, dy)))
    for s in side:
        torch.cuda.current_stream().wait_stream(s)
    for o, gr in outs:
        assert torch.equal(o, ref)
        for a, n in zip(gr, ("dx", "dgamma", "dbeta", "dres")):
            assert torch.equal(a, gref[n])


@pytest.mark.parametrize("shape,groups", [((4, 7, 7, 64), 8), ((2, 56, 56, 64), 32)])
def test_group_norm_act_captured(shape, groups):
    x, w, b, _, dy = make(shape, torch.float16, 13)
    xl = x.clone().requires_grad_(True)
    w, b = w.requires_grad_(True), b.requires_grad_(True)

    def step():
        o = ops.group_norm_act(xl, groups, w, b, None, "silu")
        return (o,) + torch.autograd.grad(o, (xl, w, b), dy)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        with torch.no_grad():
            xl.copy_(make(shape, torch.float16, 20 + i)[0])
        graph.replay()
        torch.cuda.synchronize()
        for a, r in zip(got, step()):
            assert torch.equal(a, r)
