"""act_checkpoint_int8, act_backward_int8 and checkpointed_activation against their formulas.

Codes and scales have to be equal.  Values, element by element: half a step of the
output's type, plus the fp32 evaluation: z (the sigmoid's argument) is off by 2^-22
of itself and the exponential by 2^-21, so the sigmoid by (|z| + 8) 2^-22 of itself."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
ACTS = ("gelu_tanh", "silu", "swiglu")
C0, C1 = math.sqrt(2.0 / math.pi), 0.044715


def _codes(x, k):
    """Codes and scales group by group, in fp32 with IEEE divisions, on the CPU."""
    x = x.float().cpu()
    q, scales = torch.empty_like(x), []
    for lo in range(0, x.shape[1], k):
        for at in range(lo, lo + k, 128):
            end = min(at + 128, lo + k)
            s = (x[:, at:end].abs().amax(1) / 127.0).clamp_min(1e-30)
            q[:, at:end] = torch.round(x[:, at:end] / s[:, None])
            scales.append(s)
    return q.to(torch.int8), torch.stack(scales, 1)


def _value(q, scale, k):
    s = scale.unflatten(-1, (q.shape[1] // k, -1)).repeat_interleave(128, -1)[..., :k].flatten(-2)
    return (q.float() * s).double()


def _sig(x, act):
    """(sigmoid, its argument, the argument's slope) in 64 bits."""
    z = 2 * C0 * (x + C1 * x ** 3) if act == "gelu_tanh" else x
    dz = 2 * C0 * (1 + 3 * C1 * x ** 2) if act == "gelu_tanh" else torch.ones_like(x)
    return torch.sigmoid(z), z.abs(), dz


def _forward(x, act):
    """(y, error bound of its fp32 evaluation)."""
    gate, up = x.chunk(2, -1) if act == "swiglu" else (x, 1.0)
    s, z, _ = _sig(gate, act)
    y = gate * s * up
    return y, y.abs() * (z + 8) * 2.0 ** -22


def _backward(dy, x, act):
    gate, up = x.chunk(2, -1) if act == "swiglu" else (x, torch.ones_like(x))
    s, z, dz = _sig(gate, act)
    t = gate * s * torch.sigmoid(-(2 * C0 * (gate + C1 * gate ** 3) if act == "gelu_tanh" else gate)) * dz
    dg = dy * up * (s + t)
    eg = (dy * up).abs() * (s + t.abs()) * (z + 8) * 2.0 ** -20
    if act != "swiglu":
        return dg, eg
    du = dy * gate * s
    return torch.cat([dg, du], -1), torch.cat([eg, du.abs() * (z + 8) * 2.0 ** -20], -1)


def _check(got, ref, err):
    fi = torch.finfo(got.dtype)
    tol = fi.eps / 2 * ref.abs() * (1 + 2.0 ** -8) + err + 2 * fi.tiny
    over = (got.double().cpu() - ref.cpu()).abs() - tol.cpu()
    assert bool((over <= 0).all()), f"worst excess {over.max().item():.3e}"


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 128), (3, 7), (5, 129), (77, 1200), (33, 255), (260, 1024), (2, 12288)])
def test_checkpoint_and_gradient(rows, k, dtype, act):
    import imagine_b200 as W

    t = DTYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(rows * 31 + k)
    x = (torch.randn(rows, k * (2 if act == "swiglu" else 1), generator=g, device="cuda") * 3).to(t)
    x.view(-1)[::37] *= 20
    dy = torch.randn(rows, k, generator=g, device="cuda").to(t)
    y, q, scale = W.act_checkpoint_int8(x, act)
    want_q, want_s = _codes(x, k)
    assert torch.equal(scale.cpu(), want_s) and torch.equal(q.cpu(), want_q)
    _check(y, *_forward(x.double(), act))
    dx = W.act_backward_int8(dy, q, scale, act)
    assert dx.shape == x.shape and dx.dtype == t
    _check(dx, *_backward(dy.double(), _value(q, scale, k), act))
    # rows apart, at odd starts; a batch of samples
    apart = torch.empty(rows, x.shape[1] + 9, dtype=t, device="cuda")[:, 1:1 + x.shape[1]]
    apart.copy_(x)
    for p, r in zip(W.act_checkpoint_int8(apart, act), (y, q, scale)):
        assert torch.equal(p, r)
    dya = torch.empty(rows, k + 3, dtype=t, device="cuda")[:, 2:2 + k]
    dya.copy_(dy)
    assert torch.equal(W.act_backward_int8(dya, q, scale, act), dx)
    x3 = x.view(1, rows, -1)
    assert torch.equal(W.act_checkpoint_int8(x3, act)[0][0], y)


@pytest.mark.parametrize("act", ACTS)
def test_extreme_values(act):
    """Zeros, tiny and huge values, and groups with infinity or NaN."""
    import imagine_b200 as W

    x = torch.randn(4, 512, device="cuda")
    x[0] = 0
    x[1] *= 1e-36
    x[2] *= 1e30
    x[3, :128] = 1e-45
    k = 256 if act == "swiglu" else 512
    y, q, scale = W.act_checkpoint_int8(x, act)
    want_q, want_s = _codes(x, k)
    assert torch.equal(scale.cpu(), want_s) and torch.equal(q.cpu(), want_q)
    dy = torch.ones(4, k, device="cuda")
    dx = W.act_backward_int8(dy, q, scale, act)
    assert bool(dx.isfinite().all())
    if act != "swiglu":
        assert torch.equal(dx[0], torch.full_like(dx[0], 0.5))
        assert torch.equal(dx[2][q[2] > 0], torch.ones_like(dx[2][q[2] > 0]))
        assert not bool(dx[2][q[2] < 0].any())
    z = torch.zeros(2, 512, device="cuda")
    z[0, 130], z[1, 300] = float("inf"), float("nan")
    y, q, scale = W.act_checkpoint_int8(z, act)
    bad = torch.zeros(2, 4, dtype=torch.bool)
    bad[0, 1], bad[1, 2] = True, True
    assert torch.equal(scale.isnan().cpu(), bad)
    dx = W.act_backward_int8(dy[:2], q, scale, act)
    hit = bad.repeat_interleave(128, 1)
    if act == "swiglu":  # d gate = dy up silu'(gate) needs both halves, d up = dy silu(gate) the gate alone
        hit = torch.cat([hit[:, :256] | hit[:, 256:], hit[:, :256]], 1)
    assert torch.equal(dx.isnan().cpu(), hit)


def test_differentiable_and_captured():
    import imagine_b200 as W

    for act in ACTS:
        x = torch.randn(3, 20, 320, device="cuda").bfloat16().requires_grad_()
        y = W.checkpointed_activation(x, act)
        dy = torch.randn_like(y)
        gx, = torch.autograd.grad(y, x, dy)
        y2, q, scale = W.act_checkpoint_int8(x.detach(), act)
        assert torch.equal(y, y2) and torch.equal(gx, W.act_backward_int8(dy, q, scale, act))
        # against differences of the activation itself: the checkpoint moves x by half a code
        # (scale / 2), the slope by at most 1.2 times that (|f''| < 1.2), rounding aside
        ref, _ = _backward(dy.double().view(-1, dy.shape[-1]), x.detach().double().view(-1, 320), act)
        step = scale.max().item() / 2
        big = x.detach().abs().max().item() + 1
        tol = dy.abs().max().item() * (1.2 * step * (big if act == "swiglu" else 1) + step) + 2.0 ** -7 * ref.abs()
        assert bool(((gx.double().view(-1, 320) - ref).abs() <= tol).all())
    data = torch.randn(64, 512, device="cuda").bfloat16()
    dy = torch.randn(64, 512, device="cuda").bfloat16()

    def step_():
        y, q, scale = W.act_checkpoint_int8(data)
        return y, W.act_backward_int8(dy, q, scale)
    step_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step_()
    data.copy_(torch.randn_like(data))
    graph.replay()
    assert all(torch.equal(p, r) for p, r in zip(held, step_()))


def test_empty():
    import imagine_b200 as W

    y, q, scale = W.act_checkpoint_int8(torch.empty(0, 256, device="cuda").half(), "swiglu")
    assert y.shape == (0, 128) and q.shape == (0, 256) and scale.shape == (0, 2)
    assert W.act_backward_int8(y, q, scale, "swiglu").shape == (0, 256)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("k", [512, 200, 333])
def test_output_next_to_nan_and_infinity(k, dtype, act):
    """y is a function of the element itself: what stands beside a NaN or an infinity, at even and odd
    places, has the bits of the same row without it; the element itself has the formula's value."""
    import imagine_b200 as W

    t = DTYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(k)
    x = torch.randn(24, k * (2 if act == "swiglu" else 1), generator=g, device="cuda").to(t)
    clean = W.act_checkpoint_int8(x, act)[0]
    spots = [0, 1, 2, 63, 64, 127, 128, k - 2, k - 1, 31, 100, 165]
    for half in range(2 if act == "swiglu" else 1):
        for v in (float("nan"), float("inf"), -float("inf")):
            z = x.clone()
            hit = torch.zeros(24, k, dtype=torch.bool, device="cuda")
            for row in range(24):
                at = spots[row % len(spots)]
                z[row, half * k + at] = v
                hit[row, at] = True
            y, q, scale = W.act_checkpoint_int8(z, act)
            assert torch.equal(y[~hit], clean[~hit])
            want = _forward(z.double(), act)[0][hit]
            # -inf times a sigmoid of zero is NaN, as in the formula
            assert torch.equal(y[hit].isnan(), want.isnan())
            known = ~want.isnan()
            assert torch.equal(y[hit][known].double(), want[known])
            # and the gradient of such a group is NaN, of the others finite
            dx = W.act_backward_int8(torch.ones_like(y), q, scale, act)
            groups = -(-k // 128)
            of = scale.isnan().unflatten(-1, (-1, groups)).repeat_interleave(128, -1)[..., :k]
            assert bool((of.any(1) == dx.unflatten(-1, (-1, k)).isnan().any(1)).all())


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_zeros_tiny_and_huge_values_of_sixteen_bits(dtype, act):
    import imagine_b200 as W

    t = DTYPES[dtype]
    fi = torch.finfo(t)
    x = torch.randn(6, 512, device="cuda").to(t)
    x[0] = 0
    x[1] = x[1].sign() * fi.tiny
    x[2, ::3] = fi.max
    x[3, 1::3] = -fi.max
    x[4] *= fi.smallest_normal ** 0.5
    x[5] *= 60
    k = 256 if act == "swiglu" else 512
    y, q, scale = W.act_checkpoint_int8(x, act)
    want_q, want_s = _codes(x, k)
    assert torch.equal(scale.cpu(), want_s) and torch.equal(q.cpu(), want_q)
    ref, err = _forward(x.double(), act)
    fits = ref.abs() <= float(fi.max)
    # a value below the type's normal range is off by half of its last place there
    tol = fi.eps / 2 * ref.abs() * (1 + 2.0 ** -8) + err + 2 * fi.tiny
    assert bool(((y.double() - ref).abs() <= tol)[fits].all())
    assert bool((y[~fits].double().sign() == ref[~fits].sign()).all())
    dx = W.act_backward_int8(torch.ones(6, k, dtype=t, device="cuda"), q, scale, act)
    want, err = _backward(torch.ones(6, k, device="cuda").double(), _value(q, scale, k), act)
    fits = want.abs() <= float(fi.max)
    _check(torch.where(fits, dx, 0), torch.where(fits, want, 0), torch.where(fits, err, 0))
