"""lora_add, lora_backward, int8_linear_backward and int8_linear_lora against
their formulas in 64 bits.

Tolerances, element by element: half a step of the output's type on the result
(u = eps / 2), plus what the fp32 sums and the bf16 pieces may be off, relative
to the sum of the products' absolute values.  A contraction of n products adds at
most n / 16 + 1 tensor-core sums, each off by 2^-22 of what it holds (the products of a
sum are cut to its largest one's last kept bit, and so is the sum).
Pieces: a rank-side value next to 16-bit data keeps 16 bits (2^-16); f16 drops the
product of two second pieces, each below 2^-7 (2^-14 a product); fp32 drops those below
the third (2 * 2^-22 a product)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
PIECES = {torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -16 + 2.0 ** -14, torch.float32: 2.0 ** -21}


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _sums(*lengths):
    return sum(n / 16 + 2 for n in lengths) * 2.0 ** -22


def _case(m, k, n, s, r, dtype, seed=0, none=True):
    g = torch.Generator(device="cuda").manual_seed(seed + m * 131 + k * 7 + n)
    def rn(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)
    x, y, dy = rn(m, k), rn(m, n), rn(m, n)
    a, b = rn(s, r, k, std=max(k, 1) ** -0.5), rn(s, n, r, std=0.5)
    c = torch.rand(s, generator=g, device="cuda") + 0.5
    idx = torch.randint(-1 if none else 0, s, (m,), generator=g, device="cuda", dtype=torch.int32)
    return x, y, dy, a, b, c, idx


def _add_ref(x, y, a, b, c, idx):
    """(out, sum of absolute products) in 64 bits."""
    out, size = y.double().clone(), torch.zeros_like(y, dtype=torch.float64)
    for s in range(a.shape[0]):
        rows = (idx == s).nonzero().flatten()
        h = x[rows].double() @ a[s].double().t()
        hs = x[rows].double().abs() @ a[s].double().abs().t()
        out[rows] += c[s].double() * (h @ b[s].double().t())
        size[rows] = c[s].double().abs() * (hs @ b[s].double().abs().t())
    return out, size


def _check(got, ref, size, rel, name=""):
    tol = _u(got.dtype) * ref.abs() * (1 + 2.0 ** -8) + rel * size + 2.0 * torch.finfo(got.dtype).tiny
    over = (got.double() - ref).abs() - tol
    assert bool((over <= 0).all()), f"{name}: worst excess {over.max().item():.3e} at {over.argmax().item()}"


def _grad_ref(x, dy, a, b, c, idx):
    x, dy, a, b, c = x.double(), dy.double(), a.double(), b.double(), c.double()
    out = {}
    dx, da, db = torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    sx, sa, sb = torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    for s in range(a.shape[0]):
        rows = (idx == s).nonzero().flatten()
        g, gs = dy[rows] @ b[s], dy[rows].abs() @ b[s].abs()
        h, hs = x[rows] @ a[s].t(), x[rows].abs() @ a[s].abs().t()
        cs = c[s].abs()
        dx[rows], sx[rows] = c[s] * (g @ a[s]), cs * (gs @ a[s].abs())
        da[s], sa[s] = c[s] * (g.t() @ x[rows]), cs * (gs.t() @ x[rows].abs())
        db[s], sb[s] = c[s] * (dy[rows].t() @ h), cs * (dy[rows].abs().t() @ hs)
    out["dx"], out["da"], out["db"] = (dx, sx), (da, sa), (db, sb)
    return out


def _check_grads(got, x, dy, a, b, c, idx):
    ref = _grad_ref(x, dy, a, b, c, idx)
    m, k, n, r = x.shape[0], x.shape[1], dy.shape[1], a.shape[1]
    rel = {"dx": _sums(n, r), "da": _sums(n, m), "db": _sums(k, m)}
    for name, t in zip(("dx", "da", "db"), got):
        # twice: the rank-side sum and the product it enters drop pieces each
        _check(t, *ref[name], 2 * PIECES[dy.dtype] + rel[name], name)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("m,k,n,s,r", [
    (1, 64, 128, 1, 16), (1, 4096, 4096, 8, 16), (2, 1, 1, 2, 1), (7, 33, 65, 3, 5), (64, 512, 384, 40, 8),
    (65, 200, 129, 2, 12), (130, 1000, 257, 4, 31), (333, 768, 520, 5, 64), (200, 640, 1100, 3, 128),
    (1030, 1024, 512, 9, 33)])
def test_lora_add(m, k, n, s, r, dtype):
    import imagine_b200 as W

    x, y, _, a, b, c, idx = _case(m, k, n, s, r, DTYPES[dtype])
    out = W.lora_add(y, x, a, b, idx, c)
    ref, size = _add_ref(x, y, a, b, c, idx)
    _check(out, ref, size, 2 * PIECES[x.dtype] + _sums(k, r), "out")
    assert torch.equal(out[idx < 0], y[idx < 0])
    assert torch.equal(out, W.lora_add(y, x, a, b, idx.long(), c))  # int64, and the same bits again
    assert torch.equal(out, W.lora_add(y.clone(), x, a, b, idx, c, out=y))  # written into y itself


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("m,k,n,s,r", [
    (1, 64, 128, 1, 16), (3, 1, 1, 2, 1), (7, 33, 65, 3, 5), (65, 200, 136, 2, 12), (190, 520, 257, 6, 31),
    (700, 768, 512, 2, 64), (1500, 256, 1024, 3, 128), (64, 4096, 256, 1, 8)])
def test_lora_backward(m, k, n, s, r, codes, dtype):
    import imagine_b200 as W

    x, _, dy, a, b, c, idx = _case(m, k, n, s, r, DTYPES[dtype], seed=1)
    xs = None
    data = x
    if codes:
        x, xs = W.quantize_int8_rowwise(x)
        data = x.double() * xs.double()
    got = W.lora_backward(dy, x, a, b, idx, c, x_scale=xs)
    _check_grads(got, data, dy, a, b, c, idx)
    again = W.lora_backward(dy, x, a, b, idx, c, x_scale=xs)
    assert all(torch.equal(p, q) for p, q in zip(got, again))
    base = torch.randn(m, k, device="cuda").to(dy.dtype)
    dx, da, db = W.lora_backward(dy, x, a, b, idx, c, x_scale=xs, dx=base.clone(), need_weights=False)
    assert da is None and db is None
    ref, size = _grad_ref(data, dy, a, b, c, idx)["dx"]
    _check(dx, ref + base.double(), size, 2 * PIECES[dy.dtype] + _sums(n, r), "dx added")
    assert torch.equal(dx[idx < 0], base[idx < 0])


def test_long_and_wide():
    """A long batch of ragged requests, the split contractions joined over many blocks."""
    import imagine_b200 as W

    x, y, dy, a, b, c, _ = _case(5856, 1536, 2048, 3, 16, torch.bfloat16)
    idx = torch.repeat_interleave(torch.tensor([0, -1, 2, 1], device="cuda", dtype=torch.int32),
                                  torch.tensor([256, 100, 5000, 500], device="cuda"))
    _check(W.lora_add(y, x, a, b, idx, c), *_add_ref(x, y, a, b, c, idx), 2 * PIECES[x.dtype] + _sums(1536, 16))
    _check_grads(W.lora_backward(dy, x, a, b, idx, c), x, dy, a, b, c, idx)


def test_index_forms_and_strides():
    import imagine_b200 as W

    bt, t, k, n, s, r = 3, 50, 136, 200, 4, 12
    x, y, dy, a, b, c, _ = _case(bt * t, k, n, s, r, torch.bfloat16)
    sample = torch.tensor([2, -1, 0], device="cuda")
    token = sample.repeat_interleave(t)
    x3, y3, dy3 = x.view(bt, t, k), y.view(bt, t, n), dy.view(bt, t, n)
    want = W.lora_add(y, x, a, b, token, c)
    assert torch.equal(W.lora_add(y3, x3, a, b, sample, c).view(-1, n), want)
    assert torch.equal(W.lora_add(y3, x3, a, b, token.view(bt, t), c).view(-1, n), want)
    grads = W.lora_backward(dy, x, a, b, token, c)
    for p, q in zip(W.lora_backward(dy3, x3, a, b, sample, c), grads):
        assert torch.equal(p.reshape(q.shape), q)
    # no index: adapter 0; no scaling: ones; one number
    zero = torch.zeros_like(token)
    one = torch.ones_like(c)
    assert torch.equal(W.lora_add(y, x, a, b), W.lora_add(y, x, a, b, zero, one))
    assert torch.equal(W.lora_add(y, x, a, b, None, 0.5), W.lora_add(y, x, a, b, zero, one * 0.5))
    # rows apart (odd strides, unaligned starts), every second adapter of a stack
    def apart(v, pad, at):
        big = torch.full((v.shape[0], v.shape[1] + pad), float("nan"), dtype=v.dtype, device="cuda")
        big[:, at:at + v.shape[1]] = v
        return big[:, at:at + v.shape[1]]
    xa, ya, dya = apart(x, 5, 1), apart(y, 3, 2), apart(dy, 7, 3)
    a2 = torch.full((2 * s, r, k), float("nan"), dtype=a.dtype, device="cuda")
    b2 = torch.full((2 * s, n, r), float("nan"), dtype=a.dtype, device="cuda")
    a2[::2], b2[::2] = a, b
    assert torch.equal(W.lora_add(ya, xa, a2[::2], b2[::2], token, c), want)
    wide = torch.full((bt * t, n + 9), 7.0, dtype=y.dtype, device="cuda")
    W.lora_add(ya, xa, a, b, token, c, out=wide[:, 4:4 + n])
    assert torch.equal(wide[:, 4:4 + n], want) and bool((wide[:, :4] == 7).all()) and bool((wide[:, 4 + n:] == 7).all())
    for p, q in zip(W.lora_backward(dya, xa, a2[::2], b2[::2], token, c), grads):
        assert torch.equal(p, q)
    # transposed operands are copied
    assert torch.equal(W.lora_add(y.t().contiguous().t(), x.t().contiguous().t(), a, b, token, c), want)


def test_indices_outside_the_stack_mean_no_adapter():
    import imagine_b200 as W

    x, y, dy, a, b, c, _ = _case(70, 64, 96, 2, 8, torch.bfloat16)
    idx = torch.randint(0, 2, (70,), device="cuda")
    off = idx.clone()
    for i, v in enumerate((-1, 2, -7, 1 << 32, (1 << 32) + 1, -(1 << 40), 65536)):
        off[5 * i] = v
    none = (off < 0) | (off > 1)
    want = torch.where(none, -1, off)
    assert torch.equal(W.lora_add(y, x, a, b, off, c), W.lora_add(y, x, a, b, want, c))
    for p, q in zip(W.lora_backward(dy, x, a, b, off, c), W.lora_backward(dy, x, a, b, want, c)):
        assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_nan_stays_in_its_rows_and_adapters(dtype):
    import imagine_b200 as W

    x, y, dy, a, b, c, idx = _case(150, 128, 192, 3, 8, DTYPES[dtype], none=True)
    clean = W.lora_add(y, x, a, b, idx, c)
    grads = W.lora_backward(dy, x, a, b, idx, c)
    bad = idx == 1
    for v in (float("nan"), float("inf")):
        xb, yb, dyb, ab, bb = x.clone(), y.clone(), dy.clone(), a.clone(), b.clone()
        xb[bad], yb[bad], dyb[bad], ab[1], bb[1] = v, v, v, v, v
        xb[idx < 0], dyb[idx < 0] = v, v  # rows without an adapter are not read at all
        out = W.lora_add(yb, xb, ab, bb, idx, c)
        assert torch.equal(out[~bad], clean[~bad]) and not bool(out[bad].isfinite().any())
        dx, da, db = W.lora_backward(dyb, xb, ab, bb, idx, c)
        assert torch.equal(dx[~bad], grads[0][~bad]) and not bool(dx[bad].isfinite().any())
        for t, ref in ((da, grads[1]), (db, grads[2])):
            assert torch.equal(t[[0, 2]], ref[[0, 2]]) and not bool(t[1].isfinite().any())


def test_large_values():
    """fp32 values near the type's end, f16 sums beyond f16's range: no overflow on the way."""
    import imagine_b200 as W

    x, y, dy, a, b, c, idx = _case(40, 96, 64, 2, 4, torch.float16, none=False)
    x, b = x * 8000, (b.float() * 1e-5).half()
    out = W.lora_add(y, x, a * 30, b, idx, c)  # h reaches 10^6
    _check(out, *_add_ref(x, y, a * 30, b, c, idx), 2 * PIECES[x.dtype] + _sums(96, 4))
    x = torch.full((3, 16), 3.4e38, device="cuda")
    a = torch.zeros(1, 1, 16, device="cuda")
    a[0, 0, 5] = 0.5
    out = W.lora_add(torch.zeros(3, 8, device="cuda"), x, a, torch.ones(1, 8, 1, device="cuda"))
    assert torch.allclose(out, torch.full_like(out, 1.7e38), rtol=1e-6)


def test_empty():
    import imagine_b200 as W

    x, y, dy, a, b, c, idx = _case(0, 64, 32, 2, 8, torch.bfloat16)
    assert W.lora_add(y, x, a, b, idx, c).shape == (0, 32)
    dx, da, db = W.lora_backward(dy, x, a, b, idx, c)
    assert dx.shape == (0, 64) and not bool(da.any()) and not bool(db.any())
    x, y, dy, a, b, c, idx = _case(5, 64, 32, 2, 8, torch.bfloat16)
    none = torch.full_like(idx, -1)
    assert torch.equal(W.lora_add(y, x, a, b, none, c), y)
    assert all(not bool(t.any()) for t in W.lora_backward(dy, x, a, b, none, c))
    assert torch.equal(W.lora_add(y, x[:, :0], a[:, :, :0], b, idx, c), y)
    assert W.int8_linear_backward(dy[:0], torch.zeros(32, 64, dtype=torch.int8, device="cuda"),
                                  torch.ones(32, device="cuda")).shape == (0, 64)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("m,k,n,scalar", [(1, 64, 128, False), (1, 17, 3, True), (3, 4096, 4096, False),
                                          (77, 200, 333, False), (250, 512, 1040, True), (640, 768, 512, False),
                                          (1100, 1536, 768, False), (300, 130, 4100, False)])
def test_int8_linear_backward(m, k, n, scalar, dtype):
    import imagine_b200 as W

    t = DTYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(m + k + n)
    dy = torch.randn(m, n, generator=g, device="cuda").to(t)
    w = torch.randint(-128, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    ws = torch.rand(1 if scalar else n, generator=g, device="cuda") * 1e-3 + 1e-4
    dx = W.int8_linear_backward(dy, w, ws)
    wd = w.double() * ws.double().view(-1, 1)
    ref, size = dy.double() @ wd, dy.double().abs() @ wd.abs()
    # one rounding of dy * ws (bf16), of its second or third piece (f16, fp32)
    rel = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -16, torch.float32: 2.0 ** -23}[t]
    _check(dx, ref, size, rel + _sums(n) + 2.0 ** -23, "dx")
    # the roundings are independent: over a whole output they come to far less
    off = float((dx.double() - ref).norm() / ref.norm())
    assert off < {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 1e-6}[t], off
    assert torch.equal(dx, W.int8_linear_backward(dy, w, ws))
    apart = torch.empty(m, n + 3, dtype=t, device="cuda")[:, 1:1 + n]
    apart.copy_(dy)
    wide = torch.empty(n, k + 5, dtype=torch.int8, device="cuda")[:, 2:2 + k]
    wide.copy_(w)
    other = W.int8_linear_backward(apart, wide, ws)
    assert float((other.double() - dx.double()).norm() / ref.norm()) < 2 * off + 2.0 ** -20


def test_int8_linear_lora_trains():
    """The run of them as a training step makes it: forward, backward, and the gradients against
    the formula in 64 bits (straight through the quantiser, adapters' inputs as kept)."""
    import imagine_b200 as W

    g = torch.Generator(device="cuda").manual_seed(3)
    bt, t, k, n, s, r = 2, 60, 256, 384, 3, 16
    x = torch.randn(bt, t, k, generator=g, device="cuda").bfloat16().requires_grad_()
    w, ws = W.quantize_weight((torch.randn(n, k, generator=g, device="cuda") * 0.02).bfloat16())
    bias = torch.randn(n, generator=g, device="cuda").bfloat16()
    a = (torch.randn(s, r, k, generator=g, device="cuda") * 0.06).bfloat16().requires_grad_()
    b = (torch.randn(s, n, r, generator=g, device="cuda") * 0.1).bfloat16().requires_grad_()
    idx = torch.tensor([1, 2], device="cuda")
    c = torch.tensor([1.0, 0.5, 2.0], device="cuda")
    dy = torch.randn(bt, t, n, generator=g, device="cuda").bfloat16()
    rows = idx.repeat_interleave(t)
    q, xs = W.quantize_int8_rowwise(x.detach().view(-1, k))
    for keep in (False, True):
        y = W.int8_linear_lora(x, w, ws, bias, a, b, idx, c, keep_input=keep)
        plain = W.int8_linear(x.detach(), w, ws, bias)
        assert torch.equal(y, W.lora_add(plain, x.detach(), a.detach(), b.detach(), idx, c))
        gx, ga, gb = torch.autograd.grad(y, (x, a, b), dy)
        data = x.detach().view(-1, k).double() if keep else q.double() * xs.double()
        ref = _grad_ref(data, dy.view(-1, n), a.detach(), b.detach(), c, rows)
        _check(ga, *ref["da"], 2 * PIECES[torch.bfloat16] + _sums(n, bt * t), "da")
        _check(gb, *ref["db"], 2 * PIECES[torch.bfloat16] + _sums(k, bt * t), "db")
        wd = w.double() * ws.double().view(-1, 1)
        base = dy.view(-1, n).double() @ wd
        want = (base + ref["dx"][0]).view(bt, t, k)
        # the base gradient is rounded to bf16 before the adapters' is added
        tol = 2.0 ** -8 * (want.abs() + 1.01 * base.abs().view(bt, t, k) +
                           (dy.view(-1, n).double().abs() @ wd.abs()).view(bt, t, k))
        assert bool(((gx.double() - want).abs() <= 1.02 * tol).all())
    only = torch.autograd.grad(W.int8_linear_lora(x.detach(), w, ws, bias, a, b, idx, c), (a,), dy)[0]
    q_again = torch.autograd.grad(W.int8_linear_lora(x, w, ws, bias, a, b, idx, c), (a,), dy)[0]
    assert torch.equal(only, q_again)


def test_int8_linear_lora_captured_and_frozen():
    """A captured training step on its own stream, replayed with new contents; what is frozen says so."""
    import imagine_b200 as W

    g = torch.Generator(device="cuda").manual_seed(12)
    m, k, n, r = 40, 512, 768, 8
    x = torch.randn(m, k, generator=g, device="cuda").bfloat16()
    w, ws = W.quantize_weight((torch.randn(n, k, generator=g, device="cuda") * 0.02).bfloat16())
    a = (torch.randn(1, r, k, generator=g, device="cuda") * 0.05).bfloat16().requires_grad_()
    b = (torch.randn(1, n, r, generator=g, device="cuda") * 0.1).bfloat16().requires_grad_()
    dy = torch.randn(m, n, generator=g, device="cuda").bfloat16()

    def step():
        y = W.int8_linear_lora(x, w, ws, None, a, b)
        return (y, *torch.autograd.grad(y, (a, b), dy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(2):
        x.copy_(torch.randn(m, k, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, step()))
    for kw in (dict(weight_scale=ws.clone().requires_grad_()), dict(bias=torch.zeros(n, device="cuda", requires_grad=True)),
               dict(scaling=torch.ones(1, device="cuda", requires_grad=True))):
        args = dict(weight_scale=ws, bias=None, scaling=None)
        args.update(kw)
        with pytest.raises(ValueError, match="frozen"):
            W.int8_linear_lora(x, w, args["weight_scale"], args["bias"], a, b, None, args["scaling"])


def test_gradient_against_differences():
    """fp32: the adapters' gradient against differences of the forward operator, which is linear
    in each of x, a and b (so a difference is the slope, up to the rounding of its two ends)."""
    import imagine_b200 as W

    x, y, dy, a, b, c, idx = _case(40, 72, 56, 2, 6, torch.float32)
    grads = W.lora_backward(dy, x, a, b, idx, c)

    def loss(x, a, b):
        return (W.lora_add(y, x, a, b, idx, c).double() * dy.double()).sum()
    g = torch.Generator(device="cuda").manual_seed(5)
    for i, t in enumerate((x, a, b)):
        v = torch.randn(t.shape, generator=g, device="cuda")
        args = [x, a, b]
        args[i] = t + v
        up = loss(*args)
        args[i] = t - v
        slope = float(up - loss(*args)) / 2
        want = float((grads[i].double() * v.double()).sum())
        # each end: m * n outputs off by 2^-20 of their size, weighted by dy; 4 for the moved operand's size
        room = 4 * 2.0 ** -20 * float((W.lora_add(y, x, a, b, idx, c).abs() * dy.abs()).sum()) + 1e-3
        assert abs(slope - want) <= room, (i, slope, want, room)


def test_other_stream_and_graph():
    """On a side stream, and captured: a replay reads the new contents of the same buffers."""
    import imagine_b200 as W

    x, y, dy, a, b, c, idx = _case(100, 256, 192, 3, 16, torch.bfloat16)
    w = torch.randint(-127, 128, (192, 256), device="cuda", dtype=torch.int8)
    ws = torch.rand(192, device="cuda") * 1e-3

    def step():
        base = W.int8_linear_backward(dy, w, ws)
        return (W.lora_add(y, x, a, b, idx, c), *W.lora_backward(dy, x, a, b, idx, c, dx=base))
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (1, 2):
        x2, y2, dy2, a2, b2, c2, idx2 = _case(100, 256, 192, 3, 16, torch.bfloat16, seed=seed)
        for dst, src in zip((x, y, dy, a, b, c, idx), (x2, y2, dy2, a2, b2, c2, idx2)):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, step()))


def test_output_beside_the_projection_in_one_tensor():
    """Columns of one tensor as y, out and x: rows interleave and share nothing."""
    import imagine_b200 as W
    m, n, k, s, r = 70, 64, 64, 2, 16
    gen = torch.Generator("cuda").manual_seed(5)
    big, a, b = (torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16)
                 for shape in ((m, 3 * 64), (s, r, k), (s, n, r)))
    y, x, out = big[:, :64], big[:, 64:128], big[:, 128:]
    want = W.lora_add(y.contiguous(), x.contiguous(), a, b)
    got = W.lora_add(y, x, a, b, out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(got, want)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("m", [0, 1, 16, 30, 100])
def test_input_gradient_of_a_weight_without_rows_or_columns(m, dtype):
    import imagine_b200 as W

    t = DTYPES[dtype]
    for n, k in ((64, 0), (0, 40), (0, 0)):
        w = torch.zeros(n, k, dtype=torch.int8, device="cuda")
        dx = W.int8_linear_backward(torch.ones(m, n, dtype=t, device="cuda"), w, torch.ones(n, device="cuda"))
        assert dx.shape == (m, k) and dx.dtype == t and not bool(dx.any())


def test_output_beside_the_adapters_in_one_tensor():
    """Columns between which other operands lie share nothing with them; an operand's own memory is refused."""
    import imagine_b200 as W

    m, n, k, s, r = 30, 64, 64, 2, 16
    gen = torch.Generator("cuda").manual_seed(6)
    x, y, a, b = (torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16)
                  for shape in ((m, k), (m, n), (s, r, k), (s, n, r)))
    want = W.lora_add(y, x, a, b)
    grads = W.lora_backward(y, x, a, b)
    # a row of the buffer: 64 columns of out, then 2048 in which an adapter's a (rows 0 and 1) and b (2 and 3) lie
    big = torch.zeros(m, 64 + 2048, dtype=torch.bfloat16, device="cuda")
    out, tail = big[:, :64], big[:, 64:]
    tail[:2].copy_(a.flatten(1, 2)[:, :1024].repeat(1, 2))
    tail[2:4].copy_(b.flatten(1, 2)[:, :1024].repeat(1, 2))
    ab, bb = tail[:2, :1024].unflatten(1, (r, k)), tail[2:4, :1024].unflatten(1, (n, r))
    assert not ab.is_contiguous() and ab.data_ptr() == big.data_ptr() + 128
    assert torch.equal(W.lora_add(y, x, ab, bb, out=out), want)
    out.zero_()
    dx, da, db = W.lora_backward(y, x, ab, bb, dx=out)
    assert torch.equal(dx, grads[0]) and torch.equal(da, grads[1]) and torch.equal(db, grads[2])
    for t in (a, b):
        part = t.flatten()[:m * 64].view(-1, 64)
        if part.shape[0] == m:
            with pytest.raises(ValueError, match="operand's memory"):
                W.lora_add(y, x, a, b, out=part)
            with pytest.raises(ValueError, match="operand's memory"):
                W.lora_backward(y, x, a, b, dx=part)


@pytest.mark.parametrize("scalar", [False, True])
@pytest.mark.parametrize("k,n", [(264, 4096), (130, 333), (1024, 1040)])
def test_bf16_input_gradient_is_the_same_product_in_every_form(k, n, scalar):
    """bf16: dy times the weight dequantised to bf16, whatever the rows and strides (and so the kernel);
    with one scale for the whole weight, dy times the codes, the scale on the sum: nothing rounded on
    the way.  What is left beside the output's rounding is the fp32 sum: its products, at most sixteen
    splits and eight warps joined (2^-24 each) and the scale's product."""
    import imagine_b200 as W

    g = torch.Generator(device="cuda").manual_seed(k)
    m = 300
    dy = torch.randn(m, n, generator=g, device="cuda").bfloat16()
    w = torch.randint(-128, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    ws = torch.rand(1 if scalar else n, generator=g, device="cuda") * 1e-3 + 1e-4
    if scalar:
        wd = w.double() * ws.double()
    else:
        wd = (w.float() * ws.view(-1, 1)).bfloat16().double()
    ref, size = dy.double() @ wd, dy.double().abs() @ wd.abs()
    rel = _sums(n) + 6 * 2.0 ** -22 + 2.0 ** -23
    apart = torch.empty(m, n + 3, dtype=dy.dtype, device="cuda")[:, 1:1 + n]
    apart.copy_(dy)
    wide = torch.empty(n, k + 5, dtype=torch.int8, device="cuda")[:, 2:2 + k]
    wide.copy_(w)
    for rows in (1, 10, 16, 17, 64, 65, 300):
        for d in (dy, apart):
            for v in (w, wide):
                _check(W.int8_linear_backward(d[:rows], v, ws), ref[:rows], size[:rows], rel, f"{rows} rows")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("m,s,r", [(1, 1, 128), (8, 1, 128), (9, 1, 128), (64, 1, 16), (64, 1, 17), (33, 1, 100), (64, 4, 28),
                                   (64, 4, 29), (64, 64, 128), (64, 1, 72), (64, 8, 128), (2, 70, 5)])
def test_lora_add_of_up_to_64_rows_in_either_form(m, s, r, dtype):
    """Row by row or as a tile, by the rows' share of each adapter; k and n that vectors take and not."""
    import imagine_b200 as W

    for k, n in ((512, 384), (130, 257)):
        x, y, _, a, b, c, idx = _case(m, k, n, s, r, DTYPES[dtype], seed=9)
        out = W.lora_add(y, x, a, b, idx, c)
        _check(out, *_add_ref(x, y, a, b, c, idx), 2 * PIECES[x.dtype] + _sums(k, r), "out")
        assert torch.equal(out[idx < 0], y[idx < 0])
        assert torch.equal(out, W.lora_add(y.clone(), x, a, b, idx, c, out=y))


def test_writing_into_a_saved_tensor_is_noticed():
    """An output written in place counts as a change of it: a graph that saved its old values for the
    backward pass raises instead of going on with the new ones."""
    import imagine_b200 as W

    x, y, dy, a, b, c, idx = _case(20, 64, 64, 2, 8, torch.float32)
    leaf = y.clone().requires_grad_()
    for write in (lambda t: W.lora_add(t, x, a, b, idx, c, out=t), lambda t: W.lora_backward(dy, x, a, b, idx, c, dx=t)):
        held = leaf * 2
        z = held * held
        before = held._version
        write(held.detach())
        assert held._version == before + 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.sum().backward()
    # what is not written stays as it was
    before = [t._version for t in (x, y, dy, a, b, c, idx)]
    W.lora_add(y, x, a, b, idx, c)
    W.lora_backward(dy, x, a, b, idx, c)
    assert before == [t._version for t in (x, y, dy, a, b, c, idx)]
