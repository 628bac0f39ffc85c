"""The adapters' kernels for long bf16 batches (tiles of 128 rows, TMA operands): mixed tiles,
ragged ends, every padded rank, and the batches beside them that take the other form.
Tolerances as in test_gpu_adapters."""
import pytest
import torch

from tests.test_gpu_adapters import PIECES, _add_ref, _case, _check, _check_grads, _grad_ref, _sums

pytestmark = pytest.mark.gpu


def _ragged(m, s, seed, none=True):
    """Adapters of ragged requests: runs of rows, some without an adapter."""
    g = torch.Generator().manual_seed(seed)
    idx = torch.empty(m, dtype=torch.int32)
    at = 0
    while at < m:
        run = int(torch.randint(1, max(2, m // 3), (1,), generator=g))
        idx[at:at + run] = int(torch.randint(-1 if none else 0, s, (1,), generator=g))
        at += run
    return idx.cuda()


def _quiet():
    import imagine_b200 as W

    assert W.device_error() == 0


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("m,k,n,s,r", [
    (256, 64, 64, 1, 8), (257, 136, 72, 2, 16), (300, 512, 264, 3, 24), (511, 1032, 520, 5, 32), (640, 192, 1544, 4, 64),
    (1000, 1024, 776, 7, 40), (777, 256, 512, 2, 128), (384, 2056, 200, 64, 16), (1290, 320, 328, 3, 104)])
def test_every_rank_and_ragged_ends(m, k, n, s, r, codes):
    import imagine_b200 as W

    x, y, dy, a, b, c, _ = _case(m, k, n, s, r, torch.bfloat16, seed=2)
    idx = _ragged(m, s, m + r)
    if not codes:
        out = W.lora_add(y, x, a, b, idx, c)
        _check(out, *_add_ref(x, y, a, b, c, idx), 2 * PIECES[x.dtype] + _sums(k, r), "out")
        assert torch.equal(out[idx < 0], y[idx < 0])
        assert torch.equal(out, W.lora_add(y.clone(), x, a, b, idx.long(), c, out=y))
    xs, data = None, x
    if codes:
        x, xs = W.quantize_int8_rowwise(x)
        data = x.double() * xs.double()
    got = W.lora_backward(dy, x, a, b, idx, c, x_scale=xs)
    _check_grads(got, data, dy, a, b, c, idx)
    assert not bool(got[0][idx < 0].any())
    assert all(torch.equal(p, q) for p, q in zip(got, W.lora_backward(dy, x, a, b, idx, c, x_scale=xs)))
    base = torch.randn(m, k, device="cuda").bfloat16()
    dx = W.lora_backward(dy, x, a, b, idx, c, x_scale=xs, dx=base.clone(), need_weights=False)[0]
    ref, size = _grad_ref(data, dy, a, b, c, idx)["dx"]
    _check(dx, ref + base.double(), size, 2 * PIECES[dy.dtype] + _sums(n, r), "dx added")
    assert torch.equal(dx[idx < 0], base[idx < 0])
    _quiet()


@pytest.mark.parametrize("s,r", [(64, 16), (64, 64), (9, 128), (70, 8)])
def test_every_row_another_adapter(s, r):
    """Rows of all adapters in every tile (more than there are accumulators for); over 64 adapters
    the other form runs."""
    import imagine_b200 as W

    m, k, n = 400, 264, 392
    x, y, dy, a, b, c, idx = _case(m, k, n, s, r, torch.bfloat16)
    _check(W.lora_add(y, x, a, b, idx, c), *_add_ref(x, y, a, b, c, idx), 2 * PIECES[x.dtype] + _sums(k, r))
    _check_grads(W.lora_backward(dy, x, a, b, idx, c), x, dy, a, b, c, idx)
    _quiet()


def test_nan_stays_in_its_rows_and_adapters():
    import imagine_b200 as W

    m, k, n, s, r = 700, 256, 384, 3, 16
    x, y, dy, a, b, c, _ = _case(m, k, n, s, r, torch.bfloat16)
    idx = _ragged(m, s, 11)
    idx[100:140], idx[600:650], idx[300:310] = 1, 1, -1
    clean, grads = W.lora_add(y, x, a, b, idx, c), W.lora_backward(dy, x, a, b, idx, c)
    bad = idx == 1
    for v in (float("nan"), float("inf")):
        xb, yb, dyb, ab, bb = x.clone(), y.clone(), dy.clone(), a.clone(), b.clone()
        xb[bad], yb[bad], dyb[bad], ab[1], bb[1] = v, v, v, v, v
        xb[idx < 0], dyb[idx < 0] = v, v
        out = W.lora_add(yb, xb, ab, bb, idx, c)
        assert torch.equal(out[~bad], clean[~bad]) and not bool(out[bad].isfinite().any())
        dx, da, db = W.lora_backward(dyb, xb, ab, bb, idx, c)
        assert torch.equal(dx[~bad], grads[0][~bad]) and not bool(dx[bad].isfinite().any())
        for t, ref in ((da, grads[1]), (db, grads[2])):
            assert torch.equal(t[[0, 2]], ref[[0, 2]]) and not bool(t[1].isfinite().any())
    _quiet()


def test_operands_that_lie_elsewhere():
    """Rows apart (16-byte strides: the same form; odd ones: the other), a stack's every second adapter,
    samples of a batch, and rows of the output's surroundings left as they were."""
    import imagine_b200 as W

    bt, t, k, n, s, r = 3, 130, 136, 200, 4, 16
    m = bt * t
    x, y, dy, a, b, c, _ = _case(m, k, n, s, r, torch.bfloat16)
    sample = torch.tensor([2, -1, 0], device="cuda")
    token = sample.repeat_interleave(t)
    want, grads = W.lora_add(y, x, a, b, token, c), W.lora_backward(dy, x, a, b, token, c)
    for p, q in zip(W.lora_backward(dy.view(bt, t, n), x.view(bt, t, k), a, b, sample, c), grads):
        assert torch.equal(p.reshape(q.shape), q)
    assert torch.equal(W.lora_add(y.view(bt, t, n), x.view(bt, t, k), a, b, sample, c).view(m, n), want)

    def apart(v, pad, at):
        big = torch.full((v.shape[0], v.shape[1] + pad), float("nan"), dtype=v.dtype, device="cuda")
        big[:, at:at + v.shape[1]] = v
        return big[:, at:at + v.shape[1]]
    a2 = torch.full((2 * s, r, k), float("nan"), dtype=a.dtype, device="cuda")
    b2 = torch.full((2 * s, n, r), float("nan"), dtype=a.dtype, device="cuda")
    a2[::2], b2[::2] = a, b
    xa, ya, dya = apart(x, 24, 8), apart(y, 16, 16), apart(dy, 8, 0)
    wide = torch.full((m, n + 24), 7.0, dtype=y.dtype, device="cuda")
    W.lora_add(ya, xa, a2[::2], b2[::2], token, c, out=wide[:, 8:8 + n])
    assert torch.equal(wide[:, 8:8 + n], want)
    assert bool((wide[:, :8] == 7).all()) and bool((wide[:, 8 + n:] == 7).all())
    for p, q in zip(W.lora_backward(dya, xa, a2[::2], b2[::2], token, c), grads):
        assert torch.equal(p, q)
    # rows that TMA cannot take: other kernels, the same values up to the order of the sums
    for p, q in zip(W.lora_backward(apart(dy, 3, 1), apart(x, 5, 2), a, b, token, c), grads):
        assert float((p.double() - q.double()).norm() / q.double().norm()) < 2.0 ** -8
    odd = W.lora_add(apart(y, 1, 0), apart(x, 3, 1), a, b, token, c)
    _check(odd, *_add_ref(x, y, a, b, c, token), 2 * PIECES[x.dtype] + _sums(k, r))
    assert torch.equal(odd[token < 0], y[token < 0])


@pytest.mark.parametrize("rows", [64, 65, 255, 256, 2048 * 64 + 70])
def test_borders_of_the_forms(rows):
    """Row counts where another kernel, or another split of a long batch, takes over."""
    import imagine_b200 as W

    k, n, s, r = 64, 72, 2, 8
    x, y, dy, a, b, c, _ = _case(rows, k, n, s, r, torch.bfloat16)
    idx = (torch.arange(rows, device="cuda") * s // rows).int()
    idx[rows // 3] = -1
    _check(W.lora_add(y, x, a, b, idx, c), *_add_ref(x, y, a, b, c, idx), 2 * PIECES[x.dtype] + _sums(k, r))
    _check_grads(W.lora_backward(dy, x, a, b, idx, c), x, dy, a, b, c, idx)
    _quiet()


def test_two_streams_and_a_graph():
    """Two calls at once on two streams, and a captured step whose replay reads new contents."""
    import imagine_b200 as W

    sets = [_case(500, 512, 640, 3, 32, torch.bfloat16, seed=q) for q in (1, 2)]
    idx = _ragged(500, 3, 5)
    w = torch.randint(-127, 128, (640, 512), device="cuda", dtype=torch.int8)
    ws = torch.rand(640, device="cuda") * 1e-3

    def step(x, y, dy, a, b, c, _):
        base = W.int8_linear_backward(dy, w, ws)
        return (W.lora_add(y, x, a, b, idx, c), *W.lora_backward(dy, x, a, b, idx, c, dx=base))
    want = [step(*q) for q in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(step(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for run in got[i]:
            assert all(torch.equal(p, q) for p, q in zip(run, want[i]))
    held_in = [t.clone() for t in sets[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(*held_in)
    for i in (1, 0):
        for dst, src in zip(held_in, sets[i]):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, want[i]))
    _quiet()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_long_batches_of_the_other_types(dtype):
    import imagine_b200 as W

    m, k, n, s, r = 1100, 520, 264, 3, 24
    x, y, dy, a, b, c, _ = _case(m, k, n, s, r, dtype)
    idx = _ragged(m, s, 3)
    _check(W.lora_add(y, x, a, b, idx, c), *_add_ref(x, y, a, b, c, idx), 2 * PIECES[dtype] + _sums(k, r))
    _check_grads(W.lora_backward(dy, x, a, b, idx, c), x, dy, a, b, c, idx)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_a_layer_as_it_is_trained(dtype):
    """MLP up, activation, MLP down with adapters: the run of the operators together, its gradients
    against the same layer in 64 bits with the inputs that the operators kept."""
    import imagine_b200 as W

    g = torch.Generator(device="cuda").manual_seed(9)
    t, k, f, s, r = 320, 256, 512, 2, 16
    def rn(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)
    x = rn(t, k).requires_grad_()
    up, ups = W.quantize_weight(rn(f, k, std=0.05).bfloat16())
    down, downs = W.quantize_weight(rn(k, f, std=0.05).bfloat16())
    leaves = [rn(s, r, k, std=0.05), rn(s, f, r, std=0.1), rn(s, r, f, std=0.05), rn(s, k, r, std=0.1)]
    for q in leaves:
        q.requires_grad_()
    idx = _ragged(t, s, 4)
    c = torch.tensor([1.0, 0.5], device="cuda")
    u = W.int8_linear_lora(x, up, ups, None, leaves[0], leaves[1], idx, c)
    h = W.checkpointed_activation(u)
    z = W.int8_linear_lora(h, down, downs, None, leaves[2], leaves[3], idx, c)
    dz = rn(t, k)
    grads = torch.autograd.grad(z, (x, *leaves), dz)
    # the same backward in 64 bits, from what was kept
    def kept(v):
        q, sc = W.quantize_int8_rowwise(v.detach())
        return q.double() * sc.double()
    hk, xk = kept(h), kept(x)
    uq, us = W.act_checkpoint_int8(u.detach())[1:]
    uk = (uq.float() * us.repeat_interleave(128, 1)).double().requires_grad_()
    a1, b1, a2, b2 = (q.detach().double() for q in leaves)
    dz64 = dz.double()

    def through(d, wq, wsc, a, b, inp):
        ref = _grad_ref(inp, d, a, b, c, idx)
        return d @ (wq.double() * wsc.double().view(-1, 1)) + ref["dx"][0], ref["da"][0], ref["db"][0]
    dh, da2, db2 = through(dz64, down, downs, a2, b2, hk)
    du = torch.autograd.grad(torch.nn.functional.gelu(uk, approximate="tanh"), uk, dh)[0]
    dx, da1, db1 = through(du, up, ups, a1, b1, xk)
    # per operator: its inputs' and its own rounding (u each), seven of them in the longest chain
    u_ = torch.finfo(dtype).eps / 2
    for name, got, ref in zip(("x", "a1", "b1", "a2", "b2"), grads, (dx, da1, db1, da2, db2)):
        off = float((got.double() - ref).norm() / ref.norm())
        assert off < 7 * u_ + 1e-5, (name, off)


@pytest.mark.parametrize("r", [8, 16, 24, 32, 64, 128])
@pytest.mark.parametrize("s", [16, 33, 64])
@pytest.mark.parametrize("codes", [False, True])
def test_as_many_adapters_in_a_block_as_tensor_memory_holds(s, r, codes):
    """A long contraction of rows of many adapters: a block's accumulators take all of its columns, and
    several passes where there are more adapters."""
    import imagine_b200 as W

    m, wide, narrow = 1500, 2048, 64
    x, y, _, a, b, c, idx = _case(m, wide, narrow, s, r, torch.bfloat16, seed=5)
    _check(W.lora_add(y, x, a, b, idx, c), *_add_ref(x, y, a, b, c, idx), 2 * PIECES[x.dtype] + _sums(wide, r))
    _quiet()
    x, _, dy, a, b, c, idx = _case(m, narrow, wide, s, r, torch.bfloat16, seed=6)
    xs, data = None, x
    if codes:
        x, xs = W.quantize_int8_rowwise(x)
        data = x.double() * xs.double()
    _check_grads(W.lora_backward(dy, x, a, b, idx, c, x_scale=xs), data, dy, a, b, c, idx)
    _quiet()
    x, _, dy, a, b, c, idx = _case(m, wide, narrow, s, r, torch.bfloat16, seed=7)
    if codes:
        x, xs = W.quantize_int8_rowwise(x)
        data = x.double() * xs.double()
    else:
        data = x
    ref = _grad_ref(data, dy, a, b, c, idx)
    dx, da, db = W.lora_backward(dy, x, a, b, idx, c, x_scale=xs, need_dx=False)
    assert dx is None
    _check(da, *ref["da"], 2 * PIECES[dy.dtype] + _sums(narrow, m), "da")
    _check(db, *ref["db"], 2 * PIECES[dy.dtype] + _sums(wide, m), "db")
    _quiet()


@pytest.mark.parametrize("m,k,n,s,r", [
    (2000, 264, 4096, 4, 16), (700, 4096, 512, 16, 64), (1500, 264, 2048, 64, 16), (1500, 2048, 264, 9, 128),
    (3100, 512, 520, 64, 64), (3300, 1032, 1544, 5, 40)])
@pytest.mark.parametrize("order", ["mixed", "runs", "some"])
def test_many_adapters_in_tiles_of_blocks_with_several(m, k, n, s, r, order):
    """More tiles than multiprocessors, so that a block goes through several, each with as many products
    as its 128 rows have adapters: every row another one, short runs, or tiles of one, none and many."""
    import imagine_b200 as W

    x, y, dy, a, b, c, idx = _case(m, k, n, s, r, torch.bfloat16, seed=4)
    if order == "runs":
        idx = (torch.arange(m, device="cuda") // 11 % (s + 1) - 1).int()
    elif order == "some":
        tile = torch.arange(m, device="cuda") // 128
        idx = torch.where(tile % 3 == 0, idx, torch.where(tile % 3 == 1, tile.int() % s, -1)).int()
    out = W.lora_add(y, x, a, b, idx, c)
    _quiet()
    _check(out, *_add_ref(x, y, a, b, c, idx), 2 * PIECES[x.dtype] + _sums(k, r), "out")
    assert torch.equal(out, W.lora_add(y.clone(), x, a, b, idx, c, out=y))
    got = W.lora_backward(dy, x, a, b, idx, c)
    _quiet()
    _check_grads(got, x, dy, a, b, c, idx)
    base = torch.randn(m, k, device="cuda").bfloat16()
    dx = W.lora_backward(dy, x, a, b, idx, c, dx=base.clone(), need_weights=False)[0]
    _quiet()
    ref, size = _grad_ref(x, dy, a, b, c, idx)["dx"]
    _check(dx, ref + base.double(), size, 2 * PIECES[dy.dtype] + _sums(n, r), "dx added")


# The tcgen05 form takes batches from 256 rows on of 5 to 8 Mi elements (2 to 3 Mi with more than eight
# adapters): the smallest and oddest of those, of every padded rank.
LONG = [
    (1300, 4104, 2568, 1, 8), (2049, 4096, 72, 2, 16), (2049, 72, 4096, 2, 24), (257, 16400, 16392, 3, 24),
    (511, 8200, 8328, 5, 32), (1000, 1544, 7000, 4, 64), (777, 5504, 5512, 2, 128), (3001, 2048, 776, 7, 40),
    (1290, 3208, 3320, 3, 104), (256, 8200, 4200, 64, 16)]


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("m,k,n,s,r", LONG)
def test_every_rank_and_ragged_ends_of_long_batches(m, k, n, s, r, codes):
    test_every_rank_and_ragged_ends(m, k, n, s, r, codes)


def test_nan_stays_in_its_rows_and_adapters_of_long_batches():
    import imagine_b200 as W

    m, k, n, s, r = 2100, 2048, 2056, 3, 16
    x, y, dy, a, b, c, _ = _case(m, k, n, s, r, torch.bfloat16)
    idx = _ragged(m, s, 11)
    idx[100:140], idx[600:650], idx[300:310], idx[1900:1905] = 1, 1, -1, 1
    clean, grads = W.lora_add(y, x, a, b, idx, c), W.lora_backward(dy, x, a, b, idx, c)
    bad = idx == 1
    for v in (float("nan"), float("inf")):
        xb, yb, dyb, ab, bb = x.clone(), y.clone(), dy.clone(), a.clone(), b.clone()
        xb[bad], yb[bad], dyb[bad], ab[1], bb[1] = v, v, v, v, v
        xb[idx < 0], dyb[idx < 0] = v, v
        out = W.lora_add(yb, xb, ab, bb, idx, c)
        assert torch.equal(out[~bad], clean[~bad]) and not bool(out[bad].isfinite().any())
        dx, da, db = W.lora_backward(dyb, xb, ab, bb, idx, c)
        assert torch.equal(dx[~bad], grads[0][~bad]) and not bool(dx[bad].isfinite().any())
        for t, ref in ((da, grads[1]), (db, grads[2])):
            assert torch.equal(t[[0, 2]], ref[[0, 2]]) and not bool(t[1].isfinite().any())
    _quiet()


def test_operands_of_long_batches_that_lie_elsewhere():
    """Rows a multiple of 16 bytes apart, a stack's every second adapter, samples of a batch: the same
    bits; the output's surroundings left as they were; rows that TMA cannot take: the same values."""
    import imagine_b200 as W

    bt, t, k, n, s, r = 3, 700, 2056, 2040, 4, 16
    m = bt * t
    x, y, dy, a, b, c, _ = _case(m, k, n, s, r, torch.bfloat16)
    sample = torch.tensor([2, -1, 0], device="cuda")
    token = sample.repeat_interleave(t)
    want, grads = W.lora_add(y, x, a, b, token, c), W.lora_backward(dy, x, a, b, token, c)
    for p, q in zip(W.lora_backward(dy.view(bt, t, n), x.view(bt, t, k), a, b, sample, c), grads):
        assert torch.equal(p.reshape(q.shape), q)
    assert torch.equal(W.lora_add(y.view(bt, t, n), x.view(bt, t, k), a, b, sample, c).view(m, n), want)

    def apart(v, pad, at):
        big = torch.full((v.shape[0], v.shape[1] + pad), float("nan"), dtype=v.dtype, device="cuda")
        big[:, at:at + v.shape[1]] = v
        return big[:, at:at + v.shape[1]]
    a2 = torch.full((2 * s, r, k), float("nan"), dtype=a.dtype, device="cuda")
    b2 = torch.full((2 * s, n, r), float("nan"), dtype=a.dtype, device="cuda")
    a2[::2], b2[::2] = a, b
    xa, ya, dya = apart(x, 24, 8), apart(y, 16, 16), apart(dy, 8, 0)
    wide = torch.full((m + 1, n + 24), 7.0, dtype=y.dtype, device="cuda")
    W.lora_add(ya, xa, a2[::2], b2[::2], token, c, out=wide[:m, 8:8 + n])
    assert torch.equal(wide[:m, 8:8 + n], want) and bool((wide[m] == 7).all())
    assert bool((wide[:, :8] == 7).all()) and bool((wide[:, 8 + n:] == 7).all())
    base = torch.full((m + 1, k + 16), 7.0, dtype=y.dtype, device="cuda")
    base[:m, 8:8 + k] = 0
    got = W.lora_backward(dya, xa, a2[::2], b2[::2], token, c, dx=base[:m, 8:8 + k])
    assert all(torch.equal(p, q) for p, q in zip(got, grads))
    assert bool((base[:, :8] == 7).all()) and bool((base[:, 8 + k:] == 7).all()) and bool((base[m] == 7).all())
    for p, q in zip(W.lora_backward(apart(dy, 3, 1), apart(x, 5, 2), a, b, token, c), grads):
        assert float((p.double() - q.double()).norm() / q.double().norm()) < 2.0 ** -8
    odd = W.lora_add(apart(y, 1, 0), apart(x, 3, 1), a, b, token, c)
    _check(odd, *_add_ref(x, y, a, b, c, token), 2 * PIECES[x.dtype] + _sums(k, r))
    # a dx or an out alone that TMA cannot take: the contraction's sums go to the other form's product
    out = torch.empty(m, n + 3, dtype=y.dtype, device="cuda")[:, 1:1 + n]
    _check(W.lora_add(y, x, a, b, token, c, out=out), *_add_ref(x, y, a, b, c, token), 2 * PIECES[x.dtype] + _sums(k, r))
    odd = torch.zeros(m, k + 3, dtype=y.dtype, device="cuda")[:, 1:1 + k]
    _check_grads(W.lora_backward(dy, x, a, b, token, c, dx=odd), x, dy, a, b, c, token)
    _quiet()


@pytest.mark.parametrize("m,n,k,s", [
    (1279, 2048, 2048, 1), (1280, 2048, 2048, 1), (2047, 2048, 2048, 8), (2048, 2048, 2048, 8), (767, 2048, 2048, 9),
    (768, 2048, 2048, 9), (511, 2048, 2048, 9), (512, 2048, 2048, 64), (2048, 2048, 2048, 65), (255, 20000, 20000, 2)])
def test_borders_between_the_forms_by_work(m, n, k, s):
    import imagine_b200 as W

    r = 16
    x, y, dy, a, b, c, idx = _case(m, k, n, s, r, torch.bfloat16, seed=8)
    _check(W.lora_add(y, x, a, b, idx, c), *_add_ref(x, y, a, b, c, idx), 2 * PIECES[x.dtype] + _sums(k, r))
    _check_grads(W.lora_backward(dy, x, a, b, idx, c), x, dy, a, b, c, idx)
    _quiet()


def test_long_calls_on_three_streams():
    """Contractions, products and sums over rows of three streams at once, with the linear and its input
    gradient among them: each run has the bits of the call alone."""
    import imagine_b200 as W

    steps = []
    for seed, (m, k, n, s, r) in enumerate(((1500, 4096, 2048, 3, 16), (3100, 512, 2048, 64, 64), (5000, 1024, 1024, 2, 128))):
        x, y, dy, a, b, c, idx = _case(m, k, n, s, r, torch.bfloat16, seed=seed)
        w = torch.randint(-127, 128, (n, k), device="cuda", dtype=torch.int8)
        ws = torch.rand(n, device="cuda") * 1e-3
        q, xs = W.quantize_int8_rowwise(x)

        def step(x=x, dy=dy, a=a, b=b, c=c, idx=idx, w=w, ws=ws, q=q, xs=xs):
            base = W.int8_linear_backward(dy, w, ws)
            z = W.lora_add(W.int8_linear(x, w, ws), x, a, b, idx, c)
            return (z, *W.lora_backward(dy, q, a, b, idx, c, x_scale=xs, dx=base), *W.act_checkpoint_int8(z))
        steps.append(step)
    want = [f() for f in steps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(4):
        got = []
        for f, st in zip(steps, streams):
            with torch.cuda.stream(st):
                got.append(f())
        torch.cuda.synchronize()
        for run, ref in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(run, ref))
    _quiet()


@pytest.mark.parametrize("m,k,n", [(200000, 512, 12288), (1100000, 2048, 2040)])
def test_offsets_beyond_32_bits(m, k, n):
    """Operands of more than 2^31 elements: the last rows against the formula."""
    import imagine_b200 as W

    s, r = 3, 16
    x, y, a, b = (torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(0, std)
                  for shape, std in (((m, k), 1), ((m, n), 1), ((s, r, k), k ** -0.5), ((s, n, r), 0.5)))
    assert y.numel() > 1 << 31
    c = torch.ones(s, device="cuda")
    idx = torch.arange(m, device="cuda") * s // m
    last = slice(m - 300, m)
    out = W.lora_add(y, x, a, b, idx, c)
    _check(out[last], *_add_ref(x[last], y[last], a, b, c, idx[last]), 2 * PIECES[x.dtype] + _sums(k, r))
    assert torch.equal(W.lora_add(y, x, a, b, torch.full_like(idx, -1), c, out=out)[last], y[last])
    del out
    dx = W.lora_backward(y, None, a, b, idx, c, need_weights=False)[0]
    ref, size = _grad_ref(x[last], y[last], a, b, c, idx[last])["dx"]
    _check(dx[last], ref, size, 2 * PIECES[y.dtype] + _sums(n, r))
    w = torch.randint(-127, 128, (n, k), device="cuda", dtype=torch.int8)
    dx = W.int8_linear_backward(y, w, torch.ones(1, device="cuda"))
    _check(dx[last], y[last].double() @ w.double(), y[last].double().abs() @ w.double().abs(), _sums(n) + 8 * 2.0 ** -22)
    o, q, scale = W.act_checkpoint_int8(y)
    few = W.act_checkpoint_int8(y[last])
    assert all(torch.equal(p[last], v) for p, v in zip((o, q, scale), few))
    assert torch.equal(W.act_backward_int8(y, q, scale)[last], W.act_backward_int8(y[last], *few[1:]))
    _quiet()
