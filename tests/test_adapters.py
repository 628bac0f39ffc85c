"""What the adapter, input-gradient and checkpointed-activation operators refuse, on
the host: nothing is launched."""
import ctypes

import pytest
import torch

from imagine_b200 import _native as N

P = 0x10000  # any aligned non-null address: never dereferenced on these paths


def _err():
    return N.LIB.w8a8_last_error().decode()


def _add(**kw):
    d = dict(y=P, ldy=64, x=P, ldx=32, dtype=N.BF16, a=P, slot_a=256, b=P, slot_b=512, adapter=P, is64=0, per=1,
             scaling=P, out=P, ldo=64, m=10, n=64, k=32, s=2, r=8, ws=P, ws_bytes=1 << 30)
    d.update(kw)
    return N.LIB.w8a8_lora_add(d["y"], d["ldy"], d["x"], d["ldx"], d["dtype"], d["a"], d["slot_a"], d["b"], d["slot_b"],
                               d["adapter"], d["is64"], d["per"], d["scaling"], d["out"], d["ldo"], d["m"], d["n"],
                               d["k"], d["s"], d["r"], d["ws"], d["ws_bytes"], None)


@pytest.mark.parametrize("kw,word", [
    (dict(m=-1), "negative"), (dict(r=0), "rank"), (dict(r=129), "rank"), (dict(s=0), "adapters"),
    (dict(s=70000), "adapters"), (dict(y=None), "NULL"), (dict(x=None), "NULL"), (dict(out=None), "NULL"),
    (dict(a=None), "NULL"), (dict(b=None), "NULL"), (dict(ldx=31), "stride"), (dict(ldy=63), "stride"),
    (dict(ldo=63), "stride"), (dict(ldo=80), "another row stride"), (dict(dtype=N.S8), "floating"),
    (dict(per=0), "rows_per_index"), (dict(slot_a=255), "overlap"), (dict(slot_b=511), "overlap"),
    (dict(x=P + 1), "aligned"), (dict(adapter=P + 4, is64=1), "aligned"), (dict(scaling=P + 2), "aligned"),
    (dict(ws_bytes=16), "workspace"), (dict(ws=None), "workspace"), (dict(ws=P + 16), "workspace"),
    (dict(m=1 << 40), "sizes"), (dict(m=1 << 30, n=1 << 30), "tiles")])
def test_lora_add_refuses(kw, word):
    assert _add(**kw) == N.ERR_VALUE
    assert word in _err()


def test_lora_add_with_nothing_to_do():
    assert _add(m=0) == 0 and _add(n=0) == 0


def _back(**kw):
    d = dict(dy=P, lddy=64, x=P, ldx=32, xs=None, dtype=N.BF16, a=P, slot_a=256, b=P, slot_b=512, adapter=P, is64=0,
             per=1, scaling=P, dx=2 * P, lddx=32, acc=0, da=P, db=P, m=10, n=64, k=32, s=2, r=8, ws=P, ws_bytes=1 << 30)
    d.update(kw)
    return N.LIB.w8a8_lora_backward(d["dy"], d["lddy"], d["x"], d["ldx"], d["xs"], d["dtype"], d["a"], d["slot_a"],
                                    d["b"], d["slot_b"], d["adapter"], d["is64"], d["per"], d["scaling"], d["dx"],
                                    d["lddx"], d["acc"], d["da"], d["db"], d["m"], d["n"], d["k"], d["s"], d["r"],
                                    d["ws"], d["ws_bytes"], None)


@pytest.mark.parametrize("kw,word", [
    (dict(r=200), "rank"), (dict(da=None), "go together"), (dict(db=None), "go together"), (dict(n=0), "N > 0"),
    (dict(k=0), "N > 0"), (dict(dy=None), "NULL"), (dict(x=None), "NULL"), (dict(lddy=3), "stride"),
    (dict(ldx=3), "stride"), (dict(lddx=3), "stride"), (dict(dtype=N.E4M3), "floating"), (dict(a=None), "NULL"),
    (dict(x=P + 1), "aligned"), (dict(xs=P + 1), "aligned"), (dict(dx=2 * P + 1), "aligned"), (dict(da=P + 1), "aligned"),
    (dict(ws_bytes=100), "workspace"), (dict(dx=P + 64, dy=P + 64), "operand"), (dict(dx=P + 64, x=P + 64), "operand")])
def test_lora_backward_refuses(kw, word):
    assert _back(**kw) == N.ERR_VALUE
    assert word in _err()
    assert _back(dx=None, da=None, db=None) == 0  # nothing wanted


def test_workspace_sizes():
    need = N.LIB.w8a8_lora_workspace_bytes
    assert need(10, 64, 32, 2, 8, 0) >= 10 * 8 * 4
    assert need(10, 64, 32, 2, 200, 0) == N.ERR_VALUE and need(-1, 64, 32, 2, 8, 1) == N.ERR_VALUE
    assert need(10, 64, 32, 2, 8, 3) == N.ERR_VALUE
    # the input gradient alone takes no room for the adapters' sums
    assert need(4096, 4096, 4096, 4, 64, 2) < need(4096, 4096, 4096, 4, 64, 1)
    # partial sums of the adapters' gradients stay bounded
    assert need(100000, 12288, 12288, 64, 128, 1) < 10 << 30
    assert N.LIB.w8a8_input_grad_workspace_bytes(10, 64, 32, N.S8) == N.ERR_VALUE
    assert N.LIB.w8a8_input_grad_workspace_bytes(-1, 64, 32, N.BF16) == N.ERR_VALUE


@pytest.mark.parametrize("kw,word", [
    (dict(dy=None), "NULL"), (dict(w=None), "NULL"), (dict(ws=None), "NULL"), (dict(dx=None), "NULL"),
    (dict(lddy=63), "stride"), (dict(ldw=31), "stride"), (dict(lddx=31), "stride"), (dict(wsn=3), "per-output"),
    (dict(dtype=N.S32), "floating"), (dict(dy=P + 1), "aligned"), (dict(work=None, work_bytes=0), "workspace"),
    (dict(m=-1), "negative")])
def test_input_grad_refuses(kw, word):
    d = dict(dy=P, lddy=4096, w=P, ldw=32, ws=P, wsn=4096, dtype=N.BF16, dx=P, lddx=32, m=10, n=4096, k=32, work=P,
             work_bytes=1 << 30)
    if "lddy" in kw or "wsn" in kw:
        d.update(n=64, wsn=64)
    d.update(kw)
    rc = N.LIB.w8a8_input_grad(d["dy"], d["lddy"], d["w"], d["ldw"], d["ws"], d["wsn"], d["dtype"], d["dx"], d["lddx"],
                               d["m"], d["n"], d["k"], d["work"], d["work_bytes"], None)
    assert rc == N.ERR_VALUE and word in _err()


def test_activation_refuses():
    f, g = N.LIB.w8a8_act_checkpoint, N.LIB.w8a8_act_backward
    assert f(P, N.BF16, 64, 4, 64, 9, P, P, P, None) == N.ERR_VALUE and "activation" in _err()
    assert f(P, N.S8, 64, 4, 64, 1, P, P, P, None) == N.ERR_VALUE and "floating" in _err()
    assert f(P, N.BF16, 64, -4, 64, 1, P, P, P, None) == N.ERR_VALUE
    assert f(None, N.BF16, 64, 4, 64, 1, P, P, P, None) == N.ERR_VALUE and "NULL" in _err()
    assert f(P, N.BF16, 64, 4, 64, N.CKPT_SWIGLU, P, P, P, None) == N.ERR_VALUE and "stride" in _err()
    assert f(P + 1, N.BF16, 64, 4, 64, 1, P, P, P, None) == N.ERR_VALUE and "aligned" in _err()
    assert g(P, N.BF16, 63, 4, 64, 1, P, P, P, None) == N.ERR_VALUE and "stride" in _err()
    assert g(P, N.BF16, 64, 4, 64, 1, None, P, P, None) == N.ERR_VALUE and "NULL" in _err()
    assert f(None, N.BF16, 64, 0, 64, 1, None, None, None, None) == 0


def test_cpu_tensors_are_refused():
    import imagine_b200 as W

    x, y, a, b = torch.zeros(2, 8), torch.zeros(2, 4), torch.zeros(1, 2, 8), torch.zeros(1, 4, 2)
    w, ws = torch.zeros(4, 8, dtype=torch.int8), torch.ones(4)
    for call in (lambda: W.lora_add(y, x, a, b), lambda: W.lora_backward(y, x, a, b),
                 lambda: W.int8_linear_backward(y, w, ws), lambda: W.int8_linear_lora(x, w, ws, None, a, b),
                 lambda: W.act_checkpoint_int8(x), lambda: W.act_backward_int8(x, x, x),
                 lambda: W.checkpointed_activation(x)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="unknown activation"):
        W.act_checkpoint_int8(x, "relu")


def test_argument_helpers():
    """Host-side checks of shapes, strides and indices (device-independent parts)."""
    from imagine_b200 import adapters as A

    t = torch.zeros(4, 6)
    assert A._rows(t)[1] == 6 and A._rows(t[:, :3])[1] == 6 and A._rows(t.t())[0].is_contiguous()
    assert A._rows(t[:1].expand(3, 6))[0].is_contiguous()  # rows that overlap are copied
    assert A._rows(torch.zeros(2, 3, 0))[1] == 1 and A._rows(torch.zeros(2, 0, 5))[1] == 5
    assert A._rows(torch.zeros(1, 9)[:, ::2])[0].is_contiguous()  # elements apart are copied
    assert A._rows(torch.zeros(3, 2, 8)[:, :, :4])[1] == 8  # samples whose rows stay one stride apart
    assert A._index(None, (4,), 4, None) == (None, 0, 1)
    assert A._scaling(None, 3, None) is None


@pytest.mark.parametrize("kw", [
    dict(out=P + 2 * 64),                         # y a row further
    dict(y=P, out=P + 64, ldy=128, ldo=128),      # half of y's columns
    dict(y=P + (1 << 20), out=P + 2 * 16, x=P),   # inside x
    dict(y=P + 2 * 64, out=P, ldo=70, ldy=64)])   # another stride in one range
def test_lora_add_refuses_an_output_that_overlaps(kw):
    assert _add(**{**dict(y=P, x=P + (1 << 21), out=P, m=10, n=64), **kw}) == N.ERR_VALUE
    assert "operand's memory" in _err()


@pytest.mark.parametrize("kw", [
    dict(dx=P + 2 * 32, dy=P, lddy=64), dict(dx=P + 2 * 32, x=P), dict(dx=P + 16, x=P, xs=P)])
def test_lora_backward_refuses_a_gradient_that_overlaps(kw):
    assert _back(**{**dict(dy=P + (1 << 20), x=P + (1 << 21), dx=P + (1 << 22)), **kw}) == N.ERR_VALUE
    assert "operand's memory" in _err()


@pytest.mark.parametrize("dtype", [N.BF16, N.F16, N.F32])
@pytest.mark.parametrize("m", [0, 1, 10, 16, 30, 65, 100])
def test_input_grad_of_a_dimension_of_zero(m, dtype):
    """No output: no workspace and nothing to do, whatever the kernel the row count would choose."""
    need = N.LIB.w8a8_input_grad_workspace_bytes
    for n in (0, 64, 4096):
        assert need(m, n, 0, dtype) == 0 and need(0, n, 64, dtype) == 0
        assert N.LIB.w8a8_input_grad(P, n, P, 0, P, n, dtype, None, 0, m, n, 0, None, 0, None) == 0
        assert N.LIB.w8a8_input_grad(None, n, P, 64, P, n, dtype, None, 64, 0, n, 64, None, 0, None) == 0
    assert need(m, 0, 64, dtype) >= 0  # an empty sum: dx is zero


@pytest.mark.parametrize("backward", [0, 1, 2])
def test_lora_workspace_of_a_dimension_of_zero(backward):
    need = N.LIB.w8a8_lora_workspace_bytes
    for m in (0, 1, 64, 100, 300):
        for n, k in ((0, 64), (64, 0), (0, 0), (64, 64)):
            assert need(m, n, k, 2, 8, backward) >= 0


@pytest.mark.parametrize("kw", [dict(dy=P), dict(dy=P + 2 * 64 * 9 + 2 * 31), dict(w=P + 2 * 32 * 9), dict(w=P - 63 * 32),
                                dict(ws=P + 16)])
def test_input_grad_refuses_a_gradient_in_an_operands_memory(kw):
    d = dict(dy=P + (1 << 22), w=P + (2 << 22), ws=P + (3 << 22))
    d.update(kw)
    rc = N.LIB.w8a8_input_grad(d["dy"], 64, d["w"], 32, d["ws"], 64, N.BF16, P, 64, 10, 64, 32, P + (4 << 22), 1 << 22, None)
    assert rc == N.ERR_VALUE and "operand's memory" in _err()


# Addresses far from each other for whatever a case does not name.
FAR = dict(a=P + (1 << 22), b=P + (2 << 22), adapter=P + (3 << 22), scaling=P + (4 << 22))


@pytest.mark.parametrize("name", list(FAR))
@pytest.mark.parametrize("at", [0, 2 * 64 * 9])  # the output's first row, and its last
def test_lora_add_refuses_an_output_in_the_adapters_memory(name, at):
    far = dict(FAR, y=P + (5 << 22), x=P + (6 << 22))
    assert _add(**{**far, name: P + at, "out": P}) == N.ERR_VALUE
    assert "operand's memory" in _err()
    # the second adapter of a stack alone
    if name in ("a", "b"):
        assert _add(**{**far, name: P - 2 * 4096, f"slot_{name}": 4096, "out": P}) == N.ERR_VALUE
        assert "operand's memory" in _err()


@pytest.mark.parametrize("name", [*FAR, "xs"])
@pytest.mark.parametrize("at", [0, 2 * 32 * 9])
def test_lora_backward_refuses_a_gradient_in_the_adapters_memory(name, at):
    far = dict(FAR, dy=P + (5 << 22), x=P + (6 << 22), xs=P + (7 << 22))
    assert _back(**{**far, name: P + at, "dx": P}) == N.ERR_VALUE
    assert "operand's memory" in _err()
    if name in ("a", "b"):
        assert _back(**{**far, name: P - 2 * 4096, f"slot_{name}": 4096, "dx": P}) == N.ERR_VALUE
        assert "operand's memory" in _err()


def test_sizes_whose_steps_would_pass_31_bits_are_refused():
    """A block steps through a dimension in 32 bits, by up to 2048 elements at a time."""
    most = (1 << 31) - (1 << 20)
    need = N.LIB.w8a8_lora_workspace_bytes
    grad = N.LIB.w8a8_input_grad_workspace_bytes
    for big in (most + 1, 0x7fffff00, 1 << 31):
        for sizes in ((big, 64, 64), (1, big, 64), (1, 64, big)):
            for backward in (0, 1, 2):
                assert need(*sizes, 1, 1, backward) == N.ERR_VALUE and "sizes" in _err()
            for dtype in (N.BF16, N.F16, N.F32):
                assert grad(*sizes, dtype) == N.ERR_VALUE and "sizes" in _err()
        assert N.LIB.w8a8_act_checkpoint(P, N.BF16, 64, big, 64, 1, P, P, P, None) == N.ERR_VALUE
        assert N.LIB.w8a8_act_backward(P, N.BF16, big, 1, big // 2 + 1, 1, P, P, P, None) == N.ERR_VALUE
    for sizes in ((most, 64, 64), (1, most, 64), (1, 64, most)):
        assert need(*sizes, 1, 1, 0) >= 0 and grad(*sizes, N.BF16) >= 0


@pytest.mark.parametrize("size", [(1 << 31) - (1 << 20), (1 << 31) - (1 << 20) - 1, (1 << 30) + 7, 4096, 1])
def test_last_steps_of_the_largest_sizes_stay_below_31_bits(size):
    """The kernels' index arithmetic, restated: each loop's counter after its last step."""
    top = (1 << 31) - 1
    sms = 148
    # few rows: 256 threads of eight elements
    assert size - 1 + 256 * 8 <= top
    # contractions cut into at most 16 splits of whole steps of 64 or 128
    for step in (64, 128):
        steps = -(-size // step)
        for want in range(1, 17):
            per = -(-steps // want)
            assert -(-steps // per) * per * step + 2 * step <= top
    # column ranges: up to six blocks a multiprocessor, of whole tiles of 128
    tiles = -(-size // 128)
    for want in range(1, 6 * sms + 1):
        per = -(-tiles // min(want, tiles))
        assert -(-tiles // per) * per * 128 + 128 <= top
