"""The operators of adapter training and serving beside the W8A8 linears, as they are measured.

Four operators, each in its plain form (elementary torch operations in 32 bits, rounded once at the
end) and, with ``own``, as a user calls it:

* ``add``   ``lora_add(y, x, a, b, adapter, scaling)``: the low-rank adapters of many requests
  beside one shared projection, ``out = y + scaling[s] * (x a[s]^T) b[s]^T`` with ``s`` the row's
  adapter (-1: none, the row of y is returned as it is).
* ``grad``  ``lora_backward(dy, x, a, b, adapter, scaling, x_scale)``: its gradients (dx, da, db),
  from x itself or from its 8-bit checkpoint (int8 codes and one scale a row, what the W8A8 linear
  made of it in the forward pass).
* ``act``   ``act_checkpoint_int8(x, act)`` and ``act_backward_int8(dy, q, scale, act)``: an
  activation that keeps its input in 8 bits (groups of 128 along a row, one fp32 scale each), and
  the gradient from those bits.
* ``dx``    ``int8_linear_backward(dy, weight, weight_scale)``: the gradient of the W8A8 linear's
  input, ``dx = dy (weight_scale * weight)``.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
GROUP = 128  # elements of a row that share one scale in an activation's 8-bit checkpoint


def listed():
    return [
        # one request decodes one token: latency is all
        dict(name="add_token", op="add", dtype="bf16", rows=1, requests=1, adapters=8, rank=16, k=4096, n=4096),
        # a decode batch, each row another request, 32 adapters and a few rows without one
        dict(name="add_decode", op="add", dtype="bf16", rows=64, requests=64, adapters=32, rank=32, k=4096, n=12288),
        # 256 text and 5600 image tokens a sample, two samples, each with an adapter of its own
        dict(name="add_image", op="add", dtype="bf16", rows=11712, requests=3, adapters=3, rank=64, k=4096, n=12288),
        # half precision, odd sizes, ragged requests
        dict(name="add_odd", op="add", dtype="f16", rows=777, requests=5, adapters=4, rank=12, k=1000, n=1501),
        # one adapter trained on one sample, x kept as it was
        dict(name="grad_one", op="grad", dtype="bf16", int8=False, rows=5856, requests=1, adapters=1, rank=16, k=4096, n=4096),
        # four adapters trained at once on a batch, x kept as the linear's int8 codes
        dict(name="grad_int8", op="grad", dtype="bf16", int8=True, rows=11712, requests=5, adapters=4, rank=64, k=4096, n=12288),
        # a short text, full precision, odd sizes
        dict(name="grad_odd", op="grad", dtype="f32", int8=False, rows=77, requests=3, adapters=3, rank=8, k=650, n=1283),
        # the MLP's activation: forward, its 8-bit checkpoint and the gradient from it
        dict(name="act_gelu", op="act", act="gelu_tanh", step=True, dtype="bf16", rows=5856, k=12288),
        # the gated activation's gradient from a checkpoint that the forward pass left
        dict(name="act_swiglu", op="act", act="swiglu", step=False, dtype="bf16", rows=5856, k=12288),
        # a short text, half precision, a last group that is not whole
        dict(name="act_text", op="act", act="silu", step=True, dtype="f16", rows=77, k=1200),
        # the MLP-up projection's input gradient over the joint sequence
        dict(name="dx_up", op="dx", dtype="bf16", rows=5856, k=4096, n=12288),
        # the text stream's out-projection, sizes off the tiles
        dict(name="dx_text", op="dx", dtype="f16", rows=250, k=4112, n=4080),
    ]


def _spread(rng, low, high, step=1):
    """A whole number in [low, high], spread over its logarithm, a multiple of ``step``."""
    v = math.exp(rng.uniform(math.log(low), math.log(high + 0.999)))
    return max(low, min(high, int(v) // step * step)) if step > 1 else max(low, min(high, int(v)))


def draw(rng):
    op = rng.choice(["add", "add", "grad", "grad", "act", "dx"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f32"])
    step = rng.choice([1, 8, 16, 128])
    if op == "act":
        return dict(op=op, act=rng.choice(["gelu_tanh", "silu", "swiglu"]), step=rng.random() < 0.6, dtype=dtype,
                    rows=_spread(rng, 1, 4096), k=_spread(rng, max(64, step), 12288, step))
    k, n = _spread(rng, 256, 4096, step), _spread(rng, 256, 8192, step)
    if op == "dx":
        return dict(op=op, dtype=dtype, rows=_spread(rng, 1, 2048 if dtype == "f32" else 4096), k=k, n=n)
    rows = _spread(rng, 1, 8192)
    # short batches are decode steps (a request a row), long ones a few ragged requests
    requests = rows if rows <= 128 else rng.randint(1, 8)
    case = dict(op=op, dtype=dtype, rows=rows, requests=requests, adapters=rng.randint(1, 16 if op == "add" else 4),
                rank=rng.choice([4, 8, 12, 16, 16, 32, 64]), k=k, n=n)
    if op == "grad":
        case["int8"] = rng.random() < 0.5
    return case


def _adapter_of_request(case):
    """Request i's adapter: the adapters in turn, every eighth request has none."""
    return [-1 if i % 8 == 5 else i % case["adapters"] for i in range(case["requests"])]


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed * 7919 + 17)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dtype):
        return (torch.randn(*shape, generator=gen, device=dev) * std).to(dtype)

    rows, k = case["rows"], case["k"]
    st = dict(case=case)
    if case["op"] == "act":
        width = 2 * k if case["act"] == "swiglu" else k
        x = normal(rows, width, std=2.0)
        st["dy"] = normal(rows, k)
        if case["step"]:
            st["x"] = x
        else:
            st["q"], st["scale"] = _quantise_groups(x.float(), k)
        return st
    n = case["n"]
    if case["op"] == "dx":
        st["dy"] = normal(rows, n)
        st["w"] = torch.randn(n, k, generator=gen, device=dev).mul_(40.0).round_().clamp_(-127, 127).to(torch.int8)
        st["ws"] = torch.rand(n, generator=gen, device=dev) * 4e-4 + 4e-4
        return st
    s, r = case["adapters"], case["rank"]
    x = normal(rows, k)
    st["a"] = normal(s, r, k, std=k ** -0.5)
    st["b"] = normal(s, n, r, std=0.5 * r ** -0.5)
    st["scaling"] = torch.rand(s, generator=gen, device=dev) + 0.5
    # ragged requests: consecutive rows of one request share its adapter
    cuts = torch.rand(case["requests"] - 1, generator=gen, device=dev).mul_(rows).long() if rows > case["requests"] else \
        torch.arange(1, case["requests"], device=dev)
    request = torch.zeros(rows, dtype=torch.long, device=dev).index_add_(0, cuts, torch.ones_like(cuts)).cumsum(0)
    st["adapter"] = torch.tensor(_adapter_of_request(case), dtype=torch.int32, device=dev)[request]
    if case["op"] == "add":
        st["x"], st["y"] = x, normal(rows, n)
        return st
    st["dy"] = normal(rows, n)
    if case["int8"]:
        scale = (x.float().abs().amax(1, keepdim=True) / 127.0).clamp_min(1e-30)
        st["x"], st["x_scale"] = torch.round(x.float() / scale).to(torch.int8), scale
    else:
        st["x"], st["x_scale"] = x, None
    return st


# ------------------------------------------------------------------ plain forms
def _quantise_groups(x, k):
    """fp32 rows -> int8 codes and the scale of every group of 128 (the last of k elements, or of
    each half of a gated pair, may be shorter)."""
    halves = x.unflatten(-1, (-1, k))
    pad = -k % GROUP
    g = torch.nn.functional.pad(halves, (0, pad)).unflatten(-1, (-1, GROUP))
    scale = (g.abs().amax(-1) / 127.0).clamp_min(1e-30)
    q = torch.round(g / scale.unsqueeze(-1)).to(torch.int8)
    return q.flatten(-2)[..., :k].flatten(-2).contiguous(), scale.flatten(-2).contiguous()


def _dequantise_groups(q, scale, k):
    s = scale.unflatten(-1, (q.shape[-1] // k, -1)).repeat_interleave(GROUP, -1)[..., :k].flatten(-2)
    return q.to(scale.dtype) * s


def _act(x, act):
    if act == "gelu_tanh":
        return 0.5 * x * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (x + 0.044715 * x * x * x)))
    if act == "silu":
        return x / (1.0 + torch.exp(-x))
    gate, up = x.chunk(2, -1)
    return gate / (1.0 + torch.exp(-gate)) * up


def _act_grad(dy, x, act):
    if act == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (x + 0.044715 * x * x * x))
        return dy * (0.5 * (1.0 + t) + 0.5 * x * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * x * x))
    gate, up = (x, None) if act == "silu" else x.chunk(2, -1)
    sig = 1.0 / (1.0 + torch.exp(-gate))
    slope = sig * (1.0 + gate * (1.0 - sig))
    if act == "silu":
        return dy * slope
    return torch.cat([dy * up * slope, dy * gate * sig], -1)


def _plain_act(st):
    case, dy = st["case"], st["dy"]
    if not case["step"]:
        return {"dx": _act_grad(dy.float(), _dequantise_groups(st["q"], st["scale"], case["k"]), case["act"]).to(dy.dtype)}
    x = st["x"].float()
    q, scale = _quantise_groups(x, case["k"])
    return {"y": _act(x, case["act"]).to(dy.dtype),
            "dx": _act_grad(dy.float(), _dequantise_groups(q, scale, case["k"]), case["act"]).to(dy.dtype)}


def _chosen(st):
    """[rows, adapters * rank]: the scaling where the column belongs to the row's adapter, else 0."""
    r = st["a"].shape[1]
    of = torch.arange(st["a"].shape[0], device=st["a"].device)
    return torch.where(st["adapter"].unsqueeze(1) == of, st["scaling"], 0.0).repeat_interleave(r, 1)


def _plain_add(st):
    # the adapters side by side as one matrix, the columns of other rows' adapters taken out
    a = st["a"].float().flatten(0, 1)
    b = st["b"].float().transpose(1, 2).flatten(0, 1)
    delta = ((st["x"].float() @ a.t()) * _chosen(st)) @ b
    return (st["y"].float() + delta).to(st["y"].dtype)


def _plain_grad(st):
    dtype = st["dy"].dtype
    s, r, k = st["a"].shape
    a = st["a"].float().flatten(0, 1)
    b = st["b"].float().transpose(1, 2).flatten(0, 1)
    x, dy = st["x"].float(), st["dy"].float()
    if st["x_scale"] is not None:
        x = x * st["x_scale"]
    chosen = _chosen(st)
    h = (x @ a.t()) * chosen
    g = (dy @ b.t()) * chosen
    da = (g.t() @ x).view(s, r, k)
    db = (dy.t() @ h).view(-1, s, r).transpose(0, 1)
    return {"dx": (g @ a).to(dtype), "da": da.to(dtype), "db": db.to(dtype).contiguous()}


def _plain_dx(st):
    return (st["dy"].float() @ (st["w"].float() * st["ws"].unsqueeze(1))).to(st["dy"].dtype)


# ------------------------------------------------------------------ the framework's calls
def _own(st):
    import imagine_b200 as W

    case = st["case"]
    if case["op"] == "add":
        return W.lora_add(st["y"], st["x"], st["a"], st["b"], st["adapter"], st["scaling"])
    if case["op"] == "grad":
        dx, da, db = W.lora_backward(st["dy"], st["x"], st["a"], st["b"], st["adapter"], st["scaling"], x_scale=st["x_scale"])
        return {"dx": dx, "da": da, "db": db}
    if case["op"] == "dx":
        return W.int8_linear_backward(st["dy"], st["w"], st["ws"])
    if not case["step"]:
        return {"dx": W.act_backward_int8(st["dy"], st["q"], st["scale"], case["act"])}
    y, q, scale = W.act_checkpoint_int8(st["x"], case["act"])
    return {"y": y, "dx": W.act_backward_int8(st["dy"], q, scale, case["act"])}


def run(state):
    if own:
        return _own(state)
    return {"add": _plain_add, "grad": _plain_grad, "act": _plain_act, "dx": _plain_dx}[state["case"]["op"]](state)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    m, k = case["rows"], case["k"]
    if case["op"] == "act":
        width = 2 * k if case["act"] == "swiglu" else k
        groups = width // k * -(-k // GROUP)
        held = m * (width + 4 * groups)  # codes and scales
        back = held + m * (k + width) * size  # dy in, dx out
        if not case["step"]:
            return {"bytes": back, "flops": 20 * m * width}
        return {"bytes": back + held + m * (width + k) * size, "flops": 40 * m * width}
    n = case["n"]
    if case["op"] == "dx":
        return {"bytes": n * k + 4 * n + m * (n + k) * size, "flops": 2 * m * n * k}
    r = case["rank"]
    used = len(set(_adapter_of_request(case)) - {-1})
    weights = used * r * (k + n) * size
    if case["op"] == "add":
        return {"bytes": m * (k + 2 * n) * size + weights + 4 * m, "flops": 2 * m * r * (k + n)}
    x = m * (k + 4) if case["int8"] else m * k * size
    grads = case["adapters"] * r * (k + n) * size
    return {"bytes": x + m * (n + k) * size + weights + grads + 4 * m, "flops": 2 * m * r * (3 * k + 2 * n)}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "act":
        k, act = case["k"], case["act"]
        dy = st["dy"].double()
        x = st["x" if case["step"] else "q"].double()
        codes = torch.empty_like(x)
        group = 0
        for lo in range(0, x.shape[1], k):
            for at in range(lo, lo + k, GROUP):
                end = min(at + GROUP, lo + k)
                if case["step"]:  # the scale is held in 32 bits
                    scale = (x[:, at:end].abs().amax(1, keepdim=True) / 127.0).float().double().clamp_min(1e-30)
                    codes[:, at:end] = torch.round(x[:, at:end] / scale) * scale
                else:
                    codes[:, at:end] = x[:, at:end] * st["scale"][:, group:group + 1].double()
                group += 1
        out = {"y": _exact_act(x, act)} if case["step"] else {}
        codes.requires_grad_(True)
        out["dx"] = torch.autograd.grad(_exact_act(codes, act), codes, dy)[0]
        return out
    if case["op"] == "dx":
        return (st["dy"].double() * st["ws"].double()) @ st["w"].double()
    a, b, adapter, scaling = st["a"].double(), st["b"].double(), st["adapter"].long(), st["scaling"].double()
    x = st["x"].double()
    if case["op"] == "add":
        out = st["y"].double()
        for s in range(case["adapters"]):
            rows = (adapter == s).nonzero().flatten()
            out[rows] += scaling[s] * (x[rows] @ a[s].t() @ b[s].t())
        return out
    if st["x_scale"] is not None:
        x = x * st["x_scale"].double()
    dy = st["dy"].double()
    dx, da, db = torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    for s in range(case["adapters"]):
        rows = (adapter == s).nonzero().flatten()
        g = scaling[s] * (dy[rows] @ b[s])
        dx[rows] = g @ a[s]
        da[s] = g.t() @ x[rows]
        db[s] = scaling[s] * (dy[rows].t() @ (x[rows] @ a[s].t()))
    return {"dx": dx, "da": da, "db": db}


def _exact_act(x, act):
    if act == "gelu_tanh":
        return 0.5 * x * (1.0 + torch.tanh((2.0 / math.pi) ** 0.5 * (x + 0.044715 * x.pow(3))))
    if act == "silu":
        return x * torch.sigmoid(x)
    gate, up = x.chunk(2, -1)
    return gate * torch.sigmoid(gate) * up
