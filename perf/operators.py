"""Cases of the transformer-block operators around the attention: layer norm and its
backward pass, the linear layer with bias, activation and residual in its epilogue
and its backward pass, and activation checkpoints in 8 bits.

``run`` computes each in plain torch operations in 32 bits; with ``own`` set it calls
the package's kernels. ``exact`` states the definitions once more in 64 bits.

An 8-bit checkpoint holds each row in blocks of 32 values: one power-of-two scale
2^e (a byte, e + 127) and 32 signed codes. With amax = f 2^q (1/2 <= f < 1) the
largest magnitude of the block, e = max(q - 7, -126) and code = round(x / 2^e), ties
to even, limited to [-127, 127]. The value it stands for is code 2^e.
"""
import math

import torch

own = False

BLOCK = 32
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # one 8x8-patch window's tokens through a norm: the smallest call, latency counts
        dict(name="norm_window", op="norm", rows=64, width=1280, dtype="bf16", params="bf16", strided=False),
        # all 9216 tokens of a 1344x1344 image, norm weights kept in 32 bits as in training
        dict(name="norm_image", op="norm", rows=9216, width=1280, dtype="bf16", params="f32", strided=False),
        # the same image's norm in the backward pass
        dict(name="norm_bwd_image", op="norm_bwd", rows=9216, width=1280, dtype="bf16", params="bf16", packed=False),
        # a norm over the MLP width, a ragged number of rows, its input kept as an 8-bit checkpoint
        dict(name="norm_bwd_packed_ragged", op="norm_bwd", rows=4097, width=3420, dtype="f16", params="f32",
             packed=True),
        # a single token through the first MLP matrix: reading the weight is all there is
        dict(name="linear_token", op="linear", rows=1, k=1280, n=3424, dtype="bf16", act="silu", bias=True,
             residual=False, save="none", strided=False),
        # a small ragged batch of tokens, output rows that are not 16-byte multiples, training forward
        dict(name="linear_ragged_train", op="linear", rows=333, k=1280, n=3420, dtype="f16", act="gelu", bias=True,
             residual=False, save="full", strided=True),
        # the first MLP matrix of a 1344x1344 image, pre-activation kept in 8 bits for the backward pass
        dict(name="linear_image_gelu_packed", op="linear", rows=9216, k=1280, n=3424, dtype="bf16", act="gelu",
             bias=True, residual=False, save="packed", strided=False),
        # the second MLP matrix with the residual stream added in the epilogue
        dict(name="linear_image_residual", op="linear", rows=9216, k=3424, n=1280, dtype="bf16", act="none",
             bias=True, residual=True, save="none", strided=False),
        # its backward pass for the first MLP matrix: the largest case
        dict(name="linear_bwd_image", op="linear_bwd", rows=9216, k=1280, n=3424, dtype="bf16", act="gelu_tanh",
             packed=False),
        # an 896x896 image, the MLP's own odd width, input and pre-activation from 8-bit checkpoints
        dict(name="linear_bwd_packed", op="linear_bwd", rows=4096, k=1280, n=3420, dtype="bf16", act="silu",
             packed=True),
        # hidden activations of an image written to 8 bits and read back
        dict(name="checkpoint_image", op="checkpoint", rows=9216, width=3424, dtype="bf16"),
        # a few rows of an odd width
        dict(name="checkpoint_ragged", op="checkpoint", rows=1000, width=1281, dtype="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size over [lo, hi] by its logarithm: mostly multiples of 16, the others as they fall."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.35 else max(lo, n // 16 * 16)


def draw(rng):
    op = rng.choice(["norm", "norm_bwd", "linear", "linear", "linear_bwd", "linear_bwd", "checkpoint"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op in ("norm", "norm_bwd", "checkpoint"):
        width = _size(rng, 64, 8192)
        rows = min(_log(rng, 1, 32768), 9216 * 3424 // width)
        if op == "norm":
            return dict(op=op, rows=rows, width=width, dtype=rng.choice([dtype, "f32"]),
                        params=rng.choice(["same", "f32"]), strided=rng.random() < 0.3)
        if op == "norm_bwd":
            return dict(op=op, rows=rows, width=width, dtype=dtype, params=rng.choice(["same", "f32"]),
                        packed=rng.random() < 0.4)
        return dict(op=op, rows=rows, width=width, dtype=dtype)
    k, n = _size(rng, 64, 5120), _size(rng, 64, 5120)
    rows = min(_log(rng, 1, 16384), 9216 * 1280 * 3424 // (k * n))
    act = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
    if op == "linear":
        return dict(op=op, rows=rows, k=k, n=n, dtype=dtype, act=act, bias=rng.random() < 0.8,
                    residual=rng.random() < 0.4, save=rng.choice(["none", "full", "packed"]),
                    strided=rng.random() < 0.3)
    return dict(op=op, rows=rows, k=k, n=n, dtype=dtype, act=act, packed=rng.random() < 0.4)


def _params(case):
    return DTYPES[case["dtype"] if case["params"] == "same" else case["params"]]


def work(case):
    e = DTYPES[case["dtype"]].itemsize
    r = case["rows"]
    if case["op"] in ("norm", "norm_bwd", "checkpoint"):
        c = case["width"]
        q = 1 + 1 / BLOCK
        if case["op"] == "norm":
            return {"bytes": 2 * r * c * e + 2 * c * _params(case).itemsize + 8 * r, "flops": 8 * r * c}
        if case["op"] == "norm_bwd":
            x = q if case["packed"] else e
            return {"bytes": r * c * (2 * e + x) + 3 * c * _params(case).itemsize + 8 * r, "flops": 14 * r * c}
        return {"bytes": r * c * (2 * e + 2 * q), "flops": 4 * r * c}
    k, n = case["k"], case["n"]
    q = 1 + 1 / BLOCK
    if case["op"] == "linear":
        z = {"none": 0, "full": e, "packed": q}[case["save"]]
        extra = (e if case["residual"] else 0) + z
        return {"bytes": r * k * e + n * k * e + (n * e if case["bias"] else 0) + r * n * (e + extra),
                "flops": 2 * r * n * k}
    x = q if case["packed"] else e
    z = 0 if case["act"] == "none" else x
    return {"bytes": r * n * (e + z) + r * k * (x + e) + 2 * n * k * e + n * e, "flops": 4 * r * n * k}


# --------------------------------------------------------------------------- inputs
def _inputs(case, seed):
    """The inputs of a case on the GPU, from the seed alone."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    r = case["rows"]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    def stream(rows, width):
        """Rows of a residual stream: channels of different spread and offset, a few large ones."""
        spread = torch.exp(0.5 * randn(width))
        spread[torch.rand(width, generator=g, device=dev) < 0.01] *= 8
        return randn(rows, width) * spread + 0.2 * randn(width)

    def rows_of(t, strided):
        """t in the case's type; strided: as the rows of a wider buffer."""
        t = t.to(dt)
        if not strided:
            return t
        wide = torch.zeros(t.shape[0], t.shape[1] + 16 + (-t.shape[1]) % 8, dtype=t.dtype, device=dev)
        wide[:, :t.shape[1]] = t
        return wide[:, :t.shape[1]]

    if case["op"] in ("norm", "norm_bwd"):
        c, pt = case["width"], _params(case)
        s = {"x": rows_of(stream(r, c), case.get("strided", False)), "weight": (1 + 0.2 * randn(c)).to(pt),
             "bias": (0.1 * randn(c)).to(pt), "eps": 1e-6}
        if case["op"] == "norm_bwd":
            xf = s["x"].float()
            s["mean"] = xf.mean(1)
            s["rstd"] = torch.rsqrt((xf - s["mean"][:, None]).square().mean(1) + s["eps"])
            s["dout"] = (0.1 * randn(r, c)).to(dt)
            if case["packed"]:
                s["codes"], s["scales"] = _pack(s.pop("x"))
        return s
    if case["op"] == "checkpoint":
        return {"x": stream(r, case["width"]).to(dt)}
    k, n = case["k"], case["n"]
    s = {"x": rows_of(randn(r, k), case.get("strided", False)), "weight": (randn(n, k) / math.sqrt(k)).to(dt)}
    if case["op"] == "linear":
        s["bias"] = (0.2 * randn(n)).to(dt) if case["bias"] else None
        s["residual"] = stream(r, n).to(dt) if case["residual"] else None
        return s
    s["dout"] = (0.1 * randn(r, n)).to(dt)
    s["preact"] = (1.2 * randn(r, n)).to(dt) if case["act"] != "none" else None
    if case["packed"]:
        s["x_codes"], s["x_scales"] = _pack(s.pop("x"))
        if s["preact"] is not None:
            s["z_codes"], s["z_scales"] = _pack(s.pop("preact"))
    return s


def prepare(case, seed):
    return dict(_inputs(case, seed), case=dict(case))


# --------------------------------------------------------------------------- plain forms (32 bits)
def _pow2(e):
    """2^e in 32 bits for integer e in [-126, 127]."""
    return ((e + 127) << 23).view(torch.float32)


def _pack(x):
    """Codes [rows, blocks * 32] int8 and scale bytes [rows, blocks] uint8 of a checkpoint of x."""
    r, c = x.shape
    nb = -(-c // BLOCK)
    xf = torch.zeros(r, nb * BLOCK, dtype=torch.float32, device=x.device)
    xf[:, :c] = x
    xf = xf.view(r, nb, BLOCK)
    _, q = torch.frexp(xf.abs().amax(-1))
    e = (q.to(torch.int32) - 7).clamp_min(-126)
    codes = torch.round(xf * _pow2(-e)[..., None]).clamp(-127, 127).to(torch.int8)
    return codes.view(r, nb * BLOCK), (e + 127).to(torch.uint8)


def _unpack(codes, scales, width):
    """The values of a checkpoint in 32 bits."""
    r, nb = scales.shape
    v = codes.view(r, nb, BLOCK).float() * _pow2(scales.to(torch.int32) - 127)[..., None]
    return v.view(r, nb * BLOCK)[:, :width]


def _act(z, act):
    if act == "none":
        return z
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z / (1 + torch.exp(-z))


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def _run_plain(s):
    case = s["case"]
    dt = DTYPES[case["dtype"]]
    if case["op"] == "norm":
        x = s["x"].float()
        mean = x.mean(1)
        d = x - mean[:, None]
        rstd = torch.rsqrt((d * d).mean(1) + s["eps"])
        return (d * rstd[:, None] * s["weight"].float() + s["bias"].float()).to(dt), mean, rstd
    if case["op"] == "norm_bwd":
        x = _unpack(s["codes"], s["scales"], case["width"]) if case["packed"] else s["x"].float()
        dy = s["dout"].float()
        xh = (x - s["mean"][:, None]) * s["rstd"][:, None]
        gy = dy * s["weight"].float()
        dx = s["rstd"][:, None] * (gy - gy.mean(1, keepdim=True) - xh * (gy * xh).mean(1, keepdim=True))
        pt = s["weight"].dtype
        return dx.to(dt), (dy * xh).sum(0).to(pt), dy.sum(0).to(pt)
    if case["op"] == "checkpoint":
        return _unpack(*_pack(s["x"]), case["width"]).to(dt)
    if case["op"] == "linear":
        z = s["x"].float() @ s["weight"].float().t()
        if s["bias"] is not None:
            z = z + s["bias"].float()
        y = _act(z, case["act"])
        if s["residual"] is not None:
            y = y + s["residual"].float()
        if case["save"] == "full":
            return y.to(dt), z.to(dt)
        if case["save"] == "packed":
            return y.to(dt), _unpack(*_pack(z), case["n"]).to(dt)
        return y.to(dt)
    dz = s["dout"].float()
    if case["packed"]:
        x = _unpack(s["x_codes"], s["x_scales"], case["k"])
        z = _unpack(s["z_codes"], s["z_scales"], case["n"]) if case["act"] != "none" else None
    else:
        x, z = s["x"].float(), s["preact"].float() if s["preact"] is not None else None
    if case["act"] != "none":
        dz = dz * _act_grad(z, case["act"])
    return (dz @ s["weight"].float()).to(dt), (dz.t() @ x).to(dt), dz.sum(0).to(dt)


# --------------------------------------------------------------------------- the package's operators
def _run_own(s):
    import fused_rope_attn_b200 as fr

    case = s["case"]
    dt = DTYPES[case["dtype"]]
    if case["op"] == "norm":
        return fr.layer_norm(s["x"], s["weight"], s["bias"], eps=s["eps"], return_stats=True)
    if case["op"] == "norm_bwd":
        x = fr.PackedActivation(s["codes"], s["scales"], case["width"], dt) if case["packed"] else s["x"]
        return fr.layer_norm_backward(s["dout"], x, s["weight"], s["mean"], s["rstd"])
    if case["op"] == "checkpoint":
        return fr.unpack_activation(fr.pack_activation(s["x"]))
    if case["op"] == "linear":
        if case["save"] == "none":
            return fr.linear_act(s["x"], s["weight"], s["bias"], activation=case["act"], residual=s["residual"])
        y, z = fr.linear_act(s["x"], s["weight"], s["bias"], activation=case["act"], residual=s["residual"],
                             save_preact=case["save"])
        return y, fr.unpack_activation(z) if case["save"] == "packed" else z
    if case["packed"]:
        x = fr.PackedActivation(s["x_codes"], s["x_scales"], case["k"], dt)
        z = fr.PackedActivation(s["z_codes"], s["z_scales"], case["n"], dt) if case["act"] != "none" else None
    else:
        x, z = s["x"], s["preact"]
    return fr.linear_act_backward(s["dout"], x, s["weight"], z, activation=case["act"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# --------------------------------------------------------------------------- definitions in 64 bits
def _pack64(x):
    """The values of a checkpoint of x (64 bits), from the definition."""
    r, c = x.shape
    pad = torch.nn.functional.pad(x, (0, (-c) % BLOCK)).reshape(r, -1, BLOCK)
    _, q = torch.frexp(pad.abs().max(dim=2).values)
    step = torch.ldexp(torch.ones_like(pad[..., :1]), (q - 7).clamp(min=-126).unsqueeze(2))
    return (torch.round(pad / step).clamp(-127, 127) * step).reshape(r, -1)[:, :c]


def _values64(codes, scales, width):
    e = scales.double() - 127
    return (codes.double().reshape(scales.shape[0], -1, BLOCK) * torch.exp2(e).unsqueeze(2)).flatten(1)[:, :width]


def exact(case, seed):
    s = _inputs(case, seed)
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    op, act = case["op"], case.get("act")
    if op == "norm":
        mean = d["x"].sum(1) / case["width"]
        var = ((d["x"] - mean.unsqueeze(1)) ** 2).sum(1) / case["width"]
        rstd = 1 / torch.sqrt(var + s["eps"])
        return ((d["x"] - mean.unsqueeze(1)) * rstd.unsqueeze(1)) * d["weight"] + d["bias"], mean, rstd
    if op == "norm_bwd":
        x = _values64(s["codes"], s["scales"], case["width"]) if case["packed"] else d["x"]
        r = d["rstd"].unsqueeze(1)
        h = (x - d["mean"].unsqueeze(1)) * r
        u = d["dout"] * d["weight"]
        n = case["width"]
        dx = r * (u - u.sum(1, keepdim=True) / n - h * ((u * h).sum(1, keepdim=True) / n))
        return dx, (d["dout"] * h).sum(0), d["dout"].sum(0)
    if op == "checkpoint":
        return _pack64(d["x"])
    if op == "linear":
        z = torch.einsum("mk,nk->mn", d["x"], d["weight"]) + (d["bias"] if s["bias"] is not None else 0)
    else:
        z = d.get("preact")
        if case["packed"] and act != "none":
            z = _values64(s["z_codes"], s["z_scales"], case["n"])
        if z is not None:
            z = z.clone().requires_grad_(True)
    if act == "relu":
        y = z.clamp(min=0)
    elif act == "gelu":
        y = z * torch.special.erfc(-z / math.sqrt(2)) / 2
    elif act == "gelu_tanh":
        y = z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    elif act == "silu":
        y = z * torch.sigmoid(z)
    else:
        y = z
    if op == "linear":
        out = y + d["residual"] if s["residual"] is not None else y
        if case["save"] == "full":
            return out, z
        # The packed pre-activation is a step function of a sum: one that lies within its own
        # rounding of a step's edge moves by a whole step, so no value here is the right one.
        return (out, None) if case["save"] == "packed" else out
    dz = d["dout"] if act == "none" else torch.autograd.grad(y, z, d["dout"])[0]
    x = _values64(s["x_codes"], s["x_scales"], case["k"]) if case["packed"] else d["x"]
    return torch.einsum("mn,nk->mk", dz, d["weight"]), torch.einsum("mn,mk->nk", dz, x), dz.sum(0)
