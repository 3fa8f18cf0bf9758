"""The token operators of rt_pose_amd on their own: root-mean-square norm with the residual's addition (values or 8 bits out),
quantising to 8 bits with block scales, the 8-bit matrix product that reads both, and cross attention to an encoder's states.

`run` computes an operator in plain torch operations (32 bits inside, rounded once at the end); with `own = True` it makes the calls
that a user of the framework makes.  `exact` is the same operator from its definition in 64 bits.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
AMAX_FLOOR = 2.0 ** -100
EPS = 1e-6


# --------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # training step's norm over the tokens of a batch of 8 volumes of 4 x 16 x 40, width 1024
        dict(name="norm-train", op="norm", mode="train", rows=20480, h=1024, type="bf16", residual=True),
        # the same where nothing is even: an odd number of tokens of an odd width
        dict(name="norm-train-odd", op="norm", mode="train", rows=1237, h=777, type="fp16", residual=True),
        # serving, one token for each of 8 streams: nothing but latency
        dict(name="norm-fp8-token", op="norm", mode="fp8", rows=8, h=4096, type="bf16", residual=True),
        # serving, a long prompt or a whole volume, written straight in 8 bits for the product behind it
        dict(name="norm-fp8-prompt", op="norm", mode="fp8", rows=16384, h=8192, type="bf16", residual=True),
        # weights laid out once per update: one scale for each 128 x 128 block
        dict(name="quant-weight", op="quant", rows=8192, cols=4096, type="bf16", square=True, turned=False),
        # a gradient's transpose for the weight gradient's product, ragged: blocks of 128 run down the columns of what is in memory
        dict(name="quant-turned", op="quant", rows=1000, cols=20481, type="bf16", square=False, turned=True),
        # serving, a handful of tokens: the weights' bytes are the time
        dict(name="matmul-token", op="matmul", m=4, n=4096, k=4096, square=True, out="bf16"),
        # the 384 -> 256 channel 1x1x1 product of the widest configuration over one full-resolution volume
        dict(name="matmul-voxels", op="matmul", m=163840, n=256, k=384, square=True, out="bf16"),
        # a large layer's product
        dict(name="matmul-large", op="matmul", m=8192, n=8192, k=8192, square=True, out="bf16"),
        # serving: one query token for each of 8 streams against its encoder's states, grouped heads
        dict(name="attn-token", op="attn", mode="infer", b=8, sq=1, sk=2560, hq=32, hkv=8, d=128, type="bf16", lens=True, mask=False),
        # training 15 key-point queries against the tokens of a volume, ragged and masked
        dict(name="attn-joints", op="attn", mode="train", b=8, sq=15, sk=20480, hq=8, hkv=8, d=32, type="bf16", lens=True, mask=True),
        # training one sensor's tokens against another's
        dict(name="attn-train", op="attn", mode="train", b=4, sq=2560, sk=5120, hq=8, hkv=8, d=64, type="bf16", lens=True, mask=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the listed ones' ranges that has no more to read, write and compute than the largest of its operator."""
    cost = lambda c: work(dict(c, mode="train") if c["op"] == "attn" else c)  # noqa: E731
    top = {}
    for c in listed():
        for k, v in cost(c).items():
            top[c["op"], k] = max(v, top.get((c["op"], k), 0.0))
    op = rng.choice(["norm", "norm", "quant", "matmul", "matmul", "attn", "attn", "attn"])
    while True:
        if op == "norm":
            c = dict(op=op, mode=rng.choice(["train", "fp8"]), rows=_log(rng, 1, 20480), h=_log(rng, 32, 8192),
                     type=rng.choice(["bf16", "fp16", "fp32"]), residual=rng.random() < 0.75)
        elif op == "quant":
            c = dict(op=op, rows=_log(rng, 1, 8192), cols=_log(rng, 16, 20481), type=rng.choice(["bf16", "fp16", "fp32"]),
                     square=rng.random() < 0.5, turned=rng.random() < 0.5)
        elif op == "matmul":
            c = dict(op=op, m=_log(rng, 1, 163840), n=_log(rng, 16, 8192), k=_log(rng, 32, 8192), square=rng.random() < 0.7,
                     out=rng.choice(["bf16", "fp16", "fp32"]))
        else:
            hkv = rng.choice([1, 2, 4, 8])
            c = dict(op=op, mode=rng.choice(["train", "infer"]), b=_log(rng, 1, 16), sq=rng.choice([1, _log(rng, 1, 64), _log(rng, 16, 2560)]),
                     sk=_log(rng, 16, 20480), hq=hkv * rng.choice([1, 1, 2, 4]), hkv=hkv, d=rng.choice([32, 40, 64, 96, 128]),
                     type=rng.choice(["bf16", "fp16"]), lens=rng.random() < 0.7, mask=rng.random() < 0.4)
        if all(v <= top[op, k] for k, v in cost(c).items()):
            return c


def work(c):
    """What one pass cannot do without: every input read once, every output written once, and the products' operations."""
    op = c["op"]
    if op == "norm":
        n, s, res = c["rows"] * c["h"], SIZE[c["type"]], int(c["residual"])
        if c["mode"] == "fp8":     # x (, residual) in; q, scales (, stream) out
            return dict(bytes=n * (s * (1 + 2 * res) + 1) + 4 * c["rows"] * -(-c["h"] // 128) + s * c["h"], flops=6.0 * n)
        # x, residual in, y, stream out; y's gradient (, the stream's) and the stream in, the inputs' gradient out; the weight's two
        return dict(bytes=n * s * (2 + 2 * res) + n * s * (3 + res) + 2 * s * c["h"], flops=16.0 * n)
    if op == "quant":
        n = c["rows"] * c["cols"]
        blocks = -(-c["cols"] // 128) * (-(-c["rows"] // 128) if c["square"] else c["rows"])
        return dict(bytes=n * (SIZE[c["type"]] + 1) + 4 * blocks, flops=3.0 * n)
    if op == "matmul":
        m, n, k = c["m"], c["n"], c["k"]
        kb = -(-k // 128)
        return dict(bytes=m * k + n * k + 4 * m * kb + 4 * kb * (-(-n // 128) if c["square"] else n) + m * n * SIZE[c["out"]], flops=2.0 * m * n * k)
    seen = sum(_lens(c)) if c["lens"] else c["b"] * c["sk"]
    q, kv = c["b"] * c["sq"] * c["hq"] * c["d"], seen * c["hkv"] * c["d"]
    pairs = c["sq"] * c["hq"] * seen * (0.75 if c["mask"] else 1.0)
    s = SIZE[c["type"]]
    if c["mode"] == "infer":       # q, k, v in; o out; two products
        return dict(bytes=s * (2 * q + 2 * kv), flops=4.0 * pairs * c["d"])
    # o's gradient in besides, the gradients of q, k and v out (k's and v's whole); six products, the scores' counted once
    return dict(bytes=s * (4 * q + 2 * kv + 2 * c["b"] * c["sk"] * c["hkv"] * c["d"]), flops=12.0 * pairs * c["d"])


def _lens(c):
    """Keys of each batch entry: from none to all, in steps; the last has all."""
    b, sk = c["b"], c["sk"]
    return [sk if i == b - 1 else (sk * (2 * i + 1) // (2 * b) if i else (0 if b > 3 else (sk + 1) // 2)) for i in range(b)]


# -------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, *shape, type="fp32", scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(TYPES[type])


def _tokens(g, rows, cols, type):
    """Activations: rows of different size, some channels ten times the others."""
    x = torch.randn(rows, cols, generator=g, device=DEV)
    x *= torch.exp(0.5 * torch.randn(rows, 1, generator=g, device=DEV))
    x *= torch.where(torch.rand(1, cols, generator=g, device=DEV) < 0.01, 10.0, 1.0)
    return x.to(TYPES[type])


def _eight_bits(g, rows, cols, blocks_rows):
    """An operand in 8 bits as quantising leaves it: values over the whole range, a scale for each block."""
    q = torch.randn(rows, cols, generator=g, device=DEV).mul_(120.0).clamp_(-FP8_MAX, FP8_MAX).to(FP8)
    scale = torch.exp(0.3 * torch.randn(blocks_rows, -(-cols // 128), generator=g, device=DEV)) * (0.02 / 120.0)
    return q, scale


def _padded(q):
    """The 8-bit operand in rows of a multiple of 16 bytes, as the framework's own quantising operators write it."""
    rows, cols = q.shape
    wide = torch.zeros(rows, -(-cols // 16) * 16, dtype=torch.uint8, device=q.device)
    wide[:, :cols] = q.view(torch.uint8)
    return wide.view(FP8)[:, :cols]


def prepare(c, seed):
    g = _gen(seed)
    s = {"case": c}
    if c["op"] == "norm":
        s["x"] = _tokens(g, c["rows"], c["h"], c["type"])
        s["r"] = _tokens(g, c["rows"], c["h"], c["type"]) if c["residual"] else None
        s["w"] = (1.0 + 0.2 * torch.randn(c["h"], generator=g, device=DEV)).to(TYPES[c["type"]])
        if c["mode"] == "train":
            s["dy"] = _normal(g, c["rows"], c["h"], type=c["type"], scale=0.1)
            s["dh"] = _normal(g, c["rows"], c["h"], type=c["type"], scale=0.1) if c["residual"] else None
            for n in ("x", "r", "w"):
                if s[n] is not None:
                    s[n].requires_grad_(True)
    elif c["op"] == "quant":
        x = _tokens(g, c["cols"], c["rows"], c["type"]).t() if c["turned"] else _tokens(g, c["rows"], c["cols"], c["type"])
        s["x"] = x
    elif c["op"] == "matmul":
        a, sa = _eight_bits(g, c["m"], c["k"], c["m"])
        b, sb = _eight_bits(g, c["n"], c["k"], -(-c["n"] // 128) if c["square"] else c["n"])
        s.update(a=_padded(a), sa=sa, b=_padded(b), sb=sb)
    else:
        t = c["type"]
        s["q"] = _normal(g, c["b"], c["sq"], c["hq"], c["d"], type=t, scale=1.5)
        s["k"] = _normal(g, c["b"], c["sk"], c["hkv"], c["d"], type=t)
        s["v"] = _normal(g, c["b"], c["sk"], c["hkv"], c["d"], type=t)
        s["lens"] = torch.tensor(_lens(c), dtype=torch.int32, device=DEV) if c["lens"] else None
        s["mask"] = torch.rand(c["b"], c["sk"], generator=g, device=DEV) < 0.75 if c["mask"] else None
        if c["mode"] == "train":
            s["do"] = _normal(g, c["b"], c["sq"], c["hq"], c["d"], type=t, scale=0.1)
            for n in ("q", "k", "v"):
                s[n].requires_grad_(True)
    return s


# ----------------------------------------------------------------------------------------------------------- plain form
def _plain_norm(s):
    c, t = s["case"], TYPES[s["case"]["type"]]
    x, w = s["x"].detach().float(), s["w"].detach().float()
    stream = x
    out = {}
    if s["r"] is not None:
        out["stream"] = (x + s["r"].detach().float()).to(t)    # the stream as it is written is what is normed
        stream = out["stream"].float()
    rstd = (stream.square().mean(1, keepdim=True) + EPS).rsqrt()
    xhat = stream * rstd
    y = xhat * w
    if c["mode"] == "fp8":
        out["q"], out["scale"] = _plain_quant(y, False)
        return out
    out["y"] = y.to(t)
    dy = s["dy"].float()
    gy = dy * w
    dx = rstd * (gy - xhat * (gy * xhat).mean(1, keepdim=True))
    if s["r"] is not None:
        dx = dx + s["dh"].float()
    out["dx"] = dx.to(t)
    if s["r"] is not None:
        out["dr"] = out["dx"].clone()
    out["dw"] = (dy * xhat).sum(0).to(t)
    return out


def _plain_quant(x, square):
    rows, cols = x.shape
    kb = -(-cols // 128)
    x = x.float()
    whole = torch.nn.functional.pad(x, (0, kb * 128 - cols))
    if square:
        rb = -(-rows // 128)
        whole = torch.nn.functional.pad(whole, (0, 0, 0, rb * 128 - rows))
        amax = whole.abs().reshape(rb, 128, kb, 128).amax((1, 3)).clamp_min(AMAX_FLOOR)
        up = (FP8_MAX / amax).repeat_interleave(128, 0)[:rows]
    else:
        amax = whole.abs().reshape(rows, kb, 128).amax(2).clamp_min(AMAX_FLOOR)
        up = FP8_MAX / amax
    return (x * up.repeat_interleave(128, 1)[:, :cols]).to(FP8), amax / FP8_MAX


def _plain_matmul(s):
    c = s["case"]
    sa = s["sa"].repeat_interleave(128, 1)[:, :c["k"]]
    sb = s["sb"].repeat_interleave(128, 1)[:, :c["k"]]
    if c["square"]:
        sb = sb.repeat_interleave(128, 0)[:c["n"]]
    return ((s["a"].float() * sa) @ (s["b"].float() * sb).t()).to(TYPES[c["out"]])


def _seen(s):
    """[B, Sk] truth values: the keys that count."""
    c = s["case"]
    seen = torch.ones(c["b"], c["sk"], dtype=torch.bool, device=DEV)
    if s["lens"] is not None:
        seen &= torch.arange(c["sk"], device=DEV) < s["lens"][:, None]
    if s["mask"] is not None:
        seen &= s["mask"]
    return seen


def _plain_attn(s):
    c, t = s["case"], TYPES[s["case"]["type"]]
    b, sq, sk, hq, hkv, d = (c[n] for n in ("b", "sq", "sk", "hq", "hkv", "d"))
    grp = hq // hkv
    scale = d ** -0.5
    seen = _seen(s)
    # [B, Hkv, group * Sq, D] and [B, Hkv, Sk, D]; keys that do not count are zeros
    rows = lambda x: x.detach().float().reshape(b, sq, hkv, grp, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, grp * sq, d)  # noqa: E731
    back = lambda x: x.reshape(b, hkv, grp, sq, d).permute(0, 3, 1, 2, 4).reshape(b, sq, hq, d).to(t)                    # noqa: E731
    keys = lambda x: torch.where(seen[:, :, None, None], x.detach().float(), 0.0).transpose(1, 2).contiguous()           # noqa: E731
    q, k, v = rows(s["q"]), keys(s["k"]), keys(s["v"])
    p = (q @ k.transpose(2, 3)).mul_(scale)
    p.masked_fill_(~seen[:, None, None, :], -math.inf)
    p.sub_(p.amax(3, keepdim=True).clamp_min(-1e30)).exp_()
    p.div_(p.sum(3, keepdim=True).clamp_min(1e-30))
    o = p @ v
    if c["mode"] == "infer":
        return back(o)
    do = rows(s["do"])
    dv = p.transpose(2, 3) @ do
    ds = do @ v.transpose(2, 3)
    ds.sub_((o * do).sum(3, keepdim=True)).mul_(p).mul_(scale)
    return {"o": back(o), "dq": back(ds @ k), "dk": (ds.transpose(2, 3) @ q).transpose(1, 2).to(t).contiguous(), "dv": dv.transpose(1, 2).to(t).contiguous()}


# ---------------------------------------------------------------------------------------------------------------- runs
def _own(s):
    c = s["case"]
    if c["op"] == "norm":
        from rt_pose_amd import rmsnorm
        if c["mode"] == "fp8":
            q, scale, stream = rmsnorm.add_rms_norm_fp8(s["x"], s["r"], s["w"], EPS)
            return {"q": q, "scale": scale, "stream": stream} if c["residual"] else {"q": q, "scale": scale}
        if c["residual"]:
            y, stream = rmsnorm.add_rms_norm(s["x"], s["r"], s["w"], EPS)
            dx, dr, dw = torch.autograd.grad((y, stream), (s["x"], s["r"], s["w"]), (s["dy"], s["dh"]))
            return {"y": y, "stream": stream, "dx": dx, "dr": dr, "dw": dw}
        y = rmsnorm.rms_norm(s["x"], s["w"], EPS)
        dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
        return {"y": y, "dx": dx, "dw": dw}
    if c["op"] == "attn":
        from rt_pose_amd import attention
        o = attention.cross_attention(s["q"], s["k"], s["v"], key_lens=s["lens"], key_mask=s["mask"])
        if c["mode"] == "infer":
            return o
        dq, dk, dv = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])
        return {"o": o, "dq": dq, "dk": dk, "dv": dv}
    from rt_pose_amd import fp8
    if c["op"] == "quant":
        q, scale = fp8.quantize_fp8(s["x"], (128, 128) if c["square"] else (1, 128))
        return {"q": q, "scale": scale}
    return fp8.matmul_fp8(s["a"], s["sa"], s["b"], s["sb"], out_dtype=TYPES[c["out"]])


def run(s):
    if own:
        return _own(s)
    op = s["case"]["op"]
    if op == "norm":
        return _plain_norm(s)
    if op == "quant":
        q, scale = _plain_quant(s["x"], s["case"]["square"])
        return {"q": q, "scale": scale}
    return _plain_matmul(s) if op == "matmul" else _plain_attn(s)


# --------------------------------------------------------------------------------------------------------------- exact
def _exact_scale(y, square):
    """Largest magnitude of each block over 448, block by block along the columns."""
    rows, cols = y.shape
    tall = 128 if square else 1
    got = torch.empty(-(-rows // tall), -(-cols // 128), dtype=torch.float64, device=y.device)
    for j in range(got.shape[1]):
        top = y[:, j * 128:(j + 1) * 128].abs().max(1).values
        if square:
            top = torch.stack([part.max() for part in top.split(128)])
        got[:, j] = torch.maximum(top, torch.tensor(AMAX_FLOOR, dtype=torch.float64, device=y.device)) / FP8_MAX
    return got


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "quant":
        return {"q": None, "scale": _exact_scale(s["x"].double(), c["square"])}
    if c["op"] == "matmul":
        a, b = s["a"].double(), s["b"].double()
        out = torch.zeros(c["m"], c["n"], dtype=torch.float64, device=DEV)
        for j in range(-(-c["k"] // 128)):
            part = a[:, j * 128:(j + 1) * 128] @ b[:, j * 128:(j + 1) * 128].t()
            part *= s["sa"][:, j:j + 1].double()
            sb = s["sb"][:, j].double()
            part *= (sb.repeat_interleave(128)[:c["n"]] if c["square"] else sb)[None]
            out += part
        return out
    if c["op"] == "norm":
        x, w = s["x"].detach().double(), s["w"].detach().double()
        out = {}
        if c["residual"]:
            written = (x + s["r"].detach().double()).to(s["x"].dtype)
            x = written.double()
            out["stream"] = x
        root = torch.sqrt((x * x).sum(1) / c["h"] + EPS)[:, None]
        if c["mode"] == "fp8":
            out.update(q=None, scale=_exact_scale(x / root * w, False))
            return out
        dy = s["dy"].double()
        out["y"] = x / root * w
        # y_i = w_i x_i / root with root^2 = mean(x^2) + eps: dx_j = w_j dy_j / root - x_j sum_i(w_i dy_i x_i) / (h root^3)
        dx = w * dy / root - x * ((w * dy * x).sum(1, keepdim=True) / (c["h"] * root ** 3))
        if c["residual"]:
            dx = dx + s["dh"].double()
            out["dr"] = dx
        out["dx"] = dx
        out["dw"] = (dy * x / root).sum(0)
        return out
    b, sq, sk, hq, hkv, d = (c[n] for n in ("b", "sq", "sk", "hq", "hkv", "d"))
    if work(c)["flops"] > 6e11:
        return None
    train = c["mode"] == "train"
    o = torch.zeros(b, sq, hq, d, dtype=torch.float64, device=DEV)
    dq, dk, dv = torch.zeros_like(o), *(torch.zeros(b, sk, hkv, d, dtype=torch.float64, device=DEV) for _ in range(2))
    for i in range(b):
        at = torch.arange(sk, device=DEV)
        if s["mask"] is not None:
            at = at[s["mask"][i]]
        if s["lens"] is not None:
            at = at[at < s["lens"][i]]
        if at.numel() == 0:
            continue
        for h in range(hq):
            j = h * hkv // hq
            q, k, v = s["q"][i, :, h].detach().double(), s["k"][i, at, j].detach().double(), s["v"][i, at, j].detach().double()
            p = torch.softmax(q @ k.t() / math.sqrt(d), 1)
            o[i, :, h] = p @ v
            if train:
                do = s["do"][i, :, h].double()
                dp = do @ v.t()
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) / math.sqrt(d)
                dq[i, :, h] = ds @ k
                dk[i, at, j] += ds.t() @ q
                dv[i, at, j] += p.t() @ do
    return {"o": o, "dq": dq, "dk": dk, "dv": dv} if train else o
