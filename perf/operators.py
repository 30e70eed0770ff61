"""Cases of the dense operators around the expert block: ``block_norm`` (the norms before and after a block with its
gate and residual scale), ``int8_linear`` and ``int8_gated`` (W8A8 products, plain and gated).

``run`` computes a case in plain torch operations, or, where ``own`` is set, through the package's entry points.
"""
import torch

own = False

TINY = 2.0 ** -120          # a row whose largest magnitude is below this counts as a row of zeros
EPS = 1e-5
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one decoded token between two blocks: bf16 residual stream, post-norm, per-channel gate, next norm
        dict(name="norm-1x4096", op="norm", T=1, H=4096, res="bf16", blk="bf16", post=True, gate="channel", out="bf16"),
        # a decode batch over an f32 residual stream, a sigmoid gate per token, rows leave as int8 for the next product
        dict(name="norm-32x7168-int8", op="norm", T=32, H=7168, res="f32", blk="bf16", post=True, gate="token", out="int8"),
        # a long prompt: everything bf16, a gate value per element
        dict(name="norm-4096x5120", op="norm", T=4096, H=5120, res="bf16", blk="bf16", post=True, gate="element", out="bf16"),
        # odd width, the block's f32 partial sums straight from the expert-parallel sum, no post-norm
        dict(name="norm-509x2879", op="norm", T=509, H=2879, res="f32", blk="f32", post=False, gate="none", out="f32"),
        # one decoded token through a square projection
        dict(name="linear-1x4096x4096", op="linear", T=1, K=4096, N=4096, x="bf16", bias=False, out="bf16"),
        # a decode batch into a wide model
        dict(name="linear-32x4096x7168", op="linear", T=32, K=4096, N=7168, x="bf16", bias=False, out="bf16"),
        # ragged prompt chunk, odd widths, bias, f32 activations and f32 result (a head that feeds a sampler)
        dict(name="linear-333x1000x1537", op="linear", T=333, K=1000, N=1537, x="f32", bias=True, out="f32"),
        # a long prompt through a square projection of a wide model
        dict(name="linear-4096x7168x7168", op="linear", T=4096, K=7168, N=7168, x="bf16", bias=False, out="bf16"),
        # one decoded token through the gated projections of a shared expert's width
        dict(name="gated-1x7168x2048", op="gated", T=1, K=7168, I=2048, x="bf16", out="bf16"),
        # an odd small block with f32 result
        dict(name="gated-77x1000x523", op="gated", T=77, K=1000, I=523, x="f32", out="f32"),
        # the batch of the expert-parallel layer
        dict(name="gated-128x7168x2048", op="gated", T=128, K=7168, I=2048, x="bf16", out="bf16"),
        # a long prompt through the dense feed-forward
        dict(name="gated-4096x5120x2048", op="gated", T=4096, K=5120, I=2048, x="bf16", out="bf16"),
    ]


def _spread(rng, lo, hi):
    """A size between lo and hi, even over the logarithm; half of them whole multiples of 64 where that is possible."""
    n = int(round(lo * (hi / lo) ** rng.random()))
    if n >= 128 and rng.random() < 0.5:
        n = n // 64 * 64
    return max(lo, min(hi, n))


def draw(rng):
    op = rng.choice(["norm", "linear", "gated"])
    T = _spread(rng, 1, 4096)
    if op == "norm":
        return dict(op=op, T=T, H=_spread(rng, 64, 8192), res=rng.choice(["bf16", "f32"]), blk=rng.choice(["bf16", "f32"]),
                    post=rng.random() < 0.7, gate=rng.choice(["none", "channel", "token", "element"]),
                    out=rng.choice(["bf16", "f32", "int8"]))
    K = _spread(rng, 64, 7168)
    x, out = rng.choice(["bf16", "f32"]), rng.choice(["bf16", "bf16", "f32"])
    if op == "linear":
        return dict(op=op, T=T, K=K, N=_spread(rng, 64, 7168), x=x, bias=rng.random() < 0.4, out=out)
    return dict(op=op, T=T, K=K, I=_spread(rng, 32, 3584), x=x, out=out)


def _rows(shape, kind, g):
    """Activations: N(0, 1) with every hundredth channel or so 20 times as wide, as hidden states are."""
    x = torch.randn(shape, generator=g, device="cuda")
    wide = torch.rand(shape[-1], generator=g, device="cuda") < 0.01
    return (x * torch.where(wide, 20.0, 1.0)).to(TYPES[kind])


def _weight(rows, cols, g):
    """int8 rows with a scale each, rows 16-byte aligned: a weight of N(0, 0.02) quantised once at load time."""
    q = torch.zeros((rows, (cols + 15) // 16 * 16), dtype=torch.int8, device="cuda")
    w = torch.randn((rows, cols), generator=g, device="cuda") * 0.02
    scale = w.abs().amax(dim=1) / 127
    q[:, :cols] = torch.round(w / scale[:, None]).clamp(-127, 127).to(torch.int8)
    return q[:, :cols], scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case)
    if case["op"] == "norm":
        T, H = case["T"], case["H"]
        s["residual"] = _rows((T, H), case["res"], g)
        s["block"] = _rows((T, H), case["blk"], g)
        s["post_gain"] = 1 + 0.1 * torch.randn(H, generator=g, device="cuda") if case["post"] else None
        s["pre_gain"] = 1 + 0.1 * torch.randn(H, generator=g, device="cuda")
        shape = {"none": None, "channel": (H,), "token": (T, 1), "element": (T, H)}[case["gate"]]
        s["gate_value"] = None if shape is None else torch.randn(shape, generator=g, device="cuda").to(
            torch.float32 if case["gate"] == "channel" else torch.bfloat16)
        return s
    rows = case["N"] if case["op"] == "linear" else 2 * case["I"]
    s["tokens"] = _rows((case["T"], case["K"]), case["x"], g)
    s["weight"] = _weight(rows, case["K"], g)
    s["bias_value"] = torch.randn(rows, generator=g, device="cuda") if case.get("bias") else None
    return s


RES_SCALE, BLK_SCALE = 0.9, 1.25      # residual and block scale of the norm cases


def _quantise(x):
    """f32 rows -> integer rows (as f32) and the scale of each row."""
    a = x.abs().amax(dim=1, keepdim=True)
    fine = a >= TINY
    steps = torch.full_like(a, 127)        # a tensor: torch multiplies by a reciprocal where one side is a number
    q = torch.where(fine & torch.isfinite(a), torch.round(x * (steps / a)), 0.0)
    scale = torch.where(fine, a / steps, 0.0)
    return q, torch.where(torch.isfinite(a), scale, float("nan"))


def _plain_norm(s):
    r, y = s["residual"].float(), s["block"].float()
    if s["post_gain"] is not None:
        y = y * torch.rsqrt((y * y).mean(dim=1, keepdim=True) + EPS) * s["post_gain"]
    if s["gate_value"] is not None:
        gate = s["gate_value"].float()
        y = y * (1 / (1 + torch.exp(-gate)) if s["gate"] == "token" else gate)
    r = RES_SCALE * r + BLK_SCALE * y
    x = r * torch.rsqrt((r * r).mean(dim=1, keepdim=True) + EPS) * s["pre_gain"]
    if s["out"] == "int8":
        q, scale = _quantise(x)
        x = (q * scale).to(torch.bfloat16)
    else:
        x = x.to(TYPES[s["out"]])
    return r.to(s["residual"].dtype), x


def _plain_product(s):
    q, scale = _quantise(s["tokens"].float())
    w, w_scale = s["weight"]
    y = (q @ w.float().t()) * (scale * w_scale)
    if s["op"] == "gated":
        gate, up = y[:, :s["I"]], y[:, s["I"]:]
        y = gate / (1 + torch.exp(-gate)) * up
    elif s["bias_value"] is not None:
        y = y + s["bias_value"]
    return y.to(TYPES[s["out"]])


def _own(s):
    import okc_muse_kernels_b200 as okc
    if s["op"] == "norm":
        r, x = okc.block_norm(s["residual"], s["block"], post_gain=s["post_gain"], gate=s["gate_value"],
                              gate_sigmoid=s["gate"] == "token", residual_scale=RES_SCALE, block_scale=BLK_SCALE,
                              pre_gain=s["pre_gain"], eps=EPS, out=s["out"])
        if s["out"] == "int8":      # the values that the int8 rows stand for
            x = (x.q * x.scale[:, None]).to(torch.bfloat16)
        return r, x
    if s["op"] == "linear":
        return okc.int8_linear(s["tokens"], s["weight"], bias=s["bias_value"], out_f32=s["out"] == "f32")
    return okc.int8_gated(s["tokens"], s["weight"], out_f32=s["out"] == "f32")


def run(state):
    if own:
        return _own(state)
    return _plain_norm(state) if state["op"] == "norm" else _plain_product(state)


def work(case):
    size = {"bf16": 2, "f32": 4}
    T = case["T"]
    if case["op"] == "norm":
        H = case["H"]
        gate = {"none": 0, "channel": 4 * H, "token": 2 * T, "element": 2 * T * H}[case["gate"]]
        out = T * H + 4 * T if case["out"] == "int8" else T * H * size[case["out"]]
        return {"bytes": T * H * (2 * size[case["res"]] + size[case["blk"]]) + out + gate + (8 if case["post"] else 4) * H,
                "flops": 12 * T * H}
    K = case["K"]
    rows, n = (case["N"], case["N"]) if case["op"] == "linear" else (2 * case["I"], case["I"])
    return {"bytes": rows * K + (8 if case.get("bias") else 4) * rows + T * K * size[case["x"]] + T * n * size[case["out"]],
            "flops": 2 * T * K * rows}


def exact(case, seed):
    """The same outputs from the definitions, in 64 bits.  Where an operator's definition rounds (the int8 values of
    a row: multiplier and product in f32, halves to even), the same rounding stands here."""
    s = prepare(case, seed)

    def sigmoid(v):
        return torch.special.expit(v)

    def int8_values(x):
        peak = torch.linalg.vector_norm(x, ord=float("inf"), dim=1)
        multiplier = (127.0 / peak).float().double()
        q = torch.einsum("tk,t->tk", x, multiplier).float().double().round()
        q[peak < TINY] = 0
        return q, torch.where(peak < TINY, 0.0, (peak / 127.0).float().double())

    if case["op"] == "norm":
        r = s["residual"].double() * RES_SCALE
        y = s["block"].double()
        if case["post"]:
            y = torch.einsum("th,t,h->th", y, (y.pow(2).mean(1) + EPS).pow(-0.5), s["post_gain"].double())
        if case["gate"] == "token":
            y = y * sigmoid(s["gate_value"].double())
        elif case["gate"] != "none":
            y = y * s["gate_value"].double()
        r = r + BLK_SCALE * y
        x = torch.einsum("th,t,h->th", r, (r.pow(2).mean(1) + EPS).pow(-0.5), s["pre_gain"].double())
        if case["out"] == "int8":
            q, scale = int8_values(x)
            x = q * scale[:, None]
        return r, x
    q, scale = int8_values(s["tokens"].double())
    w, w_scale = s["weight"]
    y = torch.einsum("tk,nk->tn", q * scale[:, None], w.double() * w_scale.double()[:, None])
    if case["op"] == "gated":
        return torch.nn.functional.silu(y[:, :case["I"]]) * y[:, case["I"]:]
    return y if s["bias_value"] is None else y + s["bias_value"].double()
