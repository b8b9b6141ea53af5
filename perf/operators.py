"""Timed and checked cases of the operators beside the convolution.

* ``linear``     quantise rows to int8, int8 matrix product with its epilogue
* ``matmul``     the product alone, on int8 operands that are already there
* ``mlp``        quantise, product with an activation to int8, product with a residual
* ``experts``    gather and quantise rows, matrix products grouped by expert
* ``norm``       group norm with an activation, channels last
* ``norm_proj``  group norm to int8, then the 1x1 projection that reads it

Where ``own`` is false, ``run`` computes them in elementary torch operations.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "int32": 4}


def listed():
    return [
        # One token through a square projection, added to the residual stream:
        # latency and the weights' bytes are all that counts.
        dict(name="token_square", op="linear", m=1, n=4096, k=4096, type="bf16", act="none",
             bias=False, residual=True),
        # A batch of single tokens through a widening layer.
        dict(name="tokens_wide", op="linear", m=16, n=16384, k=4096, type="bf16", act="silu",
             bias=True, residual=False),
        # A prompt through a square layer.
        dict(name="prompt_linear", op="linear", m=2048, n=4096, k=4096, type="fp16", act="gelu",
             bias=True, residual=False),
        # The largest product: many packed prompts, wide layer, residual.
        dict(name="prompt_large", op="matmul", m=16384, n=8192, k=8192, type="bf16", act="none",
             bias=True, residual=True),
        # Odd sizes that end inside every tile, 32-bit output.
        dict(name="ragged_fp32", op="matmul", m=777, n=1111, k=1234, type="fp32", act="gelu",
             bias=True, residual=False),
        # A whole feed-forward block: the hidden layer stays in int8.
        dict(name="mlp_block", op="mlp", m=4096, n=8192, k=2048, type="bf16", act="gelu_tanh",
             bias=True, residual=True),
        # 16 tokens, two experts each, of 32 experts: some experts get none.
        dict(name="experts_tokens", op="experts", m=32, n=4096, k=2048, groups=32, type="bf16",
             act="silu", bias=False, spread=1.0),
        # A long prompt over the same experts, unevenly.
        dict(name="experts_prompt", op="experts", m=16384, n=4096, k=2048, groups=32, type="bf16",
             act="silu", bias=False, spread=0.3),
        # More and smaller experts, odd sizes, 16-bit floats.
        dict(name="experts_ragged", op="experts", m=1500, n=1408, k=1000, groups=60, type="fp16",
             act="none", bias=True, spread=0.6),
        # The int32 output of a small convolution of one image.
        dict(name="norm_small", op="norm", m=1, p=196, c=256, groups=32, source="int32",
             type="bf16", act="silu"),
        # An image model's attention block: norm to int8, 1x1 projection.
        dict(name="norm_project", op="norm_proj", m=8, p=4096, c=320, groups=32, source="bf16",
             n=320, type="bf16", act="none"),
        # The int32 output of the benchmark's convolution (256 images, 56 x 56 x 256).
        dict(name="norm_conv_output", op="norm", m=256, p=3136, c=256, groups=32, source="int32",
             type="fp16", act="relu"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "matmul", "matmul", "mlp", "experts", "experts", "norm",
                     "norm", "norm_proj"])
    kind = rng.choice(["bf16", "bf16", "fp16"])
    act = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
    if op in ("linear", "matmul", "mlp"):
        n, k = _log(rng, 64, 16384), _log(rng, 64, 16384)
        m = _log(rng, 1, min(16384, max(1, 16384 * 8192 * 8192 // (2 * n * k))))
        if rng.random() < 0.5:
            n, k = (n + 63) // 64 * 64, (k + 63) // 64 * 64
        return dict(op=op, m=m, n=n, k=k, type=rng.choice([kind, "fp32"]) if op == "matmul" else kind,
                    act=act, bias=rng.random() < 0.5, residual=rng.random() < 0.5)
    if op == "experts":
        n, k, e = _log(rng, 64, 8192), _log(rng, 64, 4096), _log(rng, 2, 128)
        m = _log(rng, 1, 16384)
        return dict(op=op, m=m, n=n, k=k, groups=e, type=kind, act=act, bias=rng.random() < 0.5,
                    spread=rng.choice([0.2, 0.5, 1.0]))
    groups = rng.choice([1, 8, 16, 32])
    c = groups * _log(rng, 2, 64)
    p = _log(rng, 1, 16384)
    m = _log(rng, 1, min(64, max(1, (1 << 27) // (p * c))))
    if op == "norm_proj":
        return dict(op=op, m=m, p=p, c=c, groups=groups, source=rng.choice(["bf16", "int32"]),
                    n=_log(rng, 32, 1024), type="bf16", act=rng.choice(["none", "silu"]))
    return dict(op=op, m=m, p=p, c=c, groups=groups,
                source=rng.choice(["int32", "bf16", "fp16", "fp32"]),
                type=rng.choice([kind, "fp32"]), act=act)


def _ints(g, rows, k):
    """int8 values of a quantised matrix, in rows of 16-byte pitch as the products take them."""
    pitch = (k + 15) // 16 * 16
    v = torch.empty(rows, pitch, dtype=torch.int8, device="cuda")
    step = max(1, (1 << 26) // pitch)
    for i in range(0, rows, step):
        part = torch.randn(min(step, rows - i), pitch, generator=g, device="cuda")
        v[i:i + step] = (part * 36).round_().clamp_(-127, 127).to(torch.int8)
    return v[:, :k]


def _sizes(case, seed):
    """Rows of each expert: every row drawn from uneven weights."""
    g = torch.Generator().manual_seed(seed * 7 + 1)
    w = torch.exp(case["spread"] * torch.randn(case["groups"], generator=g))
    which = torch.multinomial(w, case["m"], replacement=True, generator=g)
    return torch.bincount(which, minlength=case["groups"])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def floats(*shape, scale=1.0, add=0.0):
        return torch.randn(*shape, generator=g, device="cuda") * scale + add

    def positive(*shape, about=1.0):
        return (torch.rand(*shape, generator=g, device="cuda") + 0.5) * about

    op, m, kind = case["op"], case["m"], _TYPES[case["type"]]
    s = {"case": case}
    if op in ("norm", "norm_proj"):
        c = case["c"]
        offset = floats(c, scale=0.5)
        if case["source"] == "int32":  # accumulators of a convolution, and what one step is worth
            s["x"] = torch.empty(m, case["p"], c, dtype=torch.int32, device="cuda")
            for i in range(0, m, 16):
                s["x"][i:i + 16] = ((floats(min(16, m - i), case["p"], c) + offset) * 2000).round()
            s["scale"] = positive(c, about=1 / 2000)
        else:
            s["x"] = (floats(m, case["p"], c) + offset).to(_TYPES[case["source"]])
            s["scale"] = None
        s["gamma"], s["beta"] = positive(c), floats(c, scale=0.3)
        if op == "norm_proj":
            n = case["n"]
            s["w"], s["step"] = _ints(g, n, c), 4.5 / 127
            s["col"] = positive(n, about=1 / (36 * math.sqrt(c))) * s["step"]
            s["bias"] = floats(n, scale=0.1)
        return s
    n, k = case["n"], case["k"]
    e = case.get("groups")
    about = 1 / (36 * math.sqrt(k))  # a product's values come out near one
    s["w"] = _ints(g, n * (e or 1), k)
    if e:
        s["w"] = s["w"].as_strided((e, n, k), (n * s["w"].stride(0), s["w"].stride(0), 1))
    s["col"] = positive(*((e, n) if e else (n,)), about=about)
    s["bias"] = floats(*((e, n) if e else (n,)), scale=0.2) if case["bias"] else None
    s["residual"] = floats(m, n).to(kind) if case.get("residual") and op != "mlp" else None
    if op == "matmul":
        s["a"], s["row"] = _ints(g, m, k), positive(m, about=1 / 36)
        return s
    loud = torch.ones(k, device="cuda")  # a few channels are far louder, as activations' are
    loud[torch.randint(0, k, (max(1, k // 256),), generator=g, device="cuda")] = 6.0
    if op == "experts":
        sizes = _sizes(case, seed)
        tokens = max(1, m // 2)
        s["x"] = (floats(tokens, k) * loud).to(kind)
        s["index"] = torch.randint(0, tokens, (m,), generator=g, device="cuda", dtype=torch.int32)
        s["most"] = int(sizes.max())
        s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), sizes.cumsum(0)]).to(torch.int32).cuda()
        return s
    s["x"] = (floats(m, k) * loud).to(kind)
    if op == "mlp":
        s["step"] = 4.0 / 127  # the hidden layer's scale, known from calibration
        s["w2"] = _ints(g, k, n)
        s["col2"] = positive(k, about=1 / (36 * math.sqrt(n))) * s["step"]
    return s


def _act(y, act):
    if act == "relu":
        return y.clamp_min(0)
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y * 0.7071067811865476))
    if act == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y * y * y)))
    if act == "silu":
        return y / (1 + torch.exp(-y))
    return y


def _quantize(x):
    x = x.float()
    scale = x.abs().amax(1) / 127
    q = torch.round(x / torch.where(scale > 0, scale, 1.0)[:, None])
    return q, scale


def _product(q, w, row, col, bias, act):
    y = q @ w.float().transpose(-1, -2)
    y = y * col.unsqueeze(-2)
    if row is not None:
        y = y * row.unsqueeze(-1)
    if bias is not None:
        y = y + bias.unsqueeze(-2)
    return _act(y, act)


def _normalised(s):
    case = s["case"]
    x = s["x"].float()
    if s["scale"] is not None:
        x = x * s["scale"]
    m, p, c = x.shape
    x = x.view(m, p, case["groups"], c // case["groups"])
    x = x - x.mean((1, 3), keepdim=True)
    x = x * torch.rsqrt((x * x).mean((1, 3), keepdim=True) + 1e-5)
    return _act(x.view(m, p, c) * s["gamma"] + s["beta"], case["act"])


def run(s):
    case = s["case"]
    op, kind, act = case["op"], _TYPES[case["type"]], case["act"]
    if own:
        return _run_own(s, op, kind, act)
    if op == "norm":
        return _normalised(s).to(kind)
    if op == "norm_proj":
        q = torch.round(_normalised(s) * (1 / s["step"])).clamp(-128, 127)
        return _product(q.view(-1, case["c"]), s["w"], None, s["col"], s["bias"], "none").to(kind)
    if op == "experts":
        q, row = _quantize(s["x"][s["index"]])
        # Every expert's rows side by side, padded to the longest; one batched product.
        start = s["offsets"][:-1].long()
        at = torch.arange(case["m"], device="cuda")
        expert = torch.searchsorted(s["offsets"][1:].long(), at, right=True)
        place = at - start[expert]
        wide = torch.zeros(case["groups"], s["most"], case["k"], device="cuda")
        wide[expert, place] = q
        rows = torch.zeros(case["groups"], s["most"], device="cuda")
        rows[expert, place] = row
        return _product(wide, s["w"], rows, s["col"], s["bias"], act)[expert, place].to(kind)
    if op == "matmul":
        y = _product(s["a"].float(), s["w"], s["row"], s["col"], s["bias"], act)
    else:
        q, row = _quantize(s["x"])
        y = _product(q, s["w"], row, s["col"], s["bias"], act)
        if op == "mlp":
            q = torch.round(y * (1 / s["step"])).clamp(-128, 127)
            return (_product(q, s["w2"], None, s["col2"], None, "none") + s["x"].float()).to(kind)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(kind)


def _run_own(s, op, kind, act):
    import int8_kernel_lab_b200 as lab

    if op == "norm":
        return lab.group_norm(s["x"], s["case"]["groups"], s["gamma"], s["beta"], eps=1e-5,
                              activation=act, scale=s["scale"], dtype=kind)
    if op == "norm_proj":
        q = lab.group_norm(s["x"], s["case"]["groups"], s["gamma"], s["beta"], eps=1e-5,
                           activation=act, scale=s["scale"], dtype=torch.int8, out_scale=s["step"])
        return lab.matmul(q.view(-1, s["case"]["c"]), s["w"], col_scale=s["col"], bias=s["bias"],
                          dtype=kind)
    if op == "matmul":
        return lab.matmul(s["a"], s["w"], row_scale=s["row"], col_scale=s["col"], bias=s["bias"],
                          activation=act, residual=s["residual"], dtype=kind)
    if op == "experts":
        q, row = lab.quantize_rows(s["x"], s["index"])
        return lab.grouped_matmul(q, s["w"], s["offsets"], row_scale=row, col_scale=s["col"],
                                  bias=s["bias"], activation=act, dtype=kind)
    q, row = lab.quantize_rows(s["x"])
    if op == "mlp":
        q = lab.matmul(q, s["w"], row_scale=row, col_scale=s["col"], bias=s["bias"],
                       activation=act, dtype=torch.int8, out_scale=s["step"])
        return lab.matmul(q, s["w2"], col_scale=s["col2"], residual=s["x"], dtype=kind)
    return lab.matmul(q, s["w"], row_scale=row, col_scale=s["col"], bias=s["bias"],
                      activation=act, residual=s["residual"], dtype=kind)


def work(case):
    op, m, out = case["op"], case["m"], _BYTES[case["type"]]
    if op in ("norm", "norm_proj"):
        cells = m * case["p"] * case["c"]
        read = cells * _BYTES[case["source"]] + 12 * case["c"]
        if op == "norm":
            return {"bytes": read + cells * out, "flops": 8 * cells}
        rows, n = m * case["p"], case["n"]
        return {"bytes": read + n * case["c"] + 8 * n + rows * n * out,
                "flops": 8 * cells + 2 * rows * n * case["c"]}
    n, k = case["n"], case["k"]
    if op == "mlp":
        return {"bytes": 2 * m * k * out + 2 * n * k + 8 * (n + k), "flops": 4 * m * n * k}
    reached, source = 1, m * k * (1 if op == "matmul" else out)
    if op == "experts":
        reached = int((_sizes(case, 0) > 0).sum())
        source = max(1, m // 2) * k * out + 4 * m  # the gathered rows are read once each
    extra = m * n * out if case.get("residual") else 0
    return {"bytes": source + reached * (n * k + 8 * n) + m * n * out + extra,
            "flops": 2 * m * n * k}


def exact(case, seed):
    """The operators' definitions, in 64 bits."""
    s = prepare(case, seed)
    act = {"none": lambda v: v,
           "relu": lambda v: torch.where(v > 0, v, torch.zeros_like(v)),
           "gelu": lambda v: v * torch.special.ndtr(v),
           "gelu_tanh": lambda v: v * torch.sigmoid(math.sqrt(8 / math.pi) * (v + 0.044715 * v ** 3)),
           "silu": lambda v: v * torch.sigmoid(v)}[case["act"]]

    def levels(x):
        x = x.double()
        unit = x.abs().max(dim=1, keepdim=True).values / 127
        unit[unit == 0] = 1
        return (x / unit).round(), unit

    op = case["op"]
    if op in ("norm", "norm_proj"):
        c, parts = case["c"], []
        for x in s["x"]:
            x = x.double() * (1 if s["scale"] is None else s["scale"].double())
            x = x.reshape(-1, case["groups"], c // case["groups"])
            var, mean = torch.var_mean(x, dim=(0, 2), unbiased=False, keepdim=True)
            x = ((x - mean) / (var + 1e-5).sqrt()).reshape(-1, c)
            y = act(torch.addcmul(s["beta"].double(), x, s["gamma"].double()))
            if op == "norm_proj":
                y = (y / s["step"]).round().clamp(-128, 127)
                y = torch.addmm(s["bias"].double(), y, (s["w"].double() * s["col"].double()[:, None]).t())
            parts.append(y)
        return torch.cat(parts) if op == "norm_proj" else torch.stack(parts)
    if op == "experts":
        a, unit = levels(s["x"][s["index"].long()])
        out, ends = torch.empty(case["m"], case["n"], dtype=torch.float64, device="cuda"), s["offsets"].tolist()
        for e, (lo, hi) in enumerate(zip(ends, ends[1:])):
            y = (a[lo:hi] * unit[lo:hi]) @ (s["w"][e].double() * s["col"][e].double()[:, None]).t()
            out[lo:hi] = act(y if s["bias"] is None else y + s["bias"][e].double())
        return out
    a, unit = (s["a"].double(), s["row"].double()[:, None]) if op == "matmul" else levels(s["x"])
    y = (a * unit) @ (s["w"].double() * s["col"].double()[:, None]).t()
    y = act(y if s["bias"] is None else y + s["bias"].double())
    if op == "mlp":
        y = (y / s["step"]).round().clamp(-128, 127)
        return y @ (s["w2"].double() * s["col2"].double()[:, None]).t() + s["x"].double()
    return y if s["residual"] is None else y + s["residual"].double()
