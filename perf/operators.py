"""The work that the operators of dream_go_amd.ops are measured on: dense, group_norm and adjust_logits.

`run` computes an operator in its plain form (elementary torch operations in 32 bits, one rounding at the end) or, where `own` is
true, through the library.  `exact` states the same definitions in 64 bits."""
import math

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
TAU = 1.0 / 0.709888            # the policy head's temperature as a factor on its logits

_ops = None


def _library():
    global _ops
    if _ops is None:
        import __graft_entry__
        __graft_entry__.package()
        from dream_go_amd import ops
        _ops = ops
    return _ops


def listed():
    return [
        # the policy head's dense layer (361 points x 8 planes -> 362 moves) for one position and for a full leaf batch
        dict(name="dense policy head, 1", op="dense", m=1, k=2888, n=362, type="fp16", out="fp32", act="identity", alpha1=TAU, bias=True, residual=False),
        dict(name="dense policy head, 256", op="dense", m=256, k=2888, n=362, type="fp16", out="fp16", act="identity", alpha1=TAU, bias=True, residual=False),
        # a wide layer on the tokens of one serving step: the weights are all there is to read
        dict(name="dense 16 tokens, wide", op="dense", m=16, k=4096, n=16384, type="bf16", out="bf16", act="gelu", alpha1=1.0, bias=True, residual=False),
        # a ragged batch through an odd layer: no row of either operand is aligned
        dict(name="dense odd sizes", op="dense", m=1021, k=2027, n=1531, type="bf16", out="bf16", act="silu", alpha1=1.0, bias=True, residual=True),
        # the second layer of a wide block over a long prompt, its residual added on the way
        dict(name="dense 8192 tokens, wide", op="dense", m=8192, k=16384, n=4096, type="bf16", out="bf16", act="identity", alpha1=1.0, bias=True, residual=True),
        # one position behind a narrow convolution
        dict(name="group norm, one board", op="group_norm", n=1, p=361, c=64, groups=8, type="fp16", act="relu", residual=False),
        # the end of a residual block for a leaf batch: norm, skip, ReLU
        dict(name="group norm, 256 boards", op="group_norm", n=256, p=361, c=256, groups=32, type="fp16", act="relu", residual=True),
        # large feature maps with groups of ten channels
        dict(name="group norm, large maps", op="group_norm", n=8, p=16384, c=320, groups=32, type="bf16", act="silu", residual=False),
        # fp32 maps whose rows are not a multiple of 16 bytes
        dict(name="group norm, odd sizes", op="group_norm", n=13, p=1021, c=90, groups=9, type="fp32", act="gelu", residual=False),
        # one position's moves: what is legal, and a discount on what was just played
        dict(name="logits, one position", op="logits", b=1, v=362, t=8, type="fp16", mask="row", bias="none", penalties=True),
        # an odd vocabulary, one bias for all rows, a grammar for each
        dict(name="logits, odd vocabulary", op="logits", b=32, v=50257, t=700, type="fp32", mask="row", bias="vocabulary", penalties=True),
        # a serving step of many long sequences
        dict(name="logits, 256 sequences", op="logits", b=256, v=131072, t=8192, type="bf16", mask="row", bias="vocabulary", penalties=True),
    ]


def _spread(rng, low, high):
    """A size between low and high, spread over its logarithm, one in three odd."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.34:
        v |= 1
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(("dense", "group_norm", "logits"))
    if op == "dense":
        while True:
            m, n, k = _spread(rng, 1, 8192), _spread(rng, 1, 16384), _spread(rng, 1, 16384)
            if rng.random() < 0.6:
                n, k = -(-n // 8) * 8, -(-k // 8) * 8
            if m * n * k <= 8192 * 16384 * 4096 and m * n <= 1 << 26:
                break
        t = rng.choice(("fp16", "bf16"))
        return dict(op=op, m=m, k=k, n=n, type=t, out=rng.choice((t, t, t, "fp32")), act=rng.choice(("identity", "relu", "tanh", "gelu", "silu")),
                    alpha1=rng.choice((1.0, 0.5, TAU)), bias=rng.random() < 0.7, residual=rng.random() < 0.5)
    if op == "group_norm":
        while True:
            groups, per = rng.choice((1, 2, 4, 8, 9, 16, 32)), rng.choice((1, 2, 3, 4, 8, 10, 16, 20, 32, 64))
            n, p = _spread(rng, 1, 512), _spread(rng, 1, 16384)
            if n * p * groups * per <= 8 * 16384 * 320:
                break
        return dict(op=op, n=n, p=p, c=groups * per, groups=groups, type=rng.choice(("fp16", "bf16", "fp32")),
                    act=rng.choice(("identity", "relu", "tanh", "gelu", "silu")), residual=rng.random() < 0.5)
    b, v, t = _spread(rng, 1, 256), _spread(rng, 100, 131072), _spread(rng, 1, 8192)
    return dict(op=op, b=b, v=v, t=t, type=rng.choice(("fp16", "bf16", "fp32")), mask=rng.choice(("none", "row", "row", "shared")),
                bias=rng.choice(("none", "vocabulary", "row")), penalties=rng.random() < 0.75)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["type"]]

    def normal(*shape, scale=1.0, shift=0.0, to=dtype):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(to)

    s = dict(case)
    if case["op"] == "dense":
        m, n, k = case["m"], case["n"], case["k"]
        s["x"], s["w"] = normal(m, k), normal(n, k, scale=1.0 / math.sqrt(k))
        s["b"] = normal(n, scale=0.5) if case["bias"] else None
        s["z"] = normal(m, n, to=TYPES[case["out"]]) if case["residual"] else None
    elif case["op"] == "group_norm":
        n, p, c = case["n"], case["p"], case["c"]
        s["x"] = (torch.randn(n, p, c, generator=g, device="cuda") * normal(c, scale=0.5, shift=1.5, to=torch.float32)
                  + normal(n, 1, c, to=torch.float32)).to(dtype)
        s["w"], s["b"] = normal(c, scale=0.2, shift=1.0), normal(c, scale=0.2)
        s["z"] = normal(n, p, c) if case["residual"] else None
    else:
        b, v, t = case["b"], case["v"], case["t"]
        s["logits"] = normal(b, v, scale=3.0)
        s["mask"] = s["bias_t"] = s["history"] = None
        if case["mask"] != "none":
            rows, words = b if case["mask"] == "row" else 1, -(-v // 32)
            # a grammar leaves a few tokens in some places and most in others; the last of several rows has nothing left
            some = [torch.randint(-(1 << 31), 1 << 31, (rows, words), generator=g, device="cuda") for _ in range(2)]
            s["mask"] = torch.where(torch.rand(rows, 1, generator=g, device="cuda") < 0.5, some[0] & some[1], some[0] | some[1]).to(torch.int32)
            if rows > 1:
                s["mask"][-1] = 0
        if case["bias"] != "none":
            s["bias_t"] = normal(*((v,) if case["bias"] == "vocabulary" else (b, v)), scale=0.7, to=torch.float32)
        if case["penalties"]:
            # words come back as they do in text: the frequent ones often
            s["history"] = (torch.rand(b, t, generator=g, device="cuda").pow(3) * v).to(torch.int32).clamp_(max=v - 1)
            s["lengths"] = torch.randint(0, t + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
            s["prompts"] = (s["lengths"] * torch.rand(b, generator=g, device="cuda")).to(torch.int32)
            s["repetition"] = 1.0 + torch.rand(b, generator=g, device="cuda")
            s["presence"], s["frequency"] = (torch.rand(b, generator=g, device="cuda") for _ in range(2))
    return s


def _activate(v, name):
    if name == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if name == "tanh":
        return torch.tanh(v)
    if name == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    return v


def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "dense":
        y = (s["x"].float() @ s["w"].float().t()) * s["alpha1"]
        if s["z"] is not None:
            y = y + s["z"].float()
        if s["b"] is not None:
            y = y + s["b"].float()
        return _activate(y, s["act"]).to(TYPES[s["out"]])
    if s["op"] == "group_norm":
        n, p, c, groups = s["n"], s["p"], s["c"], s["groups"]
        x = s["x"].float().view(n, p, groups, c // groups)
        x = x - x.mean((1, 3), keepdim=True)
        y = x * torch.rsqrt((x * x).mean((1, 3), keepdim=True) + 1e-5)
        y = y.view(n, p, c) * s["w"].float() + s["b"].float()
        if s["z"] is not None:
            y = y + s["z"].float()
        return _activate(y, s["act"]).to(s["x"].dtype)
    b, v, t = s["b"], s["v"], s["t"]
    y = s["logits"].float()
    if s["history"] is not None:
        at = torch.arange(t, device=y.device)
        within = at < s["lengths"][:, None]
        answer = within & (at >= s["prompts"][:, None])
        tokens = s["history"].long()
        seen, count = (torch.zeros(b, v, device=y.device).scatter_add_(1, tokens, w.float()) for w in (within, answer))
        r = s["repetition"][:, None]
        y = torch.where(seen > 0, torch.where(y > 0, y / r, y * r), y)
        y = y - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias_t"] is not None:
        y = y + s["bias_t"]
    if s["mask"] is not None:
        bits = (s["mask"][:, :, None] >> torch.arange(32, device=y.device, dtype=torch.int32)) & 1
        y = torch.where(bits.view(s["mask"].shape[0], -1)[:, :v] != 0, y, -math.inf)
    return y.to(s["logits"].dtype)


def _run_own(s):
    ops = _library()
    if s["op"] == "dense":
        return ops.dense(s["x"], s["w"], s["b"], s["z"], alpha1=s["alpha1"], activation=s["act"], out_dtype=TYPES[s["out"]])
    if s["op"] == "group_norm":
        return ops.group_norm(s["x"], s["groups"], s["w"], s["b"], s["z"], eps=1e-5, activation=s["act"])
    if s["history"] is None:
        return ops.adjust_logits(s["logits"], mask=s["mask"], bias=s["bias_t"])
    return ops.adjust_logits(s["logits"], mask=s["mask"], bias=s["bias_t"], history=s["history"], lengths=s["lengths"], prompt_lengths=s["prompts"],
                             repetition=s["repetition"], presence=s["presence"], frequency=s["frequency"])


def work(case):
    size = {"fp16": 2, "bf16": 2, "fp32": 4}
    e = size[case["type"]]
    if case["op"] == "dense":
        m, n, k = case["m"], case["n"], case["k"]
        o = size[case["out"]]
        return {"bytes": (m * k + n * k) * e + m * n * o * (2 if case["residual"] else 1) + (n * e if case["bias"] else 0), "flops": 2 * m * n * k}
    if case["op"] == "group_norm":
        elements = case["n"] * case["p"] * case["c"]
        return {"bytes": elements * e * (3 if case["residual"] else 2) + 2 * case["c"] * e, "flops": 8 * elements}
    b, v = case["b"], case["v"]
    bits = {"none": 0, "shared": 1, "row": b}[case["mask"]] * -(-v // 32) * 4
    bias = {"none": 0, "vocabulary": 1, "row": b}[case["bias"]] * v * 4
    return {"bytes": 2 * b * v * e + bits + bias + (b * (case["t"] * 4 + 20) if case["penalties"] else 0), "flops": 4 * b * v}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "dense":
        y = torch.mm(s["w"].double(), s["x"].double().t().contiguous()).t() * case["alpha1"]
        for extra in (s["b"], s["z"]):
            if extra is not None:
                y = y + extra.double()
        return _exact_activation(y, case["act"])
    if case["op"] == "group_norm":
        groups, per = case["groups"], case["c"] // case["groups"]
        out = torch.empty(case["n"], case["p"], case["c"], dtype=torch.float64, device="cuda")
        for j in range(groups):
            at = slice(j * per, (j + 1) * per)
            x = s["x"][:, :, at].double()
            var, mean = torch.var_mean(x, dim=(1, 2), unbiased=False, keepdim=True)
            y = (x - mean) / torch.sqrt(var + 1e-5) * s["w"][at].double() + s["b"][at].double()
            out[:, :, at] = y if s["z"] is None else y + s["z"][:, :, at].double()
        return _exact_activation(out, case["act"])
    rows = []
    for i in range(case["b"]):
        y = s["logits"][i].double()
        if case["penalties"]:
            length, prompt = int(s["lengths"][i]), int(s["prompts"][i])
            whole = torch.bincount(s["history"][i, :length], minlength=case["v"])
            answer = torch.bincount(s["history"][i, prompt:length], minlength=case["v"])
            r = s["repetition"][i].double()
            y = torch.where(whole.bool(), torch.minimum(y * r, y / r) if float(r) >= 1 else torch.maximum(y * r, y / r), y)
            y = y - answer * s["frequency"][i].double() - answer.clamp(max=1) * s["presence"][i].double()
        if s["bias_t"] is not None:
            y = y + (s["bias_t"] if s["bias_t"].dim() == 1 else s["bias_t"][i]).double()
        if s["mask"] is not None:
            words = s["mask"][i if s["mask"].shape[0] > 1 else 0].long() & 0xFFFFFFFF
            token = torch.arange(case["v"], device="cuda")
            y = y.masked_fill((words[token // 32] // 2 ** (token % 32)) % 2 == 0, -math.inf)
        rows.append(y)
    return torch.stack(rows)


def _exact_activation(y, name):
    if name == "relu":
        return y.clamp(min=0)
    if name == "tanh":
        return 1 - 2 / (torch.exp(2 * y) + 1)
    if name == "gelu":
        return y * torch.special.ndtr(y)
    if name == "silu":
        return y * torch.sigmoid(y)
    return y
