"""Workloads of three operators: the RMSNorm with the residual's addition and an FP8 output, the 16-bit
linear layer, and the block-scaled FP8 linear layer on activations that are already quantized, the last
two with bias, activation and residual in their epilogue.

`own` chooses between the operators' plain forms (elementary torch operations) and the library's calls.
Cases are dicts with an "op":

  norm    s = x + residual, rounded to x's type; y = s / sqrt(mean(s^2) + eps) * weight, rounded once;
          codes = e4m3(y / scale) per row and 128 columns with scale = max(absmax, 1e-10) / 448, taken
          from y before its rounding
  linear  act(x W^T + bias) + residual, 16-bit x and W, 32-bit sums, rounded once
  fp8     act(sum_b (code_x . code_w over 128 columns b) scale_x[t, b] scale_w[r / 128, b] + bias) +
          residual, rounded once; "qkv" is the checkpoint's fused QKV row and scale map
"""
import math

import torch

own = False

EPS = 1e-5
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
QKV_ROWS, QKV_COLS = 13568, 4096  # the fused full-attention QKV projection


def listed():
    return [
        # the decode step's norm: one token of a 4096-wide model, everything asked for
        {"name": "norm decode", "op": "norm", "rows": 1, "hidden": 4096, "dtype": "bf16", "residual": True, "y": True,
         "codes": True, "pad": 0},
        # a 2048-token prompt on its way into the FP8 projections: the stream and the codes, no y
        {"name": "norm prompt", "op": "norm", "rows": 2048, "hidden": 4096, "dtype": "bf16", "residual": True,
         "y": False, "codes": True, "pad": 0},
        # an odd width in rows cut from a wider buffer, in 32 bits: no vector fits
        {"name": "norm odd f32", "op": "norm", "rows": 777, "hidden": 5003, "dtype": "f32", "residual": True, "y": True,
         "codes": True, "pad": 6},
        # the final norm of a long batch, no residual
        {"name": "norm batch f16", "op": "norm", "rows": 16384, "hidden": 8192, "dtype": "f16", "residual": False,
         "y": True, "codes": False, "pad": 0},
        # the attention output projection of one token, onto the stream
        {"name": "linear decode", "op": "linear", "width": 1, "rows": 4096, "cols": 8192, "dtype": "bf16",
         "out": "bf16", "bias": False, "act": "none", "residual": True, "pad": 0},
        # the vocabulary's logits of a verifier's eight tokens, in 32 bits
        {"name": "linear logits", "op": "linear", "width": 8, "rows": 152576, "cols": 4096, "dtype": "bf16",
         "out": "f32", "bias": False, "act": "none", "residual": False, "pad": 0},
        # a ragged batch through odd sizes
        {"name": "linear odd f16", "op": "linear", "width": 77, "rows": 5001, "cols": 1003, "dtype": "f16",
         "out": "f16", "bias": True, "act": "silu", "residual": True, "pad": 5},
        # the attention output projection of a 2048-token prompt
        {"name": "linear prompt", "op": "linear", "width": 2048, "rows": 4096, "cols": 8192, "dtype": "bf16",
         "out": "bf16", "bias": False, "act": "none", "residual": True, "pad": 0},
        # a feed-forward's first projection over a long batch
        {"name": "linear batch gelu", "op": "linear", "width": 8192, "rows": 16384, "cols": 4096, "dtype": "bf16",
         "out": "bf16", "bias": True, "act": "gelu", "residual": False, "pad": 0},
        # the fused QKV projection of a verifier's eight tokens, from the norm's codes
        {"name": "fp8 qkv verify", "op": "fp8", "width": 8, "rows": QKV_ROWS, "cols": QKV_COLS, "qkv": True,
         "out": "bf16", "bias": False, "act": "none", "residual": False},
        # one expert-sized down projection of a ragged batch, onto the stream
        {"name": "fp8 down ragged", "op": "fp8", "width": 203, "rows": 4096, "cols": 2048, "qkv": False,
         "out": "f32", "bias": True, "act": "none", "residual": True},
        # a wide projection with its activation over a prompt
        {"name": "fp8 prompt silu", "op": "fp8", "width": 2048, "rows": 16384, "cols": 4096, "qkv": False,
         "out": "bf16", "bias": True, "act": "silu", "residual": False},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "linear", "fp8"])
    if op == "norm":
        hidden = _log(rng, 64, 16384)
        if rng.random() < 0.6:
            hidden = max(128, hidden // 128 * 128)
        rows = _log(rng, 1, min(16384, max(1, (1 << 27) // hidden)))
        y = rng.random() < 0.7
        return {"op": op, "rows": rows, "hidden": hidden, "dtype": rng.choice(["bf16", "f16", "f32"]),
                "residual": rng.random() < 0.7, "y": y, "codes": not y or rng.random() < 0.6,
                "pad": rng.choice([0, 0, 8, rng.randint(1, 40)])}
    act = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
    more = {"bias": rng.random() < 0.5, "act": act, "residual": rng.random() < 0.5}
    if op == "linear":
        width, rows, cols = _log(rng, 1, 8192), _log(rng, 64, 16384), _log(rng, 64, 8192)
        if rng.random() < 0.6:
            rows, cols = max(64, rows // 64 * 64), max(64, cols // 64 * 64)
        dtype = rng.choice(["bf16", "bf16", "f16"])
        return {"op": op, "width": min(width, max(1, (1 << 39) // (rows * cols))), "rows": rows, "cols": cols,
                "dtype": dtype, "out": rng.choice([dtype, dtype, "f32"]), "pad": rng.choice([0, 0, rng.randint(1, 40)]),
                **more}
    qkv = rng.random() < 0.2
    return {"op": op, "width": _log(rng, 1, 2048), "rows": QKV_ROWS if qkv else 128 * _log(rng, 1, 128),
            "cols": QKV_COLS if qkv else 128 * _log(rng, 1, 32), "qkv": qkv, "out": rng.choice(["bf16", "f16", "f32"]),
            **more}


# ------------------------------------------------------------------ inputs
def _padded(rows, cols, pad, dtype, g, scale=1.0):
    """[rows, cols] normal values in rows of a buffer that is `pad` columns wider, its row stride a multiple of 8."""
    width = cols if not pad else (cols + pad + 7) // 8 * 8
    t = torch.empty((rows, width), dtype=dtype, device="cuda")
    for r in range(0, rows, 16384):  # in pieces: no second copy of a large matrix in 32 bits
        n = min(16384, rows - r)
        t[r:r + n] = torch.randn((n, width), generator=g, device="cuda").mul_(scale)
    return t[:, :cols]


def _stream(rows, cols, pad, dtype, g):
    """A residual stream: a few channels carry most of the energy."""
    t = _padded(rows, cols, pad, dtype, g, 2.0)
    loud = torch.randint(0, cols, (max(1, cols // 512),), generator=g, device="cuda")
    t[:, loud] *= 12.0
    return t


def _row_codes(x):
    """e4m3 codes per row and 128 columns, and their scales."""
    rows, cols = x.shape
    v = x.view(rows, cols // 128, 128)
    scale = v.abs().amax(-1).clamp_min(1e-10) / 448.0
    codes = (v / scale[..., None]).to(torch.float8_e4m3fn).view(torch.uint8).view(rows, cols)
    return codes, scale.contiguous()


def _block_codes(w):
    """e4m3 codes and scales per 128 x 128 block."""
    rows, cols = w.shape
    v = w.view(rows // 128, 128, cols // 128, 128)
    scale = v.abs().amax((1, 3)).clamp_min(1e-10) / 448.0
    codes = (v / scale[:, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8).view(rows, cols)
    return codes, scale.contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "norm":
        t = TYPES[case["dtype"]]
        rows, hidden = case["rows"], case["hidden"]
        return {"case": case, "x": _stream(rows, hidden, case["pad"], t, g),
                "residual": _stream(rows, hidden, case["pad"], t, g) if case["residual"] else None,
                "weight": (1.0 + 0.2 * torch.randn(hidden, generator=g, device="cuda")).to(torch.bfloat16)}
    width, rows, cols = case["width"], case["rows"], case["cols"]
    out = TYPES[case["out"]]
    s = {"case": case,
         "bias": torch.randn(rows, generator=g, device="cuda").to(out) if case["bias"] else None,
         "residual": torch.randn((width, rows), generator=g, device="cuda").to(out) if case["residual"] else None}
    if op == "linear":
        t = TYPES[case["dtype"]]
        s["x"] = _padded(width, cols, case["pad"], t, g)
        # a weight's rows start at multiples of 16 bytes
        s["weight"] = _padded(rows, cols, case["pad"] or (-cols) % 8, t, g, cols ** -0.5)
        if s["x"].stride(0) % 8:
            s["x"] = _padded(width, cols, 1, t, g)
        return s
    x = torch.randn((width, cols), generator=g, device="cuda")
    s["codes"], s["scales"] = _row_codes(x)
    if case["qkv"]:
        # checkpoint order: 108 scale rows, each shard's second K block has 64 rows of its own
        w = torch.randn((108 * 128, cols), generator=g, device="cuda").mul_(cols ** -0.5)
        codes, s["weight_scale"] = _block_codes(w)
        blocks = torch.tensor([64 if b % 27 == 25 else 128 for b in range(108)])
        keep = torch.cat([torch.arange(n) + 128 * b for b, n in enumerate(blocks.tolist())]).cuda()
        s["weight"] = codes[keep].contiguous()
    else:
        s["weight"], s["weight_scale"] = _block_codes(
            torch.randn((rows, cols), generator=g, device="cuda").mul_(cols ** -0.5))
    return s


# ------------------------------------------------------------------ the library's calls
_runtimes = {}  # by device: [the runtime, the stream that it runs on]


def _runtime():
    """The current device's runtime, on the current stream."""
    device = torch.cuda.current_device()
    stream = torch._C._cuda_getCurrentRawStream(device)  # torch.cuda.current_stream() takes as long as a short call
    kept = _runtimes.get(device)
    if kept is None:
        from mimo_prismwing_b200.runtime import WideMoeRuntime
        kept = _runtimes[device] = [WideMoeRuntime.compile_with_fused_gate_up(device), None]
    if kept[1] != stream:
        kept[0].set_stream(torch.cuda.current_stream())
        kept[1] = stream
    return kept[0]


def _own(s):
    from mimo_prismwing_b200.runtime import LAYOUT_FULL_QKV, LAYOUT_PLAIN, WideProjectionBinding
    rt = _runtime()
    c = s["case"]
    if c["op"] == "norm":
        r = rt.add_rms_norm(s["x"], s["weight"], EPS, residual=s["residual"], want_y=c["y"],
                            want_codes=c["codes"], asynchronous=True)
        return _norm_outputs(c, r.sum, r.y, r.codes, r.scales)
    out = TYPES[c["out"]]
    if c["op"] == "linear":
        return rt.linear(s["x"], s["weight"], bias=s["bias"], activation=c["act"], residual=s["residual"],
                         out_dtype=out, asynchronous=True).output
    return rt.fp8_linear_codes(s["codes"], s["scales"], WideProjectionBinding(s["weight"], s["weight_scale"]),
                               layout=LAYOUT_FULL_QKV if c["qkv"] else LAYOUT_PLAIN, bias=s["bias"],
                               activation=c["act"], residual=s["residual"], out_dtype=out, asynchronous=True).output


def _norm_outputs(c, total, y, codes, scales):
    out = {}
    if c["residual"]:
        out["sum"] = total
    if c["y"]:
        out["y"] = y
    if c["codes"]:
        out["codes"] = codes.view(torch.float8_e4m3fn) if codes.dtype == torch.uint8 else codes
        out["scales"] = scales
    return out


# ------------------------------------------------------------------ plain forms
def _activate(v, act):
    if act == "relu":
        return v.clamp_min(0.0)
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    return v


def _epilogue(v, s):
    if s["bias"] is not None:
        v = v + s["bias"].float()
    v = _activate(v, s["case"]["act"])
    if s["residual"] is not None:
        v = v + s["residual"].float()
    return v.to(TYPES[s["case"]["out"]])


def _qkv_rows(device):
    """(checkpoint row, scale row) of each of the 13568 output rows: Q, K, V from four shards of [3072|192|128]."""
    r = torch.arange(QKV_ROWS, device=device)
    k, v = r - 12288, r - 13056
    q_at, k_at, v_at = (r // 3072, r % 3072), (k // 192, 3072 + k % 192), (v // 128, 3264 + v % 128)
    shard = torch.where(r < 12288, q_at[0], torch.where(r < 13056, k_at[0], v_at[0]))
    local = torch.where(r < 12288, q_at[1], torch.where(r < 13056, k_at[1], v_at[1]))
    block = torch.where(local < 3264, local // 128, 26)
    return shard * 3392 + local, shard * 27 + block


def _plain(s):
    c = s["case"]
    if c["op"] == "norm":
        total = s["x"]
        if c["residual"]:
            total = (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
        v = total.float()
        y = v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS) * s["weight"].float()
        codes = scales = None
        if c["codes"]:
            rows, hidden = y.shape
            groups = -(-hidden // 128)
            full = torch.zeros((rows, groups * 128), device=y.device)
            full[:, :hidden] = y
            full = full.view(rows, groups, 128)
            scales = full.abs().amax(-1).clamp_min(1e-10) / 448.0
            codes = (full / scales[..., None]).to(torch.float8_e4m3fn).view(rows, groups * 128)[:, :hidden]
        return _norm_outputs(c, total, y.to(total.dtype), codes, scales)
    if c["op"] == "linear":
        return _epilogue(s["x"].float() @ s["weight"].float().t(), s)
    x = s["codes"].view(torch.float8_e4m3fn).float() * s["scales"].repeat_interleave(128, 1)
    w = s["weight"].view(torch.float8_e4m3fn).float()
    if c["qkv"]:
        at, block = _qkv_rows(w.device)
        w = w[at] * s["weight_scale"][block].repeat_interleave(128, 1)
    else:
        w = w * s["weight_scale"].repeat_interleave(128, 0).repeat_interleave(128, 1)
    return _epilogue(x @ w.t(), s)


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    if case["op"] == "norm":
        n, z = case["rows"] * case["hidden"], SIZE[case["dtype"]]
        b = n * z * (3 if case["residual"] else 1) + 2 * case["hidden"]  # x, residual, sum; the weight
        b += n * z if case["y"] else 0
        b += n + 4 * case["rows"] * -(-case["hidden"] // 128) if case["codes"] else 0
        return {"bytes": b, "flops": 8 * n}
    width, rows, cols = case["width"], case["rows"], case["cols"]
    z = SIZE[case["out"]]
    b = width * rows * z * (2 if case["residual"] else 1) + (rows * z if case["bias"] else 0)
    if case["op"] == "linear":
        b += 2 * cols * (rows + width)
    else:
        b += cols * (rows + width) + 4 * (cols // 128) * (width + -(-rows // 128))
    return {"bytes": b, "flops": 2 * width * rows * cols}


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x = s["x"].double()
        out = {}
        if s["residual"] is not None:
            x = (x + s["residual"].double()).to(s["x"].dtype).double()  # the stream is kept in x's type
            out["sum"] = x
        rms = (x.square().sum(1) / case["hidden"] + EPS).sqrt()
        y = torch.einsum("rc,r,c->rc", x, 1.0 / rms, s["weight"].double())
        if case["y"]:
            out["y"] = y
        if case["codes"]:
            scales, codes = [], []
            for c0 in range(0, case["hidden"], 128):
                part = y[:, c0:c0 + 128]
                top = torch.maximum(part.max(1).values, (-part).max(1).values).clamp(min=1e-10) / 448
                scales.append(top)
                codes.append(part / top.unsqueeze(1))
            out["codes"], out["scales"] = torch.cat(codes, 1), torch.stack(scales, 1)
        return out
    width, rows, cols = case["width"], case["rows"], case["cols"]
    got = torch.empty((width, rows), dtype=torch.float64, device="cuda")
    if case["op"] == "linear":
        x = s["x"].double()
        for r in range(0, rows, 16384):
            got[:, r:r + 16384] = torch.einsum("tc,rc->tr", x, s["weight"][r:r + 16384].double())
    else:
        values = torch.arange(256, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).double()
        got.zero_()
        order = torch.arange(rows)
        block = order // 128
        if case["qkv"]:  # (shard, place in the shard) of Q, then K, then V
            parts = [(0, 3072), (3072, 192), (3264, 128)]
            order = torch.cat([h * 3392 + a + torch.arange(n) for a, n in parts for h in range(4)])
            block = torch.cat([h * 27 + torch.div(a, 128, rounding_mode="floor") + torch.arange(n) // 128
                               if a < 3264 else torch.full((n,), h * 27 + 26) for a, n in
                               [(torch.tensor(a), n) for a, n in parts] for h in range(4)])
        order, block = order.cuda(), block.cuda()
        for b in range(cols // 128):
            at = slice(128 * b, 128 * b + 128)
            x = values[s["codes"][:, at].long()] * s["scales"][:, b:b + 1].double()
            w = values[s["weight"][:, at][order].long()] * s["weight_scale"][block, b].double().unsqueeze(1)
            got += x @ w.t()
    if s["bias"] is not None:
        got += s["bias"].double()
    act = case["act"]
    if act == "relu":
        got = torch.where(got > 0, got, torch.zeros_like(got))
    elif act == "gelu":
        got = got * torch.special.ndtr(got)
    elif act == "gelu_tanh":
        # (1 + tanh(u)) / 2 = 1 / (1 + exp(-2 u))
        u = (got + 0.044715 * got ** 3) * (2.0 / math.pi) ** 0.5
        got = got / (1.0 + torch.exp(-2.0 * u))
    elif act == "silu":
        got = got * torch.sigmoid(got)
    if s["residual"] is not None:
        got += s["residual"].double()
    return got
