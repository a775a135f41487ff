"""The 8-bit expert layer's operators as cases that can be timed and compared: quantising to 8-bit floating point with
a scale for each block of 128, the matrix products on such operands (dense, per expert, one token, and both
directions of a training step), and the router's balance loss with its per-expert counts and gradient.

Each case has a plain form in elementary torch operations (`own` false) and the calls of libtextsift_cuda's entry
points (`own` true), on the same inputs.

The 8-bit format.  A row is cut into blocks of 128 values.  A block's scale is s = max(a / 448, 2^-100), a the largest
finite magnitude in it.  The scale is stored in 32 bits, as a times the f32 nearest 1/448, and r is the f32 nearest its
reciprocal: the codes are e4m3(f32(x r)), rounded to nearest even and clamped to +-448.  (These three roundings belong
to the format: x / s often lies halfway between two codes.)  Weights have one scale for each block of 128 rows by 128
columns.
"""
import math

import torch

own = False

BLOCK = 128
SMALLEST = 2.0 ** -100  # a block of zeros has this scale
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
CODES = {"f16": 1, "f32": 2, "bf16": 4}  # the library's TS_DTYPE_* of each


def _up(n, m):
    return -(-n // m) * m


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one token's hidden state before a projection: the smallest call, all latency
        {"name": "quant_token", "op": "quant", "rows": 1, "cols": 640, "dtype": "f16", "transpose": False},
        # the hidden states of a full packed forward (65,536 tokens of 640)
        {"name": "quant_packed", "op": "quant", "rows": 65536, "cols": 640, "dtype": "f16", "transpose": False},
        # a weight gradient's operand: blocks run along the tokens, whose number is odd
        {"name": "quant_columns", "op": "quant", "rows": 16391, "cols": 1280, "dtype": "bf16", "transpose": True},
        # one token through a square projection: the weight is read once
        {"name": "mm_token", "op": "matvec", "m": 1, "n": 4096, "k": 4096, "dtype": "f16"},
        # the fused Q/K/V projection of a full packed forward, with bias
        {"name": "mm_qkv", "op": "matmul", "m": 65536, "n": 1152, "k": 640, "bias": True, "dtype": "f16"},
        # a short document through a layer whose sizes fit no tile
        {"name": "mm_odd", "op": "matmul", "m": 517, "n": 1001, "k": 1500, "bias": True, "dtype": "bf16"},
        # a large square product
        {"name": "mm_square", "op": "matmul", "m": 8192, "n": 8192, "k": 8192, "bias": False, "dtype": "bf16"},
        # the gate and up products of 128 experts over the four routes of each of 65,536 tokens, unevenly spread
        {"name": "mm_experts", "op": "experts", "m": 262144, "n": 1280, "k": 640, "e": 128, "dtype": "f16"},
        # the gradient of a layer's input: the output's gradient is quantised, then multiplied with the weight
        {"name": "grad_input", "op": "dx", "m": 16384, "n": 2048, "k": 2048, "dtype": "bf16"},
        # the gradient of an expert's weight from an odd number of tokens: both operands quantised along them
        {"name": "grad_weight", "op": "dw", "m": 16391, "n": 1280, "k": 640, "dtype": "bf16"},
        # the router's balance over one short document
        {"name": "balance_document", "op": "balance", "tokens": 80, "seqs": 1, "e": 128, "k": 4, "dtype": "f32"},
        # the router's balance over the documents of a full packed forward, each for itself
        {"name": "balance_packed", "op": "balance", "tokens": 65536, "seqs": 44, "e": 128, "k": 4, "dtype": "f32"},
    ]


def _between(rng, lo, hi):
    """A whole number from lo to hi, evenly spread over its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["quant", "quant", "matvec", "matmul", "matmul", "experts", "dx", "dw", "balance", "balance"])
    dtype = rng.choice(["f16", "bf16", "f32"])
    if op == "quant":
        rows, cols = _between(rng, 1, 65536), _between(rng, 16, 8192)
        while rows * cols > 65536 * 1280:
            rows = max(1, rows // 3)
        return {"op": op, "rows": rows, "cols": cols, "dtype": dtype, "transpose": rng.random() < 0.4}
    if op == "matvec":
        return {"op": op, "m": _between(rng, 1, 16), "n": _between(rng, 16, 8192), "k": _between(rng, 16, 8192),
                "dtype": dtype}
    if op == "balance":
        tokens = _between(rng, 1, 65536)
        e = _between(rng, 2, 256)
        return {"op": op, "tokens": tokens, "seqs": min(tokens, _between(rng, 1, 256)), "e": e,
                "k": rng.randint(1, min(e, 8)), "dtype": dtype}
    n, k = _between(rng, 16, 8192), _between(rng, 16, 8192)
    m = _between(rng, 1, 65536)
    if op == "experts":
        e = _between(rng, 1, 128)
        n, k = _between(rng, 16, 2048), _between(rng, 16, 2048)
        while m * max(n, k) > 65536 * 1280:
            m = max(1, m // 3)
        return {"op": op, "m": m, "n": n, "k": k, "e": e, "dtype": dtype}
    while m * n * k > 2 ** 36 or m * max(n, k) > 2 ** 26:
        m = max(1, m // 3)
        n, k = max(16, n * 2 // 3), max(16, k * 2 // 3)
    if op == "matmul":
        return {"op": op, "m": m, "n": n, "k": k, "bias": rng.random() < 0.5, "dtype": dtype}
    return {"op": op, "m": m, "n": n, "k": k, "dtype": dtype}


# ---------------------------------------------------------------------------
# The plain forms' pieces, in 32 bits
# ---------------------------------------------------------------------------

def _e4m3(v):
    return v.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def _pad_blocks(v):
    """The last dimension filled up with zeros to whole blocks."""
    cols = v.shape[-1]
    full = torch.zeros(v.shape[:-1] + (_up(cols, BLOCK),), dtype=v.dtype, device=v.device)
    full[..., :cols] = v
    return full


def _quant_rows(x):
    """x [rows, cols], any type -> codes [rows, cols] (e4m3), scales [blocks, rows] (f32)."""
    rows, cols = x.shape
    v = _pad_blocks(x.float()).view(rows, -1, BLOCK)
    a = torch.where(v.isfinite(), v.abs(), torch.zeros_like(v)).amax(-1)
    s = (a * (1.0 / 448.0)).clamp_min(SMALLEST)
    inv = torch.ones_like(s) / s
    codes = _e4m3(v * inv[:, :, None]).view(rows, -1)[:, :cols]
    return codes, s.t()


def _quant_weight(w):
    """w f32 [E, N, K] -> codes [E, N, K], scales [E, N blocks, K blocks]."""
    e, n, k = w.shape
    full = torch.zeros(e, _up(n, BLOCK), _up(k, BLOCK), device=w.device)
    full[:, :n, :k] = w
    v = full.view(e, -1, BLOCK, full.shape[2] // BLOCK, BLOCK)
    s = (v.abs().amax((2, 4)) * (1.0 / 448.0)).clamp_min(SMALLEST)
    codes = _e4m3(v / s[:, :, None, :, None]).view(e, full.shape[1], full.shape[2])[:, :n, :k]
    return codes, s


def _rows_back(codes, scales):
    """f32 values of codes [rows, cols] with scales [blocks, rows]."""
    return codes.float() * scales.t().repeat_interleave(BLOCK, 1)[:, :codes.shape[1]]


def _weight_back(codes, scales):
    """f32 values of codes [N, K] with scales [N blocks, K blocks]."""
    n, k = codes.shape
    return codes.float() * scales.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _activations(g, rows, cols, dtype):
    """Hidden states: each row with a size of its own and a few channels that stand out."""
    x = torch.randn(rows, cols, device="cuda", generator=g)
    x *= torch.exp(0.5 * torch.randn(rows, 1, device="cuda", generator=g))
    x *= torch.where(torch.rand(1, cols, device="cuda", generator=g) < 0.01, 12.0, 1.0)
    return x.to(dtype)


def _pitched(codes):
    """codes [..., cols] as bytes with rows that start at multiples of 16 bytes, as the products take them."""
    cols = codes.shape[-1]
    full = torch.zeros(codes.shape[:-1] + (_up(cols, 16),), dtype=torch.uint8, device=codes.device)
    full[..., :cols] = codes.view(torch.uint8)
    return full


def _operand(g, rows, cols):
    """A quantised operand as a layer before has left it: bytes [rows, pitch], scales [blocks, rows rounded up to 4]."""
    codes, scales = _quant_rows(_activations(g, rows, cols, torch.float16))
    s = torch.zeros(scales.shape[0], _up(rows, 4), device="cuda")
    s[:, :rows] = scales
    return _pitched(codes), s


def _weights(g, e, n, k):
    """Expert weights: bytes [e, n, pitch], scales [e, n blocks, k blocks]."""
    codes, scales = _quant_weight(torch.randn(e, n, k, device="cuda", generator=g) * (1.0 / math.sqrt(k)))
    return _pitched(codes), scales.contiguous()


def _f8(raw, cols):
    return raw.view(torch.float8_e4m3fn)[..., :cols]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, dt = case["op"], DTYPES[case["dtype"]]
    st = {"case": case, "op": op, "dt": dt, "code": CODES[case["dtype"]],
          "stream": torch.cuda.current_stream().cuda_stream}
    empty = lambda *shape, dtype=torch.float32: torch.empty(*shape, dtype=dtype, device="cuda")  # noqa: E731
    if op == "quant":
        rows, cols = case["rows"], case["cols"]
        st["x"] = _activations(g, rows, cols, dt)
        out_rows, out_cols = (cols, rows) if case["transpose"] else (rows, cols)
        st["codes"] = empty(out_rows, _up(out_cols, 16), dtype=torch.uint8)
        st["scales"] = empty(_up(out_cols, BLOCK) // BLOCK, _up(out_rows, 4))
    elif op == "balance":
        t, e, k, s = case["tokens"], case["e"], case["k"], case["seqs"]
        # some experts are liked more than others, and the last tokens of some documents are padding
        logits = torch.randn(t, e, device="cuda", generator=g) * 1.5 + torch.randn(e, device="cuda", generator=g) * 0.7
        st["logits"] = logits.to(dt)
        st["idx"] = st["logits"].float().topk(k, dim=1).indices.to(torch.int32).contiguous()
        cuts = (torch.randperm(t - 1, device="cuda", generator=g)[: s - 1] + 1).sort().values
        st["seq"] = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), t)]).to(torch.int32)
        place = torch.rand(t, device="cuda", generator=g)
        st["mask"] = (place < 0.95).to(torch.uint8)
        st["counts"], st["prob"], st["loss"] = empty(s, e, dtype=torch.int32), empty(s, e), empty(1)
        st["grad"] = empty(t, e, dtype=dt)
        # a loss scale that keeps an fp16 gradient in range, as a training loop has it
        st["alpha"], st["grad_scale"] = 0.01, 65536.0
        st["work"] = empty(_balance_work(s, e), dtype=torch.uint8)
    else:
        m, n, k = case["m"], case["n"], case["k"]
        if op == "dw":
            st["dy"], st["x"] = _activations(g, m, n, dt), _activations(g, m, k, dt)
            pitch, blocks = _up(m, 16), _up(m, BLOCK) // BLOCK
            st["dyt"], st["xt"] = empty(n, pitch, dtype=torch.uint8), empty(k, pitch, dtype=torch.uint8)
            st["dys"], st["xs"] = empty(blocks, _up(n, 4)), empty(blocks, _up(k, 4))
            st["out"] = empty(n, k)
        elif op == "dx":
            st["dy"] = _activations(g, m, n, dt)
            # the weight [n, k] laid out by its columns once, for the products with it from the other side
            w, ws = _weights(g, 1, n, k)
            st["w"] = _pitched(_f8(w, k)[0].view(torch.uint8).t().contiguous())[None]
            st["ws"] = ws.transpose(1, 2).contiguous()
            st["dyc"], st["dys"] = empty(m, _up(n, 16), dtype=torch.uint8), empty(_up(n, BLOCK) // BLOCK, _up(m, 4))
            st["out"] = empty(m, k, dtype=dt)
        else:
            e = case.get("e", 1)
            st["w"], st["ws"] = _weights(g, e, n, k)
            st["bias"] = (torch.randn(e, n, device="cuda", generator=g) * 0.1).half() if case.get("bias") else None
            if op == "matvec":
                st["x"] = _activations(g, m, k, dt)
            else:
                st["a"], st["as"] = _operand(g, m, k)
            if op == "experts":
                like = (torch.arange(1, e + 1, device="cuda").float() ** -0.5)
                like = like[torch.randperm(e, device="cuda", generator=g)]
                like[torch.rand(e, device="cuda", generator=g) < 0.03] = 0  # experts that no token chose
                like[0] += 1e-3
                picks = torch.multinomial(like, m, replacement=True, generator=g)
                sizes = torch.zeros(e, dtype=torch.int64, device="cuda").scatter_add_(0, picks, torch.ones_like(picks))
                st["seg"] = torch.cat([sizes.new_zeros(1), sizes.cumsum(0)]).to(torch.int32)
                st["ends"] = st["seg"].tolist()
            st["out"] = empty(m, n, dtype=dt)
    return st


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_plain(st):
    op, dt, case = st["op"], st["dt"], st["case"]
    if op == "quant":
        codes, scales = _quant_rows(st["x"].t() if case["transpose"] else st["x"])
        return {"codes": codes, "scales": scales}
    if op == "balance":
        return _balance_plain(st)
    if op == "dw":
        dy, dys = _quant_rows(st["dy"].t())
        x, xs = _quant_rows(st["x"].t())
        return {"dw": _rows_back(dy, dys) @ _rows_back(x, xs).t()}
    if op == "dx":
        dy, dys = _quant_rows(st["dy"])
        return {"dx": (_rows_back(dy, dys) @ _weight_back(_f8(st["w"][0], case["n"]), st["ws"][0]).t()).to(dt)}
    n, k = case["n"], case["k"]
    if op == "matvec":
        x, xs = _quant_rows(st["x"])
        return {"y": (_rows_back(x, xs) @ _weight_back(_f8(st["w"][0], k), st["ws"][0]).t()).to(dt)}
    a = _rows_back(_f8(st["a"], k), st["as"][:, :case["m"]])
    if op == "experts":
        ends = st["ends"]
        y = torch.empty(case["m"], n, device="cuda")
        for e in range(case["e"]):
            y[ends[e]:ends[e + 1]] = a[ends[e]:ends[e + 1]] @ _weight_back(_f8(st["w"][e], k), st["ws"][e]).t()
        return {"y": y.to(dt)}
    y = a @ _weight_back(_f8(st["w"][0], k), st["ws"][0]).t()
    if st["bias"] is not None:
        y = y + st["bias"].float()
    return {"y": y.to(dt)}


def _balance_plain(st):
    case = st["case"]
    t, e, k, s = case["tokens"], case["e"], case["k"], case["seqs"]
    z = st["logits"].float()
    z = (z - z.amax(1, keepdim=True)).exp()
    p = z / z.sum(1, keepdim=True)
    at = torch.arange(t, device=z.device)
    of = (at[:, None] >= st["seq"][None, 1:-1]).sum(1)  # the document of each token
    live = st["mask"].long()
    counts = torch.zeros(s * e, dtype=torch.int64, device=z.device)
    counts.scatter_add_(0, (of[:, None] * e + st["idx"]).view(-1), live[:, None].expand(t, k).reshape(-1))
    counts = counts.view(s, e)
    tokens = torch.zeros(s, dtype=torch.int64, device=z.device).scatter_add_(0, of, live)
    member = ((of[None] == torch.arange(s, device=z.device)[:, None]) & (live[None] > 0)).float()  # [s, t]
    inv = 1.0 / tokens.clamp_min(1).float()
    prob = (member @ p) * inv[:, None]
    share = counts.float() * (inv * (e / k))[:, None]
    docs = (tokens > 0).sum().clamp_min(1).float()
    loss = (st["alpha"] / docs) * (share * prob).sum()
    c = share[of]
    grad = p * (c - (p * c).sum(1, keepdim=True)) * (st["grad_scale"] * st["alpha"] / docs)
    grad = grad * (live.float() * inv[of])[:, None]
    return {"counts": counts.int(), "prob": prob, "loss": loss.view(1), "grad": grad.to(st["dt"])}


def _balance_work(seqs, experts):
    """Bytes of scratch: the accumulators of seqs x experts sums and each sequence's length."""
    return 16 * seqs * (experts + 2) + 256


def _run_own(st):
    from textsift_b200 import abi
    lib = abi.lib()
    op, case, stream = st["op"], st["case"], st["stream"]
    if op == "quant":
        x, codes, scales = st["x"], st["codes"], st["scales"]
        abi.check(lib.ts_cuda_op_quant_fp8(
            x.data_ptr(), st["code"], x.stride(0), x.shape[0], x.shape[1], int(case["transpose"]), codes.data_ptr(),
            codes.stride(0), scales.data_ptr(), scales.stride(0), stream))
        shape = x.shape[::-1] if case["transpose"] else x.shape
        return {"codes": _f8(codes, shape[1]), "scales": scales[:, :shape[0]]}
    if op == "balance":
        abi.check(lib.ts_cuda_op_router_balance(
            st["logits"].data_ptr(), st["code"], case["e"], st["idx"].data_ptr(), st["mask"].data_ptr(),
            st["seq"].data_ptr(), case["seqs"], case["tokens"], case["e"], case["k"], st["alpha"], st["grad_scale"],
            st["counts"].data_ptr(), st["prob"].data_ptr(), st["loss"].data_ptr(), st["grad"].data_ptr(), case["e"],
            st["work"].data_ptr(), st["work"].numel(), stream))
        return {"counts": st["counts"], "prob": st["prob"], "loss": st["loss"], "grad": st["grad"]}
    m, n, k = case["m"], case["n"], case["k"]
    if op == "dw":
        for x, codes, scales in ((st["dy"], st["dyt"], st["dys"]), (st["x"], st["xt"], st["xs"])):
            abi.check(lib.ts_cuda_op_quant_fp8(
                x.data_ptr(), st["code"], x.stride(0), x.shape[0], x.shape[1], 1, codes.data_ptr(), codes.stride(0),
                scales.data_ptr(), scales.stride(0), stream))
        # dW [n, k] = dY^T X: the tokens are the axis that is summed, and both operands have a scale for each row
        abi.check(lib.ts_cuda_op_matmul_fp8(
            st["dyt"].data_ptr(), st["dyt"].stride(0), st["dys"].data_ptr(), st["dys"].stride(0),
            st["xt"].data_ptr(), st["xt"].stride(0), st["xs"].data_ptr(), st["xs"].stride(0), 1, None, None, 1,
            st["out"].data_ptr(), CODES["f32"], k, 0, n, k, m, stream))
        return {"dw": st["out"]}
    w, ws, out = st["w"], st["ws"], st["out"]
    if op == "matvec":
        abi.check(lib.ts_cuda_op_matvec_fp8(
            st["x"].data_ptr(), st["code"], k, w.data_ptr(), w.stride(1), ws.data_ptr(), None, out.data_ptr(),
            st["code"], n, m, n, k, stream))
        return {"y": out}
    if op == "dx":
        dy, codes, scales = st["dy"], st["dyc"], st["dys"]
        abi.check(lib.ts_cuda_op_quant_fp8(
            dy.data_ptr(), st["code"], n, m, n, 0, codes.data_ptr(), codes.stride(0), scales.data_ptr(),
            scales.stride(0), stream))
        abi.check(lib.ts_cuda_op_matmul_fp8(
            codes.data_ptr(), codes.stride(0), scales.data_ptr(), scales.stride(0), w.data_ptr(), w.stride(1),
            ws.data_ptr(), 0, BLOCK, None, None, 1, out.data_ptr(), st["code"], k, 0, m, k, n, stream))
        return {"dx": out}
    abi.check(lib.ts_cuda_op_matmul_fp8(
        st["a"].data_ptr(), st["a"].stride(0), st["as"].data_ptr(), st["as"].stride(0), w.data_ptr(), w.stride(1),
        ws.data_ptr(), 0, BLOCK, None if st["bias"] is None else st["bias"].data_ptr(),
        st["seg"].data_ptr() if op == "experts" else None, case.get("e", 1), out.data_ptr(), st["code"], n, 0, m, n,
        k, stream))
    return {"y": out}


# ---------------------------------------------------------------------------
# Bytes and operations that a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    op, b = case["op"], DTYPES[case["dtype"]].itemsize
    blocks = lambda v: _up(v, BLOCK) // BLOCK  # noqa: E731
    if op == "quant":
        r, c = case["rows"], case["cols"]
        long, short = (r, c) if case["transpose"] else (c, r)
        return {"bytes": r * c * (b + 1) + 4 * blocks(long) * short, "flops": 3 * r * c}
    if op == "balance":
        t, e, k, s = case["tokens"], case["e"], case["k"], case["seqs"]
        return {"bytes": 2 * t * e * b + t * (4 * k + 1) + 8 * s * e, "flops": 9 * t * e}
    m, n, k = case["m"], case["n"], case["k"]
    flops = 2 * m * n * k
    if op == "dw":
        return {"bytes": m * (n + k) * b + 4 * n * k, "flops": flops}
    weight = case.get("e", 1) * (n * k + 4 * blocks(n) * blocks(k))
    if op == "dx":
        return {"bytes": m * (n + k) * b + weight, "flops": flops}
    if op == "matvec":
        return {"bytes": m * (n + k) * b + weight, "flops": flops}
    return {"bytes": m * k + 4 * m * blocks(k) + weight + m * n * b, "flops": flops}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_e4m3(v):
    """The nearest e4m3 value of each v (f64), ties to the even one: steps of 2^(e-3), e at least -6, at most 448."""
    mag = v.abs().clamp(min=2.0 ** -60)
    step = torch.exp2(torch.floor(torch.log2(mag)).clamp(min=-6) - 3)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def _exact_rows(x):
    """Quantised values (without their scales) and the scales [rows, blocks] of x [rows, cols], in f64 but for the
    format's roundings to 32 bits."""
    x = x.double()
    rows, cols = x.shape
    parts = [x[:, b:b + BLOCK] for b in range(0, cols, BLOCK)]
    most = torch.stack([p.abs().max(1).values for p in parts], 1)
    per448 = torch.tensor(1.0 / 448.0, dtype=torch.float32, device=x.device).double()
    s = (most * per448).float().double().clamp(min=SMALLEST)
    r = (1.0 / s).float().double()
    q = torch.cat([_exact_e4m3((p * r[:, i:i + 1]).float().double()) for i, p in enumerate(parts)], 1)
    return q, s


def _spread(s, dim, size):
    at = torch.arange(size, device=s.device) // BLOCK
    return s.double().index_select(dim, at)


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "quant":
        q, s = _exact_rows(st["x"].t() if case["transpose"] else st["x"])
        return {"codes": q, "scales": s.t()}
    if op == "balance":
        return _balance_exact(st)
    m, n, k = case["m"], case["n"], case["k"]
    if op == "dw":
        (dy, dys), (x, xs) = _exact_rows(st["dy"].t()), _exact_rows(st["x"].t())
        return {"dw": (dy * _spread(dys, 1, m)) @ (x * _spread(xs, 1, m)).t()}
    if op == "dx":
        dy, dys = _exact_rows(st["dy"])
        w = _f8(st["w"][0], n).double() * _spread(_spread(st["ws"][0], 0, k), 1, n)
        return {"dx": (dy * _spread(dys, 1, n)) @ w.t()}
    if op == "matvec":
        x, xs = _exact_rows(st["x"])
        a = x * _spread(xs, 1, k)
    else:
        a = _f8(st["a"], k).double() * _spread(st["as"][:, :m].t(), 1, k)
    ends = st["ends"] if op == "experts" else [0, m]
    y = torch.zeros(m, n, dtype=torch.float64, device="cuda")
    for e in range(len(ends) - 1):
        w = _f8(st["w"][e], k).double() * _spread(_spread(st["ws"][e], 0, n), 1, k)
        y[ends[e]:ends[e + 1]] = torch.einsum("mk,nk->mn", a[ends[e]:ends[e + 1]], w)
    if st.get("bias") is not None:
        y += st["bias"].double()
    return {"y": y}


def _balance_exact(st):
    case = st["case"]
    e, k, ends = case["e"], case["k"], st["seq"].tolist()
    p = torch.softmax(st["logits"].double(), 1)
    live = st["mask"].bool()
    docs = [live[a:b] for a, b in zip(ends, ends[1:])]
    used = max(1, sum(bool(d.any()) for d in docs))
    grad, prob, loss = torch.zeros_like(p), [], torch.zeros(1, dtype=torch.float64, device=p.device)
    for (a, b), d in zip(zip(ends, ends[1:]), docs):
        tokens = max(1, int(d.sum()))
        f = torch.bincount(st["idx"][a:b][d].flatten().long(), minlength=e).double() * e / (k * tokens)
        mean = p[a:b][d].sum(0) / tokens
        prob.append(mean)
        loss += st["alpha"] / used * (f * mean).sum()
        g = p[a:b] * (f - (p[a:b] @ f)[:, None]) * (st["grad_scale"] * st["alpha"] / (used * tokens))
        grad[a:b] = g * d[:, None]
    return {"counts": None, "prob": torch.stack(prob), "loss": loss, "grad": grad}
