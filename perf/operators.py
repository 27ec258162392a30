"""Cases for the block-scaled fp8 and expert-grouped GEMM operators of k8s_gpu_monitor_amd.ops.diag.

Three operators that a mixture-of-experts training step or server runs one after the other:

quantize  x [rows, cols] (bf16 or f32) -> e4m3 values with one f32 scale per block of 128: a block is 128 consecutive
          elements of a row ("rows", activations and gradients) or 128 x 128 elements ("tiles", weights); with `transpose`
          the transposed matrix is what is laid out and blocked.
              amax = max |x| over the block, at least 2^-96;  scale = f32(amax / 448);  q = e4m3(f32(x * f32(448 / amax)))
gemm      C [m, n] = sum over blocks kb of sa[m, kb] * sb[n, kb] * sum over the 128 k of the block of A[m, k] * B[n, k];
          B's scales are per tile (forward, input gradient) or per row (weight gradient).
grouped   rows sorted by expert, expert e owning rows offsets[e] .. offsets[e + 1]; forward y[t] = W[e] x[t], bf16 or
          block-scaled fp8; backward (bf16) dx[t] = W[e]^T dy[t] and dW[e] = sum over its rows of dy[t] x[t]^T.

`own` chooses between the framework's kernels and the plain form in elementary torch operations.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
AMAX_MIN = 2.0 ** -96


def _up(x, to):
    return -(-x // to) * to


def listed():
    return [
        # one decode step of eight sequences: the activations on their way into an fp8 product; launch latency
        {"name": "quantize_decode", "kind": "quantize", "rows": 8, "cols": 7168, "dtype": "bf16", "blocks": "rows", "transpose": False},
        # a training batch's or a prefill's activations: memory bandwidth
        {"name": "quantize_activations", "kind": "quantize", "rows": 16384, "cols": 7168, "dtype": "bf16", "blocks": "rows", "transpose": False},
        # master weights for the input gradient's product, which contracts over their rows; sizes off the block grid
        {"name": "quantize_weights_t", "kind": "quantize", "rows": 8200, "cols": 4100, "dtype": "f32", "blocks": "tiles", "transpose": True},
        # one token through one projection: the weights are read once
        {"name": "gemm_one_token", "kind": "gemm", "m": 1, "n": 4096, "k": 7168, "b_blocks": "tiles", "out": "bf16"},
        # a short prompt; nothing a multiple of a tile, K ending inside a block
        {"name": "gemm_short_prompt", "kind": "gemm", "m": 203, "n": 4120, "k": 2064, "b_blocks": "tiles", "out": "bf16"},
        # training forward at the size the GEMM soak runs
        {"name": "gemm_training", "kind": "gemm", "m": 8192, "n": 8192, "k": 8192, "b_blocks": "tiles", "out": "bf16"},
        # weight gradient: both operands blocked along the tokens, f32 out for the optimizer
        {"name": "gemm_weight_gradient", "kind": "gemm", "m": 2048, "n": 7168, "k": 8192, "b_blocks": "rows", "out": "f32"},
        # a decode step of eight sequences, eight experts each, out of 64: the weights of the experts that were picked
        {"name": "grouped_decode", "kind": "grouped", "pass": "forward", "dtype": "bf16", "rows": 64, "used": 64, "groups": 64, "n": 2048, "k": 2048, "out": "bf16"},
        # the same with block-scaled fp8 weights
        {"name": "grouped_decode_fp8", "kind": "grouped", "pass": "forward", "dtype": "fp8", "rows": 72, "used": 69, "groups": 64, "n": 4096, "k": 7168, "out": "bf16"},
        # a training batch over 32 experts with uneven loads
        {"name": "grouped_training", "kind": "grouped", "pass": "forward", "dtype": "bf16", "rows": 32768, "used": 32768, "groups": 32, "n": 4096, "k": 2048, "out": "bf16"},
        # its backward pass: input and weight gradients
        {"name": "grouped_backward", "kind": "grouped", "pass": "backward", "dtype": "bf16", "rows": 16384, "used": 16001, "groups": 16, "n": 4096, "k": 2048, "out": "f32"},
        # a prefill through fp8 experts
        {"name": "grouped_prefill_fp8", "kind": "grouped", "pass": "forward", "dtype": "fp8", "rows": 16384, "used": 16161, "groups": 32, "n": 4096, "k": 7168, "out": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["quantize", "gemm", "grouped"])
    if kind == "quantize":
        return {"kind": kind, "rows": _log(rng, 1, 16384), "cols": _log(rng, 64, 7168), "dtype": rng.choice(["bf16", "f32"]),
                "blocks": rng.choice(["rows", "tiles"]), "transpose": rng.random() < 0.5}
    if kind == "gemm":
        return {"kind": kind, "m": _log(rng, 1, 8192), "n": 8 * _log(rng, 16, 1024), "k": 16 * _log(rng, 8, 512),
                "b_blocks": rng.choice(["tiles", "tiles", "rows"]), "out": rng.choice(["bf16", "f32"])}
    dtype, backward = rng.choice(["bf16", "fp8"]), False
    if dtype == "bf16":
        backward = rng.random() < 0.5
    rows, n, k = _log(rng, 1, 32768), 16 * _log(rng, 16, 256), 16 * _log(rng, 16, 256)
    while rows * n * k > 2.5e11:
        rows //= 2
    groups = _log(rng, 1, max(1, min(128, int(3e8 / (n * k)))))
    return {"kind": kind, "pass": "backward" if backward else "forward", "dtype": dtype, "rows": rows,
            "used": max(1, rows - rng.choice([0, 0, rows // 50])), "groups": groups, "n": n, "k": k,
            "out": rng.choice(["bf16", "f32"]) if backward else "bf16"}


# ------------------------------------------------------------------------------------------------------ inputs --
def _e4m3_blocks(x, blocks):
    """x [r, c] f32, c a multiple of 16 -> (e4m3 [r, c], scales): the formula at the head of the file."""
    r, c = x.shape
    cb = _up(c, BLOCK)
    rb = _up(r, BLOCK) if blocks == "tiles" else r
    p = torch.zeros(rb, cb, device=x.device)
    p[:r, :c] = x
    if blocks == "rows":
        amax = p.view(rb, cb // BLOCK, BLOCK).abs().amax(2).clamp_min(AMAX_MIN)
        inv = torch.full_like(amax, E4M3_MAX) / amax
        q = (p.view(rb, cb // BLOCK, BLOCK) * inv[:, :, None]).view(rb, cb)
        scales = (amax / torch.full_like(amax, E4M3_MAX)).t().contiguous()  # [blocks, rows]: a block's scales lie together
    else:
        v = p.view(rb // BLOCK, BLOCK, cb // BLOCK, BLOCK)
        amax = v.abs().amax(3).amax(1).clamp_min(AMAX_MIN)
        inv = torch.full_like(amax, E4M3_MAX) / amax
        q = (v * inv[:, None, :, None]).view(rb, cb)
        scales = (amax / torch.full_like(amax, E4M3_MAX)).contiguous()      # [row blocks, blocks]
    return q[:r, :c].to(torch.float8_e4m3fn).contiguous(), scales


def _activations(rows, cols, gen, dev):
    """Normal values with a few channels that are far larger, as layers' outputs have."""
    x = torch.randn(rows, cols, device=dev, generator=gen)
    big = torch.rand(cols, device=dev, generator=gen) < 0.01
    return x * torch.where(big, 20.0, 1.0)


def _weights(rows, cols, gen, dev):
    return torch.randn(rows, cols, device=dev, generator=gen) / math.sqrt(cols)


def _offsets(case, seed):
    """Uneven expert loads: some experts get several times the mean, some none."""
    r = np.random.RandomState(seed % (1 << 31))
    w = np.exp(0.7 * r.randn(case["groups"]))
    counts = r.multinomial(case["used"], w / w.sum())
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def _inputs(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    kind = case["kind"]
    if kind == "quantize":
        x = _activations(case["rows"], case["cols"], gen, dev)
        return {"x": x.bfloat16() if case["dtype"] == "bf16" else x}
    if kind == "gemm":
        a, sa = _e4m3_blocks(_activations(case["m"], case["k"], gen, dev), "rows")
        make = _activations if case["b_blocks"] == "rows" else _weights
        b, sb = _e4m3_blocks(make(case["n"], case["k"], gen, dev), case["b_blocks"])
        return {"a": a, "sa": sa, "b": b, "sb": sb}
    rows, g, n, k = case["rows"], case["groups"], case["n"], case["k"]
    at = _offsets(case, seed)
    s = {"at": at.tolist(), "offsets": torch.from_numpy(at).to(dev)}
    x = _activations(rows, k, gen, dev)
    if case["dtype"] == "fp8":
        s["x"], s["sx"] = _e4m3_blocks(x, "rows")
        s["w"] = torch.empty(g, n, k, dtype=torch.float8_e4m3fn, device=dev)
        s["sw"] = torch.empty(g, _up(n, BLOCK) // BLOCK, _up(k, BLOCK) // BLOCK, device=dev)
        for e in range(g):
            s["w"][e], s["sw"][e] = _e4m3_blocks(_weights(n, k, gen, dev), "tiles")
        return s
    s["x"] = x.bfloat16()
    s["w"] = torch.empty(g, n, k, dtype=torch.bfloat16, device=dev)
    for e in range(g):
        s["w"][e] = _weights(n, k, gen, dev)
    if case["pass"] == "backward":
        s["dy"] = _activations(rows, n, gen, dev).bfloat16()
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    dev = torch.device("cuda")
    out = {"bf16": torch.bfloat16, "f32": torch.float32}
    kind = case["kind"]
    if not own:
        return s
    from k8s_gpu_monitor_amd.ops import diag  # the outputs are buffers that the program keeps
    s["diag"] = diag
    if kind == "quantize":
        r, c = (case["cols"], case["rows"]) if case["transpose"] else (case["rows"], case["cols"])
        s["q"] = torch.zeros(r, _up(c, 16), dtype=torch.float8_e4m3fn, device=dev)
        kb = _up(c, BLOCK) // BLOCK
        s["scales"] = torch.zeros((kb, r) if case["blocks"] == "rows" else (_up(r, BLOCK) // BLOCK, kb), device=dev)
    elif kind == "gemm":
        s["c"] = torch.zeros(case["m"], case["n"], dtype=out[case["out"]], device=dev)
    elif case["pass"] == "forward":
        s["y"] = torch.zeros(case["rows"], case["n"], dtype=torch.bfloat16, device=dev)
    else:
        s["dx"] = torch.zeros(case["rows"], case["k"], dtype=torch.bfloat16, device=dev)
        s["dw"] = torch.zeros(case["groups"], case["n"], case["k"], dtype=out[case["out"]], device=dev)
    return s


# --------------------------------------------------------------------------------------------------- one pass --
def _run_own(s):
    case, diag = s["case"], s["diag"]
    stream = torch.cuda.current_stream().cuda_stream
    kind = case["kind"]
    if kind == "quantize":
        diag.block_quantize_launch(s["x"].data_ptr(), s["q"].data_ptr(), s["scales"].data_ptr(), case["rows"], case["cols"],
                                   dtype=case["dtype"], blocks=case["blocks"], transpose=case["transpose"], stream=stream)
        return {"q": s["q"], "scales": s["scales"]}
    if kind == "gemm":
        diag.gemm_block_launch(s["a"].data_ptr(), s["sa"].data_ptr(), s["b"].data_ptr(), s["sb"].data_ptr(), s["c"].data_ptr(),
                               case["m"], case["n"], case["k"], b_blocks=case["b_blocks"], out=case["out"], stream=stream)
        return {"c": s["c"]}
    shape = (s["offsets"].data_ptr(), case["groups"], case["rows"], case["n"], case["k"])
    if case["pass"] == "forward":
        scales = {"scale_a": s["sx"].data_ptr(), "scale_b": s["sw"].data_ptr()} if case["dtype"] == "fp8" else {}
        diag.grouped_gemm_launch("forward", case["dtype"], s["x"].data_ptr(), s["w"].data_ptr(), s["y"].data_ptr(), *shape, stream=stream, **scales)
        return {"y": s["y"]}
    diag.grouped_gemm_launch("dgrad", "bf16", s["dy"].data_ptr(), s["w"].data_ptr(), s["dx"].data_ptr(), *shape, stream=stream)
    diag.grouped_gemm_launch("wgrad", "bf16", s["dy"].data_ptr(), s["x"].data_ptr(), s["dw"].data_ptr(), *shape, out=case["out"], stream=stream)
    return {"dx": s["dx"], "dw": s["dw"]}


def _values(q, scales, blocks):
    """The f32 values that block-scaled e4m3 stands for."""
    r, c = q.shape
    if blocks == "rows":
        return q.float() * scales.t().repeat_interleave(BLOCK, 1)[:, :c]
    return q.float() * scales.repeat_interleave(BLOCK, 0)[:r].repeat_interleave(BLOCK, 1)[:, :c]


def _run_plain(s):
    case = s["case"]
    kind = case["kind"]
    out = {"bf16": torch.bfloat16, "f32": torch.float32}
    if kind == "quantize":
        x = s["x"].float()
        x = x.t() if case["transpose"] else x
        p = torch.zeros(x.shape[0], _up(x.shape[1], 16), device=x.device)
        p[:, :x.shape[1]] = x
        q, scales = _e4m3_blocks(p, case["blocks"])
        return {"q": q, "scales": scales}
    if kind == "gemm":
        c = _values(s["a"], s["sa"], "rows") @ _values(s["b"], s["sb"], case["b_blocks"]).t()
        return {"c": c.to(out[case["out"]])}
    rows, g, n, k = case["rows"], case["groups"], case["n"], case["k"]
    dev = s["x"].device
    at = s["at"]
    if case["pass"] == "forward":
        y = torch.zeros(rows, n, dtype=torch.bfloat16, device=dev)
        x = _values(s["x"], s["sx"], "rows") if case["dtype"] == "fp8" else s["x"].float()
        for e in range(g):
            if at[e + 1] > at[e]:
                w = _values(s["w"][e], s["sw"][e], "tiles") if case["dtype"] == "fp8" else s["w"][e].float()
                y[at[e]:at[e + 1]] = (x[at[e]:at[e + 1]] @ w.t()).bfloat16()
        return {"y": y}
    dx = torch.zeros(rows, k, dtype=torch.bfloat16, device=dev)
    dw = torch.zeros(g, n, k, dtype=out[case["out"]], device=dev)
    x, dy = s["x"].float(), s["dy"].float()
    for e in range(g):
        if at[e + 1] > at[e]:
            i = slice(at[e], at[e + 1])
            dx[i] = (dy[i] @ s["w"][e].float()).bfloat16()
            dw[e] = dy[i].t().contiguous() @ x[i]
    return {"dx": dx, "dw": dw}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------------- work --
def work(case):
    kind = case["kind"]
    size = {"bf16": 2, "f32": 4, "fp8": 1}
    if kind == "quantize":
        r, c = (case["cols"], case["rows"]) if case["transpose"] else (case["rows"], case["cols"])
        blocks = _up(c, BLOCK) // BLOCK * (r if case["blocks"] == "rows" else _up(r, BLOCK) // BLOCK)
        return {"bytes": r * c * size[case["dtype"]] + r * _up(c, 16) + 4 * blocks, "flops": 2 * r * c}
    if kind == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        kb = _up(k, BLOCK) // BLOCK
        sb = kb * (n if case["b_blocks"] == "rows" else _up(n, BLOCK) // BLOCK)
        return {"bytes": (m + n) * k + 4 * (m * kb + sb) + m * n * size[case["out"]], "flops": 2 * m * n * k}
    t, g, n, k = case["used"], case["groups"], case["n"], case["k"]
    active = g * (1 - (1 - 1 / g) ** t)  # experts with a row, were the loads even
    if case["pass"] == "forward":
        e = size[case["dtype"]]
        scales = 4 * _up(k, BLOCK) // BLOCK * (t + active * _up(n, BLOCK) // BLOCK) if case["dtype"] == "fp8" else 0
        return {"bytes": int(e * (t * k + active * n * k) + scales + 2 * t * n), "flops": 2 * t * n * k}
    return {"bytes": int(2 * t * (n + k) + 2 * active * n * k + 2 * t * k + 2 * t * (n + k) + g * n * k * size[case["out"]]),
            "flops": 4 * t * n * k}


# ------------------------------------------------------------------------------------------------------ exact --
def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        x = s["x"].double()
        if case["transpose"]:
            x = x.t()
        r, c = x.shape
        kb = _up(c, BLOCK) // BLOCK
        tall = 1 if case["blocks"] == "rows" else BLOCK
        q = torch.zeros(r, _up(c, 16), dtype=torch.float64, device=x.device)
        scales = torch.zeros(-(-r // tall), kb, dtype=torch.float64, device=x.device)
        for j in range(kb):
            part = x[:, j * BLOCK:(j + 1) * BLOCK]
            top = part.abs().max(dim=1).values
            if tall > 1:
                pad = torch.zeros(_up(r, tall), dtype=torch.float64, device=x.device)
                pad[:r] = top
                top = pad.view(-1, tall).max(dim=1).values
            top = torch.clamp(top, min=AMAX_MIN)
            scales[:, j] = top / E4M3_MAX
            # the definition holds 448 / amax and the product to 24 bits; both are exact in 64 before that rounding
            factor = (E4M3_MAX / top).float().double().repeat_interleave(tall)[:r]
            y = (part * factor[:, None]).float().double()
            # e4m3: four significant bits down to 2^-6, steps of 2^-9 below; ties to the even step
            step = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.clamp(y.abs(), min=2.0 ** -20))), min=-6) - 3)
            q[:, j * BLOCK:j * BLOCK + part.shape[1]] = torch.clamp(torch.round(y / step) * step, -E4M3_MAX, E4M3_MAX)
        return {"q": q, "scales": scales.t().contiguous() if case["blocks"] == "rows" else scales}

    def wide(q, scales, blocks):
        v = q.double()
        for j in range(0, v.shape[1], BLOCK):
            if blocks == "rows":
                v[:, j:j + BLOCK] *= scales[j // BLOCK].double()[:, None]
            else:
                for i in range(0, v.shape[0], BLOCK):
                    v[i:i + BLOCK, j:j + BLOCK] *= scales[i // BLOCK, j // BLOCK].double()
        return v

    if kind == "gemm":
        return {"c": torch.mm(wide(s["a"], s["sa"], "rows"), wide(s["b"], s["sb"], case["b_blocks"]).t())}
    at, fp8 = s["at"], case["dtype"] == "fp8"
    x = wide(s["x"], s["sx"], "rows") if fp8 else s["x"].double()
    if case["pass"] == "forward":
        y = torch.zeros(case["rows"], case["n"], dtype=torch.float64, device=x.device)
        for e, (lo, hi) in enumerate(zip(at, at[1:])):
            if hi > lo:
                w = wide(s["w"][e], s["sw"][e], "tiles") if fp8 else s["w"][e].double()
                y[lo:hi] = torch.mm(x[lo:hi], w.t())
        return {"y": y}
    dy = s["dy"].double()
    dx = torch.zeros(case["rows"], case["k"], dtype=torch.float64, device=x.device)
    dw = torch.zeros(case["groups"], case["n"], case["k"], dtype=torch.float64, device=x.device)
    for e, (lo, hi) in enumerate(zip(at, at[1:])):
        if hi > lo:
            torch.mm(dy[lo:hi], s["w"][e].double(), out=dx[lo:hi])
            dw[e] = torch.mm(dy[lo:hi].t(), x[lo:hi])
    return {"dx": dx, "dw": dw}
