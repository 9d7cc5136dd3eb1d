"""Measured cases of the block-scaled 8-bit linear layers and of the linear layers grouped by expert.

Operators (A: weights, M output features by K; B: activations, N tokens by K, one token per row; C: N by M):

  quantize          X -> e4m3 codes and fp32 scales, one scale for each 1 x 128 block (activations) or 128 x 128 block (weights)
  fp8_linear        C = B * A^T from codes and scales
  grouped_linear    C rows of group e = B rows of group e * A[e]^T, fp16 or bf16, group sizes known on the device only
  grouped_fp8       the same from codes and scales
"""
import math

import numpy as np
import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
SCALE_MIN = 2.0 ** -64
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one token's activations before a layer: nothing but latency
        dict(name="quantize_1x9216", op="quantize", rows=1, cols=9216, block_rows=1, groups=1, type="fp16"),
        # a prefill batch of odd length
        dict(name="quantize_4099x12288", op="quantize", rows=4099, cols=12288, block_rows=1, groups=1, type="bf16"),
        # a layer's weights at load time, the last block of rows not full
        dict(name="quantize_weights_9208x36864", op="quantize", rows=9208, cols=36864, block_rows=128, groups=1, type="fp16"),
        # one token through an output projection
        dict(name="fp8_1_m9216_k9216", op="fp8_linear", n=1, m=9216, k=9216, type="fp16"),
        # a decode batch through the first layer of a feed-forward block
        dict(name="fp8_16_m36864_k9216", op="fp8_linear", n=16, m=36864, k=9216, type="bf16"),
        # a ragged chunk of a prompt
        dict(name="fp8_333_m7168_k7168", op="fp8_linear", n=333, m=7168, k=7168, type="bf16"),
        # prefill, bound by arithmetic
        dict(name="fp8_8192_m36864_k9216", op="fp8_linear", n=8192, m=36864, k=9216, type="fp16"),
        # decode through experts: most groups hold a token or two, some none
        dict(name="grouped_96_e64_m2048_k4096", op="grouped_linear", n=96, groups=64, m=2048, k=4096, routing=3, pad=0, type="bf16"),
        # prefill through experts of very unequal load, in a batch padded at its end
        dict(name="grouped_8205_e16_m4096_k7168", op="grouped_linear", n=8205, groups=16, m=4096, k=7168, routing=5, pad=13, type="fp16"),
        # the smallest call: a short prompt's rows through a few small experts
        dict(name="grouped_fp8_24_e8_m1032_k1040", op="grouped_fp8", n=24, groups=8, m=1032, k=1040, routing=7, pad=0, type="bf16"),
        # decode through many experts
        dict(name="grouped_fp8_256_e128_m4096_k2048", op="grouped_fp8", n=256, groups=128, m=4096, k=2048, routing=11, pad=0, type="fp16"),
        # prefill through experts
        dict(name="grouped_fp8_16384_e32_m4096_k7168", op="grouped_fp8", n=16384, groups=32, m=4096, k=7168, routing=13, pad=0, type="bf16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["quantize", "fp8_linear", "grouped_linear", "grouped_fp8"])
    kind = rng.choice(["fp16", "bf16"])
    if op == "quantize":
        block_rows = rng.choice([1, 1, 128])
        groups = rng.choice([1, 1, 4, 16]) if block_rows == 128 else 1
        cols = 16 * _log(rng, 64, 2304)
        most = (1 << 28) // (cols * groups)
        return dict(op=op, rows=_log(rng, 1 if block_rows == 1 else 64, max(65, min(36864, most))), cols=cols, block_rows=block_rows, groups=groups, type=kind)
    k = 16 * _log(rng, 64, 2304 if op == "fp8_linear" else 512)
    m = 8 * _log(rng, 64, 4608 if op == "fp8_linear" else 512)
    if op == "fp8_linear":
        while m * k > (1 << 29):
            m, k = max(512, m // 16 * 8), max(1024, k // 32 * 16)
        return dict(op=op, n=_log(rng, 1, 8192), m=m, k=k, type=kind)
    groups = rng.randint(2, 64)
    while groups * m * k > (1 << 30):
        groups = max(2, groups // 2)
    n = _log(rng, 1, 16384)
    return dict(op=op, n=n, groups=groups, m=m, k=k, routing=rng.randint(1, 1 << 20), pad=rng.choice([0, 0, min(7, n - 1)]), type=kind)


def _group_sizes(case):
    """Rows of each group, most of them unequal, some empty; their order is left to the seed."""
    r = np.random.RandomState(case["routing"])
    load = np.exp(r.randn(case["groups"]) * 0.7)
    return r.multinomial(case["n"] - case["pad"], load / load.sum())


# ---------------------------------------------------------------- inputs
def _values(shape, kind, sigma, g):
    return (torch.randn(shape, device="cuda", generator=g, dtype=torch.float32) * sigma).to(TYPES[kind])


def _codes(shape, sigma, block_rows, g):
    """Codes and scales as a checkpoint or an earlier call leaves them: [.., rows, K] -> codes, scales."""
    rows, k = shape[-2:]
    kb = -(-k // BLOCK)
    if block_rows == 1:
        top = (torch.rand((kb, rows), device="cuda", generator=g) * 2.0 + 2.0) * sigma
        per = top.t().repeat_interleave(BLOCK, 1)[:, :k]
    else:
        rb = -(-rows // BLOCK)
        top = (torch.rand((*shape[:-2], rb, kb), device="cuda", generator=g) + 3.5) * sigma
        per = top.repeat_interleave(BLOCK, -2)[..., :rows, :].repeat_interleave(BLOCK, -1)[..., :k]
    x = torch.randn(shape, device="cuda", generator=g, dtype=torch.float32)
    scales = top / E4M3_MAX
    x.mul_(sigma * E4M3_MAX).div_(per).clamp_(-E4M3_MAX, E4M3_MAX)
    return x.to(torch.float8_e4m3fn), scales.contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = dict(case)
    if case["op"] == "quantize":
        rows, cols = case["rows"], case["cols"]
        shape = (rows, cols) if case["groups"] == 1 else (case["groups"], rows, cols)
        x = torch.randn(shape, device="cuda", generator=g, dtype=torch.float32)
        if case["block_rows"] == 1:  # some features of activations are far larger than the others
            x *= torch.exp(torch.randn((cols,), device="cuda", generator=g) * 1.5)
        else:
            x *= 0.02
        s["x"] = x.to(TYPES[case["type"]])
        kb = -(-cols // BLOCK)
        s["codes"] = torch.zeros(shape, device="cuda", dtype=torch.float8_e4m3fn)
        s["scales"] = torch.zeros((kb, rows) if case["block_rows"] == 1 else (*shape[:-2], -(-rows // BLOCK), kb), device="cuda")
        return s
    n, m, k = case["n"], case["m"], case["k"]
    groups = case.get("groups", 0)
    weights = (groups, m, k) if groups else (m, k)
    if case["op"] == "grouped_linear":
        s["a"], s["b"] = _values(weights, case["type"], 0.02, g), _values((n, k), case["type"], 1.0, g)
    else:
        s["a"], s["a_scales"] = _codes(weights, 0.02, BLOCK, g)
        s["b"], s["b_scales"] = _codes((n, k), 1.0, 1, g)
    s["c"] = torch.zeros((n, m), device="cuda", dtype=TYPES[case["type"]])
    if groups:
        sizes = np.random.RandomState(int(seed) % (1 << 31)).permutation(_group_sizes(case))
        offsets = np.concatenate([[0], np.cumsum(sizes)])
        s["offsets"] = torch.from_numpy(offsets.astype(np.int32)).cuda()
        s["rows_used"], s["rows_most"] = int(offsets[-1]), int(sizes.max())
    if own:
        import graphneuralnetproj_b200 as sp
        nbytes = sp.linear_workspace_bytes(max(groups, 1), m, n, k, case["op"] != "grouped_linear")
        s["workspace"] = torch.zeros(nbytes, device="cuda", dtype=torch.uint8)
    return s


# ---------------------------------------------------------------- one pass
def _e4m3(y):
    """fp64 values rounded to the nearest e4m3 value, ties to even."""
    _, e = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), torch.clamp(e - 1, min=-6) - 3)
    return torch.clamp(torch.round(y / step) * step, -E4M3_MAX, E4M3_MAX)


def _blocks(x, block_rows):
    """x padded with zeros to whole blocks: [.., row blocks, block_rows, column blocks, 128]."""
    rows, cols = x.shape[-2:]
    rb, cb = -(-rows // block_rows), -(-cols // BLOCK)
    full = torch.zeros((*x.shape[:-2], rb * block_rows, cb * BLOCK), device=x.device, dtype=torch.float32)
    full[..., :rows, :cols] = x
    return full.view(*x.shape[:-2], rb, block_rows, cb, BLOCK)


def _quantize(s):
    x = s["x"]
    rows, cols = x.shape[-2:]
    blocks = _blocks(x, s["block_rows"])
    top = blocks.abs().amax(dim=(-3, -1))
    scales = torch.clamp(top / torch.full_like(top, E4M3_MAX), min=SCALE_MIN)  # by a tensor: a division, rounded once
    values = _e4m3(blocks.double() / scales.double()[..., :, None, :, None])
    values = values.to(torch.float32).reshape(*x.shape[:-2], blocks.shape[-4] * s["block_rows"], -1)[..., :rows, :cols]
    return {"codes": values.to(torch.float8_e4m3fn), "scales": scales.t().contiguous() if s["block_rows"] == 1 else scales}


def _decoded(codes, scales, block_rows):
    """The fp32 values that codes and scales stand for."""
    rows, cols = codes.shape[-2:]
    blocks = _blocks(codes.to(torch.float32), block_rows)
    per = scales.t()[:, None, :, None] if block_rows == 1 else scales[..., :, None, :, None]
    return (blocks * per).reshape(*codes.shape[:-2], blocks.shape[-4] * block_rows, -1)[..., :rows, :cols]


def _grouped(a, b, s):
    """Rows of each group padded to the longest group, one batched product, rows taken back."""
    rows = torch.arange(s["rows_used"], device="cuda")
    offsets = s["offsets"].long()
    group = torch.searchsorted(offsets[1:], rows, right=True)
    place = rows - offsets[group]
    padded = torch.zeros((s["groups"], s["rows_most"], s["k"]), device="cuda")
    padded[group, place] = b[:s["rows_used"]]
    c = torch.bmm(padded, a.transpose(1, 2))
    out = torch.zeros_like(s["c"])
    out[:s["rows_used"]] = c[group, place].to(out.dtype)
    return out


def run(state):
    s = state
    if own:
        import graphneuralnetproj_b200 as sp
        if s["op"] == "quantize":
            rc = sp.quantize_fp8(None, s["x"], s["codes"], s["scales"], s["block_rows"])
        elif s["op"] == "fp8_linear":
            rc = sp.fp8_linear(None, s["a"], s["a_scales"], s["b"], s["b_scales"], s["c"], s["m"], s["n"], s["k"], s["workspace"])
        elif s["op"] == "grouped_linear":
            rc = sp.grouped_linear(None, s["a"], s["b"], s["c"], s["offsets"], s["groups"], s["m"], s["n"], s["k"], s["workspace"])
        else:
            rc = sp.grouped_fp8_linear(None, s["a"], s["a_scales"], s["b"], s["b_scales"], s["c"], s["offsets"], s["groups"],
                                       s["m"], s["n"], s["k"], s["workspace"])
        if rc != 0:
            raise RuntimeError("cudaError %d" % rc)
        return {"codes": s["codes"], "scales": s["scales"]} if s["op"] == "quantize" else s["c"]
    if s["op"] == "quantize":
        return _quantize(s)
    if s["op"] == "grouped_linear":
        return _grouped(s["a"].float(), s["b"].float(), s)
    a, b = _decoded(s["a"], s["a_scales"], BLOCK), _decoded(s["b"], s["b_scales"], 1)
    if s["op"] == "fp8_linear":
        return (b @ a.t()).to(s["c"].dtype)
    return _grouped(a, b, s)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "quantize":
        rows, cols = case["rows"], case["cols"]
        blocks = -(-rows // case["block_rows"]) * -(-cols // BLOCK)
        return {"bytes": case["groups"] * (3 * rows * cols + 4 * blocks), "flops": case["groups"] * 2 * rows * cols}
    n, m, k = case["n"], case["m"], case["k"]
    sizes = _group_sizes(case) if "groups" in case else np.array([n])
    rows, active = int(sizes.sum()), int((sizes > 0).sum())
    width = 2 if case["op"] == "grouped_linear" else 1
    nbytes = active * m * k * width + rows * k * width + rows * m * 2
    if width == 1:
        nbytes += 4 * -(-k // BLOCK) * (active * -(-m // BLOCK) + rows)
    return {"bytes": nbytes + 4 * (len(sizes) + 1), "flops": 2 * rows * m * k}


# ---------------------------------------------------------------- definitions in 64 bits
def _e4m3_values():
    small = [i * 2.0 ** -9 for i in range(8)]
    return small + [(8 + f) * 2.0 ** (e - 3) for e in range(-6, 9) for f in range(8)][:119]  # 126 * 2^.. = 448 is the last


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        x = s["x"]
        lead = x.shape[:-2]
        x = x.reshape(-1, *x.shape[-2:])
        grid = torch.tensor(_e4m3_values(), device="cuda", dtype=torch.float64)
        codes, scales = torch.empty(x.shape, device="cuda", dtype=torch.float32), []
        for c0 in range(0, x.shape[2], BLOCK):
            part = x[:, :, c0:c0 + BLOCK].double()
            top = part.abs().amax(2)
            if case["block_rows"] != 1:
                pad = torch.nn.functional.pad(top, (0, -top.shape[1] % BLOCK))
                top = pad.view(top.shape[0], -1, BLOCK).amax(2)
            scale = torch.clamp(top / E4M3_MAX, min=SCALE_MIN)
            scales.append(scale)
            stored = scale.float().double()
            if case["block_rows"] != 1:
                stored = stored.repeat_interleave(BLOCK, 1)[:, :x.shape[1]]
            y = part / stored[:, :, None]
            mag = y.abs().contiguous()
            above = torch.searchsorted(grid, mag).clamp(max=len(grid) - 1)
            below = (above - 1).clamp(min=0)
            up, down = grid[above] - mag, mag - grid[below]
            pick = torch.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
            codes[:, :, c0:c0 + BLOCK] = torch.copysign(grid[pick], y).float()
        scales = torch.stack(scales, 2)
        codes = codes.reshape(*lead, *x.shape[1:])
        return {"codes": codes, "scales": scales[0].t().contiguous() if case["block_rows"] == 1 else scales.reshape(*lead, *scales.shape[1:])}

    def wide(codes, scales, rows_per):
        out = codes.double()
        for i in range(scales.shape[1] if rows_per != 1 else scales.shape[0]):
            if rows_per == 1:
                out[:, i * BLOCK:(i + 1) * BLOCK] *= scales[i].double()[:, None]
            else:
                out[:, i * BLOCK:(i + 1) * BLOCK] *= scales[:, i].double().repeat_interleave(BLOCK)[:out.shape[0], None]
        return out

    eight = case["op"] != "grouped_linear"
    b = wide(s["b"], s["b_scales"], 1) if eight else s["b"].double()
    if case["op"] == "fp8_linear":
        return b @ wide(s["a"], s["a_scales"], BLOCK).t()
    c = torch.zeros((case["n"], case["m"]), device="cuda", dtype=torch.float64)
    ends = s["offsets"].tolist()
    for e in range(case["groups"]):
        if ends[e + 1] > ends[e]:
            a = wide(s["a"][e], s["a_scales"][e], BLOCK) if eight else s["a"][e].double()
            c[ends[e]:ends[e + 1]] = b[ends[e]:ends[e + 1]] @ a.t()
    return c
