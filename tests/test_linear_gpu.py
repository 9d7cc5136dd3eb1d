"""The 8-bit block-scaled and grouped linear layers against their definitions in 64 bits.

Tolerance of a product, from the arithmetic alone: the values that codes and scales stand for are exact in 64 bits; the
kernel's sums are fp32.  A sum of K products in fp32, in whatever order and with each addition cut off rather than rounded
(what a tensor core may do), is off by at most K * 2^-23 * sum |a b|; the scales multiply in with three more roundings
(their product, the product with the block's sum, the addition), which the same bound with K + 4 covers; C is rounded
once, by half a step of its type (2^-11 or 2^-8 of the value, 2^-25 where fp16 is subnormal)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
E4M3 = np.array([i * 2.0 ** -9 for i in range(8)] + [(8 + f) * 2.0 ** (e - 3) for e in range(-6, 9) for f in range(8)][:119])


@pytest.fixture(scope="module", autouse=True)
def cuda():
    assert torch.cuda.is_available(), "these tests need a CUDA device"


def rng(*seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(hash(seed) % (1 << 31))
    return g


def kb_of(k):
    return -(-k // 128)


def random_operands(groups, m, n, k, dtype, seed):
    """Random codes with random scales (8 bits) or random values: tensors for the call and their fp64 values."""
    g = rng(groups, m, n, k, seed)
    a = torch.randn((groups, m, k), device="cuda", generator=g)
    b = torch.randn((n, k), device="cuda", generator=g)
    if dtype is not None:
        a, b = a.to(dtype), b.to(dtype)
        return a, None, b, None, a.double(), b.double()
    a8, b8 = (a * 30).to(torch.float8_e4m3fn), (b * 30).to(torch.float8_e4m3fn)
    sa = torch.rand((groups, kb_of(m), kb_of(k)), device="cuda", generator=g) + 0.5
    sb = torch.rand((kb_of(k), n), device="cuda", generator=g) * 0.01 + 1e-3
    av = a8.double() * sa.double().repeat_interleave(128, 1)[:, :m].repeat_interleave(128, 2)[:, :, :k]
    bv = b8.double() * sb.double().t().repeat_interleave(128, 1)[:, :k]
    return a8, sa, b8, sb, av, bv


def integer_operands(groups, m, n, k, dtype, seed):
    """Small whole numbers and powers of two as scales: every partial sum is exact, so C must be too.  Values -1, 0, 1 on
    a tenth of the places of A: sums stay below 2^8 with room, exact in bf16 as well."""
    g = rng(groups, m, n, k, seed, 1)
    a = (torch.rand((groups, m, k), device="cuda", generator=g) < 40.0 / k).float() * torch.randint(-1, 2, (groups, m, k), device="cuda", generator=g)
    b = torch.randint(-1, 2, (n, k), device="cuda", generator=g).float()
    if dtype is not None:
        return a.to(dtype), None, b.to(dtype), None, a.double(), b.double()
    sa = torch.full((groups, kb_of(m), kb_of(k)), 0.5, device="cuda")
    sb = torch.full((kb_of(k), n), 2.0, device="cuda")
    return a.to(torch.float8_e4m3fn), sa, b.to(torch.float8_e4m3fn), sb, a.double(), b.double()


def workspace_for(sp, groups, m, n, k, eight):
    return torch.zeros(sp.linear_workspace_bytes(groups, m, n, k, eight), dtype=torch.uint8, device="cuda")


def call(sp, a, sa, b, sb, c, offsets, groups, m, n, k, ws, stream=None):
    if offsets is None:
        return sp.fp8_linear(stream, a, sa, b, sb, c, m, n, k, ws)
    if sa is None:
        return sp.grouped_linear(stream, a, b, c, offsets, groups, m, n, k, ws)
    return sp.grouped_fp8_linear(stream, a, sa, b, sb, c, offsets, groups, m, n, k, ws)


def check(c, av, bv, offsets, k, out, exact=False):
    """c against the definition; rows outside all groups still hold 7."""
    n, m = c.shape
    borders = [0, n] if offsets is None else offsets
    covered = torch.zeros(n, dtype=torch.bool, device="cuda")
    for e in range(len(borders) - 1):
        rows = slice(borders[e], borders[e + 1])
        if borders[e + 1] <= borders[e]:
            continue
        covered[rows] = True
        want = bv[rows] @ av[e].t()
        got = c[rows].double()
        if exact:
            assert torch.equal(got, want), "group %d" % e
            continue
        size = bv[rows].abs() @ av[e].abs().t()
        bound = (k + 4) * 2.0 ** -23 * size + HALF_STEP[out] * want.abs() * 1.001 + 2.0 ** -25
        worst = ((got - want).abs() / bound).max().item()
        assert worst <= 1.0, "group %d: %.3f of the bound" % (e, worst)
    assert bool((c[~covered].double() == 7).all())


def run_case(sp, groups, m, n, k, dtype, out, offsets, with_workspace, make, exact):
    a, sa, b, sb, av, bv = make(groups, m, n, k, dtype, 5)
    c = torch.full((n, m), 7.0, dtype=out, device="cuda")
    ws = workspace_for(sp, groups, m, n, k, dtype is None) if with_workspace else None
    off = None if offsets is None else torch.tensor(offsets, dtype=torch.int32, device="cuda")
    assert call(sp, a, sa, b, sb, c, off, groups, m, n, k, ws) == 0
    torch.cuda.synchronize()
    assert sp.device_status() == 0
    check(c, av, bv, offsets, k, out, exact)


DENSE = [(128, 1, 128), (1, 1, 16), (130, 17, 144), (1032, 24, 1040), (257, 129, 272), (384, 300, 2048), (2304, 16, 4608), (1000, 64, 8192),
         (128, 3, 36864), (640, 513, 640), (7168, 40, 1024), (4104, 1031, 528)]


@pytest.mark.parametrize("make", [integer_operands, random_operands], ids=["integers", "random"])
@pytest.mark.parametrize("with_workspace", [True, False], ids=["workspace", "alone"])
@pytest.mark.parametrize("out", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("m,n,k", DENSE)
def test_fp8_linear(sp, m, n, k, out, with_workspace, make):
    run_case(sp, 1, m, n, k, None, out, None, with_workspace, make, make is integer_operands)


def borders(sizes, start=0):
    return [start] + [start + int(x) for x in np.cumsum(sizes)]


GROUPED = [  # m, n, k, group sizes, first row
    (128, 1, 128, [1], 0),
    (128, 4, 64, [0, 0, 4, 0], 0),
    (200, 37, 272, [5, 0, 17, 1, 14], 0),           # odd sizes
    (136, 50, 1040, [3, 2, 40], 2),                 # rows before the first group and behind the last
    (1032, 700, 528, [0, 300, 129, 1, 256, 0, 14], 0),
    (256, 16, 4096, [1] * 16, 0),                   # a token each, K cut between blocks
    (520, 2000, 144, [0] * 30 + [1990] + [0] * 33, 5),  # one group has nearly everything
    (64, 1024, 48, [1] * 1024, 0),                  # as many groups as there may be
    (384, 9, 2064, [0, 0, 0], 4),                   # nothing to do
    (264, 900, 528, [300, 0, 1, 257, 300], 7),      # many tokens per group: pairs of SMs
    (1000, 1400, 1040, [1393], 0),
    (513, 2100, 272, [33, 512, 129, 1400], 3),      # M odd
    (256, 520, 8192, [257, 263], 0),                # K cut between pairs
    (128, 700, 16, [160, 540], 0),
]


@pytest.mark.parametrize("make", [integer_operands, random_operands], ids=["integers", "random"])
@pytest.mark.parametrize("kind", ["fp16", "bf16", "e4m3-fp16", "e4m3-bf16"])
@pytest.mark.parametrize("case", range(len(GROUPED)))
def test_grouped(sp, case, kind, make):
    m, n, k, sizes, start = GROUPED[case]
    out = torch.bfloat16 if kind.endswith("bf16") else torch.float16
    dtype = None if kind.startswith("e4m3") else out
    for with_workspace in (True, False):
        run_case(sp, len(sizes), m, n, k, dtype, out, borders(sizes, start), with_workspace, make, make is integer_operands)


@pytest.mark.parametrize("eight", [True, False], ids=["e4m3", "fp16"])
def test_repeated_calls_are_bitwise_reproducible(sp, eight):
    """Tiles cut between blocks are added in a fixed order; the workspace is ready for the next call, of another size too."""
    ws = workspace_for(sp, 4, 1152, 40, 9216, eight)
    results = {}
    for turn in range(3):
        for n, k in ((40, 9216), (7, 4096)):
            m, sizes = 1152, [n - 4, 0, 3, 1]
            a, sa, b, sb, _, _ = random_operands(4, m, n, k, None if eight else torch.float16, 9)
            c = torch.zeros((n, m), dtype=torch.float16, device="cuda")
            off = torch.tensor(borders(sizes), dtype=torch.int32, device="cuda")
            assert call(sp, a, sa, b, sb, c, off, 4, m, n, k, ws) == 0
            first = results.setdefault(n, c)
            assert torch.equal(first, c), turn


def test_values_outside_a_group_do_not_reach_it(sp):
    """NaN in the rows of other groups, behind the last group, and in the weights of an empty group."""
    m, n, k, sizes = 192, 60, 256, [20, 0, 21]
    for dtype in (None, torch.bfloat16):
        a, sa, b, sb, av, bv = random_operands(3, m, n, k, dtype, 3)
        a, b = a.clone(), b.clone()
        bits = torch.uint8 if dtype is None else torch.int16
        a[1].view(bits).fill_(0x7f if dtype is None else 0x7fff)
        b[41:].view(bits).fill_(0x7f if dtype is None else 0x7fff)
        b[20:41].view(bits)[3, 5] = 0x7f if dtype is None else 0x7fff
        c = torch.full((n, m), 7.0, dtype=torch.bfloat16, device="cuda")
        off = torch.tensor(borders(sizes), dtype=torch.int32, device="cuda")
        assert call(sp, a, sa, b, sb, c, off, 3, m, n, k, workspace_for(sp, 3, m, n, k, dtype is None)) == 0
        assert bool(c[23].isnan().all())
        c[23] = (bv[23] @ av[2].t()).to(c.dtype)
        check(c, av, bv, borders(sizes), k, torch.bfloat16)


def test_corrupt_group_borders_touch_nothing_outside(sp):
    m, n, k, groups = 136, 40, 128, 4
    a, sa, b, sb, _, _ = random_operands(groups, m, n, k, None, 4)
    for table in ([-5, 3, 2000000000, 10, 41], [40, 30, 20, 10, 0], [-1, -2, -3, -4, -5], [2147483647, -2147483648, 2147483647, 0, 100]):
        whole = torch.full((3 * n, m), 7.0, dtype=torch.float16, device="cuda")
        off = torch.tensor(table, dtype=torch.int32, device="cuda")
        assert call(sp, a, sa, b, sb, whole[n:2 * n], off, groups, m, n, k, None) == 0
        torch.cuda.synchronize()
        assert sp.device_status() == 0
        assert bool((whole[:n] == 7).all()) and bool((whole[2 * n:] == 7).all())


def test_far_offsets(sp):
    """Weights and results beyond 2^31 elements."""
    groups, m, k, n = 9, 16384, 16384, 3
    a = torch.zeros((groups, m, k), dtype=torch.float8_e4m3fn, device="cuda")
    a.view(torch.uint8)[8, m - 1, k - 16:] = 0x38  # 1.0
    sa = torch.ones((groups, m // 128, k // 128), device="cuda")
    b, sb = torch.ones((n, k), device="cuda").to(torch.float8_e4m3fn), torch.ones((k // 128, n), device="cuda")
    c = torch.zeros((n, m), dtype=torch.float16, device="cuda")
    off = torch.tensor([0] * 9 + [n], dtype=torch.int32, device="cuda")
    assert call(sp, a, sa, b, sb, c, off, groups, m, n, k, workspace_for(sp, groups, m, n, k, True)) == 0
    assert bool((c[:, m - 1] == 16).all()) and bool((c[:, :m - 1] == 0).all())
    del a
    m, n, k = 65544, 32896, 16
    a, sa, b, sb, av, bv = integer_operands(1, m, n, k, None, 6)
    c = torch.full((n, m), 7.0, dtype=torch.float16, device="cuda")
    assert call(sp, a, sa, b, sb, c, None, 1, m, n, k, None) == 0
    for rows in (slice(0, 130), slice(n - 130, n)):
        assert torch.equal(c[rows].double(), bv[rows] @ av[0].t())


def test_two_streams_at_once_and_graph_replay(sp):
    m, k, sizes = 1152, 4608, [9, 0, 30]
    n = sum(sizes)
    off = torch.tensor(borders(sizes), dtype=torch.int32, device="cuda")
    jobs = []
    for seed, dtype in ((1, None), (2, torch.float16)):
        a, sa, b, sb, av, bv = random_operands(3, m, n, k, dtype, seed)
        jobs.append((a, sa, b, sb, torch.full((n, m), 7.0, dtype=torch.float16, device="cuda"), workspace_for(sp, 3, m, n, k, dtype is None), av, bv))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for s, (a, sa, b, sb, c, ws, _, _) in zip(streams, jobs):
            assert call(sp, a, sa, b, sb, c, off, 3, m, n, k, ws, s) == 0
    torch.cuda.synchronize()
    assert sp.device_status() == 0
    for a, sa, b, sb, c, ws, av, bv in jobs:
        check(c, av, bv, borders(sizes), k, torch.float16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for a, sa, b, sb, c, ws, _, _ in jobs:
            assert call(sp, a, sa, b, sb, c, off, 3, m, n, k, ws) == 0
    other = [30, 9, 0]  # the borders are read when the graph runs
    for table in (sizes, other, sizes):
        off.copy_(torch.tensor(borders(table), dtype=torch.int32))
        for job in jobs:
            job[4].fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        for a, sa, b, sb, c, ws, av, bv in jobs:
            check(c, av, bv, borders(table), k, torch.float16)


@pytest.mark.parametrize("kind", ["e4m3", "bf16"])
def test_pairs_on_two_streams_and_in_a_graph(sp, kind):
    """Many tokens per group: two calls at once with a workspace each, then both in one graph, K cut between pairs."""
    m, k, sizes = 512, 8192, [200, 0, 310]
    n, dtype = sum(sizes), None if kind == "e4m3" else torch.bfloat16
    off = torch.tensor(borders(sizes), dtype=torch.int32, device="cuda")
    jobs = []
    for seed in (1, 2):
        a, sa, b, sb, av, bv = random_operands(3, m, n, k, dtype, seed)
        jobs.append((a, sa, b, sb, torch.full((n, m), 7.0, dtype=torch.bfloat16, device="cuda"), workspace_for(sp, 3, m, n, k, dtype is None), av, bv))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for s, (a, sa, b, sb, c, ws, _, _) in zip(streams, jobs):
            assert call(sp, a, sa, b, sb, c, off, 3, m, n, k, ws, s.cuda_stream) == 0  # a raw handle
    torch.cuda.synchronize()
    first = [job[4].clone() for job in jobs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for a, sa, b, sb, c, ws, _, _ in jobs:
            assert call(sp, a, sa, b, sb, c, off, 3, m, n, k, ws) == 0
    for job in jobs:
        job[4].fill_(7.0)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert sp.device_status() == 0
    for (_, _, _, _, c, _, av, bv), before in zip(jobs, first):
        assert torch.equal(c, before)
        check(c, av, bv, borders(sizes), k, torch.bfloat16)


def test_smallest_depth_and_codes_as_bytes(sp):
    """K of one 16-byte row; codes passed as uint8."""
    run_case(sp, 2, 3, 5, 8, torch.float16, torch.float16, [0, 2, 5], True, integer_operands, True)
    m, n, k = 72, 9, 16
    a, sa, b, sb, av, bv = integer_operands(1, m, n, k, None, 2)
    c = torch.full((n, m), 7.0, dtype=torch.bfloat16, device="cuda")
    assert sp.fp8_linear(None, a.view(torch.uint8), sa, b.view(torch.uint8), sb, c, m, n, k, None) == 0
    assert torch.equal(c.double(), bv @ av[0].t())


def test_nothing_to_do(sp):
    """No tokens, no rows: nothing is written."""
    m, k = 128, 128
    a, sa, _, _, _, _ = random_operands(2, m, 1, k, None, 3)
    empty8, empty = torch.empty((0, k), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((0, m), dtype=torch.float16, device="cuda")
    scales, off = torch.empty((1, 0), device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    assert sp.fp8_linear(None, a[0], sa[0], empty8, scales, empty, m, 0, k, None) == 0
    assert sp.grouped_fp8_linear(None, a, sa, empty8, scales, empty, off, 2, m, 0, k, None) == 0
    assert sp.grouped_linear(None, a.to(torch.float16), empty8.to(torch.float16), empty, off, 2, m, 0, k, None) == 0
    assert sp.quantize_fp8(None, torch.empty((0, k), dtype=torch.float16, device="cuda"), empty8, scales, 1) == 0


def test_not_finite_operands_reach_their_rows_only(sp):
    """Infinite activations or scales spoil the tokens they belong to, at few and at many tokens."""
    for n in (20, 300):
        m, k = 136, 400
        a, sa, b, sb, av, bv = random_operands(1, m, n, k, None, 8)
        sb = sb.clone()
        sb[1, 7] = float("inf")
        sb[3, 11] = float("nan")
        c = torch.full((n, m), 7.0, dtype=torch.bfloat16, device="cuda")
        assert sp.fp8_linear(None, a[0], sa[0], b, sb, c, m, n, k, workspace_for(sp, 1, m, n, k, True)) == 0
        assert not bool(c[[7, 11]].isfinite().any())
        good = torch.ones(n, dtype=torch.bool, device="cuda")
        good[[7, 11]] = False
        check(c[good], av, bv[good], None, k, torch.bfloat16)


# ---------------------------------------------------------------- quantiser
def reference_codes(x, block_rows):
    """(values, scales) by the definition: the e4m3 value nearest to x / scale, ties to the even code."""
    rows, cols = x.shape
    kb, rb = kb_of(cols), -(-rows // block_rows)
    mag = np.where(np.isfinite(x), np.abs(x), 0.0)
    full = np.zeros((rb * block_rows, kb * 128))
    full[:rows, :cols] = mag
    top = full.reshape(rb, block_rows, kb, 128).max(axis=(1, 3))
    scales = np.maximum((top / 448.0).astype(np.float32), np.float32(2.0 ** -64))
    per = np.repeat(np.repeat(scales.astype(np.float64), block_rows, 0)[:rows], 128, 1)[:, :cols]
    y = mag / per
    above = np.minimum(np.searchsorted(E4M3, y), 126)
    below = np.maximum(above - 1, 0)
    up, down = E4M3[above] - y, y - E4M3[below]
    value = np.where((up < down) | ((up == down) & (above % 2 == 0)), E4M3[above], E4M3[below])
    return np.where(np.isfinite(x), np.copysign(value, x), np.nan), scales


def quantize(sp, x, block_rows):
    rows, cols = x.shape
    codes = torch.zeros((rows, cols), dtype=torch.float8_e4m3fn, device="cuda")
    shape = (kb_of(cols), rows) if block_rows == 1 else (-(-rows // 128), kb_of(cols))
    scales = torch.zeros(shape, device="cuda")
    assert sp.quantize_fp8(None, x, codes, scales, block_rows) == 0
    return codes, scales


def check_quantized(x, codes, scales, block_rows):
    want, want_scales = reference_codes(x.double().cpu().numpy(), block_rows)
    got_scales = scales.cpu().numpy()
    assert np.array_equal(got_scales.T if block_rows == 1 else got_scales, want_scales)
    got = codes.float().double().cpu().numpy()
    assert np.array_equal(got, want, equal_nan=True)
    assert np.array_equal(np.signbit(got[~np.isnan(want)]), np.signbit(want[~np.isnan(want)]))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,cols", [(1, 16), (1, 9216), (7, 144), (8, 1024), (129, 400), (300, 2064), (1025, 1040)])
def test_quantize(sp, rows, cols, block_rows, dtype):
    g = rng(rows, cols)
    x = torch.randn((rows, cols), device="cuda", generator=g) * torch.exp(2 * torch.randn((cols,), device="cuda", generator=g))
    x[rows // 2, : cols // 2] = 0.0
    x = x.to(dtype)
    check_quantized(x, *quantize(sp, x, block_rows), block_rows)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_quantize_borders(sp, dtype):
    """Ties, their neighbours, the smallest codes, zeros of both signs, infinities, NaN, blocks of nothing, extreme blocks."""
    mids = (E4M3[1:] + E4M3[:-1]) / 2
    rows = []
    for power in (0, -3, 4 if dtype is torch.float16 else 60):  # amax = 448 * 2^power: the scale is a power of two
        t = torch.tensor(np.concatenate([mids, -mids, E4M3, [0.0, -0.0]]) * 2.0 ** power).to(dtype)
        up, down = (t.view(torch.int16) + 1).view(dtype), (t.view(torch.int16) - 1).view(dtype)
        for v in (t, up, down):
            v = v[torch.isfinite(v) & (v.abs() <= 448.0 * 2.0 ** power)]
            v = torch.cat([v, torch.zeros(-len(v) % 127, dtype=dtype)]).view(-1, 127)
            rows.append(torch.cat([v, torch.full((len(v), 1), 448.0 * 2.0 ** power, dtype=dtype)], 1))
    special = torch.zeros((9, 128), dtype=dtype)
    special[0, 3] = float("inf")
    special[0, 4] = 1.0
    special[1, 100] = float("nan")
    special[1, :50] = torch.linspace(-3, 3, 50).to(dtype)
    special[2] = float("-inf")
    special[3, 7] = torch.finfo(dtype).max
    special[3, 8] = torch.finfo(dtype).tiny
    special[4] = torch.finfo(dtype).smallest_normal / 4
    special[5, 0] = torch.finfo(dtype).max
    special[5, 1:] = -torch.finfo(dtype).max
    special[6, 64:] = -0.0
    special[7, 1] = 2.0 ** -24
    special[8, ::2] = 1.0 / 3
    rows.append(special)
    x = torch.cat(rows).cuda().contiguous()
    check_quantized(x, *quantize(sp, x, 1), 1)
    check_quantized(x[:, :].contiguous(), *quantize(sp, x, 128), 128)


def test_quantize_every_fp16_value(sp):
    """All finite halves under 32 different scales."""
    values = torch.arange(0, 65536, dtype=torch.int32).to(torch.int16).view(torch.float16)
    values = values[torch.isfinite(values)]
    for step in range(32):
        top = float(values.abs().max()) * (1.0 - step / 67.0)
        v = values[values.abs() <= top]
        v = torch.cat([v, torch.zeros(-len(v) % 127, dtype=v.dtype)]).view(-1, 127)
        x = torch.cat([v, torch.full((len(v), 1), top, dtype=v.dtype)], 1).cuda()
        check_quantized(x, *quantize(sp, x, 1), 1)


def test_quantize_groups_of_weights(sp):
    x = torch.randn((3, 200, 272), device="cuda", generator=rng(3)).to(torch.bfloat16)
    codes, scales = torch.zeros(x.shape, dtype=torch.uint8, device="cuda"), torch.zeros((3, 2, 3), device="cuda")
    assert sp.quantize_fp8(None, x, codes, scales, 128) == 0
    for e in range(3):
        check_quantized(x[e], codes[e].view(torch.float8_e4m3fn), scales[e], 128)


# ---------------------------------------------------------------- as they are used
def test_feed_forward_through_experts(sp):
    """Tokens sorted by expert through two 8-bit layers with a ReLU between them, all on one stream, the group borders and
    the second layer's operands written by the kernels just ahead.  Each stage against its definition on the stage's inputs."""
    tokens, hidden, inner, groups = 45, 512, 1040, 6
    g = rng(77)
    x = torch.randn((tokens, hidden), device="cuda", generator=g).to(torch.bfloat16)
    weights = [torch.randn(s, device="cuda", generator=g).mul_(0.05).to(torch.bfloat16) for s in ((groups, inner, hidden), (groups, hidden, inner))]
    packed = []
    for w in weights:
        codes = torch.empty(w.shape, dtype=torch.float8_e4m3fn, device="cuda")
        scales = torch.empty((groups, kb_of(w.shape[1]), kb_of(w.shape[2])), device="cuda")
        assert sp.quantize_fp8(None, w, codes, scales, 128) == 0
        packed.append((codes, scales))
    expert = torch.randint(0, groups - 1, (tokens,), device="cuda", generator=g)
    order = torch.argsort(expert, stable=True)
    off = torch.searchsorted(expert[order].contiguous(), torch.arange(groups + 1, device="cuda")).to(torch.int32)
    rows = x[order].contiguous()
    for layer, (codes, scales) in enumerate(packed):
        m, k = codes.shape[1:]
        b, sb = quantize(sp, rows, 1)
        c = torch.full((tokens, m), 7.0, dtype=torch.bfloat16, device="cuda")
        assert sp.grouped_fp8_linear(None, codes, scales, b, sb, c, off, groups, m, tokens, k, workspace_for(sp, groups, m, tokens, k, True)) == 0
        av = codes.double() * scales.double().repeat_interleave(128, 1)[:, :m].repeat_interleave(128, 2)[:, :, :k]
        bv = b.double() * sb.double().t().repeat_interleave(128, 1)[:, :k]
        check(c, av, bv, off.tolist(), k, torch.bfloat16)
        check_quantized(rows, b, sb, 1)
        rows = torch.relu(c)
    assert sp.device_status() == 0


def test_python_refusals(sp):
    m, n, k = 128, 4, 128
    a, sa, b, sb, _, _ = random_operands(1, m, n, k, None, 1)
    c = torch.zeros((n, m), dtype=torch.float16, device="cuda")
    off = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    ok = dict(A=a, A_scales=sa, B=b, B_scales=sb, C=c)
    for name, bad in [("A", a.float()), ("A", a.cpu()), ("A", a[:, :64]), ("B", b.t()), ("B", b[:3]), ("A_scales", sa.half()), ("B_scales", sb[:, :3]),
                      ("C", c.float()), ("C", torch.zeros((m, n), dtype=torch.float16, device="cuda").t()), ("C", c[:3])]:
        with pytest.raises(ValueError):
            t = dict(ok, **{name: bad})
            sp.fp8_linear(None, t["A"], t["A_scales"], t["B"], t["B_scales"], t["C"], m, n, k, None)
    with pytest.raises(ValueError):
        sp.grouped_linear(None, a.half(), b.bfloat16(), c, off, 1, m, n, k, None)
    with pytest.raises(ValueError):
        sp.grouped_fp8_linear(None, a, sa, b, sb, c, off.long(), 1, m, n, k, None)
    with pytest.raises(ValueError):
        sp.grouped_fp8_linear(None, a, sa, b, sb, c, off, 2, m, n, k, None)
    with pytest.raises(ValueError):
        sp.quantize_fp8(None, c, b, sb, 2)
    with pytest.raises(ValueError):
        sp.quantize_fp8(None, c.float(), b, sb, 1)
    assert sp.fp8_linear(None, a[:, :120].contiguous(), sa, b[:, :120].contiguous(), sb, c, m, n, 120, None) == 1
    small = torch.zeros(64, dtype=torch.uint8, device="cuda")  # too small a workspace is not used
    assert sp.fp8_linear(None, a, sa, b, sb, c, m, n, k, small) == 0
    assert not bool(small.any())


@pytest.mark.parametrize("eight", [True, False], ids=["e4m3", "fp16"])
def test_as_many_tokens_as_there_may_be(sp, eight):
    """2^31 - 513 tokens of the smallest depth, in one group but for a few: counts and widths of tiles near the end of an
    int.  Values 0, 1 and 128, whose sums (16 of them at most) are exact in fp16."""
    m, n, k = 1, 2 ** 31 - 513, 16 if eight else 8
    free = torch.cuda.mem_get_info()[0]
    if free < 64 << 30:
        pytest.skip("needs 64 GB of device memory, %d GB are free" % (free >> 30))
    bits = 0x38 if eight else 0x3c00  # 1.0; twice the bits are 128 (e4m3), 2^15 would be too much for fp16: halves take 0 and 1
    b = torch.randint(0, 3 if eight else 2, (n, k), dtype=torch.uint8 if eight else torch.int16, device="cuda", generator=rng(n, k))
    b.mul_(bits)
    b = b.view(torch.float8_e4m3fn if eight else torch.float16)
    a = torch.ones((2, m, k), device="cuda").to(b.dtype)
    c = torch.full((n, m), 7.0, dtype=torch.float16, device="cuda")
    off = torch.tensor([2, 7, n - 1], dtype=torch.int32, device="cuda")
    sa = sb = None
    if eight:
        sa, sb = torch.ones((2, 1, 1), device="cuda"), torch.ones((1, n), device="cuda")
    assert call(sp, a, sa, b, sb, c, off, 2, m, n, k, None) == 0
    assert sp.device_status() == 0
    assert bool((c[:2] == 7).all()) and bool((c[n - 1] == 7).all())
    for first in range(2, n - 1, 1 << 26):
        last = min(n - 1, first + (1 << 26))
        assert torch.equal(c[first:last, 0], b[first:last].to(torch.float16).sum(1)), first
    del a, b, c, sa, sb
    torch.cuda.empty_cache()


@pytest.mark.parametrize("kb", [1, 3, 4, 7], ids=lambda kb: "%d-blocks" % kb)
@pytest.mark.parametrize("n", [1, 20, 50, 100, 300])
def test_infinite_scales_at_the_end_of_k(sp, n, kb):
    """Infinite scales of the last k-block give what the formula gives, whether the number of k-blocks is odd or even: codes
    are positive, so it is an infinity, and NaN for the scale that is NaN."""
    m, k = 264, 128 * kb - 48
    a = torch.full((1, m, k), 0x38, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    b = torch.full((n, k), 0x40, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    sa, sb = torch.full((1, kb_of(m), kb), 0.25, device="cuda"), torch.full((kb, n), 0.5, device="cuda")
    sa[0, 1, kb - 1] = float("inf")
    sb[kb - 1, n // 2] = float("-inf")
    sb[kb - 1, n // 3] = float("nan")
    depth = torch.full((kb,), 128.0, dtype=torch.float64, device="cuda")
    depth[kb - 1] = 80
    want = 2 * torch.einsum("b,ob,bn->no", depth, sa[0].double(), sb.double()).repeat_interleave(128, 1)[:, :m]
    assert bool(want.isinf().any()) or n < 3
    for groups in (None, [0, n // 2, n]):
        c = torch.full((n, m), 7.0, dtype=torch.bfloat16, device="cuda")
        off = None if groups is None else torch.tensor(groups, dtype=torch.int32, device="cuda")
        count = 1 if groups is None else 2
        assert call(sp, a.expand(count, -1, -1).contiguous(), sa.repeat(count, 1, 1), b, sb, c, off, count, m, n, k,
                    workspace_for(sp, count, m, n, k, True)) == 0
        finite = want.isfinite()
        assert torch.equal(c[~finite].double().nan_to_num(nan=5.0), want[~finite].nan_to_num(nan=5.0))
        assert bool(((c[finite].double() - want[finite]).abs() <= HALF_STEP[torch.bfloat16] * want[finite].abs()).all())
    assert sp.device_status() == 0


def test_chain_of_calls_on_buffers_written_just_ahead(sp):
    """Quantiser, product, quantiser, experts back to back, every launch starting while the one that writes its operands,
    scales or group borders may still run, all in buffers that the turn before has used with other values: the same as with the
    device idle between the calls."""
    n, hidden, inner, groups, turns = 24, 1024, 1536, 3, 12
    g = rng(5)
    w1, s1, _, _, _, _ = random_operands(1, inner, 1, hidden, None, 1)
    w2, s2, _, _, _, _ = random_operands(groups, hidden, 1, inner, None, 2)
    w3 = torch.randn((groups, hidden, hidden), device="cuda", generator=g).mul_(0.05).to(torch.bfloat16)
    inputs = [torch.randn((n, hidden), device="cuda", generator=g).mul_(2.0 ** (t % 5)).to(torch.bfloat16) for t in range(turns)]
    tables = [torch.tensor([t % 3, 5 + t % 7, 20 - t % 8, n - t % 2], dtype=torch.int32, device="cuda") for t in range(turns)]
    ws = torch.zeros(max(sp.linear_workspace_bytes(e, inner, n, inner, True) for e in (1, groups)), dtype=torch.uint8, device="cuda")
    x, off = torch.empty_like(inputs[0]), torch.empty_like(tables[0])
    c1, c2, c3 = (torch.empty((n, m), dtype=torch.bfloat16, device="cuda") for m in (inner, hidden, hidden))
    codes = [torch.empty((n, k), dtype=torch.float8_e4m3fn, device="cuda") for k in (hidden, inner)]
    scales = [torch.empty((kb_of(k), n), device="cuda") for k in (hidden, inner)]

    def turn(t, idle, keep):
        steps = [lambda: x.copy_(inputs[t]) is None, lambda: off.copy_(tables[t]) is None, lambda: c2.zero_() is None, lambda: c3.zero_() is None,
                 lambda: sp.quantize_fp8(None, x, codes[0], scales[0], 1),
                 lambda: sp.fp8_linear(None, w1, s1, codes[0], scales[0], c1, inner, n, hidden, ws),
                 lambda: sp.quantize_fp8(None, c1, codes[1], scales[1], 1),
                 lambda: sp.grouped_fp8_linear(None, w2, s2, codes[1], scales[1], c2, off, groups, hidden, n, inner, ws),
                 lambda: sp.grouped_linear(None, w3, c2, c3, off, groups, hidden, n, hidden, ws)]
        for step in steps:
            assert step() == 0
            if idle:
                torch.cuda.synchronize()
        keep[t].copy_(c3)

    want, got, replayed = (torch.empty((turns, n, hidden), dtype=torch.bfloat16, device="cuda") for _ in range(3))
    for t in range(turns):
        turn(t, True, want)
    for _ in range(3):
        for t in range(turns):
            turn(t, False, got)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for t in range(turns):
            turn(t, False, replayed)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert sp.device_status() == 0
    assert bool(want.isfinite().all()) and bool((want != 0).any(2).any(1).all())
    assert torch.equal(want, got) and torch.equal(want, replayed)


def test_a_wait_that_runs_out_is_reported_and_cleared(sp):
    """Failure detection without a fault: two warps wait with the linear layers' bounded wait for something that nothing does.
    One gives up after 50 ms, the other follows, the block ends, the status word says so until it is reset, and the
    layers keep working."""
    assert sp.device_status(reset=True) == 0
    assert sp.selftest_linear_wait_timeout(50) == 0
    assert sp.device_status() == 1
    assert sp.device_status(reset=True) == 1
    assert sp.device_status() == 0
    for n in (20, 300):
        run_case(sp, 1, 264, n, 528, None, torch.float16, None, True, integer_operands, True)


def test_errors_of_other_calls_are_not_reported(sp):
    """An error that an earlier call has returned already (here: a status is asked for while a stream is capturing) is not
    returned again by a product, a quantiser or an SpMM that runs."""
    import ctypes
    runtime = ctypes.CDLL("libcudart.so.12")
    m, n, k = 128, 4, 128
    a, sa, b, sb, av, bv = random_operands(1, m, n, k, None, 1)
    x = torch.ones((n, k), dtype=torch.float16, device="cuda")
    c = torch.full((n, m), 7.0, dtype=torch.float16, device="cuda")
    assert sp.fp8_linear(None, a, sa, b, sb, c, m, n, k, None) == 0 and sp.device_status() == 0
    words, offsets, _ = sp.InitSparseMatrixA_API(sp.synth_fp16((m, k), 1, 0.02, 0.8), m, 16, k)
    words, offsets = torch.from_numpy(words.view(np.int32)).cuda(), torch.from_numpy(offsets).cuda()
    dense, out = torch.ones((k, 16), dtype=torch.float16, device="cuda"), torch.empty((m, 16), dtype=torch.float16, device="cuda")
    calls = [lambda: sp.quantize_fp8(None, x, b, sb, 1), lambda: sp.fp8_linear(None, a, sa, b, sb, c, m, n, k, None),
             lambda: sp.SpMM_SplitK_API(None, None, words, None, None, offsets, dense, out, m, 16, k, None, 1)]
    statuses = [sp.device_status, lambda: sp.spmm_api.LIB.spmm_b200_allreduce_status(0)]
    for run, ask in [(run, ask) for run in calls for ask in statuses]:
        stream, graph = torch.cuda.Stream(), ctypes.c_void_p()
        torch.cuda.synchronize()
        assert runtime.cudaStreamBeginCapture(ctypes.c_void_p(stream.cuda_stream), 2) == 0
        try:
            status = ask()
        finally:
            runtime.cudaStreamEndCapture(ctypes.c_void_p(stream.cuda_stream), ctypes.byref(graph))
            runtime.cudaGetLastError()
        assert status < 0
        assert run() == 0
    assert sp.device_status() == 0
    assert bool((b.float() == 448).all()) and bool((sb == 1 / torch.tensor(448.0, device="cuda")).all())


# ---------------------------------------------------------------- scales, depth, many groups and bands of tiles
def scaled_integer_operands(groups, m, n, k, dtype, seed):
    """As integer_operands (A has about 40 places that are not zero in a row, whatever K is), but with scales drawn per block
    and per token: 1 or 2 for A; 1/2, 1 or 2 for B.  Sums are multiples of 1/2 that stay below 128, exact in bf16, and a
    scale of another k-block, row block, group or token, or a k-block left out, changes them at every depth."""
    a, sa, b, sb, av, bv = integer_operands(groups, m, n, k, dtype, seed)
    if dtype is not None:
        return a, sa, b, sb, av, bv
    g = rng(groups, m, n, k, seed, 2)
    sa = torch.randint(0, 2, sa.shape, device="cuda", generator=g).float().exp2()
    sb = torch.randint(-1, 2, sb.shape, device="cuda", generator=g).float().exp2()
    av = a.double() * sa.double().repeat_interleave(128, 1)[:, :m].repeat_interleave(128, 2)[:, :, :k]
    bv = b.double() * sb.double().t().repeat_interleave(128, 1)[:, :k]
    return a, sa, b, sb, av, bv


def exact_case(sp, groups, m, n, k, dtype, out, offsets, with_workspace):
    """run_case on scaled_integer_operands, after a look at the oracle: its values have to fit the type of C."""
    _, _, _, _, av, bv = scaled_integer_operands(groups, m, n, k, dtype, 5)
    for e in range(groups):
        want = bv[:256] @ av[e].t()
        assert torch.equal(want.to(out).double(), want)
    run_case(sp, groups, m, n, k, dtype, out, offsets, with_workspace, scaled_integer_operands, True)


@pytest.mark.parametrize("with_workspace", [True, False], ids=["workspace", "alone"])
@pytest.mark.parametrize("out", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("m,n,k", DENSE + [(264, 150, 16400), (520, 33, 9232), (640, 520, 4112)])
def test_fp8_linear_with_scales_of_their_own(sp, m, n, k, out, with_workspace):
    exact_case(sp, 1, m, n, k, None, out, None, with_workspace)


@pytest.mark.parametrize("out", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("case", range(len(GROUPED)))
def test_grouped_fp8_with_scales_of_their_own(sp, case, out):
    m, n, k, sizes, start = GROUPED[case]
    exact_case(sp, len(sizes), m, n, k, None, out, borders(sizes, start), True)


DEEP = [(128, 3, 36864), (2304, 16, 9216), (1000, 64, 8192), (264, 120, 16400), (640, 513, 8192)]


@pytest.mark.parametrize("kind", ["e4m3-fp16", "e4m3-bf16", "fp16", "bf16"])
@pytest.mark.parametrize("m,n,k", DEEP)
def test_deep_products_by_their_mean_square_error(sp, m, n, k, kind):
    """At large K the bound for each element, which adds up the largest error of every addition, hides whole k-blocks.  Of the
    root of the mean square the triangle inequality gives more: an addition is off by 2^-23 of the sum there is at most,
    K of them by K * 2^-23 times the largest root mean square that the sums have on their way (taken behind each 128; half as
    much again for what lies between), and C by half a step.  A k-block left out is sqrt(128 / K) of C, more than five times that."""
    out = torch.bfloat16 if kind.endswith("bf16") else torch.float16
    dtype = None if kind.startswith("e4m3") else out
    a, sa, b, sb, av, bv = random_operands(1, m, n, k, dtype, 7)
    rms = lambda t: t.square().mean().sqrt().item()  # noqa: E731
    total, largest = torch.zeros((n, m), dtype=torch.float64, device="cuda"), 0.0
    for first in range(0, k, 128):
        total += bv[:, first:first + 128] @ av[0][:, first:first + 128].t()
        largest = max(largest, rms(total))
    bound = HALF_STEP[out] * rms(total) + k * 2.0 ** -23 * 1.5 * largest
    assert 5 * bound < (128.0 / k) ** 0.5 * rms(total)
    off = None if dtype is None else torch.tensor([0, n], dtype=torch.int32, device="cuda")
    for ws in (None, workspace_for(sp, 1, m, n, k, dtype is None)):
        c = torch.full((n, m), 7.0, dtype=out, device="cuda")
        assert call(sp, a, sa, b, sb, c, off, 1, m, n, k, ws) == 0
        assert rms(c.double() - total) <= bound


@pytest.mark.parametrize("kind", ["fp16", "bf16", "e4m3-fp16", "e4m3-bf16"])
def test_many_groups_of_many_tokens(sp, kind):
    """More groups than are sorted by width (256), with 130 tokens on average: pairs of SMs."""
    out = torch.bfloat16 if kind.endswith("bf16") else torch.float16
    groups, m, k = 300, 264, 144
    sizes = np.random.RandomState(3).multinomial(groups * 130, np.random.RandomState(4).dirichlet(np.full(groups, 0.7)))
    sizes[17] = sizes[299] = 0
    n = int(sizes.sum()) + 9
    assert n // groups > 128 and (sizes > 512).any() and (sizes[:256] == 0).any()
    run_case(sp, groups, m, n, k, None if kind.startswith("e4m3") else out, out, borders(sizes, 4), True, scaled_integer_operands, True)


@pytest.mark.parametrize("kind", ["fp16", "bf16", "e4m3-fp16", "e4m3-bf16"])
def test_several_bands_of_tiles(sp, kind):
    """More tiles of tokens than a band holds (8), on pairs of SMs and in single blocks; every row is compared."""
    out = torch.bfloat16 if kind.endswith("bf16") else torch.float16
    dtype = None if kind.startswith("e4m3") else out
    run_case(sp, 2, 776, 6300, 272, dtype, out, [3, 6221, 6290], True, scaled_integer_operands, True)
    sizes = [0] * 20 + [4900] + [0] * 30
    run_case(sp, len(sizes), 520, 4907, 272, dtype, out, borders(sizes, 7), True, scaled_integer_operands, True)


@pytest.mark.parametrize("kind,n,m,k,cut", [
    ("bf16", 16, 4096, 4096, True), ("bf16", 64, 7168, 7168, True), ("bf16", 33, 4096, 2048, False), ("bf16", 100, 7168, 7168, True),
    ("bf16", 128, 4096, 2048, False), ("bf16", 200, 1024, 8192, True), ("bf16", 200, 4096, 2048, False), ("bf16", 200, 7168, 7168, False),
    ("e4m3", 16, 2048, 4096, True), ("e4m3", 16, 4096, 2048, False), ("e4m3", 33, 7168, 7168, True), ("e4m3", 64, 4096, 2048, False),
    ("e4m3", 128, 4096, 4096, True), ("e4m3", 128, 4096, 2048, False), ("e4m3", 200, 7168, 7168, True), ("e4m3", 512, 4096, 4096, False)])
def test_tiles_are_cut_where_that_is_faster(sp, kind, n, m, k, cut):
    """Sizes at which whole and cut tiles were timed on a B200: pieces are parked in the workspace where cutting won, for each
    width of the operands, and it stays as it is where whole tiles did.  The results are the same up to the order of sums."""
    dtype = None if kind == "e4m3" else torch.bfloat16
    a, sa, b, sb, av, bv = scaled_integer_operands(1, m, n, k, dtype, 5)
    off = None if dtype is None else torch.tensor([0, n], dtype=torch.int32, device="cuda")
    c = torch.full((n, m), 7.0, dtype=torch.bfloat16, device="cuda")
    ws = workspace_for(sp, 1, m, n, k, dtype is None)
    assert call(sp, a, sa, b, sb, c, off, 1, m, n, k, ws) == 0
    check(c, av, bv, None, k, torch.bfloat16, True)
    assert bool(ws.any()) == cut


@pytest.mark.parametrize("eight", [True, False], ids=["e4m3", "fp16"])
def test_as_many_features_as_an_int_holds(sp, eight):
    """2^31 - 8 rows of A of the smallest depth, one token: the same values and sums as with as many tokens."""
    m, n, k = 2 ** 31 - 8, 1, 16 if eight else 8
    free = torch.cuda.mem_get_info()[0]
    if free < 64 << 30:
        pytest.skip("needs 64 GB of device memory, %d GB are free" % (free >> 30))
    a = torch.randint(0, 3 if eight else 2, (m, k), dtype=torch.uint8 if eight else torch.int16, device="cuda", generator=rng(m, k))
    a.mul_(0x38 if eight else 0x3c00)
    a = a.view(torch.float8_e4m3fn if eight else torch.float16)
    b = torch.ones((n, k), device="cuda").to(a.dtype)
    c = torch.full((n, m), 7.0, dtype=torch.float16, device="cuda")
    off = None if eight else torch.tensor([0, n], dtype=torch.int32, device="cuda")
    sa, sb = (torch.ones((kb_of(m), 1), device="cuda"), torch.ones((1, n), device="cuda")) if eight else (None, None)
    assert call(sp, a, sa, b, sb, c, off, 1, m, n, k, workspace_for(sp, 1, m, n, k, eight)) == 0
    assert sp.device_status() == 0
    for first in range(0, m, 1 << 26):
        rows = slice(first, min(m, first + (1 << 26)))
        assert torch.equal(c[0, rows], a[rows].to(torch.float16).sum(1)), first
    del a, b, c, sa, sb
    torch.cuda.empty_cache()


@pytest.mark.parametrize("with_workspace", [True, False], ids=["workspace", "alone"])
@pytest.mark.parametrize("kind,n", [("bf16", 1), ("bf16", 129), ("e4m3", 1)])
def test_as_deep_as_there_may_be(sp, kind, n, with_workspace):
    """The largest K: one accumulation of 2^27 in 16 bits ends before a wait gives up, on one SM and on a pair.  Ones in 64
    places of A, the first and the last among them, and one of 0, 1, -1 in each place of B: sums are exact."""
    eight = kind == "e4m3"
    m, k, dtype = 2, 2 ** 29 if eight else 2 ** 27, torch.float8_e4m3fn if eight else torch.bfloat16
    free = torch.cuda.mem_get_info()[0]
    if free < 48 << 30:
        pytest.skip("needs 48 GB of device memory, %d GB are free" % (free >> 30))
    places = torch.randint(0, k, (62,), device="cuda", generator=rng(k, n)).cpu().tolist() + [0, k - 1]
    one = 0x38 if eight else 0x3f80
    minus = (0x38 | 0x80) if eight else 0x3f80 - 0x8000  # as the stored integer
    bits = torch.uint8 if eight else torch.int16
    a, b = torch.zeros((1, m, k), dtype=bits, device="cuda"), torch.zeros((n, k), dtype=bits, device="cuda")
    a[0, 1, places] = one
    b[:, ::3] = one
    b[:, 1::3] = minus
    a, b = a.view(dtype), b.view(dtype)
    sa, sb = (torch.ones((1, 1, kb_of(k)), device="cuda"), torch.ones((kb_of(k), n), device="cuda")) if eight else (None, None)
    off = None if eight else torch.tensor([0, n], dtype=torch.int32, device="cuda")
    c = torch.full((n, m), 7.0, dtype=torch.bfloat16, device="cuda")
    assert call(sp, a, sa, b, sb, c, off, 1, m, n, k, workspace_for(sp, 1, m, n, k, eight) if with_workspace else None) == 0
    assert sp.device_status() == 0
    assert bool((c[:, 0] == 0).all()) and bool((c[:, 1] == sum((1, -1, 0)[p % 3] for p in set(places))).all())
    del a, b, c, sa, sb
    torch.cuda.empty_cache()
