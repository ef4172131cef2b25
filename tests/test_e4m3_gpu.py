"""GPU tests of the e4m3 quantiser (exact, against float64) and of the block-scaled e4m3 product.

Tolerance of the product, element by element, with S = the sum of the absolute scaled products: a product of two e4m3
values is exact in fp32; a block's sum of 128 is off by at most 128 * 2^-23 of its part of S (one error of 2^-23 per
addition, truncation allowed), the product of two scales by 2^-24, each of the block-wise multiply-adds by 2^-24 of the
running sum; so (128 + blocks + 2) * 2^-23 * S in all, and the bf16 rounding of the result, half a step: 2^-8 of the value."""
import pytest

pytestmark = pytest.mark.gpu


def gen(seed):
    import torch
    return torch.Generator(device="cuda").manual_seed(seed)


def e4m3_of(v):
    """float64 -> the nearest e4m3 value, ties to even, as float64 (|v| <= 448)."""
    import torch
    unit = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))) / 8
    return torch.round(v / unit) * unit


def plain_quantize(x, block_rows):
    """The definition in float64: (values, scales)."""
    import torch
    rows, cols = x.shape
    v = x.double()
    finite = torch.isfinite(v)
    size = torch.where(finite, v.abs(), 0.0)
    size = torch.nn.functional.pad(size, (0, -cols % 128, 0, -rows % block_rows))
    top = size.view(size.shape[0] // block_rows, block_rows, size.shape[1] // 128, 128).amax((1, 3))
    scale = torch.full_like(top, 2.0 ** -126)
    for p in range(-126, 128):  # smallest power of two that holds the block
        scale = torch.where(top > 448.0 * scale, torch.full_like(top, 2.0 ** (p + 1)), scale)
    scale = torch.where(top == 0, 1.0, scale)
    wide = scale.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :cols]
    q = e4m3_of(torch.where(finite, v, 0.0) / wide)
    return torch.where(finite, q, float("nan")), scale


def same(a, b):
    import torch
    return bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


def check_quantize(ctx, x, block_rows, **kw):
    q, s = ctx.quantize_e4m3(x, block_rows, **kw)
    ctx.poll()
    want, scale = plain_quantize(x, block_rows)
    assert s.shape == scale.shape and same(s.double(), scale)
    assert same(q.double(), want)
    return q, s


def spread(g, rows, cols):
    import torch
    x = torch.randn((rows, cols), generator=g, device="cuda")
    return (x * torch.exp2(torch.randint(-20, 20, (rows, 1), generator=g, device="cuda").float())).to(torch.bfloat16)


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8), (1, 128), (3, 127), (2, 129), (128, 128), (129, 136), (127, 1000),
                                       (300, 264), (17, 4104), (5, 4103), (1000, 384), (131, 2049)])
def test_quantize_sizes(ctx, rows, cols, block_rows):
    check_quantize(ctx, spread(gen(rows * 7 + cols), rows, cols), block_rows)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_every_bf16_value(ctx, block_rows):
    """All 65536 bit patterns, NaN, infinities and subnormals among them: as blocks of neighbours (one scale suits all) and
    strided, so that every block spans all magnitudes."""
    import torch
    bits = torch.arange(65536, device="cuda", dtype=torch.int32)
    for order in (bits, bits.view(128, 512).t().reshape(-1)):
        x = (order - 65536 * (order >= 32768)).to(torch.int16).view(torch.bfloat16).view(256, 256)
        check_quantize(ctx, x, block_rows)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_special_blocks(ctx, block_rows):
    import torch
    x = spread(gen(3), 256, 512)
    x[:128, :128] = 0
    x[130, 5] = float("inf")
    x[131, 6] = float("-inf")
    x[132, 7] = float("nan")
    x[133, 128:256] = float("nan")
    x[134, 128:256] = float("inf")
    x[140, :] = 448.0   # exactly on the border of a scale
    x[141, :] = 450.0   # the next bf16 above it
    x[142, :] = 2.0 ** -133
    x[143, :] = 3.3e38
    check_quantize(ctx, x, block_rows)
    x[:] = float("inf")
    check_quantize(ctx, x, block_rows)


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("cols,shift,ldx,ldq", [(264, 0, 272, 272), (264, 3, 272, 270), (261, 1, 263, 265), (256, 8, 272, 264),
                                                (1000, 5, 1011, 1000), (128, 2, 134, 131)])
def test_quantize_strided(ctx, cols, shift, ldx, ldq, block_rows):
    """Any row pitch and alignment, nothing around Q or the scales is touched."""
    import torch
    rows = 131
    x = spread(gen(4), rows, ldx)[:, shift:shift + cols] if shift + cols <= ldx else spread(gen(4), rows, ldx + 8)[:, shift:shift + cols]
    buf = torch.full((rows, ldq + shift), 7.0, device="cuda").to(torch.float8_e4m3fn)
    q = buf[:, shift:shift + cols]
    sr, sc = -(-rows // block_rows), -(-cols // 128)
    sbuf = torch.full((sr, sc + 2), 7.0, device="cuda")
    check_quantize(ctx, x, block_rows, out=q, scales=sbuf[:, 1:1 + sc])
    around = buf.float()
    around[:, shift:shift + cols] = 7.0
    assert (around == 7).all() and (sbuf[:, 0] == 7).all() and (sbuf[:, -1] == 7).all()


def operands(seed, m, n, k, spread_scales=True):
    import torch
    g = gen(seed)
    f8 = torch.float8_e4m3fn
    a = (torch.randn((m, k), generator=g, device="cuda") * 60).clamp(-448, 448).to(f8)
    b = (torch.randn((n, k), generator=g, device="cuda") * 60).clamp(-448, 448).to(f8)
    kb = -(-k // 128)
    sa = torch.rand((m, kb), generator=g, device="cuda") + 0.25
    sb = torch.rand((-(-n // 128), kb), generator=g, device="cuda") + 0.25
    if spread_scales:  # blocks of very different sizes next to each other
        sa *= torch.exp2(torch.randint(-8, 8, sa.shape, generator=g, device="cuda").float())
        sb *= torch.exp2(torch.randint(-8, 8, sb.shape, generator=g, device="cuda").float())
    return a, sa, b, sb


def plain_product(a, sa, b, sb):
    af = a.double() * sa.double().repeat_interleave(128, 1)[:, :a.shape[1]]
    bf = b.double() * sb.double().repeat_interleave(128, 0)[:b.shape[0]].repeat_interleave(128, 1)[:, :b.shape[1]]
    return af @ bf.T, af.abs() @ bf.abs().T


def close(out, ref, size, k, what=""):
    import torch
    blocks = -(-k // 128)
    tol = 2.0 ** -8 * ref.abs() + (1 + 2.0 ** -8) * (128 + blocks + 2) * 2.0 ** -23 * size
    err = (out.double() - ref).abs()
    assert torch.isfinite(out.double()).all(), what
    bad = err > tol
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}, "
                           f"worst ratio {float((err / tol).max()):.3g}")


SHAPES = [(1, 1, 16), (1, 128, 128), (16, 256, 128), (128, 128, 256), (256, 256, 128), (257, 130, 144), (3, 1000, 272),
          (130, 7, 1024), (300, 520, 2064), (64, 384, 128 * 13), (1030, 776, 400), (2500, 2304, 256), (33, 4096, 512),
          (5, 9000, 256), (16, 300, 4096),
          # K over two or four CTAs: one, few and many rows of A, tiles that touch two scale blocks, K not cut evenly
          (1, 4096, 4096), (16, 512, 8192), (17, 500, 2064), (32, 9001, 1040), (33, 700, 8192), (64, 1001, 4096), (65, 1000, 1024),
          (128, 520, 8192), (100, 1001, 4112), (129, 1000, 4000), (300, 1001, 4000), (500, 77, 8192), (1000, 64, 2048),
          (16, 16384, 256), (127, 20000, 128)]


@pytest.fixture
def parts(ctx, request):
    """The number of CTAs that share a tile's K, forced for a test."""
    ctx.set("k_parts", request.param)
    yield request.param
    ctx.set("k_parts", 0)


EVERY_KERNEL = pytest.mark.parametrize("parts", [0, 1, 2, 4], indirect=True)


@EVERY_KERNEL
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product_sizes(ctx, m, n, k, parts):
    a, sa, b, sb = operands(m + n + k, m, n, k)
    out = ctx.gemm_e4m3(a, sa, b, sb)
    ctx.poll()
    ref, size = plain_product(a, sa, b, sb)
    close(out, ref, size, k, f"{m} x {n} x {k}")


@EVERY_KERNEL
@pytest.mark.parametrize("m", [5, 40, 200])
@pytest.mark.parametrize("n,pad", [(264, 8), (264, 6), (257, 7), (257, 3), (100, 4)])
def test_product_strided(ctx, m, n, pad, parts):
    """Padded operands, scales and result; nothing around C is touched."""
    import torch
    k = 272
    a, sa, b, sb = operands(5, m, n, k)
    wide = lambda t, left, right: torch.nn.functional.pad(t.view(torch.uint8) if t.element_size() == 1 else t, (left, right), value=0x7f)  # noqa: E731
    f8 = torch.float8_e4m3fn
    a2, b2 = wide(a, 16, 32).view(f8)[:, 16:16 + k], wide(b, 32, 0).view(f8)[:, 32:32 + k]
    sa2, sb2 = wide(sa, 1, 2)[:, 1:1 + sa.shape[1]], wide(sb, 0, 3)[:, :sb.shape[1]]
    buf = torch.full((m + 2, n + pad), 7.0, dtype=torch.bfloat16, device="cuda")
    out = buf[1:-1, :n]
    ctx.gemm_e4m3(a2, sa2, b2, sb2, out=out)
    ctx.poll()
    ref, size = plain_product(a, sa, b, sb)
    close(out, ref, size, k)
    out.fill_(7.0)
    assert (buf == 7).all()


@EVERY_KERNEL
@pytest.mark.parametrize("m", [7, 50, 300])
def test_nan_stays_in_its_row_and_column(ctx, m, parts):
    import torch
    n, k = 300, 272
    a, sa, b, sb = operands(6, m, n, k)
    a.view(torch.uint8)[3, 200] = 0x7f
    b.view(torch.uint8)[70, 5] = 0x7f
    out = ctx.gemm_e4m3(a, sa, b, sb)
    ctx.poll()
    bad = torch.isnan(out)
    want = torch.zeros_like(bad)
    want[3] = True
    want[:, 70] = True
    assert torch.equal(bad, want)


@EVERY_KERNEL
@pytest.mark.parametrize("m", [2, 300])
def test_extreme_scales(ctx, m, parts):
    """Scales far from one, and zeros, in single blocks."""
    import torch
    n, k = 200, 512
    a, sa, b, sb = operands(7, m, n, k)
    sa[:, 0] *= 2.0 ** 60
    sb[:, 0] *= 2.0 ** -60
    sa[:, 1] = 0
    sb[1, 2] = 0
    out = ctx.gemm_e4m3(a, sa, b, sb)
    ctx.poll()
    ref, size = plain_product(a, sa, b, sb)
    close(out, ref, size, k)


@EVERY_KERNEL
@pytest.mark.parametrize("m", [3, 50, 100, 300])
@pytest.mark.parametrize("kind", ["over", "under", "lost", "mixed"])
def test_scales_whose_product_is_no_normal_number(ctx, m, kind, parts):
    """Each pair of scales times a block's sum is in range, their product alone is not: above 2^128, below 2^-149, or between that and
    2^-126, where it would lose bits.  Beside the tolerance above: half of the smallest bf16 step, 2^-134, and for every block half
    of the smallest fp32 step."""
    import torch
    n, k = 300, 512
    g = gen(91)
    f8 = torch.float8_e4m3fn
    kb = k // 128
    rand = lambda *s: torch.rand(s, generator=g, device="cuda")  # noqa: E731
    a, b = (256 + 192 * rand(m, k)).to(f8), (256 + 192 * rand(n, k)).to(f8)
    sa, sb = 1 + rand(m, kb), 1 + rand(3, kb)
    if kind == "over":
        # block 0: sums of 0; block 1: sums of 2^-9 at least, times 2^130
        a[:, :128] = 0
        sa[:, 0] *= 2.0 ** 100
        sb[:, 0] *= 2.0 ** 60
        a[:, 128:256] = 0
        b[:, 128:256] = 0
        a[:, 130:134] = (2.0 ** -9)
        b[:, 130:134] = (1.0 + rand(n, 4)).to(f8)
        sa[::2, 1] *= 2.0 ** 125
        sa[1::2, 1] *= 2.0 ** 5
        sb[:, 1] *= 2.0 ** 5
        sb[1, 1] *= 2.0 ** -9
    elif kind == "under":   # 2^-152 times sums of 2^24
        sa *= 2.0 ** -100
        sb *= 2.0 ** -52
    elif kind == "lost":    # 2^-145: a product of four bits
        sa *= 2.0 ** -45
        sb *= 2.0 ** -100
    else:                   # every other row, and one block of columns; zeros beside them
        sa[::2] *= 2.0 ** -60
        sa[1::4] = 0
        sa[3::4] *= 2.0 ** -40
        sb[1] *= 2.0 ** -85
        sb[2, 1] = 0
        sb[2, 0] = 2.0 ** 127
    out = ctx.gemm_e4m3(a, sa, b, sb)
    ctx.poll()
    ref, size = plain_product(a, sa, b, sb)
    assert torch.isfinite(out.double()).all()
    tol = 2.0 ** -8 * ref.abs() + (1 + 2.0 ** -8) * (128 + kb + 2) * 2.0 ** -23 * size + 2.0 ** -134 + 2 * kb * 2.0 ** -150
    assert ((out.double() - ref).abs() <= tol).all()
    if parts == 1:  # a row's result does not depend on what stands in the rows beside it
        assert torch.equal(ctx.gemm_e4m3(a[1:2], sa[1:2], b, sb), out[1:2])


@EVERY_KERNEL
@pytest.mark.parametrize("m", [2, 40, 300])
def test_infinite_and_nan_scales(ctx, m, parts):
    """As the formula has it: infinite where a block's sum is not zero, NaN where it is; no other row or column is touched."""
    import torch
    n, k = 300, 512
    f8 = torch.float8_e4m3fn
    a, b = torch.ones((m, k), device="cuda").to(f8), torch.ones((n, k), device="cuda").to(f8)
    sa, sb = torch.ones((m, 4), device="cuda"), torch.ones((3, 4), device="cuda")
    sa[1, 2] = float("inf")
    sb[1, 3] = float("nan")
    out = ctx.gemm_e4m3(a, sa, b, sb).float()
    b.view(torch.uint8)[5, 256:384] = 0
    zero = ctx.gemm_e4m3(a, sa, b, sb).float()
    ctx.poll()
    want = torch.full((m, n), 512.0, device="cuda")
    want[1] = float("inf")
    want[:, 128:256] = float("nan")
    assert same(out, want)
    want[:, 5] = 384.0
    want[1, 5] = float("nan")
    assert same(zero, want)


@pytest.mark.parametrize("m", [1, 16, 300])
def test_quantized_linear_layer(ctx, m):
    """As they are used together: weights quantised once in 128 x 128 blocks, activations row by row, one product; against
    the float64 product of the dequantised operands, and within the quantisation error of the bf16 product."""
    import torch
    g = gen(8)
    n, k = 520, 1040
    x = torch.randn((m, k), generator=g, device="cuda").to(torch.bfloat16)
    w = (torch.randn((n, k), generator=g, device="cuda") * 0.02).to(torch.bfloat16)
    qw, sw = ctx.quantize_e4m3(w, 128)
    qx, sx = ctx.quantize_e4m3(x)
    out = ctx.gemm_e4m3(qx, sx, qw, sw)
    ctx.poll()
    ref, size = plain_product(qx, sx, qw, sw)
    close(out, ref, size, k)
    # each operand moved by at most 2^-4 of itself, or half of the smallest step 2^-9 of its scale
    xd, wd = x.double(), w.double()
    ex = xd.abs() * 2.0 ** -4 + 2.0 ** -10 * sx.double().repeat_interleave(128, 1)[:, :k]
    ew = wd.abs() * 2.0 ** -4 + 2.0 ** -10 * sw.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    bound = ex @ wd.abs().T + xd.abs() @ ew.T + ex @ ew.T
    assert ((ref - xd @ wd.T).abs() <= bound).all()


def test_results_do_not_vary_and_graphs_do_not_meet(ctx):
    """Twice the same, on a side stream, and from two captured graphs replayed at once."""
    import torch
    a, sa, b, sb = operands(9, 300, 520, 1040)
    a2, sa2, b2, sb2 = operands(10, 4, 2056, 1040)
    x = spread(gen(11), 64, 520)
    call = lambda: (ctx.gemm_e4m3(a, sa, b, sb), ctx.gemm_e4m3(a2, sa2, b2, sb2), *ctx.quantize_e4m3(x), *ctx.quantize_e4m3(x, 128))  # noqa: E731
    eq = lambda p, q: all(torch.equal(u.view(torch.uint8), v.view(torch.uint8)) for u, v in zip(p, q))  # noqa: E731
    want = call()
    assert eq(want, call())
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = ctx.gemm_e4m3(a, sa, b, sb, stream=side), ctx.gemm_e4m3(a2, sa2, b2, sb2, stream=side), *ctx.quantize_e4m3(x, stream=side)
    side.synchronize()
    assert eq(got, want[:4])
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(call())
        graphs.append(graph)
    for _ in range(5):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    ctx.poll()
    assert all(eq(o, want) for o in outs)


def test_empty(ctx):
    import torch
    f8 = torch.float8_e4m3fn
    e = lambda *s, d=f8: torch.empty(s, dtype=d, device="cuda")  # noqa: E731
    f = torch.float32
    assert ctx.gemm_e4m3(e(0, 32), e(0, 1, d=f), e(8, 32), e(1, 1, d=f)).shape == (0, 8)
    assert ctx.gemm_e4m3(e(8, 32), e(8, 1, d=f), e(0, 32), e(0, 1, d=f)).shape == (8, 0)
    out = torch.full((3, 5), 7.0, dtype=torch.bfloat16, device="cuda")
    ctx.gemm_e4m3(e(3, 0), e(3, 0, d=f), e(5, 0), e(1, 0, d=f), out=out)
    ctx.poll()
    assert (out == 0).all()
    q, s = ctx.quantize_e4m3(e(0, 64, d=torch.bfloat16))
    assert q.shape == (0, 64) and s.shape == (0, 1)
    q, s = ctx.quantize_e4m3(e(5, 0, d=torch.bfloat16), 128)
    assert q.shape == (5, 0) and s.shape == (1, 0)


def test_refusals(ctx):
    import torch
    import maize_b200
    a, sa, b, sb = operands(12, 16, 256, 128)
    x = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda")
    before = ctx.launch_count
    bad = [
        lambda: ctx.gemm_e4m3(a, sa, b[:, :64], sb),
        lambda: ctx.gemm_e4m3(a, sa[:8], b, sb),
        lambda: ctx.gemm_e4m3(a, sa, b, sb[:1]),
        lambda: ctx.gemm_e4m3(a, sa.double(), b, sb),
        lambda: ctx.gemm_e4m3(a.view(torch.uint8), sa, b, sb),
        lambda: ctx.gemm_e4m3(a.cpu(), sa, b, sb),
        lambda: ctx.gemm_e4m3(a, sa.cpu(), b, sb),
        lambda: ctx.gemm_e4m3(a, sa, b, sb, out=torch.zeros((16, 255), dtype=torch.bfloat16, device="cuda")),
        lambda: ctx.gemm_e4m3(a, sa, b, sb, out=torch.zeros((16, 256), device="cuda")),
        lambda: ctx.gemm_e4m3(a[:, :120], sa, b[:, :120], sb),      # K no multiple of 16
        lambda: ctx.gemm_e4m3(a[:, 8:120], sa, b[:, 8:120], sb),    # not 16-byte aligned
        lambda: ctx.quantize_e4m3(x, 2),
        lambda: ctx.quantize_e4m3(x.float()),
        lambda: ctx.quantize_e4m3(x.cpu()),
        lambda: ctx.quantize_e4m3(x.t()),
        lambda: ctx.quantize_e4m3(x, out=torch.zeros((4, 64), device="cuda")),
        lambda: ctx.quantize_e4m3(x, scales=torch.zeros((4, 2), device="cuda")),
    ]
    for call in bad:
        with pytest.raises(maize_b200.MaizeError) as e:
            call()
        assert e.value.status in (maize_b200._ffi.INVALID_ARG, maize_b200._ffi.UNSUPPORTED)
    assert ctx.launch_count == before


@EVERY_KERNEL
@pytest.mark.parametrize("ctas", [1, 2, 5, 20])
def test_few_ctas_many_rounds(ctx, ctas, parts):
    """A limit on the CTAs makes every one of them go through many tiles, with odd and even numbers of k-blocks."""
    ctx.set("max_ctas", ctas)
    try:
        for m, n, k in ((600, 1000, 400), (300, 777, 128), (20, 2000, 1040), (50, 1500, 640), (1030, 520, 256)):
            a, sa, b, sb = operands(m + n + k, m, n, k)
            ref, size = plain_product(a, sa, b, sb)
            close(ctx.gemm_e4m3(a, sa, b, sb), ref, size, k, f"{m} {n} {k}")
        ctx.poll()
    finally:
        ctx.set("max_ctas", 0)


@pytest.mark.parametrize("parts", [1], indirect=True)
@pytest.mark.parametrize("k", [16, 128, 272])
@pytest.mark.parametrize("m,n,ctas", [(1030, 520, 2), (2048, 1032, 4), (1000, 1080, 6), (600, 904, 2), (520, 1856, 2), (4096, 4104, 0),
                                      (8192, 8200, 0), (8192, 8256, 0)])
def test_edge_tiles_between_whole_ones(ctx, m, n, ctas, k, parts):
    """Short sums, so that a tile's stores are still on their way when the next tile's begin; the last columns are half a tile's or
    less (N % 128 of 8 to 64), so that a warp has one store there and two in the tiles before and after."""
    import torch
    a, sa, b, sb = operands(m + n + k, m, n, k)
    ref, size = plain_product(a, sa, b, sb)
    ctx.set("max_ctas", ctas)
    try:
        first = ctx.gemm_e4m3(a, sa, b, sb)
        close(first, ref, size, k, f"{m} x {n} x {k}")
        outs = [torch.empty_like(first) for _ in range(4)]
        for _ in range(10):
            for out in outs:
                ctx.gemm_e4m3(a, sa, b, sb, out=out.fill_(7.0))
            assert all(torch.equal(out, first) for out in outs)
        ctx.poll()
    finally:
        ctx.set("max_ctas", 0)


@EVERY_KERNEL
def test_product_past_32_bits(ctx, parts):
    """The last rows of operands and of a result that lie more than 2^32 bytes behind the start."""
    import torch
    f8 = torch.float8_e4m3fn
    for m, n, k in ((300_000, 8193, 144), (270_001, 40, 16_384), (40, 270_001, 16_384)):  # C, A, B beyond 4 GiB
        a, sa, b, sb = operands(71, 40 if m > 40 else m, 40 if n > 8193 else n, k, False)
        if m > 40:
            big = torch.zeros((m, k), dtype=torch.uint8, device="cuda").view(f8)
            big[-40:] = a
            big_s = torch.ones((m, sa.shape[1]), device="cuda")
            big_s[-40:] = sa
            out = ctx.gemm_e4m3(big, big_s, b, sb)[-40:]
        elif n > 8193:
            # rows of B in two scale blocks: the last 40 start inside the block before the last
            big = torch.zeros((n, k), dtype=torch.uint8, device="cuda").view(f8)
            big[-40:] = b
            big_s = torch.ones((-(-n // 128), sb.shape[1]), device="cuda")
            out = ctx.gemm_e4m3(a, sa, big, big_s)[:, -40:]
            sb = torch.ones_like(sb)
        ctx.poll()
        ref, size = plain_product(a, sa, b, sb)
        close(out, ref, size, k, f"{m} {n} {k}")
        del big, big_s, out


@EVERY_KERNEL
@pytest.mark.parametrize("m", [1, 16, 48, 100])
def test_operands_written_by_the_call_before(ctx, m, parts):
    """Quantiser and product one behind the other, the same buffers again and again: no product sees the values before."""
    import torch
    g = gen(81)
    n, k, rounds = 1000, 4096, 12
    xs = [torch.randn((m, k), generator=g, device="cuda").to(torch.bfloat16) for _ in range(rounds)]
    ws = [(torch.randn((n, k), generator=g, device="cuda") * 2.0 ** (i % 5)).to(torch.bfloat16) for i in range(rounds)]
    want = []
    for x, w in zip(xs, ws):
        given = *ctx.quantize_e4m3(x), *ctx.quantize_e4m3(w, 128)
        torch.cuda.synchronize()
        want.append(ctx.gemm_e4m3(*given))
        torch.cuda.synchronize()
    qx, sx = ctx.quantize_e4m3(xs[0])
    qw, sw = ctx.quantize_e4m3(ws[0], 128)
    torch.cuda.synchronize()
    for order in (0, 1):  # the weights, then the rows of A, quantised last
        got = []
        for x, w in zip(xs, ws):
            for last in (order, 1 - order):
                if last:
                    ctx.quantize_e4m3(w, 128, out=qw, scales=sw)
                else:
                    ctx.quantize_e4m3(x, out=qx, scales=sx)
            got.append(ctx.gemm_e4m3(qx, sx, qw, sw))
        ctx.poll()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("parts", [0, 1, 4], indirect=True)
@pytest.mark.parametrize("first", ["gemm", "grouped_gemm", "gemm_e4m3"])
@pytest.mark.parametrize("m,k", [(4, 2048), (64, 1040), (300, 2056)])
def test_chain_of_products_and_quantisers(ctx, m, k, first, parts):
    """Product -> quantiser -> product -> quantiser (by rows and by blocks) -> product over the same buffers again and again, eager
    and from a captured graph: every call reads what the one right before it wrote, at the values that a chain with a
    synchronisation behind each call gives.  The rounds' sizes differ by powers of two, so that a stale scale shows."""
    import torch
    g = gen(82)
    n, inner, rounds = 1040, 512, 8
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    k16 = k // 16 * 16  # of X's columns, what the products by e4m3 take
    us = [(rand(m, inner) * 2.0 ** (3 * i % 7)).to(torch.bfloat16) for i in range(rounds)]
    v = rand(k, inner).to(torch.bfloat16)
    qw, sw = ctx.quantize_e4m3(rand(n, k16).to(torch.bfloat16), 128)
    qv, sv = ctx.quantize_e4m3(v, 128)
    qus = [ctx.quantize_e4m3(u) for u in us]
    offsets = torch.tensor([0, m // 2, m], dtype=torch.int32, device="cuda")
    stack = torch.stack([v, v.flip(0)])
    torch.cuda.synchronize()
    f8, f32 = torch.float8_e4m3fn, torch.float32
    new = lambda *s, d=torch.bfloat16: torch.zeros(s, dtype=d, device="cuda")  # noqa: E731
    x, y = new(m, k), new(m, n)
    qx, sx = new(m, k16, d=f8), new(m, -(-k16 // 128), d=f32)
    qy, sy, qb, sb = new(m, n, d=f8), new(m, -(-n // 128), d=f32), new(m, n, d=f8), new(-(-m // 128), -(-n // 128), d=f32)
    held = [new(m, m) for _ in range(rounds)]

    def one(i, wait=lambda: None):
        if first == "gemm":
            ctx.gemm(us[i], v, out=x)
        elif first == "grouped_gemm":
            ctx.grouped_gemm(us[i], stack, offsets, out=x)
        else:
            ctx.gemm_e4m3(*qus[i], qv, sv, out=x)
        wait()
        ctx.quantize_e4m3(x[:, :k16], out=qx, scales=sx)
        wait()
        ctx.gemm_e4m3(qx, sx, qw, sw, out=y)
        wait()
        ctx.quantize_e4m3(y, 128, out=qb, scales=sb)
        wait()
        ctx.quantize_e4m3(y, out=qy, scales=sy)
        wait()
        ctx.gemm_e4m3(qy, sy, qb, sb, out=held[i])
        wait()
        return held[i]

    want = []
    for i in range(rounds):
        want.append(one(i, torch.cuda.synchronize).clone())
        torch.cuda.synchronize()
    assert len({float(w.float().abs().max()) for w in want}) == rounds
    right = lambda: all(torch.equal(h, w) for h, w in zip(held, want))  # noqa: E731
    for _ in range(6):
        for h in held:
            h.zero_()
        for i in range(rounds):
            one(i)
        ctx.poll()
        assert right()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for i in range(rounds):
            one(i)
    for _ in range(6):
        for h in held:
            h.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert right()
    ctx.poll()


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("cols", [16_384, 16_391])
def test_quantize_past_32_bits(ctx, cols, block_rows):
    import torch
    rows = 270_000
    x = torch.zeros((rows, cols), dtype=torch.bfloat16, device="cuda")
    tail = rows % 128  # whole blocks of 128 rows before it
    x[-tail:] = spread(gen(72), tail, cols)
    q, s = ctx.quantize_e4m3(x, block_rows)
    ctx.poll()
    want, scale = plain_quantize(x[-tail:], block_rows)
    assert same(s[-scale.shape[0]:].double(), scale) and same(q[-tail:].double(), want)
    assert (s[:-scale.shape[0]] == 1).all() and not q[:256].view(torch.uint8).any()


def test_module_functions(ctx):
    import torch
    import maize_b200
    a, sa, b, sb = operands(13, 20, 300, 144)
    assert torch.equal(maize_b200.gemm_e4m3(a, sa, b, sb), ctx.gemm_e4m3(a, sa, b, sb))
    x = spread(gen(14), 9, 300)
    q, s = maize_b200.quantize_e4m3(x, block_rows=128)
    want, scale = plain_quantize(x, 128)
    assert same(q.double(), want) and same(s.double(), scale)
