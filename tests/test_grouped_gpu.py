"""GPU tests of the grouped (expert) products against plain float64 products, group by group.

Tolerance, element by element: the bf16 rounding of the result, half a step (2^-8 of the value), plus the fp32 sums.  A
sum of K products accumulated in fp32 with one error of at most 2^-23 of the running sum's bound per addition (truncation
allowed) is off by at most K * 2^-23 * sum |a_i b_i|; the rounding of a value that is off by that adds a factor 1 + 2^-8."""
import pytest

pytestmark = pytest.mark.gpu


def bf16(gen, shape, scale=1.0):
    import torch
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(torch.bfloat16)


def gen(seed):
    import torch
    return torch.Generator(device="cuda").manual_seed(seed)


def offsets_of(sizes, first=0):
    import torch
    o = [first]
    for s in sizes:
        o.append(o[-1] + s)
    return torch.tensor(o, dtype=torch.int32, device="cuda")


def close(got, ref, size, terms, what=""):
    """`size` = sum of the products' absolute values, `terms` = their number (both may be tensors)."""
    import torch
    err = (got.double() - ref).abs()
    tol = 2.0 ** -8 * ref.abs() + (1 + 2.0 ** -8) * terms * 2.0 ** -23 * size
    assert torch.isfinite(got.double()).all(), f"{what}: not finite"
    bad = err > tol
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} elements off, first at {bad.nonzero()[0].tolist()}, "
                           f"worst excess {float((err - tol).max()):.3g}")


def plain_grouped(a, w, o, kn):
    """Rows of each group times its matrix in float64; (result, sum of absolute products)."""
    import torch
    n = w.shape[2] if kn else w.shape[1]
    ref = torch.zeros((a.shape[0], n), dtype=torch.float64, device="cuda")
    size = torch.zeros_like(ref)
    o = o.tolist()
    for g in range(w.shape[0]):
        x, m = a[o[g]:o[g + 1]].double(), w[g].double()
        m = m if kn else m.T
        ref[o[g]:o[g + 1]] = x @ m
        size[o[g]:o[g + 1]] = x.abs() @ m.abs()
    return ref, size


def check_grouped(ctx, sizes, n, k, kn, seed=1, first=0, behind=0):
    import torch
    g = gen(seed)
    rows = first + sum(sizes) + behind
    a = bf16(g, (rows, k))
    w = bf16(g, (len(sizes), k, n) if kn else (len(sizes), n, k), 0.1)
    o = offsets_of(sizes, first)
    # rows outside the groups: their content may not matter, their rows of C stay as they were
    a[:first] = float("nan")
    a[first + sum(sizes):] = float("inf")
    out = torch.full((rows, n), 7.0, dtype=torch.bfloat16, device="cuda")
    (ctx.grouped_gemm_kn if kn else ctx.grouped_gemm)(a, w, o, out=out)
    ctx.poll()
    inside = slice(first, first + sum(sizes))
    ref, size = plain_grouped(a, w, o, kn)
    close(out[inside], ref[inside], size[inside], k, f"{sizes} n {n} k {k} kn {kn}")
    assert (out[:first] == 7).all() and (out[first + sum(sizes):] == 7).all()
    return out


SIZES = [
    [1], [128], [256], [257], [0, 1, 0], [3, 0, 5, 64], [256, 257, 255, 1, 0, 33], [31, 32, 33], [15, 16, 17, 0, 0],
    [700], [0, 0, 513, 1], [1] * 70, [2, 40, 0, 100] * 12,
]


@pytest.fixture
def parts(ctx, request):
    """The number of CTAs that share a tile's K, forced for a test."""
    ctx.set("k_parts", request.param)
    yield request.param
    ctx.set("k_parts", 0)


EVERY_KERNEL = pytest.mark.parametrize("parts", [0, 1, 2, 4, 8], indirect=True)


@EVERY_KERNEL
@pytest.mark.parametrize("kn", [False, True])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "-".join(map(str, s[:7])))
def test_group_sizes(ctx, sizes, kn, parts):
    check_grouped(ctx, sizes, 520, 264, kn)


@EVERY_KERNEL
@pytest.mark.parametrize("kn", [False, True])
@pytest.mark.parametrize("n,k", [(8, 8), (256, 64), (256, 384), (40, 8), (264, 520), (2048, 72), (512, 2056), (136, 64 * 21)])
def test_matrix_sizes(ctx, n, k, kn, parts):
    check_grouped(ctx, [5, 300, 0, 33], n, k, kn, seed=2)


@EVERY_KERNEL
@pytest.mark.parametrize("n", [1, 7, 31, 33, 257, 1031])
def test_odd_result_rows(ctx, n, parts):
    """C needs no alignment: odd N, where B is N x K."""
    check_grouped(ctx, [5, 70, 0, 33], n, 136, False, seed=3)


@EVERY_KERNEL
@pytest.mark.parametrize("k", [1, 3, 63, 65, 127])
def test_any_k_where_b_is_k_by_n(ctx, k, parts):
    """K x N matrices: K is free as long as the rows' pitch is a multiple of 8."""
    import torch
    g = gen(4)
    sizes, n = [9, 0, 40], 72
    a = bf16(g, (49, 128))
    a[:, k:] = float("nan")  # what lies behind a row's end takes no part
    a = a[:, :k]
    w = bf16(g, (3, k, n), 0.1)
    o = offsets_of(sizes)
    out = ctx.grouped_gemm_kn(a, w, o)
    ctx.poll()
    ref, size = plain_grouped(a, w, o, True)
    close(out, ref, size, k)


@EVERY_KERNEL
@pytest.mark.parametrize("kn", [False, True])
def test_rows_outside_the_groups_stay(ctx, kn, parts):
    check_grouped(ctx, [30, 0, 41], 256, 128, kn, seed=5, first=3, behind=500)
    check_grouped(ctx, [0, 0], 256, 128, kn, seed=5, first=2, behind=9)


@EVERY_KERNEL
@pytest.mark.parametrize("kn", [False, True])
def test_other_groups_values_do_not_leak(ctx, kn, parts):
    """One group's rows or weights are NaN or infinite: the other groups' results do not change."""
    import torch
    g = gen(6)
    sizes, n, k = [70, 50, 60], 200, 136
    a = bf16(g, (180, k))
    w = bf16(g, (3, k, n) if kn else (3, n, k), 0.1)
    o = offsets_of(sizes)
    f = ctx.grouped_gemm_kn if kn else ctx.grouped_gemm
    clean = f(a, w, o)
    a[70:120] = float("nan")
    w[1] = float("inf")
    out = f(a, w, o)
    ctx.poll()
    assert torch.equal(out[:70], clean[:70]) and torch.equal(out[120:], clean[120:])
    assert not torch.isfinite(out[70:120].float()).any()


@EVERY_KERNEL
@pytest.mark.parametrize("kn", [False, True])
def test_strided_operands(ctx, kn, parts):
    """Padded rows of A, C and the weights, and matrices with a gap between them; nothing around C is touched."""
    import torch
    g = gen(7)
    sizes, n, k = [33, 0, 90, 7], 264, 200
    rows = sum(sizes)
    a = bf16(g, (rows, k + 24))[:, 8:8 + k]
    wr, wc = (k, n) if kn else (n, k)
    w = bf16(g, (4, wr + 5, wc + 16), 0.1)[:, :wr, :wc]
    o = offsets_of(sizes)
    ref, size = plain_grouped(a, w, o, kn)
    for pad, shift in ((8, 0), (6, 2), (3, 1)):  # 16-byte rows, 4-byte rows, odd rows
        buf = torch.full((rows + 2, n + pad), 7.0, dtype=torch.bfloat16, device="cuda")
        out = buf[1:-1, shift:shift + n]
        (ctx.grouped_gemm_kn if kn else ctx.grouped_gemm)(a, w, o, out=out)
        ctx.poll()
        close(out, ref, size, k, f"pad {pad}")
        out.fill_(7.0)
        assert (buf == 7).all()


@pytest.mark.parametrize("kn", [False, True])
def test_large_ragged(ctx, kn):
    check_grouped(ctx, [1000, 17, 0, 2100, 300, 5, 689], 2056, 1032, kn, seed=8)


@EVERY_KERNEL
def test_many_tiles_per_cta(ctx, parts):
    """More tiles than clusters: accumulator buffers, the exchange and their phases go round."""
    check_grouped(ctx, [200, 3, 0, 129, 64] * 4, 1032, 328, False, seed=9)
    check_grouped(ctx, [70] * 40, 776, 72, True, seed=10)


@pytest.mark.parametrize("sizes", [[8], [2, 2, 2, 1, 1], [26, 26, 26], [0, 0, 1, 0]])
def test_few_rows_long_k(ctx, sizes):
    """The sizes that K is split for by itself."""
    check_grouped(ctx, sizes, 144, 6936, False, seed=11)
    check_grouped(ctx, sizes, 144, 6936, True, seed=12)


def test_empty_sum_clears_the_groups_rows(ctx):
    import torch
    a = torch.empty((20, 0), dtype=torch.bfloat16, device="cuda")
    w = torch.empty((2, 24, 0), dtype=torch.bfloat16, device="cuda")
    out = torch.full((20, 24), 7.0, dtype=torch.bfloat16, device="cuda")
    ctx.grouped_gemm(a, w, offsets_of([3, 9], first=2), out=out)
    ctx.poll()
    assert (out[2:14] == 0).all() and (out[:2] == 7).all() and (out[14:] == 7).all()


def test_nothing_to_do(ctx):
    import torch
    w = torch.zeros((2, 24, 16), dtype=torch.bfloat16, device="cuda")
    assert ctx.grouped_gemm(torch.empty((0, 16), dtype=torch.bfloat16, device="cuda"), w, offsets_of([0, 0])).shape == (0, 24)
    none = torch.empty((0, 24, 16), dtype=torch.bfloat16, device="cuda")
    out = torch.full((5, 24), 7.0, dtype=torch.bfloat16, device="cuda")
    ctx.grouped_gemm(torch.zeros((5, 16), dtype=torch.bfloat16, device="cuda"), none, offsets_of([]), out=out)
    ctx.poll()
    assert (out == 7).all()


def test_results_do_not_vary(ctx):
    import torch
    g = gen(9)
    sizes = [400, 3, 0, 130]
    a, w, dy = bf16(g, (533, 264)), bf16(g, (4, 520, 264)), bf16(g, (533, 520))
    o = offsets_of(sizes)
    first = ctx.grouped_gemm(a, w, o), ctx.grouped_gemm_wgrad(a, dy, o)
    for _ in range(3):
        again = ctx.grouped_gemm(a, w, o), ctx.grouped_gemm_wgrad(a, dy, o)
        assert all(torch.equal(x, y) for x, y in zip(first, again))
    ctx.poll()


# ------------------------------------------------------------- weight gradient --
def check_wgrad(ctx, sizes, n, k, seed=11, first=0, behind=0):
    import torch
    g = gen(seed)
    rows = first + sum(sizes) + behind
    a, dy = bf16(g, (rows, k)), bf16(g, (rows, n), 0.1)
    o = offsets_of(sizes, first)
    # a block of 64 rows that crosses the end of the groups meets these
    for t in (a, dy):
        t[:first] = float("nan")
        t[first + sum(sizes):] = float("inf")
    out = ctx.grouped_gemm_wgrad(a, dy, o)
    ctx.poll()
    at = first
    for i, s in enumerate(sizes):
        x, y = a[at:at + s].double(), dy[at:at + s].double()
        close(out[i], y.T @ x, y.abs().T @ x.abs(), max(s, 1), f"{sizes} group {i} n {n} k {k}")
        if s == 0:
            assert (out[i] == 0).all()
        at += s


@EVERY_KERNEL
@pytest.mark.parametrize("sizes", SIZES + [[64, 128, 192], [16, 32, 48], [63, 65, 127, 1], [320, 0, 321, 15]],
                         ids=lambda s: "-".join(map(str, s[:7])))
def test_wgrad_group_sizes(ctx, sizes, parts):
    check_wgrad(ctx, sizes, 264, 520, behind=70)


@EVERY_KERNEL
@pytest.mark.parametrize("n,k", [(8, 8), (256, 256), (256, 64), (64, 256), (40, 264), (1032, 72), (776, 2056)])
def test_wgrad_matrix_sizes(ctx, n, k, parts):
    check_wgrad(ctx, [5, 300, 0, 33], n, k, seed=12, first=3)


@EVERY_KERNEL
def test_wgrad_neighbours_do_not_leak(ctx, parts):
    """Rows of the next group are infinite or NaN in both operands: a block that crosses the border drops them."""
    import torch
    g = gen(13)
    a, dy = bf16(g, (150, 136)), bf16(g, (150, 264))
    o = offsets_of([37, 70, 43])
    clean = ctx.grouped_gemm_wgrad(a, dy, o)
    a[37:107] = float("inf")
    dy[37:107] = float("nan")
    out = ctx.grouped_gemm_wgrad(a, dy, o)
    ctx.poll()
    assert torch.equal(out[0], clean[0]) and torch.equal(out[2], clean[2])


@EVERY_KERNEL
@pytest.mark.parametrize("n,k", [(264, 200), (33, 57)])
def test_wgrad_strided(ctx, n, k, parts):
    """Padded operand rows; results with 16-byte rows (TMA stores), odd rows (plain stores) and gaps between matrices."""
    import torch
    g = gen(14)
    sizes = [33, 0, 90, 7]
    a = bf16(g, (130, 272))[:, 8:8 + k]
    dy = bf16(g, (130, 288), 0.1)[:, 16:16 + n]
    o = offsets_of(sizes)
    for pad, extra, shift in ((8, 2, 0), (8, 0, 0), (3, 1, 1)):
        width = -(-k // 8) * 8 + pad
        buf = torch.full((4, n + extra, width), 7.0, dtype=torch.bfloat16, device="cuda")
        out = buf[:, :n, shift:shift + k]
        ctx.grouped_gemm_wgrad(a, dy, o, out=out)
        ctx.poll()
        at = 0
        for i, s in enumerate(sizes):
            x, y = a[at:at + s].double(), dy[at:at + s].double()
            close(out[i], y.T @ x, y.abs().T @ x.abs(), max(s, 1), f"pad {pad} group {i}")
            at += s
        out.fill_(7.0)
        assert (buf == 7).all()


def test_wgrad_of_one_long_group(ctx):
    """The sizes that the rows are split for by themselves."""
    check_wgrad(ctx, [5003], 136, 544, seed=15)
    check_wgrad(ctx, [2100, 0, 900], 200, 104, seed=16, first=7, behind=9)


@EVERY_KERNEL
def test_wgrad_many_tiles_per_cta(ctx, parts):
    check_wgrad(ctx, [200, 3, 0, 129, 64] * 4, 520, 776, seed=17)


def test_wgrad_without_rows_is_zero(ctx):
    import torch
    e = torch.empty((0, 16), dtype=torch.bfloat16, device="cuda")
    out = torch.full((3, 16, 16), 7.0, dtype=torch.bfloat16, device="cuda")
    ctx.grouped_gemm_wgrad(e, e, offsets_of([0, 0, 0]), out=out)
    ctx.poll()
    assert (out == 0).all()


# ------------------------------------------------------------------ as they are used --
def test_expert_layer_forward_and_backward(ctx):
    """Two grouped products with a gate between them, forward and backward, against float64 autograd."""
    import torch
    g = gen(21)
    sizes, d, h = [70, 0, 129, 41], 136, 264
    rows = sum(sizes)
    o = offsets_of(sizes)
    x, up, down = bf16(g, (rows, d)), bf16(g, (4, h, d), 0.1), bf16(g, (4, d, h), 0.1)
    dy = bf16(g, (rows, d))
    mid = ctx.grouped_gemm(x, up, o)
    act = torch.relu(mid)
    y = ctx.grouped_gemm(act, down, o)
    d_act = ctx.grouped_gemm_kn(dy, down, o)
    d_down = ctx.grouped_gemm_wgrad(act, dy, o)
    d_mid = torch.where(mid > 0, d_act, 0)
    d_x = ctx.grouped_gemm_kn(d_mid, up, o)
    d_up = ctx.grouped_gemm_wgrad(x, d_mid, o)
    ctx.poll()
    at = 0
    for i, s in enumerate(sizes):
        r = slice(at, at + s)
        at += s
        xx, uu, dd = (t.double().requires_grad_() for t in (x[r], up[i], down[i]))
        m = xx @ uu.T
        # the layer's own roundings are the operands of its next product: they are put in, and pass gradients through
        m_r = m + (mid[r].double() - m).detach()
        a_r = torch.relu(m_r)
        (a_r @ dd.T).backward(dy[r].double())
        close(y[r], (a_r @ dd.T).detach(), a_r.detach().abs() @ dd.detach().abs().T, h, "y")
        close(d_down[i], dd.grad, dy[r].double().abs().T @ a_r.detach().abs(), max(s, 1), "d_down")
        # d_mid was rounded to bf16 (2^-8 of each) before the last two products
        size = d_mid[r].double().abs() @ uu.detach().abs()
        tol = 2.0 ** -8 * (xx.grad.abs() + size) + 2 * (h + d) * 2.0 ** -23 * size + 1e-30
        carried = (dy[r].double().abs() @ dd.detach().abs()) @ uu.detach().abs() * (d * 2.0 ** -23)
        assert ((d_x[r].double() - xx.grad).abs() <= tol * (1 + 2.0 ** -7) + carried).all()
        size = d_mid[r].double().abs().T @ xx.detach().abs()
        carried = (dy[r].double().abs() @ dd.detach().abs()).T @ xx.detach().abs() * (d * 2.0 ** -23)
        tol = 2.0 ** -8 * (uu.grad.abs() + size) + 2 * (s + d) * 2.0 ** -23 * size + 1e-30
        assert ((d_up[i].double() - uu.grad).abs() <= tol * (1 + 2.0 ** -7) + carried).all()


def test_gradients_against_differences(ctx):
    """The input's and the weights' gradients predict how a scalar of the forward product changes along a direction."""
    import torch
    g = gen(22)
    sizes, n, k = [40, 0, 23], 64, 72
    o = offsets_of(sizes)
    x, w, dy = bf16(g, (63, k)), bf16(g, (3, n, k), 0.2), bf16(g, (63, n))
    dx, dw = ctx.grouped_gemm_kn(dy, w, o).double(), ctx.grouped_gemm_wgrad(x, dy, o).double()
    ctx.poll()

    def f(x, w):
        at, total = 0, 0.0
        for i, s in enumerate(sizes):
            total = total + ((x[at:at + s] @ w[i].T) * dy[at:at + s].double()).sum()
            at += s
        return total

    vx, vw = bf16(g, x.shape).double(), bf16(g, w.shape).double()
    eps = 2.0 ** -10
    for grad, v, diff in ((dx, vx, (f(x.double() + eps * vx, w.double()) - f(x.double() - eps * vx, w.double())) / (2 * eps)),
                          (dw, vw, (f(x.double(), w.double() + eps * vw) - f(x.double(), w.double() - eps * vw)) / (2 * eps))):
        # f is linear in each argument: the difference is exact but for float64; the gradients carry 2^-8 each, and fp32 sums
        assert abs(float((grad * v).sum() - diff)) <= (2.0 ** -8 + 72 * 2.0 ** -20) * float((grad * v).abs().sum())


def test_other_stream_and_graphs(ctx):
    """Calls on a side stream, and two captured graphs replayed at the same time, give what the default stream gives."""
    import torch
    g = gen(23)
    o = offsets_of([30, 0, 100, 3])
    x, w, dy = bf16(g, (133, 264)), bf16(g, (4, 520, 264)), bf16(g, (133, 520))
    want = ctx.grouped_gemm(x, w, o), ctx.grouped_gemm_kn(dy, w, o), ctx.grouped_gemm_wgrad(x, dy, o)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = ctx.grouped_gemm(x, w, o, stream=side), ctx.grouped_gemm_kn(dy, w, o, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append((ctx.grouped_gemm(x, w, o), ctx.grouped_gemm_kn(dy, w, o), ctx.grouped_gemm_wgrad(x, dy, o)))
        graphs.append(graph)
    for _ in range(5):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    # the graphs read the offsets when they run: other group sizes, same graph
    o.copy_(offsets_of([0, 64, 1, 68]))
    graphs[0].replay()
    torch.cuda.synchronize()
    again = ctx.grouped_gemm(x, w, o), ctx.grouped_gemm_kn(dy, w, o), ctx.grouped_gemm_wgrad(x, dy, o)
    ctx.poll()
    assert all(torch.equal(a, b) for a, b in zip(outs[0], again))


@EVERY_KERNEL
@pytest.mark.parametrize("bad", [[0, 5, 4, 10], [0, 5, 8, 11], [-1, 2, 3, 4]])
def test_wrong_offsets_are_reported(ctx, bad, parts):
    """Offsets that descend or leave the rows: the kernels' own check reports them, nothing is written."""
    import torch
    import maize_b200
    x, w = torch.ones((10, 16), dtype=torch.bfloat16, device="cuda"), torch.ones((3, 24, 16), dtype=torch.bfloat16, device="cuda")
    o = torch.tensor(bad, dtype=torch.int32, device="cuda")
    out = torch.full((10, 24), 7.0, dtype=torch.bfloat16, device="cuda")
    dw = torch.full((3, 24, 16), 7.0, dtype=torch.bfloat16, device="cuda")
    for call in (lambda: ctx.grouped_gemm(x, w, o, out=out), lambda: ctx.grouped_gemm_wgrad(x, out, o, out=dw)):
        call()
        with pytest.raises(maize_b200.MaizeError) as e:
            ctx.poll()
        assert e.value.status == maize_b200._ffi.DEVICE_ABORT
    assert (out == 7).all() and (dw == 7).all()
    ctx.poll()


def test_refusals(ctx):
    """What is refused on the host: nothing is launched."""
    import torch
    import maize_b200
    t = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    o = offsets_of([4, 6])
    before = ctx.launch_count
    bad = [
        lambda: ctx.grouped_gemm(t(10, 16), t(2, 24, 8), o),                        # K differs
        lambda: ctx.grouped_gemm(t(10, 16), t(3, 24, 16), o),                       # offsets for other groups
        lambda: ctx.grouped_gemm(t(10, 16), t(2, 24, 16), o.long()),                # offsets of another type
        lambda: ctx.grouped_gemm(t(10, 16), t(2, 24, 16), o.cpu()),
        lambda: ctx.grouped_gemm(t(10, 16).float(), t(2, 24, 16), o),
        lambda: ctx.grouped_gemm(t(10, 16), t(24, 16), o),
        lambda: ctx.grouped_gemm(t(16, 10).T, t(2, 24, 16), o),                     # columns not contiguous
        lambda: ctx.grouped_gemm(t(10, 16), t(2, 24, 16), o, out=t(10, 23)),
        lambda: ctx.grouped_gemm(t(10, 16).cpu(), t(2, 24, 16), o),
        lambda: ctx.grouped_gemm(t(10, 12), t(2, 24, 12), o),                       # K no multiple of 8
        lambda: ctx.grouped_gemm(t(10, 24)[:, 4:20], t(2, 24, 16), o),              # A not 16-byte aligned
        lambda: ctx.grouped_gemm(t(10, 16), t(1, 24, 16).expand(2, 24, 16), o),     # overlapping matrices
        lambda: ctx.grouped_gemm_kn(t(10, 16), t(2, 16, 20), o),                    # N no multiple of 8
        lambda: ctx.grouped_gemm_wgrad(t(10, 16), t(9, 24), o),
        lambda: ctx.grouped_gemm_wgrad(t(10, 12), t(10, 24), o),
        lambda: ctx.grouped_gemm_wgrad(t(10, 16), t(10, 24), o, out=t(2, 16, 24)),
        lambda: ctx.grouped_gemm(t(10, 16), t(1025, 8, 16), offsets_of([0] * 1025)),
    ]
    for call in bad:
        with pytest.raises(maize_b200.MaizeError) as e:
            call()
        assert e.value.status in (maize_b200._ffi.INVALID_ARG, maize_b200._ffi.UNSUPPORTED)
    assert ctx.launch_count == before


def test_most_groups(ctx):
    """1024 groups, most of them empty."""
    sizes = [0] * 1024
    for i in range(0, 1024, 37):
        sizes[i] = 1 + i % 5
    check_grouped(ctx, sizes, 40, 24, False, seed=31)
    check_wgrad(ctx, sizes, 40, 24, seed=32)


@EVERY_KERNEL
@pytest.mark.parametrize("sizes", [
    [(37 * i) % 200 for i in range(90)],                       # all different, some empty, several rounds of tiles
    [0, 0, 300, 0, 1, 0, 0, 129, 0] * 10,                      # the same sizes again and again: ties in the order
    [0] * 500 + [70] + [0] * 400 + [500, 1] + [0] * 121,       # 1024 groups, three with rows
    [64 * (1 << i) + d for i in range(6) for d in (-1, 0, 1)], # around the borders between the classes
], ids=["different", "ties", "sparse", "borders"])
def test_order_of_uneven_groups(ctx, parts, sizes):
    """The groups are listed, and for the weight gradient sorted, by their rows: every one is still computed once."""
    check_grouped(ctx, sizes, 264, 72, False, seed=51)
    check_wgrad(ctx, sizes, 264, 72, seed=52)


@EVERY_KERNEL
@pytest.mark.parametrize("ctas", [1, 2, 5, 20])
def test_few_ctas_many_rounds(ctx, ctas, parts):
    """A limit on the CTAs makes every one of them go through many tiles, of rows that differ."""
    ctx.set("max_ctas", ctas)
    try:
        sizes = [70, 0, 1, 300, 33, 64, 129, 5, 0, 31]
        check_grouped(ctx, sizes, 520, 200, False, seed=55)
        check_grouped(ctx, sizes, 520, 200, True, seed=56)
        check_wgrad(ctx, sizes, 520, 200, seed=57)
    finally:
        ctx.set("max_ctas", 0)


def test_first_calls_of_a_context_inside_a_capture():
    """What a context finds out with its first call of a kind is found out while a graph is captured, too."""
    import torch
    import maize_b200
    g = gen(58)
    sizes = [30, 0, 7]
    o = offsets_of(sizes)
    x, w, dy = bf16(g, (37, 1024)), bf16(g, (3, 136, 1024), 0.1), bf16(g, (37, 136))
    usual = maize_b200.Context(0)
    for parts in (0, 1, 2, 4, 8):
        usual.set("k_parts", parts)
        qx, sx = usual.quantize_e4m3(x)
        qw, sw = usual.quantize_e4m3(w[0], 128)
        want = (usual.grouped_gemm(x, w, o), usual.grouped_gemm_kn(dy, w, o), usual.grouped_gemm_wgrad(x, dy, o), qx, sx, qw, sw,
                usual.gemm_e4m3(qx, sx, qw, sw))
        usual.poll()
        fresh = maize_b200.Context(0)
        fresh.set("k_parts", parts)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = (fresh.grouped_gemm(x, w, o), fresh.grouped_gemm_kn(dy, w, o), fresh.grouped_gemm_wgrad(x, dy, o),
                   *fresh.quantize_e4m3(x), *fresh.quantize_e4m3(w[0], 128), fresh.gemm_e4m3(qx, sx, qw, sw))
        graph.replay()
        fresh.poll()
        for a, b in zip(got, want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        del graph, got
        fresh.close()
    usual.close()


@EVERY_KERNEL
def test_elements_past_32_bits(ctx, parts):
    """Rows of A and C, matrices of B and of DB that lie more than 2^32 bytes behind the start: a group at the very end."""
    import torch
    g = gen(61)
    rows, k, n = 300_000, 8192, 8192  # A and C of 4.9e9 bytes each
    a = torch.zeros((rows, k), dtype=torch.bfloat16, device="cuda")
    a[-100:] = bf16(g, (100, k))
    w = bf16(g, (2, n, k), 0.1)
    o = torch.tensor([rows - 100, rows - 70, rows], dtype=torch.int32, device="cuda")
    out = torch.full((rows, n), 7.0, dtype=torch.bfloat16, device="cuda")
    near = torch.tensor([0, 30, 100], dtype=torch.int32, device="cuda")
    for kn in (False, True):
        (ctx.grouped_gemm_kn if kn else ctx.grouped_gemm)(a, w, o, out=out)
        ctx.poll()
        ref, size = plain_grouped(a[-100:], w, near, kn)
        close(out[-100:], ref, size, k)
        assert (out[:64] == 7).all() and (out[-164:-100] == 7).all()
    dw = ctx.grouped_gemm_wgrad(a, out, o)  # rows in front of the groups hold sevens
    ctx.poll()
    for i, (b, e) in enumerate(((0, 30), (30, 100))):
        x, y = a[-100:][b:e].double(), out[-100:][b:e].double()
        close(dw[i, :256], y[:, :256].T @ x, y[:, :256].abs().T @ x.abs(), e - b)
        close(dw[i, -256:], y[:, -256:].T @ x, y[:, -256:].abs().T @ x.abs(), e - b)
    del a, out, w, dw
    # stacks of matrices: 33 of 8192 x 8192, rows for the first and the last
    a, w, dy = bf16(g, (20, k)), torch.zeros((33, n, k), dtype=torch.bfloat16, device="cuda"), bf16(g, (20, n))
    w[0], w[-1] = bf16(g, (n, k), 0.1), bf16(g, (n, k), 0.1)
    o = torch.tensor([0] + [7] * 32 + [20], dtype=torch.int32, device="cuda")
    for kn in (False, True):
        out = (ctx.grouped_gemm_kn if kn else ctx.grouped_gemm)(a, w, o)
        ctx.poll()
        ref, size = plain_grouped(a, w[[0, -1]], torch.tensor([0, 7, 20]), kn)
        close(out, ref, size, k)
    dw = ctx.grouped_gemm_wgrad(a, dy, o, out=w.fill_(7.0))
    ctx.poll()
    assert not dw[1:-1].any()
    for i, (b, e) in ((0, (0, 7)), (32, (7, 20))):
        x, y = a[b:e].double(), dy[b:e].double()
        close(dw[i, -256:], y[:, -256:].T @ x, y[:, -256:].abs().T @ x.abs(), e - b)


def test_module_functions_use_the_tensors_device():
    import torch
    import maize_b200
    g = gen(41)
    o = offsets_of([4, 6])
    x, w, dy = bf16(g, (10, 16)), bf16(g, (2, 24, 16)), bf16(g, (10, 24))
    ref, size = plain_grouped(x, w, o, False)
    close(maize_b200.grouped_gemm(x, w, o), ref, size, 16)
    ref, size = plain_grouped(dy, w, o, True)
    close(maize_b200.grouped_gemm_kn(dy, w, o), ref, size, 24)
    assert maize_b200.grouped_gemm_wgrad(x, dy, o).shape == (2, 24, 16)
    maize_b200.default_context(0).poll()
