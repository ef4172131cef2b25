"""Measured cases of the expert (grouped) products, their weight gradient, and the 8-bit block-scaled product with its quantiser.

``run`` computes a case in its plain form (elementary torch operations in fp32, rounded once at the end) or, with ``own``
set, with the calls a user of the package makes.
"""
import math

import torch

own = False

BLOCK = 128


# ------------------------------------------------------------------ cases --
def listed():
    return [
        # the smallest call: three rows left for four small experts; latency is all that counts
        {"name": "experts 3 rows", "op": "grouped", "layout": "nk", "rows": 3, "groups": 4, "n": 512, "k": 256},
        # one decoding step of a batch: 32 routed rows over 16 experts, bound by reading the weights
        {"name": "experts decode 32", "op": "grouped", "layout": "nk", "rows": 32, "groups": 16, "n": 4096, "k": 2048},
        # a prompt or training batch through the up projection of eight experts
        {"name": "experts 16384 rows", "op": "grouped", "layout": "nk", "rows": 16384, "groups": 8, "n": 4096, "k": 4096},
        # the input's gradient (the same weights read as K x N), many experts, nothing a multiple of a tile
        {"name": "experts dX ragged", "op": "grouped", "layout": "kn", "rows": 4111, "groups": 32, "n": 1032, "k": 1416},
        # weight gradient of a training batch
        {"name": "experts dW 8192 rows", "op": "wgrad", "rows": 8192, "groups": 16, "n": 4096, "k": 2048},
        # weight gradient of a small micro-batch: short and empty groups, odd sizes
        {"name": "experts dW ragged", "op": "wgrad", "rows": 777, "groups": 24, "n": 520, "k": 264},
        # activations of one decoding step
        {"name": "quantize 16 rows", "op": "quantize", "rows": 16, "cols": 4096, "block_rows": 1},
        # activations of a prompt
        {"name": "quantize 8192 rows", "op": "quantize", "rows": 8192, "cols": 8192, "block_rows": 1},
        # a weight matrix in 128 x 128 blocks, edges inside a block
        {"name": "quantize weight ragged", "op": "quantize", "rows": 3967, "cols": 4104, "block_rows": 128},
        # decoding step: 16 rows against a large weight, bound by reading it
        {"name": "e4m3 decode 16", "op": "e4m3", "m": 16, "n": 16384, "k": 4096},
        # ragged in every direction, the last block of K cut short
        {"name": "e4m3 ragged", "op": "e4m3", "m": 4111, "n": 3967, "k": 4112},
        # a large square product: bound by the tensor cores
        {"name": "e4m3 8192", "op": "e4m3", "m": 8192, "n": 8192, "k": 8192},
    ]


def _spread(rng, lo, hi, step=1):
    """A size between lo and hi, uniform in its logarithm, a multiple of step."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + step)))
    return max(lo, min(hi, int(v) // step * step))


def draw(rng):
    op = rng.choice(("grouped", "grouped", "wgrad", "quantize", "e4m3"))
    while True:
        if op == "quantize":
            case = {"op": op, "rows": _spread(rng, 1, 16384), "cols": _spread(rng, 8, 16384),
                    "block_rows": rng.choice((1, BLOCK))}
            if case["rows"] * case["cols"] <= 8192 * 8192:
                return case
        elif op == "e4m3":
            case = {"op": op, "m": _spread(rng, 1, 8192), "n": _spread(rng, 16, 16384), "k": _spread(rng, 64, 8192, 16)}
            if case["m"] * case["n"] * case["k"] <= 8192 ** 3:
                return case
        else:
            case = {"op": op, "rows": _spread(rng, 1, 16384), "groups": _spread(rng, 1, 64),
                    "n": _spread(rng, 128, 8192, 8), "k": _spread(rng, 128, 8192, 8)}
            if op == "grouped":
                case["layout"] = rng.choice(("nk", "kn"))
            if case["rows"] * case["n"] * case["k"] <= 8192 * 4096 * 4096 and case["groups"] * case["n"] * case["k"] <= 8 * 4096 * 4096:
                return case


# ----------------------------------------------------------------- inputs --
def _normal(gen, shape, scale):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(torch.bfloat16)


def _offsets(gen, rows, groups):
    """Offsets of rows dealt to experts by a skewed router: some experts get several times the mean, some nothing."""
    p = torch.softmax(0.7 * torch.randn(groups, generator=gen, device="cuda"), 0)
    choice = torch.multinomial(p, rows, replacement=True, generator=gen)
    counts = torch.bincount(choice, minlength=groups)
    offsets = torch.zeros(groups + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = counts.cumsum(0)
    return offsets, int(counts.max())


def _scaled(gen, rows, cols, block_rows, scale):
    """A matrix held in e4m3 with a scale for each block, as a checkpoint or a quantiser gives it."""
    x = torch.randn((rows, cols), generator=gen, device="cuda")
    q = (x * 100.0).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    s = (0.5 + torch.rand((-(-rows // block_rows), -(-cols // BLOCK)), generator=gen, device="cuda")) * (scale / 100.0)
    return q, s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, state = case["op"], {"op": case["op"]}
    if op == "grouped":
        rows, groups, n, k = case["rows"], case["groups"], case["n"], case["k"]
        state["kn"] = case["layout"] == "kn"
        state["x"] = _normal(gen, (rows, k), 1.0)
        state["w"] = _normal(gen, (groups, k, n) if state["kn"] else (groups, n, k), 0.02)
        state["offsets"], state["largest"] = _offsets(gen, rows, groups)
    elif op == "wgrad":
        rows, groups, n, k = case["rows"], case["groups"], case["n"], case["k"]
        state["x"] = _normal(gen, (rows, k), 1.0)
        state["dy"] = _normal(gen, (rows, n), 0.01)
        state["offsets"], state["largest"] = _offsets(gen, rows, groups)
    elif op == "quantize":
        # rows of different sizes and a few outliers, as activations have them
        size = torch.exp(torch.randn((case["rows"], 1), generator=gen, device="cuda"))
        x = torch.randn((case["rows"], case["cols"]), generator=gen, device="cuda") * size
        far = torch.rand(x.shape, generator=gen, device="cuda") < 1e-3
        state["x"] = torch.where(far, 30.0 * x, x).to(torch.bfloat16)
        state["block_rows"] = case["block_rows"]
    else:
        state["a"], state["sa"] = _scaled(gen, case["m"], case["k"], 1, 1.0)
        state["b"], state["sb"] = _scaled(gen, case["n"], case["k"], BLOCK, 0.02)
    return state


# ------------------------------------------------------------ plain forms --
def _rows_by_group(offsets, largest, rows):
    """[groups, largest] row numbers, which of them are rows of the group, and each row's group."""
    start, end = offsets[:-1, None].long(), offsets[1:, None].long()
    at = start + torch.arange(largest, device=offsets.device)
    group = torch.searchsorted(offsets[1:].long(), torch.arange(rows, device=offsets.device), right=True)
    return at.clamp(max=rows - 1), at < end, group


def _padded(x, at, real):
    return torch.where(real[..., None], x[at].float(), 0.0)


def _plain_grouped(x, w, offsets, largest, kn):
    at, real, group = _rows_by_group(offsets, largest, x.shape[0])
    wf = w.float()
    y = torch.bmm(_padded(x, at, real), wf if kn else wf.transpose(1, 2))
    place = torch.arange(x.shape[0], device=x.device) - offsets[:-1].long()[group]
    return y[group, place].to(torch.bfloat16)


def _plain_wgrad(x, dy, offsets, largest):
    at, real, _ = _rows_by_group(offsets, largest, x.shape[0])
    return torch.bmm(_padded(dy, at, real).transpose(1, 2), _padded(x, at, real)).to(torch.bfloat16)


def _blocks(x, block_rows):
    """x padded with zeros to whole blocks, as [blocks down, block_rows, blocks across, 128]."""
    rows, cols = x.shape
    down, across = -(-rows // block_rows), -(-cols // BLOCK)
    full = x.new_zeros((down * block_rows, across * BLOCK))
    full[:rows, :cols] = x
    return full.view(down, block_rows, across, BLOCK)


def _plain_quantize(x, block_rows):
    rows, cols = x.shape
    b = _blocks(x.float(), block_rows)
    amax = b.abs().amax((1, 3))
    m, e = torch.frexp(amax)
    p = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-126)  # 448 = 0.875 * 2^9
    scale = torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), p), 1.0)
    q = (b / scale[:, None, :, None]).to(torch.float8_e4m3fn)
    return q.view(-1, b.shape[2] * BLOCK)[:rows, :cols].contiguous(), scale


def _widen(s, rows, cols, block_rows):
    return s.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]


def _plain_e4m3(a, sa, b, sb):
    af = a.float() * _widen(sa, *a.shape, 1)
    bf = b.float() * _widen(sb, *b.shape, BLOCK)
    return torch.matmul(af, bf.t()).to(torch.bfloat16)


def run(state):
    op = state["op"]
    if own:
        import maize_b200
        if op == "grouped":
            f = maize_b200.grouped_gemm_kn if state["kn"] else maize_b200.grouped_gemm
            return f(state["x"], state["w"], state["offsets"])
        if op == "wgrad":
            return maize_b200.grouped_gemm_wgrad(state["x"], state["dy"], state["offsets"])
        if op == "quantize":
            return maize_b200.quantize_e4m3(state["x"], block_rows=state["block_rows"])
        return maize_b200.gemm_e4m3(state["a"], state["sa"], state["b"], state["sb"])
    if op == "grouped":
        return _plain_grouped(state["x"], state["w"], state["offsets"], state["largest"], state["kn"])
    if op == "wgrad":
        return _plain_wgrad(state["x"], state["dy"], state["offsets"], state["largest"])
    if op == "quantize":
        return _plain_quantize(state["x"], state["block_rows"])
    return _plain_e4m3(state["a"], state["sa"], state["b"], state["sb"])


# -------------------------------------------------------------- reckoning --
def work(case):
    op = case["op"]
    if op == "quantize":
        blocks = -(-case["rows"] // case["block_rows"]) * -(-case["cols"] // BLOCK)
        return {"bytes": 3 * case["rows"] * case["cols"] + 4 * blocks, "flops": 2 * case["rows"] * case["cols"]}
    if op == "e4m3":
        m, n, k = case["m"], case["n"], case["k"]
        scales = 4 * -(-k // BLOCK) * (m + -(-n // BLOCK))
        return {"bytes": m * k + n * k + scales + 2 * m * n, "flops": 2 * m * n * k}
    rows, groups, n, k = case["rows"], case["groups"], case["n"], case["k"]
    # grouped: a weight matrix is read where its group has a row (as many as even chances give); its gradient is always written
    matrices = groups if op == "wgrad" else groups * (1.0 - (1.0 - 1.0 / groups) ** rows)
    return {"bytes": 2 * rows * (n + k) + 2 * matrices * n * k + 4 * (groups + 1), "flops": 2 * rows * n * k}


def exact(case, seed):
    """The same from the definitions, in 64 bits: group by group, block by block."""
    s = prepare(case, seed)
    op = case["op"]
    if op in ("grouped", "wgrad"):
        ends = s["offsets"].tolist()
        x = s["x"].double()
        if op == "grouped":
            out = torch.zeros((case["rows"], case["n"]), dtype=torch.float64, device="cuda")
            for g in range(case["groups"]):
                mine = slice(ends[g], ends[g + 1])
                weight = s["w"][g].double()
                out[mine] = x[mine] @ (weight if s["kn"] else weight.T)
        else:
            out = torch.zeros((case["groups"], case["n"], case["k"]), dtype=torch.float64, device="cuda")
            for g in range(case["groups"]):
                mine = slice(ends[g], ends[g + 1])
                out[g] = s["dy"][mine].double().T @ x[mine]
        return out
    if op == "quantize":
        x, step = s["x"].double(), case["block_rows"]
        pad = torch.nn.functional.pad(x, (0, -x.shape[1] % BLOCK, 0, -x.shape[0] % step))
        tops = pad.abs().reshape(pad.shape[0] // step, step, pad.shape[1] // BLOCK, BLOCK).amax(3).amax(1)
        scale = torch.where(tops > 0, torch.exp2(torch.ceil(torch.log2(tops / 448.0))).clamp(min=2.0 ** -126), 1.0)
        # the logarithm may miss a whole number by a rounding: put right by comparison
        scale = torch.where((tops > 0) & (tops <= 224.0 * scale) & (scale > 2.0 ** -126), scale / 2, scale)
        scale = torch.where(tops > 448.0 * scale, scale * 2, scale)
        wide = scale.repeat_interleave(step, 0)[: x.shape[0]].repeat_interleave(BLOCK, 1)[:, : x.shape[1]]
        v = x / wide
        # e4m3: steps of an eighth of the binade, no finer than 2^-9
        unit = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))) / 8
        return torch.round(v / unit) * unit, scale
    a, b = s["a"].double(), s["b"].double()
    out = torch.zeros((case["m"], case["n"]), dtype=torch.float64, device="cuda")
    for j in range(s["sa"].shape[1]):
        part = slice(j * BLOCK, (j + 1) * BLOCK)
        column = s["sb"][:, j].double().repeat_interleave(BLOCK)[: case["n"]]
        out += (a[:, part] * s["sa"][:, j : j + 1].double()) @ (b[:, part] * column[:, None]).T
    return out
