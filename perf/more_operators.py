"""The operators around experts whose weights are microscaled 4-bit floating point, as cases that can be timed.

A row of k values is held in blocks of 32: a 4-bit floating value (one sign, two exponent and one mantissa bit: 0, 0.5, 1, 1.5, 2, 3,
4, 6) for each, two to a byte, the even one in the low half, and a power of two for the block, 2^(byte - 127).

  * quantize: rows of floating values into that form, and back: the values that the codes stand for.
  * product: a token batch against one matrix in that form (a shared expert, a projection); the tokens come as floating rows and
    are quantized in the call.
  * experts: the same product over the runs of slots that a router made. "gate": the tokens' rows, quantized once, every slot
    reading its token's; "down": the gate's and the up's rows, joined by silu(g) * u and quantized.
  * layer: the experts' whole step for a few tokens, whose values stay in floating point: gate and up, silu(g) * u, down, and the
    weighted sum onto the residual.

Shapes are the repository's two layers (hidden 2048, 128 experts of 768, top-8; hidden 7168, 256 experts of 2048, top-8) and
sizes between and around them. The router's logits come out near N(0, 1) plus a bias an expert, so some experts are popular and
a few get nothing; "here" is the number of experts that this card holds: the slots of the others are served elsewhere.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _quantize(name, tokens, k, dtype):
    c = {"kind": "quantize", "tokens": tokens, "k": k, "type": dtype}
    return dict(c, name=name) if name else c


def _product(name, tokens, rows, k, dtype):
    c = {"kind": "product", "tokens": tokens, "rows": rows, "k": k, "type": dtype}
    return dict(c, name=name) if name else c


def _experts(name, half, tokens, rows, k, dtype, experts=128, here=128, top_k=8, skew=0.5):
    c = {"kind": "experts", "half": half, "tokens": tokens, "rows": rows, "k": k, "type": dtype, "experts": experts, "here": here,
         "top_k": top_k, "skew": skew}
    return dict(c, name=name) if name else c


def _layer(name, tokens, hidden, ff, dtype, experts=128, here=128, top_k=8, skew=0.5):
    c = {"kind": "layer", "tokens": tokens, "hidden": hidden, "ff": ff, "type": dtype, "experts": experts, "here": here, "top_k": top_k,
         "skew": skew}
    return dict(c, name=name) if name else c


def listed():
    return [
        # a decode batch's rows in f32: latency counts
        _quantize("quantize_16", 16, 2048, "f32"),
        # a long prompt's chunk of the larger layer
        _quantize("quantize_4096", 4096, 7168, "bf16"),
        # one token through an expert-sized matrix: latency counts
        _product("product_1", 1, 768, 2048, "f32"),
        # a decode batch through a projection of the larger layer
        _product("product_24", 24, 7168, 2048, "bf16"),
        # a ragged prompt through a matrix whose sizes are no multiples of a tile's or of a block's
        _product("product_777", 777, 2000, 1996, "f16"),
        # a long prompt's chunk through the larger layer's square projection
        _product("product_4096", 4096, 7168, 7168, "bf16"),
        # a decode batch: most experts that are hit have one slot or two
        _experts("experts_gate_16", "gate", 16, 768, 2048, "bf16"),
        # a ragged prompt on a card that holds a quarter of the larger layer's experts
        _experts("experts_down_333", "down", 333, 7168, 2048, "f16", experts=256, here=64),
        # a prompt's chunk through the gates of a layer, a popular expert among them
        _experts("experts_gate_2048", "gate", 2048, 768, 2048, "bf16", skew=1.0),
        # a decode step of one sequence: latency counts
        _layer("layer_1", 1, 2048, 768, "bf16"),
        # a decode batch in f32
        _layer("layer_16", 16, 2048, 768, "f32"),
        # a larger batch on a card that holds a quarter of the larger layer's experts
        _layer("layer_64", 64, 7168, 2048, "bf16", experts=256, here=64),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["quantize", "product", "product", "experts", "experts", "layer", "layer"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    if kind == "quantize":
        k = spread(64, 8192) if rng.random() < 0.4 else 32 * spread(2, 256)
        return _quantize(None, max(1, min(spread(1, 8000), 29000000 // k)), k, dtype)
    if kind == "product":
        rows, k = spread(64, 8192), spread(64, 8192)
        rows, k = (rows, k) if rng.random() < 0.4 else (16 * -(-rows // 16), 64 * -(-k // 64))
        return _product(None, max(1, min(spread(1, 6000), int(2e11 / (rows * k)))), rows, k, dtype)
    experts, top_k = spread(8, 256), rng.randint(1, 8)
    here = experts if rng.random() < 0.7 else max(1, experts // 4)
    skew = rng.choice([0.5, 0.5, 1.0])
    if kind == "layer":
        hidden, ff = spread(64, 7168), spread(64, 4096)
        hidden, ff = (hidden, ff) if rng.random() < 0.3 else (32 * -(-hidden // 32), 32 * -(-ff // 32))
        while here * hidden * ff > 1 << 29:
            experts, here = max(8, experts // 2), max(1, here // 2)
        return _layer(None, spread(1, 64), hidden, ff, dtype, experts, here, top_k, skew)
    rows, k = 16 * spread(8, 448), 32 * spread(4, 224)
    while here * rows * k > 1 << 30:
        experts, here = max(8, experts // 2), max(1, here // 2)
    tokens = max(1, min(spread(1, 2500), int(4e10 / (rows * k * top_k)), int(2e11 / (rows * k * here))))
    half = rng.choice(["gate", "down"])
    return _experts(None, half, tokens, rows, k, rng.choice(["f16", "bf16"]) if half == "down" else dtype, experts, here, top_k, skew)


class _State:
    """What a program has in hand before the call."""


def _normal(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def _token_rows(gen, m, k, dtype):
    """Rows whose sizes differ from token to token, with a few large channels."""
    x = _normal(gen, m, k) * torch.exp(0.5 * _normal(gen, m, 1))
    return (x * torch.exp(0.7 * _normal(gen, k))).to(TYPES[dtype])


def _row_bytes(k):
    """Bytes of a row's codes and of its scales."""
    blocks = -(-k // 32)
    return 16 * blocks, 16 * -(-blocks // 16)


def _matrix(gen, rows, k):
    """A matrix as codes and scales, as a file of weights holds it: what rows of a spread of 0.02 give."""
    nb, ns = _row_bytes(k)
    codes = torch.zeros(rows, nb, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(rows, ns, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 27) // k)
    for r in range(0, rows, step):
        n = min(step, rows - r)
        x = torch.zeros(n, 2 * nb, device="cuda")
        x[:, :k] = 0.02 * _normal(gen, n, k)
        levels, exponent = _to_blocks(x)
        code = torch.bucketize(levels.abs(), torch.tensor(LEVELS, device="cuda"), out_int32=True).to(torch.uint8)
        code += torch.signbit(levels).to(torch.uint8) * 8
        code = code.view(n, nb, 2)
        codes[r:r + n] = code[:, :, 0] + 16 * code[:, :, 1]
        scales[r:r + n, :nb // 16] = (exponent + 127).to(torch.uint8)
    return codes, scales


def _ids(gen, c):
    """A router's picks and weights: ids at or past `here` are served elsewhere."""
    m, n = c["tokens"], c["experts"]
    top_k = min(c["top_k"], n)
    logits = _normal(gen, m, n) + c["skew"] * _normal(gen, n)
    picked, ids = torch.topk(torch.softmax(logits, 1), top_k, dim=1)
    ids = torch.where(ids < c["here"], ids, torch.full_like(ids, -1)).to(torch.int32).contiguous()
    return ids, (picked / picked.sum(1, keepdim=True)).contiguous()


def _tables(ids, here):
    """order and start of the slots by expert, in 64 bits; entries behind the last listed one are the unlisted slots."""
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < here), flat, torch.full_like(flat, here))
    order = torch.argsort(key, stable=True)
    return order, torch.searchsorted(key[order], torch.arange(here + 1, device=ids.device))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    c, s = case, _State()
    s.case = c
    m, dtype = c["tokens"], TYPES[c["type"]]

    def columns(n, k):
        nb, ns = _row_bytes(k)
        s.codes = torch.zeros(n, nb, dtype=torch.uint8, device="cuda")
        s.scales = torch.zeros(n, ns, dtype=torch.uint8, device="cuda")

    if c["kind"] == "quantize":
        s.x = _token_rows(gen, m, c["k"], c["type"])
        columns(m, c["k"])
        s.y = torch.zeros(m, c["k"], dtype=dtype, device="cuda")
        return s
    if c["kind"] == "product":
        s.w, s.w_scales = _matrix(gen, c["rows"], c["k"])
        s.x = _token_rows(gen, m, c["k"], c["type"])
        columns(m, c["k"])
        s.y = torch.zeros(m, c["rows"], dtype=dtype, device="cuda")
        return s
    s.ids, s.weights = _ids(gen, c)
    s.top_k = s.ids.shape[1]
    n, here = s.ids.numel(), c["here"]
    if c["kind"] == "layer":
        hidden, ff = c["hidden"], c["ff"]
        s.gate, s.gate_scales = _matrix(gen, here * ff, hidden)
        s.up, s.up_scales = _matrix(gen, here * ff, hidden)
        s.down, s.down_scales = _matrix(gen, here * hidden, ff)
        s.x = _token_rows(gen, m, hidden, c["type"])
        s.resid = _token_rows(gen, m, hidden, c["type"])
        s.y = torch.zeros(m, hidden, dtype=dtype, device="cuda")
        s.work = torch.zeros(n * (8 * ff + 8 * hidden + 1024) + 65536, dtype=torch.uint8, device="cuda")
        return s
    rows, k = c["rows"], c["k"]
    s.w, s.w_scales = _matrix(gen, here * rows, k)
    order, start = _tables(s.ids, here)
    s.order, s.start = order.to(torch.int32), start.to(torch.int32)
    if c["half"] == "gate":
        s.x = _token_rows(gen, m, k, c["type"])
        columns(m, k)
    else:
        s.g, s.u = _token_rows(gen, n, k, c["type"]), _token_rows(gen, n, k, c["type"])
        columns(n, k)
    s.y = torch.zeros(n, rows, dtype=dtype, device="cuda")
    return s


_context = None


def _run_own(s):
    """The framework's calls, on torch's stream."""
    global _context
    import bloomery_amd as bm
    if _context is None:
        _context = bm.Gpu(0, stream=torch.cuda.current_stream().cuda_stream)
    gpu, c = _context, s.case
    p = torch.Tensor.data_ptr
    t, m = {"f32": bm.F32, "f16": bm.F16, "bf16": bm.BF16}[c["type"]], c["tokens"]
    if c["kind"] == "quantize":
        gpu.enqueue_mx4_quantize(p(s.x), t, m, c["k"], p(s.codes), p(s.scales))
        gpu.enqueue_mx4_dequantize(p(s.codes), p(s.scales), m, c["k"], p(s.y), t)
        return s.y
    if c["kind"] == "product":
        gpu.enqueue_mx4_gemm_x(p(s.w), p(s.w_scales), c["rows"], c["k"], p(s.x), t, m, p(s.codes), p(s.scales), p(s.y), t)
        return s.y
    if c["kind"] == "layer":
        gpu.enqueue_mx4_moe((p(s.gate), p(s.gate_scales)), (p(s.up), p(s.up_scales)), (p(s.down), p(s.down_scales)), c["here"], c["hidden"], c["ff"],
                            p(s.x), t, m, p(s.ids), p(s.weights), s.top_k, p(s.resid), p(s.y), p(s.work))
        return s.y
    n = s.ids.numel()
    if c["half"] == "gate":
        gpu.enqueue_mx4_quantize(p(s.x), t, m, c["k"], p(s.codes), p(s.scales))
    else:
        gpu.enqueue_mx4_swiglu_quantize(p(s.g), p(s.u), t, n, c["k"], p(s.codes), p(s.scales), live=p(s.start) + 4 * c["here"])
    gpu.enqueue_mx4_gemm_experts(p(s.w), p(s.w_scales), c["here"], c["rows"], c["k"], p(s.codes), p(s.scales), p(s.order), p(s.start), n,
                                 s.top_k if c["half"] == "gate" else 0, p(s.y), t)
    return s.y


def _to_blocks(x):
    """Rows of whole blocks: the levels, and the blocks' exponents of two."""
    v = x.view(x.shape[0], -1, 32)
    exponent = (torch.frexp(v.abs().amax(2))[1] - 3).clamp(-127, 127)  # the largest value's power of two, less the 4's
    exponent = torch.where(v.abs().amax(2) > 0, exponent, torch.full_like(exponent, -127))
    small = torch.exp2(-exponent.double())[:, :, None] * v
    step = torch.where(small.abs() < 2, 0.5, torch.where(small.abs() < 4, 1.0, 2.0))
    return (torch.round(small / step) * step).clamp(-6, 6).float().view_as(x), exponent


def _rounded(x):
    """Rows as the values that their codes stand for, in 32 bits."""
    k = x.shape[1]
    v = torch.zeros(x.shape[0], 32 * -(-k // 32), device="cuda")
    v[:, :k] = x
    levels, exponent = _to_blocks(v)
    return (levels.view(x.shape[0], -1, 32) * torch.exp2(exponent.double()).float()[:, :, None]).view_as(v)[:, :k]


def _values(codes, scales, k):
    """What codes and scales stand for, in 32 bits."""
    level = torch.tensor(LEVELS, device="cuda")
    level = torch.cat([level, -level])
    pair = torch.stack([level.repeat(16), level.repeat_interleave(16)], 1)
    v = pair[codes.int()].view(codes.shape[0], -1, 32)
    return (v * torch.exp2(scales[:, :v.shape[1]].double() - 127.0).float()[:, :, None]).view(codes.shape[0], -1)[:, :k]


def _entries(order, start, n):
    """Every expert's run padded to the longest: its entries, and where they are there; and for each entry of n its expert, its place in the run, and whether it is listed."""
    order, start = order.long(), start.long()
    most = max(1, int((start[1:] - start[:-1]).max()))
    entry = start[:-1, None] + torch.arange(most, device="cuda")[None, :]
    live = entry < start[1:, None]
    j = torch.arange(n, device="cuda")
    listed_rows = j < start[-1]
    e = torch.where(listed_rows, torch.searchsorted(start, j, right=True) - 1, torch.zeros_like(j))
    return torch.where(live, entry, torch.zeros_like(entry)), e, torch.where(listed_rows, j - start[e], torch.zeros_like(j)), listed_rows


def _times(w, columns, table):
    """Experts' matrices (experts x rows x k) with their entries' columns: entries x rows."""
    entry, e, at, _ = table
    return torch.bmm(w, columns[entry].transpose(1, 2).contiguous()).transpose(1, 2)[e, at]


def run(s):
    if own:
        return _run_own(s)
    c = s.case
    m, dtype = c["tokens"], TYPES[c["type"]]
    if c["kind"] == "quantize":
        return _rounded(s.x.float()).to(dtype)
    if c["kind"] == "product":
        return (_rounded(s.x.float()) @ _values(s.w, s.w_scales, c["k"]).t()).to(dtype)
    n, here = s.ids.numel(), c["here"]
    if c["kind"] == "experts":
        table = _entries(s.order, s.start, n)
        if c["half"] == "gate":
            columns = _rounded(s.x.float())[s.order.long() // s.top_k]
        else:
            g = s.g.float()
            columns = _rounded(g / (1.0 + torch.exp(-g)) * s.u.float())
        y = _times(_values(s.w, s.w_scales, c["k"]).view(here, c["rows"], -1), columns, table)
        return torch.where(table[3][:, None], y.to(dtype), s.y)
    hidden, ff = c["hidden"], c["ff"]
    order, start = _tables(s.ids, here)
    table = _entries(order, start, n)
    x = s.x.float()[order // s.top_k]
    g = _times(_values(s.gate, s.gate_scales, hidden).view(here, ff, -1), x, table)
    u = _times(_values(s.up, s.up_scales, hidden).view(here, ff, -1), x, table)
    y = _times(_values(s.down, s.down_scales, ff).view(here, hidden, -1), g / (1.0 + torch.exp(-g)) * u, table)
    y = torch.where(table[3][:, None], y * s.weights.view(-1)[order][:, None], torch.zeros_like(y))
    back = torch.empty_like(order)
    back[order] = torch.arange(n, device="cuda")
    return (s.resid.float() + y[back].view(m, s.top_k, hidden).sum(1)).to(dtype)


def exact(case, seed):
    s, c = prepare(case, seed), case
    middles = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64, device="cuda")
    level = torch.tensor(LEVELS, dtype=torch.float64, device="cuda")

    def rounded(x):
        """The nearest value of every block's scale, the even code where two are as near."""
        out = torch.zeros(x.shape[0], 32 * -(-x.shape[1] // 32), dtype=torch.float64, device="cuda")
        out[:, :x.shape[1]] = x
        step = max(1, (1 << 24) // out.shape[1])
        for r in range(0, x.shape[0], step):
            v = out[r:r + step].reshape(-1, 32)
            most = v.abs().max(1, keepdim=True).values
            scale = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.where(most > 0, most, torch.ones_like(most)))) - 2.0, -127.0, 127.0))
            size = v.abs() / scale
            code = torch.bucketize(size, middles)
            tie = (code < 7) & (size == middles[code.clamp(max=6)]) & (code % 2 == 1)
            out[r:r + step] = (torch.sign(v) * level[code + tie.long()] * scale).view(-1, out.shape[1])
        return out[:, :x.shape[1]]

    def matrix(codes, scales, k):
        """A matrix' values, byte by byte."""
        low, high = (codes % 16).long(), (codes // 16).long()
        v = torch.stack([level[low % 8] * (1.0 - 2.0 * (low // 8)), level[high % 8] * (1.0 - 2.0 * (high // 8))], dim=2)
        blocks = codes.shape[1] // 16
        return (v.reshape(-1, blocks, 32) * torch.exp2(scales[:, :blocks].double() - 127.0).unsqueeze(2)).reshape(codes.shape[0], -1)[:, :k]

    if c["kind"] == "quantize":
        return rounded(s.x.double())
    if c["kind"] == "product":
        return torch.matmul(rounded(s.x.double()), matrix(s.w, s.w_scales, c["k"]).t().contiguous())
    runs = [[] for _ in range(c["here"])]
    for slot, e in enumerate(s.ids.view(-1).tolist()):
        if e >= 0:
            runs[e].append(slot)

    def of(stack, scales, e, rows, k):
        return matrix(stack[e * rows:(e + 1) * rows], scales[e * rows:(e + 1) * rows], k).t().contiguous()

    if c["kind"] == "experts":
        rows, k = c["rows"], c["k"]
        y, at = torch.zeros(s.ids.numel(), rows, dtype=torch.float64, device="cuda"), 0
        g = None if c["half"] == "gate" else s.g.double()
        columns = rounded(s.x.double() if g is None else g * torch.sigmoid(g) * s.u.double())
        for e, r in enumerate(runs):
            if r:
                j = torch.arange(at, at + len(r), device="cuda")
                y[j] = torch.matmul(columns[torch.tensor(r, device="cuda") // s.top_k if g is None else j], of(s.w, s.w_scales, e, rows, k))
                at += len(r)
        return y
    y, x, weights = s.resid.double(), s.x.double(), s.weights.double().view(-1)
    for e, r in enumerate(runs):
        if r:
            slots = torch.tensor(r, device="cuda")
            g = torch.matmul(x[slots // s.top_k], of(s.gate, s.gate_scales, e, c["ff"], c["hidden"]))
            h = g * torch.sigmoid(g) * torch.matmul(x[slots // s.top_k], of(s.up, s.up_scales, e, c["ff"], c["hidden"]))
            y.index_add_(0, slots // s.top_k, weights[slots][:, None] * torch.matmul(h, of(s.down, s.down_scales, e, c["hidden"], c["ff"])))
    return y


def work(case):
    c, m = case, case["tokens"]
    e, held = SIZE[c["type"]], 17 / 32  # bytes of a value in blocks
    if c["kind"] == "quantize":
        # the rows and the values that the codes stand for (in between, the codes go out and come back in)
        return {"bytes": m * c["k"] * (2 * e + 2 * held), "flops": 0}
    if c["kind"] == "product":
        rows, k = c["rows"], c["k"]
        return {"bytes": rows * k * held + e * m * (k + rows), "flops": 2 * m * rows * k}
    top_k = min(c["top_k"], c["experts"])
    n = m * top_k * c["here"] / c["experts"]  # slots that this card serves
    # the experts that m tokens hit when every expert is as likely (a skewed router hits somewhat fewer)
    hit = c["here"] * (1.0 - (1.0 - top_k / c["experts"]) ** m)
    if c["kind"] == "experts":
        rows, k = c["rows"], c["k"]
        return {"bytes": hit * rows * k * held + e * k * (min(m, n) if c["half"] == "gate" else 2 * n) + e * n * rows, "flops": 2 * n * rows * k}
    hidden, ff = c["hidden"], c["ff"]
    return {"bytes": 3 * hit * hidden * ff * held + 3 * e * m * hidden + 8 * m * top_k, "flops": 6 * n * hidden * ff}
