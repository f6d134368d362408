"""The operators around experts that are not held in GGUF blocks, as cases that can be timed.

  * product: a token batch against one matrix of 8-bit integers, a scale a token and a scale a row of the matrix (a shared
    expert, a projection); the tokens come as floating rows and are quantized in the call.
  * experts: the same product over the runs of slots that a router made. "gate": the tokens' rows, quantized once, every slot
    reading its token's; "down": the gate's and the up's rows, joined by silu(g) * u and quantized.
  * sort: tokens sorted by expert: the tables and the moved rows, and the gradient of the move.
  * combine: the experts' rows back at their tokens, weighted and summed onto the residual, and its gradients.

Shapes are the repository's two layers (hidden 2048, 128 experts of 768, top-8; hidden 7168, 256 experts of 2048, top-8) and
sizes between and around them. The router's logits come out near N(0, 1) plus a bias an expert, so some experts are popular and
a few get nothing; "here" is the number of experts that this card holds: the slots of the others are served elsewhere.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _product(name, tokens, rows, k, dtype):
    c = {"kind": "product", "tokens": tokens, "rows": rows, "k": k, "type": dtype}
    return dict(c, name=name) if name else c


def _experts(name, half, tokens, rows, k, dtype, experts=128, here=128, top_k=8, skew=0.5):
    c = {"kind": "experts", "half": half, "tokens": tokens, "rows": rows, "k": k, "type": dtype, "experts": experts, "here": here,
         "top_k": top_k, "skew": skew}
    return dict(c, name=name) if name else c


def _rows(name, kind, tokens, width, dtype, grad=False, experts=128, here=128, top_k=8, skew=0.5):
    c = {"kind": kind, "grad": grad, "tokens": tokens, "width": width, "type": dtype, "experts": experts, "here": here, "top_k": top_k,
         "skew": skew}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token through an expert-sized matrix: latency counts
        _product("product_1", 1, 768, 2048, "f32"),
        # a decode batch through a projection of the larger layer
        _product("product_24", 24, 7168, 2048, "bf16"),
        # a ragged prompt through a matrix whose sizes are no multiples of a tile's
        _product("product_777", 777, 2000, 1996, "f16"),
        # a long prompt's chunk through the larger layer's square projection
        _product("product_4096", 4096, 7168, 7168, "bf16"),
        # a decode batch: most experts that are hit have one slot or two
        _experts("experts_gate_16", "gate", 16, 768, 2048, "bf16"),
        # a ragged prompt on a card that holds a quarter of the larger layer's experts
        _experts("experts_down_333", "down", 333, 7168, 2048, "f16", experts=256, here=64),
        # a prompt's chunk through the gates of a layer, a popular expert among them
        _experts("experts_gate_2048", "gate", 2048, 768, 2048, "bf16", skew=1.0),
        # a decode batch's rows in f32
        _rows("sort_16", "sort", 16, 2048, "f32"),
        # a training batch, forward and backward
        _rows("sort_4096", "sort", 4096, 2048, "bf16"),
        _rows("sort_grad_1500", "sort", 1500, 7168, "f16", grad=True, experts=256, here=256),
        # a decode batch's rows onto the residual in f32
        _rows("combine_16", "combine", 16, 2048, "f32"),
        # a training batch, backward: the gradients of the rows and of the router's weights
        _rows("combine_grad_4096", "combine", 4096, 2048, "bf16", grad=True),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["product", "product", "experts", "experts", "sort", "combine"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    if kind == "product":
        rows, k = spread(64, 8192), spread(64, 8192)
        rows, k = (rows, k) if rng.random() < 0.4 else (16 * -(-rows // 16), 64 * -(-k // 64))
        return _product(None, max(1, min(spread(1, 6000), int(2e11 / (rows * k)))), rows, k, dtype)
    experts, top_k = spread(8, 256), rng.randint(1, 8)
    here = experts if rng.random() < 0.7 else max(1, experts // 4)
    skew = rng.choice([0.5, 0.5, 1.0])
    if kind == "experts":
        rows, k = 16 * spread(8, 448), 16 * spread(8, 448)
        while here * rows * k > 1 << 30:
            experts, here = max(8, experts // 2), max(1, here // 2)
        tokens = max(1, min(spread(1, 2500), int(4e10 / (rows * k * top_k)), int(2e11 / (rows * k * here))))
        half = rng.choice(["gate", "down"])
        return _experts(None, half, tokens, rows, k, rng.choice(["f16", "bf16"]) if half == "down" else dtype, experts, here, top_k, skew)
    width = spread(64, 7168) if rng.random() < 0.4 else 64 * spread(1, 112)
    tokens = max(1, min(spread(1, 8000), int(3.2e8 / (top_k * width * SIZE[dtype]))))
    return _rows(None, kind, tokens, width, dtype, rng.random() < 0.5, experts, here, top_k, skew)


class _State:
    """What a program has in hand before the call."""


def _normal(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def _token_rows(gen, m, k, dtype):
    """Rows whose sizes differ from token to token, with a few large channels."""
    x = _normal(gen, m, k) * torch.exp(0.5 * _normal(gen, m, 1))
    return (x * torch.exp(0.7 * _normal(gen, k))).to(TYPES[dtype])


def _matrix(gen, n, rows, k):
    """n matrices as codes (rows padded with zeros to 16 bytes) and a scale a row: what rows of a spread of 0.02 give."""
    pad = -(-k // 16) * 16
    w = torch.zeros(n * rows, pad, dtype=torch.int8, device="cuda")
    step = max(1, (1 << 26) // k)
    for r in range(0, n * rows, step):
        some = _normal(gen, min(step, n * rows - r), k)
        w[r:r + step, :k] = (some * 31.0).round_().clamp_(-127, 127).to(torch.int8)
    return w, 0.02 / 31.0 * (0.75 + 0.5 * torch.rand(n * rows, device="cuda", generator=gen))


def _ids(gen, c):
    """A router's picks and weights: ids at or past `here` are served elsewhere."""
    m, n = c["tokens"], c["experts"]
    top_k = min(c["top_k"], n)
    logits = _normal(gen, m, n) + c["skew"] * _normal(gen, n)
    picked, ids = torch.topk(torch.softmax(logits, 1), top_k, dim=1)
    ids = torch.where(ids < c["here"], ids, torch.full_like(ids, -1)).to(torch.int32).contiguous()
    return ids, (picked / picked.sum(1, keepdim=True)).contiguous()


def _tables(ids, here):
    """order, start, place of the slots by expert, in 64 bits; entries behind the last listed one are the unlisted slots."""
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < here), flat, torch.full_like(flat, here))
    order = torch.argsort(key, stable=True)
    start = torch.searchsorted(key[order], torch.arange(here + 1, device=ids.device))
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device=ids.device)
    return order, start, torch.where(key < here, place, torch.full_like(place, -1))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    c, s = case, _State()
    s.case = c
    m, dtype = c["tokens"], TYPES[c["type"]]
    if c["kind"] == "product":
        rows, k = c["rows"], c["k"]
        s.w, s.w_scales = _matrix(gen, 1, rows, k)
        s.x = _token_rows(gen, m, k, c["type"])
        s.codes = torch.zeros(m, s.w.shape[1], dtype=torch.int8, device="cuda")
        s.scales = torch.zeros(m, device="cuda")
        s.y = torch.zeros(m, rows, dtype=dtype, device="cuda")
        return s
    s.ids, s.weights = _ids(gen, c)
    s.top_k = s.ids.shape[1]
    n, here = s.ids.numel(), c["here"]
    if c["kind"] == "experts":
        rows, k = c["rows"], c["k"]
        s.w, s.w_scales = _matrix(gen, here, rows, k)
        order, start, _ = _tables(s.ids, here)
        s.order, s.start = order.to(torch.int32), start.to(torch.int32)
        columns = m if c["half"] == "gate" else n
        if c["half"] == "gate":
            s.x = _token_rows(gen, m, k, c["type"])
        else:
            s.g, s.u = _token_rows(gen, n, k, c["type"]), _token_rows(gen, n, k, c["type"])
        s.codes = torch.zeros(columns, s.w.shape[1], dtype=torch.int8, device="cuda")
        s.scales = torch.zeros(columns, device="cuda")
        s.y = torch.zeros(n, rows, dtype=dtype, device="cuda")
        return s
    width = c["width"]
    if c["kind"] == "sort" and not c["grad"]:
        s.x = _token_rows(gen, m, width, c["type"])
        s.order, s.place = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(2))
        s.start = torch.zeros(here + 1, dtype=torch.int32, device="cuda")
        s.moved = torch.zeros(n, width, dtype=dtype, device="cuda")
        s.work = torch.zeros(n + 4096, dtype=torch.int32, device="cuda")
        return s
    s.place = _tables(s.ids, here)[2].to(torch.int32)
    s.moved = _token_rows(gen, n, width, c["type"])  # the experts' rows, or the gradients that came back to them
    if c["kind"] == "sort":
        s.dx = torch.zeros(m, width, dtype=dtype, device="cuda")
        return s
    s.rows = _token_rows(gen, m, width, c["type"])  # the residual, or the gradient of the sum
    s.y = torch.zeros(m, width, dtype=dtype, device="cuda")
    if c["grad"]:
        s.d_moved, s.d_weights = torch.zeros_like(s.moved), torch.zeros_like(s.weights)
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
    if c["kind"] == "product":
        gpu.enqueue_i8_gemm_x(p(s.w), p(s.w_scales), c["rows"], c["k"], p(s.x), t, m, p(s.codes), p(s.scales), p(s.y), t)
        return s.y
    if c["kind"] == "experts":
        n = s.ids.numel()
        if c["half"] == "gate":
            gpu.enqueue_i8_quantize(p(s.x), t, m, c["k"], p(s.codes), p(s.scales))
        else:
            live = p(s.start) + 4 * c["here"]
            gpu.enqueue_i8_swiglu_quantize(p(s.g), p(s.u), t, n, c["k"], p(s.codes), p(s.scales), live=live)
        gpu.enqueue_i8_gemm_experts(p(s.w), p(s.w_scales), c["here"], c["rows"], c["k"], p(s.codes), p(s.scales), p(s.order), p(s.start), n,
                                    s.top_k if c["half"] == "gate" else 0, p(s.y), t)
        return s.y
    if c["kind"] == "sort":
        if c["grad"]:
            gpu.enqueue_expert_sort_grad(p(s.moved), t, p(s.place), m, s.top_k, c["width"], p(s.dx))
            return s.dx
        gpu.enqueue_expert_sort(p(s.ids), m, s.top_k, c["here"], p(s.x), t, c["width"], p(s.order), p(s.start), p(s.place), p(s.moved), p(s.work))
        return {"order": s.order, "start": s.start, "place": s.place, "rows": s.moved}
    if c["grad"]:
        gpu.enqueue_expert_combine_grad(p(s.rows), t, p(s.moved), p(s.place), p(s.weights), m, s.top_k, c["width"], p(s.d_moved), p(s.d_weights))
        return {"rows": s.d_moved, "weights": s.d_weights}
    gpu.enqueue_expert_combine(p(s.moved), t, p(s.place), p(s.weights), p(s.rows), m, s.top_k, c["width"], p(s.y))
    return s.y


def _codes(x):
    """Rows as whole numbers in f32 and their scales: the quotients in 64 bits, for those next to a half."""
    scales = (x.double().abs().amax(1) / 127.0).float()  # a quotient in 64 bits: torch multiplies by a 32-bit scalar's reciprocal
    q = torch.round(x.double() / scales.double()[:, None]).clamp(-127, 127)
    return torch.where(scales[:, None] > 0, q, torch.zeros_like(q)).float(), scales


def run(s):
    if own:
        return _run_own(s)
    c = s.case
    m, dtype = c["tokens"], TYPES[c["type"]]
    if c["kind"] == "product":
        q, scales = _codes(s.x)
        sums = q @ s.w[:, :c["k"]].float().t()
        return (sums * scales[:, None] * s.w_scales[None, :]).to(dtype)
    if c["kind"] == "experts":
        here, rows, k = c["here"], c["rows"], c["k"]
        if c["half"] == "gate":
            q, scales = _codes(s.x)
            column = s.order.long() // s.top_k
            q, scales = q[column], scales[column]
        else:
            g = s.g.float()
            q, scales = _codes(g / (1.0 + torch.exp(-g)) * s.u.float())
        # every run padded to the longest, one batched product
        start = s.start.long()
        most = max(1, int((start[1:] - start[:-1]).max()))
        entry = start[:-1, None] + torch.arange(most, device="cuda")[None, :]
        live = entry < start[1:, None]
        batch = q[torch.where(live, entry, torch.zeros_like(entry))].transpose(1, 2).contiguous()
        sums = torch.bmm(s.w.view(here, rows, -1)[:, :, :k].float(), batch)
        # and back: entry j is column j - start of its expert
        j = torch.arange(s.y.shape[0], device="cuda")
        expert = torch.searchsorted(start, j, right=True) - 1
        listed_rows = j < start[here]
        e = torch.where(listed_rows, expert, torch.zeros_like(expert))
        at = torch.where(listed_rows, j - start[e], torch.zeros_like(j))
        y = sums.transpose(1, 2)[e, at] * scales[:, None] * s.w_scales.view(here, rows)[e]
        return torch.where(listed_rows[:, None], y.to(dtype), s.y)
    if c["kind"] == "sort" and not c["grad"]:
        order, start, place = _tables(s.ids, c["here"])
        there = torch.arange(order.numel(), device="cuda") < start[c["here"]]
        return {"order": torch.where(there, order.to(torch.int32), s.order), "start": start.to(torch.int32), "place": place.to(torch.int32),
                "rows": torch.where(there[:, None], s.x[order // s.top_k], s.moved)}
    place = s.place.long().view(m, s.top_k)
    there = place >= 0
    at = torch.where(there, place, torch.zeros_like(place))
    mine = s.moved.float()[at]  # tokens x slots x width
    if c["kind"] == "sort":
        return torch.where(there[:, :, None], mine, torch.zeros_like(mine)).sum(1).to(dtype)
    if not c["grad"]:
        weighted = torch.where(there[:, :, None], mine * s.weights[:, :, None], torch.zeros_like(mine))
        return (s.rows.float() + weighted.sum(1)).to(dtype)
    dy = s.rows.float()[:, None, :]
    d_weights = torch.where(there, (mine * dy).sum(2), torch.zeros_like(s.weights))
    d_rows = torch.zeros(s.moved.shape[0] + 1, c["width"], device="cuda")  # unlisted slots meet in the row behind the last
    d_rows[torch.where(there, place, torch.full_like(place, s.moved.shape[0])).view(-1)] = (s.weights[:, :, None] * dy).view(-1, c["width"])
    n = s.moved.shape[0]
    listed_rows = torch.arange(n, device="cuda") < there.sum()
    return {"rows": torch.where(listed_rows[:, None], d_rows[:n], torch.zeros_like(d_rows[:n])).to(dtype), "weights": d_weights}


def exact(case, seed):
    s, c = prepare(case, seed), case
    k = c.get("k")

    def columns(x):
        x = x.double()
        scale = (x.abs().max(1).values / 127.0).float().double()
        return torch.where(scale[:, None] > 0, torch.round(x / scale[:, None]).clamp(-127.0, 127.0), 0.0 * x), scale

    if c["kind"] == "product":
        q, scale = columns(s.x)
        return scale[:, None] * torch.matmul(q, s.w.double()[:, :k].t().contiguous()) * s.w_scales.double()
    ids = s.ids.view(-1).tolist()
    runs = [[] for _ in range(c["here"])]
    for slot, e in enumerate(ids):
        if e >= 0:
            runs[e].append(slot)
    order = [slot for r in runs for slot in r]
    if c["kind"] == "experts":
        if c["half"] == "gate":
            q, scale = columns(s.x)
        else:
            g, u = s.g.double(), s.u.double()
            q, scale = columns(g * torch.sigmoid(g) * u)
        y = torch.zeros(len(ids), c["rows"], dtype=torch.float64, device="cuda")
        w, ws, at = s.w.view(c["here"], c["rows"], -1), s.w_scales.double().view(c["here"], c["rows"]), 0
        for e, r in enumerate(runs):
            if r:
                j = torch.arange(at, at + len(r), device="cuda")
                col = torch.tensor(r, device="cuda") // s.top_k if c["half"] == "gate" else j
                y[j] = torch.matmul(q[col], w[e][:, :k].double().t().contiguous()) * scale[col][:, None] * ws[e]
                at += len(r)
        return y
    where = torch.tensor(order, dtype=torch.int64, device="cuda")
    token = where // s.top_k
    n = len(order)
    if c["kind"] == "sort" and not c["grad"]:
        rows = torch.zeros(len(ids), c["width"], dtype=torch.float64, device="cuda")
        rows[:n] = s.x.double()[token]
        return {"order": None, "start": None, "place": None, "rows": rows}
    moved = s.moved.double()[:n]
    y = torch.zeros(c["tokens"], c["width"], dtype=torch.float64, device="cuda")
    if c["kind"] == "sort":
        return y.index_add_(0, token, moved)
    w = s.weights.double().view(-1)
    if not c["grad"]:
        return y.index_add_(0, token, w[where][:, None] * moved) + s.rows.double()
    dy = s.rows.double()[token]
    d_rows = torch.zeros(len(ids), c["width"], dtype=torch.float64, device="cuda")
    d_rows[:n] = dy * w[where][:, None]
    d_w = torch.zeros_like(w)
    d_w[where] = torch.linalg.vecdot(dy, moved)
    return {"rows": d_rows, "weights": d_w.view(s.weights.shape)}


def work(case):
    c, m = case, case["tokens"]
    e = SIZE[c["type"]]
    if c["kind"] == "product":
        rows, k = c["rows"], c["k"]
        return {"bytes": rows * k + 4 * rows + e * m * (k + rows), "flops": 2 * m * rows * k}
    top_k = min(c["top_k"], c["experts"])
    n = m * top_k * c["here"] / c["experts"]  # slots that this card serves
    if c["kind"] == "experts":
        rows, k = c["rows"], c["k"]
        # the experts that m tokens hit when every expert is as likely (a skewed router hits somewhat fewer)
        hit = c["here"] * (1.0 - (1.0 - top_k / c["experts"]) ** m)
        return {"bytes": hit * rows * (k + 4) + e * k * (min(m, n) if c["half"] == "gate" else 2 * n) + e * n * rows, "flops": 2 * n * rows * k}
    row = c["width"] * e
    if c["kind"] == "sort":
        return {"bytes": n * row + min(m, n) * row + 12 * m * top_k, "flops": n * c["width"] if c["grad"] else 0}
    if c["grad"]:
        return {"bytes": 2 * n * row + m * row + 12 * m * top_k, "flops": 3 * n * c["width"]}
    return {"bytes": n * row + 2 * m * row + 8 * m * top_k, "flops": 2 * n * c["width"]}
