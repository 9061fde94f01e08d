"""Expert routing and int8 (W8A8) operators, as a serving program calls them, and their plain forms.

Weights are int8 with one fp32 scale per output channel, rows int8 with one fp32 scale per token. A
case is one call of:

  * ``route`` - the choice of experts from a router's logits: softmax or sigmoid scores, a bias for
    balance, groups of experts, top-k, renormalised weights (``route_topk``);
  * ``dense`` - one linear layer (``int8_gemm``), from int8 rows or from 16-bit rows that the call quantises;
  * ``layer`` - a gated expert layer from routed tokens (``moe_int8_apply``).

``own`` chooses between the package's kernels and the plain forms below, which compute with
elementary torch operations (in fp32; the router's scores in fp64: a choice between two experts may
hang on their last bits). ``exact`` restates each operator in float64.
"""
import math
import os
import sys

import torch

own = False

INT8_MAX = 127.0
LEAST = INT8_MAX * 2.0 ** -100                     # what a row's largest value counts as at least
# the largest listed weights and products
MOST_WEIGHTS = 64 * 3 * 4096 * 1024
MOST_DENSE = 2 * 4096 * 12288 * 4096
MOST_LAYER = 6 * 2048 * 8 * 4096 * 1024


def listed():
    route = dict(op="route", E=256, k=8, dtype="fp32", masked=0)
    layer = dict(op="layer", H=2048, I=512, E=256, k=8, dtype="bf16", rows8=False, zipf=False)
    return [
        # one user decoding, a softmax router: latency alone
        dict(route, name="route_t1", T=1, scoring="softmax", bias=False, groups=1, top_groups=1, renorm=True, scale=1.0),
        # a decode batch, sigmoid scores with the balance bias, four of eight groups
        dict(route, name="route_t77", T=77, scoring="sigmoid", bias=True, groups=8, top_groups=4, renorm=True, scale=2.5),
        # prompt processing, the same router with 16-bit logits, whose values are often equal
        dict(route, name="route_t16384", T=16384, dtype="bf16", scoring="sigmoid", bias=True, groups=8, top_groups=4,
             renorm=True, scale=2.5),
        # an attention projection while one user decodes
        dict(op="dense", name="int8_m1", M=1, N=4096, K=4096, dtype="bf16", rows8=False, bias=False),
        # a down projection of long rows for a few users
        dict(op="dense", name="int8_m8", M=8, N=4096, K=12288, dtype="bf16", rows8=True, bias=False),
        # a wide projection with a bias for a decode batch, from 16-bit rows
        dict(op="dense", name="int8_m77", M=77, N=12288, K=4096, dtype="bf16", rows8=False, bias=True),
        # a chunk of a prompt with an odd number of tokens
        dict(op="dense", name="int8_m333", M=333, N=4096, K=12288, dtype="fp16", rows8=True, bias=False),
        # prompt processing, a wide projection
        dict(op="dense", name="int8_m4096", M=4096, N=12288, K=4096, dtype="bf16", rows8=True, bias=False),
        # an expert layer while one user decodes
        dict(layer, name="layer_t1", T=1),
        # a decode batch: the weights of most experts are streamed
        dict(layer, name="layer_t32", T=32),
        # prompt processing with a trained router's skew
        dict(layer, name="layer_t4096", T=4096, zipf=True),
        # prompt processing over fewer, wide experts: the largest call
        dict(layer, name="layer_t2048", T=2048, H=4096, I=1024, E=64),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("route", "dense", "dense", "layer", "layer"))
    if op == "route":
        E, groups, top = rng.choice(((256, 8, 4), (256, 1, 1), (160, 8, 3), (128, 1, 1), (64, 1, 1), (60, 1, 1),
                                     (384, 1, 1), (512, 16, 4), (32, 4, 2), (8, 1, 1)))
        scoring = rng.choice(("softmax", "sigmoid"))
        return dict(op=op, T=_log(rng, 1, min(32768, 16384 * 256 // E)), E=E, k=rng.choice((1, 2, 4, 6, 8)), scoring=scoring,
                    bias=rng.random() < (0.8 if scoring == "sigmoid" else 0.3), groups=groups, top_groups=top,
                    renorm=rng.random() < 0.8, scale=rng.choice((1.0, 1.0, 2.5, 16.0)),
                    dtype=rng.choice(("fp32", "bf16", "fp16")), masked=rng.choice((0, 0, 0, E // 2, E - 3)))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if op == "dense":
        K = 16 * _log(rng, 8, 768)
        N = _log(rng, 64, 12288)
        return dict(op=op, M=_log(rng, 1, min(4096, MOST_DENSE // (2 * N * K))), N=N, K=K, dtype=dtype,
                    rows8=rng.random() < 0.5, bias=rng.random() < 0.3)
    E, k = rng.choice(((256, 8), (128, 8), (64, 6), (32, 4), (8, 2)))
    H, I = rng.choice(((2048, 512), (2048, 768), (1024, 704), (2048, 256), (4096, 1024), (512, 384), (1536, 1408)))
    while 3 * E * H * I > MOST_WEIGHTS:
        E //= 2
    return dict(op=op, T=_log(rng, 1, min(4096, MOST_LAYER // (6 * k * H * I))), H=H, I=I, E=E, k=min(k, E), dtype=dtype,
                rows8=rng.random() < 0.3, zipf=rng.random() < 0.5)


# --------------------------------------------------------------------------- inputs
_TYPES = dict(fp32=torch.float32, bf16=torch.bfloat16, fp16=torch.float16)


def _gen(seed, part):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1013 + part)


def _hidden(g, T, H, dtype):
    """Hidden states: normal values, one channel in 64 eight times as wide, tokens of other sizes."""
    x = torch.randn((T, H), generator=g, device="cuda")
    x *= torch.where(torch.rand((H,), generator=g, device="cuda") < 1 / 64, 8.0, 1.0)
    x *= torch.exp(torch.randn((T, 1), generator=g, device="cuda") * 0.5)
    return x.to(dtype)


def _weight(g, E, N, K):
    """int8 weights (E, N, K) and channel scales (E, N): normal weights of standard deviation 0.02,
    channels of other sizes, each channel's largest value at 127."""
    w = torch.empty((E, N, K), dtype=torch.int8, device="cuda")
    s = torch.empty((E, N), dtype=torch.float32, device="cuda")
    step = max(1, (1 << 27) // (N * K))
    for lo in range(0, E, step):
        hi = min(E, lo + step)
        v = torch.randn((hi - lo, N, K), generator=g, device="cuda").mul_(0.02)
        v.mul_(torch.rand((hi - lo, N, 1), generator=g, device="cuda").add_(0.5))
        sc = v.abs().amax(2, keepdim=True).div_(INT8_MAX)
        w[lo:hi] = v.div_(sc).round_().to(torch.int8)
        s[lo:hi] = sc[..., 0]
    return w, s


def _logits(g, T, E, zipf):
    """A router's logits: normal, or with some experts far more popular (Zipf 1.1)."""
    if not zipf:
        return torch.randn((T, E), generator=g, device="cuda")
    p = torch.arange(1, E + 1, device="cuda", dtype=torch.float32).log_().mul_(-1.1)
    u = torch.rand((T, E), generator=g, device="cuda").clamp_(1e-7, 1 - 1e-7)
    return p[torch.randperm(E, generator=g, device="cuda")] - torch.log(-torch.log(u))


def prepare(case, seed):
    g, op, dt = _gen(seed, 1), case["op"], _TYPES[case["dtype"]]
    if op == "route":
        T, E = case["T"], case["E"]
        logits = torch.randn((T, E), generator=g, device="cuda") * 2 - 1
        if case["masked"]:
            # experts that a token must not reach
            rank = torch.rand((T, E), generator=g, device="cuda").argsort(1)
            logits = torch.where(rank < case["masked"], -math.inf, logits)
        bias = torch.randn((E,), generator=g, device="cuda") * 0.1 if case["bias"] else None
        return dict(case, logits=logits.to(dt), b=bias)
    if op == "dense":
        w, ws = _weight(g, 1, case["N"], case["K"])
        x, xs = _hidden(g, case["M"], case["K"], dt), None
        if case["rows8"]:
            # as a layer before this one leaves them
            x, xs = _quant(x.float())
        b = torch.randn((case["N"],), generator=g, device="cuda").to(dt) if case["bias"] else None
        return dict(case, x=x, xs=xs, w=w[0], ws=ws[0], b=b, out_dtype=dt)
    T, H, I, E = case["T"], case["H"], case["I"], case["E"]
    w13, s13 = _weight(g, E, 2 * I, H)
    w2, s2 = _weight(g, E, H, I)
    top, ids = torch.softmax(_logits(g, T, E, case["zipf"]), 1).topk(case["k"], 1)
    tw = (top / top.sum(1, keepdim=True)).contiguous()
    x, xs = _hidden(g, T, H, dt), None
    if case["rows8"]:
        x, xs = _quant(x.float())
    return dict(case, x=x, xs=xs, w13=w13, s13=s13, w2=w2, s2=s2, tw=tw, ids=ids.to(torch.int32).contiguous(),
                out_dtype=dt)


# --------------------------------------------------------------------------- plain forms
def _quant(v):
    """fp32 rows -> int8 rows, one fp32 scale each (rows, 1). (127 times a 16-bit value is an fp32
    number, so that its quotient by the row's largest value lies on a border between two whole
    numbers only where the true one does.)"""
    top = v.abs().amax(-1, keepdim=True).clamp_min(LEAST)
    # (divided by a tensor: a quotient by a number is a product with its rounded inverse)
    return torch.round(v * INT8_MAX / top).to(torch.int8), top / torch.full_like(top, INT8_MAX)


def _plain_route(st):
    E, k, groups = st["E"], st["k"], st["groups"]
    l = st["logits"].double()
    p = torch.sigmoid(l) if st["scoring"] == "sigmoid" else torch.softmax(l, 1)
    c = p if st["b"] is None else p + st["b"].double()
    c = torch.where(l == -math.inf, -math.inf, c)
    if groups > 1:
        by = c.view(-1, groups, E // groups)
        best = by.amax(2)
        if st["b"] is not None:
            second = by.topk(2, 2).values[:, :, 1]
            best = best + torch.where(second == -math.inf, 0.0, second)
        kept = best.sort(dim=1, descending=True, stable=True).indices[:, : st["top_groups"]]
        keep = torch.zeros_like(best).scatter_(1, kept, 1.0)
        c = torch.where((keep > 0)[:, :, None], by, -math.inf).view(-1, E)
    c, ids = c.sort(dim=1, descending=True, stable=True)
    c, ids = c[:, :k], ids[:, :k]
    none = c == -math.inf
    w = torch.where(none, 0.0, p.gather(1, ids))
    if st["renorm"]:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    return [(w * st["scale"]).float(), torch.where(none, -1, ids).to(torch.int32)]


def _plain_dense(st):
    x, xs = (st["x"], st["xs"]) if st["xs"] is not None else _quant(st["x"].float())
    y = (x.float() @ st["w"].float().t()) * (xs * st["ws"])
    return (y if st["b"] is None else y + st["b"].float()).to(st["out_dtype"])


def _by_expert(ids, E, block):
    """Slots by expert, each expert's run padded to whole blocks: (slot of each padded row, the number
    of slots for padding; expert of each block)."""
    flat = ids.reshape(-1).long()
    n = flat.numel()
    P = -(-(n + min(E, n) * (block - 1)) // block) * block
    counts = torch.zeros(E, dtype=torch.long, device=flat.device).scatter_add_(0, flat, torch.ones_like(flat))
    pad = (counts + block - 1) // block * block
    ends = pad.cumsum(0)
    order = torch.argsort(flat, stable=True)
    by = flat[order]
    row = (ends - pad)[by] + torch.arange(n, device=flat.device) - (counts.cumsum(0) - counts)[by]
    slots = torch.full((P,), n, dtype=torch.long, device=flat.device)
    slots[row] = order
    start = torch.arange(0, P, block, device=flat.device)
    return slots, torch.searchsorted(ends, start, right=True).clamp_max(E - 1)


def _products(rows, experts, w, block):
    """Padded rows (P, K) times the transposed weight of each block's expert -> (P, N)."""
    y = rows.view(-1, block, rows.shape[1]) @ w[experts].float().transpose(1, 2)
    return y.reshape(rows.shape[0], -1)


def _plain_layer(st):
    T, k, I = st["T"], st["k"], st["I"]
    n, block = T * k, 16 if T * k <= 16 * st["E"] else 64
    x, xs = (st["x"], st["xs"]) if st["xs"] is not None else _quant(st["x"].float())
    slots, experts = _by_expert(st["ids"], st["E"], block)
    token = slots.clamp_max(n - 1) // k
    y = _products(x.float()[token], experts, st["w13"], block) * xs[token]
    y *= st["s13"][experts].repeat_interleave(block, 0)
    gate, up = y[:, :I], y[:, I:]
    h, hs = _quant(gate / (1.0 + torch.exp(-gate)) * up)
    y = _products(h.float(), experts, st["w2"], block) * hs
    y *= st["s2"][experts].repeat_interleave(block, 0)
    by_slot = torch.empty((n + 1, st["H"]), device=y.device)
    by_slot[slots] = y
    return (by_slot[:n].view(T, k, -1) * st["tw"][:, :, None]).sum(1).to(st["out_dtype"])


_package = None


def _own():
    """The package, imported on first use."""
    global _package
    if _package is None:
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rdna4-vllm_amd")
        if at not in sys.path:
            sys.path.insert(0, at)
        import w4a8_fp8_wmma
        _package = w4a8_fp8_wmma
    return _package


def run(st):
    op = st["op"]
    if own:
        W = _own()
        if op == "route":
            return list(W.route_topk(st["logits"], st["k"], scoring=st["scoring"], bias=st["b"],
                                     num_groups=st["groups"], top_groups=st["top_groups"],
                                     renormalize=st["renorm"], scale=st["scale"]))
        if op == "dense":
            return W.int8_gemm(st["x"], st["xs"], st["w"], st["ws"], bias=st["b"], out_dtype=st["out_dtype"])
        return W.moe_int8_apply(st["x"], st["w13"], st["w2"], st["s13"], st["s2"], st["tw"], st["ids"],
                                x_scales=st["xs"], out_dtype=st["out_dtype"])
    if op == "route":
        return _plain_route(st)
    if op == "dense":
        return _plain_dense(st)
    return _plain_layer(st)


# --------------------------------------------------------------------------- what a pass needs
def _touched(T, k, E, zipf):
    """Expected number of distinct experts among T tokens' k different choices."""
    if not zipf:
        return E * (1 - (1 - k / E) ** T)
    p = [1 / (e + 1) ** 1.1 for e in range(E)]
    total = sum(p)
    # choices without replacement, as if k (at most E / 2) draws were independent
    return sum(1 - (1 - v / total) ** (T * k) for v in p)


def work(case):
    op = case["op"]
    if op == "route":
        T, E = case["T"], case["E"]
        return dict(bytes=T * E * (4 if case["dtype"] == "fp32" else 2) + 8 * T * case["k"], flops=8 * T * E)
    if op == "dense":
        M, N, K = case["M"], case["N"], case["K"]
        return dict(bytes=M * K * (1 if case["rows8"] else 2) + N * K + 4 * N + 2 * M * N, flops=2 * M * N * K)
    T, H, I, n = case["T"], case["H"], case["I"], case["T"] * case["k"]
    experts = _touched(T, case["k"], case["E"], case["zipf"])
    return dict(bytes=experts * (3 * H * I + 4 * (2 * I + H)) + T * H * (3 if case["rows8"] else 4), flops=6 * n * H * I)


# --------------------------------------------------------------------------- float64
def _exact_rows(v):
    """float64 rows -> (whole numbers, scales) of their int8 form: to the nearest, ties to even. The
    scale is an fp32 number by definition."""
    top = torch.clamp(v.abs().max(1).values, min=LEAST)[:, None]
    return torch.round(v * INT8_MAX / top), (top / INT8_MAX).float().double()


def _exact_route(case, st):
    """One expert after the other: the best that is left, the lowest index of equal ones."""
    l, T, E, size = st["logits"].double(), case["T"], case["E"], case["E"] // case["groups"]
    if case["scoring"] == "sigmoid":
        p = 1 / (1 + torch.exp(-l))
    else:
        e = torch.exp(l - l.max(1, keepdim=True).values)
        p = e / e.sum(1, keepdim=True)
    c = p.clone() if st["b"] is None else p + st["b"].double()
    c[torch.isinf(l)] = -math.inf
    index = torch.arange(E, device=l.device)

    def best(score):
        top = score.max(1, keepdim=True).values
        at = torch.where(score == top, index[: score.shape[1]], E).min(1, keepdim=True).values
        return top, at

    if case["groups"] > 1:
        g = torch.empty((T, case["groups"]), dtype=torch.float64, device=l.device)
        for j in range(case["groups"]):
            part = c[:, j * size:(j + 1) * size].clone()
            top, at = best(part)
            g[:, j] = top[:, 0]
            if st["b"] is not None:
                second = part.scatter(1, at, -math.inf).max(1).values
                g[:, j] += torch.where(torch.isinf(second), 0.0, second)
        out = torch.ones_like(g, dtype=torch.bool)
        # (a group is taken once, whatever its score)
        for _ in range(case["top_groups"]):
            score = torch.where(out, g, -math.inf)
            top = score.max(1, keepdim=True).values
            at = torch.where(out & (score == top), index[: case["groups"]], E).min(1, keepdim=True).values
            out = out.scatter(1, at, False)
        c = torch.where(out.repeat_interleave(size, 1), -math.inf, c)
    w = torch.zeros((T, case["k"]), dtype=torch.float64, device=l.device)
    ids = torch.full((T, case["k"]), -1, dtype=torch.int32, device=l.device)
    for j in range(case["k"]):
        top, at = best(c)
        real = top[:, 0] > -math.inf
        w[:, j] = torch.where(real, p.gather(1, at)[:, 0], 0.0)
        ids[:, j] = torch.where(real, at[:, 0], -1).to(torch.int32)
        c = c.scatter(1, at, -math.inf)
    if case["renorm"]:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    return [w * case["scale"], ids]


def exact(case, seed):
    st, op = prepare(case, seed), case["op"]
    if op == "route":
        return _exact_route(case, st)
    x, xs = (st["x"].double(), st["xs"].double()) if st["xs"] is not None else _exact_rows(st["x"].double())
    if op == "dense":
        y = (x @ st["w"].double().t()) * xs * st["ws"].double()
        return y if st["b"] is None else y + st["b"].double()
    I, out, ids = case["I"], torch.zeros_like(x), st["ids"].long()
    for e in torch.unique(ids).tolist():
        t, j = torch.nonzero(ids == e, as_tuple=True)
        gu = (x[t] @ st["w13"][e].double().t()) * xs[t] * st["s13"][e].double()
        h, hs = _exact_rows(gu[:, :I] * torch.sigmoid(gu[:, :I]) * gu[:, I:])
        y = (h @ st["w2"][e].double().t()) * hs * st["s2"][e].double()
        out.index_add_(0, t, y * st["tw"][t, j].double()[:, None])
    return out
