"""The serving-side operators beside the experts, with their plain forms: rows and weights quantised to
MXFP4, products with a resident MXFP4 matrix, the choice of experts by other rules than the path's own
(with its gradient), and the choice of a token from logits.

Sizes: the matrices, experts and vocabulary of GPT-OSS (2880, 5760, 32 experts, 201088 tokens) next to
shapes that are generic. Inputs: rows of unit variance as behind an RMSNorm, with a spread of scales over
the channels; weights that keep results of order one; router logits of a standard deviation of 1.5 with a
bias as a balance rule leaves it; logits of the vocabulary with a few tokens far above the rest.
"""
import math

import torch

own = False

VOCAB = 201088
FP8_MAX = 448.0


def _quant(name, T, C, dtype):
    return dict(name=name, op="quant", T=T, C=C, dtype=dtype)


def _mm(name, op, T, R, C, dtype):
    return dict(name=name, op=op, T=T, R=R, C=C, dtype=dtype)


def _route(name, op, T, E, k, score, groups=0, top_groups=0, two=False, bias=False, normalize=True):
    return dict(name=name, op=op, T=T, E=E, k=k, score=score, groups=groups, top_groups=top_groups, two=two, bias=bias,
                normalize=normalize)


def _sample(name, T, V, rule):
    return dict(name=name, op="sample", T=T, V=V, rule=rule)


def listed():
    return [
        # the row of one decoded token, quantised and read back
        _quant("quant_1_f32", 1, 2880, "f32"),
        # four experts' gate and up matrices, from a bf16 checkpoint
        _quant("quant_23040_bf16", 23040, 2880, "bf16"),
        # a quantised dense layer for one token while decoding
        _mm("mm_1_f32", "mm", 1, 5760, 2880, "f32"),
        # a short prompt on a model of other dimensions, in f32
        _mm("mm_333_f32", "mm", 333, 2064, 1056, "f32"),
        # a long prompt's bf16 rows, as they are
        _mm("mm_4096_bf16", "mm", 4096, 2880, 2880, "bf16"),
        # a batch of decoding sequences with rows of 8 bits
        _mm("mm8_128_bf16", "mm8", 128, 5760, 2880, "bf16"),
        # a long prompt with rows of 4 bits, both operands microscaled
        _mm("mm4_4096_bf16", "mm4", 4096, 5760, 2880, "bf16"),
        # one token's experts: softmax of the chosen
        _route("route_1_softmax", "route", 1, 32, 4, "softmax"),
        # a training batch: sigmoid scores, a balance bias, groups, and the gradient of the weights
        _route("routegrad_16384_sigmoid", "routegrad", 16384, 256, 8, "sigmoid", 8, 4, True, True),
        # the next token of one sequence: temperature, top-k, top-p and min-p
        _sample("sample_1", 1, VOCAB, "all"),
        # a small vocabulary, odd, only a temperature
        _sample("sample_37_plain", 37, 32003, "temperature"),
        # a batch of requests, each with settings of its own
        _sample("sample_256_mixed", 256, VOCAB, "mixed"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.random()
    dtype = "bf16" if rng.random() < 0.6 else "f32"
    if kind < 0.2:
        return dict(op="quant", T=_log_int(rng, 1, 8192), C=32 * rng.randint(4, 180), dtype=dtype)
    if kind < 0.55:
        op = rng.choice(("mm", "mm", "mm8", "mm4"))
        top = 4096 if dtype == "bf16" or op != "mm" else 1024
        C = 2880 if rng.random() < 0.4 else 32 * rng.randint(4, 90)
        return dict(op=op, T=_log_int(rng, 1, top), R=16 * _log_int(rng, 8, 360), C=C, dtype=dtype)
    if kind < 0.75:
        score = rng.choice(("softmax", "sigmoid"))
        groups = rng.choice((0, 0, 4, 8))
        E = groups * rng.randint(2, 32) if groups else _log_int(rng, 8, 256)
        top_groups = rng.randint(1, groups) if groups else 0
        most = E // groups * top_groups if groups else E
        return dict(op=rng.choice(("route", "routegrad")), T=_log_int(rng, 1, 16384), E=E, k=rng.randint(1, min(16, most)), score=score,
                    groups=groups, top_groups=top_groups, two=bool(groups) and rng.random() < 0.5, bias=rng.random() < 0.5,
                    normalize=rng.random() < 0.7)
    return dict(op="sample", T=_log_int(rng, 1, 256), V=VOCAB if rng.random() < 0.3 else _log_int(rng, 1000, VOCAB),
                rule=rng.choice(("all", "temperature", "mixed", "mixed")))


# ---------------------------------------------------------------- inputs, from the seed alone


def _gen(seed, *tags):
    g = torch.Generator(device="cuda")
    s = int(seed) * 1_000_003
    for t in tags:
        s = (s * 1009 + t + 17) % (1 << 62)
    return g.manual_seed(s)


def _type(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _rows(case, seed, tag):
    g = _gen(seed, tag)
    spread = torch.exp(0.3 * torch.randn(case["C"], device="cuda", generator=g))
    return (torch.randn((case["T"], case["C"]), device="cuda", generator=g) * spread).to(_type(case))


def _inputs(case, seed):
    op, T = case["op"], case["T"]
    if op == "quant":
        return dict(x=_rows(case, seed, 1))
    if op in ("mm", "mm8", "mm4"):
        R, C, g = case["R"], case["C"], _gen(seed, 2)
        # any codes, scales around 1 / sqrt(C) of unit values
        s0 = 127 - round(math.log2(math.sqrt(C) * 2.5))
        return dict(x=_rows(case, seed, 1),
                    blocks=torch.randint(0, 256, (R, C // 32, 16), device="cuda", generator=g, dtype=torch.uint8),
                    scales=torch.randint(s0 - 1, s0 + 2, (R, C // 32), device="cuda", generator=g, dtype=torch.uint8),
                    bias=torch.randn(R, device="cuda", generator=g) * 0.1)
    if op in ("route", "routegrad"):
        E, g = case["E"], _gen(seed, 3)
        d = dict(logits=torch.randn((T, E), device="cuda", generator=g) * 1.5 + torch.randn(E, device="cuda", generator=g) * 0.5)
        if case["bias"]:
            d["bias"] = torch.randn(E, device="cuda", generator=g) * (0.1 if case["score"] == "sigmoid" else 0.3 / E)
        if op == "routegrad":
            d["dweights"] = torch.randn((T, case["k"]), device="cuda", generator=g)
        return d
    V, rule, g = case["V"], case["rule"], _gen(seed, 4)
    logits = torch.randn((T, V), device="cuda", generator=g) * 2.0
    raised = torch.randint(0, V, (T, 64), device="cuda", generator=g)
    up = -4.0 * torch.log(1.0 - torch.rand((T, 64), device="cuda", generator=g)) + 4.0
    logits.scatter_reduce_(1, raised, up, "amax")
    share = {"all": 1.0, "mixed": 0.5, "temperature": 0.0}[rule]

    def some(values, off):  # of the rows that have this setting
        return torch.where(torch.rand(T, device="cuda", generator=g) < share, values, torch.full_like(values, off))

    def uniform(lo, hi):
        return lo + (hi - lo) * torch.rand(T, device="cuda", generator=g)

    temperature = uniform(0.6, 1.2)
    if rule == "mixed":  # some requests decode greedily
        temperature = torch.where(torch.rand(T, device="cuda", generator=g) < 0.15, torch.zeros_like(temperature), temperature)
    top_k = torch.randint(20, 400, (T,), device="cuda", generator=g, dtype=torch.int32)
    top_p, min_p = uniform(0.8, 0.98), uniform(0.005, 0.05)
    return dict(logits=logits, temperature=temperature,
                top_k=some(top_k, 0), top_p=some(top_p, 1.0), min_p=some(min_p, 0.0), u=torch.rand(T, device="cuda", generator=g))


_side = None


def _stream():
    """The stream that every call of the program is enqueued on."""
    global _side
    if _side is None:
        _side = torch.cuda.Stream()
    return _side.cuda_stream


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if own:
        s["framework"] = _Program(case, s)
    return s


# ---------------------------------------------------------------- the framework's calls


class _Program:
    """What a program that uses the library keeps: its context, the resident matrix, its buffers."""

    def __init__(self, case, s):
        import silentotithrandousha_amd as pkg

        self.case, self.op, self.T = case, case["op"], case["T"]
        self.d = pkg.GpuMoeDispatcher(32, 32)
        self.f32, self.mxfp4, self.mxfp8 = pkg.MOE_F32, pkg.MOE_MXFP4, pkg.MOE_MXFP8
        self.p = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
        self.out, self.buf = {}, {}
        T, f, i, b = self.T, torch.float32, torch.int32, torch.uint8
        torch.cuda.synchronize()
        if "dtype" in case:
            self.dtype = pkg.MOE_F32 if case["dtype"] == "f32" else pkg.MOE_BF16
        if self.op in ("quant", "mm4"):
            self._new(self.buf, "x_blocks", (T, case["C"] // 32, 16), b)
            self._new(self.buf, "x_scales", (T, case["C"] // 32), b)
        if self.op == "mm8":
            self._new(self.buf, "x8", (self.d.act8_bytes(T, case["C"]),), b)
        if self.op == "quant":
            self._new(self.out, "x4", (T, case["C"]), f)
        elif "R" in case:
            self._new(self.buf, "packed", (self.d.mxfp4_packed_size(case["R"], case["C"]),), b)
            self.d.mxfp4_pack_device(self.p["blocks"], self.p["scales"], case["R"], case["C"], self.p["packed"])
            self.d.synchronize()
            self._new(self.out, "y", (T, case["R"]), _type(case))
        elif "E" in case:
            self.rule = pkg.Routing(score=pkg.MOE_SCORE_SIGMOID if case["score"] == "sigmoid" else pkg.MOE_SCORE_SOFTMAX,
                                    normalize=case["normalize"], top_k=case["k"], n_groups=case["groups"],
                                    top_groups=case["top_groups"], group_score=pkg.MOE_GROUP_TOP2 if case["two"] else pkg.MOE_GROUP_MAX,
                                    scale=2.5 if case["score"] == "sigmoid" else 1.0, bias=self.p.get("bias"))
            self._new(self.out, "idx", (T, case["k"]), i)
            self._new(self.out, "weights", (T, case["k"]), f)
            self._new(self.out, "counts", (case["E"],), i)
            if self.op == "routegrad":
                self._new(self.out, "dlogits", (T, case["E"]), f)
        else:
            self.rule = pkg.Sampling(*(self.p[k] for k in ("temperature", "top_k", "top_p", "min_p")))
            self._new(self.out, "tokens", (T,), i)
            self._new(self.out, "logprob", (T,), f)

    def _new(self, where, name, shape, dtype):
        where[name] = torch.empty(shape, dtype=dtype, device="cuda")
        self.p[name] = where[name].data_ptr()

    def call(self):
        d, p, T, c, st = self.d, self.p, self.T, self.case, _stream()
        if self.op == "quant":
            d.mxfp4_quantize_device(p["x"], self.dtype, T, c["C"], p["x_blocks"], p["x_scales"], st)
            d.mxfp4_dequant_device(p["x_blocks"], p["x_scales"], T, c["C"], p["x4"], st)
        elif "R" in c:
            x, x_type, x_scales = p["x"], self.dtype, None
            if self.op == "mm4":
                d.mxfp4_quantize_device(x, self.dtype, T, c["C"], p["x_blocks"], p["x_scales"], st)
                x, x_type, x_scales = p["x_blocks"], self.mxfp4, p["x_scales"]
            elif self.op == "mm8":
                d.act8_pack_device(x, self.dtype, T, c["C"], p["x8"], st)
                x, x_type = p["x8"], self.mxfp8
            d.mxfp4_matmul_device(p["packed"], c["R"], c["C"], p["bias"], x, x_type, x_scales, T, p["y"], self.dtype, st)
        elif "E" in c:
            d.route_device(self.rule, p["logits"], T, c["E"], p["idx"], p["weights"], p["counts"], st)
            if self.op == "routegrad":
                d.route_backward_device(self.rule, p["logits"], p["idx"], p["dweights"], T, c["E"], p["dlogits"], st)
        else:
            d.sample_device(self.rule, p["logits"], c["V"], p["u"], T, c["V"], p["tokens"], p["logprob"], st)
        return self.out


# ---------------------------------------------------------------- the plain forms


def _plain_x4(x):
    """The values that MXFP4 rows stand for: blocks of 32 over 2^(floor(log2 of the largest) - 2), E2M1 to
    nearest even, at most 6. Steps of a power of two: exact."""
    b = x.float().unflatten(-1, (-1, 32))
    _, e = torch.frexp(b.abs().amax(-1, keepdim=True))  # the largest is m 2^e, m in [1/2, 1)
    e = (e - 3).clamp(min=-126)
    v = (b.double() * torch.exp2(-e.double())).float()
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return ((torch.round(v / step) * step).clamp(-6.0, 6.0) * torch.exp2(e.double())).float().flatten(-2)


def _plain_x8(x):
    """The values that the 8-bit form stands for: the smallest power of two that leaves nothing above 448, e4m3."""
    b = x.float().unflatten(-1, (-1, 32))
    m, e = torch.frexp(b.abs().amax(-1, keepdim=True))
    e = (e - 9 + (m > 0.875).int()).clamp(min=-127)
    v = (b.double() * torch.exp2(-e.double())).float()
    _, ve = torch.frexp(v.abs().clamp(min=2.0 ** -6))
    step = torch.exp2(ve.double() - 4).float()
    return (torch.round(v / step) * step * torch.exp2(e.double())).float().flatten(-2)


def _plain_weights(blocks, scales):
    lut = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device="cuda")
    codes = torch.stack((blocks & 15, blocks >> 4), -1).flatten(-2).int()
    return (lut[codes] * torch.exp2(scales.float() - 127.0)[..., None]).flatten(-2)


def _plain_route(s):
    """Scores in 64 bits: which experts are chosen hangs on their order."""
    case, l64 = s["case"], s["logits"].double()
    T, E, k = case["T"], case["E"], case["k"]
    if case["score"] == "softmax":
        ex = torch.exp(l64 - l64.amax(1, keepdim=True))
        scores = ex / ex.sum(1, keepdim=True)
    else:
        scores = 1.0 / (1.0 + torch.exp(-l64))
    key = scores + s["bias"].double() if case["bias"] else scores
    order_by = key if case["bias"] else l64  # without a bias the logits' order is the scores'
    if case["groups"]:
        per = key.view(T, case["groups"], -1).sort(dim=-1, descending=True).values
        group = per[..., 0] + per[..., 1] if case["two"] else per[..., 0]
        kept = group.sort(dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        mask = torch.zeros((T, case["groups"]), dtype=torch.bool, device="cuda").scatter_(1, kept, True)
        order_by = torch.where(mask.repeat_interleave(E // case["groups"], 1), order_by, -math.inf)
    idx = order_by.sort(dim=1, descending=True, stable=True).indices[:, :k]
    w = scores.gather(1, idx)
    scale = 2.5 if case["score"] == "sigmoid" else 1.0
    total = w.sum(1, keepdim=True) if case["normalize"] else torch.ones_like(w[:, :1])
    out = dict(idx=idx.int(), weights=(scale * w / total).float(), counts=torch.bincount(idx.flatten(), minlength=E).int())
    if case["op"] == "routegrad":
        dw = s["dweights"].double() * scale
        dscore = dw / total
        if case["normalize"]:
            dscore = dscore - (dw * w).sum(1, keepdim=True) / total ** 2
        full = torch.zeros_like(scores).scatter_add_(1, idx, dscore)
        if case["score"] == "softmax":
            out["dlogits"] = (scores * (full - (full * scores).sum(1, keepdim=True))).float()
        else:
            out["dlogits"] = (full * scores / (1.0 + torch.exp(l64))).float()
    return out


def _plain_sample(s):
    """In 64 bits: a token is drawn by where a sum over the vocabulary passes the random number."""
    l64, V = s["logits"].double(), s["logits"].shape[1]
    greedy = s["temperature"] <= 0
    tau = torch.where(greedy, torch.ones_like(s["temperature"]), s["temperature"]).double()[:, None]
    sorted_l, order = l64.sort(dim=1, descending=True, stable=True)
    e = torch.exp((sorted_l - sorted_l[:, :1]) / tau)
    k = torch.where(s["top_k"] > 0, s["top_k"], torch.full_like(s["top_k"], V))[:, None]
    e = torch.where(torch.arange(V, device="cuda")[None, :] < k, e, torch.zeros_like(e))
    before = torch.cumsum(e, 1) - e
    p = s["top_p"].double()[:, None]
    e = torch.where(((before < p * e.sum(1, keepdim=True)) | (p >= 1)) & (e >= s["min_p"].double()[:, None]), e, torch.zeros_like(e))
    total = e.sum(1, keepdim=True)
    e = torch.zeros_like(e).scatter_(1, order, e)  # in the vocabulary's order
    token = ((torch.cumsum(e, 1) > s["u"].double()[:, None] * total) & (e > 0)).to(torch.int8).argmax(1)
    token = torch.where(greedy, order[:, 0], token)
    logprob = torch.log(e.gather(1, token[:, None])[:, 0] / total[:, 0])
    return dict(tokens=token.int(), logprob=torch.where(greedy, torch.zeros_like(logprob), logprob).float())


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "quant":
        return dict(x4=_plain_x4(s["x"]))
    if op in ("route", "routegrad"):
        return _plain_route(s)
    if op == "sample":
        return _plain_sample(s)
    x = _plain_x4(s["x"]) if op == "mm4" else _plain_x8(s["x"]) if op == "mm8" else s["x"].float()
    return dict(y=(x @ _plain_weights(s["blocks"], s["scales"]).T + s["bias"]).to(_type(case)))


def run(state):
    if own:
        return state["framework"].call()
    return _plain(state)


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    T, op = case["T"], case["op"]
    if "C" in case:
        C, b = case["C"], 4 if case["dtype"] == "f32" else 2
        if op == "quant":  # written and read back
            return {"bytes": (b + 4) * T * C + 2 * T * C * 17 // 32, "flops": 0}
        R = case["R"]
        return {"bytes": b * T * (C + R) + R * C * 17 // 32 + 4 * R, "flops": 2 * T * R * C}
    if op == "sample":
        return {"bytes": 4 * T * case["V"] + 28 * T, "flops": 0}
    one = 4 * T * case["E"]
    bytes_ = one + 8 * T * case["k"] + 8 * case["E"]
    if op == "routegrad":
        bytes_ += 2 * one + 8 * T * case["k"]
    return {"bytes": bytes_, "flops": 0}


# ---------------------------------------------------------------- the same in 64 bits


def _nearest(v, grid):
    """The nearest of the grid's values (codes in order) to v >= 0, ties to the even code, at most the last."""
    hi = torch.searchsorted(grid, v).clamp(max=len(grid) - 1)
    lo = (hi - 1).clamp(min=0)
    down, up = v - grid[lo], grid[hi] - v
    return grid[torch.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)]


def _exact_x4(x):
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top)).nan_to_num(neginf=-126.0)
    e = torch.where(torch.exp2(e) > top, e - 1, torch.where(torch.exp2(e + 1) <= top, e + 1, e))
    s = torch.exp2((e - 2).clamp(min=-126.0))
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
    return (_nearest(b.abs() / s, grid) * torch.sign(b) * s).flatten(-2)


def _exact_x8(x):
    pos = [m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** (k - 7) for k in range(1, 16) for m in range(8)]
    grid = torch.tensor(pos[:127], dtype=torch.float64, device="cuda")  # the last code is NaN
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / FP8_MAX)).nan_to_num(neginf=-127.0)
    e = torch.where(top > FP8_MAX * torch.exp2(e), e + 1, e)
    e = torch.where(top <= FP8_MAX * torch.exp2(e - 1), e - 1, e).clamp(min=-127)
    return (_nearest(b.abs() / torch.exp2(e), grid) * torch.sign(b) * torch.exp2(e)).flatten(-2)


def _exact_weights(d):
    byte = d["blocks"].long()
    codes = torch.empty(byte.shape[:-1] + (32,), dtype=torch.long, device="cuda")
    codes[..., 0::2], codes[..., 1::2] = byte % 16, byte // 16
    m, e = codes % 2, (codes // 2) % 4
    size = torch.where(e == 0, m.double() / 2, (1 + m.double() / 2) * torch.exp2(e.double() - 1))
    w = torch.where(codes >= 8, -size, size) * torch.exp2(d["scales"].double() - 127)[..., None]
    return w.flatten(-2)


def _exact_route(case, d):
    """The k largest one after the other, and the gradient by the chain rule of log weights."""
    z = d["logits"].double()
    T, E, k, rows = case["T"], case["E"], case["k"], torch.arange(case["T"], device="cuda")
    scores = torch.softmax(z, 1) if case["score"] == "softmax" else torch.sigmoid(z)
    bias = d["bias"].double() if case["bias"] else torch.zeros(E, dtype=torch.float64, device="cuda")
    left = scores + bias if case["bias"] else z.clone()
    if case["groups"]:
        per = (scores + bias).reshape(T, case["groups"], -1)
        best = per.amax(2)
        if case["two"]:
            rest = per.scatter(2, per.argmax(2, keepdim=True), -math.inf)
            best = best + rest.amax(2)
        allowed = torch.zeros_like(best, dtype=torch.bool)
        for _ in range(case["top_groups"]):
            at = best.argmax(1)
            allowed[rows, at] = True
            best[rows, at] = -math.inf
        left = left.masked_fill(~allowed.repeat_interleave(E // case["groups"], 1), -math.inf)
    idx = torch.empty((T, k), dtype=torch.long, device="cuda")
    for j in range(k):
        idx[:, j] = left.argmax(1)
        left[rows, idx[:, j]] = -math.inf
    chosen = scores.gather(1, idx)
    w = chosen / chosen.sum(1, keepdim=True) if case["normalize"] else chosen
    w = w * (2.5 if case["score"] == "sigmoid" else 1.0)
    counts = (idx.flatten()[:, None] == torch.arange(E, device="cuda")[None, :]).sum(0) if T * k * E < 1 << 26 else \
        torch.zeros(E, dtype=torch.long, device="cuda").scatter_add_(0, idx.flatten(), torch.ones(T * k, dtype=torch.long, device="cuda"))
    out = dict(idx=idx, weights=w, counts=counts)
    if case["op"] == "routegrad":
        g = d["dweights"].double() * w  # d / d log w
        if case["normalize"]:  # log w_j = log s_j - log sum s
            g = g - chosen / chosen.sum(1, keepdim=True) * g.sum(1, keepdim=True)
        dz = torch.zeros_like(z)
        if case["score"] == "softmax":  # log s_j = z_j - log sum exp z
            dz.scatter_(1, idx, g)
            dz -= scores * g.sum(1, keepdim=True)
        else:
            dz.scatter_(1, idx, g * torch.sigmoid(-z).gather(1, idx))
        out["dlogits"] = dz
    return out


def _exact_sample(case, d):
    """Row by row, in probabilities."""
    T, V = case["T"], case["V"]
    tokens, logprob = torch.empty(T, dtype=torch.long, device="cuda"), torch.zeros(T, dtype=torch.float64, device="cuda")
    settings = torch.stack([d[k].double() for k in ("temperature", "top_k", "top_p", "min_p", "u")]).tolist()
    for t, (tau, k, top_p, min_p, u) in enumerate(zip(*settings)):
        row = d["logits"][t].double()
        if tau <= 0:
            tokens[t] = torch.nonzero(row == row.max())[0, 0]
            continue
        order = torch.argsort(-row, stable=True)
        n = min(int(k), V) if k > 0 else V
        p = torch.softmax(row[order[:n]] / tau, 0)
        keep = p >= min_p * p[0]
        if top_p < 1:
            keep &= torch.cumsum(p, 0) - p < top_p
        kept, at = order[:n][keep].sort()
        p = p[keep][at]
        p = p / p.sum()
        pos = int((torch.cumsum(p, 0) <= u).sum().clamp(max=len(p) - 1))
        tokens[t], logprob[t] = kept[pos], torch.log(p[pos])
    return dict(tokens=tokens, logprob=logprob)


def exact(case, seed):
    d, op = _inputs(case, seed), case["op"]
    if op == "quant":
        return dict(x4=_exact_x4(d["x"]))
    if op in ("route", "routegrad"):
        return _exact_route(case, d)
    if op == "sample":
        return _exact_sample(case, d)
    x = _exact_x4(d["x"]) if op == "mm4" else _exact_x8(d["x"]) if op == "mm8" else d["x"].double()
    return dict(y=x @ _exact_weights(d).T + d["bias"].double())
