"""The training-side operators of the library, with their plain forms: the loss over the LM head and
its gradient, the gated feed-forward block with bf16 weights and its backward pass, and the 8-bit
activation checkpoints that the backward pass reads.

Sizes: the LM head of GPT-OSS (201088 rows of 2880) and the 2880 x 2880 block, next to shapes that are
generic. Inputs: rows of unit variance as behind an RMSNorm (with a spread of scales over the
channels), weights that keep gate and up of order one, LM head rows that give logits a standard
deviation of 2, a tenth of the targets ignored (prompt parts and padding).
"""
import math

import torch

own = False

CLAMP = 7.0
ALPHA = 1.702
VOCAB = 201088
GPT_OSS = dict(H=2880, I=2880)
FP8_MAX = 448.0


def _loss(name, op, T, dtype, V=VOCAB, H=2880):
    return dict(name=name, op=op, T=T, dtype=dtype, V=V, H=H)


def _ffn(name, op, T, dtype, H=2880, I=2880):  # noqa: E741
    return dict(name=name, op=op, T=T, dtype=dtype, H=H, I=I)


def listed():
    return [
        # the log-probability of one decoded token, from the rows that the layers return
        _loss("loss_1_f32", "loss", 1, "f32"),
        # a short odd prompt scored on a model of other dimensions, an odd vocabulary
        _loss("loss_333_f32", "loss", 333, "f32", V=50257, H=2048),
        # a long prompt scored
        _loss("loss_4096_bf16", "loss", 4096, "bf16"),
        # a training step's loss and gradient: rows and LM head
        _loss("lossgrad_2048_bf16", "lossgrad", 2048, "bf16"),
        # the same for a handful of tokens in f32, odd sizes
        _loss("lossgrad_19_f32", "lossgrad", 19, "f32", V=32003, H=1024),
        # the dense block for one token while decoding
        _ffn("ffn_1_bf16", "ffn", 1, "bf16"),
        # the dense block over a long prompt
        _ffn("ffn_4096_bf16", "ffn", 4096, "bf16"),
        # its backward pass, a training batch
        _ffn("ffngrad_4096_bf16", "ffngrad", 4096, "bf16"),
        # a short sequence, f32 rows, other dimensions
        _ffn("ffngrad_333_f32", "ffngrad", 333, "f32", H=2048, I=1536),
        # a checkpointed layer's step: forward that keeps its input in 8 bits, backward from that
        _ffn("ffn8_4096_bf16", "ffn8", 4096, "bf16"),
        _ffn("ffn8_257_f32", "ffn8", 257, "f32", H=1024, I=2056),
        # checkpoints alone: written and read back
        dict(name="act8_4096_f32", op="act8", T=4096, dtype="f32", H=2880),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.random()
    dtype = "bf16" if rng.random() < 0.6 else "f32"
    H = 2880 if rng.random() < 0.4 else 32 * rng.randint(4, 90)
    if kind < 0.40:
        op = "loss" if rng.random() < 0.5 else "lossgrad"
        V = VOCAB if rng.random() < 0.4 else _log_int(rng, 1000, VOCAB)
        top = 4096 if op == "loss" else 2048
        if dtype == "f32":
            top //= 4
        return dict(op=op, T=_log_int(rng, 1, top), dtype=dtype, V=V, H=H)
    if kind < 0.90:
        op = rng.choice(("ffn", "ffngrad", "ffn8"))
        return dict(op=op, T=_log_int(rng, 1, 4096 if dtype == "bf16" else 1024), dtype=dtype, H=H, I=8 * rng.randint(16, 400))
    return dict(op="act8", T=_log_int(rng, 1, 8192), dtype=dtype, H=H)


# ---------------------------------------------------------------- inputs, from the seed alone


def _gen(seed, *tags):
    g = torch.Generator(device="cuda")
    s = int(seed) * 1_000_003
    for t in tags:
        s = (s * 1009 + t + 17) % (1 << 62)
    return g.manual_seed(s)


def _type(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _rows(case, seed, tag, scale=1.0):
    g = _gen(seed, tag)
    spread = torch.exp(0.3 * torch.randn(case["H"], device="cuda", generator=g))
    return (torch.randn((case["T"], case["H"]), device="cuda", generator=g) * spread * scale).to(_type(case))


def _inputs(case, seed):
    T, H = case["T"], case["H"]
    d = dict(x=_rows(case, seed, 1))
    if case["op"] in ("loss", "lossgrad"):
        V, g = case["V"], _gen(seed, 2)
        w = torch.empty((V, H), dtype=torch.bfloat16, device="cuda")
        for part in w.split(32768):  # in pieces, to keep the f32 numbers small
            part.copy_(torch.randn(part.shape, device="cuda", generator=g) * (1.9 / math.sqrt(H)))
        targets = torch.randint(0, V, (T,), device="cuda", generator=g, dtype=torch.int32)
        ignored = torch.rand(T, device="cuda", generator=g) < 0.1
        ignored[0] = False
        d.update(w=w, targets=torch.where(ignored, torch.full_like(targets, -1), targets))
        if case["op"] == "lossgrad":  # of the mean over the tokens that count
            d["dloss"] = (d["targets"] >= 0).float() / (d["targets"] >= 0).sum()
    elif case["op"] != "act8":
        I, g = case["I"], _gen(seed, 3)  # noqa: E741

        def weight(rows, cols):
            return (torch.randn((rows, cols), device="cuda", generator=g) * (1.1 / math.sqrt(cols))).bfloat16()

        d.update(gate_up=weight(2 * I, H), gate_up_bias=torch.randn(2 * I, device="cuda", generator=g) * 0.1,
                 down=weight(H, I), down_bias=torch.randn(H, device="cuda", generator=g) * 0.1)
        if case["op"] != "ffn":
            d["dy"] = _rows(case, seed, 4, scale=1e-3)
    return d


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
    """What a program that uses the library keeps: its context, the resident LM head, its buffers."""

    def __init__(self, case, s):
        import silentotithrandousha_amd as pkg

        self.T, self.H, self.V, self.op = case["T"], case["H"], case.get("V"), case["op"]
        self.dtype = pkg.MOE_F32 if case["dtype"] == "f32" else pkg.MOE_BF16
        self.mxfp8 = pkg.MOE_MXFP8
        self.d = pkg.GpuMoeDispatcher(self.H, 32, CLAMP)
        self.p = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
        self.out = {}
        t, f = _type(case), torch.float32
        torch.cuda.synchronize()
        if self.V:
            self.d.init_lm_head_bf16_device(self.p["w"], self.V)
            self._new("loss", (self.T,), f)
            self._new("lse", (self.T,), f)
        if self.op == "lossgrad":
            self._new("dx", (self.T, self.H), t)
            self._new("dw", (self.V, self.H), t)
        if "I" in case:
            I = case["I"]  # noqa: E741
            self.block = pkg.GatedFfn(I, *(self.p[k] for k in ("gate_up", "gate_up_bias", "down", "down_bias")))
            if self.op != "ffngrad":
                self._new("y", (self.T, self.H), t)
            if self.op != "ffn":
                self._new("dx", (self.T, self.H), t)
                self._new("dgate_up", (2 * I, self.H), t)
                self._new("dgate_up_bias", (2 * I,), f)
                self._new("ddown", (self.H, I), t)
                self._new("ddown_bias", (self.H,), f)
                self.grads = pkg.GatedFfnGrads(*(self.p[k] for k in ("dx", "dgate_up", "dgate_up_bias", "ddown", "ddown_bias")))
        if self.op in ("ffn8", "act8"):
            self.x8 = torch.empty(self.d.act8_bytes(self.T, self.H), dtype=torch.uint8, device="cuda")
            self.p["packed"] = self.x8.data_ptr()
            self._new("x8", (self.T, self.H), t)

    def _new(self, name, shape, dtype):
        self.out[name] = torch.empty(shape, dtype=dtype, device="cuda")
        self.p[name] = self.out[name].data_ptr()

    def call(self):
        d, p, T, dt, st = self.d, self.p, self.T, self.dtype, _stream()
        if self.V:
            d.lm_head_loss_device(p["x"], dt, p["targets"], T, self.V, p["loss"], p["lse"], st)
            if self.op == "lossgrad":
                d.lm_head_loss_backward_device(p["x"], dt, p["targets"], p["lse"], p["dloss"], T, self.V, p["dx"], p["dw"], st)
        elif self.op == "ffn":
            d.ffn_forward_device(self.block, p["x"], dt, T, p["y"], stream=st)
        elif self.op == "ffngrad":
            d.ffn_backward_device(self.block, p["x"], dt, p["dy"], dt, T, self.grads, st)
        elif self.op == "ffn8":
            d.ffn_forward_device(self.block, p["x"], dt, T, p["y"], x8=p["packed"], stream=st)
            d.ffn_backward_device(self.block, p["packed"], self.mxfp8, p["dy"], dt, T, self.grads, st)
            d.act8_unpack_device(p["packed"], T, self.H, p["x8"], dt, st)
        else:
            d.act8_pack_device(p["x"], dt, T, self.H, p["packed"], st)
            d.act8_unpack_device(p["packed"], T, self.H, p["x8"], dt, st)
        return self.out


# ---------------------------------------------------------------- the plain forms


def _plain_x8(x):
    """The values that the 8-bit form of x [T, H] stands for: blocks of 32, a power-of-two scale (the
    smallest that leaves nothing above 448), e4m3 to nearest even. Steps of a power of two: exact."""
    b = x.float().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)  # top = m 2^e, m in [1/2, 1); 448 = 0.875 2^9
    e = (e - 9 + (m > 0.875).int()).clamp(min=-127)
    scaled = (b.double() * torch.exp2(-e.double())).float()
    _, se = torch.frexp(scaled.abs().clamp(min=2.0 ** -6))
    step = torch.exp2(se.double() - 4).float()
    return (torch.round(scaled / step) * step * torch.exp2(e.double())).float().flatten(-2)


def _plain_block(x, s):
    gu = x @ s["gate_up"].float().T + s["gate_up_bias"]
    g, u = gu[:, 0::2], gu[:, 1::2]
    G, U = g.clamp(max=CLAMP), u.clamp(-CLAMP, CLAMP)
    sig = 1.0 / (1.0 + torch.exp(-ALPHA * G))
    return g, u, G, U, sig, (U + 1.0) * G * sig


def _plain_block_backward(x, s, t):
    g, u, G, U, sig, h = _plain_block(x, s)
    dy = s["dy"].float()
    dh = dy @ s["down"].float()
    du = dh * G * sig * (u.abs() <= CLAMP)
    dg = dh * (U + 1.0) * sig * (1.0 + ALPHA * G * (1.0 - sig)) * (g <= CLAMP)
    dgu = torch.stack((dg, du), -1).flatten(-2)
    return dict(dx=(dgu @ s["gate_up"].float()).to(t), dgate_up=(dgu.T @ x).to(t), dgate_up_bias=dgu.sum(0),
                ddown=(dy.T @ h).to(t), ddown_bias=dy.sum(0))


def _plain(s):
    case = s["case"]
    op, t = case["op"], _type(case)
    x = s["x"].float()
    if op in ("loss", "lossgrad"):
        w = s["w"].float()
        logits = x @ w.T
        top = logits.amax(-1, keepdim=True)
        lse = torch.log(torch.exp(logits - top).sum(-1)) + top[:, 0]
        counts = s["targets"] >= 0
        at = s["targets"].clamp(min=0).long()[:, None]
        out = dict(loss=torch.where(counts, lse - logits.gather(1, at)[:, 0], torch.zeros_like(lse)), lse=lse)
        if op == "lossgrad":
            scale = (s["dloss"] * counts)[:, None]
            dl = torch.exp(logits - lse[:, None]) * scale
            dl.scatter_add_(1, at, -scale)
            out.update(dx=(dl @ w).to(t), dw=(dl.T @ x).to(t))
        return out
    if op == "act8":
        return dict(x8=_plain_x8(x).to(t))
    if op == "ffngrad":
        return _plain_block_backward(x, s, t)
    out = dict(y=(_plain_block(x, s)[-1] @ s["down"].float().T + s["down_bias"]).to(t))
    if op == "ffn8":
        x8 = _plain_x8(x)
        out.update(_plain_block_backward(x8, s, t), x8=x8.to(t))
    return out


def run(state):
    if own:
        return state["framework"].call()
    return _plain(state)


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    T, H, op = case["T"], case["H"], case["op"]
    b = 4 if case["dtype"] == "f32" else 2
    rows = b * T * H
    if op in ("loss", "lossgrad"):
        w = case["V"] * H
        if op == "loss":
            return {"bytes": 2 * w + rows + 12 * T, "flops": 2 * T * w}
        return {"bytes": (2 + b) * w + 2 * rows + 16 * T, "flops": 6 * T * w}
    if op == "act8":
        return {"bytes": 2 * rows + 2 * T * H * 33 // 32, "flops": 0}
    w = H * case["I"]
    forward = {"bytes": 6 * w + 2 * rows + 4 * (2 * case["I"] + H), "flops": 6 * T * w}
    if op == "ffn":
        return forward
    back = {"bytes": 6 * w + 3 * rows + 3 * b * w + 8 * (2 * case["I"] + H), "flops": 16 * T * w}
    if op == "ffngrad":
        return back
    # forward and backward, the checkpoint written and read between them and its values returned
    return {"bytes": forward["bytes"] + back["bytes"] + 3 * T * H * 33 // 32, "flops": forward["flops"] + back["flops"]}


# ---------------------------------------------------------------- the same in 64 bits


def _exact_x8(x):
    """Nearest of the e4m3 values (by their list) under the block's scale; ties to the even code."""
    pos = [m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** (k - 7) for k in range(1, 16) for m in range(8)]
    grid = torch.tensor(pos[:127], dtype=torch.float64, device="cuda")  # the last code is NaN
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / FP8_MAX)).nan_to_num(neginf=-127.0)
    e = torch.where(top > FP8_MAX * torch.exp2(e), e + 1, e)
    e = torch.where(top <= FP8_MAX * torch.exp2(e - 1), e - 1, e).clamp(min=-127)
    v = b.abs() / torch.exp2(e)
    hi = torch.searchsorted(grid, v).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    down, up = v - grid[lo], grid[hi] - v
    pick = torch.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    return (grid[pick] * torch.sign(b) * torch.exp2(e)).flatten(-2)


def _exact_loss(case, d):
    x, w, targets = d["x"].double(), d["w"], d["targets"]
    T, H, V = case["T"], case["H"], case["V"]
    top = torch.full((T,), -math.inf, dtype=torch.float64, device="cuda")
    total = torch.zeros_like(top)
    picked = torch.zeros_like(top)
    for first in range(0, V, 16384):
        logits = x @ w[first:first + 16384].double().T
        new = torch.maximum(top, logits.amax(1))
        total = total * torch.exp(top - new) + torch.exp(logits - new[:, None]).sum(1)
        top = new
        here = (targets >= first) & (targets < first + logits.shape[1])
        picked[here] = logits[here, (targets[here] - first).long()]
    lse = top + torch.log(total)
    out = dict(loss=torch.where(targets >= 0, lse - picked, torch.zeros_like(lse)), lse=lse)
    if case["op"] == "lossgrad":
        scale = d["dloss"].double() * (targets >= 0)
        dx = torch.zeros_like(x)
        dw = torch.empty((V, H), dtype=torch.float64, device="cuda")
        for first in range(0, V, 16384):
            part = w[first:first + 16384].double()
            p = torch.exp(x @ part.T - lse[:, None])
            p -= (targets[:, None] == torch.arange(first, first + part.shape[0], device="cuda")[None, :]).double()
            p *= scale[:, None]
            dx += p @ part
            dw[first:first + part.shape[0]] = p.T @ x
        out.update(dx=dx, dw=dw)
    return out


def _exact_block(x, d, dy=None):
    wg, wu = d["gate_up"][0::2].double(), d["gate_up"][1::2].double()
    bias, wd = d["gate_up_bias"].double(), d["down"].double()
    g, u = x @ wg.T + bias[0::2], x @ wu.T + bias[1::2]
    low, mid = torch.minimum(g, torch.full_like(g, CLAMP)), torch.clip(u, -CLAMP, CLAMP)
    sig = torch.sigmoid(ALPHA * low)
    glu = low * sig
    h = (mid + 1) * glu
    if dy is None:
        return dict(y=h @ wd.T + d["down_bias"].double())
    dh = dy @ wd
    du = torch.where(u.abs() <= CLAMP, dh * glu, torch.zeros_like(dh))
    dg = torch.where(g <= CLAMP, dh * (mid + 1) * (sig + ALPHA * glu * (1 - sig)), torch.zeros_like(dh))
    n, H = d["gate_up"].shape
    dw, db = torch.empty((n, H), dtype=torch.float64, device="cuda"), torch.empty(n, dtype=torch.float64, device="cuda")
    dw[0::2], dw[1::2] = dg.T @ x, du.T @ x
    db[0::2], db[1::2] = dg.sum(0), du.sum(0)
    return dict(dx=dg @ wg + du @ wu, dgate_up=dw, dgate_up_bias=db, ddown=dy.T @ h, ddown_bias=dy.sum(0))


def exact(case, seed):
    d, op = _inputs(case, seed), case["op"]
    if op in ("loss", "lossgrad"):
        return _exact_loss(case, d)
    x = d["x"].double()
    if op == "act8":
        return dict(x8=_exact_x8(x))
    if op == "ffn":
        return _exact_block(x, d)
    if op == "ffngrad":
        return _exact_block(x, d, d["dy"].double())
    x8 = _exact_x8(x)
    return dict(_exact_block(x, d), **_exact_block(x8, d, d["dy"].double()), x8=x8)
