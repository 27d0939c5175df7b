"""Operators that serve a model in 8 bits: products of 8-bit integers with a
scale for each token and output channel, the gated feed-forward block built of
them, and attention over keys and values cached in 8 bits with a scale for each
block of 64 tokens and head.

Rows in 8 bits (c the codes, s the row's scale):
    s = max|x| / 127,  c = rint(127 x / max|x|), ties to even
Projection (kind "linear"), x quantised within the pass, W beforehand:
    y = act(s_x s_w (c_x c_w^T) + b); act is nothing or the tanh form of GELU
Gated block (kind "mlp"), behind no norm or one of the two adaLN norms, whose
32-bit rows are quantised, as are the rows of h:
    [g | u] = product with W1,  h = silu(g) u,  y = product with W2
Cache (kind "store"): rows of K and V into blocks of 64 tokens; tokens behind
those that a block has widen its scale where they need to,
    s' = max(s, max|new| / 127),  c' = rint(c s / s')
Attention (kind "attend"): the query rows of request i attend to its own rows
of the cache, in `heads` heads that share `kv_heads` key heads.

Widths are the repository's two model families' (hidden 5376 with an FFN of
14336, hidden 5120 with one of 13824, 40 or 56 heads of 128) or generic ones;
rows are those of their clips (778, 1536, 2378, 6144), prompts of up to 512
tokens, and single rows.  Inputs are N(0, 1) activations and 0.02 N(0, 1)
weights, as in the repository's benchmark.
"""
import ctypes
import math
import os
import sys

import torch
import numpy as np

own = False


def listed():
    return [
        # a pooled or time embedding of one request: the smallest product,
        # bound by the weight
        {"name": "linear_row_1", "kind": "linear", "rows": 1, "in": 5120,
         "out": 5120, "gelu": False},
        # two prompts through a projection of odd widths
        {"name": "linear_odd_197", "kind": "linear", "rows": 197, "in": 1283,
         "out": 2051, "gelu": True},
        # the QKV projection of one 512x512 clip
        {"name": "linear_qkv_2378", "kind": "linear", "rows": 2378,
         "in": 5376, "out": 21504, "gelu": False},
        # the first projection of the ungated FFN, a longer clip
        {"name": "linear_ffn_6144", "kind": "linear", "rows": 6144,
         "in": 5120, "out": 13824, "gelu": True},
        # the gated FFN of a single row
        {"name": "mlp_row_1", "kind": "mlp", "rows": 1, "in": 5376,
         "hidden": 14336, "out": 5376, "norm": "none"},
        # the text refiner's kind of block on a prompt, odd widths
        {"name": "mlp_odd_300", "kind": "mlp", "rows": 300, "in": 1001,
         "hidden": 2675, "out": 1001, "norm": "layer"},
        # the gated FFN behind its norm, two 512x512 clips
        {"name": "mlp_clips_4756", "kind": "mlp", "rows": 4756, "in": 5376,
         "hidden": 14336, "out": 5376, "norm": "rms"},
        # the text keys and values of three requests
        {"name": "store_text_3", "kind": "store", "has": "0,0,0",
         "new": "512,77,300", "kv_heads": 40, "dim": 128},
        # the next token of 16 requests
        {"name": "store_next_16", "kind": "store",
         "has": "20,33,511,77,126,1,300,64,65,63,200,411,90,18,256,150",
         "new": ",".join(["1"] * 16), "kv_heads": 8, "dim": 128},
        # one row of each of 16 requests against its prompt
        {"name": "attend_rows_16", "kind": "attend",
         "q": ",".join(["1"] * 16),
         "kv": "20,33,512,77,126,1,300,64,65,63,200,411,90,18,256,150",
         "heads": 40, "kv_heads": 40, "dim": 128},
        # one row of each of 8 requests against long contexts, shared heads:
        # bound by reading the cache
        {"name": "attend_rows_8_long", "kind": "attend",
         "q": ",".join(["1"] * 8),
         "kv": "9720,6144,8191,4096,5000,9001,7777,6145", "heads": 64,
         "kv_heads": 8, "dim": 128},
        # four 512x512 clips against their prompts, one of them empty
        {"name": "attend_cross_4", "kind": "attend",
         "q": "6144,6144,6144,6144", "kv": "512,77,300,0", "heads": 40,
         "kv_heads": 40, "dim": 128},
    ]


def draw(rng):
    def between(low, high):
        return int(round(math.exp(rng.uniform(math.log(low),
                                              math.log(high)))))

    def text(values):
        return ",".join(str(v) for v in values)

    kind = rng.choice(["linear", "linear", "mlp", "store", "attend",
                       "attend"])
    largest = 4756 * 3 * 5376 * 14336  # multiplications of the largest block
    if kind == "linear":
        k, n = rng.choice([(5120, 5120), (5120, 13824), (5376, 21504),
                           (7168, 5376), (2688, 10752),
                           (between(32, 6000), between(32, 6000)),
                           (between(32, 6000), between(32, 6000))])
        return {"kind": kind, "rows": between(1, min(6144, largest // (k * n))),
                "in": k, "out": n, "gelu": rng.random() < 0.3}
    if kind == "mlp":
        k, h = rng.choice([(5376, 14336), (5120, 13824), (512, 1536),
                           (between(32, 2000), between(32, 6000)),
                           (between(32, 2000), between(32, 6000))])
        return {"kind": kind,
                "rows": between(1, min(4756, largest // (3 * k * h))),
                "in": k, "hidden": h, "out": k,
                "norm": rng.choice(["none", "rms", "layer"])}
    heads, kv_heads, dim = rng.choice(
        [(40, 40, 128), (56, 56, 128), (64, 8, 128), (32, 8, 64), (16, 2, 128),
         (12, 12, 64), (24, 4, 96), (10, 5, 80)])
    n = rng.choice([1, 2, 3, 4, 7, 8, 16])
    if kind == "store":
        begun = rng.random() < 0.5
        return {"kind": kind, "has": text(
                    [rng.randint(0, 1536 // n) if begun else 0
                     for _ in range(n)]),
                "new": text([rng.choice([1, between(1, 1536 // n)])
                             for _ in range(n)]),
                "kv_heads": kv_heads, "dim": dim}
    high = rng.choice([1, 4, 6144])  # single rows, a few, whole clips
    q = [between(1, min(high, 24576 // n)) for _ in range(n)]
    kv = [between(1, 512 if high > 4 else 9720) for _ in range(n)]
    if rng.random() < 0.3:
        kv[rng.randrange(n)] = 0
    return {"kind": kind, "q": text(q), "kv": text(kv), "heads": heads,
            "kv_heads": kv_heads, "dim": dim}


BLOCK = 64  # tokens that share a scale
SLOTS, SHIFT, SCALE, EPSILON = 6, 3, 4, 1e-5  # of the adaLN norms


def _numbers(text):
    return [int(v) for v in text.split(",")]


def _starts(counts):
    return [sum(counts[:i]) for i in range(len(counts))]


def _blocks(counts):
    return [(n + BLOCK - 1) // BLOCK for n in counts]


# ------------------------------------------------------------- the inputs

class _Make:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape, std=1.0):
        x = torch.randn(shape, generator=self.g, device="cuda")
        return x.mul_(std).to(torch.bfloat16)


def _inputs(case, seed):
    """The tensors a pass starts from, by name."""
    m = _Make(seed)
    if case["kind"] == "linear":
        k, n = case["in"], case["out"]
        return {"x": m.normal(case["rows"], k), "w": m.normal(n, k, std=0.02),
                "b": m.normal(n, std=0.02)}
    if case["kind"] == "mlp":
        k, h, n = case["in"], case["hidden"], case["out"]
        x = {"x": m.normal(case["rows"], k),
             "w1": m.normal(2 * h, k, std=0.02),
             "w2": m.normal(n, h, std=0.02)}
        if case["norm"] != "none":  # two time rows
            host = np.random.RandomState(seed % (1 << 31))
            x["nw"] = m.normal(k, std=0.1) + 1
            x["nb"] = m.normal(k, std=0.1)
            x["mod"] = m.normal(2, SLOTS, k, std=0.1)
            x["map"] = torch.from_numpy(
                host.randint(0, 2, case["rows"]).astype(np.int32)).cuda()
        return x
    g, d = case["kv_heads"], case["dim"]
    if case["kind"] == "store":
        # K and V side by side: the rows that the cache has, and the new ones
        return {"had": m.normal(max(1, sum(_numbers(case["has"]))),
                                2 * g * d),
                "kv": m.normal(sum(_numbers(case["new"])), 2 * g * d)}
    return {"q": m.normal(sum(_numbers(case["q"])), case["heads"] * d),
            "kv": m.normal(max(1, sum(_numbers(case["kv"]))), 2 * g * d)}


class _State:
    pass


def prepare(case, seed):
    """The activations, and what a program keeps: weights in 8 bits, the cache
    as it stands, the attention's plan."""
    s = _State()
    s.case = dict(case)
    if own:
        torch.cuda.synchronize()  # freed tensors may be handed out again
    s.x = _inputs(case, seed)
    if own:
        s.device = _Device(s.case, s.x)
        torch.cuda.synchronize()
        return s
    for name in ("w", "w1", "w2"):
        if name in s.x:
            s.x[name] = _codes(s.x[name].float())
    if case["kind"] == "store":
        has = _numbers(case["has"])
        s.new_at, starts = _places(case)
        s.x["cache"] = _into_blocks(case, s.x["had"], _rows_at(starts, has),
                                    starts[-1])
    if case["kind"] == "attend":
        kv = _numbers(case["kv"])
        starts = [BLOCK * b for b in _starts(_blocks(kv) + [0])]
        s.x["cache"] = _into_blocks(case, s.x["kv"], _rows_at(starts, kv),
                                    max(BLOCK, starts[-1]))
    return s


def _rows_at(starts, counts):
    """The cache rows of each request's tokens, in order."""
    return torch.cat([torch.arange(s, s + n) for s, n in zip(starts, counts)]
                     + [torch.arange(0)]).cuda()


def _places(case):
    """The cache rows that a store's new rows go to, and each request's first
    one, with the end behind them."""
    has, new = _numbers(case["has"]), _numbers(case["new"])
    both = [a + b for a, b in zip(has, new)]
    starts = [BLOCK * b for b in _starts(_blocks(both) + [0])]
    return _rows_at([s + a for s, a in zip(starts, has)], new), starts


def run(s):
    if own:
        return s.device.run()
    return {"linear": _linear, "mlp": _mlp, "store": _store,
            "attend": _attend}[s.case["kind"]](s)


# -------------------------------------------------------- the plain forms

def _codes(x):
    """Rows of x in 8 bits: codes, and a scale a row."""
    most = x.abs().amax(dim=1, keepdim=True)
    c = torch.round(x * 127 / torch.where(most == 0, 1.0, most))
    return c.to(torch.int8), most / 127


def _product(x, w):
    """Of rows in 8 bits, in F32."""
    return (x[0].float() @ w[0].float().T) * x[1] * w[1].T


def _linear(s):
    x = s.x
    y = _product(_codes(x["x"].float()), x["w"]) + x["b"].float()
    if s.case["gelu"]:
        y = 0.5 * y * (1 + torch.tanh(
            math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    return y.to(torch.bfloat16)


def _mlp(s):
    x, v = s.x, s.x["x"].float()
    if s.case["norm"] != "none":
        if s.case["norm"] == "layer":
            v = v - v.mean(dim=1, keepdim=True)
        v = v * torch.rsqrt((v * v).mean(dim=1, keepdim=True) + EPSILON) * \
            x["nw"].float()
        if s.case["norm"] == "layer":
            v = v + x["nb"].float()
        mod = x["mod"].float()[x["map"]]
        v = v * (1 + mod[:, SCALE]) + mod[:, SHIFT]
    g, u = _product(_codes(v), x["w1"]).chunk(2, dim=1)
    h = g / (1 + torch.exp(-g)) * u
    return _product(_codes(h), x["w2"]).to(torch.bfloat16)


def _as_blocks(case, rows, at, size):
    """Rows of K and V at their places in the blocks, F32, zeros elsewhere:
    [block][token][2][head][dim]."""
    full = torch.zeros(size, rows.shape[1], device="cuda")
    full[at] = rows.float()
    return full.reshape(-1, BLOCK, 2, case["kv_heads"], case["dim"])


def _into_blocks(case, rows, at, size):
    """A cache: codes as above, scales [block][1][2][head][1]."""
    full = _as_blocks(case, rows[:len(at)], at, size)
    most = full.abs().amax(dim=(1, 4), keepdim=True)
    c = torch.round(full * 127 / torch.where(most == 0, 1.0, most))
    return c.to(torch.int8), most / 127


def _store(s):
    """The values of the cache's rows; those behind a request's tokens are 0."""
    codes, scales = s.x["cache"]
    g, d = s.case["kv_heads"], s.case["dim"]
    size = codes.shape[0] * BLOCK
    full = _as_blocks(s.case, s.x["kv"], s.new_at, size)
    most = full.abs().amax(dim=(1, 4), keepdim=True)
    wide = torch.maximum(scales, most / 127)
    new = torch.zeros(size, dtype=torch.bool, device="cuda")
    new[s.new_at] = True
    # values next to a border: in 64 bits
    top = torch.where(wide > scales, most.double(), 127 * scales.double())
    unit = torch.where(top == 0, 1.0, top)
    kept = torch.round(codes.double() * torch.where(
        wide > scales, 127 * scales.double() / unit, 1.0))
    c = torch.where(new.reshape(-1, BLOCK, 1, 1, 1),
                    torch.round(127 * full.double() / unit), kept)
    kv = (c.float() * wide).to(torch.bfloat16).reshape(size, 2, g * d)
    return kv[:, 0].contiguous(), kv[:, 1].contiguous()


def _attend(s):
    """In F32: the requests' rows gathered into one padded batch."""
    case = s.case
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    q_rows, kv_rows = _numbers(case["q"]), _numbers(case["kv"])
    kv = (s.x["cache"][0].float() * s.x["cache"][1]).reshape(-1, 2, g * d)
    qf, qn, kf, kn = (torch.tensor(v, device="cuda") for v in (
        _starts(q_rows), q_rows,
        [BLOCK * b for b in _starts(_blocks(kv_rows))], kv_rows))
    n, most_q, most_k = len(q_rows), max(q_rows), max(1, max(kv_rows))
    q_pos = torch.arange(most_q, device="cuda")
    k_pos = torch.arange(most_k, device="cuda")
    q_live, k_live = q_pos < qn[:, None], k_pos < kn[:, None]
    q_at = torch.where(q_live, qf[:, None] + q_pos, 0)
    k_at = torch.where(k_live, kf[:, None] + k_pos, 0)
    # [request][key head][query row, head of the group][dim]
    qb = s.x["q"][q_at].float().reshape(n, most_q, g, h // g, d).permute(
        0, 2, 1, 3, 4).reshape(n, g, most_q * (h // g), d)
    kb = kv[:, 0][k_at].reshape(n, most_k, g, d).permute(0, 2, 3, 1)
    vb = (kv[:, 1][k_at] * k_live[:, :, None]).reshape(
        n, most_k, g, d).permute(0, 2, 1, 3)
    p = (qb @ kb.contiguous()) * (1 / math.sqrt(d))
    p.masked_fill_(~k_live[:, None, None, :], -math.inf)
    top = p.amax(dim=-1, keepdim=True)
    e = p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = e.sum(dim=-1, keepdim=True)
    o = (e @ vb.contiguous()) / torch.where(total == 0, 1.0, total)
    o = o.reshape(n, g, most_q, h // g, d).permute(0, 2, 1, 3, 4).reshape(
        n, most_q, h * d)
    return o[q_live].to(torch.bfloat16)  # in the order of the rows


# ---------------------------------------------------- the framework's calls

_gpu = None


def _context():
    """The process's one context, with a batch open as in a forward: launches
    queue up and nothing waits between them."""
    global _gpu
    if _gpu is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "h3.c_amd"))
        import h3hip
        torch.cuda.init()
        _gpu = h3hip.Gpu()
        _gpu.begin()
    return _gpu


class _Memory:
    """Device memory behind a tensor handle, as torch takes it.  The handle
    is freed with the last view of the memory."""

    def __init__(self, handle, shape, typestr, free):
        # a tensor handle starts with its device address
        self.handle, self.free = handle, free
        self.__cuda_array_interface__ = {
            "shape": tuple(shape), "typestr": typestr, "version": 2,
            "data": (ctypes.c_void_p.from_address(handle).value, False),
            "strides": None}

    def __del__(self):
        self.free(self.handle)


class _Tensor:
    """A backend tensor: .h is the handle that entry points take, .t the same
    memory as a torch tensor."""

    def __init__(self, gpu, shape, dtype, values=None):
        n = int(np.prod(shape))
        bf16 = dtype == torch.bfloat16
        h = gpu.L.h3_gpu_tensor_new_bf16(gpu.h, n) if bf16 else \
            gpu.L.h3_gpu_tensor_from_u32(gpu.h, None, n)
        gpu.check(h, "tensor")
        self.h = h
        self.t = torch.as_tensor(
            _Memory(h, shape, "<i2" if bf16 else "<i4",
                    gpu.L.h3_gpu_tensor_free), device="cuda")
        if bf16:
            self.t = self.t.view(torch.bfloat16)
        if values is not None:
            self.t.copy_(values)


class _Device:
    """What a program of the framework has in hand before the call: inputs and
    outputs as the framework's tensors, weights in 8 bits, the cache, the
    attention's plan."""

    def __init__(self, case, x):
        gpu = self.gpu = _context()
        self.case, self.made = case, []
        self.i = {name: _Tensor(gpu, v.shape, v.dtype, v)
                  for name, v in x.items()}
        torch.cuda.synchronize()
        getattr(self, "_keep_" + case["kind"])()
        self.run = getattr(self, "_run_" + case["kind"])

    def _int8(self, rows, columns):
        t = self.gpu.int8(rows, columns)
        self.made.append(t)
        return t

    def _weight(self, name, rows, columns):
        w = self._int8(rows, columns)
        self._call("h3_hip_quantize_int8", w, self.i[name].h, rows, columns)
        return w

    def _output(self, *shape):
        return _Tensor(self.gpu, shape, torch.bfloat16)

    def _call(self, name, *args):
        if not getattr(self.gpu.L, name)(self.gpu.h, *args):
            raise RuntimeError(self.gpu.error())

    def _keep_linear(self):
        case = self.case
        self.w = self._weight("w", case["out"], case["in"])
        self.q = self._int8(case["rows"], case["in"])
        self.y = self._output(case["rows"], case["out"])

    def _run_linear(self):
        case, i = self.case, self.i
        rows, k, n = case["rows"], case["in"], case["out"]
        self._call("h3_hip_quantize_int8", self.q, i["x"].h, rows, k)
        self._call("h3_hip_linear_gelu_int8_bf16" if case["gelu"] else
                   "h3_hip_linear_int8_bf16", self.y.h, self.q, self.w,
                   i["b"].h, rows, k, n)
        return self.y.t

    def _keep_mlp(self):
        case = self.case
        self.w1 = self._weight("w1", 2 * case["hidden"], case["in"])
        self.w2 = self._weight("w2", case["out"], case["hidden"])
        self.q = self._int8(case["rows"], case["in"])
        self.y = self._output(case["rows"], case["out"])

    def _run_mlp(self):
        case, i = self.case, self.i
        rows, k = case["rows"], case["in"]
        if case["norm"] == "none":
            self._call("h3_hip_quantize_int8", self.q, i["x"].h, rows, k)
        elif case["norm"] == "rms":
            self._call("h3_hip_adaln_int8", self.q, i["x"].h, i["nw"].h,
                       i["mod"].h, i["map"].h, rows, k, SLOTS, SHIFT, SCALE,
                       EPSILON)
        else:
            self._call("h3_hip_layer_adaln_int8", self.q, i["x"].h,
                       i["nw"].h, i["nb"].h, i["mod"].h, i["map"].h, rows, k,
                       SLOTS, SHIFT, SCALE, EPSILON)
        self._call("h3_hip_mlp_int8_bf16", self.y.h, self.q, self.w1, self.w2,
                   rows, k, case["hidden"], case["out"])
        return self.y.t

    def _cache(self, rows):
        t = self.gpu.kv_int8(rows, self.case["kv_heads"], self.case["dim"])
        self.made.append(t)
        return t

    def _ranges(self, *lists):
        """Host arrays of row numbers, as the store takes them."""
        return [(ctypes.c_uint32 * len(v))(*v) for v in lists]

    def _store(self, rows, ranges, count):
        width = self.case["kv_heads"] * self.case["dim"]
        self._call("h3_hip_kv_int8_store", self.cache, *ranges, count, rows.h,
                   0, rows.h, width, 2 * width)

    def _keep_store(self):
        case = self.case
        has, new = _numbers(case["has"]), _numbers(case["new"])
        _, starts = _places(case)
        self.rows = starts[-1]
        self.cache = self._cache(self.rows)
        # the cache as it stands, then where the new rows go
        self._store(self.i["had"], self._ranges(starts[:-1], _starts(has),
                                                has), len(has))
        self.ranges = self._ranges([s + n for s, n in zip(starts, has)],
                                   _starts(new), new)
        width = case["kv_heads"] * case["dim"]
        self.k = self._output(self.rows, width)
        self.v = self._output(self.rows, width)

    def _run_store(self):
        self._store(self.i["kv"], self.ranges, len(self.ranges[0]))
        self._call("h3_hip_kv_int8_read", self.k.h, self.v.h, self.cache, 0,
                   self.rows)
        return self.k.t, self.v.t

    def _keep_attend(self):
        case = self.case
        q, kv = _numbers(case["q"]), _numbers(case["kv"])
        starts = [BLOCK * b for b in _starts(_blocks(kv) + [0])]
        self.cache = self._cache(max(BLOCK, starts[-1]))
        self._store(self.i["kv"], self._ranges(starts[:-1], _starts(kv), kv),
                    len(kv))
        self.plan = self.gpu.sdpa_packed_plan(
            _starts(q), q, starts[:-1], kv, case["heads"], case["kv_heads"],
            case["dim"])
        self.made.append(self.plan)
        self.y = self._output(sum(q), case["heads"] * case["dim"])

    def _run_attend(self):
        case = self.case
        self._call("h3_hip_sdpa_packed_int8_bf16", self.y.h, self.i["q"].h, 0,
                   case["heads"] * case["dim"], self.cache, self.plan,
                   1 / math.sqrt(case["dim"]))
        return self.y.t

    def __del__(self):
        for t in self.made:
            self.gpu.free(t)


# ------------------------------------------------------ what a pass costs

def work(case):
    if case["kind"] == "linear":
        m, k, n = case["rows"], case["in"], case["out"]
        return {"bytes": 2 * m * k + n * k + 6 * n + 2 * m * n,
                "flops": 2 * m * n * k}
    if case["kind"] == "mlp":
        m, k, h, n = case["rows"], case["in"], case["hidden"], case["out"]
        norm = 0 if case["norm"] == "none" else 2 * k * (2 + 2 * 2) + 4 * m
        return {"bytes": 2 * m * k + 2 * h * (k + 4) + n * (h + 4) +
                2 * m * n + norm, "flops": 2 * m * h * (2 * k + n)}
    g, d = case["kv_heads"], case["dim"]
    if case["kind"] == "store":
        # new rows in, their codes out, begun blocks both ways, and all values
        # that the cache then holds, out
        has, new = _numbers(case["has"]), _numbers(case["new"])
        rows = BLOCK * sum(_blocks([a + b for a, b in zip(has, new)]))
        begun = sum(a % BLOCK for a in has)
        return {"bytes": 2 * g * d * (3 * sum(new) + 2 * begun + 2 * rows),
                "flops": 4 * g * d * rows}
    q, kv, h = _numbers(case["q"]), _numbers(case["kv"]), case["heads"]
    return {"bytes": 4 * d * h * sum(q) + 2 * g * (d * sum(kv) +
                                                   4 * sum(_blocks(kv))),
            "flops": 4 * d * h * sum(a * b for a, b in zip(q, kv))}


# -------------------------------------------------- the same in 64 bits

def _exact_rows(x):
    x = x.double()
    top = x.abs().max(dim=1).values.clamp_min(1e-300).unsqueeze(1)
    return (127 * x / top).round_(), top / 127


def _exact_cache(case, kv, has, new):
    """Each request's K and V, [whole blocks][2][heads][dim], as its blocks
    hold them after the tokens that it has and then the new ones."""
    def largest(rows):
        if not len(rows):
            return torch.zeros_like(out[0, :, :, :1])
        return rows.abs().amax(dim=3).amax(dim=0).unsqueeze(-1)

    def step(rows, top):
        return (127 * rows / top.clamp_min(1e-300)).round()

    kept, fresh = kv
    for i, (a, b) in enumerate(zip(has, new)):
        shape = (-1, 2, case["kv_heads"], case["dim"])
        old = kept[sum(has[:i]):sum(has[:i + 1])].double().reshape(shape)
        more = fresh[sum(new[:i]):sum(new[:i + 1])].double().reshape(shape)
        out = torch.zeros(BLOCK * _blocks([a + b])[0], 2, case["kv_heads"],
                          case["dim"], dtype=torch.float64, device="cuda")
        for first in range(0, a + b, BLOCK):
            o = old[first:first + BLOCK]
            m = more[max(0, first - a):max(0, first + BLOCK - a)]
            before = largest(o)
            top = torch.maximum(before, largest(m))
            c = torch.cat([
                (step(o, before) * (before / top.clamp_min(1e-300))).round(),
                step(m, top)])
            out[first:first + len(c)] = c * top / 127
        yield out, a + b


def exact(case, seed):
    x = _inputs(case, seed)
    if case["kind"] == "linear":
        c, s = _exact_rows(x["x"])
        w, t = _exact_rows(x["w"])
        y = torch.mm(c, w.t()).mul_(s).mul_(t.t()).add_(x["b"].double())
        if case["gelu"]:
            return torch.nn.functional.gelu(y, approximate="tanh")
        return y
    if case["kind"] == "mlp":
        v = x["x"].double()
        if case["norm"] != "none":
            k = case["in"]
            if case["norm"] == "layer":
                v = torch.nn.functional.layer_norm(
                    v, (k,), x["nw"].double(), x["nb"].double(), EPSILON)
            else:
                v = v / (v.square().mean(dim=1, keepdim=True) +
                         EPSILON).sqrt() * x["nw"].double()
            rows = x["map"].long()
            v = v + v * x["mod"][:, SCALE].double()[rows] + \
                x["mod"][:, SHIFT].double()[rows]
        c, s = _exact_rows(v)
        w, t = _exact_rows(x["w1"])
        gu = torch.mm(c, w.t()).mul_(s).mul_(t.t())
        h = case["hidden"]
        c, s = _exact_rows(torch.nn.functional.silu(gu[:, :h]) * gu[:, h:])
        w, t = _exact_rows(x["w2"])
        return torch.mm(c, w.t()).mul_(s).mul_(t.t())
    g, d = case["kv_heads"], case["dim"]
    if case["kind"] == "store":
        rows = torch.cat([out for out, _ in _exact_cache(
            case, (x["had"], x["kv"]), _numbers(case["has"]),
            _numbers(case["new"]))])
        return (rows[:, 0].reshape(-1, g * d).contiguous(),
                rows[:, 1].reshape(-1, g * d).contiguous())
    h, q, kv = case["heads"], _numbers(case["q"]), _numbers(case["kv"])
    out = torch.zeros(sum(q), h, d, dtype=torch.float64, device="cuda")
    caches = _exact_cache(case, (x["kv"][:0], x["kv"]), [0] * len(kv), kv)
    for first, n, (rows, tokens) in zip(_starts(q), q, caches):
        rows = rows[:tokens]
        if not tokens:
            continue
        for head in range(h):
            k, v = rows[:, 0, head // (h // g)], rows[:, 1, head // (h // g)]
            p = torch.softmax(torch.mm(
                x["q"][first:first + n, head * d:(head + 1) * d].double(),
                k.t()) / math.sqrt(d), dim=1)
            out[first:first + n, head] = torch.mm(p, v)
    return out.reshape(-1, h * d)
