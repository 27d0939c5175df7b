"""The operators of a forward that serves several requests at once, packed into
one sequence of rows: projections with each request's own low-rank adapter, and
attention of each request's rows to its own keys.

Adapters (kind "adapters"):
    y[r] = act(x[r] W^T + b + s_a (x[r] A_a^T) B_a^T),  a = map[r]
with no adapter where the map names none; act is nothing or the tanh form of
GELU.  Attention (kind "packed"): the query rows of request i attend to its own
key rows, in `heads` heads that share `kv_heads` key heads; a request without
keys gets zeros.

Widths are the repository's two model families' (hidden 5376 with 56 heads of
128 and 5120 with 40 heads of 128, FFN 13824, time features 2688) or generic
ones; rows are those of their clips (778, 1536, 2378, 6144 rows), prompts of up
to 512 tokens, and single rows.

Inputs are N(0, 1) activations and 0.02 N(0, 1) weights, as in the repository's
benchmark; adapter scales lie between 0.5 and 2.
"""
import ctypes
import math
import os
import sys

import torch
import numpy as np

own = False


def listed():
    one = ",".join(["1"] * 8)
    return [
        # one row of each of eight requests (a pooled or time embedding), each
        # with its own adapter: the smallest call, bound by the weight
        {"name": "adapters_rows_8", "kind": "adapters", "rows": one,
         "use": "0,1,2,3,4,5,6,7", "ranks": ",".join(["16"] * 8),
         "in": 5120, "out": 5120, "gelu": False, "mixed": False},
        # the adaLN projection of three requests' time rows
        {"name": "adapters_modulation_39", "kind": "adapters",
         "rows": "13,13,13", "use": "0,-,1", "ranks": "16,16", "in": 2688,
         "out": 96768, "gelu": False, "mixed": False},
        # the condition projection of two prompts, ranks that differ
        {"name": "adapters_text_197", "kind": "adapters", "rows": "120,77",
         "use": "0,1", "ranks": "32,8", "in": 5120, "out": 5376,
         "gelu": False, "mixed": False},
        # the attention output projection of one 256x256 clip
        {"name": "adapters_out_778", "kind": "adapters", "rows": "778",
         "use": "0", "ranks": "16", "in": 7168, "out": 5376, "gelu": False,
         "mixed": False},
        # the QKV projection of two 512x512 clips
        {"name": "adapters_qkv_4756", "kind": "adapters", "rows": "2378,2378",
         "use": "0,1", "ranks": "64,4", "in": 5376, "out": 21504,
         "gelu": False, "mixed": False},
        # the FFN's first projection of four clips, one without an adapter,
        # one of an odd rank
        {"name": "adapters_ffn_6144", "kind": "adapters",
         "rows": "1536,1536,1536,1536", "use": "0,1,-,2",
         "ranks": "128,16,33", "in": 5120, "out": 13824, "gelu": True,
         "mixed": False},
        # one row of each of 16 requests against its prompt
        {"name": "packed_rows_16", "kind": "packed",
         "q": ",".join(["1"] * 16),
         "kv": "20,33,512,77,126,1,300,64,65,63,200,411,90,18,256,150",
         "heads": 40, "kv_heads": 40, "dim": 128, "self": False},
        # one row of each of 8 requests against long contexts, shared heads:
        # bound by reading the keys and values
        {"name": "packed_rows_8_long", "kind": "packed",
         "q": ",".join(["1"] * 8),
         "kv": "9720,6144,8191,4096,5000,9001,7777,6145", "heads": 64,
         "kv_heads": 8, "dim": 128, "self": False},
        # two clips of unlike size, a full prompt and a short one
        {"name": "packed_cross_pair", "kind": "packed",
         "q": "1536,778", "kv": "512,126", "heads": 40, "kv_heads": 40,
         "dim": 128, "self": False},
        # four 512x512 clips against their prompts, one of them empty
        {"name": "packed_cross_4", "kind": "packed",
         "q": "6144,6144,6144,6144", "kv": "512,77,300,0", "heads": 40,
         "kv_heads": 40, "dim": 128, "self": False},
        # self-attention of three packed clips
        {"name": "packed_self_3", "kind": "packed", "q": "778,1536,2378",
         "kv": "778,1536,2378", "heads": 56, "kv_heads": 56, "dim": 128,
         "self": True},
        # the same of five ragged sequences with shared heads of 64
        {"name": "packed_self_shared_64", "kind": "packed",
         "q": "1000,33,517,1,2048", "kv": "1000,33,517,1,2048", "heads": 32,
         "kv_heads": 8, "dim": 64, "self": True},
    ]


def draw(rng):
    def between(low, high):
        return int(round(math.exp(rng.uniform(math.log(low),
                                              math.log(high)))))

    def text(values):
        return ",".join(str(v) for v in values)

    n = rng.choice([1, 2, 3, 4, 7, 8, 16])
    if rng.random() < 0.5:
        # widths of the two models' projections, and generic ones
        k, out = rng.choice([(5120, 5120), (5120, 13824), (5376, 21504),
                             (7168, 5376), (2688, 10752), (512, 1536),
                             (1280, 3420), (320, 5120)])
        # at most the flops of the largest projection listed
        most = min(6144, 4756 * 5376 * 21504 // (k * out))
        rows = [between(1, most) // n + 1 for _ in range(n)]
        count = rng.randint(1, n)
        ranks = [rng.choice([4, 8, 16, 16, 32, 64, 128, rng.randint(1, 100)])
                 for _ in range(count)]
        use = [rng.choice(list(range(count)) * 3 + ["-"]) for _ in range(n)]
        return {"kind": "adapters", "rows": text(rows), "use": text(use),
                "ranks": text(ranks), "in": k, "out": out,
                "gelu": rng.random() < 0.3,
                "mixed": sum(rows) < 600 and rng.random() < 0.3}
    heads, kv_heads, dim = rng.choice(
        [(40, 40, 128), (56, 56, 128), (64, 8, 128), (32, 8, 64), (16, 2, 128),
         (12, 12, 64), (24, 4, 96), (10, 5, 80)])
    if rng.random() < 0.4:
        q = [between(1, 4000) // n + 1 for _ in range(n)]
        return {"kind": "packed", "q": text(q), "kv": text(q), "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "self": True}
    high = rng.choice([1, 4, 6144])  # single rows, a few, whole clips
    q = [between(1, min(high, 24576 // n)) for _ in range(n)]
    kv = [between(1, 512 if high > 4 else 9720) for _ in range(n)]
    if rng.random() < 0.3:
        kv[rng.randrange(n)] = 0
    return {"kind": "packed", "q": text(q), "kv": text(kv), "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "self": False}


def _numbers(text):
    return [None if v == "-" else int(v) for v in text.split(",")]


# ------------------------------------------------------------- the inputs

NO_ADAPTER = 0xFFFFFFFF


class _Make:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape, std=1.0):
        x = torch.randn(shape, generator=self.g, device="cuda")
        return x.mul_(std).to(torch.bfloat16)


def _row_starts(counts):
    return [sum(counts[:i]) for i in range(len(counts))]


def _inputs(case, seed):
    """The tensors a call reads, by name, and its host-side numbers."""
    m = _Make(seed)
    if case["kind"] == "adapters":
        rows, use = _numbers(case["rows"]), _numbers(case["use"])
        ranks, k, n = _numbers(case["ranks"]), case["in"], case["out"]
        ids = np.repeat(np.array([NO_ADAPTER if u is None else u
                                  for u in use], np.uint32), rows)
        host = np.random.RandomState(seed % (1 << 31))
        if case["mixed"]:  # rows of the requests in any order
            host.shuffle(ids)
        x = {"x": m.normal(len(ids), k), "w": m.normal(n, k, std=0.02),
             "b": m.normal(n, std=0.02),
             "map": torch.from_numpy(ids.view(np.int32)).cuda()}
        for a, r in enumerate(ranks):
            x[f"down.{a}"] = m.normal(r, k, std=0.02)
            x[f"up.{a}"] = m.normal(n, r, std=0.02)
        return x, {"ranks": ranks, "scales": [
            float(np.float32(s)) for s in host.uniform(0.5, 2, len(ranks))]}
    q, kv = _numbers(case["q"]), _numbers(case["kv"])
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    numbers = {"q_first": _row_starts(q), "q_rows": q,
               "kv_first": _row_starts(kv), "kv_rows": kv}
    if case["self"]:  # rows of a fused projection: queries, keys, values
        return {"qkv": m.normal(sum(q), (h + 2 * g) * d)}, numbers
    # keys and values of a fused projection of the text
    return {"q": m.normal(sum(q), h * d),
            "kv": m.normal(max(1, sum(kv)), 2 * g * d)}, numbers


class _State:
    pass


def prepare(case, seed):
    s = _State()
    s.case = dict(case)
    if own:
        torch.cuda.synchronize()  # freed tensors may be handed out again
    s.x, s.numbers = _inputs(case, seed)
    if own:
        s.device = _Device(s.case, s.x, s.numbers)
        torch.cuda.synchronize()
    return s


def run(s):
    if own:
        return s.device.run()
    if s.case["kind"] == "adapters":
        return _adapters(s.case, s.x, s.numbers)
    return _packed(s.case, s.x, s.numbers)


# -------------------------------------------------------- the plain forms

def _adapters(case, x, numbers):
    """In F32: the shared product, the products with all adapters' rows side
    by side, those of other adapters than the row's own masked out."""
    y = x["x"].float() @ x["w"].float().T + x["b"].float()
    count = len(numbers["ranks"])
    ranks = torch.tensor(numbers["ranks"], device="cuda")
    down = torch.cat([x[f"down.{a}"] for a in range(count)]).float()
    up = torch.cat([x[f"up.{a}"] for a in range(count)], dim=1).float()
    owner = torch.repeat_interleave(torch.arange(count, device="cuda"), ranks)
    scale = torch.tensor(numbers["scales"], device="cuda")[owner]
    u = x["x"].float() @ down.T * scale
    u = u * (owner[None, :] == x["map"][:, None])
    y = y + u @ up.T
    if case["gelu"]:
        y = 0.5 * y * (1 + torch.tanh(
            math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    return y.to(torch.bfloat16)


def _packed(case, x, numbers):
    """In F32: the requests' rows gathered into one padded batch."""
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    if case["self"]:
        q, k, v = torch.split(x["qkv"], [h * d, g * d, g * d], dim=1)
    else:
        q, (k, v) = x["q"], torch.split(x["kv"], [g * d, g * d], dim=1)
    qf, qn, kf, kn = (torch.tensor(numbers[name], device="cuda") for name in
                      ("q_first", "q_rows", "kv_first", "kv_rows"))
    n, most_q, most_k = len(qn), max(numbers["q_rows"]), \
        max(1, max(numbers["kv_rows"]))
    q_pos = torch.arange(most_q, device="cuda")
    k_pos = torch.arange(most_k, device="cuda")
    q_live, k_live = q_pos < qn[:, None], k_pos < kn[:, None]
    q_at = torch.where(q_live, qf[:, None] + q_pos, 0)
    k_at = torch.where(k_live, kf[:, None] + k_pos, 0)
    # [request][key head][query row, head of the group][dim]
    qb = q[q_at].float().reshape(n, most_q, g, h // g, d).permute(
        0, 2, 1, 3, 4).reshape(n, g, most_q * (h // g), d)
    kb = k[k_at].float().reshape(n, most_k, g, d).permute(0, 2, 3, 1)
    vb = (v[k_at].float() * k_live[:, :, None]).reshape(
        n, most_k, g, d).permute(0, 2, 1, 3)
    s = (qb @ kb.contiguous()) * (1 / math.sqrt(d))
    s.masked_fill_(~k_live[:, None, None, :], -math.inf)
    top = s.amax(dim=-1, keepdim=True)
    e = s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
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
    """What a program of the framework has in hand before the call: the
    inputs and the output as the framework's tensors, and the adapters' table
    or the attention's plan."""

    def __init__(self, case, x, numbers):
        gpu = self.gpu = _context()
        self.case = case
        self.i = {name: _Tensor(gpu, v.shape, v.dtype, v)
                  for name, v in x.items()}
        torch.cuda.synchronize()  # the table copies the adapters
        if case["kind"] == "adapters":
            self.rows = len(x["map"])
            self.y = _Tensor(gpu, (self.rows, case["out"]), torch.bfloat16)
            count = len(numbers["ranks"])
            self.made = gpu.lora_table(
                [self.i[f"down.{a}"].h for a in range(count)],
                [self.i[f"up.{a}"].h for a in range(count)],
                numbers["ranks"], numbers["scales"], case["in"], case["out"])
        else:
            d = case["dim"]
            self.rows = sum(numbers["q_rows"])
            self.y = _Tensor(gpu, (self.rows, case["heads"] * d),
                             torch.bfloat16)
            self.made = gpu.sdpa_packed_plan(
                numbers["q_first"], numbers["q_rows"], numbers["kv_first"],
                numbers["kv_rows"], case["heads"], case["kv_heads"], d)

    def run(self):
        case, gpu, L, i = self.case, self.gpu, self.gpu.L, self.i
        if case["kind"] == "adapters":
            call = L.h3_hip_linear_lora_gelu_bf16 if case["gelu"] else \
                L.h3_hip_linear_lora_bf16
            ok = call(gpu.h, self.y.h, i["x"].h, i["w"].h, i["b"].h,
                      self.made, i["map"].h, self.rows, case["in"],
                      case["out"])
        else:
            q, k, d = case["heads"] * case["dim"], \
                case["kv_heads"] * case["dim"], case["dim"]
            if case["self"]:
                t, stride = i["qkv"].h, q + 2 * k
                ok = L.h3_hip_sdpa_packed_bf16(
                    gpu.h, self.y.h, t, 0, stride, t, q, t, q + k, stride,
                    self.made, 1 / math.sqrt(d))
            else:
                t = i["kv"].h
                ok = L.h3_hip_sdpa_packed_bf16(
                    gpu.h, self.y.h, i["q"].h, 0, q, t, 0, t, k, 2 * k,
                    self.made, 1 / math.sqrt(d))
        if not ok:
            raise RuntimeError(gpu.error())
        return self.y.t

    def __del__(self):
        self.gpu.free(self.made)


# ------------------------------------------------------ what a pass costs

def work(case):
    if case["kind"] == "adapters":
        rows, use = _numbers(case["rows"]), _numbers(case["use"])
        ranks, k, n = _numbers(case["ranks"]), case["in"], case["out"]
        m = sum(rows)
        used = sum(ranks[a] for a in {u for u in use if u is not None})
        low = sum(r * ranks[u] for r, u in zip(rows, use) if u is not None)
        return {"bytes": 2 * (m * k + n * k + n + m * n + used * (k + n)) +
                4 * m, "flops": 2 * m * n * k + 2 * low * (k + n)}
    q, kv = _numbers(case["q"]), _numbers(case["kv"])
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    return {"bytes": 2 * d * (2 * h * sum(q) + 2 * g * sum(kv)),
            "flops": 4 * d * h * sum(a * b for a, b in zip(q, kv))}


# -------------------------------------------------- the same in 64 bits

def exact(case, seed):
    x, numbers = _inputs(case, seed)
    if case["kind"] == "adapters":
        wide = {name: v.double() for name, v in x.items() if name != "map"}
        y = torch.addmm(wide["b"], wide["x"], wide["w"].t())
        for a, scale in enumerate(numbers["scales"]):
            at = torch.nonzero(x["map"] == a).reshape(-1)
            rows = wide["x"].index_select(0, at)
            low = torch.mm(rows, wide[f"down.{a}"].t()).mul_(scale)
            y.index_add_(0, at, torch.mm(low, wide[f"up.{a}"].t()))
        if case["gelu"]:
            return torch.nn.functional.gelu(y, approximate="tanh")
        return y
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros(sum(numbers["q_rows"]), h, d, dtype=torch.float64,
                      device="cuda")
    for qf, qn, kf, kn in zip(*(numbers[name] for name in (
            "q_first", "q_rows", "kv_first", "kv_rows"))):
        if not kn:
            continue
        for head in range(h):
            at, kv_at = head * d, head // (h // g) * d
            if case["self"]:
                rows = x["qkv"][qf:qf + qn].double()
                q = rows[:, at:at + d]
                k = rows[:, h * d + kv_at:h * d + kv_at + d]
                v = rows[:, (h + g) * d + kv_at:(h + g) * d + kv_at + d]
            else:
                q = x["q"][qf:qf + qn, at:at + d].double()
                kv = x["kv"][kf:kf + kn].double()
                k, v = kv[:, kv_at:kv_at + d], \
                    kv[:, g * d + kv_at:g * d + kv_at + d]
            p = torch.softmax(torch.mm(q, k.t()) / math.sqrt(d), dim=1)
            out[qf:qf + qn, head] = torch.mm(p, v)
    return out.reshape(-1, h * d)
