"""Microscaled 4-bit (MXFP4) rows, products and expert products: what is measured of them, in plain form and through the backend.

A block of 32 values is a byte e and 16 bytes of codes (value j in the low nibble of byte j, value 16 + j in the high nibble): E2M1(code) 2^(e - 127), e = 255 for NaN.

  store    SET_ROWS of f32 rows into an MXFP4 table, then GET_ROWS of the whole table in another order
  convert  CPY of a dense f32 matrix into MXFP4 and back: the quantisation and the reading of whole matrices
  read     GET_ROWS of an MXFP4 matrix: token embeddings
  product  MUL_MAT by an MXFP4 matrix, from one column (a decode step) to a prompt's
  experts  MUL_MAT_ID by the matrices of MXFP4 experts, and ADD_ID of the experts' bias rows: a decode step, a few tokens, a prompt

A product takes its activations as whole numbers q of -255 .. 255 times a power of two, a block of 32 each (q = rint(x 2^-s), s the exponent of the block's largest magnitude rounded to 8
significant bits, less 7, within -120 .. 120): the counterpart of the 8-bit activation blocks that the products by the other block formats use.
"""
import ctypes as C
import math

import numpy as np
import torch

own = False  # True: the framework's operators; False: the plain form of the same

VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
STEPS = 120  # exponents of an activation block's step: -STEPS .. STEPS


def _rows(name, kind, width, rows, taken):
    return {"name": name, "kind": kind, "width": width, "rows": rows, "taken": taken}


def _product(name, width, out, cols):
    return {"name": name, "kind": "product", "width": width, "out": out, "cols": cols}


def _experts(name, width, out, experts, used, tokens, shared):
    return {"name": name, "kind": "experts", "width": width, "out": out, "experts": experts, "used": used, "tokens": tokens, "shared": shared}


def listed():
    return [
        _rows("store 3 rows", "store", 1056, 129, 3),                           # a few rows into a small table: latency
        _rows("convert matrix", "convert", 4096, 14336, 14336),                 # a feed-forward matrix quantised when a model is made, and expanded again
        _rows("read embeddings", "read", 4096, 32000, 512),                     # a micro-batch's token embeddings
        _product("one column", 4096, 4096, 1),                                  # decode: an attention projection
        _product("one long column", 14336, 4096, 1),                            # decode: a down projection
        _product("odd columns", 2080, 1001, 5),                                 # a few drafts, rows and widths that fill no tile
        _product("batch 32", 4096, 14336, 32),                                  # continuous batching with all slots busy
        _product("prompt 512", 4096, 14336, 512),                               # the engine's micro-batch
        _product("prompt 1900", 4096, 14336, 1900),                             # a long prompt in one batch
        _experts("experts decode", 2048, 4096, 32, 4, 1, True),                 # one user's token: four experts' gate or up rows
        _experts("experts few tokens", 1056, 333, 5, 3, 7, False),              # a down projection of a few tokens, odd sizes
        _experts("experts prompt", 2048, 4096, 32, 4, 1000, True),              # a prompt: ragged groups over all experts
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def width(lo, hi):
        return 32 * max(1, log_int(lo, hi) // 32)

    kind = rng.choice(["store", "convert", "read"] + ["product"] * 4 + ["experts"] * 4)
    if kind in ("store", "read"):
        rows = log_int(16, 20000)
        c = _rows("", kind, width(32, 8192), rows, min(rows, log_int(1, 2000)))
    elif kind == "convert":
        rows = log_int(1, 10000)
        c = _rows("", kind, width(32, 4096), rows, rows)
    elif kind == "product":
        cols = rng.choice([1, log_int(2, 40), log_int(33, 1800)])
        c = _product("", width(64, 14336 if cols < 33 else 4096), log_int(32, 14336), cols)
    else:
        tokens = rng.choice([1, log_int(2, 60), log_int(33, 900)])
        n = log_int(2, 32)
        c = _experts("", width(64, 2048), log_int(32, 4096), n, rng.randint(1, min(4, n)), tokens, rng.random() < 0.5)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------ the plain form
def _quantise(x):
    """f32 [..., K] -> packed blocks, uint8 [..., K / 32 * 17]"""
    b = x.unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    good = torch.isfinite(top)
    e = torch.frexp(torch.where(good, top, torch.ones_like(top)))[1] - 1 - 2 + 127
    e = torch.where(top > 0, e, torch.zeros_like(e)).clamp(min=0)
    m = torch.ldexp(torch.ldexp(b.abs(), (64 - e // 2).unsqueeze(-1)), (63 - (e - e // 2)).unsqueeze(-1))  # (2^(127 - e), in two steps that 32 bits hold)
    code = torch.zeros_like(m, dtype=torch.uint8)
    for border in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0):
        code += m > border
    code = torch.where((b < 0) & (code > 0), code + 8, code)
    code = torch.where(good.unsqueeze(-1), code, torch.zeros_like(code))
    e = torch.where(good, e, torch.full_like(e, 255)).to(torch.uint8)
    return torch.cat([e.unsqueeze(-1), code[..., :16] | (code[..., 16:] << 4)], -1).flatten(-2)


def _values(p):
    """packed blocks, uint8 [..., K / 32 * 17] -> f32 [..., K]"""
    b = p.unflatten(-1, (-1, 17))
    e, q = b[..., :1].int(), b[..., 1:]
    code = torch.cat([q & 15, q >> 4], -1)
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), device=p.device)
    scale = torch.where(e == 255, torch.full_like(e, 1, dtype=torch.float32) * math.nan, torch.ldexp(torch.ones_like(e, dtype=torch.float32), e - 127))
    return (table[code.int()] * scale).flatten(-2)


def _activations(x):
    """f32 [..., K] -> the values that a product takes for them"""
    b = x.unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    good = torch.isfinite(top)
    frac, e = torch.frexp(torch.where(good, top, torch.ones_like(top)))
    step = (e + (frac >= 255.5 / 256) - 8).clamp(-STEPS, STEPS)
    q = torch.round(torch.ldexp(b, -step)).clamp(-255, 255)
    return torch.where(good, torch.ldexp(q, step), torch.full_like(q, math.nan)).flatten(-2)


def _plain_experts(s):
    c = s["case"]
    ids, x = s["ids"], _activations(s["x"])  # ids [T, U], x [T, 1 or U, K]
    T, U = ids.shape
    if T * U <= c["experts"]:  # a few columns: each with its expert's matrix
        w = _values(s["w"][ids.flatten().long()])
        y = torch.bmm(w, x.expand(T, U, -1).reshape(T * U, -1, 1)).view(T, U, -1)
    else:  # columns sorted by expert, every expert's padded to the longest group
        flat = ids.flatten().long()
        count = torch.bincount(flat, minlength=c["experts"])
        order = torch.argsort(flat, stable=True)
        place = torch.arange(T * U, device=flat.device) - (torch.cumsum(count, 0) - count)[flat[order]]
        groups = torch.zeros((c["experts"], int(count.max()), x.shape[-1]), device=x.device)
        groups[flat[order], place] = x.expand(T, U, -1).reshape(T * U, -1)[order]
        g = torch.bmm(groups, _values(s["w"]).transpose(1, 2).contiguous())
        y = torch.empty((T * U, g.shape[-1]), device=x.device)
        y[order] = g[flat[order], place]
        y = y.view(T, U, -1)
    return y + s["bias"][ids.long()]


def _plain(s):
    kind = s["case"]["kind"]
    if kind == "store":
        s["table"][s["slots"]] = _quantise(s["x"])
        return _values(s["table"][s["order"].long()])
    if kind == "convert":
        return _values(_quantise(s["x"]))
    if kind == "read":
        return _values(s["table"][s["order"].long()])
    if kind == "product":
        return torch.matmul(_activations(s["x"]), _values(s["w"]).t())
    return _plain_experts(s)


# ------------------------------------------------------------------------------------------ the framework's operators
class _Event(C.Structure):
    """struct ggml_backend_event (include/ggml_abi.h) around an event of torch's: its context is the hipEvent_t"""

    _fields_ = [("device", C.c_void_p), ("context", C.c_void_p)]

    def __init__(self, device):
        self.torch = torch.cuda.Event()
        self.torch.record()  # (its first record makes it)
        super().__init__(device, self.torch.cuda_event)


class _Graph:
    """The graph of one case, as an engine keeps it. Its tensors lie where the state's lie: every call takes their addresses anew and reads and writes them there."""

    backend = None  # one for the process, as an engine has, with the two events that order its stream and torch's

    def __init__(self, s):
        import llama_box_amd as L

        self.H = H = L.host()
        if _Graph.backend is None:
            _Graph.backend = L.Backend(0)
            _Graph.begun, _Graph.done = _Event(_Graph.backend.dev), _Event(_Graph.backend.dev)
            for f in (H.ggml_backend_event_wait, H.ggml_backend_event_record):
                f.restype, f.argtypes = None, [C.c_void_p, C.c_void_p]
        self.ctx = ctx = H.ggml_init(L.InitParams(0, None, True))
        self.theirs, self.room = [], []  # (tensor, the state's name for it); memory between two operators

        def of_state(t, key):
            self.theirs.append((t.contents, key))
            return t

        def leaf(kind, ne, key):
            return of_state(H.ggml_new_tensor_4d(ctx, kind, *(list(ne) + [1] * (4 - len(ne)))), key)

        def between(t):
            self.room.append(torch.empty(H.ggml_nbytes(t), dtype=torch.uint8, device="cuda"))
            t.contents.data = self.room[-1].data_ptr()
            return t

        c = s["case"]
        k, K = c["kind"], c["width"]
        if k == "store":
            n = s["order"].numel()
            stored = of_state(H.ggml_set_rows(ctx, leaf(L.MXFP4, (K, c["rows"]), "table"), leaf(L.F32, (K, c["taken"]), "x"), leaf(L.I64, (c["taken"],), "slots")), "table")
            out, shape = H.ggml_get_rows(ctx, stored, leaf(L.I32, (n,), "order")), (n, K)
        elif k == "convert":
            out, shape = H.ggml_cast(ctx, between(H.ggml_cast(ctx, leaf(L.F32, (K, c["rows"]), "x"), L.MXFP4)), L.F32), (c["rows"], K)
        elif k == "read":
            n = s["order"].numel()
            out, shape = H.ggml_get_rows(ctx, leaf(L.MXFP4, (K, c["rows"]), "table"), leaf(L.I32, (n,), "order")), (n, K)
        elif k == "product":
            out, shape = H.ggml_mul_mat(ctx, leaf(L.MXFP4, (K, c["out"]), "w"), leaf(L.F32, (K, c["cols"]), "x")), (c["cols"], c["out"])
        else:
            T, U, N = c["tokens"], c["used"], c["out"]
            ids = leaf(L.I32, (U, T), "ids")
            y = between(H.ggml_mul_mat_id(ctx, leaf(L.MXFP4, (K, N, c["experts"]), "w"), leaf(L.F32, (K, 1 if c["shared"] else U, T), "x"), ids))
            out, shape = H.ggml_add_id(ctx, y, leaf(L.F32, (N, c["experts"]), "bias"), ids), (T, U, N)
        H.ggml_set_output(out)
        self.graph = H.ggml_new_graph(ctx)
        H.ggml_build_forward_expand(self.graph, out)
        self.out = torch.empty(shape, device="cuda")
        out.contents.data = self.out.data_ptr()

    def __del__(self):
        self.H.ggml_free(self.ctx)

    def __call__(self, s):
        for t, key in self.theirs:
            t.data = s[key].data_ptr()
        # the backend's stream behind what torch's stream holds (the last reader of the output, too), torch's behind the graph
        H, backend, begun, done = self.H, _Graph.backend.backend, _Graph.begun, _Graph.done
        stream = torch.cuda.current_stream()
        begun.torch.record(stream)
        H.ggml_backend_event_wait(backend, C.addressof(begun))
        if H.ggml_backend_graph_compute_async(backend, self.graph) != 0:
            raise RuntimeError("graph_compute failed")
        H.ggml_backend_event_record(C.addressof(done), backend)
        stream.wait_event(done.torch)
        return self.out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def activations(*shape):  # normed rows with a few channels that stand out, as a model's have
        x = normal(*shape)
        x[..., torch.randint(0, shape[-1], (max(1, shape[-1] // 100),), generator=g, device="cuda")] *= 12.0
        return x

    s, K, kind = {"case": case}, case["width"], case["kind"]
    if kind in ("store", "read"):
        s["table"] = _quantise(normal(case["rows"], K))
        if kind == "store":
            s["x"] = activations(case["taken"], K)
            s["slots"] = torch.randperm(case["rows"], generator=g, device="cuda")[: case["taken"]].contiguous()
            s["order"] = torch.randperm(case["rows"], generator=g, device="cuda").int()
        else:
            s["order"] = torch.randint(0, case["rows"], (case["taken"],), generator=g, device="cuda").int()
    elif kind == "convert":
        s["x"] = normal(case["rows"], K) * (0.02 * torch.exp(0.5 * normal(case["rows"], 1)))
    elif kind == "product":
        s["w"] = _quantise(normal(case["out"], K) / math.sqrt(K))
        s["x"] = activations(case["cols"], K)
    else:
        n, T, U = case["experts"], case["tokens"], case["used"]
        s["w"] = torch.stack([_quantise(normal(case["out"], K) / math.sqrt(K)) for _ in range(n)])
        s["bias"] = 0.1 * normal(n, case["out"])
        s["ids"] = torch.topk(normal(T, n) + 0.7 * normal(n), U, dim=-1)[1].int().contiguous()  # some experts are chosen more often than others
        s["x"] = activations(T, 1 if case["shared"] else U, K)
    if own:
        s["graph"] = _Graph(s)
    return s


def run(s):
    return s["graph"](s) if own else _plain(s)


# ------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    K, kind = case["width"], case["kind"]
    packed = 17 / 32
    if kind == "store":
        return {"bytes": case["taken"] * (K * 4 + 8) + case["rows"] * (K * (packed + 4) + 4), "flops": 0}
    if kind == "convert":
        return {"bytes": case["rows"] * K * 8, "flops": 0}
    if kind == "read":
        return {"bytes": case["taken"] * (K * (packed + 4) + 4), "flops": 0}
    N = case["out"]
    if kind == "product":
        return {"bytes": N * K * packed + case["cols"] * (K + N) * 4, "flops": 2 * N * K * case["cols"]}
    n, T, U = case["experts"], case["tokens"], case["used"]
    met = n * (1 - (1 - U / n) ** T)  # experts that at least one token chooses, on average
    return {"bytes": met * N * (K * packed + 4) + T * ((1 if case["shared"] else U) * K * 4 + U * (N * 4 + 4)), "flops": 2 * N * K * T * U}


# ------------------------------------------------------------------------------------------ the same in 64 bits
def _exact_values(p):
    n = p.shape[-1] // 17
    b = p.reshape(*p.shape[:-1], n, 17)
    e = b[..., 0].double()
    q = b[..., 1:].to(torch.int64)
    c = torch.stack([q % 16, q // 16], -2).reshape(*q.shape[:-1], 32)
    exponent, half = (c % 8) // 2, (c % 2).double()
    mag = torch.where(exponent == 0, 0.5 * half, (1.0 + 0.5 * half) * torch.pow(2.0, (exponent - 1).double()))
    v = torch.where(c >= 8, -mag, mag) * torch.where(e == 255, torch.nan, torch.pow(2.0, e - 127)).unsqueeze(-1)
    return v.reshape(*p.shape[:-1], n * 32)


def _exact_rounded(x):
    """what an MXFP4 row made of x stands for"""
    b = x.double().reshape(*x.shape[:-1], -1, 32)
    top = b.abs().max(-1, keepdim=True)[0]
    unit = torch.pow(2.0, torch.floor(torch.log2(torch.where(top > 0, top, 1.0))).sub(2).clamp(min=-127))
    grid = torch.tensor(VALUES, dtype=torch.float64, device=x.device)
    near = torch.bucketize((b.abs() / unit).contiguous(), (grid[1:] + grid[:-1]) / 2)  # (a tie belongs to the value below)
    return torch.where(torch.isfinite(top), torch.sign(b) * grid[near] * unit, torch.nan).reshape(x.shape)


def _exact_activations(x):
    b = x.double().reshape(*x.shape[:-1], -1, 32)
    top = b.abs().max(-1, keepdim=True)[0]
    s = torch.floor(torch.log2(torch.where(top > 0, top, 2.0**-200))) - 7
    s = torch.where(torch.round(top / torch.pow(2.0, s)) > 255, s + 1, s).clamp(-STEPS, STEPS)
    unit = torch.pow(2.0, s)
    return torch.where(torch.isfinite(top), torch.round(b / unit).clamp(-255, 255) * unit, torch.nan).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "store":
        table = _exact_values(s["table"])
        table[s["slots"]] = _exact_rounded(s["x"])
        return table[s["order"].long()]
    if kind == "convert":
        return _exact_rounded(s["x"])
    if kind == "read":
        return _exact_values(s["table"][s["order"].long()])
    x = _exact_activations(s["x"])
    if kind == "product":
        return x @ _exact_values(s["w"]).T
    x = x.expand(-1, case["used"], -1)
    y = s["bias"].double()[s["ids"].long()]
    for e in range(case["experts"]):
        at = s["ids"] == e
        y[at] += x[at] @ _exact_values(s["w"][e]).T
    return y
