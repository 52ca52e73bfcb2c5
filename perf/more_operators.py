"""Operators over weights held in 8-bit floating point with one scale per block of 128 x 128, and over rows sorted by expert, as cases that
can be timed and compared.

* ``quantize``: rows become e4m3 codes with one scale, a power of two, per row and block of 128 columns (`swlm_op_f8_quantize_dev`).
* ``product``: such rows times a matrix of such weights, or the gated pair of two (`swlm_op_f8_product_dev`).
* ``sort``: (token, choice) pairs sorted by expert (`swlm_op_expert_sort_dev`).
* ``sum``: the experts' rows back at their tokens, weighted and added up (`swlm_op_expert_sum_dev`).
* ``routed``: all of them as a routed feed-forward runs them: sort, gather and quantize, gated product into codes, product, sum.

A held value is code * scale. `run` returns codes as they are held beside the scales; together they are the values. Widths are those of the
framework's own shapes (2048 with 64 experts of 1024, 4096 with 32 experts of 1792, feed-forwards of 8192 and 14336) and generic ones.
"""
import math

import torch

own = False

BLOCK, TOP = 128, 448.0
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ALPHA, LIMIT = 1.702, 7.0   # of the clamped activation


def listed():
    return [
        # the token of one decoding user in front of a product: the smallest call
        {"name": "quantize_1x4096", "kind": "quantize", "rows": 1, "width": 4096, "dtype": "bf16"},
        # a portion of prompts, the residual stream's norm kept in 32 bits
        {"name": "quantize_8192x4096", "kind": "quantize", "rows": 8192, "width": 4096, "dtype": "fp32"},
        # one decoding user, the projection back to the stream: latency and the weights' bytes
        {"name": "product_1x4096x14336", "kind": "product", "rows": 1, "n": 4096, "k": 14336, "dtype": "bf16", "act": "none"},
        # a serving batch of no round size, gate and up of a feed-forward
        {"name": "product_41x8192x2048_gated", "kind": "product", "rows": 41, "n": 8192, "k": 2048, "dtype": "bf16", "act": "silu"},
        # a ragged portion, sizes that no tile divides
        {"name": "product_777x5000x4100", "kind": "product", "rows": 777, "n": 5000, "k": 4100, "dtype": "fp16", "act": "none"},
        # a large batch of prompts through a large matrix
        {"name": "product_8192x4096x14336", "kind": "product", "rows": 8192, "n": 4096, "k": 14336, "dtype": "bf16", "act": "none"},
        # a small serving batch's choices
        {"name": "sort_16x8_of_64", "kind": "sort", "tokens": 16, "top": 8, "experts": 64, "skew": 0.5, "parked": 0.0},
        # a batch of prompts, an eighth of the choices identity experts
        {"name": "sort_16384x8_of_256", "kind": "sort", "tokens": 16384, "top": 8, "experts": 256, "skew": 1.0, "parked": 0.125},
        # a small serving batch
        {"name": "sum_7x8x2048", "kind": "sum", "tokens": 7, "top": 8, "width": 2048, "dtype": "bf16", "add": True},
        # a batch of prompts, added to the residual stream in 32 bits
        {"name": "sum_4096x8x4096", "kind": "sum", "tokens": 4096, "top": 8, "width": 4096, "dtype": "fp32", "add": True},
        # a serving batch's step through a routed feed-forward
        {"name": "routed_32x2048_8_of_64", "kind": "routed", "tokens": 32, "width": 2048, "ff": 1024, "experts": 64, "top": 8, "act": "clamped", "skew": 0.5},
        # a batch of prompts, experts of unequal load
        {"name": "routed_4096x4096_8_of_32", "kind": "routed", "tokens": 4096, "width": 4096, "ff": 1792, "experts": 32, "top": 8, "act": "silu", "skew": 0.5},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["quantize", "product", "product", "product", "sort", "sum", "routed", "routed"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "quantize":
        width = _log(rng, 64, 16384)
        return {"kind": kind, "rows": _log(rng, 1, min(16384, 8192 * 4096 // width)), "width": width, "dtype": dtype}
    if kind == "product":
        act = rng.choice(["none", "none", "silu", "gelu", "clamped"])
        n, k = (_log(rng, 128, 16384) // step * step for step in (rng.choice([1, 8, 128]), rng.choice([1, 16, 128])))
        most = 8192 * 4096 * 14336 // (n * k * (1 if act == "none" else 2))
        return {"kind": kind, "rows": _log(rng, 1, max(1, min(8192, most))), "n": n, "k": k, "dtype": dtype, "act": act}
    if kind == "sort":
        experts = _log(rng, 2, 512)
        return {"kind": kind, "tokens": _log(rng, 1, 16384), "top": rng.randint(1, min(8, experts)), "experts": experts, "skew": rng.choice([0.0, 0.5, 1.0, 2.0]),
                "parked": rng.choice([0.0, 0.0, 0.125, 0.5])}
    if kind == "sum":
        top, width = rng.randint(1, 8), _log(rng, 64, 8192)
        return {"kind": kind, "tokens": _log(rng, 1, 4096 * 8 * 4096 // (top * max(width, 4096))), "top": top, "width": width, "dtype": dtype, "add": rng.random() < 0.5}
    width, ff, experts = _log(rng, 256, 4096), _log(rng, 128, 1792), _log(rng, 2, 64)
    top = rng.randint(1, min(8, experts))
    return {"kind": kind, "tokens": _log(rng, 1, 4096), "width": width, "ff": ff, "experts": experts, "top": top, "act": rng.choice(["silu", "gelu", "clamped"]),
            "skew": rng.choice([0.0, 0.5, 1.0])}


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _generator(seed, salt):
    return torch.Generator(device="cuda").manual_seed((seed * 1000003 + salt) & 0x7FFFFFFF)


def _blocks(width):
    return (width + BLOCK - 1) // BLOCK


def _pitch(width):
    return (width + 15) // 16 * 16


def _codes(generator, *shape):
    """Codes whose spread is a quarter of the range, as in a block whose largest value is four deviations out; rows start at multiples of 16 bytes."""
    out = torch.empty((*shape[:-1], _pitch(shape[-1])), dtype=torch.float8_e4m3fn, device="cuda")
    for part in out if out.ndim == 3 else [out]:
        part.copy_((torch.randn(part.shape, generator=generator, device="cuda") * (TOP / 4)).clamp_(-TOP, TOP))
    return out[..., :shape[-1]]


def _weight(seed, salt, n, k, experts=1):
    """A matrix whose products with values of deviation 1 have deviation 1; its blocks' scales differ by some tenths."""
    g = _generator(seed, salt)
    scale = 4.0 / TOP / math.sqrt(k) * torch.exp(0.3 * torch.randn((experts, _blocks(n), _blocks(k)), generator=g, device="cuda"))
    return _codes(g, experts, n, k), scale


def _rows(seed, salt, rows, width):
    g = _generator(seed, salt)
    scale = 4.0 / TOP * torch.exp(0.3 * torch.randn((_blocks(width), rows), generator=g, device="cuda"))
    return _codes(g, rows, width), scale


def _values(seed, salt, rows, width, dtype):
    """Activations: some columns are several times as large as the others, as in a residual stream's."""
    g = _generator(seed, salt)
    x = torch.randn((rows, (width + 7) // 8 * 8), generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn((x.shape[1],), generator=g, device="cuda"))
    return x.to(DTYPES[dtype])[:, :width]


def _choices(case, seed):
    """Every token's experts, no two alike, some more popular than others; a parked choice is none of them."""
    g = _generator(seed, 5)
    popular = case["skew"] * torch.randn((case["experts"],), generator=g, device="cuda")
    choice = torch.empty((case["tokens"], case["top"]), dtype=torch.int32, device="cuda")
    for part in choice.split(4096):
        part.copy_((torch.randn((part.shape[0], case["experts"]), generator=g, device="cuda") + popular).topk(case["top"], dim=1).indices)
    if case.get("parked"):
        choice[torch.rand(choice.shape, generator=g, device="cuda") < case["parked"]] = -1
    return choice


def _shares(case, seed):
    return torch.softmax(torch.randn((case["tokens"], case["top"]), generator=_generator(seed, 6), device="cuda"), dim=1)


def _inputs(case, seed):
    kind = case["kind"]
    if kind == "quantize":
        return {"x": _values(seed, 1, case["rows"], case["width"], case["dtype"])}
    if kind == "product":
        state = {"x": _rows(seed, 1, case["rows"], case["k"]), "w": _weight(seed, 2, case["n"], case["k"])}
        if case["act"] != "none":
            state["up"] = _weight(seed, 3, case["n"], case["k"])
        return state
    if kind == "sort":
        return {"choice": _choices(case, seed)}
    if kind == "sum":
        entries = case["tokens"] * case["top"]
        g = _generator(seed, 7)
        # rows in the order that a sort leaves them in, one pair in sixteen parked
        place = torch.rand((entries,), generator=g, device="cuda").argsort().int()
        place[torch.rand((entries,), generator=g, device="cuda") < 0.0625] = -1
        state = {"y": _values(seed, 8, entries, case["width"], "bf16"), "place": place.view(case["tokens"], case["top"]), "share": _shares(case, seed)}
        if case["add"]:
            state["add"] = _values(seed, 9, case["tokens"], case["width"], case["dtype"])
        return state
    width, ff, experts = case["width"], case["ff"], case["experts"]
    return {"x": _values(seed, 1, case["tokens"], width, "bf16"), "choice": _choices(case, seed), "share": _shares(case, seed),
            "w": _weight(seed, 2, ff, width, experts), "up": _weight(seed, 3, ff, width, experts), "down": _weight(seed, 4, width, ff, experts)}


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if own:
        _prepare_own(state)
    torch.cuda.synchronize()
    return state


# ---- the framework's calls ----------------------------------------------------------------------------------------------

def _context():
    """The package and the context of the device: a program makes them once."""
    if not hasattr(_context, "made"):
        import __graft_entry__
        pkg = __graft_entry__.load_package()
        _context.made = pkg, pkg.WeightStore(0)
    return _context.made


def _room(rows, width, dtype):
    return torch.zeros((rows, (width + 15) // 16 * 16), device="cuda").to(dtype)[:, :width]


def _code_room(rows, width):
    return _room(rows, width, torch.float8_e4m3fn), torch.zeros((_blocks(width), rows), device="cuda")


def _prepare_own(state):
    """Results and what lies between two calls, as a program keeps them from step to step."""
    _context()
    case, kind = state["case"], state["case"]["kind"]
    if kind == "quantize":
        state["out"] = _code_room(case["rows"], case["width"])
    elif kind == "product":
        state["out"] = _room(case["rows"], case["n"], DTYPES[case["dtype"]])
    elif kind == "sum":
        state["out"] = _room(case["tokens"], case["width"], DTYPES[case["dtype"]])
    if kind in ("sort", "routed"):
        entries = case["tokens"] * case["top"]
        state["offsets"] = torch.zeros((case["experts"] + 1,), dtype=torch.int32, device="cuda")
        state["source"], state["place"] = (torch.zeros((entries,), dtype=torch.int32, device="cuda") for _ in range(2))
    if kind == "routed":
        state["rows"], state["mid"] = _code_room(entries, case["width"]), _code_room(entries, case["ff"])
        state["y"] = _room(entries, case["width"], torch.bfloat16)
        state["out"] = _room(case["tokens"], case["width"], torch.bfloat16)


class _Calls:
    """The library's calls on torch's stream."""

    def __init__(self):
        self.pkg, store = _context()
        # (a null stream stands for the context's own; 1 is CUDA's handle of the default stream that torch works on)
        self.lib, self.handle, self.stream = store.lib, store.handle, torch.cuda.current_stream().cuda_stream or 1
        self.types = {torch.bfloat16: self.pkg.F8_BF16, torch.float16: self.pkg.F8_FP16, torch.float32: self.pkg.F8_FP32, torch.float8_e4m3fn: self.pkg.F8_E4M3}
        self.acts = {"none": 0, "silu": self.pkg.F8_SILU, "gelu": self.pkg.F8_GELU, "clamped": self.pkg.F8_CLAMPED}

    def rows(self, x):
        return self.pkg.F8Rows(codes=x[0].data_ptr(), scale=x[1].data_ptr(), stride=x[0].stride(0), scale_stride=x[1].stride(0))

    def weight(self, w):
        return self.pkg.F8Weight(codes=w[0].data_ptr(), scale=w[1].data_ptr(), stride=w[0].stride(1))

    def quantize(self, x, out, source=None):
        call = self.pkg.F8Quantize(x=x.data_ptr(), x_stride=x.stride(0), source=source.data_ptr() if source is not None else None, out=self.rows(out),
                                   dtype=self.types[x.dtype], rows=out[0].shape[0], width=x.shape[1], x_rows=x.shape[0])
        self.lib.check(self.lib.swlm_op_f8_quantize_dev(self.handle, call, self.stream))

    def product(self, x, w, y, up=None, act="none", offsets=None):
        call = self.pkg.F8Product(x=self.rows(x), w=self.weight(w), offsets=offsets.data_ptr() if offsets is not None else None, rows=x[0].shape[0],
                                  n=w[0].shape[1], k=w[0].shape[2], experts=w[0].shape[0] if offsets is not None else 0, act=self.acts[act], alpha=ALPHA, limit=LIMIT)
        if up is not None:
            call.up = self.weight(up)
        room = y[0] if isinstance(y, tuple) else y
        call.y, call.y_stride, call.dtype = room.data_ptr(), room.stride(0), self.types[room.dtype]
        if isinstance(y, tuple):
            call.y_scale, call.y_scale_stride = y[1].data_ptr(), y[1].stride(0)
        self.lib.check(self.lib.swlm_op_f8_product_dev(self.handle, call, self.stream))

    def sort(self, state):
        case = state["case"]
        call = self.pkg.ExpertSort(choice=state["choice"].data_ptr(), offsets=state["offsets"].data_ptr(), source=state["source"].data_ptr(),
                                   place=state["place"].data_ptr(), tokens=case["tokens"], top=case["top"], experts=case["experts"])
        self.lib.check(self.lib.swlm_op_expert_sort_dev(self.handle, call, self.stream))

    def sum(self, y, place, share, out, add=None):
        call = self.pkg.ExpertSum(y=y.data_ptr(), y_stride=y.stride(0), place=place.data_ptr(), weight=share.data_ptr(), out=out.data_ptr(), out_stride=out.stride(0),
                                  tokens=share.shape[0], top=share.shape[1], width=y.shape[1], y_rows=y.shape[0], y_dtype=self.types[y.dtype], dtype=self.types[out.dtype])
        if add is not None:
            call.add, call.add_stride = add.data_ptr(), add.stride(0)
        self.lib.check(self.lib.swlm_op_expert_sum_dev(self.handle, call, self.stream))


def _run_own(state):
    case, kind, calls = state["case"], state["case"]["kind"], _Calls()
    if kind == "quantize":
        calls.quantize(state["x"], state["out"])
        return {"codes": state["out"][0], "scale": state["out"][1]}
    if kind == "product":
        calls.product(state["x"], state["w"], state["out"], state.get("up"), case["act"])
        return {"out": state["out"]}
    if kind == "sum":
        calls.sum(state["y"], state["place"], state["share"], state["out"], state.get("add"))
        return {"out": state["out"]}
    calls.sort(state)
    if kind == "sort":
        return {"offsets": state["offsets"], "source": state["source"], "place": state["place"]}
    calls.quantize(state["x"], state["rows"], state["source"])
    calls.product(state["rows"], state["w"], state["mid"], state["up"], case["act"], state["offsets"])
    calls.product(state["mid"], state["down"], state["y"], offsets=state["offsets"])
    calls.sum(state["y"], state["place"], state["share"], state["out"])
    return {"out": state["out"]}


def run(state):
    if own:
        return _run_own(state)
    case, kind = state["case"], state["case"]["kind"]
    if kind == "quantize":
        codes, scale = _plain_quantize(state["x"].float())
        return {"codes": codes, "scale": scale}
    if kind == "product":
        return {"out": _plain_product(case["act"], _plain_rows(state["x"]), state["w"], state.get("up")).to(DTYPES[case["dtype"]])}
    if kind == "sort":
        offsets, source, place = _plain_sort(case, state["choice"])
        return {"offsets": offsets.int(), "source": source.int(), "place": place.int()}
    if kind == "sum":
        out = _plain_sum(state["y"], state["place"], state["share"])
        return {"out": (out + state["add"].float() if case["add"] else out).to(DTYPES[case["dtype"]])}
    return {"out": _plain_routed(state)}


# ---- the plain forms ----------------------------------------------------------------------------------------------------

def _plain_quantize(x):
    """The scale of a block is the smallest power of two that is at least its largest |value| / 448, and not below 2^-126."""
    rows, width = x.shape
    wide = torch.nn.functional.pad(x, (0, _blocks(width) * BLOCK - width)).view(rows, -1, BLOCK)
    fraction, exponent = torch.frexp(wide.abs().amax(dim=2))   # 448 = 0.875 * 2^9
    exponent = torch.where(fraction > 0, exponent - torch.where(fraction > 0.875, 8, 9), -126).clamp(min=-126)
    scale = torch.where(fraction.isfinite(), ((exponent + 127) << 23).int().view(torch.float32), math.nan)
    codes = (wide / scale[:, :, None]).clamp(-TOP, TOP).to(torch.float8_e4m3fn)
    return codes.view(rows, -1)[:, :width], scale.t().contiguous()


def _plain_rows(x):
    return x[0].float() * x[1].t().repeat_interleave(BLOCK, dim=1)[:, :x[0].shape[1]]


def _plain_matrix(w, expert=0):
    codes, scale = w[0][expert], w[1][expert]
    return codes.float() * scale.repeat_interleave(BLOCK, dim=0)[:codes.shape[0]].repeat_interleave(BLOCK, dim=1)[:, :codes.shape[1]]


def _plain_product(act, x, w, up=None, expert=0):
    g = x @ _plain_matrix(w, expert).t()
    if act == "none":
        return g
    u = x @ _plain_matrix(up, expert).t()
    if act == "gelu":
        return 0.5 * g * (1.0 + torch.tanh(0.7978845608 * (g + 0.044715 * g * g * g))) * u
    if act == "clamped":
        g, u = g.clamp(max=LIMIT), u.clamp(-LIMIT, LIMIT) + 1.0
    return g / (1.0 + torch.exp(-(ALPHA if act == "clamped" else 1.0) * g)) * u


def _plain_sort(case, choice):
    flat, experts = choice.reshape(-1).long(), case["experts"]
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    order = key.sort(stable=True).indices
    counts = (key[:, None] == torch.arange(experts, device="cuda")).sum(dim=0) if flat.numel() * experts <= 1 << 24 else torch.bincount(key, minlength=experts + 1)[:experts]
    offsets = torch.nn.functional.pad(counts.cumsum(dim=0), (1, 0))
    row = torch.arange(flat.numel(), device="cuda")
    source = torch.where(row < offsets[-1], order // case["top"], -1)
    place = torch.empty_like(order)
    place[order] = torch.where(row < offsets[-1], row, -1)
    return offsets, source, place


def _plain_sum(y, place, share):
    out = torch.zeros((place.shape[0], y.shape[1]), device="cuda")
    for j in range(place.shape[1]):
        at = place[:, j].long()
        out += torch.where(at[:, None] >= 0, y[at.clamp(min=0)].float() * share[:, j, None], 0.0)
    return out


def _plain_routed(state):
    case = state["case"]
    offsets, source, place = _plain_sort(case, state["choice"])
    rows = _plain_rows(_plain_quantize(state["x"][source.clamp(min=0)].float()))
    y = torch.zeros((rows.shape[0], case["width"]), dtype=torch.bfloat16, device="cuda")
    bounds = offsets.tolist()
    for e in range(case["experts"]):
        if bounds[e] < bounds[e + 1]:
            mid = _plain_product(case["act"], rows[bounds[e]:bounds[e + 1]], state["w"], state["up"], e)
            y[bounds[e]:bounds[e + 1]] = _plain_product("none", _plain_rows(_plain_quantize(mid)), state["down"], None, e).bfloat16()
    return _plain_sum(y, place.view(case["tokens"], case["top"]), state["share"]).bfloat16()


# ---- what it takes, and the values in 64 bits ------------------------------------------------------------------------------

def _size(dtype):
    return 4.0 if dtype == "fp32" else 2.0


def _reached(case):
    """Experts that some token is expected to choose."""
    return case["experts"] * (1.0 - (1.0 - case["top"] / case["experts"]) ** case["tokens"])


def _matrix_bytes(n, k):
    return n * k + 4.0 * _blocks(n) * _blocks(k)


def work(case):
    kind = case["kind"]
    if kind == "quantize":
        return {"bytes": case["rows"] * (case["width"] * (_size(case["dtype"]) + 1) + 4.0 * _blocks(case["width"])), "flops": 3.0 * case["rows"] * case["width"]}
    if kind == "product":
        rows, n, k, pair = case["rows"], case["n"], case["k"], 1 if case["act"] == "none" else 2
        return {"bytes": rows * (k + 4.0 * _blocks(k)) + pair * _matrix_bytes(n, k) + rows * n * _size(case["dtype"]), "flops": 2.0 * pair * rows * n * k}
    entries = case["tokens"] * case["top"]
    if kind == "sort":
        return {"bytes": 12.0 * entries + 4.0 * (case["experts"] + 1), "flops": 4.0 * entries}
    width = case["width"]
    if kind == "sum":
        return {"bytes": entries * (2.0 * width + 8.0) + case["tokens"] * width * _size(case["dtype"]) * (2 if case["add"] else 1), "flops": 2.0 * entries * width}
    # the tokens in, the chosen experts' weights, the result out: what lies between could stay on the chip
    return {"bytes": 4.0 * case["tokens"] * width + 8.0 * entries + _reached(case) * 3 * _matrix_bytes(case["ff"], width), "flops": 6.0 * entries * width * case["ff"]}


def _double_quantize(x):
    """Codes and scales of x in 64 bits."""
    codes, scales = torch.empty_like(x), []
    for at in range(0, x.shape[1], BLOCK):
        part = x[:, at:at + BLOCK]
        fraction, exponent = torch.frexp(part.abs().amax(dim=1, keepdim=True) / TOP)
        s = torch.exp2(torch.where(fraction > 0, exponent - (fraction == 0.5).int(), -126).clamp(min=-126).double())
        y = part / s
        step = torch.exp2((torch.frexp(y).exponent - 1).clamp(min=-6).double() - 3)
        codes[:, at:at + BLOCK] = (y / step).round() * step
        scales.append(s[:, 0])
    return codes, torch.stack(scales)


def _double_times(codes, scale, w, expert=0):
    """Rows (codes, scales [blocks][rows]) times an expert's matrix, block by block of 128 columns of the rows."""
    matrix, grid = w[0][expert].double(), w[1][expert].double()
    per_row = grid[torch.arange(matrix.shape[0], device="cuda") // BLOCK]
    column = torch.arange(matrix.shape[1], device="cuda") // BLOCK
    return (codes.double() * scale.double()[column].t()) @ (matrix * per_row[:, column]).t()


def _double_act(act, g, u):
    if act == "silu":
        return g * torch.sigmoid(g) * u
    if act == "gelu":
        return g * torch.sigmoid(2.0 * 0.7978845608 * (g + 0.044715 * g ** 3)) * u   # (1 + tanh z) / 2 = sigmoid(2 z)
    g, u = torch.minimum(g, torch.full_like(g, LIMIT)), u.clamp(-LIMIT, LIMIT)
    return g * torch.sigmoid(ALPHA * g) * (u + 1.0)


def exact(case, seed):
    given, kind = _inputs(case, seed), case["kind"]
    if kind == "quantize":
        codes, scale = _double_quantize(given["x"].double())
        return {"codes": codes, "scale": scale}
    if kind == "product":
        g = _double_times(*given["x"], given["w"])
        return {"out": g if case["act"] == "none" else _double_act(case["act"], g, _double_times(*given["x"], given["up"]))}
    if kind == "sort":
        return None
    if kind == "sum":
        out = given["add"].double() if case["add"] else torch.zeros((case["tokens"], case["width"]), dtype=torch.float64, device="cuda")
        for token in range(0, case["tokens"], 256):
            place, share = given["place"][token:token + 256].long(), given["share"][token:token + 256].double()
            picked = given["y"][place.clamp(min=0).reshape(-1)].double().view(*place.shape, -1)
            out[token:token + 256] += (picked * (share * (place >= 0))[:, :, None]).sum(dim=1)
        return {"out": out}
    out = torch.zeros((case["tokens"], case["width"]), dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        token, j = (given["choice"] == e).nonzero(as_tuple=True)
        if token.numel():
            rows = _double_quantize(given["x"][token].double())
            mid = _double_act(case["act"], _double_times(*rows, given["w"], e), _double_times(*rows, given["up"], e))
            # a row of an expert's result is held in 16 bits
            y = _double_times(*_double_quantize(mid), given["down"], e).bfloat16().double()
            out.index_add_(0, token, y * given["share"][token, j].double()[:, None])
    return {"out": out}
