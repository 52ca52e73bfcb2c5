"""Plain forms in 64 bits of the operators over 8-bit float weights and over rows sorted by expert, and bounds on what fp32 sums may be off."""
import torch

TOP = 448.0
E4M3 = torch.float8_e4m3fn
ACTS = {"plain": 0, "silu": 1, "gelu": 2, "clamped": 3}
ALPHA, LIMIT = 1.702, 7.0


def blocks(width):
    return (width + 127) // 128


def room(rows, width, dtype, fill=None):
    """Rows that start at multiples of 16 bytes, with a gap behind each."""
    size = torch.empty((), dtype=dtype).element_size()
    out = torch.zeros((rows, (width * size + 15) // 16 * 16 // size + 32 // size), device="cuda").to(dtype)
    if fill is not None:
        out.view(torch.uint8).fill_(fill)
    return out[:, :width]


def codes(g, *shape, spread=100.0):
    """Codes in rows of a multiple of 16 bytes and a gap behind them, both of which hold NaN."""
    wide = torch.full((*shape[:-1], (shape[-1] + 15) // 16 * 16 + 16), 0x7F, dtype=torch.uint8, device="cuda")
    wide[..., :shape[-1]] = (torch.randn(shape, generator=g, device="cuda") * spread).clamp(-TOP, TOP).to(E4M3).view(torch.uint8)
    return wide.view(E4M3)[..., :shape[-1]]


def rows_of(g, rows, k):
    wide = torch.full((blocks(k), rows + 3), float("nan"), device="cuda")
    wide[:, :rows] = torch.exp(torch.randn((blocks(k), rows), generator=g, device="cuda")) / 100
    return codes(g, rows, k), wide[:, :rows]


def matrix(g, n, k, experts=1):
    return codes(g, experts, n, k), torch.exp(0.5 * torch.randn((experts, blocks(n), blocks(k)), generator=g, device="cuda")) / 100


def row_values(x):
    return x[0].double() * x[1].double().t().repeat_interleave(128, dim=1)[:, :x[0].shape[1]]


def matrix_values(w, e=0):
    n, k = w[0].shape[1:]
    return w[0][e].double() * w[1][e].double().repeat_interleave(128, dim=0)[:n].repeat_interleave(128, dim=1)[:, :k]


def quantized(x):
    """Codes as numbers, and scales [blocks][rows], of x in 64 bits."""
    out, scales = torch.empty_like(x), []
    for c in range(0, x.shape[1], 128):
        part = x[:, c:c + 128]
        fraction, exponent = torch.frexp(part.abs().amax(dim=1, keepdim=True) / TOP)
        s = torch.ldexp(torch.ones_like(fraction), torch.where(fraction == 0, -126, exponent - (fraction == 0.5).int()).clamp(min=-126))
        y = part / s
        step = torch.ldexp(torch.ones_like(y), (torch.frexp(y).exponent - 1).clamp(min=-6) - 3)
        out[:, c:c + 128] = torch.where(part.isfinite().all(dim=1, keepdim=True), (y / step).round() * step, torch.nan)
        scales.append(torch.where(fraction.isfinite(), s, torch.nan)[:, 0])
    return out, torch.stack(scales)


def product(x, w, e=0):
    """Values, and a bound on what sums in fp32 may be off: a block's products are exact, its sum of 128 of them, the product of two scales, the one with
    it and the sum over blocks each round once per addend, by 2^-24 of what the addends come to at most (2^-23 where an adder truncates)."""
    xv, wv = row_values(x), matrix_values(w, e)
    return xv @ wv.t(), (xv.abs() @ wv.abs().t()) * ((128 + blocks(wv.shape[1]) + 4) * 2.0 ** -23)


def activated(act, g, u, off_g, off_u):
    """The gated result and its bound. The slope of all three activations is at most 1.13; an exponential's argument z is off by some 2^-23 |z|, which
    is off its value by as much, and the other operations are fewer than 16."""
    if act == "silu":
        z = g
    elif act == "gelu":
        z = 2 * 0.7978845608 * (g + 0.044715 * g ** 3)
    else:
        g, u = g.clamp(max=LIMIT), u.clamp(-LIMIT, LIMIT) + 1.0
        z = ALPHA * g
    a = g * torch.sigmoid(z)
    off = 1.13 * off_g * (u.abs() + off_u) + (a.abs() + 1.13 * off_g) * off_u
    return a * u, off + (16 + 4 * z.abs()) * 2.0 ** -24 * (a * u).abs() + 1e-35


def expected(act, x, w, up=None, e=0):
    g, off = product(x, w, e)
    return (g, off) if act == "plain" else activated(act, g, *[product(x, up, e)[i] for i in (0,)], off, product(x, up, e)[1])


def check(got, want, off):
    """A result of 16 or 32 bits: `off`, and half a step of its type."""
    half = torch.finfo(got.dtype).eps / 2
    assert got.isfinite().all()
    assert ((got.double() - want).abs() <= off + half * (want.abs() + off) + torch.finfo(got.dtype).smallest_normal * half).all()


def check_codes(got, scale, want, off):
    """Codes and scales of a result: the scale is that of some largest value within the bound, values are half a step of a code off at most. (The scale grows
    with the largest value, which is off by the bound at most either way: it is a power of two between those of the two ends.)"""
    for b in range(scale.shape[0]):
        part, slack = want[:, 128 * b:128 * b + 128], off[:, 128 * b:128 * b + 128]
        low = quantized((part.abs() - slack).clamp(min=0).amax(dim=1, keepdim=True))[1][0]
        high = quantized((part.abs() + slack).amax(dim=1, keepdim=True))[1][0]
        s = scale[b].double()
        assert ((s >= low) & (s <= high) & (torch.frexp(s).mantissa == 0.5)).all()
        values = got[:, 128 * b:128 * b + 128].double() * s[:, None]
        # e4m3 has 3 bits behind the leading one: half a step is 2^-4 of the number, or 2^-10 of the scale below the normal ones
        assert ((values - part).abs() <= slack + torch.maximum(2.0 ** -4 * (part.abs() + slack), 2.0 ** -10 * s[:, None])).all()


def sort(choice, experts):
    """offsets, source, place of choices [tokens][top] (on the CPU)."""
    flat = choice.reshape(-1).cpu().long()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    order = key.sort(stable=True).indices
    counts = torch.bincount(key, minlength=experts + 1)[:experts]
    total = int(counts.sum())
    source, place = torch.full_like(flat, -1), torch.full_like(flat, -1)
    source[:total] = order[:total] // choice.shape[1]
    place[order[:total]] = torch.arange(total)
    return torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)]).int(), source.int(), place.view(choice.shape).int()


class Calls:
    """The library's calls on torch's current stream, or on another."""

    def __init__(self, pkg, store, stream=None):
        self.pkg, self.lib, self.handle, self.other = pkg, store.lib, store.handle, stream
        self.types = {torch.bfloat16: pkg.F8_BF16, torch.float16: pkg.F8_FP16, torch.float32: pkg.F8_FP32, E4M3: pkg.F8_E4M3}

    @property
    def stream(self):
        return self.other if self.other is not None else torch.cuda.current_stream().cuda_stream or 1

    def rows(self, x):
        return self.pkg.F8Rows(codes=x[0].data_ptr(), scale=x[1].data_ptr(), stride=x[0].stride(0), scale_stride=x[1].stride(0))

    def weight(self, w):
        return self.pkg.F8Weight(codes=w[0].data_ptr(), scale=w[1].data_ptr(), stride=w[0].stride(1))

    def quantize(self, x, out, source=None):
        self.lib.check(self.lib.swlm_op_f8_quantize_dev(self.handle, self.pkg.F8Quantize(
            x=x.data_ptr(), x_stride=x.stride(0), source=source.data_ptr() if source is not None else None, out=self.rows(out), dtype=self.types[x.dtype],
            rows=out[0].shape[0], width=x.shape[1], x_rows=x.shape[0]), self.stream))

    def product_call(self, x, w, y, up=None, act="plain", offsets=None):
        call = self.pkg.F8Product(x=self.rows(x), w=self.weight(w), offsets=offsets.data_ptr() if offsets is not None else None, rows=x[0].shape[0], n=w[0].shape[1],
                                  k=w[0].shape[2], experts=w[0].shape[0] if offsets is not None else 0, act=ACTS[act], alpha=ALPHA, limit=LIMIT)
        if up is not None:
            call.up = self.weight(up)
        held = y[0] if isinstance(y, tuple) else y
        call.y, call.y_stride, call.dtype = held.data_ptr(), held.stride(0), self.types[held.dtype]
        if isinstance(y, tuple):
            call.y_scale, call.y_scale_stride = y[1].data_ptr(), y[1].stride(0)
        return call

    def product(self, *args, **more):
        self.lib.check(self.lib.swlm_op_f8_product_dev(self.handle, self.product_call(*args, **more), self.stream))

    def sort(self, choice, offsets, source, place):
        self.lib.check(self.lib.swlm_op_expert_sort_dev(self.handle, self.pkg.ExpertSort(
            choice=choice.data_ptr(), offsets=offsets.data_ptr(), source=source.data_ptr(), place=place.data_ptr(), tokens=choice.shape[0], top=choice.shape[1],
            experts=offsets.shape[0] - 1), self.stream))

    def sum(self, y, place, weight, out, add=None):
        call = self.pkg.ExpertSum(y=y.data_ptr(), y_stride=y.stride(0), place=place.data_ptr(), weight=weight.data_ptr(), out=out.data_ptr(), out_stride=out.stride(0),
                                  tokens=place.shape[0], top=place.shape[1], width=y.shape[1], y_rows=y.shape[0], y_dtype=self.types[y.dtype], dtype=self.types[out.dtype])
        if add is not None:
            call.add, call.add_stride = add.data_ptr(), add.stride(0)
        self.lib.check(self.lib.swlm_op_expert_sum_dev(self.handle, call, self.stream))
