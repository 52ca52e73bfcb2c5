"""The operators over an 8-bit cache in plain torch operations and 64 bits, sequence by sequence, and how far results may be from them."""
import math

import torch

TOP = {0: 127.0, 1: 448.0}   # KV8_INT8, KV8_E4M3
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # half a step of a rounding, relative


class Cache:
    """One layer's cache: arrays on the device and the structure that describes them. Everything behind the tokens that a test puts there is
    garbage: codes of all bit patterns, scales that are NaN, weights and positions of -7."""

    def __init__(self, pkg, batch, kv_heads, head_dim, capacity, block, code, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.pkg, self.code, self.block = pkg, code, block
        shape = (batch, kv_heads, capacity)
        for x in "kv":
            setattr(self, x, torch.randint(0, 256, (*shape, head_dim), generator=g, device="cuda", dtype=torch.uint8))
            setattr(self, x + "_scale", torch.full((batch, kv_heads, capacity // block), math.nan, device="cuda"))
        self.weight = torch.full(shape, -7.0, device="cuda")
        self.slot_pos = torch.full(shape, -7, device="cuda", dtype=torch.int32)

    def arrays(self):
        return [self.k, self.v, self.k_scale, self.v_scale, self.weight, self.slot_pos]

    def clone(self):
        other = object.__new__(Cache)
        other.pkg, other.code, other.block = self.pkg, self.code, self.block
        other.k, other.v, other.k_scale, other.v_scale, other.weight, other.slot_pos = (x.clone() for x in self.arrays())
        return other

    def described(self, **changes):
        b, h, cap, d = self.k.shape
        fields = dict(zip(("k", "v", "k_scale", "v_scale", "weight", "slot_pos"), (x.data_ptr() for x in self.arrays())), batch=b, kv_heads=h, head_dim=d,
                      capacity=cap, block=self.block, code=self.code)
        return self.pkg.Kv8Cache(**{**fields, **changes})

    def fill(self, lengths, seed=1, key=2.0, spread=0.3):
        """Tokens 0..lengths[b]-1 of every sequence: codes of all sizes, block scales that differ; weights from tiny to large, positions in order."""
        g = torch.Generator(device="cuda").manual_seed(seed)
        b, h, cap, d = self.k.shape
        for i, n in enumerate(lengths):
            n = max(n, 0)
            blocks = -(-n // self.block)
            for x, unit in (("k", key), ("v", 1.0)):
                values = torch.randn((h, n, d), generator=g, device="cuda") * (TOP[self.code] / 4)
                getattr(self, x)[i, :, :n] = to_codes(values, self.code)
                getattr(self, x + "_scale")[i, :, :blocks] = unit * 4 / TOP[self.code] * torch.exp(spread * torch.randn((h, blocks), generator=g, device="cuda"))
            self.weight[i, :, :n] = torch.exp(2 * torch.randn((h, n), generator=g, device="cuda"))
            self.slot_pos[i, :, :n] = torch.arange(n, device="cuda", dtype=torch.int32)
        return self

    def values(self, x, b, n):
        """The first n tokens' values [kv_heads, n, head_dim] in 64 bits."""
        each = getattr(self, x + "_scale")[b].double().repeat_interleave(self.block, dim=1)[:, :n, None]
        return numbers(getattr(self, x)[b, :, :n], self.code) * each


def numbers(codes, code):
    return codes.view(torch.int8 if code == 0 else torch.float8_e4m3fn).double()


def to_codes(x, code):
    """The nearest codes of fp32 numbers, as bytes."""
    top = TOP[code]
    return (x.round().clamp(-top, top).to(torch.int8) if code == 0 else x.clamp(-top, top).to(torch.float8_e4m3fn)).view(torch.uint8)


def half_step(y, code):
    """How far the nearest code is from y at most, in units of the scale."""
    return 0.5 if code == 0 else torch.clamp(y.abs() * 2.0 ** -4, min=2.0 ** -10)


def expected_append(cache, x, b, new, length):
    """(codes, scales) of sequence b behind an append of new [tokens, kv_heads, head_dim] at `length`: the formula's IEEE operations in fp32."""
    codes, scales, t = getattr(cache, x)[b].clone(), getattr(cache, x + "_scale")[b].clone(), cache.block
    top = torch.tensor(TOP[cache.code], device="cuda")
    n = new.shape[0]
    for blk in range(length // t, (length + n - 1) // t + 1 if n else 0):
        low, mid, high = blk * t, max(blk * t, length), min(blk * t + t, length + n)
        fresh = new[mid - length:high - length].transpose(0, 1).float()
        s0 = scales[:, blk] if mid > low else torch.zeros_like(scales[:, blk])
        m = fresh.abs().amax(dim=(1, 2))
        s = torch.where(torch.isfinite(m) & ~torch.isnan(s0), torch.maximum(s0, m / top), math.nan)
        s_, s0_ = s[:, None, None], s0[:, None, None]
        old = codes[:, low:mid]
        again = to_codes(numbers(old, cache.code).float() * s0_ / s_, cache.code)
        codes[:, low:mid] = torch.where(s_ > s0_, again, old)
        codes[:, mid:high] = torch.where(s_ > 0, to_codes(fresh / s_, cache.code), 0)
        scales[:, blk] = s
    return codes, scales


def attend(cache, q, b, length, scale, span):
    """Queries q [n, heads, d] of sequence b, of which `length` tokens lie before the first: results, weights [kv_heads, span] that they add, and
    bounds of both: (out, out_tol, weight, weight_tol)."""
    n, heads, d = q.shape
    h = cache.k.shape[1]
    group = heads // h
    total = max(0, min(length + n, span))
    qd = q.double()
    k, v = cache.values("k", b, total), cache.values("v", b, total)
    limit = torch.clamp(length + torch.arange(n, device="cuda") + 1, 0, total)
    hidden = torch.arange(total, device="cuda")[None, :] >= limit[:, None]
    out, tol = torch.zeros_like(qd), torch.zeros_like(qd)
    weight, weight_tol = torch.zeros((h, span), dtype=torch.float64, device="cuda"), torch.zeros((h, span), dtype=torch.float64, device="cuda")
    if total == 0:
        return out, tol, weight, weight_tol
    top = TOP[cache.code]
    for head in range(heads):
        kv = head // group
        s = (qd[:, head] @ k[kv].T * scale).masked_fill(hidden, -math.inf)
        m = s.amax(dim=-1, keepdim=True)
        p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
        p = p / p.sum(dim=-1, keepdim=True).clamp(min=1e-300)
        out[:, head] = p @ v[kv]
        size = p @ v[kv].abs()
        # A score's error: 16 products at a time are added to an fp32 sum (2^-22 of the magnitudes met so far, d / 16 times), then two products with
        # the scale and the factor, the difference from the maximum and the exponential (another four such steps)
        reach = (qd[:, head].abs() @ k[kv].abs().T * scale).masked_fill(hidden, 0.0).amax(dim=-1, keepdim=True)
        score = (d / 16 + 4) * 2.0 ** -22 * (reach + 1)
        # A probability's: its own and its sum's score error, and the order of the sum (64 partial sums at least, 2^-24 for each addition)
        prob = 2 * score + (total / 64 + 32) * 2.0 ** -24
        # The products with the values: probabilities as fp16 (2^-11, and 2^-25 of a unit of the largest value scale / 128), fp32 sums of 16 at a time
        vs = cache.v_scale[b, kv, :-(-total // cache.block)].double().max()
        tol[:, head] = (prob + 2.0 ** -11 + (total / 128 + 32) * 2.0 ** -22) * size + total * 2.0 ** -25 * vs * top / 128
        weight[kv, :total] += p.sum(dim=0)
        weight_tol[kv, :total] += (prob * p).sum(dim=0)
    tol += out.abs() * HALF[q.dtype] + 2.0 ** -25   # (results that are subnormal in fp16)
    weight_tol += (n * group) * 2.0 ** -24 * weight
    return out, tol, weight, weight_tol


def chosen(cache, b, h, length, keep, sink, recent, seen):
    """Where the tokens of slots 0..min(length, keep)-1 come from behind an eviction."""
    n = min(length, keep)
    if length <= keep:
        return list(range(n))
    weight, pos = cache.weight[b, h, :length].tolist(), cache.slot_pos[b, h, :length].tolist()

    def rank(j):
        if pos[j] < sink or pos[j] >= seen - recent:
            return (2, 0.0)
        return (0, 0.0) if math.isnan(weight[j]) else (1, weight[j])

    order = sorted(range(length), key=lambda j: (tuple(-x for x in rank(j)), j))[:keep]
    stays = {j for j in order if j < keep}
    comes = iter(sorted(j for j in order if j >= keep))
    return [j if j in stays else next(comes) for j in range(n)]
